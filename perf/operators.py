"""The operators that a decode step in 8 and 4 bits is made of, as cases that can be timed and compared.

The cache holds K and V in 8 bits (int8 or e4m3) with a scale for each block and key/value head, the weights hold 4 bits with a
scale (and a zero point) for each group of columns:

  append  rotary positions on Q and K, K and V quantised into the paged cache; blocks that were begun grow their scale
  decode  one query row a sequence over that cache
  prompt  the rows of prompt chunks over that cache, cached tokens in front of them
  w4      products of few rows with 4-bit weights

Head layouts, widths and the block of 64 tokens are those of `llama3-8b` (32 query heads, 8 key/value heads, width 4096, 14336 in
the feed-forward), `llama3-70b` (64, 8, 8192, 28672) and the bench's `1b-shapes` (16, 4, 2048)."""
import math
import random

import torch

own = False

DEV = "cuda"
D = 128
SCALE = 1.0 / math.sqrt(D)
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
HEADS = [(32, 8), (16, 4), (64, 8), (8, 8), (8, 1), (14, 2), (12, 4), (16, 1)]
BLOCKS = [16, 32, 64, 128]
LAYERS = [(4096, 4096), (6144, 4096), (28672, 4096), (4096, 14336), (8192, 8192), (2048, 2048)]  # N, K


# ---------------------------------------------------------------- cases
def _attn(name, kind, codes, heads, batch, ctx, rows=1, block=64):
    return {"name": name, "kind": kind, "codes": codes, "nq": heads[0], "nkv": heads[1], "batch": batch, "ctx": ctx, "rows": rows, "block": block}


def _w4(name, m, n, k, group, zeros):
    return {"name": name, "kind": "w4", "m": m, "n": n, "k": k, "group": group, "zeros": zeros}


def listed():
    return [
        # a decode step of 64 streams writes its tokens; each block was begun by earlier steps
        _attn("append, 64 streams, int8", "append", "int8", (32, 8), 64, 3150),
        # prompt chunks of an engine step of 8192 tokens, some behind cached tokens that end inside a block
        _attn("append, prompt chunks, e4m3", "append", "e4m3", (32, 8), 4, 3000, rows=2000),
        # one chat: what a token waits for
        _attn("decode, one stream, int8", "decode", "int8", (32, 8), 1, 700),
        # a full server at the benchmark's lengths
        _attn("decode, 96 streams, int8", "decode", "int8", (32, 8), 96, 3150),
        # a few long documents, eight query heads a key/value head
        _attn("decode, 3 long, e4m3", "decode", "e4m3", (64, 8), 3, 60001),
        # short chats of a small model in small pages
        _attn("decode, 44 short, int8", "decode", "int8", (16, 4), 44, 76, block=16),
        # drafted tokens checked, or the short end of a prompt, behind a long cached document
        _attn("prompt, 16 rows, int8", "prompt", "int8", (32, 8), 1, 20016, rows=16),
        # new turns of chats behind their cached prefixes
        _attn("prompt, chunks, e4m3", "prompt", "e4m3", (32, 8), 6, 1200, rows=379),
        # whole prompts
        _attn("prompt, 2 of 5000, int8", "prompt", "int8", (32, 8), 2, 5000, rows=5000),
        # one chat's attention output projection
        _w4("w4, 1 row, 4096 x 4096", 1, 4096, 4096, 128, False),
        # one chat's gate and up projection
        _w4("w4, 1 row, 28672 x 4096", 1, 28672, 4096, 64, True),
        # sixteen chats' down projection
        _w4("w4, 16 rows, 4096 x 14336", 16, 4096, 14336, 32, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "prompt", "w4"])
    if kind == "w4":
        m = _log(rng, 1, 64)
        group = rng.choice([32, 64, 128])
        if rng.random() < 0.5:
            n, k = rng.choice(LAYERS)
        else:
            k = group * _log(rng, 1, 16000 // group)
            n = _log(rng, 17, min(16000, 110000000 // k))
        return {"kind": "w4", "m": m, "n": n, "k": k, "group": group, "zeros": rng.random() < 0.5}
    heads = rng.choice(HEADS)
    c = {"kind": kind, "codes": rng.choice(["int8", "e4m3"]), "nq": heads[0], "nkv": heads[1], "block": rng.choice(BLOCKS)}
    if kind == "decode":
        c |= {"ctx": _log(rng, 1, 60001), "rows": 1}
        c["batch"] = _log(rng, 1, max(1, min(128, 2400000 // (c["ctx"] * heads[1]))))
    elif kind == "append":
        c |= {"rows": _log(rng, 1, 4000), "ctx": 0}
        c["batch"] = _log(rng, 1, max(1, min(128, 8000 // c["rows"])))
        c["ctx"] = c["rows"] + rng.randint(0, 4000)
    else:
        c |= {"rows": _log(rng, 1, 5000)}
        c["ctx"] = c["rows"] + (rng.randint(0, 5000) if rng.random() < 0.7 else 0)
        most = max(1, 1300000000 // (heads[0] * c["rows"] * c["ctx"]))
        c["batch"] = _log(rng, 1, min(16, most))
    return c


def _lens(c):
    """New tokens and whole lengths of a case's sequences: ragged, the first as long as the case says; a padded row last where a
    decode step has several."""
    r = random.Random("%(kind)s %(batch)d %(ctx)d %(rows)d" % c)
    new, ctx = [], []
    for i in range(c["batch"]):
        n = c["rows"] if i == 0 or c["rows"] == 1 else max(1, int(c["rows"] * r.uniform(0.6, 1.0)))
        past = c["ctx"] - c["rows"]
        p = past if i == 0 else int(past * r.uniform(0.6, 1.0))
        new.append(n)
        ctx.append(n + p)
    if c["kind"] == "decode" and c["batch"] > 2:
        ctx[-1] = 0
    return new, ctx


def work(case):
    c = case
    if c["kind"] == "w4":
        groups = c["n"] * (c["k"] // c["group"])
        return {"bytes": c["n"] * c["k"] // 2 + groups * (3 if c["zeros"] else 2) + 2 * c["m"] * (c["k"] + c["n"]), "flops": 2 * c["m"] * c["n"] * c["k"]}
    new, ctx = _lens(c)
    rows = sum(new)
    if c["kind"] == "append":
        # Q, K, V rows in, Q out, codes out, and the touched blocks' values as they are handed back
        blocks = sum(-(-x // c["block"]) - (x - n) // c["block"] for n, x in zip(new, ctx))
        held = 2 * blocks * c["block"] * c["nkv"] * D
        return {"bytes": rows * D * (4 * c["nq"] + 6 * c["nkv"]) + rows * (16 + 4 * D) + 3 * held, "flops": 6 * rows * (c["nq"] + c["nkv"]) * D // 2}
    held = 2 * sum(ctx) * c["nkv"] * D
    seen = sum(ctx) if c["kind"] == "decode" else sum(n * (x - n) + n * (n + 1) // 2 for n, x in zip(new, ctx))
    return {"bytes": held + 4 * rows * c["nq"] * D, "flops": 4 * D * c["nq"] * seen}


# ---------------------------------------------------------------- inputs
def _power(amax, most):
    """The smallest power of two whose `most`-fold holds amax (2^-126 at least)."""
    m, e = torch.frexp(amax)
    top = math.frexp(most)
    e = torch.where(amax > 0, e - top[1] + (m > top[0]).int(), -126)
    return torch.ldexp(torch.ones_like(amax), e.clamp(min=-126))


def _bytes(t):
    return t.view(torch.uint8)


def _cache(g, c, blocks):
    """Codes and scales of `blocks` blocks of rows as a model writes them: a few wide channels, blocks of unlike size."""
    dtype, most = CODES[c["codes"]]
    shape = (blocks, c["nkv"], c["block"], D)
    x = torch.randn(shape, generator=g, device=DEV) * torch.exp(0.7 * torch.randn((1, c["nkv"], 1, D), generator=g, device=DEV))
    x *= torch.exp(0.5 * torch.randn((blocks, c["nkv"], 1, 1), generator=g, device=DEV))
    scale = _power(x.abs().amax((2, 3)), most)
    x /= scale[:, :, None, None]
    return (x.round().to(dtype) if dtype == torch.int8 else x.to(dtype)), scale


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "w4":
        n, k, groups = c["n"], c["k"], c["k"] // c["group"]
        s["x"] = torch.randn((c["m"], k), generator=g, device=DEV).to(torch.bfloat16)
        s["codes"] = torch.randint(0, 16, (n, k), generator=g, device=DEV, dtype=torch.uint8)
        s["scales"] = (0.004 * torch.exp(0.3 * torch.randn((n, groups), generator=g, device=DEV))).to(torch.bfloat16)
        s["zeros"] = torch.randint(5, 11, (n, groups), generator=g, device=DEV, dtype=torch.uint8) if c["zeros"] else None
        if own:  # laid out once, as a model is loaded
            from dynamo_exp_amd import ops
            s["weight"] = ops.w4_pack(s["codes"], s["scales"], s["zeros"], c["group"])
        return s
    nq, nkv, bs = c["nq"], c["nkv"], c["block"]
    new, ctx = _lens(c)
    need = [-(-x // bs) for x in ctx]
    blocks = sum(need) + 3
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))
    table = torch.zeros((c["batch"], max(need + [1])), dtype=torch.int64)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    s["table"] = table.to(DEV, torch.int32)
    s["ctx"] = i32(ctx)
    if c["kind"] == "append":
        touched, inside, live, slots, pos = [], [], [], [], []
        for i, (n, x) in enumerate(zip(new, ctx)):
            first = (x - n) // bs
            for b in range(first, need[i]):
                live.append((x - n) % bs if b == first else 0)
                touched.append(int(table[i, b]))
            p = torch.arange(x - n, x)
            inside.append(len(touched) - (need[i] - first) + p // bs - first)
            slots.append(table[i][p // bs] * bs + p % bs)
            pos.append(p)
        pad = 3 if c["rows"] == 1 else 0  # a graph's rows that hold no stream
        s["rows"] = torch.arange(sum(new), device=DEV)  # the rows that have a place
        s["slots"] = torch.cat(slots + [torch.full((pad,), -1)]).to(DEV)
        s["pos"] = torch.cat(pos + [torch.zeros(pad, dtype=torch.int64)]).to(DEV)
        s["inside"] = torch.cat(inside).to(DEV)
        s["touched"] = torch.tensor(touched, device=DEV)
        s["live"] = torch.tensor(live, device=DEV)
        s["read"], s["read_ctx"] = s["touched"].int()[None].contiguous(), i32([len(touched) * bs])
        most = max(ctx) + 1
        inv = 500000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        angle = torch.outer(torch.arange(most, dtype=torch.float64), inv)
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], -1).float().to(DEV)
        row = torch.randn((sum(new) + pad, (nq + 2 * nkv) * D), generator=g, device=DEV)
        row *= torch.exp(0.7 * torch.randn((1, row.shape[1]), generator=g, device=DEV)) * torch.exp(0.3 * torch.randn((row.shape[0], 1), generator=g, device=DEV))
        s["qkv"] = row.to(torch.bfloat16)
        s["q_out"] = torch.empty((row.shape[0], nq * D), dtype=torch.bfloat16, device=DEV)
    else:
        s["q"] = torch.randn((sum(new), nq, D), generator=g, device=DEV).to(torch.bfloat16)
        s["out"] = torch.empty_like(s["q"])
        s["cu"] = i32([sum(new[:i]) for i in range(len(new) + 1)])
        # row by row: its sequence and its place among that sequence's rows
        s["seq"] = torch.cat([torch.full((n,), i) for i, n in enumerate(new)]).to(DEV)
        s["nth"] = torch.cat([torch.arange(n) for n in new]).to(DEV)
        s["most"] = max(new)
        if own and c["kind"] == "prompt":  # planned once for a step's layers
            from dynamo_exp_amd import ops
            s["plan"] = ops.prefill_plan(new, ctx, nq, nkv, DEV)
    s["k"], s["ks"] = _cache(g, c, blocks)
    s["v"], s["vs"] = _cache(g, c, blocks)
    if c["kind"] != "append" and c["codes"] == "e4m3":  # whatever was left behind a sequence's last row
        for i, x in enumerate(ctx):
            if x % bs:
                last = int(table[i, x // bs])
                _bytes(s["k"])[last, :, x % bs:] = 0x7F
                _bytes(s["v"])[last, :, x % bs:] = 0x7F
    return s


# ---------------------------------------------------------------- plain forms
def _rotate(x, cos_sin):
    a, b = x[..., : D // 2], x[..., D // 2:]
    cos, sin = cos_sin[:, None, : D // 2], cos_sin[:, None, D // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _append_plain(codes, scales, x, s, dtype, most):
    """x [tokens, heads, D] into the touched blocks; their values afterwards."""
    n, heads = s["touched"].numel(), x.shape[1]
    at = s["inside"][:, None].expand(-1, heads)
    amax = torch.zeros((n, heads), device=DEV).scatter_reduce(0, at, x.abs().amax(-1), "amax")
    begun = (s["live"] > 0)[:, None]
    old = torch.where(begun, scales[s["touched"]], 0.0)
    scale = torch.maximum(old, _power(amax, most))
    held = _bytes(codes)[s["touched"]].view(dtype).float()
    moved = held * (old / scale)[:, :, None, None]
    moved = moved.round() if dtype == torch.int8 else moved
    held = torch.where((torch.arange(held.shape[2], device=DEV) < s["live"][:, None])[:, None, :, None], moved, held)
    y = (x / scale[s["inside"]][:, :, None])
    y = y.round() if dtype == torch.int8 else y
    held[s["inside"], :, s["slots"][s["rows"]] % held.shape[2]] = y.clamp(-most, most)
    held = held.to(dtype)
    _bytes(codes)[s["touched"]] = _bytes(held)
    scales[s["touched"]] = scale
    return (held.float() * scale[:, :, None, None]).to(torch.bfloat16)


def _values(codes, scales, table, dtype):
    """[sequences, heads, tokens, D] in 32 bits."""
    x = _bytes(codes)[table].view(dtype).float() * scales[table][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _attention_plain(s, causal_rows):
    """q over the cache for rows of [sequences, rows]; `causal_rows`: each row's last key."""
    c = s["case"]
    dtype = CODES[c["codes"]][0]
    table = s["table"].long()
    k, v = _values(s["k"], s["ks"], table, dtype), _values(s["v"], s["vs"], table, dtype)
    j = torch.arange(k.shape[2], device=DEV)
    live = (j < s["ctx"][:, None])[:, None, :, None]
    k, v = torch.where(live, k, 0.0), torch.where(live, v, 0.0)
    group = c["nq"] // c["nkv"]
    q = torch.zeros((c["batch"], s["most"], c["nq"], D), device=DEV)
    q[s["seq"], s["nth"]] = s["q"].float()
    q = q.transpose(1, 2).reshape(c["batch"], c["nkv"], group * s["most"], D)
    t = torch.matmul(q, k.transpose(-1, -2).contiguous()) * SCALE
    t = t.view(c["batch"], c["nkv"], group, s["most"], -1)
    t = t.masked_fill_((j > causal_rows[:, :, None])[:, None, None], float("-inf"))
    top = t.amax(-1, keepdim=True)
    t = t.sub_(torch.where(top.isinf(), 0.0, top)).exp_()
    total = t.sum(-1, keepdim=True)
    o = torch.matmul(t.view(c["batch"], c["nkv"], group * s["most"], -1), v).view(c["batch"], c["nkv"], group, s["most"], D)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(c["batch"], s["most"], c["nq"], D)
    return o[s["seq"], s["nth"]].to(torch.bfloat16)


def run(s):
    c = s["case"]
    if own:
        from dynamo_exp_amd import ops
        if c["kind"] == "w4":
            return ops.w4_linear(s["x"], s["weight"])
        scales = (s["ks"], s["vs"])
        if c["kind"] == "append":
            q = ops.rope_cache(s["qkv"], s["pos"], s["cos_sin"], s["slots"], s["k"], s["v"], c["nq"], c["nkv"], D, c["block"], kv_scales=scales, out=s["q_out"])
            k, v, _ = ops.kv_dequant_scratch(s["k"], s["v"], s["read"], s["read_ctx"], kv_scales=scales)
            return q, k, v
        if c["kind"] == "decode":
            return ops.decode_attention(s["q"], s["k"], s["v"], s["table"], s["ctx"], SCALE, s["out"], None, kv_scales=scales)
        return ops.prefill_attention(s["q"], s["k"], s["v"], s["table"], s["cu"], s["ctx"], SCALE, s["out"], work=s["plan"], kv_scales=scales)
    if c["kind"] == "w4":
        n, k = s["codes"].shape
        w = s["codes"].float().view(n, -1, c["group"])
        w = w - (8.0 if s["zeros"] is None else s["zeros"].float()[..., None])
        w = (w * s["scales"].float()[..., None]).view(n, k)
        return torch.matmul(s["x"].float(), w.t()).to(torch.bfloat16)
    if c["kind"] == "append":
        dtype, most = CODES[c["codes"]]
        x = s["qkv"].float().view(s["qkv"].shape[0], -1, D)
        turned = _rotate(x[:, : c["nq"] + c["nkv"]], s["cos_sin"][s["pos"]])
        q = turned[:, : c["nq"]].to(torch.bfloat16).flatten(1)
        k = _append_plain(s["k"], s["ks"], turned[s["rows"], c["nq"]:], s, dtype, most)
        v = _append_plain(s["v"], s["vs"], x[s["rows"], c["nq"] + c["nkv"]:], s, dtype, most)
        return q, k, v
    if c["kind"] == "decode":
        return _attention_plain(s, s["ctx"][:, None] - 1)
    new = (s["cu"][1:] - s["cu"][:-1])[:, None]
    return _attention_plain(s, s["ctx"][:, None] - new + torch.arange(s["most"], device=DEV))


# ---------------------------------------------------------------- the definitions in 64 bits, sequence by sequence
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "w4":
        out = []
        z = torch.full_like(s["scales"], 8) if s["zeros"] is None else s["zeros"]
        for a in range(0, c["n"], 4096):
            w = s["codes"][a:a + 4096].double()
            w -= z[a:a + 4096].double().repeat_interleave(c["group"], 1)
            w *= s["scales"][a:a + 4096].double().repeat_interleave(c["group"], 1)
            out.append(s["x"].double() @ w.T.contiguous())
        return torch.cat(out, 1)
    bs, nq, nkv = c["block"], c["nq"], c["nkv"]
    new, ctx = _lens(c)
    dtype, most = CODES[c["codes"]]
    if c["kind"] == "append":
        half = D // 2
        x = s["qkv"].double().view(-1, nq + 2 * nkv, D)
        angle = s["cos_sin"].double()[s["pos"]]
        z = torch.complex(x[:, : nq + nkv, :half], x[:, : nq + nkv, half:]) * torch.complex(angle[:, :half], angle[:, half:])[:, None]
        turned = torch.cat([z.real, z.imag], -1)
        inside, slots, live = s["inside"].tolist(), s["slots"].tolist(), s["live"].tolist()
        first = [inside.index(b) for b in range(len(live))]
        first.append(len(inside))
        result = []
        for codes, scales, fresh in ((s["k"], s["ks"], turned[:, nq:]), (s["v"], s["vs"], x[:, nq + nkv:])):
            got = []
            for b, block in enumerate(s["touched"].tolist()):
                rows, off = fresh[first[b]:first[b + 1]], slots[first[b]] % bs
                held = codes[block].double()
                a = rows.abs().amax((0, 2))
                need = torch.exp2(torch.ceil(torch.log2(a / most)).clamp(min=-126))
                was = scales[block].double() if live[b] else torch.zeros_like(need)
                now = torch.maximum(need, was)
                both = torch.cat([held[:, :off] * (was / now)[:, None, None], rows.transpose(0, 1) / now[:, None, None]], 1)
                both = both.round() if c["codes"] == "int8" else both.float().to(dtype).double()
                held[:, : both.shape[1]] = both
                got.append(held * now[:, None, None])
            result.append(torch.stack(got))
        return [turned[:, :nq].flatten(1), *result]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for i, (n, x) in enumerate(zip(new, ctx)):
        if x:
            blocks = s["table"][i, : -(-x // bs)].long()
            k, v = ((_bytes(a)[blocks].view(dtype).double() * b.double()[blocks][:, :, None, None]).transpose(1, 2).flatten(0, 1)[:x]
                    for a, b in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            hidden = torch.arange(x, device=DEV) > torch.arange(x - n, x, device=DEV)[:, None]
            for h in range(nq):
                t = s["q"][at:at + n, h].double() @ k[:, h * nkv // nq].T.contiguous() * SCALE
                p = torch.softmax(t.masked_fill_(hidden, float("-inf")), -1)
                out[at:at + n, h] = p @ v[:, h * nkv // nq]
        at += n
    return out
