"""The 8-bit KV cache with a scale for each block and head (ops/block8.py; csrc/kernels/block_cache.hip, block_decode.hip,
block_prefill.hip): the append against its definition in 64 bits, both attentions against a plain softmax in 64 bits, refusals, and
a run of all of them together as a server makes it."""
from __future__ import annotations

import math

import pytest
import torch

from dynamo_exp_amd import ops
from dynamo_exp_amd.ops import block8
from dynamo_exp_amd.ops import reference as ref

D = 128
SCALE = 1 / math.sqrt(D)
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
both = pytest.mark.parametrize("codes", ["int8", "e4m3"])
NAN, INF = float("nan"), float("inf")


def bits(t):
    return t.view(torch.uint8)


def table_of(need, seed=0, extra=3):
    """Blocks in an order of no order: [sequences, columns] int32 and how many blocks there are."""
    order = torch.randperm(sum(need) + extra, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    t = torch.zeros((len(need), max(need + [1])), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    return t, len(order)


def slots_of(table, spans, bs):
    """The slots of positions lo .. hi - 1 of each sequence, behind one another."""
    out = [table[i].long()[torch.arange(lo, hi) // bs] * bs + torch.arange(lo, hi) % bs for i, (lo, hi) in enumerate(spans)]
    return torch.cat(out)


def random_cache(blocks, nkv, bs, dtype, seed, pow2=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((blocks, nkv, bs, D), generator=g) * torch.exp(torch.randn((blocks, nkv, 1, 1), generator=g))
    s = ref.power_scale(x.abs().amax((2, 3)), dtype) * (1.0 if pow2 else 1.37)
    return ref.to_codes(x / s[..., None, None], dtype), s


def on_gpu(*ts):
    return [t.cuda() for t in ts]


# ---------------------------------------------------------------- the definition, in 64 bits, for one sequence's rows of one head
def check_rows(got, want, scale, dtype):
    """New rows' values against the unrounded ones: half a step of the code.  The values themselves come from products in fp32 (three
    roundings of 2^-24 relative to values of at most `most` steps: under 2^-13 steps)."""
    err = (got - want).abs()
    if dtype == torch.int8:
        tol = scale * (0.5 + 2 ** -13)
    else:  # normal codes 2^-4 of the value, subnormal ones half of 2^-9
        tol = torch.maximum(want.abs() * (2 ** -4 + 2 ** -20), scale * (2 ** -10 + 2 ** -13))
    assert bool((err <= tol).all()), float((err / tol).max())


def rotated(x, pos, cs):
    c, s = cs.double()[pos.long()][:, None, :64], cs.double()[pos.long()][:, None, 64:]
    a, b = x.double()[..., :64], x.double()[..., 64:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def append_case(codes, bs, spans, nq=4, nkv=2, seed=1, pad=0, device="cpu", pos32=False, grow=1.0):
    dtype = CODES[codes]
    table, blocks = table_of([-(-hi // bs) for _, hi in spans], seed)
    k8, ks = random_cache(blocks, nkv, bs, dtype, seed)
    v8, vs = random_cache(blocks, nkv, bs, dtype, seed + 1)
    g = torch.Generator().manual_seed(seed + 2)
    T = sum(hi - lo for lo, hi in spans)
    qkv = (torch.randn((T + pad, (nq + 2 * nkv) * D), generator=g) * grow).bfloat16()
    pos = torch.cat([torch.arange(lo, hi) for lo, hi in spans] + [torch.zeros(pad, dtype=torch.int64)])
    slots = torch.cat([slots_of(table, spans, bs), torch.full((pad,), -1)])
    cs = ref.rope_cos_sin(D, int(pos.max()) + 1, 500000.0)
    before = [t.clone() for t in (k8, v8, ks, vs)]
    args = [t.to(device) for t in (qkv, pos.int() if pos32 else pos, cs, slots, k8, v8)]
    scales = (ks.to(device), vs.to(device))
    q_out = torch.full((T + pad, nq * D), NAN, dtype=torch.bfloat16, device=device)
    r = ops.rope_cache(*args, nq, nkv, D, bs, kv_scales=scales, out=q_out)
    assert r is q_out and torch.equal(args[0].cpu(), qkv)
    return dict(dtype=dtype, table=table, qkv=qkv, pos=pos, cs=cs, slots=slots, before=before, q=q_out.cpu(), k8=args[4].cpu(), v8=args[5].cpu(),
                ks=scales[0].cpu(), vs=scales[1].cpu(), T=T, bs=bs, nq=nq, nkv=nkv, spans=spans)


def check_append(c):
    dtype, bs, nq, nkv, T = c["dtype"], c["bs"], c["nq"], c["nkv"], c["T"]
    x = c["qkv"].view(-1, nq + 2 * nkv, D)
    q64 = rotated(x[:, :nq], c["pos"], c["cs"])
    # one rounding to bf16 and three in fp32
    assert bool(((c["q"].view(-1, nq, D).double() - q64).abs() <= q64.abs() * 2 ** -8 + 2 ** -20).all())
    new = {"k": rotated(x[:T, nq:nq + nkv], c["pos"][:T], c["cs"]), "v": x[:T, nq + nkv:].double()}
    seen = set()
    at = 0
    for i, (lo, hi) in enumerate(c["spans"]):
        for first in range(lo // bs * bs, hi, bs):
            a, b = max(lo, first), min(hi, first + bs)
            if a >= b:
                continue
            block = int(c["table"][i, first // bs])
            seen.add(block)
            for w, n_codes, n_scale, o_codes, o_scale in (("k", c["k8"], c["ks"], c["before"][0], c["before"][2]), ("v", c["v8"], c["vs"], c["before"][1], c["before"][3])):
                rows = new[w][at + a - lo:at + b - lo].transpose(0, 1)
                need = ref.power_scale(rows.abs().amax((1, 2)), dtype)
                off = a - first
                old = o_scale[block] if off else torch.zeros(nkv)
                assert torch.equal(n_scale[block], torch.maximum(old, need))
                s = n_scale[block].double()[:, None, None]
                check_rows(n_codes[block].double()[:, off:off + b - a] * s, rows, s, dtype)
                ratio = (old.double() / n_scale[block].double())[:, None, None]
                moved = ref.to_codes((o_codes[block].double()[:, :off] * ratio).float(), dtype)
                assert torch.equal(bits(n_codes[block][:, :off]), bits(moved))
                assert torch.equal(bits(n_codes[block][:, off + b - a:]), bits(o_codes[block][:, off + b - a:]))  # rows behind
        at += hi - lo
    others = [b for b in range(c["k8"].shape[0]) if b not in seen]
    for n, o in zip((c["k8"], c["v8"], c["ks"], c["vs"]), c["before"]):
        assert torch.equal(n[others].view(torch.uint8), o[others].view(torch.uint8))


SPANS = [
    [(0, 1)],
    [(5, 6), (63, 64), (64, 65), (127, 128), (16, 17)],  # one token each, at blocks' edges
    [(0, 300), (17, 130), (250, 251), (40, 48)],  # ragged chunks, some behind cached tokens
    [(1, 260), (511, 530)],  # more rows than a decode step has
]


@both
@pytest.mark.parametrize("bs", [16, 64, 128])
@pytest.mark.parametrize("spans", SPANS)
def test_append_cpu(codes, bs, spans):
    check_append(append_case(codes, bs, spans, pad=2, seed=len(spans) + bs))


@pytest.mark.gpu
@both
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("spans", SPANS)
def test_append(codes, bs, spans):
    check_append(append_case(codes, bs, spans, pad=2, seed=len(spans) + bs, device="cuda"))


@pytest.mark.gpu
@both
@pytest.mark.parametrize("nq,nkv", [(32, 8), (14, 2), (1, 1), (5, 5)])
@pytest.mark.parametrize("grow", [2.0 ** -40, 9.0])
def test_append_heads_and_growth(codes, nq, nkv, grow):
    """Tokens far smaller than their block's (its scale stays) and larger (its codes move)."""
    check_append(append_case(codes, 32, [(30, 37), (9, 10), (64, 200)], nq, nkv, device="cuda", pos32=True, grow=grow))


@pytest.mark.gpu
@both
def test_append_in_place_and_twice(codes):
    """Without `out` Q is rotated where it lies; the same tokens appended again change nothing."""
    c = append_case(codes, 64, [(70, 90), (3, 4)], device="cuda")
    qkv, k8, v8 = c["qkv"].cuda(), c["k8"].cuda(), c["v8"].cuda()
    scales = (c["ks"].cuda(), c["vs"].cuda())
    ops.rope_cache(qkv, c["pos"].cuda(), c["cs"].cuda(), c["slots"].cuda(), k8, v8, 4, 2, D, 64, kv_scales=scales)
    assert torch.equal(qkv[:, : 4 * D].cpu(), c["q"]) and torch.equal(qkv[:, 4 * D:].cpu(), c["qkv"][:, 4 * D:])
    for a, b in ((k8, c["k8"]), (v8, c["v8"])):
        assert torch.equal(bits(a.cpu()), bits(b))
    assert torch.equal(scales[0].cpu(), c["ks"]) and torch.equal(scales[1].cpu(), c["vs"])


def special_append(codes, device):
    """Infinities, NaN, zeros, the largest and smallest numbers, slots past the cache, a scale that is none: kv_write."""
    dtype, bs = CODES[codes], 16
    k8, v8, scales = block8.alloc(4, 2, bs, dtype, device)
    scales[0].fill_(NAN)
    scales[1].fill_(-1.0)
    k = torch.zeros((7, 2, D), dtype=torch.bfloat16)
    k[0, 0, :4] = torch.tensor([1.0, INF, -INF, NAN])
    k[0, 1, 0] = 3e38
    k[1, 0, 0] = 1e-39
    v = k.flip(1)
    slots = torch.tensor([0, 17, 18, -5, 64, 2 ** 40, 60])  # the second and third begin inside a block whose scale is none
    dev = [t.to(device) for t in (k, v, slots)]
    ops.kv_write(*dev, k8, v8, bs, kv_scales=scales)
    return [t.cpu() for t in (k8, v8, *scales)]


def check_special(got, codes):
    k8, v8, ks, vs = got
    most = MOST[CODES[codes]]
    f = k8[0, 0, 0].float()
    assert f[0] * ks[0, 0] == 1.0 and f[1] == most and f[2] == -most and (f[3] == 0 if codes == "int8" else bool(f[3].isnan()))
    assert 3e38 / most <= float(ks[0, 1]) <= 6.1e38 / most and abs(float(k8[0, 1, 0].float()[0] * ks[0, 1]) / 3e38 - 1) <= (2 ** -7 if codes == "int8" else 2 ** -4)
    tiny = float(torch.tensor(1e-39).bfloat16())
    assert ks[1, 0] == 2.0 ** -126 and bool((k8[1, 0].float()[2:] == 0).all())
    assert abs(float(k8[1, 0].float()[1, 0]) * 2.0 ** -126 - tiny) <= (2.0 ** -127 if codes == "int8" else tiny * 2 ** -4)
    assert ks[3, 0] == 2.0 ** -126 and ks[2].isnan().all() and bool((vs[2] == -1).all())  # a block that no token went into
    assert torch.equal(bits(v8[0, 1, 0]), bits(k8[0, 0, 0])) and vs[0, 1] == ks[0, 0]


@both
def test_append_special_cpu(codes):
    check_special(special_append(codes, "cpu"), codes)


@pytest.mark.gpu
@both
def test_append_special(codes):
    got = special_append(codes, "cuda")
    check_special(got, codes)
    for a, b in zip(got, special_append(codes, "cpu")):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
def test_growth_loses_less_than_a_step():
    """A block filled token by token, each twice the one before: every int8 row ends less than a step from what was written."""
    k8, v8, scales = block8.alloc(1, 1, 64, torch.int8, "cuda")
    g = torch.Generator().manual_seed(3)
    x = (torch.randn((64, 1, D), generator=g) * 2.0 ** (torch.arange(64)[:, None, None] / 6)).bfloat16()
    for t in range(64):
        row = x[t:t + 1].cuda()
        ops.kv_write(row, row, torch.tensor([t], device="cuda"), k8, v8, 64, kv_scales=scales)
    s = float(scales[0][0, 0])
    assert s == float(ref.power_scale(x.float().abs().max()[None], torch.int8)[0])
    assert float((k8[0, 0].cpu().double() * s - x[:, 0].double()).abs().max()) < s


@pytest.mark.gpu
@both
def test_read_back(codes):
    """kv_dequant_scratch: whole blocks as bf16 (a power of two's products are exact), those past a sequence's length left."""
    dtype = CODES[codes]
    k8, ks = random_cache(9, 3, 32, dtype, 4)
    v8, vs = random_cache(9, 3, 32, dtype, 5, pow2=False)
    table = torch.tensor([[4, 2, 8], [0, 7, 1]], dtype=torch.int32)
    ctx = torch.tensor([65, 31], dtype=torch.int32)
    a = on_gpu(k8, v8, table, ctx)
    gk, gv, t = ops.kv_dequant_scratch(*a, kv_scales=tuple(on_gpu(ks, vs)))
    for i, n in ((0, 3), (1, 1)):
        for j in range(n):
            b, to = int(table[i, j]), int(t[i, j])
            assert torch.equal(gk[to].cpu(), ref.block_values(k8[b], ks[b]).bfloat16())
            assert torch.equal(gv[to].cpu(), ref.block_values(v8[b], vs[b]).bfloat16())


# ---------------------------------------------------------------- attention
def attention64(q, k8, v8, ks, vs, table, new, ctx, causal=True):
    """(result, sum p |v|) in 64 bits, rows of all sequences behind one another."""
    bs, nkv = k8.shape[2], k8.shape[1]
    out, size = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    at = 0
    for i, (n, x) in enumerate(zip(new, ctx)):
        if n and x:
            b = table[i, : -(-x // bs)].long()
            k, v = ((c.view(torch.uint8)[b].view(c.dtype).double() * s.double()[b][..., None, None]).transpose(1, 2).reshape(-1, nkv, D)[:x] for c, s in ((k8, ks), (v8, vs)))
            hide = torch.arange(x) > torch.arange(x - n, x)[:, None]
            for h in range(q.shape[1]):
                kv = h * nkv // q.shape[1]
                t = q[at:at + n, h].double() @ k[:, kv].T * SCALE
                p = torch.softmax(t.masked_fill(hide, -INF) if causal else t, -1)
                out[at:at + n, h], size[at:at + n, h] = p @ v[:, kv], p @ v[:, kv].abs()
        at += n
    return out, size


def near(got, want, size, roundings, floor=0.0):
    """Weights rounded to bf16 `roundings` times (in the sum, and where the row sum is of the rounded ones), the result once; scores of
    128 products in fp32, of size 30 at most here: 128 2^-24 30 < 2^-12 of a weight, twice.  Weights under 2^-126 are no normal numbers
    and may be 0: at most 2^14 of them meet values of at most 2^11 here, 2^-101 in all."""
    tol = (roundings * 2 ** -8 + 2 ** -11) * size + 2 ** -8 * want.abs() * 1.01 + 2 ** -101 + floor
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp(min=1e-300)).max())


def cache_of(codes, nkv, bs, ctx, seed, junk=True, pow2=True):
    dtype = CODES[codes]
    table, blocks = table_of([-(-x // bs) for x in ctx], seed)
    k8, ks = random_cache(blocks, nkv, bs, dtype, seed, pow2)
    v8, vs = random_cache(blocks, nkv, bs, dtype, seed + 1, pow2)
    if junk:  # rows behind a sequence, and scales of blocks that are none's
        used = set()
        for i, x in enumerate(ctx):
            used |= set(table[i, : -(-x // bs)].tolist())
            if x % bs:
                b = int(table[i, x // bs])
                bits(k8)[b, :, x % bs:] = 0x7F
                bits(v8)[b, :, x % bs:] = 0x7F
        for b in range(blocks):
            if b not in used:
                ks[b], vs[b] = NAN, INF
                bits(k8)[b] = 0x7F
                bits(v8)[b] = 0x7F
    return table, k8, v8, ks, vs


def run_decode(codes, nq, nkv, bs, ctx, n_parts, seed=0, workspace=None, pow2=True):
    table, k8, v8, ks, vs = cache_of(codes, nkv, bs, ctx, seed, pow2=pow2)
    q = torch.randn((len(ctx), nq, D), generator=torch.Generator().manual_seed(seed + 9)).bfloat16()
    dev = on_gpu(q, k8, v8, table, torch.tensor(ctx, dtype=torch.int32))
    out = torch.full((len(ctx), nq, D), NAN, dtype=torch.bfloat16, device="cuda")
    r = ops.decode_attention(*dev, SCALE, out, n_parts, workspace=workspace, kv_scales=tuple(on_gpu(ks, vs)))
    assert r is out
    want, size = attention64(q, k8, v8, ks, vs, table, [1] * len(ctx), ctx)
    near(out.cpu(), want, size, 1 if pow2 else 2)
    assert all(bool((out[i] == 0).all()) for i, x in enumerate(ctx) if x == 0)
    return dev, (ks, vs), out


@pytest.mark.gpu
@both
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("ctx", [[1], [700], [0, 15, 16, 17, 31, 32, 33, 63, 64, 65], [129, 0, 2100, 511]])
@pytest.mark.parametrize("n_parts", [None, 1, 3])
def test_decode(codes, bs, ctx, n_parts):
    run_decode(codes, 8, 2, bs, ctx, n_parts, seed=bs)


@pytest.mark.gpu
@both
@pytest.mark.parametrize("nq,nkv", [(1, 1), (32, 8), (14, 2), (12, 4), (16, 1), (5, 1), (64, 8), (8, 8), (22, 2)])
def test_decode_heads(codes, nq, nkv):
    run_decode(codes, nq, nkv, 64, [333, 20, 1500], None, seed=nq)


@pytest.mark.gpu
@both
@pytest.mark.parametrize("n_parts", [1, 17, 65])
def test_decode_long(codes, n_parts):
    """More than 64 blocks a part (their numbers are fetched 64 at a time), more parts than a wave has lanes."""
    run_decode(codes, 4, 1, 16, [9001, 5, 4096], n_parts, seed=3)


@pytest.mark.gpu
@both
def test_decode_scales_that_are_no_powers(codes):
    run_decode(codes, 8, 2, 32, [500, 33], None, seed=8, pow2=False)


@pytest.mark.gpu
@both
def test_decode_unlike_scales(codes):
    """Blocks 2^30 apart: a large value under no weight must not cost a small one its digits, nor the other way round."""
    nkv, bs, ctx = 1, 16, [256]
    table, k8, v8, ks, vs = cache_of(codes, nkv, bs, ctx, 5)
    vs *= 2.0 ** torch.randint(-15, 16, vs.shape, generator=torch.Generator().manual_seed(1))
    q = torch.randn((1, 4, D)).bfloat16()
    dev = on_gpu(q, k8, v8, table, torch.tensor(ctx, dtype=torch.int32))
    out = torch.empty_like(dev[0])
    ops.decode_attention(*dev, SCALE, out, None, kv_scales=tuple(on_gpu(ks, vs)))
    near(out.cpu(), *attention64(q, k8, v8, ks, vs, table, [1], ctx), 1)


@pytest.mark.gpu
def test_decode_strides_workspaces_and_pages():
    """Rows of a fused projection, tables with more columns than blocks and rows farther apart, a workspace full of NaN, numbers in the
    table that are no blocks (only rows that use them suffer)."""
    nq, nkv, bs, ctx = 8, 2, 64, [300, 70]
    table, k8, v8, ks, vs = cache_of("int8", nkv, bs, ctx, 2)
    wide = torch.full((2, 40), -7, dtype=torch.int32)
    wide[:, : table.shape[1]] = table
    wide[1, 2:] = 2 ** 30
    row = torch.randn((2, (nq + 2 * nkv) * D)).bfloat16()
    q = row[:, : nq * D].unflatten(1, (nq, D))
    n = 5
    ws = (torch.full((4, nq, n, D), NAN, device="cuda"), torch.full((4, nq, n, 2), NAN, device="cuda"))
    out = torch.full((2, nq, D), NAN, dtype=torch.bfloat16, device="cuda")
    dev = row.cuda()[:, : nq * D].unflatten(1, (nq, D))
    ops.decode_attention(dev, k8.cuda(), v8.cuda(), wide.cuda()[:, :17], torch.tensor(ctx, dtype=torch.int32).cuda(), SCALE, out, n, workspace=ws,
                         kv_scales=tuple(on_gpu(ks, vs)))
    near(out.cpu(), *attention64(q, k8, v8, ks, vs, table, [1, 1], ctx), 1)
    # a length past the table is cut to it
    long = torch.tensor([300, 99999], dtype=torch.int32)
    for parts in (1, 7):
        ops.decode_attention(dev, k8.cuda(), v8.cuda(), table.cuda(), long.cuda(), SCALE, out, parts, kv_scales=tuple(on_gpu(ks, vs)))
        near(out[:1].cpu(), *[t[:1] for t in attention64(q, k8, v8, ks, vs, table, [1, 1], ctx)], 1)


def run_prefill(codes, nq, nkv, bs, new, ctx, seed=0, causal=True, planned=True, pow2=True):
    table, k8, v8, ks, vs = cache_of(codes, nkv, bs, ctx, seed, pow2=pow2)
    T = sum(new)
    q = torch.randn((T, nq, D), generator=torch.Generator().manual_seed(seed + 9)).bfloat16()
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
    plan = ops.prefill_plan(new, ctx, nq, nkv, "cuda", causal) if planned else None
    dev = on_gpu(q, k8, v8, table, cu, torch.tensor(ctx, dtype=torch.int32))
    out = torch.full((T, nq, D), NAN, dtype=torch.bfloat16, device="cuda")
    r = ops.prefill_attention(*dev, SCALE, out, work=plan, kv_scales=tuple(on_gpu(ks, vs)), causal=causal)
    assert r is out
    want, size = attention64(q, k8, v8, ks, vs, table, new, ctx, causal)
    near(out.cpu(), want, size, 2)
    return plan


@pytest.mark.gpu
@both
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("new,ctx", [([1], [1]), ([1, 64, 3], [200, 64, 67]), ([130, 0, 33], [130, 5, 400]), ([16], [4000])])
def test_prefill(codes, bs, new, ctx):
    run_prefill(codes, 8, 2, bs, new, ctx, seed=bs)


@pytest.mark.gpu
@both
@pytest.mark.parametrize("nq,nkv", [(1, 1), (14, 2), (12, 4), (16, 1), (5, 1), (3, 3), (24, 1), (32, 8)])
def test_prefill_heads(codes, nq, nkv):
    run_prefill(codes, nq, nkv, 64, [100, 7], [333, 7], seed=nq)


@pytest.mark.gpu
@both
def test_prefill_tiles_of_eight_waves(codes):
    plan = run_prefill(codes, 32, 8, 64, [1100, 900, 1300, 1000], [1100, 1000, 1300, 1001], seed=4)
    assert plan.tile == 256 and plan.places == 0


@pytest.mark.gpu
@both
def test_prefill_parts(codes):
    """Few rows behind many keys: parts, joined; some see none of a part's keys."""
    plan = run_prefill(codes, 8, 2, 16, [70, 3], [3000, 900], seed=6)
    assert plan.n_joins and plan.places


@pytest.mark.gpu
@both
def test_prefill_bidirectional_and_unplanned(codes):
    run_prefill(codes, 8, 2, 32, [90, 5], [90, 500], seed=7, causal=False)
    run_prefill(codes, 8, 2, 32, [90, 5], [90, 500], seed=7, planned=False)
    run_prefill(codes, 8, 2, 32, [90, 5], [90, 500], seed=7, planned=False, causal=False)


@pytest.mark.gpu
@both
def test_prefill_scales_that_are_no_powers(codes):
    run_prefill(codes, 8, 2, 32, [90, 5], [90, 500], seed=7, pow2=False)


@pytest.mark.gpu
@both
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("new,ctx", [([200, 30], [700, 300]), ([8], [600])])
def test_prefill_unlike_scales(codes, bs, new, ctx):
    """Value scales up to 2^20 apart, from block to block and (small blocks) within a tile of keys; a block of zeros, whose scale is 0."""
    nq, nkv = 8, 2
    table, k8, v8, ks, vs = cache_of(codes, nkv, bs, ctx, 5, junk=False)
    vs *= 2.0 ** torch.randint(-10, 11, vs.shape, generator=torch.Generator().manual_seed(1))
    ks *= 2.0 ** torch.randint(-3, 2, ks.shape, generator=torch.Generator().manual_seed(2))
    zero = int(table[0, 1])
    bits(v8)[zero] = 0
    vs[zero] = 0
    T = sum(new)
    q = torch.randn((T, nq, D), generator=torch.Generator().manual_seed(3)).bfloat16()
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
    out = torch.empty((T, nq, D), dtype=torch.bfloat16, device="cuda")
    dev = on_gpu(q, k8, v8, table, cu, torch.tensor(ctx, dtype=torch.int32))
    ops.prefill_attention(*dev, SCALE, out, work=ops.prefill_plan(new, ctx, nq, nkv), kv_scales=tuple(on_gpu(ks, vs)))
    near(out.cpu(), *attention64(q, k8, v8, ks, vs, table, new, ctx), 2)


@pytest.mark.gpu
def test_long_flat_weights():
    """40000 keys whose weights are alike but for one that is 2^15 times theirs: together the small ones are worth as much."""
    nq, nkv, bs, ctx = 4, 1, 64, [40000]
    table, k8, v8, ks, vs = cache_of("int8", nkv, bs, ctx, 5)
    bits(k8)[:] = 0
    ks[:] = 1.0
    k8[int(table[0, 3]), 0, 5] = 1
    for new in ([1], [12], [30]):
        T = new[0]
        q = torch.full((T, nq, D), 15 * math.log(2) / (D * SCALE), dtype=torch.float32).bfloat16()
        cu = torch.tensor([0, T], dtype=torch.int32)
        out = torch.empty((T, nq, D), dtype=torch.bfloat16, device="cuda")
        dev = on_gpu(q, k8, v8, table, cu, torch.tensor(ctx, dtype=torch.int32))
        scales = tuple(on_gpu(ks, vs))
        ops.prefill_attention(*dev, SCALE, out, work=ops.prefill_plan(new, ctx, nq, nkv), kv_scales=scales)
        near(out.cpu(), *attention64(q, k8, v8, ks, vs, table, new, ctx), 2)
        if T == 1:
            ops.decode_attention(dev[0], dev[1], dev[2], dev[3], dev[5], SCALE, out, None, kv_scales=scales)
            near(out.cpu(), *attention64(q, k8, v8, ks, vs, table, new, ctx), 2)


# ---------------------------------------------------------------- together
def server(device, codes, steps=6):
    """Two prompts in chunks beside a decoding stream: append and attend, step by step; the attention results of all steps."""
    nq, nkv, bs = 8, 2, 16
    k8, v8, scales = block8.alloc(40, nkv, bs, CODES[codes], device)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(5)).to(torch.int32)[:36].view(3, 12)
    cs = ref.rope_cos_sin(D, 200, 500000.0)
    have, got = [0, 0, 0], []
    g = torch.Generator().manual_seed(11)
    for step in range(steps):
        new = [[23, 40], [30, 1], [1, 33], [17, 17], [40, 2], [5, 5]][step] + [1]
        T = sum(new)
        qkv = torch.randn((T, (nq + 2 * nkv) * D), generator=g).bfloat16().to(device)
        spans = [(h, h + n) for h, n in zip(have, new)]
        have = [h + n for h, n in zip(have, new)]
        pos = torch.cat([torch.arange(a, b) for a, b in spans]).to(device)
        slots = slots_of(table, spans, bs).to(device)
        ops.rope_cache(qkv, pos, cs.to(device), slots, k8, v8, nq, nkv, D, bs, kv_scales=scales)
        q = qkv[:, : nq * D].view(T, nq, D)
        out = torch.empty((T, nq, D), dtype=torch.bfloat16, device=device)
        cu = torch.tensor([0, new[0], new[0] + new[1]], dtype=torch.int32, device=device)
        ctx = torch.tensor(have, dtype=torch.int32, device=device)
        bt = table.to(device)
        work = ops.prefill_plan(new[:2], have[:2], nq, nkv, device)
        ops.prefill_attention(q[: T - 1], k8, v8, bt[:2], cu, ctx[:2], SCALE, out[: T - 1], work=work, kv_scales=scales)
        ops.decode_attention(q[T - 1:], k8, v8, bt[2:], ctx[2:], SCALE, out[T - 1:], None, kv_scales=scales)
        got.append(out.float().cpu())
    return got, k8.cpu(), scales[0].cpu()


@both
def test_served_steps_keep_to_the_unquantised_attention(codes):
    """On the CPU: the whole run against attention over the values as written (their codes' roundings alone lie between)."""
    got, k8, ks = server("cpu", codes)
    assert all(bool(x.isfinite().all()) for x in got) and float(ks.max()) <= 2.0 ** -4


@pytest.mark.gpu
@both
def test_served_steps(codes):
    """The same run on the GPU: every step's results within the roundings of the kernels', and codes within one of the CPU's (a value
    next to a code's border may fall on either side; its neighbours' weights move by less than a step's worth)."""
    got, k8, ks = server("cuda", codes)
    want, k8c, ksc = server("cpu", codes)
    assert torch.equal(ks, ksc)
    differ = (k8.float() - k8c.float()).abs() > 0
    assert float(differ.float().mean()) < 1e-4
    for a, b in zip(got, want):
        # 3 roundings to bf16 of weights or results on the GPU, 2 on the CPU, of values below 4.5, halved by the mean over keys; a
        # first token's result is one value
        assert float((a - b).abs().max()) <= 5 * 2 ** -8 * 4.5


@pytest.mark.gpu
def test_captured_step_replays():
    """Append, decode attention and the read-back captured, replayed with other inputs between eager work; a second graph beside it."""
    nq, nkv, bs, B = 8, 2, 16, 3
    graphs = []
    for n in range(2):
        k8, v8, scales = block8.alloc(30, nkv, bs, torch.int8, "cuda")
        table = torch.randperm(30, generator=torch.Generator().manual_seed(n)).to(torch.int32).view(3, 10).cuda()
        cs = ref.rope_cos_sin(D, 200, 500000.0).cuda()
        st = dict(qkv=torch.zeros((B, (nq + 2 * nkv) * D), dtype=torch.bfloat16, device="cuda"), pos=torch.zeros(B, dtype=torch.int64, device="cuda"),
                  slots=torch.full((B,), -1, device="cuda"), ctx=torch.zeros(B, dtype=torch.int32, device="cuda"),
                  out=torch.zeros((B, nq, D), dtype=torch.bfloat16, device="cuda"))

        def step(st=st, k8=k8, v8=v8, scales=scales, table=table, cs=cs):
            ops.rope_cache(st["qkv"], st["pos"], cs, st["slots"], k8, v8, nq, nkv, D, bs, kv_scales=scales)
            ops.decode_attention(st["qkv"][:, : nq * D].view(B, nq, D), k8, v8, table, st["ctx"], SCALE, st["out"], 4, kv_scales=scales)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.inference_mode(), torch.cuda.graph(graph):
            step()
        graphs.append((graph, st, step, table, k8, v8, scales))
    g = torch.Generator().manual_seed(4)
    rows = [torch.randn((B, (nq + 2 * nkv) * D), generator=g).bfloat16() for _ in range(20)]
    eager = block8.alloc(30, nkv, bs, torch.int8, "cuda")
    for t, row in enumerate(rows):
        live = torch.tensor([True, True, t % 3 != 2])  # a padded row now and then: its stream stays away
        for graph, st, step, table, k8, v8, scales in graphs:
            st["qkv"].copy_(row)
            st["pos"].fill_(t)
            st["slots"].copy_(torch.where(live.cuda(), table[:, t // bs].long() * bs + t % bs, -1))
            st["ctx"].copy_(torch.where(live.cuda(), t + 1, 0))
            graph.replay()
        outs = [st["out"].clone() for _, st, *_ in graphs]
        _, st, _, table, *_ = graphs[0]
        q = row.cuda()
        ops.rope_cache(q, st["pos"], cs, st["slots"], eager[0], eager[1], nq, nkv, D, bs, kv_scales=eager[2])
        out = torch.empty_like(st["out"])
        ops.decode_attention(q[:, : nq * D].view(B, nq, D), eager[0], eager[1], table, st["ctx"], SCALE, out, 4, kv_scales=eager[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], out) and torch.equal(outs[1], out)
        assert torch.equal(graphs[0][4], eager[0])


@pytest.mark.gpu
def test_other_stream():
    """The kernels go to the current stream, with their workspace: results on a side stream are those of the default one."""
    dev, (ks, vs), want = run_decode("int8", 8, 2, 64, [2100, 300], 9)
    scales = tuple(on_gpu(ks, vs))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = torch.empty_like(want)
        for _ in range(3):
            ops.decode_attention(*dev, SCALE, out, 9, kv_scales=scales)
    s.synchronize()
    assert torch.equal(out, want)


# ---------------------------------------------------------------- refusals (CPU tensors stand for the GPU's: the checks are the host's)
def test_refusals():
    k8, v8, scales = block8.alloc(4, 2, 16, torch.int8, "cpu")
    chk = block8._check_cache
    chk(k8, v8, scales)
    with pytest.raises(TypeError):
        chk(k8.float(), v8.float(), scales)
    with pytest.raises(TypeError):
        chk(k8, v8.view(torch.uint8), scales)
    with pytest.raises(TypeError):
        chk(k8, v8, (scales[0].half(), scales[1]))
    with pytest.raises(ValueError):
        chk(k8, v8, (scales[0][:3], scales[1]))
    with pytest.raises(ValueError):
        chk(k8, v8, (scales[0].t().contiguous().t(), scales[1]))
    with pytest.raises(ValueError):
        chk(k8[:, :, :, :64].contiguous(), v8[:, :, :, :64].contiguous(), scales)
    with pytest.raises(ValueError):
        chk(k8.view(4, 2, 128, 16)[:, :, :24].contiguous(), v8.view(4, 2, 128, 16)[:, :, :24].contiguous(), scales)
    with pytest.raises(ValueError):
        chk(k8.transpose(0, 1).contiguous().transpose(0, 1), v8, scales)
    with pytest.raises(TypeError):
        block8.alloc(4, 2, 16, torch.bfloat16, "cpu")
    q, out = torch.zeros((3, 8, D), dtype=torch.bfloat16), torch.zeros((3, 8, D), dtype=torch.bfloat16)
    bt, ctx = torch.zeros((3, 2), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    rd = lambda **k: block8._check_reader(**{**dict(q=q, out=out, k_cache=k8, v_cache=v8, kv_scales=scales, block_tables=bt, ctx_lens=ctx, n=3), **k})  # noqa: E731
    rd()
    for bad in (dict(q=q[:, :7]), dict(out=out[:2]), dict(block_tables=bt[:2]), dict(ctx_lens=ctx[:2]), dict(block_tables=bt[:, :0]),
                dict(block_tables=bt.t().contiguous().t()), dict(out=out.transpose(0, 1).contiguous().transpose(0, 1)), dict(ctx_lens=torch.ones(6, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError):
            rd(**bad)
    for bad in (dict(q=q.float()), dict(block_tables=bt.long()), dict(ctx_lens=ctx.long()), dict(out=out.float())):
        with pytest.raises(TypeError):
            rd(**bad)
    with pytest.raises(ValueError):
        ops.prefill_plan([3], [2], 8, 2, "cpu")
    with pytest.raises(ValueError):
        ops.prefill_plan([3], [4, 5], 8, 2, "cpu")
    with pytest.raises(ValueError):
        ops.prefill_plan([3], [4], 8, 3, "cpu")


@pytest.mark.gpu
def test_refusals_gpu():
    k8, v8, scales = block8.alloc(4, 2, 16, torch.int8)
    cs = ref.rope_cos_sin(D, 32, 500000.0).cuda()
    qkv = torch.zeros((3, 8 * D), dtype=torch.bfloat16, device="cuda")
    pos, slots = torch.arange(3, device="cuda"), torch.arange(3, device="cuda")
    call = lambda **k: ops.rope_cache(**{**dict(qkv=qkv, positions=pos, cos_sin=cs, slot_mapping=slots, k_cache=k8, v_cache=v8, n_q=4, n_kv=2, head_dim=D,  # noqa: E731
                                                block_size=16, kv_scales=scales), **k})
    call()
    for bad in (dict(n_q=5), dict(block_size=32), dict(slot_mapping=slots[:2]), dict(positions=pos[:2]), dict(cos_sin=cs[:, :64].contiguous()),
                dict(qkv=torch.zeros((3, 8 * D + 4), dtype=torch.bfloat16, device="cuda")[:, : 8 * D]), dict(slot_mapping=slots.cpu()), dict(row_scale=torch.ones(2, device="cuda")),
                dict(qkv=torch.zeros(3 * 8 * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 8 * D)), dict(slot_mapping=slots.int())):
        with pytest.raises((ValueError, TypeError)):
            call(**bad)
    q, out = qkv[:, : 4 * D].view(3, 4, D), torch.empty((3, 4, D), dtype=torch.bfloat16, device="cuda")
    bt, ctx = torch.zeros((3, 2), dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    for parts, ws in ((0, None), (2, (torch.empty((3, 4, 3, D), device="cuda"), torch.empty((3, 4, 3, 2), device="cuda")))):
        with pytest.raises(ValueError):
            ops.decode_attention(q, k8, v8, bt, ctx, SCALE, out, parts, workspace=ws, kv_scales=scales)
    wide = torch.zeros((1, 34, D), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        ops.decode_attention(wide, k8, v8, bt[:1], ctx[:1], SCALE, torch.empty_like(wide), None, kv_scales=scales)
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    for plan, e in ((ops.prefill_plan([2], [3], 4, 2), ValueError), (ops.prefill_plan([3], [3], 4, 2, causal=False), ValueError), (torch.zeros(2, dtype=torch.int32, device="cuda"), TypeError)):
        with pytest.raises(e):
            ops.prefill_attention(q, k8, v8, bt[:1], cu, ctx[:1], SCALE, out, work=plan, kv_scales=scales)


@pytest.mark.gpu
def test_nothing_to_do():
    k8, v8, scales = block8.alloc(4, 2, 16, torch.int8)
    qkv = torch.zeros((0, 8 * D), dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    ops.rope_cache(qkv, none, ref.rope_cos_sin(D, 32, 500000.0).cuda(), none, k8, v8, 4, 2, D, 16, kv_scales=scales)
    q = torch.zeros((0, 4, D), dtype=torch.bfloat16, device="cuda")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.decode_attention(q, k8, v8, i32(0, 2), i32(0), SCALE, torch.empty_like(q), None, kv_scales=scales)
    ops.prefill_attention(q, k8, v8, i32(1, 2), i32(2), i32(1), SCALE, torch.empty_like(q), work=ops.prefill_plan([0], [0], 4, 2), kv_scales=scales)


@pytest.mark.parametrize("beside", [-1, block8.BESIDE_KEYS])
def test_plan_covers_every_row_and_key(beside, monkeypatch):
    """The plan's items: each row tile's keys once, in whole tiles of 64, parts behind one another in the workspace; sequences of few rows
    as a kind of their own, or with the others where they have few keys."""
    monkeypatch.setattr(block8, "BESIDE_KEYS", beside)
    g = torch.Generator().manual_seed(2)
    for nq, nkv in ((32, 8), (14, 2), (16, 1), (8, 8)):
        for n in range(1, 5):
            new = torch.randint(0, 700, (n,), generator=g).tolist()
            ctx = [a + b for a, b in zip(new, torch.randint(0, 9000, (n,), generator=g).tolist())]
            p = ops.prefill_plan(new, ctx, nq, nkv, "cpu")
            flat, G, tile = p.work.tolist(), nq // nkv, p.tile
            n_items, n_joins = p.n_work + p.n_few, p.n_joins + p.n_few_joins
            items = [flat[6 * i:6 * i + 6] for i in range(n_items)]
            joins = [flat[6 * n_items + 4 * i:][:4] for i in range(n_joins)]
            assert len(flat) == max(1, 6 * n_items + 4 * n_joins)
            for w, j, places in ((items[:p.n_work], joins[:p.n_joins], p.places), (items[p.n_work:], joins[p.n_joins:], p.few_places)):
                assert sorted(x[4] for x in w if x[4] >= 0) == list(range(places)) and sum(x[3] for x in j) == places
            for s, (ql, cl) in enumerate(zip(new, ctx)):
                few = any(x[0] == s for x in items[p.n_work:])
                assert few == (0 < ql * G <= block8.FEW_ROWS) or (beside > 0 and not p.n_few)
                assert not few or ql * G <= 16 * p.few_groups
                w, j, step = (items[p.n_work:], joins[p.n_joins:], block8.FEW_ROWS) if few else (items[:p.n_work], joins[:p.n_joins], tile)
                assert sum(x[0] == s for x in items) == sum(x[0] == s for x in w)
                for r0 in range(0, ql * G, step):
                    mine = sorted(x[2:5] for x in w if x[0] == s and x[1] == r0)
                    assert mine[0][0] == 0 and all(x[1] == y[0] and x[1] % 64 == 0 for x, y in zip(mine, mine[1:]))
                    assert mine[-1][1] > cl - ql + (min(r0 + step, ql * G) - 1) // G
                    if len(mine) > 1:
                        k = [x for x in j if x[:2] == [s, r0]]
                        assert len(k) == 1 and [m[2] for m in mine] == list(range(k[0][2], k[0][2] + k[0][3]))
                    else:
                        assert mine[0][2] == -1


@pytest.mark.gpu
@both
@pytest.mark.parametrize("nq,nkv", [(8, 2), (14, 2), (32, 8), (48, 1), (3, 3)])
@pytest.mark.parametrize("bs", [16, 64])
def test_prefill_few_rows(codes, nq, nkv, bs, monkeypatch):
    """Sequences of 1 to 64 rows a key/value head (few, or a tile of 64), in one part and in many, beside one of many rows."""
    for beside in (-1, block8.BESIDE_KEYS):
        monkeypatch.setattr(block8, "BESIDE_KEYS", beside)
        for new, ctx in (([1, 2, 5], [1, 3, 400]), ([16, 1, 100, 3], [2100, 900, 300, 70]), ([4], [9000])):
            plan = run_prefill(codes, nq, nkv, bs, new, ctx, seed=nq + bs)
            few = [0 < n * nq // nkv <= block8.FEW_ROWS for n in new]
            assert bool(plan.n_few) == any(few) or (beside > 0 and not all(few))
    run_prefill(codes, nq, nkv, bs, [3, 1], [777, 1], seed=2, causal=False)


@pytest.mark.gpu
@both
def test_append_mixed_step(codes):
    """Chunks and decode rows in one call of more than 512 tokens: runs of every length up to nine and whole blocks, at every place of a
    window."""
    spans = [(3, 700)] + [(16 * i + i % 7, 16 * i + i % 7 + 1 + i % 9) for i in range(60)] + [(640 + i, 641 + i) for i in range(9)]
    check_append(append_case(codes, 16, spans, nkv=1, nq=1, seed=3, pad=5, device="cuda"))
    check_append(append_case(codes, 64, spans, nkv=2, nq=2, seed=4, pad=0, device="cuda"))


@pytest.mark.gpu
@both
def test_append_rows_without_a_place_between(codes):
    """Rows that have no place lie between the others': they end runs, and nothing of them is written."""
    dtype, bs, nkv = CODES[codes], 16, 2
    none = [-1, 10 ** 12, 96, -7]  # the cache has 96 slots
    slots = none[:1] + list(range(3, 8)) + none[:2] + list(range(16, 32)) + none[2:3] + [33] + none[3:] + list(range(48, 57)) + none + list(range(71, 79)) + none[1:2] + [80]
    slots = torch.tensor(slots)
    T = len(slots)
    k = torch.randn((T, nkv, D), generator=torch.Generator().manual_seed(1)).bfloat16()
    got = []
    for device in ("cuda", "cpu"):
        k8, v8, scales = block8.alloc(6, nkv, bs, dtype, device)
        ops.kv_write(k.to(device), k.flip(1).contiguous().to(device), slots.to(device), k8, v8, bs, kv_scales=scales)
        got.append([t.cpu() for t in (k8, v8, *scales)])
    for a, b in zip(*got):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 64])
def test_prefill_tiny_scores_beside_a_block_of_zeros(bs):
    """Keys of zeros (scale 2^-126) behind queries of 2^-40: a score's factor is no number that fp32 holds, and masked scores are
    infinities times it."""
    nq, nkv, new, ctx = 8, 2, [90], [200]
    table, k8, v8, ks, vs = cache_of("int8", nkv, bs, ctx, 5)
    for j in range(-(-ctx[0] // bs)):
        if j != 1:
            bits(k8)[int(table[0, j])] = 0
            ks[int(table[0, j])] = 2.0 ** -126
    q = (torch.randn((90, nq, D), generator=torch.Generator().manual_seed(3)) * 2.0 ** -40).bfloat16()
    cu = torch.tensor([0, 90], dtype=torch.int32)
    out = torch.empty((90, nq, D), dtype=torch.bfloat16, device="cuda")
    dev = on_gpu(q, k8, v8, table, cu, torch.tensor(ctx, dtype=torch.int32))
    ops.prefill_attention(*dev, SCALE, out, work=ops.prefill_plan(new, ctx, nq, nkv), kv_scales=tuple(on_gpu(ks, vs)))
    near(out.cpu(), *attention64(q, k8, v8, ks, vs, table, new, ctx), 2)


@pytest.mark.gpu
@both
@pytest.mark.parametrize("T", [3, 600])
def test_positions_past_the_table(codes, T):
    """A position that cos_sin has no row for takes its last (or first) one."""
    cs = ref.rope_cos_sin(D, 50, 500000.0)
    qkv = torch.randn((T, 4 * D), generator=torch.Generator().manual_seed(T)).bfloat16()
    slots = torch.arange(T)
    wild = torch.where(torch.arange(T) % 3 == 0, 2 ** 40, -(2 ** 33))
    got = []
    for pos in (wild, torch.where(torch.arange(T) % 3 == 0, 49, 0), torch.where(torch.arange(T) % 3 == 0, 2 ** 31 - 1, -5).int()):
        k8, v8, scales = block8.alloc(40, 1, 16, CODES[codes])
        row = qkv.cuda()
        ops.rope_cache(row, pos.cuda(), cs.cuda(), slots.cuda(), k8, v8, 2, 1, D, 16, kv_scales=scales)
        got.append([t.cpu().view(torch.uint8) for t in (row, k8, v8, *scales)])
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


@both
def test_read_back_cpu(codes):
    k8, ks = random_cache(9, 3, 32, CODES[codes], 4)
    v8, vs = random_cache(9, 3, 32, CODES[codes], 5, pow2=False)
    table, ctx = torch.tensor([[4, 2, 8], [0, 7, 1]], dtype=torch.int32), torch.tensor([65, 31], dtype=torch.int32)
    packed = torch.tensor([[0, 1, 2], [3, 0, 0]], dtype=torch.int32)
    for scratch in (None, (packed, 4)):
        gk, gv, t = ops.kv_dequant_scratch(k8, v8, table, ctx, kv_scales=(ks, vs), scratch=scratch)
        for i, n in ((0, 3), (1, 1)):
            for j in range(n):
                b, to = int(table[i, j]), int(t[i, j])
                assert torch.equal(gk[to], ref.block_values(k8[b], ks[b]).bfloat16())
                assert torch.equal(gv[to], ref.block_values(v8[b], vs[b]).bfloat16())


@pytest.mark.gpu
def test_captured_read_back_has_its_own_workspace():
    """A graph's copies lie in memory of the graph: eager calls, small and so large that their workspace is made anew, leave them, and
    two graphs leave each other's."""
    k8, ks = random_cache(200, 2, 16, torch.int8, 4)
    v8, vs = random_cache(200, 2, 16, torch.int8, 5)
    dev = on_gpu(k8, v8)
    scales = tuple(on_gpu(ks, vs))
    tables = [torch.arange(n, dtype=torch.int32, device="cuda").view(1, n) + at for at, n in ((3, 5), (20, 7))]
    lens = [torch.tensor([16 * t.shape[1]], dtype=torch.int32, device="cuda") for t in tables]
    call = lambda t, n: ops.kv_dequant_scratch(*dev, t, n, kv_scales=scales)  # noqa: E731
    s = torch.cuda.Stream()
    with torch.inference_mode(), torch.cuda.stream(s):
        call(tables[0], lens[0])
        s.synchronize()
        graphs = []
        for t, n in zip(tables, lens):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                got = call(t, n)
            graphs.append((graph, got))
        for turn in range(3):
            for graph, _ in graphs:
                graph.replay()
            s.synchronize()
            held = [[x.clone() for x in got[:2]] for _, got in graphs]
            wide = torch.arange(70 + 40 * turn, dtype=torch.int32, device="cuda").view(1, -1) + 10
            eager = call(wide, torch.tensor([16 * wide.shape[1]], dtype=torch.int32, device="cuda"))
            s.synchronize()
            assert torch.equal(eager[0][0].cpu(), ref.block_values(k8[10], ks[10]).bfloat16())
            for (_, got), old, t in zip(graphs, held, tables):
                b = t[0].cpu().long()
                for x, o, codes, sc in zip(got, old, (k8, v8), (ks, vs)):
                    assert torch.equal(x[:len(b)], o[:len(b)]) and torch.equal(x[:len(b)].cpu(), ref.block_values(codes[b], sc[b]).bfloat16())


def test_readers_refuse_a_cache_without_blocks():
    k8, v8, scales = block8.alloc(0, 2, 16, torch.int8, "cpu")
    q = torch.zeros((1, 4, D), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no block"):
        block8._check_reader(q, q.clone(), k8, v8, scales, torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32), 1)


def test_prefill_refuses_a_negative_scale():
    k8, v8, scales = block8.alloc(4, 2, 16, torch.int8, "cpu")
    q = torch.zeros((3, 4, D), dtype=torch.bfloat16)
    cu, ctx, bt = torch.tensor([0, 3], dtype=torch.int32), torch.tensor([3], dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32)
    for scale in (-SCALE, NAN):
        with pytest.raises(ValueError, match="not negative"):
            block8.prefill(q, k8, v8, bt, cu, ctx, scale, q.clone(), ops.prefill_plan([3], [3], 4, 2, "cpu"), scales, True)


@pytest.mark.gpu
@both
@pytest.mark.parametrize("bs", [16, 64, 128])
@pytest.mark.parametrize("nq,nkv,new,ctx", [
    (32, 8, [41], [41]), (32, 8, [64], [64]), (32, 8, [65, 64], [65, 129]), (8, 2, [130, 257, 80], [200, 5000, 80]), (16, 2, [90], [6000]),
    (14, 2, [300, 1, 45], [310, 700, 4200]), (3, 3, [700], [900])])
def test_prefill_wide_tiles(codes, bs, nq, nkv, new, ctx, monkeypatch):
    """256 rows a workgroup whatever the sizes: one tile of keys, two, many, parts of them that begin anywhere, more than 64 blocks a
    part, waves without rows, rows that end in a wave."""
    monkeypatch.setattr(block8, "WIDE_TILES", 0)
    monkeypatch.setattr(block8, "WIDE_WASTE", 9)
    plan = run_prefill(codes, nq, nkv, bs, new, ctx, seed=nq + bs)
    assert plan.tile == 256
    monkeypatch.setattr(block8, "PREFILL_KEYS", 10 ** 8)  # (keys in one part)
    run_prefill(codes, nq, nkv, bs, new, ctx, seed=nq)
    run_prefill(codes, nq, nkv, bs, new, ctx, seed=nq, causal=False)


@pytest.mark.gpu
@both
@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("apart", [24, 60])
def test_prefill_scales_that_rise_and_fall(codes, bs, wide, apart, monkeypatch):
    """Value scales 2^apart from one end of 9000 tokens to the other, either way round: the unit that sums are held in rises where the
    64 blocks whose scales are at hand do."""
    monkeypatch.setattr(block8, "PREFILL_KEYS", 10 ** 8)  # (keys in one part)
    if wide:
        monkeypatch.setattr(block8, "WIDE_TILES", 0)
        monkeypatch.setattr(block8, "WIDE_WASTE", 9)
    nq, nkv, new, ctx = 8, 2, [70, 90], [9000, 5000]
    table, k8, v8, ks, vs = cache_of(codes, nkv, bs, ctx, 5, junk=False)
    for s, up in ((0, 1), (1, -1)):
        n = -(-ctx[s] // bs)
        vs[table[s, :n].long()] *= 2.0 ** (up * (torch.arange(n) * apart // n - apart // 2).float())[:, None]
    q = torch.randn((160, nq, D), generator=torch.Generator().manual_seed(3)).bfloat16()
    cu = torch.tensor([0, 70, 160], dtype=torch.int32)
    out = torch.empty((160, nq, D), dtype=torch.bfloat16, device="cuda")
    dev = on_gpu(q, k8, v8, table, cu, torch.tensor(ctx, dtype=torch.int32))
    plan = ops.prefill_plan(new, ctx, nq, nkv)
    assert (plan.tile == 256) == wide
    ops.prefill_attention(*dev, SCALE, out, work=plan, kv_scales=tuple(on_gpu(ks, vs)))
    want, size = attention64(q, k8, v8, ks, vs, table, new, ctx)
    # weights of blocks 2^-apart of the unit: what falls under 2^-126 may be lost, 2^(apart - 126) of a row's largest weight a key
    near(out.cpu(), want, size, 2, 9000 * 2.0 ** (apart - 126) * float((v8.float().abs().amax() * vs).max()))


@pytest.mark.gpu
@both
def test_join_of_few_and_many_parts(codes):
    """Parts up to four are joined eight rows a workgroup, more by a workgroup a row; rows that are not a multiple of eight."""
    plan = run_prefill(codes, 8, 2, 64, [33, 45], [700, 900], seed=6)
    assert plan.n_joins and 1 < plan.parts <= 4
    plan = run_prefill(codes, 8, 2, 64, [21], [700], seed=6)
    assert 1 < plan.parts <= 4 and plan.join_rows == 84
    plan = run_prefill(codes, 4, 1, 64, [33], [6000], seed=6)
    assert plan.parts > 4


@pytest.mark.gpu
@both
def test_prefill_captured_and_on_two_streams(codes, monkeypatch):
    """A step of prompts (tiles, parts and their join, few rows in parts) captured, replayed with other rows and another cache's codes between
    eager calls; and two such calls at once on two streams, each with its workspace."""
    monkeypatch.setattr(block8, "BESIDE_KEYS", -1)
    nq, nkv, bs, new, ctx = 8, 2, 64, [70, 3, 40], [900, 2000, 40]
    table, k8, v8, ks, vs = cache_of(codes, nkv, bs, ctx, 3)
    plan = ops.prefill_plan(new, ctx, nq, nkv)
    assert plan.n_joins and plan.n_few_joins
    cu = torch.tensor([0, 70, 73, 113], dtype=torch.int32)
    q, k, v, t, c, n, s0, s1 = on_gpu(torch.zeros((113, nq, D), dtype=torch.bfloat16), k8, v8, table, cu, torch.tensor(ctx, dtype=torch.int32), ks, vs)
    out = torch.zeros_like(q)
    call = lambda q, out: ops.prefill_attention(q, k, v, t, c, n, SCALE, out, work=plan, kv_scales=(s0, s1))  # noqa: E731
    call(q, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        call(q, out)
    g = torch.Generator().manual_seed(8)
    for turn in range(3):
        rows = torch.randn((113, nq, D), generator=g).bfloat16()
        bits(k).copy_(bits(k8).roll(turn, 0) if turn else bits(k8))
        s0.copy_(ks.roll(turn, 0))
        q.copy_(rows)
        graph.replay()
        got = out.clone()
        eager = torch.empty_like(out)
        call(q, eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), eager.view(torch.int16)) and torch.equal(out.view(torch.int16), eager.view(torch.int16))
        if turn == 0:
            near(got.cpu(), *attention64(rows, k8, v8, ks, vs, table, new, ctx), 2)
    bits(k).copy_(bits(k8))
    s0.copy_(ks)
    qs = [torch.randn((113, nq, D), generator=g).bfloat16() for _ in range(2)]
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    ins = [x.cuda() for x in qs]
    torch.cuda.synchronize()
    for x, s in zip(ins, streams):
        with torch.cuda.stream(s):
            outs.append([torch.empty_like(out) for _ in range(4)])
            for o in outs[-1]:
                call(x, o)
    torch.cuda.synchronize()
    for x, os in zip(qs, outs):
        near(os[0].cpu(), *attention64(x, k8, v8, ks, vs, table, new, ctx), 2)
        assert all(torch.equal(o.view(torch.int16), os[0].view(torch.int16)) for o in os)


@pytest.mark.gpu
@both
def test_blocks_past_32_bits(codes):
    """The last blocks of a cache of 2.7 GB a side: the same results, bit for bit, as at the front of a small one."""
    nq, nkv, bs, blocks = 16, 8, 64, 41000
    small = block8.alloc(24, nkv, bs, CODES[codes])
    big = (*(torch.empty((blocks, nkv, bs, D), dtype=torch.uint8, device="cuda").view(CODES[codes]) for _ in range(2)),
           tuple(torch.zeros((blocks, nkv), device="cuda") for _ in range(2)))
    order = torch.randperm(24, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(2, 12)
    cs = ref.rope_cos_sin(D, 800, 500000.0).cuda()
    g = torch.Generator().manual_seed(2)
    spans = [(0, 700), (0, 333)]
    qkv = torch.randn((1033, (nq + 2 * nkv) * D), generator=g).bfloat16()
    pos = torch.cat([torch.arange(a, b) for a, b in spans]).cuda()
    got = []
    for (k8, v8, scales), first in ((small, 0), (big, blocks - 24)):
        table = order + first
        row = qkv.cuda()
        ops.rope_cache(row, pos, cs, slots_of(table, spans, bs).cuda(), k8, v8, nq, nkv, D, bs, kv_scales=scales)
        q = row[:, : nq * D].unflatten(1, (nq, D))
        ctx, cu, bt = torch.tensor([700, 333], dtype=torch.int32).cuda(), torch.tensor([0, 700, 1033], dtype=torch.int32).cuda(), table.cuda()
        outs = [torch.empty((1033, nq, D), dtype=torch.bfloat16, device="cuda"), torch.empty((2, nq, D), dtype=torch.bfloat16, device="cuda")]
        ops.prefill_attention(q, k8, v8, bt, cu, ctx, SCALE, outs[0], work=ops.prefill_plan([700, 333], [700, 333], nq, nkv), kv_scales=scales)
        ops.decode_attention(q[699:701], k8, v8, bt, ctx, SCALE, outs[1], 3, kv_scales=scales)
        few = torch.empty((3, nq, D), dtype=torch.bfloat16, device="cuda")
        ops.prefill_attention(q[:3], k8, v8, bt[:1], torch.tensor([0, 3], dtype=torch.int32).cuda(), ctx[:1], SCALE, few, work=ops.prefill_plan([3], [700], nq, nkv), kv_scales=scales)
        back = ops.kv_dequant_scratch(k8, v8, bt, ctx, kv_scales=scales)
        got.append([x.clone().cpu() for x in (row, *outs, few, back[0][:10], back[1][:10], scales[0][bt[0, :11].long()], scales[1][bt[0, :11].long()])])
    for a, b in zip(*got):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    near(got[1][1][:700], *attention64(got[1][0][:700, : nq * D].view(700, nq, D), *(x.cpu() for x in (small[0], small[1], *small[2])), order, [700, 0], [700, 333]), 2)


@pytest.mark.gpu
@both
def test_read_backs_are_their_callers(codes):
    """Results of eager calls on one stream, held at once: each is memory of its own, its table too."""
    dtype, bs, nkv = CODES[codes], 16, 2
    caches = [(*random_cache(30, nkv, bs, dtype, seed), *random_cache(30, nkv, bs, dtype, seed + 1)) for seed in (4, 6, 8)]
    tables = [torch.randperm(30, generator=torch.Generator().manual_seed(n)).to(torch.int32)[:n].view(1, n) for n in (9, 5, 9)]
    got = []
    for (k8, ks, v8, vs), t in zip(caches, tables):
        dev = on_gpu(k8, v8, t, torch.tensor([bs * t.shape[1] - 3], dtype=torch.int32))
        got.append(ops.kv_dequant_scratch(*dev, kv_scales=tuple(on_gpu(ks, vs))))
        if len(got) == 1:
            first = got[0][2].cpu()
            got[0][2].fill_(-1)  # (the caller's to change)
    assert len({x.data_ptr() for r in got for x in r}) == 9
    for i, ((k8, ks, v8, vs), t, (gk, gv, to)) in enumerate(zip(caches, tables, got)):
        at = (first if i == 0 else to.cpu())[0].long()
        b = t[0].long()
        assert torch.equal(at, torch.arange(len(b)))
        assert torch.equal(gk.cpu()[at], ref.block_values(k8.view(torch.uint8)[b].view(dtype), ks[b]).bfloat16())
        assert torch.equal(gv.cpu()[at], ref.block_values(v8.view(torch.uint8)[b].view(dtype), vs[b]).bfloat16())


def one_element_run(device, dtype, ks, vs):
    """All ops of a cache with one scale a tensor; what they write and give."""
    bs, nkv, nq, T = 16, 2, 4, 21
    g = torch.Generator().manual_seed(3)
    k, v = (torch.zeros((4, nkv, bs, D), dtype=torch.bfloat16, device=device).to(dtype) for _ in range(2))
    qkv = torch.randn((T, (nq + 2 * nkv) * D), generator=g).bfloat16().to(device)
    slots, pos = torch.arange(16, 16 + T, device=device), torch.arange(T, device=device)
    ops.rope_cache(qkv, pos, ref.rope_cos_sin(D, 64, 500000.0).to(device), slots, k, v, nq, nkv, D, bs, kv_scales=(ks, vs))
    more = torch.randn((2, 5, nkv, D), generator=g).bfloat16().to(device)
    ops.kv_write(more[0], more[1], torch.arange(48, 53, device=device), k, v, bs, kv_scales=(ks, vs))
    bt = torch.tensor([[1, 2], [3, 0]], dtype=torch.int32, device=device)
    ctx, cu = torch.tensor([21, 5], dtype=torch.int32, device=device), torch.tensor([0, 3, 5], dtype=torch.int32, device=device)
    q = torch.randn((5, nq, D), generator=g).bfloat16().to(device)
    outs = [torch.empty_like(q[:2]), torch.empty_like(q)]
    ops.decode_attention(q[:2].contiguous(), k, v, bt, ctx, SCALE, outs[0], 1, kv_scales=(ks, vs))
    ops.prefill_attention(q, k, v, bt, cu, ctx, SCALE, outs[1], kv_scales=(ks, vs))
    if device != "cpu" and dtype != torch.bfloat16:
        outs += [t.clone() for t in ops.kv_dequant_scratch(k, v, bt[:1], ctx[:1] * 0 + 16, kv_scales=(ks, vs))[:2]]
        outs[2], outs[3] = outs[2][:1], outs[3][:1]
    return [t.float().cpu() for t in (qkv, k, v, *outs)]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("shape", [(), (1,), (1, 1)])
def test_scales_of_one_element_are_a_tensors(device, dtype, shape):
    """One scale a tensor, held as checkpoints hold it: the numbers' results, bit for bit."""
    a, b = (0.5, 0.25) if dtype != torch.bfloat16 else (1.0, 1.0)
    want = one_element_run(device, dtype, a, b)
    got = one_element_run(device, dtype, torch.full(shape, a, device=device), torch.full(shape, b, device=device))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_int8_codes_without_block_scales_are_refused():
    """int8 codes beside numbers, or one scale a tensor: no op has such a form (the bf16 kernels would read past them)."""
    k8, v8, scales = block8.alloc(4, 2, 16, torch.int8, "cpu")
    q, rows = torch.zeros((1, 4, D), dtype=torch.bfloat16), torch.zeros((1, 8 * D), dtype=torch.bfloat16)
    bt, ctx, cu = torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    zero = torch.zeros(1, dtype=torch.int64)
    for s in ((1.0, 1.0), (torch.ones(1), torch.ones(1)), (torch.ones(()), torch.ones(()))):
        for call in (lambda: ops.rope_cache(rows, zero, ref.rope_cos_sin(D, 4, 500000.0), zero, k8, v8, 4, 2, D, 16, kv_scales=s),
                     lambda: ops.kv_write(q[:, :2], q[:, :2], zero, k8, v8, 16, kv_scales=s),
                     lambda: ops.decode_attention(q, k8, v8, bt, ctx, SCALE, q.clone(), 1, kv_scales=s),
                     lambda: ops.prefill_attention(q, k8, v8, bt, cu, ctx, SCALE, q.clone(), kv_scales=s),
                     lambda: ops.kv_dequant_scratch(k8, v8, bt, ctx, kv_scales=s)):
            with pytest.raises(TypeError, match="int8"):
                call()
    with pytest.raises(TypeError):
        ops.kv_write(q[:, :2], q[:, :2], zero, k8, v8, 16, kv_scales=(scales[0], 1.0))
    assert not bool(bits(k8).any())


NANS = [  # tiles of 64, 128 and 256 rows, their parts, few rows in one part and in parts
    ([8], [600], {}), ([100, 30], [333, 300], {}), ([300], [700], {"WIDE_TILES": 0, "WIDE_WASTE": 9}), ([16], [4000], {}), ([3, 2], [90, 30], {"BESIDE_KEYS": -1}),
    ([4], [2500], {})]


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["k", "v", "q"])
@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("new,ctx,rules", NANS)
def test_prefill_nan_of_a_live_token(where, bs, new, ctx, rules, monkeypatch):
    """A NaN that the append stored: in a key, every row of its head that sees it is NaN and no other; in a value, its column of those rows
    (and perhaps of its chunk's rows in front of it, whose weights for it are zeros); in a query, its row."""
    for name, x in rules.items():
        monkeypatch.setattr(block8, name, x)
    nq, nkv = 8, 2
    table, k8, v8, ks, vs = cache_of("e4m3", nkv, bs, ctx, 5)
    T, cu = sum(new), [sum(new[:i]) for i in range(len(new) + 1)]
    q = torch.randn((T, nq, D), generator=torch.Generator().manual_seed(3)).bfloat16()
    want, size = attention64(q, k8, v8, ks, vs, table, new, ctx)
    j = ctx[0] - new[0] // 2 - 1  # a token of the first sequence's chunk; its second head's
    sees, head = torch.arange(ctx[0] - new[0], ctx[0]) >= j, slice(nq // 2, nq)
    nan, either = torch.zeros(q.shape, dtype=torch.bool), torch.zeros(q.shape, dtype=torch.bool)
    if where == "q":
        row = new[0] // 2
        q[row, 3, 7] = NAN
        nan[row, 3] = True
    else:
        codes = bits(k8 if where == "k" else v8)
        codes[int(table[0, j // bs]), 1, j % bs, 9] = 0x7F
        if where == "k":
            nan[:new[0], head] = sees[:, None, None]
        else:
            nan[:new[0], head, 9] = sees[:, None]
            either[:new[0], head, 9] = ~sees[:, None]
    out = torch.zeros((T, nq, D), dtype=torch.bfloat16, device="cuda")
    dev = on_gpu(q, k8, v8, table, torch.tensor(cu, dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32))
    ops.prefill_attention(*dev, SCALE, out, work=ops.prefill_plan(new, ctx, nq, nkv), kv_scales=tuple(on_gpu(ks, vs)))
    got = out.cpu()
    assert bool(got[nan].isnan().all())
    left = ~nan & ~(either & got.isnan())
    near(got[left], want[left], size[left], 2)


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["k", "v", "q"])
@pytest.mark.parametrize("n_parts", [1, 5])
def test_decode_nan_of_a_live_token(where, n_parts):
    nq, nkv, bs, ctx = 8, 2, 32, [700, 300]
    table, k8, v8, ks, vs = cache_of("e4m3", nkv, bs, ctx, 5)
    q = torch.randn((2, nq, D), generator=torch.Generator().manual_seed(3)).bfloat16()
    want, size = attention64(q, k8, v8, ks, vs, table, [1, 1], ctx)
    nan = torch.zeros(q.shape, dtype=torch.bool)
    if where == "q":
        q[0, 3, 7] = NAN
        nan[0, 3] = True
    else:
        bits(k8 if where == "k" else v8)[int(table[0, 500 // bs]), 1, 500 % bs, 9] = 0x7F
        nan[(0, slice(nq // 2, nq)) if where == "k" else (0, slice(nq // 2, nq), 9)] = True
    out = torch.zeros((2, nq, D), dtype=torch.bfloat16, device="cuda")
    dev = on_gpu(q, k8, v8, table, torch.tensor(ctx, dtype=torch.int32))
    ops.decode_attention(*dev, SCALE, out, n_parts, kv_scales=tuple(on_gpu(ks, vs)))
    got = out.cpu()
    assert bool(got[nan].isnan().all())
    near(got[~nan], want[~nan], size[~nan], 1)


def planned_run(codes, nq, nkv, bs, planned, new, ctx, seed=0, causal=True, cu=None, behind=0):
    """prefill_attention of rows `new` behind contexts `ctx` by a plan of others; (result, wanted, size, plan)."""
    table, k8, v8, ks, vs = cache_of(codes, nkv, bs, ctx, seed)
    T = sum(new)
    q = torch.randn((T, nq, D), generator=torch.Generator().manual_seed(seed + 9)).bfloat16()
    cu = [sum(new[:i]) for i in range(len(new) + 1)] if cu is None else cu
    plan = ops.prefill_plan(*planned, nq, nkv, "cuda", causal)
    dev = on_gpu(q, k8, v8, table, torch.tensor(cu, dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32))
    out = torch.full((T + behind, nq, D), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.prefill_attention(*dev, SCALE, out[:T], work=plan, kv_scales=tuple(on_gpu(ks, vs)), causal=causal)
    want, size = attention64(q, k8, v8, ks, vs, table, new, ctx, causal)
    return out.cpu(), want, size, plan


@pytest.mark.gpu
@both
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,was,ctx,rules", [
    ([70, 43], [500, 500], [5000, 500], {}), ([70, 43], [3000, 2000], [900, 70], {}), ([16], [4000], [16], {}), ([8], [600], [3000], {}), ([3, 5], [200, 5], [2500, 700], {"BESIDE_KEYS": -1}),
    ([4], [2500], [77], {}), ([4], [2500], [9000], {}), ([300, 200], [300, 200], [1000, 3000], {"WIDE_TILES": 0, "WIDE_WASTE": 9})])
def test_plan_of_other_contexts(codes, causal, new, was, ctx, rules, monkeypatch):
    """A plan serves contexts that have grown, or shrunk, since: it says how the work is cut, not how far a row sees."""
    for name, x in rules.items():
        monkeypatch.setattr(block8, name, x)
    got, want, size, plan = planned_run(codes, 8, 2, 64, (new, was), new, ctx, seed=3, causal=causal)
    near(got, want, size, 2)


@pytest.mark.gpu
@both
@pytest.mark.parametrize("planned,new,past,rules", [
    ([70, 43], [43, 70], [900, 100], {}), ([113, 0, 5], [43, 70, 5], [0, 0, 300], {}), ([3, 30, 9], [30, 3, 9], [2000, 1000, 40], {"BESIDE_KEYS": -1}),
    ([1, 8], [8, 1], [3000, 3000], {"BESIDE_KEYS": -1}), ([300, 10, 20], [20, 290, 20], [50, 60, 70], {"WIDE_TILES": 0, "WIDE_WASTE": 9}), ([33, 100], [100, 33], [4000, 0], {}),
    ([21, 200], [32, 189], [700, 0], {}), ([0, 12], [12, 0], [100, 100], {})])
def test_plan_of_other_rows_gives_nan(codes, planned, new, past, rules, monkeypatch):
    """As many rows in all, but not sequence by sequence: those of the sequences that differ are NaN, not what the memory held."""
    for name, x in rules.items():
        monkeypatch.setattr(block8, name, x)
    ctx = [n + p for n, p in zip(new, past)]
    got, want, size, plan = planned_run(codes, 8, 2, 16, (planned, [max(p + q, c) for p, q, c in zip(planned, past, ctx)]), new, ctx, seed=3, behind=2)
    at = 0
    for a, n in zip(planned, new):
        rows = slice(at, at + n)
        if a == n:
            near(got[rows], want[rows], size[rows], 2)
        else:
            assert bool(got[rows].isnan().all())
        at += n
    assert bool((got[at:] == 7).all())


@pytest.mark.gpu
def test_rows_past_the_queries_are_left():
    """Row numbers past the rows that there are are cut to them: as many as planned then, or NaN; nothing lies behind them."""
    for planned, cu in (([70, 43], [0, 70, 5000]), ([43, 70], [0, 70, 5000]), ([70, 43], [-9, 70, 2 ** 31 - 1])):
        got, want, size, _ = planned_run("int8", 8, 2, 16, (planned, [70, 70]), [70, 43], [70, 43], cu=cu, behind=60)
        near(got[:113], want, size, 2) if planned == [70, 43] else None
        assert bool(got[:113].isnan().all()) == (planned != [70, 43]) and bool((got[113:] == 7).all())
    for planned, cu in (([3, 2], [-7, 3, 60]), ([2, 3], [-7, 3, 60])):
        got, want, size, _ = planned_run("int8", 8, 2, 16, (planned, [3, 3]), [3, 2], [3, 2], cu=cu, behind=60)
        near(got[:5], want, size, 2) if planned == [3, 2] else None
        assert bool(got[:5].isnan().all()) == (planned != [3, 2]) and bool((got[5:] == 7).all())


@pytest.mark.gpu
@both
def test_captured_prompt_whose_contexts_grow(codes):
    """A captured call replayed behind contexts that the plan did not know."""
    nq, nkv, bs, new, most = 8, 2, 64, [40, 5], [3000, 1500]
    table, k8, v8, ks, vs = cache_of(codes, nkv, bs, most, 3)
    plan = ops.prefill_plan(new, [100, 20], nq, nkv)
    q = torch.randn((45, nq, D), generator=torch.Generator().manual_seed(8)).bfloat16()
    dev = on_gpu(q, k8, v8, table, torch.tensor([0, 40, 45], dtype=torch.int32), torch.tensor([100, 20], dtype=torch.int32))
    scales, out = tuple(on_gpu(ks, vs)), torch.zeros((45, nq, D), dtype=torch.bfloat16, device="cuda")
    call = lambda: ops.prefill_attention(*dev, SCALE, out, work=plan, kv_scales=scales)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        call()
    for ctx in ([100, 20], [1700, 64], [41, 700], most):
        dev[5].copy_(torch.tensor(ctx, dtype=torch.int32))
        out.fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        near(out.cpu(), *attention64(q, k8, v8, ks, vs, table, new, ctx), 2)


def test_plan_has_no_ends_and_knows_its_rows():
    """The last part of a tile's keys has no end, every item knows its sequence's rows, and a sequence without rows has one."""
    for new, ctx in (([70, 0, 3, 500], [3000, 9, 4000, 500]), ([3], [9000]), ([0], [0]), ([40, 2], [900, 3])):
        p = ops.prefill_plan(new, ctx, 8, 2, "cpu")
        flat = p.work.tolist()
        items = [flat[6 * i:6 * i + 6] for i in range(p.n_work + p.n_few)]
        assert {x[0] for x in items} == set(range(len(new)))
        assert all(x[5] == 4 * new[x[0]] for x in items)
        for s in [s for s, n in enumerate(new) if n]:
            for r0 in {x[1] for x in items if x[0] == s}:
                ends = sorted(x[3] for x in items if x[:2] == [s, r0])
                assert ends[-1] == 2 ** 31 - 1 and all(e % 64 == 0 for e in ends[:-1])


def test_readers_refuse_no_heads():
    """No query heads: a group of none has no last head for the lanes behind it."""
    k8, v8, scales = block8.alloc(4, 2, 16, torch.int8, "cpu")
    q = torch.zeros((1, 0, D), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        block8._check_reader(q, q.clone(), k8, v8, scales, torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32), 1)
    for heads in ((0, 2), (0, 1), (-2, 2)):
        with pytest.raises(ValueError):
            ops.prefill_plan([3], [4], *heads, "cpu")
    none = block8.alloc(4, 0, 16, torch.int8, "cpu")
    with pytest.raises(ValueError):
        block8._check_reader(q, q.clone(), none[0], none[1], none[2], torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32), 1)


def test_append_refuses_heads_of_other_widths(monkeypatch):
    """K and V of 64 columns a head: the kernel reads 128 of each.  (No GPU here: what the op would start stands still.)"""
    k8, v8, scales = block8.alloc(4, 2, 16, torch.int8, "cpu")
    started = []
    monkeypatch.setattr(block8, "append_rows", lambda *a: started.append(a))
    zero = torch.zeros(3, dtype=torch.int64)

    class Rows(torch.Tensor):  # (CPU memory that says it is the GPU's)
        is_cuda = True

    rows = lambda d: torch.zeros((3, 8, d), dtype=torch.bfloat16).as_subclass(Rows).split((4, 2, 2), 1)  # noqa: E731
    block8.append(*rows(D), None, None, zero, k8, v8, scales)
    assert len(started) == 1
    for d in (64, 32, 256):
        q, k, v = rows(d)
        with pytest.raises(ValueError, match="heads of 128"):
            block8.append(q, k, v, None, None, zero, k8, v8, scales)
        with pytest.raises(ValueError, match="heads of 128"):
            block8.append(None, k, v, None, None, zero, k8, v8, scales)
    assert len(started) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 256])
def test_append_refuses_heads_of_other_widths_gpu(d):
    k8, v8, scales = block8.alloc(4, 2, 16, torch.int8)
    k = torch.zeros((3, 2, d), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="heads of 128"):
        ops.kv_write(k, k, torch.arange(3, device="cuda"), k8, v8, 16, kv_scales=scales)


# ---------------------------------------------------------------- every key in its place
def unit_cache(codes, nkv, bs, ctx, seed):
    """Keys of zeros, so that every key that a row sees has the same weight (1 before the division: exact), and values that say where they
    lie: a token of 16-key unit u has 1 + u // 128 in column u % 128, under scales of 1."""
    table, k8, v8, ks, vs = cache_of(codes, nkv, bs, ctx, seed)
    bits(k8)[:] = 0
    v = torch.zeros(v8.shape)
    for i, x in enumerate(ctx):
        j = torch.arange(x)
        v[table[i].long()[j // bs], :, j % bs, j // 16 % 128] = (1 + j // 16 // 128).float()[:, None]
    used = torch.cat([table[i, : -(-x // bs)] for i, x in enumerate(ctx)]).long()
    ks[used], vs[used] = 0.5, 1.0
    return table, k8, v.to(CODES[codes]), ks, vs


def in_place(got, want):
    """Sums of small whole numbers over their count: fp32 holds the sum, the quotient has 2^-23, the result its rounding to bf16.  (Needles:
    one value, and e^-80 = 2^-115 of values below 2^11.)"""
    return bool(((got.double() - want).abs() <= 2 ** -8 * want.abs() * (1 + 2 ** -10) + 2 ** -100).all())


def needle_cache(codes, nkv, bs, ctx, seed):
    """Keys of +-1: a query of 16 times one of them scores 16 * 128 * SCALE = 181 there and N(0, 16) elsewhere, so that its weight is 1 and
    the others' e^-80 together, and the result that key's value."""
    table, k8, v8, ks, vs = cache_of(codes, nkv, bs, ctx, seed)
    g = torch.Generator().manual_seed(seed + 3)
    signs = (torch.randint(0, 2, k8.shape, generator=g) * 2 - 1).float().to(CODES[codes])
    for i, x in enumerate(ctx):
        j = torch.arange(x)
        b = table[i].long()[j // bs]
        bits(k8)[b, :, j % bs] = bits(signs)[b, :, j % bs]
        ks[b] = 1.0
    return table, k8, v8, ks, vs


def needles(table, k8, v8, vs, i, bs, targets, nq):
    """(queries, wanted) [rows, nq, D] that look for keys targets [rows, nq] of sequence i."""
    nkv = k8.shape[1]
    kv = (torch.arange(nq) * nkv // nq).expand_as(targets)
    b = table[i].long()[targets // bs]
    return (16 * k8.float()[b, kv, targets % bs]).bfloat16(), (v8.float()[b, kv, targets % bs] * vs[b, kv][..., None]).double()


def spread(rows, nq, nkv, seen):
    """Targets [rows, nq]: each key/value head's are spread evenly over the keys that their rows see, the last among them."""
    g = nq // nkv
    n = torch.arange(rows * g).view(rows, g).repeat(1, nkv)
    return (n * (seen[:, None] - 1) // max(rows * g - 1, 1)).long()


@pytest.mark.gpu
@both
@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("B,ctx,n_parts", [(40, 9001, 1), (40, 9001, 17), (40, 9001, 65), (40, 9001, None), (20, 700, 1), (20, 700, 6), (300, 700, 1), (20, 2100, 4), (3, 50, 2)])
def test_decode_every_key_in_its_place(codes, bs, B, ctx, n_parts):
    """Sequences that share a context: eight waves and four, parts, refills of the 64 blocks at hand, the join."""
    nq, nkv = 16, 1
    for kind in ("units", "needles"):
        table, k8, v8, ks, vs = (unit_cache if kind == "units" else needle_cache)(codes, nkv, bs, [ctx], 7)
        if kind == "units":
            q = torch.randn((B, nq, D), generator=torch.Generator().manual_seed(1)).bfloat16()
            want = attention64(q[:1], k8, v8, ks, vs, table, [1], [ctx])[0].expand(B, nq, D)
        else:
            targets = spread(B, nq, nkv, torch.full((B,), ctx))
            assert B < 40 or ctx < 9000 or len(set((targets // 16).flatten().tolist())) == -(-ctx // 16)
            q, want = needles(table, k8, v8, vs, 0, bs, targets, nq)
        dev = on_gpu(q, k8, v8, table.expand(B, -1), torch.full((B,), ctx, dtype=torch.int32))
        out = torch.empty((B, nq, D), dtype=torch.bfloat16, device="cuda")
        ops.decode_attention(*dev, SCALE, out, n_parts, kv_scales=tuple(on_gpu(ks, vs)))
        assert in_place(out.cpu(), want)


@pytest.mark.gpu
@both
@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("new,ctx,nq,nkv,rules", [
    ([70, 40], [9000, 5000], 8, 2, {}), ([16], [4000], 32, 8, {}), ([33], [6000], 4, 1, {}), ([21], [700], 8, 2, {}), ([70, 3], [3000, 900], 8, 2, {}),
    ([8, 5], [9000, 3000], 4, 1, {"BESIDE_KEYS": -1}), ([2], [9000], 8, 2, {"BESIDE_KEYS": -1}), ([4, 1], [200, 300], 4, 1, {"FEW_KEYS": 10 ** 8}),
    ([257, 130], [5000, 200], 8, 2, {"WIDE_TILES": 0, "WIDE_WASTE": 9}), ([300], [9000], 8, 2, {"WIDE_TILES": 0, "WIDE_WASTE": 9, "PREFILL_KEYS": 10 ** 8}),
    ([130], [7000], 8, 2, {"PREFILL_KEYS": 10 ** 8}), ([12], [7000], 4, 1, {"PREFILL_KEYS": 10 ** 8})])
def test_prompt_every_key_in_its_place(codes, bs, new, ctx, nq, nkv, rules, monkeypatch):
    """Tiles of 64, 128 and 256 rows and few rows, whole and in parts, few parts and many to join, refills of the 64 blocks at hand."""
    for name, x in rules.items():
        monkeypatch.setattr(block8, name, x)
    T, cu = sum(new), [sum(new[:i]) for i in range(len(new) + 1)]
    plan = ops.prefill_plan(new, ctx, nq, nkv)
    for kind in ("units", "needles"):
        table, k8, v8, ks, vs = (unit_cache if kind == "units" else needle_cache)(codes, nkv, bs, ctx, 7)
        if kind == "units":
            q = torch.randn((T, nq, D), generator=torch.Generator().manual_seed(1)).bfloat16()
            want = attention64(q, k8, v8, ks, vs, table, new, ctx)[0]
        else:
            both_ = [needles(table, k8, v8, vs, i, bs, spread(n, nq, nkv, torch.arange(x - n, x) + 1), nq) for i, (n, x) in enumerate(zip(new, ctx))]
            q, want = (torch.cat(t) for t in zip(*both_))
        dev = on_gpu(q, k8, v8, table, torch.tensor(cu, dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32))
        out = torch.empty((T, nq, D), dtype=torch.bfloat16, device="cuda")
        ops.prefill_attention(*dev, SCALE, out, work=plan, kv_scales=tuple(on_gpu(ks, vs)))
        assert in_place(out.cpu(), want)


def test_a_lost_or_doubled_chunk_is_seen():
    """The check above against an oracle without, and with twice, each 32 keys of 9001 (planted here, on the CPU)."""
    n = 9001
    u = torch.arange(n) // 16
    v = torch.zeros((n, D), dtype=torch.float64)
    v[torch.arange(n), u % 128] = (1 + u // 128).double()
    want = v.mean(0)
    for at in range(0, n, 32):
        part = v[at:at + 32]
        assert not in_place(((v.sum(0) - part.sum(0)) / (n - len(part))).bfloat16(), want)
        assert not in_place(((v.sum(0) + part.sum(0)) / (n + len(part))).bfloat16(), want)
        assert not in_place(((v.sum(0) - part.sum(0) + v[(at + 64) % 8960:][:len(part)].sum(0)) / n).bfloat16(), want)


def closer(got, q, k8, v8, ks, vs, table, new, ctx, of_rounded):
    """A weight p is off by at most 2^-8 of itself (rounded to bf16), and 2^-11 by its score's products in fp32; taken as independent, their
    sum passes 8 times the root of the sum of the squares once in 10^13 (2 exp(-8^2 / 2)); the prompt kernels' row sum has as many.  The
    result's own rounding, and weights too small to be numbers, as above."""
    bs, nkv, nq = k8.shape[2], k8.shape[1], q.shape[1]
    at = 0
    for i, (n, x) in enumerate(zip(new, ctx)):
        b = table[i, : -(-x // bs)].long()
        k, v = ((c.view(torch.uint8)[b].view(c.dtype).double() * s.double()[b][..., None, None]).transpose(1, 2).reshape(-1, nkv, D)[:x] for c, s in ((k8, ks), (v8, vs)))
        hide = torch.arange(x) > torch.arange(x - n, x)[:, None]
        for h in range(nq):
            kv = h * nkv // nq
            p = torch.softmax((q[at:at + n, h].double() @ k[:, kv].T * SCALE).masked_fill(hide, -INF), -1)
            want = p @ v[:, kv]
            root = ((p * p) @ (v[:, kv] * v[:, kv])).sqrt() + (want.abs() * (p * p).sum(-1, keepdim=True).sqrt() if of_rounded else 0)
            tol = 8 * (2 ** -8 + 2 ** -11) * root + 2 ** -8 * want.abs() * 1.01 + 2 ** -101
            err = (got[at:at + n, h].double() - want).abs()
            assert bool((err <= tol).all()), (i, h, float((err / tol).max()))
        at += n


@pytest.mark.gpu
@both
@pytest.mark.parametrize("ctx,n_parts", [([9001, 5, 4096], 1), ([9001, 5, 4096], 17), ([700, 333], None)])
def test_decode_closer(codes, ctx, n_parts):
    nq, nkv, bs = 4, 1, 16
    table, k8, v8, ks, vs = cache_of(codes, nkv, bs, ctx, 3)
    q = torch.randn((len(ctx), nq, D), generator=torch.Generator().manual_seed(12)).bfloat16()
    out = torch.empty((len(ctx), nq, D), dtype=torch.bfloat16, device="cuda")
    dev = on_gpu(q, k8, v8, table, torch.tensor(ctx, dtype=torch.int32))
    ops.decode_attention(*dev, SCALE, out, n_parts, kv_scales=tuple(on_gpu(ks, vs)))
    closer(out.cpu(), q, k8, v8, ks, vs, table, [1] * len(ctx), ctx, False)


@pytest.mark.gpu
@both
@pytest.mark.parametrize("new,ctx,rules", [([70, 3], [3000, 900], {}), ([16], [4000], {}), ([33], [6000], {}), ([8], [9000], {"BESIDE_KEYS": -1}), ([300, 200], [900, 3000], {"WIDE_TILES": 0, "WIDE_WASTE": 9})])
def test_prompt_closer(codes, new, ctx, rules, monkeypatch):
    for name, x in rules.items():
        monkeypatch.setattr(block8, name, x)
    nq, nkv, bs = 4, 1, 16
    table, k8, v8, ks, vs = cache_of(codes, nkv, bs, ctx, 3)
    T = sum(new)
    q = torch.randn((T, nq, D), generator=torch.Generator().manual_seed(12)).bfloat16()
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
    out = torch.empty((T, nq, D), dtype=torch.bfloat16, device="cuda")
    dev = on_gpu(q, k8, v8, table, cu, torch.tensor(ctx, dtype=torch.int32))
    ops.prefill_attention(*dev, SCALE, out, work=ops.prefill_plan(new, ctx, nq, nkv), kv_scales=tuple(on_gpu(ks, vs)))
    closer(out.cpu(), q, k8, v8, ks, vs, table, new, ctx, True)
