"""The paged KV cache in 8 bits with a scale for each block and key/value head: its writer and its readers.

codes [num_blocks, Hkv, BS, 128] int8 or float8_e4m3fn, scales [num_blocks, Hkv] float32, value = code * scale, for K and V each.
The engine ops of the package take such a cache where their ``kv_scales`` are tensors [num_blocks, Hkv]: ``rope_cache`` and ``kv_write`` append to it,
``decode_attention`` and ``prefill_attention`` read it, ``kv_dequant_scratch`` hands its blocks back as bf16.  GPU tensors run
csrc/kernels/block_cache.hip, block_decode.hip and block_prefill.hip, CPU tensors the PyTorch forms of :mod:`.reference`.  (These take
other widths and types too; the kernels' rows are bf16, their heads 128 wide, decode has at most 16 query heads a key/value head, and
prompt attention no negative scale: other calls are refused.)

Scales are made by the append, as powers of two, so that nothing has to be calibrated: a block's grows when a token needs it,
and the block's codes move with it (see :func:`append`).  A cache needs no clearing: a block's first token (offset 0) starts its
scale anew.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from .. import _native
from . import reference as ref

HEAD_DIM = 128
CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}
BLOCKS = (16, 32, 64, 128)  # tokens of a block
MAX_GROUP = 16  # query heads per key/value head, decode


def blocked(kv_scales, cache) -> bool:
    """Whether kv_scales are those of a cache with a scale per block and head: tensors, but not of one element, which is a scale of the
    whole cache however it is held (unless codes of one block and one head have it in that shape)."""
    if ref.blocked(kv_scales[0], cache):
        return True
    if cache.dtype is torch.int8:  # (the kernels for one scale a tensor would read two bytes a value)
        raise TypeError("KV cache: int8 codes have a scale for each block and head, kv_scales [num_blocks, Hkv] float32 each")
    return False


def alloc(num_blocks: int, n_kv: int, block_size: int, dtype=torch.int8, device="cuda"):
    """An empty cache: (k codes, v codes, (k scales, v scales))."""
    if dtype not in CODES:
        raise TypeError(f"block-scaled cache: int8 or float8_e4m3fn codes, got {dtype}")
    shape = (num_blocks, n_kv, block_size, HEAD_DIM)
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
    return k, v, tuple(torch.zeros((num_blocks, n_kv), dtype=torch.float32, device=device) for _ in range(2))


def _stream(t: torch.Tensor) -> int:
    dev = torch._C._cuda_getDevice()
    if t.get_device() != dev:
        raise ValueError(f"block-scaled cache: tensors on {t.device}, current device is cuda:{dev}")
    return torch._C._cuda_getCurrentRawStream(dev)


def _check_cache(k, v, kv_scales):
    """(blocks, heads, tokens of a block, device's number).  (A call of few tokens takes its checks as long as its kernel: what is asked of
    a tensor is asked once.)"""
    ks, vs = kv_scales
    dtype = k.dtype
    if dtype not in CODES or v.dtype is not dtype:
        raise TypeError(f"block-scaled cache: int8 or float8_e4m3fn codes, got {k.dtype} and {v.dtype}")
    if not isinstance(vs, torch.Tensor) or ks.dtype is not torch.float32 or vs.dtype is not torch.float32:
        raise TypeError("block-scaled cache: scales are float32 tensors")
    shape = k.shape
    nb, hkv, bs, d = shape
    heads = (nb, hkv)
    if v.shape != shape or ks.shape != heads or vs.shape != heads:
        raise ValueError(f"block-scaled cache: codes {tuple(k.shape)} {tuple(v.shape)}, scales {tuple(ks.shape)} {tuple(vs.shape)}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("block-scaled cache: codes and scales are contiguous")
    if d != HEAD_DIM or bs not in BLOCKS:
        raise ValueError(f"block-scaled cache: heads of {HEAD_DIM}, blocks of 16, 32, 64 or 128 tokens; got {d} and {bs}")
    if (k.data_ptr() | v.data_ptr()) % 16:
        raise ValueError("block-scaled cache: codes are 16-byte aligned")
    dev = k.get_device()
    if v.get_device() != dev or ks.get_device() != dev or vs.get_device() != dev:
        raise ValueError("block-scaled cache: codes and scales on one device")
    return nb, hkv, bs, dev


def _check_on(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name}: on {t.device}, the cache is on {device}")


def append(q, k, v, positions, cos_sin, slot_mapping, k_cache, v_cache, kv_scales, rotate_q=True, q_out=None, row_scale=None):
    """Rotate, quantise and append.  q [T, Hq, 128] (or None), k, v [T, Hkv, 128] bf16 views whose tokens lie equally far apart;
    cos_sin None: as they come; a position past its rows takes the last one.  q_out [T, Hq, 128] takes the rotated q (it may be q).

    slot_mapping [T] int64: block * BS + offset, negative (or past the cache) for rows that have no place.  Tokens that go into one
    block lie behind one another, at offsets that rise by one; what the block holds in front of them belongs to the sequence, what
    it holds behind them does not.  Each block and head, K and V each, with M = 127 (int8) or 448 (e4m3):

      need = the smallest power of two with max |finite new values| <= M need;  scale = max(old scale, need)  (offset 0: need)
      new codes = round_half_even(x / scale), +-M where x is larger or infinite; a NaN is 0 in int8, NaN in e4m3
      if the scale grew: codes in front become round_half_even(code old / scale)

    Two runs of tokens into one block in one call are not ordered; rows that no token went into keep their codes."""
    if not k.is_cuda:
        return ref.block_append(q, k, v, positions, cos_sin, slot_mapping, k_cache, v_cache, kv_scales, rotate_q, q_out, row_scale)
    T, hkv, d = k.shape
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or (q is not None and q.dtype != torch.bfloat16):
        raise TypeError("append: q, k, v are bfloat16")
    if d != HEAD_DIM or v.shape != k.shape or (q is not None and (q.dim() != 3 or q.shape[0] != T or q.shape[2] != d)):
        raise ValueError(f"append: k {tuple(k.shape)}, v {tuple(v.shape)}, heads of {HEAD_DIM}")
    stride = k.stride(0)
    for t in (q, k, v):
        if t is not None and T > 0 and (t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != d) or (T > 1 and t.stride(0) != stride)):
            raise ValueError("append: heads of a token behind one another, tokens equally far apart")
    q_out = q if q_out is None else q_out
    if q is not None and (q_out.shape != q.shape or q_out.dtype != torch.bfloat16 or (T > 0 and (
            q_out.stride(2) != 1 or (q.shape[1] > 1 and q_out.stride(1) != d)))):
        raise ValueError("append: q_out is shaped as q, heads of a token behind one another")
    _check_on(k_cache.device, q=q, k=k, v=v, q_out=q_out)
    append_rows(0 if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(), T, stride if T > 1 else 0, 0 if q is None else q.shape[1], hkv,
                0 if q is None else q_out.data_ptr(), q_out.stride(0) if q is not None and T > 1 else 0, positions, cos_sin, slot_mapping, k_cache,
                v_cache, kv_scales, rotate_q, row_scale)
    return q_out


def append_rows(qp, kp, vp, T, stride, nq, hkv, qop, q_out_stride, positions, cos_sin, slot_mapping, k_cache, v_cache, kv_scales, rotate_q, row_scale):
    """append() on rows that the caller has looked at: bf16 at qp, kp, vp, tokens `stride` elements apart, on the cache's device."""
    nb, heads, bs, number = _check_cache(k_cache, v_cache, kv_scales)
    d = HEAD_DIM
    if heads != hkv:
        raise ValueError(f"append: {hkv} heads, the cache has {heads}")
    if (qp | kp | vp | qop) % 16 or stride % 8 or q_out_stride % 8:
        raise ValueError("append: rows are 16-byte aligned")
    n_cos = 0
    if cos_sin is not None:
        table = cos_sin.shape
        n_cos = table[0]
        if cos_sin.dtype is not torch.float32 or len(table) != 2 or n_cos < 1 or table[1] != d or not cos_sin.is_contiguous() or cos_sin.data_ptr() % 16:
            raise ValueError("append: cos_sin is [positions, 128] float32, contiguous")
        if positions.dtype not in (torch.int64, torch.int32) or positions.dim() != 1 or positions.numel() != T or not positions.is_contiguous():
            raise ValueError("append: positions are [T] int64 or int32, contiguous")
        if positions.get_device() != number or cos_sin.get_device() != number:
            raise ValueError(f"append: positions on {positions.device}, cos_sin on {cos_sin.device}, the cache on {k_cache.device}")
    if slot_mapping is not None and (slot_mapping.dtype is not torch.int64 or slot_mapping.dim() != 1 or slot_mapping.numel() != T
                                     or not slot_mapping.is_contiguous() or slot_mapping.get_device() != number):
        raise ValueError("append: slot_mapping is [T] int64, contiguous, on the cache's device")
    if row_scale is not None and (row_scale.dtype != torch.float32 or row_scale.shape != (T,) or not row_scale.is_contiguous() or row_scale.get_device() != number):
        raise ValueError("append: row_scale is [T] float32, contiguous, on the cache's device")
    _native.kernels().block_append(
        qp, kp, vp, stride, qop, q_out_stride, positions.data_ptr() if cos_sin is not None else 0,
        int(cos_sin is not None and positions.dtype == torch.int64), 0 if cos_sin is None else cos_sin.data_ptr(), n_cos,
        0 if row_scale is None else row_scale.data_ptr(), 0 if slot_mapping is None else slot_mapping.data_ptr(), k_cache.data_ptr(),
        v_cache.data_ptr(), kv_scales[0].data_ptr(), kv_scales[1].data_ptr(), T, nq, hkv, d, bs, nb, int(rotate_q), CODES[k_cache.dtype],
        _stream(k_cache))


def read_back(k_cache, v_cache, kv_scales, block_tables, ctx_lens, scratch):
    """ops.kv_dequant_scratch of a block-scaled cache.  K, V and a table that is made here are the caller's, as any result; blocks that no
    sequence's length reaches may hold anything."""
    nb, hkv, bs, dev = _check_cache(k_cache, v_cache, kv_scales)
    n, cols = block_tables.shape
    rows, step = block_tables.stride()
    if block_tables.dtype is not torch.int32 or ctx_lens.dtype is not torch.int32:
        raise TypeError("kv_dequant_scratch: tables and lengths are int32")
    if (cols > 1 and step != 1) or ctx_lens.dim() != 1 or ctx_lens.numel() != n or not ctx_lens.is_contiguous():
        raise ValueError(f"kv_dequant_scratch: block_tables {tuple(block_tables.shape)}, ctx_lens {tuple(ctx_lens.shape)}")
    if block_tables.get_device() != dev or ctx_lens.get_device() != dev:
        raise ValueError(f"kv_dequant_scratch: tables on {block_tables.device}, lengths on {ctx_lens.device}, the cache on {k_cache.device}")
    need = n * cols if scratch is None else scratch[1]
    if dev < 0:
        table = torch.arange(need, dtype=torch.int32).view(n, cols) if scratch is None else scratch[0]
        ks, vs = (torch.zeros((max(need, 1), hkv, bs, HEAD_DIM), dtype=torch.bfloat16) for _ in range(2))
        for i, ctx in enumerate(ctx_lens.tolist()):
            blocks = min(-(-ctx // bs), cols)
            src, dst = block_tables[i, :blocks].long(), table[i, :blocks].long()
            ks[dst] = ref.block_values(k_cache[src], kv_scales[0][src]).bfloat16()
            vs[dst] = ref.block_values(v_cache[src], kv_scales[1][src]).bfloat16()
        return ks, vs, table
    stream, blocks = _stream(k_cache), max(need, 1)
    if scratch is None:  # (the kernel writes it)
        table = block_tables.new_empty((n, cols))
    else:
        table = scratch[0]
        if table.dtype != torch.int32 or table.shape != (n, cols) or not table.is_contiguous() or table.get_device() != dev:
            raise ValueError(f"kv_dequant_scratch: the scratch's table is [{n}, {cols}] int32, contiguous, on {k_cache.device}")
    ks = k_cache.new_empty((blocks, hkv, bs, HEAD_DIM), dtype=torch.bfloat16)
    vs = torch.empty_like(ks)
    _native.kernels().block_dequant(k_cache.data_ptr(), v_cache.data_ptr(), kv_scales[0].data_ptr(), kv_scales[1].data_ptr(), ks.data_ptr(),
                                    vs.data_ptr(), block_tables.data_ptr(), rows, ctx_lens.data_ptr(), table.data_ptr(),
                                    int(scratch is None), n, cols, nb, blocks, hkv, bs, HEAD_DIM, CODES[k_cache.dtype], stream)
    return ks, vs, table


def _check_reader(q, out, k_cache, v_cache, kv_scales, block_tables, ctx_lens, n):
    nb, hkv, bs, dev = _check_cache(k_cache, v_cache, kv_scales)
    shape = q.shape
    T, hq, d = shape
    if nb < 1:
        raise ValueError("attention over a block-scaled cache: the cache has no block")
    if q.dtype is not torch.bfloat16 or out.dtype is not torch.bfloat16:
        raise TypeError("attention over a block-scaled cache: q and out are bfloat16")
    if d != HEAD_DIM or hkv < 1 or hq < 1 or hq % hkv or out.shape != shape or not out.is_contiguous():
        raise ValueError(f"attention over a block-scaled cache: q {tuple(q.shape)}, out {tuple(out.shape)}, {hkv} key/value heads")
    rows = 0
    if T:
        rows, heads, cols = q.stride()
        if cols != 1 or (hq > 1 and heads != d) or (T > 1 and rows % 8) or (q.data_ptr() | out.data_ptr()) % 16:
            raise ValueError("attention over a block-scaled cache: q's heads behind one another, its rows and out 16-byte aligned")
    if block_tables.dtype is not torch.int32 or ctx_lens.dtype is not torch.int32:
        raise TypeError("attention over a block-scaled cache: tables and lengths are int32")
    table, strides = block_tables.shape, block_tables.stride()
    if (len(table) != 2 or table[0] != n or table[1] < 1 or (table[1] > 1 and strides[1] != 1) or ctx_lens.dim() != 1 or
            ctx_lens.numel() != n or not ctx_lens.is_contiguous()):
        raise ValueError(f"attention over a block-scaled cache: block_tables {tuple(table)}, ctx_lens {tuple(ctx_lens.shape)}, {n} sequences")
    if q.get_device() != dev or out.get_device() != dev or block_tables.get_device() != dev or ctx_lens.get_device() != dev:
        raise ValueError(f"attention over a block-scaled cache: q on {q.device}, out on {out.device}, block_tables on {block_tables.device}, "
                         f"ctx_lens on {ctx_lens.device}, the cache on {k_cache.device}")
    return T, hq, d, nb, hkv, bs, rows if T > 1 else 0, table[1], strides[0]


def decode(q, k_cache, v_cache, block_tables, ctx_lens, scale, out, n_parts, workspace, kv_scales):
    B, hq, d, nb, hkv, bs, rows, cols, table_rows = _check_reader(q, out, k_cache, v_cache, kv_scales, block_tables, ctx_lens, q.shape[0])
    if hq // hkv > MAX_GROUP:
        raise ValueError(f"decode_attention: at most {MAX_GROUP} query heads per key/value head, got {hq // hkv}")
    if n_parts is None:
        n_parts = decode_parts(B, hkv, cols * bs)
    if n_parts < 1:
        raise ValueError(f"decode_attention: {n_parts} parts")
    t0 = t1 = 0
    if n_parts > 1 and B:
        if workspace is None:
            ws = q.new_empty(B * hq * n_parts * (d + 2), dtype=torch.float32)
            t0 = ws.data_ptr()
            t1 = t0 + 4 * B * hq * n_parts * d
        else:
            o, ml = workspace
            if o.dtype != torch.float32 or ml.dtype != torch.float32 or not (o.is_contiguous() and ml.is_contiguous()):
                raise TypeError("decode_attention: the workspace is float32, contiguous")
            if o.shape[0] < B or o.shape[1:] != (hq, n_parts, d) or ml.shape[0] < B or ml.shape[1:] != (hq, n_parts, 2):
                raise ValueError(f"decode_attention: workspace {tuple(o.shape)} {tuple(ml.shape)} for {(B, hq, n_parts, d)}")
            _check_on(q.device, workspace=o, sums=ml)
            t0, t1 = o.data_ptr(), ml.data_ptr()
    _native.kernels().block_decode(out.data_ptr(), t0, t1, q.data_ptr(), rows, k_cache.data_ptr(), v_cache.data_ptr(),
                                   kv_scales[0].data_ptr(), kv_scales[1].data_ptr(), block_tables.data_ptr(), table_rows, cols,
                                   ctx_lens.data_ptr(), B, hq, hkv, d, bs, nb, int(n_parts), float(scale),
                                   CODES[k_cache.dtype], _stream(q))
    return out


CUS = 256
# Tokens that eight waves take whole where a CU has one workgroup at most.  us on the GPU, whole and in the best number of parts with their
# join: 30 sequences of 700 tokens, 8 key/value heads 11.5 and 14.6, 30 of 300 7.6 and 11.0, 16 of 700 10.4 and 10.7, but one of 400 7.2 and 6.7,
# one of 700 8.7 and 7.1, eight 9.7 and 8.8.  These too are left whole: an eager call's host takes 4 us to start the join.  A caller that captures
# few short contexts names the number of parts.
WHOLE = 768


@functools.lru_cache(maxsize=4096)
def decode_parts(batch: int, n_kv: int, max_ctx: int) -> int:
    """Parts of a context for a decode launch over the 8-bit cache of `batch` contexts of at most `max_ctx` tokens: a CU's share of the
    workgroups, times a part's tokens and the 64 tokens' time that a part takes without any, is least, and a CU with one workgroup is a
    tenth slower.  us, this and the parts next to it, 8 key/value heads: 40 sequences of 3000 tokens 4 parts 46.1 (2 50.5, 5 48.7), 3 of
    60000 32 63.3 (22 81, 48 69), one of 700 6 7.3 (3 8.4), one of 4000 32 8.1 (16 8.8), 96 of 3150 1 92 (2 94)."""
    heads = batch * n_kv
    if heads <= CUS and max_ctx <= WHOLE:
        return 1

    def cost(p):
        wgs = -(-heads * p // CUS)
        return (wgs if wgs > 1 else 1.1) * (-(-max_ctx // (32 * p)) * 32 + 64)

    return min(range(1, max(1, min(64, max_ctx // 96)) + 1), key=cost)


class PrefillPlan(NamedTuple):
    """What a step's prompt rows are cut into, for all of its layers (:func:`prefill_plan`)."""
    work: torch.Tensor  # int32: n_work + n_few items of 6, then n_joins + n_few_joins of 4
    n_work: int
    n_few: int
    n_joins: int
    n_few_joins: int
    places: int  # tiles of sums in the workspace
    few_places: int
    join_rows: int  # rows and parts that a joined item has at most
    few_join_rows: int
    parts: int
    few_parts: int
    tile: int  # rows of a work item
    few_groups: int  # 16s of rows that the sequences of few rows have at most
    rows: int
    sequences: int
    n_q: int
    n_kv: int
    causal: bool


# Key tiles of 64 a CU from which 256-row workgroups, one a CU, are worth it.  us with 128 and 256 rows, 32 / 8 heads: 300 tokens behind 3700
# (9.7 tiles a CU) 51, 65; six chunks of 1000 tokens' contexts (14) 42, 41; 2000 (16) 61.0, 57.8; 3000 (35) 91, 87; 4000 (63) 156, 130; 200
# behind 19800 (39) 148, 97; 500 (1) 18.8, 21.3; six of 700 behind 200 (18, 2.06 turns) 60, 64.
WIDE_TILES, WIDE_WASTE = 12, 1.25
# Keys of a part at least, and key tiles of a part from which two parts of 128 rows a CU hide each other's waits: 32 tokens, us with one and
# two a CU, of 20480 (5 tiles a part of two) 29.9, 32.2, of 40960 (10) 44.4, 45.2, of 81920 81, 73.
PREFILL_KEYS, PAIR_TILES = 256, 16
FEW_ROWS, FEW_WGS, FEW_KEYS = 32, 256, 256
# Keys (times heads) of sequences of few rows that go with the others' tiles, where none is longer than theirs: a launch (and its join) less.  us,
# apart and together: 5 and 4 tokens, 14 / 2 heads, alone 14.2, 7.6, behind 1700 and 1200 24.1, 12.8; 32 / 8 heads, four of 300 and eight of 4
# behind 296 23.0, 15.6, 5000 and four of 6 behind 1794 236, 220.
BESIDE_KEYS = 65536
NO_END = 2 ** 31 - 1  # the end of a tile's last part: as far as the context that the call comes with


def prefill_plan(q_lens: list[int], ctx_lens: list[int], n_q: int, n_kv: int, device="cuda", causal: bool = True) -> PrefillPlan:
    """Cuts prompt chunks (q_lens new tokens each, the last of ctx_lens tokens) into work items for ``prefill_attention`` over a
    block-scaled cache: tiles of query rows, heaviest first, and where those are too few for the chip, parts of their keys.  Sequences of
    at most 32 rows a key/value head (new tokens times query heads per key/value head) go to a kernel of their own, where they have many keys
    or are alone.

    A plan holds for these new tokens, sequence by sequence: rows of a sequence that comes with others are NaN.  Contexts may have grown or
    shrunk since (a captured call's do); the work is only less evenly cut then."""
    if len(q_lens) != len(ctx_lens) or any(q < 0 or c < q for q, c in zip(q_lens, ctx_lens)):
        raise ValueError(f"prefill_plan: {list(q_lens)} new tokens of {list(ctx_lens)}")
    if n_kv < 1 or n_q < 1 or n_q % n_kv:
        raise ValueError(f"prefill_plan: {n_q} query heads, {n_kv} key/value heads")
    g = n_q // n_kv
    few = [s for s, ql in enumerate(q_lens) if 0 < ql * g <= FEW_ROWS]
    many = [s for s, ql in enumerate(q_lens) if ql * g > FEW_ROWS]
    if many and sum(ctx_lens[s] for s in few) * n_kv <= BESIDE_KEYS and max((ctx_lens[s] for s in few), default=0) <= max(ctx_lens[s] for s in many):
        few, many = [], sorted(few + many)

    def tiles(tile):
        """[key tiles, sequence, first row] of row tiles."""
        items, keys = [], 128 if tile == 64 else 64
        for s in many:
            ql, cl = q_lens[s], ctx_lens[s]
            for r0 in range(0, ql * g, tile):
                seen = cl - ql + (min(r0 + tile, ql * g) - 1) // g + 1 if causal else cl
                items.append((-(-seen // keys), s, r0))
        return items

    tile = 128 if any(q_lens[s] * g > 64 for s in many) else 64
    items = tiles(tile)
    if tile == 128:  # (rows of 256 that are mostly none cost what they are all worth)
        wide = tiles(256)
        total = sum(i[0] for i in wide)
        if total * n_kv >= WIDE_TILES * CUS and 2 * total <= WIDE_WASTE * sum(i[0] for i in items):
            tile, items = 256, wide

    def cut(items, unit, per, most):
        """items (units of keys, sequence, first row) -> work and joins: those of over 1.5 `per` units in parts of about `per`, the last
        without an end."""
        work, joins, places, rows, cuts = [], [], 0, 0, 0
        for n, s, r0 in items:
            parts = -(-n // per) if 2 * n > 3 * per else 1
            each = -(-n // parts)
            parts = -(-n // each)
            if parts == 1:
                work.append((n, [s, r0, 0, NO_END, -1, q_lens[s] * g]))
                continue
            joins += [s, r0, places, parts]
            rows, cuts = max(rows, min(most, q_lens[s] * g - r0)), max(cuts, parts)
            for p in range(parts):
                end = min((p + 1) * each, n)
                work.append((end - p * each, [s, r0, unit * p * each, NO_END if p == parts - 1 else unit * end, places + p, q_lens[s] * g]))
            places += parts
        if len(work) > 65535:
            raise ValueError(f"prefill_plan: {len(work)} work items, at most 65535")
        work.sort(key=lambda w: -w[0])
        return [x for _, w in work for x in w], joins, places, rows, cuts

    total = sum(i[0] for i in items)
    wgs = CUS * (2 if tile == 128 and total * n_kv >= 2 * CUS * PAIR_TILES else 1)
    unit = 128 if tile == 64 else 64
    per = max(PREFILL_KEYS // unit, -(-total * n_kv // wgs)) if len(items) * n_kv < wgs else 1 << 30
    work, joins, places, rows, parts = cut(items, unit, per, tile)
    for s, ql in enumerate(q_lens):  # (a sequence without rows has an item all the same, which looks whether it has come with some)
        if ql == 0:
            work += [s, 0, 0, 0, -1, 0]
    if len(work) > 6 * 65535:
        raise ValueError(f"prefill_plan: {len(work) // 6} work items, at most 65535")
    items = [(-(-ctx_lens[s] // 128), s, 0) for s in few]
    total = sum(i[0] for i in items)
    few_work, few_joins, few_places, few_rows, few_parts = cut(items, 128, max(FEW_KEYS // 128, -(-total * n_kv // FEW_WGS)), FEW_ROWS)
    flat = work + few_work + joins + few_joins
    most = max([q_lens[s] * g for s in few], default=0)
    return PrefillPlan(torch.tensor(flat or [0], dtype=torch.int32).to(device), len(work) // 6, len(few_work) // 6, len(joins) // 4, len(few_joins) // 4,
                       places, few_places, rows, few_rows, parts, few_parts, tile, 1 if most <= 16 else 2, sum(q_lens), len(q_lens), n_q, n_kv, causal)


def prefill(q, k_cache, v_cache, block_tables, cu_seqlens_q, ctx_lens, scale, out, plan, kv_scales, causal):
    if plan is None:
        cu = cu_seqlens_q.tolist()
        plan = prefill_plan([b - a for a, b in zip(cu, cu[1:])], ctx_lens.tolist(), q.shape[1], k_cache.shape[1], q.device, causal)
    if not isinstance(plan, PrefillPlan):
        raise TypeError("prefill_attention: over a block-scaled cache `work` is a plan of prefill_plan")
    n = cu_seqlens_q.shape[0] - 1
    T, hq, d, nb, hkv, bs, rows, cols, table_rows = _check_reader(q, out, k_cache, v_cache, kv_scales, block_tables, ctx_lens, n)
    if cu_seqlens_q.dtype != torch.int32 or not cu_seqlens_q.is_contiguous():
        raise TypeError("prefill_attention: cu_seqlens_q is int32, contiguous")
    if (plan.rows, plan.sequences, plan.n_q, plan.n_kv, plan.causal) != (T, n, hq, hkv, causal):
        raise ValueError(f"prefill_attention: a plan of {plan.rows} rows, {plan.sequences} sequences, {plan.n_q} / {plan.n_kv} heads, causal "
                         f"{plan.causal} for {T}, {n}, {hq} / {hkv}, {causal}")
    if not scale >= 0:
        raise ValueError(f"prefill_attention: scale {scale}, over a block-scaled cache it is not negative")
    _check_on(q.device, cu_seqlens_q=cu_seqlens_q, work=plan.work)
    o = ml = few_o = few_ml = 0
    tiles, few = plan.places * hkv * plan.tile, plan.few_places * hkv * FEW_ROWS
    if tiles or few:
        ws = q.new_empty((tiles + few) * (d + 2), dtype=torch.float32)
        o = ws.data_ptr()
        few_o = o + 4 * tiles * d
        ml = few_o + 4 * few * d
        few_ml = ml + 8 * tiles
    work = plan.work.data_ptr()
    _native.kernels().block_prefill(out.data_ptr(), o, ml, few_o, few_ml, q.data_ptr(), rows, k_cache.data_ptr(),
                                    v_cache.data_ptr(), kv_scales[0].data_ptr(), kv_scales[1].data_ptr(), block_tables.data_ptr(),
                                    table_rows, cols, cu_seqlens_q.data_ptr(), ctx_lens.data_ptr(), work, plan.n_work,
                                    plan.n_few, work + 24 * (plan.n_work + plan.n_few), plan.n_joins, plan.n_few_joins, plan.join_rows, plan.few_join_rows, plan.parts,
                                    plan.few_parts, plan.tile, plan.few_groups,
                                    hq, hkv, d, bs, nb, T, float(scale), int(causal), CODES[k_cache.dtype], _stream(q))
    return out
