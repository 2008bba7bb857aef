"""Products of few rows with weights in 4 bits: codes 0..15, a bf16 scale and (perhaps) a zero point 0..15 for each group of 32, 64 or
128 columns of a weight row,  w[n, k] = (code[n, k] - zero[n, k / group]) * scale[n, k / group]  (zero 8 where there are none).

GPU tensors run csrc/kernels/w4_gemm.hip, CPU tensors PyTorch in fp32."""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from .. import _native

GROUPS = (32, 64, 128)
MAX_ROWS = 256
# More than 16 rows go to w4_wide_kernel, which has x in LDS, from so much work or so many weights on.  us, bands of 16 rows and wide: 64 rows of
# 2048 x 2048 5.0, 11, of 4096 x 4096 9.3, 15.6, of 8192 x 4096 14.9, 19.6, of 8192 x 8192 26.3, 25.8; 128 rows of 8192 x 4096 26.3, 25.8, of 4096 x
# 14336 43, 33; 20 rows of 28672 x 4096 24.8, 19.5.
WIDE_WORK, WIDE_WEIGHTS = 4 << 30, 80 << 20


class W4Weight(NamedTuple):
    """A weight [n, k] as the kernel reads it (:func:`w4_pack`): rows in tiles of 16, columns in chunks of 128."""
    packed: torch.Tensor  # int32 [n / 16, k / 128, 64, 4]: lane 16 q + r, word s: columns 32 s + 8 q .. of row r
    scales: torch.Tensor  # bf16 [n / 16, k / 128, 16, groups of a chunk]
    zeros: torch.Tensor | None  # uint8, as scales: 128 + zero
    n: int
    k: int
    group: int


def _tiles(t: torch.Tensor, per: int) -> torch.Tensor:
    """[n, groups] -> [n / 16, chunks, 16, per], `per` groups a chunk; rows and groups that are none 0."""
    n, g = t.shape
    p = torch.zeros((-(-n // 16) * 16, -(-g // per) * per), dtype=t.dtype, device=t.device)
    p[:n, :g] = t
    return p.view(-1, 16, p.shape[1] // per, per).transpose(1, 2).contiguous()


def _rows(t: torch.Tensor, n: int, groups: int) -> torch.Tensor:
    return t.transpose(1, 2).reshape(16 * t.shape[0], -1)[:n, :groups]


def w4_pack(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, group: int) -> W4Weight:
    """Lays a quantised weight out for :func:`w4_linear`, once: codes [n, k] uint8 in 0..15, scales [n, k / group] bf16, zeros as
    scales in uint8 0..15 or None (8).  k is a multiple of group (32, 64 or 128)."""
    if codes.dim() != 2 or group not in GROUPS or codes.shape[0] < 1 or codes.shape[1] < group or codes.shape[1] % group:
        raise ValueError(f"w4_pack: codes {tuple(codes.shape)} in groups of {group} (32, 64 or 128, a divisor of the columns)")
    n, k = codes.shape
    if codes.dtype != torch.uint8 or scales.dtype != torch.bfloat16 or (zeros is not None and zeros.dtype != torch.uint8):
        raise TypeError("w4_pack: codes and zeros are uint8, scales bfloat16")
    if scales.shape != (n, k // group) or (zeros is not None and zeros.shape != scales.shape):
        raise ValueError(f"w4_pack: scales {tuple(scales.shape)} for {(n, k // group)}")
    if int(codes.max()) > 15 or (zeros is not None and int(zeros.max()) > 15):
        raise ValueError("w4_pack: codes and zeros are 0..15")
    n16, k128 = -(-n // 16), -(-k // 128)
    c = torch.zeros((n16 * 16, k128 * 128), dtype=torch.uint8, device=codes.device)
    c[:n, :k] = codes
    # [tile, row, chunk, step, quarter, 8] -> [tile, chunk, quarter, row, step, 8]
    c = c.view(n16, 16, k128, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)
    word = torch.zeros(c.shape[:-1], dtype=torch.int32, device=codes.device)
    for j in range(8):  # column 2 i in nibble i, 2 i + 1 in nibble 4 + i
        word |= c[..., j].to(torch.int32) << (4 * (j // 2 + 4 * (j % 2)))
    packed = word.reshape(n16, k128, 64, 4).contiguous()
    return W4Weight(packed, _tiles(scales, 128 // group), None if zeros is None else _tiles(zeros + 128, 128 // group), n, k, group)


def w4_quant(w: torch.Tensor, group: int = 128, symmetric: bool = True) -> W4Weight:
    """Quantises a weight [n, k] to the nearest codes: symmetric (zero 8, scale max |w| / 7) or over each group's range, 0 in it."""
    if w.dim() != 2 or group not in GROUPS or w.shape[1] < group or w.shape[1] % group:
        raise ValueError(f"w4_quant: a weight {tuple(w.shape)} in groups of {group}")
    n, k = w.shape
    x = w.float().reshape(n, k // group, group)
    if symmetric:
        s = x.abs().amax(-1) / 7
    else:
        lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
        s = (hi - lo) / 15
    s = s.to(torch.bfloat16)
    f = torch.where(s > 0, s, 1).float()
    z = None if symmetric else (-lo / f).round().clamp(0, 15)
    c = (x / f[..., None]).round() + (8 if z is None else z[..., None])
    return w4_pack(c.clamp(0, 15).to(torch.uint8).reshape(n, k), s, None if z is None else z.to(torch.uint8), group)


def w4_unpack(weight: W4Weight) -> torch.Tensor:
    """The weight's values [n, k] in fp32."""
    p, n16, k128 = weight.packed, weight.packed.shape[0], weight.packed.shape[1]
    w = p.view(n16, k128, 4, 16, 4, 1).expand(n16, k128, 4, 16, 4, 8)
    shift = torch.tensor([4 * (j // 2 + 4 * (j % 2)) for j in range(8)], dtype=torch.int32, device=p.device)
    c = ((w >> shift) & 15).permute(0, 3, 1, 4, 2, 5).reshape(n16 * 16, k128 * 128)[: weight.n, : weight.k].float()
    rows = lambda t: _rows(t, weight.n, weight.k // weight.group).float().repeat_interleave(weight.group, 1)  # noqa: E731
    zeros = 8.0 if weight.zeros is None else rows(weight.zeros) - 128
    return (c - zeros) * rows(weight.scales)


@functools.lru_cache(maxsize=4096)
def _shape(m: int, n: int, k: int) -> tuple[int, int, int]:
    """(waves of a workgroup, 16-row tiles of weights a wave, workgroups that K is split over).  Tiles share x's way from L2, but need
    workgroups enough for 256 CUs; us with 1, 2 and 4 tiles, groups of 128, one row: 4096 x 4096 (256 tiles of rows) 4.4, 5.0, -;
    6144 x 4096 6.3, 5.2, 7.2; 28672 x 4096 13.9, 13.3, 12.4; 16 rows: 8192 x 8192 (512) -, 11.9, 13.2; 11008 x 4096 (688) -, 11.5, 9.7.
    More than 8 rows of a long K take two tiles, and halve K while a CU has one workgroup at most: 16 rows, one tile, two, two and halves, of
    4096 x 6144 9.1, 10.0, 8.8, x 8192 10.9, 11.9, 10.2, x 14336 16.9, 18.6, 13.4, of 4352 x 8192 18.1, 11.9, 14.3, x 14336 29.5, 18.7, 20.7, of
    5600 x 11008 23.7, 15.3, 17.7; 9 rows of 4096 x 8192 8.3, 9.4, 8.8, x 14336 12.7, 14.6, 11.3; 8 of 4096 x 14336 10.9, -, 10.8; 48 of 1024 x 11008
    13.2, 14.4, 11.8, of 1536 x 11008 23.2, 14.5, 16.8.  Few rows of weights
    split K until there are 256 workgroups or a wave has its one chunk: 17 x 16000 26 -> 4.6, 1000 x 8192 11 -> 5.3.  More than 16 rows are
    bands of 16, which add to the workgroups, or (0 tiles) w4_wide_kernel's, which splits K up to 16 times: 64 rows of 28672 x 4096 (224 workgroups)
    31 in one part, 42 in two."""
    tiles, chunks, bands = -(-n // 16), -(-k // 128), max(1, -(-m // 16))
    if m > 16 and (m * n * k > WIDE_WORK or n * k > WIDE_WEIGHTS):  # eight tiles a workgroup, K split until there are 256 workgroups or it has two steps of 256 columns
        return 8, 0, max(1, min(chunks // 4, 16, 256 // (-(-tiles // 8) * -(-m // 64))))
    work = tiles * bands
    rt = 4 if work >= (640 if m > 8 else 1024) else 2 if work >= 384 else 1
    splits = 1
    if work < 384 and m > 8 and k >= 8192:
        rt, splits = 2, 2 if work <= 256 else 1
    groups = -(-tiles // rt) * bands
    if groups < 128:
        splits = max(splits, min(chunks // 8, 256 // groups))
    waves = 8
    while waves > 1 and waves * splits > chunks:
        waves //= 2
    if waves * splits > chunks:
        splits = 1
    return waves, rt, splits


def _check_weight(weight: W4Weight) -> int:
    """What the kernel takes for granted of a weight's tensors; their device's number.  (Each thing is asked once: a product of one row
    takes these checks nearly as long as its kernel.)"""
    p, s, z, n, k, group = weight
    if p.dtype is not torch.int32 or s.dtype is not torch.bfloat16 or (z is not None and z.dtype is not torch.uint8):
        raise TypeError(f"w4_linear: a weight of {p.dtype}, scales of {s.dtype}{'' if z is None else f', zeros of {z.dtype}'}, not as w4_pack lays it out")
    if group not in GROUPS or n < 1 or k < group or k % group:
        raise ValueError(f"w4_linear: a weight {(n, k)} in groups of {group}")
    chunks = -(-n // 16) * -(-k // 128)
    if (p.numel() != 256 * chunks or s.numel() * group != 2048 * chunks or not p.is_contiguous() or not s.is_contiguous()
            or p.data_ptr() % 16 or s.data_ptr() % 8):
        raise ValueError(f"w4_linear: a weight {(n, k)} in groups of {group} laid out as {tuple(p.shape)} and {tuple(s.shape)}, contiguous and 16-byte aligned")
    dev = p.get_device()
    if s.get_device() != dev:
        raise ValueError(f"w4_linear: a weight on {p.device}, its scales on {s.device}")
    if z is not None and (z.numel() != s.numel() or not z.is_contiguous() or z.data_ptr() % 4 or z.get_device() != dev):
        raise ValueError(f"w4_linear: zeros {tuple(z.shape)} on {z.device} beside scales {tuple(s.shape)} on {s.device}")
    return dev


def w4_linear(x: torch.Tensor, weight: W4Weight, out: torch.Tensor | None = None) -> torch.Tensor:
    """y [m, n] = x [m, k] . w^T for up to 256 rows of bf16, sums in fp32.  (CPU tensors: any number of rows of any type.)"""
    shape, (p, s, z, n, k, group) = x.shape, weight
    if len(shape) != 2 or shape[1] != k:
        raise ValueError(f"w4_linear: x {tuple(shape)}, weight {(n, k)}")
    m = shape[0]
    if not x.is_cuda:
        y = (x.float() @ w4_unpack(weight).t()).to(x.dtype)
        return y if out is None else out.copy_(y)
    if x.dtype != torch.bfloat16:
        raise TypeError(f"w4_linear: x is bfloat16, got {x.dtype}")
    if m > MAX_ROWS:
        raise ValueError(f"w4_linear: at most {MAX_ROWS} rows, got {m}")
    rows, cols = x.stride()
    xp, number = x.data_ptr(), x.get_device()
    if m and (cols != 1 or (m > 1 and rows % 8) or xp % 16):
        raise ValueError("w4_linear: rows of x have unit stride and are 16-byte aligned")
    dev = torch._C._cuda_getDevice()
    if number != dev or _check_weight(weight) != dev:
        raise ValueError(f"w4_linear: x on {x.device}, the weight on {p.device}, current device cuda:{dev}")
    if out is None:
        out = x.new_empty((m, n))
    elif out.shape != (m, n) or out.dtype is not x.dtype or out.get_device() != dev or (m and out.stride(1) != 1):
        raise ValueError("w4_linear: bad out tensor")
    waves, rt, splits = _shape(m, n, k)
    ws = x.new_empty(splits * m * n, dtype=torch.float32) if splits > 1 and m else None
    _native.kernels().w4_gemm(out.data_ptr(), out.stride(0), xp, rows if m > 1 else 0, p.data_ptr(), s.data_ptr(),
                              0 if z is None else z.data_ptr(), 0 if ws is None else ws.data_ptr(), m, n, k, group, waves, rt, splits,
                              torch._C._cuda_getCurrentRawStream(dev))
    return out
