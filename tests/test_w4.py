"""Products of few rows with 4-bit weights (ops/w4.py, csrc/kernels/w4_gemm.hip) against the definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

from dynamo_exp_amd import ops


def make(n, k, group, zeros, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = (0.01 * torch.exp(torch.randn((n, k // group), generator=g))).bfloat16()
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    w = codes.double() - (8.0 if z is None else z.double().repeat_interleave(group, 1))
    return codes, scales, z, w * scales.double().repeat_interleave(group, 1)


def near(got, x, w, scales, group):
    """y's own rounding, and sums in fp32 of (128 + code) x and (128 + zero) x (143 at most each) over a group (its products added one
    by one at worst) and over the groups."""
    x = x.double()
    want = x @ w.T
    size = (x.abs() * 1.0) @ scales.double().repeat_interleave(group, 1).T
    tol = 2 ** -8 * want.abs() * 1.01 + (group + w.shape[1] // group + 4) * 2 ** -24 * 286 * size
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 16, 128), (1, 1, 128), (3, 17, 384), (16, 100, 896), (17, 48, 1152), (33, 250, 256), (64, 31, 4096), (65, 40, 640), (130, 64, 128), (256, 33, 256)])
def test_product(m, n, k, group, zeros):
    codes, scales, z, w = make(n, k, group, zeros, seed=m + n)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)).bfloat16()
    weight = ops.w4_pack(codes.cuda(), scales.cuda(), None if z is None else z.cuda(), group)
    near(ops.w4_linear(x.cuda(), weight).cpu(), x, w, scales, group)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [32, 96, 160, 4128])
@pytest.mark.parametrize("m", [1, 20])
def test_columns_that_end_inside_a_chunk(k, m):
    codes, scales, z, w = make(70, k, 32, True, seed=k)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)).bfloat16()
    near(ops.w4_linear(x.cuda(), ops.w4_pack(codes.cuda(), scales.cuda(), z.cuda(), 32)).cpu(), x, w, scales, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (1, 28672, 4096), (16, 4096, 14336), (5, 6144, 4096), (40, 8192, 8192), (2, 9001, 2048)])
def test_layer_sizes(m, n, k):
    codes, scales, z, w = make(n, k, 128, False, seed=n)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)).bfloat16()
    near(ops.w4_linear(x.cuda(), ops.w4_pack(codes.cuda(), scales.cuda(), None, 128)).cpu(), x, w, scales, 128)


@pytest.mark.gpu
def test_rows_with_a_common_part():
    """x far from zero on average: what the codes' offset adds to the sums is 136 times their mean."""
    codes, scales, z, w = make(64, 4096, 128, True, seed=3)
    x = (torch.randn((2, 4096), generator=torch.Generator().manual_seed(1)) + 20).bfloat16()
    near(ops.w4_linear(x.cuda(), ops.w4_pack(codes.cuda(), scales.cuda(), z.cuda(), 128)).cpu(), x, w, scales, 128)


@pytest.mark.gpu
def test_rows_apart_and_out():
    """Rows of a wider tensor, an `out` whose rows lie apart; what lies between them is left."""
    codes, scales, z, w = make(40, 256, 64, True, seed=5)
    wide = torch.randn((6, 512), generator=torch.Generator().manual_seed(2)).bfloat16()
    x = wide[:, 128:384]
    out = torch.full((6, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    weight = ops.w4_pack(codes.cuda(), scales.cuda(), z.cuda(), 64)
    r = ops.w4_linear(wide.cuda()[:, 128:384], weight, out[:, :40])
    near(r.cpu(), x, w, scales, 64)
    assert bool((out[:, 40:] == 7).all())
    assert ops.w4_linear(x[:0].cuda(), weight).shape == (0, 40)


@pytest.mark.gpu
def test_infinities_stay_in_their_rows():
    codes, scales, z, w = make(33, 256, 32, False, seed=6)
    x = torch.randn((4, 256), generator=torch.Generator().manual_seed(2)).bfloat16()
    bad = x.clone()
    bad[1, 3], bad[2, 9] = float("nan"), float("inf")
    weight = ops.w4_pack(codes.cuda(), scales.cuda(), None, 32)
    got, want = ops.w4_linear(bad.cuda(), weight).cpu(), ops.w4_linear(x.cuda(), weight).cpu()
    assert torch.equal(got[[0, 3]], want[[0, 3]]) and not bool(got[1:3].isfinite().any())


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    codes, scales, z, w = make(512, 2048, 128, True, seed=7)
    weight = ops.w4_pack(codes.cuda(), scales.cuda(), z.cuda(), 128)
    x = torch.zeros((3, 2048), dtype=torch.bfloat16, device="cuda")
    out = torch.zeros((3, 512), dtype=torch.bfloat16, device="cuda")
    ops.w4_linear(x, weight, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):  # (as the engine captures: torch keeps the generator's state of the first capture)
        ops.w4_linear(x, weight, out)
    side = torch.cuda.Stream()
    for i in range(4):
        new = torch.randn((3, 2048), generator=torch.Generator().manual_seed(i)).bfloat16()
        x.copy_(new)
        graph.replay()
        eager = ops.w4_linear(new.cuda(), weight)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = ops.w4_linear(x, weight)
        side.synchronize()
        assert torch.equal(out, eager) and torch.equal(other, eager)
        near(eager.cpu(), new, w, scales, 128)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,k,group", [(5, 96, 32), (33, 256, 128), (16, 192, 64)])
def test_pack_and_unpack(n, k, group, zeros):
    codes, scales, z, w = make(n, k, group, zeros)
    weight = ops.w4_pack(codes, scales, z, group)
    assert torch.equal(ops.w4_unpack(weight).double(), w)
    x = torch.randn((3, k)).bfloat16()
    near(ops.w4_linear(x, weight), x, w, scales, group)


@pytest.mark.parametrize("symmetric", [False, True])
def test_quantised_weights_are_near(symmetric):
    """Within half a step of the group's scale, and the scale's own rounding to bf16 (2^-8 of at most 8, or 15, steps)."""
    w = torch.randn((40, 256), generator=torch.Generator().manual_seed(1)) * 0.1
    w[3, :64] = 0
    q = ops.w4_quant(w, 64, symmetric)
    s = ops.w4_unpack(q)
    codes = torch.full((40, 256), 9 if symmetric else 1, dtype=torch.uint8)  # one step above zero: the step itself
    one = q._replace(packed=ops.w4_pack(codes, torch.ones((40, 4)).bfloat16(), None, 64).packed, zeros=None if symmetric else torch.full_like(q.zeros, 128))
    step = ops.w4_unpack(one)
    assert bool(((s - w).abs() <= step * (0.5 + (8 if symmetric else 30) * 2 ** -8) + (0 if symmetric else 0.5) * step).all())
    assert bool((s[3, :64] == 0).all())


def test_refusals():
    codes, scales, z, _ = make(16, 128, 32, True)
    for bad in ((codes, scales, z, 16), (codes, scales, z, 64), (codes[:, :100], scales, z, 32), (codes, scales[:8], z, 32), (codes, scales, z[:, :2], 32), (codes + 1, scales, z, 32),
                (codes, scales, z + 1, 32), (codes[:0], scales[:0], None, 32)):
        with pytest.raises(ValueError):
            ops.w4_pack(*bad)
    for bad in ((codes.int(), scales, z, 32), (codes, scales.float(), z, 32), (codes, scales, z.int(), 32)):
        with pytest.raises(TypeError):
            ops.w4_pack(*bad)
    with pytest.raises(ValueError):
        ops.w4_quant(torch.zeros((4, 48)), 32)
    weight = ops.w4_pack(codes, scales, z, 32)
    for x in (torch.zeros((2, 96)), torch.zeros(128)):
        with pytest.raises(ValueError):
            ops.w4_linear(x, weight)


@pytest.mark.gpu
def test_refusals_gpu():
    codes, scales, z, _ = make(16, 128, 32, True)
    weight = ops.w4_pack(codes.cuda(), scales.cuda(), z.cuda(), 32)
    b = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    for x in (b(257, 128), b(2, 132)[:, :128], b(128, 2).t(), b(257)[1:].view(2, 128)):
        with pytest.raises(ValueError):
            ops.w4_linear(x, weight)
    with pytest.raises(TypeError):
        ops.w4_linear(b(2, 128).float(), weight)
    with pytest.raises(ValueError):
        ops.w4_linear(b(2, 128), weight, b(2, 17))
    with pytest.raises(ValueError):
        ops.w4_linear(b(2, 128), ops.w4_pack(codes, scales, z, 32))


@pytest.mark.gpu
def test_refuses_a_weight_laid_out_otherwise():
    codes, scales, z, _ = make(48, 256, 32, True)
    w = ops.w4_pack(codes.cuda(), scales.cuda(), z.cuda(), 32)
    x = torch.zeros((2, 256), dtype=torch.bfloat16, device="cuda")
    for bad in (w._replace(packed=w.packed[:2]), w._replace(scales=w.scales[:, :1]), w._replace(zeros=w.zeros[:1]), w._replace(n=64), w._replace(group=64),
                w._replace(scales=w.scales.cpu()), w._replace(zeros=w.zeros.cpu())):
        with pytest.raises(ValueError):
            ops.w4_linear(x, bad)


@pytest.fixture
def wide(monkeypatch):
    """More than 16 rows through w4_wide_kernel whatever the sizes."""
    from dynamo_exp_amd.ops import w4
    monkeypatch.setattr(w4, "WIDE_WORK", -1)
    w4._shape.cache_clear()
    yield w4
    w4._shape.cache_clear()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k", [(17, 48, 1152), (33, 250, 256), (64, 31, 4096), (65, 40, 640), (130, 64, 128), (256, 33, 256), (32, 513, 2176), (48, 128, 1408)])
def test_wide_product(m, n, k, group, zeros, wide):
    assert wide._shape(m, n, k)[1] == 0
    codes, scales, z, w = make(n, k, group, zeros, seed=m + n)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)).bfloat16()
    weight = ops.w4_pack(codes.cuda(), scales.cuda(), None if z is None else z.cuda(), group)
    near(ops.w4_linear(x.cuda(), weight).cpu(), x, w, scales, group)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [32, 96, 160, 4128])
def test_wide_columns_that_end_inside_a_chunk(k, wide):
    codes, scales, z, w = make(70, k, 32, True, seed=k)
    x = torch.randn((20, k), generator=torch.Generator().manual_seed(k)).bfloat16()
    near(ops.w4_linear(x.cuda(), ops.w4_pack(codes.cuda(), scales.cuda(), z.cuda(), 32)).cpu(), x, w, scales, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(20, 28672, 4096), (256, 2048, 2048), (100, 17, 16000), (129, 1000, 8192), (17, 4096, 4096)])
def test_bands_of_rows(m, n, k):
    codes, scales, z, w = make(n, k, 64, True, seed=n)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)).bfloat16()
    near(ops.w4_linear(x.cuda(), ops.w4_pack(codes.cuda(), scales.cuda(), z.cuda(), 64)).cpu(), x, w, scales, 64)


def test_weights_that_the_kernel_cannot_read_are_refused():
    """Types, strides and alignment of a weight's tensors: what the kernel takes for granted of the memory behind them."""
    from dynamo_exp_amd.ops import w4
    codes, scales, z, _ = make(48, 256, 32, True)
    w = ops.w4_pack(codes, scales, z, 32)
    w4._check_weight(w)
    one = torch.zeros(w.packed.numel() + 1, dtype=torch.int32)
    for bad, kind in ((w._replace(packed=w.packed.to(torch.int64)), TypeError), (w._replace(packed=w.packed.to(torch.uint8)), TypeError), (w._replace(scales=w.scales.float()), TypeError),
                      (w._replace(scales=w.scales.view(torch.float16)), TypeError), (w._replace(scales=w.scales.to(torch.float8_e4m3fn)), TypeError), (w._replace(zeros=w.zeros.int()), TypeError),
                      (w._replace(packed=w.packed[:1].expand(3, -1, -1, -1)), ValueError), (w._replace(scales=w.scales[:1].expand(3, -1, -1, -1)), ValueError),
                      (w._replace(zeros=w.zeros[:1].expand(3, -1, -1, -1)), ValueError), (w._replace(packed=w.packed.transpose(0, 1)), ValueError),
                      (w._replace(packed=one[1:].view(w.packed.shape)), ValueError), (w._replace(n=64), ValueError), (w._replace(n=0), ValueError), (w._replace(k=2 ** 20), ValueError),
                      (w._replace(group=64), ValueError), (w._replace(group=0), ValueError), (w._replace(k=250), ValueError), (w._replace(zeros=w.zeros[:, :1]), ValueError)):
        with pytest.raises(kind):
            w4._check_weight(bad)


@pytest.mark.gpu
def test_weights_that_the_kernel_cannot_read_are_refused_gpu():
    codes, scales, z, _ = make(48, 256, 32, True)
    w = ops.w4_pack(codes.cuda(), scales.cuda(), z.cuda(), 32)
    x = torch.zeros((2, 256), dtype=torch.bfloat16, device="cuda")
    for bad, kind in ((w._replace(scales=w.scales.to(torch.float8_e4m3fn)), TypeError), (w._replace(packed=w.packed[:1].expand(3, -1, -1, -1)), ValueError), (w._replace(zeros=w.zeros.int()), TypeError)):
        with pytest.raises(kind):
            ops.w4_linear(x, bad)


def infinite(got, want, x, w):
    """Infinities and NaN where the definition has them; the rest within sums in fp32 of its products, one by one."""
    size = x.double().nan_to_num(0, 0, 0).abs() @ w.abs().T
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf())
    ok = want.isfinite()
    err = (got.double() - want).abs()[ok]
    assert bool((err <= 2 ** -8 * want.abs()[ok] * 1.01 + (w.shape[1] + 4) * 2 ** -24 * size[ok]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k,group", [(1, 33, 256, 32), (4, 48, 1152, 128), (7, 40, 640, 64), (16, 100, 896, 128), (16, 64, 8192, 64), (40, 48, 1152, 32), (100, 17, 16000, 128), (64, 8192, 8448, 64)])
def test_infinite_and_huge_rows(m, n, k, group, zeros):
    """x that is infinite, or so large that 128 and 143 times it is: the definition's results, as on the CPU."""
    codes, scales, z, w = make(n, k, group, zeros, seed=m)
    scales = (scales.float() * 2.0 ** -6).bfloat16()
    w = w * 2.0 ** -6
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)).bfloat16()
    x[0, 5] = float("inf")
    if m > 1:
        x[1, 9], x[1, k - 1] = float("inf"), float("-inf")
        x[2] *= 2.0 ** 119
        x[3, k // 2] = -3e38
    weight = ops.w4_pack(codes.cuda(), scales.cuda(), None if z is None else z.cuda(), group)
    want = x.double() @ w.T
    assert bool((want[0].isinf() | want[0].isnan()).all()) and (m == 1 or bool(want[2:4].isfinite().all()))
    infinite(ops.w4_linear(x.cuda(), weight).cpu(), want, x, w)


def test_a_long_k_is_halved_where_cus_are_free():
    """More than 8 rows of a long K: two tiles a wave, and halves of K only while these are a workgroup a CU at most (256)."""
    from dynamo_exp_amd.ops import w4
    for m, n, k in ((9, 4096, 8192), (16, 4097, 8192), (16, 4352, 14336), (16, 6128, 20480), (32, 2048, 11008), (32, 2304, 11008), (48, 1365, 8192), (48, 1536, 8192), (64, 1040, 14336)):
        bands = -(-m // 16)
        waves, rt, splits = w4._shape(m, n, k)
        assert rt == 2 and splits == (2 if -(-n // 16) * bands <= 256 else 1)
        assert waves == 8 and (splits == 1 or -(-n // 32) * bands * splits <= 256)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(9, 4352, 8192), (16, 4104, 11008), (32, 2304, 8192), (48, 1536, 8320)])
def test_long_rows_of_more_tiles_than_cus(m, n, k):
    codes, scales, z, w = make(n, k, 64, True, seed=n)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)).bfloat16()
    near(ops.w4_linear(x.cuda(), ops.w4_pack(codes.cuda(), scales.cuda(), z.cuda(), 64)).cpu(), x, w, scales, 64)
