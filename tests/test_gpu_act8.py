"""8-bit activation checkpoints against a definition in exact arithmetic: codes and scales have to be equal bit for bit, GELU and its
gradient are within bounds that follow from the arithmetic, the weight gradient within that of f32 sums."""
import pytest
import torch

from transcodon_amd import _lib, ops

DEV = "cuda"
gpu = pytest.mark.gpu
C = 2.0 ** -24                                                    # half a step of f32


def _half(dt):
    return 2.0 ** -8 if dt == torch.bfloat16 else C


def _pack(x):
    """(values f64, scales f64) from the definition; NaN where x is not finite."""
    x = x.double()
    M, E = x.shape
    out = torch.empty_like(x)
    scales = torch.empty(M, (E + 31) // 32, dtype=torch.float64)
    for g in range(scales.shape[1]):
        v = x[:, 32 * g:32 * g + 32]
        most = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(1, keepdim=True)
        e = torch.full_like(most, -126)
        for _ in range(260):                                      # the smallest power that fits
            e = torch.where(448.0 * torch.exp2(e) < most, e + 1, e)
        unit = torch.exp2(e)
        q = v / unit
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
        q = torch.round(q / step) * step * unit                   # torch.round: ties to even
        out[:, 32 * g:32 * g + 32] = torch.where(torch.isfinite(v), q, torch.full_like(q, float("nan")))
        scales[:, g] = unit[:, 0]
    return out, scales


def _values(codes, scales):
    s = scales.cpu().view(torch.uint8).double() - 127
    return codes.cpu().float().double() * torch.exp2(s).repeat_interleave(32, 1)[:, :codes.shape[1]]


def _input(M, E, dt, seed=0):
    """Normal values, runs of very different size, runs of zeros, exact ties and the largest code's neighbourhood."""
    gen = torch.Generator().manual_seed(seed + 31 * M + E)
    x = torch.randn(M, E, generator=gen)
    x = x * torch.exp2(torch.randint(-30, 20, (M, 1), generator=gen).float()) if M > 2 else x
    if E >= 64:
        x[0, :32] = 0.0
        x[0, 32:64] = torch.linspace(-448, 448, 32)
        if M > 3:
            x[3, :32] = torch.arange(32).float() * 2.0 ** -10      # ties among the smallest codes, next to 448
            x[3, 31] = 448.0
            x[3, 32:64] = 17.0 + torch.arange(32).float() / 2
            x[3, 63] = 449.0                                       # just past: the next power
    return x.to(dt)


SHAPES = [(1, 1), (1, 32), (1, 768), (3, 31), (5, 33), (2, 40), (7, 100), (131, 768), (64, 2048), (9, 4104), (1000, 8), (257, 96)]


@gpu
@pytest.mark.parametrize("M,E", SHAPES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_pack_and_unpack(M, E, dt):
    x = _input(M, E, dt)
    want, unit = _pack(x)
    codes, scales = ops.act8_pack(x.to(DEV))
    assert codes.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu and scales.shape == unit.shape
    assert torch.equal(torch.exp2(scales.cpu().view(torch.uint8).double() - 127), unit)
    assert torch.equal(_values(codes, scales), want)
    # e4m3: half a step is 2^-4 of the value, or 2^-10 of the unit where the code is subnormal
    per = unit.repeat_interleave(32, 1)[:, :E]
    assert bool(((want - x.double()).abs() <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * per)).all())
    for odt in (torch.float32, torch.bfloat16):
        assert torch.equal(ops.act8_unpack(codes, scales, odt).cpu().double(), want)
    # rows with a gap, and rows no vector load fits
    for first in (0, 8, 3):
        wide = torch.full((M, E + 16), float("nan"), dtype=dt, device=DEV)
        wide[:, first:first + E] = x.to(DEV)
        c2, s2 = ops.act8_pack(wide[:, first:first + E])
        assert torch.equal(c2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s2.view(torch.uint8), scales.view(torch.uint8))


@gpu
def test_pack_of_every_bf16_value():
    """All 65536 bit patterns, one at a time in a run of their own scale and 32 to a run."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    alone = torch.zeros(65536, 32, dtype=torch.bfloat16)
    alone[:, 5] = bits
    for x in (alone, bits.view(2048, 32)):
        want, unit = _pack(x)
        codes, scales = ops.act8_pack(x.to(DEV))
        assert torch.equal(torch.exp2(scales.cpu().view(torch.uint8).double() - 127), unit)
        got = _values(codes, scales)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(), want.nan_to_num())


@gpu
def test_values_that_are_not_finite_do_not_reach_their_neighbours():
    x = torch.randn(4, 70, generator=torch.Generator().manual_seed(1))
    clean = x.clone()
    x[1, 3], x[2, 40], x[3, 69] = float("inf"), float("nan"), float("-inf")
    for i, j in ((1, 3), (2, 40), (3, 69)):
        clean[i, j] = 0.0
    want, _ = _pack(clean)
    codes, scales = ops.act8_pack(x.to(DEV))
    got = _values(codes, scales)
    assert torch.equal(torch.isnan(got), ~torch.isfinite(x.double()))
    assert torch.equal(got.nan_to_num(), want)
    back = ops.act8_unpack(codes, scales, torch.float32).cpu()
    assert torch.equal(torch.isnan(back), ~torch.isfinite(x))
    _, c2, s2 = ops.gelu_act8(x.to(DEV))
    assert torch.equal(c2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s2.view(torch.uint8), scales.view(torch.uint8))


@gpu
def test_unpack_takes_scales_of_any_byte():
    codes = torch.full((256, 32), 1.5).to(torch.float8_e4m3fn).to(DEV)
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1).to(DEV).view(torch.float8_e8m0fnu)
    got = ops.act8_unpack(codes, scales, torch.float32).cpu().double()
    want = 1.5 * torch.exp2(torch.arange(256).double() - 127)
    assert bool(torch.isnan(got[255]).all())
    assert torch.equal(got[:255], want[:255, None].expand(255, 32))


def _cdf(x):
    return 0.5 * torch.special.erfc(x * -0.5 ** 0.5)             # (torch's ndtr has no relative accuracy below -7)


def _cdf_bound(x):
    """Bound of the kernel's Phi(x).  Lower tail q = Phi(-|x|): the fit is within 2.5 C, its evaluation within 16 C (8 roundings,
    the coefficients' magnitudes add up to 1.84 times the polynomial), reciprocal, exponential and products within 12 C, and the
    exponent -x^2/2 is rounded three times: 3 C x^2/2 of q.  Phi = 1 - q on the other side: C more."""
    q = _cdf(-x.abs())
    return (32 + 1.5 * x * x) * C * q + torch.where(x >= 0, C, 0.0) + 1e-37


@gpu
@pytest.mark.parametrize("M,E", SHAPES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_gelu_and_its_gradient(M, E, dt):
    gen = torch.Generator().manual_seed(M + E)
    u = (torch.randn(M, E, generator=gen) * 2.5).to(dt)
    u.view(-1)[:: 17] *= 4                                        # both tails
    dy = torch.randn(M, E, generator=gen).to(dt)
    act, codes, scales = ops.gelu_act8(u.to(DEV))
    c2, s2 = ops.act8_pack(u.to(DEV))
    assert torch.equal(c2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s2.view(torch.uint8), scales.view(torch.uint8))
    phi = _cdf

    def close(got, want, bound):
        assert got.dtype == dt
        # results below 2^-126 are rounded to whole multiples of 2^-133 (bf16; f32: 2^-149), so by up to 2^-134 whatever their size:
        # dy = 7.0e-5, v = -13 gives -7.2e-41, which lies between the neighbours 0 and -9.2e-41 = -2^-133
        assert bool(((got.cpu().double() - want).abs() <= bound + (want.abs() + bound) * (_half(dt) + C) + 2.0 ** -134).all())

    x = u.double()
    close(act, x * phi(x), x.abs() * _cdf_bound(x))
    v, d = _pack(u)[0], dy.double()
    pdf = torch.exp(-v * v / 2) * 0.3989422804014327
    # v phi(v): exponent rounded three times, exponential, constant and two products
    slope, bound = phi(v) + v * pdf, _cdf_bound(v) + (v * pdf).abs() * (8 + 1.5 * v * v) * C + 2 * C * (phi(v) + (v * pdf).abs())
    du, again = ops.dgelu_act8(dy.to(DEV), codes, scales, want_act=True)
    close(du, d * slope, d.abs() * bound)
    close(again, v * phi(v), v.abs() * _cdf_bound(v))
    assert torch.equal(ops.dgelu_act8(dy.to(DEV), codes, scales), du)
    wide = torch.zeros(M, E + 16, dtype=dt, device=DEV)
    for first in (8, 3):
        wide[:, first:first + E] = dy.to(DEV)
        assert torch.equal(ops.dgelu_act8(wide[:, first:first + E], codes, scales), du)


@gpu
def test_gelu_of_extreme_values():
    u = torch.tensor([[0.0, -0.0, 1e-40, 3e38, -3e38, 20.0, -20.0, float("inf"), float("nan"), -13.0, 5.5, -5.5]])
    act, codes, scales = ops.gelu_act8(u.to(DEV))
    want = u.double() * _cdf(u.double())
    a = act.cpu().double()
    assert bool(torch.isnan(a[0, 8])) and a[0, 7] == float("inf")
    keep = [0, 1, 2, 3, 4, 5, 6, 9, 10, 11]
    assert bool(((a - want).abs()[0, keep] <= want.abs()[0, keep] * 2e-5 + 1e-36).all())


@gpu
def test_gradient_is_that_of_differences():
    """Codes that hold exactly: multiples of 1/8 below 2.  d gelu by central differences in 64 bits."""
    u = (torch.arange(-15, 16).float() / 8).view(1, 31)
    _, codes, scales = ops.gelu_act8(u.to(DEV))
    assert torch.equal(_values(codes, scales), u.double())
    du = ops.dgelu_act8(torch.ones(1, 31, device=DEV), codes, scales).cpu().double()
    f = lambda t: t * _cdf(t)
    h = 1e-5
    slope = (f(u.double() + h) - f(u.double() - h)) / (2 * h)
    assert float((slope - du).abs().max()) < 64 * C + 1e-9        # Phi and u phi(u) below 1.2: _cdf_bound; h^2 f''' < 1e-9


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 8, 16), (1, 128, 128), (63, 8, 48), (64, 136, 112), (65, 128, 256), (131, 264, 80), (262, 768, 768),
                                   (1000, 96, 1040), (4097, 256, 256), (8192, 512, 768), (8200, 776, 784), (8192, 2304, 768), (8197, 2304, 776 + 8), (3400, 4096, 4096), (3392, 4096, 4096)])
def test_weight_gradient(M, N, K):
    gen = torch.Generator().manual_seed(M + N + K)
    dy = torch.randn(M, N, generator=gen).bfloat16()
    x = torch.randn(M, K, generator=gen) * torch.exp2(torch.randint(-6, 6, (M, 1), generator=gen).float())
    codes, scales = ops.act8_pack(x.bfloat16().to(DEV))
    v, d = _pack(x.bfloat16())[0], dy.double()
    want, size = d.t() @ v, d.abs().t() @ v.abs()
    tol = 2 * (M + 4) * C * size                                  # products are exact; M f32 additions in any order
    got = ops.gemm_tn_act8(dy.to(DEV), codes, scales)
    assert got.shape == (N, K) and got.dtype == torch.float32
    assert bool(((got.cpu().double() - want).abs() <= tol).all())
    assert float((got.cpu().double() - want).norm() / want.norm()) < 2e-6          # sums are cut into hundreds of parts
    assert torch.equal(got, ops.gemm_tn_act8(dy.to(DEV), codes, scales))
    base = torch.randn(N, K, generator=gen)
    out = base.to(DEV)
    assert ops.gemm_tn_act8(dy.to(DEV), codes, scales, out=out).data_ptr() == out.data_ptr()
    assert bool(((out.cpu().double() - base.double() - want).abs() <= tol + 2 * C * (base.double() + want).abs()).all())
    wide = torch.full((M, N + 16), float("nan"), dtype=torch.bfloat16, device=DEV)          # a NaN beside the rows is not read into them
    wide[:, 8:8 + N] = dy.to(DEV)
    assert torch.equal(ops.gemm_tn_act8(wide[:, 8:8 + N], codes, scales), got)


@gpu
@pytest.mark.parametrize("rows", [1, 128 * 64])
def test_weight_gradient_of_one_row_is_the_row(rows):
    """One row of ones among rows of zeros: every value of the activation comes out as it is, whatever its code and scale."""
    N, K = 2048, 1024
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    bits = bits[torch.isfinite(bits.float())]
    for first in range(0, 65280 - K + 1, 9 * K):
        x = torch.ones(rows, K, dtype=torch.bfloat16)
        x[rows // 2] = bits[first:first + K]
        dy = torch.zeros(rows, N, dtype=torch.bfloat16, device=DEV)
        dy[rows // 2] = 1.0
        codes, scales = ops.act8_pack(x.to(DEV))
        want = ops.act8_unpack(codes[rows // 2:rows // 2 + 1], scales[rows // 2:rows // 2 + 1], torch.float32)
        assert torch.equal(ops.gemm_tn_act8(dy, codes, scales), want.expand(N, K))


@gpu
def test_weight_gradient_keeps_a_nan_in_its_column():
    M, N, K = 200, 136, 144
    dy = torch.ones(M, N, dtype=torch.bfloat16, device=DEV)
    x = torch.ones(M, K, device=DEV)
    x[M - 1, 140] = float("nan")                                  # last row: the rows past it must not carry it on
    got = ops.gemm_tn_act8(dy, *ops.act8_pack(x))
    assert bool(torch.isnan(got[:, 140]).all())
    got[:, 140] = float(M)
    assert bool((got == float(M)).all())


@gpu
def test_empty_and_refused_calls():
    none = torch.zeros(0, 32, device=DEV)
    act, codes, scales = ops.gelu_act8(none)
    assert act.shape == (0, 32) and ops.dgelu_act8(none, codes, scales).shape == (0, 32)
    assert torch.equal(ops.gemm_tn_act8(torch.zeros(0, 8, dtype=torch.bfloat16, device=DEV), codes, scales), torch.zeros(8, 32, device=DEV))
    x = torch.zeros(4, 48, device=DEV)
    codes, scales = ops.act8_pack(x)
    dy = torch.zeros(4, 8, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: ops.act8_pack(x.half()), lambda: ops.gemm_tn_act8(dy.float(), codes, scales),
                lambda: ops.act8_unpack(codes.view(torch.uint8), scales), lambda: ops.act8_unpack(codes, scales, torch.float16),
                lambda: ops.act8_unpack(codes, scales.view(torch.uint8))):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: ops.act8_pack(x.t()), lambda: ops.act8_unpack(codes, scales[:, :1]), lambda: ops.dgelu_act8(x[:3], codes, scales),
                lambda: ops.gemm_tn_act8(dy[:3], codes, scales), lambda: ops.gemm_tn_act8(dy, codes, scales, out=torch.zeros(48, 8, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.gemm_tn_act8(dy[:, :4].contiguous(), codes, scales),
                lambda: ops.gemm_tn_act8(dy, *ops.act8_pack(torch.zeros(4, 40, device=DEV)))):
        with pytest.raises(_lib.HipLibraryError):
            bad()


def test_refusals_without_a_gpu():
    lib, one = _lib.load(), 1 << 12
    pack = lambda dt=0, x=one, ld=8, codes=one, scales=one, M=4, E=8: lib.tc_act8_pack(dt, x, ld, codes, scales, M, E, None)
    for bad in (dict(dt=4), dict(x=None), dict(ld=7), dict(codes=None), dict(scales=None), dict(M=0), dict(E=0), dict(x=one + 2), dict(E=2 ** 21)):
        assert pack(**bad) == -1, bad
    assert lib.tc_gelu_act8(0, one, 8, None, one, one, 4, 8, None) == -1
    assert lib.tc_act8_unpack(0, one, one, None, 4, 8, None) == lib.tc_act8_unpack(0, one, one, one + 1, 4, 8, None) == -1
    assert lib.tc_dgelu_act8(0, one, 7, one, one, one, None, 4, 8, None) == lib.tc_dgelu_act8(0, one, 8, one, one, None, None, 4, 8, None) == -1
    need = lib.tc_gemm_tn_act8_workspace_bytes(4, 8, 8, 16)
    assert need > 0 and lib.tc_gemm_tn_act8_workspace_bytes(4, 4, 4, 16) == lib.tc_gemm_tn_act8_workspace_bytes(4, 8, 8, 8) == 0
    tn = lambda dy=one, ld=8, codes=one, dW=one, M=4, N=8, K=16, ws=one, n=need: lib.tc_gemm_tn_act8(dy, ld, codes, one, dW, M, N, K, 0, ws, n, None)
    for bad in (dict(dy=None), dict(ld=4), dict(ld=12), dict(dy=one + 2), dict(codes=one + 8), dict(N=12), dict(K=24), dict(M=0), dict(ws=None)):
        assert tn(**bad) == -1, bad
    assert tn(n=need - 1) == -3


@gpu
@pytest.mark.parametrize("rows", [1, 128 * 64])
def test_weight_gradient_takes_scales_of_any_byte(rows):
    """One row of ones among rows of zeros, every scale byte in it: 0 stands for 2^-127, 255 for NaN."""
    N, K = 2048, 256 * 32
    codes = torch.full((rows, K), 1.5, device=DEV).to(torch.float8_e4m3fn)
    scales = torch.full((rows, 256), 127, dtype=torch.uint8, device=DEV)
    scales[rows // 2] = torch.arange(256, dtype=torch.uint8, device=DEV)
    scales = scales.view(torch.float8_e8m0fnu)
    dy = torch.zeros(rows, N, dtype=torch.bfloat16, device=DEV)
    dy[rows // 2] = 1.0
    got = ops.gemm_tn_act8(dy, codes, scales)
    want = ops.act8_unpack(codes[rows // 2:rows // 2 + 1], scales[rows // 2:rows // 2 + 1], torch.float32).expand(N, K)
    assert bool(torch.isnan(got[:, 255 * 32:]).all())
    # a product with a value below the smallest normal number may count as zero on the matrix cores
    assert bool(((got[:, :255 * 32] - want[:, :255 * 32]).abs() <= 2.0 ** -126).all())
    assert torch.equal(got[:, 2 * 32:255 * 32], want[:, 2 * 32:255 * 32])


def test_weight_gradient_workspace_is_bounded_without_a_gpu():
    """At most 128 MiB or a quarter of the operands' bytes, whatever the shape; rows behind the last whole stage take no part of
    the sum of their own."""
    need = _lib.load().tc_gemm_tn_act8_workspace_bytes
    gen = torch.Generator().manual_seed(3)
    size = lambda lo, hi: int(2.0 ** (lo + (hi - lo) * float(torch.rand(1, generator=gen))))
    shapes = [(231953, 13736, 12176), (100000, 8192, 8192), (50000, 20000, 20000), (65536, 2304, 768), (2 ** 31 - 100, 8, 16)]
    shapes += [(size(0, 24), size(0, 13) * 8, size(0, 12) * 16) for _ in range(3000)]
    for M, N, K in shapes:
        for rows in (M, M // 64 * 64 or M):
            got = need(rows, N, N, K)
            assert 0 < got <= max(128 * 2 ** 20, rows * (2 * N + K) // 4), (rows, N, K, got)
            assert got == 16 or got % (4 * N * K) == 0
    assert need(3400, 4096, 4096, 4096) == need(3392, 4096, 4096, 4096) == 16


@gpu
@pytest.mark.parametrize("M", [3393, 3400, 3455, 8193, 8255])
@pytest.mark.parametrize("N,K", [(4096, 4096), (2304, 784)])
def test_weight_gradient_counts_the_last_rows_once(M, N, K):
    """Whole stages are ones in dy, the rows behind them twos: sums of small whole numbers, exact in any order."""
    dy = torch.ones(M, N, dtype=torch.bfloat16, device=DEV)
    dy[M // 64 * 64:] = 2.0
    codes, scales = ops.act8_pack(torch.ones(M, K, device=DEV))
    want = float(M + M % 64)
    assert bool((ops.gemm_tn_act8(dy, codes, scales) == want).all())
    out = torch.full((N, K), 5.0, device=DEV)
    assert bool((ops.gemm_tn_act8(dy, codes, scales, out=out) == want + 5.0).all())


@gpu
@pytest.mark.parametrize("M,E", [(1, 1), (5, 33), (7, 100), (131, 768), (300, 96), (9, 4104), (2000, 2048)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("again", [False, True])
def test_gradient_in_place_of_the_one_it_comes_from(M, E, dt, again):
    """tc_dgelu_act8: du may be dy."""
    lib, gen = _lib.load(), torch.Generator().manual_seed(M + E)
    u, dy = torch.randn(M, E, generator=gen).to(dt).to(DEV), torch.randn(M, E, generator=gen).to(dt).to(DEV)
    codes, scales = ops.act8_pack(u)
    want, want_act = ops.dgelu_act8(dy, codes, scales, want_act=True)
    act = torch.empty_like(dy)
    assert lib.tc_dgelu_act8(int(dt == torch.bfloat16), dy.data_ptr(), E, codes.data_ptr(), scales.data_ptr(), dy.data_ptr(),
                             act.data_ptr() if again else None, M, E, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(dy, want) and (not again or torch.equal(act, want_act))
