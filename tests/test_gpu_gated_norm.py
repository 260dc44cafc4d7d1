"""Norms before and after a block with gate and residual scale, against the formulas in 64 bits.

Tolerances follow the arithmetic.  C = 2^-24 is half a step of f32.  A row sum is at most 16 additions in a lane, 6 across a wave
and 8 across waves, so with the few operations around it every f32 intermediate is within K C of the sum of the magnitudes that
enter it, K = 64; errors of inputs are carried on through the derivative.  A column sum of n rows is within n C of the sum of
its terms' magnitudes.  Results rounded to bf16 are off by another 2^-8 of the value."""
import os
import re

import pytest
import torch

from transcodon_amd import _lib, ops

DEV = "cuda"
gpu = pytest.mark.gpu
C, K = 2.0 ** -24, 64
EPS = float(torch.tensor(1e-5))                                   # the call's eps is an f32


def _half(dt):
    return 2.0 ** -8 if dt == torch.bfloat16 else C


def _case(M, E, dt, G, rms, pre=True, seed=0, gate_dt=torch.float32):
    gen = torch.Generator().manual_seed(seed + 7 * M + E)
    r = lambda *s: torch.randn(*s, generator=gen)
    return dict(y=(r(M, E) * 1.5 + 0.3).to(dt), x=r(M, E) * 2 - 0.2, post_gamma=1 + 0.1 * r(E), post_beta=None if rms else 0.1 * r(E),
                gate=None if G == 0 else (0.5 + 0.3 * r(G, E)).to(gate_dt), pre_gamma=1 + 0.1 * r(E) if pre else None,
                pre_beta=None if rms or not pre else 0.1 * r(E), dh=r(M, E).to(dt) if pre else None, dx_out=r(M, E))


def _on_gpu(c):
    return {k: None if v is None else v.to(DEV) for k, v in c.items()}


def _norm(t, err, gamma, beta, rms):
    """(norm, its error bound, t_hat, rstd) of f64 rows t known up to err."""
    mean = torch.zeros_like(t[:, :1]) if rms else t.mean(1, keepdim=True)
    rstd = ((t - mean).square().mean(1, keepdim=True) + EPS).rsqrt()
    hat = (t - mean) * rstd
    g = gamma.double()
    out = hat * g + (0 if beta is None else beta.double())
    size = (hat * g).abs() + (0 if beta is None else beta.double().abs()) + t.abs().mean(1, keepdim=True) * rstd * g.abs()
    carried = rstd * g.abs() * (err + err.mean(1, keepdim=True) + hat.abs() * (hat.abs() * err).mean(1, keepdim=True))
    return out, K * C * size + 1.5 * carried, hat, rstd


def _gated(gate, t):
    return t if gate is None else (gate.double()[:, None] * t.view(gate.shape[0], -1, t.shape[1])).view_as(t)


def _forward(c, rms, res):
    y, x = c["y"].double(), c["x"].double()
    n, e, _, _ = _norm(y, torch.zeros_like(y), c["post_gamma"], c["post_beta"], rms)
    gate_abs = None if c["gate"] is None else c["gate"].abs()
    x_out = res * x + _gated(c["gate"], n)
    ex = _gated(gate_abs, e) + 4 * C * ((res * x).abs() + _gated(c["gate"], n).abs())
    if c["pre_gamma"] is None:
        return x_out, ex, None, None
    h, eh, _, _ = _norm(x_out, ex, c["pre_gamma"], c["pre_beta"], rms)
    return x_out, ex, h, eh + (h.abs() + eh) * _half(c["y"].dtype)


SHAPES = [(1, 1), (1, 768), (2, 3), (3, 770), (131, 768), (5, 1024), (7, 1025), (4, 1028), (9, 2048), (6, 4096), (3, 4100), (2, 5001),
          (2, 8192), (600, 8), (1030, 64)]


@gpu
@pytest.mark.parametrize("M,E", SHAPES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rms", [False, True])
def test_forward(M, E, dt, rms):
    res = 0.875
    for G in sorted({0, 1, M}):
        for gate_dt in {torch.float32, dt}:
            c = _case(M, E, dt, G, rms, gate_dt=gate_dt)
            want_x, ex, want_h, eh = _forward(c, rms, res)
            g = _on_gpu(c)
            x_out, h, stats = ops.gated_residual_norm(g["y"], g["x"], g["post_gamma"], g["post_beta"], g["gate"], g["pre_gamma"],
                                                      g["pre_beta"], res_scale=res, rms=rms)
            assert x_out.dtype == torch.float32 and h.dtype == dt and stats.shape == (M, 4)
            assert bool(((x_out.cpu().double() - want_x).abs() <= ex).all())
            assert bool(((h.cpu().double() - want_h).abs() <= eh).all())
            if rms:
                assert bool((stats[:, ::2] == 0).all())


@gpu
def test_forward_without_the_second_norm_and_with_strided_rows():
    c = _case(33, 768, torch.bfloat16, 3, False, pre=False)
    want_x, ex, _, _ = _forward(c, False, 1.0)
    g = _on_gpu(c)
    x_out, h, stats = ops.gated_residual_norm(g["y"], g["x"], g["post_gamma"], g["post_beta"], g["gate"])
    assert h is None and bool((stats[:, 2:] == 0).all())
    assert bool(((x_out.cpu().double() - want_x).abs() <= ex).all())
    for first in (0, 4, 5):                                       # 5: rows no vector load fits
        wide_y = torch.zeros(33, 780, dtype=torch.bfloat16, device=DEV)
        wide_x = torch.zeros(33, 780, device=DEV)
        wide_y[:, first:first + 768], wide_x[:, first:first + 768] = g["y"], g["x"]
        again, _, _ = ops.gated_residual_norm(wide_y[:, first:first + 768], wide_x[:, first:first + 768], g["post_gamma"],
                                              g["post_beta"], g["gate"])
        assert bool(((again.cpu().double() - want_x).abs() <= ex).all())


def _norm_back(hat, rstd, mean_size, q, eq, rms):
    """Gradient through a norm and its bound: q = gradient times gamma, known up to eq; t_hat known up to K C (..)."""
    eh = K * C * (hat.abs() + mean_size * rstd)
    m = lambda t: t.mean(1, keepdim=True)
    m1 = 0.0 if rms else m(q)
    out = rstd * (q - m1 - hat * m(q * hat))
    size = q.abs() + m(q.abs()) + hat.abs() * m((q * hat).abs())
    carried = eq + m(eq) + hat.abs() * m(hat.abs() * eq) + eh * m((q * hat).abs()) + hat.abs() * m(q.abs() * eh)
    return out, rstd * (K * C * size + 1.5 * carried), eh


def _backward(c, x_out, rms, res):
    M, E = c["y"].shape
    zero = torch.zeros(M, E, dtype=torch.float64)
    y, d = c["y"].double(), zero if c["dx_out"] is None else c["dx_out"].double()
    ed, out = zero.clone(), {}
    cols = lambda t, e: (t.sum(0), (e + (M + 4) * C * t.abs()).sum(0))
    if c["pre_gamma"] is not None:
        _, _, hat, rstd = _norm(x_out, zero, c["pre_gamma"], c["pre_beta"], rms)
        dh, g2 = c["dh"].double(), c["pre_gamma"].double()
        back, eb, eh = _norm_back(hat, rstd, x_out.abs().mean(1, keepdim=True), dh * g2, C * (dh * g2).abs(), rms)
        ed = eb + 2 * C * (d.abs() + back.abs())
        d = d + back
        out["d_pre_gamma"], out["d_pre_beta"] = cols(dh * hat, dh.abs() * eh), cols(dh, zero)
    n, en, hat, rstd = _norm(y, zero, c["post_gamma"], c["post_beta"], rms)
    gate = None if c["gate"] is None else c["gate"].abs()
    dn, edn = _gated(c["gate"], d), _gated(gate, ed + 2 * C * d.abs())
    if c["gate"] is not None:
        G = c["gate"].shape[0]
        t, e = d * n, d.abs() * en + ed * n.abs() + (M // G + 4) * C * (d * n).abs()
        out["d_gate"] = t.view(G, -1, E).sum(1), e.view(G, -1, E).sum(1)
    g1 = c["post_gamma"].double()
    dy, edy, eh = _norm_back(hat, rstd, y.abs().mean(1, keepdim=True), dn * g1, edn * g1.abs() + C * (dn * g1).abs(), rms)
    out["dy"] = dy, edy + (dy.abs() + edy) * _half(c["y"].dtype)
    out["dx"] = res * d, abs(res) * ed + C * (res * d).abs()
    out["d_post_gamma"], out["d_post_beta"] = cols(dn * hat, edn * hat.abs() + dn.abs() * eh), cols(dn, edn)
    return out


NAMES = ("dy", "dx", "d_post_gamma", "d_post_beta", "d_gate", "d_pre_gamma", "d_pre_beta")
THERE = {"d_post_beta": "post_beta", "d_gate": "gate", "d_pre_gamma": "pre_gamma", "d_pre_beta": "pre_beta"}


def _stats64(c, x_out, rms):
    """Statistics as a forward pass leaves them, rounded once."""
    out = []
    for t in (c["y"].double(), x_out.double()):
        mean = torch.zeros_like(t[:, 0]) if rms else t.mean(1)
        out += [mean, ((t - mean[:, None]).square().mean(1) + EPS).rsqrt()]
    return torch.stack(out, 1).float()


def _check_backward(c, got, x_out, rms, res):
    want = _backward(c, x_out.double(), rms, res)
    for name, t in zip(NAMES, got):
        if name in THERE and c[THERE[name]] is None:
            assert t is None
            continue
        w, tol = want[name]
        assert t.shape == w.shape
        off = (t.cpu().double() - w).abs()
        assert bool((off <= tol).all()), (name, float((off / (tol + 1e-300)).max()))


@gpu
@pytest.mark.parametrize("M,E", SHAPES + [(2051, 96), (6000, 40), (4100, 770)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rms", [False, True])
def test_backward(M, E, dt, rms):
    res = 0.875
    third = [g for g in (2, 3, 5, 7, 10, 60) if M % g == 0][:2]
    for G in sorted({0, 1, M, *third}):
        c = _case(M, E, dt, G, rms, gate_dt=dt if G == M else torch.float32)
        x_out = _forward(c, rms, res)[0].float()                  # any f32 rows will do as the saved residual stream
        g = _on_gpu(c)
        args = (g["dh"], g["dx_out"], g["y"], x_out.to(DEV), _stats64(c, x_out, rms).to(DEV), g["post_gamma"], g["post_beta"],
                g["gate"], g["pre_gamma"], g["pre_beta"])
        got = ops.gated_residual_norm_bwd(*args, res_scale=res, rms=rms)
        _check_backward(c, got, x_out, rms, res)
        again = ops.gated_residual_norm_bwd(*args, res_scale=res, rms=rms)
        assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, again))


@gpu
@pytest.mark.parametrize("pre,dxo", [(False, True), (True, False), (True, True)])
def test_backward_without_one_of_the_gradients(pre, dxo):
    c = _case(131, 768, torch.bfloat16, 1, False, pre=pre)
    if not dxo:
        c["dx_out"] = None
    x_out = _forward(c, False, 1.0)[0].float()
    g = _on_gpu(c)
    stats = _stats64(c, x_out, False).to(DEV)
    got = ops.gated_residual_norm_bwd(g["dh"], g["dx_out"], g["y"], x_out.to(DEV), stats, g["post_gamma"], g["post_beta"], g["gate"],
                                      g["pre_gamma"], g["pre_beta"])
    _check_backward(c, got, x_out, False, 1.0)


@gpu
@pytest.mark.parametrize("M,E", [(37, 768), (37, 771), (9000, 96)])
def test_backward_of_strided_rows(M, E):
    c = _case(M, E, torch.bfloat16, 1, False)
    x_out = _forward(c, False, 1.0)[0].float()
    g = _on_gpu(c)
    stats = _stats64(c, x_out, False).to(DEV)
    rest = (stats, g["post_gamma"], g["post_beta"], g["gate"], g["pre_gamma"], g["pre_beta"])
    want = ops.gated_residual_norm_bwd(g["dh"], g["dx_out"], g["y"], x_out.to(DEV), *rest)
    for first in (4, 3):                                          # 3: rows no aligned vector load fits
        def wide(t):
            w = torch.full((M, E + 12), float("nan"), dtype=t.dtype, device=DEV)
            w[:, first:first + E] = t.to(DEV)
            return w[:, first:first + E]
        got = ops.gated_residual_norm_bwd(wide(g["dh"]), wide(g["dx_out"]), wide(g["y"]), wide(x_out), *rest)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("G", [1, 5, 300])
def test_backward_adds_to_given_buffers(G):
    c = _case(300, 132, torch.float32, G, False)
    x_out = _forward(c, False, 1.0)[0].float().to(DEV)
    g = _on_gpu(c)
    args = (g["dh"], g["dx_out"], g["y"], x_out, _stats64(c, x_out.cpu(), False).to(DEV), g["post_gamma"], g["post_beta"], g["gate"],
            g["pre_gamma"], g["pre_beta"])
    fresh = ops.gated_residual_norm_bwd(*args)
    into = [torch.full_like(t, 2.0) for t in fresh[2:]]
    into[1] = None                                                # this one is returned fresh
    got = ops.gated_residual_norm_bwd(*args, into=into)
    for i, (f, t) in enumerate(zip(fresh[2:], got[2:])):
        if into[i] is None:
            assert torch.equal(t, f)
        else:
            assert t.data_ptr() == into[i].data_ptr() and torch.equal(t, f + 2.0)


@gpu
@pytest.mark.parametrize("rms", [False, True])
def test_backward_is_that_of_differences(rms):
    """Central differences of <dh, h> + <dx_out, x_out> in 64 bits against the kernel's gradients."""
    c = _case(6, 40, torch.float32, 3, rms)
    res = 0.75

    def loss(**moved):
        m = {**c, **moved}
        x_out, _, h, _ = _forward({k: v if v is None else v.double() for k, v in m.items()}, rms, res)
        return float((c["dh"].double() * h).sum() + (c["dx_out"].double() * x_out).sum())

    g = _on_gpu(c)
    x_out, _, stats = ops.gated_residual_norm(g["y"], g["x"], g["post_gamma"], g["post_beta"], g["gate"], g["pre_gamma"], g["pre_beta"],
                                              res_scale=res, rms=rms)
    got = ops.gated_residual_norm_bwd(g["dh"], g["dx_out"], g["y"], x_out, stats, g["post_gamma"], g["post_beta"], g["gate"],
                                      g["pre_gamma"], g["pre_beta"], res_scale=res, rms=rms)
    step = 1e-4
    for name, grad in zip(("y", "x", "post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta"), got):
        if c[name] is None:
            continue
        flat = c[name].double().reshape(-1)
        for i in (0, flat.numel() // 2, flat.numel() - 1):
            up, down = flat.clone(), flat.clone()
            up[i] += step
            down[i] -= step
            slope = (loss(**{name: up.view(c[name].shape)}) - loss(**{name: down.view(c[name].shape)})) / (2 * step)
            # third derivatives of order 10 times step^2 = 1e-7, f32 sums of order 10: 1e-5
            assert abs(slope - float(grad.reshape(-1)[i])) <= 2e-5 * max(1.0, abs(slope)), name


@gpu
def test_rows_that_are_constant_and_values_that_are_not_finite():
    """A constant row has deviation 0: rstd = 1 / sqrt(eps), the normalised row is 0.  A NaN stays in its own row."""
    c = _case(8, 256, torch.float32, 0, False)
    c["y"][2] = 0.25                                              # exact mean: powers of two
    c["y"][5, 7] = float("nan")
    g = _on_gpu(c)
    x_out, h, stats = ops.gated_residual_norm(g["y"], g["x"], g["post_gamma"], g["post_beta"], None, g["pre_gamma"], g["pre_beta"])
    assert torch.equal(x_out[2], g["x"][2] + g["post_beta"])
    assert bool(torch.isnan(x_out[5]).all()) and bool(torch.isnan(h[5]).all())
    keep = [0, 1, 2, 3, 4, 6, 7]
    assert bool(torch.isfinite(h[keep]).all()) and bool(torch.isfinite(x_out[keep]).all())


@gpu
def test_empty_and_refused_calls():
    c = _on_gpu(_case(6, 16, torch.float32, 3, False))
    none = torch.zeros(0, 16, device=DEV)
    x_out, h, stats = ops.gated_residual_norm(none, none, c["post_gamma"], None, None, c["pre_gamma"])
    assert x_out.shape == h.shape == (0, 16) and stats.shape == (0, 4)
    back = ops.gated_residual_norm_bwd(none, None, none, none, stats, c["post_gamma"], None, None, c["pre_gamma"])
    assert back[0].shape == (0, 16) and torch.equal(back[2], torch.zeros(16, device=DEV))
    call = lambda **k: ops.gated_residual_norm(**{**{n: c[n] for n in ("y", "x", "post_gamma", "post_beta", "gate", "pre_gamma",
                                                                       "pre_beta")}, **k})
    call()
    for bad in (dict(gate=torch.ones(4, 16, device=DEV)), dict(gate=torch.ones(3, 15, device=DEV)), dict(x=c["x"][:5]),
                dict(x=c["x"].bfloat16()), dict(post_gamma=c["post_gamma"][:8]), dict(pre_gamma=None), dict(y=c["y"].t())):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(y=c["y"].half()), dict(gate=c["gate"].bfloat16()), dict(post_gamma=c["post_gamma"].double())):
        with pytest.raises(TypeError):
            call(**bad)
    with pytest.raises(_lib.HipLibraryError):
        ops.gated_residual_norm(torch.zeros(1, 8193, device=DEV), torch.zeros(1, 8193, device=DEV), torch.ones(8193, device=DEV))


def test_refusals_without_a_gpu():
    lib, one = _lib.load(), 1 << 12
    fwd = lambda dt=0, y=one, ldy=8, x=one, gdt=0, gate=one, G=2, pre=one, h=one, stats=one, M=4, E=8: lib.tc_gated_residual_norm_fwd(
        dt, y, ldy, x, 8, one, one, gdt, gate, G, 1.0, pre, None, one, h, stats, M, E, 0, 1e-5, 1e-5, None)
    for bad in (dict(dt=2), dict(y=None), dict(ldy=7), dict(x=one + 2), dict(gdt=1), dict(gate=None), dict(G=3), dict(G=0), dict(h=None),
                dict(pre=None), dict(stats=one + 4), dict(M=0), dict(E=0), dict(E=8193)):
        assert fwd(**bad) == -1, bad
    need = lib.tc_gated_residual_norm_bwd_workspace_bytes(4, 8, 2)
    assert need > 0 and lib.tc_gated_residual_norm_bwd_workspace_bytes(4, 8, 3) == 0
    bwd = lambda dh=one, dxo=one, pre=one, d_gate=one, ws=one, n=need, ldy=8: lib.tc_gated_residual_norm_bwd(
        0, dh, 8, dxo, 8, one, ldy, one, 8, one, one, one, 0, one, 2, 1.0, pre, one, one, one, one, d_gate, pre, None, 0, 4, 8, 0, ws, n,
        None)
    for bad in (dict(dh=None), dict(pre=None), dict(dh=None, pre=None, dxo=None), dict(d_gate=None), dict(ws=None), dict(ws=one + 4),
                dict(ldy=4)):
        assert bwd(**bad) == -1, bad
    assert bwd(n=need - 1) == -3


def test_gradients_that_overlap_are_refused_without_a_gpu():
    """Two sums into one buffer would lose one of them (one parameter for both norms, say)."""
    lib, one = _lib.load(), 1 << 12
    need = lib.tc_gated_residual_norm_bwd_workspace_bytes(4, 8, 2)

    def bwd(d_post_gamma, d_post_beta, d_pre_gamma, d_pre_beta, d_gate):
        return lib.tc_gated_residual_norm_bwd(0, one, 8, one, 8, one, 8, one, 8, one, one, one, 0, one, 2, 1.0, one, one, one,
                                              d_post_gamma, d_post_beta, d_gate, d_pre_gamma, d_pre_beta, 31, 4, 8, 0, one, need, None)

    far = [one * 2, one * 3, one * 4, one * 5, one * 6]
    for a in range(5):
        for b in range(5):
            if a == b:
                continue
            bad = list(far)
            bad[a] = bad[b]
            assert bwd(*bad) == -1, (a, b)
            bad[a] = bad[b] + 28                                  # the last of eight values
            assert bwd(*bad) == -1, (a, b)
    for a in range(4):                                            # into the gate's second row
        bad = list(far)
        bad[a] = far[4] + 32
        assert bwd(*bad) == -1, a


@gpu
def test_backward_refuses_one_buffer_for_two_gradients():
    c = _on_gpu(_case(6, 16, torch.float32, 0, False))
    x_out, h, stats = ops.gated_residual_norm(c["y"], c["x"], c["post_gamma"], None, None, c["pre_gamma"])
    call = lambda into: ops.gated_residual_norm_bwd(c["dh"], c["dx_out"], c["y"], x_out, stats, c["post_gamma"], None, None,
                                                    c["pre_gamma"], None, into=into)
    shared = torch.zeros(16, device=DEV)
    with pytest.raises(_lib.HipLibraryError, match="overlap"):
        call([shared, None, None, shared, None])
    with pytest.raises(ValueError):
        call([shared])
    next_to = torch.zeros(2, 16, device=DEV)
    got, fresh = call([next_to[0], None, None, next_to[1], None]), call(None)
    assert torch.equal(got[2], fresh[2]) and torch.equal(got[5], fresh[5])


@gpu
@pytest.mark.parametrize("E", [3, 6, 300, 515, 766, 768, 1022, 1030, 2048, 2053, 4096, 4098, 8000, 8190, 8192])
@pytest.mark.parametrize("second", [True, False])
def test_results_in_place_of_the_residual_stream(E, second):
    """x_out may be x, and dx may be dx_out: a row's last columns may be read by two lanes, in two waves."""
    M, lib = 700, _lib.load()
    c = _on_gpu(_case(M, E, torch.bfloat16, 7, False))
    pre = (c["pre_gamma"], c["pre_beta"]) if second else (None, None)
    dh = c["dh"] if second else None
    P = lambda t: None if t is None else t.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    x_out, h, stats = ops.gated_residual_norm(c["y"], c["x"], c["post_gamma"], c["post_beta"], c["gate"], *pre, res_scale=0.5)
    want = ops.gated_residual_norm_bwd(dh, c["dx_out"], c["y"], x_out, stats, c["post_gamma"], c["post_beta"], c["gate"], *pre,
                                       res_scale=0.5)
    need = lib.tc_gated_residual_norm_bwd_workspace_bytes(M, E, 7)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    for _ in range(3):
        x, d, h2, stats2, dy = c["x"].clone(), c["dx_out"].clone(), torch.empty_like(c["y"]), torch.empty_like(stats), torch.empty_like(c["y"])
        assert lib.tc_gated_residual_norm_fwd(1, P(c["y"]), E, P(x), E, P(c["post_gamma"]), P(c["post_beta"]), 0, P(c["gate"]), 7, 0.5, P(pre[0]),
                                              P(pre[1]), P(x), P(h2) if second else None, P(stats2), M, E, 0, 1e-5, 1e-5, stream) == 0
        assert torch.equal(x, x_out) and torch.equal(stats2, stats) and (not second or torch.equal(h2, h))
        grads = [torch.empty_like(t) for t in want[2:] if t is not None]
        g = grads + [None] * (5 - len(grads))
        assert lib.tc_gated_residual_norm_bwd(1, P(dh), E, P(d), E, P(c["y"]), E, P(x_out), E, P(stats), P(c["post_gamma"]), P(c["post_beta"]), 0,
                                              P(c["gate"]), 7, 0.5, P(pre[0]), P(dy), P(d), P(g[0]), P(g[1]), P(g[2]), P(g[3]), P(g[4]), 0, M, E, 0,
                                              P(ws), need, stream) == 0
        for a, b in zip([dy, d, *grads], [t for t in want if t is not None]):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("E", [1, 2, 3, 5, 257, 513, 769, 1025, 2049, 4097, 8191])
@pytest.mark.parametrize("G", [0, 1, 5, 40])
def test_a_row_end_behind_the_last_whole_piece(E, G):
    """The columns that two lanes hold count once in every sum."""
    c = _case(40, E, torch.float32, G, False)
    g = _on_gpu(c)
    x_out, h, stats = ops.gated_residual_norm(g["y"], g["x"], g["post_gamma"], g["post_beta"], g["gate"], g["pre_gamma"], g["pre_beta"])
    got = ops.gated_residual_norm_bwd(g["dh"], g["dx_out"], g["y"], x_out, stats, g["post_gamma"], g["post_beta"], g["gate"], g["pre_gamma"],
                                      g["pre_beta"])
    into = [None if t is None else torch.ones_like(t) for t in got[2:]]
    again = ops.gated_residual_norm_bwd(g["dh"], g["dx_out"], g["y"], x_out, stats, g["post_gamma"], g["post_beta"], g["gate"], g["pre_gamma"],
                                        g["pre_beta"], into=into)
    for a, b in zip(got[2:], again[2:]):
        assert a is None and b is None or torch.equal(a + 1.0, b)
    # a gradient of beta is a plain sum over the rows of dh: 40 values of size up to 4, f32
    assert float((got[6].double().cpu() - c["dh"].double().sum(0)).abs().max()) <= 40 * 4 * 40 * 2.0 ** -24


@gpu
@pytest.mark.parametrize("E", [1, 3, 5, 255, 514, 769, 1025, 2050, 4099, 8191])
@pytest.mark.parametrize("first", [0, 1])
def test_what_lies_around_the_results_is_left_as_it_was(E, first):
    """Dense results at any address, guards of 64 values on both sides."""
    M, G, lib = 30, 5, _lib.load()
    c = _on_gpu(_case(M, E, torch.bfloat16, G, False))
    guards = []

    def result(*shape, dtype=torch.float32):
        size = torch.Size(shape).numel()
        buf = torch.full((size + 129,), 7.0, dtype=dtype, device=DEV)
        guards.append((buf, 64 + first, 64 + first + size))
        return buf[64 + first:64 + first + size].view(shape)

    P = lambda t: t.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    x_out, h, stats = result(M, E), result(M, E, dtype=torch.bfloat16), torch.empty(M, 4, device=DEV)
    assert lib.tc_gated_residual_norm_fwd(1, P(c["y"]), E, P(c["x"]), E, P(c["post_gamma"]), P(c["post_beta"]), 0, P(c["gate"]), G, 1.0,
                                          P(c["pre_gamma"]), P(c["pre_beta"]), P(x_out), P(h), P(stats), M, E, 0, 1e-5, 1e-5, stream) == 0
    want = ops.gated_residual_norm(c["y"], c["x"], c["post_gamma"], c["post_beta"], c["gate"], c["pre_gamma"], c["pre_beta"])
    assert torch.equal(x_out, want[0]) and torch.equal(h, want[1]) and torch.equal(stats, want[2])
    dy, dx, d_gate, vectors = result(M, E, dtype=torch.bfloat16), result(M, E), result(G, E), [result(E) for _ in range(4)]
    need = lib.tc_gated_residual_norm_bwd_workspace_bytes(M, E, G)
    ws = torch.full((need + 64,), 77, dtype=torch.uint8, device=DEV)
    assert lib.tc_gated_residual_norm_bwd(1, P(c["dh"]), E, P(c["dx_out"]), E, P(c["y"]), E, P(x_out), E, P(stats), P(c["post_gamma"]),
                                          P(c["post_beta"]), 0, P(c["gate"]), G, 1.0, P(c["pre_gamma"]), P(dy), P(dx), P(vectors[0]),
                                          P(vectors[1]), P(d_gate), P(vectors[2]), P(vectors[3]), 0, M, E, 0, P(ws), need, stream) == 0
    back = ops.gated_residual_norm_bwd(c["dh"], c["dx_out"], c["y"], want[0], stats, c["post_gamma"], c["post_beta"], c["gate"],
                                       c["pre_gamma"], c["pre_beta"])
    for a, b in zip([dy, dx, vectors[0], vectors[1], d_gate, vectors[2], vectors[3]], back):
        assert torch.equal(a, b)
    assert bool((ws[need:] == 77).all())
    for buf, begin, end in guards:
        assert bool((buf[:begin] == 7.0).all()) and bool((buf[end:] == 7.0).all())


# ---- every layout of rows over waves ----------------------------------------------------------------
# The kernels exist for (waves a row, loads a lane), each for aligned rows and for any rows.  Widths and row counts below reach all of
# them in both directions; the tolerances are those above (a row sum of at most 16 waves: 8 additions in a lane, 6 across a
# wave, 16 across waves, or of one wave 16 and 6: below K).
def _shape(M, E, backward):
    """(waves, loads of four columns a lane) as the dispatch takes them."""
    if backward and 512 < E <= 768 and M < 8192:
        return 3, 1
    W = 1 if E <= ((768 if M >= 8192 else 512) if backward else 1024) else 4
    if W > 1:
        for more in (5, 6, 8, 10, 12, 16):
            if E > 512 * W:
                W = more
    return W, -(-E // (256 * W))


FEW_ROWS = [(5, E) for E in (96, 255, 260, 511, 600, 767, 1000, 1023, 1500, 1501, 2304, 2305, 2820, 3001, 3500, 3501, 5000, 5001, 6000,
                             6143, 7000, 8191)]
MANY_ROWS = [(8192, 768), (8195, 766), (8200, 600)]


def test_every_layout_is_tested_without_a_gpu():
    source = open(os.path.join(os.path.dirname(_lib.__file__), "csrc", "gated_norm.hip")).read()
    common, fwd, bwd = (source[source.index(f"#define {n}("):].split("\n\n")[0].split("#define")[1] for n in
                        ("TC_GN_COMMON", "TC_GN_FWD", "TC_GN_BWD"))
    built = lambda text: {(int(w), int(n)) for w, n in re.findall(r"TC_GN\(T, TG, LOOSE, (\d+), (\d+)\)", text)}
    for backward, text in ((False, fwd), (True, bwd)):
        there = built(common) | built(text)
        reached = {_shape(M, E, backward) for M in (1, 700, 8191, 8192) for E in range(4, 8193)}
        assert reached == there                                   # nothing is built that no call takes, nothing falls to the default
        for loose in (False, True):
            tested = {_shape(M, E, backward) for M, E in FEW_ROWS + MANY_ROWS if (E % 4 != 0) == loose}
            assert tested == there, (backward, loose, there - tested)


def _both_directions(M, E, dt, G, rms, gate_dt):
    res = 0.875
    c = _case(M, E, dt, G, rms, gate_dt=gate_dt)
    want_x, ex, want_h, eh = _forward(c, rms, res)
    g = _on_gpu(c)
    x_out, h, _ = ops.gated_residual_norm(g["y"], g["x"], g["post_gamma"], g["post_beta"], g["gate"], g["pre_gamma"], g["pre_beta"],
                                          res_scale=res, rms=rms)
    assert bool(((x_out.cpu().double() - want_x).abs() <= ex).all())
    assert bool(((h.cpu().double() - want_h).abs() <= eh).all())
    x_out = want_x.float()
    args = (g["dh"], g["dx_out"], g["y"], x_out.to(DEV), _stats64(c, x_out, rms).to(DEV), g["post_gamma"], g["post_beta"], g["gate"],
            g["pre_gamma"], g["pre_beta"])
    got = ops.gated_residual_norm_bwd(*args, res_scale=res, rms=rms)
    _check_backward(c, got, x_out, rms, res)
    again = ops.gated_residual_norm_bwd(*args, res_scale=res, rms=rms)
    assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, again))


@gpu
@pytest.mark.parametrize("M,E", FEW_ROWS)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rms", [False, True])
def test_every_width_class(M, E, dt, rms):
    for G, gate_dt in ((0, torch.float32), (1, dt), (M, torch.float32), (M, dt)):
        _both_directions(M, E, dt, G, rms, gate_dt)


@gpu
@pytest.mark.parametrize("M,E,G,rms", [(8192, 768, 0, False), (8192, 768, 64, False), (8192, 768, 8192, True), (8195, 766, 1, False),
                                       (8195, 766, 5, True), (8195, 766, 8195, False), (8200, 600, 0, True), (8200, 600, 8, False),
                                       (8200, 600, 4100, False)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_many_rows_of_one_wave_each(M, E, G, rms, dt):
    _both_directions(M, E, dt, G, rms, dt if G == M else torch.float32)


@gpu
@pytest.mark.parametrize("M,E", [(700, E) for _, E in FEW_ROWS if E > 1024] + MANY_ROWS + [(8192, 511)])
@pytest.mark.parametrize("second", [True, False])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_results_in_place_in_every_layout(M, E, second, dt):
    """x_out may be x, and dx may be dx_out."""
    G, lib = 5 if M % 5 == 0 else 64, _lib.load()
    c = _on_gpu(_case(M, E, dt, G, False))
    pre = (c["pre_gamma"], c["pre_beta"]) if second else (None, None)
    dh = c["dh"] if second else None
    P = lambda t: None if t is None else t.data_ptr()
    code, stream = int(dt == torch.bfloat16), torch.cuda.current_stream().cuda_stream
    x_out, h, stats = ops.gated_residual_norm(c["y"], c["x"], c["post_gamma"], c["post_beta"], c["gate"], *pre, res_scale=0.5)
    want = ops.gated_residual_norm_bwd(dh, c["dx_out"], c["y"], x_out, stats, c["post_gamma"], c["post_beta"], c["gate"], *pre,
                                       res_scale=0.5)
    need = lib.tc_gated_residual_norm_bwd_workspace_bytes(M, E, G)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    x, d, h2, stats2, dy = c["x"].clone(), c["dx_out"].clone(), torch.empty_like(c["y"]), torch.empty_like(stats), torch.empty_like(c["y"])
    assert lib.tc_gated_residual_norm_fwd(code, P(c["y"]), E, P(x), E, P(c["post_gamma"]), P(c["post_beta"]), 0, P(c["gate"]), G, 0.5, P(pre[0]),
                                          P(pre[1]), P(x), P(h2) if second else None, P(stats2), M, E, 0, 1e-5, 1e-5, stream) == 0
    assert torch.equal(x, x_out) and torch.equal(stats2, stats) and (not second or torch.equal(h2, h))
    grads = [torch.empty_like(t) for t in want[2:] if t is not None]
    g = grads + [None] * (5 - len(grads))
    assert lib.tc_gated_residual_norm_bwd(code, P(dh), E, P(d), E, P(c["y"]), E, P(x_out), E, P(stats), P(c["post_gamma"]), P(c["post_beta"]), 0,
                                          P(c["gate"]), G, 0.5, P(pre[0]), P(dy), P(d), P(g[0]), P(g[1]), P(g[2]), P(g[3]), P(g[4]), 0, M, E, 0,
                                          P(ws), need, stream) == 0
    for a, b in zip([dy, d, *grads], [t for t in want if t is not None]):
        assert torch.equal(a, b)
