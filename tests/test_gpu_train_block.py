"""The training-block operators together, as a block's forward and backward pass use them: embedding lookup, feed-forward block with
8-bit checkpoints, norms with gate and residual scale; on another stream, in a captured graph, and past 32-bit offsets."""
import pytest
import torch

from transcodon_amd import _lib, ops

DEV = "cuda"
pytestmark = pytest.mark.gpu
B, T, E, F, V = 3, 67, 256, 512, 37
RES, SCALE = 0.9, 16.0


def _weights(seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    tok = torch.randint(0, V, (B, T), generator=gen)
    tok[1, 50:] = 1                                               # padding
    w = dict(table=r(V, E) * 0.06, g0=1 + 0.1 * r(E), b0=0.1 * r(E), W1=(r(F, E) * E ** -0.5).bfloat16(), c1=0.1 * r(F),
             W2=(r(E, F) * F ** -0.5).bfloat16(), c2=0.1 * r(E), g1=1 + 0.1 * r(E), b1=0.1 * r(E), gate=0.5 + 0.2 * r(B, E),
             g2=1 + 0.1 * r(E), b2=0.1 * r(E), dh=r(B * T, E).bfloat16(), dx=r(B * T, E))
    return tok, w


def _forward(tok, w):
    s = {}
    s["x0"] = ops.embedding(tok, w["table"], SCALE, pad_idx=1)
    h0 = ops.layernorm(s["x0"], w["g0"], w["b0"], out_dtype=torch.bfloat16)
    s["h0"] = ops.act8_pack(h0)
    u = ops.gemm(h0, w["W1"], w["c1"])
    act, *s["u"] = ops.gelu_act8(u)
    s["y"] = ops.gemm(act, w["W2"], w["c2"])
    s["x1"], h1, s["stats"] = ops.gated_residual_norm(s["y"], s["x0"], w["g1"], w["b1"], w["gate"], w["g2"], w["b2"], res_scale=RES)
    return h1, s


def _backward(tok, w, s):
    dy, dx0, d_g1, d_b1, d_gate, d_g2, d_b2 = ops.gated_residual_norm_bwd(
        w["dh"], w["dx"], s["y"], s["x1"], s["stats"], w["g1"], w["b1"], w["gate"], w["g2"], w["b2"], res_scale=RES)
    none = torch.zeros(F, device=DEV), torch.zeros(E, device=DEV)
    d_act = ops.gemm(dy, w["W2"].t().contiguous(), none[0])
    du, act = ops.dgelu_act8(d_act, *s["u"], want_act=True)
    dW2 = ops.gemm_tn(dy, act)[0]
    dW1 = ops.gemm_tn_act8(du, *s["h0"])
    d_h0 = ops.gemm(du, w["W1"].t().contiguous(), none[1])
    d_g0, d_b0 = torch.zeros(E, device=DEV), torch.zeros(E, device=DEV)
    ops.layernorm_bwd(s["x0"], w["g0"], d_h0, d_g0, d_b0, dx=dx0, accumulate=True)
    d_table = ops.embedding_bwd(tok, dx0, V, SCALE, pad_idx=1)
    return dict(d_table=d_table, dW1=dW1, dW2=dW2, d_g0=d_g0, d_b0=d_b0, d_g1=d_g1, d_b1=d_b1, d_gate=d_gate, d_g2=d_g2, d_b2=d_b2)


def _reference(tok, w):
    """The same block in 64 bits by autograd; rounding to 8 bits passes its gradient through, and is what the weight gradient and
    gelu' see."""
    p = {k: v.double().requires_grad_() for k, v in w.items() if k not in ("dh", "dx")}
    ln = lambda t, g, b: (t - t.mean(1, keepdim=True)) * ((t - t.mean(1, keepdim=True)).square().mean(1, keepdim=True) + 1e-5).rsqrt() * g + b
    x0 = p["table"][tok.view(-1)] * SCALE * (tok.view(-1, 1) != 1)
    h0 = ln(x0, p["g0"], p["b0"])

    def eight(t):
        g = t.detach().view(t.shape[0], -1, 32)
        unit = torch.exp2(torch.ceil(torch.log2(g.abs().amax(2, keepdim=True) / 448)).clamp(min=-126))
        return ((g / unit).float().to(torch.float8_e4m3fn).double() * unit).view(t.shape)

    class Linear8(torch.autograd.Function):       # weight gradient from the 8-bit input
        @staticmethod
        def forward(ctx, t, W):
            ctx.save_for_backward(eight(t), W)
            return t @ W.t()

        @staticmethod
        def backward(ctx, d):
            t8, W = ctx.saved_tensors
            return d @ W, d.t() @ t8

    class Gelu8(torch.autograd.Function):         # gelu' at the 8-bit input
        @staticmethod
        def forward(ctx, t):
            ctx.save_for_backward(eight(t))
            return torch.nn.functional.gelu(t)

        @staticmethod
        def backward(ctx, d):
            with torch.enable_grad():
                t8 = ctx.saved_tensors[0].requires_grad_()
                return torch.autograd.grad(torch.nn.functional.gelu(t8), t8, d)[0]

    class LinearOf(torch.autograd.Function):      # second product: its weight gradient sees gelu of the 8-bit input
        @staticmethod
        def forward(ctx, t, W, again):
            ctx.save_for_backward(again, W)
            return t @ W.t()

        @staticmethod
        def backward(ctx, d):
            again, W = ctx.saved_tensors
            return d @ W, d.t() @ again, None

    u = Linear8.apply(h0, p["W1"]) + p["c1"]
    y = LinearOf.apply(Gelu8.apply(u), p["W2"], torch.nn.functional.gelu(eight(u))) + p["c2"]
    n = ln(y, p["g1"], p["b1"])
    x1 = RES * x0 + (p["gate"][:, None] * n.view(B, T, E)).view(-1, E)
    h1 = ln(x1, p["g2"], p["b2"])
    ((h1 * w["dh"].double()).sum() + (x1 * w["dx"].double()).sum()).backward()
    names = dict(d_table="table", dW1="W1", dW2="W2", d_g0="g0", d_b0="b0", d_g1="g1", d_b1="b1", d_gate="gate", d_g2="g2", d_b2="b2")
    return h1.detach(), {k: p[v].grad for k, v in names.items()}


def test_forward_and_backward_of_a_block():
    tok, w = _weights()
    want_h, want = _reference(tok, w)
    g = {k: v.to(DEV) for k, v in w.items()}
    h1, s = _forward(tok.to(DEV), g)
    got = _backward(tok.to(DEV), g, s)
    # bf16 rounds h0, u, act, y, h1 on the way forward and d_act, du, d_h0 back: each by at most 2^-8 of its value, and a value that
    # falls on the other side of an e4m3 border moves by 2^-3 (one in 2^-8 / 2^-4 of them): in the 2-norm below 9 * 2^-8
    off = lambda a, b: float((a.cpu().double() - b).norm() / b.norm())
    assert off(h1, want_h) < 9 * 2.0 ** -8
    for k, t in got.items():
        assert t.shape == want[k].shape
        assert off(t, want[k]) < 9 * 2.0 ** -8, (k, off(t, want[k]))


NEW = ("dW1", "d_table", "d_g1", "d_b1", "d_gate", "d_g2", "d_b2")         # (the LayerNorm gradient in between adds with atomics)


def _new_only(tok, w, s):
    """Outputs of the operators under test alone: the same bits every time."""
    dy, dx0, *vec = ops.gated_residual_norm_bwd(w["dh"], w["dx"], s["y"], s["x1"], s["stats"], w["g1"], w["b1"], w["gate"], w["g2"],
                                                w["b2"], res_scale=RES)
    d_act = ops.gemm(dy, w["W2"].t().contiguous(), w["c1"])
    du, act = ops.dgelu_act8(d_act, *s["u"], want_act=True)
    return [dy, dx0, *vec, du, act, ops.gemm_tn_act8(du, *s["h0"]), ops.act8_unpack(*s["h0"]), ops.embedding_bwd(tok, dx0, V, SCALE, pad_idx=1)]


def test_on_another_stream():
    tok, w = _weights(1)
    tok, w = tok.to(DEV), {k: v.to(DEV) for k, v in w.items()}
    h1, s = _forward(tok, w)
    want = [h1, *_new_only(tok, w, s)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        h2, s2 = _forward(tok, w)
        got = [h2, *_new_only(tok, w, s2)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_captured_graphs_replayed():
    """Two graphs of the same calls on different inputs, replayed in turn with eager work between; every replay is checked."""
    cases = []
    for seed in (2, 3):
        tok, w = _weights(seed)
        tok, w = tok.to(DEV), {k: v.to(DEV) for k, v in w.items()}
        h1, s = _forward(tok, w)                                  # also what a program does before it captures
        want = [t.clone() for t in (h1, *_new_only(tok, w, s))]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            h1, s = _forward(tok, w)
            got = [h1, *_new_only(tok, w, s)]
        cases.append((graph, got, want, tok, w))                  # a graph reads its inputs where they were
    for turn in range(4):
        for graph, got, want, *_ in (cases if turn % 2 else cases[::-1]):
            for t in got:
                t.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
            ops.gelu_act8(torch.randn(300, 320, device=DEV))     # eager work of the same operators
            ops.embedding_bwd(torch.zeros(5000, dtype=torch.int64, device=DEV), torch.randn(5000, 64, device=DEV), 9)


def test_many_positions_in_a_captured_graph():
    """The sorted form of the embedding gradient: counts and partial rows of one replay must not reach the next."""
    tok = torch.randint(0, 700, (20000,), device=DEV)
    dy = torch.randn(20000, 96, device=DEV)
    want = ops.embedding_bwd(tok, dy, 700)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.embedding_bwd(tok, dy, 700)
    for seed in range(3):
        graph.replay()
        assert torch.equal(got, want)
        tok.copy_(torch.randint(0, 700 if seed % 2 else 5, (20000,), device=DEV))
        want = ops.embedding_bwd(tok, dy, 700)


PERIOD = 1009


def _periodic(rows, width, dtype):
    base = torch.randn(PERIOD, width, device=DEV, dtype=torch.float32).to(dtype)
    return base, base.repeat(-(-rows // PERIOD), 1)[:rows]


def test_offsets_past_32_bits():
    """Rows repeat with a period; what comes out behind 2^31 elements (2^32 for bytes) must repeat as well."""
    width, rows = 4096, 2 ** 20 + 4097
    last = (rows - PERIOD) // PERIOD * PERIOD                     # a whole period near the end
    base, u = _periodic(rows, width, torch.bfloat16)
    act, codes, scales = ops.gelu_act8(u)
    want = ops.gelu_act8(base)
    for a, b in zip((act, codes, scales), want):
        assert torch.equal(a[last:last + PERIOD].view(torch.uint8), b.view(torch.uint8))
    du, again = ops.dgelu_act8(act, codes, scales, want_act=True)
    want = ops.dgelu_act8(want[0], *want[1:], want_act=True)
    assert torch.equal(du[last:last + PERIOD], want[0]) and torch.equal(again[last:last + PERIOD], want[1])
    del du, again
    # weight gradient of the last rows alone: all others are zero
    dy = torch.zeros(rows, 8, dtype=torch.bfloat16, device=DEV)
    dy[-70:] = torch.randn(70, 8, device=DEV).bfloat16()
    got = ops.gemm_tn_act8(dy, codes, scales)
    want = dy[-70:].double().t() @ (codes[-70:].float() * scales[-70:].float().repeat_interleave(32, 1)).double()
    assert float((got.double() - want).abs().max()) < 1e-4
    wide = torch.zeros(rows, width, dtype=torch.bfloat16, device=DEV)
    wide[-70:, :8] = dy[-70:]
    got = ops.gemm_tn_act8(wide, codes[:, :64].contiguous(), scales[:, :2].contiguous())
    assert float((got[:8].double() - want[:, :64]).abs().max()) < 1e-4 and bool((got[8:] == 0).all())
    del act, codes, scales, wide
    torch.cuda.empty_cache()
    # norms: the same rows as y and, in f32, as the residual stream
    x = u.float()
    ones = torch.ones(width, device=DEV)
    x_out, h, stats = ops.gated_residual_norm(u, x, ones, ones, ones, ones, ones)
    want = ops.gated_residual_norm(base, base.float(), ones, ones, ones, ones, ones)
    for a, b in zip((x_out, h, stats), want):
        assert torch.equal(a[last:last + PERIOD], b)
    del x
    dy, dx, *_ = ops.gated_residual_norm_bwd(h, x_out, u, x_out, stats, ones, ones, ones, ones, ones)
    back = ops.gated_residual_norm_bwd(want[1], want[0], base, want[0], want[2], ones, ones, ones, ones, ones)
    assert torch.equal(dy[last:last + PERIOD], back[0]) and torch.equal(dx[last:last + PERIOD], back[1])
    del x_out, h, dy, dx
    torch.cuda.empty_cache()
    # lookup, and a gradient that comes from the last rows only
    tok = (torch.arange(rows, device=DEV) % PERIOD)
    out = ops.embedding(tok, base, out_dtype=torch.bfloat16)
    assert torch.equal(out[last:last + PERIOD], base)
    del out
    grad = ops.embedding_bwd(torch.where(torch.arange(rows, device=DEV) < rows - 7, torch.ones_like(tok), tok), u, PERIOD, pad_idx=1)
    want = torch.zeros(PERIOD, width, device=DEV)
    want.index_add_(0, tok[-7:], u[-7:].float())
    want[1] = 0
    assert torch.equal(grad, want)


def test_tensors_on_the_cpu_are_refused():
    x = torch.zeros(4, 32)
    for call in (lambda: ops.act8_pack(x), lambda: ops.gelu_act8(x), lambda: ops.gated_residual_norm(x, x, torch.ones(32)),
                 lambda: ops.embedding_bwd(torch.zeros(4, dtype=torch.int64), x, 3)):
        with pytest.raises(_lib.HipLibraryError):
            call()
