"""Cases and plain forms of the training-block operators: embedding lookup with scaling and its gradient by
sorted tokens, a block's two norms with gate and residual scale, and 8-bit activation checkpoints.

With ``own`` false, ``run`` computes an operator from elementary torch operations; with ``own`` true it makes the
calls that a program makes of ``transcodon_amd.ops``.  Both take what ``prepare`` returns.
"""

import math

import torch

own = False

GROUP = 32            # values that share one scale of an 8-bit checkpoint
PAD = 1               # <pad> of the nucleotide alphabet


def listed():
    return [
        # one species row for a single sequence: the smallest lookup, all latency
        dict(name="embedding-one", op="embedding", rows=1, vocab=1438, width=768, dtype="f32", ids=32, pad=0.0),
        # the tokens of one training batch (64 sequences of 1024) over the 10 nucleotide symbols, padded tails
        dict(name="embedding-batch", op="embedding", rows=65536, vocab=10, width=768, dtype="f32", ids=32, pad=0.1),
        # gradient of the species table for one batch of sequences: few rows, all others zero
        dict(name="embedding-grad-species", op="embedding_bwd", rows=64, vocab=1438, width=768, dtype="f32", ids=32, pad=0.0),
        # gradient of the nucleotide table: every symbol has thousands of rows
        dict(name="embedding-grad-bases", op="embedding_bwd", rows=65536, vocab=10, width=768, dtype="f32", ids=32, pad=0.1),
        # a word-sized vocabulary with a few frequent and many rare tokens, 64-bit ids, an odd token count
        dict(name="embedding-grad-words", op="embedding_bwd", rows=49153, vocab=50021, width=1024, dtype="bf16", ids=64, pad=0.1),
        # one sequence through the end of a block in full precision, one learned gate for all rows
        dict(name="norm-one-sequence", op="norm", rows=131, width=768, dtype="f32", gates=1, rms=False),
        # a training batch, one gate vector for each of its 64 sequences
        dict(name="norm-batch", op="norm", rows=65536, width=768, dtype="bf16", gates=64, rms=False),
        # a ragged width that no vector load divides, root-mean-square norms, a gate for each of three sequences
        dict(name="norm-grad-odd", op="norm_bwd", rows=4101, width=770, dtype="f32", gates=3, rms=True),
        # the gradient for the same training batch
        dict(name="norm-grad-batch", op="norm_bwd", rows=65536, width=768, dtype="bf16", gates=64, rms=False),
        # activation of a feed-forward block, forward and backward through the 8-bit checkpoint of its input
        dict(name="act8-gelu-batch", op="act8_gelu", rows=32768, width=4096, dtype="bf16"),
        # weight gradient of the output projection for two sequences of one batch row of 131 tokens
        dict(name="act8-wgrad-short", op="act8_wgrad", rows=262, out=768, width=768),
        # weight gradient of the stacked q/k/v projection for a training batch, its input kept in 8 bits
        dict(name="act8-wgrad-batch", op="act8_wgrad", rows=65536, out=2304, width=768),
    ]


def _between(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embedding", "embedding_bwd", "norm", "norm_bwd", "act8_gelu", "act8_wgrad"])
    dtype = rng.choice(["f32", "bf16"])
    if op in ("embedding", "embedding_bwd"):
        width = _between(rng, 8, 4096)
        if rng.random() < 0.7:
            width = -(-width // 8) * 8
        return dict(op=op, rows=_between(rng, 1, min(65536, 50331648 // width)), vocab=_between(rng, 2, min(65536, 50331648 // width)),
                    width=width, dtype=dtype, ids=rng.choice([32, 64]), pad=rng.choice([0.0, 0.1, 0.5]))
    if op in ("norm", "norm_bwd"):
        width = _between(rng, 8, 8192)
        if rng.random() < 0.7:
            width = -(-width // 8) * 8
        gates = rng.choice([0, 1, _between(rng, 2, 64), -1])          # -1: a gate row for each row
        rows = _between(rng, 1, min(65536, 50331648 // width))
        if gates > 1:
            rows = max(1, rows // gates) * gates
            if rows * width > 50331648:
                gates, rows = 1, 50331648 // width
        return dict(op=op, rows=rows, width=width, dtype=dtype, gates=rows if gates < 0 else gates, rms=rng.random() < 0.5)
    if op == "act8_gelu":
        width = _between(rng, 8, 8192)
        if rng.random() < 0.7:
            width = -(-width // 8) * 8
        return dict(op=op, rows=_between(rng, 1, min(65536, (134217728 if dtype == "bf16" else 67108864) // width)), width=width, dtype=dtype)
    out, width = 8 * _between(rng, 1, 512), 16 * _between(rng, 1, 256)
    return dict(op=op, rows=_between(rng, 1, min(65536, 115964116992 // (out * width), 134217728 // max(out, width))), out=out, width=width)


_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _tokens(case, gen):
    """Ids that a few rows share often and many rarely (even over a handful of symbols), and <pad> at the end."""
    rows, vocab = case["rows"], case["vocab"]
    u = torch.rand(rows, generator=gen, device="cuda", dtype=torch.float64)
    ids = (u * vocab) if vocab < 64 else torch.exp(u * math.log(vocab + 1.0)) - 1.0
    ids = ids.long().clamp_(0, vocab - 1)
    n_pad = int(rows * case["pad"])
    if n_pad:
        ids[rows - n_pad:] = PAD
    return ids.to(torch.int32 if case["ids"] == 32 else torch.int64)


def _normal(gen, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda") * std + mean).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, rows, width = case["op"], case["rows"], case["width"]
    s = dict(case)
    if op == "embedding":
        s["tokens"] = _tokens(case, gen)
        s["table"] = _normal(gen, case["vocab"], width, std=0.02)               # f32 parameters
        s["scale"] = math.sqrt(width)
    elif op == "embedding_bwd":
        s["tokens"] = _tokens(case, gen)
        s["dy"] = _normal(gen, rows, width, dtype=_DTYPE[case["dtype"]])
        s["scale"] = math.sqrt(width)
    elif op in ("norm", "norm_bwd"):
        dt = _DTYPE[case["dtype"]]
        s["y"] = _normal(gen, rows, width, std=1.5, mean=0.2, dtype=dt)
        s["post_gamma"] = _normal(gen, width, std=0.1, mean=1.0)
        s["pre_gamma"] = _normal(gen, width, std=0.1, mean=1.0)
        s["post_beta"] = None if case["rms"] else _normal(gen, width, std=0.1)
        s["pre_beta"] = None if case["rms"] else _normal(gen, width, std=0.1)
        s["gate"] = None if case["gates"] == 0 else _normal(gen, case["gates"], width, std=0.3, mean=0.5)
        s["res_scale"] = 0.875
        if op == "norm":
            s["x"] = _normal(gen, rows, width, std=2.0, mean=-0.3)
        else:
            s["x_out"] = _normal(gen, rows, width, std=2.0, mean=-0.3)          # residual stream, as the forward left it
            s["dh"] = _normal(gen, rows, width, dtype=dt)
            s["dx_out"] = _normal(gen, rows, width)
            s["stats"] = torch.stack(_stats(s["y"], case["rms"]) + _stats(s["x_out"], case["rms"]), 1).float()
    elif op == "act8_gelu":
        dt = _DTYPE[case["dtype"]]
        s["u"] = _normal(gen, rows, width, std=1.2, mean=-0.4, dtype=dt)
        s["dy"] = _normal(gen, rows, width, dtype=dt)
    else:
        s["x"] = _normal(gen, rows, width, dtype=torch.bfloat16)
        s["dy"] = _normal(gen, rows, case["out"], std=0.05, dtype=torch.bfloat16)
    return s


def _stats(t, rms, eps=1e-5):
    """Mean and reciprocal deviation of each row, as a forward pass has left them."""
    t = t.double()
    mean = torch.zeros_like(t[:, 0]) if rms else t.mean(1)
    return mean, ((t - mean[:, None]).square().mean(1) + eps).rsqrt()


# ---- what a program calls ---------------------------------------------------------------------------------
def _run_own(s):
    from transcodon_amd import ops
    op = s["op"]
    if op == "embedding":
        return ops.embedding(s["tokens"], s["table"], s["scale"], pad_idx=PAD, out_dtype=_DTYPE[s["dtype"]])
    if op == "embedding_bwd":
        return ops.embedding_bwd(s["tokens"], s["dy"], s["vocab"], s["scale"], pad_idx=PAD)
    if op == "norm":
        x_out, h, stats = ops.gated_residual_norm(s["y"], s["x"], s["post_gamma"], s["post_beta"], s["gate"], s["pre_gamma"],
                                                  s["pre_beta"], res_scale=s["res_scale"], rms=s["rms"])
        return dict(x_out=x_out, h=h)
    if op == "norm_bwd":
        dy, dx, d_post_gamma, d_post_beta, d_gate, d_pre_gamma, d_pre_beta = ops.gated_residual_norm_bwd(
            s["dh"], s["dx_out"], s["y"], s["x_out"], s["stats"], s["post_gamma"], s["post_beta"], s["gate"], s["pre_gamma"],
            s["pre_beta"], res_scale=s["res_scale"], rms=s["rms"])
        return dict(dy=dy, dx=dx, d_post_gamma=d_post_gamma, d_post_beta=d_post_beta, d_gate=d_gate, d_pre_gamma=d_pre_gamma,
                    d_pre_beta=d_pre_beta)
    if op == "act8_gelu":
        act, codes, scales = ops.gelu_act8(s["u"])
        du, again = ops.dgelu_act8(s["dy"], codes, scales, want_act=True)
        return dict(act=act, du=du, again=again)
    codes, scales = ops.act8_pack(s["x"])
    return ops.gemm_tn_act8(s["dy"], codes, scales)


# ---- plain forms ------------------------------------------------------------------------------------------
def _plain_norm(t, gamma, beta, rms, eps=1e-5):
    mean = 0.0 if rms else t.mean(1, keepdim=True)
    n = (t - mean) * ((t - mean).square().mean(1, keepdim=True) + eps).rsqrt() * gamma
    return n if beta is None else n + beta


def _plain_norm_bwd(t_hat, rstd, g, gamma, rms):
    """Gradient of a norm's input: t_hat normalised rows, g the gradient of its output."""
    p = g * gamma
    back = p - t_hat * (p * t_hat).mean(1, keepdim=True)
    if not rms:
        back = back - p.mean(1, keepdim=True)
    return rstd * back


def _gated(gate, n):
    return n if gate is None else (gate[:, None] * n.view(gate.shape[0], -1, n.shape[1])).view_as(n)


def _power(e):
    """2^e in f32 for whole e in [-126, 127]."""
    return ((e + 127) << 23).view(torch.float32)


def _plain_pack(x):
    """The values that the 8-bit checkpoint of x stands for: groups of 32 along a row share the smallest power of two (at least
    2^-126) with which no value passes 448, each value is rounded once to e4m3."""
    rows, width = x.shape
    pad = -width % GROUP
    g = torch.nn.functional.pad(x.float(), (0, pad)).view(rows, -1, GROUP)
    m, e = torch.frexp(g.abs().amax(2, keepdim=True))
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-126)
    e = torch.where(m == 0, torch.full_like(e, -126), e)
    q = (g * _power(-e)).to(torch.float8_e4m3fn).float() * _power(e)
    return q.view(rows, -1)[:, :width]


def _plain_gelu(x):
    return x * 0.5 * torch.erfc(x * -0.7071067811865476)


def _run_plain(s):
    op = s["op"]
    if op == "embedding":
        keep = (s["tokens"] != PAD).float()[:, None]
        return (s["table"][s["tokens"]] * s["scale"] * keep).to(_DTYPE[s["dtype"]])
    if op == "embedding_bwd":
        g = s["dy"].float() * s["scale"] * (s["tokens"] != PAD).float()[:, None]
        return torch.zeros(s["vocab"], s["width"], device="cuda").index_add_(0, s["tokens"], g)
    rms = s.get("rms")
    if op == "norm":
        n = _plain_norm(s["y"].float(), s["post_gamma"], s["post_beta"], rms)
        x_out = s["res_scale"] * s["x"] + _gated(s["gate"], n)
        h = _plain_norm(x_out, s["pre_gamma"], s["pre_beta"], rms).to(s["y"].dtype)
        return dict(x_out=x_out, h=h)
    if op == "norm_bwd":
        mean1, rstd1, mean2, rstd2 = s["stats"][:, :, None].unbind(1)
        dh = s["dh"].float()
        x_hat = (s["x_out"] - mean2) * rstd2
        d = s["dx_out"] + _plain_norm_bwd(x_hat, rstd2, dh, s["pre_gamma"], rms)
        y_hat = (s["y"].float() - mean1) * rstd1
        n = y_hat * s["post_gamma"]
        if s["post_beta"] is not None:
            n = n + s["post_beta"]
        dn = _gated(s["gate"], d)
        dy = _plain_norm_bwd(y_hat, rstd1, dn, s["post_gamma"], rms).to(s["y"].dtype)
        d_gate = None if s["gate"] is None else (d * n).view(s["gates"], -1, s["width"]).sum(1)
        return dict(dy=dy, dx=s["res_scale"] * d, d_post_gamma=(dn * y_hat).sum(0), d_post_beta=None if rms else dn.sum(0),
                    d_gate=d_gate, d_pre_gamma=(dh * x_hat).sum(0), d_pre_beta=None if rms else dh.sum(0))
    if op == "act8_gelu":
        u, dt = s["u"].float(), s["u"].dtype
        kept = _plain_pack(u)
        slope = 0.5 * torch.erfc(kept * -0.7071067811865476) + kept * torch.exp(-0.5 * kept * kept) * 0.3989422804014327
        return dict(act=_plain_gelu(u).to(dt), du=(s["dy"].float() * slope).to(dt), again=_plain_gelu(kept).to(dt))
    return s["dy"].float().t() @ _plain_pack(s["x"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------
def work(case):
    op, m, e = case["op"], case["rows"], case["width"]
    t = 2 if case.get("dtype") == "bf16" else 4
    if op == "embedding":       # ids, the rows of the table that they can name, the output
        return dict(bytes=m * case["ids"] // 8 + 4 * e * min(m, case["vocab"]) + t * m * e, flops=m * e)
    if op == "embedding_bwd":   # ids, the rows that are not <pad>, the dense gradient
        kept = m - int(m * case["pad"])
        return dict(bytes=m * case["ids"] // 8 + t * kept * e + 4 * e * case["vocab"], flops=kept * e)
    vectors = 4 * e * ((2 if case.get("rms") else 4) + case.get("gates", 0))
    if op == "norm":            # y, x, x_out, h
        return dict(bytes=m * e * (t + 4 + 4 + t) + vectors, flops=20 * m * e)
    if op == "norm_bwd":        # dh, dx_out, y, x_out, dy, dx, and the gradients of the vectors
        return dict(bytes=m * e * (t + 4 + t + 4 + t + 4) + 16 * m + 2 * vectors, flops=40 * m * e)
    kept = m * (e + -(-e // GROUP))
    if op == "act8_gelu":       # u, act, the checkpoint written and read, dy, du, act again
        return dict(bytes=5 * t * m * e + 2 * kept, flops=80 * m * e)
    # x, the checkpoint written and read, dy, the gradient
    return dict(bytes=2 * m * e + 2 * kept + 2 * m * case["out"] + 4 * case["out"] * e, flops=2 * m * e * case["out"])


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------
def _exact_pack(x):
    rows, width = x.shape
    x = x.double()
    out = torch.empty_like(x)
    for first in range(0, width, GROUP):
        g = x[:, first:first + GROUP]
        most = g.abs().amax(1, keepdim=True)
        unit = torch.full_like(most, 2.0 ** -126)
        e = torch.ceil(torch.log2((most / 448.0).clamp(min=2.0 ** -126)))
        e = torch.where(torch.exp2(e - 1) * 448.0 >= most, e - 1, e)
        e = torch.where(torch.exp2(e) * 448.0 < most, e + 1, e)
        unit = torch.maximum(unit, torch.exp2(e))
        v = g / unit
        # e4m3: three bits behind the leading one, steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        out[:, first:first + GROUP] = torch.round(v / step) * step * unit
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "embedding":
        out = s["table"].double().index_select(0, s["tokens"].long()) * s["scale"]
        out[s["tokens"] == PAD] = 0.0
        return out
    if op == "embedding_bwd":
        order = s["tokens"].long().argsort(stable=True)
        ids, dy = s["tokens"].long()[order], s["dy"].double()[order]
        out = torch.zeros(s["vocab"], s["width"], dtype=torch.float64, device="cuda")
        out.index_add_(0, ids[ids != PAD], dy[ids != PAD])
        return out * s["scale"]
    if op in ("norm", "norm_bwd"):
        vec = {k: None if s[k] is None else s[k].double() for k in ("post_gamma", "post_beta", "pre_gamma", "pre_beta", "gate")}
        y = s["y"].double().requires_grad_(op == "norm_bwd")
        for v in vec.values():
            if v is not None:
                v.requires_grad_(op == "norm_bwd")

        def norm(t, gamma, beta):
            c = t if s["rms"] else t - t.mean(1, keepdim=True)
            t_hat = c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt()
            return t_hat * gamma if beta is None else t_hat * gamma + beta

        def gated(n):
            return n if vec["gate"] is None else (vec["gate"][:, None] * n.view(s["gates"], -1, s["width"])).view_as(n)

        if op == "norm":
            x_out = s["res_scale"] * s["x"].double() + gated(norm(y, vec["post_gamma"], vec["post_beta"]))
            return dict(x_out=x_out, h=norm(x_out, vec["pre_gamma"], vec["pre_beta"]))
        x_out = s["x_out"].double().requires_grad_()
        h = norm(x_out, vec["pre_gamma"], vec["pre_beta"])
        wanted = [x_out, vec["pre_gamma"]] + ([] if s["rms"] else [vec["pre_beta"]])
        got = torch.autograd.grad(h, wanted, s["dh"].double())
        d = s["dx_out"].double() + got[0]
        branch = gated(norm(y, vec["post_gamma"], vec["post_beta"]))
        names = ["post_gamma"] + ([] if s["rms"] else ["post_beta"]) + ([] if s["gate"] is None else ["gate"])
        back = dict(zip(["y"] + names, torch.autograd.grad(branch, [y] + [vec[k] for k in names], d)))
        return dict(dy=back["y"], dx=s["res_scale"] * d, d_post_gamma=back["post_gamma"], d_post_beta=back.get("post_beta"),
                    d_gate=back.get("gate"), d_pre_gamma=got[1], d_pre_beta=None if s["rms"] else got[2])
    if op == "act8_gelu":
        u = s["u"].double()
        kept = _exact_pack(s["u"]).requires_grad_()
        again = kept * torch.special.ndtr(kept)
        du, = torch.autograd.grad(again, kept, s["dy"].double())
        return dict(act=u * torch.special.ndtr(u), du=du, again=again.detach())
    return s["dy"].double().t() @ _exact_pack(s["x"])
