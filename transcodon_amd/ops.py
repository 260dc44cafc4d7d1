"""Torch-tensor front ends of the C-ABI kernels (device pointers + current HIP stream).

PyTorch only provides device memory and the stream here; all arithmetic runs in
libtranscodon_hip.so.  Every function requires CUDA(HIP) tensors and raises otherwise.
"""

import torch

from . import _lib
from ._lib import TC_BF16, TC_F32, check

AA_ORDER = "FLIMVPTAY_HQNKDECWRSG"      # amino-acid codes of tc_codon_decode
_AA_CODE = {c: i for i, c in enumerate(AA_ORDER)}


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return TC_BF16
    if t.dtype == torch.float32:
        return TC_F32
    raise TypeError(f"unsupported element type {t.dtype}")


def _dev(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise _lib.HipLibraryError("transcodon_amd kernels need tensors on the GPU (no CPU fallback)")
        if t is not None and not t.is_contiguous():
            raise ValueError("tensor must be contiguous")


def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def embed(tokens, species, tok_table, species_table, pad_idx=1):
    """x[B*T,E] f32, pad_flags[B*T] u8, bad[1] i32   (model.py:178-206)."""
    tokens = tokens.to(torch.int32).contiguous()
    species = species.to(torch.int32).contiguous()
    _dev(tokens, species, tok_table, species_table)
    B, T = tokens.shape
    E = tok_table.shape[1]
    x = torch.empty(B * T, E, dtype=torch.float32, device=tokens.device)
    pad = torch.empty(B * T, dtype=torch.uint8, device=tokens.device)
    bad = torch.zeros(1, dtype=torch.int32, device=tokens.device)
    check(_lib.load().tc_embed_fwd(_p(tokens), _p(species), _p(tok_table), _p(species_table), _p(x),
                                   _p(pad), _p(bad), B, T, E, tok_table.shape[0],
                                   species_table.shape[0], pad_idx, _stream()), "tc_embed_fwd")
    return x, pad, bad


def layernorm(x, gamma, beta, eps=1e-5, out_dtype=torch.float32):
    _dev(x, gamma, beta)
    M, E = x.shape
    out = torch.empty(M, E, dtype=out_dtype, device=x.device)
    f32 = out if out_dtype == torch.float32 else None
    b16 = out if out_dtype == torch.bfloat16 else None
    check(_lib.load().tc_layernorm_fwd(_p(x), _p(gamma), _p(beta), _p(f32), _p(b16), M, E, eps,
                                       _stream()), "tc_layernorm_fwd")
    return out


def gemm(a, w, bias, epilogue=_lib.EPI_BIAS, residual=None, out=None, q_scale=1.0,
         rope_cos=None, rope_sin=None, T=0, head_dim=0):
    """epilogue(a[M,K] @ w[N,K]^T + bias[N]); see tc_gemm."""
    _dev(a, w, bias, residual, out, rope_cos, rope_sin)
    M, K = a.shape
    N = w.shape[0]
    assert w.shape[1] == K and a.dtype == w.dtype
    if out is None:
        odt = torch.float32 if epilogue == _lib.EPI_BIAS_RESIDUAL else a.dtype
        out = torch.empty(M, N, dtype=odt, device=a.device)
    check(_lib.load().tc_gemm(_dt(a), epilogue, _p(a), a.stride(0), _p(w), _p(bias), _p(residual),
                              _p(out), out.stride(0), M, N, K, q_scale, _p(rope_cos), _p(rope_sin),
                              T, head_dim, _stream()), "tc_gemm")
    return out


def key_mask_words(pad_flags, B, T):
    _dev(pad_flags)
    words = torch.empty(B, (T + 63) // 64, dtype=torch.int64, device=pad_flags.device)
    check(_lib.load().tc_key_mask_words(_p(pad_flags), _p(words), B, T, _stream()), "tc_key_mask_words")
    return words


def attention(qkv, B, T, H, key_words=None, q2=False):
    """qkv[B*T, 3*H*64] (q scaled, q/k rotated) -> out[B*T, H*64].  q2: the q columns carry
    log2(e) / sqrt(64) instead of 1 / sqrt(64) (tc_attn_fwd_q2, bf16 only)."""
    _dev(qkv, key_words)
    E = H * 64
    out = torch.empty(B * T, E, dtype=qkv.dtype, device=qkv.device)
    fn = _lib.load().tc_attn_fwd_q2 if q2 else _lib.load().tc_attn_fwd
    check(fn(_dt(qkv), _p(qkv), qkv.stride(0), _p(key_words), _p(out), B, T, H, 64, _stream()),
          "tc_attn_fwd_q2" if q2 else "tc_attn_fwd")
    return out


def attention_scores(qkv, B, T, H, pad_flags=None):
    _dev(qkv, pad_flags)
    s = torch.empty(B, H, T, T, dtype=torch.float32, device=qkv.device)
    check(_lib.load().tc_attn_scores(_dt(qkv), _p(qkv), qkv.stride(0), _p(pad_flags), _p(s), B, T, H, 64,
                                     _stream()), "tc_attn_scores")
    return s


def head_logits(g, col0, E, gamma, beta, W, bias, eps=1e-5):
    _dev(g, gamma, beta, W, bias)
    M = g.shape[0]
    V = W.shape[0]
    out = torch.empty(M, V, dtype=torch.float32, device=g.device)
    check(_lib.load().tc_head_logits_fwd(_dt(g), _p(g), g.stride(0), col0, _p(gamma), _p(beta), _p(W),
                                         _p(bias), _p(out), M, E, V, eps, _stream()),
          "tc_head_logits_fwd")
    return out


def mean_pool(rep, start, length):
    """rep f32 [B,T,E]; start,length int32 [B] -> pooled f32 [B,E] (tc_mean_pool)."""
    start = start.to(torch.int32).contiguous()
    length = length.to(torch.int32).contiguous()
    _dev(rep, start, length)
    B, T, E = rep.shape
    out = torch.empty(B, E, dtype=torch.float32, device=rep.device)
    check(_lib.load().tc_mean_pool(_p(rep), _p(start), _p(length), _p(out), B, T, E, _stream()), "tc_mean_pool")
    return out


def mean_pool_packed(rep, row_start, length):
    """rep f32 [M,E] (packed rows); row_start, length int32 [n] -> pooled f32 [n,E] (tc_mean_pool_packed)."""
    row_start = row_start.to(torch.int32).contiguous()
    length = length.to(torch.int32).contiguous()
    _dev(rep, row_start, length)
    M, E = rep.shape
    n = row_start.numel()
    out = torch.empty(n, E, dtype=torch.float32, device=rep.device)
    check(_lib.load().tc_mean_pool_packed(_p(rep), _p(row_start), _p(length), _p(out), n, M, E, _stream()),
          "tc_mean_pool_packed")
    return out


def encode_amino_acids(aa_seq: str) -> bytes:
    """Protein letters -> tc_codon_decode codes; unknown letters raise KeyError like
    the reference's dict lookup (infer_utr.py:108)."""
    return bytes(_AA_CODE[c] for c in aa_seq)


def codon_decode(logits2d, aa_codes, aa_off, row0):
    """logits2d f32 [rows, >=10]; aa_codes u8 [n]; aa_off i32 [n_seq+1]; row0 i32 [n_seq]
    -> bases u8 [3n] (ASCII).  See tc_codon_decode."""
    _dev(logits2d, aa_codes, aa_off, row0)
    assert logits2d.dtype == torch.float32
    n = aa_codes.numel()
    bases = torch.empty(3 * n, dtype=torch.uint8, device=logits2d.device)
    check(_lib.load().tc_codon_decode(_p(logits2d), logits2d.stride(0), _p(aa_codes), _p(aa_off),
                                      _p(row0), _p(bases), row0.numel(), n, _stream()),
          "tc_codon_decode")
    return bases


def ce_loss(logits2d, labels, want_grad=False, grad_scale=1.0):
    """Returns (loss_sum f32[1], count i32[1], dlogits or None); mean = sum / count."""
    labels = labels.to(torch.int32).contiguous()
    _dev(logits2d, labels)
    M, V = logits2d.shape
    loss = torch.zeros(1, dtype=torch.float32, device=logits2d.device)
    cnt = torch.zeros(1, dtype=torch.int32, device=logits2d.device)
    dl = torch.empty_like(logits2d) if want_grad else None
    check(_lib.load().tc_ce_loss_fwd_bwd(_p(logits2d), _p(labels), _p(loss), _p(cnt), _p(dl),
                                         grad_scale, M, V, _stream()), "tc_ce_loss_fwd_bwd")
    return loss, cnt, dl


# ---- training-step kernels -----------------------------------------------------------------
def gemm_train(a, w, epilogue, bias=None, aux=None, out=None, out2=None, splits=1):
    """tc_gemm_train: EPI_PLAIN_F32 (f32 out, optional split-K slabs [splits, M, N]),
    EPI_BIAS_GELU_SAVE (returns (gelu, pre)), EPI_DGELU (aux = pre-activation; out2: optional f32 [N]
    that receives += column sums of the result)."""
    _dev(a, w, bias, aux, out, out2)
    M, K = a.shape
    N = w.shape[0]
    assert w.shape[1] == K and a.dtype == w.dtype
    if out is None:
        if epilogue == _lib.EPI_PLAIN_F32:
            out = torch.empty((splits, M, N) if splits > 1 else (M, N), dtype=torch.float32, device=a.device)
        else:
            out = torch.empty(M, N, dtype=a.dtype, device=a.device)
    if epilogue == _lib.EPI_BIAS_GELU_SAVE and out2 is None:
        out2 = torch.empty(M, N, dtype=a.dtype, device=a.device)
    check(_lib.load().tc_gemm_train(_dt(a), epilogue, _p(a), a.stride(0), _p(w), _p(bias), _p(aux), _p(out),
                                    _p(out2), N, M, N, K, splits, _stream()), "tc_gemm_train")
    return (out, out2) if epilogue == _lib.EPI_BIAS_GELU_SAVE else out


def transpose_cast(x, out_dtype, want_rowmajor=False, want_colsum=False, colsum=None, pad_to=64):
    """x [M,N] -> (x^T [N, ldt] zero-padded to a multiple of pad_to columns, row-major copy or
    None, column sums f32 [N] or None)."""
    _dev(x, colsum)
    M, N = x.shape
    ldt = (M + pad_to - 1) // pad_to * pad_to
    out_t = torch.empty(N, ldt, dtype=out_dtype, device=x.device)
    rm = torch.empty(M, N, dtype=out_dtype, device=x.device) if want_rowmajor else None
    if want_colsum and colsum is None:
        colsum = torch.zeros(N, dtype=torch.float32, device=x.device)
    check(_lib.load().tc_transpose_cast(_dt(x), TC_BF16 if out_dtype == torch.bfloat16 else TC_F32, _p(x),
                                        x.stride(0), _p(out_t), ldt, _p(rm), N, _p(colsum), M, N, _stream()),
          "tc_transpose_cast")
    return out_t, rm, colsum


def reduce_slabs(slabs, out=None, accumulate=False):
    _dev(slabs, out)
    S = slabs.shape[0]
    n = slabs[0].numel()
    if out is None:
        out = torch.empty_like(slabs[0])
        accumulate = False
    check(_lib.load().tc_reduce_slabs(_p(slabs), _p(out), S, n, int(accumulate), _stream()), "tc_reduce_slabs")
    return out


def layernorm_bwd(x, gamma, dy, dgamma, dbeta, dx=None, accumulate=False, eps=1e-5, dx_bf16=None, dx_colsum=None):
    """x and dy may be column slices of wider buffers (row stride = leading dimension); dy f32 or bf16.
    dx_bf16 [M,E] bf16 / dx_colsum [E] f32 (accumulated): optional bf16 copy and column sums of the final dx."""
    _dev(gamma, dy, dgamma, dbeta, dx, dx_bf16, dx_colsum)
    if not x.is_cuda or x.stride(1) != 1 or dy.stride(1) != 1:
        raise ValueError("x must be a GPU tensor, x and dy with unit column stride")
    M, E = dy.shape
    if dx is None:
        dx = torch.empty(M, E, dtype=torch.float32, device=dy.device)
        accumulate = False
    check(_lib.load().tc_layernorm_bwd_dy(_dt(x), _p(x), x.stride(0), _p(gamma), _dt(dy), _p(dy), dy.stride(0), _p(dx),
                                          int(accumulate), _p(dgamma), _p(dbeta), _p(dx_bf16), _p(dx_colsum), M, E, eps,
                                          _stream()),
          "tc_layernorm_bwd")
    return dx


def dgelu(dy, u):
    _dev(dy, u)
    out = torch.empty_like(u)
    check(_lib.load().tc_dgelu(_dt(u), _p(dy), _p(u), _p(out), u.numel(), _stream()), "tc_dgelu")
    return out


def head_logits_bwd(g, col0, E, gamma, beta, W, dlogits, dW, dbias, eps=1e-5):
    _dev(g, gamma, beta, W, dlogits, dW, dbias)
    M, V = dlogits.shape
    d_ln = torch.empty(M, E, dtype=torch.float32, device=g.device)
    check(_lib.load().tc_head_logits_bwd(_dt(g), _p(g), g.stride(0), col0, _p(gamma), _p(beta), _p(W), _p(dlogits),
                                         _p(d_ln), _p(dW), _p(dbias), M, E, V, eps, _stream()),
          "tc_head_logits_bwd")
    return d_ln


def embed_bwd(tokens, species, dx, d_tok, d_sp, pad_idx=1):
    tokens = tokens.to(torch.int32).contiguous()
    species = species.to(torch.int32).contiguous()
    _dev(tokens, species, dx, d_tok, d_sp)
    B, T = tokens.shape
    E = dx.shape[-1]
    check(_lib.load().tc_embed_bwd(_p(tokens), _p(species), _p(dx), _p(d_tok), _p(d_sp), B, T, E, d_tok.shape[0],
                                   d_sp.shape[0], pad_idx, _stream()), "tc_embed_bwd")


def rope_bwd(dqkv, cos, sin, T, E, head_dim, q_scale):
    _dev(dqkv, cos, sin)
    check(_lib.load().tc_rope_bwd(_dt(dqkv), _p(dqkv), dqkv.stride(0), _p(cos), _p(sin), dqkv.shape[0], T, E,
                                  head_dim, q_scale, _stream()), "tc_rope_bwd")
    return dqkv


def attention_train(qkv, B, T, H, key_words=None):
    """Forward that also returns lse f32 [B,H,T] for attention_bwd (tc_attn_fwd_train)."""
    _dev(qkv, key_words)
    E = H * 64
    out = torch.empty(B * T, E, dtype=qkv.dtype, device=qkv.device)
    lse = torch.empty(B, H, T, dtype=torch.float32, device=qkv.device)
    check(_lib.load().tc_attn_fwd_train(_dt(qkv), _p(qkv), qkv.stride(0), _p(key_words), _p(out), _p(lse),
                                        B, T, H, 64, _stream()), "tc_attn_fwd_train")
    return out, lse


def attention_bwd(qkv, out, d_out, lse, B, T, H, key_words=None, rope_cos=None, rope_sin=None, q_scale=1.0):
    """Gradient of attention() with respect to its qkv input (tc_attn_bwd) -> d_qkv like qkv; with
    rope tables, with respect to the unrotated, unscaled q/k/v projections."""
    _dev(qkv, out, d_out, lse, key_words, rope_cos, rope_sin)
    E = H * 64
    if out.shape != (B * T, E) or d_out.shape != (B * T, E) or not out.is_contiguous() or not d_out.is_contiguous():
        raise ValueError("attention_bwd: out and d_out must be contiguous [B*T, E]")
    if d_out.dtype != qkv.dtype or out.dtype != qkv.dtype:
        raise ValueError("attention_bwd: out/d_out dtype must match qkv")
    d_qkv = torch.empty(B * T, 3 * E, dtype=qkv.dtype, device=qkv.device)
    delta = torch.empty(B, H, T, dtype=torch.float32, device=qkv.device)
    check(_lib.load().tc_attn_bwd(_dt(qkv), _p(qkv), qkv.stride(0), _p(key_words), _p(out), _p(d_out), _p(lse),
                                  _p(delta), _p(d_qkv), d_qkv.stride(0), _p(rope_cos), _p(rope_sin), q_scale,
                                  B, T, H, 64, _stream()), "tc_attn_bwd")
    return d_qkv


def gemm_tn(a, b, splits=1):
    """slabs[s] = partial a^T b over the s-th part of the rows; a [M,I], b [M,J] bf16 (tc_gemm_tn)."""
    _dev(a, b)
    M, I = a.shape
    J = b.shape[1]
    assert b.shape[0] == M and a.dtype == torch.bfloat16 and b.dtype == torch.bfloat16
    out = torch.empty(splits, I, J, dtype=torch.float32, device=a.device)
    check(_lib.load().tc_gemm_tn(_p(a), a.stride(0), _p(b), b.stride(0), _p(out), J, M, I, J, splits, _stream()),
          "tc_gemm_tn")
    return out


def colsum(x, want_bf16_copy=False, out=None):
    """Column sums f32 [N] of x [M,N] (added to ``out`` when given) and, for f32 x, a bf16 copy."""
    _dev(x, out)
    M, N = x.shape
    if out is None:
        out = torch.zeros(N, dtype=torch.float32, device=x.device)
    copy = torch.empty(M, N, dtype=torch.bfloat16, device=x.device) if want_bf16_copy else None
    check(_lib.load().tc_colsum(_dt(x), _p(x), x.stride(0), _p(copy), N, _p(out), M, N, _stream()), "tc_colsum")
    return (out, copy) if want_bf16_copy else out


# ---- operators of a training block ---------------------------------------------------------------
def _same_device(*tensors):
    """The common device of GPU tensors (None entries skipped); raises otherwise."""
    first, index = None, -1
    for t in tensors:
        if t is None:
            continue
        i = t.get_device()
        if i < 0:
            raise _lib.HipLibraryError("transcodon_amd kernels need tensors on the GPU (no CPU fallback)")
        if first is None:
            first, index = t, i
        elif i != index:
            raise ValueError(f"tensors on {first.device} and {t.device}")
    return first.device


# handle of a device's current stream without a Stream object around it (2 us of a call's 7)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _call(name, dev, *args):
    """One library call on ``dev``'s current stream, also where another device is the current one."""
    fn = getattr(_lib.load(), name)
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev.index))
    if rc:
        check(rc, name)


def _rows(t, name):
    """Row stride of a 2-d tensor whose columns are neighbours in memory."""
    if t.dim() == 2:
        (M, E), (ld, step) = t.shape, t.stride()
        if (step == 1 or E <= 1) and (ld >= E or M <= 1):
            return ld if ld > E else E
    raise ValueError(f"{name} must be 2-d with unit column stride and rows that do not overlap")


def _scratch(need, out, dev):
    """Workspace of ``need`` bytes; 16 stand for "none is used", where the output's address does."""
    if need <= 16 and out.data_ptr() % 16 == 0:
        return out
    return torch.empty(max(need, 16), dtype=torch.uint8, device=dev)


def _dense(t, name, shape=None, dtype=None):
    """Checks a dense operand: its shape and element type where they are given."""
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} has type {t.dtype}, expected {dtype}")


def _pad(pad_idx):
    if pad_idx is None:
        return -1
    if pad_idx < 0:
        raise ValueError(f"pad_idx must be None or at least 0, got {pad_idx}")
    return pad_idx


def _id_bytes(tokens):
    if tokens.dtype == torch.int32:
        return 4
    if tokens.dtype == torch.int64:
        return 8
    raise TypeError(f"token ids must be int32 or int64, got {tokens.dtype}")


def embedding(tokens, table, scale=1.0, pad_idx=None, out_dtype=None, bad=None):
    """scale * table[tokens] -> [tokens.numel(), E] in ``out_dtype`` (default: the table's type), zeros for ``pad_idx`` and for
    ids outside the table; the latter also set ``bad`` (int32 [1], optional, never cleared here).  tc_embedding_fwd; the lookup
    of model.py:178-206 for a table of any size."""
    dev = _same_device(tokens, table, bad)
    idb = _id_bytes(tokens)
    _dense(tokens, "tokens")
    if table.dim() != 2:
        raise ValueError("table must be [vocab, E]")
    _dense(table, "table")
    if bad is not None:
        _dense(bad, "bad", (1,), torch.int32)
    V, E = table.shape
    M = tokens.numel()
    out = torch.empty(M, E, dtype=out_dtype or table.dtype, device=dev)
    dts = _dt(table), _dt(out)
    if M and E:
        _call("tc_embedding_fwd", dev, *dts, idb, tokens.data_ptr(), table.data_ptr(), out.data_ptr(), M, E, V, scale,
              _pad(pad_idx), _p(bad))
    return out


def embedding_bwd(tokens, dy, vocab, scale=1.0, pad_idx=None, out=None):
    """Gradient of :func:`embedding` with respect to its table: f32 [vocab, E], summed by sorted tokens in a fixed order
    (added to ``out`` when given).  dy [tokens.numel(), E] f32 or bf16, rows may be strided.  tc_embedding_bwd."""
    dev = _same_device(tokens, dy, out)
    idb = _id_bytes(tokens)
    _dense(tokens, "tokens")
    ld = _rows(dy, "dy")
    M, E = dy.shape
    if tokens.numel() != M:
        raise ValueError(f"{tokens.numel()} tokens but {M} rows of dy")
    accumulate = out is not None
    if accumulate:
        _dense(out, "out", (vocab, E), torch.float32)
    elif M == 0 or E == 0:
        return torch.zeros(vocab, E, dtype=torch.float32, device=dev)
    else:
        out = torch.empty(vocab, E, dtype=torch.float32, device=dev)
    dt = _dt(dy)
    if M and E:
        need = _lib.load().tc_embedding_bwd_workspace_bytes(M, E, vocab)
        ws = _scratch(need, out, dev)
        _call("tc_embedding_bwd", dev, dt, idb, tokens.data_ptr(), dy.data_ptr(), ld, out.data_ptr(), M, E, vocab, scale,
              _pad(pad_idx), int(accumulate), ws.data_ptr(), need)
    return out


def _vector(t, name, E):
    if t is not None:
        _dense(t, name, (E,), torch.float32)


def _gate(gate, M, E, dtype):
    """(type code, rows) of a gate [E] or [G, E] with G dividing M; (f32, 0) for none."""
    if gate is None:
        return TC_F32, 0
    _dense(gate, "gate")
    G = 1 if gate.dim() == 1 else gate.shape[0]
    if gate.dim() not in (1, 2) or gate.shape[-1] != E or G == 0 or M % G:
        raise ValueError(f"gate of shape {tuple(gate.shape)} for {M} rows of {E}: [E] or [G, E] with G dividing the rows")
    if gate.dtype != torch.float32 and gate.dtype != dtype:
        raise TypeError(f"gate has type {gate.dtype}, expected float32 or {dtype}")
    return _dt(gate), G


def gated_residual_norm(y, x, post_gamma, post_beta=None, gate=None, pre_gamma=None, pre_beta=None, res_scale=1.0, eps=1e-5,
                        rms=False):
    """The end of a block and the start of the next in one pass over y (the block's output, [M, E] f32 or bf16) and the f32
    residual stream x [M, E]:

        x_out = res_scale * x + gate * norm(y; post)        h = norm(x_out; pre)

    norm: LayerNorm, or root-mean-square norm with ``rms``; betas are optional.  gate: None, [E], or [G, E] whose row g is for rows
    g M/G .. (g+1) M/G - 1 (one per sequence, or one per row).  Without ``pre_gamma`` there is no h.
    Returns (x_out f32, h of y's type or None, stats f32 [M, 4] for the backward pass).  tc_gated_residual_norm_fwd."""
    dev = _same_device(y, x, post_gamma, post_beta, gate, pre_gamma, pre_beta)
    dt, ldy, ldx = _dt(y), _rows(y, "y"), _rows(x, "x")
    M, E = y.shape
    if x.shape != y.shape or x.dtype != torch.float32:
        raise ValueError(f"x must be float32 {tuple(y.shape)}, got {x.dtype} {tuple(x.shape)}")
    for t, n in ((post_gamma, "post_gamma"), (post_beta, "post_beta"), (pre_gamma, "pre_gamma"), (pre_beta, "pre_beta")):
        _vector(t, n, E)
    if pre_gamma is None and pre_beta is not None:
        raise ValueError("pre_beta without pre_gamma")
    gdt, G = _gate(gate, M, E, y.dtype)
    x_out = torch.empty(M, E, dtype=torch.float32, device=dev)
    h = None if pre_gamma is None else torch.empty(M, E, dtype=y.dtype, device=dev)
    stats = torch.empty(M, 4, dtype=torch.float32, device=dev)
    if M and E:
        _call("tc_gated_residual_norm_fwd", dev, dt, y.data_ptr(), ldy, x.data_ptr(), ldx, post_gamma.data_ptr(), _p(post_beta),
              gdt, _p(gate), G, res_scale, _p(pre_gamma), _p(pre_beta), x_out.data_ptr(), _p(h), stats.data_ptr(), M, E, int(rms),
              eps, eps)
    return x_out, h, stats


def gated_residual_norm_bwd(dh, dx_out, y, x_out, stats, post_gamma, post_beta=None, gate=None, pre_gamma=None, pre_beta=None,
                            res_scale=1.0, rms=False, into=None):
    """Gradient of :func:`gated_residual_norm`: dh (of y's type) and dx_out (f32) are those of h and x_out, either may be None
    (dh is None exactly where there is no second norm); y, x_out and stats are those of the forward pass.

    Returns (dy, dx, d_post_gamma, d_post_beta, d_gate, d_pre_gamma, d_pre_beta), f32 but for dy, None where there is no such
    vector.  into: five f32 buffers or None in the order of the last five, which are added to instead; no two
    may overlap.
    tc_gated_residual_norm_bwd."""
    dev = _same_device(dh, dx_out, y, x_out, stats, post_gamma, post_beta, gate, pre_gamma, pre_beta, *(into or ()))
    dt, ldy, ldx = _dt(y), _rows(y, "y"), _rows(x_out, "x_out")
    M, E = y.shape
    if x_out.shape != y.shape or x_out.dtype != torch.float32:
        raise ValueError(f"x_out must be float32 {tuple(y.shape)}, got {x_out.dtype} {tuple(x_out.shape)}")
    if (dh is None) != (pre_gamma is None):
        raise ValueError("dh and pre_gamma go together")
    if dh is None and dx_out is None:
        raise ValueError("neither dh nor dx_out")
    if dh is not None and (dh.shape != y.shape or dh.dtype != y.dtype):
        raise ValueError(f"dh must be {y.dtype} {tuple(y.shape)}, got {dh.dtype} {tuple(dh.shape)}")
    if dx_out is not None and (dx_out.shape != y.shape or dx_out.dtype != torch.float32):
        raise ValueError(f"dx_out must be float32 {tuple(y.shape)}, got {dx_out.dtype} {tuple(dx_out.shape)}")
    _dense(stats, "stats", (M, 4), torch.float32)
    for t, n in ((post_gamma, "post_gamma"), (post_beta, "post_beta"), (pre_gamma, "pre_gamma"), (pre_beta, "pre_beta")):
        _vector(t, n, E)
    gdt, G = _gate(gate, M, E, y.dtype)
    dy = torch.empty(M, E, dtype=y.dtype, device=dev)
    dx = torch.empty(M, E, dtype=torch.float32, device=dev)
    vectors = (post_gamma, post_beta, gate, pre_gamma, pre_beta)
    if into is not None and len(into) != len(vectors):
        raise ValueError(f"into has {len(into)} buffers, expected {len(vectors)}")
    empty = torch.empty if M and E else torch.zeros
    # one allocation for the gradients of length E
    fresh = iter(empty(4, E, dtype=torch.float32, device=dev).unbind(0))
    got, accumulate = [], 0
    for i, v in enumerate(vectors):
        given = into[i] if into else None
        if given is not None:
            if v is None:
                raise ValueError("into has a buffer for a vector that is not there")
            _dense(given, "buffer in into", v.shape, torch.float32)
            accumulate |= (1, 2, 16, 4, 8)[i]
        elif v is not None:
            given = empty(v.shape, dtype=torch.float32, device=dev) if i == 2 else next(fresh)
        got.append(given)
    if M and E:
        need = _lib.load().tc_gated_residual_norm_bwd_workspace_bytes(M, E, G)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        d_post_gamma, d_post_beta, d_gate, d_pre_gamma, d_pre_beta = got
        _call("tc_gated_residual_norm_bwd", dev, dt, _p(dh), 0 if dh is None else _rows(dh, "dh"), _p(dx_out),
              0 if dx_out is None else _rows(dx_out, "dx_out"), y.data_ptr(), ldy, x_out.data_ptr(), ldx, stats.data_ptr(),
              post_gamma.data_ptr(), _p(post_beta), gdt, _p(gate), G, res_scale, _p(pre_gamma), dy.data_ptr(), dx.data_ptr(),
              _p(d_post_gamma), _p(d_post_beta), _p(d_gate), _p(d_pre_gamma), _p(d_pre_beta), accumulate, M, E, int(rms),
              ws.data_ptr(), need)
    return (dy, dx, *got)


ACT8_GROUP = 32      # neighbouring values of a row that share a scale


def _act8(codes, scales):
    """(M, E) of an 8-bit activation: codes float8_e4m3fn [M, E], scales float8_e8m0fnu [M, ceil(E / 32)]."""
    if codes.dim() != 2:
        raise ValueError("codes must be [M, E]")
    M, E = codes.shape
    _dense(codes, "codes", dtype=torch.float8_e4m3fn)
    _dense(scales, "scales", (M, (E + ACT8_GROUP - 1) // ACT8_GROUP), torch.float8_e8m0fnu)
    return M, E


def _act8_empty(M, E, dev):
    return (torch.empty(M, E, dtype=torch.float8_e4m3fn, device=dev),
            torch.empty(M, (E + ACT8_GROUP - 1) // ACT8_GROUP, dtype=torch.float8_e8m0fnu, device=dev))


def act8_pack(x):
    """8-bit form of an activation x [M, E] (f32 or bf16, rows may be strided) kept for the backward pass: codes
    (float8_e4m3fn [M, E]) and scales (float8_e8m0fnu, one power of two per row and 32 columns); a value is
    code * scale, at most half an e4m3 step from x.  tc_act8_pack."""
    dev = _same_device(x)
    dt, ld = _dt(x), _rows(x, "x")
    M, E = x.shape
    codes, scales = _act8_empty(M, E, dev)
    if M and E:
        _call("tc_act8_pack", dev, dt, x.data_ptr(), ld, codes.data_ptr(), scales.data_ptr(), M, E)
    return codes, scales


def act8_unpack(codes, scales, out_dtype=torch.bfloat16):
    """The values of an 8-bit activation, [M, E] f32 or bf16 (exact in both but below 2^-133 in bf16).  tc_act8_unpack."""
    dev = _same_device(codes, scales)
    M, E = _act8(codes, scales)
    out = torch.empty(M, E, dtype=out_dtype, device=dev)
    dt = _dt(out)
    if M and E:
        _call("tc_act8_unpack", dev, dt, codes.data_ptr(), scales.data_ptr(), out.data_ptr(), M, E)
    return out


def gelu_act8(u):
    """(gelu(u) in u's type, codes, scales): the activation of a feed-forward block and the 8-bit form of its input in one pass
    over u [M, E].  tc_gelu_act8."""
    dev = _same_device(u)
    dt, ld = _dt(u), _rows(u, "u")
    M, E = u.shape
    act = torch.empty(M, E, dtype=u.dtype, device=dev)
    codes, scales = _act8_empty(M, E, dev)
    if M and E:
        _call("tc_gelu_act8", dev, dt, u.data_ptr(), ld, act.data_ptr(), codes.data_ptr(), scales.data_ptr(), M, E)
    return act, codes, scales


def dgelu_act8(dy, codes, scales, want_act=False):
    """dy * gelu'(v) in dy's type, v being the values of the 8-bit activation; with ``want_act`` also gelu(v), which the weight
    gradient of the next linear layer reads, from the same pass.  tc_dgelu_act8."""
    dev = _same_device(dy, codes, scales)
    dt, ld = _dt(dy), _rows(dy, "dy")
    M, E = _act8(codes, scales)
    if dy.shape != (M, E):
        raise ValueError(f"dy has shape {tuple(dy.shape)}, the codes {(M, E)}")
    du = torch.empty(M, E, dtype=dy.dtype, device=dev)
    act = torch.empty(M, E, dtype=dy.dtype, device=dev) if want_act else None
    if M and E:
        _call("tc_dgelu_act8", dev, dt, dy.data_ptr(), ld, codes.data_ptr(), scales.data_ptr(), du.data_ptr(), _p(act), M, E)
    return (du, act) if want_act else du


def gemm_tn_act8(dy, codes, scales, out=None):
    """Weight gradient dy^T v -> f32 [N, K] of a linear layer whose input v [M, K] is kept in 8 bits (added to ``out`` when given);
    dy [M, N] bf16, rows may be strided; N a multiple of 8, K of 16.  tc_gemm_tn_act8."""
    dev = _same_device(dy, codes, scales, out)
    if dy.dtype != torch.bfloat16:
        raise TypeError(f"dy must be bfloat16, got {dy.dtype}")
    ld = _rows(dy, "dy")
    M, K = _act8(codes, scales)
    N = dy.shape[1]
    if dy.shape[0] != M:
        raise ValueError(f"dy has {dy.shape[0]} rows, the codes {M}")
    accumulate = out is not None
    if accumulate:
        _dense(out, "out", (N, K), torch.float32)
    elif M == 0:
        return torch.zeros(N, K, dtype=torch.float32, device=dev)
    else:
        out = torch.empty(N, K, dtype=torch.float32, device=dev)
    if M:
        need = _lib.load().tc_gemm_tn_act8_workspace_bytes(M, ld, N, K)
        ws = _scratch(need, out, dev)
        _call("tc_gemm_tn_act8", dev, dy.data_ptr(), ld, codes.data_ptr(), scales.data_ptr(), out.data_ptr(), M, N, K,
              int(accumulate), ws.data_ptr(), need)
    return out
