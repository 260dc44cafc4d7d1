"""Training with 8-bit activation checkpoints (model.act8_checkpoints): the same forward pass, less memory, gradients near those of the
bf16 checkpoints."""
import ctypes as C
import dataclasses

import pytest
import torch

import transcodon_amd as ta
from oracle import transcodon_ref as O
from oracle.weights import seeded_state_dict
from transcodon_amd import _lib
from transcodon_amd import train as TR

DEV = "cuda"
gpu = pytest.mark.gpu


def _model(cfg, seed=11, dtype=torch.bfloat16):
    args = ta.default_args(num_layers=cfg.num_layers, embed_dim=cfg.embed_dim, ffn_embed_dim=cfg.ffn_embed_dim,
                           attention_heads=cfg.attention_heads, species_vocab_size=cfg.species_vocab_size)
    m = ta.ProteinBertModel(args, ta.Alphabet.from_architecture("CodonModel"))
    m.load_state_dict(seeded_state_dict(cfg, seed, perturb=True), strict=True)
    return m.to(DEV).train().set_compute_dtype(dtype)


def _batch(cfg, B, T, seed=5):
    gen = torch.Generator().manual_seed(seed)
    tok = torch.randint(5, 9, (B, T), generator=gen)
    labels = torch.where(torch.rand(B, T, generator=gen) < 0.25, tok, torch.full_like(tok, -100))
    tok = torch.where((labels >= 0) & (torch.rand(B, T, generator=gen) < 0.8), torch.full_like(tok, 9), tok)
    tok[:, 0] = 0
    tok[-1, T - T // 4:] = 1                                      # padded tail
    labels[-1, T - T // 4:] = -100
    struct = torch.randint(0, 3, (B, T), generator=gen)
    struct[tok == 1] = -100
    sp = torch.randint(0, cfg.species_vocab_size, (B,), generator=gen)
    return [t.to(DEV) for t in (tok, sp, labels, struct)]


def _step(m, batch, act8, switch=None):
    tok, sp, labels, struct = batch
    m.act8_checkpoints = act8
    for p in m.parameters():
        p.grad = None
    out = m(tok, sp)
    if switch is not None:
        m.act8_checkpoints = switch
    loss = TR.mlm_loss(out["logits"], labels, out["struct_label_output"], struct)
    loss.backward()
    return out["logits"].detach().clone(), float(loss.detach()), {k: p.grad.clone() for k, p in m.named_parameters() if p.grad is not None}


@gpu
@pytest.mark.parametrize("B,T", [(3, 40), (1, 1), (2, 131), (5, 64)])
def test_gradients_are_near_those_of_bf16_checkpoints(B, T):
    """What enters a weight gradient in 8 bits is off by at most 2^-4 of itself (2^-4 / sqrt 3 in the mean square), gelu' by at
    most max |u gelu''(u)| 2^-4 < 2^-5 of dy for each layer above; terms of random sign keep that share of the sum's norm, so 0.12 in the 2-norm
    covers two layers.  (One token alone is left out: every sum is one term and LayerNorm's projections cancel it.)"""
    m = _model(O.TINY)
    batch = _batch(O.TINY, B, T)
    if T == 1:
        batch[2][:] = 5
        batch[0][:] = 9
    logits16, loss16, want = _step(m, batch, False)
    logits8, loss8, got = _step(m, batch, True)
    assert torch.equal(logits8, logits16)                         # the forward pass computes the same values
    assert abs(loss8 - loss16) <= B * T * 2.0 ** -24 * abs(loss16)         # (the loss is summed with atomics, in any order)
    assert set(got) == set(want)
    for k, w in want.items():
        assert bool(torch.isfinite(got[k]).all()), k
        if T > 1:
            off = float((got[k] - w).norm() / (w.norm() + 1e-12))
            assert off <= 0.12, (k, off)
    again = _step(m, batch, True, switch=False)[2]                # the switch moved between the passes: the forward's holds
    for k, w in got.items():
        assert float((again[k] - w).norm()) <= 1e-4 * float(w.norm()) + 1e-12, k
    back = _step(m, batch, False)[2]
    for k, w in want.items():                                     # and bf16 checkpoints are as before
        assert float((back[k] - w).norm()) <= 1e-4 * float(w.norm()) + 1e-12, k


@gpu
def test_with_a_parameter_store():
    m = _model(O.TINY)
    batch = _batch(O.TINY, 3, 40)
    want = _step(m, batch, True)[2]
    store = TR.FlatParameters(m)
    opt = TR.AdamW(store)
    store.zero_grad()
    tok, sp, labels, struct = batch
    m.act8_checkpoints = True
    out = m(tok, sp)
    TR.mlm_loss(out["logits"], labels, out["struct_label_output"], struct).backward()
    for k, p in m.named_parameters():
        if k in want:
            assert float((p.grad - want[k]).norm()) <= 1e-4 * float(want[k].norm()) + 1e-12, k
    opt.step()
    assert bool(torch.isfinite(store.data).all())


@gpu
def test_f32_is_refused():
    m = _model(O.TINY, dtype=torch.float32)
    m.act8_checkpoints = True
    tok, sp, _, _ = _batch(O.TINY, 2, 16)
    with pytest.raises(ValueError):
        m(tok, sp)
    m.act8_checkpoints = False
    assert bool(torch.isfinite(m(tok, sp)["logits"]).all())


def test_workspace_is_smaller():
    """12 layers of 768 / 3072, 64 x 1024 tokens: 36 E bytes a token and layer with bf16 checkpoints, 22.2 E with 8-bit ones."""
    lib = _lib.load()
    d = _lib.EncoderDesc()
    d.dtype, d.num_layers, d.E, d.F, d.H = _lib.TC_BF16, 12, 768, 4 * 768, 12
    d.vocab, d.n_species, d.n_struct = 10, 1438, 3
    size = {}
    for d.act8 in (0, 1):
        size[d.act8] = lib.tc_train_workspace_bytes(C.byref(d), 64, 1024)
    saved = size[0] - size[1]
    tokens = 12 * 64 * 1024
    assert abs(saved - tokens * (36 - 22.1875) * 768 - tokens * 256) < 2 ** 20 * 64       # the rows' 128-byte gaps; split-sum buffers
    d.dtype = _lib.TC_F32
    assert lib.tc_train_workspace_bytes(C.byref(d), 64, 1024) == 0


ABOVE = ("lm_head.", "structure_linear.", "emb_layer_norm_after.")            # no 8-bit value on the way to these


def _gradients_change_where_they_should(cfg, B, T):
    m = _model(cfg)
    batch = _batch(cfg, B, T)
    logits16, _, want = _step(m, batch, False)
    logits8, _, got = _step(m, batch, True)
    assert torch.equal(logits8, logits16)
    assert set(got) == set(want)
    off = {k: float((got[k] - w).norm() / (w.norm() + 1e-12)) for k, w in want.items()}
    top = f"layers.{cfg.num_layers - 1}.fc2.bias"
    assert top in off
    for k, d in off.items():
        assert bool(torch.isfinite(got[k]).all()), k
        if k.startswith(ABOVE) or k == top:
            assert d <= 1e-4, (k, d)                              # additions by atomics, in any order
        else:
            assert d <= 0.12, (k, d)                              # as derived above for two layers
        if k.startswith("layers.") and k.endswith(("q_proj.weight", "k_proj.weight", "v_proj.weight", "fc1.weight", "fc2.weight")):
            assert d > 2e-4, (k, d)                               # 8-bit values did enter: more than the atomics explain


@gpu
@pytest.mark.parametrize("B,T", [(3, 40), (5, 64), (2, 131)])
def test_gradients_change_where_the_8_bit_values_enter(B, T):
    _gradients_change_where_they_should(O.TINY, B, T)


@gpu
@pytest.mark.parametrize("B,T", [(7, 1171), (5, 500)])
def test_one_layer_of_full_width(B, T):
    """Enough rows for the weight gradients' 256 x 256 tiles in several parts, with rows behind the last whole stage (8197 = 128 * 64 + 5),
    beside the buffers that they share with the rest of the step; 2500 rows take the small tiles."""
    _gradients_change_where_they_should(dataclasses.replace(O.FULL, num_layers=1), B, T)
