"""Embedding lookup with scaling and its gradient by sorted tokens, against the formulas in 64 bits."""
import pytest
import torch

from transcodon_amd import _lib, ops

DEV = "cuda"
gpu = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}      # half a step, relative to the value


def _ids(n, vocab, gen, kind):
    if kind == "even":
        return torch.randint(0, vocab, (n,), generator=gen)
    if kind == "one":                                             # every position the same id
        return torch.full((n,), vocab // 2)
    return (torch.exp(torch.rand(n, generator=gen, dtype=torch.float64) * torch.log(torch.tensor(vocab + 1.0))) - 1).long().clamp(
        0, vocab - 1)                                             # few frequent, many rare ids


def _want_grad(tok, dy, vocab, scale, pad):
    keep = (tok >= 0) & (tok < vocab)
    if pad is not None:
        keep &= tok != pad
    out = torch.zeros(vocab, dy.shape[1], dtype=torch.float64)
    out.index_add_(0, tok[keep], dy.double()[keep])
    size = torch.zeros(vocab, dy.shape[1], dtype=torch.float64)
    size.index_add_(0, tok[keep], dy.double()[keep].abs())
    n = torch.bincount(tok[keep], minlength=vocab)[:vocab].double()
    # a sum of n terms in f32, in any order, is off by at most (n - 1) 2^-24 sum|terms| to first order; times scale: one more
    return out * scale, (n[:, None] + 1) * 2.0 ** -24 * 1.01 * size * abs(scale) + 1e-37


@gpu
@pytest.mark.parametrize("tdt,odt", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                     (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("rows,vocab,width", [(1, 2, 1), (1, 1438, 768), (131, 10, 768), (257, 1000, 770), (70, 33, 4096),
                                              (4099, 70000, 24), (5, 3, 12)])
@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_lookup(tdt, odt, rows, vocab, width, idt):
    gen = torch.Generator().manual_seed(rows * 7 + width)
    tok = _ids(rows, vocab, gen, "few")
    table = torch.randn(vocab, width, generator=gen).to(tdt)
    scale = 27.7128
    got = ops.embedding(tok.to(idt).to(DEV), table.to(DEV), scale, pad_idx=1, out_dtype=odt).cpu()
    want = table.double()[tok] * float(torch.tensor(scale))       # the call's scale is an f32
    want[tok == 1] = 0
    assert got.dtype == odt and got.shape == (rows, width)
    err = (got.double() - want).abs()
    assert bool((err <= want.abs() * (HALF[odt] + 2.0 ** -24) * 1.001).all())
    assert bool((got[tok == 1] == 0).all())


@gpu
def test_lookup_flags_ids_out_of_range():
    table = torch.full((5, 8), float("nan"), device=DEV)
    table[2:] = 1.0
    big = 2 ** 32 + 2                                             # would name row 2 if its upper half were dropped
    for ids, flag in (([2, 3, 4], 0), ([2, 5], 1), ([-1, 2], 1), ([big, 2], 1), ([9, 2], 0)):
        bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = ops.embedding(torch.tensor(ids, device=DEV), table, 2.0, pad_idx=9, bad=bad).cpu()
        assert int(bad) == flag
        want = torch.tensor([[2.0 if 2 <= i < 5 else 0.0] * 8 for i in ids])
        assert torch.equal(out, want), ids


@gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,width", [
    (1, 1, 1), (1, 1438, 768), (2, 2, 4), (63, 10, 768), (64, 10, 768), (65, 10, 768), (128, 3, 256), (129, 1, 260), (1023, 1438, 770),
    (1024, 255, 96), (1025, 256, 33), (4096, 511, 64), (5000, 512, 64), (256, 50, 260), (257, 50, 260), (511, 9, 65), (512, 300, 128), (513, 300, 128), (700, 524286, 4), (700, 524287, 4), (700, 524288, 4),
    (4097, 40, 8), (8191, 1000, 512), (8192, 70000, 12), (8193, 70000, 12), (9001, 70000, 40), (20000, 10, 768), (140000, 600, 8), (600000, 5000, 4), (2500000, 3, 1), (300000, 300000, 4)])
@pytest.mark.parametrize("kind", ["even", "one", "few"])
def test_gradient(dt, rows, vocab, width, kind):
    gen = torch.Generator().manual_seed(rows + 3 * width)
    tok = _ids(rows, vocab, gen, kind)
    dy = torch.randn(rows, width, generator=gen).to(dt)
    pad = 1 if vocab > 2 else None
    want, tol = _want_grad(tok, dy, vocab, 0.5, pad)
    for idt in (torch.int32, torch.int64):
        got = ops.embedding_bwd(tok.to(idt).to(DEV), dy.to(DEV), vocab, 0.5, pad_idx=pad)
        assert got.dtype == torch.float32 and got.shape == (vocab, width)
        assert bool(((got.cpu().double() - want).abs() <= tol).all())
        again = ops.embedding_bwd(tok.to(idt).to(DEV), dy.to(DEV), vocab, 0.5, pad_idx=pad)
        assert torch.equal(got, again)


@gpu
def test_gradient_leaves_out_padding_and_ids_out_of_range():
    gen = torch.Generator().manual_seed(5)
    rows, vocab, width = 700, 20, 132
    tok = torch.randint(-2, vocab + 2, (rows,), generator=gen)
    tok[400:] = 1
    dy = torch.randn(rows, width, generator=gen)
    dy[400:] = float("nan")                                       # padding
    dy[(tok < 0) | (tok >= vocab)] = float("inf")
    want, tol = _want_grad(tok, torch.nan_to_num(dy, nan=0.0, posinf=0.0), vocab, 3.0, 1)
    got = ops.embedding_bwd(tok.to(DEV), dy.to(DEV), vocab, 3.0, pad_idx=1).cpu()
    assert bool(((got.double() - want).abs() <= tol).all())
    # nothing but padding: every row is written, and is zero
    got = ops.embedding_bwd(torch.ones(700, dtype=torch.int64, device=DEV), dy.to(DEV), vocab, 3.0, pad_idx=1)
    assert bool((got == 0).all())


@gpu
def test_gradient_adds_to_a_given_buffer_and_takes_strided_rows():
    gen = torch.Generator().manual_seed(6)
    rows, vocab, width = 333, 40, 64
    tok = torch.randint(0, vocab - 5, (rows,), generator=gen)
    wide = torch.randn(rows, width + 8, generator=gen)
    for first in (0, 3, 8):                                       # 3: rows no 16-byte load fits
        dy = wide[:, first:first + width]
        want, tol = _want_grad(tok, dy, vocab, 1.0, None)
        base = torch.randn(vocab, width, generator=gen)
        out = base.to(DEV)
        got = ops.embedding_bwd(tok.to(DEV), wide.to(DEV)[:, first:first + width], vocab, out=out)
        assert got.data_ptr() == out.data_ptr()
        total = base.double() + want
        assert bool(((got.cpu().double() - total).abs() <= tol + total.abs() * 2.0 ** -23).all())
        assert torch.equal(got.cpu()[vocab - 5:], base[vocab - 5:])        # rows that no token names


@gpu
@pytest.mark.parametrize("rows", [50, 333, 6000])
def test_gradient_into_a_buffer_that_is_aligned_to_a_value_only(rows):
    gen = torch.Generator().manual_seed(rows)
    vocab, width = 40, 64
    tok, dy = torch.randint(0, vocab, (rows,), generator=gen).to(DEV), torch.randn(rows, width, generator=gen).to(DEV)
    want = ops.embedding_bwd(tok, dy, vocab)
    store = torch.full((vocab * width + 9,), 5.0, device=DEV)
    out = store[3:3 + vocab * width].view(vocab, width)
    out.zero_()
    assert torch.equal(ops.embedding_bwd(tok, dy, vocab, out=out), want)
    assert bool((store[:3] == 5).all()) and bool((store[3 + vocab * width:] == 5).all())
    table = store[3:3 + vocab * width].view(vocab, width)
    assert torch.equal(ops.embedding(tok, table), table[tok])


@gpu
def test_gradient_is_that_of_differences():
    """The lookup is linear in its table: moving one entry by d moves <dy, out> by d * gradient."""
    gen = torch.Generator().manual_seed(7)
    tok = torch.randint(0, 9, (50,), generator=gen).to(DEV)
    table = torch.randn(9, 16, generator=gen).to(DEV)
    dy = torch.randn(50, 16, generator=gen).to(DEV)
    grad = ops.embedding_bwd(tok, dy, 9, 1.5, pad_idx=4)
    loss = lambda t: float((ops.embedding(tok, t, 1.5, pad_idx=4).double() * dy.double()).sum())
    for v, c in ((0, 0), (4, 3), (8, 15)):
        up, down = table.clone(), table.clone()
        up[v, c] += 1.0
        down[v, c] -= 1.0
        slope = (loss(up) - loss(down)) / 2
        # out differs from exact by 2^-24 a value, |out| < 8 over 50 rows: 50 * 8 * 2^-24 * |dy| < 1e-4
        assert abs(slope - float(grad[v, c])) < 1e-4


@gpu
def test_empty_calls():
    table = torch.randn(4, 8, device=DEV)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    assert ops.embedding(none, table).shape == (0, 8)
    assert torch.equal(ops.embedding_bwd(none, torch.zeros(0, 8, device=DEV), 4), torch.zeros(4, 8, device=DEV))


@gpu
def test_refusals():
    tok = torch.zeros(4, dtype=torch.int64, device=DEV)
    table, dy = torch.zeros(3, 8, device=DEV), torch.zeros(4, 8, device=DEV)
    with pytest.raises(TypeError):
        ops.embedding(tok.to(torch.int16), table)
    with pytest.raises(TypeError):
        ops.embedding(tok, table.half())
    with pytest.raises(ValueError):
        ops.embedding(tok, table.t())
    with pytest.raises(ValueError):
        ops.embedding(torch.zeros(4, 2, dtype=torch.int64, device=DEV)[:, 0], table)
    with pytest.raises(ValueError):
        ops.embedding_bwd(tok[:3], dy, 3)
    with pytest.raises(ValueError):
        ops.embedding_bwd(tok, dy.t().contiguous().t(), 3)
    with pytest.raises(ValueError):
        ops.embedding_bwd(tok, dy, 3, out=torch.zeros(4, 8, device=DEV))
    for call in (lambda: ops.embedding(tok, table, pad_idx=-1), lambda: ops.embedding_bwd(tok, dy, 3, pad_idx=-1),
                 lambda: ops.embedding_bwd(tok, dy[:1].expand(4, 8), 3)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_lib.HipLibraryError):
        ops.embedding_bwd(tok, dy, 0)


def test_refusals_without_a_gpu():
    lib = _lib.load()
    one = 1 << 12                                                 # any aligned non-null address: refused before it is used
    for args in ((0, 0, 4, None, one, one, 4, 8, 3), (0, 7, 4, one, one, one, 4, 8, 3), (0, 0, 2, one, one, one, 4, 8, 3),
                 (0, 0, 4, one, one, one, 0, 8, 3), (0, 0, 4, one, one, one, 4, 8, 0), (0, 0, 4, one, one + 2, one, 4, 8, 3),
                 (0, 0, 4, one, one, one, 2 ** 33, 8, 3), (0, 0, 4, one, one, one, 4, 65537, 3)):
        assert lib.tc_embedding_fwd(*args, 1.0, -1, None, None) == -1, args
        assert lib.tc_last_error()
    assert lib.tc_embedding_bwd_workspace_bytes(0, 8, 3) == 0 and lib.tc_embedding_bwd_workspace_bytes(4, 8, 2 ** 40) == 0
    need = lib.tc_embedding_bwd_workspace_bytes(4, 8, 3)
    assert need > 0
    bwd = lambda dt=0, idb=4, tok=one, dy=one, ld=8, out=one, M=4, E=8, V=3, ws=one, n=need: lib.tc_embedding_bwd(
        dt, idb, tok, dy, ld, out, M, E, V, 1.0, -1, 0, ws, n, None)
    assert bwd(dt=3) == bwd(idb=1) == bwd(tok=None) == bwd(ld=7) == bwd(out=one + 2) == bwd(M=0) == bwd(V=0) == bwd(ws=one + 4) == -1
    assert bwd(n=need - 1) == -3
    with pytest.raises(_lib.HipLibraryError):
        ops.embedding(torch.zeros(4, dtype=torch.int64), torch.zeros(3, 8))


@gpu
@pytest.mark.parametrize("rows", [100, 600])
def test_rows_without_a_position_are_zeros_for_any_scale(rows):
    tok = torch.full((rows,), 3, device=DEV)
    got = ops.embedding_bwd(tok, torch.ones(rows, 8, device=DEV), 6, scale=float("inf"))
    want = torch.zeros(6, 8, device=DEV)
    want[3] = float("inf")
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("pad", [None, 1])
def test_the_smallest_ids_are_flagged_and_left_out(pad):
    """The ends of the id types (what a bad conversion from a float leaves) are out of range like any other, with and without
    a padding id."""
    table = torch.ones(5, 8, device=DEV)
    for idt in (torch.int32, torch.int64):
        ends = torch.iinfo(idt)
        for odd in (ends.min, ends.min + 1, -2, -1, 5, ends.max):
            ids = torch.tensor([2, odd, 3], dtype=idt, device=DEV)
            bad = torch.zeros(1, dtype=torch.int32, device=DEV)
            out = ops.embedding(ids, table, 2.0, pad_idx=pad, bad=bad).cpu()
            assert int(bad) == 1, (idt, odd)
            assert torch.equal(out, torch.tensor([2.0, 0.0, 2.0])[:, None].expand(3, 8))
            for rows in (3, 600):                                 # without and with a sort
                dy = torch.ones(rows, 8, device=DEV)
                got = ops.embedding_bwd(ids.repeat(rows // 3), dy, 5, 1.0, pad_idx=pad).cpu()
                assert torch.equal(got[:, 0], torch.tensor([0.0, 0.0, rows / 3, rows / 3, 0.0])), (idt, odd, rows)


@gpu
def test_any_negative_padding_id_stands_for_none():
    """tc_embedding_fwd: pad_idx < 0 is no padding id, so an id of that very value is out of range."""
    lib, table = _lib.load(), torch.ones(5, 8, device=DEV)
    for pad in (-1, -7, -2 ** 63):
        ids = torch.tensor([2, pad], device=DEV)
        bad, out = torch.zeros(1, dtype=torch.int32, device=DEV), torch.full((2, 8), 3.0, device=DEV)
        assert lib.tc_embedding_fwd(0, 0, 8, ids.data_ptr(), table.data_ptr(), out.data_ptr(), 2, 8, 5, 1.0, pad, bad.data_ptr(),
                                    torch.cuda.current_stream().cuda_stream) == 0
        assert int(bad) == 1 and torch.equal(out.cpu(), torch.tensor([1.0, 0.0])[:, None].expand(2, 8))
