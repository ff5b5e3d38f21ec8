"""Scaled lookup, dropout and the gradient of token embeddings on the GPU against their restatement in 64 bits.

Tolerances count roundings.  A value is input * factor (the factor rounded to fp32, the product rounded to fp32: 2^-24
each) and then rounded to its type (half a step: eps / 2, and half of the smallest subnormal).  A sum of m terms in any order
is within (m - 1) 2^-24 of the sum of their magnitudes."""
import math

import numpy as np
import pytest
import torch

from oracle import token_oracle as oracle

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ROUND = 2.0 ** -24
TINY = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}


@pytest.fixture(scope="module")
def E(cuda_lib):
    from hades_b200 import EmbCacheLib

    return EmbCacheLib


def status():
    from hades_b200 import _lib

    return _lib.device_status()


def f64(t):
    return t.detach().double().cpu().numpy()


def rows_like(rng, shape, dtype, sigma=1.0):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * sigma).to(dtype).cuda()


def close(got, want, dtype, size=None, terms=0):
    """size: sum of the magnitudes of the terms of a sum of so many."""
    size = np.abs(want) if size is None else size
    bound = (2 * ROUND + np.maximum(terms - 1, 0) * ROUND) * size
    bound = bound * (1 + 2.0 ** -20) + torch.finfo(dtype).eps / 2 * (np.abs(want) + bound) + TINY[dtype]
    got = f64(got).reshape(want.shape)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])


# ---- lookup -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [1, 7, 8, 9, 64, 100, 250, 1001, 1024, 8200])
@pytest.mark.parametrize("wt,ot", [(F32, F32), (F16, F32), (BF16, BF16), (F32, BF16), (F16, F16), (BF16, F16)])
def test_lookup(E, dim, wt, ot):
    rng = np.random.default_rng(dim)
    w = rows_like(rng, (53, dim), wt)
    for n, idt, pad, p in ((1, torch.int64, None, 0.0), (2, torch.int32, None, 0.4), (33, torch.int64, 5, 0.1),
                           (1000, torch.int64, -1, 0.0), (700, torch.int32, -1, 0.25)):
        ids = rng.integers(0, 53, n)
        if pad is not None:
            ids[rng.random(n) < 0.3] = pad
        out = E.cudaEmbedding(w, torch.from_numpy(ids).to(idt).cuda(), 1.5, pad, p, seed=11, offset=n, dtype=ot)
        assert out.dtype == ot and out.shape == (n, dim)
        close(out, oracle.embedding(f64(w), ids, padding_idx=pad, scale=1.5, p=p, seed=11, offset=n), ot)
    assert status() == 0


def test_lookup_without_change_is_a_copy(E):
    for t in (F32, F16, BF16):
        w = torch.randn(100, 96, device="cuda").to(t)
        ids = torch.randint(0, 100, (4, 5, 3), device="cuda")
        assert torch.equal(E.cudaEmbedding(w, ids), w[ids])
        assert E.cudaEmbedding(w, ids[:0]).shape == (0, 5, 3, 96)
        assert torch.equal(E.cudaEmbedding(w, ids[0, 0, 0]), w[ids[0, 0, 0]])  # one token


@pytest.mark.parametrize("n", [3, 5000])
@pytest.mark.parametrize("first,dim,wide", [(1, 64, 80), (2, 63, 72), (4, 40, 44), (8, 128, 136), (3, 1001, 1010)])
@pytest.mark.parametrize("t", [F32, BF16])
def test_lookup_of_rows_at_a_distance(E, n, first, dim, wide, t):
    rng = np.random.default_rng(first)
    base, ids = rows_like(rng, (41, wide), t), rng.integers(0, 41, n)
    w, given = base[:, first:first + dim], torch.from_numpy(ids).cuda()
    out = torch.full((n, wide), 7.0, dtype=t, device="cuda")
    back = E.cudaEmbedding(w, given, 2.0, dropout=0.2, seed=1, offset=2, out=out[:, first:first + dim])
    assert back.data_ptr() == out[:, first:].data_ptr()
    close(back, oracle.embedding(f64(w), ids, scale=2.0, p=0.2, seed=1, offset=2), t)
    assert bool((out[:, :first] == 7).all()) and bool((out[:, first + dim:] == 7).all())
    spread = torch.empty(2 * n, dtype=torch.int64, device="cuda")[::2].copy_(given)
    assert torch.equal(E.cudaEmbedding(w, spread, 2.0), E.cudaEmbedding(w, given, 2.0))


def test_lookup_of_a_pinned_table(E):
    w = torch.randn(20, 40).pin_memory()
    ids = torch.randint(0, 20, (100,), device="cuda")
    assert torch.equal(E.cudaEmbedding(w, ids, 2.0).cpu(), 2 * w[ids.cpu()])


def test_ids_outside_of_the_table(E):
    w = torch.randn(10, 24, device="cuda")
    ids = torch.tensor([3, 10, -1, 9, 1 << 40, -(1 << 62)], device="cuda")
    g = torch.randn(6, 24, device="cuda")
    assert status() == 0
    out = E.cudaEmbedding(w, ids)
    assert status() == 1
    assert torch.equal(out[[0, 3]], w[[3, 9]]) and not out[[1, 2, 4, 5]].any()
    grad = E.cudaEmbeddingGrad(ids, g, 10)
    assert status() == 1
    want = torch.zeros(10, 24, device="cuda")
    want[3], want[9] = g[0], g[3]
    assert torch.equal(grad, want)
    tokens, rows = E.cudaEmbeddingGradRows(ids, g, 10)
    assert status() == 1 and tokens.tolist() == [3, 9] and torch.equal(rows, g[[0, 3]])
    # as padding they are nothing unusual
    ids = torch.tensor([3, -1, -1, 9], device="cuda")
    E.cudaEmbedding(w, ids, padding_idx=-1)
    E.cudaEmbeddingGrad(ids, g[:4], 10, padding_idx=-1)
    # an empty table has no rows for any id
    assert not E.cudaEmbedding(w[:0], ids, padding_idx=-1).any() and status() == 1
    assert E.cudaEmbeddingGrad(ids, g[:4], 0, padding_idx=-1).shape == (0, 24) and status() == 1


def test_a_table_beyond_32_bits(E):
    # 2.6e9 values: the last rows lie more than 2^32 bytes and 2^31 values behind the first
    rows, dim = 640_000, 4096
    w = torch.zeros((rows, dim), dtype=BF16, device="cuda")
    w[-3:] = torch.randn(3, dim, device="cuda").to(BF16)
    ids = torch.tensor([rows - 1, rows - 3, 0, rows - 2], device="cuda")
    out = E.cudaEmbedding(w, ids)
    assert torch.equal(out, w[ids])
    grad = E.cudaEmbeddingGrad(ids, out, rows, out=w, accumulate=True)
    assert torch.equal(grad[ids], 2 * out) and not grad[1:1000].any()


# ---- dropout ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("n,dim", [(1, 1), (1, 4097), (5, 8), (300, 100), (77, 1001), (4099, 64), (600, 2048)])
def test_dropout(E, n, dim, t):
    rng = np.random.default_rng(n + dim)
    x = rows_like(rng, (n, dim), t)
    for p, seed, offset in ((0.1, 1, 1), (0.5, (1 << 64) - 1, 1 << 33), (0.999, 1 << 40, (1 << 64) - 5), (1e-9, 3, 4)):
        y = E.cudaDropout(x, p, seed, offset, scale=0.75)
        close(y, oracle.dropped(f64(x), 0.75, p, seed, offset), t)
        kept = oracle.kept(n, dim, p, seed, offset)
        assert np.array_equal((y != 0).cpu().numpy(), kept & (f64(x) != 0))
    assert torch.equal(E.cudaDropout(x, 0.0), x)
    assert not E.cudaDropout(x, 1.0).any()


def test_dropped_values_are_zeros_whatever_they_were(E):
    x = torch.full((64, 48), math.nan, device="cuda")
    x[::2] = math.inf
    keep = torch.from_numpy(oracle.kept(64, 48, 0.5, 9, 9)).cuda()
    for t in (F32, F16, BF16):
        y = E.cudaDropout(x.to(t), 0.5, 9, 9)
        assert not y[~keep].any() and not torch.signbit(y[~keep]).any() and not torch.isfinite(y[keep]).any()
        w = E.cudaEmbedding(x.to(t), torch.arange(64, device="cuda"), dropout=0.5, seed=9, offset=9)
        assert torch.equal(w.nan_to_num(5.0), y.nan_to_num(5.0))
    ids = torch.zeros(64, dtype=torch.int64, device="cuda")
    g = torch.where(keep, 1.0, math.nan)  # NaN only where values are dropped
    grad = E.cudaEmbeddingGrad(ids, g, 2, dropout=0.5, seed=9, offset=9)
    assert torch.equal(grad[0], 2.0 * keep.sum(0)) and not grad[1].any()
    # and of padding, whatever its rows and gradients hold
    ids[:] = 1
    assert not E.cudaEmbedding(x, ids, padding_idx=1).any()
    assert not E.cudaEmbeddingGrad(ids, x, 2, padding_idx=1).any()


def test_dropout_in_place_and_of_other_shapes(E):
    x = torch.randn(30, 7, 72, device="cuda").to(BF16)
    want = E.cudaDropout(x, 0.3, 5, 6)
    assert torch.equal(want.view(210, 72), E.cudaDropout(x.view(210, 72), 0.3, 5, 6))
    assert torch.equal(want[0], E.cudaDropout(x[0], 0.3, 5, 6))  # rows count from the first
    y = x.clone()
    assert E.cudaDropout(y, 0.3, 5, 6, out=y) is not None and torch.equal(y, want)
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)  # rows in another order: copied
    assert torch.equal(E.cudaDropout(turned, 0.3, 5, 6), want)
    lone = torch.randn(72, device="cuda")
    assert torch.equal(E.cudaDropout(lone, 0.3, 5, 6), E.cudaDropout(lone[None], 0.3, 5, 6)[0])
    row = torch.randn(1, 72, device="cuda").expand(30, 72)  # one row for all
    assert torch.equal(E.cudaDropout(row, 0.3, 5, 6), E.cudaDropout(row.contiguous(), 0.3, 5, 6))
    wide = torch.randn(30, 80, device="cuda")
    kept = wide.clone()
    E.cudaDropout(wide[:, 3:75], 0.3, 5, 6, out=wide[:, 3:75])
    assert torch.equal(wide[:, 3:75], E.cudaDropout(kept[:, 3:75].contiguous(), 0.3, 5, 6))
    assert torch.equal(wide[:, :3], kept[:, :3]) and torch.equal(wide[:, 75:], kept[:, 75:])
    assert E.cudaDropout(x[:0], 0.3).shape == (0, 7, 72)
    assert E.cudaDropout(x, 0.3, 5, 6, dtype=F32).dtype == F32


def test_more_rows_than_a_launch_counts(E):
    n = (1 << 31) + 1001  # blocks of one launch count in 31 bits, rows of a mask in 32
    if torch.cuda.mem_get_info()[0] < 3 * 16 * n:
        pytest.skip("needs some 100 GB")
    x = torch.ones((n, 8), dtype=BF16, device="cuda")
    E.cudaDropout(x, 0.5, 3, 4, out=x)
    for row in (0, 5, (1 << 31) - 1, 1 << 31, n - 1):
        words = oracle.philox4x32((0, row, 4, 0), (3, 0))
        draws = np.array([int(w) >> s & 0xFFFF for w in words for s in (0, 16)])
        assert np.array_equal(f64(x[row]), np.where(draws >= 32768, 2.0, 0.0))
    del x
    torch.cuda.empty_cache()


def test_numbers_on_the_device(E):
    x = torch.randn(100, 64, device="cuda")
    for seed, offset in ((1, 2), (-1, -2), (1 << 62, 1 << 40)):
        rng = torch.tensor([seed, offset], device="cuda")
        mask = {"seed": seed % (1 << 64), "offset": offset % (1 << 64)}
        assert torch.equal(E.cudaDropout(x, 0.5, rng=rng), E.cudaDropout(x, 0.5, **mask))
        ids = torch.arange(100, device="cuda")
        assert torch.equal(E.cudaEmbedding(x, ids, dropout=0.5, rng=rng), E.cudaDropout(x, 0.5, **mask))
        assert torch.equal(E.cudaEmbeddingGrad(ids, x, 100, dropout=0.5, rng=rng), E.cudaDropout(x, 0.5, **mask))


# ---- gradient ---------------------------------------------------------------------------------------------------------------
def tokens_of(rng, kind, n, vocab):
    if kind == "one":
        return np.full(n, vocab - 1)
    if kind == "distinct":
        return rng.permutation(max(n, vocab))[:n] % vocab
    return np.minimum(vocab - 1, (rng.pareto(0.7, n) * 3).astype(np.int64))


def check_grad(E, ids, g, vocab, ot=F32, pad=None, idt=torch.int64, **drop):
    given = torch.from_numpy(np.asarray(ids)).to(idt).cuda()
    want, size, terms = oracle.embedding_grad(ids, f64(g), vocab, padding_idx=pad, **drop)
    call = {"scale": drop.get("scale", 1.0), "padding_idx": pad, "dropout": drop.get("p", 0.0), "seed": drop.get("seed", 0),
            "offset": drop.get("offset", 0)}
    dense = E.cudaEmbeddingGrad(given, g, vocab, dtype=ot, **call)
    close(dense, want, ot, size, terms[:, None])
    assert not dense[torch.from_numpy(terms == 0).cuda()].any()
    tokens, rows = E.cudaEmbeddingGradRows(given, g, vocab, **call)
    present = np.flatnonzero(terms)
    assert np.array_equal(tokens.cpu().numpy(), present) and rows.dtype == F32
    close(rows, want[present], F32, size[present], terms[present][:, None])
    full = E.cudaEmbeddingGradRows(given, g, vocab, sync=False, **call)
    u = int(full[2].item())
    assert u == present.size and torch.equal(full[0][:u], tokens) and torch.equal(full[1][:u], rows)
    # added to a gradient that is there: rows of other tokens as they were
    start = torch.randn(vocab, g.shape[-1], device="cuda").to(ot)
    both = E.cudaEmbeddingGrad(given, g, vocab, out=start.clone(), accumulate=True, **call)
    close(both, want + f64(start), ot, size + np.abs(f64(start)), terms[:, None] + 1)
    rest = torch.from_numpy(terms == 0).cuda()
    assert torch.equal(both[rest], start[rest])
    # the same bits every time
    assert torch.equal(dense, E.cudaEmbeddingGrad(given, g, vocab, dtype=ot, **call))
    assert status() == 0


@pytest.mark.parametrize("kind", ["one", "distinct", "zipf"])
@pytest.mark.parametrize("n,dim,vocab", [(1, 1, 1), (1, 40, 9), (2, 9, 3), (7, 64, 5), (8, 256, 100), (9, 250, 100), (255, 257, 64),
                                         (513, 100, 1000), (1000, 1001, 300), (3000, 8, 50), (4097, 33, 5000), (2500, 512, 700)])
def test_grad(E, kind, n, dim, vocab):
    rng = np.random.default_rng(n)
    check_grad(E, tokens_of(rng, kind, n, vocab), rows_like(rng, (n, dim), F32), vocab, scale=3.0)


@pytest.mark.parametrize("times", [2, 8, 15, 16, 17, 32, 33, 300, 1000])
def test_grad_of_tokens_that_repeat(E, times):
    rng = np.random.default_rng(times)
    for n, dim in ((1900, 136), (1000, 72), (500, 1000), (3000, 300)):
        check_grad(E, rng.permutation(n) // times, rows_like(rng, (n, dim), BF16), n, scale=0.5)


@pytest.mark.parametrize("gt,ot", [(F32, BF16), (F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("n,dim", [(3, 17), (700, 320), (1500, 1002)])
def test_grad_of_types_with_dropout_and_padding(E, n, dim, gt, ot):
    rng = np.random.default_rng(dim)
    for kind, pad, idt in (("zipf", 0, torch.int32), ("zipf", -1, torch.int64), ("one", 0, torch.int64)):
        ids = tokens_of(rng, kind, n, 90)
        ids[rng.random(n) < 0.3] = pad
        check_grad(E, ids, rows_like(rng, (n, dim), gt), 90, ot, pad, idt, scale=0.5, p=0.2, seed=77, offset=n)


@pytest.mark.parametrize("kind", ["one", "zipf", "distinct"])
def test_grad_of_many_tokens(E, kind):
    # beyond what one cluster sorts; pieces of the sums in all lengths
    rng = np.random.default_rng(5)
    for n, dim in ((66_001, 24), (20_011, 264)):
        check_grad(E, tokens_of(rng, kind, n, 30_000), rows_like(rng, (n, dim), BF16), 30_000, p=0.1, seed=1, offset=1)


@pytest.mark.parametrize("n,dim,vocab,t", [(300, 1, 5000, F16), (77, 3, 700_000, F32), (500, 5, 9_001, BF16), (2048, 2, 40, F32),
                                           (100, 1024, 60_000, F32), (2048, 4096, 30, BF16), (2000, 4001, 30, F16)])
def test_grad_of_narrow_rows_and_large_tables(E, n, dim, vocab, t):
    """Both forms that few tokens can take, and zeros in rows of all widths."""
    rng = np.random.default_rng(dim)
    ids, g = rng.integers(0, vocab, n), rows_like(rng, (n, dim), t)
    out = torch.full((vocab, dim), math.nan, dtype=t, device="cuda")
    E.cudaEmbeddingGrad(torch.from_numpy(ids).cuda(), g, vocab, out=out)
    want, size, terms = oracle.embedding_grad(ids, f64(g), vocab)
    close(out, want, t, size, terms[:, None])
    # two rows, one of them written over by a single token, at every place of memory that rows can begin
    for first in range(1, 9):
        base = torch.full((3 * dim + 16,), 5.0, dtype=t, device="cuda")
        E.cudaEmbeddingGrad(torch.ones(1, dtype=torch.int64, device="cuda"), g[:1], 3, out=base[first:first + 3 * dim].view(3, dim))
        assert torch.equal(base[first:first + 3 * dim].view(3, dim)[1], g[0])
        assert not base[first:first + dim].any() and not base[first + 2 * dim:first + 3 * dim].any()
        assert bool((base[:first] == 5).all()) and bool((base[first + 3 * dim:] == 5).all())


def test_grad_of_tokens_of_any_size(E):
    rng = np.random.default_rng(9)
    for n in (50, 3000):
        ids = torch.from_numpy(rng.integers(0, 40, n) * (1 << 34) + 7).cuda()
        g = torch.randn(n, 48, device="cuda")
        tokens, rows = E.cudaEmbeddingGradRows(ids, g, 1 << 50, padding_idx=7)
        small, same = E.cudaEmbeddingGradRows((ids - 7) >> 34, g, 40, padding_idx=0)
        assert torch.equal(tokens, (small << 34) + 7)
        # (50 tokens take two forms, which add in another order: some six terms of at most 5 each, 6 * 30 * 2^-24 = 1.1e-5)
        torch.testing.assert_close(rows, same, rtol=0, atol=1.1e-5)
        assert status() == 0
        assert E.cudaEmbeddingGradRows(ids, g, 1 << 30, padding_idx=7)[0].numel() == 0 and status() == 1
        assert E.cudaEmbeddingGrad(ids, g, 0, padding_idx=7).shape == (0, 48) and status() == 1


@pytest.mark.parametrize("n", [700, 5000])
@pytest.mark.parametrize("dim,first", [(64, 8), (63, 3), (100, 4), (264, 1)])
@pytest.mark.parametrize("t", [F32, F16])
def test_grad_added_to_rows_at_a_distance(E, n, dim, first, t):
    rng = np.random.default_rng(n + dim)
    ids, g = tokens_of(rng, "zipf", n, 400), rows_like(rng, (n, dim), t, 0.25)
    base = rows_like(rng, (400, dim + 24), t)
    start, out = base.clone(), base[:, first:first + dim]
    E.cudaEmbeddingGrad(torch.from_numpy(ids).cuda(), g, 400, out=out, accumulate=True, dropout=0.25, seed=2, offset=3)
    want, size, terms = oracle.embedding_grad(ids, f64(g), 400, p=0.25, seed=2, offset=3)
    there = f64(start[:, first:first + dim])
    close(out, want + there, t, size + np.abs(there), terms[:, None] + 1)
    assert torch.equal(base[:, :first], start[:, :first]) and torch.equal(base[:, first + dim:], start[:, first + dim:])
    full = torch.full_like(base, 3.0)
    E.cudaEmbeddingGrad(torch.from_numpy(ids).cuda(), g, 400, out=full[:, first:first + dim])
    assert torch.equal(full[:, first:first + dim], E.cudaEmbeddingGrad(torch.from_numpy(ids).cuda(), g, 400))
    assert bool((full[:, :first] == 3).all()) and bool((full[:, first + dim:] == 3).all())


def test_grad_of_nothing(E):
    ids, g = torch.zeros(0, dtype=torch.int64, device="cuda"), torch.zeros(0, 32, device="cuda")
    assert not E.cudaEmbeddingGrad(ids, g, 10).any()
    tokens, rows = E.cudaEmbeddingGradRows(ids, g, 10)
    assert tokens.numel() == 0 and rows.shape == (0, 32)
    assert int(E.cudaEmbeddingGradRows(ids, g, 10, sync=False)[2].item()) == 0
    out = torch.randn(10, 32, device="cuda")
    assert torch.equal(E.cudaEmbeddingGrad(ids, g, 10, out=out.clone(), accumulate=True), out)
    # all of it padding
    ids, g = torch.full((100,), 3, device="cuda"), torch.randn(100, 32, device="cuda")
    assert not E.cudaEmbeddingGrad(ids, g, 10, padding_idx=3).any()
    assert E.cudaEmbeddingGradRows(ids, g, 10, padding_idx=3)[0].numel() == 0
    assert torch.equal(E.cudaEmbeddingGrad(ids, g, 10, padding_idx=3, out=out.clone(), accumulate=True), out)


def test_grad_strides(E):
    rng = np.random.default_rng(8)
    ids = torch.from_numpy(rng.integers(0, 40, (6, 50))).cuda()
    g = rows_like(rng, (6, 50, 96), F32)
    want = E.cudaEmbeddingGrad(ids, g, 40)
    assert torch.equal(want, E.cudaEmbeddingGrad(ids.flatten(), g.view(300, 96), 40))
    assert torch.equal(want, E.cudaEmbeddingGrad(ids, g.transpose(0, 1).contiguous().transpose(0, 1), 40))
    wide = torch.zeros(6, 50, 103, device="cuda")
    wide[..., 5:101] = g
    assert torch.equal(want, E.cudaEmbeddingGrad(ids, wide[..., 5:101], 40))
    one = torch.ones((), device="cuda").expand(6, 50, 96)  # what a sum's backward pass hands over
    count = torch.bincount(ids.flatten(), minlength=40).float()
    assert torch.equal(E.cudaEmbeddingGrad(ids, one, 40), count[:, None].expand(40, 96))
    row = torch.randn(96, device="cuda").expand(6, 50, 96)
    assert torch.allclose(E.cudaEmbeddingGrad(ids, row, 40), count[:, None] * row[0, 0], rtol=60 * ROUND, atol=0)
    out = torch.full((40, 110), 3.0, device="cuda")
    E.cudaEmbeddingGrad(ids, g, 40, out=out[:, 7:103])
    assert torch.equal(out[:, 7:103], want) and bool((out[:, :7] == 3).all()) and bool((out[:, 103:] == 3).all())


# ---- refusals that need tensors on the GPU ------------------------------------------------------------------------------------
def test_refusals(E):
    w, ids, g = torch.randn(8, 16, device="cuda"), torch.arange(4, device="cuda"), torch.randn(4, 16, device="cuda")
    out = torch.empty(4, 16, device="cuda")
    for bad in (lambda: E.cudaEmbedding(w.double(), ids), lambda: E.cudaEmbedding(w, ids.float()),
                lambda: E.cudaEmbedding(w, ids.short()), lambda: E.cudaEmbedding(w[0], ids),
                lambda: E.cudaEmbedding(w.t(), ids), lambda: E.cudaEmbedding(w.cpu(), ids), lambda: E.cudaEmbedding(w[:, :0], ids),
                lambda: E.cudaEmbedding(w, ids, dropout=1.1), lambda: E.cudaEmbedding(w, ids, scale=math.inf),
                lambda: E.cudaEmbedding(w, ids, out=out[:3]), lambda: E.cudaEmbedding(w, ids, out=out.t()),
                lambda: E.cudaEmbedding(w, ids, out=out, dtype=BF16), lambda: E.cudaEmbedding(w, ids, out=w[:4]),
                lambda: E.cudaEmbedding(w, ids, out=out[:1].expand(4, 16)), lambda: E.cudaEmbedding(w, ids, dtype=torch.int32),
                lambda: E.cudaEmbedding(w, ids, dropout=0.1, rng=torch.zeros(2, dtype=torch.int64)),
                lambda: E.cudaEmbedding(w, ids, dropout=0.1, rng=torch.zeros(3, dtype=torch.int64, device="cuda")),
                lambda: E.cudaEmbeddingGrad(ids, g[:3], 8), lambda: E.cudaEmbeddingGrad(ids, g.double(), 8),
                lambda: E.cudaEmbeddingGrad(ids, g, -1), lambda: E.cudaEmbeddingGrad(ids, g, 8, accumulate=True),
                lambda: E.cudaEmbeddingGrad(ids, g, 8, out=out), lambda: E.cudaEmbeddingGrad(ids, g, 4, out=g),
                lambda: E.cudaDropout(g, 0.1, out=g[:, :8]), lambda: E.cudaDropout(g.double(), 0.1),
                lambda: E.cudaDropout(g[:3], 0.1, out=g[1:]), lambda: E.cudaDropout(g, math.nan)):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: E.cudaEmbedding(w, ids, seed=-1), lambda: E.cudaDropout(g, 0.1, offset=1 << 64)):
        with pytest.raises((OverflowError, TypeError)):
            bad()
    with pytest.raises(TypeError):
        E.cudaEmbedding(w, [1, 2])
    assert status() == 0


# ---- autograd, layers, optimisers -----------------------------------------------------------------------------------------------
def test_autograd(E):
    from hades_b200 import token_emb

    rng = np.random.default_rng(3)
    ids = torch.from_numpy(rng.integers(0, 30, (4, 25))).cuda()
    for t in (F32, BF16):
        w = rows_like(rng, (30, 80), t).requires_grad_()
        call = {"scale": 2.0, "padding_idx": 4, "dropout": 0.25, "seed": 5, "offset": 6}
        h = token_emb.embedding(w, ids, **call)
        g = rows_like(rng, (4, 25, 80), t)
        h.backward(g)
        assert w.grad.dtype == t and torch.equal(w.grad, E.cudaEmbeddingGrad(ids, g, 30, **call))
        want, size, terms = oracle.embedding_grad(ids.cpu().numpy(), f64(g), 30, padding_idx=4, scale=2.0, p=0.25, seed=5, offset=6)
        close(w.grad, want, t, size, terms[:, None])
        x = rows_like(rng, (9, 80), t).requires_grad_()
        token_emb.dropout(x, 0.25, 5, 6, scale=2.0).backward(g[0, :9])
        assert torch.equal(x.grad, E.cudaDropout(g[0, :9], 0.25, 5, 6, scale=2.0))


def test_autograd_refusals(E):
    from hades_b200 import token_emb

    w = torch.randn(20, 16, device="cuda").requires_grad_()
    ids = torch.arange(8, device="cuda")
    h = token_emb.embedding(w, ids, dropout=0.5)
    (g,) = torch.autograd.grad((h * h).sum(), w, create_graph=False)
    h = token_emb.embedding(w, ids)
    with pytest.raises(RuntimeError, match="not differentiated again"):
        torch.autograd.grad((h * h).sum(), w, create_graph=True)
    h = token_emb.embedding(w, ids)
    assert torch.autograd.grad(h.sum(), w, create_graph=True)[0][:8].eq(1).all()  # (does not depend on anything)
    h = token_emb.embedding(w, ids)
    ids += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    rng = torch.tensor([1, 2], device="cuda")
    h = token_emb.dropout(w, 0.5, rng=rng)
    rng += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    h = token_emb.embedding(w, ids)
    h.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        h.sum().backward()
    w.grad = None
    h = token_emb.embedding(w, ids)
    h.sum().backward(retain_graph=True)
    h.sum().backward()
    assert bool((w.grad[ids] == 2).all())
    assert not token_emb.embedding(w.detach(), ids).requires_grad
    with torch.no_grad():
        assert not token_emb.embedding(w, ids).requires_grad
    # a weight that is computed, used twice
    v = torch.randn(20, 16, device="cuda").requires_grad_()
    u = v * 3
    (token_emb.embedding(u, ids) + token_emb.embedding(u, ids, scale=2.0)).sum().backward()
    want = torch.zeros_like(v)
    want[ids] = 9.0
    assert torch.equal(v.grad, want)
    # a tensor that a graph has saved is written over
    y = torch.randn(8, 16, device="cuda").requires_grad_()
    z = y * 2
    s = (z * z).sum()
    E.cudaEmbedding(w.detach(), ids, out=z.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        s.backward()
    # an output that nothing depends on
    x = torch.randn(4, 16, device="cuda").requires_grad_()
    a, b = token_emb.dropout(x, 0.5, 1, 1), token_emb.dropout(x, 0.5, 1, 2)
    a.sum().backward()
    assert torch.equal(x.grad, E.cudaDropout(torch.ones_like(x), 0.5, 1, 1)) and b.requires_grad


def test_gradient_against_differences(E):
    """Small whole numbers and a share of one half: every product and sum is exact, and so is the difference quotient."""
    from hades_b200 import token_emb

    rng = np.random.default_rng(4)
    ids = torch.from_numpy(rng.integers(-1, 12, 64)).cuda()
    w = torch.from_numpy(rng.integers(-8, 9, (12, 40)).astype(np.float32)).cuda().requires_grad_()
    call = {"scale": 0.5, "padding_idx": -1, "dropout": 0.5, "seed": 8, "offset": 1}
    g = torch.from_numpy(rng.integers(-8, 9, (64, 40)).astype(np.float32)).cuda()
    token_emb.embedding(w, ids, **call).backward(g)
    for _ in range(4):
        e = torch.from_numpy(rng.integers(-4, 5, (12, 40)).astype(np.float32)).cuda()
        change = E.cudaEmbedding(w.detach() + e, ids, **call) - E.cudaEmbedding(w.detach(), ids, **call)
        assert float((change * g).sum()) == float((w.grad * e).sum())


def test_layer_in_training_and_evaluation(E):
    from hades_b200.token_emb import TokenEmbedding

    layer = TokenEmbedding(50, 64, scale=8.0, padding_idx=0, dropout=0.5, dtype=BF16, seed=3)
    assert not layer.weight[0].any()
    ids = torch.randint(0, 50, (3, 10), device="cuda")
    a, b = layer(ids), layer(ids)
    assert not torch.equal(a, b)  # another mask every time
    assert torch.equal(a, E.cudaEmbedding(layer.weight.detach(), ids, 8.0, 0, 0.5, seed=3, offset=1))
    a.float().sum().backward()
    assert torch.equal(layer.weight.grad, E.cudaEmbeddingGrad(ids, torch.ones_like(a), 50, 8.0, 0, 0.5, 3, 1))
    layer.eval()
    assert torch.equal(layer(ids), E.cudaEmbedding(layer.weight.detach(), ids, 8.0, 0))
    import copy
    import io

    for saved in (layer.state_dict(), layer.weight):
        f = io.BytesIO()
        torch.save(saved, f)
        f.seek(0)
        torch.load(f)
    assert torch.equal(copy.deepcopy(layer).weight, layer.weight)


@pytest.mark.parametrize("kind", ["adam", "adagrad"])
def test_sparse_training_step(E, kind):
    """Lookup, dropout, backward, tokens and rows, sparse update: as with the update's own merge of repeated tokens."""
    from hades_b200.sparse_optim import ShardedEmbedding, SparseAdagrad, SparseAdam

    make = SparseAdam if kind == "adam" else SparseAdagrad
    a, b = (ShardedEmbedding(500, 64, init_sigma=0.1, seed=1) for _ in range(2))
    oa, ob = make(a, 0.01), make(b, 0.01)
    rng = np.random.default_rng(2)
    for step in range(3):
        ids = torch.from_numpy(rng.integers(0, 500, 2000)).cuda()
        call = {"scale": 2.0, "padding_idx": 7, "dropout": 0.1, "seed": 1, "offset": step}
        h = E.cudaEmbedding(a.weight, ids, **call).requires_grad_()
        (h * h).sum().backward()
        tokens, rows, num = E.cudaEmbeddingGradRows(ids, h.grad, 500, sync=False, **call)
        oa.update(tokens, rows, is_unique=True, n_dev=num)
        u, r = E.cudaEmbeddingGradRows(ids, h.grad, 500, **call)
        ob.update(u, r.clone(), is_unique=True)
        assert 7 not in u.tolist() and torch.equal(a.weight, b.weight)
        # and as the aggregation that was here before sums the same rows (another order of additions)
        v, s, _ = E.cudaUniqueSegSum(ids, E.cudaDropout(h.grad, 0.1, 1, step, scale=2.0))
        assert torch.equal(v[v != 7], u)
        torch.testing.assert_close(s[v != 7], r, rtol=1e-4, atol=1e-4)
    assert status() == 0


@pytest.mark.parametrize("scale,p", [(1.0, 0.2), (3.0, 0.0), (0.5, 0.5)])
def test_dist_emb_with_scale_and_dropout(E, scale, p):
    from hades_b200 import pipeline, synth
    from hades_b200.dist_emb import DistEmb, DistembSparseGradOptimizer

    base = synth.scaled(synth.CONFIG1, 0.05, "scaled")
    cfg = synth.CacheFetchConfig(base.name, base.config, base.table_rows, base.dim, base.cache_entries, base.batch,
                                 base.zipf_s, flush_every=2)
    plain, ours = DistEmb(pipeline.build_path(cfg)), DistEmb(pipeline.build_path(cfg), scale=scale, dropout=p, seed=4)
    opts = [DistembSparseGradOptimizer([layer.sparse_emb]) for layer in (plain, ours)]
    sampler, rng = synth.ZipfSampler(cfg.table_rows, cfg.zipf_s), synth.rng_for(1, 0, 3)
    for step in range(1, 4):
        ids = torch.from_numpy(sampler.ids(rng, cfg.batch)).cuda()
        g = torch.randn(cfg.batch, cfg.dim, device="cuda")
        h, k = plain(ids), ours(ids)
        assert torch.equal(k, E.cudaDropout(h.detach(), p, 4, step, scale=scale))
        for opt in opts:
            opt.zero_grad()
        h.backward(E.cudaDropout(g, p, 4, step, scale=scale))
        k.backward(g)
        for opt in opts:
            opt.step()
        assert torch.equal(plain.sparse_emb.path.table, ours.sparse_emb.path.table)
    plain.eval(), ours.eval()
    ids = torch.from_numpy(sampler.ids(rng, 1000)).cuda()
    assert torch.equal(ours(ids), plain(ids) * scale)


# ---- streams and graphs ---------------------------------------------------------------------------------------------------------
def test_another_stream(E):
    side = torch.cuda.Stream()
    ids = torch.randint(0, 5000, (20_000,), device="cuda")
    g = torch.randn(20_000, 128, device="cuda")
    want = E.cudaEmbeddingGrad(ids, g, 5000)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ours = [E.cudaEmbeddingGrad(ids, g * k, 5000) for k in (1, 2, 4)]
    theirs = [E.cudaEmbeddingGrad(ids, g * k, 5000) for k in (1, 2, 4)]
    torch.cuda.synchronize()
    for k, a, b in zip((1, 2, 4), ours, theirs):
        assert torch.equal(a, want * k) and torch.equal(b, want * k)


def test_two_threads(E):
    import threading

    ids = [torch.randint(0, 4000, (n,), device="cuda") for n in (9000, 300)]
    grads = [torch.randn(n, 72, device="cuda") for n in (9000, 300)]
    want = [E.cudaEmbeddingGrad(i, g, 4000, dropout=0.2, seed=1) for i, g in zip(ids, grads)]
    torch.cuda.synchronize()
    failed = []

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                got = E.cudaEmbeddingGrad(ids[k], grads[k], 4000, dropout=0.2, seed=1)
                tokens, rows = E.cudaEmbeddingGradRows(ids[k], grads[k], 4000, dropout=0.2, seed=1)
                if not (torch.equal(got, want[k]) and torch.equal(rows, want[k][tokens])):
                    failed.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1, 0, 1)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failed and status() == 0


def test_captured_layer(E):
    from hades_b200.token_emb import TokenEmbedding

    layer = TokenEmbedding(300, 128, dropout=0.3, padding_idx=0, seed=5, seed_on_device=True)
    ids = torch.randint(0, 300, (8, 40), device="cuda")
    g = torch.randn(8, 40, 128, device="cuda")

    def step():
        layer.weight.grad = None
        h = layer(ids)
        h.backward(g)
        return h.detach(), layer.weight.grad

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, grad = step()
    masks = []
    for k in range(3):
        ids.copy_(torch.randint(0, 300, (8, 40), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        offset = int(layer.seeds.state[1].item())
        assert offset == 2 + k  # one before the capture, which itself draws none
        assert torch.equal(h, E.cudaEmbedding(layer.weight.detach(), ids, 1.0, 0, 0.3, seed=5, offset=offset))
        assert torch.equal(grad, E.cudaEmbeddingGrad(ids, g, 300, 1.0, 0, 0.3, 5, offset))
        masks.append((h != 0).clone())
    assert not torch.equal(masks[0], masks[1])


def test_captured_backward_of_many_tokens(E):
    from hades_b200 import token_emb

    w = torch.randn(900, 136, device="cuda").requires_grad_()
    ids = torch.randint(0, 900, (5000,), device="cuda")
    g = torch.randn(5000, 136, device="cuda")

    def step():
        w.grad = None
        token_emb.embedding(w, ids, dropout=0.1, seed=1, offset=1).backward(g)
        return w.grad

    step()
    torch.cuda.synchronize()
    w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = step()
    for _ in range(2):
        ids.copy_(torch.randint(0, 900, (5000,), device="cuda"))
        grad.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, E.cudaEmbeddingGrad(ids, g, 900, dropout=0.1, seed=1, offset=1))
    assert status() == 0


def test_two_graphs_and_eager_calls_between(E):
    ids = [torch.randint(0, 900, (n,), device="cuda") for n in (3000, 700)]
    grads = [torch.randn(n, 260, device="cuda") for n in (3000, 700)]
    want = [E.cudaEmbeddingGrad(i, g, 900) for i, g in zip(ids, grads)]
    graphs, outs = [], []
    for i, g in zip(ids, grads):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append((E.cudaEmbeddingGrad(i, g, 900), *E.cudaEmbeddingGradRows(i, g, 900, sync=False)))
    for order in ((0, 1), (1, 0), (0, 1)):
        for k in order:
            outs[k][0].fill_(5.0)
            graphs[k].replay()
            eager = E.cudaEmbeddingGrad(ids[1 - k], grads[1 - k], 900)
            torch.cuda.synchronize()
            assert torch.equal(outs[k][0], want[k]) and torch.equal(eager, want[1 - k])
            u = int(outs[k][3].item())
            assert torch.equal(outs[k][2][:u], want[k][outs[k][1][:u]])
    assert status() == 0


def test_a_capture_refuses_what_it_cannot_wait_for(E):
    from hades_b200 import token_emb

    w = torch.randn(20, 16, device="cuda").requires_grad_()
    ids = torch.arange(8, device="cuda")
    h = token_emb.embedding(w, ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="still lives"):
            token_emb.embedding(w, ids)
        with pytest.raises(RuntimeError, match="sync=False"):
            E.cudaEmbeddingGradRows(ids, w.detach()[:8], 20)
        kept = E.cudaEmbedding(w.detach(), ids)
    del h
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, w.detach()[:8])
    # any other operator's graph of the leaf is one too; two in the same capture are none
    other = w * 2
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="still lives"):
            token_emb.embedding(w, ids)
        with pytest.raises(RuntimeError, match="still lives"):
            token_emb.dropout(w, 0.5)
        kept = E.cudaEmbedding(w.detach(), ids)
    del other
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.grad = None
        (token_emb.embedding(w, ids) + token_emb.embedding(w, ids, scale=2.0)).sum().backward()
    graph.replay()
    torch.cuda.synchronize()
    assert bool((w.grad[:8] == 3).all()) and not w.grad[8:].any()
