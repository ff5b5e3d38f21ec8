"""What the differentiable token-embedding calls refuse before they look at the device."""
import pytest
import torch


@pytest.fixture(scope="module")
def token_emb():
    from hades_b200 import _build, token_emb

    _build.build()
    return token_emb


A = 1 << 20  # made-up addresses: the calls return before anything that they point to is looked at


def test_pointers_between_values_are_refused(token_emb):
    import ctypes as C

    from hades_b200 import _lib

    lib = _lib.load()
    refused = lambda rc: rc == 1 and b"aligned" in lib.hb_last_error()  # noqa: E731
    drop = C.byref(_lib.DropDesc(0.5, 0, 0, A + 4))
    for t, between in ((0, 2), (0, 1), (1, 1), (2, 1)):
        for k in range(3):
            w, ids, out = (A * (i + 1) + (between if i == k else 0) for i in range(3))
            assert refused(lib.hb_embedding(w, t, 16, 100, 16, ids, 4, 10, -1, 1.0, None, out, t, 16, None))
            assert k == 1 or refused(lib.hb_dropout(w, t, 16, 10, 16, 1.0, None, out, t, 16, None))
            assert refused(lib.hb_embedding_grad(ids, 8, 10, -1, w, t, 16, 16, 1.0, None, 100, out, t, 16, 0, 4 * A, 1 << 30, None))
    assert refused(lib.hb_embedding(A, 0, 16, 100, 16, 2 * A, 8, 10, -1, 1.0, drop, 3 * A, 0, 16, None))
    assert refused(lib.hb_dropout(A, 0, 16, 10, 16, 1.0, drop, 2 * A, 0, 16, None))
    assert refused(lib.hb_embedding_grad(A, 8, 10, -1, 2 * A, 0, 16, 16, 1.0, drop, 100, 3 * A, 0, 16, 0, 4 * A, 1 << 30, None))
    assert refused(lib.hb_embedding_grad(A, 8, 10, -1, 2 * A, 0, 16, 16, 1.0, None, 100, 3 * A, 0, 16, 0, 4 * A + 8, 1 << 30, None))
    for k, between in enumerate((4, 2, 4, 8)):
        uniq, rows, num, ws = ((5 + i) * A + (between if i == k else 0) for i in range(4))
        assert refused(lib.hb_embedding_grad_rows(A, 8, 10, -1, 2 * A, 0, 16, 16, 1.0, None, 100, uniq, rows, num, ws, 1 << 30, None))


def test_forward_mode_is_refused(token_emb):
    import torch.autograd.forward_ad as fwd

    w, ids = torch.randn(8, 16), torch.arange(4)
    with fwd.dual_level():
        for grad in (False, True):
            dual = fwd.make_dual(w.clone().requires_grad_(grad), torch.ones_like(w))
            for call in (lambda: token_emb.embedding(dual, ids), lambda: token_emb.dropout(dual, 0.5)):
                with pytest.raises(RuntimeError, match="forward mode"):
                    call()
        with pytest.raises(RuntimeError, match="CUDA"):
            token_emb.embedding(w, ids)


def test_traces_are_refused(token_emb):
    from torch.fx.experimental.proxy_tensor import make_fx

    w, ids = torch.randn(8, 16), torch.arange(4)
    for call in (lambda a: token_emb.embedding(a, ids), lambda a: token_emb.dropout(a, 0.5)):
        with torch.no_grad(), pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(call, (w,), check_trace=False)
        with pytest.raises(RuntimeError, match="trace"):
            make_fx(call)(w)
        with pytest.raises(RuntimeError, match="CUDA"):  # (the trace is over)
            call(w)


@pytest.mark.parametrize("reentrant", [False, True])
def test_masks_of_passes_that_run_again_are_refused(token_emb, reentrant):
    from torch.utils.checkpoint import checkpoint

    seeds, drawn = token_emb.DropoutSeeds(3), []

    def layer(x):
        drawn.append(seeds.next())
        return (x * drawn[-1]["offset"]).sin()

    x = torch.ones(4, requires_grad=True)
    y = checkpoint(layer, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="another mask"):
        y.sum().backward()
    assert len(drawn) == 1 and seeds.next()["offset"] == 2
    mask = seeds.next()  # numbers of one's own
    checkpoint(lambda x: (x * mask["offset"]).sin(), x, use_reentrant=reentrant).sum().backward()
    assert x.grad is not None


def _layer(token_emb, **kw):
    return token_emb.TokenEmbedding(4, 8, device="cpu", **kw)


def test_masks_are_saved_with_the_layer(token_emb, tmp_path):
    """A run that continues from a module's state draws the next mask, not the first."""
    for make in (lambda seed: _layer(token_emb, dropout=0.5, seed=seed), lambda seed: _dist_emb(0.5, seed)):
        layer = make(7)
        model = torch.nn.Sequential(torch.nn.Linear(2, 2), layer)
        drawn = [layer.seeds.next() for _ in range(3)]
        torch.save(model.state_dict(), tmp_path / "state")
        assert drawn[-1] == {"seed": 7, "offset": 3}
        state = torch.load(tmp_path / "state")  # (tensors only)
        for seed in (7, None):
            other = torch.nn.Sequential(torch.nn.Linear(2, 2), make(seed))
            other.load_state_dict(state)
            assert other[1].seeds.next() == {"seed": 7, "offset": 4}
        largest = make((1 << 63) - 1)
        copy = make(0)
        copy.load_state_dict(largest.state_dict())
        assert copy.seeds.next() == {"seed": (1 << 63) - 1, "offset": 1}
        # as saved before the numbers were: nothing is missing, and they stay
        for key in [k for k in state if "extra" in k]:
            del state[key]
        other.load_state_dict(state)
        assert other[1].seeds.next() == {"seed": 7, "offset": 5}


def _dist_emb(dropout, seed=None):
    from types import SimpleNamespace

    from hades_b200.dist_emb import DistEmb

    return DistEmb(SimpleNamespace(dim=8, num_nodes=4), dropout=dropout, seed=seed)


def test_layers_without_dropout_save_what_they_did(token_emb):
    plain, dropping = _layer(token_emb), _layer(token_emb, dropout=0.5, seed=1)
    assert list(plain.state_dict()) == ["weight"] and not _dist_emb(0.0).state_dict()
    dropping.load_state_dict(plain.state_dict())
    plain.load_state_dict(dropping.state_dict())
    assert torch.equal(plain.weight, dropping.weight) and dropping.seeds.next() == {"seed": 1, "offset": 1}
    _dist_emb(0.0).load_state_dict(_dist_emb(0.5).state_dict())
    with pytest.raises(RuntimeError, match="Missing key"):
        plain.load_state_dict({})
    with pytest.raises(RuntimeError, match="Unexpected key"):
        plain.load_state_dict({**plain.state_dict(), "other": torch.zeros(1)})


def test_numbers_on_a_device_move_with_the_layer(token_emb):
    layer = _layer(token_emb, dropout=0.5, seed=5, seed_on_device=True)
    layer.seeds.next()
    kept = layer.seeds.state
    layer.half().to("cpu").double()
    assert layer.seeds.state is kept and kept.tolist() == [5, 1] and kept.dtype == torch.int64
    other = _layer(token_emb, dropout=0.5, seed=6, seed_on_device=True)
    at = other.seeds.state.data_ptr()
    other.load_state_dict(layer.state_dict())
    assert other.seeds.next()["rng"].tolist() == [5, 2] and other.seeds.state.data_ptr() == at
    layer.to("meta")  # has no numbers to keep
    assert layer.seeds.state.tolist() == [5, 1]
