"""The token-embedding operators without a GPU: the generator against its authors' vectors, what the calls refuse."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import token_oracle as oracle


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))])
def test_generator_gives_its_authors_vectors(counter, key, want):
    assert tuple(int(w) for w in oracle.philox4x32(counter, key)) == want


def test_share_dropped():
    keep = oracle.kept(1_000, 1_000, 0.1, 1234, 5)
    # a million draws of a share 6554 / 65536: five standard deviations
    share = 6554 / 65536
    assert abs((~keep).mean() - share) < 5 * math.sqrt(share * (1 - share) / 1e6)
    assert (oracle.kept(100, 100, 0.1, 1234, 6) != keep[:100, :100]).any()
    assert oracle.threshold(1.0) == 65536 and not oracle.kept(8, 8, 1.0, 1, 1).any()


@pytest.fixture(scope="module")
def lib():
    from hades_b200 import _build, _lib

    _build.build()
    return _lib.load()


def _drop(p, **kw):
    from hades_b200 import _lib

    return C.byref(_lib.DropDesc(p, 0, 0, None))


A = 1 << 20  # addresses here are made up: the calls return before anything that they point to is looked at


@pytest.mark.parametrize("change,why", [
    ({"n": -1}, b"bad sizes"), ({"n": (1 << 32) + 1}, b"bad sizes"), ({"dim": 0}, b"bad sizes"), ({"dim": 1 << 24}, b"bad sizes"),
    ({"rows": -1}, b"bad sizes"), ({"wt": 3}, b"value type"), ({"ot": -1}, b"value type"), ({"ib": 2}, b"idx_bytes"),
    ({"ids": None}, b"null"), ({"w": None}, b"null"), ({"out": None}, b"null"), ({"os": 15}, b"overlap"),
    ({"scale": math.nan}, b"finite"), ({"scale": 1e39}, b"finite"), ({"p": 1.5}, b"probability"), ({"p": -0.1}, b"probability"),
    ({"p": math.nan}, b"probability"), ({"out": A + 64}, b"lies in the table")])
def test_embedding_refuses(lib, change, why):
    a = {"w": A, "wt": 0, "ws": 16, "rows": 100, "dim": 16, "ids": 2 * A, "ib": 8, "n": 10, "pad": -1, "scale": 1.0, "p": 0.5,
         "out": 3 * A, "ot": 0, "os": 16, **change}
    rc = lib.hb_embedding(a["w"], a["wt"], a["ws"], a["rows"], a["dim"], a["ids"], a["ib"], a["n"], a["pad"], a["scale"],
                          _drop(a["p"]), a["out"], a["ot"], a["os"], None)
    assert rc == 1 and why in lib.hb_last_error(), lib.hb_last_error()


@pytest.mark.parametrize("change,why", [
    ({"n": -1}, b"bad sizes"), ({"dim": 0}, b"bad sizes"), ({"xt": 7}, b"value type"), ({"x": None}, b"null"),
    ({"ys": 8}, b"overlap"), ({"y": A + 4}, b"neither apart"), ({"y": A, "yt": 1}, b"neither apart"),
    ({"y": A, "ys": 32}, b"neither apart"), ({"p": 2.0}, b"probability"), ({"scale": math.inf}, b"finite")])
def test_dropout_refuses(lib, change, why):
    a = {"x": A, "xt": 0, "xs": 16, "n": 10, "dim": 16, "scale": 1.0, "p": 0.5, "y": 2 * A, "yt": 0, "ys": 16, **change}
    rc = lib.hb_dropout(a["x"], a["xt"], a["xs"], a["n"], a["dim"], a["scale"], _drop(a["p"]), a["y"], a["yt"], a["ys"], None)
    assert rc == 1 and why in lib.hb_last_error(), lib.hb_last_error()


@pytest.mark.parametrize("change,rc,why", [
    ({"n": 1 << 31}, 1, b"bad sizes"), ({"dim": -1}, 1, b"bad sizes"), ({"rows": -1}, 1, b"bad sizes"),
    ({"gt": 3}, 1, b"value type"), ({"ot": 3}, 1, b"value type"), ({"ib": 1}, 1, b"idx_bytes"), ({"ids": None}, 1, b"null"),
    ({"g": None}, 1, b"null"), ({"out": None}, 1, b"null"), ({"os": 3}, 1, b"overlap"), ({"p": -1.0}, 1, b"probability"),
    ({"scale": math.nan}, 1, b"finite"), ({"ws": None}, 3, b"workspace"), ({"wb": 16}, 3, b"workspace"),
    ({"out": 2 * A + 64}, 1, b"gradients"), ({"gs": -1}, 1, b"stride")])
def test_embedding_grad_refuses(lib, change, rc, why):
    a = {"ids": A, "ib": 8, "n": 10, "pad": -1, "g": 2 * A, "gt": 0, "gs": 16, "dim": 16, "scale": 1.0, "p": 0.5, "rows": 100,
         "out": 3 * A, "ot": 0, "os": 16, "ws": 4 * A, "wb": 1 << 30, **change}
    got = lib.hb_embedding_grad(a["ids"], a["ib"], a["n"], a["pad"], a["g"], a["gt"], a["gs"], a["dim"], a["scale"], _drop(a["p"]),
                                a["rows"], a["out"], a["ot"], a["os"], 0, a["ws"], a["wb"], None)
    assert got == rc and why in lib.hb_last_error(), lib.hb_last_error()


def test_embedding_grad_rows_refuses(lib):
    call = lambda uniq, rows, num: lib.hb_embedding_grad_rows(A, 8, 10, -1, 2 * A, 0, 16, 16, 1.0, None, 100, uniq, rows, num,
                                                              4 * A, 1 << 30, None)  # noqa: E731
    for missing in range(3):
        args = [5 * A, 6 * A, 7 * A]
        args[missing] = None
        assert call(*args) == 1 and b"null output" in lib.hb_last_error()
    assert lib.hb_embedding_grad_workspace_bytes(-1, 16) == 0 and lib.hb_embedding_grad_workspace_bytes(10, 0) == 0
    assert lib.hb_embedding_grad_workspace_bytes(10, 16) > 0


def test_host_tensors_are_refused():
    from hades_b200 import EmbCacheLib as E

    w, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        E.cudaEmbedding(w, ids)
    with pytest.raises(RuntimeError, match="CUDA"):
        E.cudaEmbeddingGrad(ids, torch.zeros(3, 8), 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        E.cudaEmbeddingGradRows(ids, torch.zeros(3, 8), 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        E.cudaDropout(w, 0.5)


def test_seeds():
    from hades_b200.token_emb import DropoutSeeds

    a, b = DropoutSeeds(7), DropoutSeeds(7)
    assert a.next() == b.next() == {"seed": 7, "offset": 1} and a.next() == {"seed": 7, "offset": 2}
    with pytest.raises(RuntimeError, match="seed"):
        DropoutSeeds(-1)
    with pytest.raises(RuntimeError, match="seed"):
        DropoutSeeds(1 << 63)
    b.load_state_dict(a.state_dict())
    assert a.state_dict() == {"seed": 7, "offset": 2} and b.next() == a.next()
    torch.manual_seed(3)
    c = DropoutSeeds().seed
    torch.manual_seed(3)
    assert DropoutSeeds().seed == c


def test_layers_refuse_shares_outside_of_one():
    from hades_b200.dist_emb import DistEmb
    from hades_b200.token_emb import TokenEmbedding

    for p in (-0.1, 1.1, math.nan):
        with pytest.raises(RuntimeError, match="dropout"):
            TokenEmbedding(4, 8, dropout=p, device="cpu")
        with pytest.raises(RuntimeError, match="dropout"):
            DistEmb(None, dropout=p)


def test_oracle_gradient_is_that_of_its_forward():
    rng = np.random.default_rng(1)
    w, ids, g = rng.standard_normal((7, 10)), rng.integers(-1, 7, 20), rng.standard_normal((20, 10))
    drop = {"scale": 1.5, "p": 0.3, "seed": 5, "offset": 2}
    grad, _, _ = oracle.embedding_grad(ids, g, 7, padding_idx=2, **drop)
    for _ in range(5):  # linear: the difference along a direction is the gradient's product with it
        e = rng.standard_normal((7, 10))
        diff = (oracle.embedding(w + e, ids, padding_idx=2, **drop) - oracle.embedding(w, ids, padding_idx=2, **drop)) * g
        assert abs(diff.sum() - (grad * e).sum()) < 1e-10
