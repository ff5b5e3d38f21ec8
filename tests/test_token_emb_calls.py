"""What the differentiable token-embedding calls refuse before they look at the device."""
import pytest
import torch


@pytest.fixture(scope="module")
def token_emb():
    from hades_b200 import _build, token_emb

    _build.build()
    return token_emb


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
