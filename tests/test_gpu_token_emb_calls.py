"""Calls of the token-embedding operators that a program may make beside the usual ones: on several streams, on outputs that
begin anywhere, by way of other parts of torch."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def E(cuda_lib):
    from hades_b200 import EmbCacheLib

    return EmbCacheLib


def test_a_gradient_does_not_wait_for_another_stream(E):
    """A kernel of half a second lies in front of one stream's gradient; gradients on others finish before it does.  (One of
    four is enough: the GPU may put any two streams into one queue.)"""
    ids, g = torch.randint(0, 5000, (5000,), device="cuda"), torch.randn(5000, 128, device="cuda")
    want = E.cudaEmbeddingGrad(ids, g, 5000)
    torch.cuda.synchronize()
    busy, *others = [torch.cuda.Stream() for _ in range(5)]
    for stream in (busy, *others):  # what a first call makes is there
        with torch.cuda.stream(stream):
            E.cudaEmbeddingGrad(ids, g, 5000)
    torch.cuda.synchronize()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(1_000_000_000)
        late = E.cudaEmbeddingGrad(ids, g, 5000)
        done = busy.record_event()
    outs = []
    for stream in others:
        with torch.cuda.stream(stream):
            outs.append((E.cudaEmbeddingGrad(ids, g, 5000), stream.record_event()))
    early = 0
    while not done.query():
        early = sum(event.query() for _, event in outs)
        if early:
            break
    torch.cuda.synchronize()
    assert early and torch.equal(late, want) and all(torch.equal(out, want) for out, _ in outs)
