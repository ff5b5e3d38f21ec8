"""Calls of the token-embedding operators that a program may make beside the usual ones: on several streams, on outputs that
begin anywhere, by way of other parts of torch."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
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


# ---- a sort that gives up ---------------------------------------------------------------------------------------------------
GIVES_UP = r"""
#include <cstdio>
#include "runsfinish.cuh"

struct Ctx {
  static constexpr int kThreads = 64;
  static constexpr uint32_t count = 100;
  __device__ uint32_t chunk_begin() const { return 0; }
  __device__ uint32_t chunk_end() const { return count; }
};
struct Source { int64_t sentinel; };
__global__ void give_up(hb::RunsFinish<false> fin) {
  Ctx ctx;
  fin.give_up(ctx, Source{(1 << 20) - 1});
}
template <class T> T* words(int n) {
  T* p = nullptr;
  cudaMallocManaged(&p, n * sizeof(T));
  memset(p, 0x55, n * sizeof(T));
  return p;
}
int main() {
  hb::RunsFinish<false> fin = {};
  fin.perm = words<uint32_t>(100);
  fin.head = words<uint8_t>(108);
  fin.uniq = words<int64_t>(101);
  fin.uniq2 = words<int64_t>(100);
  fin.run_start = words<int64_t>(101);
  fin.num_runs = words<int64_t>(1);
  fin.num_runs2 = words<int64_t>(1);
  fin.class_counts = words<int64_t>(4);
  fin.base8 = words<int32_t>(14);
  fin.n_valid = words<int64_t>(1);
  give_up<<<1, 64>>>(fin);
  if (cudaDeviceSynchronize() != cudaSuccess) return 1;
  std::printf("%lld %lld %lld %lld", (long long)*fin.num_runs, (long long)*fin.num_runs2, (long long)fin.uniq[0], (long long)fin.uniq2[0]);
  return 0;
}
"""


def test_what_a_sort_that_gives_up_leaves(tmp_path):
    (tmp_path / "up.cu").write_text(GIVES_UP)
    nvcc = "/usr/local/cuda/bin/nvcc"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr", "--extended-lambda",
                    "-I", str(ROOT / "include"), "-I", str(ROOT / "hades_b200" / "csrc"), str(tmp_path / "up.cu"),
                    "-o", str(tmp_path / "up")], check=True, capture_output=True)
    r = subprocess.run([str(tmp_path / "up")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == f"0 0 {(1 << 20) - 1} -1", r.stdout + r.stderr


# The library's call in the state that such a sort leaves: no tokens, the first of them -1.
GAVE_UP = r"""
#include <cstdint>
#include <cuda_runtime.h>
extern "C" int hb_embedding_grad_rows(const void*, int, int64_t, int64_t, const void*, int, int64_t, int64_t, double, const void*,
                                      int64_t, int64_t* uniq, float*, int64_t* num, void*, size_t, cudaStream_t stream) {
  const int64_t first = FIRST, none = 0;
  cudaMemcpyAsync(uniq, &first, 8, cudaMemcpyDefault, stream);
  cudaMemcpyAsync(num, &none, 8, cudaMemcpyDefault, stream);
  return 0;
}
"""
CALLS = """
import torch
from hades_b200 import EmbCacheLib as E
E.cudaEmbeddingGradRows(torch.zeros(20, dtype=torch.int64, device="cuda"), torch.ones(20, 8, device="cuda"), 4)
"""


def test_a_sort_that_gave_up_is_an_error(tmp_path):
    for first, raises in ((-1, True), (4, False)):
        (tmp_path / "up.cpp").write_text(GAVE_UP.replace("FIRST", str(first)))
        subprocess.run(["g++", "-shared", "-fPIC", "-I", "/usr/local/cuda/include", str(tmp_path / "up.cpp"), "-L",
                        "/usr/local/cuda/lib64", "-lcudart", "-o", str(tmp_path / f"up{first}.so")], check=True)
        r = subprocess.run([sys.executable, "-c", CALLS], cwd=ROOT, capture_output=True, text=True, timeout=300,
                           env={**os.environ, "LD_PRELOAD": str(tmp_path / f"up{first}.so")})
        assert (r.returncode != 0) == raises and ("gave up waiting" in r.stderr) == raises, r.stderr


@pytest.mark.parametrize("n", [100, 2000, 3000, 60_000, 70_000])
def test_batches_without_tokens(E, n):
    """Rows of a batch that is all padding: none, and no error; the first token says that the sort did not give up."""
    ids, g = torch.full((n,), 3, device="cuda"), torch.ones(n, 8, device="cuda")
    for pad, vocab in ((3, 10), (3, 4)):
        tokens, rows = E.cudaEmbeddingGradRows(ids, g, vocab, padding_idx=pad)
        assert tokens.numel() == 0 and rows.shape == (0, 8)
        tokens, _, number = E.cudaEmbeddingGradRows(ids, g, vocab, padding_idx=pad, sync=False)
        assert number.item() == 0 and tokens[0].item() >= vocab


# ---- what else torch can do with a call ---------------------------------------------------------------------------------------
def test_forward_mode_is_refused(E):
    import torch.autograd.forward_ad as fwd

    from hades_b200 import token_emb

    w, ids = torch.randn(8, 16, device="cuda"), torch.arange(4, device="cuda")
    with fwd.dual_level():
        for grad in (False, True):
            dual = fwd.make_dual(w.clone().requires_grad_(grad), torch.ones_like(w))
            for call in (lambda: token_emb.embedding(dual, ids), lambda: token_emb.dropout(dual, 0.5)):
                with pytest.raises(RuntimeError, match="forward mode"):
                    call()
        # of a gradient on its way back, too
        leaf = w.clone().requires_grad_()
        g = fwd.make_dual(torch.ones(4, 16, device="cuda"), torch.ones(4, 16, device="cuda"))
        for h in (token_emb.embedding(leaf, ids), token_emb.dropout(leaf, 0.5)[:4]):
            with pytest.raises(RuntimeError, match="forward mode"):
                torch.autograd.grad(h, leaf, g)
        # what has no tangent is as ever, and so is what is taken out of one
        assert torch.equal(token_emb.embedding(w, ids), w[:4])
        assert torch.equal(token_emb.embedding(fwd.unpack_dual(fwd.make_dual(w, w)).primal, ids), w[:4])


# ---- DistEmb ------------------------------------------------------------------------------------------------------------------
def small_path():
    from hades_b200 import pipeline, synth

    base = synth.scaled(synth.CONFIG1, 0.05, "small")
    return pipeline.build_path(synth.CacheFetchConfig(base.name, base.config, base.table_rows, base.dim, base.cache_entries,
                                                      base.batch, base.zipf_s, flush_every=2))


def test_dist_emb_has_one_shape(E):
    """[number of ids, dim] whatever the ids' shape, the scale and the mode."""
    from hades_b200.dist_emb import DistEmb

    path = small_path()
    ids = torch.randint(0, path.num_nodes, (7, 30), device="cuda")
    want = path.table[ids.view(-1)]
    for given in (ids, ids.t().contiguous().t(), ids.view(-1), ids.view(1, 7, 5, 6), ids.cpu()):
        for scale in (1.0, 2.0):
            layer = DistEmb(path, scale=scale, dropout=0.25).eval()
            assert torch.equal(layer(given), want * scale)
    assert DistEmb(path, scale=2.0).eval()(ids[0, 0]).shape == DistEmb(path).eval()(ids[0, 0]).shape == (1, path.dim)
    for scale in (1.0, 2.0):
        layer = DistEmb(path, scale=scale)
        assert layer(ids.view(-1)).shape == layer.eval()(ids.view(-1)).shape == (210, path.dim)


def test_checkpointed_layers(E):
    from torch.utils.checkpoint import checkpoint

    from hades_b200 import token_emb

    layer, ids = token_emb.TokenEmbedding(40, 64, dropout=0.5, seed=1), torch.randint(0, 40, (50,), device="cuda")
    for reentrant in (False, True):
        x = torch.ones((), device="cuda", requires_grad=True)
        h = checkpoint(lambda x: (layer(ids) * x).sin(), x, use_reentrant=reentrant)
        with pytest.raises(RuntimeError, match="another mask"):
            h.sum().backward()
        layer.weight.grad = None
        # with numbers of one's own, and without dropout, as without checkpoints
        for p in (0.5, 0.0):
            def passes(x, p=p):
                return (token_emb.embedding(layer.weight, ids, dropout=p, seed=1, offset=9) * x).sin()

            want = torch.autograd.grad(passes(x).sum(), layer.weight)[0]
            checkpoint(passes, x, use_reentrant=reentrant).sum().backward()
            assert torch.equal(layer.weight.grad, want)
            layer.weight.grad = None
    layer.eval()
    checkpoint(lambda x: (layer(ids) * x).sin(), x, use_reentrant=False).sum().backward()
    assert layer.weight.grad is not None


def test_a_layer_that_was_saved_draws_the_next_mask(E):
    from hades_b200.token_emb import TokenEmbedding

    ids = torch.randint(0, 40, (50,), device="cuda")
    for on_device in (False, True):
        make = lambda seed: TokenEmbedding(40, 64, dropout=0.5, seed=seed, seed_on_device=on_device)  # noqa: E731
        layer, other = make(3), make(4)
        layer(ids)
        other.load_state_dict(layer.state_dict())
        assert torch.equal(layer(ids), other(ids))
        moved = layer.cpu().cuda()
        assert torch.equal(moved(ids), other(ids)) and (not on_device or moved.seeds.state.is_cuda)


@pytest.mark.parametrize("weights,results", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                             (torch.float16, None)])
def test_the_type_of_a_layers_results(E, weights, results):
    from hades_b200.token_emb import TokenEmbedding

    layer = TokenEmbedding(40, 64, scale=2.0, padding_idx=0, dropout=0.5, dtype=weights, seed=3, out_dtype=results)
    ids = torch.randint(0, 40, (6, 50), device="cuda")
    h = layer(ids)
    assert h.dtype == (results or weights)
    assert torch.equal(h, E.cudaEmbedding(layer.weight.detach(), ids, 2.0, 0, 0.5, seed=3, offset=1, dtype=results))
    g = torch.randn_like(h)
    h.backward(g)
    want = E.cudaEmbeddingGrad(ids, g, 40, 2.0, 0, 0.5, seed=3, offset=1, dtype=weights)
    assert layer.weight.grad.dtype == weights and torch.equal(layer.weight.grad, want)
    assert layer.eval()(ids).dtype == (results or weights)


def test_empty_results_into_a_given_tensor(E):
    w = torch.randn(8, 16, device="cuda")
    for shape in ((0,), (2, 0), (0, 3), (2, 0, 3), (0, 0)):
        ids, out = torch.zeros(shape, dtype=torch.int64, device="cuda"), torch.empty((*shape, 16), device="cuda")
        assert E.cudaEmbedding(w, ids, out=out).data_ptr() == out.data_ptr()
        assert E.cudaDropout(out, 0.5, out=torch.empty_like(out)).shape == out.shape
        grad = E.cudaEmbeddingGrad(ids, out, 8, out=torch.ones_like(w), accumulate=True)
        assert bool((grad == 1).all())
        assert E.cudaEmbeddingGrad(ids, out, 0, out=w[:0]).shape == (0, 16)


def test_flags_that_are_neither_true_nor_false(E):
    ids, g = torch.arange(4, device="cuda"), torch.ones(4, 16, device="cuda")
    out = torch.zeros(8, 16, device="cuda")
    for call in (lambda: E.cudaEmbeddingGrad(ids, g, 8, out=out, accumulate=torch.ones(2)),
                 lambda: E.cudaEmbeddingGradRows(ids, g, 8, sync=torch.ones(2))):
        with pytest.raises(RuntimeError, match="ambiguous"):
            call()
    assert not out.any()


# ---- zeros of the rows that no token points to ----------------------------------------------------------------------------------
def check_every_row(E, out, ids, g, **call):
    """Into an output that held NaN, against sums in 64 bits: m terms in any order are within (m - 1) 2^-24 of the sum of their
    magnitudes, the result is rounded once more (eps / 2), and where there is no term it is +0."""
    assert bool(out.isnan().all())
    E.cudaEmbeddingGrad(ids, g, out.shape[0], out=out, **call)
    want = torch.zeros(out.shape, dtype=torch.float64, device="cuda").index_add_(0, ids, g.double())
    size = torch.zeros_like(want).index_add_(0, ids, g.double().abs())
    terms = torch.bincount(ids, minlength=out.shape[0]).double()[:, None]
    bound = (terms - 1).clamp(min=0) * 2.0 ** -24 * (1 + 2.0 ** -20) * size
    bound = bound + torch.finfo(out.dtype).eps / 2 * (want.abs() + bound) + {2: 2.0 ** -25, 4: 2.0 ** -150}[out.element_size()]
    assert bool(((out.double() - want).abs() <= bound).all())
    absent = out[terms[:, 0] == 0]
    assert not absent.any() and not torch.signbit(absent).any()


@pytest.mark.parametrize("n,vocab,dim", [
    (500, 3_000, 64), (500, 2_000, 20_011),   # few tokens; few of many bytes
    (5_000, 9_000, 100), (30_000, 60_000, 513),  # zeros beside the sort of one cluster, 123 MB of them
    (70_000, 9_000, 100), (70_000, 60_000, 513)])  # beside the sort of the whole GPU, and in front of it
@pytest.mark.parametrize("t", [torch.float32, torch.float16])
def test_every_row_is_written(E, n, vocab, dim, t):
    torch.manual_seed(n + dim)
    ids = torch.randint(0, vocab // 2, (n,), device="cuda") * 2  # every other row, the last one among the others
    g = torch.randn(n, dim, device="cuda").to(t)
    check_every_row(E, torch.full((vocab, dim), float("nan"), dtype=t, device="cuda"), ids, g)
    wide = torch.full((vocab, dim + 3), float("nan"), dtype=t, device="cuda")  # rows at a distance
    check_every_row(E, wide[:, 1:dim + 1], ids, g)
    assert bool(wide[:, 0].isnan().all()) and bool(wide[:, dim + 1:].isnan().all())


@pytest.mark.parametrize("n", [100, 3_000, 70_000])
@pytest.mark.parametrize("vocab,dim", [(50, 1001), (7, 3), (300, 1)])
def test_zeros_of_a_stretch_that_begins_anywhere(E, n, vocab, dim):
    """Two-byte values from 1 to 8 values behind a boundary of 16 bytes on; the first and the last rows have no tokens."""
    torch.manual_seed(dim)
    ids = torch.randint(2, vocab - 2, (n,), device="cuda")
    g = torch.randn(n, dim, device="cuda").half()
    for first in range(9):
        base = torch.full((vocab * dim + 24,), float("nan"), dtype=torch.float16, device="cuda")
        check_every_row(E, base[first:first + vocab * dim].view(vocab, dim), ids, g)
        assert bool(base[:first].isnan().all()) and bool(base[first + vocab * dim:].isnan().all())
