"""Token embeddings of language models with autograd: scaled lookup, dropout whose mask is not stored, gradients by
sorted tokens (``cudaEmbedding``, ``cudaDropout``, ``cudaEmbeddingGrad`` of ``EmbCacheLib``).  The reference has no such
layer; ``dist_emb.DistEmb`` takes its dropout from here.

    layer = TokenEmbedding(50_000, 1_024, scale=32.0, padding_idx=0, dropout=0.1, dtype=torch.bfloat16)
    h = layer(tokens)                 # [*tokens.shape, 1024]
    loss(h).backward()                # layer.weight.grad: every row, in the type of the weights

With a sparse optimiser the table is a ``ShardedEmbedding`` and the looked-up rows are the leaf, as in ``DistEmb``:

    h = cudaEmbedding(emb.weight, tokens, scale=s).requires_grad_()
    loss(h).backward()
    rows = cudaEmbeddingGradRows(tokens, h.grad, emb.num_embeddings, scale=s, sync=False)
    optimizer.update(rows[0], rows[1], is_unique=True, n_dev=rows[2])

Captured graphs: masks come from numbers that a graph would repeat at every replay, so that a captured layer keeps them on
the GPU (``seed_on_device=True``).  A graph of the same weights that was built outside of the capture must be gone before:
its gradient accumulation belongs to another stream, which a capture cannot wait for, so both calls below refuse it.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import EmbCacheLib as E
from . import _lib


def embedding(weight, ids, scale: float = 1.0, padding_idx: int | None = None, dropout: float = 0.0, seed: int = 0,
              offset: int = 0, rng: torch.Tensor | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``cudaEmbedding``, differentiable (once, in reverse) in weight, all of whose rows the gradient has, zeros where no token
    points.  Derivatives in forward mode and traces (``torch.jit.trace``, ``make_fx``) are refused."""
    return (_lib._NATIVE or _lib.native()).embedding_autograd(weight, ids, scale, padding_idx, dropout, seed, offset, rng, dtype)


def dropout(x, p: float, seed: int = 0, offset: int = 0, rng: torch.Tensor | None = None, scale: float = 1.0,
            dtype: torch.dtype | None = None) -> torch.Tensor:
    """``cudaDropout``, differentiable (once, in reverse) in x."""
    return (_lib._NATIVE or _lib.native()).dropout_autograd(x, scale, p, seed, offset, rng, dtype)


class DropoutSeeds:
    """The (seed, offset) of a layer's masks: a seed, and the number of masks so far.  seed None: drawn from torch's
    default generator.  on_device: both are kept on that GPU and advanced there, so that every replay of a captured graph
    draws another mask."""

    def __init__(self, seed: int | None = None, on_device=None):
        self.seed = int(torch.randint(0, 1 << 62, (1,)).item()) if seed is None else int(seed)
        E._check(0 <= self.seed < 1 << 63, "0 <= seed < 2^63")
        self.offset = 0
        self.state = None
        if on_device is not None:
            self.state = torch.tensor([self.seed, 0], dtype=torch.int64, device=on_device)

    def next(self) -> dict:
        """The next mask, as the arguments of ``cudaDropout`` and its like.  Not within a backward pass: a forward pass that
        is run again there (activation checkpointing) needs the mask that it had."""
        E._check(torch._C._current_graph_task_id() == -1,
                 "a forward pass that runs again within a backward pass (activation checkpointing) would draw another mask: "
                 "call token_emb.embedding or token_emb.dropout with a seed and an offset of your own there")
        if self.state is None:
            self.offset += 1
            return {"seed": self.seed, "offset": self.offset}
        self.state[1] += 1
        return {"rng": self.state.clone()}  # (the backward pass reads it after the next call has advanced the state)

    def state_dict(self) -> dict:
        """Seed and number of masks so far, for a run that continues (one host read where they are on the GPU)."""
        return {"seed": self.seed, "offset": self.offset if self.state is None else int(self.state[1].item())}

    def load_state_dict(self, state: dict) -> None:
        self.seed, self.offset = int(state["seed"]), int(state["offset"])
        if self.state is not None:
            self.state.copy_(torch.tensor([self.seed, self.offset]))

    def to(self, device) -> None:
        """Moves what is kept on a GPU (a captured graph goes on with the tensor that it was captured with)."""
        if self.state is not None and torch.device(device).type != "meta":
            self.state = self.state.to(device)


class MaskedModule(nn.Module):
    """A module that drops a share ``dropout`` of its values by ``seeds``: seed and number of masks are saved with it and move
    with it, so that a run that continues draws the next mask.  (Ranks that all load one state draw the same masks from
    there on.)  A state without them leaves them as they are."""

    def get_extra_state(self) -> torch.Tensor:
        s = self.seeds
        if s is None or s.state is None:
            return torch.tensor([s.seed, s.offset] if s else [])
        return s.state.clone()

    def set_extra_state(self, state: torch.Tensor) -> None:
        if self.dropout:
            seed, offset = state.tolist()
            self.seeds.load_state_dict({"seed": seed, "offset": offset})

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        if not self.dropout:
            del destination[prefix + "_extra_state"]

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, *args):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, *args)
        missing_keys[:] = [key for key in missing_keys if key != prefix + "_extra_state"]

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        if self.seeds is not None and self.seeds.state is not None:
            self.seeds.to(fn(self.seeds.state).device)
        return self


class TokenEmbedding(MaskedModule):
    """A table of [num_embeddings, embedding_dim] weights on the GPU, looked up by token, results in ``out_dtype`` (None: the
    weights').  Values are multiplied by ``scale``; in training a share ``dropout`` of them is dropped.  Every forward pass
    draws another mask; one that is run again within a backward pass (activation checkpointing) is refused: call
    ``embedding`` with numbers of your own there."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float = 1.0, padding_idx: int | None = None,
                 dropout: float = 0.0, dtype=torch.float32, device="cuda", init_sigma: float = 0.02, seed: int | None = None,
                 seed_on_device: bool = False, out_dtype: torch.dtype | None = None):
        super().__init__()
        E._check(0.0 <= dropout <= 1.0, "0 <= dropout <= 1")
        self.scale, self.padding_idx, self.dropout, self.out_dtype = float(scale), padding_idx, float(dropout), out_dtype
        weight = torch.empty((num_embeddings, embedding_dim), dtype=dtype, device=device).normal_(0.0, init_sigma)
        if padding_idx is not None and 0 <= padding_idx < num_embeddings:
            weight[padding_idx].zero_()
        self.weight = nn.Parameter(weight)
        self.seeds = DropoutSeeds(seed, device if seed_on_device else None)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        drop = {"dropout": self.dropout, **self.seeds.next()} if self.training and self.dropout else {}
        return embedding(self.weight, ids, self.scale, self.padding_idx, dtype=self.out_dtype, **drop)
