"""The token-embedding operators whose speed counts in this repository, over the sizes, types and options they are used
with, each in its plain form (elementary torch operations) and as this package's calls.

* ``lookup``   rows of a table by token, scaled, with or without dropout: ``cudaEmbedding``
* ``dropout``  rows with a share of the values dropped, the mask from a counter-based generator: ``cudaDropout``
* ``grad``     gradient of a table from the gradients of the rows that were looked up, all of its rows:
               ``cudaEmbeddingGrad``; several micro-batches add to one gradient
* ``rows``     the same as distinct tokens and their rows, what a sparse optimiser takes: ``cudaEmbeddingGradRows``
* ``step``     lookup with dropout and its backward pass through autograd: ``token_emb.embedding``

A position whose token is the padding index gives a row of zeros and no gradient.  A value is kept where the 16 bits that
Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) gives its place are at
least T = floor(65536 p + 1/2): counter (column / 8, row, offset's low and high word), key the seed; eight values share a
call, two a word, the even column in the low half.  What is kept is multiplied by scale * 65536 / (65536 - T).
"""
import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
DIMS = (64, 100, 128, 250, 256, 512, 768, 1_001, 1_024, 2_048, 4_096, 8_192)
MASK = 0xFFFFFFFF


def listed():
    return [
        # one new token of one sequence
        {"name": "lookup_token", "kind": "lookup", "vocab": 32_768, "n": 1, "dim": 4_096, "table": "bf16", "out": "bf16",
         "ids": "int64", "scale": 1.0, "padding": "none", "p": 0.0},
        # a decoding step of many sequences, wide rows scaled by the square root of their width
        {"name": "lookup_decode", "kind": "lookup", "vocab": 131_072, "n": 256, "dim": 8_192, "table": "bf16", "out": "bf16",
         "ids": "int64", "scale": 90.5, "padding": "none", "p": 0.0},
        # a padded batch of prompts, rows of an odd width that begin nowhere in particular
        {"name": "lookup_padded_odd", "kind": "lookup", "vocab": 50_021, "n": 10_007, "dim": 1_001, "table": "fp16",
         "out": "fp32", "ids": "int64", "scale": 31.64, "padding": "-1", "p": 0.0},
        # a training batch: fp32 weights, bf16 activations, dropout behind the lookup
        {"name": "lookup_train", "kind": "lookup", "vocab": 50_000, "n": 32_768, "dim": 2_048, "table": "fp32", "out": "bf16",
         "ids": "int32", "scale": 45.25, "padding": "none", "p": 0.1},
        # rows that a small graph model has fetched
        {"name": "dropout_small", "kind": "dropout", "n": 2_000, "dim": 64, "type": "fp32", "scale": 1.0, "p": 0.5},
        # rows of the width of a products feature
        {"name": "dropout_100", "kind": "dropout", "n": 30_001, "dim": 100, "type": "fp16", "scale": 1.0, "p": 0.3},
        # activations of a large training batch
        {"name": "dropout_large", "kind": "dropout", "n": 65_536, "dim": 4_096, "type": "bf16", "scale": 1.0, "p": 0.1},
        # a small model's gradient: what launches and the host cost
        {"name": "grad_small", "kind": "grad", "vocab": 5_000, "n": 512, "dim": 256, "micro": 1, "type": "fp32",
         "table": "fp32", "ids": "int64", "scale": 1.0, "padding": "none", "p": 0.0},
        # a large vocabulary of wide rows: most of the gradient is zeros
        {"name": "grad_dense", "kind": "grad", "vocab": 131_072, "n": 8_192, "dim": 4_096, "micro": 1, "type": "bf16",
         "table": "bf16", "ids": "int64", "scale": 64.0, "padding": "none", "p": 0.0},
        # two micro-batches whose gradients are added up in fp32, dropout as in the forward pass
        {"name": "grad_micro", "kind": "grad", "vocab": 32_768, "n": 16_384, "dim": 2_048, "micro": 2, "type": "bf16",
         "table": "fp32", "ids": "int64", "scale": 1.0, "padding": "first", "p": 0.1},
        # tokens and rows for a sparse optimiser
        {"name": "rows_65k", "kind": "rows", "vocab": 262_144, "n": 65_536, "dim": 1_024, "type": "fp16", "ids": "int64",
         "scale": 1.0, "padding": "none", "p": 0.0},
        # forward and backward of the layer on a padded batch, weights and gradient in bf16
        {"name": "step_padded", "kind": "step", "vocab": 50_021, "n": 16_000, "dim": 1_024, "table": "bf16", "out": "bf16",
         "ids": "int64", "scale": 32.0, "padding": "first", "p": 0.1},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("lookup", "lookup", "dropout", "dropout", "grad", "grad", "rows", "step"))
    dim = rng.choice(DIMS) if rng.random() < 0.7 else _log_int(rng, 33, 8_192)
    scale = rng.choice((1.0, round(math.sqrt(dim), 3)))
    p = rng.choice((0.0, 0.1, round(rng.uniform(0.01, 0.6), 3)))
    any_type = tuple(TYPES)
    ids, padding = rng.choice(("int64", "int64", "int32")), rng.choice(("none", "first", "-1"))
    if kind == "dropout":
        return {"kind": kind, "n": _log_int(rng, 16, 65_536 * 2_048 // max(dim, 2_048)), "dim": dim,
                "type": rng.choice(any_type), "scale": scale, "p": p or 0.1}
    vocab = _log_int(rng, 1_000, min(262_144, 131_072 * 1_024 // dim))
    if kind == "lookup":
        return {"kind": kind, "vocab": vocab, "n": _log_int(rng, 1, 65_536 * 1_024 // max(dim, 1_024)), "dim": dim,
                "table": rng.choice(any_type), "out": rng.choice(any_type), "ids": ids, "scale": scale, "padding": padding,
                "p": p}
    n = _log_int(rng, 64, 32_768 * 1_024 // max(dim, 1_024))
    if kind == "rows":
        return {"kind": kind, "vocab": vocab, "n": n, "dim": dim, "type": rng.choice(any_type), "ids": ids, "scale": scale,
                "padding": padding, "p": p}
    if kind == "step":
        table = rng.choice(any_type)
        return {"kind": kind, "vocab": vocab, "n": n, "dim": dim, "table": table, "out": table, "ids": ids, "scale": scale,
                "padding": padding, "p": p}
    return {"kind": kind, "vocab": vocab, "n": n, "dim": dim, "micro": rng.choice((1, 1, 2)), "type": rng.choice(any_type),
            "table": rng.choice(any_type), "ids": ids, "scale": scale, "padding": padding, "p": p}


# ---- inputs ---------------------------------------------------------------------------------------------------------
ZIPF = 1.1          # power law of the tokens' frequencies
PADDED = 0.25       # share of the positions behind the ends of their sequences
DISTINCT = 0.3      # share of the positions of ``rows`` that hold a token for the first time: its outputs are as long in every batch
SIGMA_TABLE = 0.02
SIGMA_GRAD = 1e-3


def _tokens(gen, case):
    """Tokens by a bounded power law over ranks, ranks scattered over the vocabulary; tails of sequences are padding."""
    vocab, n = case["vocab"], case["n"]
    u = torch.rand(n, dtype=torch.float64, device="cuda", generator=gen)
    a, b = 1.0, (vocab + 1.0) ** (1 - ZIPF)
    ranks = ((a + u * (b - a)) ** (1 / (1 - ZIPF))).to(torch.int64).sub_(1).clamp_(0, vocab - 1)
    scattered = torch.randperm(vocab, device="cuda", generator=gen)
    if case["kind"] == "rows":
        valid, distinct = _sizes(case)
        scattered, ranks = scattered[scattered != 0][:distinct], ranks % distinct
        ranks[:distinct] = torch.arange(distinct, device="cuda")
        ids = scattered[ranks]
        ids[:valid] = ids[torch.randperm(valid, device="cuda", generator=gen)]
        ids[valid:] = _padding(case) or 0
        return ids.to(torch.int32 if case["ids"] == "int32" else torch.int64)
    ids = scattered[ranks]
    if case["padding"] != "none":
        length = max(n // 16, 1)  # sixteen sequences
        ends = torch.rand(n // length + 1, device="cuda", generator=gen) * (2 * PADDED)
        at = torch.arange(n, device="cuda")
        ids[(at % length) >= ((1 - ends[at // length]) * length)] = _padding(case)
    return ids.to(torch.int32 if case["ids"] == "int32" else torch.int64)


def _sizes(case):
    """Positions of ``rows`` that are not padding, and distinct tokens among them (not the padding's)."""
    valid = case["n"] - (int(case["n"] * PADDED) if case["padding"] != "none" else 0)
    return valid, max(1, min(int(valid * DISTINCT), case["vocab"] // 2))


def _padding(case):
    return {"none": None, "first": 0, "-1": -1}[case["padding"]]


def _normal(gen, shape, sigma, name):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, sigma, generator=gen).to(TYPES[name])


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = SimpleNamespace(case=case, kind=case["kind"], scale=case["scale"], p=case["p"])
    s.seed = int(np.random.default_rng(seed).integers(0, 1 << 62))  # of the dropout
    s.offset = 1 + seed % 1000                                      # and which call it is
    n, dim = case["n"], case["dim"]
    if s.kind == "dropout":
        s.x = _normal(gen, (n, dim), 1.0, case["type"])
        return s
    s.padding, s.vocab = _padding(case), case["vocab"]
    if s.kind in ("lookup", "step"):
        s.weight = _normal(gen, (s.vocab, dim), SIGMA_TABLE, case["table"])
    micro = case.get("micro", 1)
    s.ids = [_tokens(gen, case) for _ in range(micro)]
    if s.kind != "lookup":
        s.grads = [_normal(gen, (n, dim), SIGMA_GRAD, case.get("type") or case["out"]) for _ in range(micro)]
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if s.kind == "step":
        s.weight.requires_grad_(True)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    return (_own if own else _plain)(s)


def _own(s):
    from hades_b200 import EmbCacheLib as E
    from hades_b200 import token_emb

    drop = {"dropout": s.p, "seed": s.seed, "offset": s.offset}
    if s.kind == "dropout":
        return E.cudaDropout(s.x, s.p, seed=s.seed, offset=s.offset, scale=s.scale)
    if s.kind == "lookup":
        return E.cudaEmbedding(s.weight, s.ids[0], scale=s.scale, padding_idx=s.padding, dtype=TYPES[s.case["out"]], **drop)
    if s.kind == "rows":
        return E.cudaEmbeddingGradRows(s.ids[0], s.grads[0], s.vocab, scale=s.scale, padding_idx=s.padding, **drop)
    if s.kind == "grad":
        out = None
        for k, (ids, grad) in enumerate(zip(s.ids, s.grads)):
            out = E.cudaEmbeddingGrad(ids, grad, s.vocab, scale=s.scale, padding_idx=s.padding, dtype=TYPES[s.case["table"]],
                                      dropout=s.p, seed=s.seed, offset=s.offset + k, out=out, accumulate=k > 0)
        return out
    s.weight.grad = None
    h = token_emb.embedding(s.weight, s.ids[0], scale=s.scale, padding_idx=s.padding, **drop)
    h.backward(s.grads[0])
    return h.detach(), s.weight.grad


def _threshold(p):
    return math.floor(65536 * p + 0.5)


def _factor(scale, p):
    t = _threshold(p)
    return scale * 65536 / (65536 - t) if t < 65536 else 0.0


def _kept(s, offset, n, dim):
    """[n, dim] truth values, Philox in 64-bit integers whose products wrap as the generator's do."""
    blocks = (dim + 7) // 8
    c0 = torch.arange(blocks, device="cuda").expand(n, blocks)
    c1 = torch.arange(n, device="cuda").unsqueeze(1).expand(n, blocks)
    c2, c3 = torch.full_like(c0, offset & MASK), torch.full_like(c0, offset >> 32)
    k0, k1 = s.seed & MASK, s.seed >> 32
    for _ in range(10):
        m0, m1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (m1 >> 32 & MASK) ^ c1 ^ k0, m1 & MASK, (m0 >> 32 & MASK) ^ c3 ^ k1, m0 & MASK
        k0, k1 = (k0 + 0x9E3779B9) & MASK, (k1 + 0xBB67AE85) & MASK
    halves = torch.stack([w >> shift & 0xFFFF for w in (c0, c1, c2, c3) for shift in (0, 16)], dim=2)
    return halves.reshape(n, 8 * blocks)[:, :dim] >= _threshold(s.p)


def _dropped(s, rows, offset):
    """fp32 rows, scaled, zeros where values are dropped."""
    rows = rows * _factor(s.scale, s.p)
    if _threshold(s.p):
        rows = torch.where(_kept(s, offset, *rows.shape), rows, 0.0)
    return rows


def _plain_lookup(s, ids):
    rows = _dropped(s, s.weight.detach()[ids.clamp(0, s.vocab - 1)].float(), s.offset)
    if s.padding is not None:
        rows = torch.where((ids != s.padding).unsqueeze(1), rows, 0.0)
    return rows.to(TYPES[s.case["out"]])


def _plain_grad(s, total, ids, grad, offset):
    rows = _dropped(s, grad.float(), offset)
    if s.padding is not None:
        rows, ids = rows[ids != s.padding], ids[ids != s.padding]
    return total.index_add_(0, ids, rows)


def _plain(s):
    if s.kind == "dropout":
        return _dropped(s, s.x.float(), s.offset).to(s.x.dtype)
    if s.kind == "lookup":
        return _plain_lookup(s, s.ids[0])
    dim = s.case["dim"]
    if s.kind == "rows":
        rows, ids = _dropped(s, s.grads[0].float(), s.offset), s.ids[0]
        if s.padding is not None:
            rows, ids = rows[ids != s.padding], ids[ids != s.padding]
        uniq, inverse = torch.unique(ids.long(), return_inverse=True)
        return uniq, torch.zeros((uniq.numel(), dim), device="cuda").index_add_(0, inverse, rows)
    total = torch.zeros((s.vocab, dim), device="cuda")
    if s.kind == "grad":
        out = TYPES[s.case["table"]]
        for k, (ids, grad) in enumerate(zip(s.ids, s.grads)):
            total = _plain_grad(s, total, ids, grad, s.offset + k).to(out)  # (a gradient between two calls has its type)
            total = total.float() if k + 1 < len(s.ids) else total
        return total
    h = _plain_lookup(s, s.ids[0])
    return h, _plain_grad(s, total, s.ids[0], s.grads[0], s.offset).to(s.weight.dtype)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def _distinct(case):
    """Expected number of distinct tokens of a batch."""
    if case["kind"] == "rows":
        return _sizes(case)[1]
    vocab, n = case["vocab"], case["n"] * (1 - PADDED if case["padding"] != "none" else 1)
    edges = np.arange(1, vocab + 2, dtype=np.float64) ** (1 - ZIPF)
    p = (edges[:-1] - edges[1:]) / (edges[0] - edges[-1])
    return float(-np.expm1(n * np.log1p(-np.minimum(p, 0.999999))).sum())


def work(case):
    n, dim, kind = case["n"], case["dim"], case["kind"]
    if kind == "dropout":
        return {"bytes": 2 * n * dim * BYTES[case["type"]], "flops": n * dim}
    ids = n * (4 if case["ids"] == "int32" else 8)
    valid = n * (1 - PADDED if case["padding"] != "none" else 1)
    distinct = _distinct(case)
    lookup = ids + distinct * dim * BYTES[case.get("table", "fp32")] + n * dim * BYTES[case.get("out", "fp32")]
    if kind == "lookup":
        return {"bytes": int(lookup), "flops": n * dim}
    taken = ids + valid * dim * BYTES[case.get("type") or case["out"]]
    if kind == "rows":
        return {"bytes": int(taken + distinct * (8 + dim * 4)), "flops": int(valid * dim)}
    whole = case["vocab"] * dim * BYTES[case["table"]]
    if kind == "step":
        return {"bytes": int(lookup + taken + whole), "flops": int(2 * valid * dim)}
    micro = case["micro"]
    return {"bytes": int(micro * taken + whole + (micro - 1) * 2 * distinct * dim * BYTES[case["table"]]),
            "flops": int(micro * valid * dim)}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def _mul32(a, b):
    """High and low word of a product of 32-bit numbers by the halves of b, no intermediate beyond 49 bits."""
    low, high = a * (b & 0xFFFF), a * (b >> 16)
    mid = (low >> 16) + (high & 0xFFFF)
    return (high >> 16) + (mid >> 16), ((mid & 0xFFFF) << 16) | (low & 0xFFFF)


def _exact_rows(x, case, seed, offset):
    """float64 rows, scaled, zeros where values are dropped, a stretch of rows at a time."""
    n, dim = x.shape
    p = case["p"]
    drop_below = int(math.floor(p * 2.0 ** 16 + 0.5))
    out = x.double() * (case["scale"] / (1.0 - drop_below / 2.0 ** 16))
    if drop_below == 0:
        return out
    blocks = -(-dim // 8)
    step = max(1, (1 << 23) // blocks)
    for r0 in range(0, n, step):
        r1 = min(n, r0 + step)
        at = torch.arange((r1 - r0) * blocks, device=x.device)
        ctr = [at % blocks, r0 + at // blocks, torch.full_like(at, offset % 2 ** 32), torch.full_like(at, offset // 2 ** 32)]
        for i in range(10):
            key = ((seed % 2 ** 32 + i * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + i * 0xBB67AE85) % 2 ** 32)
            h0, l0 = _mul32(ctr[0], 0xD2511F53)
            h1, l1 = _mul32(ctr[2], 0xCD9E8D57)
            ctr = [h1 ^ ctr[1] ^ key[0], l1, h0 ^ ctr[3] ^ key[1], l0]
        draws = torch.empty(((r1 - r0) * blocks, 8), dtype=torch.int64, device=x.device)
        for j in range(8):
            draws[:, j] = ctr[j // 2] // (65536 if j % 2 else 1) % 65536
        draws = draws.view(r1 - r0, blocks * 8)[:, :dim]
        out[r0:r1].masked_fill_(draws < drop_below, 0.0)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "dropout":
        return _exact_rows(s.x, case, s.seed, s.offset)
    tokens = [t.long() for t in s.ids]
    pad = -2 if s.padding is None else s.padding

    def looked_up():
        valid = tokens[0] != pad
        rows = s.weight.index_select(0, torch.where(valid, tokens[0], torch.zeros_like(tokens[0])))
        return _exact_rows(rows, case, s.seed, s.offset) * valid.unsqueeze(1)

    if kind == "lookup":
        return looked_up()
    total = torch.zeros((s.vocab, case["dim"]), dtype=torch.float64, device="cuda")
    for k, (t, g) in enumerate(zip(tokens, s.grads)):
        rows = _exact_rows(g, case, s.seed, s.offset + k)
        total.index_put_((t[t != pad],), rows[t != pad], accumulate=True)
    if kind == "rows":
        present = torch.bincount(tokens[0][tokens[0] != pad], minlength=s.vocab).nonzero().flatten()
        return present, total[present]
    return (looked_up(), total) if kind == "step" else total
