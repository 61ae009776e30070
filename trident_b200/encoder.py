"""A trainable query encoder in front of a fixed index, and a command that trains one.

A query's tokens are looked up in a table, scaled, normalised and averaged into the vector that the index
searches:

    x = sqrt(D) table[tokens];  y = layer_norm(x) weight + bias;  q = mean of y over the query's tokens.

The index stays as it is while the encoder learns to put its queries next to the rows that answer them: each
step searches the index for every query of the batch, takes the rows that it finds as negatives of a
contrastive loss, and updates the encoder by AdamW. The reference has no counterpart: it takes its vectors as
given.

    python -m trident_b200.encoder [--docs 20000] [--vocab 4096] [--dim 128] [--steps 200] [--state-bits 8]
"""
import argparse
import json
import math
import sys
import time

import torch

from .ops import embedding_grad, embedding_lookup, layer_norm, layer_norm_grad
from .optim import AdamW


class QueryEncoder:
    """Token table, layer norm and mean pooling. `parameters` lists the table [V, D], the weight and the bias
    [D]; `forward` gives the query vectors and `backward` their gradients in the same order."""

    def __init__(self, vocab: int, dim: int, device="cuda:0", dtype=torch.float32, seed: int = 0, eps: float = 1e-5):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.scale, self.eps = math.sqrt(dim), eps
        table = torch.randn((vocab, dim), generator=gen, device=device) / self.scale
        self.table = table.to(dtype)
        self.weight = torch.ones(dim, dtype=dtype, device=device)
        self.bias = torch.zeros(dim, dtype=dtype, device=device)
        self._saved = None

    @property
    def parameters(self):
        return [self.table, self.weight, self.bias]

    def forward(self, tokens):
        """tokens [B, L], padded with -1 -> float32 query vectors [B, D]. What backward needs is kept until the
        next forward."""
        x = embedding_lookup(self.table, tokens, scale=self.scale)
        y, mean, rstd = layer_norm(x, self.weight, self.bias, eps=self.eps)
        share = (tokens >= 0).float()
        share /= share.sum(1, keepdim=True).clamp_(min=1.0)  # a query without tokens has the vector 0
        self._saved = (tokens, x, mean, rstd, share)
        return torch.einsum("bl,bld->bd", share, y.float())

    def backward(self, grad):
        """Gradients of the parameters, given the gradient [B, D] of the last forward's vectors."""
        tokens, x, mean, rstd, share = self._saved
        dy = (share[:, :, None] * grad[:, None, :]).to(x.dtype)
        dx, dw, db = layer_norm_grad(dy, x, self.weight, mean, rstd)
        return [embedding_grad(dx, tokens, self.table.shape[0], scale=self.scale), dw, db]


def contrastive_step(encoder, optimizer, index, rows, tokens, answers, nprobe: int, k: int = 16, temperature: float = 16.0):
    """One training step. rows [N, D]: the index's float32 rows by id; answers [B]: the id that each query should
    find. Returns (loss, search hit rate) as device scalars.

    The candidates of a query are its answer and the k rows that the index finds for it; the loss is the cross
    entropy of softmax(-|q - x|^2 / temperature) on the answer. As the softmax minus the target sums to 0, its
    gradient is (2 / temperature) sum_j (p_j - target_j) x_j."""
    q = encoder.forward(tokens)
    _, found, _ = index.search(q.detach(), nprobe, mode=-1, k=k)
    ids = torch.cat([answers[:, None], found], 1)
    x = embedding_lookup(rows, ids)                       # a missing result (-1) is a row of zeros
    hit = found == answers[:, None]
    out = torch.cat([torch.zeros_like(hit[:, :1]), hit | (found < 0)], 1)
    logits = -(q[:, None, :] - x).square().sum(2) / temperature
    logits = torch.where(out, float("-inf"), logits)      # neither the answer again nor a missing row is a negative
    logp = torch.log_softmax(logits, 1)
    p = logp.exp()
    p[:, 0] -= 1.0
    grad = torch.einsum("bj,bjd->bd", p, x) * (2.0 / temperature / tokens.shape[0])
    optimizer.step(encoder.backward(grad))
    return -logp[:, 0].mean(), hit.any(1).float().mean()


def synthetic_corpus(docs: int, vocab: int, dim: int, length: int = 8, seed: int = 0, device="cuda:0"):
    """(rows [docs, dim], doc tokens [docs, length]): every token has a hidden vector, and a row is the mean of
    its document's, so that an encoder whose table learns the hidden vectors finds a document by its tokens."""
    gen = torch.Generator(device=device).manual_seed(seed)
    hidden = torch.randn((vocab, dim), generator=gen, device=device)
    hidden = (hidden - hidden.mean(1, keepdim=True)) / hidden.std(1, keepdim=True, unbiased=False)
    words = torch.randint(0, vocab, (docs, length), generator=gen, device=device)
    return hidden[words].mean(1).contiguous(), words


def queries_of(words, ids, keep: int, gen):
    """Queries for documents `ids`: `keep` of each one's tokens at random places, the others -1."""
    at = torch.rand(words[ids].shape, generator=gen, device=words.device).argsort(1)
    return torch.where(at < keep, words[ids], -1)


def recall(encoder, index, words, ids, keep: int, nprobe: int, gen, k: int = 10) -> float:
    """The share of queries for documents `ids` that find theirs among the first k."""
    q = encoder.forward(queries_of(words, ids, keep, gen))
    _, found, _ = index.search(q, nprobe, mode=-1, k=k)
    return float((found == ids[:, None]).any(1).float().mean())


def train(docs: int = 20_000, vocab: int = 4096, dim: int = 128, steps: int = 200, batch: int = 1000, nlist: int = 128,
          nprobe: int = 16, state_bits: int = 8, lr: float = 3e-2, seed: int = 0, device="cuda:0") -> dict:
    """Builds an index over a synthetic corpus, trains an encoder against it and reports recall@10 before and after."""
    from .clustering import train_clustering
    from .index import SharedClusterStorage, TridentV4Index, choose_tile

    rows, words = synthetic_corpus(docs, vocab, dim, seed=seed, device=device)
    cent, lids, _, mu, R, _ = train_clustering(rows, nlist, sample_size=min(docs, 64 * nlist), device=device)
    st = SharedClusterStorage(rows, torch.from_numpy(lids).to(device), None, nlist, device=device)
    index = TridentV4Index(st, cent, mu, R, tile_size=choose_tile(dim), device=device, max_batch=batch, max_nprobe=nprobe)
    gen = torch.Generator(device=device).manual_seed(seed + 1)
    encoder = QueryEncoder(vocab, dim, device=device, seed=seed + 2)
    optimizer = AdamW(encoder.parameters, lr=lr, weight_decay=0.0, state_bits=state_bits, seed=seed)
    probe = torch.randint(0, docs, (batch,), generator=gen, device=device)
    res = {"docs": docs, "vocab": vocab, "dim": dim, "steps": steps, "batch": batch, "state_bits": state_bits,
           "recall_before": recall(encoder, index, words, probe, 6, nprobe, gen), "losses": []}
    torch.cuda.synchronize(device)
    t0 = time.perf_counter()
    for step in range(steps):
        ids = torch.randint(0, docs, (batch,), generator=gen, device=device)
        loss, _ = contrastive_step(encoder, optimizer, index, rows, queries_of(words, ids, 6, gen), ids, nprobe)
        if step % max(1, steps // 10) == 0 or step == steps - 1:
            res["losses"].append(round(float(loss), 4))
    torch.cuda.synchronize(device)
    res["ms_per_step"] = round((time.perf_counter() - t0) / max(1, steps) * 1e3, 3)
    res["recall_after"] = recall(encoder, index, words, probe, 6, nprobe, gen)
    return res


def main(argv=None):
    p = argparse.ArgumentParser(description="Train a query encoder against a fixed index of synthetic documents.")
    p.add_argument("--docs", type=int, default=20_000)
    p.add_argument("--vocab", type=int, default=4096)
    p.add_argument("--dim", type=int, default=128)
    p.add_argument("--steps", type=int, default=200)
    p.add_argument("--batch", type=int, default=1000)
    p.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    a = p.parse_args(argv)
    print(json.dumps(train(a.docs, a.vocab, a.dim, a.steps, a.batch, state_bits=a.state_bits)), flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
