"""A small embedder and reader around the index: documents and queries through windowed attention, their
embeddings through the bitplane scan, and the passages found read back token by token over a paged 8-bit cache.

    python examples/embed_and_search.py

The model has random weights (two layers, 4 query and 2 key/value heads of 64): it shows the calls and their
order, not an embedding worth searching. Steps, in the manner of the reference's embedder (prefix KV cache,
ragged prefill):

  1. documents: one ragged batch through `window_attention` in every layer, mean over tokens, L2 norm;
  2. the index: EDEN fit, encoded pages, a device segment;
  3. queries: the instruction in front of every query goes into the cache once; each query forks it, appends
     its own tokens and attends over both (`reserve`, `append`, `attend`);
  4. the scan: top documents of every query (`query_scan`);
  5. the reader: the best document's tokens join the query's sequence, then single tokens are decoded, old
     pages are given back behind the window (`trim`), the sequences are dropped and the pool compacted.
"""
from __future__ import annotations

import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mrl-index-rust-vector_b200"))
import mrl_b200 as M  # noqa: E402

LAYERS, Q_HEADS, KV_HEADS, HEAD_DIM, DIMS, VOCAB = 2, 4, 2, 64, 256, 1000
WINDOW, SINKS = 128, 4


class Model:
    """Random weights; every layer is attention with a residual and a root-mean-square norm before it."""

    def __init__(self, seed: int = 0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rand = lambda *s: (torch.randn(*s, generator=g, device="cuda") / s[-2] ** 0.5).half()  # noqa: E731
        self.table = torch.randn(VOCAB, DIMS, generator=g, device="cuda").half()
        self.qkv = [rand(DIMS, (Q_HEADS + 2 * KV_HEADS) * HEAD_DIM) for _ in range(LAYERS)]
        self.out = [rand(Q_HEADS * HEAD_DIM, DIMS) for _ in range(LAYERS)]

    def run(self, tokens: torch.Tensor, attend) -> torch.Tensor:
        """Hidden states [tokens, DIMS]; attend(layer, q, k, v) is the attention of one layer."""
        x = self.table[tokens]
        for layer in range(LAYERS):
            y = (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).half()
            qkv = (y @ self.qkv[layer]).view(-1, Q_HEADS + 2 * KV_HEADS, HEAD_DIM)
            q, k, v = qkv[:, :Q_HEADS], qkv[:, Q_HEADS:Q_HEADS + KV_HEADS], qkv[:, Q_HEADS + KV_HEADS:]
            x = x + attend(layer, q, k, v).reshape(-1, Q_HEADS * HEAD_DIM) @ self.out[layer]
        return x


def ragged(parts):
    """Token lists packed into one tensor, and their offsets (int32)."""
    cu = np.concatenate([[0], np.cumsum([len(p) for p in parts])])
    return (torch.from_numpy(np.concatenate(parts)).cuda(), torch.from_numpy(cu.astype(np.int32)).cuda(), [int(c) for c in cu])


def pooled(x: torch.Tensor, cu) -> np.ndarray:
    """Mean over each sequence's rows, L2 norm."""
    e = torch.stack([x[a:b].float().mean(0) for a, b in zip(cu, cu[1:])])
    return (e / e.norm(dim=1, keepdim=True)).cpu().numpy()


def i32(values) -> torch.Tensor:
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def embed_documents(model: Model, dev, docs) -> np.ndarray:
    tokens, cu_dev, cu = ragged(docs)
    longest = max(len(d) for d in docs)

    def attend(layer, q, k, v):
        return M.window_attention(q, k, v, cu_dev, longest, causal=True, window=WINDOW, sinks=SINKS, dev=dev)

    return pooled(model.run(tokens, attend), cu)


class Reader:
    """Sequences over one cache."""

    def __init__(self, model: Model, dev, max_seqs: int = 32, pages: int = 256):
        self.model = model
        self.cache = M.KvCache.create(LAYERS, pages, KV_HEADS, HEAD_DIM, max_seqs, 32, dev=dev)

    def extend(self, seqs, parts) -> tuple:
        """Run new tokens of the sequences, into the cache and over it; hidden states and offsets."""
        tokens, cu_dev, cu = ragged(parts)
        ids, counts = i32(seqs), i32(len(p) for p in parts)
        self.cache.reserve(ids, counts)
        longest = max(len(p) for p in parts)

        def attend(layer, q, k, v):
            self.cache.append(layer, k, v, ids, cu_dev)
            return self.cache.attend(layer, q, ids, cu_dev, max_q=longest, window=WINDOW, sinks=SINKS)

        return self.model.run(tokens, attend), cu

    def decode(self, seqs, tokens: torch.Tensor) -> torch.Tensor:
        """One token per sequence: the next tokens, greedily against the embedding table."""
        ids = i32(seqs)
        self.cache.reserve(ids, torch.ones_like(ids))

        def attend(layer, q, k, v):
            self.cache.append(layer, k, v, ids)
            return self.cache.attend(layer, q, ids, window=WINDOW, sinks=SINKS)

        return (self.model.run(tokens, attend) @ self.model.table.T).argmax(1)


def main(n_docs: int = 640, n_queries: int = 5, steps: int = 70, seed: int = 1) -> dict:
    dev = M.Device(0)
    dev.use_torch_stream()
    model = Model()
    rng = np.random.default_rng(seed)
    docs = [rng.integers(0, VOCAB, int(n)) for n in rng.integers(5, 400, n_docs)]

    # 1, 2: documents, their embeddings, the index
    emb = embed_documents(model, dev, docs)
    fit = M.EdenFit.fit_prefix(emb)
    segment = M.Segment.upload(M.encode_blocks(emb, DIMS, eden=fit, dev=dev), dev)

    # 3: queries are pieces of documents behind an instruction that is cached once
    instruction = rng.integers(0, VOCAB, 150)
    targets = rng.permutation(n_docs)[:n_queries]
    queries = [docs[t][: max(4, len(docs[t]) // 2)] for t in targets]
    reader = Reader(model, dev)
    reader.extend([0], [instruction])
    seqs = list(range(1, 1 + n_queries))
    reader.cache.fork(i32([0] * n_queries), i32(seqs))
    hidden, cu = reader.extend(seqs, queries)
    q_emb = pooled(hidden, cu)

    # 4: the scan
    cfg = M.ScanConfig(shortlist_cand=16)
    ids, scores, counts, plan = M.query_scan(segment, q_emb, cfg, prefix_codec=M.PrefixCodec.EDEN_PROD, eden=fit)
    best = [int(r) >> 16 << 6 | int(r) & 0xFFFF for r in ids[:, 0]]  # VectorId to document number

    # 5: the reader
    hidden, cu = reader.extend(seqs, [docs[b] for b in best])
    token = (hidden[torch.tensor([c - 1 for c in cu[1:]], device="cuda")] @ model.table.T).argmax(1)
    answers = []
    for _ in range(steps):
        token = reader.decode(seqs, token)
        answers.append(token)
    lens = reader.cache.lens.tolist()
    held = int((reader.cache.refs > 0).sum())
    reader.cache.trim(i32(seqs), WINDOW, SINKS)
    trimmed = int((reader.cache.refs > 0).sum())
    reader.cache.release(i32(seqs[:-1]))
    reader.cache.compact()
    again = reader.decode(seqs[-1:], token[-1:])
    plan.free()
    out = dict(best=best, scores=scores[:, 0].tolist(), answers=torch.stack(answers).cpu().numpy(), lens=lens, held=held,
               trimmed=trimmed, compacted=int((reader.cache.refs > 0).sum()), again=int(again), status=int(reader.cache.status),
               doc_lens=[len(docs[b]) for b in best], query_lens=[len(q) for q in queries], emb=emb, q_emb=q_emb)
    segment.free()
    dev.close()
    return out


if __name__ == "__main__":
    r = main()
    print("best documents:", r["best"], "scores:", [round(s, 3) for s in r["scores"]])
    print("tokens per sequence:", r["lens"][:6], "pages held:", r["held"], "after trim:", r["trimmed"], "after release:", r["compacted"])
