"""Approximate search from end to end: index embeddings, look queries up, rank their candidates with rows held in 4 bits,
compare with an exhaustive search over the same rows, and take a training step of a query encoder on the candidate lists.

    python examples/rank_candidates.py [--rows 1000000] [--queries 10000] [--features 128] [--top 10]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import culsh_b200 as culsh  # noqa: E402


def main(rows=1_000_000, queries=10_000, features=128, top=10, tables=16, hashes=14, temperature=0.05, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    X = torch.nn.functional.normalize(torch.randn(rows, features, generator=gen, device="cuda"))
    source = torch.randint(0, rows, (queries,), generator=gen, device="cuda")  # the row that a query is a disturbed copy of
    noise = torch.randn(queries, features, generator=gen, device="cuda") * (0.5 / features ** 0.5)
    Q = torch.nn.functional.normalize(X[source] + noise)

    model = culsh.RPLSH(tables, hashes, seed=seed).fit(X)
    held = culsh.MXRows(X)  # 17 bytes for 32 values: what a service keeps of the rows
    candidates = model.query(Q)
    best = culsh.rank(held, Q, candidates, top_k=top, metric="cosine", temperature=temperature, targets=source)
    found = float((best.top_ids[:, 0] == source).float().mean())

    few = min(queries, 256)
    every = culsh.rank(held, Q[:few], top_k=top, metric="cosine", temperature=temperature)
    hits = (best.top_ids[:few, :, None] == every.top_ids[:, None, :]) & (best.top_ids[:few, :, None] >= 0)
    recall = float(hits.any(1).float().mean())

    # one step of a linear query encoder: raise the log probability of the source among the candidates
    scores = held.score(Q, candidates, metric="dot")
    before = culsh.log_probs(scores, source, candidates, temperature=temperature)
    seen = torch.isfinite(before.log_probs)
    grad = culsh.log_probs_backward(scores, source, before.lse, before.entropy, -seen.float() / seen.sum().clamp(min=1), lists=candidates,
                                    temperature=temperature)
    owner = torch.repeat_interleave(torch.arange(queries, device="cuda"), candidates.get_counts(as_torch=True).long())
    ids = candidates.get_indices(as_torch=True).long()
    grad_Q = torch.zeros_like(Q).index_add_(0, owner, grad[:, None] * held.dequantize()[ids])
    W = torch.eye(features, device="cuda") - 0.1 * (grad_Q.T @ Q)
    after = culsh.log_probs(held.score(Q @ W.T, candidates, metric="dot"), source, candidates, temperature=temperature)
    loss = [float(-r.log_probs[seen].mean()) for r in (before, after)]

    print(f"{rows} rows of {features} values in {held.size_bytes() / 1e6:.1f} MB, {candidates.n_total_candidates} candidates for {queries} queries")
    print(f"the query's own row comes first for {100 * found:.1f} %; {100 * recall:.1f} % of the {top} best of all rows are among the candidates' {top} best")
    print(f"mean entropy {float(best.entropy.mean()):.2f} nats; loss of the encoder {loss[0]:.4f}, after a step {loss[1]:.4f}")
    return found, recall, loss


if __name__ == "__main__":
    p = argparse.ArgumentParser()
    for name, value in (("rows", 1_000_000), ("queries", 10_000), ("features", 128), ("top", 10)):
        p.add_argument("--" + name, type=int, default=value)
    main(**vars(p.parse_args()))
