"""Trains the vectors that an index holds, then searches them.

A catalogue of items is learned as a table of unit vectors together with a
small encoder (a projection and a layer norm) that maps an item's features to
its vector: softmax cross entropy of every query against the whole catalogue
(vector_cuda.ops.linear_cross_entropy), without keeping the scores. The learned
table then becomes a cosine index (DistributedKnnEngine) and new queries are
answered from it. Synthetic data; needs a CUDA GPU and torch.

    python examples/train_and_search.py [--items N] [--dim D] [--batch B] [--steps S]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vector-rs_b200", "python"))
import vector_cuda as vc  # noqa: E402
from vector_cuda import ops  # noqa: E402


class Encoder(torch.nn.Module):
    """Features -> vector: projection, layer norm (32-bit parameters), unit length."""

    def __init__(self, features: int, dim: int):
        super().__init__()
        self.project = torch.nn.Parameter(torch.randn(features, dim, device="cuda") / features ** 0.5)
        self.weight = torch.nn.Parameter(torch.ones(dim, device="cuda"))
        self.bias = torch.nn.Parameter(torch.zeros(dim, device="cuda"))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        h = x.bfloat16() @ self.project.bfloat16()
        h = ops.layer_norm(h, self.weight, self.bias)
        return torch.nn.functional.normalize(h.float(), dim=1).bfloat16()


def main(items: int = 20000, dim: int = 128, batch: int = 1024, steps: int = 60, features: int = 96, seed: int = 7,
         quiet: bool = False):
    """Returns (first loss, last loss, share of new queries whose item is among their 10 nearest)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    torch.manual_seed(seed)
    truth = torch.randn(items, features, generator=g, device="cuda")  # what the items are like

    def queries(n):
        ids = torch.randint(0, items, (n,), generator=g, device="cuda")
        return truth[ids] + 0.5 * torch.randn(n, features, generator=g, device="cuda"), ids

    encoder = Encoder(features, dim)
    table = torch.nn.Parameter(torch.nn.functional.normalize(torch.randn(items, dim, device="cuda"), dim=1))
    params = [*encoder.parameters(), table]
    adam = torch.optim.Adam(params, lr=0.02)
    losses = []
    for step in range(steps):
        x, ids = queries(batch)
        vectors = torch.nn.functional.normalize(table, dim=1).bfloat16()
        loss = ops.linear_cross_entropy(encoder(x), vectors, ids, scale=20.0)
        adam.zero_grad(set_to_none=True)
        loss.backward()
        adam.step()
        losses.append(loss.detach())
        if not quiet and step % 20 == 0:
            print(f"step {step}: loss {losses[-1].item():.4f}")

    ops.check()

    # The same encoder at the start of a search: the index answers from the learned table.
    with torch.no_grad():
        x, ids = queries(512)
        q = encoder(x).float().cpu().numpy()
        base = torch.nn.functional.normalize(table, dim=1).cpu().numpy()
    index = vc.DistributedKnnEngine.try_new(base, dim, 1, vc.GpuShardMode.Sharded, vc.DistanceMetric.CosineSimilarity)
    _, found = index.search_arrays(q, 10)
    index.close()
    hit = float((found == ids.cpu().numpy()[:, None]).any(1).mean())
    first, last = losses[0].item(), losses[-1].item()
    if not quiet:
        print(f"loss {first:.4f} -> {last:.4f}; item among its query's 10 nearest: {hit:.3f}")
    return first, last, hit


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--items", type=int, default=20000)
    p.add_argument("--dim", type=int, default=128)
    p.add_argument("--batch", type=int, default=1024)
    p.add_argument("--steps", type=int, default=60)
    a = p.parse_args()
    main(a.items, a.dim, a.batch, a.steps)
