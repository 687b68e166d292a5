"""A sequence model from lookup to serving, on synthetic events.

Training: the rows of a sequence feature (one per event, PoolingMode NONE) go
through a projection to queries, keys and values, causal attention within each
user's list, and a loss on a vector of the next event; the backward updates the
projection and, by the fused rowwise Adagrad, the table.  Serving: the users'
histories fill a paged cache, then every new event costs one appended row and
one pass over the user's own cache; the results are those of the attention over
the whole lists.  With --positions queries and keys turn by their events'
positions, in training and on the way into the cache; with --bits 4 the cache
holds rows of 4 bits.

    python examples/sequence_model.py [--users 64] [--events 200] [--steps 20] [--positions] [--bits 4]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "torchlib-xpu_amd"))

import mx_fbgemm  # noqa: E402,F401  (registers torch.ops.fbgemm.* and torch.ops.mx_fbgemm.*)
from mx_fbgemm import ComputeDevice, EmbeddingLocation, PoolingMode  # noqa: E402
from mx_fbgemm.sequence_attention import PagedSequenceCache, rotary_table  # noqa: E402
from mx_fbgemm.split_table_batched_embeddings_ops_training import (  # noqa: E402
    SplitTableBatchedEmbeddingBagsCodegen,
)


class SequenceModel(torch.nn.Module):
    """One attention layer over one sequence feature's rows."""

    def __init__(self, rows: int, dim: int = 64, heads: int = 4, kv_heads: int = 2, device="cuda",
                 positions: int = 0):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, dim // heads * 2
        self.table = SplitTableBatchedEmbeddingBagsCodegen(
            [(rows, dim, EmbeddingLocation.DEVICE, ComputeDevice.CUDA)], pooling_mode=PoolingMode.NONE,
            learning_rate=0.05, device=torch.device(device))
        with torch.no_grad():
            self.table.weights_dev.normal_(0, 0.5)
        width = (heads + 2 * kv_heads) * self.head_dim
        self.project = torch.nn.Linear(dim, width, bias=False, device=device)
        self.out = torch.nn.Linear(heads * self.head_dim, dim, bias=False, device=device)
        # Angles of up to `positions` events (0: the model knows no positions).
        self.register_buffer("rotary", rotary_table(positions, self.head_dim, device=device) if positions else None)
        self.register_buffer("targets", torch.randn(rows, dim, device=device))  # of each event

    def qkv(self, rows: torch.Tensor):
        """Queries, keys and values as views of one projection's output."""
        x = self.project(rows).to(torch.bfloat16).view(rows.size(0), -1, self.head_dim)
        return x.split([self.heads, self.kv_heads, self.kv_heads], dim=1)

    def attend(self, rows: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        q, k, v = self.qkv(rows)
        if self.rotary is not None:
            q, k = (torch.ops.mx_fbgemm.jagged_rotary(x, offsets, self.rotary) for x in (q, k))
        return torch.ops.mx_fbgemm.jagged_attention(q, k, v, offsets)

    def forward(self, ids: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        return self.out(self.attend(self.table(ids, offsets), offsets).flatten(1).float())


def synthetic_batch(users: int, events: int, rows: int, seed: int):
    """Histories of 1 .. events ids, each id following from the one before."""
    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(1, events + 1, (users,), generator=g)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), lengths.cumsum(0)])
    ids = torch.randint(0, rows, (int(offsets[-1]),), generator=g).tolist()
    for b, e in zip(offsets[:-1].tolist(), offsets[1:].tolist()):
        for i in range(b + 1, e):
            ids[i] = (5 * ids[i - 1] + 17) % rows
    return torch.tensor(ids), offsets


def train(model: SequenceModel, users: int, events: int, rows: int, steps: int) -> list[float]:
    opt = torch.optim.Adam([*model.project.parameters(), *model.out.parameters()], lr=5e-3)
    ids, offsets = (x.cuda() for x in synthetic_batch(users, events, rows, 0))
    last = torch.zeros(ids.numel(), dtype=torch.bool, device="cuda")
    last[offsets[1:] - 1] = True  # a list's last event has no next one
    losses = []
    for _ in range(steps):
        y = model(ids, offsets)
        loss = (y - model.targets[ids].roll(-1, 0))[~last].square().mean()
        opt.zero_grad()
        loss.backward()  # the table's rows are updated here
        opt.step()
        losses.append(float(loss.detach()))
    return losses


@torch.no_grad()
def serve(model: SequenceModel, users: int, events: int, rows: int, new: int, bits: int = 16):
    """Histories into the cache, then `new` events per user one at a time; the
    outputs of the new events, and those of attention over the whole lists."""
    ids, offsets = (x.cuda() for x in synthetic_batch(users, events, rows, 1))
    more = torch.randint(0, rows, (new, users), generator=torch.Generator().manual_seed(2)).cuda()
    counts = offsets.diff().tolist()
    cache = PagedSequenceCache(pages=sum(-(-(n + new) // 16) for n in counts), page_size=16,
                               heads=model.kv_heads, head_dim=model.head_dim, max_sequences=users,
                               max_length=max(counts) + new, bits=bits, rotary=model.rotary)
    names = [cache.add() for _ in range(users)]
    q, k, v = model.qkv(model.table(ids, offsets))
    cache.append(names, counts, k, v)
    one_each = torch.arange(users + 1, device="cuda")
    steps = []
    for t in range(new):
        q, k, v = model.qkv(model.table(more[t], one_each))
        q = cache.append(names, [1] * users, k, v, q)  # (turned, if the cache turns keys)
        steps.append(cache.attend(names, q).clone())
    # The same from the whole lists.
    lists = [torch.cat([ids[offsets[u]:offsets[u + 1]], more[:, u]]) for u in range(users)]
    whole = torch.tensor([0, *counts]).cumsum(0).cuda() + torch.arange(users + 1, device="cuda") * new
    y = model.attend(model.table(torch.cat(lists), whole), whole)
    at = whole[1:, None] - new + torch.arange(new, device="cuda")[None, :]
    return torch.stack(steps, 1), y[at]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--users", type=int, default=64)
    ap.add_argument("--events", type=int, default=200)
    ap.add_argument("--rows", type=int, default=1000)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--new", type=int, default=8)
    ap.add_argument("--positions", action="store_true", help="rotate queries and keys by position")
    ap.add_argument("--bits", type=int, choices=(16, 4), default=16, help="of the cache")
    a = ap.parse_args()
    torch.manual_seed(0)
    model = SequenceModel(a.rows, positions=a.events + a.new if a.positions else 0)
    losses = train(model, a.users, a.events, a.rows, a.steps)
    print(f"training loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps")
    got, want = serve(model, a.users, a.events, a.rows, a.new, a.bits)
    off = float((got - want).float().norm() / want.float().norm())
    print(f"{a.new} served events of {a.users} users against the whole lists: {off:.1e} apart")


if __name__ == "__main__":
    main()
