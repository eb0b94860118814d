"""Trains bucket layers on a residual stream, with the operators that stand around them.

The features are those of a LayerStack (examples/learned_buckets.py), which form the
residual; a position's stage of the game, a whole number that the features do not hold,
adds a row of a table to it:

    s = features + dropout(table[stage])
    h = RMS norm(s)
    bucket, gate = the best top_k of h W^T and their shares
    y = sum over them of gate * U_bucket clipped relu(L_bucket h)
    value = mean over the columns of (s + y) v

with layers L_e (hidden x width) and U_e (width x hidden) a bucket.  The positions of each
bucket lie side by side, with room for a fixed number of them, so that a batched product
takes all buckets at once and nothing waits for a count: a step can be recorded into a
graph.  Embedding, dropout, norm, gate, rows and the Muon updates are this package's
operators; the products are torch's.

    python examples/bucket_layers.py --steps 60
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
    sys.path.insert(0, str(Path(__file__).resolve().parent))

from learned_buckets import features  # noqa: E402
from tatara_amd import ops  # noqa: E402


class BucketLayers:
    """The model, its gradients and its updates, for batches of one size."""

    def __init__(self, positions: int, width: int, buckets: int, top_k: int, stages: int, hidden: int = 32,
                 p: float = 0.1, balance: float = 0.01, room: float = 1.5, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n, k, e = positions, top_k, buckets

        def empty(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device="cuda")

        def normal(*shape):
            return torch.randn(shape, device="cuda", generator=g) / math.sqrt(shape[-1])

        self.embedding = ops.Embedding(stages, width, n)
        self.dropout = ops.Dropout(width, p, seed=seed)
        self.norm = ops.RMSNorm(width)
        self.gate = ops.BucketGate(e, k, renormalise=True, balance=balance)
        self.rows = ops.BucketRows(e, width, k, capacity=math.ceil(room * n * k / e))
        self.table, self.weight = normal(stages, width), torch.ones(width, device="cuda")
        self.w, self.l, self.u, self.v = normal(1, e, width), normal(e, hidden, width), normal(e, width, hidden), \
            torch.randn(width, device="cuda", generator=g)
        self.muon = [ops.Muon(*x.shape) for x in (self.w, self.l, self.u)]
        self.momentum = [torch.zeros_like(x) for x in (self.w, self.l, self.u)]
        m = self.rows.rows(n)
        self.step_count = torch.zeros(1, dtype=torch.int64, device="cuda")  # other masks every step
        self.looked_up, self.dropped, self.s, self.h = (empty(n, width) for _ in range(4))
        self.rstd = empty(n)
        self.bucket, self.share = empty(n, k, dtype=torch.int32), empty(n, k)
        self.count, self.prob = empty(e, dtype=torch.int32), empty(e)
        self.counted, self.balance_loss = empty(1, dtype=torch.int32), empty(1)
        self.slot, self.source, self.offset = (empty(*shape, dtype=torch.int32) for shape in ((n, k), (m,), (e + 1,)))
        self.sorted, self.dup = empty(m, width), empty(m, width)
        self.y, self.dshare, self.dlogits = empty(n, width), empty(n, k), empty(n, e)
        self.dh, self.ds, self.dlooked_up = (empty(n, width) for _ in range(3))
        self.dtable, self.dweight = torch.empty_like(self.table), torch.empty_like(self.weight)
        for op in (self.embedding, self.norm, self.gate, self.rows, *self.muon):
            op.prepare()

    def forward(self, x: torch.Tensor, stage: torch.Tensor) -> torch.Tensor:
        """The positions' values [n]."""
        e = self.w.shape[1]
        self.embedding.forward(stage, self.table, self.looked_up)
        self.dropout.forward(self.looked_up, self.dropped, more_steps=self.step_count)
        self.norm.forward(self.dropped, self.weight, self.h, self.rstd, residual=x, total=self.s)
        self.logits = self.h @ self.w[0].t().contiguous()
        self.gate.forward(self.logits, self.bucket, self.share, self.count, self.prob, self.counted,
                          self.balance_loss)
        self.rows.sort(self.bucket, self.slot, self.source, self.offset)
        self.rows.gather(self.h, self.slot, self.source, self.sorted)
        self.a = torch.bmm(self.sorted.view(e, -1, self.sorted.shape[1]), self.l.transpose(1, 2).contiguous())
        self.up = torch.bmm(self.a.clamp(0.0, 1.0), self.u.transpose(1, 2).contiguous()).view(self.sorted.shape)
        self.rows.combine(self.up, self.slot, self.share, self.y)
        return (self.s + self.y) @ self.v / len(self.v)

    def backward(self, dout: torch.Tensor, stage: torch.Tensor) -> None:
        """The gradients of dw, dl, du, dv, dweight and dtable from that of the values."""
        e, width = self.w.shape[1], len(self.v)
        self.dv = dout @ (self.s + self.y) / width
        dy = dout[:, None] * (self.v / width)
        self.rows.combine_backward(dy, self.up, self.slot, self.source, self.share, self.dup, dgate=self.dshare)
        dup = self.dup.view(e, -1, width)
        self.du = torch.bmm(dup.transpose(1, 2).contiguous(), self.a.clamp(0.0, 1.0))
        da = torch.bmm(dup, self.u) * ((self.a > 0.0) & (self.a < 1.0))
        self.dl = torch.bmm(da.transpose(1, 2).contiguous(), self.sorted.view(e, -1, width))
        self.rows.gather_backward(torch.bmm(da, self.l).view(-1, width), self.slot, self.dh)
        self.gate.backward(self.logits, self.bucket, self.count, self.counted, self.dlogits, dgate=self.dshare)
        self.dw = (self.dlogits.t().contiguous() @ self.h).view_as(self.w)
        self.dh += self.dlogits @ self.w[0]
        self.norm.backward(self.dh, self.s, self.weight, self.rstd, self.ds, self.dweight, dtotal=dy)
        self.dropout.backward(self.ds, self.dlooked_up, more_steps=self.step_count)
        self.embedding.backward(self.dlooked_up, stage, self.dtable)

    def step(self, x: torch.Tensor, stage: torch.Tensor, target: torch.Tensor, lr: float) -> torch.Tensor:
        """One training step; the squared error before it."""
        error = self.forward(x, stage) - target
        self.backward(2.0 * error / len(error), stage)
        for muon, weights, momentum, d in zip(self.muon, (self.w, self.l, self.u), self.momentum,
                                              (self.dw, self.dl, self.du)):
            muon.step(weights, momentum, d, lr)
        for weights, d in ((self.table, self.dtable), (self.weight, self.dweight), (self.v, self.dv)):
            weights.sub_(lr * d)
        self.step_count += 1
        return (error * error).mean()


def train(steps: int = 60, positions: int = 2048, width: int = 256, buckets: int = 9, top_k: int = 2,
          stages: int = 32, lr: float = 0.02) -> list[dict]:
    """Trains the model on seeded values; one record a step."""
    model = BucketLayers(positions, width, buckets, top_k, stages)
    g = torch.Generator(device="cuda").manual_seed(9)
    bonus = torch.randn(stages, device="cuda", generator=g)
    direction = torch.randn(width, device="cuda", generator=g) / math.sqrt(width)
    history = []
    for step in range(steps):
        x = features(positions, width, step % 8)
        stage = torch.randint(0, stages, (positions,), device="cuda", generator=g, dtype=torch.int32)
        target = (x - 0.4) @ direction + 0.2 * bonus[stage.long()]
        error = model.step(x, stage, target, lr * (1.0 - step / steps))
        history.append(dict(step=step, error=float(error), balance=float(model.balance_loss),
                            counts=model.count.tolist(), dropped=int((model.slot < 0).sum())))
    return history


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--positions", type=int, default=2048)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--buckets", type=int, default=9)
    ap.add_argument("--top-k", type=int, default=2)
    a = ap.parse_args()
    for r in train(a.steps, a.positions, a.width, a.buckets, a.top_k):
        if r["step"] % 10 == 0 or r["step"] + 1 == a.steps:
            print(f"step {r['step']:4d}  squared error {r['error']:.5f}  balance loss {r['balance']:.5f}  "
                  f"positions a bucket {r['counts']}, {r['dropped']} without a row")


if __name__ == "__main__":
    main()
