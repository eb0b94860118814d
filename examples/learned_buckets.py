"""Learns which bucket a position's dense layer comes from, instead of a fixed rule.

The features are those of a LayerStack: the pairwise feature-transformer output of
seeded positions (tatara_op_ft_forward_pairwise).  On them stands a small model that
is trained here:

    h = layer norm(features)
    logits = h W^T                     the scores of the buckets
    bucket, gate = the best top_k buckets and their shares
    value = sum over them of gate * mean(clipped relu(L_bucket h))

with one layer L_e (16 x ft_out) a bucket, as LayerStack's first layers are.  It
learns a seeded teacher's values under squared error and the loss that keeps the
buckets balanced.  Layer norm, gate and both updates (Muon of W and of all L_e as one
batch) are this package's operators; the products between them are torch's.

    python examples/learned_buckets.py --steps 60
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from tatara_amd import _lib, ops  # noqa: E402
from tatara_amd.synthetic import small_spec, structured_batch  # noqa: E402

HIDDEN = 16


def features(positions: int, ft_out: int, seed: int) -> torch.Tensor:
    """[positions, ft_out] pairwise FT activations of seeded positions."""
    spec = small_spec(king_buckets=6, piece_inputs=64)
    batch, _ = structured_batch(positions, spec, seed=seed, nnz_min=32)
    g = torch.Generator(device="cuda").manual_seed(1)  # one table for all batches
    table = torch.randn(spec["ft_in"], ft_out, device="cuda", generator=g) * 0.08
    bias = torch.full((ft_out,), 0.4, device="cuda")
    rows = [torch.from_numpy(a).cuda() for a in (batch.stm_indices, batch.nstm_indices, batch.nnz)]
    raw = [torch.empty(positions, ft_out, device="cuda") for _ in range(2)]
    out = torch.empty(positions, ft_out, device="cuda")
    torch.cuda.synchronize()
    _lib.check(_lib.load().tatara_op_ft_forward_pairwise(
        table.data_ptr(), rows[0].data_ptr(), rows[1].data_ptr(), rows[2].data_ptr(), bias.data_ptr(),
        raw[0].data_ptr(), raw[1].data_ptr(), out.data_ptr(), positions, ft_out, spec["ft_in"], spec["max_active"], 0,
        127.0 / 128.0))
    return out


class LearnedBuckets:
    """The model, its gradients and its updates, for batches of one size."""

    def __init__(self, positions: int, ft_out: int, buckets: int, top_k: int, balance: float, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def empty(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device="cuda")

        self.norm = ops.LayerNorm(ft_out)
        self.gate = ops.BucketGate(buckets, top_k, renormalise=True, balance=balance)
        self.weight, self.bias = torch.ones(ft_out, device="cuda"), torch.zeros(ft_out, device="cuda")
        self.w = torch.randn(1, buckets, ft_out, device="cuda", generator=g) / math.sqrt(ft_out)
        self.layers = torch.randn(buckets, HIDDEN, ft_out, device="cuda", generator=g) / math.sqrt(ft_out)
        self.muon_w = ops.Muon(1, buckets, ft_out)
        self.muon_layers = ops.Muon(buckets, HIDDEN, ft_out)
        self.m_w, self.m_layers = torch.zeros_like(self.w), torch.zeros_like(self.layers)
        n, k = positions, top_k
        self.h, self.mean, self.rstd = empty(n, ft_out), empty(n), empty(n)
        self.bucket, self.share = empty(n, k, dtype=torch.int32), empty(n, k)
        self.count, self.prob = empty(buckets, dtype=torch.int32), empty(buckets)
        self.counted, self.balance_loss = empty(1, dtype=torch.int32), empty(1)
        self.dlogits, self.dx = empty(n, buckets), empty(n, ft_out)
        self.dweight, self.dbias = empty(ft_out), empty(ft_out)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """The positions' values [n]."""
        self.norm.forward(x, self.weight, self.bias, self.h, self.mean, self.rstd)
        self.logits = self.h @ self.w[0].t().contiguous()
        self.gate.forward(self.logits, self.bucket, self.share, self.count, self.prob, self.counted,
                          self.balance_loss)
        n, k = self.bucket.shape
        buckets = self.layers.shape[0]
        # every bucket's layer, of which the chosen ones count
        self.a = (self.h @ self.layers.view(buckets * HIDDEN, -1).t().contiguous()).view(n, buckets, HIDDEN)
        self.at = self.bucket.long().view(n, k, 1).expand(n, k, HIDDEN)
        self.chosen = self.a.gather(1, self.at)
        self.value = self.chosen.clamp(0.0, 1.0).mean(2)  # [n, k]
        return (self.share * self.value).sum(1)

    def step(self, x: torch.Tensor, target: torch.Tensor, lr: float) -> tuple[float, float]:
        """One training step; the squared error and the balance loss before it."""
        out = self.forward(x)
        n, buckets = x.shape[0], self.layers.shape[0]
        error = out - target
        dout = 2.0 * error / n
        dshare = dout[:, None] * self.value
        inside = ((self.chosen > 0.0) & (self.chosen < 1.0)) / HIDDEN
        da = torch.zeros_like(self.a).scatter_add_(1, self.at, (dout[:, None] * self.share)[:, :, None] * inside)
        da = da.view(n, buckets * HIDDEN)
        self.gate.backward(self.logits, self.bucket, self.count, self.counted, self.dlogits, dgate=dshare)
        dw = (self.dlogits.t().contiguous() @ self.h).view_as(self.w)
        dlayers = (da.t().contiguous() @ self.h).view_as(self.layers)
        dh = self.dlogits @ self.w[0] + da @ self.layers.view(buckets * HIDDEN, -1)
        self.norm.backward(dh, x, self.weight, self.mean, self.rstd, self.dx, self.dweight, self.dbias)
        self.muon_w.step(self.w, self.m_w, dw, lr)
        self.muon_layers.step(self.layers, self.m_layers, dlayers, lr)
        self.weight -= lr * self.dweight
        self.bias -= lr * self.dbias
        return float((error * error).mean()), float(self.balance_loss)


def train(steps: int = 60, positions: int = 2048, ft_out: int = 256, buckets: int = 9, top_k: int = 2,
          balance: float = 0.01, lr: float = 0.02) -> list[dict]:
    """Trains the model; one record a step."""
    model = LearnedBuckets(positions, ft_out, buckets, top_k, balance)
    g = torch.Generator(device="cuda").manual_seed(9)
    teacher = torch.randn(ft_out, 3, device="cuda", generator=g) / math.sqrt(ft_out)
    history = []
    for step in range(steps):
        x = features(positions, ft_out, step % 8)
        z = (x - x.mean(1, keepdim=True)) / (x.std(1, keepdim=True) + 1e-5) @ teacher
        target = 0.3 + 0.1 * torch.where(z[:, 0] > 0, z[:, 1], z[:, 2])  # which of two rules holds is for the gate to find
        error, balance_loss = model.step(x, target, lr * (1.0 - step / steps))
        history.append(dict(step=step, error=error, balance=balance_loss, counts=model.count.tolist()))
    return history


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--positions", type=int, default=2048)
    ap.add_argument("--ft-out", type=int, default=256)
    ap.add_argument("--buckets", type=int, default=9)
    ap.add_argument("--top-k", type=int, default=2)
    a = ap.parse_args()
    for r in train(a.steps, a.positions, a.ft_out, a.buckets, a.top_k):
        if r["step"] % 10 == 0 or r["step"] + 1 == a.steps:
            print(f"step {r['step']:4d}  squared error {r['error']:.5f}  balance loss {r['balance']:.5f}  "
                  f"positions a bucket {r['counts']}")


if __name__ == "__main__":
    main()
