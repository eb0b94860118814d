"""The operators of a learned bucket choice and of orthogonalised updates, as cases that can be timed and compared.

A LayerStack's position goes to one of a few buckets, each with dense layers of
its own.  A program that learns this choice normalises the position's features
(layer norm), scores the buckets (a product), takes the best few of them with a
loss that keeps the buckets balanced (the gate), and updates its matrices, the
stack's per-bucket layers and the feature transformer's king blocks among them,
by orthogonalised momentum (Muon).  The cases take these calls over the sizes of
this repository's networks and over generic ones.

With `own` false the operators are computed from elementary torch operations in
32 bits; with `own` true by tatara_amd.ops.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
BALANCE = 0.01
MUON = dict(beta=0.95, nesterov=True, weight_decay=0.01)
NORM_EPS = 1e-7
A, B, C = 3.4445, -4.7750, 2.0315  # the quintic of the Newton-Schulz steps
STEPS = 5
CLAMP = 127.0 / 64.0  # the dense layers' weight range
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed() -> list[dict]:
    return [
        # A batch's feature activations at the headline width, normalised.
        dict(name="norm_f32_65536x1536", kind="norm", rows=65536, cols=1536, pad=0, dtype="f32"),
        # One position that is scored on its own.
        dict(name="norm_bf16_1x1536", kind="norm", rows=1, cols=1536, pad=0, dtype="bf16"),
        # The training step's other half, in half the bytes.
        dict(name="norm_grad_bf16_65536x1536", kind="norm_grad", rows=65536, cols=1536, pad=0, dtype="bf16"),
        # A small odd batch of rows that lie inside wider ones, as the column
        # range of a concatenated activation does.
        dict(name="norm_grad_f32_1009x769", kind="norm_grad", rows=1009, cols=769, pad=10, dtype="f32"),
        # The choice among the nine buckets for the headline batch.
        dict(name="gate_f32_65536x9", kind="gate", rows=65536, buckets=9, top=1, pad=0, dtype="f32", masked=False,
             share=False),
        # One position, blended over its two best buckets.
        dict(name="gate_f32_1x8_top2", kind="gate", rows=1, buckets=8, top=2, pad=0, dtype="f32", masked=False,
             share=True),
        # The gradient of the same choice.
        dict(name="gate_grad_f32_65536x9", kind="gate_grad", rows=65536, buckets=9, top=1, pad=0, dtype="f32",
             masked=False, share=False),
        # Many buckets, several of them a position; an odd batch with positions
        # that do not count and buckets that a position may not take.
        dict(name="gate_grad_bf16_16381x64_top4", kind="gate_grad", rows=16381, buckets=64, top=4, pad=0,
             dtype="bf16", masked=True, share=True),
        # The per-bucket first layers (9 x 16 x 1536): small, so latency counts.
        dict(name="muon_f32_9x16x1536", kind="muon", batch=9, rows=16, cols=1536, dtype="f32"),
        # The feature transformer: every king block's table as a matrix.
        dict(name="muon_f32_45x1629x1536", kind="muon", batch=45, rows=1629, cols=1536, dtype="f32"),
        # The orthogonal factor alone, of one generic matrix in 16 bits.
        dict(name="ortho_bf16_1x2048x1024", kind="ortho", batch=1, rows=2048, cols=1024, dtype="bf16"),
        # The same of a few odd ones in 32 bits.
        dict(name="ortho_f32_5x257x391", kind="ortho", batch=5, rows=257, cols=391, dtype="f32"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "norm_grad", "gate", "gate_grad", "muon", "ortho"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind in ("norm", "norm_grad"):
        cols = rng.choice([256, 512, 768, 1024, 1536, 2048, _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)])
        rows = _log_int(rng, 1, min(65536, 65536 * 1536 // cols))
        return dict(kind=kind, rows=rows, cols=cols, pad=rng.choice([0, 0, 8, rng.randint(1, 40)]), dtype=dtype)
    if kind in ("gate", "gate_grad"):
        buckets = rng.choice([8, 9, _log_int(rng, 2, 256), _log_int(rng, 2, 256)])
        return dict(kind=kind, rows=_log_int(rng, 1, 65536), buckets=buckets,
                    top=rng.randint(1, min(8, buckets)), pad=rng.choice([0, 0, rng.randint(1, 9)]), dtype=dtype,
                    masked=rng.random() < 0.4, share=rng.random() < 0.5)
    rows, cols = _log_int(rng, 16, 2048), _log_int(rng, 16, 2048)
    most = max(1, min(64, int(45 * _products(1629, 1536) / _products(rows, cols))))
    return dict(kind=kind, batch=_log_int(rng, 1, most), rows=rows, cols=cols, dtype=dtype)


def _products(rows: int, cols: int) -> float:
    """Operations of one matrix's Newton-Schulz steps: the two symmetric
    products' halves and the full one, on the smaller side."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (3.0 * m * m * n + 1.0 * m * m * m)


def work(case: dict) -> dict:
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind in ("norm", "norm_grad"):
        r, c = case["rows"], case["cols"]
        if kind == "norm":  # x in, y, mean and rstd out
            return dict(bytes=2 * r * c * e + 8 * r + 8 * c, flops=8 * r * c)
        return dict(bytes=3 * r * c * e + 8 * r + 12 * c, flops=13 * r * c)
    if kind in ("gate", "gate_grad"):
        t, b, k = case["rows"], case["buckets"], case["top"]
        mask = t if case["masked"] else 0
        if kind == "gate":  # logits in; bucket, gate, counts, sums, loss out
            return dict(bytes=t * b * e + 8 * t * k + 8 * b + mask, flops=6 * t * b)
        return dict(bytes=2 * t * b * e + 8 * t * k + 4 * b + mask, flops=9 * t * b)
    n = case["batch"] * case["rows"] * case["cols"]
    flops = case["batch"] * _products(case["rows"], case["cols"])
    if kind == "ortho":
        return dict(bytes=2 * n * e, flops=flops)
    return dict(bytes=n * (e + 16), flops=flops)  # gradient in, weights and momentum in and out


# ---------------------------------------------------------------------------
# what a program holds before the call
# ---------------------------------------------------------------------------

def _rows(g, rows: int, cols: int, pad: int, dtype: str, scale=1.0, shift=0.0) -> torch.Tensor:
    """[rows, cols] inside rows of cols + pad values."""
    x = torch.randn(rows, cols + pad, device=DEV, generator=g) * scale + shift
    return x.to(TORCH[dtype])[:, :cols]


def _matrices(g, case: dict) -> torch.Tensor:
    """Gradients as a layer meets them: a few strong directions of falling
    size over a wide floor, and inputs that the batch never had."""
    b, r, c = case["batch"], case["rows"], case["cols"]
    rank = min(16, r, c)
    size = torch.arange(1, rank + 1, device=DEV, dtype=torch.float32) ** -0.7
    left = torch.randn(b, r, rank, device=DEV, generator=g) * size
    right = torch.randn(b, rank, c, device=DEV, generator=g)
    x = left @ right
    x += 0.5 * torch.randn(b, r, c, device=DEV, generator=g)
    x *= (torch.rand(b, r, 1, device=DEV, generator=g) < 0.93) * 1e-3
    return x


def _choice(logits: torch.Tensor, valid, top: int):
    """The positions that count, and the buckets of the `top` largest logits
    (ties to the lowest bucket; -1 where the rest is masked)."""
    value, bucket = torch.sort(logits, dim=1, descending=True, stable=True)
    counted = logits.amax(dim=1) > -math.inf
    if valid is not None:
        counted = counted & (valid != 0)
    taken = (value[:, :top] > -math.inf) & counted[:, None]
    return counted, torch.where(taken, bucket[:, :top], -1)


def prepare(case: dict, seed: int) -> dict:
    kind, dtype = case["kind"], case["dtype"]
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    s = dict(case=case)
    if kind in ("norm", "norm_grad"):
        r, c, pad = case["rows"], case["cols"], case["pad"]
        s["x"] = _rows(g, r, c, pad, dtype, 0.6, 0.4)
        s["weight"] = 1.0 + 0.2 * torch.randn(c, device=DEV, generator=g)
        s["bias"] = 0.1 * torch.randn(c, device=DEV, generator=g)
        if kind == "norm":
            s["out"] = dict(y=_empty(r, c, dtype), mean=_empty(r), rstd=_empty(r))
        else:
            x = s["x"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square().mean(1) + EPS)
            s["dy"] = _rows(g, r, c, pad, dtype, 1e-2)
            s["out"] = dict(dx=_empty(r, c, dtype), dweight=_empty(c), dbias=_empty(c))
    elif kind in ("gate", "gate_grad"):
        t, b, k = case["rows"], case["buckets"], case["top"]
        logits = torch.randn(t, b + case["pad"], device=DEV, generator=g) * 1.5
        logits += torch.randn(b + case["pad"], device=DEV, generator=g)
        s["valid"] = None
        if case["masked"]:
            logits[torch.rand(t, b + case["pad"], device=DEV, generator=g) < 0.05] = -math.inf
            logits[torch.rand(t, device=DEV, generator=g) < 0.01] = -math.inf
            s["valid"] = (torch.rand(t, device=DEV, generator=g) < 0.95).to(torch.uint8)
        s["logits"] = logits.to(TORCH[dtype])[:, :b]
        if kind == "gate":
            s["out"] = dict(bucket=_whole(t, k), gate=_empty(t, k), count=_whole(b), prob=_empty(b),
                            counted=_whole(1), loss=_empty(1))
        else:
            counted, bucket = _choice(s["logits"].float(), s["valid"], k)
            s["bucket"] = bucket.int()
            s["count"] = torch.bincount(bucket[bucket >= 0], minlength=b).int()
            s["counted"] = counted.sum(dtype=torch.int32).reshape(1)
            # 16-bit floats of 5 exponent bits take a scaled loss, as training in them does
            s["dloss"] = float(t) if dtype == "f16" else 1.0
            s["dgate"] = torch.randn(t, k, device=DEV, generator=g) * (s["dloss"] / t)
            s["out"] = dict(dlogits=_empty(t, b, dtype))
    else:
        s["grad"] = _matrices(g, case).to(TORCH[dtype])
        if kind == "ortho":
            s["out"] = torch.empty_like(s["grad"])
        else:
            s["weights"] = 0.04 * torch.randn(s["grad"].shape, device=DEV, generator=g)
            s["momentum"] = _matrices(g, case)
            s["lr"] = 0.02
            s["scale"] = math.sqrt(max(1.0, case["rows"] / case["cols"]))
    return s


def _empty(*shape) -> torch.Tensor:
    dtype = TORCH[shape[-1]] if isinstance(shape[-1], str) else torch.float32
    return torch.empty([n for n in shape if not isinstance(n, str)], dtype=dtype, device=DEV)


def _whole(*shape) -> torch.Tensor:
    return torch.empty(shape, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------
# the operators in their plain form
# ---------------------------------------------------------------------------

def _plain_norm(s: dict) -> dict:
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    y = d * rstd * s["weight"] + s["bias"]
    return dict(y=y.to(s["x"].dtype), mean=mean[:, 0], rstd=rstd[:, 0])


def _plain_norm_grad(s: dict) -> dict:
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    h = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["weight"]
    dx = (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)) * rstd
    return dict(dx=dx.to(s["x"].dtype), dweight=(dy * h).sum(0), dbias=dy.sum(0))


def _probabilities(logits: torch.Tensor, counted: torch.Tensor) -> torch.Tensor:
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - torch.where(top > -math.inf, top, 0.0))
    return torch.where(counted[:, None], e / e.sum(1, keepdim=True), 0.0)


def _plain_gate(s: dict) -> dict:
    c, logits = s["case"], s["logits"].float()
    counted, bucket = _choice(logits, s["valid"], c["top"])
    p = _probabilities(logits, counted)
    gate = torch.where(bucket >= 0, p.gather(1, bucket.clamp(min=0)), 0.0)
    if c["share"]:
        gate = gate / torch.where(counted, gate.sum(1), 1.0)[:, None]
    count = (bucket[:, :, None] == torch.arange(c["buckets"], device=DEV)).sum((0, 1))
    prob, n = p.sum(0), counted.sum()
    loss = BALANCE * c["buckets"] / c["top"] * (count.float() * prob).sum() / n.float().clamp(min=1).square()
    return dict(bucket=bucket.int(), gate=gate, count=count.int(), prob=prob, counted=n.int().reshape(1),
                loss=loss.reshape(1))


def _plain_gate_grad(s: dict) -> dict:
    c, logits = s["case"], s["logits"].float()
    counted = logits.amax(1) > -math.inf
    if s["valid"] is not None:
        counted = counted & (s["valid"] != 0)
    p = _probabilities(logits, counted)
    taken, at = s["bucket"] >= 0, s["bucket"].clamp(min=0).long()
    dgate = torch.where(taken, s["dgate"], 0.0)
    if c["share"]:
        chosen = torch.where(taken, p.gather(1, at), 0.0)
        total = torch.where(counted, chosen.sum(1), 1.0)[:, None]
        dgate = torch.where(taken, (dgate - (dgate * chosen / total).sum(1, keepdim=True)) / total, 0.0)
    n = s["counted"].float().clamp(min=1)
    h = s["dloss"] * BALANCE * c["buckets"] / c["top"] * s["count"].float() / n.square()
    h = h.expand_as(p).contiguous()
    h = h.scatter_add(1, at, dgate)
    d = p * (h - (p * h).sum(1, keepdim=True))
    return dict(dlogits=d.to(s["logits"].dtype))


def _plain_orthogonal(u: torch.Tensor) -> torch.Tensor:
    x = u.transpose(1, 2) if u.shape[1] > u.shape[2] else u
    x = (x / ((x * x).sum((1, 2), keepdim=True).sqrt() + NORM_EPS)).contiguous()
    for _ in range(STEPS):  # each step needs the one before
        gram = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = A * x + torch.matmul(B * gram + C * torch.matmul(gram, gram), x)
    return x.transpose(1, 2) if u.shape[1] > u.shape[2] else x


def _plain_muon(s: dict) -> dict:
    g, beta = s["grad"].float(), MUON["beta"]
    s["momentum"].mul_(beta).add_((1.0 - beta) * g)
    o = _plain_orthogonal((1.0 - beta) * g + beta * s["momentum"])
    w = s["weights"] * (1.0 - s["lr"] * MUON["weight_decay"]) - s["lr"] * s["scale"] * o
    s["weights"].copy_(w.clamp(-CLAMP, CLAMP))
    return dict(weights=s["weights"], momentum=s["momentum"])


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _operator(kind: str, dtype: str, *shape):
    """The operator's handle, one for a shape as a program keeps one a layer."""
    from tatara_amd import ops

    if kind == "norm":
        return ops.LayerNorm(cols=shape[0], dtype=dtype, eps=EPS)
    if kind == "gate":
        return ops.BucketGate(buckets=shape[0], top_k=shape[1], renormalise=shape[2], balance=BALANCE, dtype=dtype)
    if kind == "ortho":
        return ops.Orthogonaliser(batch=shape[0], rows=shape[1], cols=shape[2], dtype=dtype, steps=STEPS)
    return ops.Muon(batch=shape[0], rows=shape[1], cols=shape[2], grad_dtype=dtype, steps=STEPS, min_w=-CLAMP,
                    max_w=CLAMP, **MUON)


def _own(s: dict):
    c, o = s["case"], s.get("out")
    kind, dtype = c["kind"], c["dtype"]
    if kind == "norm":
        _operator("norm", dtype, c["cols"]).forward(s["x"], s["weight"], s["bias"], o["y"], o["mean"], o["rstd"])
    elif kind == "norm_grad":
        _operator("norm", dtype, c["cols"]).backward(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"], o["dx"],
                                                     o["dweight"], o["dbias"])
    elif kind == "gate":
        _operator("gate", dtype, c["buckets"], c["top"], c["share"]).forward(
            s["logits"], o["bucket"], o["gate"], o["count"], o["prob"], o["counted"], o["loss"], valid=s["valid"])
    elif kind == "gate_grad":
        _operator("gate", dtype, c["buckets"], c["top"], c["share"]).backward(
            s["logits"], s["bucket"], s["count"], s["counted"], o["dlogits"], dgate=s["dgate"], dloss=s["dloss"],
            valid=s["valid"])
    elif kind == "ortho":
        _operator("ortho", dtype, c["batch"], c["rows"], c["cols"])(s["grad"], o)
    else:
        _operator("muon", dtype, c["batch"], c["rows"], c["cols"]).step(s["weights"], s["momentum"], s["grad"],
                                                                        lr=s["lr"], scale=s["scale"])
        return dict(weights=s["weights"], momentum=s["momentum"])
    return o


def run(s: dict):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind == "norm":
        return _plain_norm(s)
    if kind == "norm_grad":
        return _plain_norm_grad(s)
    if kind == "gate":
        return _plain_gate(s)
    if kind == "gate_grad":
        return _plain_gate_grad(s)
    if kind == "ortho":
        return _plain_orthogonal(s["grad"].float()).to(s["grad"].dtype)
    return _plain_muon(s)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_orthogonal(u: torch.Tensor) -> torch.Tensor:
    """The same polynomial from the other side, X (a + b G + c G^2) with G the
    Gram matrix of the shorter dimension, so X stands with its longer one first."""
    tall = u if u.shape[1] >= u.shape[2] else u.transpose(1, 2)
    x = tall / (torch.linalg.vector_norm(tall, dim=(1, 2), keepdim=True) + NORM_EPS)
    eye = torch.eye(x.shape[2], dtype=torch.float64, device=DEV)
    for _ in range(STEPS):
        gram = x.transpose(1, 2) @ x
        x = x @ (A * eye + gram @ (B * eye + C * gram))
    return x if u.shape[1] >= u.shape[2] else x.transpose(1, 2)


def exact(case: dict, seed: int):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("norm", "norm_grad"):
        x, w = s["x"].double(), s["weight"].double()
        if kind == "norm":
            var, mean = torch.var_mean(x, dim=1, correction=0)
            rstd = (var + EPS) ** -0.5
            return dict(y=((x - mean[:, None]) * (rstd[:, None] * w)).add_(s["bias"].double()), mean=mean, rstd=rstd)
        dy, rstd = s["dy"].double(), s["rstd"].double()
        h = (x - s["mean"].double()[:, None]).mul_(rstd[:, None])
        del x
        dweight, dbias = (dy * h).sum(0), dy.sum(0)
        g = dy.mul_(w)
        along = (g * h).sum(1) / case["cols"]
        dx = (g - g.mean(1)[:, None]).sub_(h.mul_(along[:, None])).mul_(rstd[:, None])
        return dict(dx=dx, dweight=dweight, dbias=dbias)
    if kind in ("gate", "gate_grad"):
        l, b, k = s["logits"].double().cpu(), case["buckets"], case["top"]
        counted = (l != -math.inf).any(1)
        if s["valid"] is not None:
            counted &= s["valid"].cpu() != 0
        p = torch.zeros_like(l)
        p[counted] = torch.exp(l[counted] - torch.logsumexp(l[counted], 1, keepdim=True))
        if kind == "gate":
            _, bucket = _choice(s["logits"].float(), s["valid"], k)
            bucket = bucket.cpu()
            gate = torch.gather(torch.cat([p, torch.zeros(len(p), 1, dtype=p.dtype)], 1), 1, bucket % (b + 1))
            if case["share"]:
                gate[counted] /= gate[counted].sum(1, keepdim=True)
            count, n = torch.bincount(bucket[bucket >= 0], minlength=b), int(counted.sum())
            loss = BALANCE * b / k * float(count.double() @ p.sum(0)) / max(n, 1) ** 2
            return dict(bucket=None, gate=gate, count=None, prob=p.sum(0), counted=None,
                        loss=torch.tensor([loss], dtype=torch.float64))
        n, bucket = max(int(s["counted"]), 1), s["bucket"].cpu().long()
        dgate = torch.where(bucket >= 0, s["dgate"].double().cpu(), 0.0)
        wide = torch.cat([p, torch.zeros(len(p), 1, dtype=p.dtype)], 1)
        if case["share"]:  # gate = chosen / total
            chosen = torch.gather(wide, 1, bucket % (b + 1))
            total = torch.where(counted, chosen.sum(1), torch.ones(len(p), dtype=p.dtype))[:, None]
            dgate = dgate / total - (dgate * chosen).sum(1, keepdim=True) / total ** 2
        h = torch.zeros_like(wide).scatter_add_(1, bucket % (b + 1), dgate)[:, :b]
        h += s["dloss"] * BALANCE * b / k / n ** 2 * s["count"].cpu().double()
        return dict(dlogits=p * h - p * (p * h).sum(1, keepdim=True))
    g = s["grad"].double()
    if kind == "ortho":
        return _exact_orthogonal(g)
    beta, lr = MUON["beta"], s["lr"]
    momentum = beta * s["momentum"].double() + (1.0 - beta) * g
    o = _exact_orthogonal(beta * momentum + (1.0 - beta) * g)
    weights = s["weights"].double() * (1.0 - lr * MUON["weight_decay"]) - lr * s["scale"] * o
    return dict(weights=weights.clamp(-CLAMP, CLAMP), momentum=momentum)
