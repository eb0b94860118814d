"""The operators around a learned choice's bucket layers, as cases that can be timed and compared.

Beside the bucket gate, a network whose positions choose their dense layers needs
the rows of each bucket side by side and back in their positions' order with the
gate's shares (bucket rows), a norm with the residual's addition in front of it
(RMS norm, in 8 bits for layers that take them), dropout on the branch, and rows
of a table for a position's discrete values, such as a king's square (embedding).
The cases take these calls over the sizes of this repository's networks and over
generic ones.

With `own` false the operators are computed from elementary torch operations in
32 bits; with `own` true by tatara_amd.ops.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
E4M3_MAX = 448.0
SCALE_FLOOR = 2.0 ** -100  # the largest value that a group's scale stands for is at least this
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
VALUES = 65536 * 1536  # of a case's rows at most: the headline batch at the headline width


def listed() -> list[dict]:
    return [
        # A training batch at the headline width: the branch is added to the
        # residual and the sum normalised for the next layer.
        dict(name="rms_add_bf16_65536x1536", kind="rms", rows=65536, cols=1536, pad=0, dtype="bf16", residual=True),
        # One position that is scored on its own, for layers that take 8 bits.
        dict(name="rms8_bf16_1x1536", kind="rms8", rows=1, cols=1536, pad=0, dtype="bf16", residual=True, group=0),
        # A batch that is scored by layers with a scale for every 128 columns.
        dict(name="rms8_f16_16381x2048_g128", kind="rms8", rows=16381, cols=2048, pad=0, dtype="f16", residual=False,
             group=128),
        # A small odd batch of rows that lie inside wider ones, on its way back,
        # where the residual's own gradient joins.
        dict(name="rms_grad_f32_1009x769", kind="rms_grad", rows=1009, cols=769, pad=10, dtype="f32", residual=True),
        # The branch of a training batch, dropped out and added to the residual.
        dict(name="dropout_add_bf16_65536x1536", kind="dropout", rows=65536, cols=1536, pad=0, dtype="bf16", p=0.1,
             residual=True),
        # The gradient of a small odd batch through the same mask.
        dict(name="dropout_grad_f32_1021x130", kind="dropout_grad", rows=1021, cols=130, pad=3, dtype="f32", p=0.25,
             residual=False),
        # The headline batch, sorted by its nine buckets.
        dict(name="gather_f32_65536x1536_9", kind="gather", rows=65536, cols=1536, pad=0, dtype="f32", buckets=9, top=1,
             room=0.0, masked=False),
        # One position for its two best buckets.
        dict(name="gather_bf16_1x1536_8_top2", kind="gather", rows=1, cols=1536, pad=0, dtype="bf16", buckets=8, top=2,
             room=0.0, masked=False),
        # Many buckets with room for a fixed number of rows each, four of them a
        # position, blended back; some positions do not count.
        dict(name="combine_bf16_16381x512_64_top4", kind="combine", rows=16381, cols=512, pad=0, dtype="bf16",
             buckets=64, top=4, room=1.25, masked=True),
        # The gradient of blending two buckets a position: of the rows and of the shares.
        dict(name="combine_grad_f16_32768x768_9_top2", kind="combine_grad", rows=32768, cols=768, pad=0, dtype="f16",
             buckets=9, top=2, room=0.0, masked=False),
        # A batch's positions look up a row for one discrete value of theirs each.
        dict(name="embed_bf16_65536x768_1629", kind="embed", rows=65536, cols=768, pad=0, dtype="bf16", vocab=1629,
             hot=False),
        # The gradient of a table as large as the feature transformer's.
        dict(name="embed_grad_f32_65536x1536_73305", kind="embed_grad", rows=65536, cols=1536, pad=0, dtype="f32",
             vocab=73305, hot=True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["rms", "rms8", "rms_grad", "dropout", "dropout_grad", "gather", "gather_grad", "combine",
                       "combine_grad", "embed", "embed_grad"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    cols = rng.choice([256, 512, 768, 1024, 1536, 2048, _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)])
    pad = rng.choice([0, 0, 8, rng.randint(1, 40)])
    c = dict(kind=kind, rows=0, cols=cols, pad=pad, dtype=dtype)
    if kind in ("gather", "gather_grad", "combine", "combine_grad"):
        buckets = rng.choice([8, 9, _log_int(rng, 2, 256), _log_int(rng, 2, 256)])
        top = rng.randint(1, min(4, buckets))
        c.update(buckets=buckets, top=top, room=rng.choice([0.0, 0.0, 1.0, 1.25]), masked=rng.random() < 0.4)
        c["rows"] = _log_int(rng, 1, min(65536, VALUES // (2 * cols * top)))
        return c
    c["rows"] = _log_int(rng, 1, min(65536, VALUES // cols))
    if kind == "rms8":
        c["group"] = rng.choice([0, 32, 64, 128])
    if kind in ("rms", "rms8", "rms_grad"):
        c["residual"] = rng.random() < 0.5
    elif kind in ("dropout", "dropout_grad"):
        c["p"] = rng.choice([0.0625, 0.1, 0.25, 0.5])
        c["residual"] = kind == "dropout" and rng.random() < 0.5
    else:
        c["vocab"] = _log_int(rng, 2, min(73305, VALUES // cols))
        c["hot"] = rng.random() < 0.5
    return c


def _room(case: dict):
    """Rows that each bucket has room for, or None: as many as it has."""
    if not case["room"]:
        return None
    return max(1, math.ceil(case["room"] * case["rows"] * case["top"] / case["buckets"]))


def _sorted_rows(case: dict) -> int:
    room = _room(case)
    return case["rows"] * case["top"] if room is None else case["buckets"] * room


def work(case: dict) -> dict:
    kind, r, c, e = case["kind"], case["rows"], case["cols"], SIZE[case["dtype"]]
    n = r * c
    if kind == "rms":  # x and the residual in, their sum and y out
        return dict(bytes=n * e * (4 if case["residual"] else 2) + 4 * r + 4 * c, flops=5 * n)
    if kind == "rms8":
        groups = -(-c // case["group"]) if case["group"] else 1
        return dict(bytes=n * (e * (3 if case["residual"] else 1) + 1) + 4 * r * groups + 4 * c, flops=8 * n)
    if kind == "rms_grad":  # dy, the sum and its own gradient in, dx out
        return dict(bytes=n * e * (4 if case["residual"] else 3) + 4 * r + 8 * c, flops=10 * n)
    if kind in ("dropout", "dropout_grad"):  # ten rounds of two products and four exclusive ors for four values
        return dict(bytes=n * e * (3 if case["residual"] else 2), flops=17 * n)
    if kind in ("embed", "embed_grad"):
        v = case["vocab"]
        if kind == "embed":
            return dict(bytes=4 * r + min(r, v) * c * e + n * e, flops=n)
        return dict(bytes=4 * r + n * e + 4 * v * c, flops=2 * n)
    k, s = case["top"], _sorted_rows(case)
    taken = min(s, r * k) * c * e  # rows that a bucket has
    if kind == "gather":  # buckets and x in; slot, source, offset and rows out
        return dict(bytes=8 * r * k + 4 * s + 4 * case["buckets"] + n * e + s * c * e, flops=r * k)
    if kind == "gather_grad":
        return dict(bytes=4 * r * k + taken + n * e, flops=n * k)
    if kind == "combine":
        return dict(bytes=8 * r * k + taken + n * e, flops=2 * n * k)
    return dict(bytes=12 * r * k + 4 * s + n * e + taken + s * c * e, flops=3 * n * k)


# ---------------------------------------------------------------------------
# what a program holds before the call
# ---------------------------------------------------------------------------

def _rows(g, rows: int, cols: int, pad: int, dtype: str, scale=1.0) -> torch.Tensor:
    """[rows, cols] inside rows of cols + pad values."""
    x = torch.randn(rows, cols + pad, device=DEV, generator=g) * scale
    return x.to(TORCH[dtype])[:, :cols]


def _empty(*shape) -> torch.Tensor:
    dtype = TORCH[shape[-1]] if isinstance(shape[-1], str) else torch.float32
    return torch.empty([n for n in shape if not isinstance(n, str)], dtype=dtype, device=DEV)


def _whole(*shape) -> torch.Tensor:
    return torch.empty(shape, dtype=torch.int32, device=DEV)


def _chosen(g, case: dict) -> torch.Tensor:
    """Each position's buckets as a gate leaves them: distinct, some buckets
    liked better than others, -1 where a position has none."""
    t, b, k = case["rows"], case["buckets"], case["top"]
    liking = torch.randn(t, b, device=DEV, generator=g) + torch.randn(b, device=DEV, generator=g)
    bucket = liking.topk(k, dim=1).indices.int()
    if case["masked"]:
        bucket[torch.rand(t, device=DEV, generator=g) < 0.05] = -1
        bucket[:, k - 1][torch.rand(t, device=DEV, generator=g) < 0.05] = -1
    return bucket.contiguous()


def _tokens(g, case: dict) -> torch.Tensor:
    """Values that all come alike, or a few of them far more often; some rows have none (-1)."""
    u = torch.rand(case["rows"], device=DEV, generator=g, dtype=torch.float64)
    v = case["vocab"]
    token = ((v + 1.0) ** u - 1.0 if case["hot"] else u * v).long().clamp(max=v - 1)
    token = (token * 7919) % v if math.gcd(7919, v) == 1 else token  # the frequent ones lie anywhere in the table
    token[torch.rand(case["rows"], device=DEV, generator=g) < 0.01] = -1
    return token.int()


def prepare(case: dict, seed: int) -> dict:
    kind, r, c, pad, dtype = case["kind"], case["rows"], case["cols"], case["pad"], case["dtype"]
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    s = dict(case=case, residual=None)
    if kind in ("rms", "rms8", "rms_grad"):
        s["x"] = _rows(g, r, c, pad, dtype, 0.8)
        s["weight"] = 1.0 + 0.2 * torch.randn(c, device=DEV, generator=g)
        if case["residual"]:
            s["residual"] = _rows(g, r, c, pad, dtype, 0.01 if kind == "rms_grad" else 1.5)
        if kind == "rms_grad":
            s["rstd"] = torch.rsqrt(s["x"].float().square().mean(1) + EPS)
            s["dy"] = _rows(g, r, c, pad, dtype, 1e-2)
            s["out"] = dict(dx=_empty(r, c, dtype), dweight=_empty(c))
        else:
            s["out"] = dict(rstd=_empty(r))
            if case["residual"]:
                s["out"]["total"] = _empty(r, c, dtype)
            if kind == "rms":
                s["out"]["y"] = _empty(r, c, dtype)
            else:
                groups = -(-c // case["group"]) if case["group"] else 1
                s["out"]["q"] = torch.empty(r, c, dtype=torch.float8_e4m3fn, device=DEV)
                s["out"]["scale"] = _empty(r, groups)
    elif kind in ("dropout", "dropout_grad"):
        s["x"] = _rows(g, r, c, pad, dtype, 1e-2 if kind == "dropout_grad" else 0.8)
        if case["residual"]:
            s["residual"] = _rows(g, r, c, pad, dtype, 1.5)
        s["seed"], s["step"] = 0x9E3779B97F4A7C15 + 2 * seed & (1 << 63) - 1, 1000 + 3 * seed
        s["out"] = dict(y=_empty(r, c, dtype))
    elif kind in ("embed", "embed_grad"):
        s["token"] = _tokens(g, case)
        s["scale"] = math.sqrt(c)
        if kind == "embed":
            s["table"] = _rows(g, case["vocab"], c, pad, dtype, c ** -0.5)
            s["out"] = dict(y=_empty(r, c, dtype))
        else:
            s["dy"] = _rows(g, r, c, pad, dtype, 1e-2)
            s["out"] = dict(dtable=_empty(case["vocab"], c))
    else:
        t, k, n = r, case["top"], _sorted_rows(case)
        s["bucket"] = _chosen(g, case)
        if kind == "gather":
            s["x"] = _rows(g, r, c, pad, dtype, 0.8)
            s["out"] = dict(slot=_whole(t, k), source=_whole(n), offset=_whole(case["buckets"] + 1),
                            rows=_empty(n, c, dtype))
            return s
        s["slot"], s["source"], _ = _sorted(s["bucket"], case["buckets"], _room(case))
        s["rows"] = _rows(g, n, c, pad, dtype, 1e-2 if kind == "gather_grad" else 0.8)
        s["rows"][s["source"] < 0] = 0.0
        if kind != "gather_grad":
            share = torch.rand(t, k, device=DEV, generator=g) + 0.1
            s["gate"] = torch.where(s["bucket"] >= 0, share / share.sum(1, keepdim=True), 0.0)
        if kind == "combine_grad":
            s["dy"] = _rows(g, r, c, pad, dtype, 1e-2)
            s["out"] = dict(drows=_empty(n, c, dtype), dgate=_empty(t, k))
        else:
            s["out"] = dict(y=_empty(r, c, dtype))
    return s


# ---------------------------------------------------------------------------
# the operators in their plain form
# ---------------------------------------------------------------------------

def _sorted(bucket: torch.Tensor, buckets: int, room):
    """slot [positions, top], source [rows] and offset [buckets + 1]: the choices
    by bucket, and in a bucket by position and choice."""
    key = bucket.reshape(-1).long()
    taken = (key >= 0) & (key < buckets)
    key = torch.where(taken, key, buckets)
    count = (key[:, None] == torch.arange(buckets, device=DEV)).sum(0)
    offset = torch.cat([count.new_zeros(1), count.cumsum(0)])
    by, order = torch.sort(key, stable=True)
    rank = torch.arange(len(key), device=DEV) - offset[by]
    if room is None:
        row, rows = torch.where(by < buckets, offset[by] + rank, -1), len(key)
    else:
        row, rows = torch.where((by < buckets) & (rank < room), by * room + rank, -1), buckets * room
    slot = torch.empty_like(key)
    slot[order] = row
    source = torch.full((rows + 1,), -1, dtype=torch.int64, device=DEV)
    source[torch.where(row >= 0, row, rows)] = order
    return slot.int().view(bucket.shape), source[:rows].int(), offset.int()


def _plain_gather(s: dict) -> dict:
    c = s["case"]
    slot, source, offset = _sorted(s["bucket"], c["buckets"], _room(c))
    rows = s["x"][source.clamp(min=0).long() // c["top"]]
    return dict(slot=slot, source=source, offset=offset, rows=torch.where(source[:, None] >= 0, rows, 0.0).to(rows.dtype))


def _at_slots(rows: torch.Tensor, slot: torch.Tensor) -> torch.Tensor:
    """[positions, top, cols] in f32, zeros where a choice has no row."""
    at = rows[slot.clamp(min=0).long()].float()
    return torch.where(slot[:, :, None] >= 0, at, 0.0)


def _plain_combine(s: dict) -> dict:
    at = _at_slots(s["rows"], s["slot"])
    if "gate" in s:
        at = at * s["gate"][:, :, None]
    return dict(y=at.sum(1).to(s["rows"].dtype))


def _plain_combine_grad(s: dict) -> dict:
    dy, top, source = s["dy"].float(), s["case"]["top"], s["source"].clamp(min=0).long()
    dgate = (_at_slots(s["rows"], s["slot"]) * dy[:, None, :]).sum(2)
    drows = s["gate"].reshape(-1)[source][:, None] * dy[source // top]
    drows = torch.where(s["source"][:, None] >= 0, drows, 0.0)
    return dict(drows=drows.to(s["rows"].dtype), dgate=dgate)


def _plain_rms(s: dict) -> dict:
    c, x = s["case"], s["x"]
    out = {}
    if s["residual"] is not None:
        out["total"] = x = (x.float() + s["residual"].float()).to(x.dtype)
    x = x.float()
    out["rstd"] = torch.rsqrt((x * x).mean(1) + EPS)
    y = x * out["rstd"][:, None] * s["weight"]
    if c["kind"] == "rms":
        out["y"] = y.to(s["x"].dtype)
        return out
    rows, cols, group = c["rows"], c["cols"], c["group"] or c["cols"]
    groups = -(-cols // group)
    wide = torch.zeros(rows, groups * group, device=DEV)
    wide[:, :cols] = y
    wide = wide.view(rows, groups, group)
    out["scale"] = wide.abs().amax(2).clamp(min=SCALE_FLOOR) / E4M3_MAX
    q = (wide / out["scale"][:, :, None]).view(rows, -1)[:, :cols].clamp(-E4M3_MAX, E4M3_MAX)
    out["q"] = q.contiguous().to(torch.float8_e4m3fn)
    return out


def _plain_rms_grad(s: dict) -> dict:
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    h = s["x"].float() * rstd
    g = dy * s["weight"]
    dx = (g - h * (g * h).mean(1, keepdim=True)) * rstd
    if s["residual"] is not None:
        dx = dx + s["residual"].float()
    return dict(dx=dx.to(s["x"].dtype), dweight=(dy * h).sum(0))


def _philox(rows: int, blocks: int, seed: int, step: int) -> torch.Tensor:
    """[rows, 4 * blocks] 32-bit numbers of Philox4x32 with ten rounds: counter
    (column / 4, row, step's low and high half), key the seed's halves."""
    low = 0xFFFFFFFF
    a = torch.arange(blocks, device=DEV).expand(rows, blocks)
    b = torch.arange(rows, device=DEV)[:, None].expand(rows, blocks)
    c, d = torch.full_like(a, step & low), torch.full_like(a, step >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):  # each round needs the one before
        p, q = a * 0xD2511F53, c * 0xCD9E8D57  # of 64 bits, which wrap as they should
        a, b, c, d = (q >> 32 & low) ^ b ^ k0, q & low, (p >> 32 & low) ^ d ^ k1, p & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    return torch.stack([a, b, c, d], 2).view(rows, -1)


def _plain_dropout(s: dict) -> dict:
    c, x = s["case"], s["x"]
    u = _philox(c["rows"], -(-c["cols"] // 4), s["seed"], s["step"])[:, :c["cols"]]
    y = torch.where(u >= round(c["p"] * 2.0 ** 32), x.float() * (1.0 / (1.0 - c["p"])), 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return dict(y=y.to(x.dtype))


def _plain_embed(s: dict) -> dict:
    y = s["table"][s["token"].clamp(min=0).long()].float() * s["scale"]
    return dict(y=torch.where(s["token"][:, None] >= 0, y, 0.0).to(s["table"].dtype))


def _plain_embed_grad(s: dict) -> dict:
    v = s["case"]["vocab"]
    d = torch.zeros(v + 1, s["case"]["cols"], device=DEV)
    d.index_add_(0, torch.where(s["token"] >= 0, s["token"], v).long(), s["dy"].float())
    return dict(dtable=d[:v] * s["scale"])


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _operator(kind: str, dtype: str, *shape):
    """The operator's handle, one for a shape as a program keeps one a layer."""
    from tatara_amd import ops

    if kind == "rms":
        return ops.RMSNorm(cols=shape[0], dtype=dtype, eps=EPS)
    if kind == "rms8":
        return ops.RMSNorm(cols=shape[0], dtype=dtype, eps=EPS, out8="e4m3", group=shape[1])
    if kind == "dropout":
        return ops.Dropout(cols=shape[0], p=shape[1], dtype=dtype, seed=shape[2])
    if kind == "embed":
        return ops.Embedding(vocab=shape[0], cols=shape[1], positions=shape[2], dtype=dtype, scale=shape[3])
    return ops.BucketRows(buckets=shape[0], cols=shape[1], top_k=shape[2], dtype=dtype, capacity=shape[3])


def _own(s: dict) -> dict:
    c, o = s["case"], s["out"]
    kind, dtype, cols = c["kind"], c["dtype"], c["cols"]
    if kind == "rms":
        _operator("rms", dtype, cols).forward(s["x"], s["weight"], o["y"], rstd=o["rstd"], residual=s["residual"],
                                              total=o.get("total"))
    elif kind == "rms8":
        _operator("rms8", dtype, cols, c["group"]).forward_8bit(
            s["x"], s["weight"], o["q"], o["scale"], rstd=o["rstd"], residual=s["residual"], total=o.get("total"))
    elif kind == "rms_grad":
        _operator("rms", dtype, cols).backward(s["dy"], s["x"], s["weight"], s["rstd"], o["dx"], dweight=o["dweight"],
                                               dtotal=s["residual"])
    elif kind == "dropout":
        _operator("dropout", dtype, cols, c["p"], s["seed"]).forward(s["x"], o["y"], step=s["step"],
                                                                     residual=s["residual"])
    elif kind == "dropout_grad":
        _operator("dropout", dtype, cols, c["p"], s["seed"]).backward(s["x"], o["y"], step=s["step"])
    elif kind == "embed":
        op = _operator("embed", dtype, c["vocab"], cols, c["rows"], s["scale"])
        op.forward(s["token"], s["table"], o["y"])
    elif kind == "embed_grad":
        op = _operator("embed", dtype, c["vocab"], cols, c["rows"], s["scale"])
        op.backward(s["dy"], s["token"], o["dtable"])
    else:
        op = _operator("rows", dtype, c["buckets"], cols, c["top"], _room(c))
        if kind == "gather":
            op.sort(s["bucket"], o["slot"], o["source"], o["offset"])
            op.gather(s["x"], o["slot"], o["source"], o["rows"])
        elif kind == "gather_grad":
            op.gather_backward(s["rows"], s["slot"], o["y"])
        elif kind == "combine":
            op.combine(s["rows"], s["slot"], s["gate"], o["y"])
        else:
            op.combine_backward(s["dy"], s["rows"], s["slot"], s["source"], s["gate"], o["drows"], dgate=o["dgate"])
    return o


def run(s: dict):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind in ("rms", "rms8"):
        return _plain_rms(s)
    if kind == "rms_grad":
        return _plain_rms_grad(s)
    if kind in ("dropout", "dropout_grad"):
        return _plain_dropout(s)
    if kind == "gather":
        return _plain_gather(s)
    if kind in ("gather_grad", "combine"):
        return _plain_combine(s)
    if kind == "combine_grad":
        return _plain_combine_grad(s)
    return _plain_embed(s) if kind == "embed" else _plain_embed_grad(s)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_kept(case: dict, seed: int, step: int) -> torch.Tensor:
    """The same mask with the products' halves from limbs of 16 bits, a value at a time."""
    def product(x, m):
        lo, hi = x * (m & 0xFFFF), x * (m >> 16)  # below 2^48
        full = (lo >> 16) + hi
        return full >> 16, (full << 16 | lo & 0xFFFF) & 0xFFFFFFFF

    rows, cols = case["rows"], case["cols"]
    word = torch.zeros(4, rows, -(-cols // 4), dtype=torch.int64, device=DEV)
    word[0] = torch.arange(word.shape[2], device=DEV)
    word[1] = torch.arange(rows, device=DEV)[:, None]
    word[2], word[3] = step % 2 ** 32, step // 2 ** 32
    for r in range(10):
        hi0, lo0 = product(word[0], 0xD2511F53)
        hi1, lo1 = product(word[2], 0xCD9E8D57)
        key = ((seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32)
        word[0] = hi1.bitwise_xor_(word[1]).bitwise_xor_(key[0])
        word[2] = hi0.bitwise_xor_(word[3]).bitwise_xor_(key[1])
        word[1], word[3] = lo1, lo0
    return (word.permute(1, 2, 0).reshape(rows, -1)[:, :cols].double() / 2.0 ** 32) >= round(case["p"] * 2.0 ** 32) / 2.0 ** 32


def exact(case: dict, seed: int):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("rms", "rms8"):
        out, x = {}, s["x"]
        if case["residual"]:
            out["total"] = x.double() + s["residual"].double()
            x = out["total"].to(x.dtype)  # the norm is that of the sum as it is stored
        x = x.double()
        out["rstd"] = (torch.linalg.vector_norm(x, dim=1).square() / case["cols"] + EPS) ** -0.5
        y = x.mul_(out["rstd"][:, None]).mul_(s["weight"].double())
        if kind == "rms":
            out["y"] = y
            return out
        group = case["group"] or case["cols"]
        parts = y.split(group, dim=1)
        out["scale"] = torch.stack([p.abs().amax(1) for p in parts], 1).clamp(min=SCALE_FLOOR) / E4M3_MAX
        out["q"] = y / out["scale"].repeat_interleave(group, 1)[:, :case["cols"]]
        return out
    if kind == "rms_grad":
        dy, w, rstd = s["dy"].double(), s["weight"].double(), s["rstd"].double()[:, None]
        h = s["x"].double().mul_(rstd)
        dweight = torch.linalg.vecdot(dy, h, dim=0)
        along = torch.linalg.vecdot(dy * w, h, dim=1)[:, None] / case["cols"]
        dx = dy.mul_(w).sub_(h.mul_(along)).mul_(rstd)
        if case["residual"]:
            dx += s["residual"].double()
        return dict(dx=dx, dweight=dweight)
    if kind in ("dropout", "dropout_grad"):
        y = s["x"].double() / (1.0 - case["p"])
        y[~_exact_kept(case, s["seed"], s["step"])] = 0.0
        if case["residual"]:
            y += s["residual"].double()
        return dict(y=y)
    if kind in ("embed", "embed_grad"):
        known = s["token"] >= 0
        at = s["token"][known].long()
        if kind == "embed":
            y = torch.zeros(case["rows"], case["cols"], dtype=torch.float64, device=DEV)
            y[known] = s["table"].double()[at] * s["scale"]
            return dict(y=y)
        order = torch.argsort(at)
        dy = s["dy"].double()[known][order].mul_(s["scale"])
        lengths = torch.bincount(at, minlength=case["vocab"])
        return dict(dtable=torch.segment_reduce(dy, "sum", lengths=lengths, axis=0, unsafe=True))
    if kind == "gather":
        key, room = s["bucket"].flatten(), _room(case)
        rows = torch.zeros(_sorted_rows(case), case["cols"], dtype=torch.float64, device=DEV)
        first = 0
        for e in range(case["buckets"]):
            at = torch.nonzero(key == e)[:room, 0]  # in the positions' order
            rows[first:first + len(at)] = s["x"][torch.div(at, case["top"], rounding_mode="floor")].double()
            first += len(at) if room is None else room
        return dict(slot=None, source=None, offset=None, rows=rows)
    t, k = s["slot"].shape
    none = len(s["rows"])  # a row of zeros behind the others
    at = torch.where(s["slot"] < 0, none, s["slot"]).long()
    rows = torch.cat([s["rows"].double(), s["rows"].new_zeros(1, case["cols"]).double()])
    if kind in ("gather_grad", "combine"):
        y = torch.zeros(t, case["cols"], dtype=torch.float64, device=DEV)
        for j in range(k):
            y += rows[at[:, j]] * (s["gate"][:, j:j + 1].double() if kind == "combine" else 1.0)
        return dict(y=y)
    dy = s["dy"].double()
    dgate = torch.stack([torch.linalg.vecdot(rows[at[:, j]], dy) for j in range(k)], 1)
    drows = torch.zeros_like(rows)
    for j in range(k):  # the row of zeros takes what has none, and is left out
        drows[at[:, j]] = dy * s["gate"][:, j:j + 1].double()
    return dict(drows=drows[:none], dgate=dgate)
