"""Caches, rows and the cache-attention operators' formulas in 64 bits (numpy)."""
import numpy as np

import lfm_hip

HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative
# what the weights lose where they meet V: two binary16 numbers hold 22 bits
WEIGHT = {"f32": 2.0 ** -21, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def to_bf16(x):
    """float32 -> bfloat16 bit patterns, to nearest even (finite values, infinities, NaN)."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(b):
    return (np.ascontiguousarray(b, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32)


def encode(x, kind):
    return to_bf16(x) if kind == "bf16" else np.asarray(x).astype(np.float16 if kind == "f16" else np.float32)


def decode(a, kind):
    return from_bf16(a) if kind == "bf16" else np.asarray(a, dtype=np.float32)


NP = {"f32": np.float32, "f16": np.float16, "bf16": "bf16"}


def tensor(x, kind):
    """A row-major device tensor of x's values in this type, and the values it holds."""
    e = encode(x, kind)
    return lfm_hip.DeviceTensor.from_array(e, NP[kind]), decode(e, kind).astype(np.float64)


def i32(x):
    return lfm_hip.DeviceTensor.from_array(np.asarray(x, dtype=np.int32))


def f32(x):
    return lfm_hip.DeviceTensor.from_array(np.asarray(x, dtype=np.float32))


class Cache:
    """A seeded cache: .view for the operators, .k and .v [n][kv][slots][d] in 64 bits.
    order "head": the engine's [kv][slots][d]; "slot": [slots][kv][d]; "mixed": K and V of a
    slot side by side, with unused elements between the slots."""

    def __init__(self, rng, length, kv, slots, dim, kind, order="head", edit=None):
        n = len(length)
        self.k, self.v = (rng.standard_normal((n, kv, slots, dim)).astype(np.float32) for _ in range(2))
        if edit:
            edit(self.k, self.v)
        self.kind, self.length = kind, np.asarray(length)
        e = [encode(x, kind) for x in (self.k, self.v)]
        self.k, self.v = (decode(x, kind).astype(np.float64) for x in e)
        if order == "head":
            t = [lfm_hip.DeviceTensor.from_array(x, NP[kind]) for x in e]
        elif order == "slot":
            bufs = [lfm_hip.DeviceBuffer.from_array(x.transpose(0, 2, 1, 3)) for x in e]
            st = (slots * kv * dim, dim, kv * dim, 1)
            t = [lfm_hip.DeviceTensor(b, (n, kv, slots, dim), NP[kind], 0, st) for b in bufs]
        else:
            row = 2 * kv * dim + 8
            host = np.full((n, slots, row), 0x7FFF, dtype=np.uint16)  # NaN between the slots
            for i, x in enumerate(e):
                host[:, :, i * kv * dim:(i + 1) * kv * dim] = \
                    x.view(np.uint16).transpose(0, 2, 1, 3).reshape(n, slots, kv * dim)
            buf = lfm_hip.DeviceBuffer.from_array(host)
            st = (slots * row, dim, row, 1)
            t = [lfm_hip.DeviceTensor(buf, (n, kv, slots, dim), NP[kind], i * kv * dim, st) for i in range(2)]
        self.tk, self.tv, self.tl = t[0], t[1], i32(self.length)
        self.view = lfm_hip.KvCache(self.tk, self.tv, self.tl)


def reference(q, cache, start=None, window=0, sinks=0, scale=None, prefix=None, dim=None):
    """Formulas in 64 bits.  Returns out, lse, acc [n][kv][slots] and, for the tolerances,
    the sums of w |v|, the largest sum of |q k| * scale and the slots seen, per row and head."""
    rows, heads, dim = q.shape
    n, kv, slots, _ = cache.k.shape
    scale = dim ** -0.5 if scale is None else float(np.float32(scale))
    g = heads // kv
    start = np.arange(n + 1) if start is None else np.asarray(start)
    out, size = np.zeros_like(q), np.zeros_like(q)
    lse = np.full((rows, heads), -np.inf)
    reach, seen = np.zeros((rows, heads)), np.zeros((rows, heads))
    acc = np.zeros((n, kv, slots))
    for b in range(n):
        length = min(max(int(cache.length[b]), 0), slots)
        lo, hi = max(0, min(int(start[b]), rows)), max(0, min(int(start[b + 1]), rows))
        for row in range(lo, hi):
            p = length - hi + row
            j = np.arange(max(p + 1, 0))
            if window:
                j = j[(j < sinks) | (j > p - window)]
            for h in range(heads):
                k, v = cache.k[b, h // g][j], cache.v[b, h // g][j]
                if prefix is not None:
                    m = min(max(int(prefix.length[0]), 0), prefix.k.shape[2])
                    k = np.concatenate([prefix.k[0, h // g][:m], k])
                    v = np.concatenate([prefix.v[0, h // g][:m], v])
                if not len(k):
                    continue
                with np.errstate(invalid="ignore", over="ignore"):
                    s = k @ q[row, h] * scale
                    top = s.max()
                    w = np.exp(s - top)
                    lse[row, h] = top + np.log(w.sum())
                    w = w / w.sum()
                    out[row, h] = w @ v
                    size[row, h] = w @ np.abs(v)
                    reach[row, h] = (np.abs(k) @ np.abs(q[row, h])).max() * scale
                seen[row, h] = len(k)
                if prefix is None:
                    acc[b, h // g, j] += w
    return out, lse, acc, (size, reach, seen)


def score_error(reach, dim):
    """Of a score: rows as 22 bits or exact, sums of dim products in 32 bits, three more
    roundings of a number no larger than reach (scaling, the distance from the maximum)."""
    return ((dim + 4) * 2.0 ** -24 + 2.0 ** -21) * reach


def out_tolerance(out, extra, kind, dim):
    """Per element.  Weights: relative exp(2 score_error) - 1 each, their 16-bit form, one
    step of the hardware's 2^x each for weight and rescaling; sums over the slots seen in 32
    bits in any order; the division; the output's own rounding.  Weights under 2^-24 of the
    largest may vanish in 16 bits."""
    size, reach, seen = extra
    rel = 2.1 * score_error(reach, dim) + WEIGHT[kind] + 2.0 ** -20 + 2 * (seen + 16) * 2.0 ** -24
    biggest = size.max(axis=-1, keepdims=True) + 6.0
    return rel[..., None] * size + HALF[kind] * 1.01 * np.abs(out) + (seen * 2.0 ** -24)[..., None] * \
        (0 if kind == "bf16" else 1) * biggest * 2.0 ** -8 + 1e-7


def lse_tolerance(lse, extra, dim):
    _, reach, seen = extra
    return score_error(reach, dim) + (seen + 16) * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * np.abs(
        np.where(np.isfinite(lse), lse, 0))


def check_out(got, want, extra, kind, dim):
    tol = out_tolerance(want, extra, kind, dim)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5], tol[bad][:5])


def keep_slots(acc, pos, length, keep, sinks, recent):
    """The eviction's rule for one (sequence, kv head): the source slot of each slot that
    stays, or None for a sequence that is short enough."""
    n = max(0, int(length))
    if n <= keep:
        return None
    newest = max(int(p) for p in pos[:n])

    def rank(j):
        protected = pos[j] < sinks or int(pos[j]) > newest - recent
        nan = np.isnan(acc[j])
        return (0 if protected else 2 if nan else 1, 0.0 if protected or nan else -float(acc[j]), j)

    kept = set(sorted(range(n), key=rank)[:keep])
    late = iter(sorted(j for j in kept if j >= keep))
    return np.array([j if j in kept else next(late) for j in range(keep)])
