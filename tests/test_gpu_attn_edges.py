"""Cache-attention operators at the edges of what their calls allow, against the formulas in
64 bits with attn_util's tolerances."""
import numpy as np
import pytest

import attn_util as U
from attn_util import Cache, check_out, decode, encode, f32, i32
from test_gpu_attn import Rows, check_prefix, check_scored, check_window, workspace

pytestmark = pytest.mark.gpu


class NarrowRows(Rows):
    """Rows with no more than the 16-byte alignment that calls promise: base, head and row
    strides are odd multiples of 16 bytes."""

    def __init__(self, gpu, rng, n, heads, dim, kind):
        super().__init__(gpu, rng, n, heads, dim, kind)
        e = 4 if kind == "f32" else 8
        st = (heads * (dim + e) + (heads + 1) % 2 * e, dim + e, 1)
        self.at = e + np.arange(n)[:, None, None] * st[0] + np.arange(heads)[:, None] * st[1] + np.arange(dim)
        host = np.full(e + n * st[0], 7, dtype=np.uint16 if kind == "bf16" else U.NP[kind])
        host[self.at] = encode(self.values, kind)
        self.q = gpu.DeviceTensor(gpu.DeviceBuffer.from_array(host), self.shape, U.NP[kind], e, st)
        host[:] = 77
        self.out = gpu.DeviceTensor(gpu.DeviceBuffer.from_array(host), self.shape, U.NP[kind], e, st)
        assert all(x * (4 if kind == "f32" else 2) % 32 == 16 for x in (e, st[0], st[1]))


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f32", 128), ("f16", 64), ("bf16", 128)])
def test_rows_of_16_byte_alignment(gpu, kind, dim):
    rng = np.random.default_rng([dim, 30])
    cached = "bf16" if kind == "bf16" else "f16"
    cache = Cache(rng, [90, 7, 41], 2, 101, dim, cached)
    prefix = Cache(rng, [130], 2, 131, dim, cached)
    start = [0, 60, 67, 100]
    for heads in (6, 40):
        single, many = (NarrowRows(gpu, rng, n, heads, dim, kind) for n in (3, 100))
        check_window(gpu, single, cache, None, 30, 3)
        check_window(gpu, many, cache, start, 30, 3)
        check_scored(gpu, single, cache, None, None)
        check_scored(gpu, many, cache, start, None)
        check_prefix(gpu, single, prefix, cache)
        check_prefix(gpu, many, prefix, cache, start)


def tight_scored(gpu, r, cache, start=None, scale=None, acc_in=None, nan_rows=None):
    """Runs the scored operator and checks out, lse and acc; acc with a bound of its own for
    every slot: each pair's weight times that pair's relative error (its score and its lse, the
    exponentials, the sum over the slots it sees), and the adding up of the sequence's pairs
    of one kv head, in 32 bits in any order.  nan_rows: [row][head] whose outputs are not checked."""
    n, kv, slots, dim = cache.k.shape
    rows, heads, _ = r.shape
    g = heads // kv
    st = None if start is None else i32(start)
    dst = f32(np.full((n, kv, slots), 55.0, np.float32))
    ws = workspace(gpu, gpu.attn_scored_workspace(r.q, cache.view, start=st))
    gpu.attn_scored(r.q, cache.view, r.out, None if acc_in is None else f32(acc_in), dst, ws, start=st, lse=r.lse,
                    scale=scale)
    got = dst.download().reshape(n, kv, slots).astype(np.float64)
    with np.errstate(invalid="ignore"):
        out, lse, acc, extra = U.reference(r.values, cache, start, scale=scale)
    size, reach, seen = extra
    first = np.arange(n + 1) if start is None else np.asarray(start)
    all_rows = slice(first[0], first[-1])
    fine = np.ones((rows, heads), bool) if nan_rows is None else ~nan_rows
    o, tol = r.result(), U.out_tolerance(np.nan_to_num(out), tuple(np.nan_to_num(x) for x in extra), r.kind, dim)
    bad = ~(np.abs(o - out) <= tol) & fine[..., None]
    assert not bad[all_rows].any(), (np.argwhere(bad)[:5], o[bad][:5], out[bad][:5], tol[bad][:5])
    z, ztol = r.lse.download().reshape(rows, heads), U.lse_tolerance(lse, extra, dim)
    with np.errstate(invalid="ignore"):
        assert ((np.abs(z - lse) <= ztol) | ((lse == -np.inf) & (z == -np.inf)))[all_rows].all()
    rel = 2.2 * U.score_error(reach, dim) + 2.0 ** -20 + (seen + 16) * 2.0 ** -24 + \
        2.0 ** -21 * np.abs(np.where(np.isfinite(lse), lse, 0))
    for b in range(n):
        lo, hi, length = first[b], first[b + 1], min(max(int(cache.length[b]), 0), slots)
        err = np.zeros((kv, slots))
        for row in range(lo, hi):
            p = length - hi + row
            for h in range(heads):
                if p >= 0:
                    s = cache.k[b, h // g, :p + 1] @ r.values[row, h] * (
                        dim ** -0.5 if scale is None else float(np.float32(scale)))
                    err[h // g, :p + 1] += rel[row, h] * np.exp(s - lse[row, h])
        base = np.zeros((kv, slots)) if acc_in is None else acc_in[b].astype(np.float64)
        err += ((hi - lo) * g + 16) * 2.0 ** -24 * acc[b] + 2.0 ** -23 * np.abs(base + acc[b]) + 1e-12
        bad = ~(np.abs(got[b] - base - acc[b]) <= err)
        bad[:, length:] = got[b][:, length:] != 55.0
        assert not bad.any(), (b, np.argwhere(bad)[:5], got[b][bad][:5], (base + acc[b])[bad][:5], err[bad][:5])
    return got


@pytest.mark.parametrize("spread, scale", [(1e-38, 1e-8), (0.0, 3e38), (1e38, 1e-38), (1e36, 2e-37), (2e-38, 5e37),
                                           (1.0, 1e-45)])
def test_scales_and_rows_at_the_ends_of_32_bits(gpu, spread, scale):
    """Rows times scale are in range where neither is: masked slots stay masked (an infinity
    times a factor that has become 0 is no number), and kept scores are in range too."""
    rng = np.random.default_rng(31)
    cache = Cache(rng, [77, 5, 40], 2, 101, 64, "f16")
    prefix = Cache(rng, [130], 2, 131, 64, "f16")
    for kind in ("f32",) if 0 < spread != 1 else ("f32", "f16"):
        for start, n in ((None, 3), ([0, 60, 65, 100], 100)):
            # of as many normal numbers as 100 rows have some are past 3.4
            r = Rows(gpu, rng, n, 6, 64, kind, spread=spread if n == 3 else min(spread, 1e37))
            check_window(gpu, r, cache, start, 30, 3, scale=scale)
            tight_scored(gpu, r, cache, start, scale=scale)
            st = None if start is None else i32(start)
            ws = workspace(gpu, gpu.attn_prefix_workspace(r.q, prefix.view, cache.view, start=st))
            gpu.attn_prefix(r.q, prefix.view, cache.view, r.out, ws, start=st, lse=r.lse, scale=scale)
            out, _, _, extra = U.reference(r.values, cache, start, prefix=prefix, scale=scale)
            check_out(r.result(), out, extra, kind, 64)


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("n_rows", [1, 40])
def test_nan_where_weights_vanish(gpu, kind, dim, n_rows):
    """V is no number in seen slots whose weights are 0 beside the others': 0 times NaN is NaN,
    however the slots are cut into ranges (2000 slots: several), and all other dims are fine."""
    rng = np.random.default_rng([dim, 32])
    cached = "bf16" if kind == "bf16" else "f16"
    q = rng.standard_normal(dim)
    for slots in (400, 2000):
        def near(k, v):
            k[:] = np.where(np.arange(k.shape[2]) < slots // 2, 10.0, -10.0)[:, None] * q
            v[:, :, slots - 60, :3] = np.nan

        cache = Cache(rng, [slots], 1, slots, dim, cached, edit=near)
        r = Rows(gpu, rng, n_rows, 2, dim, kind)
        r.values[:] = decode(encode(np.broadcast_to(q, r.shape), kind), kind)
        r.q = U.tensor(r.values, kind)[0]
        start = None if n_rows == 1 else i32([0, n_rows])
        for run in ("window", "scored", "prefix"):
            if run == "window":
                ws = workspace(gpu, gpu.attn_window_workspace(r.q, cache.view, start=start))
                gpu.attn_window(r.q, cache.view, r.out, ws, start=start)
            elif run == "scored":
                ws = workspace(gpu, gpu.attn_scored_workspace(r.q, cache.view, start=start))
                acc = f32(np.zeros((1, 1, slots)))
                gpu.attn_scored(r.q, cache.view, r.out, None, acc, ws, start=start)
                a = acc.download()
                # each of the 2 n_rows pairs' weights add up to 1, but for each one's relative error
                reach = 10 * np.abs(q).max() * np.abs(q).sum() * dim ** -0.5
                err = 2.2 * U.score_error(reach, dim) + 2.0 ** -20 + (slots + 2 * n_rows + 32) * 2.0 ** -24
                assert np.isfinite(a).all() and abs(a.astype(np.float64).sum() - 2 * n_rows) < 2 * n_rows * err
            else:
                own = Cache(rng, [n_rows], 1, n_rows, dim, cached, edit=lambda k, v: k.fill(0))
                ws = workspace(gpu, gpu.attn_prefix_workspace(r.q, cache.view, own.view, start=start))
                gpu.attn_prefix(r.q, cache.view, own.view, r.out, ws, start=start)
            got = r.result()
            where = np.argwhere(np.isnan(got) != (np.arange(dim) < 3))
            assert not len(where), (slots, run, len(where), where[:3])
