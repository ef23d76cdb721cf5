"""Cache-attention operators on the GPU against their formulas in 64 bits.  Tolerances are
derived per element in attn_util."""
import ctypes as C
from types import SimpleNamespace

import numpy as np
import pytest

import attn_util as U
from attn_util import Cache, check_out, encode, decode, f32, i32, tensor

pytestmark = pytest.mark.gpu

LAYOUTS = [("f32", 64, 32, 8, "head"), ("f16", 64, 4, 2, "slot"), ("bf16", 64, 9, 3, "mixed"),
           ("f32", 128, 6, 6, "mixed"), ("f16", 128, 28, 4, "head"), ("bf16", 128, 20, 1, "slot")]


def ids(v):
    return "-".join(map(str, v)) if isinstance(v, tuple) else str(v)


class Rows:
    """q and out of a call; out starts as a pattern, so that what is left alone shows."""

    def __init__(self, gpu, rng, n, heads, dim, kind, padded=False, spread=1.5):
        x = (spread * rng.standard_normal((n, heads, dim))).astype(np.float32)
        self.kind, self.shape = kind, (n, heads, dim)
        e = encode(x, kind)
        self.values = decode(e, kind).astype(np.float64)
        st = (heads * (dim + 8) + 16, dim + 8, 1) if padded else (heads * dim, dim, 1)
        size = max(1, n * st[0])
        self.at = np.arange(n)[:, None, None] * st[0] + np.arange(heads)[:, None] * st[1] + np.arange(dim)
        host = np.full(size, 0x7F if kind == "bf16" else 7, dtype=np.uint16 if kind == "bf16" else U.NP[kind])
        host[self.at] = e
        self.q = gpu.DeviceTensor(gpu.DeviceBuffer.from_array(host), self.shape, U.NP[kind], 0, st)
        host[:] = 77
        self.out = gpu.DeviceTensor(gpu.DeviceBuffer.from_array(host), self.shape, U.NP[kind], 0, st)
        self.lse = f32(np.full((n, heads), 77.0, np.float32))

    def result(self):
        flat = self.out.download()
        rest = np.delete(flat, self.at.reshape(-1))
        assert (rest == 77).all(), "elements between the rows were written"
        return decode(flat[self.at], self.kind).astype(np.float64)

    def untouched(self, rows):
        flat = self.out.download()
        return (flat[self.at[rows]] == 77).all() and (self.lse.download().reshape(self.shape[:2])[rows] == 77).all()


def workspace(gpu, n, fill=0xFF):
    """Bytes that were used before: NaN wherever a kernel would read what it did not write."""
    return gpu.DeviceBuffer.from_array(np.full(max(n, 16), fill, np.uint8))


def run_window(gpu, r, cache, stream=0, **kw):
    ws = workspace(gpu, gpu.attn_window_workspace(r.q, cache.view, **{k: v for k, v in kw.items() if k in (
        "window", "sinks", "start")}))
    gpu.attn_window(r.q, cache.view, r.out, ws, lse=r.lse, stream=stream, **kw)
    return ws


def check_window(gpu, r, cache, start, window, sinks, scale=None):
    run_window(gpu, r, cache, window=window, sinks=sinks, start=None if start is None else i32(start), scale=scale)
    out, lse, _, extra = U.reference(r.values, cache, start, window, sinks, scale)
    rows = slice(None) if start is None else slice(max(0, start[0]), min(start[-1], r.shape[0]))
    got = r.result()
    check_out(got[rows], out[rows], tuple(x[rows] for x in extra), r.kind, r.shape[2])
    g = r.lse.download().reshape(lse.shape)
    tol = U.lse_tolerance(lse, extra, r.shape[2])
    ok = (np.abs(g - lse) <= tol) | ((lse == -np.inf) & (g == -np.inf))
    assert ok[rows].all(), (g[rows][~ok[rows]][:5], lse[rows][~ok[rows]][:5])
    return got


# ------------------------------------------------------------------ window
@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 0), (1, 3), (7, 0), (64, 4), (100, 70), (300, 1000)], ids=ids)
@pytest.mark.parametrize("layout", LAYOUTS, ids=ids)
def test_window_single_rows(gpu, layout, window, sinks):
    kind, dim, heads, kv, order = layout
    rng = np.random.default_rng([dim, heads, window, sinks])
    length = [0, 1, 2, 15, 16, 17, 63, 64, 65, 200, 333, 129]
    cache = Cache(rng, length, kv, 333, dim, kind if kind == "bf16" else "f16", order)
    r = Rows(gpu, rng, len(length), heads, dim, kind, padded=order == "mixed")
    check_window(gpu, r, cache, None, window, sinks)


@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 0), (1, 2), (33, 0), (64, 5), (40, 200)], ids=ids)
@pytest.mark.parametrize("layout", LAYOUTS, ids=ids)
def test_window_ragged_rows(gpu, layout, window, sinks):
    kind, dim, heads, kv, order = layout
    rng = np.random.default_rng([dim, heads, window, sinks, 1])
    # a sequence without rows, rows that have no position, prompts, chunks onto a past
    counts, length = [0, 1, 2, 31, 70, 5, 3, 9], [9, 1, 2, 31, 150, 140, 1, 0]
    start = np.concatenate([[2], 2 + np.cumsum(counts)])
    cache = Cache(rng, length, kv, 157, dim, kind if kind == "bf16" else "f16", order)
    r = Rows(gpu, rng, int(start[-1]) + 3, heads, dim, kind, padded=order == "mixed")
    check_window(gpu, r, cache, start, window, sinks)
    assert r.untouched([0, 1, -1, -2, -3])


@pytest.mark.parametrize("kind, dim, heads, kv", [("f32", 64, 8, 2), ("bf16", 128, 7, 1), ("f16", 64, 2, 2)], ids=ids)
@pytest.mark.parametrize("window, sinks", [(0, 0), (500, 4)], ids=ids)
def test_window_long_single_rows(gpu, kind, dim, heads, kv, window, sinks):
    rng = np.random.default_rng([heads, window])
    cache = Cache(rng, [5001, 4096, 1, 2977], kv, 5003, dim, "bf16" if kind == "bf16" else "f16")
    r = Rows(gpu, rng, 4, heads, dim, kind)
    check_window(gpu, r, cache, None, window, sinks)


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f16", 128), ("bf16", 64)], ids=ids)
@pytest.mark.parametrize("window, sinks", [(0, 0), (129, 4)], ids=ids)
def test_window_long_prompt(gpu, kind, dim, window, sinks):
    rng = np.random.default_rng([dim, window])
    cache = Cache(rng, [700, 1500], 1, 1501, dim, "bf16" if kind == "bf16" else "f16", "slot")
    r = Rows(gpu, rng, 700 + 130, 3, dim, kind)
    check_window(gpu, r, cache, [0, 700, 830], window, sinks)


@pytest.mark.parametrize("heads, kv", [(128, 1), (130, 2), (33, 1)])
def test_many_heads_a_group(gpu, heads, kv):
    """More query heads than a row tile holds, in single rows and in chunks."""
    rng = np.random.default_rng(heads)
    cache = Cache(rng, [70, 300, 5], kv, 301, 64, "f16")
    check_window(gpu, Rows(gpu, rng, 3, heads, 64, "f16"), cache, None, 90, 3)
    check_window(gpu, Rows(gpu, rng, 9, heads, 64, "f32"), cache, [0, 3, 7, 9], 90, 3)
    check_scored(gpu, Rows(gpu, rng, 3, heads, 64, "f32"), cache, None, None)
    check_scored(gpu, Rows(gpu, rng, 9, heads, 64, "f16"), cache, [0, 3, 7, 9], None)


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f16", 64), ("bf16", 64), ("f32", 128), ("bf16", 128)])
def test_window_large_prompts(gpu, kind, dim):
    """Enough rows for the larger tiles: some rows of them, against single rows in 64 bits.
    Slot 3000 of the first prompt holds NaN in V: rows before it and those whose window has
    passed it do not see it."""
    rng = np.random.default_rng([dim, 19])
    length, counts, heads, kv = [3907, 333], [3850, 130], 24, 8

    def edit(k, v):
        v[0, :, 3000] = np.nan

    cache = Cache(rng, length, kv, 3911, dim, "bf16" if kind == "bf16" else "f16", "slot", edit)
    start = np.concatenate([[0], np.cumsum(counts)])
    r = Rows(gpu, rng, int(start[-1]), heads, dim, kind)
    for window, sinks in ((0, 0), (700, 5)):
        run_window(gpu, r, cache, window=window, sinks=sinks, start=i32(start))
        got, lse = r.result(), r.lse.download().reshape(r.shape[:2])
        rows = np.concatenate([rng.choice(r.shape[0], 25, replace=False), [0, 1, 2942, 2943, 3642, 3643, 3849, 3850, 3979]])
        for row in rows:
            b = int(row >= start[1])
            pos = length[b] - start[b + 1] + row
            one = SimpleNamespace(k=cache.k[b:b + 1], v=cache.v[b:b + 1], length=[pos + 1])
            out, want, _, extra = U.reference(r.values[row:row + 1], one, None, window, sinks)
            if b == 0 and pos >= 3000 and (window == 0 or pos < 3700):
                assert np.isnan(got[row]).all()
            else:
                check_out(got[row:row + 1], out, extra, kind, dim)
            assert (np.abs(lse[row] - want[0]) <= U.lse_tolerance(want, extra, dim)[0]).all()


@pytest.mark.parametrize("kind, dim", [("f16", 64), ("bf16", 128)])
def test_many_prompts(gpu, kind, dim):
    """The larger tiles over many short sequences, each ending inside one."""
    rng = np.random.default_rng([dim, 20])
    counts = rng.integers(40, 80, 68 if dim == 64 else 50)
    start = np.concatenate([[0], np.cumsum(counts)])
    cache = Cache(rng, counts + rng.integers(-20, 40, len(counts)), 8, 120, dim, kind)
    r = Rows(gpu, rng, int(start[-1]), 24, dim, kind)
    check_scored(gpu, r, cache, start, None)


@pytest.mark.parametrize("heads, kv", [(128, 1), (33, 1), (34, 2)])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_many_heads_a_group_of_128_dims(gpu, heads, kv, kind):
    rng = np.random.default_rng([heads, 21])
    cache = Cache(rng, [70, 700, 5], kv, 701, 128, "bf16" if kind == "bf16" else "f16")
    check_window(gpu, Rows(gpu, rng, 3, heads, 128, kind), cache, None, 0, 0)
    check_window(gpu, Rows(gpu, rng, 3, heads, 128, kind), cache, None, 90, 3)
    check_scored(gpu, Rows(gpu, rng, 3, heads, 128, kind), cache, None, None)


def test_many_sequences(gpu):
    """More sequences than a wave has lanes, most of few rows, some of none."""
    rng = np.random.default_rng(17)
    counts = rng.choice([0, 1, 1, 2, 5, 40], 150)
    start = np.concatenate([[0], np.cumsum(counts)])
    cache = Cache(rng, rng.integers(0, 60, 150), 2, 60, 64, "f16", "slot")
    check_window(gpu, Rows(gpu, rng, int(start[-1]), 2, 64, "f16"), cache, start, 0, 0)
    check_window(gpu, Rows(gpu, rng, int(start[-1]), 2, 64, "f16"), cache, start, 11, 2)
    check_scored(gpu, Rows(gpu, rng, int(start[-1]), 2, 64, "f32"), cache, start, None)
    prefix = Cache(rng, [77], 2, 80, 64, "f16", "slot")
    check_prefix(gpu, Rows(gpu, rng, int(start[-1]), 2, 64, "f16"), prefix, cache, start)


def test_window_and_sinks_past_every_length(gpu):
    rng = np.random.default_rng(18)
    cache = Cache(rng, [70, 130], 2, 150, 64, "f16")
    for window, sinks in ((0xFFFFFFFF, 0), (0xFFFFFFFF, 0xFFFFFFFF), (0x80000000, 5), (1, 0xFFFFFFFF)):
        check_window(gpu, Rows(gpu, rng, 2, 4, 64, "f16"), cache, None, window, sinks)
        check_window(gpu, Rows(gpu, rng, 80, 4, 64, "f16"), cache, [0, 30, 80], window, sinks)


def test_window_lengths_out_of_range_count_as_their_ends(gpu):
    rng = np.random.default_rng(5)
    cache = Cache(rng, [-3, 500, 60, 2147483647, -2147483648], 2, 60, 64, "f16")
    r = Rows(gpu, rng, 5, 4, 64, "f16")
    check_window(gpu, r, cache, None, 20, 2)


def test_window_starts_out_of_range(gpu):
    """Starts below 0 and past the rows count as the ends, a descending one as no rows."""
    rng = np.random.default_rng(6)
    cache = Cache(rng, [40, 50, 60, 30], 2, 60, 64, "f16")
    r = Rows(gpu, rng, 20, 4, 64, "f16")
    start = [-5, 6, 4, 12, 500]
    run_window(gpu, r, cache, window=9, sinks=1, start=i32(start))
    out, _, _, extra = U.reference(r.values, cache, start, 9, 1)
    # rows 4 and 5 belong to two sequences: either's answer; the rest to one
    got = r.result()
    rows = [i for i in range(20) if i not in (4, 5)]
    check_out(got[rows], out[rows], tuple(x[rows] for x in extra), "f16", 64)


def test_window_large_scores(gpu):
    """Scores far apart and far from zero: no overflow, weights of one slot alone."""
    rng = np.random.default_rng(7)
    for kind in ("f32", "f16"):
        cache = Cache(rng, [257, 100], 2, 300, 64, "f16")
        r = Rows(gpu, rng, 2, 4, 64, kind, spread=60)
        check_window(gpu, r, cache, None, 0, 0, scale=0.5)
    r = Rows(gpu, rng, 2, 4, 64, "f32", spread=3e5)  # past binary16's range
    check_window(gpu, r, cache, None, 0, 0, scale=1e-6)
    r = Rows(gpu, rng, 2, 4, 64, "f32", spread=1e-9)  # below it
    check_window(gpu, r, cache, None, 0, 0, scale=1e9)


@pytest.mark.parametrize("kind, dim, first", [("f32", 64, 0), ("f16", 64, 300), ("bf16", 64, 0), ("f32", 128, 300),
                                              ("bf16", 128, -300)])
def test_scores_that_rise_and_fall(gpu, kind, dim, first):
    """K of slot j is (first + j / 2) times one vector: for some rows every block's scores pass
    all before them, for others the first slots' are the largest, far below zero or above."""
    rng = np.random.default_rng([dim, abs(first), 23])
    length = [500, 130, 33]

    def edit(k, v):
        k[:] = (first + 0.5 * np.arange(k.shape[2]))[:, None] * k[:, :, :1]

    cache = Cache(rng, length, 2, 501, dim, "bf16" if kind == "bf16" else "f16", edit=edit)
    check_window(gpu, Rows(gpu, rng, 3, 8, dim, kind), cache, None, 0, 0)
    check_scored(gpu, Rows(gpu, rng, 3, 40, dim, kind), cache, None, None)
    check_window(gpu, Rows(gpu, rng, 99, 6, dim, kind), cache, [0, 60, 66, 99], 70, 3)
    check_scored(gpu, Rows(gpu, rng, 99, 6, dim, kind), cache, [0, 60, 66, 99], None)
    prefix = Cache(rng, [700], 2, 700, dim, "bf16" if kind == "bf16" else "f16", edit=edit)
    check_prefix(gpu, Rows(gpu, rng, 3, 40, dim, kind), prefix, cache)
    check_prefix(gpu, Rows(gpu, rng, 3, 10, dim, kind), prefix, cache)


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f16", 128), ("bf16", 64)], ids=ids)
def test_window_unseen_slots_hold_anything(gpu, kind, dim):
    """NaN and infinities in slots that a row does not see: past the length, before the
    window, and (for earlier rows of a prompt) after its position."""
    rng = np.random.default_rng(8)
    bad = [np.nan, np.inf, -np.inf, 65504.0]

    def edit(k, v):
        for x in (k, v):
            for b, n in ((0, 90), (1, 41)):
                x[b, :, n:] = np.resize(bad, x[b, :, n:].shape)  # past the length
            x[0, :, 5:60] = np.resize(bad, x[0, :, 5:60].shape)  # between sinks and window

    cache = Cache(rng, [90, 41], 2, 133, dim, "bf16" if kind == "bf16" else "f16", edit=edit)
    r = Rows(gpu, rng, 2, 6, dim, kind)
    check_window(gpu, r, cache, None, 30, 5)
    # a prompt: slots 20, 21 of sequence 1 are NaN and infinite; rows 0..19 do not see them
    def late(k, v):
        for x in (k, v):
            x[1, :, 41:] = np.nan
        v[1, :, 20] = np.nan
        v[1, :, 21, :3] = np.inf
        k[1, :, 25] = np.inf

    cache = Cache(rng, [90, 41], 2, 133, dim, "bf16" if kind == "bf16" else "f16", edit=late)
    r = Rows(gpu, rng, 33 + 41, 6, dim, kind)
    start = [0, 33, 74]
    for window, sinks in ((0, 0), (4, 2)):
        run_window(gpu, r, cache, window=window, sinks=sinks, start=i32(start))
        out, lse, _, extra = U.reference(r.values, cache, start, window, sinks)
        got = r.result()
        fine = np.isfinite(out) & np.isfinite(extra[0]) & np.isfinite(extra[1])[..., None]
        assert fine[:53].all() and not fine[53:].all()
        tol = U.out_tolerance(np.where(fine, out, 0), tuple(np.nan_to_num(x, posinf=0) for x in extra), kind, dim)
        assert (np.abs(got - out)[fine] <= tol[fine]).all()
        assert not np.isfinite(got[~np.isfinite(out)]).any()
        if window:  # the rows whose window has passed them see numbers again
            assert fine[33 + 30:].all()


@pytest.mark.parametrize("stride", ["seq", "head", "slot"])
def test_window_offsets_past_32_bits(gpu, stride):
    rng = np.random.default_rng(9)
    far = (1 << 31) + 8 * 1013  # elements
    n, kv, slots, dim = (2, 1, 40, 64) if stride == "seq" else (1, 2, 40, 64) if stride == "head" else (1, 1, 40, 64)
    small = Cache(rng, [40] * n, kv, slots, dim, "f16")
    if stride == "slot":
        step = (far // 39 + 8) // 8 * 8
        st, count = (0, 0, step, 1), 39 * step + 64
    else:
        st, count = ((far, 0, 64, 1) if stride == "seq" else (0, far, 64, 1)), far + 40 * 64
    bufs = [gpu.DeviceBuffer(2 * count) for _ in range(2)]
    t = []
    for buf, x in zip(bufs, (small.k, small.v)):
        for b in range(n):
            for h in range(kv):
                for s in range(slots if stride == "slot" else 1):
                    rows = x[b, h, s] if stride == "slot" else x[b, h]
                    buf.upload(rows.astype(np.float16), 2 * (b * st[0] + h * st[1] + s * st[2]))
        t.append(gpu.DeviceTensor(buf, (n, kv, slots, dim), np.float16, 0, st))
    small.view = gpu.KvCache(t[0], t[1], small.tl)
    for start, rows in ((None, n), (list(range(0, 11 * n, 10)), 10 * n)):
        r = Rows(gpu, rng, rows, 2 * kv, dim, "f16")
        check_window(gpu, r, small, start, 0, 0)
    for b in bufs:
        b.free()


# ------------------------------------------------------------------ scored
def check_scored(gpu, r, cache, start, acc_in, in_place=False):
    shape = cache.k.shape[:3]
    dst = f32(np.full(shape, 55.0, np.float32) if not in_place else acc_in)
    src = dst if in_place else None if acc_in is None else f32(acc_in)
    st = None if start is None else i32(start)
    ws = workspace(gpu, gpu.attn_scored_workspace(r.q, cache.view, start=st))
    gpu.attn_scored(r.q, cache.view, r.out, src, dst, ws, start=st, lse=r.lse)
    out, lse, acc, extra = U.reference(r.values, cache, start)
    rows = slice(None) if start is None else slice(start[0], start[-1])
    check_out(r.result()[rows], out[rows], tuple(x[rows] for x in extra), r.kind, r.shape[2])
    got = dst.download().reshape(shape)
    base = np.zeros(shape) if acc_in is None else acc_in.astype(np.float64)
    used = np.arange(shape[2]) < np.clip(cache.length, 0, shape[2])[:, None, None]
    left = acc_in if in_place else np.full(shape, 55.0)
    assert (got == left)[~np.broadcast_to(used, shape)].all()
    # each weight's relative error: of its score, of the lse and of the exponential; the sums
    err = 2.2 * U.score_error(extra[1].max(initial=0), r.shape[2]) + 2.0 ** -20 + (extra[2].max(initial=0) + r.shape[0] * r.shape[1] + 32) \
        * 2.0 ** -24 + 2.0 ** -21 * np.abs(lse[np.isfinite(lse)]).max(initial=0)
    tol = err * acc + 2.0 ** -23 * np.abs(base + acc) + 1e-12
    bad = ~(np.abs(got - base - acc) <= tol) & used
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], (base + acc)[bad][:5], tol[bad][:5])
    return got


@pytest.mark.parametrize("layout", LAYOUTS, ids=ids)
@pytest.mark.parametrize("given", ["none", "apart", "in_place"])
def test_scored_single_rows(gpu, layout, given):
    kind, dim, heads, kv, order = layout
    rng = np.random.default_rng([dim, heads, 2])
    length = [0, 1, 16, 17, 64, 65, 200, 333, 700]
    cache = Cache(rng, length, kv, 701, dim, kind if kind == "bf16" else "f16", order)
    r = Rows(gpu, rng, len(length), heads, dim, kind, padded=order == "mixed")
    acc = None if given == "none" else rng.random((len(length), kv, 701), dtype=np.float32) * 3
    check_scored(gpu, r, cache, None, acc, given == "in_place")


@pytest.mark.parametrize("layout", LAYOUTS, ids=ids)
def test_scored_ragged_rows(gpu, layout):
    kind, dim, heads, kv, order = layout
    rng = np.random.default_rng([dim, heads, 3])
    counts, length = [0, 1, 2, 31, 70, 5, 3, 9], [9, 1, 2, 31, 150, 140, 1, 0]
    start = np.concatenate([[1], 1 + np.cumsum(counts)])
    cache = Cache(rng, length, kv, 157, dim, kind if kind == "bf16" else "f16", order)
    r = Rows(gpu, rng, int(start[-1]) + 2, heads, dim, kind)
    check_scored(gpu, r, cache, start, rng.random((8, kv, 157), dtype=np.float32))
    assert r.untouched([0, -1, -2])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_scored_long(gpu, kind):
    rng = np.random.default_rng(10)
    cache = Cache(rng, [4999, 2500], 2, 5003, 64, "bf16" if kind == "bf16" else "f16")
    r = Rows(gpu, rng, 2, 8, 64, kind)
    a = check_scored(gpu, r, cache, None, None)
    assert np.array_equal(a.view(np.uint32), check_scored(gpu, r, cache, None, None).view(np.uint32))
    cache = Cache(rng, [900, 411], 1, 901, 64, "bf16" if kind == "bf16" else "f16")
    r = Rows(gpu, rng, 900 + 200, 2, 64, kind)
    a = check_scored(gpu, r, cache, [0, 900, 1100], None)
    assert np.array_equal(a.view(np.uint32), check_scored(gpu, r, cache, [0, 900, 1100], None).view(np.uint32))


def test_scored_without_rows_keeps_acc(gpu):
    rng = np.random.default_rng(11)
    cache = Cache(rng, [5, 0], 2, 9, 64, "f16")
    r = Rows(gpu, rng, 0, 4, 64, "f16")
    check_scored(gpu, r, cache, [0, 0, 0], rng.random((2, 2, 9), dtype=np.float32))


# ------------------------------------------------------------------ prefix
def check_prefix(gpu, r, prefix, cache, start=None):
    st = None if start is None else i32(start)
    ws = workspace(gpu, gpu.attn_prefix_workspace(r.q, prefix.view, cache.view, start=st))
    gpu.attn_prefix(r.q, prefix.view, cache.view, r.out, ws, start=st, lse=r.lse)
    out, lse, _, extra = U.reference(r.values, cache, start, prefix=prefix)
    rows = slice(None) if start is None else slice(start[0], start[-1])
    check_out(r.result()[rows], out[rows], tuple(x[rows] for x in extra), r.kind, r.shape[2])
    g = r.lse.download().reshape(lse.shape)[rows]
    tol = U.lse_tolerance(lse, extra, r.shape[2])[rows]
    assert ((np.abs(g - lse[rows]) <= tol) | ((lse[rows] == -np.inf) & (g == -np.inf))).all()


@pytest.mark.parametrize("n_prefix", [0, 1, 31, 64, 65, 500, 3001])
@pytest.mark.parametrize("layout", LAYOUTS, ids=ids)
def test_prefix_single_rows(gpu, layout, n_prefix):
    kind, dim, heads, kv, order = layout
    rng = np.random.default_rng([dim, heads, n_prefix])
    cached = kind if kind == "bf16" else "f16"
    length = [0, 1, 2, 17, 64, 65, 100, 3, 0, 33, 7]

    def edit(k, v):
        for x in (k, v):
            x[:, :, n_prefix:] = np.nan

    prefix = Cache(rng, [n_prefix], kv, n_prefix + 9, dim, cached, order, edit)
    cache = Cache(rng, length, kv, 100, dim, cached, order)
    r = Rows(gpu, rng, len(length), heads, dim, kind, padded=order == "mixed")
    check_prefix(gpu, r, prefix, cache)


@pytest.mark.parametrize("layout", LAYOUTS, ids=ids)
def test_prefix_ragged_rows(gpu, layout):
    kind, dim, heads, kv, order = layout
    rng = np.random.default_rng([dim, heads, 4])
    cached = kind if kind == "bf16" else "f16"
    counts, length = [0, 1, 2, 31, 45, 3], [9, 1, 2, 31, 70, 1]
    start = np.concatenate([[1], 1 + np.cumsum(counts)])
    prefix = Cache(rng, [300], kv, 300, dim, cached, order)
    cache = Cache(rng, length, kv, 71, dim, cached, order)
    r = Rows(gpu, rng, int(start[-1]) + 2, heads, dim, kind)
    check_prefix(gpu, r, prefix, cache, start)
    assert r.untouched([0, -1, -2])


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("bf16", 128), ("f16", 64)])
def test_prefix_of_few_ragged_rows(gpu, kind, dim):
    rng = np.random.default_rng([dim, 6])
    cached = kind if kind == "bf16" else "f16"
    prefix = Cache(rng, [1200], 3, 1201, dim, cached)
    for counts, heads in (([2, 0, 3], 3), ([1, 1, 1], 6), ([4, 3, 9], 12)):
        start = np.concatenate([[0], np.cumsum(counts)])
        cache = Cache(rng, [5, 9, 40], 3, 41, dim, cached)
        check_prefix(gpu, Rows(gpu, rng, int(start[-1]), heads, dim, kind), prefix, cache, start)


@pytest.mark.parametrize("kind, dim, heads, kv, n", [("f32", 64, 8, 2, 70), ("bf16", 128, 3, 1, 41), ("f16", 64, 2, 2, 1)])
def test_prefix_batches(gpu, kind, dim, heads, kv, n):
    rng = np.random.default_rng([n, 5])
    cached = kind if kind == "bf16" else "f16"
    prefix = Cache(rng, [2049], kv, 2100, dim, cached)
    cache = Cache(rng, rng.integers(0, 30, n), kv, 30, dim, cached)
    check_prefix(gpu, Rows(gpu, rng, n, heads, dim, kind), prefix, cache)


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f16", 64), ("f32", 128), ("bf16", 128)])
@pytest.mark.parametrize("heads, kv, n, n_prefix, slots", [
    (3, 1, 40, 2203, 1000),  # own slots in several ranges, longer than the prefix
    (4, 2, 45, 9001, 70),    # the prefix in many ranges
    (34, 2, 9, 700, 150),    # more query heads than a row tile, in a launch of their own
    (10, 2, 13, 2500, 700)])
def test_prefix_and_own_slots_together(gpu, kind, dim, heads, kv, n, n_prefix, slots):
    """Prefix of many rows and their own slots in one launch, each in key ranges."""
    rng = np.random.default_rng([heads, dim, 22])
    cached = kind if kind == "bf16" else "f16"
    prefix = Cache(rng, [n_prefix], kv, n_prefix + 5, dim, cached)
    length = rng.integers(0, slots + 1, n)
    length[[0, 1, -1]] = 0, slots, 1
    check_prefix(gpu, Rows(gpu, rng, n, heads, dim, kind), prefix, Cache(rng, length, kv, slots, dim, cached, "slot"))


# ------------------------------------------------------------------ eviction
def evict_inputs(rng, n, kv, slots, pattern):
    acc = rng.random((n, kv, slots), dtype=np.float32) ** 4
    if pattern == "ties":
        acc = rng.integers(0, 3, acc.shape).astype(np.float32)
    if pattern == "equal":
        acc[:] = 0.0
    if pattern == "odd":
        acc = rng.standard_normal(acc.shape).astype(np.float32)
        odd = np.array([np.nan, np.inf, -np.inf, -0.0, 0.0, 1e-42, -1e-42, 3.4e38, -3.4e38], np.float32)
        where = rng.random(acc.shape) < 0.5
        acc[where] = rng.choice(odd, where.sum())
    pos = np.cumsum(rng.integers(1, 4, acc.shape), -1).astype(np.int32) - 1
    if pattern == "odd":  # out of order, as an eviction in place leaves them
        pos = rng.permuted(pos, axis=-1)
    return acc, pos


def bits(x):
    return np.ascontiguousarray(x).view(np.uint32)


@pytest.mark.parametrize("place", ["apart", "in_place"])
@pytest.mark.parametrize("pattern", ["plain", "ties", "equal", "odd"])
@pytest.mark.parametrize("slots, keep, sinks, recent, dim, kind, order", [
    (1, 1, 0, 0, 64, "f16", "head"), (65, 64, 4, 16, 64, "f16", "slot"), (300, 1, 0, 0, 128, "bf16", "head"),
    (300, 1, 0, 1, 64, "f16", "mixed"), (1100, 1090, 10, 1000, 64, "bf16", "slot"), (2500, 700, 3, 100, 128, "f16", "mixed"),
    (9000, 33, 0, 33, 64, "f16", "head"), (513, 512, 0, 0, 64, "f16", "head"), (70, 70, 70, 0, 64, "f16", "head")],
    ids=ids)
def test_evict(gpu, slots, keep, sinks, recent, dim, kind, order, pattern, place):
    rng = np.random.default_rng([slots, keep, len(pattern)])
    kv = 3
    length = [slots, max(0, keep - 1), keep, min(slots, keep + 1), 0, slots + 5, -1, (slots + keep) // 2]
    n = len(length)
    acc, pos = evict_inputs(rng, n, kv, slots, pattern)
    cache = Cache(rng, length, kv, slots, dim, kind, order)
    src = lambda t: t.download().copy()  # noqa: E731
    ta, tp = f32(acc), i32(pos)
    ws = workspace(gpu, gpu.kv_evict_workspace(cache.view, keep))
    if place == "in_place":
        out, oa, op, ol, out_slots = cache.view, ta, tp, cache.tl, slots
        before = (cache.k, cache.v, acc, pos)
    else:
        out_slots = keep + 2
        base = Cache(rng, [0] * n, kv, out_slots, dim, kind, order)
        out, ol = base.view, base.tl
        before = (base.k, base.v, np.full((n, kv, out_slots), 9.0, np.float32), np.full((n, kv, out_slots), 9, np.int32))
        oa, op = f32(before[2]), i32(before[3])
    gpu.kv_evict(cache.view, ta, tp, keep, out, oa, op, ws, sinks=sinks, recent=recent)
    want = [x.copy() for x in before]
    for b in range(n):
        m = min(max(length[b], 0), slots)
        for h in range(kv):
            s = U.keep_slots(acc[b, h], pos[b, h], m, keep, sinks, recent)
            s = np.arange(m) if s is None else s
            for w, x in zip(want, (cache.k, cache.v, acc, pos)):
                w[b, h, :len(s)] = x[b, h][s]
    got = read_cache(out, kind, order)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    assert np.array_equal(bits(src(oa).reshape(want[2].shape)), bits(want[2]))
    assert np.array_equal(src(op).reshape(want[3].shape), want[3])
    assert np.array_equal(ol.download(), np.minimum(np.clip(length, 0, slots), keep))


@pytest.mark.parametrize("pattern", ["plain", "ties"])
def test_evict_long(gpu, pattern):
    """Past the slots whose ranks are held in registers and in shared memory."""
    rng = np.random.default_rng(19)
    slots, keep = 41003, 20011
    length = [slots, 33000]
    acc, pos = evict_inputs(rng, 2, 1, slots, pattern)
    cache = Cache(rng, length, 1, slots, 64, "f16")
    ta, tp = f32(acc), i32(pos)
    ws = workspace(gpu, gpu.kv_evict_workspace(cache.view, keep))
    gpu.kv_evict(cache.view, ta, tp, keep, cache.view, ta, tp, ws, sinks=4, recent=1000)
    p = tp.download().reshape(pos.shape)
    k, _ = read_cache(cache.view, "f16", "head")
    for b in range(2):
        s = U.keep_slots(acc[b, 0], pos[b, 0], length[b], keep, 4, 1000)
        assert np.array_equal(p[b, 0, :keep], pos[b, 0][s])
        assert np.array_equal(k[b, 0, :keep], cache.k[b, 0][s])
        assert np.array_equal(k[b, 0, keep:], cache.k[b, 0, keep:])


def read_cache(view, kind, order):
    n, kv, slots, dim = view.n_seq, view.kv_heads, view.slots, view.head_dim
    out = []
    for t in (view.k, view.v):
        flat = t.download()
        st = t.stride()
        at = (t.offset + np.arange(n)[:, None, None, None] * st[0] + np.arange(kv)[:, None, None] * st[1]
              + np.arange(slots)[:, None] * st[2] + np.arange(dim))
        out.append(decode(flat[at], kind).astype(np.float64))
    return out


def test_evict_again_and_again(gpu):
    """A cache at its limit: one token more, one slot less, ten times; what is left is what
    the rule leaves, whatever order the slots are in by then."""
    rng = np.random.default_rng(12)
    n, kv, keep, slots, dim = 2, 2, 50, 52, 64
    cache = Cache(rng, [keep, keep], kv, slots, dim, "f16")
    acc = rng.random((n, kv, slots), dtype=np.float32)
    pos = np.tile(np.arange(slots, dtype=np.int32), (n, kv, 1))
    ta, tp = f32(acc), i32(pos)
    ws = workspace(gpu, gpu.kv_evict_workspace(cache.view, keep))
    held = [[set(range(keep)) for _ in range(kv)] for _ in range(n)]
    weight = {(b, h, j): acc[b, h, j] for b in range(n) for h in range(kv) for j in range(keep)}
    for step in range(10):
        new = rng.random((n, kv), dtype=np.float32)
        a, p = (t.download().reshape(n, kv, slots) for t in (ta, tp))
        a[:, :, keep], p[:, :, keep] = new, keep + step
        ta.buf.upload(a), tp.buf.upload(p)
        cache.tl.buf.upload(np.full(n, keep + 1, np.int32))
        gpu.kv_evict(cache.view, ta, tp, keep, cache.view, ta, tp, ws, sinks=2, recent=8)
        p = tp.download().reshape(n, kv, slots)
        for b in range(n):
            for h in range(kv):
                held[b][h].add(keep + step)
                weight[b, h, keep + step] = new[b, h]
                free = [j for j in held[b][h] if j >= 2 and j <= keep + step - 8]
                held[b][h].remove(min(free, key=lambda j: weight[b, h, j]))
                assert set(p[b, h, :keep].tolist()) == held[b][h]


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("kind, dim, heads, kv", [("f32", 64, 8, 2), ("bf16", 128, 6, 3)], ids=ids)
def test_prompt_evicted_then_continued(gpu, kind, dim, heads, kv):
    """A prompt scored, cut to its heaviest slots, then a step over what stays: scored again
    and, as the shared prefix of three sequences, attended by each."""
    rng = np.random.default_rng(13)
    cached = kind if kind == "bf16" else "f16"
    T, keep = 150, 60
    cache = Cache(rng, [T], kv, T + 1, dim, cached)
    r = Rows(gpu, rng, T, heads, dim, kind)
    acc = check_scored(gpu, r, cache, [0, T], None)
    pos = np.tile(np.arange(T + 1, dtype=np.int32), (1, kv, 1))
    ta, tp = f32(acc), i32(pos)
    ws = workspace(gpu, gpu.kv_evict_workspace(cache.view, keep))
    gpu.kv_evict(cache.view, ta, tp, keep, cache.view, ta, tp, ws, sinks=4, recent=16)
    k, v = cache.k.copy(), cache.v.copy()
    for h in range(kv):
        s = U.keep_slots(acc[0, h], pos[0, h], T, keep, 4, 16)
        cache.k[0, h, :keep], cache.v[0, h, :keep] = k[0, h][s], v[0, h][s]
        assert np.array_equal(tp.download().reshape(pos.shape)[0, h, :keep], pos[0, h][s])
    cache.length = np.array([keep])
    step = Rows(gpu, rng, 1, heads, dim, kind)
    check_scored(gpu, step, cache, None, ta.download().reshape(acc.shape))
    own = Cache(rng, [1, 5, 9], kv, 9, dim, cached)
    check_prefix(gpu, Rows(gpu, rng, 3, heads, dim, kind), cache, own)


# ------------------------------------------------------------------ streams, graphs, refusals
class Hip:
    """The few HIP calls that streams and graphs need, of the runtime the library uses."""

    def __init__(self):
        self.L = C.CDLL("libamdhip64.so.7")

    def ok(self, name, *args):
        rc = getattr(self.L, name)(*args)
        assert rc == 0, (name, rc)

    def stream(self):
        s = C.c_void_p()
        self.ok("hipStreamCreateWithFlags", C.byref(s), C.c_uint(1))  # does not wait for the null stream
        return s

    def graph(self, s, enqueue):
        self.ok("hipStreamBeginCapture", s, C.c_int(2))
        enqueue()
        g, e = C.c_void_p(), C.c_void_p()
        self.ok("hipStreamEndCapture", s, C.byref(g))
        self.ok("hipGraphInstantiate", C.byref(e), g, None, None, C.c_size_t(0))
        return e


def test_captured_calls_follow_their_inputs(gpu):
    """Two graphs, each with a workspace of its own, replayed in turn with eager calls between
    them while lengths and rows change: every replay equals the eager call's bits."""
    hip = Hip()
    rng = np.random.default_rng(14)
    n, heads, kv, dim, slots, keep = 3, 8, 2, 64, 900, 300
    s = hip.stream()
    cache = Cache(rng, [900, 30, 500], kv, slots, dim, "f16")
    prefix = Cache(rng, [700], kv, 700, dim, "f16")
    r, out2 = Rows(gpu, rng, n, heads, dim, "f32"), Rows(gpu, rng, n, heads, dim, "f32")
    acc, acc2 = f32(np.zeros((n, kv, slots))), f32(np.zeros((n, kv, slots)))
    pos = i32(np.tile(np.arange(slots), (n, kv, 1)))
    kept = Cache(rng, [0] * n, kv, keep, dim, "f16")
    ka, kp = f32(np.zeros((n, kv, keep))), i32(np.zeros((n, kv, keep)))

    def spaces():
        return [workspace(gpu, m) for m in (
            gpu.attn_window_workspace(r.q, cache.view, window=100, sinks=4), gpu.attn_scored_workspace(r.q, cache.view),
            gpu.attn_prefix_workspace(r.q, prefix.view, cache.view), gpu.kv_evict_workspace(cache.view, keep))]

    def first(ws, stream):
        gpu.attn_window(r.q, cache.view, r.out, ws[0], window=100, sinks=4, lse=r.lse, stream=stream)
        gpu.attn_scored(r.q, cache.view, out2.out, None, acc, ws[1], stream=stream)

    def second(ws, stream):
        gpu.attn_prefix(r.q, prefix.view, cache.view, r.out, ws[2], lse=r.lse, stream=stream)
        gpu.kv_evict(cache.view, acc2, pos, keep, kept.view, ka, kp, ws[3], sinks=4, recent=20, stream=stream)

    def state():
        gpu.lib().lfm_dev_synchronize()
        return [x.download().tobytes() for x in (r.out, r.lse, out2.out, acc, ka, kp, kept.tk, kept.tv, kept.tl)]

    eager_ws = spaces()
    first(eager_ws, 0), second(eager_ws, 0)
    gpu.lib().lfm_dev_synchronize()
    graphs = []
    for fn in (first, second):
        ws = spaces()
        graphs.append((fn, ws, hip.graph(s, lambda: fn(ws, s.value))))
    for turn in range(4):
        cache.tl.buf.upload(rng.integers(0, slots + 1, n).astype(np.int32))
        r.q.buf.upload(rng.standard_normal((n, heads, dim)).astype(np.float32))
        acc2.buf.upload(rng.random((n, kv, slots), dtype=np.float32))
        for fn, ws, e in graphs:
            fn(eager_ws, 0)
            want = state()
            for x in (r.out, r.lse):
                x.buf.upload(np.full(x.buf.nbytes, 0xEE, np.uint8))
            hip.ok("hipGraphLaunch", e, s)
            hip.ok("hipStreamSynchronize", s)
            assert state() == want, (turn, fn.__name__)


def test_two_streams_at_once(gpu):
    hip = Hip()
    rng = np.random.default_rng(15)
    jobs = []
    for i in range(2):
        cache = Cache(rng, [2000, 1500, 900], 2, 2000, 64, "f16")
        r = Rows(gpu, rng, 3, 8, 64, "f16")
        jobs.append((hip.stream(), cache, r, workspace(gpu, gpu.attn_window_workspace(r.q, cache.view))))
    for _ in range(5):
        for s, cache, r, ws in jobs:
            gpu.attn_window(r.q, cache.view, r.out, ws, lse=r.lse, stream=s.value)
    for s, cache, r, ws in jobs:
        hip.ok("hipStreamSynchronize", s)
        out, _, _, extra = U.reference(r.values, cache)
        check_out(r.result(), out, extra, "f16", 64)


def test_bad_pointers_are_refused(gpu):
    rng = np.random.default_rng(16)
    cache = Cache(rng, [9], 2, 9, 64, "f16")
    r = Rows(gpu, rng, 1, 4, 64, "f16")
    ws = workspace(gpu, gpu.attn_scored_workspace(r.q, cache.view))
    L = gpu.lib()
    host = np.zeros(1 << 12)
    good = gpu.Rows.from_buffer_copy(gpu._rows(r.q, cache.view, r.out, None, None, r.lse))

    def rows(**kw):
        x = gpu.Rows.from_buffer_copy(good)
        for k, v in kw.items():
            setattr(x, k, v)
        return x

    def kv(**kw):
        x = gpu.Kv.from_buffer_copy(cache.view._c)
        for k, v in kw.items():
            setattr(x, k, v)
        return x

    def status(k, x, w=ws.ptr, n=ws.nbytes, stream=None):
        return L.lfm_attn_window(C.byref(k), C.byref(x), 0, 0, w, n, stream)

    assert status(kv(), rows()) == 0
    for name in ("q", "out", "lse", "start"):
        assert status(kv(), rows(**{name: host.ctypes.data})) == gpu.LFM_EINVAL, name
        assert b"device memory" in L.lfm_last_error()
    assert status(kv(), rows(q=good.q + 2)) == gpu.LFM_EINVAL
    assert status(kv(), rows(out=good.q)) == gpu.LFM_EINVAL
    assert status(kv(), rows(out=None)) == gpu.LFM_EINVAL
    for name in ("k", "v", "len"):
        assert status(kv(**{name: host.ctypes.data}), rows()) == gpu.LFM_EINVAL, name
        assert status(kv(**{name: None}), rows()) == gpu.LFM_EINVAL, name
    f = C.byref
    for bad in (None, host.ctypes.data):
        assert L.lfm_attn_scored(f(kv()), f(rows()), None, bad, ws.ptr, ws.nbytes, None) == gpu.LFM_EINVAL
    a = f32(np.zeros((1, 2, 9)))
    assert L.lfm_attn_scored(f(kv()), f(rows(lse=None)), None, a.data_ptr(), ws.ptr, 0, None) == gpu.LFM_EINVAL
    assert b"workspace" in L.lfm_last_error()
    assert L.lfm_attn_scored(f(kv()), f(rows(lse=None)), None, a.data_ptr(), host.ctypes.data, host.nbytes,
                             None) == gpu.LFM_EINVAL
    L.lfm_dev_synchronize()
