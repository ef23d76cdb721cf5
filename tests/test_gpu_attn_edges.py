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


# ------------------------------------------------------------------ rows of many tokens in key ranges
@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f16", 64), ("bf16", 64), ("f32", 128), ("f16", 128), ("bf16", 128)])
def test_scored_chunks_in_ranges(gpu, kind, dim):
    """Few rows over more than 1024 slots: their states come from joined key ranges."""
    rng = np.random.default_rng([dim, 33])
    cache = Cache(rng, [2203, 1, 1025, 40, 0], 2, 2207, dim, "bf16" if kind == "bf16" else "f16", "slot")
    start = np.concatenate([[1], 1 + np.cumsum([37, 1, 3, 45, 2])])
    r = Rows(gpu, rng, int(start[-1]) + 2, 6, dim, kind)
    tight_scored(gpu, r, cache, start, acc_in=rng.random((5, 2, 2207), dtype=np.float32))
    assert r.untouched([0, -1, -2])


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f16", 64), ("bf16", 128)])
def test_scored_prompt_in_parts_and_ranges(gpu, kind, dim):
    """A prompt whose weights are added in 16 parts, its rows in three key ranges."""
    rng = np.random.default_rng([dim, 34])
    cache = Cache(rng, [2100], 1, 2101, dim, "bf16" if kind == "bf16" else "f16")
    r = Rows(gpu, rng, 2060, 4, dim, kind)
    a = tight_scored(gpu, r, cache, [0, 2060])
    assert np.array_equal(a, tight_scored(gpu, r, cache, [0, 2060]))


@pytest.mark.parametrize("kind, dim", [("f16", 64), ("bf16", 128)])
def test_scored_many_prompts_slot_by_slot(gpu, kind, dim):
    """The larger tiles over many short sequences: what one slot receives from its sequence's
    rows, each of which weighs far more than the bound."""
    rng = np.random.default_rng([dim, 35])
    counts = rng.integers(40, 80, 68 if dim == 64 else 50)
    start = np.concatenate([[0], np.cumsum(counts)])
    cache = Cache(rng, counts + rng.integers(-20, 40, len(counts)), 8, 120, dim, kind)
    tight_scored(gpu, Rows(gpu, rng, int(start[-1]), 24, dim, kind), cache, start)


@pytest.mark.parametrize("group", [1, 7, 16, 17, 50, 128])
def test_scored_groups(gpu, group):
    rng = np.random.default_rng([group, 36])
    cache = Cache(rng, [90, 300, 5], 2, 301, 64, "f16")
    tight_scored(gpu, Rows(gpu, rng, 3, 2 * group, 64, "f16"), cache)
    tight_scored(gpu, Rows(gpu, rng, 24, 2 * group, 64, "f32"), cache, [0, 13, 19, 24])


def check_seen(got, want, extra, kind, dim, rows, slots_nan, dims=3):
    """got of rows: no number in the first dims where a row sees one of slots_nan, else the
    formula's."""
    out, size, reach, seen = want.copy(), *(x.copy() for x in extra)
    hit = np.zeros(got.shape[0], bool)
    for row, see in rows:
        hit[row] = any(see(j) for j in slots_nan)
    listed = np.array([row for row, _ in rows])
    assert hit[listed].any() and not hit[listed].all()
    expected = hit[:, None, None] & (np.arange(dim) < dims) & np.ones(got.shape, bool)
    assert np.array_equal(np.isnan(out)[listed], expected[listed])  # the formula's NaN are these
    assert np.array_equal(np.isnan(got)[listed], expected[listed])
    tol = U.out_tolerance(np.nan_to_num(out), tuple(np.nan_to_num(x) for x in (size, reach, seen)), kind, dim)
    bad = ~(np.abs(got - out) <= tol) & ~expected
    assert not bad[listed].any(), (np.argwhere(bad)[:5], got[bad][:5], out[bad][:5], tol[bad][:5])


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f16", 64), ("bf16", 64), ("f32", 128), ("f16", 128), ("bf16", 128)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (300, 4)])
def test_masked_nan_in_ranges(gpu, kind, dim, window, sinks):
    """V is no number in slots that some rows of a chunk see and others do not, over more than
    1024 slots: those rows' partial outputs come from the rows computed one by one."""
    rng = np.random.default_rng([dim, window, 37])
    length, counts, heads = [2000, 1300, 1100], [40, 25, 30], 3
    odd = {0: [1975], 1: [1290]}
    if window:  # and one that the window of later rows has passed
        odd[0].append(1672), odd[1].append(981)

    def edit(k, v):
        for b, js in odd.items():
            v[b, :, js, :3] = np.nan

    cache = Cache(rng, length, 1, 2003, dim, "bf16" if kind == "bf16" else "f16", "slot", edit)
    start = np.concatenate([[0], np.cumsum(counts)])
    r = Rows(gpu, rng, int(start[-1]), heads, dim, kind)
    check = []
    for b in odd:
        for row in range(start[b], start[b + 1]):
            p = length[b] - int(start[b + 1]) + row
            check.append((row, lambda j, p=p, b=b: j in odd[b] and j <= p and (
                not window or j < sinks or j > p - window)))
    ws = workspace(gpu, gpu.attn_window_workspace(r.q, cache.view, window=window, sinks=sinks, start=i32(start)))
    gpu.attn_window(r.q, cache.view, r.out, ws, window=window, sinks=sinks, start=i32(start), lse=r.lse)
    with np.errstate(invalid="ignore"):
        out, lse, _, extra = U.reference(r.values, cache, start, window, sinks)
    js = sorted({j for b in odd for j in odd[b]})
    check_seen(r.result(), out, extra, kind, dim, check, js)
    rest = slice(start[2], start[3])
    check_out(r.result()[rest], out[rest], tuple(x[rest] for x in extra), kind, dim)
    assert (np.abs(r.lse.download().reshape(lse.shape) - lse) <= U.lse_tolerance(lse, extra, dim)).all()
    if window:
        return
    # the same scored: what slots receive has nothing to do with V
    nan = np.zeros(r.shape[:2], bool)
    for row, see in check:
        nan[row] = any(see(j) for j in js)
    tight_scored(gpu, r, cache, start, nan_rows=nan)
    check_seen(r.result(), out, extra, kind, dim, check, js)


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f16", 64), ("bf16", 64), ("f32", 128), ("f16", 128), ("bf16", 128)])
@pytest.mark.parametrize("slots", [200, 1300])
def test_masked_nan_behind_a_prefix(gpu, kind, dim, slots):
    """The same for own slots behind a shared prefix, in one range of their own and in several."""
    rng = np.random.default_rng([dim, slots, 38])
    cached = "bf16" if kind == "bf16" else "f16"
    length, counts, heads = [slots, slots - 40], [40, 25], 3
    odd = [slots - 20, slots - 50]

    def edit(k, v):
        v[0, :, odd[0], :3] = v[1, :, odd[1], :3] = np.nan

    prefix = Cache(rng, [600], 2, 610, dim, cached)
    cache = Cache(rng, length, 2, slots + 3, dim, cached, "head", edit)
    start = np.concatenate([[0], np.cumsum(counts)])
    r = Rows(gpu, rng, int(start[-1]), 2 * heads, dim, kind)
    ws = workspace(gpu, gpu.attn_prefix_workspace(r.q, prefix.view, cache.view, start=i32(start)))
    gpu.attn_prefix(r.q, prefix.view, cache.view, r.out, ws, start=i32(start), lse=r.lse)
    with np.errstate(invalid="ignore"):
        out, lse, _, extra = U.reference(r.values, cache, start, prefix=prefix)
    check = []
    for b in range(2):
        for row in range(start[b], start[b + 1]):
            p = length[b] - int(start[b + 1]) + row
            check.append((row, lambda j, p=p, b=b: j == odd[b] and j <= p))
    check_seen(r.result(), out, extra, kind, dim, check, odd)
    assert (np.abs(r.lse.download().reshape(lse.shape) - lse) <= U.lse_tolerance(lse, extra, dim)).all()


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("bf16", 128)])
def test_masked_infinite_keys_in_ranges(gpu, kind, dim):
    """K is no number or infinite in a slot that later rows of a chunk see: earlier ones do not
    take part."""
    rng = np.random.default_rng([dim, 39])

    def edit(k, v):
        k[0, :, 1980] = np.nan
        k[0, :, 1990] = np.inf

    cache = Cache(rng, [2000], 1, 2003, dim, "bf16" if kind == "bf16" else "f16", "slot", edit)
    r = Rows(gpu, rng, 40, 3, dim, kind)
    ws = workspace(gpu, gpu.attn_window_workspace(r.q, cache.view, start=i32([0, 40])))
    gpu.attn_window(r.q, cache.view, r.out, ws, start=i32([0, 40]), lse=r.lse)
    got = r.result()
    assert np.isnan(got[20:]).all() and np.isfinite(got[:20]).all()
    sane = Cache(np.random.default_rng([dim, 39]), [1980], 1, 2003, dim, "bf16" if kind == "bf16" else "f16", "slot")
    out, lse, _, extra = U.reference(r.values[:20], sane, [0, 20])
    check_out(got[:20], out, extra, kind, dim)
    z = r.lse.download().reshape(40, 3)[:20]
    assert (np.abs(z - lse) <= U.lse_tolerance(lse, extra, dim)).all()


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f16", 128), ("bf16", 64)])
def test_equal_calls_give_equal_bits(gpu, kind, dim):
    rng = np.random.default_rng([dim, 40])
    cached = "bf16" if kind == "bf16" else "f16"
    cache = Cache(rng, [2500, 700], 2, 2500, dim, cached)
    prefix = Cache(rng, [3001], 2, 3001, dim, cached)
    for n, start in ((2, None), (900, [0, 600, 900])):
        r = Rows(gpu, rng, n, 8, dim, kind)
        st = None if start is None else i32(start)
        acc = f32(np.zeros((2, 2, 2500)))
        for call in (lambda ws: gpu.attn_window(r.q, cache.view, r.out, ws, window=900, sinks=3, start=st, lse=r.lse),
                     lambda ws: gpu.attn_scored(r.q, cache.view, r.out, None, acc, ws, start=st, lse=r.lse),
                     lambda ws: gpu.attn_prefix(r.q, prefix.view, cache.view, r.out, ws, start=st, lse=r.lse)):
            bits = []
            for fill in (0xFF, 0x00, 0x3C):  # whatever the workspace held
                ws = workspace(gpu, 1 << 26, fill)
                call(ws)
                bits.append([x.download().tobytes() for x in (r.out, r.lse, acc)])
            assert bits[0] == bits[1] == bits[2]


# ------------------------------------------------------------------ what else the calls allow
@pytest.mark.parametrize("kind, dim", [("f32", 64), ("bf16", 128)])
def test_one_cache_shared_by_all_sequences(gpu, kind, dim):
    """A sequence stride of 0, and a head stride of 0 (one kv head for several)."""
    rng = np.random.default_rng([dim, 50])
    cached = "bf16" if kind == "bf16" else "f16"
    one = Cache(rng, [1], 1, 901, dim, cached)
    cache = Cache(rng, [900, 3, 0, 77], 2, 901, dim, cached)
    cache.k, cache.v = (np.broadcast_to(x, cache.k.shape) for x in (one.k, one.v))
    cache.view = gpu.KvCache(*(gpu.DeviceTensor(x.buf, cache.k.shape, x.dtype, 0, (0, 0, dim, 1))
                               for x in (one.tk, one.tv)), cache.tl)
    check_window(gpu, Rows(gpu, rng, 4, 6, dim, kind), cache, None, 90, 2)
    check_window(gpu, Rows(gpu, rng, 50, 6, dim, kind), cache, [0, 30, 33, 40, 50], 90, 2)
    tight_scored(gpu, Rows(gpu, rng, 4, 6, dim, kind), cache)
    tight_scored(gpu, Rows(gpu, rng, 50, 6, dim, kind), cache, [0, 30, 33, 40, 50])


@pytest.mark.parametrize("kind, dim", [("f32", 128), ("f16", 64)])
def test_one_query_for_all_rows_and_heads(gpu, kind, dim):
    rng = np.random.default_rng([dim, 51])
    cache = Cache(rng, [90, 7, 41], 2, 101, dim, "f16")
    for n, start in ((3, None), (60, [0, 30, 37, 60])):
        r = Rows(gpu, rng, n, 6, dim, kind)
        r.values[:] = r.values[0, 0]
        r.q = gpu.DeviceTensor(r.q.buf, r.shape, r.q.dtype, 0, (0, 0, 1))
        check_window(gpu, r, cache, start, 30, 3)
        tight_scored(gpu, r, cache, start)


class Space:
    """A workspace of exactly n bytes with a guard behind it."""

    def __init__(self, gpu, n):
        self.n, self.buf = n, gpu.DeviceBuffer.from_array(np.full(n + 4096, 0x5A, np.uint8))

    def data_ptr(self):
        return self.buf.ptr

    def numel(self):
        return self.n

    def element_size(self):
        return 1

    def intact(self):
        return (self.buf.download(np.uint8)[self.n:] == 0x5A).all()


@pytest.mark.parametrize("heads, kv, dim, kind", [(6, 2, 64, "f32"), (34, 2, 64, "f16"), (9, 3, 128, "bf16"),
                                                  (128, 1, 128, "f32")])
def test_workspaces_are_large_enough(gpu, heads, kv, dim, kind):
    rng = np.random.default_rng([heads, dim, 52])
    cached = "bf16" if kind == "bf16" else "f16"
    cache = Cache(rng, [1499, 700, 1033], kv, 1499, dim, cached)
    prefix = Cache(rng, [2300], kv, 2300, dim, cached)
    for n, start in ((3, None), (70, [0, 30, 30, 70]), (1100, [0, 700, 1000, 1100])):
        r = Rows(gpu, rng, n, heads, dim, kind)
        st = None if start is None else i32(start)
        acc = f32(np.zeros((3, kv, 1499)))
        ws = [Space(gpu, x) for x in (gpu.attn_window_workspace(r.q, cache.view, start=st),
                                      gpu.attn_window_workspace(r.q, cache.view, window=1100, sinks=3, start=st),
                                      gpu.attn_scored_workspace(r.q, cache.view, start=st),
                                      gpu.attn_prefix_workspace(r.q, prefix.view, cache.view, start=st))]
        gpu.attn_window(r.q, cache.view, r.out, ws[0], start=st)
        gpu.attn_window(r.q, cache.view, r.out, ws[1], window=1100, sinks=3, start=st)
        gpu.attn_scored(r.q, cache.view, r.out, None, acc, ws[2], start=st)
        gpu.attn_prefix(r.q, prefix.view, cache.view, r.out, ws[3], start=st)
        assert all(w.intact() for w in ws), n
    for keep in (1, 77, 1499):
        w = Space(gpu, gpu.kv_evict_workspace(cache.view, keep))
        pos = i32(np.tile(np.arange(1499), (3, kv, 1)))
        cache.tl.buf.upload(np.array([1499, 700, 1033], np.int32))
        gpu.kv_evict(cache.view, acc, pos, keep, cache.view, acc, pos, w)
        assert w.intact()


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_bad_row_stays_alone(gpu, kind, dim, bad):
    """Queries that are no numbers, between others: the rest are the formula's."""
    rng = np.random.default_rng([dim, 53])
    cached = "bf16" if kind == "bf16" else "f16"
    cache = Cache(rng, [90, 700, 41], 2, 701, dim, cached)
    prefix = Cache(rng, [130], 2, 131, dim, cached)
    for n, start in ((3, None), (100, [0, 40, 60, 100])):
        r = Rows(gpu, rng, n, 6, dim, kind)
        r.values[1, 2, 5] = r.values[1, 3] = bad
        r.q = U.tensor(r.values, kind)[0]
        st = None if start is None else i32(start)
        rest = np.ones((n, 6), bool)
        rest[1, 2:4] = False
        for pre in (None, prefix):
            if pre is None:
                ws = workspace(gpu, gpu.attn_window_workspace(r.q, cache.view, start=st))
                gpu.attn_window(r.q, cache.view, r.out, ws, start=st)
            else:
                ws = workspace(gpu, gpu.attn_prefix_workspace(r.q, pre.view, cache.view, start=st))
                gpu.attn_prefix(r.q, pre.view, cache.view, r.out, ws, start=st)
            with np.errstate(invalid="ignore"):
                out, _, _, extra = U.reference(r.values, cache, start, prefix=pre)
            got = r.result()
            assert np.isnan(got[~rest]).all()
            check_out(got[rest], out[rest], tuple(x[rest] for x in extra), kind, dim)
        acc = f32(np.zeros((3, 2, 701)))
        ws = workspace(gpu, gpu.attn_scored_workspace(r.q, cache.view, start=st))
        gpu.attn_scored(r.q, cache.view, r.out, None, acc, ws, start=st)
        a = acc.download().reshape(3, 2, 701)
        b, p = (1, 699) if start is None else (0, 90 - 40 + 1)  # the bad row's sequence and position
        used = np.arange(701) < cache.length[:, None]
        nan = np.zeros(a.shape, bool)
        nan[b, :, :p + 1] = True  # heads 2 and 3 are of kv heads 0 and 1
        assert np.array_equal(np.isnan(a), nan & used[:, None])


def test_captured_prompts_follow_their_starts(gpu):
    """Graphs of ragged calls: lengths, starts and rows change between replays, and eager calls
    of the same run between them."""
    from test_gpu_attn import Hip
    hip = Hip()
    rng = np.random.default_rng(54)
    cache = Cache(rng, [1400, 900, 2], 2, 1400, 64, "f16")
    prefix = Cache(rng, [700], 2, 700, 64, "f16")
    n, heads = 90, 6
    st = i32([0, 50, 80, 90])
    outs = [Rows(gpu, rng, n, heads, 64, "f32") for _ in range(3)]
    q = outs[0].q
    acc = f32(np.zeros((3, 2, 1400)))

    def spaces():
        return [workspace(gpu, m) for m in (gpu.attn_window_workspace(q, cache.view, window=1200, sinks=4, start=st),
                                            gpu.attn_scored_workspace(q, cache.view, start=st),
                                            gpu.attn_prefix_workspace(q, prefix.view, cache.view, start=st))]

    def calls(ws, stream):
        gpu.attn_window(q, cache.view, outs[0].out, ws[0], window=1200, sinks=4, start=st, lse=outs[0].lse, stream=stream)
        gpu.attn_scored(q, cache.view, outs[1].out, acc, acc, ws[1], start=st, stream=stream)
        gpu.attn_prefix(q, prefix.view, cache.view, outs[2].out, ws[2], start=st, stream=stream)

    def clear():
        for x in (outs[0].out, outs[1].out, outs[2].out, outs[0].lse, acc):
            x.buf.upload(np.zeros(x.buf.nbytes, np.uint8))

    def state():
        gpu.lib().lfm_dev_synchronize()
        return [x.download().tobytes() for x in (outs[0].out, outs[1].out, outs[2].out, outs[0].lse, acc)]

    eager, own = spaces(), spaces()
    calls(eager, 0)
    gpu.lib().lfm_dev_synchronize()
    s = hip.stream()
    graph = hip.graph(s, lambda: calls(own, s.value))
    for turn in range(5):
        cuts = np.sort(rng.integers(0, n + 1, 2))
        st.buf.upload(np.array([0, *cuts, n] if turn % 2 else [3, *np.maximum(cuts, 3), n], np.int32))
        cache.tl.buf.upload(rng.integers(0, 1401, 3).astype(np.int32))
        q.buf.upload(rng.standard_normal((n, heads, 64)).astype(np.float32))
        clear()
        calls(eager, 0)
        want = state()
        clear()
        hip.ok("hipGraphLaunch", graph, s)
        hip.ok("hipStreamSynchronize", s)
        assert state() == want, turn


@pytest.mark.parametrize("place", ["acc", "pos", "both"])
def test_evict_apart_with_acc_or_pos_in_place(gpu, place):
    rng = np.random.default_rng(55)
    n, kv, slots, keep, dim = 3, 2, 400, 150, 64
    length = [400, 151, 90]
    cache, out = Cache(rng, length, kv, slots, dim, "f16"), Cache(rng, [0] * n, kv, slots, dim, "f16", "slot")
    acc = rng.random((n, kv, slots), dtype=np.float32)
    pos = np.cumsum(rng.integers(1, 4, acc.shape), -1).astype(np.int32)
    ta, tp, oa, op = f32(acc), i32(pos), f32(np.full(acc.shape, 9.0)), i32(np.full(acc.shape, 9))
    da, dp = ta if place != "pos" else oa, tp if place != "acc" else op
    want_a, want_p = (acc.copy() if place != "pos" else np.full_like(acc, 9)), (pos.copy() if place != "acc" else np.full_like(pos, 9))
    ws = workspace(gpu, gpu.kv_evict_workspace(cache.view, keep))
    gpu.kv_evict(cache.view, ta, tp, keep, out.view, da, dp, ws, sinks=5, recent=30)
    from test_gpu_attn import read_cache
    got = read_cache(out.view, "f16", "slot")
    for b in range(n):
        for h in range(kv):
            s = U.keep_slots(acc[b, h], pos[b, h], length[b], keep, 5, 30)
            s = np.arange(length[b]) if s is None else s
            want_a[b, h, :len(s)], want_p[b, h, :len(s)] = acc[b, h][s], pos[b, h][s]
            for x, w in zip(got, (cache.k, cache.v)):
                assert np.array_equal(x[b, h, :len(s)], w[b, h][s])
    assert np.array_equal(da.download().reshape(acc.shape), want_a)
    assert np.array_equal(dp.download().reshape(acc.shape), want_p)
    assert np.array_equal(out.tl.download(), [150, 150, 90])


def test_evict_positions_at_the_ends_of_32_bits(gpu):
    """Positions that are negative, the largest and the smallest; keep larger than the cache."""
    rng = np.random.default_rng(56)
    n, kv, slots, dim = 4, 1, 130, 64
    acc = rng.random((n, kv, slots), dtype=np.float32)
    pos = rng.integers(-(1 << 31), 1 << 31, (n, kv, slots)).astype(np.int32)
    pos[0, 0, 7], pos[0, 0, 9] = (1 << 31) - 1, -(1 << 31)
    pos[1] = np.abs(pos[1])
    pos[2] = -1 - np.abs(pos[2] // 2)
    pos[3] = np.arange(slots)
    length = [slots] * n
    for keep, sinks, recent in ((60, 0, 60), (60, 60, 0), (60, 7, 9), (1, 0, 1), (500, 3, 400)):
        cache = Cache(rng, length, kv, slots, dim, "f16")
        out = Cache(rng, [0] * n, kv, 501, dim, "f16")
        oa, op = f32(np.zeros((n, kv, 501))), i32(np.zeros((n, kv, 501)))
        ws = workspace(gpu, gpu.kv_evict_workspace(cache.view, keep))
        gpu.kv_evict(cache.view, f32(acc), i32(pos), keep, out.view, oa, op, ws, sinks=sinks, recent=recent)
        p = op.download().reshape(n, kv, 501)
        for b in range(n):
            s = U.keep_slots(acc[b, 0], pos[b, 0], slots, keep, sinks, recent)
            s = np.arange(slots) if s is None else s
            assert np.array_equal(p[b, 0, :len(s)], pos[b, 0][s]), (b, keep, sinks, recent)
        assert np.array_equal(out.tl.download(), [min(slots, keep)] * n)


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("bf16", 128)])
def test_window_of_chunks_in_ranges(gpu, kind, dim):
    rng = np.random.default_rng([dim, 57])
    cache = Cache(rng, [2400, 1300, 40], 2, 2407, dim, "bf16" if kind == "bf16" else "f16", "mixed")
    r = Rows(gpu, rng, 90, 6, dim, kind)
    for window, sinks in ((1500, 0), (1100, 70), (2300, 2000)):
        check_window(gpu, r, cache, [0, 40, 75, 90], window, sinks)


@pytest.mark.parametrize("kind, dim", [("f32", 64), ("f16", 64), ("f16", 128)])
@pytest.mark.parametrize("size", [65504.0, 60000.0, 3e-5, 6e-8])
def test_values_at_the_ends_of_binary16(gpu, kind, dim, size):
    """V of one size, the largest number and subnormal ones among them: the outputs are that size
    and no infinity, in every kernel that writes some."""
    rng = np.random.default_rng([dim, 60])

    def edit(k, v):
        v[:] = np.where(rng.random(v.shape[:2] + (1, v.shape[3])) < 0.5, size, -size)

    cache = Cache(rng, [1900, 45, 301], 2, 1900, dim, "f16", edit=edit)
    prefix = Cache(rng, [700], 2, 700, dim, "f16")
    prefix.v[:] = cache.v[:1, :, :1]
    prefix.tv.buf.upload(np.broadcast_to(prefix.v, prefix.k.shape).astype(np.float16))
    cache.v[1:] = cache.v[:1]
    cache.tv.buf.upload(cache.v.astype(np.float16))
    want = np.repeat(cache.v[0, :, 0], 3, axis=0)  # [heads][dim], every row's
    for n, start in ((3, None), (100, [0, 40, 70, 100])):
        r = Rows(gpu, rng, n, 6, dim, kind)
        st = None if start is None else i32(start)
        acc = f32(np.zeros((3, 2, 1900)))
        for call in (lambda: gpu.attn_window(r.q, cache.view, r.out, ws, start=st),
                     lambda: gpu.attn_window(r.q, cache.view, r.out, ws, window=40, start=st),
                     lambda: gpu.attn_scored(r.q, cache.view, r.out, None, acc, ws, start=st),
                     lambda: gpu.attn_prefix(r.q, prefix.view, cache.view, r.out, ws, start=st)):
            ws = workspace(gpu, 1 << 25)
            call()
            # |sum w v| is |v| but for the weights' rounding; the output's own (of a subnormal an absolute one)
            rel = U.WEIGHT[kind] + 2.0 ** -20 + 2 * (2600 + 16) * 2.0 ** -24
            tol = rel * np.abs(want) + 1.01 * (U.HALF[kind] * np.abs(want) + (2.0 ** -25 if kind == "f16" else 2.0 ** -149))
            got = r.result()
            bad = ~(np.abs(got - want) <= tol)
            assert not bad.any(), (n, int(bad.sum()), got[bad][:5], np.broadcast_to(want, got.shape)[bad][:5])


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_keys_that_are_subnormal(gpu, kind):
    rng = np.random.default_rng(61)

    def edit(k, v):
        k *= 1e-6

    cache = Cache(rng, [190, 45, 3], 2, 190, 64, "f16", edit=edit)
    for n, start in ((3, None), (100, [0, 67, 97, 100])):
        r = Rows(gpu, rng, n, 6, 64, kind)
        check_window(gpu, r, cache, start, 60, 3, scale=1e5)
        tight_scored(gpu, r, cache, start, scale=1e5)
