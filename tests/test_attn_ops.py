"""Refusals of the cache-attention operators: sizes, types and strides are checked before
any device is touched (the pointers here are never dereferenced)."""
import ctypes as C

import numpy as np
import pytest

FAKE = 1 << 20


def kv(lfm, **kw):
    a = dict(k=FAKE, v=2 * FAKE, len=3 * FAKE, seq_stride=8 * 100 * 64, head_stride=100 * 64, slot_stride=64,
             type=lfm.TYPE_F16, n_seq=3, kv_heads=8, slots=100, head_dim=64)
    a.update(kw)
    return lfm.Kv(**a)


def rows(lfm, **kw):
    a = dict(q=4 * FAKE, out=5 * FAKE, q_row_stride=32 * 64, q_head_stride=64, out_row_stride=32 * 64,
             out_head_stride=64, type=lfm.TYPE_F16, heads=32, n_rows=3, scale=0.125)
    a.update(kw)
    return lfm.Rows(**a)


def calls(lfm, k, r, prefix=None):
    """The status of every attention entry point, workspace queries first."""
    L, n = lfm.lib(), C.c_size_t()
    p = kv(lfm, n_seq=1, type=k.type, head_dim=k.head_dim, kv_heads=k.kv_heads) if prefix is None else prefix
    k, r, p = C.byref(k), C.byref(r), C.byref(p)
    return [L.lfm_attn_window_workspace(k, r, 5, 1, C.byref(n)), L.lfm_attn_window(k, r, 5, 1, FAKE, 1 << 40, None),
            L.lfm_attn_scored_workspace(k, r, C.byref(n)), L.lfm_attn_scored(k, r, None, FAKE, FAKE, 1 << 40, None),
            L.lfm_attn_prefix_workspace(p, k, r, C.byref(n)), L.lfm_attn_prefix(p, k, r, FAKE, 1 << 40, None)]


def test_workspace_sizes_without_a_device(lfm):
    L, n = lfm.lib(), C.c_size_t(1 << 50)
    k, r, p = kv(lfm), rows(lfm), kv(lfm, n_seq=1)
    assert L.lfm_attn_window_workspace(C.byref(k), C.byref(r), 0, 0, C.byref(n)) == 0 and n.value < 1 << 30
    assert L.lfm_attn_scored_workspace(C.byref(k), C.byref(r), C.byref(n)) == 0 and 0 < n.value < 1 << 30
    assert L.lfm_attn_prefix_workspace(C.byref(p), C.byref(k), C.byref(r), C.byref(n)) == 0
    assert L.lfm_kv_evict_workspace(C.byref(k), 50, C.byref(n)) == 0 and 3 * 8 * 50 * 8 <= n.value < 1 << 20
    assert L.lfm_kv_evict_workspace(C.byref(k), 50, None) == lfm.LFM_EINVAL


@pytest.mark.parametrize("change", [
    dict(type=0), dict(type=3), dict(head_dim=0), dict(head_dim=96), dict(head_dim=256), dict(kv_heads=0),
    dict(kv_heads=7), dict(slots=0), dict(slots=1 << 31), dict(seq_stride=-8), dict(slot_stride=60),
    dict(head_stride=4), dict(n_seq=4), dict(n_seq=70000)], ids=str)
def test_bad_caches(lfm, change):
    assert set(calls(lfm, kv(lfm, **change), rows(lfm), kv(lfm, n_seq=1))) == {lfm.LFM_EINVAL}
    assert lfm.lib().lfm_last_error()


@pytest.mark.parametrize("change", [
    dict(type=2), dict(type=3), dict(heads=0), dict(heads=33), dict(heads=80000), dict(n_rows=2),
    dict(n_rows=1 << 31, start=FAKE), dict(n_rows=1 << 19, start=FAKE), dict(heads=8 * 129), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(q_row_stride=-64), dict(q_head_stride=4), dict(out_row_stride=63),
    dict(out_row_stride=0), dict(out_head_stride=0)], ids=str)
def test_bad_rows(lfm, change):
    assert set(calls(lfm, kv(lfm), rows(lfm, **change))) == {lfm.LFM_EINVAL}
    assert lfm.lib().lfm_last_error()


def test_bf16_and_f32_rows_pair_with_their_caches(lfm):
    assert set(calls(lfm, kv(lfm, type=lfm.TYPE_BF16), rows(lfm, type=lfm.TYPE_F32))) == {lfm.LFM_EINVAL}
    assert set(calls(lfm, kv(lfm, type=lfm.TYPE_BF16), rows(lfm))) == {lfm.LFM_EINVAL}
    # strides of F32 rows go by 4 elements, those of 16-bit ones by 8
    n = C.c_size_t()
    q = rows(lfm, type=lfm.TYPE_F32, q_head_stride=68)
    assert lfm.lib().lfm_attn_window_workspace(C.byref(kv(lfm)), C.byref(q), 0, 0, C.byref(n)) == 0


def test_null_structs(lfm):
    L, n = lfm.lib(), C.c_size_t()
    k, r = C.byref(kv(lfm)), C.byref(rows(lfm))
    assert L.lfm_attn_window_workspace(None, r, 0, 0, C.byref(n)) == lfm.LFM_EINVAL
    assert L.lfm_attn_window_workspace(k, None, 0, 0, C.byref(n)) == lfm.LFM_EINVAL
    assert L.lfm_attn_window_workspace(k, r, 0, 0, None) == lfm.LFM_EINVAL
    assert L.lfm_attn_prefix(None, k, r, FAKE, 1 << 40, None) == lfm.LFM_EINVAL


@pytest.mark.parametrize("change", [dict(n_seq=2), dict(n_seq=0), dict(kv_heads=4), dict(head_dim=128),
                                    dict(type=2)], ids=str)
def test_prefix_pairs_with_the_cache(lfm, change):
    p = kv(lfm, **dict(dict(n_seq=1), **change))
    assert calls(lfm, kv(lfm), rows(lfm), p)[4:] == [lfm.LFM_EINVAL] * 2


@pytest.mark.parametrize("out, keep, sinks, recent", [
    (dict(), 101, 0, 0),                                            # more than out holds
    (dict(), 0, 0, 0), (dict(), 50, 30, 21), (dict(), 50, 0xFFFFFFFF, 1), (dict(n_seq=2), 50, 0, 0),
    (dict(kv_heads=4), 50, 0, 0), (dict(head_dim=128), 50, 0, 0), (dict(type=2), 50, 0, 0),
    (dict(slots=49), 50, 0, 0), (dict(slot_stride=0), 50, 0, 0), (dict(head_stride=0), 50, 0, 0),
    (dict(k=FAKE), 50, 0, 0),                                       # k in place, v not
    (dict(k=FAKE, v=2 * FAKE, slot_stride=72), 50, 0, 0)], ids=str)
def test_bad_evictions(lfm, out, keep, sinks, recent):
    o = kv(lfm, **dict(dict(k=6 * FAKE, v=7 * FAKE, len=8 * FAKE), **out))
    c, f = kv(lfm), FAKE
    L = lfm.lib()
    assert L.lfm_kv_evict(C.byref(c), f, f, keep, sinks, recent, C.byref(o), 9 * f, 9 * f, f, 1 << 40,
                          None) == lfm.LFM_EINVAL
    assert L.lfm_last_error()


def test_grids_that_cannot_be_launched_are_refused(lfm):
    n = C.c_size_t()
    k = kv(lfm, slots=0x7FFFFF00, kv_heads=8)
    r = rows(lfm, start=FAKE)
    assert lfm.lib().lfm_attn_scored_workspace(C.byref(k), C.byref(r), C.byref(n)) == lfm.LFM_EINVAL
    assert lfm.lib().lfm_attn_window_workspace(C.byref(k), C.byref(r), 0, 0, C.byref(n)) == 0
    assert lfm.lib().lfm_kv_evict_workspace(C.byref(k), (1 << 28) + 1, C.byref(n)) == lfm.LFM_EINVAL


def test_acc_in_place_needs_equal_slots(lfm):
    c, o = kv(lfm), kv(lfm, k=6 * FAKE, v=7 * FAKE, slots=80)
    L = lfm.lib()
    for acc, pos in ((FAKE, 9 * FAKE), (9 * FAKE, 2 * FAKE)):
        assert L.lfm_kv_evict(C.byref(c), FAKE, 2 * FAKE, 50, 0, 0, C.byref(o), acc, pos, FAKE, 1 << 40,
                              None) == lfm.LFM_EINVAL


class Host:
    """Stands for a device tensor: shape, strides and type without memory."""

    def __init__(self, shape, dtype="torch.float16", strides=None):
        self.shape, self.dtype, self.st = tuple(shape), dtype, strides

    def stride(self):
        if self.st:
            return self.st
        return tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))

    def data_ptr(self):
        return FAKE

    def numel(self):
        return int(np.prod(self.shape))

    def element_size(self):
        return 2


def test_binding_checks_shapes_and_types(lfm):
    length = Host((3,), "torch.int32")
    k = Host((3, 8, 100, 64))
    cache = lfm.KvCache(k, k, length)
    q = Host((3, 32, 64))
    assert lfm.attn_window_workspace(q, cache) >= 0
    bad = [lambda: lfm.KvCache(k, Host((3, 8, 99, 64)), length), lambda: lfm.KvCache(k, k, Host((4,), "torch.int32")),
           lambda: lfm.KvCache(k, k, Host((3,), "torch.int64")),
           lambda: lfm.KvCache(Host(k.shape, "torch.float32"), Host(k.shape, "torch.float32"), length),
           lambda: lfm.KvCache(Host(k.shape, strides=(1, 64 * 100, 64, 2)), k, length),
           lambda: lfm.KvCache(Host(k.shape, strides=(8 * 64 * 100, 64 * 100, 2 * 64, 1)), k, length),
           lambda: lfm.attn_window_workspace(Host((3, 32, 128)), cache),
           lambda: lfm.attn_window_workspace(Host((3, 64)), cache),
           lambda: lfm.attn_window_workspace(Host((4, 32, 64)), cache),
           lambda: lfm.attn_window_workspace(Host((3, 32, 64), "torch.float64"), cache),
           lambda: lfm.attn_window_workspace(Host((3, 32, 64), strides=(64 * 32, 1, 32)), cache),
           lambda: lfm.attn_window_workspace(q, cache, start=Host((3,), "torch.int32")),
           lambda: lfm.attn_window(q, cache, Host((3, 32, 64), "torch.float32"), Host((1,))),
           lambda: lfm.attn_window(q, cache, q, Host((1,)), lse=Host((3, 31), "torch.float32")),
           lambda: lfm.attn_scored(q, cache, q, None, Host((3, 8, 99), "torch.float32"), Host((1,)))]
    for call in bad:
        with pytest.raises(lfm.LfmError) as e:
            call()
        assert e.value.code == lfm.LFM_EINVAL
