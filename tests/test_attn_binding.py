"""The Python binding of the cache-attention operators, without a device."""
import numpy as np
import pytest

from test_attn_ops import Host


class OnGpu(Host):
    """Stands for a torch tensor on a device."""
    is_cuda = True

    def get_device(self):
        return 0


def test_binding_takes_torchs_current_stream(lfm, monkeypatch):
    """Without a stream, calls on torch tensors go to torch's current stream, where those are
    made; calls on others to the default stream; a stream that is given is taken as it is."""
    calls, devices = [], []

    class Library:
        def __getattr__(self, name):
            return lambda *args: calls.append((name, args[-1])) or 0

    monkeypatch.setattr(lfm, "lib", Library)
    monkeypatch.setattr(lfm, "_torch_stream", lambda index: devices.append(index) or 4711)
    for tensor, given, want in ((OnGpu, None, 4711), (OnGpu, 0, 0), (OnGpu, 99, 99), (Host, None, 0), (Host, 99, 99)):
        kw = {} if given is None else {"stream": given}
        k, ws = tensor((3, 8, 100, 64)), tensor((1 << 20,))
        cache = lfm.KvCache(k, k, tensor((3,), "torch.int32"))
        prefix = lfm.KvCache(tensor((1, 8, 100, 64)), tensor((1, 8, 100, 64)), tensor((1,), "torch.int32"))
        q, acc = tensor((3, 32, 64)), tensor((3, 8, 100), "torch.float32")
        pos = tensor((3, 8, 100), "torch.int32")
        del calls[:]
        lfm.attn_window(q, cache, q, ws, window=5, **kw)
        lfm.attn_scored(q, cache, q, None, acc, ws, **kw)
        lfm.attn_prefix(q, prefix, cache, q, ws, **kw)
        lfm.kv_evict(cache, acc, pos, 50, cache, acc, pos, ws, **kw)
        assert calls == [(n, want) for n in ("lfm_attn_window", "lfm_attn_scored", "lfm_attn_prefix", "lfm_kv_evict")]
    assert set(devices) == {0}


def test_binding_refuses_numbers_past_32_bits(lfm):
    """ctypes would take their low 32 bits: window -1 as a large one, keep 2^32 + 50 as 50."""
    k, ws = Host((3, 8, 100, 64)), Host((1 << 20,))
    cache = lfm.KvCache(k, k, Host((3,), "torch.int32"))
    q, acc, pos = Host((3, 32, 64)), Host((3, 8, 100), "torch.float32"), Host((3, 8, 100), "torch.int32")

    def evict(**kw):
        a = dict(keep=50, sinks=0, recent=0)
        a.update(kw)
        lfm.kv_evict(cache, acc, pos, a.pop("keep"), cache, acc, pos, ws, **a)

    for bad in (-1, 1 << 32, (1 << 32) + 50, 3.0, None):
        for call in (lambda: lfm.attn_window_workspace(q, cache, window=bad),
                     lambda: lfm.attn_window_workspace(q, cache, sinks=bad),
                     lambda: lfm.attn_window(q, cache, q, ws, window=bad), lambda: lfm.attn_window(q, cache, q, ws, sinks=bad),
                     lambda: lfm.kv_evict_workspace(cache, bad), lambda: evict(keep=bad), lambda: evict(sinks=bad),
                     lambda: evict(recent=bad)):
            with pytest.raises(lfm.LfmError) as e:
                call()
            assert e.value.code == lfm.LFM_EINVAL and "32 bits" in str(e.value)
    assert lfm.attn_window_workspace(q, cache, window=np.int64(7), sinks=0xFFFFFFFF) >= 0


def test_workspace_of_one_query_for_all(lfm):
    """q may have strides of 0 (one query for all rows, or all heads); outputs may not."""
    cache = lfm.KvCache(Host((3, 8, 100, 64)), Host((3, 8, 100, 64)), Host((3,), "torch.int32"))
    prefix = lfm.KvCache(Host((1, 8, 100, 64)), Host((1, 8, 100, 64)), Host((1,), "torch.int32"))
    dense = Host((3, 32, 64))
    for strides in ((0, 0, 1), (0, 64, 1), (64 * 32, 0, 1)):
        q = Host((3, 32, 64), strides=strides)
        assert lfm.attn_window_workspace(q, cache) == lfm.attn_window_workspace(dense, cache)
        assert lfm.attn_scored_workspace(q, cache) == lfm.attn_scored_workspace(dense, cache)
        assert lfm.attn_prefix_workspace(q, prefix, cache) == lfm.attn_prefix_workspace(dense, prefix, cache)
        with pytest.raises(lfm.LfmError) as e:
            lfm.attn_window(dense, cache, q, Host((1,)))
        assert e.value.code == lfm.LFM_EINVAL and "out stride" in str(e.value)


def test_workspaces_that_are_strided_views_are_refused(lfm):
    """A call would write the bytes between the view's own."""
    cache = lfm.KvCache(Host((3, 8, 100, 64)), Host((3, 8, 100, 64)), Host((3,), "torch.int32"))
    q, acc, pos = Host((3, 32, 64)), Host((3, 8, 100), "torch.float32"), Host((3, 8, 100), "torch.int32")

    class View(Host):
        def is_contiguous(self):
            return False

    ws = View((1 << 20,))
    for call in (lambda: lfm.attn_window(q, cache, q, ws), lambda: lfm.attn_scored(q, cache, q, None, acc, ws),
                 lambda: lfm.attn_prefix(q, cache, cache, q, ws),
                 lambda: lfm.kv_evict(cache, acc, pos, 50, cache, acc, pos, ws)):
        with pytest.raises(lfm.LfmError) as e:
            call()
        assert e.value.code == lfm.LFM_EINVAL and "workspace" in str(e.value)
