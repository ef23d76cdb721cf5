"""The cache-attention operators' host side on the CPU: which device pointers are refused
and what a call enqueues, over stand-ins for the HIP calls (hip_stub.cpp)."""
import ctypes as C
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(os.path.dirname(HERE), "lfm2-w9100-rust_amd", "csrc")
MB = 1 << 20
HOST = 1 << 40  # an address that is no device memory


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("attn_host") / "attn_host.so")
    rocm = os.environ.get("ROCM", "/opt/rocm")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-D__HIP_PLATFORM_AMD__",
                    "-I" + os.path.join(rocm, "include"), "-I" + SRC, os.path.join(SRC, "attn_ops.cpp"),
                    os.path.join(HERE, "hip_stub.cpp"), "-o", so], check=True)
    L = C.CDLL(so)
    L.stub_launch.restype = C.c_char_p
    L.stub_error.restype = C.c_char_p
    L.stub_memory.argtypes = [C.c_size_t, C.c_size_t, C.c_int]
    L.stub_reset.argtypes = [C.c_size_t]
    return L


@pytest.fixture
def call(host, lfm):
    """Calls an operator; returns its status and the kernels that it enqueued.  Device memory
    is [1 MB, 64 MB)."""
    def run(name, *args):
        host.stub_reset(0)
        host.stub_memory(MB, 63 * MB, 0)
        f = getattr(host, name)
        f.argtypes = getattr(lfm.lib(), name).argtypes
        rc = f(*args)
        grid, block, names = (C.c_uint32 * 3)(), C.c_uint32(), []
        for i in range(host.stub_launches()):
            names.append(host.stub_launch(i, grid, C.byref(block)).decode())
        return rc, names
    return run


def kv(lfm, **kw):
    a = dict(k=MB, v=2 * MB, len=3 * MB, seq_stride=8 * 100 * 64, head_stride=100 * 64, slot_stride=64,
             type=lfm.TYPE_F16, n_seq=3, kv_heads=8, slots=100, head_dim=64)
    a.update(kw)
    return lfm.Kv(**a)


def rows(lfm, **kw):
    a = dict(q=4 * MB, out=5 * MB, q_row_stride=32 * 64, q_head_stride=64, out_row_stride=32 * 64,
             out_head_stride=64, type=lfm.TYPE_F16, heads=32, n_rows=3, scale=0.125)
    a.update(kw)
    return lfm.Rows(**a)


WS = (16 * MB, 40 * MB)


def scored(call, k, r):
    return call("lfm_attn_scored", C.byref(k), C.byref(r), None, 6 * MB, *WS, None)


@pytest.mark.parametrize("start", [HOST, 7 * MB + 2])
def test_scored_checks_start_without_rows(call, lfm, start):
    """A call without rows still reads start on the device: it copies acc to acc_out."""
    assert scored(call, kv(lfm), rows(lfm, n_rows=0, start=7 * MB)) == (0, ["k_attn_weights_f16_64"])
    assert scored(call, kv(lfm), rows(lfm, n_rows=0, start=start)) == (lfm.LFM_EINVAL, [])
    # q, out and lse are not read then
    assert scored(call, kv(lfm), rows(lfm, n_rows=0, start=7 * MB, q=None, out=None))[0] == 0


# ------------------------------------------------------------------ every pointer of every call
def window(call, p):
    return call("lfm_attn_window", C.byref(p["kv"]), C.byref(p["rows"]), 0, 0, *p["ws"], None)


def scored_of(call, p):
    return call("lfm_attn_scored", C.byref(p["kv"]), C.byref(p["rows"]), p["acc_in"], p["acc_out"], *p["ws"], None)


def prefix(call, p):
    return call("lfm_attn_prefix", C.byref(p["prefix"]), C.byref(p["kv"]), C.byref(p["rows"]), *p["ws"], None)


def evict(call, p):
    return call("lfm_kv_evict", C.byref(p["kv"]), p["acc_in"], p["pos"], 50, 4, 8, C.byref(p["out"]), p["acc_out"],
                p["pos_out"], *p["ws"], None)


def arguments(lfm, **kw):
    a = dict(kv=kv(lfm, slots=2000), rows=rows(lfm, lse=11 * MB, start=7 * MB, n_rows=9), ws=(16 * MB, 40 * MB),
             prefix=kv(lfm, n_seq=1, k=8 * MB, v=9 * MB, len=10 * MB), acc_in=6 * MB, acc_out=12 * MB, pos=13 * MB,
             pos_out=14 * MB, out=kv(lfm, k=8 * MB, v=9 * MB, len=10 * MB))
    a.update(kw)
    return a


POINTERS = [(window, s, f) for s, f in (("kv", "k"), ("kv", "v"), ("kv", "len"), ("rows", "q"), ("rows", "out"),
                                        ("rows", "lse"), ("rows", "start"), ("ws", None))]
POINTERS += [(scored_of, s, f) for s, f in (("kv", "k"), ("rows", "start"), ("acc_in", None), ("acc_out", None), ("ws", None))]
POINTERS += [(prefix, s, f) for s, f in (("kv", "v"), ("rows", "q"), ("prefix", "k"), ("prefix", "v"), ("prefix", "len"),
                                         ("ws", None))]
POINTERS += [(evict, s, f) for s, f in (("kv", "k"), ("kv", "v"), ("kv", "len"), ("out", "k"), ("out", "v"), ("out", "len"),
                                        ("acc_in", None), ("acc_out", None), ("pos", None), ("pos_out", None), ("ws", None))]
OPTIONAL = {("rows", "lse"), ("acc_in", None)}


@pytest.mark.parametrize("op, struct, field", POINTERS,
                         ids=lambda v: v if isinstance(v, str) else "" if v is None else v.__name__)
def test_every_pointer_is_checked(host, call, lfm, op, struct, field):
    """A host address, another device's memory, one byte off and null: refused, nothing enqueued."""
    rc, names = op(call, arguments(lfm))
    assert rc == 0 and names, host.stub_error()
    far = 100 * MB  # memory of device 1
    for bad in (HOST, far, 1, None):
        if bad is None and (op is not evict and (struct, field) in OPTIONAL or (struct, field) == ("rows", "start")):
            continue
        a = arguments(lfm)

        def change(old):
            return old + 1 if bad == 1 else bad
        if field:
            setattr(a[struct], field, change(getattr(a[struct], field)))
        else:
            a[struct] = (change(a[struct][0]), a[struct][1]) if struct == "ws" else change(a[struct])

        def run(name, *args):
            host.stub_reset(0)
            host.stub_memory(MB, 63 * MB, 0)
            host.stub_memory(far, MB, 1)
            f = getattr(host, name)
            f.argtypes = getattr(lfm.lib(), name).argtypes
            return f(*args), [None] * host.stub_launches()
        assert op(run, a) == (lfm.LFM_EINVAL, []), (bad, host.stub_error())
        assert host.stub_error()


def test_workspaces_one_byte_short(host, call, lfm):
    n = C.c_size_t()
    a = arguments(lfm)
    k, r, p = C.byref(a["kv"]), C.byref(a["rows"]), C.byref(a["prefix"])
    for op, size in ((window, lambda: host.lfm_attn_window_workspace(k, r, 0, 0, C.byref(n))),
                     (scored_of, lambda: host.lfm_attn_scored_workspace(k, r, C.byref(n))),
                     (prefix, lambda: host.lfm_attn_prefix_workspace(p, k, r, C.byref(n))),
                     (evict, lambda: host.lfm_kv_evict_workspace(k, 50, C.byref(n)))):
        a["ws"] = (16 * MB, 1 << 40)
        assert size() == 0 and op(call, a)[0] == 0
        a["ws"] = (16 * MB, n.value)
        assert op(call, a)[0] == 0
        if n.value:
            a["ws"] = (16 * MB, n.value - 1)
            assert op(call, a) == (lfm.LFM_EINVAL, [])


def test_nothing_to_do_enqueues_nothing(call, lfm):
    """No sequences, or no rows: fine, whatever the pointers are."""
    none = arguments(lfm, kv=kv(lfm, n_seq=0, k=None, v=None, len=None), out=kv(lfm, n_seq=0, k=None, v=None, len=None),
                     rows=rows(lfm, n_rows=0, q=None, out=None), ws=(None, 0), acc_in=None, acc_out=None, pos=None,
                     pos_out=None)
    # k and v alike are in place there
    for op in (window, scored_of, prefix, evict):
        assert op(call, none) == (0, []), op.__name__
    rowless = arguments(lfm, rows=rows(lfm, n_rows=0, start=7 * MB, q=None, out=None))
    assert window(call, rowless) == (0, []) and prefix(call, rowless) == (0, [])


def test_a_failing_runtime_leaves_no_error_behind(host, call, lfm, tmp_path):
    """A call that the runtime fails returns LFM_EDEVICE, and the error is not there for the
    caller's next check to find; a refused pointer leaves none either."""
    import shutil
    so = shutil.copy(host._name, tmp_path / "fresh.so")  # one that has loaded no code object yet
    fresh = C.CDLL(str(so))
    a = arguments(lfm)
    for which in (1, 2, 3, 0):
        fresh.stub_reset.argtypes, fresh.stub_memory.argtypes = [C.c_size_t], [C.c_size_t, C.c_size_t, C.c_int]
        fresh.stub_reset(0)
        fresh.stub_memory(MB, 63 * MB, 0)
        fresh.stub_refuse(which)

        def run(name, *args):
            f = getattr(fresh, name)
            f.argtypes = getattr(lfm.lib(), name).argtypes
            return f(*args)
        for op in (window, scored_of, prefix, evict):
            assert op(run, a) == (lfm.LFM_EDEVICE if which else 0)
            assert fresh.stub_left() == 0, (which, op.__name__)
    assert window(call, arguments(lfm, rows=rows(lfm, q=HOST)))[0] == lfm.LFM_EINVAL
    assert host.stub_left() == 0
