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
        f.argtypes = lfm.lib().__getattr__(name).argtypes
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
