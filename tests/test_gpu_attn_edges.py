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
