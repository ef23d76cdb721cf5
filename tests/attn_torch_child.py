"""The cache-attention binding over torch tensors, in a process of its own (torch loaded
first, so that both use one HIP runtime): torch's current stream, a torch graph, views."""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lfm2-w9100-rust_amd"))
import lfm_hip  # noqa: E402

DEV = "cuda:0"


def attend(q, k, v, length, window, sinks):
    """[n][heads][d] in 64 bits on the host; one row per sequence."""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    out = torch.zeros_like(q)
    g = q.shape[1] // k.shape[1]
    for b, n in enumerate(length.tolist()):
        j = torch.arange(n)
        j = j[(j < sinks) | (j > n - 1 - window)] if window else j
        for h in range(q.shape[1]):
            w = torch.softmax(k[b, h // g, j] @ q[b, h] * q.shape[2] ** -0.5, 0)
            out[b, h] = w @ v[b, h // g, j]
    return out


def close(got, want, v):
    """F16 rows: weights and output rounded to 11 bits, and scores' 32-bit sums."""
    err = (got.cpu().double() - want).abs().max().item()
    assert err <= 2.0 ** -10 * v.abs().max().item(), err


def main():
    torch.manual_seed(3)
    n, heads, kv, slots, d = 5, 8, 2, 700, 64
    # caches slot by slot, seen as [n][kv][slots][d]; q a slice of a fused projection's output
    k, v = (torch.randn(n, slots, kv, d, device=DEV).half().transpose(1, 2) for _ in range(2))
    length = torch.tensor([700, 1, 33, 512, 690], dtype=torch.int32, device=DEV)
    fused = torch.randn(n, heads + 2 * kv, d, device=DEV).half()
    q, out = fused[:, :heads], torch.empty(n, heads, d, device=DEV).half()
    cache = lfm_hip.KvCache(k, v, length)
    ws = torch.empty(max(1, lfm_hip.attn_window_workspace(q, cache, window=100, sinks=4)), dtype=torch.uint8, device=DEV)
    lfm_hip.attn_window(q, cache, out, ws, window=100, sinks=4)
    torch.cuda.synchronize()
    close(out, attend(q, k, v, length, 100, 4), v)
    print("views ok", flush=True)

    # q is made on a side stream, late: the call has to come after it
    side, new = torch.cuda.Stream(), torch.randn(n, heads, d, device=DEV).half()
    a = torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            a = (a @ a) * 1e-3
        q.copy_(new)
        lfm_hip.attn_window(q, cache, out, ws, window=100, sinks=4)
    side.synchronize()
    close(out, attend(new, k, v, length, 100, 4), v)
    print("side stream ok", flush=True)

    # captured by torch: the graph's stream is the current one
    scored = torch.empty(n, kv, slots, device=DEV)
    ws2 = torch.empty(max(1, lfm_hip.attn_scored_workspace(q, cache)), dtype=torch.uint8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lfm_hip.attn_scored(q, cache, out, None, scored, ws2)
    for i in range(4):
        q.copy_(torch.randn(n, heads, d, device=DEV).half())
        scored.zero_()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        close(out, attend(q, k, v, length, 0, 0), v)
        for b, m in enumerate(length.tolist()):
            assert abs(scored[b, :, :m].double().sum().item() - heads) < 1e-3
            assert (scored[b, :, m:] == 0).all()
    print("graph ok", flush=True)

    # tensors of the host are refused
    try:
        lfm_hip.attn_window(q, cache, torch.empty(n, heads, d).half(), ws)
    except lfm_hip.LfmError as e:
        assert e.code == lfm_hip.LFM_EINVAL
        print("host tensor refused", flush=True)
    torch.cuda.synchronize()


main()
