"""Attention over key/value caches, and a cache's eviction, as cases that can be timed and compared.

A cache holds K and V of n_seq sequences, each [kv_heads][slots][head_dim] (the engine's
order) or slot by slot, in binary16 or bfloat16, with the number of slots in use per
sequence.  The rows of a call are new tokens whose own K and V are in the cache already.
"f32" rows over a binary16 cache are the engine's pair.  Queries are scaled so that a
row's weights are as uneven as attention's are: the scores' standard deviation is 1.5.
"""
import math
import os
import random
import sys

import torch

own = False
PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lfm2-w9100-rust_amd")

ENGINE = {"heads": 32, "kv_heads": 8, "dim": 64, "type": "f32", "order": "head"}
WIDE = {"heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "order": "slot"}


def listed():
    return [
        # One step of one chat on the engine's heads: the newest 1024 positions and the
        # first four of a full context.  The smallest attention call.
        {"name": "window_step", "op": "window", **ENGINE, "seqs": 1, "rows": 1, "slots": 4096, "shortest": 3900,
         "window": 1024, "sinks": 4},
        # A server's step: 64 chats of mixed lengths, some shorter than the window.
        {"name": "window_batch", "op": "window", **WIDE, "seqs": 64, "rows": 1, "slots": 16384, "shortest": 700,
         "window": 4096, "sinks": 16},
        # A whole context as one prompt.
        {"name": "window_prompt", "op": "window", **ENGINE, "type": "f16", "seqs": 1, "rows": 4096, "slots": 4096,
         "shortest": 4096, "window": 1024, "sinks": 4},
        # Chunks of several chats at once, of odd lengths, onto what each holds already.
        {"name": "window_chunks", "op": "window", **WIDE, "heads": 28, "kv_heads": 4, "seqs": 13, "rows": 611,
         "slots": 5000, "shortest": 900, "window": 2048, "sinks": 1},
        # A step of eight chats that keep the weights their tokens received.
        {"name": "scored_step", "op": "scored", **ENGINE, "seqs": 8, "rows": 1, "slots": 4096, "shortest": 1500},
        # The same for a few long documents.
        {"name": "scored_long", "op": "scored", **WIDE, "seqs": 6, "rows": 1, "slots": 32768, "shortest": 20000},
        # A prompt whose weights decide what stays of it.
        {"name": "scored_prompt", "op": "scored", **ENGINE, "type": "f16", "seqs": 1, "rows": 2048, "slots": 2048,
         "shortest": 2048},
        # Ten slots too many in one chat's cache.
        {"name": "evict_step", "op": "evict", **ENGINE, "seqs": 1, "slots": 1034, "shortest": 1034, "keep": 1024,
         "sinks": 4, "recent": 256},
        # Prompts cut down to the cache that their answers are made from.
        {"name": "evict_prompts", "op": "evict", **WIDE, "seqs": 16, "slots": 8192, "shortest": 3001, "keep": 2048,
         "sinks": 16, "recent": 512},
        # Four chats under one short system prompt, at their first words.
        {"name": "prefix_small", "op": "prefix", **ENGINE, "seqs": 4, "prefix": 512, "slots": 128, "shortest": 1},
        # Sixty-four chats under a long one.
        {"name": "prefix_batch", "op": "prefix", **WIDE, "seqs": 64, "prefix": 8192, "slots": 1024, "shortest": 17},
        # Many short questions about one long document.
        {"name": "prefix_document", "op": "prefix", **ENGINE, "type": "f16", "seqs": 150, "prefix": 32000,
         "slots": 257, "shortest": 2},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["window", "window", "scored", "evict", "prefix"])
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (16, 16), (28, 4), (4, 2), (24, 2), (9, 3)])
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([64, 64, 128]),
         "type": rng.choice(["f32", "f16", "bf16"]), "order": rng.choice(["head", "slot"])}
    if op == "evict":
        c["seqs"] = _log_uniform(rng, 1, 24)
        c["keep"] = _log_uniform(rng, 48, 2048)
        c["slots"] = c["keep"] + _log_uniform(rng, 1, 6000)
        c["shortest"] = rng.randint(c["keep"], c["slots"])
        c["sinks"] = rng.randint(0, 16)
        c["recent"] = rng.randint(0, c["keep"] - 16)
        return c
    if op == "prefix":
        c["seqs"] = _log_uniform(rng, 1, 128)
        c["prefix"] = _log_uniform(rng, 1, 16384)
        c["slots"] = _log_uniform(rng, 1, 1024)
        c["shortest"] = rng.randint(1, c["slots"])
        return c
    if rng.random() < 0.5:  # a step
        c["rows"] = 1
        c["seqs"] = _log_uniform(rng, 1, 64)
        c["slots"] = _log_uniform(rng, 1, min(32768, 120000 // c["seqs"]))
    else:  # chunks or prompts: 3 x 1024 x 2048 pairs of a row and a slot at most
        c["rows"] = _log_uniform(rng, 2, 2048)
        c["slots"] = c["rows"] + _log_uniform(rng, 1, 2048) - 1
        c["seqs"] = _log_uniform(rng, 1, max(1, min(32, 3 * 1024 * 2048 // (c["rows"] * c["slots"]))))
    c["shortest"] = rng.randint(1, c["slots"])
    if op == "window":
        c["window"] = rng.choice([0, _log_uniform(rng, 1, 8192)])
        c["sinks"] = rng.choice([0, 1, 4, rng.randint(0, 200)])
    return c


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Slots in use and new rows of each sequence: part of the case, the same for every seed."""
    r = random.Random(case["seqs"] * 1000003 + case["slots"])
    n = case["seqs"]
    length = [r.randint(case["shortest"], case["slots"]) for _ in range(n)]
    if case["op"] == "prefix" or case.get("rows", 1) == 1:
        return length, [1] * n
    rows = [min(l, r.randint(1, case["rows"])) for l in length]
    rows[0] = min(length[0], case["rows"])
    return length, rows


def _cache(case, n, slots, gen, kind):
    kv, d = case["kv_heads"], case["dim"]
    shape = (n, kv, slots, d) if case["order"] == "head" else (n, slots, kv, d)
    t = [torch.randn(shape, generator=gen, device=gen.device).to(kind) for _ in range(2)]
    return t if case["order"] == "head" else [x.transpose(1, 2) for x in t]


TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind = torch.bfloat16 if case["type"] == "bf16" else torch.float16
    n, kv, slots = case["seqs"], case["kv_heads"], case["slots"]
    length, rows = _lengths(case)
    s = {"case": case}
    s["k"], s["v"] = _cache(case, n, slots, gen, kind)
    s["length"] = torch.tensor(length, dtype=torch.int32, device=dev)
    if case["op"] == "evict":
        # weights received so far: heavy for a few slots, slight for most
        s["acc"] = torch.rand(n, kv, slots, generator=gen, device=dev).pow(6) * 50
        # a cache that was evicted from before holds every few positions
        gaps = torch.randint(1, 4, (n, kv, slots), generator=gen, device=dev)
        s["pos"] = (gaps.cumsum(-1) - 1).to(torch.int32)
        s["k_out"], s["v_out"] = (torch.zeros_like(x[:, :, :case["keep"]]) for x in (s["k"], s["v"]))
        s["acc_out"], s["pos_out"] = (torch.zeros_like(x[:, :, :case["keep"]]).contiguous()
                                      for x in (s["acc"], s["pos"]))
        s["length_out"], s["most"] = torch.zeros_like(s["length"]), 1
        return s
    total = sum(rows)
    s["scale"] = 1 / math.sqrt(case["dim"])
    s["q"] = (1.5 * torch.randn(total, case["heads"], case["dim"], generator=gen, device=dev)).to(TYPES[case["type"]])
    s["start"] = torch.tensor([sum(rows[:i]) for i in range(n + 1)], dtype=torch.int32, device=dev)
    s["most"] = max(rows)  # a program that lays out a batch knows the longest part
    s["out"] = torch.zeros_like(s["q"])
    s["lse"] = torch.zeros(s["q"].shape[:2], device=dev)
    if case["op"] == "scored":
        s["acc"] = torch.rand(n, kv, slots, generator=gen, device=dev)
        s["acc_out"] = torch.zeros_like(s["acc"])
    if case["op"] == "prefix":
        s["pk"], s["pv"] = _cache(case, 1, case["prefix"], gen, kind)
        s["plength"] = torch.tensor([case["prefix"]], dtype=torch.int32, device=dev)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state)
    if op == "evict":
        return _plain_evict(state)
    if op == "prefix":
        return _plain_prefix(state)
    return _plain_attention(state)


def _own(s):
    """The framework's calls, on device pointers, with the outputs and the workspace that
    the program keeps."""
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import lfm_hip

    case, op = s["case"], s["case"]["op"]
    start = s["start"] if s["most"] > 1 else None
    if "cache" not in s:  # made once by a program: the views of its caches and a workspace
        cache = s["cache"] = lfm_hip.KvCache(s["k"], s["v"], s["length"])
        if op == "evict":
            s["kept"] = lfm_hip.KvCache(s["k_out"], s["v_out"], s["length_out"])
            n = lfm_hip.kv_evict_workspace(cache, case["keep"])
        elif op == "window":
            n = lfm_hip.attn_window_workspace(s["q"], cache, window=case["window"], sinks=case["sinks"], start=start)
        elif op == "scored":
            n = lfm_hip.attn_scored_workspace(s["q"], cache, start=start)
        else:
            s["prefix"] = lfm_hip.KvCache(s["pk"], s["pv"], s["plength"])
            n = lfm_hip.attn_prefix_workspace(s["q"], s["prefix"], cache, start=start)
        s["workspace"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    cache, workspace = s["cache"], s["workspace"]
    if op == "evict":
        lfm_hip.kv_evict(cache, s["acc"], s["pos"], case["keep"], s["kept"], s["acc_out"], s["pos_out"], workspace,
                         sinks=case["sinks"], recent=case["recent"])
        return {"k": s["k_out"], "v": s["v_out"], "acc": s["acc_out"], "pos": s["pos_out"],
                "length": s["length_out"]}
    if op == "window":
        lfm_hip.attn_window(s["q"], cache, s["out"], workspace, window=case["window"], sinks=case["sinks"],
                            start=start, scale=s["scale"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if op == "scored":
        lfm_hip.attn_scored(s["q"], cache, s["out"], s["acc"], s["acc_out"], workspace, start=start,
                            scale=s["scale"])
        return {"out": s["out"], "acc": s["acc_out"]}
    lfm_hip.attn_prefix(s["q"], s["prefix"], cache, s["out"], workspace, start=start, scale=s["scale"])
    return {"out": s["out"]}


def _rows(s):
    """Index of row i of sequence b in the batch, where it is one, and its position."""
    count = (s["start"][1:] - s["start"][:-1]).unsqueeze(1)
    i = torch.arange(s["most"], device=count.device)
    valid = i < count
    index = torch.where(valid, s["start"][:-1].unsqueeze(1) + i, torch.zeros_like(valid, dtype=torch.int32))
    return index.long(), valid, s["length"].unsqueeze(1) - count + i


def _grouped(x, kv):
    """[b][rows][heads][d] -> [b][kv][rows * group][d]"""
    b, r, h, d = x.shape
    return x.view(b, r, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(b, kv, r * (h // kv), d)


def _plain_attention(s):
    case = s["case"]
    kv, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    index, valid, pos = _rows(s)
    b, r = index.shape
    score = _grouped(s["q"].float()[index], kv) @ s["k"].float().transpose(-1, -2) * s["scale"]
    slot = torch.arange(case["slots"], device=index.device)
    seen = (slot <= pos.unsqueeze(-1)) & valid.unsqueeze(-1)
    if case.get("window"):
        seen = seen & ((slot < case["sinks"]) | (slot > pos.unsqueeze(-1) - case["window"]))
    score = score.view(b, kv, r, group, -1).masked_fill(~seen.view(b, 1, r, 1, -1), -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3.0e38)
    w = (score - top).exp()
    total = w.sum(-1, keepdim=True)
    lse = (top + total.log()).squeeze(-1)
    w = w / total.clamp(min=1e-30)
    out = (w.reshape(b, kv, r * group, -1) @ s["v"].float()).view(b, kv, r, group, -1)
    out = out.permute(0, 2, 1, 3, 4)[valid].reshape(s["q"].shape).to(s["q"].dtype)
    if case["op"] == "window":
        return {"out": out, "lse": lse.permute(0, 2, 1, 3)[valid].reshape(s["q"].shape[:2])}
    acc = torch.where(slot < s["length"].view(-1, 1, 1), s["acc"] + w.sum((2, 3)), s["acc_out"])
    return {"out": out, "acc": acc}  # the slots past the length as they were


def _plain_prefix(s):
    case = s["case"]
    n, kv, group, d = case["seqs"], case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    q = _grouped(s["q"].float().unsqueeze(1), kv)  # [n][kv][group][d]: one row each
    flat = q.transpose(0, 1).reshape(kv, n * group, d)
    first = (flat @ s["pk"][0].float().transpose(-1, -2)).view(kv, n, group, -1).transpose(0, 1) * s["scale"]
    second = q @ s["k"].float().transpose(-1, -2) * s["scale"]
    slot = torch.arange(case["slots"], device=q.device)
    second = second.masked_fill(slot >= s["length"].view(-1, 1, 1, 1), -math.inf)
    w = torch.cat([first, second], -1)
    w = (w - w.amax(-1, keepdim=True)).exp()
    w = w / w.sum(-1, keepdim=True)
    first, second = w.split([case["prefix"], case["slots"]], -1)
    out = first.transpose(0, 1).reshape(kv, n * group, -1) @ s["pv"][0].float()
    out = out.view(kv, n, group, d).transpose(0, 1) + second @ s["v"].float()
    return {"out": out.reshape(n, kv * group, d).to(s["q"].dtype)}


def _plain_evict(s):
    case = s["case"]
    keep, slots = case["keep"], case["slots"]
    slot = torch.arange(slots, device=s["pos"].device)
    used = slot < s["length"].view(-1, 1, 1)
    newest = s["pos"].masked_fill(~used, -1).amax(-1, keepdim=True)
    protected = (s["pos"] < case["sinks"]) | (s["pos"] > newest - case["recent"])
    score = s["acc"].masked_fill(protected, math.inf).masked_fill(~used, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(used.expand_as(score)).scatter(-1, order[..., :keep], True)
    # the i-th kept slot at or past `keep` goes into the i-th hole below it
    moved = torch.where(kept[..., keep:], slot[keep:], slots).sort(-1).values
    hole = ~kept[..., :keep]
    rank = (hole.cumsum(-1) - 1).clamp(min=0, max=moved.shape[-1] - 1)
    source = torch.where(hole, moved.gather(-1, rank), slot[:keep])
    rows = source.unsqueeze(-1).expand(-1, -1, -1, case["dim"])
    return {"k": s["k"].gather(2, rows), "v": s["v"].gather(2, rows), "acc": s["acc"].gather(2, source),
            "pos": s["pos"].gather(2, source), "length": s["length"].clamp(max=keep)}


# ------------------------------------------------------------------ work
def work(case):
    length, rows = _lengths(case)
    kv, d, heads = case["kv_heads"], case["dim"], case["heads"]
    slot_bytes = 2 * kv * d * 2
    if case["op"] == "evict":
        # every slot's weight and position; the kept rows read and written, with theirs
        return {"bytes": 8 * kv * sum(length) + case["seqs"] * case["keep"] * (2 * slot_bytes + 8 * kv), "flops": 0}
    wide = 4 if case["type"] == "f32" else 2
    moved = 2 * wide * sum(rows) * heads * d
    if case["op"] == "prefix":
        pairs = sum(length) + case["seqs"] * case["prefix"]
        return {"bytes": moved + slot_bytes * (sum(length) + case["prefix"]), "flops": 4 * heads * d * pairs}
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    pairs = touched = 0
    for l, r in zip(length, rows):
        if window:
            pairs += sum(min(p + 1, sinks + window) for p in range(l - r, l))
            touched += min(l, sinks + window + r - 1)
        else:
            pairs += sum(range(l - r + 1, l + 1))
            touched += l
    total = moved + slot_bytes * touched
    if case["op"] == "window":
        total += 4 * sum(rows) * heads
    else:
        total += 8 * kv * sum(length)
    return {"bytes": total, "flops": 4 * heads * d * pairs}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_evict(s) if case["op"] == "evict" else _exact_attention(s)


def _exact_attention(s):
    """Each sequence and kv head by itself, its visible slots alone where rows are single."""
    case = s["case"]
    length, rows = _lengths(case)
    kv, group, d = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    acc = torch.zeros(s["k"].shape[:3], dtype=torch.float64, device=q.device)
    at = 0
    for b, (l, r) in enumerate(zip(length, rows)):
        j = torch.arange(l, device=q.device)
        p = torch.arange(l - r, l, device=q.device).unsqueeze(1)
        hidden = j > p
        if case.get("window"):
            hidden |= (j >= case["sinks"]) & (p - j >= case["window"])
        for h in range(kv):
            k, v = s["k"][b, h, :l].double(), s["v"][b, h, :l].double()
            mask = hidden
            if case["op"] == "prefix":
                k, v = torch.cat([s["pk"][0, h].double(), k]), torch.cat([s["pv"][0, h].double(), v])
                mask = torch.cat([hidden.new_zeros(r, case["prefix"]), hidden], 1)
            here = slice(h * group, (h + 1) * group)
            logit = torch.einsum("rgd,jd->rgj", q[at:at + r, here], k) / math.sqrt(d)
            logit = logit.masked_fill(mask.unsqueeze(1), -math.inf)
            z = torch.logsumexp(logit, -1)
            w = torch.exp(logit - z.unsqueeze(-1))
            out[at:at + r, here] = torch.einsum("rgj,jd->rgd", w, v)
            lse[at:at + r, here] = z
            if case["op"] == "scored":
                acc[b, h, :l] = s["acc"][b, h, :l].double() + w.sum((0, 1))
        at += r
    if case["op"] == "window":
        return {"out": out, "lse": lse}
    return {"out": out, "acc": acc} if case["op"] == "scored" else {"out": out}


def _exact_evict(s):
    case = s["case"]
    length, _ = _lengths(case)
    keep = case["keep"]
    acc, pos = s["acc"].double().cpu(), s["pos"].long().cpu()
    source = torch.zeros(*acc.shape[:2], keep, dtype=torch.int64)
    for b, l in enumerate(length):
        for h in range(case["kv_heads"]):
            a, p = acc[b, h, :l].tolist(), pos[b, h, :l].tolist()
            newest = max(p)
            rank = sorted(range(l), key=lambda j: (not (p[j] < case["sinks"] or newest - p[j] < case["recent"]),
                                                   -a[j] if not (p[j] < case["sinks"] or newest - p[j] < case["recent"])
                                                   else 0.0, j))
            kept = set(rank[:keep])
            late = iter(sorted(j for j in kept if j >= keep))
            source[b, h] = torch.tensor([j if j in kept else next(late) for j in range(keep)])
    source = source.to(s["k"].device)
    wide = source.unsqueeze(-1).expand(-1, -1, -1, case["dim"])
    return {"k": s["k"].gather(2, wide).double(), "v": s["v"].gather(2, wide).double(),
            "acc": s["acc"].gather(2, source).double(), "pos": s["pos"].gather(2, source),
            "length": s["length"].clamp(max=keep)}
