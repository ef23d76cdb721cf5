// attn_ops.cpp -- C ABI of the cache-attention operators: argument checks, work splits and
// launches of the kernels in lfm_attn.hip.
#include <float.h>
#include <hip/hip_runtime_api.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <exception>
#include <mutex>
#include <unordered_map>

#include "../../include/lfm_hip.h"
#include "attn_args.h"
#include "host_err.h"
#include "launch_host.h"

#define RC(call)                                                                              \
    do {                                                                                      \
        int _rc = (call);                                                                     \
        if (_rc != LFM_OK)                                                                    \
            return _rc;                                                                       \
    } while (0)

// ------------------------------------------------------------------ code object
// Row tiles of 16 of the larger forms, as many as the registers hold.
static uint32_t step_tiles(uint32_t dim) { return dim == 64 ? 4 : 2; }

// Kernels by [type pair][head_dim 64, 128]; the pair is the rows' type.
struct AttnKernels {
    hipModule_t mod = nullptr;
    hipFunction_t tile_1[3][2], tile_most[3][2], tile_prefix[3][2], weights[3][2];
    hipFunction_t step_1[3][2], step_most[3][2], merge[3][2], scored_join[3][2];
    hipFunction_t sums, kv_select, kv_move;
};

static std::mutex g_mu;
static std::unordered_map<int, AttnKernels *> g_attn;

// A call of the runtime that failed: its error is not left for the caller's next check.
static int device_error(const char *what, const char *of, hipError_t e)
{
    (void)hipGetLastError();
    return fail(LFM_EDEVICE, "%s%s: %s", what, of, hipGetErrorString(e));
}

static int load_attn(int dev)
{
    const std::string path = lfm_beside_code_object("lfm_attn.hsaco");
    AttnKernels k;
    hipError_t e = hipModuleLoad(&k.mod, path.c_str());
    if (e != hipSuccess)
        return device_error("hipModuleLoad of ", path.c_str(), e);
    static const char *const types[3] = {"f32", "f16", "bf16"};
    auto get = [&](hipFunction_t *f, const std::string &name) -> int {
        const hipError_t r = hipModuleGetFunction(f, k.mod, name.c_str());
        return r == hipSuccess ? LFM_OK : device_error("hipModuleGetFunction of ", name.c_str(), r);
    };
    int rc = LFM_OK;
    for (int t = 0; t < 3 && rc == LFM_OK; ++t)
        for (int d = 0; d < 2 && rc == LFM_OK; ++d) {
            const std::string tag = std::string("_") + types[t] + (d ? "_128" : "_64");
            struct {
                hipFunction_t *f;
                std::string name;
            } fns[] = {{&k.tile_1[t][d], "k_attn_tile" + tag + "_r1"},
                       {&k.tile_most[t][d], "k_attn_tile" + tag + "_r" + std::to_string(TILE_TILES)},
                       {&k.tile_prefix[t][d], "k_attn_prefix" + tag},
                       {&k.weights[t][d], "k_attn_weights" + tag},
                       {&k.step_1[t][d], "k_attn_step" + tag + "_r1"},
                       {&k.step_most[t][d], "k_attn_step" + tag + "_r" + std::to_string(step_tiles(d ? 128 : 64))},
                       {&k.merge[t][d], "k_attn_merge" + tag},
                       {&k.scored_join[t][d], "k_scored_join" + tag}};
            for (auto &f : fns)
                if (rc == LFM_OK)
                    rc = get(f.f, f.name);
        }
    if (rc == LFM_OK)
        rc = get(&k.sums, "k_attn_sums");
    if (rc == LFM_OK)
        rc = get(&k.kv_select, "k_kv_select");
    if (rc == LFM_OK)
        rc = get(&k.kv_move, "k_kv_move");
    if (rc != LFM_OK) {
        (void)hipModuleUnload(k.mod);
        return rc;
    }
    g_attn[dev] = new AttnKernels(k);
    return LFM_OK;
}

// The code object on the current device, loaded by the device's first call.
static int attn_kernels(int dev, AttnKernels **out)
{
    try {
        std::lock_guard<std::mutex> lk(g_mu);
        auto it = g_attn.find(dev);
        if (it == g_attn.end()) {
            RC(load_attn(dev));
            it = g_attn.find(dev);
        }
        *out = it->second;
        return LFM_OK;
    } catch (const std::exception &x) {
        return fail(LFM_EINTERNAL, "loading the attention kernels: %s", x.what());
    }
}

template <typename A> static int launch(hipFunction_t f, dim3 grid, uint32_t threads, hipStream_t s, const A &args)
{
    void *params[] = {(void *)&args};
    const hipError_t e = hipModuleLaunchKernel(f, grid.x, grid.y, grid.z, threads, 1, 1, 0, s, params, nullptr);
    return e == hipSuccess ? LFM_OK : device_error("kernel launch", "", e);
}

// ------------------------------------------------------------------ argument checks
// A grid of 256 threads each stays below 2^32 threads.
#define MOST_WORKGROUPS 0xFFFFFFu

// Sizes and strides; they decide the workspace and need no device.
static int check_kv(const char *op, const char *name, const lfm_kv *c)
{
    if (!c)
        return fail(LFM_EINVAL, "%s: %s is null", op, name);
    if (c->type != LFM_TYPE_F16 && c->type != LFM_TYPE_BF16)
        return fail(LFM_EINVAL, "%s: %s: type %u (a cache is F16 or BF16)", op, name, c->type);
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(LFM_EINVAL, "%s: %s: head_dim %u (64 or 128)", op, name, c->head_dim);
    if (c->kv_heads == 0 || c->kv_heads > 65535 || c->n_seq > 65535)
        return fail(LFM_EINVAL, "%s: %s: %u sequences of %u kv heads (at most 65535, 1..65535)", op, name, c->n_seq,
                    c->kv_heads);
    if (c->slots == 0 || c->slots > 0x7FFFFF00u)
        return fail(LFM_EINVAL, "%s: %s: %u slots (1..%u)", op, name, c->slots, 0x7FFFFF00u);
    for (int64_t s : {c->seq_stride, c->head_stride, c->slot_stride})
        if (s < 0 || s % 8)
            return fail(LFM_EINVAL, "%s: %s: stride %lld (multiples of 8 elements, not negative)", op, name,
                        (long long)s);
    return LFM_OK;
}

static int check_rows(const char *op, const lfm_kv *c, const lfm_rows *r)
{
    if (!r)
        return fail(LFM_EINVAL, "%s: rows is null", op);
    if (r->type > LFM_TYPE_BF16 || (r->type == LFM_TYPE_BF16) != (c->type == LFM_TYPE_BF16))
        return fail(LFM_EINVAL, "%s: rows of type %u over a cache of type %u (F32 or F16 over F16, BF16 over BF16)",
                    op, r->type, c->type);
    if (r->heads == 0 || r->heads % c->kv_heads || r->heads / c->kv_heads > MAX_GROUP || r->heads > 65535)
        return fail(LFM_EINVAL, "%s: %u heads over %u kv heads (a multiple, at most %u times)", op, r->heads,
                    c->kv_heads, MAX_GROUP);
    if ((uint64_t)r->n_rows * r->heads > MOST_WORKGROUPS)
        return fail(LFM_EINVAL, "%s: %u rows of %u heads (%u of them at most)", op, r->n_rows, r->heads,
                    MOST_WORKGROUPS);
    if (!r->start && r->n_rows != c->n_seq)
        return fail(LFM_EINVAL, "%s: %u rows for %u sequences without start (one row each)", op, r->n_rows, c->n_seq);
    if (!(r->scale > 0.f) || !(r->scale < INFINITY))
        return fail(LFM_EINVAL, "%s: scale %g (a positive number)", op, (double)r->scale);
    const int64_t q = r->type == LFM_TYPE_F32 ? 4 : 8;
    for (int64_t s : {r->q_row_stride, r->q_head_stride, r->out_row_stride, r->out_head_stride})
        if (s < 0 || s % q)
            return fail(LFM_EINVAL, "%s: row or head stride %lld (multiples of 16 bytes, not negative)", op,
                        (long long)s);
    if ((r->n_rows > 1 && r->out_row_stride == 0) || (r->heads > 1 && r->out_head_stride == 0))
        return fail(LFM_EINVAL, "%s: an out stride of 0", op);
    return LFM_OK;
}

// A device pointer of the current device (or managed memory), aligned.
static int check_ptr(const char *op, const char *name, const void *p, size_t align, int dev)
{
    if (!p)
        return fail(LFM_EINVAL, "%s: %s is null", op, name);
    if ((uintptr_t)p % align)
        return fail(LFM_EINVAL, "%s: %s is not %zu-byte aligned", op, name, align);
    hipPointerAttribute_t at;
    if (hipPointerGetAttributes(&at, p) != hipSuccess) {
        (void)hipGetLastError();
        return fail(LFM_EINVAL, "%s: %s is not device memory", op, name);
    }
    if (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged)
        return fail(LFM_EINVAL, "%s: %s is not device memory", op, name);
    if (at.type == hipMemoryTypeDevice && at.device != dev)
        return fail(LFM_EINVAL, "%s: %s lies on device %d, the current one is %d", op, name, at.device, dev);
    return LFM_OK;
}

// The current device; `stream` has to be its own.
static int current_device(const char *op, hipStream_t s, int *dev)
{
    if (hipGetDevice(dev) != hipSuccess) {
        (void)hipGetLastError();
        return fail(LFM_EDEVICE, "%s: no current device", op);
    }
    hipDevice_t of;
    if (s && (hipStreamGetDevice(s, &of) != hipSuccess || of != *dev)) {
        (void)hipGetLastError();
        return fail(LFM_EINVAL, "%s: the stream is not one of the current device (%d)", op, *dev);
    }
    return LFM_OK;
}

static int check_kv_ptrs(const char *op, const char *const (&names)[3], const lfm_kv *c, int dev)
{
    RC(check_ptr(op, names[0], c->k, 16, dev));
    RC(check_ptr(op, names[1], c->v, 16, dev));
    return check_ptr(op, names[2], c->len, 4, dev);
}
static const char *const KV_NAMES[3] = {"kv->k", "kv->v", "kv->len"};
static const char *const PREFIX_NAMES[3] = {"prefix->k", "prefix->v", "prefix->len"};
static const char *const OUT_NAMES[3] = {"out->k", "out->v", "out->len"};

// start is read without rows too: a scored call then still copies acc.
static int check_rows_ptrs(const char *op, const lfm_rows *r, int dev)
{
    if (r->start)
        RC(check_ptr(op, "rows->start", r->start, 4, dev));
    if (r->n_rows == 0)
        return LFM_OK;
    RC(check_ptr(op, "rows->q", r->q, 16, dev));
    RC(check_ptr(op, "rows->out", r->out, 16, dev));
    if (r->q == r->out)
        return fail(LFM_EINVAL, "%s: out is q", op);
    return r->lse ? check_ptr(op, "rows->lse", r->lse, 4, dev) : LFM_OK;
}

static int check_workspace(const char *op, void *p, size_t have, size_t need, int dev)
{
    if (have < need)
        return fail(LFM_EINVAL, "%s: %zu bytes of workspace, %zu needed", op, have, need);
    return need ? check_ptr(op, "workspace", p, 16, dev) : LFM_OK;
}

static KvView view(const lfm_kv *c)
{
    KvView v;
    memset(&v, 0, sizeof(v));
    v.k = (const uint16_t *)c->k;
    v.v = (const uint16_t *)c->v;
    v.len = c->len;
    v.ss = c->seq_stride, v.hs = c->head_stride, v.ts = c->slot_stride;
    v.n_seq = c->n_seq, v.kv_heads = c->kv_heads, v.slots = c->slots;
    return v;
}

static RowsView view(const lfm_rows *r)
{
    RowsView v;
    memset(&v, 0, sizeof(v));
    v.q = r->q, v.out = r->out, v.lse = r->lse, v.start = r->start;
    v.q_rs = r->q_row_stride, v.q_hs = r->q_head_stride;
    v.o_rs = r->out_row_stride, v.o_hs = r->out_head_stride;
    v.heads = r->heads, v.n_rows = r->n_rows;
    // Kept a normal number at both ends of 32 bits, so that a masked score of -infinity and one of
    // 0 stay such; the scores of 16-bit rows are no others for it.
    const double c = (double)r->scale * 1.4426950408889634;
    v.cexp = (float)std::min(std::max(c, (double)FLT_MIN), (double)FLT_MAX);
    int cpow;
    v.cfrac = frexpf(v.cexp, &cpow);
    return v;
}

static size_t round256(size_t n) { return (n + 255) / 256 * 256; }

static int dim_index(const lfm_kv *c) { return c->head_dim == 128; }

// ------------------------------------------------------------------ attention
// How a call's work is cut, from sizes alone.
struct Plan {
    uint32_t own_splits = 1, prefix_splits = 0, own_groups = 1, prefix_groups = 0;
    bool most = false;      // the step kernel's larger form
    bool tile_most = false; // the tile kernel's
    bool tile_prefix = false; // the prefix goes through the tile kernel too
    uint64_t tile_items = 0;
    bool join = false; // a second kernel joins the key ranges
    uint32_t sum_parts = 1; // of the rows, in the slots' weights
    size_t ml_bytes = 0, o_bytes = 0, score_bytes = 0, stat_bytes = 0, sum_bytes = 0;
    size_t bytes() const { return ml_bytes + o_bytes + score_bytes + stat_bytes + sum_bytes; }
};


#define TARGET_GROUPS 512 // workgroups of four waves: two to a CU
#define MOST_RANGES 32    // key ranges of one kind: 64 lanes join a row's

static uint32_t ranges(uint64_t wanted, uint64_t worth)
{
    return (uint32_t)std::min<uint64_t>({std::max<uint64_t>(1, wanted), std::max<uint64_t>(1, worth), MOST_RANGES});
}

static uint32_t score_row(const lfm_kv *kv) { return (kv->slots + 31) / 32 * 32; }

static Plan plan(const lfm_kv *prefix, const lfm_kv *kv, const lfm_rows *r, uint32_t window, uint32_t sinks, bool scored)
{
    Plan p;
    const uint32_t G = r->heads / kv->kv_heads;
    const uint64_t pairs = (uint64_t)r->n_rows * r->heads;
    // from four tiles of 16 rows on, workgroups that share K and V in shared memory
    p.tile_prefix = prefix && (uint64_t)r->n_rows * G > 64;
    p.most = prefix && !p.tile_prefix ? (uint64_t)r->n_rows * G > 16 : G > 16;
    const uint32_t per = p.most ? 16 * step_tiles(kv->head_dim) : 16;
    if (!r->start) {
        const uint64_t span = window ? std::min<uint64_t>(kv->slots, (uint64_t)window + sinks + 63) : kv->slots;
        const uint64_t blocks = (span + 31) / 32;
        p.own_groups = (G + per - 1) / per;
        const uint64_t items = (uint64_t)std::max(1u, r->n_rows) * p.own_groups * kv->kv_heads;
        // A second launch that joins ranges takes 2-3 us: up to 512 slots one range is faster
        // (512 slots of one sequence, 64 dims, F16: 4.9 us against 6.0 in four ranges; 1024: 7.1
        // against 5.9 in eight; 128 dims: 7.6 and 7.1, 11.9 and 7.0), where no join follows
        // anyway.  A workgroup's four waves take a block of 32 each at least, two of a longer
        // cache (4096 slots: 7.5 us in 32 ranges, 7.0 in 16).
        if (scored || blocks > 16)
            p.own_splits = ranges(TARGET_GROUPS / items, blocks / (blocks > 64 ? 8 : 4));
    } else {
        // sequences end inside tiles: at most one more tile each
        const uint64_t cut = (uint64_t)r->n_rows * G;
        // The larger tile reads K and V half as often; it is taken where there are enough of
        // them to fill the CUs (a CU holds four at 64 dims, two at 128).  One prompt, 32 heads
        // over 8, small and large tile: 64 dims, 2048 tokens (512 large tiles) 38 and 43 us,
        // 2700 (675) 54 and 57, 3200 (800) 74 and 70, 8192 411 and 325; 128 dims, 1024 (256)
        // 27 and 32, 2048 65 and 60, 8192 789 and 584.
        const uint32_t most = 64 * TILE_TILES;
        p.tile_most = cut / most * kv->kv_heads >= (kv->head_dim == 64 ? 720 : 512);
        const uint64_t rows = p.tile_most ? most : 64;
        p.tile_items = cut / rows + std::min<uint64_t>(kv->n_seq, r->n_rows);
        const uint64_t span = window ? std::min<uint64_t>(kv->slots, (uint64_t)window + sinks + rows / G + 128)
                                     : kv->slots;
        p.own_splits = ranges(TARGET_GROUPS / std::max<uint64_t>(1, p.tile_items * kv->kv_heads), span / 512);
    }
    if (prefix) {
        const uint32_t rows = p.tile_prefix ? 64 * TILE_TILES : per;
        p.prefix_groups = (uint32_t)(((uint64_t)r->n_rows * G + rows - 1) / rows);
        const uint64_t pitems = (uint64_t)std::max(1u, p.prefix_groups) * kv->kv_heads;
        const uint64_t blocks = (prefix->slots + 31) / 32;
        uint64_t target = TARGET_GROUPS, least = blocks > 64 ? 8 : 4;
        if (p.tile_prefix) {
            // At 64 dims a CU holds four tiles: 600 rows over 32000 slots take 74 us as 480
            // tiles, 70 as 760, 73 as 1000.  A range of 16 blocks and more (8192 slots for 64
            // sequences: 60 us with 16, 70 with 8, which have to be joined); of 32 where the
            // sequences' own slots are read meanwhile for longer than the prefix takes (the
            // same: 53; where own and prefix are alike, 24 sequences of 2000 after 30000, 39 and 42).
            if (kv->head_dim == 64)
                target = TARGET_GROUPS * 3 / 2;
            if (blocks > 64)
                least = (uint64_t)r->n_rows * kv->slots >= 3 * (uint64_t)prefix->slots * p.prefix_groups ? 32 : 16;
        }
        p.prefix_splits = ranges(target / pitems, blocks / least);
    }
    const uint32_t splits = p.own_splits + p.prefix_splits;
    const bool steps = scored && !r->start; // scores are kept from the step to the join
    p.join = steps || splits > 1;
    if (p.join) {
        p.ml_bytes = round256((size_t)splits * pairs * 8);
        p.o_bytes = round256((size_t)splits * pairs * kv->head_dim * 4);
    }
    if (steps)
        p.score_bytes = round256((size_t)pairs * score_row(kv) * 4);
    else if (scored) {
        p.stat_bytes = round256((size_t)pairs * 8);
        // parts of eight steps of 64 pairs and more (one sequence's rows are at most all of them)
        const uint64_t groups = (uint64_t)((kv->slots + SUM_KEYS - 1) / SUM_KEYS) * kv->kv_heads * std::max(1u, kv->n_seq);
        p.sum_parts = (uint32_t)std::min<uint64_t>(
            {MOST_SUM_PARTS, std::max<uint64_t>(1, 2 * TARGET_GROUPS / groups),
             std::max<uint64_t>(1, (uint64_t)r->n_rows * G / 512)});
        if (p.sum_parts > 1)
            p.sum_bytes = round256((size_t)p.sum_parts * kv->n_seq * kv->kv_heads * kv->slots * 4);
    }
    return p;
}

static AttnOpArgs op_args(const Plan &p, const lfm_kv *prefix, const lfm_kv *kv, const lfm_rows *rows, uint32_t window,
                          uint32_t sinks, void *ws)
{
    AttnOpArgs a;
    memset(&a, 0, sizeof(a));
    a.own = view(kv);
    if (prefix)
        a.prefix = view(prefix);
    a.r = view(rows);
    a.window = window, a.sinks = sinks;
    a.group = rows->heads / kv->kv_heads;
    a.own_splits = p.own_splits, a.prefix_splits = p.prefix_splits;
    a.own_groups = p.own_groups, a.prefix_groups = p.prefix_groups;
    uint8_t *w = (uint8_t *)ws;
    a.ml = (float2 *)w;
    a.o = (float *)(w += p.ml_bytes);
    w += p.o_bytes;
    a.score_row = score_row(kv);
    a.scores = p.score_bytes ? (float *)w : nullptr;
    w += p.score_bytes;
    a.stats = p.stat_bytes ? (float2 *)w : nullptr;
    w += p.stat_bytes;
    a.sum_parts = p.sum_parts;
    a.sums = (float *)w;
    return a;
}

// Grids are flat, kv heads fastest: with 8 of them each XCD's cache serves one.
static int launch_items(hipFunction_t f, uint64_t items, uint32_t kv_heads, hipStream_t s, const AttnOpArgs &a)
{
    return launch(f, dim3((uint32_t)items * kv_heads), 256, s, a);
}

// Whether the grids of a call can be launched.
static int check_grids(const char *op, const Plan &p, const lfm_kv *kv, const lfm_rows *r, bool scored)
{
    const uint64_t most = std::max({(uint64_t)p.prefix_groups * p.prefix_splits +
                                        (r->start ? 0 : (uint64_t)r->n_rows * p.own_groups * p.own_splits),
                                    p.tile_items * p.own_splits,
                                    scored && r->start ? (uint64_t)(kv->slots + SUM_KEYS - 1) / SUM_KEYS : 0});
    if (most * kv->kv_heads > MOST_WORKGROUPS)
        return fail(LFM_EINVAL, "%s: %llu pieces of work for each of %u kv heads", op, (unsigned long long)most,
                    kv->kv_heads);
    return LFM_OK;
}

// Launches over (kv head, rows, key range): the prefix of many rows, then single rows (and the
// prefix of few), then rows of many tokens; then the ranges are joined.
static int attend(AttnKernels *K, const Plan &p, AttnOpArgs a, const lfm_kv *kv, const lfm_rows *rows,
                  hipStream_t s)
{
    const int t = rows->type, d = dim_index(kv);
    uint64_t steps = rows->start ? 0 : (uint64_t)rows->n_rows * p.own_groups * p.own_splits;
    a.step_prefix = 0;
    if (p.tile_prefix) {
        const uint64_t with = p.most ? 0 : steps; // in the same launch
        RC(launch_items(K->tile_prefix[t][d], (uint64_t)p.prefix_groups * p.prefix_splits + with, kv->kv_heads, s, a));
        steps -= with;
    } else {
        a.step_prefix = p.prefix_groups * p.prefix_splits;
        steps += a.step_prefix;
    }
    if (steps)
        RC(launch_items(p.most ? K->step_most[t][d] : K->step_1[t][d], steps, kv->kv_heads, s, a));
    if (rows->start)
        RC(launch_items(p.tile_most ? K->tile_most[t][d] : K->tile_1[t][d], p.tile_items * p.own_splits, kv->kv_heads,
                        s, a));
    if (a.scores)
        return launch(K->scored_join[t][d],
                      dim3((kv->slots + SCORED_SLOTS - 1) / SCORED_SLOTS, kv->kv_heads, kv->n_seq), 256, s, a);
    if (p.join)
        return launch(K->merge[t][d], dim3((rows->n_rows * rows->heads + 3) / 4), 256, s, a);
    return LFM_OK;
}

extern "C" int lfm_attn_window_workspace(const lfm_kv *kv, const lfm_rows *rows, uint32_t window, uint32_t sinks,
                                         size_t *bytes)
{
    const char *op = "lfm_attn_window_workspace";
    RC(check_kv(op, "kv", kv));
    RC(check_rows(op, kv, rows));
    if (!bytes)
        return fail(LFM_EINVAL, "%s: bytes is null", op);
    const Plan p = plan(nullptr, kv, rows, window, sinks, false);
    RC(check_grids(op, p, kv, rows, false));
    *bytes = p.bytes();
    return LFM_OK;
}

extern "C" int lfm_attn_window(const lfm_kv *kv, const lfm_rows *rows, uint32_t window, uint32_t sinks,
                               void *workspace, size_t workspace_bytes, void *stream)
{
    const char *op = "lfm_attn_window";
    size_t need;
    RC(lfm_attn_window_workspace(kv, rows, window, sinks, &need));
    if (rows->n_rows == 0 || kv->n_seq == 0)
        return LFM_OK;
    int dev;
    RC(current_device(op, (hipStream_t)stream, &dev));
    RC(check_kv_ptrs(op, KV_NAMES, kv, dev));
    RC(check_rows_ptrs(op, rows, dev));
    RC(check_workspace(op, workspace, workspace_bytes, need, dev));
    AttnKernels *K;
    RC(attn_kernels(dev, &K));
    const Plan p = plan(nullptr, kv, rows, window, sinks, false);
    return attend(K, p, op_args(p, nullptr, kv, rows, window, sinks, workspace), kv, rows, (hipStream_t)stream);
}

extern "C" int lfm_attn_scored_workspace(const lfm_kv *kv, const lfm_rows *rows, size_t *bytes)
{
    const char *op = "lfm_attn_scored_workspace";
    RC(check_kv(op, "kv", kv));
    RC(check_rows(op, kv, rows));
    if (!bytes)
        return fail(LFM_EINVAL, "%s: bytes is null", op);
    const Plan p = plan(nullptr, kv, rows, 0, 0, true);
    RC(check_grids(op, p, kv, rows, true));
    *bytes = p.bytes();
    return LFM_OK;
}

extern "C" int lfm_attn_scored(const lfm_kv *kv, const lfm_rows *rows, const float *acc_in, float *acc_out,
                               void *workspace, size_t workspace_bytes, void *stream)
{
    const char *op = "lfm_attn_scored";
    size_t need;
    RC(lfm_attn_scored_workspace(kv, rows, &need));
    if (kv->n_seq == 0)
        return LFM_OK;
    int dev;
    RC(current_device(op, (hipStream_t)stream, &dev));
    RC(check_kv_ptrs(op, KV_NAMES, kv, dev));
    RC(check_rows_ptrs(op, rows, dev));
    if (acc_in)
        RC(check_ptr(op, "acc_in", acc_in, 4, dev));
    RC(check_ptr(op, "acc_out", acc_out, 4, dev));
    RC(check_workspace(op, workspace, workspace_bytes, need, dev));
    hipStream_t s = (hipStream_t)stream;
    AttnKernels *K;
    RC(attn_kernels(dev, &K));
    const Plan p = plan(nullptr, kv, rows, 0, 0, true);
    AttnOpArgs a = op_args(p, nullptr, kv, rows, 0, 0, workspace);
    a.acc = acc_in, a.acc_out = acc_out;
    if (rows->n_rows)
        RC(attend(K, p, a, kv, rows, s));
    if (!rows->start)
        return LFM_OK;
    const uint32_t blocks = (kv->slots + SUM_KEYS - 1) / SUM_KEYS * kv->kv_heads;
    RC(launch(K->weights[rows->type][dim_index(kv)], dim3(blocks, kv->n_seq * p.sum_parts), 256, s, a));
    if (p.sum_parts == 1)
        return LFM_OK;
    return launch(K->sums, dim3((kv->slots + 255) / 256, kv->kv_heads, kv->n_seq), 256, s, a);
}

static int check_prefix(const char *op, const lfm_kv *prefix, const lfm_kv *kv)
{
    RC(check_kv(op, "prefix", prefix));
    RC(check_kv(op, "kv", kv));
    if (prefix->n_seq != 1)
        return fail(LFM_EINVAL, "%s: a prefix of %u sequences (1)", op, prefix->n_seq);
    if (prefix->kv_heads != kv->kv_heads || prefix->head_dim != kv->head_dim || prefix->type != kv->type)
        return fail(LFM_EINVAL, "%s: prefix and kv differ in kv_heads, head_dim or type", op);
    return LFM_OK;
}

extern "C" int lfm_attn_prefix_workspace(const lfm_kv *prefix, const lfm_kv *kv, const lfm_rows *rows, size_t *bytes)
{
    const char *op = "lfm_attn_prefix_workspace";
    RC(check_prefix(op, prefix, kv));
    RC(check_rows(op, kv, rows));
    if (!bytes)
        return fail(LFM_EINVAL, "%s: bytes is null", op);
    const Plan p = plan(prefix, kv, rows, 0, 0, false);
    RC(check_grids(op, p, kv, rows, false));
    *bytes = p.bytes();
    return LFM_OK;
}

extern "C" int lfm_attn_prefix(const lfm_kv *prefix, const lfm_kv *kv, const lfm_rows *rows, void *workspace,
                               size_t workspace_bytes, void *stream)
{
    const char *op = "lfm_attn_prefix";
    size_t need;
    RC(lfm_attn_prefix_workspace(prefix, kv, rows, &need));
    if (rows->n_rows == 0 || kv->n_seq == 0)
        return LFM_OK;
    int dev;
    RC(current_device(op, (hipStream_t)stream, &dev));
    RC(check_kv_ptrs(op, PREFIX_NAMES, prefix, dev));
    RC(check_kv_ptrs(op, KV_NAMES, kv, dev));
    RC(check_rows_ptrs(op, rows, dev));
    RC(check_workspace(op, workspace, workspace_bytes, need, dev));
    AttnKernels *K;
    RC(attn_kernels(dev, &K));
    const Plan p = plan(prefix, kv, rows, 0, 0, false);
    return attend(K, p, op_args(p, prefix, kv, rows, 0, 0, workspace), kv, rows, (hipStream_t)stream);
}

// ------------------------------------------------------------------ eviction
static size_t evict_list_bytes(const lfm_kv *kv, uint32_t keep)
{
    return ((size_t)kv->n_seq * kv->kv_heads * keep * 4 + 255) / 256 * 256;
}

extern "C" int lfm_kv_evict_workspace(const lfm_kv *kv, uint32_t keep, size_t *bytes)
{
    const char *op = "lfm_kv_evict_workspace";
    RC(check_kv(op, "kv", kv));
    if (keep == 0 || keep > 0x10000000u)
        return fail(LFM_EINVAL, "%s: keep %u (1..2^28)", op, keep);
    if (!bytes)
        return fail(LFM_EINVAL, "%s: bytes is null", op);
    *bytes = 2 * evict_list_bytes(kv, keep) + (size_t)kv->n_seq * kv->kv_heads * 8;
    return LFM_OK;
}

extern "C" int lfm_kv_evict(const lfm_kv *kv, const float *acc, const int32_t *pos, uint32_t keep, uint32_t sinks,
                            uint32_t recent, const lfm_kv *out, float *acc_out, int32_t *pos_out, void *workspace,
                            size_t workspace_bytes, void *stream)
{
    const char *op = "lfm_kv_evict";
    size_t need;
    RC(lfm_kv_evict_workspace(kv, keep, &need));
    RC(check_kv(op, "out", out));
    if (out->n_seq != kv->n_seq || out->kv_heads != kv->kv_heads || out->head_dim != kv->head_dim ||
        out->type != kv->type)
        return fail(LFM_EINVAL, "%s: out and kv differ in n_seq, kv_heads, head_dim or type", op);
    if ((uint64_t)sinks + recent > keep)
        return fail(LFM_EINVAL, "%s: sinks %u and recent %u do not fit into keep %u", op, sinks, recent, keep);
    if (keep > out->slots)
        return fail(LFM_EINVAL, "%s: keep %u, out holds %u slots", op, keep, out->slots);
    const bool in_place = out->k == kv->k;
    if (in_place != (out->v == kv->v) ||
        (in_place && (out->seq_stride != kv->seq_stride || out->head_stride != kv->head_stride ||
                      out->slot_stride != kv->slot_stride)))
        return fail(LFM_EINVAL, "%s: in place needs both k and v, with the same strides", op);
    if (((acc_out == acc && acc) || (pos_out == pos && pos)) && out->slots != kv->slots)
        return fail(LFM_EINVAL, "%s: acc or pos in place needs out of %u slots", op, kv->slots);
    if ((out->n_seq > 1 && out->seq_stride == 0) || (out->kv_heads > 1 && out->head_stride == 0) ||
        (keep > 1 && out->slot_stride == 0))
        return fail(LFM_EINVAL, "%s: out has a stride of 0", op);
    if (kv->n_seq == 0)
        return LFM_OK;
    int dev;
    RC(current_device(op, (hipStream_t)stream, &dev));
    RC(check_kv_ptrs(op, KV_NAMES, kv, dev));
    RC(check_kv_ptrs(op, OUT_NAMES, out, dev));
    RC(check_ptr(op, "acc", acc, 4, dev));
    RC(check_ptr(op, "pos", pos, 4, dev));
    RC(check_ptr(op, "acc_out", acc_out, 4, dev));
    RC(check_ptr(op, "pos_out", pos_out, 4, dev));
    RC(check_workspace(op, workspace, workspace_bytes, need, dev));
    AttnKernels *K;
    RC(attn_kernels(dev, &K));
    EvictArgs a;
    memset(&a, 0, sizeof(a));
    a.c = view(kv);
    a.k_out = out->k, a.v_out = out->v;
    a.oss = out->seq_stride, a.ohs = out->head_stride, a.ots = out->slot_stride;
    a.acc = acc, a.pos = pos, a.acc_out = acc_out, a.pos_out = pos_out, a.len_out = out->len;
    a.keep = keep, a.sinks = sinks, a.recent = recent, a.out_slots = out->slots, a.dim = kv->head_dim;
    a.in_place = in_place, a.acc_in_place = acc == acc_out, a.pos_in_place = pos == pos_out;
    a.map = (int32_t *)workspace;
    a.movers = (int32_t *)((uint8_t *)workspace + evict_list_bytes(kv, keep));
    a.head = (int32_t *)((uint8_t *)workspace + 2 * evict_list_bytes(kv, keep));
    RC(launch(K->kv_select, dim3(kv->kv_heads, kv->n_seq), 1024, (hipStream_t)stream, a));
    return launch(K->kv_move, dim3((keep + 31) / 32, kv->kv_heads, kv->n_seq), 256, (hipStream_t)stream, a);
}
