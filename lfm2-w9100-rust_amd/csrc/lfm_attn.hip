// lfm_attn.hip -- attention over key/value caches as operators: a sliding window with first
// tokens that stay visible, accumulated attention weights, a shared prefix, and the
// eviction of cache slots.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_args.h"
#include "wave_ops.h"

struct F32 {
    typedef float type;
};
struct F16 {
    typedef _Float16 type;
};
struct BF16 {
    typedef __bf16 type;
};

__device__ __forceinline__ int32_t clamp_len(const KvView &c, uint32_t b)
{
    return max(0, min(c.len[b], (int32_t)c.slots));
}

// Rows [lo, hi) of a sequence.
__device__ __forceinline__ void seq_rows(const RowsView &r, uint32_t b, int32_t *lo, int32_t *hi)
{
    if (!r.start) {
        *lo = (int32_t)b;
        *hi = (int32_t)b + 1;
        return;
    }
    *lo = max(0, min(r.start[b], (int32_t)r.n_rows));
    *hi = max(*lo, min(r.start[b + 1], (int32_t)r.n_rows));
}

// Sequence and position of a row; false where the row belongs to none.
__device__ __forceinline__ bool find_row(const AttnOpArgs &a, uint32_t row, uint32_t *b, int32_t *pos)
{
    if (!a.r.start) {
        *b = row;
        *pos = clamp_len(a.own, row) - 1;
        return true;
    }
    for (uint32_t s = 0; s < a.own.n_seq; ++s) {
        int32_t lo, hi;
        seq_rows(a.r, s, &lo, &hi);
        if ((int32_t)row >= lo && (int32_t)row < hi) {
            *b = s;
            *pos = clamp_len(a.own, s) - hi + (int32_t)row;
            return true;
        }
    }
    return false;
}

// One wave per row and head: 64 slots at a time, a lane's score each, then every lane its
// dims of the weighted sum.
template <typename TQ, typename TK, int D> __device__ void attn_simple(const AttnOpArgs &a)
{
    typedef typename TQ::type tq;
    typedef typename TK::type tk;
    const uint32_t row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, kh = h / (a.r.heads / a.own.kv_heads);
    uint32_t b;
    int32_t pos;
    if (!find_row(a, row, &b, &pos))
        return;
    __shared__ float qs[D], ps[64];
    for (int d = lane; d < D; d += 64)
        qs[d] = (float)((const tq *)a.r.q)[(int64_t)row * a.r.q_rs + (int64_t)h * a.r.q_hs + d];
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[D / 64];
    for (int i = 0; i < D / 64; ++i)
        o[i] = 0.f;
    for (int part = 0; part < 2; ++part) {
        if (part == 0 && !a.prefix.k)
            continue;
        const KvView &c = part ? a.own : a.prefix;
        const int32_t n = part ? pos + 1 : clamp_len(c, 0);
        const int64_t base = (part ? (int64_t)b * c.ss : 0) + (int64_t)kh * c.hs;
        const tk *k = (const tk *)c.k + base, *v = (const tk *)c.v + base;
        for (int32_t j0 = 0; j0 < n; j0 += 64) {
            const int32_t j = j0 + (int32_t)lane;
            bool seen = j < n;
            if (part && a.window)
                seen = seen && (j < (int64_t)a.sinks || j > (int64_t)pos - a.window);
            float s = -INFINITY;
            if (seen) {
                s = 0.f;
                for (int d = 0; d < D; ++d)
                    s += qs[d] * (float)k[(int64_t)j * c.ts + d];
            }
            const uint64_t any = __ballot(seen);
            if (!any)
                continue;
            const float mn = fmaxf(m, wave_max(s));
            const float r = m > -INFINITY ? exp2f((m - mn) * a.r.cexp) : 0.f;
            const float p = seen ? exp2f((s - mn) * a.r.cexp) : 0.f;
            l = l * r + wave_sum(p);
            m = mn;
            __syncthreads();
            ps[lane] = p;
            __syncthreads();
            for (int i = 0; i < D / 64; ++i)
                o[i] *= r;
            for (int jj = 0; jj < 64; ++jj)
                if ((any >> jj) & 1)
                    for (int i = 0; i < D / 64; ++i)
                        o[i] += ps[jj] * (float)v[(int64_t)(j0 + jj) * c.ts + lane + 64 * i];
        }
    }
    const bool empty = pos < 0 && (!a.prefix.k || clamp_len(a.prefix, 0) == 0);
    for (int i = 0; i < D / 64; ++i)
        ((tq *)a.r.out)[(int64_t)row * a.r.o_rs + (int64_t)h * a.r.o_hs + lane + 64 * i] =
            (tq)(empty ? 0.f : o[i] / l);
    if (a.r.lse && lane == 0)
        a.r.lse[(size_t)row * a.r.heads + h] = empty ? -INFINITY : m * a.r.scale + logf(l);
}

// One wave per 64 slots of a (sequence, kv head): a lane adds the weights its slot gets
// from every row and head, in order.
template <typename TQ, typename TK, int D> __device__ void colsum_simple(const ColsumArgs &a)
{
    typedef typename TQ::type tq;
    typedef typename TK::type tk;
    const uint32_t kh = blockIdx.y, b = blockIdx.z, G = a.r.heads / a.own.kv_heads;
    const int32_t n = clamp_len(a.own, b), j = (int32_t)(blockIdx.x * 64 + threadIdx.x);
    if (j >= n)
        return;
    int32_t lo, hi;
    seq_rows(a.r, b, &lo, &hi);
    const tk *k = (const tk *)a.own.k + (int64_t)b * a.own.ss + (int64_t)kh * a.own.hs + (int64_t)j * a.own.ts;
    float sum = 0.f;
    for (int32_t row = lo; row < hi; ++row) {
        if (j > n - hi + row)
            continue;
        for (uint32_t g = 0; g < G; ++g) {
            const uint32_t h = kh * G + g;
            const tq *q = (const tq *)a.r.q + (int64_t)row * a.r.q_rs + (int64_t)h * a.r.q_hs;
            float s = 0.f;
            for (int d = 0; d < D; ++d)
                s += (float)q[d] * (float)k[d];
            sum += expf(s * a.r.scale - a.r.lse[(size_t)row * a.r.heads + h]);
        }
    }
    const size_t at = ((size_t)b * a.own.kv_heads + kh) * a.own.slots + j;
    a.acc_out[at] = (a.acc ? a.acc[at] : 0.f) + sum;
}

#define INSTANCES(TQ, TK, tag, D)                                                                              \
    extern "C" __global__ __launch_bounds__(64) void k_attn_simple_##tag##_##D(const AttnOpArgs a)             \
    {                                                                                                          \
        attn_simple<TQ, TK, D>(a);                                                                             \
    }                                                                                                          \
    extern "C" __global__ __launch_bounds__(64) void k_colsum_simple_##tag##_##D(const ColsumArgs a)           \
    {                                                                                                          \
        colsum_simple<TQ, TK, D>(a);                                                                           \
    }
INSTANCES(F32, F16, f32, 64)
INSTANCES(F32, F16, f32, 128)
INSTANCES(F16, F16, f16, 64)
INSTANCES(F16, F16, f16, 128)
INSTANCES(BF16, BF16, bf16, 64)
INSTANCES(BF16, BF16, bf16, 128)

// ------------------------------------------------------------------ eviction
// Rank of a slot as an integer: NaN below every number, the protected slots above all.
__device__ __forceinline__ uint32_t evict_key(const EvictArgs &a, float acc, int32_t pos, int64_t newest)
{
    if (pos < (int64_t)a.sinks || (int64_t)pos > newest - a.recent)
        return 0xFFFFFFFFu;
    if (acc != acc)
        return 0u;
    const uint32_t u = __float_as_uint(acc + 0.0f); // -0 ranks as 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

#define SEL_THREADS 1024
// The `keep` slots of highest rank of one (sequence, kv head), ties to the lowest slot:
// the rank of the last one by four 8-bit histograms from the top, then each wave counts
// and places its own run of slots.
extern "C" __global__ __launch_bounds__(SEL_THREADS) void k_kv_select(const EvictArgs a)
{
    const uint32_t kh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const size_t bh = (size_t)b * a.c.kv_heads + kh;
    const uint32_t n = (uint32_t)clamp_len(a.c, b), keep = a.keep;
    if (tid == 0) {
        a.head[2 * bh] = (int32_t)min(n, keep);
        a.head[2 * bh + 1] = n > keep;
    }
    if (n <= keep)
        return;
    const float *acc = a.acc + bh * a.c.slots;
    const int32_t *pos = a.pos + bh * a.c.slots;
    int32_t *map = a.map + bh * keep, *movers = a.movers + bh * keep;
    __shared__ uint32_t hist[256];
    __shared__ int32_t wmax[16];
    __shared__ uint32_t sh_prefix, sh_need, cnt_eq[16], cnt_hole[16], cnt_move[16];
    int32_t newest = INT32_MIN;
    for (uint32_t j = tid; j < n; j += SEL_THREADS)
        newest = max(newest, pos[j]);
    newest = wave_max_i(newest);
    if (lane == 0)
        wmax[wave] = newest;
    if (tid == 0)
        sh_prefix = 0, sh_need = keep;
    __syncthreads();
    for (int w = 0; w < 16; ++w)
        newest = max(newest, wmax[w]);
    for (int pass = 3; pass >= 0; --pass) {
        if (tid < 256)
            hist[tid] = 0;
        __syncthreads();
        const uint32_t prefix = sh_prefix, mask = pass == 3 ? 0u : 0xFFFFFFFFu << (8 * (pass + 1));
        for (uint32_t j = tid; j < n; j += SEL_THREADS) {
            const uint32_t k = evict_key(a, acc[j], pos[j], newest);
            if ((k & mask) == prefix)
                atomicAdd(&hist[(k >> (8 * pass)) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t need = sh_need;
            int d = 255;
            for (; d > 0 && hist[d] < need; --d)
                need -= hist[d];
            sh_prefix = prefix | (uint32_t)d << (8 * pass);
            sh_need = need;
        }
        __syncthreads();
    }
    const uint32_t last = sh_prefix, need = sh_need; // the need lowest slots of rank `last` stay
    const uint32_t run = ((n + 15) / 16 + 63) / 64 * 64, j0 = wave * run, j1 = min(n, j0 + run);
    const uint64_t below = (1ull << lane) - 1;
    uint32_t eq = 0;
    for (uint32_t j = j0; j < j1; j += 64) {
        const bool in = j + lane < j1;
        const uint32_t k = in ? evict_key(a, acc[j + lane], pos[j + lane], newest) : 0;
        eq += __popcll(__ballot(in && k == last));
    }
    if (lane == 0)
        cnt_eq[wave] = eq;
    __syncthreads();
    uint32_t eq0 = 0;
    for (uint32_t w = 0; w < wave; ++w)
        eq0 += cnt_eq[w];
    uint32_t holes = 0, moves = 0, hole0 = 0, move0 = 0;
    for (int place = 0; place < 2; ++place) {
        uint32_t e = eq0;
        for (uint32_t j = j0; j < j1; j += 64) {
            const uint32_t s = j + lane;
            const bool in = s < j1;
            const uint32_t k = in ? evict_key(a, acc[s], pos[s], newest) : 0;
            const uint64_t meq = __ballot(in && k == last);
            const bool kept = in && (k > last || (k == last && e + __popcll(meq & below) < need));
            e += __popcll(meq);
            const uint64_t mh = __ballot(in && s < keep && !kept), mm = __ballot(s >= keep && kept);
            if (place) {
                if (in && s < keep)
                    map[s] = kept ? (int32_t)s : ~(int32_t)(hole0 + holes + __popcll(mh & below));
                else if (kept)
                    movers[move0 + moves + __popcll(mm & below)] = (int32_t)s;
            }
            holes += __popcll(mh);
            moves += __popcll(mm);
        }
        if (place)
            break;
        if (lane == 0)
            cnt_hole[wave] = holes, cnt_move[wave] = moves;
        __syncthreads();
        for (uint32_t w = 0; w < wave; ++w)
            hole0 += cnt_hole[w], move0 += cnt_move[w];
        holes = moves = 0;
    }
}

#define MOVE_ROWS 32
// Copies `keep` slots (in place: only the moved ones) of one (sequence, kv head), 32 per
// workgroup, 16 bytes a lane.  A moved slot's source is at or past `keep` and its target
// below: in place, nothing is read that another thread writes.
extern "C" __global__ __launch_bounds__(256) void k_kv_move(const EvictArgs a)
{
    const uint32_t kh = blockIdx.y, b = blockIdx.z, n0 = blockIdx.x * MOVE_ROWS;
    const size_t bh = (size_t)b * a.c.kv_heads + kh;
    const uint32_t remain = (uint32_t)a.head[2 * bh];
    const bool evicts = a.head[2 * bh + 1]; // else every slot stays where it is
    const int32_t *map = a.map + bh * a.keep, *movers = a.movers + bh * a.keep;
    if (blockIdx.x == 0 && kh == 0 && threadIdx.x == 0)
        a.len_out[b] = (int32_t)remain;
    const uint32_t lanes = a.dim / 8, per = 256 / lanes, piece = threadIdx.x % lanes;
    for (uint32_t i = threadIdx.x / lanes; i < MOVE_ROWS; i += per) {
        const uint32_t n = n0 + i;
        if (n >= remain)
            return;
        int32_t s = evicts ? map[n] : (int32_t)n;
        if (s < 0)
            s = movers[~s];
        const bool moved = (uint32_t)s != n;
        if (moved || !a.in_place) {
            const int64_t from = (int64_t)b * a.c.ss + (int64_t)kh * a.c.hs + (int64_t)s * a.c.ts + piece * 8;
            const int64_t to = (int64_t)b * a.oss + (int64_t)kh * a.ohs + (int64_t)n * a.ots + piece * 8;
            const uint4 k = *(const uint4 *)(a.c.k + from), v = *(const uint4 *)(a.c.v + from);
            *(uint4 *)((uint16_t *)a.k_out + to) = k;
            *(uint4 *)((uint16_t *)a.v_out + to) = v;
        }
        if (piece == 0) {
            const size_t src = bh * a.c.slots + (uint32_t)s, dst = bh * a.out_slots + n;
            if (moved || !a.acc_in_place)
                a.acc_out[dst] = a.acc[src];
            if (moved || !a.pos_in_place)
                a.pos_out[dst] = a.pos[src];
        }
    }
}
