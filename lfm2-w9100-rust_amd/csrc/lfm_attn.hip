// lfm_attn.hip -- attention over key/value caches as operators: a sliding window with first
// tokens that stay visible, accumulated attention weights, a shared prefix, and the
// eviction of cache slots.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_args.h"
#include "wave_ops.h"

template <int N> struct Const {
    static constexpr int value = N;
};

// ------------------------------------------------------------------ types
// Queries and weights meet K and V on the 16x16x32 matrix instruction: lane l holds 8
// numbers of row (A) or column (B) l % 16, at inner places 8 (l / 16) + i, and 4 results,
// rows 4 (l / 16) + e of column l % 16.
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4v lds_short4;

struct F16 {
    typedef _Float16 type, kv;
    typedef f16x8 vec;
    static constexpr int parts = 1;
    // A weight is 2^7 or more times its value relative to the largest (see Weights), so that
    // binary16's subnormals start 21 binary orders below it and not 14.
    static constexpr float offset = 7.f;
};
struct F32 { // rows of 32 bits over a binary16 cache: two binary16 numbers each, 22 bits
    typedef float type;
    typedef _Float16 kv;
    typedef f16x8 vec;
    static constexpr int parts = 2;
    static constexpr float offset = 7.f;
};
struct BF16 {
    typedef __bf16 type, kv;
    typedef bf16x8 vec;
    static constexpr int parts = 1;
    static constexpr float offset = 0.f; // the exponent has 8 bits
};

__device__ __forceinline__ floatx4 mma(f16x8 a, f16x8 b, floatx4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mma(bf16x8 a, bf16x8 b, floatx4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Largest and sum of a value over the lanes l, l ^ 16, l ^ 32, l ^ 48 (one query row).
__device__ __forceinline__ float quarter_other(float v)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t lo = r[0], hi = r[1];
    return (threadIdx.x & 16) ? __builtin_bit_cast(float, lo) : __builtin_bit_cast(float, hi);
}
__device__ __forceinline__ float row_max(float v)
{
    v = fmaxf(v, quarter_other(v));
    const float2v h = wave_halves(v);
    return fmaxf(h[0], h[1]);
}
__device__ __forceinline__ float row_sum(float v)
{
    v += quarter_other(v);
    const float2v h = wave_halves(v);
    return h[0] + h[1];
}

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

// Sequence and position of a row, the same for a whole wave; false where the row belongs to
// no sequence.
__device__ __forceinline__ bool find_row(const AttnOpArgs &a, uint32_t row, uint32_t *b, int32_t *pos)
{
    if (!a.r.start) {
        *b = row;
        *pos = clamp_len(a.own, row) - 1;
        return true;
    }
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t s0 = 0; s0 < a.own.n_seq; s0 += 64) {
        int32_t lo = 0, hi = 0;
        if (s0 + lane < a.own.n_seq)
            seq_rows(a.r, s0 + lane, &lo, &hi);
        const uint64_t in = __ballot((int32_t)row >= lo && (int32_t)row < hi);
        if (in) {
            const uint32_t at = (uint32_t)__ffsll((unsigned long long)in) - 1;
            *b = s0 + at;
            *pos = clamp_len(a.own, *b) - __builtin_amdgcn_readlane(hi, at) + (int32_t)row;
            return true;
        }
    }
    return false;
}

// An output before its rounding to the rows' type.  A mean of binary16 numbers is no larger than
// the largest of them, but rounded weights may carry it past that, from where it would round to an
// infinity.  (An infinity that V holds stays one.)
template <typename TQ> __device__ __forceinline__ float in_range(float v)
{
    constexpr float MOST = 65504.f;
    if constexpr (__is_same(typename TQ::type, _Float16))
        return fabsf(v) < INFINITY ? fminf(fmaxf(v, -MOST), MOST) : v;
    return v;
}

// Four outputs of a row and head, rounded to the rows' type.
template <typename TQ>
__device__ __forceinline__ void store_out(const RowsView &r, uint32_t row, uint32_t h, uint32_t d, floatx4 v)
{
#pragma unroll
    for (int e = 0; e < 4; ++e)
        v[e] = in_range<TQ>(v[e]);
    typedef typename TQ::type tq;
    typedef tq tq4 __attribute__((ext_vector_type(4)));
    *(tq4 *)((tq *)r.out + (int64_t)row * r.o_rs + (int64_t)h * r.o_hs + d) = __builtin_convertvector(v, tq4);
}

// ------------------------------------------------------------------ rows in matrix form
// Pairs of a row and one of a kv head's G query heads, counted through: pair x after
// (row, rem) is row + (rem + x) / G, head (rem + x) % G.  rem + x stays below 384, where the
// product with ceil(2^16 / G) gives the quotient exactly (G <= 128).
struct Pairs {
    uint32_t row, rem, G, inv;
    __device__ __forceinline__ Pairs(uint32_t first_row, uint32_t pair, uint32_t group)
    {
        G = group;
        inv = (65535 + G) / G;
        const uint32_t q = G == 1 ? pair : pair / G;
        row = first_row + q;
        rem = pair - q * G;
    }
    __device__ __forceinline__ uint32_t row_of(uint32_t x) const { return row + (((rem + x) * inv) >> 16); }
    __device__ __forceinline__ uint32_t head_of(uint32_t x) const
    {
        const uint32_t y = rem + x;
        return y - ((y * inv) >> 16) * G;
    }
};

// RT tiles of 16 query rows as B operands (the lane's row: lane % 16).  An F32 row is scaled
// by the power of two that brings its largest value into binary16's range, and its scores
// back by c = cfrac * back.
template <typename TQ, int D, int RT> struct Queries {
    static constexpr int N = TQ::parts == 2 ? RT : 1;
    typename TQ::vec q[RT][TQ::parts][D / 32];
    float c[N], back[N];
    __device__ __forceinline__ float c_of(int t) const { return c[N == 1 ? 0 : t]; }
};

__device__ __forceinline__ int power_up(float top)
{
    int ex = 14;
    if (top > 0.f && top < INFINITY)
        frexpf(top, &ex);
    return min(14 - ex, 126);
}

// 2^cpow over the power that a row was scaled by.  Row and scale may each be far out of the
// scores' range: the two powers meet here first, and where their quotient would be no normal
// number (the scores are 0 or past 32 bits then) it stays one, so that a masked score remains
// an infinity and no 0 becomes NaN.
__device__ __forceinline__ float power_back(const RowsView &r, int up)
{
    int cpow;
    frexpf(r.cexp, &cpow);
    return ldexpf(1.f, max(-125, min(cpow - up, 127)));
}

template <typename TQ, int D, int RT>
__device__ __forceinline__ void load_row(Queries<TQ, D, RT> &Q, int t, const RowsView &r, bool valid, uint32_t row,
                                         uint32_t h)
{
    typedef typename TQ::type tq;
    const uint32_t g = (threadIdx.x & 63) >> 4;
    const tq *p = (const tq *)r.q + (int64_t)row * r.q_rs + (int64_t)h * r.q_hs + 8 * g;
    if constexpr (TQ::parts == 1) {
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            typename TQ::vec v = {};
            if (valid)
                v = *(const typename TQ::vec *)(p + 32 * j);
            Q.q[t][0][j] = v;
        }
        Q.c[0] = r.cexp;
    } else {
        float x[D / 32][8], top = 0.f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            floatx4 a = {}, b = {};
            if (valid) {
                a = *(const floatx4 *)(p + 32 * j);
                b = *(const floatx4 *)(p + 32 * j + 4);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[j][i] = a[i], x[j][4 + i] = b[i];
                top = fmaxf(top, fmaxf(fabsf(a[i]), fabsf(b[i])));
            }
        }
        top = row_max(top);
        const int up = power_up(top);
        const float s = ldexpf(1.f, up);
        Q.back[t] = power_back(r, up);
        Q.c[t] = r.cfrac * Q.back[t];
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = x[j][i] * s;
                const _Float16 hi = (_Float16)y;
                Q.q[t][0][j][i] = hi;
                Q.q[t][1][j][i] = (_Float16)(y - (float)hi);
            }
    }
}

// ------------------------------------------------------------------ softmax state
// Of RT tiles of 16 rows: o[t][n] are dims 16 n + 4 (lane / 16) + e of row lane % 16, l the
// lane's own part of the sum of the weights 2^(s c - mc), whose four parts are added at the
// end.  mc is UNSEEN while no number was seen: then the weight of any number is infinite.
#define UNSEEN (-3.4028235e38f)
template <typename TQ, int D, int RT> struct State {
    floatx4 o[RT][D / 16];
    float mc[RT], l[RT];
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
                o[t][n] = floatx4{0.f, 0.f, 0.f, 0.f};
            mc[t] = UNSEEN, l[t] = 0.f;
        }
    }
    __device__ __forceinline__ bool seen(int t) const { return mc[t] > UNSEEN; }
    // for joining: -inf where there is nothing to join
    __device__ __forceinline__ float offset(int t) const { return seen(t) ? mc[t] : -INFINITY; }
};

// Scores of 32 slots and NT row tiles (s[t][0]: slots 4 (lane / 16) + e, s[t][1]: the same +
// 16) -> weights as B operands: inner place 8 (lane / 16) + i is slot 16 (i / 4) + 4 (lane /
// 16) + i % 4.  The largest weight is 2^offset when mc is set, and mc follows the scores only
// when the weights of a lane's eight slots pass that by RISE binary orders together: after
// the first block hardly ever, and a weight stays at or below 2^15.  So their sum, which is
// needed anyway, stands for the maximum (2700 tokens of 64 dims 54.8 us with it, 53.1 without).
// Two tiles share a check, where four would keep more in registers than there are.
//
// The matrix instruction takes V and the weights as 16-bit numbers, so a weight is rounded to 11 or
// 8 bits, half a step of the rows' own type, while the sum keeps 32: outputs of 16-bit rows are
// 1.3 to 1.4 times as far from 64 bits as their own rounding alone.  Two numbers a weight would
// double the products with V; F32 rows, whose outputs would show it, have them (22 bits).
#define RISE 8.f
template <int NT, typename TQ, int D, int RT>
__device__ __forceinline__ void weigh(State<TQ, D, RT> &S, const floatx4 (&s)[RT][2], const Queries<TQ, D, RT> &Q,
                                      typename TQ::vec (&p)[RT][TQ::parts])
{
    constexpr float MOST = 1 << (int)(TQ::offset + RISE);
    constexpr int AT_ONCE = NT < 2 ? NT : 2;
    typedef typename TQ::kv kv2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int t0 = 0; t0 < NT; t0 += AT_ONCE) {
        float w[AT_ONCE][8], sum[AT_ONCE];
        bool passes = false;
        auto weights = [&](int u) {
            const int t = t0 + u;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                w[u][i] = exp2_hw(fmaf(s[t][i / 4][i % 4], Q.c_of(t), -S.mc[t]));
            sum[u] = ((w[u][0] + w[u][1]) + (w[u][2] + w[u][3])) + ((w[u][4] + w[u][5]) + (w[u][6] + w[u][7]));
        };
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            weights(u);
            passes |= !(sum[u] <= MOST);
        }
        if (__ballot(passes)) {
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int t = t0 + u;
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    top = fmaxf(top, s[t][i / 4][i % 4] * Q.c_of(t));
                const float mc = fmaxf(S.mc[t], row_max(top) - TQ::offset),
                            r = S.seen(t) ? exp2_hw(S.mc[t] - mc) : 1.f;
                S.mc[t] = mc, S.l[t] *= r;
#pragma unroll
                for (int n = 0; n < D / 16; ++n)
                    S.o[t][n] *= r;
                weights(u);
            }
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int t = t0 + u;
            S.l[t] += sum[u];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const kv2 hi = __builtin_convertvector((float2v){w[u][i], w[u][i + 1]}, kv2);
                p[t][0][i] = hi[0], p[t][0][i + 1] = hi[1];
                if constexpr (TQ::parts == 2) {
                    const float2v back = __builtin_convertvector(hi, float2v);
                    const kv2 lo = __builtin_convertvector((float2v){w[u][i] - back[0], w[u][i + 1] - back[1]}, kv2);
                    p[t][1][i] = lo[0], p[t][1][i + 1] = lo[1];
                }
            }
        }
    }
}

// ------------------------------------------------------------------ V in shared memory
// 32 rows of D, each row's 16-byte pieces in the order piece ^ (row % pieces), so that the
// 16 rows that a transposed read touches lie in different banks.
template <int D> __device__ __forceinline__ uint32_t v_piece(uint32_t row, uint32_t piece)
{
    return row * (D / 8) + (piece ^ (row & (D / 8 - 1)));
}

// The lane's address for transposed_read: row 4 (lane / 16) + (lane % 16) / 4, dims 4 (lane % 4).
template <int D> __device__ __forceinline__ uint32_t v_lane(uint32_t lane)
{
    const uint32_t row = 4 * (lane >> 4) + ((lane & 15) >> 2);
    return v_piece<D>(row, (lane & 3) >> 1) * 16 + (lane & 1) * 8;
}

// V^T of dims 16 n .. 16 n + 15 as an A operand in the order of weigh(): two transposed
// reads, each giving the lane dim 16 n + lane % 16 of four rows.
template <typename TQ, int D>
__device__ __forceinline__ typename TQ::vec v_operand(const uint8_t *tile, uint32_t at, int n)
{
    const uint8_t *p = tile + (at ^ (uint32_t)(n << 5));
    const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)p);
    const short4v b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(p + 16 * D * 2));
    const short8v v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return __builtin_bit_cast(typename TQ::vec, v);
}

// ------------------------------------------------------------------ visible blocks
// Blocks of N slots that rows at positions lo .. hi see: those of the first tokens, then
// those of the window (all in one run where the two meet).  A slot is taken to be seen where
// the earliest row's window and the latest row's position allow it; with lo and hi exchanged,
// where every row does.
template <int N> struct Blocks {
    uint32_t hi, wlo, sinks; // slot j: j < hi and (j < sinks or j >= wlo)
    uint32_t first, skip, count;
    __device__ __forceinline__ void set(int32_t pos_lo, int32_t pos_hi, uint32_t window, uint32_t s)
    {
        hi = (uint32_t)max(pos_hi + 1, 0);
        const uint32_t end = (uint32_t)max(pos_lo + 1, 0);
        wlo = window && window < end ? end - window : 0;
        if (s >= wlo)
            wlo = 0;
        sinks = wlo ? s : 0;
        first = (min(sinks, hi) + N - 1) / N;
        const uint32_t from = max(wlo / N, first);
        skip = from - first;
        count = max((hi + N - 1) / N, from) - skip;
    }
    __device__ __forceinline__ uint32_t block(uint32_t i) const { return i < first ? i : i + skip; }
    __device__ __forceinline__ bool seen(uint32_t j) const { return j < hi && (j < sinks || j >= wlo); }
    __device__ __forceinline__ bool covers(uint32_t j, uint32_t n) const
    {
        return j + n <= hi && (j + n <= sinks || j >= wlo);
    }
    __device__ __forceinline__ bool touches(uint32_t j, uint32_t n) const
    {
        return j < hi && (j < sinks || j + n > wlo);
    }
    __device__ __forceinline__ bool whole(uint32_t blk) const { return covers(blk * N, N); }
};

// A key range's share [lo, hi) of n blocks.
__device__ __forceinline__ void share(uint32_t n, uint32_t part, uint32_t parts, uint32_t *lo, uint32_t *hi)
{
    if (parts == 1) {
        *lo = 0, *hi = n;
        return;
    }
    const uint32_t each = n / parts, more = n - each * parts;
    *lo = each * part + min(part, more);
    *hi = *lo + each + (part < more);
}

// 1 / l by the hardware (one unit in the last place of 32 bits).
__device__ __forceinline__ float inverse(float l) { return __builtin_amdgcn_rcpf(l); }

// A row's state once it is whole: its lse, and what attn_weights needs of it.
__device__ __forceinline__ void finish_row(const AttnOpArgs &a, size_t id, bool empty, float offset, float l)
{
    if (a.r.lse)
        a.r.lse[id] = empty ? -INFINITY : (offset + log2f(l)) * 0.6931471805599453f;
    if (a.stats)
        a.stats[id] = empty ? make_float2(0.f, 0.f) : make_float2(offset, inverse(l));
}

// ------------------------------------------------------------------ rows that see the same slots
// One workgroup: up to 16 RT (row, head) pairs of one kv head that see the same slots (a
// token's query heads, or any rows over the prefix), over one key range.  Its waves take
// blocks of 32 slots in turn, each with a softmax state of its own, joined at the end: a
// wave streams K straight into A operands and V through a piece of shared memory of its own
// (the transposed read), the next block's loads in flight, and no wave waits for another.
//
// Many sequences are bound by memory: 64 of up to 4112 visible slots, 32 heads over 8 of 128
// dims, take 177 us, 5.55 TB/s (reading 1 GB and nothing else 6.2).  One is bound by latency: 1028 slots, 32
// heads over 8 of 64 dims, 5.8 us, of which a launch is 2 and a half.  (Sixteen waves, or
// eight, with no join after them are slower: 1024 slots take 9.4 and 8.0 us against 6.7
// with a join, 256 slots 6.3 and 5.3 against 4.5.)
constexpr int STEP_WAVES = 4;
template <int D, int RT> struct StepShared {
    static constexpr uint32_t V_BYTES = 32 * D * 2, O_BYTES = 16 * RT * D * 4;
    __attribute__((aligned(16))) uint8_t bytes[STEP_WAVES * (V_BYTES > O_BYTES ? V_BYTES : O_BYTES)];
    float2 ml[STEP_WAVES][16 * RT];
};

template <typename TQ, int D, int RT>
__device__ __forceinline__ void attn_step(const AttnOpArgs &a, StepShared<D, RT> &shared, uint32_t item)
{
    constexpr int NW = STEP_WAVES;
    typedef typename TQ::vec vec;
    constexpr int VL = D / 16;                   // 16-byte loads of V a lane and block
    constexpr uint32_t ROWS = 16 * RT, PIECES = D / 8, V_BYTES = StepShared<D, RT>::V_BYTES;
    uint8_t *const smem = shared.bytes;
    auto &sml = shared.ml;
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4;
    const uint32_t kh = blockIdx.x % a.own.kv_heads, G = a.group;
    const bool pre = item < a.step_prefix;
    uint32_t group = 0, part, parts, row0, total;
    const uint16_t *kp, *vp;
    int64_t ts;
    Blocks<32> bl;
    if (pre) {
        part = item;
        if (a.prefix_groups > 1) {
            part = item / a.prefix_groups;
            group = item - part * a.prefix_groups;
        }
        parts = a.prefix_splits;
        row0 = 0, total = a.r.n_rows * G;
        bl.set(0, clamp_len(a.prefix, 0) - 1, 0, 0);
        const int64_t at = (int64_t)kh * a.prefix.hs;
        kp = a.prefix.k + at, vp = a.prefix.v + at, ts = a.prefix.ts;
    } else {
        item -= a.step_prefix;
        if (a.own_groups > 1) {
            const uint32_t q = item / a.own_groups;
            group = item - q * a.own_groups, item = q;
        }
        row0 = item, part = 0, parts = a.own_splits;
        if (parts > 1) {
            row0 = item / parts;
            part = item - row0 * parts;
        }
        total = G;
        const int32_t pos = clamp_len(a.own, row0) - 1;
        bl.set(pos, pos, a.window, a.sinks);
        const int64_t at = (int64_t)row0 * a.own.ss + (int64_t)kh * a.own.hs;
        kp = a.own.k + at, vp = a.own.v + at, ts = a.own.ts;
    }
    const uint32_t i0 = group * ROWS;
    uint32_t b0, b1;
    share(bl.count, part, parts, &b0, &b1);
    const uint32_t rows = min(ROWS, total - i0);
    const Pairs pairs(row0, i0, G);

    uint8_t *const vt = smem + wave * V_BYTES;
    const uint32_t at = v_lane<D>(lane);
    vec kr[2][D / 32];
    u32x4 vr[VL];
    auto load = [&](uint32_t blk) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t j = min(blk * 32 + 16 * u + (lane & 15), bl.hi - 1);
            const uint16_t *p = kp + (int64_t)j * ts + 8 * g;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
                kr[u][i] = *(const vec *)(p + 32 * i);
        }
#pragma unroll
        for (int i = 0; i < VL; ++i) {
            const uint32_t j = min(blk * 32 + (i * 64 + lane) / PIECES, bl.hi - 1);
            vr[i] = *(const u32x4 *)(vp + (int64_t)j * ts + (lane % PIECES) * 8);
        }
    };
    uint32_t b = b0 + wave;
    if (b < b1)
        load(bl.block(b));
    Queries<TQ, D, RT> Q;
    State<TQ, D, RT> S;
    S.clear();
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const uint32_t x = 16 * t + (lane & 15);
        load_row<TQ, D, RT>(Q, t, a.r, x < rows, pairs.row_of(x), kh * G + pairs.head_of(x));
    }
    // NT: the row tiles in use (all, or the first)
    auto stream = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        for (; b < b1; b += NW) {
            const uint32_t blk = bl.block(b);
            const bool whole = bl.whole(blk);
            // V to shared memory; slots that are not seen become zeros, whatever they hold
#pragma unroll
            for (int i = 0; i < VL; ++i) {
                const uint32_t row = (i * 64 + lane) / PIECES;
                if (!whole && !bl.seen(blk * 32 + row))
                    vr[i] = u32x4{0, 0, 0, 0};
                *(u32x4 *)(vt + v_piece<D>(row, lane % PIECES) * 16) = vr[i];
            }
            floatx4 s[RT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    s[t][u] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < D / 32; ++i)
#pragma unroll
                        for (int x = 0; x < TQ::parts; ++x)
                            s[t][u] = mma(kr[u][i], Q.q[t][x][i], s[t][u]);
                }
            if (b + NW < b1)
                load(bl.block(b + NW));
            if (a.scores && !pre) { // uniform; rows of whole blocks, slots past the length among them
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    if (16 * t + (lane & 15) < rows) {
                        float *to = a.scores + ((size_t)row0 * a.r.heads + kh * G + i0 + 16 * t + (lane & 15)) * a.score_row +
                                    blk * 32 + 4 * g;
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            if constexpr (TQ::parts == 2)
                                *(floatx4 *)(to + 16 * u) = s[t][u] * Q.back[t];
                            else
                                *(floatx4 *)(to + 16 * u) = s[t][u];
                        }
                    }
            }
            if (!whole) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool seen = bl.seen(blk * 32 + 16 * u + 4 * g + e);
#pragma unroll
                        for (int t = 0; t < NT; ++t)
                            s[t][u][e] = seen ? s[t][u][e] : -INFINITY;
                    }
            }
            vec p[RT][TQ::parts];
            weigh<NT>(S, s, Q, p);
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
                const vec v = v_operand<TQ, D>(vt, at, n);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int x = 0; x < TQ::parts; ++x)
                        S.o[t][n] = mma(v, p[t][x], S.o[t][n]);
            }
        }
    };
    if (RT == 1 || rows <= 16)
        stream(Const<1>());
    else
        stream(Const<RT>());
    // join the waves: offsets and sums first, then the outputs at the common offset
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        S.l[t] = row_sum(S.l[t]);
        if (lane < 16)
            sml[wave][16 * t + lane] = make_float2(S.offset(t), S.l[t]);
    }
    __syncthreads();
    float *const so = (float *)smem; // [wave][row][D]
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w)
            top = fmaxf(top, sml[w][16 * t + (lane & 15)].x);
        const float f = S.seen(t) ? exp2_hw(S.mc[t] - top) : 0.f;
        float *to = so + ((size_t)wave * ROWS + 16 * t + (lane & 15)) * D + 4 * g;
        if (16 * t + (lane & 15) < rows)
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
                *(floatx4 *)(to + 16 * n) = S.o[t][n] * f;
    }
    __syncthreads();
    const bool final = !a.scores && a.own_splits + a.prefix_splits == 1;
    constexpr uint32_t QD = D / 4;
    for (uint32_t x = tid; x < rows * QD; x += NW * 64) {
        const uint32_t i = x / QD, d = (x % QD) * 4;
        float top = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w)
            top = fmaxf(top, sml[w][i].x);
        floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float2 e = sml[w][i];
            l += e.x > -INFINITY ? e.y * exp2_hw(e.x - top) : e.y;
            o += *(const floatx4 *)(so + ((size_t)w * ROWS + i) * D + d);
        }
        const uint32_t row = pairs.row_of(i), h = kh * G + pairs.head_of(i);
        if (final) {
            const bool empty = bl.hi == 0;
            store_out<TQ>(a.r, row, h, d, empty ? o : o * inverse(l));
            if (d == 0)
                finish_row(a, (size_t)row * a.r.heads + h, empty, top, l);
        } else {
            const size_t to = ((size_t)(pre ? a.own_splits + part : part) * a.r.n_rows + row) * a.r.heads + h;
            *(floatx4 *)(a.o + to * D + d) = o;
            if (d == 0)
                a.ml[to] = make_float2(top, l);
        }
    }
}

// The key ranges (64 at most) of one row and head, joined by a wave: the common offset and
// the sum, the same in every lane, and the lane's D / 64 dims of the output before its
// division by the sum.  Lane s holds range s's state; eight ranges' outputs are loaded
// before the first is used.
template <int D>
__device__ __forceinline__ void join(const AttnOpArgs &a, uint32_t id, uint32_t n, bool outputs, float *top, float *sum,
                                     float (&o)[D / 64])
{
    constexpr int E = D / 64;
    const uint32_t lane = threadIdx.x & 63, pairs = a.r.n_rows * a.r.heads;
    float2 e = make_float2(-INFINITY, 0.f);
    if (lane < n)
        e = a.ml[(size_t)lane * pairs + id];
    *top = wave_max(e.x);
    const float f = e.x > -INFINITY ? exp2_hw(e.x - *top) : 0.f;
    // a range without a number adds its sum (0, or NaN from its scores) as it is
    *sum = wave_sum(e.x > -INFINITY ? e.y * f : e.y);
#pragma unroll
    for (int i = 0; i < E; ++i)
        o[i] = 0.f;
    if (!outputs)
        return;
    for (uint32_t s0 = 0; s0 < n; s0 += 8) {
        float x[8][E];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < E; ++i)
                x[j][i] = a.o[((size_t)min(s0 + j, n - 1) * pairs + id) * D + lane * E + i];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // a range whose weights vanish beside the others' counts too: its NaN stays
            const float w = lane_f32(f, min(s0 + j, 63u));
            if (s0 + j < n)
#pragma unroll
                for (int i = 0; i < E; ++i)
                    o[i] += w * x[j][i];
        }
    }
}

template <typename TQ, int D>
__device__ __forceinline__ void store_row(const AttnOpArgs &a, uint32_t row, uint32_t h, bool empty, float top, float sum,
                                          const float (&o)[D / 64])
{
    constexpr int E = D / 64;
    const uint32_t lane = threadIdx.x & 63;
    typedef typename TQ::type tq;
    tq *to = (tq *)a.r.out + (int64_t)row * a.r.o_rs + (int64_t)h * a.r.o_hs + lane * E;
    const float f = inverse(sum);
#pragma unroll
    for (int i = 0; i < E; ++i)
        to[i] = (tq)(empty ? 0.f : in_range<TQ>(o[i] * f));
    if (lane == 0)
        finish_row(a, (size_t)row * a.r.heads + h, empty, top, sum);
}

// Joins the key ranges of a row and head: a wave each, so that one row of 32 heads takes 8
// CUs.  Bound by latency: 3.1 us there, 5.1 for 64 rows of 32 heads, 128 dims and 9 ranges.
template <typename TQ, int D> __device__ __forceinline__ void attn_merge(const AttnOpArgs &a)
{
    const uint32_t id = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (id >= a.r.n_rows * a.r.heads)
        return;
    const uint32_t row = id / a.r.heads, h = id - row * a.r.heads;
    uint32_t b;
    int32_t pos;
    if (!find_row(a, row, &b, &pos))
        return;
    float top, sum, o[D / 64];
    join<D>(a, id, a.own_splits + a.prefix_splits, true, &top, &sum, o);
    store_row<TQ, D>(a, row, h, pos < 0 && (!a.prefix.k || clamp_len(a.prefix, 0) == 0), top, sum, o);
}

// After a scored step: joins the key ranges of one (sequence, kv head) and adds every
// slot's weights, SCORED_SLOTS slots a workgroup, four a thread.  Scores were kept as they
// left the matrix cores, so a weight is one exponential here: 16 bytes a slot and kv head at
// four query heads, where reading K again would be 128 or 256.  The first four heads' scores
// are loaded before the ranges are joined.  Six sequences of up to 32768 slots, 32 heads over
// 8: 10 us after the step's 139; eight of up to 4096: 4.9 after 12.1, mostly latency.
template <typename TQ, int D> __device__ __forceinline__ void scored_join(const AttnOpArgs &a)
{
    const uint32_t chunk = blockIdx.x, kh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x,
                   wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const uint32_t G = a.group, n = (uint32_t)clamp_len(a.own, b);
    if (chunk && chunk * SCORED_SLOTS >= n)
        return;
    constexpr int EACH = SCORED_SLOTS / 256, EARLY = 4;
    const float *scores = a.scores + ((size_t)b * a.r.heads + kh * G) * a.score_row;
    const size_t at = ((size_t)b * a.own.kv_heads + kh) * a.own.slots;
    uint32_t j[EACH];
    float had[EACH] = {}, s[EACH][EARLY] = {};
    if (n) // uniform
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            j[i] = min(chunk * SCORED_SLOTS + i * 256 + tid, n - 1);
            if (a.acc)
                had[i] = a.acc[at + j[i]];
#pragma unroll
            for (int g = 0; g < EARLY; ++g)
                s[i][g] = scores[(size_t)min((uint32_t)g, G - 1) * a.score_row + j[i]];
        }
    __shared__ float2 st[MAX_GROUP]; // offset and 1 / sum
    // the outputs of the G heads are spread over the workgroups in use
    const uint32_t chunks = max(1u, (n + SCORED_SLOTS - 1) / SCORED_SLOTS);
    for (uint32_t g = wave; g < G; g += 4) {
        const bool mine = chunk == g % chunks;
        float top, sum, o[D / 64];
        join<D>(a, b * a.r.heads + kh * G + g, a.own_splits, mine, &top, &sum, o);
        if (lane == 0)
            st[g] = make_float2(top, inverse(sum));
        if (mine)
            store_row<TQ, D>(a, b, kh * G + g, n == 0, top, sum, o);
    }
    __syncthreads();
    const float c = TQ::parts == 2 ? a.r.cfrac : a.r.cexp;
    if (n)
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            float sum = 0.f;
#pragma unroll
            for (int g = 0; g < EARLY; ++g)
                if (g < (int)G)
                    sum += exp2_hw(fmaf(s[i][g], c, -st[g].x)) * st[g].y;
            for (uint32_t g = EARLY; g < G; ++g)
                sum += exp2_hw(fmaf(scores[(size_t)g * a.score_row + j[i]], c, -st[g].x)) * st[g].y;
            if (chunk * SCORED_SLOTS + i * 256 + tid < n)
                a.acc_out[at + j[i]] = had[i] + sum;
        }
}

// ------------------------------------------------------------------ rows of many tokens
// The (sequence, part) of a flat item where sequence b has ceil(rows_b * per / of) of them;
// false past the last.  64 sequences at a time, the same in every wave.
__device__ __forceinline__ bool find_item(const RowsView &r, uint32_t n_seq, uint32_t item, uint32_t per, uint32_t of,
                                          uint32_t *b, uint32_t *part, uint32_t *parts)
{
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t s0 = 0; s0 < n_seq; s0 += 64) {
        uint32_t n = 0;
        if (s0 + lane < n_seq) {
            int32_t lo, hi;
            seq_rows(r, s0 + lane, &lo, &hi);
            n = (uint32_t)(((uint64_t)(hi - lo) * per + of - 1) / of);
        }
        uint32_t upto = n; // inclusive sums over the lanes
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(upto, d);
            upto += lane >= (uint32_t)d ? o : 0;
        }
        const uint32_t all = __builtin_amdgcn_readlane(upto, 63);
        if (item < all) {
            const uint32_t at = (uint32_t)__ffsll((unsigned long long)__ballot(upto > item)) - 1;
            *b = s0 + at;
            *parts = __builtin_amdgcn_readlane(n, at);
            *part = item - (__builtin_amdgcn_readlane(upto, at) - *parts);
            return true;
        }
        item -= all;
    }
    return false;
}

template <typename TQ> __device__ __forceinline__ bool has_nonfinite(u32x4 v)
{
    constexpr uint32_t E = TQ::offset == 0.f ? 0x7F807F80u : 0x7C007C00u; // exponents of two numbers
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        bad = bad || (w[i] & E & 0xFFFF0000u) == (E & 0xFFFF0000u) || (w[i] & E & 0xFFFFu) == (E & 0xFFFFu);
    return bad;
}

// 16 bytes a lane from memory to shared memory, lane x's to byte `to` + 16 x (uniform),
// with no register between.  Written out because the compiler makes every read of shared
// memory wait for such loads, the other buffer's too: whoever reads waits with wait_loads
// and a barrier.  The place in shared memory is an operand in M0, which the compiler so
// knows to be in use (the load may follow M0's writing after one wait state; with M0 written
// in the statement, as a clobber that the compiler warns of, a scored prompt of 2048 tokens
// takes 66.1 us for 67.1, the other cases within 0.6 %).
__device__ __forceinline__ void load_to_lds(const void *from, uint32_t to)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(to), "v"(from) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(void *p)
{
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)p;
}

// Until this wave's loads into shared memory have arrived.
__device__ __forceinline__ void wait_loads()
{
    __builtin_amdgcn_s_waitcnt(0x0f70); // vmcnt(0)
    asm volatile("" ::: "memory");
}

// A barrier that leaves loads from memory in flight.
__device__ __forceinline__ void lds_barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f); // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// One row and head over blocks b0 .. b1 of 64 slots, by a wave: a lane's score each, then
// every lane its dims of the weighted sum, a slot that the row does not see left out whatever
// it holds.
template <typename TQ, int D, typename B>
__device__ void attn_row(const AttnOpArgs &a, const B &bl, uint32_t b0, uint32_t b1, const uint16_t *kp,
                         const uint16_t *vp, uint32_t row, uint32_t h, int32_t pos, uint32_t split, float *weights)
{
    typedef typename TQ::kv tk;
    constexpr int E = D / 64;
    const uint32_t lane = threadIdx.x & 63;
    const typename TQ::type *q = (const typename TQ::type *)a.r.q + (int64_t)row * a.r.q_rs + (int64_t)h * a.r.q_hs;
    float mc = 0.f, l = 0.f, o[E] = {};
    bool none = true; // no number yet
    for (uint32_t i = b0; i < b1; ++i) {
        const uint32_t j0 = bl.block(i) * 64;
        const int64_t j = j0 + lane;
        const bool seen = j <= pos && (!a.window || j < (int64_t)a.sinks || j > (int64_t)pos - a.window);
        float x = -INFINITY;
        if (seen) {
            const tk *k = (const tk *)kp + j * a.own.ts;
            x = 0.f;
            if constexpr (TQ::parts == 2) { // q . k alone may be out of range
                for (int d = 0; d < D; ++d)
                    x = fmaf(q[d] * a.r.cexp, (float)k[d], x);
            } else {
                for (int d = 0; d < D; ++d)
                    x = fmaf((float)q[d], (float)k[d], x);
                x *= a.r.cexp;
            }
        }
        const uint64_t any = __ballot(seen);
        const float top = wave_max(x);
        if (top > (none ? -INFINITY : mc)) {
            const float r = none ? 0.f : exp2_hw(mc - top);
            mc = top, l *= r, none = false;
#pragma unroll
            for (int e = 0; e < E; ++e)
                o[e] *= r;
        }
        const float w = seen ? exp2_hw(x - mc) : 0.f;
        l += wave_sum(w);
        __builtin_amdgcn_wave_barrier();
        weights[lane] = w;
        __builtin_amdgcn_wave_barrier();
        for (uint64_t m = any; m; m &= m - 1) {
            const uint32_t s = (uint32_t)__ffsll((unsigned long long)m) - 1;
#pragma unroll
            for (int e = 0; e < E; ++e)
                o[e] += weights[s] * (float)((const tk *)vp)[(int64_t)(j0 + s) * a.own.ts + lane * E + e];
        }
    }
    const float off = none ? -INFINITY : mc;
    if (a.own_splits + a.prefix_splits == 1) {
        store_row<TQ, D>(a, row, h, pos < 0, off, l, o);
        return;
    }
    const size_t to = ((size_t)split * a.r.n_rows + row) * a.r.heads + h;
#pragma unroll
    for (int e = 0; e < E; ++e)
        a.o[to * D + lane * E + e] = o[e];
    if (lane == 0)
        a.ml[to] = make_float2(off, l);
}

#define TILE_KEYS 64
// One workgroup: 64 RT (token, head) pairs of one sequence and kv head, 16 RT a wave, over
// one key range; PRE: of the whole batch over the prefix.  Blocks of 64 slots pass through two
// buffers of shared memory, K and V as they lie in the cache with their 16-byte pieces
// exchanged (v_piece); every wave reads K as A operands and V through the transposed read.
// The next block's loads are in flight while a block is used.  Blocks that no row of a wave
// sees are passed over by it, those that all its rows see whole are used without masks.
//
// Bound by a SIMD's issue, which vector and matrix work share: products and other work hardly
// overlap (8 products and 32 multiply-adds of four waves take 194 cycles together, 132 and 82
// alone).  For 32 rows and 32 slots a wave has 16 products of 16 cycles at 64 dims, 32 at 128, and
// 111 and 123 other vector instructions (4096 tokens, window 1024; chunks, window 2048): some 70
// are the softmax, 16 exponentials among them; the rest are the loads' addresses, masks at the
// diagonal and the window's edge, and the loop's own.  Products and vector issue fill 30 and 68 %
// of the cycles at 64 dims, 37 and 49 (the products' own issue among them) at 128, where shared
// memory is busy for 28 % and a fifth is neither's.  4096 tokens, window 1024, 32
// heads over 8 of 64 dims: 50 us, 600 TFLOP/s; 8192 causal: 323 us, 850; of 128 dims, with
// half as much softmax a product, 589 us, 930.  Two groups of 32 slots in one softmax take more
// registers than four waves a SIMD have (72 us for 60), four row tiles a wave leave two waves
// (55 for 53), and V's operands before the softmax cost 71 for 59.
//
// A slot that some rows of a wave see and others do not may hold an infinity or NaN in V,
// which times a weight of 0 would reach all of them: a wave that met such numbers in a
// masked block computes its rows again, one by one (attn_row).
template <int D> struct TileShared {
    static constexpr uint32_t BYTES = TILE_KEYS * D * 2;
    __attribute__((aligned(16))) uint8_t k[2][BYTES], v[2][BYTES];
    uint64_t odd[4];      // slots of a block whose V is not all finite
    float weights[4][64]; // attn_row's
};

template <typename TQ, int D, int RT, bool PRE>
__device__ __forceinline__ void attn_tile(const AttnOpArgs &a, TileShared<D> &shared, uint32_t flat)
{
    typedef typename TQ::vec vec;
    constexpr uint32_t ROWS = 64 * RT, PIECES = D / 8, BYTES = TileShared<D>::BYTES;
    constexpr int LD = TILE_KEYS * PIECES / 256; // 16-byte pieces of K, and of V, a thread and block
    auto &ks = shared.k, &vs = shared.v;
    auto &odd = shared.odd;
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4;
    const uint32_t kh = blockIdx.x % a.own.kv_heads, G = a.group;
    const KvView &c = PRE ? a.prefix : a.own;
    const uint32_t splits = PRE ? a.prefix_splits : a.own_splits;
    const uint32_t split = splits == 1 ? 0 : flat % splits;
    // rows lo .. hi of one sequence, row lo at position `first` and each next one `step` further;
    // over the prefix all rows, each at its last position
    uint32_t b = 0, tile, tiles;
    int32_t lo = 0, hi = (int32_t)a.r.n_rows, first, step = PRE ? 0 : 1;
    if (PRE) {
        tile = splits == 1 ? flat : flat / splits;
        first = clamp_len(c, 0) - 1;
    } else {
        if (!find_item(a.r, a.own.n_seq, splits == 1 ? flat : flat / splits, G, ROWS, &b, &tile, &tiles))
            return;
        // The longest first, every second 32 (an XCD's CUs) in reverse: a CU's workgroups add
        // up to about the same.
        if (tile & 32 && (tile | 31) < tiles)
            tile ^= 31;
        tile = tiles - 1 - tile;
        seq_rows(a.r, b, &lo, &hi);
        first = clamp_len(c, b) - (hi - lo);
    }
    const uint32_t total = (uint32_t)(hi - lo) * G, p0 = tile * ROWS, window = PRE ? 0 : a.window,
                   sinks = PRE ? 0 : a.sinks;
    const int32_t pos_lo = first + step * (int32_t)(p0 / G),
                  pos_hi = first + step * (int32_t)((min(p0 + ROWS, total) - 1) / G);
    Blocks<TILE_KEYS> bl;
    bl.set(pos_lo, pos_hi, window, sinks);
    uint32_t b0, b1;
    share(bl.count, split, splits, &b0, &b1);

    Queries<TQ, D, RT> Q;
    State<TQ, D, RT> S;
    S.clear();
    int32_t pos[RT];
    const uint32_t w0 = p0 + wave * 16 * RT;
    const Pairs pairs((uint32_t)lo, w0, G);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const uint32_t x = 16 * t + (lane & 15), row = pairs.row_of(x);
        const bool in = w0 + x < total;
        load_row<TQ, D, RT>(Q, t, a.r, in, row, kh * G + pairs.head_of(x));
        pos[t] = in ? first + step * ((int32_t)row - lo) : -1;
    }
    // what this wave's rows see: some row of it, every row of it
    const bool any_row = w0 < total;
    const int32_t wpos_lo = first + step * (int32_t)(w0 / G),
                  wpos_hi = first + step * (int32_t)((min(w0 + 16 * RT, total) - 1) / G);
    Blocks<32> some, each;
    some.set(wpos_lo, wpos_hi, window, sinks);
    each.set(wpos_hi, wpos_lo, window, sinks);
    Blocks<TILE_KEYS> all; // every row of the workgroup
    all.set(pos_hi, pos_lo, window, sinks);

    const int64_t at0 = (int64_t)b * c.ss + (int64_t)kh * c.hs;
    const uint16_t *kp = c.k + at0, *vp = c.v + at0;
    // A block's K and V from memory straight into shared memory: thread x's piece i goes to
    // place 256 i + x, so the exchange of pieces is made in the address that it reads.  Past
    // the last visible slot that one is read again.
    const uint32_t row_in = tid / PIECES, piece_in = (tid % PIECES) ^ (row_in & (PIECES - 1));
    const uint16_t *const kl = kp + (int64_t)row_in * c.ts + piece_in * 8, *const vl = vp + (kl - kp);
    const uint32_t ks_at = __builtin_amdgcn_readfirstlane(lds_address(ks)),
                   vs_at = __builtin_amdgcn_readfirstlane(lds_address(vs));
    auto fetch = [&](uint32_t blk, uint32_t buf) {
        const bool inside = blk * TILE_KEYS + TILE_KEYS <= bl.hi;
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const uint32_t row = blk * TILE_KEYS + i * (256 / PIECES);
            int64_t o = (int64_t)row * c.ts;
            if (!inside)
                o = ((int64_t)min(row + row_in, bl.hi - 1) - row_in) * c.ts;
            const uint32_t to = buf * BYTES + (i * 256 + wave * 64) * 16;
            load_to_lds(kl + o, ks_at + to);
            load_to_lds(vl + o, vs_at + to);
        }
    };
    if (tid < 4)
        odd[tid] = 0;
    if (b0 < b1)
        fetch(bl.block(b0), 0);
    const uint32_t at = v_lane<D>(lane);
    bool again = false;
    for (uint32_t i = b0; i < b1; ++i) {
        const uint32_t blk = bl.block(i), buf = (i - b0) & 1;
        wait_loads();
        __syncthreads();
        if (i + 1 < b1)
            fetch(bl.block(i + 1), buf ^ 1);
        if (tid == 0)
            odd[(i + 2) & 3] = 0; // used last at i - 2, filled next at i + 2
        if (!all.whole(blk)) {
            // V of slots that no row sees becomes zeros; numbers that are not finite are noted
#pragma unroll
            for (int x = 0; x < LD; ++x) {
                const uint32_t row = (x * 256 + tid) / PIECES;
                u32x4 *const v = (u32x4 *)(vs[buf] + (x * 256 + tid) * 16);
                if (!bl.seen(blk * TILE_KEYS + row))
                    *v = u32x4{0, 0, 0, 0};
                else if (!PRE && has_nonfinite<TQ>(*v))
                    atomicOr((unsigned long long *)&odd[i & 3], 1ull << row);
            }
            lds_barrier();
        }
#pragma unroll
        for (uint32_t sub = 0; sub < 2; ++sub) {
            const uint32_t j0 = blk * TILE_KEYS + 32 * sub;
            if (!any_row || !some.touches(j0, 32))
                continue;
            const bool whole = each.covers(j0, 32);
            const uint8_t *kb = ks[buf] + sub * 32 * D * 2, *vb = vs[buf] + sub * 32 * D * 2;
            vec k[2][D / 32];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int x = 0; x < D / 32; ++x)
                    k[u][x] = *(const vec *)(kb + v_piece<D>(16 * u + (lane & 15), g + 4 * x) * 16);
            vec p[RT][TQ::parts];
            if (!PRE && !whole)
                again |= __builtin_amdgcn_readfirstlane((uint32_t)(odd[i & 3] >> (32 * sub)));
            floatx4 s[RT][2];
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    s[t][u] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int x = 0; x < D / 32; ++x)
#pragma unroll
                        for (int y = 0; y < TQ::parts; ++y)
                            s[t][u] = mma(k[u][x], Q.q[t][y][x], s[t][u]);
                }
            if (!whole) {
                // row at pos sees j <= pos, and j < sinks or j > pos - window
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    const int32_t from =
                        window && (uint32_t)max(pos[t], 0) >= window ? pos[t] - (int32_t)window : -1;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int32_t j = (int32_t)j0 + 16 * u + 4 * g + e;
                            const bool hidden = (j > pos[t]) | ((j <= from) & ((uint32_t)j >= sinks));
                            s[t][u][e] = hidden ? -INFINITY : s[t][u][e];
                        }
                }
            }
            // matrix work of other waves goes before this one's softmax (2 % of a long call)
            __builtin_amdgcn_s_setprio(0);
            weigh<RT>(S, s, Q, p);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
                const vec v = v_operand<TQ, D>(vb, at, n);
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int y = 0; y < TQ::parts; ++y)
                        S.o[t][n] = mma(v, p[t][y], S.o[t][n]);
            }
        }
    }
    const bool final = !PRE && a.own_splits + a.prefix_splits == 1;
    if (!PRE && again) { // uniform; rare (over the prefix all rows see the same slots)
        for (uint32_t x = 0; x < 16 * RT && w0 + x < total; ++x) {
            const uint32_t row = pairs.row_of(x);
            attn_row<TQ, D>(a, bl, b0, b1, kp, vp, row, kh * G + pairs.head_of(x), first + (int32_t)row - lo, split,
                            shared.weights[wave]);
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float l = row_sum(S.l[t]);
        const uint32_t x = 16 * t + (lane & 15);
        if (w0 + x >= total)
            continue;
        const uint32_t row = pairs.row_of(x), h = kh * G + pairs.head_of(x);
        const float off = S.offset(t);
        if (final) {
            const bool empty = pos[t] < 0;
            const float f = empty ? 0.f : inverse(l);
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
                store_out<TQ>(a.r, row, h, 16 * n + 4 * g, S.o[t][n] * f);
            if (g == 0)
                finish_row(a, row * a.r.heads + h, empty, off, l);
        } else {
            const size_t to = ((size_t)(PRE ? a.own_splits + split : split) * a.r.n_rows + row) * a.r.heads + h;
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
                *(floatx4 *)(a.o + to * D + 16 * n + 4 * g) = S.o[t][n];
            if (g == 0)
                a.ml[to] = make_float2(off, l);
        }
    }
}

// The weights that SUM_KEYS slots of one (sequence, kv head) receive from a part of its rows:
// scores once more, a wave's 32 slots as A operands in registers and (token, head) pairs, 64
// at a time through two buffers of shared memory, as B operands.  A lane's scores are of one
// row (its softmax state: offset and 1 / sum) and four slots a tile; it adds its slots'
// weights 2^(s c - offset) / sum over its rows, and the 16 lanes of a slot are added at the
// end, all in a fixed order.  (Rows read as operands by every wave for itself, 16 rows a load,
// kept the first-level cache busy with 64-byte pieces: a prompt of 2048 tokens, 32 heads over
// 8 of 64 dims, took 42 us so, 28 this way and 5 for the adding of the parts.)  Bound by vector
// instructions, 5.9 a score at 64 dims: three are the softmax, one of them an exponential, most of
// the rest the addresses and the staging of rows.  They fill 31 of 50 thousand cycles of a SIMD,
// the products 8; waits at a step's barrier and for loads are the rest.
template <typename TQ, int D> __device__ __forceinline__ void attn_weights(const AttnOpArgs &a)
{
    typedef typename TQ::vec vec;
    typedef typename TQ::type tq;
    constexpr uint32_t STEP = 64, PIECES = D / 8, BYTES = STEP * D * 2;
    constexpr int PER = STEP * PIECES / 256; // pieces of 8 numbers a thread and step
    constexpr int KT = SUM_KEYS / 4 / 16;    // tiles of 16 slots a wave
    struct Row {
        float c, offset, inverse;
        int32_t pos;
    };
    __shared__ __attribute__((aligned(16))) uint8_t qs[2][TQ::parts][BYTES];
    __shared__ __attribute__((aligned(16))) Row rows[2][STEP];
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4;
    const uint32_t kh = blockIdx.x % a.own.kv_heads, G = a.group;
    uint32_t tile = blockIdx.x / a.own.kv_heads;
    const uint32_t b = a.sum_parts == 1 ? blockIdx.y : blockIdx.y / a.sum_parts, part = blockIdx.y - b * a.sum_parts;
    const uint32_t n = (uint32_t)clamp_len(a.own, b), tiles = (n + SUM_KEYS - 1) / SUM_KEYS;
    if (tile >= tiles)
        return;
    // early slots are seen by more rows: each part starts with another one, so that a CU's
    // workgroups differ
    tile = (tile + blockIdx.y + blockIdx.y / 4) % tiles;
    const uint32_t j0 = tile * SUM_KEYS;
    int32_t lo, hi;
    seq_rows(a.r, b, &lo, &hi);
    const uint32_t total = (uint32_t)(hi - lo) * G;
    const int32_t first = (int32_t)n - (hi - lo);
    // steps of 64 pairs: those before the first that sees slot j0 add nothing; of the others
    // this part's
    const uint32_t skipped = (int32_t)j0 > first ? (uint32_t)((int32_t)j0 - first) * G / STEP : 0;
    uint32_t s0, s1;
    share((total + STEP - 1) / STEP - min(skipped, (total + STEP - 1) / STEP), part, a.sum_parts, &s0, &s1);
    s0 += skipped, s1 += skipped;
    const uint32_t jw = j0 + 16 * KT * wave; // the wave's slots
    vec k[KT][D / 32];
    const uint16_t *kp = a.own.k + (int64_t)b * a.own.ss + (int64_t)kh * a.own.hs + 8 * g;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        const uint16_t *p = kp + (int64_t)min(jw + 16 * t + (lane & 15), n - 1) * a.own.ts;
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
            k[t][x] = *(const vec *)(p + 32 * x);
    }
    floatx4 sum[KT] = {};
    // a thread's pieces of a step, and the state of the row that it holds for thread < 64
    // rows are 16-byte aligned; the natural alignment of eight floats is 32
    typedef tq tq8 __attribute__((ext_vector_type(8), aligned(16)));
    static_assert(alignof(tq8) == 16, "no more than the rows' own alignment");
    tq8 piece[PER];
    float2 st;
    int32_t pos = -1;
    auto load = [&](uint32_t step) {
        const Pairs pairs((uint32_t)lo, step * STEP, G);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t x = (i * 256 + tid) / PIECES, in = step * STEP + x < total ? x : 0;
            piece[i] = *(const tq8 *)((const tq *)a.r.q + (int64_t)pairs.row_of(in) * a.r.q_rs +
                                      (int64_t)(kh * G + pairs.head_of(in)) * a.r.q_hs + (tid % PIECES) * 8);
        }
        if (tid < STEP) {
            const uint32_t in = step * STEP + tid < total ? tid : 0, row = pairs.row_of(in);
            st = a.stats[(size_t)row * a.r.heads + kh * G + pairs.head_of(in)];
            pos = in == tid ? first + (int32_t)row - lo : -1;
        }
    };
    auto store = [&](uint32_t buf) {
        if (tid < STEP) {
            rows[buf][tid].offset = st.x, rows[buf][tid].inverse = st.y, rows[buf][tid].pos = pos;
            if constexpr (TQ::parts == 1)
                rows[buf][tid].c = a.r.cexp;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t x = (i * 256 + tid) / PIECES, to = v_piece<D>(x, tid % PIECES) * 16;
            if constexpr (TQ::parts == 1) {
                *(vec *)(qs[buf][0] + to) = piece[i];
            } else { // as load_row does, a row in PIECES neighbouring lanes
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    top = fmaxf(top, fabsf(piece[i][e]));
#pragma unroll
                for (uint32_t d = 1; d < PIECES; d <<= 1)
                    top = fmaxf(top, __shfl_xor(top, d));
                const int up = power_up(top);
                const float scale = ldexpf(1.f, up);
                vec hi, lo_;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float y = piece[i][e] * scale;
                    hi[e] = (_Float16)y;
                    lo_[e] = (_Float16)(y - (float)hi[e]);
                }
                *(vec *)(qs[buf][0] + to) = hi;
                *(vec *)(qs[buf][1] + to) = lo_;
                if (tid % PIECES == 0)
                    rows[buf][x].c = a.r.cfrac * power_back(a.r, up);
            }
        }
    };
    if (s0 < s1) {
        load(s0);
        store(0);
    }
    for (uint32_t s = s0; s < s1; ++s) {
        const uint32_t buf = (s - s0) & 1;
        __syncthreads();
        if (s + 1 < s1)
            load(s + 1);
#pragma unroll 2
        for (uint32_t x = 0; x < STEP / 16; ++x) {
            const Row row = rows[buf][16 * x + (lane & 15)];
            if (__ballot(row.pos >= (int32_t)jw) == 0) // uniform: no row sees the wave's first slot
                continue;
            const bool whole = __ballot(row.pos < (int32_t)(jw + 16 * KT - 1)) == 0;
            vec q[TQ::parts][D / 32];
#pragma unroll
            for (int y = 0; y < TQ::parts; ++y)
#pragma unroll
                for (int i = 0; i < D / 32; ++i)
                    q[y][i] = *(const vec *)(qs[buf][y] + v_piece<D>(16 * x + (lane & 15), g + 4 * i) * 16);
            floatx4 v[KT] = {};
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int y = 0; y < TQ::parts; ++y)
#pragma unroll
                    for (int t = 0; t < KT; ++t)
                        v[t] = mma(k[t][i], q[y][i], v[t]);
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[t][e] = exp2_hw(fmaf(v[t][e], row.c, -row.offset));
            if (whole) { // uniform
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sum[t][e] = fmaf(v[t][e], row.inverse, sum[t][e]);
                continue;
            }
            // a row's NaN stays with the slots it sees
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float to = fmaf(v[t][e], row.inverse, sum[t][e]);
                    sum[t][e] = (int32_t)(jw + 16 * t + 4 * g + e) <= row.pos ? to : sum[t][e];
                }
        }
        if (s + 1 < s1)
            store(buf ^ 1);
    }
    // the 16 lanes of a slot are its rows' sums
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float v = sum[t][e];
            v += dpp_mov<0xb1>(v, 0.f);  // quad_perm [1,0,3,2]
            v += dpp_mov<0x4e>(v, 0.f);  // quad_perm [2,3,0,1]
            v += dpp_mov<0x114>(v, 0.f); // row_shr:4
            v += dpp_mov<0x118>(v, 0.f); // row_shr:8: the row's sum in lane 15 of 16
            const uint32_t j = jw + 16 * t + 4 * g + e;
            if ((lane & 15) == 15 && j < n) {
                const size_t at = ((size_t)b * a.own.kv_heads + kh) * a.own.slots + j;
                if (a.sum_parts == 1)
                    a.acc_out[at] = (a.acc ? a.acc[at] : 0.f) + v;
                else
                    a.sums[(size_t)part * a.own.n_seq * a.own.kv_heads * a.own.slots + at] = v;
            }
        }
}

// acc_out = acc + the parts of attn_weights, in their order: equal calls give equal bits, which
// atomic additions would not.  A launch and little more, 4.6 us for 16 parts of 2048 slots and
// 8 kv heads.
extern "C" __global__ __launch_bounds__(256) void k_attn_sums(const AttnOpArgs a)
{
    const uint32_t j = blockIdx.x * 256 + threadIdx.x, kh = blockIdx.y, b = blockIdx.z;
    if (j >= (uint32_t)clamp_len(a.own, b))
        return;
    const size_t at = ((size_t)b * a.own.kv_heads + kh) * a.own.slots + j,
                 part = (size_t)a.own.n_seq * a.own.kv_heads * a.own.slots;
    float v[MOST_SUM_PARTS];
#pragma unroll
    for (uint32_t p = 0; p < MOST_SUM_PARTS; ++p)
        v[p] = p < a.sum_parts ? a.sums[p * part + at] : 0.f;
    float sum = 0.f;
#pragma unroll
    for (uint32_t p = 0; p < MOST_SUM_PARTS; ++p)
        sum += v[p];
    a.acc_out[at] = (a.acc ? a.acc[at] : 0.f) + sum;
}

// RT: row tiles of a workgroup of rows that see the same slots, as many as the registers hold
// beside the next block's K and V at one wave a SIMD (64 sequences over 8192 slots, 32 heads
// over 1 of 128 dims, F32 rows: 58 us; held to two waves, with what spills in memory, 85).  At
// 64 dims and 16-bit rows two waves find room (28 us; 32 with one).
#define STEP(TQ, tag, D, RT)                                                                                   \
    extern "C" __global__ __launch_bounds__(256, RT == 4 && TQ::parts == 1 ? 2 : 1) void                          \
    k_attn_step_##tag##_##D##_r##RT(const AttnOpArgs a)                                                        \
    {                                                                                                          \
        __shared__ StepShared<D, RT> shared;                                                                   \
        attn_step<TQ, D, RT>(a, shared, blockIdx.x / a.own.kv_heads);                                          \
    }
#define STEPS(TQ, tag, D, MOST)                                                                                \
    STEP(TQ, tag, D, 1)                                                                                        \
    STEP(TQ, tag, D, MOST)                                                                                     \
    extern "C" __global__ __launch_bounds__(256) void k_attn_merge_##tag##_##D(const AttnOpArgs a)             \
    {                                                                                                          \
        attn_merge<TQ, D>(a);                                                                                  \
    }                                                                                                          \
    extern "C" __global__ __launch_bounds__(256) void k_scored_join_##tag##_##D(const AttnOpArgs a)            \
    {                                                                                                          \
        scored_join<TQ, D>(a);                                                                                 \
    }
STEPS(F32, f32, 64, 4)
STEPS(F32, f32, 128, 2)
STEPS(F16, f16, 64, 4)
STEPS(F16, f16, 128, 2)
STEPS(BF16, bf16, 64, 4)
STEPS(BF16, bf16, 128, 2)

// The prefix of many rows, and single rows' own slots (where the call has such) in the same
// launch, the prefix first: one or two of its workgroups come to a CU, which then has matrix
// work and loads from memory at once.  64 sequences of 8192 + up to 1024 slots, 32 heads over 8
// of 128 dims: 53 us (66 in two launches); 150 of 32000 + up to 257, 64 dims: 69 (77).  In turn,
// a workgroup of the prefix and one of the own slots, the second takes 103: the prefix's come to
// the same CUs.
template <typename TQ, int D> __device__ __forceinline__ void attn_prefix(const AttnOpArgs &a)
{
    union Shared {
        TileShared<D> tile;
        StepShared<D, 1> step;
    };
    __shared__ Shared shared;
    const uint32_t item = blockIdx.x / a.own.kv_heads, tiles = a.prefix_groups * a.prefix_splits;
    if (item < tiles)
        attn_tile<TQ, D, TILE_TILES, true>(a, shared.tile, item);
    else
        attn_step<TQ, D, 1>(a, shared.step, item - tiles);
}

#define TILE_BOUNDS(TQ, D) __launch_bounds__(256, D == 128 ? 2 : TQ::parts == 2 ? 3 : 4)
#define TILE(TQ, tag, D, RT)                                                                                   \
    extern "C" __global__ TILE_BOUNDS(TQ, D) void k_attn_tile_##tag##_##D##_r##RT(const AttnOpArgs a)          \
    {                                                                                                          \
        __shared__ TileShared<D> shared;                                                                       \
        attn_tile<TQ, D, RT, false>(a, shared, blockIdx.x / a.own.kv_heads);                                   \
    }
#define TILES(TQ, tag, D)                                                                                      \
    TILE(TQ, tag, D, 1)                                                                                        \
    TILE(TQ, tag, D, 2)                                                                                        \
    extern "C" __global__ TILE_BOUNDS(TQ, D) void k_attn_prefix_##tag##_##D(const AttnOpArgs a)                \
    {                                                                                                          \
        attn_prefix<TQ, D>(a);                                                                                 \
    }                                                                                                          \
    extern "C" __global__ __launch_bounds__(256) void k_attn_weights_##tag##_##D(const AttnOpArgs a)           \
    {                                                                                                          \
        attn_weights<TQ, D>(a);                                                                                \
    }
TILES(F32, f32, 64)
TILES(F32, f32, 128)
TILES(F16, f16, 64)
TILES(F16, f16, 128)
TILES(BF16, bf16, 64)
TILES(BF16, bf16, 128)

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
#define SEL_HELD 24576 // ranks held in shared memory beside the registers'; further ones are made again
#define SEL_COPIES 16  // of each histogram, by lane: ranks share their upper bits
// The `keep` slots of highest rank of one (sequence, kv head), ties to the lowest slot.  Each
// of 16 waves has a run of slots, 64 at a time, the first eight times with their ranks in
// registers.  The rank of the last slot that stays is found by 8-bit histograms from the top
// (as many as it takes until a bin is taken whole); then each wave counts and places its run.
// Bound by the chain of its steps, some ten barriers: 8 us for 1034 slots, 14 for 16 times 8
// of up to 8192.
extern "C" __global__ __launch_bounds__(SEL_THREADS) void k_kv_select(const EvictArgs a)
{
    constexpr uint32_t IN_REGS = 8;
    const uint32_t kh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63,
                   wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
    __shared__ uint32_t held[SEL_HELD];
    __shared__ __attribute__((aligned(16))) uint32_t hist[256 * SEL_COPIES], bins[256];
    __shared__ int32_t wmax[16];
    __shared__ uint32_t cnt_eq[16], cnt_hole[16], cnt_move[16];
    const uint32_t run = ((n + 15) / 16 + 63) / 64 * 64, j0 = min(n, wave * run), j1 = min(n, j0 + run);
    const uint32_t rounds = (j1 - j0 + 63) / 64; // of this wave
    const uint32_t hold = wave * (SEL_HELD / 16); // its part of held: rounds from IN_REGS on
    uint32_t key[IN_REGS];
    float weight[IN_REGS];
    int32_t newest = INT32_MIN;
#pragma unroll
    for (uint32_t i = 0; i < IN_REGS; ++i)
        if (i < rounds) { // uniform
            const uint32_t j = min(j0 + 64 * i + lane, n - 1);
            weight[i] = acc[j];
            key[i] = (uint32_t)pos[j];
        }
    for (uint32_t i = IN_REGS; i < rounds; ++i)
        newest = max(newest, pos[min(j0 + 64 * i + lane, n - 1)]);
#pragma unroll
    for (uint32_t i = 0; i < IN_REGS; ++i)
        if (i < rounds)
            newest = max(newest, (int32_t)key[i]);
    newest = wave_max_i(newest);
    if (lane == 0)
        wmax[wave] = newest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w)
        newest = max(newest, wmax[w]);
#pragma unroll
    for (uint32_t i = 0; i < IN_REGS; ++i)
        if (i < rounds)
            key[i] = evict_key(a, weight[i], (int32_t)key[i], newest);
    auto made = [&](uint32_t i) { // the rank of a later round's slot, from memory
        const uint32_t j = min(j0 + 64 * i + lane, n - 1);
        return evict_key(a, acc[j], pos[j], newest);
    };
    for (uint32_t i = IN_REGS; i < rounds && (i - IN_REGS) * 64 < SEL_HELD / 16; ++i)
        held[hold + (i - IN_REGS) * 64 + lane] = made(i);
    // f(round, slot, rank) for every round; lanes past the run have slots from j1 on
    auto each = [&](auto &&f) {
#pragma unroll
        for (uint32_t i = 0; i < IN_REGS; ++i)
            if (i < rounds)
                f(j0 + 64 * i + lane, key[i]);
        for (uint32_t i = IN_REGS; i < rounds; ++i)
            f(j0 + 64 * i + lane,
              (i - IN_REGS) * 64 < SEL_HELD / 16 ? held[hold + (i - IN_REGS) * 64 + lane] : made(i));
    };
    uint32_t last = 0, mask = 0, need = keep; // kept: rank & mask above `last`, and `need` of those at it
    bool exact = false;
    for (int pass = 3; pass >= 0 && !exact; --pass) {
        for (uint32_t i = tid; i < 256 * SEL_COPIES / 4; i += SEL_THREADS)
            ((u32x4 *)hist)[i] = u32x4{0, 0, 0, 0};
        __syncthreads();
        each([&](uint32_t j, uint32_t k) {
            if (j < j1 && (k & mask) == last)
                atomicAdd(&hist[((k >> (8 * pass)) & 255) * SEL_COPIES + (lane & (SEL_COPIES - 1))], 1u);
        });
        __syncthreads();
        if (tid < 256) {
            uint32_t v = 0;
#pragma unroll
            for (int i = 0; i < SEL_COPIES / 4; ++i) {
                const u32x4 x = ((const u32x4 *)hist)[tid * (SEL_COPIES / 4) + i];
                v += x[0] + x[1] + x[2] + x[3];
            }
            bins[tid] = v;
        }
        __syncthreads();
        // every wave: lane l holds bins 255 - 4 l downwards; the bin where the count from the
        // top reaches `need`
        const u32x4 x = ((const u32x4 *)bins)[63 - lane];
        const uint32_t four = x[0] + x[1] + x[2] + x[3];
        uint32_t upto = four;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(upto, d);
            upto += lane >= (uint32_t)d ? o : 0;
        }
        const uint32_t at = (uint32_t)__ffsll((unsigned long long)__ballot(upto >= need)) - 1;
        uint32_t left = need - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(four, at));
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c[i] = __builtin_amdgcn_readlane(x[3 - i], at);
        uint32_t bin = 255 - 4 * at, count = c[0];
#pragma unroll
        for (int i = 1; i < 4; ++i)
            if (left > count && bin + i == 256 - 4 * at) { // still passing bins
                left -= count;
                count = c[i];
                --bin;
            }
        last |= bin << (8 * pass);
        mask |= 255u << (8 * pass);
        need = left;
        exact = left == count;
    }
    const uint64_t below = (1ull << lane) - 1;
    uint32_t eq0 = 0;
    if (!exact) { // uniform: only some of the slots at the last rank stay, the lowest
        uint32_t eq = 0;
        each([&](uint32_t j, uint32_t k) { eq += __popcll(__ballot(j < j1 && (k & mask) == last)); });
        if (lane == 0)
            cnt_eq[wave] = eq;
        __syncthreads();
        for (uint32_t w = 0; w < wave; ++w)
            eq0 += cnt_eq[w];
    }
    uint32_t holes = 0, moves = 0, hole0 = 0, move0 = 0;
    for (int place = 0; place < 2; ++place) {
        uint32_t e = eq0;
        each([&](uint32_t j, uint32_t rank) {
            const bool in = j < j1;
            const uint32_t k = rank & mask;
            const uint64_t meq = __ballot(in && k == last);
            const bool kept = in && (k > last || (k == last && (exact || e + __popcll(meq & below) < need)));
            e += __popcll(meq);
            const uint64_t mh = __ballot(in && j < keep && !kept), mm = __ballot(j >= keep && kept);
            if (place) {
                if (in && j < keep)
                    map[j] = kept ? (int32_t)j : ~(int32_t)(hole0 + holes + __popcll(mh & below));
                else if (kept)
                    movers[move0 + moves + __popcll(mm & below)] = (int32_t)j;
            }
            holes += __popcll(mh);
            moves += __popcll(mm);
        });
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
// below: in place, nothing is read that another thread writes.  Bound by memory: 16 sequences of
// 8 kv heads cut to 2048 slots of 128 dims take 47 us, 5.7 TB/s.
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
            const u32x4 k = *(const u32x4 *)(a.c.k + from), v = *(const u32x4 *)(a.c.v + from);
            *(u32x4 *)((uint16_t *)a.k_out + to) = k;
            *(u32x4 *)((uint16_t *)a.v_out + to) = v;
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
