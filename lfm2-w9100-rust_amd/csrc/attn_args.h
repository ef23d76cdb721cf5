// attn_args.h -- kernel arguments of the cache-attention operators, shared by the host
// launcher (attn_ops.cpp) and the gfx950 kernels (lfm_attn.hip).  Every kernel takes one
// of these structs by value.
#pragma once
#include <hip/hip_vector_types.h>
#include <stdint.h>

// K and V of n_seq sequences: element (b, h, slot, d) at b * ss + h * hs + slot * ts + d.
struct KvView {
    const uint16_t *k, *v;
    const int32_t *len; // slots in use per sequence, clamped to [0, slots] by the kernels
    int64_t ss, hs, ts;
    uint32_t n_seq, kv_heads, slots;
};

// The rows of a call: q[row][head][d] and out alike.  start (n_seq + 1 entries) gives each
// sequence's rows; null: row b is sequence b's.
struct RowsView {
    const void *q;
    void *out;
    float *lse; // nullable: [row][head], natural logarithm
    const int32_t *start;
    int64_t q_rs, q_hs, o_rs, o_hs;
    uint32_t heads, n_rows;
    float cfrac, cexp; // cexp = scale * log2(e), a normal number = cfrac * 2^cpow, cfrac in [0.5, 1)
};

#define MAX_GROUP 128     // query heads of a kv head
#define TILE_TILES 2      // row tiles a wave of the larger tile kernel
#define SCORED_SLOTS 1024 // slots a workgroup of k_scored_join
#define SUM_KEYS 256      // slots a workgroup of k_attn_weights: four waves of 64
#define MOST_SUM_PARTS 16 // parts of the rows that k_attn_weights sums apart

struct AttnOpArgs {
    KvView own;    // slots of the row's own sequence, causal
    KvView prefix; // k null: none; else one sequence, visible to every row
    RowsView r;
    uint32_t window, sinks; // window 0: unlimited
    uint32_t group;         // query heads of a kv head
    // Key ranges, 64 at most: own_splits of the own slots, then prefix_splits of the prefix.  Where
    // there is more than one in all, range s of row r, head h writes its softmax state to
    // ml[(s * n_rows + r) * heads + h] = {log2 offset, sum} and its unnormalized output
    // beside it in o, and k_attn_merge joins them.
    uint32_t own_splits, prefix_splits;
    uint32_t prefix_groups, own_groups; // row groups: of the whole batch, of one token
    uint32_t step_prefix;               // items of the step kernel that are the prefix's
    float2 *ml;
    float *o;
    // scored: scores[(b * heads + h) * score_row + j] = q . k (F32 rows: 2^cpow q . k, which is in
    // range where the score is); score_row is slots rounded up to whole blocks
    float *scores;
    uint32_t score_row;
    uint32_t sum_parts;
    float *sums;   // [sum_parts][n_seq][kv_heads][slots] where there is more than one
    float2 *stats; // nullable: per row and head {log2 offset, 1 / sum} of its weights
    const float *acc; // nullable
    float *acc_out;   // [n_seq][kv_heads][slots]
};

// Eviction, both steps: the choice, per (sequence, kv head) the source slot of each of the
// `keep` slots that stay, and the move.
struct EvictArgs {
    KvView c;
    void *k_out, *v_out; // may be c.k and c.v (then with its strides): in place
    int64_t oss, ohs, ots;
    const float *acc;    // [n_seq][kv_heads][slots]
    const int32_t *pos;
    float *acc_out;      // [n_seq][kv_heads][out_slots]
    int32_t *pos_out, *len_out;
    uint32_t keep, sinks, recent, out_slots, dim;
    uint32_t in_place, acc_in_place, pos_in_place;
    // workspace, per (sequence, kv head): map[n] (n < keep) is slot n itself, or ~i for
    // the i-th hole, which movers[i] fills; head = {slots that remain, whether any leaves}
    int32_t *map, *movers, *head;
};
