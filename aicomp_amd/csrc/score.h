// Attention over the paged pools whose scores follow a rule: what its kernels share.
//
// Row at position p of its sequence, key j:
//   s = scale (q . k_j);  cap > 0: s = cap tanh(s / cap);  slopes: s -= slope_h |p - j|
//   visible: first <= j, window > 0: p - j < window, and (j <= p or j < prefix)
// so that the visible keys of a row are one interval.  out = sum e^s v / sum e^s over them; 0 where there are none.
#pragma once

#include "common.h"

namespace aicomp {

struct ScoreArgs {
    void* out;
    const void* query;
    const void* k_pool;
    const void* v_pool;
    const int32_t* block_table;
    int64_t block_table_stride;
    const int32_t* context_lens;
    const int32_t* cu_q_lens;   // NULL: one query row per sequence (decode)
    int num_seqs;
    int64_t rows;               // query rows
    int max_q_len;
    int hq, hkv, d, bs, max_blocks;
    int64_t num_blocks;
    float scale;
    int q_dtype, kv_dtype;
    const float* k_scale;
    const float* v_scale;
    float cap;                  // 0: none
    const float* slopes;        // [Hq] or NULL
    int window;                 // 0: none
    const int32_t* first_keys;  // [rows] or NULL
    const int32_t* prefix_lens; // [num_seqs] or NULL (not with decode)
    int partition_size, num_parts;      // decode: tokens per partition of a row's visible keys; the last takes what is left
    int part_align;             // the first partition begins at the multiple of this at or below the first visible key
    int64_t span;               // chunks: a bound of the keys that a row sees, by which its call is laid out (no row is cut by it)
    float* ws_acc;              // decode: [rows][Hq][num_parts][D]; chunks: [parts][rows][Hq][D], NULL: keys are not divided
    float* ws_ml;               // decode: [rows][Hq][num_parts][2]; chunks: [parts][rows][Hq][2]
    hipStream_t stream;
};

// the rule as the kernels take it
struct ScoreRule {
    int window;
    const int32_t* first_keys;
    const int32_t* prefix_lens;
    const float* slopes;
    float mul;                  // cap == 0: scale * log2(e)
    float cap_mul;              // cap > 0: scale / cap
    float cap_log2;             // cap * log2(e); 0: no cap
};

inline ScoreRule rule_of(const ScoreArgs& a) {
    ScoreRule r;
    r.window = a.window; r.first_keys = a.first_keys; r.prefix_lens = a.prefix_lens; r.slopes = a.slopes;
    r.mul = a.scale * LOG2E;
    r.cap_mul = a.cap > 0.f ? a.scale / a.cap : 0.f;
    r.cap_log2 = a.cap * LOG2E;
    return r;
}

// visible keys [lo, hi) of query row `row` at position pos of sequence seq, whose context is ctx
__device__ __forceinline__ void visible_keys(const ScoreRule& r, int64_t row, int seq, int pos, int ctx, int& lo, int& hi) {
    hi = pos + 1;
    if (r.prefix_lens != nullptr) hi = max(hi, min(r.prefix_lens[seq], ctx));
    lo = r.window > 0 ? max(0, pos - r.window + 1) : 0;
    if (r.first_keys != nullptr) lo = max(lo, r.first_keys[row]);
    lo = min(lo, hi);
}

int launch_score_generic(const ScoreArgs& a);
int launch_score_merge(const ScoreArgs& a);
bool score_prefill_supported(const ScoreArgs& a);
// How a chunk call is laid out: column groups of 16 rows per wave, and the parts that the keys of its rows are divided into.
struct ScoreChunkPlan { int R, parts; };
ScoreChunkPlan score_chunk_plan(const ScoreArgs& a);
int launch_score_prefill(const ScoreArgs& a);

}  // namespace aicomp
