// Attention of query rows over cached rows, as the latent and the tree kernels share it.
//
// Sequence s has n = cu_q_lens[s+1] - cu_q_lens[s] query tokens, the last n of its ctx = context_lens[s] tokens (one each without
// cu_q_lens), hq / hkv heads to a KV head.  Query token i sees key j if
//   j < ctx - n                                        (what was cached before), or
//   j = ctx - n + b, b <= i                            (causal), or with masks: bit b of the token's mask words
// out = softmax(scale q . k_j) v_j over those; a row that sees nothing is zero, as are all rows of a sequence with n > ctx.
#pragma once

#include "common.h"

namespace aicomp {

constexpr int MAX_KEY = 1280, MAX_VALUE = 1024;     // elements of a key and of a value row, which the entry points hold to

struct RowAttnArgs {
    void* out;                  // [rows, hq, dv]
    const void* query;          // [rows, hq, dk]
    const void* k_pool;         // [num_blocks, hkv, bs, dk]
    const void* v_pool;         // rows of v_row elements, the first dv of them the value (latent rows: k_pool, v_row == dk)
    const int32_t* block_table;
    int64_t block_table_stride;
    const int32_t* context_lens;
    const int32_t* cu_q_lens;   // NULL: one query token per sequence
    const int64_t* masks;       // [rows, mask_words] or NULL: causal
    int mask_words;
    int num_seqs;
    int64_t rows;
    int max_q_len;
    int hq, hkv, dk, dv, v_row, bs, max_blocks;
    int64_t num_blocks;
    float scale;
    int q_dtype, kv_dtype;
    const float* k_scale;
    const float* v_scale;
    int longest_context;        // what the caller knows of context_lens (0: nothing); lays the call out, bounds nothing
    void* workspace;
    hipStream_t stream;
};

// Keys and values of expanded latent rows, dense: key token u of sequence s is row cu_k_lens[s] + u.
struct PromptAttnArgs {
    void* out;                  // [rows, heads, dv]
    const void* query;          // [rows, heads, nope + rope]
    const void* key;            // nope elements at u * key_ts + h * key_hs
    int64_t key_ts, key_hs;
    const void* rope_key;       // rope elements at u * rope_ts, for all heads
    int64_t rope_ts;
    const void* value;          // dv elements at u * value_ts + h * value_hs
    int64_t value_ts, value_hs;
    const int32_t* cu_q_lens;
    const int32_t* cu_k_lens;
    int num_seqs;
    int64_t rows, keys;
    int max_q_len;
    int heads, nope, rope, dv;
    float scale;
    int dtype;
    hipStream_t stream;
};

int launch_rows_generic(const RowAttnArgs& a);
bool row_attn_mfma_supported(const RowAttnArgs& a);
size_t row_attn_mfma_workspace_bytes(const RowAttnArgs& a);
int launch_row_attn_mfma(const RowAttnArgs& a);
int launch_prompt_generic(const PromptAttnArgs& a);
bool prompt_attn_mfma_supported(const PromptAttnArgs& a);
int launch_prompt_attn_mfma(const PromptAttnArgs& a);

struct LatentAppendArgs {
    const void* latent; int64_t latent_stride;          // [tokens, latent_dim + rope_dim]
    const float* weight; float eps;                     // [latent_dim]; NULL: not normed
    const float* cos_tab; const float* sin_tab;
    int64_t tab_stride, tab_rows;
    int interleaved;
    const int64_t* positions;                           // NULL: row t of the tables belongs to token t
    const void* q_in; void* q_out;                      // [tokens, heads, rope_dim]; NULL: none
    int64_t q_ts, q_hs, qo_ts, qo_hs;
    void* rows_out; int64_t rows_stride;                // NULL: none
    void* pool; const int64_t* slot_mapping;
    int64_t num_tokens;
    int heads, latent_dim, rope_dim;
    int64_t num_slots;
    int dtype;
    hipStream_t stream;
};
int launch_latent_append(const LatentAppendArgs& a);

struct KeepRowsArgs {
    void* const* pools; int num_pools;
    int64_t row_bytes; int hkv, bs;
    int64_t num_blocks;
    const int32_t* block_table; int64_t block_table_stride; int max_blocks;
    const int32_t* first; const int32_t* keep; const int32_t* cu_keep;
    int num_seqs; int64_t total;
    hipStream_t stream;
};
int launch_keep_rows(const KeepRowsArgs& a);

}  // namespace aicomp
