// C entry points of the latent rows, the trees of drafts and the accepted rows (include/aicomp_kv.h): checks, then the launchers.
#include "row_attn.h"

#include <math.h>
#include <string.h>

#include <algorithm>
#include <memory>
#include <new>

using namespace aicomp;

// tokens that a 32-bit place counts, with a tile beyond the last
static const int64_t MAX_TOKENS = INT32_MAX - 1023;

// Whether a key of two parts fits, whose sum may pass 32 bits.
static bool key_fits(int a, int b) { return (int64_t)a + b <= MAX_KEY; }

static bool float_type(int dt) { return dt == AICOMP_KV_F32 || is_16bit_float(dt); }

// What both paged calls check; the sizes of a row are the caller's.
static int check_rows(const RowAttnArgs& a, const char* who) {
    AICOMP_REQUIRE(a.hq > 0 && a.hkv > 0 && a.hq % a.hkv == 0 && a.hq <= 65535, AICOMP_KV_EINVAL,
                   "%s: %d query heads are not a multiple of %d KV heads, or more than 65535", who, a.hq, a.hkv);
    AICOMP_REQUIRE(a.bs > 0 && a.max_blocks > 0 && a.num_blocks > 0 && (int64_t)a.max_blocks * a.bs <= MAX_TOKENS, AICOMP_KV_EINVAL,
                   "%s: bad sizes (block_size %d, max_blocks %d, num_blocks %lld)", who, a.bs, a.max_blocks, (long long)a.num_blocks);
    AICOMP_REQUIRE(a.block_table_stride >= a.max_blocks, AICOMP_KV_EINVAL, "%s: block table stride %lld < width %d", who,
                   (long long)a.block_table_stride, a.max_blocks);
    AICOMP_REQUIRE(isfinite(3.f * a.scale), AICOMP_KV_EINVAL, "%s: scale must be finite (got %g)", who, (double)a.scale);
    AICOMP_REQUIRE(a.longest_context >= 0, AICOMP_KV_EINVAL, "%s: negative longest context", who);
    if (a.cu_q_lens != nullptr)
        AICOMP_REQUIRE(a.max_q_len > 0 && a.max_q_len <= a.rows && a.rows <= MAX_TOKENS, AICOMP_KV_EINVAL,
                       "%s: max_q_len %d out of range (total %lld)", who, a.max_q_len, (long long)a.rows);
    else
        AICOMP_REQUIRE(a.rows == a.num_seqs, AICOMP_KV_EINVAL, "%s: without cu_q_lens there is one row per sequence", who);
    AICOMP_REQUIRE(a.masks == nullptr ? a.mask_words == 0 : a.cu_q_lens != nullptr && a.mask_words > 0 && (uintptr_t)a.masks % 8 == 0,
                   AICOMP_KV_EINVAL, "%s: masks of %d words need cu_q_lens, and words their masks", who, a.mask_words);
    AICOMP_REQUIRE(((uintptr_t)a.query | (uintptr_t)a.out | (uintptr_t)a.k_pool | (uintptr_t)a.v_pool) % 16 == 0, AICOMP_KV_EUNSUPPORTED,
                   "%s: pointers must be 16-byte aligned", who);
    return AICOMP_KV_OK;
}

// The call of checked arguments.
static int attend(const RowAttnArgs& a, size_t workspace_bytes, const char* who) {
    if (!row_attn_mfma_supported(a)) return launch_rows_generic(a);
    const size_t need = row_attn_mfma_workspace_bytes(a);
    AICOMP_REQUIRE(need == 0 || (a.workspace && workspace_bytes >= need), AICOMP_KV_EWORKSPACE,
                   "%s: workspace of %zu bytes needed, %zu given", who, need, a.workspace ? workspace_bytes : (size_t)0);
    AICOMP_REQUIRE(need == 0 || (uintptr_t)a.workspace % 16 == 0, AICOMP_KV_EINVAL, "%s: workspace must be 16-byte aligned", who);
    return launch_row_attn_mfma(a);
}

// The sizes of a call, for its workspace: 0 for what the call refuses.
static size_t workspace_of(const RowAttnArgs& a) {
    if (a.num_seqs <= 0 || a.rows <= 0 || a.max_q_len <= 0 || a.max_q_len > a.rows || a.hq <= 0 || a.hkv <= 0 || a.hq % a.hkv ||
        a.bs <= 0 || a.max_blocks <= 0 || a.longest_context < 0 || !row_attn_mfma_supported(a))
        return 0;
    return row_attn_mfma_workspace_bytes(a);
}

extern "C" {

int aicomp_latent_kv_append(const void* latent, int64_t latent_stride, const float* weight, float eps, const float* cos, const float* sin,
                            int64_t table_stride, int64_t table_rows, int interleaved, const int64_t* positions, const void* q_in,
                            void* q_out, int64_t q_token_stride, int64_t q_head_stride, int64_t qo_token_stride, int64_t qo_head_stride,
                            void* rows_out, int64_t rows_stride, void* pool, const int64_t* slot_mapping, int64_t num_tokens,
                            int num_heads, int latent_dim, int rope_dim, int block_size, int64_t num_blocks, int dtype, void* stream) {
    const char* who = "latent_kv_append";
    AICOMP_REQUIRE(num_tokens >= 0, AICOMP_KV_EINVAL, "%s: negative token count", who);
    if (num_tokens == 0) return AICOMP_KV_OK;
    AICOMP_REQUIRE(latent && cos && sin && pool && slot_mapping && !q_in == !q_out, AICOMP_KV_EINVAL, "%s: null pointer", who);
    AICOMP_REQUIRE(num_heads >= 0 && (num_heads > 0 || !q_in) && block_size > 0 && num_blocks > 0 &&
                   num_blocks <= INT64_MAX / block_size, AICOMP_KV_EINVAL,
                   "%s: bad sizes (heads %d, block_size %d, blocks %lld)", who, num_heads, block_size, (long long)num_blocks);
    AICOMP_REQUIRE(float_type(dtype), AICOMP_KV_EUNSUPPORTED, "%s: rows must be float32, bfloat16 or float16 (got %d)", who, dtype);
    AICOMP_REQUIRE(latent_dim > 0 && latent_dim % 16 == 0 && rope_dim > 0 && rope_dim % 16 == 0, AICOMP_KV_EUNSUPPORTED,
                   "%s: latent and rotated parts of %d and %d elements are not multiples of 16", who, latent_dim, rope_dim);
    AICOMP_REQUIRE(table_rows > 0 && table_stride >= rope_dim / 2, AICOMP_KV_EINVAL, "%s: cos / sin tables of %d columns are needed", who,
                   rope_dim / 2);
    AICOMP_REQUIRE(!weight || (eps >= 0.f && isfinite(eps)), AICOMP_KV_EINVAL, "%s: eps must be finite and not negative (got %g)", who,
                   (double)eps);
    const int64_t width = (int64_t)latent_dim + rope_dim, v = 16 / dtype_size(dtype);
    AICOMP_REQUIRE(latent_stride >= width && (!rows_out || rows_stride >= width) && (!q_in || (q_token_stride >= 0 && qo_token_stride >= 0 &&
                   q_head_stride >= rope_dim && qo_head_stride >= rope_dim)), AICOMP_KV_EINVAL, "%s: strides overlap rows", who);
    AICOMP_REQUIRE((latent_stride | (rows_out ? rows_stride : 0) |
                    (q_in ? q_token_stride | q_head_stride | qo_token_stride | qo_head_stride : 0)) % v == 0 && table_stride % 4 == 0,
                   AICOMP_KV_EUNSUPPORTED, "%s: strides must be multiples of %lld elements (16 bytes)", who, (long long)v);
    AICOMP_REQUIRE(((uintptr_t)latent | (uintptr_t)weight | (uintptr_t)cos | (uintptr_t)sin | (uintptr_t)q_in | (uintptr_t)q_out |
                    (uintptr_t)rows_out | (uintptr_t)pool) % 16 == 0, AICOMP_KV_EUNSUPPORTED, "%s: pointers must be 16-byte aligned", who);
    LatentAppendArgs a;
    a.latent = latent; a.latent_stride = latent_stride; a.weight = weight; a.eps = eps; a.cos_tab = cos; a.sin_tab = sin;
    a.tab_stride = table_stride; a.tab_rows = table_rows; a.interleaved = interleaved ? 1 : 0; a.positions = positions;
    a.q_in = q_in; a.q_out = q_out; a.q_ts = q_token_stride; a.q_hs = q_head_stride; a.qo_ts = qo_token_stride; a.qo_hs = qo_head_stride;
    a.rows_out = rows_out; a.rows_stride = rows_stride; a.pool = pool; a.slot_mapping = slot_mapping; a.num_tokens = num_tokens;
    a.heads = num_heads; a.latent_dim = latent_dim; a.rope_dim = rope_dim; a.num_slots = num_blocks * block_size; a.dtype = dtype;
    a.stream = (hipStream_t)stream;
    return launch_latent_append(a);
}

size_t aicomp_paged_latent_workspace_bytes(int num_seqs, int64_t total_q, int max_q_len, int num_heads, int latent_dim, int rope_dim,
                                           int block_size, int max_blocks_per_seq, int dtype, int longest_context) {
    if (latent_dim <= 0 || rope_dim < 0 || latent_dim > MAX_VALUE || !key_fits(latent_dim, rope_dim)) return 0;
    RowAttnArgs a;
    memset(&a, 0, sizeof(a));
    a.num_seqs = num_seqs; a.rows = total_q; a.max_q_len = max_q_len; a.hq = num_heads; a.hkv = 1; a.dk = latent_dim + rope_dim;
    a.dv = latent_dim; a.v_row = a.dk; a.bs = block_size; a.max_blocks = max_blocks_per_seq; a.q_dtype = a.kv_dtype = dtype;
    a.longest_context = longest_context;
    return workspace_of(a);
}

int aicomp_paged_latent_attn(void* out, const void* query, const void* pool, const int32_t* block_table, int64_t block_table_stride,
                             const int32_t* context_lens, const int32_t* cu_q_lens, const int64_t* tree_masks, int mask_words,
                             int num_seqs, int64_t total_q, int max_q_len, int num_heads, int latent_dim, int rope_dim, int block_size,
                             int max_blocks_per_seq, int64_t num_blocks, float scale, int dtype, int longest_context, void* workspace,
                             size_t workspace_bytes, void* stream) {
    const char* who = "paged_latent_attn";
    AICOMP_REQUIRE(num_seqs >= 0 && total_q >= 0, AICOMP_KV_EINVAL, "%s: negative sizes", who);
    if (num_seqs == 0 || total_q == 0) return AICOMP_KV_OK;
    AICOMP_REQUIRE(out && query && pool && block_table && context_lens, AICOMP_KV_EINVAL, "%s: null pointer", who);
    AICOMP_REQUIRE(latent_dim > 0 && latent_dim % 16 == 0 && rope_dim >= 0 && rope_dim % 16 == 0, AICOMP_KV_EUNSUPPORTED,
                   "%s: latent and rotated parts of %d and %d elements are not multiples of 16", who, latent_dim, rope_dim);
    AICOMP_REQUIRE(latent_dim <= MAX_VALUE && key_fits(latent_dim, rope_dim), AICOMP_KV_EUNSUPPORTED,
                   "%s: rows of %d + %d elements, at most %d of the latent part and %d in all", who, latent_dim, rope_dim, MAX_VALUE, MAX_KEY);
    AICOMP_REQUIRE(float_type(dtype), AICOMP_KV_EUNSUPPORTED, "%s: rows must be float32, bfloat16 or float16 (got %d)", who, dtype);
    RowAttnArgs a;
    memset(&a, 0, sizeof(a));
    a.out = out; a.query = query; a.k_pool = pool; a.v_pool = pool; a.block_table = block_table; a.block_table_stride = block_table_stride;
    a.context_lens = context_lens; a.cu_q_lens = cu_q_lens; a.masks = tree_masks; a.mask_words = mask_words; a.num_seqs = num_seqs;
    a.rows = total_q; a.max_q_len = cu_q_lens ? max_q_len : 1; a.hq = num_heads; a.hkv = 1; a.dk = latent_dim + rope_dim; a.dv = latent_dim;
    a.v_row = a.dk; a.bs = block_size; a.max_blocks = max_blocks_per_seq; a.num_blocks = num_blocks; a.scale = scale; a.q_dtype = dtype;
    a.kv_dtype = dtype; a.longest_context = longest_context; a.workspace = workspace; a.stream = (hipStream_t)stream;
    const int rc = check_rows(a, who);
    if (rc) return rc;
    return attend(a, workspace_bytes, who);
}

size_t aicomp_paged_tree_workspace_bytes(int num_seqs, int64_t total_q, int max_q_len, int num_q_heads, int num_kv_heads, int head_dim,
                                         int block_size, int max_blocks_per_seq, int q_dtype, int kv_dtype, int longest_context) {
    RowAttnArgs a;
    memset(&a, 0, sizeof(a));
    a.num_seqs = num_seqs; a.rows = total_q; a.max_q_len = max_q_len; a.hq = num_q_heads; a.hkv = num_kv_heads;
    a.dk = a.dv = a.v_row = head_dim; a.bs = block_size; a.max_blocks = max_blocks_per_seq; a.q_dtype = q_dtype; a.kv_dtype = kv_dtype;
    a.longest_context = longest_context;
    return workspace_of(a);
}

int aicomp_paged_tree_attn(void* out, const void* query, const void* k_pool, const void* v_pool, const int32_t* block_table,
                           int64_t block_table_stride, const int32_t* context_lens, const int32_t* cu_q_lens, const int64_t* tree_masks,
                           int mask_words, int num_seqs, int64_t total_q, int max_q_len, int num_q_heads, int num_kv_heads, int head_dim,
                           int block_size, int max_blocks_per_seq, int64_t num_blocks, float scale, int q_dtype, int kv_dtype,
                           const float* k_scale, const float* v_scale, int longest_context, void* workspace, size_t workspace_bytes,
                           void* stream) {
    const char* who = "paged_tree_attn";
    AICOMP_REQUIRE(num_seqs >= 0 && total_q >= 0, AICOMP_KV_EINVAL, "%s: negative sizes", who);
    if (num_seqs == 0 || total_q == 0) return AICOMP_KV_OK;
    AICOMP_REQUIRE(out && query && k_pool && v_pool && block_table && context_lens && cu_q_lens && tree_masks, AICOMP_KV_EINVAL,
                   "%s: null pointer", who);
    AICOMP_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, AICOMP_KV_EUNSUPPORTED,
                   "%s: head_dim %d not supported (64, 128, 256)", who, head_dim);
    AICOMP_REQUIRE((q_dtype == AICOMP_KV_F32 && kv_dtype == AICOMP_KV_F32) ||
                   (is_16bit_float(q_dtype) && (kv_dtype == q_dtype || kv_dtype == AICOMP_KV_FP8_E4M3)), AICOMP_KV_EUNSUPPORTED,
                   "%s: unsupported type pair (query %d, pool %d); supported: f32/f32, bf16/bf16, f16/f16, bf16/fp8, f16/fp8", who, q_dtype,
                   kv_dtype);
    const bool fp8 = kv_dtype == AICOMP_KV_FP8_E4M3;
    AICOMP_REQUIRE(!fp8 || (k_scale && v_scale), AICOMP_KV_EINVAL, "%s: an fp8 pool needs k_scale and v_scale", who);
    RowAttnArgs a;
    memset(&a, 0, sizeof(a));
    a.out = out; a.query = query; a.k_pool = k_pool; a.v_pool = v_pool; a.block_table = block_table;
    a.block_table_stride = block_table_stride; a.context_lens = context_lens; a.cu_q_lens = cu_q_lens; a.masks = tree_masks;
    a.mask_words = mask_words; a.num_seqs = num_seqs; a.rows = total_q; a.max_q_len = max_q_len; a.hq = num_q_heads; a.hkv = num_kv_heads;
    a.dk = a.dv = a.v_row = head_dim; a.bs = block_size; a.max_blocks = max_blocks_per_seq; a.num_blocks = num_blocks; a.scale = scale;
    a.q_dtype = q_dtype; a.kv_dtype = kv_dtype; a.k_scale = fp8 ? k_scale : nullptr; a.v_scale = fp8 ? v_scale : nullptr;
    a.longest_context = longest_context; a.workspace = workspace; a.stream = (hipStream_t)stream;
    const int rc = check_rows(a, who);
    if (rc) return rc;
    return attend(a, workspace_bytes, who);
}

int aicomp_latent_prompt_attn(void* out, const void* query, const void* key, int64_t key_token_stride, int64_t key_head_stride,
                              const void* rope_key, int64_t rope_token_stride, const void* value, int64_t value_token_stride,
                              int64_t value_head_stride, const int32_t* cu_q_lens, const int32_t* cu_k_lens, int num_seqs,
                              int64_t total_q, int64_t total_k, int max_q_len, int num_heads, int nope_dim, int rope_dim, int value_dim,
                              float scale, int dtype, void* stream) {
    const char* who = "latent_prompt_attn";
    AICOMP_REQUIRE(num_seqs >= 0 && total_q >= 0 && total_k >= 0, AICOMP_KV_EINVAL, "%s: negative sizes", who);
    if (num_seqs == 0 || total_q == 0) return AICOMP_KV_OK;
    AICOMP_REQUIRE(out && query && cu_q_lens && cu_k_lens && (total_k == 0 || (key && rope_key && value)), AICOMP_KV_EINVAL,
                   "%s: null pointer", who);
    AICOMP_REQUIRE(num_heads > 0 && num_heads <= 65535 && total_q <= MAX_TOKENS && total_k <= MAX_TOKENS, AICOMP_KV_EINVAL,
                   "%s: bad sizes (heads %d, rows %lld, keys %lld)", who, num_heads, (long long)total_q, (long long)total_k);
    AICOMP_REQUIRE(nope_dim > 0 && nope_dim % 16 == 0 && rope_dim > 0 && rope_dim % 16 == 0 && value_dim > 0 && value_dim % 16 == 0,
                   AICOMP_KV_EUNSUPPORTED, "%s: heads of %d + %d key and %d value elements are not multiples of 16", who, nope_dim,
                   rope_dim, value_dim);
    AICOMP_REQUIRE(key_fits(nope_dim, rope_dim) && value_dim <= MAX_VALUE, AICOMP_KV_EUNSUPPORTED,
                   "%s: heads of %d + %d key and %d value elements, at most %d and %d", who, nope_dim, rope_dim, value_dim, MAX_KEY, MAX_VALUE);
    AICOMP_REQUIRE(float_type(dtype), AICOMP_KV_EUNSUPPORTED, "%s: rows must be float32, bfloat16 or float16 (got %d)", who, dtype);
    AICOMP_REQUIRE(max_q_len > 0 && max_q_len <= total_q, AICOMP_KV_EINVAL, "%s: max_q_len %d out of range (total %lld)", who, max_q_len,
                   (long long)total_q);
    AICOMP_REQUIRE(isfinite(3.f * scale), AICOMP_KV_EINVAL, "%s: scale must be finite (got %g)", who, (double)scale);
    AICOMP_REQUIRE(key_head_stride >= 0 && value_head_stride >= 0 && key_token_stride >= 0 && value_token_stride >= 0 &&
                   rope_token_stride >= 0, AICOMP_KV_EINVAL, "%s: negative strides", who);
    const int64_t v = 16 / dtype_size(dtype);
    AICOMP_REQUIRE((key_token_stride | key_head_stride | value_token_stride | value_head_stride | rope_token_stride) % v == 0,
                   AICOMP_KV_EUNSUPPORTED, "%s: strides must be multiples of %lld elements (16 bytes)", who, (long long)v);
    AICOMP_REQUIRE(((uintptr_t)out | (uintptr_t)query | (uintptr_t)key | (uintptr_t)rope_key | (uintptr_t)value) % 16 == 0,
                   AICOMP_KV_EUNSUPPORTED, "%s: pointers must be 16-byte aligned", who);
    PromptAttnArgs a;
    a.out = out; a.query = query; a.key = key; a.key_ts = key_token_stride; a.key_hs = key_head_stride; a.rope_key = rope_key;
    a.rope_ts = rope_token_stride; a.value = value; a.value_ts = value_token_stride; a.value_hs = value_head_stride;
    a.cu_q_lens = cu_q_lens; a.cu_k_lens = cu_k_lens; a.num_seqs = num_seqs; a.rows = total_q; a.keys = total_k; a.max_q_len = max_q_len;
    a.heads = num_heads; a.nope = nope_dim; a.rope = rope_dim; a.dv = value_dim; a.scale = scale; a.dtype = dtype;
    a.stream = (hipStream_t)stream;
    return prompt_attn_mfma_supported(a) ? launch_prompt_attn_mfma(a) : launch_prompt_generic(a);
}

int aicomp_kv_keep_rows(void* const* pools, int num_pools, int64_t row_bytes, int num_kv_heads, int block_size, int64_t num_blocks,
                        const int32_t* block_table, int64_t block_table_stride, int max_blocks_per_seq, const int32_t* first,
                        const int32_t* keep, const int32_t* cu_keep, int num_seqs, int64_t total_keep, void* stream) {
    const char* who = "keep_rows";
    AICOMP_REQUIRE(num_pools >= 0 && num_seqs >= 0 && total_keep >= 0, AICOMP_KV_EINVAL, "%s: negative sizes", who);
    if (num_pools == 0 || num_seqs == 0 || total_keep == 0) return AICOMP_KV_OK;
    AICOMP_REQUIRE(pools && block_table && first && keep && cu_keep, AICOMP_KV_EINVAL, "%s: null pointer", who);
    for (int i = 0; i < num_pools; ++i)
        AICOMP_REQUIRE(pools[i], AICOMP_KV_EINVAL, "%s: pool %d is a null pointer", who, i);
    AICOMP_REQUIRE(row_bytes > 0 && row_bytes <= INT32_MAX && num_kv_heads > 0 && block_size > 0 && num_blocks > 0 &&
                   max_blocks_per_seq > 0 && (int64_t)max_blocks_per_seq * block_size <= MAX_TOKENS &&
                   block_table_stride >= max_blocks_per_seq && total_keep <= MAX_TOKENS, AICOMP_KV_EINVAL,
                   "%s: bad sizes (row of %lld bytes, Hkv %d, BS %d, blocks %lld, table %d)", who, (long long)row_bytes, num_kv_heads,
                   block_size, (long long)num_blocks, max_blocks_per_seq);
    AICOMP_REQUIRE(row_bytes <= INT32_MAX / num_kv_heads && num_seqs <= 16777215, AICOMP_KV_EINVAL,
                   "%s: %d sequences, or %d heads of %lld bytes, exceed one launch", who, num_seqs, num_kv_heads, (long long)row_bytes);
    // Two workgroups that moved the rows of one pool would read what the other has moved already
    int64_t bytes = row_bytes;
    AICOMP_REQUIRE(!__builtin_mul_overflow(bytes, (int64_t)num_kv_heads * block_size, &bytes) &&
                   !__builtin_mul_overflow(bytes, num_blocks, &bytes), AICOMP_KV_EINVAL, "%s: pools of more than 2^63 bytes", who);
    std::unique_ptr<uintptr_t[]> places(new (std::nothrow) uintptr_t[num_pools]);
    AICOMP_REQUIRE(places, AICOMP_KV_EINVAL, "%s: no host memory for %d pools", who, num_pools);
    std::copy((const uintptr_t*)pools, (const uintptr_t*)pools + num_pools, places.get());
    if (!std::is_sorted(places.get(), places.get() + num_pools)) std::sort(places.get(), places.get() + num_pools);
    for (int i = 1; i < num_pools; ++i)
        AICOMP_REQUIRE(places[i] - places[i - 1] >= (uintptr_t)bytes, AICOMP_KV_EINVAL, "%s: two of the pools overlap", who);
    KeepRowsArgs a;
    a.pools = pools; a.num_pools = num_pools; a.row_bytes = row_bytes; a.hkv = num_kv_heads; a.bs = block_size; a.num_blocks = num_blocks;
    a.block_table = block_table; a.block_table_stride = block_table_stride; a.max_blocks = max_blocks_per_seq; a.first = first;
    a.keep = keep; a.cu_keep = cu_keep; a.num_seqs = num_seqs; a.total = total_keep; a.stream = (hipStream_t)stream;
    return launch_keep_rows(a);
}

}  // extern "C"
