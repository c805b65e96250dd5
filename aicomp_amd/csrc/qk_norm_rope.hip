// RMS norm of every query and key head, rotary positions, append to the paged pools: one launch.
//
//   r = 1 / sqrt(mean_d x_d^2 + eps),  y = x r w                    (w: the query's or the key's weight, D values)
//   (a, b) -> (a cos - b sin, b cos + a sin) for the R / 2 pairs of the first R elements of a head, which are
//   (j, j + R/2) or, interleaved, (2j, 2j + 1); elements R .. D-1 stay y.
//
// Everything is held in float32 and rounded once, to the tensor's type (or to the e4m3 code of an fp8 pool), where the
// rotation by itself (rope_append.hip) repeats the roundings of an eager evaluation.  The tables are float32 too, one angle per
// pair: a bf16 cosine would be the largest error of the result.
//
// Bound by HBM: a row is read once and written once.  A lane has sixteen elements of a row, both elements of each of
// its eight pairs among them: two chunks of eight, R/2 or half a row apart, so that a rotation needs no other lane, the norm's sum
// crosses D/16 of them, and the lanes of a load or store have neighbouring addresses (sixteen elements in a row per lane took
// 47 us where this takes 42).  8192 tokens of 32 / 8 heads of 128, 16-bit: 42.5 us, 4.7 TB/s, where a large copy reaches 5.2; one
// token: 4.3 us, a launch.
#include "rope_math.h"

namespace aicomp {

namespace {

struct NormRopeParams {
    const void* q_in; void* q_out;
    int64_t q_ts, q_hs, qo_ts, qo_hs;          // element strides (token, head)
    const void* key; const void* value;
    int64_t kv_ts, kv_hs;
    const float* q_weight; const float* k_weight;
    float eps;
    const float* cos_tab; const float* sin_tab;
    int64_t tab_stride, tab_rows;
    const int64_t* positions;                  // null: row t of the table belongs to token t
    void* k_pool; void* v_pool;
    const int64_t* slot_mapping;
    const float* k_scale; const float* v_scale;
    int hq, hkv, d, rotary, interleaved, bs;
    int64_t num_slots;
};

// 8 floats -> 8 e4m3 codes: e4m3_rne(clamp(x / scale, +-448)), the plain append's rule
__device__ __forceinline__ uint2 codes8(const float* f, float scale) {
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = fminf(fmaxf(f[j] / scale, -448.f), 448.f);
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// One workgroup per token and slice of its heads (blockIdx.y).  LPR = lanes per row, the power of two at or above D / 16.
template <typename T, bool FP8POOL, int LPR, int NI>
__global__ void __launch_bounds__(256)
qk_norm_rope_append_kernel(NormRopeParams p) {
    const int64_t t = blockIdx.x;
    const int c = (int)threadIdx.x & (LPR - 1);
    const int rows_it = (int)blockDim.x / LPR;                        // heads per pass of the workgroup
    const int hs0 = blockIdx.y * (NI * rows_it) + (int)threadIdx.x / LPR;
    const int nh = p.hq + 2 * p.hkv;
    const int chunks = p.d / 16, turned = p.rotary / 16;              // of a row; of its rotated part
    const bool here = c < chunks;                                     // (a head_dim that is no power of two leaves lanes over)
    // columns of this lane's two chunks: the halves of a region, eight columns in each; the rotated part and the rest are regions
    // of their own where elements R/2 apart are pairs
    const int from = !p.interleaved && c >= turned ? p.rotary : 0, to = !p.interleaved && c < turned ? p.rotary : p.d;
    const int a_col = from + 8 * (c - from / 16), b_col = a_col + (to - from) / 2;

    Raw8<T> ra[NI], rb[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int hs = hs0 + i * rows_it;
        if (hs < nh && here) {
            const bool is_q = hs < p.hq, is_k = hs < p.hq + p.hkv;
            const T* src = is_q ? (const T*)p.q_in + t * p.q_ts + hs * p.q_hs
                                : (is_k ? (const T*)p.key + t * p.kv_ts + (hs - p.hq) * p.kv_hs
                                        : (const T*)p.value + t * p.kv_ts + (hs - p.hq - p.hkv) * p.kv_hs);
            ra[i].load(src + a_col);
            rb[i].load(src + b_col);
        }
    }
    const int64_t pos = p.positions ? p.positions[t] : t;
    const int64_t slot = p.slot_mapping[t];
    if (p.rotary > 0 && (pos < 0 || pos >= p.tab_rows)) return;       // no table row: the token is left alone
    const bool stored = slot >= 0 && slot < p.num_slots;              // otherwise a padding row: the query alone
    const int64_t blk = stored ? slot / p.bs : 0;
    const int off = stored ? (int)(slot - blk * p.bs) : 0;
    float cs[8], sn[8];
    const float* cos_row = p.cos_tab + pos * p.tab_stride;
    const float* sin_row = p.sin_tab + pos * p.tab_stride;
    if (!p.interleaved) {
        if (c < turned) { Row8<float>::load(cos_row + 8 * c, cs); Row8<float>::load(sin_row + 8 * c, sn); }
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int col = k ? b_col : a_col;
            if (col >= p.rotary) continue;
            const float4 x = *(const float4*)(cos_row + col / 2), y = *(const float4*)(sin_row + col / 2);
            cs[4 * k] = x.x; cs[4 * k + 1] = x.y; cs[4 * k + 2] = x.z; cs[4 * k + 3] = x.w;
            sn[4 * k] = y.x; sn[4 * k + 1] = y.y; sn[4 * k + 2] = y.z; sn[4 * k + 3] = y.w;
        }
    }

#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int hs = hs0 + i * rows_it;
        if (hs >= nh) break;                                          // (the lanes of a row leave together)
        const bool is_q = hs < p.hq, is_k = !is_q && hs < p.hq + p.hkv;
        if (!is_q && !stored) break;
        const int h = is_q ? hs : (is_k ? hs - p.hq : hs - p.hq - p.hkv);
        const int64_t row = (blk * p.hkv + h) * p.bs + off;           // pool row of D elements
        if constexpr (!FP8POOL) {
            if (!is_q && !is_k) {                                     // V into a pool of its own type: raw bytes
                if (here) {
                    T* dst = (T*)p.v_pool + row * p.d;
                    ra[i].store(dst + a_col);
                    rb[i].store(dst + b_col);
                }
                continue;
            }
        }
        float a[8], b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.f;
        if (here) { ra[i].unpack(a); rb[i].unpack(b); }
        const float* weight = is_q ? p.q_weight : (is_k ? p.k_weight : nullptr);
        if (weight != nullptr) {
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(b[j], b[j], fmaf(a[j], a[j], sum));
#pragma unroll
            for (int o = 1; o < LPR; o <<= 1) sum += __shfl_xor(sum, o);
            const float r = rsqrtf(sum / (float)p.d + p.eps);
            if (here) {
                float wa[8], wb[8];
                Row8<float>::load(weight + a_col, wa);
                Row8<float>::load(weight + b_col, wb);
#pragma unroll
                for (int j = 0; j < 8; ++j) { a[j] = a[j] * r * wa[j]; b[j] = b[j] * r * wb[j]; }
            }
        }
        if (is_q || is_k) {
            if (p.interleaved) {
                auto turn = [&](float* x, int col, int k) __attribute__((always_inline)) {
                    if (col >= p.rotary) return;
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float u = x[j];
                        x[j] = u * cs[k + j / 2] - x[j + 1] * sn[k + j / 2];
                        x[j + 1] = x[j + 1] * cs[k + j / 2] + u * sn[k + j / 2];
                    }
                };
                turn(a, a_col, 0);
                turn(b, b_col, 4);
            } else if (c < turned) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = a[j];
                    a[j] = x * cs[j] - b[j] * sn[j];
                    b[j] = b[j] * cs[j] + x * sn[j];
                }
            }
        }
        if (!here) continue;
        if (is_q) {
            T* dst = (T*)p.q_out + t * p.qo_ts + h * p.qo_hs;
            Row8<T>::store(dst + a_col, a);
            Row8<T>::store(dst + b_col, b);
        } else if constexpr (FP8POOL) {
            const float sc = (is_k ? p.k_scale : p.v_scale)[h];
            uint8_t* dst = (uint8_t*)(is_k ? p.k_pool : p.v_pool) + row * p.d;
            *(uint2*)(dst + a_col) = codes8(a, sc);
            *(uint2*)(dst + b_col) = codes8(b, sc);
        } else {
            T* dst = (T*)p.k_pool + row * p.d;
            Row8<T>::store(dst + a_col, a);
            Row8<T>::store(dst + b_col, b);
        }
    }
}

template <typename T, bool FP8POOL, int LPR>
void launch_lanes(const NormRopeParams& p, int ni, dim3 grid, dim3 block, hipStream_t stream) {
    if (ni == 1) hipLaunchKernelGGL((qk_norm_rope_append_kernel<T, FP8POOL, LPR, 1>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((qk_norm_rope_append_kernel<T, FP8POOL, LPR, 2>), grid, block, 0, stream, p);
}

template <typename T>
void launch_type(const NormRopeParams& p, bool fp8, int lanes, int ni, dim3 grid, dim3 block, hipStream_t stream) {
#define AICOMP_NORM_ROPE(LPR)                                                                       \
    do {                                                                                            \
        if (fp8) launch_lanes<T, true, LPR>(p, ni, grid, block, stream);                            \
        else launch_lanes<T, false, LPR>(p, ni, grid, block, stream);                               \
    } while (0)
    switch (lanes) {
        case 1: AICOMP_NORM_ROPE(1); break;
        case 2: AICOMP_NORM_ROPE(2); break;
        case 4: AICOMP_NORM_ROPE(4); break;
        case 8: AICOMP_NORM_ROPE(8); break;
        default: AICOMP_NORM_ROPE(16); break;
    }
#undef AICOMP_NORM_ROPE
}

}  // namespace

int launch_qk_norm_rope_kv_append(const NormRopeArgs& a) {
    NormRopeParams p;
    p.q_in = a.q_in; p.q_out = a.q_out; p.q_ts = a.q_ts; p.q_hs = a.q_hs; p.qo_ts = a.qo_ts; p.qo_hs = a.qo_hs;
    p.key = a.key; p.value = a.value; p.kv_ts = a.kv_ts; p.kv_hs = a.kv_hs;
    p.q_weight = a.q_weight; p.k_weight = a.k_weight; p.eps = a.eps;
    p.cos_tab = a.cos_tab; p.sin_tab = a.sin_tab; p.tab_stride = a.tab_stride; p.tab_rows = a.tab_rows;
    p.positions = a.positions; p.k_pool = a.k_pool; p.v_pool = a.v_pool; p.slot_mapping = a.slot_mapping;
    p.k_scale = a.k_scale; p.v_scale = a.v_scale;
    p.hq = a.hq; p.hkv = a.hkv; p.d = a.d; p.rotary = a.rotary; p.interleaved = a.interleaved; p.bs = a.bs;
    p.num_slots = a.num_blocks * a.bs;
    int lanes = 1;
    while (16 * lanes < a.d) lanes *= 2;
    // two heads per lane once there are tokens enough to fill the chip (rope_append.hip has the measurements)
    constexpr int LANES = 128, TOKENS_TWO = 256;
    const int64_t items = (int64_t)(a.hq + 2 * a.hkv) * lanes;
    const int ni = items > LANES && a.num_tokens >= TOKENS_TWO ? 2 : 1;
    const int64_t slices = (items + ni * LANES - 1) / (ni * LANES);
    const int threads = (int)((items + ni * slices * 64 - 1) / (ni * slices * 64)) * 64;
    AICOMP_REQUIRE(a.num_tokens * threads <= UINT32_MAX && slices <= 65535, AICOMP_KV_EINVAL,
                   "qk_norm_rope_kv_append: %lld tokens of %d / %d heads exceed one launch", (long long)a.num_tokens, a.hq, a.hkv);
    dim3 grid((unsigned)a.num_tokens, (unsigned)slices), block(threads);
    const bool fp8 = a.pool_dtype == AICOMP_KV_FP8_E4M3;
    if (a.in_dtype == AICOMP_KV_BF16) launch_type<bf16_t>(p, fp8, lanes, ni, grid, block, a.stream);
    else if (a.in_dtype == AICOMP_KV_F16) launch_type<f16_t>(p, fp8, lanes, ni, grid, block, a.stream);
    else launch_type<float>(p, fp8, lanes, ni, grid, block, a.stream);
    AICOMP_HIP_LAUNCH_CHECK();
    return AICOMP_KV_OK;
}

}  // namespace aicomp
