// The cache row of a token of latent attention, and the rotated part of its queries, in one launch:
//
//   c <- c / sqrt(mean(c^2) + eps) * w                          the latent part, C elements, shared by all heads
//   (a, b) -> (a cos - b sin, b cos + a sin)                    pairs of the row's last D elements and of D elements of each query head,
//                                                               (j, j + D/2) or, interleaved, (2j, 2j + 1)
// and the row into its slot of the paged pool [num_blocks, block_size, C + D].  Float32 throughout, rounded once.
//
// Bound by HBM for long prompts and by the launch for one token.  Two kinds of workgroups in the one launch: a wave has a token's
// latent part, whose squares it sums by lane moves; or each lane has sixteen elements of a rotated row (two chunks of eight that
// hold both elements of each of its pairs), rows of all tokens one after the other, so that no lane is idle whatever the heads are.
// 8192 tokens of 16 heads: 12.4 us, 4.4 TB/s; one token: 2.6 us.
#include "row_attn.h"
#include "rope_math.h"

namespace aicomp {

namespace {

constexpr int MAX_LATENT = 1024;           // two chunks of eight elements to a lane
constexpr int MAX_ROPE = 65536;            // (a row's elements are counted in 32 bits)

struct LatentAppendParams {
    LatentAppendArgs a;
    uint32_t latent_wgs;                   // workgroups of latent parts; those of rotated rows follow
    uint32_t items;                        // lanes that rotated rows take
};

template <typename T>
__global__ void __launch_bounds__(256)
latent_append_kernel(LatentAppendParams p) {
    const LatentAppendArgs& a = p.a;
    const int width = a.latent_dim + a.rope_dim;
    if (blockIdx.x < p.latent_wgs) {
        const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
        if (t >= a.num_tokens) return;
        const int lane = threadIdx.x & 63, chunks = a.latent_dim / 8;
        const int64_t pos = a.positions ? a.positions[t] : t, slot = a.slot_mapping[t];
        const bool stored = slot >= 0 && slot < a.num_slots;
        Raw8<T> raw[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (lane + 64 * k < chunks) raw[k].load((const T*)a.latent + t * a.latent_stride + 8 * (lane + 64 * k));
        if (pos < 0 || pos >= a.tab_rows) return;                    // no table row: the token is left alone
        float x[2][8], sum = 0.f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (lane + 64 * k >= chunks) continue;
            raw[k].unpack(x[k]);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(x[k][e], x[k][e], sum);
        }
        if (a.weight != nullptr) {
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
            const float r = rsqrtf(sum / (float)a.latent_dim + a.eps);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (lane + 64 * k >= chunks) continue;
                float w[8];
                Row8<float>::load(a.weight + 8 * (lane + 64 * k), w);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[k][e] = x[k][e] * r * w[e];
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int col = 8 * (lane + 64 * k);
            if (lane + 64 * k >= chunks) continue;
            if (stored) Row8<T>::store((T*)a.pool + slot * width + col, x[k]);
            if (a.rows_out != nullptr) Row8<T>::store((T*)a.rows_out + t * a.rows_stride + col, x[k]);
        }
        return;
    }
    const uint32_t item = (blockIdx.x - p.latent_wgs) * 256 + threadIdx.x;
    if (item >= p.items) return;
    const uint32_t per = a.rope_dim / 16, row = item / per, c = item - row * per;       // lanes to a row
    const uint32_t rows = (a.q_in ? (uint32_t)a.heads : 0) + 1;                         // of a token; row 0 is the shared key
    const int64_t t = row / rows;
    const int h = (int)(row - (uint32_t)t * rows) - 1;
    const int a_col = 8 * c, b_col = a_col + a.rope_dim / 2;
    const T* src = h < 0 ? (const T*)a.latent + t * a.latent_stride + a.latent_dim : (const T*)a.q_in + t * a.q_ts + h * a.q_hs;
    Raw8<T> ra, rb;
    ra.load(src + a_col);
    rb.load(src + b_col);
    const int64_t pos = a.positions ? a.positions[t] : t;
    if (pos < 0 || pos >= a.tab_rows) return;
    float x[8], y[8], cs[8], sn[8];
    const float* cos_row = a.cos_tab + pos * a.tab_stride;
    const float* sin_row = a.sin_tab + pos * a.tab_stride;
    ra.unpack(x);
    rb.unpack(y);
    if (!a.interleaved) {
        Row8<float>::load(cos_row + a_col, cs);
        Row8<float>::load(sin_row + a_col, sn);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float u = x[e];
            x[e] = u * cs[e] - y[e] * sn[e];
            y[e] = y[e] * cs[e] + u * sn[e];
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int col = (k ? b_col : a_col) / 2;
            const float4 u = *(const float4*)(cos_row + col), v = *(const float4*)(sin_row + col);
            cs[4 * k] = u.x; cs[4 * k + 1] = u.y; cs[4 * k + 2] = u.z; cs[4 * k + 3] = u.w;
            sn[4 * k] = v.x; sn[4 * k + 1] = v.y; sn[4 * k + 2] = v.z; sn[4 * k + 3] = v.w;
        }
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float u = x[e], v = y[e];
            x[e] = u * cs[e / 2] - x[e + 1] * sn[e / 2];
            x[e + 1] = x[e + 1] * cs[e / 2] + u * sn[e / 2];
            y[e] = v * cs[4 + e / 2] - y[e + 1] * sn[4 + e / 2];
            y[e + 1] = y[e + 1] * cs[4 + e / 2] + v * sn[4 + e / 2];
        }
    }
    if (h >= 0) {
        T* dst = (T*)a.q_out + t * a.qo_ts + h * a.qo_hs;
        Row8<T>::store(dst + a_col, x);
        Row8<T>::store(dst + b_col, y);
        return;
    }
    const int64_t slot = a.slot_mapping[t];
    if (slot >= 0 && slot < a.num_slots) {
        T* dst = (T*)a.pool + slot * width + a.latent_dim;
        Row8<T>::store(dst + a_col, x);
        Row8<T>::store(dst + b_col, y);
    }
    if (a.rows_out != nullptr) {
        T* dst = (T*)a.rows_out + t * a.rows_stride + a.latent_dim;
        Row8<T>::store(dst + a_col, x);
        Row8<T>::store(dst + b_col, y);
    }
}

}  // namespace

int launch_latent_append(const LatentAppendArgs& a) {
    AICOMP_REQUIRE(a.latent_dim <= MAX_LATENT && a.rope_dim <= MAX_ROPE, AICOMP_KV_EUNSUPPORTED,
                   "latent_kv_append: latent and rotated parts of %d and %d elements, at most %d and %d", a.latent_dim, a.rope_dim, MAX_LATENT,
                   MAX_ROPE);
    LatentAppendParams p;
    p.a = a;
    const int64_t rows = a.num_tokens < ((int64_t)1 << 32) ? a.num_tokens * ((a.q_in ? (int64_t)a.heads : 0) + 1) : INT64_MAX;
    const int64_t items = rows < ((int64_t)1 << 32) ? rows * (a.rope_dim / 16) : INT64_MAX;
    AICOMP_REQUIRE(items < UINT32_MAX - 256, AICOMP_KV_EINVAL, "latent_kv_append: %lld tokens of %d heads exceed one launch",
                   (long long)a.num_tokens, a.heads);
    const int64_t latent_wgs = (a.num_tokens + 3) / 4, wgs = latent_wgs + (items + 255) / 256;
    AICOMP_REQUIRE(wgs * 256 <= UINT32_MAX, AICOMP_KV_EINVAL,
                   "latent_kv_append: %lld tokens of %d heads exceed one launch", (long long)a.num_tokens, a.heads);
    p.latent_wgs = (uint32_t)latent_wgs;
    p.items = (uint32_t)items;
    const dim3 grid((unsigned)wgs), block(256);
    if (a.dtype == AICOMP_KV_BF16) hipLaunchKernelGGL(latent_append_kernel<bf16_t>, grid, block, 0, a.stream, p);
    else if (a.dtype == AICOMP_KV_F16) hipLaunchKernelGGL(latent_append_kernel<f16_t>, grid, block, 0, a.stream, p);
    else hipLaunchKernelGGL(latent_append_kernel<float>, grid, block, 0, a.stream, p);
    AICOMP_HIP_LAUNCH_CHECK();
    return AICOMP_KV_OK;
}

}  // namespace aicomp
