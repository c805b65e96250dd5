// Attention of query rows over cached or expanded latent rows on the vector ALU: every type, head and row size.  The path of what
// the matrix-core kernels do not take: float32, other sizes than theirs, blocks of fewer than 16 tokens or of no power of two.
//
// One workgroup per (query row, head).  Tiles of 256 keys: a thread has one key's score (a row of the pool is read by one thread, 16
// bytes at a time, so that the lines are taken whole from the L1), the tile's weights go through LDS, and the output's
// columns are divided among the threads in quads, the keys of a tile among as many threads as there are quads to spare.  An online
// softmax in float32, exponents in base 2.  Keys that the row does not see are neither multiplied nor read.
//
// Bound by the reads of every (row, head) for itself, out of the caches: 16 rows of 16 heads over 1024 latent rows of float32 387 us, of
// bfloat16 in blocks of 48 tokens 310 (in blocks of 16, on the matrix cores, 21).
#include "row_attn.h"

#include <algorithm>

namespace aicomp {

namespace {

// four elements as floats
template <typename T> __device__ __forceinline__ float4 load_quad(const T* p);
template <> __device__ __forceinline__ float4 load_quad<float>(const float* p) { return *(const float4*)p; }
template <> __device__ __forceinline__ float4 load_quad<bf16_t>(const bf16_t* p) {
    const uint2 r = *(const uint2*)p;
    return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
                       __uint_as_float(r.y & 0xffff0000u));
}
template <> __device__ __forceinline__ float4 load_quad<f16_t>(const f16_t* p) {
    const uint2 r = *(const uint2*)p;
    return make_float4(f16_to_f32((uint16_t)r.x), f16_to_f32((uint16_t)(r.x >> 16)), f16_to_f32((uint16_t)r.y),
                       f16_to_f32((uint16_t)(r.y >> 16)));
}
template <> __device__ __forceinline__ float4 load_quad<fp8_t>(const fp8_t* p) {
    const uint32_t r = *(const uint32_t*)p;
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)r, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)r, true);
    return make_float4(lo[0], lo[1], hi[0], hi[1]);
}

// sum of n products (n a multiple of 16)
template <typename KV_T> __device__ __forceinline__ float dot(const float* q, const KV_T* k, int n, float s) {
    for (int d = 0; d < n; d += Vec16<KV_T>::N) {
        float f[Vec16<KV_T>::N];
        Vec16<KV_T>::unpack(*(const uint4*)(k + d), f);
#pragma unroll
        for (int e = 0; e < Vec16<KV_T>::N; ++e) s = fmaf(q[d + e], f[e], s);
    }
    return s;
}

// the sequence s with cu[s] <= t < cu[s + 1], -1 if there is none
__device__ __forceinline__ int sequence_of(const int32_t* cu, int num_seqs, int64_t t) {
    if (t < cu[0] || t >= cu[num_seqs]) return -1;
    int lo = 0, hi = num_seqs;                                  // cu[lo] <= t < cu[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (cu[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

template <typename KV_T> struct PagedRows {
    RowAttnArgs a;
    int seq, prior, i, ctx, kvh;
    int64_t t;
    __device__ __forceinline__ bool open(int64_t row, int head) {        // false: no row of any sequence
        t = row;
        seq = a.cu_q_lens ? sequence_of(a.cu_q_lens, a.num_seqs, row) : (int)row;
        if (seq < 0) return false;
        const int begin = a.cu_q_lens ? a.cu_q_lens[seq] : (int)row, n = a.cu_q_lens ? a.cu_q_lens[seq + 1] - begin : 1;
        ctx = (int)min((int64_t)a.context_lens[seq], (int64_t)a.max_blocks * a.bs);
        prior = ctx - n;
        i = (int)(row - begin);
        kvh = head / (a.hq / a.hkv);
        return true;
    }
    __device__ __forceinline__ int keys() const { return prior < 0 ? 0 : a.masks ? ctx : prior + i + 1; }
    __device__ __forceinline__ bool sees(int j) const {
        if (a.masks == nullptr || j < prior) return true;
        const int b = j - prior;
        return b < 64 * a.mask_words && ((a.masks[t * a.mask_words + (b >> 6)] >> (b & 63)) & 1);
    }
    __device__ __forceinline__ int64_t row_of(int j) const {
        const int64_t blk = max((int64_t)0, min((int64_t)a.block_table[seq * a.block_table_stride + j / a.bs], a.num_blocks - 1));
        return (blk * a.hkv + kvh) * a.bs + j % a.bs;
    }
    __device__ __forceinline__ float score(const float* q, int j) const {
        return dot((const float*)q, (const KV_T*)a.k_pool + row_of(j) * a.dk, a.dk, 0.f);
    }
    __device__ __forceinline__ const KV_T* value(int j) const { return (const KV_T*)a.v_pool + row_of(j) * a.v_row; }
    __device__ __forceinline__ int dk() const { return a.dk; }
    __device__ __forceinline__ int heads() const { return a.hq; }
    __device__ __forceinline__ float k_mul() const { return a.k_scale ? a.k_scale[kvh] : 1.f; }
    __device__ __forceinline__ float v_mul() const { return a.v_scale ? a.v_scale[kvh] : 1.f; }
};

template <typename KV_T> struct DenseRows {
    PromptAttnArgs a;
    int head, visible;
    int64_t k0;
    __device__ __forceinline__ bool open(int64_t row, int h) {
        const int seq = sequence_of(a.cu_q_lens, a.num_seqs, row);
        if (seq < 0) return false;
        const int begin = a.cu_q_lens[seq], n = a.cu_q_lens[seq + 1] - begin;
        k0 = max(0, a.cu_k_lens[seq]);
        const int ctx = (int)min((int64_t)a.cu_k_lens[seq + 1], a.keys) - (int)k0;
        head = h;
        visible = ctx < n ? 0 : ctx - n + (int)(row - begin) + 1;
        return true;
    }
    __device__ __forceinline__ int keys() const { return visible; }
    __device__ __forceinline__ bool sees(int) const { return true; }
    __device__ __forceinline__ float score(const float* q, int j) const {
        const float s = dot(q, (const KV_T*)a.key + (k0 + j) * a.key_ts + head * a.key_hs, a.nope, 0.f);
        return dot(q + a.nope, (const KV_T*)a.rope_key + (k0 + j) * a.rope_ts, a.rope, s);
    }
    __device__ __forceinline__ const KV_T* value(int j) const { return (const KV_T*)a.value + (k0 + j) * a.value_ts + head * a.value_hs; }
    __device__ __forceinline__ int dk() const { return a.nope + a.rope; }
    __device__ __forceinline__ int heads() const { return a.heads; }
    __device__ __forceinline__ float k_mul() const { return 1.f; }
    __device__ __forceinline__ float v_mul() const { return 1.f; }
};

template <typename Q_T, typename KV_T, typename ROWS>
__global__ void __launch_bounds__(256)
rows_generic_kernel(ROWS r, int64_t row0) {
    __shared__ __attribute__((aligned(16))) float q[MAX_KEY];
    __shared__ float weight[256];
    __shared__ float4 sums[256];
    __shared__ float red[4];
    const int head = blockIdx.x, tid = threadIdx.x, dv = r.a.dv;
    const int64_t row = row0 + blockIdx.y;
    if (!r.open(row, head)) return;
    Q_T* out = (Q_T*)r.a.out + (row * r.heads() + head) * dv;
    const int dk = r.dk(), keys = r.keys();
    for (int d = tid; d < dk; d += 256) q[d] = load_elem<Q_T>((const Q_T*)r.a.query + (row * r.heads() + head) * dk + d);
    __syncthreads();
    const float mul = r.a.scale * LOG2E * r.k_mul();
    // this thread's quad of columns, and which of the keys it takes (`lanes` threads share a quad)
    const int quads = dv / 4, lanes = 256 / quads, quad = tid % quads, lane = tid / quads;
    const bool busy = lane < lanes;
    float m = -INFINITY, l = 0.f;                              // m: alike in all threads
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int base = 0; base < keys; base += 256) {
        const int j = base + tid;
        const bool live = j < keys && r.sees(j);
        const float s = live ? r.score(q, j) * mul : 0.f;
        float mx = live ? s : -INFINITY;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        if ((tid & 63) == 0) red[tid >> 6] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
        // (nothing seen yet: any finite reference will do)
        const float ref = mx == -INFINITY ? 0.f : mx, alpha = m == -INFINITY ? 0.f : exp2f(m - ref);
        const float w = live ? exp2f(s - ref) : 0.f;
        weight[tid] = live ? w : -1.f;                         // (weights are not negative: the mark of a key that is not seen)
        l = l * alpha + w;
        acc.x *= alpha; acc.y *= alpha; acc.z *= alpha; acc.w *= alpha;
        m = mx;
        __syncthreads();
        const int here = min(256, keys - base);
        if (busy)
            for (int k = lane; k < here; k += lanes) {
                const float w_k = weight[k];
                if (w_k < 0.f) continue;
                const float4 v = load_quad<KV_T>(r.value(base + k) + 4 * quad);
                acc.x = fmaf(w_k, v.x, acc.x); acc.y = fmaf(w_k, v.y, acc.y);
                acc.z = fmaf(w_k, v.z, acc.z); acc.w = fmaf(w_k, v.w, acc.w);
            }
        __syncthreads();
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o);
    if ((tid & 63) == 0) red[tid >> 6] = l;
    sums[tid] = acc;
    __syncthreads();
    if (lane != 0) return;
    l = red[0] + red[1] + red[2] + red[3];
    for (int k = 1; k < lanes; ++k) {
        const float4 o = sums[tid + k * quads];
        acc.x += o.x; acc.y += o.y; acc.z += o.z; acc.w += o.w;
    }
    const float inv = r.v_mul() / l;
    const bool none = l == 0.f;
    store_elem<Q_T>(out + 4 * quad, none ? 0.f : acc.x * inv);
    store_elem<Q_T>(out + 4 * quad + 1, none ? 0.f : acc.y * inv);
    store_elem<Q_T>(out + 4 * quad + 2, none ? 0.f : acc.z * inv);
    store_elem<Q_T>(out + 4 * quad + 3, none ? 0.f : acc.w * inv);
}

// (a grid's second dimension holds 65535 rows, a launch less than 2^32 threads)
template <typename Q_T, typename KV_T, typename ROWS>
void launch_rows(const ROWS& r, int heads, int64_t rows, hipStream_t stream) {
    const int64_t per = std::max<int64_t>(1, std::min<int64_t>(65535, ((int64_t)1 << 24) / heads - 1));
    for (int64_t row0 = 0; row0 < rows; row0 += per)
        hipLaunchKernelGGL((rows_generic_kernel<Q_T, KV_T, ROWS>), dim3((unsigned)heads, (unsigned)std::min(per, rows - row0)), dim3(256), 0,
                           stream, r, row0);
}

template <typename Q_T, typename KV_T> void launch_paged(const RowAttnArgs& a) {
    PagedRows<KV_T> r;
    r.a = a;
    launch_rows<Q_T, KV_T>(r, a.hq, a.rows, a.stream);
}

template <typename T> void launch_dense(const PromptAttnArgs& a) {
    DenseRows<T> r;
    r.a = a;
    launch_rows<T, T>(r, a.heads, a.rows, a.stream);
}

}  // namespace

int launch_rows_generic(const RowAttnArgs& a) {
    const bool fp8 = a.kv_dtype == AICOMP_KV_FP8_E4M3;
    if (a.q_dtype == AICOMP_KV_F32) launch_paged<float, float>(a);
    else if (a.q_dtype == AICOMP_KV_BF16) { if (fp8) launch_paged<bf16_t, fp8_t>(a); else launch_paged<bf16_t, bf16_t>(a); }
    else { if (fp8) launch_paged<f16_t, fp8_t>(a); else launch_paged<f16_t, f16_t>(a); }
    AICOMP_HIP_LAUNCH_CHECK();
    return AICOMP_KV_OK;
}

int launch_prompt_generic(const PromptAttnArgs& a) {
    if (a.dtype == AICOMP_KV_F32) launch_dense<float>(a);
    else if (a.dtype == AICOMP_KV_BF16) launch_dense<bf16_t>(a);
    else launch_dense<f16_t>(a);
    AICOMP_HIP_LAUNCH_CHECK();
    return AICOMP_KV_OK;
}

}  // namespace aicomp
