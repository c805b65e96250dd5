// What the matrix-core kernels of chunks by a score rule share (score_prefill.hip, score_prefill_f32.hip).
#pragma once

#include "score.h"

#include <atomic>
#include <type_traits>

namespace aicomp {

namespace {

constexpr int BS = 16;
constexpr float NEG_BIG = -1.0e30f;
constexpr int PART_KEYS = 256;         // least keys of a part where they are divided

struct ScorePrefillParams {
    void* out;
    const void* query;
    const void* k_pool;
    const void* v_pool;
    const int32_t* block_table;
    int64_t block_table_stride;
    const int32_t* context_lens;
    const int32_t* cu_q_lens;
    int hq, hkv, group, gpack, max_blocks;
    int num_blocks;
    int num_cus;
    const float* k_scale;
    const float* v_scale;
    ScoreRule rule;
    // divided keys (parts > 1): sums, reference and weight of part i of (row, head) at [(i rows + row) hq + head]
    int hgroups, parts;
    int64_t rows;
    float* ws_acc;
    float2* ws_ml;
};

// (but what a kernel's variants differ in)
inline ScorePrefillParams chunk_params(const ScoreArgs& a) {
    ScorePrefillParams p;
    p.out = a.out; p.query = a.query; p.k_pool = a.k_pool; p.v_pool = a.v_pool;
    p.block_table = a.block_table; p.block_table_stride = a.block_table_stride;
    p.context_lens = a.context_lens; p.cu_q_lens = a.cu_q_lens;
    p.hq = a.hq; p.hkv = a.hkv; p.group = a.hq / a.hkv; p.max_blocks = a.max_blocks; p.num_blocks = (int)a.num_blocks;
    p.gpack = 16 % p.group == 0 ? p.group : 1;
    p.k_scale = a.k_scale; p.v_scale = a.v_scale;
    p.rule = rule_of(a);
    static std::atomic<int> cached_cus{-1};                    // (of the first device used: every GPU of a node is the same part)
    p.num_cus = cached_cus.load(std::memory_order_relaxed);
    if (p.num_cus < 0) {
        int dev = 0, cus = 0;
        if (hipGetDevice(&dev) != hipSuccess ||
            hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 0)
            cus = 0;
        p.num_cus = cus;
        cached_cus.store(cus, std::memory_order_relaxed);
    }
    p.hgroups = a.hq / p.gpack;
    p.parts = a.ws_acc != nullptr ? score_chunk_plan(a).parts : 1;
    p.rows = a.rows; p.ws_acc = a.ws_acc; p.ws_ml = (float2*)a.ws_ml;
    return p;
}

#define GLOBAL_PTR(p) ((const __attribute__((address_space(1))) void*)(p))
#define LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

// Sequence and query tile of a workgroup.  Where two of a grid share a CU from the start (prefill_tile_of_slice), they are an expensive
// and a cheap tile of one sequence there; here the second is of the sequence at the other end of the batch, whose contexts or windows
// may be of another length (4 x 512 behind 0 .. 2048, a window of 1024: 54.6 -> 52.3 us).
__device__ __forceinline__ void place_of(const ScorePrefillParams& p, int& seq, int& qtile) {
    const int per = gridDim.x * gridDim.y;
    qtile = prefill_tile_of_slice(blockIdx.z, gridDim.z, p.num_cus, per);
    seq = blockIdx.y;
    if (p.num_cus > 0 && p.num_cus % per == 0 && gridDim.z * per <= 2 * p.num_cus && (int)blockIdx.z >= p.num_cus / per)
        seq = gridDim.y - 1 - seq;
}

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x = min(x, __shfl_xor(x, o));
    return __builtin_amdgcn_readfirstlane(x);
}

// One row key by key, by a whole wave: what the matrix cores cannot give where a key that the row does not see, but a neighbour
// does, has a value that is not finite (a weight of 0 times it is not 0).
template <typename E, bool FP8, int DH, bool PARTS>
__device__ void score_row(const ScorePrefillParams& p, int seq, int64_t q_row, int head, int kvh, int pos, int lo, int hi, int part,
                          int lane) {
    constexpr int NV = DH / 64;
    typedef typename E::elem Elem;
    const Elem* q = (const Elem*)p.query + (q_row * p.hq + head) * DH;
    const bool capped = p.rule.cap_log2 > 0.f;
    const float mul = (capped ? p.rule.cap_mul : p.rule.mul) * (FP8 ? p.k_scale[kvh] : 1.f);
    const float slope = p.rule.slopes != nullptr ? p.rule.slopes[head] * LOG2E : 0.f;
    auto key_row = [&](int j) {
        const int64_t blk = max(0, min(p.block_table[(int64_t)seq * p.block_table_stride + j / BS], p.num_blocks - 1));
        return ((blk * p.hkv + kvh) * BS + j % BS) * DH;
    };
    float m = NEG_BIG, l = 0.f, acc[NV] = {};
    for (int base = lo; base < hi; base += 64) {
        const int j = min(base + lane, hi - 1);
        const int64_t at = key_row(j);
        float s = 0.f;
        for (int d = 0; d < DH; ++d) {
            float k;
            if constexpr (FP8) k = fp8_to_f32(((const uint8_t*)p.k_pool)[at + d]);
            else k = load_elem<Elem>((const Elem*)p.k_pool + at + d);
            s = fmaf(load_elem<Elem>(q + d), k, s);
        }
        s *= mul;
        if (capped) s = p.rule.cap_log2 * tanhf(s);
        s = fmaf(-slope, fabsf((float)(pos - j)), s);
        const bool live = base + lane < hi;
        float mx = live ? s : NEG_BIG;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        const float m_new = fmaxf(m, mx), alpha = exp2f(m - m_new), pr = live ? exp2f(s - m_new) : 0.f;
        m = m_new;
        l = l * alpha + pr;
#pragma unroll
        for (int e = 0; e < NV; ++e) acc[e] *= alpha;
        for (int k = 0; k < min(64, hi - base); ++k) {
            const float w = __shfl(pr, k);
            const int64_t v_at = key_row(base + k) + lane;
#pragma unroll
            for (int e = 0; e < NV; ++e) {
                float v;
                if constexpr (FP8) v = fp8_to_f32(((const uint8_t*)p.v_pool)[v_at + 64 * e]);
                else v = load_elem<Elem>((const Elem*)p.v_pool + v_at + 64 * e);
                acc[e] = fmaf(w, v, acc[e]);
            }
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o);
    if (PARTS && p.parts > 1) {
        const int64_t slot = (part * p.rows + q_row) * p.hq + head;
#pragma unroll
        for (int e = 0; e < NV; ++e) p.ws_acc[slot * DH + lane + 64 * e] = acc[e];
        if (lane == 0) p.ws_ml[slot] = make_float2(m, l);
        return;
    }
    const float inv = (FP8 ? p.v_scale[kvh] : 1.f) / l;
    Elem* o = (Elem*)p.out + (q_row * p.hq + head) * DH + lane;
#pragma unroll
    for (int e = 0; e < NV; ++e) store_elem<Elem>(o + 64 * e, l == 0.f ? 0.f : acc[e] * inv);
}

// The parts of divided rows joined: out = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i over the parts in which the row sees keys.
// DH / 4 lanes per (row, head), 16-byte loads; every part's loads are in flight together.
template <typename E, int DH>
__global__ void __launch_bounds__(256) score_prefill_join_kernel(ScorePrefillParams p) {
    constexpr int LPR = DH / 4;
    const int seq = blockIdx.y, begin = p.cu_q_lens[seq], n = p.cu_q_lens[seq + 1] - begin;
    const int64_t at = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;      // (row of the chunk, head)
    if (at >= (int64_t)n * p.hq) return;
    const int64_t first = begin * (int64_t)p.hq + at, step = p.rows * p.hq;
    const int e = 4 * (threadIdx.x % LPR);
    float mx = NEG_BIG, den = 0.f;
    for (int i = 0; i < p.parts; ++i) {
        const float2 ml = p.ws_ml[first + i * step];
        if (ml.y != 0.f) mx = fmaxf(mx, ml.x);
    }
    f32x4_t num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < p.parts; ++i) {
        const float2 ml = p.ws_ml[first + i * step];
        const f32x4_t a = *(const f32x4_t*)(p.ws_acc + (first + i * step) * DH + e);
        if (ml.y != 0.f) {                                     // (a part without keys wrote no sums)
            const float w = exp2f(ml.x - mx);
            den = fmaf(w, ml.y, den);
#pragma unroll
            for (int k = 0; k < 4; ++k) num[k] = fmaf(w, a[k], num[k]);
        }
    }
    const float inv = (p.v_scale != nullptr ? p.v_scale[(int)(at % p.hq) / p.group] : 1.f) / den;
    if (den == 0.f) num = f32x4_t{0.f, 0.f, 0.f, 0.f};
    else num *= inv;
    if constexpr (sizeof(typename E::raw) == 4) *(f32x4_t*)((float*)p.out + first * DH + e) = num;
    else *(uint2*)((uint16_t*)p.out + first * DH + e) = make_uint2(E::pack(num[0], num[1]), E::pack(num[2], num[3]));
}

template <typename E>
void launch_join(const ScorePrefillParams& p, const ScoreArgs& a) {
    const dim3 grid((unsigned)(((int64_t)a.max_q_len * a.hq + 1024 / a.d - 1) / (1024 / a.d)), (unsigned)a.num_seqs);
    if (a.d == 64) hipLaunchKernelGGL((score_prefill_join_kernel<E, 64>), grid, dim3(256), 0, a.stream, p);
    else if (a.d == 128) hipLaunchKernelGGL((score_prefill_join_kernel<E, 128>), grid, dim3(256), 0, a.stream, p);
    else hipLaunchKernelGGL((score_prefill_join_kernel<E, 256>), grid, dim3(256), 0, a.stream, p);
}

}  // namespace

int launch_score_prefill_f32(const ScoreArgs& a);

}  // namespace aicomp
