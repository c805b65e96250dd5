// Attention by a score rule (score.h) on the vector ALU: every type pair, head_dim 64 / 128 / 256, any group and block size,
// decode and chunks.  The path of what the matrix-core kernels do not take, and the merge of split decode rows.
//
// One workgroup (4 waves) per (query row, KV head, partition of the row's visible keys).  A K/V row is read by LPR consecutive
// lanes, 16 bytes each (8 of an fp8 row), so that a wave's load is 64 / LPR whole rows; each lane group runs an online softmax
// of its own over the tokens that it visits (reference and sum in float32, exponents in base 2), all heads of the group
// share a loaded chunk, and the groups' states are merged by shuffles, the waves' through LDS.
//
// Bound by the loads in flight for groups of one to four heads, by the vector ALU (2 D multiply-adds a score, and what a score takes
// itself in every lane of its group) above.  64 rows of 512 .. 4096 tokens, head_dim 256, bf16 under a cap: 16 / 8 heads 271 us, 4.5 TB/s
// (583 with one token in flight, two of four heads computed for nothing, sums through the LDS's lane moves and a maximum per
// token); 16 / 4 and 32 / 4 heads 256 and 560, where the bytes take 116; one row of 4096, 24.  Block sizes other than 16 (D 128, 32 / 8
// heads) 225, head_dim 64 117, where the tiles of blocks of 16 take 97 and 54.
// Chunks come here for their block size alone, a workgroup per row and KV head that reads the row's keys for itself: 512 and 2048
// tokens from none, D 128, a cap, blocks of 8 or 32: 115 and 1304 us, where blocks of 16 take 15 and 62; 64 behind 4000 271, and 27.
#include "score.h"

namespace aicomp {

namespace {

template <typename KV_T> struct RowChunk {
    static constexpr int N = Vec16<KV_T>::N;
    typedef uint4 Raw;
    __device__ __forceinline__ static void unpack(const Raw& r, float* f) { Vec16<KV_T>::unpack(r, f); }
};
template <> struct RowChunk<fp8_t> {
    static constexpr int N = 8;
    typedef uint2 Raw;
    __device__ __forceinline__ static void unpack(const Raw& r, float* f) {
        const uint32_t w[2] = {r.x, r.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
            auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
            f[4 * i] = lo[0]; f[4 * i + 1] = lo[1];
            f[4 * i + 2] = hi[0]; f[4 * i + 3] = hi[1];
        }
    }
};

struct GenericScoreParams {
    void* out;
    const void* query;
    const void* k_pool;
    const void* v_pool;
    const int32_t* block_table;
    int64_t block_table_stride;
    const int32_t* context_lens;
    const int32_t* cu_q_lens;
    int num_seqs;
    int hq, hkv, group, bs, max_blocks;
    int64_t num_blocks;
    const float* k_scale;
    const float* v_scale;
    ScoreRule rule;
    int partition_size, num_parts;
    float* ws_acc;
    float* ws_ml;
};

// sequence, position and visible keys of a query row; false: the row belongs to no sequence
__device__ __forceinline__ bool row_of(const int32_t* cu, const int32_t* ctx_lens, int num_seqs, int max_tokens, const ScoreRule& rule,
                                       int64_t row, int& seq, int& pos, int& lo, int& hi) {
    int n = 1, i = 0;
    if (cu == nullptr) {
        seq = (int)row;
    } else {
        int a = 0, b = num_seqs;             // largest s with cu[s] <= row
        while (b - a > 1) {
            const int mid = (a + b) >> 1;
            if (cu[mid] <= row) a = mid; else b = mid;
        }
        seq = a;
        n = cu[a + 1] - cu[a];
        i = (int)(row - cu[a]);
        if (i < 0 || i >= n) return false;
    }
    const int ctx = min(ctx_lens[seq], max_tokens);
    pos = ctx - n + i;
    lo = hi = 0;
    if (ctx >= n) visible_keys(rule, row, seq, pos, ctx, lo, hi);        // (a context shorter than its chunk: no keys)
    return true;
}

constexpr float NEG_BIG = -1.0e30f;

// Sum over LPR consecutive lanes, in each of them: within sixteen by the vector ALU's own lane moves.
template <int CTRL> __device__ __forceinline__ float add_moved(float s) {
    return s + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, s), CTRL, 0xf, 0xf, true));
}
template <int LPR> __device__ __forceinline__ float lanes_sum(float s) {
    if constexpr (LPR >= 2) s = add_moved<0xB1>(s);            // lanes 1 0 3 2
    if constexpr (LPR >= 4) s = add_moved<0x4E>(s);            // lanes 2 3 0 1
    if constexpr (LPR >= 8) s = add_moved<0x141>(s);           // half rows mirrored
    if constexpr (LPR >= 16) s = add_moved<0x140>(s);          // rows mirrored
    if constexpr (LPR >= 32) s += __shfl_xor(s, 16);
    if constexpr (LPR >= 64) s += __shfl_xor(s, 32);
    return s;
}

// U: tokens of a lane group whose loads are in flight together
template <typename KV_T, typename Q_T, int D, int GMAX, int U>
__global__ void __launch_bounds__(256)
score_generic_kernel(GenericScoreParams p) {
    constexpr int N = RowChunk<KV_T>::N;
    constexpr int LPR = D / N;            // lanes per K/V row
    constexpr int TPW = WAVE / LPR;       // rows per wave per load
    constexpr int NW = 4;
    static_assert(LPR >= 1 && LPR <= 64 && (LPR & (LPR - 1)) == 0, "row must split over 2^k lanes");

    const int64_t row = blockIdx.x;
    const int groups_per_kv = (p.group + GMAX - 1) / GMAX;
    const int kvh = blockIdx.y / groups_per_kv;
    const int g0 = (blockIdx.y % groups_per_kv) * GMAX;      // first head of the group handled here
    const int gn = min(GMAX, p.group - g0);
    const int part = blockIdx.z;

    int seq, pos, lo, hi;
    if (!row_of(p.cu_q_lens, p.context_lens, p.num_seqs, p.max_blocks * p.bs, p.rule, row, seq, pos, lo, hi)) return;
    const int64_t start64 = lo + (int64_t)part * p.partition_size;
    const int tid = threadIdx.x;
    const int head0 = kvh * p.group + g0;
    if (start64 >= hi) {
        if (part == 0) {                       // nothing visible: the row is zero
            Q_T* o = (Q_T*)p.out + (row * p.hq + head0) * D;
            for (int i = tid; i < gn * D; i += blockDim.x) store_elem<Q_T>(o + i, 0.f);
        }
        return;
    }
    const int start = (int)start64;
    const int end = part + 1 == p.num_parts ? hi : min(hi, start + p.partition_size);

    const int w = tid / WAVE, lane = tid % WAVE;
    const int sub = lane / LPR, lr = lane % LPR;
    const float ks = p.k_scale ? p.k_scale[kvh] : 1.f;
    const bool capped = p.rule.cap_log2 > 0.f;
    const float mul = (capped ? p.rule.cap_mul : p.rule.mul) * ks;

    float q[GMAX][N], slope[GMAX];
#pragma unroll
    for (int g = 0; g < GMAX; ++g) {
        slope[g] = g < gn && p.rule.slopes ? p.rule.slopes[head0 + g] * LOG2E : 0.f;
        const Q_T* qp = (const Q_T*)p.query + (row * p.hq + head0 + min(g, gn - 1)) * D + lr * N;
#pragma unroll
        for (int e = 0; e < N; ++e) q[g][e] = load_elem<Q_T>(qp + e);
    }

    float m[GMAX], l[GMAX], acc[GMAX][N];
#pragma unroll
    for (int g = 0; g < GMAX; ++g) {
        m[g] = NEG_BIG; l[g] = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[g][e] = 0.f;
    }

    const int32_t* table = p.block_table + (int64_t)seq * p.block_table_stride;
    typedef typename RowChunk<KV_T>::Raw Raw;
    for (int64_t tok0 = start; tok0 < end; tok0 += NW * TPW * U) {
        Raw kr[U], vr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = (int)min(tok0 + (w * U + u) * TPW + sub, (int64_t)end - 1);        // clamped: always loadable
            int64_t blk = table[at / p.bs];
            blk = blk < 0 ? 0 : (blk >= p.num_blocks ? p.num_blocks - 1 : blk);
            const int64_t base = ((blk * p.hkv + kvh) * p.bs + at % p.bs) * D + lr * N;
            kr[u] = *(const Raw*)((const KV_T*)p.k_pool + base);
            vr[u] = *(const Raw*)((const KV_T*)p.v_pool + base);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t tok = tok0 + (w * U + u) * TPW + sub;
            float k[N], v[N];
            RowChunk<KV_T>::unpack(kr[u], k);
            RowChunk<KV_T>::unpack(vr[u], v);
            const float dist = fabsf((float)(pos - tok));
#pragma unroll
            for (int g = 0; g < GMAX; ++g) {
                float s = 0.f;
#pragma unroll
                for (int e = 0; e < N; ++e) s = fmaf(q[g][e], k[e], s);
                s = lanes_sum<LPR>(s) * mul;
                if (capped) {
                    // (16-bit queries: the form of the matrix-core kernels, good to 2^-22 of the cap)
                    if constexpr (sizeof(Q_T) == 2)
                        s = fmaf(-2.f * p.rule.cap_log2, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(2.f * LOG2E * s)), p.rule.cap_log2);
                    else s = p.rule.cap_log2 * tanhf(s);
                }
                s = fmaf(-slope[g], dist, s);
                const bool up = tok < end && s > m[g] + 8.f;                 // the reference moves by more than 2^8 only
                if (__any(up)) {
                    const float m_new = up ? s : m[g], alpha = __builtin_amdgcn_exp2f(m[g] - m_new);
                    m[g] = m_new;
                    l[g] *= alpha;
#pragma unroll
                    for (int e = 0; e < N; ++e) acc[g][e] *= alpha;
                }
                if (tok < end) {
                    const float pr = __builtin_amdgcn_exp2f(s - m[g]);
                    l[g] += pr;
#pragma unroll
                    for (int e = 0; e < N; ++e) acc[g][e] = fmaf(pr, v[e], acc[g][e]);
                }
            }
        }
    }

    // merge the TPW lane groups of the wave
#pragma unroll
    for (int o = LPR; o < WAVE; o <<= 1) {
#pragma unroll
        for (int g = 0; g < GMAX; ++g) {
            const float mo = __shfl_xor(m[g], o);
            const float lo_ = __shfl_xor(l[g], o);
            const float mn = fmaxf(m[g], mo);
            const float a = exp2f(m[g] - mn), b = exp2f(mo - mn);
            l[g] = l[g] * a + lo_ * b;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float ao = __shfl_xor(acc[g][e], o);
                acc[g][e] = acc[g][e] * a + ao * b;
            }
            m[g] = mn;
        }
    }

    // merge the waves through LDS
    __shared__ float sm_m[NW][GMAX];
    __shared__ float sm_l[NW][GMAX];
    __shared__ float sm_acc[NW][GMAX][D];
    if (sub == 0) {
#pragma unroll
        for (int g = 0; g < GMAX; ++g) {
            if (lr == 0) { sm_m[w][g] = m[g]; sm_l[w][g] = l[g]; }
#pragma unroll
            for (int e = 0; e < N; ++e) sm_acc[w][g][lr * N + e] = acc[g][e];
        }
    }
    __syncthreads();

    const float vs = p.v_scale ? p.v_scale[kvh] : 1.f;
    for (int i = tid; i < gn * D; i += blockDim.x) {
        const int g = i / D, dd = i % D;
        float mx = sm_m[0][g];
#pragma unroll
        for (int ww = 1; ww < NW; ++ww) mx = fmaxf(mx, sm_m[ww][g]);
        float num = 0.f, den = 0.f;
#pragma unroll
        for (int ww = 0; ww < NW; ++ww) {
            const float f = exp2f(sm_m[ww][g] - mx);
            num = fmaf(f, sm_acc[ww][g][dd], num);
            den = fmaf(f, sm_l[ww][g], den);
        }
        const int head = head0 + g;
        if (p.num_parts == 1) {
            store_elem<Q_T>((Q_T*)p.out + (row * p.hq + head) * D + dd, den == 0.f ? 0.f : vs * num / den);
        } else {
            const int64_t slot = (row * p.hq + head) * p.num_parts + part;
            p.ws_acc[slot * D + dd] = num;
            if (dd == 0) { p.ws_ml[slot * 2] = mx; p.ws_ml[slot * 2 + 1] = den; }
        }
    }
}

// Split rows: out = sum_p 2^(m_p - M) acc_p / sum_p 2^(m_p - M) l_p over the partitions that hold visible keys.  One wave per
// (row, head); NV dims per lane.  The weights are computed by one lane each and handed round by shuffles, 64 partitions at a time.
template <typename Q_T, int NV>
__global__ void __launch_bounds__(256)
score_merge_kernel(Q_T* __restrict__ out, const float* __restrict__ ws_acc, const float* __restrict__ ws_ml,
                   const int32_t* __restrict__ context_lens, ScoreRule rule, int64_t pairs, int hq, int group, int max_tokens,
                   int partition_size, int num_parts, int part_align, const float* __restrict__ v_scale) {
    constexpr int D = 64 * NV;
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);         // (row, head)
    if (at >= pairs) return;
    const int64_t row = at / hq;
    const int head = (int)(at - row * hq);
    int seq, pos, lo, hi;
    row_of(nullptr, context_lens, 0, max_tokens, rule, row, seq, pos, lo, hi);
    if (lo >= hi) return;                                                    // the main kernel wrote the zero row
    lo -= lo % part_align;
    const int np = min(num_parts, (int)((hi - lo + (int64_t)partition_size - 1) / partition_size));
    const float* ml = ws_ml + at * num_parts * 2;
    const float* acc = ws_acc + at * num_parts * D + lane;
    float mx = NEG_BIG;
    for (int i = lane; i < np; i += 64) mx = fmaxf(mx, ml[2 * i]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    float den = 0.f, num[NV] = {};
    for (int i0 = 0; i0 < np; i0 += 64) {
        const int i = i0 + lane;
        const float wgt = i < np ? exp2f(ml[2 * i] - mx) : 0.f;
        if (i < np) den = fmaf(wgt, ml[2 * i + 1], den);
        const int n = min(64, np - i0);
        for (int u0 = 0; u0 < n; u0 += 4) {
            float a[4][NV];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int e = 0; e < NV; ++e) a[u][e] = acc[(int64_t)(i0 + min(u0 + u, n - 1)) * D + 64 * e];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float f = __shfl(wgt, min(u0 + u, 63));
#pragma unroll
                for (int e = 0; e < NV; ++e) num[e] = u0 + u < n ? fmaf(f, a[u][e], num[e]) : num[e];
            }
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) den += __shfl_xor(den, o);
    const float inv = den == 0.f ? 0.f : (v_scale ? v_scale[head / group] : 1.f) / den;
#pragma unroll
    for (int e = 0; e < NV; ++e) store_elem<Q_T>(out + at * D + lane + 64 * e, num[e] * inv);
}

template <typename KV_T, typename Q_T, int D>
void launch_d(const ScoreArgs& a, const GenericScoreParams& p) {
    const int group = a.hq / a.hkv;
    const dim3 grid((unsigned)a.rows, (unsigned)(a.hkv * ((group + 7) / 8)), (unsigned)a.num_parts);
    // us, 1, 2, 4 and 8 tokens in flight, 64 rows of 512 .. 4096, head_dim 256, 8 KV heads: groups of two 400, 311, 293, 307 (fp8 355,
    // 251, 253, 214); groups of four, 4 KV heads, 255, 308, 288
    constexpr int U = sizeof(KV_T) == 1 ? 8 : 4;
    if (group <= 2) hipLaunchKernelGGL((score_generic_kernel<KV_T, Q_T, D, 2, U>), grid, dim3(256), 0, a.stream, p);
    else if (group <= 4) hipLaunchKernelGGL((score_generic_kernel<KV_T, Q_T, D, 4, 1>), grid, dim3(256), 0, a.stream, p);
    else hipLaunchKernelGGL((score_generic_kernel<KV_T, Q_T, D, 8, 1>), grid, dim3(256), 0, a.stream, p);
}

template <typename KV_T, typename Q_T>
void launch_t(const ScoreArgs& a, const GenericScoreParams& p) {
    if (a.d == 64) launch_d<KV_T, Q_T, 64>(a, p);
    else if (a.d == 128) launch_d<KV_T, Q_T, 128>(a, p);
    else launch_d<KV_T, Q_T, 256>(a, p);
}

template <typename Q_T>
void launch_merge_t(const ScoreArgs& a) {
    const int64_t pairs = a.rows * a.hq;
    const dim3 grid((unsigned)((pairs + 3) / 4));
#define AICOMP_MERGE(NV)                                                                                                       \
    hipLaunchKernelGGL((score_merge_kernel<Q_T, NV>), grid, dim3(256), 0, a.stream, (Q_T*)a.out, a.ws_acc, a.ws_ml,            \
                       a.context_lens, rule_of(a), pairs, a.hq, a.hq / a.hkv, a.max_blocks * a.bs, a.partition_size,           \
                       a.num_parts, a.part_align, a.v_scale)
    if (a.d == 64) AICOMP_MERGE(1);
    else if (a.d == 128) AICOMP_MERGE(2);
    else AICOMP_MERGE(4);
#undef AICOMP_MERGE
}

}  // namespace

int launch_score_merge(const ScoreArgs& a) {
    if (a.q_dtype == AICOMP_KV_F32) launch_merge_t<float>(a);
    else if (a.q_dtype == AICOMP_KV_F16) launch_merge_t<f16_t>(a);
    else launch_merge_t<bf16_t>(a);
    AICOMP_HIP_LAUNCH_CHECK();
    return AICOMP_KV_OK;
}

int launch_score_generic(const ScoreArgs& a) {
    // (a launch dimension holds less than 2^32 lanes)
    AICOMP_REQUIRE(a.rows <= UINT32_MAX / 256 && a.num_parts <= 65535 && (int64_t)a.hkv * ((a.hq / a.hkv + 7) / 8) <= 65535,
                   AICOMP_KV_EINVAL, "paged_score_attn: grid too large");
    GenericScoreParams p;
    p.out = a.out; p.query = a.query; p.k_pool = a.k_pool; p.v_pool = a.v_pool;
    p.block_table = a.block_table; p.block_table_stride = a.block_table_stride;
    p.context_lens = a.context_lens; p.cu_q_lens = a.cu_q_lens; p.num_seqs = a.num_seqs;
    p.hq = a.hq; p.hkv = a.hkv; p.group = a.hq / a.hkv; p.bs = a.bs; p.max_blocks = a.max_blocks; p.num_blocks = a.num_blocks;
    p.k_scale = a.k_scale; p.v_scale = a.v_scale;
    p.rule = rule_of(a);
    p.partition_size = a.partition_size; p.num_parts = a.num_parts;
    p.ws_acc = a.ws_acc; p.ws_ml = a.ws_ml;
    const int q = a.q_dtype, kv = a.kv_dtype;
    if (q == AICOMP_KV_F32) launch_t<float, float>(a, p);
    else if (q == AICOMP_KV_BF16 && kv == AICOMP_KV_BF16) launch_t<bf16_t, bf16_t>(a, p);
    else if (q == AICOMP_KV_BF16) launch_t<fp8_t, bf16_t>(a, p);
    else if (kv == AICOMP_KV_F16) launch_t<f16_t, f16_t>(a, p);
    else launch_t<fp8_t, f16_t>(a, p);
    AICOMP_HIP_LAUNCH_CHECK();
    return a.num_parts > 1 ? launch_score_merge(a) : AICOMP_KV_OK;
}

}  // namespace aicomp
