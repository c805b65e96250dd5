// The line of work of the matrix-core kernels of row_attn.h (row_attn_mfma.hip, row_attn_shared.hip): which piece of it a workgroup has,
// what a row sees of a tile, and how the pieces of an item are joined.
//
// All (sequence, KV head, row tile, key tile) in this order are one line, of which every workgroup has a piece of equal length, whatever
// the sequences' lengths are.  An item (sequence, KV head, row tile) that one workgroup has whole is finished by it; of others each
// leaves (m, l, O) of its rows in the workspace: in its slot 0 where it does not have the item's first key tile, else in its slot 1.
#pragma once

#include "row_attn.h"

namespace aicomp {

struct RowParams {
    void* out;
    const void* query;
    const void* k_pool;
    const void* v_pool;
    const int32_t* block_table;
    int64_t block_table_stride;
    const int32_t* context_lens;
    const int32_t* cu_q_lens;
    const int64_t* masks;
    int mask_words;
    int num_seqs;
    int rows, max_q_len;
    int hq, hkv, group, max_blocks, num_blocks;
    float mul;                         // scale * log2(e)
    const float* k_scale;
    const float* v_scale;
    int workers;                       // workgroups
    int least;                         // key tiles that a workgroup has at least
    int row_tiles;                     // of the longest sequence (the join's grid)
    float* ws_acc;                     // [2 workers][rows of a tile][DV]
    float2* ws_ml;                     // [2 workers][rows of a tile]
};

// d: head_dim; R: groups of 16 rows to a wave; items: of the join's grid
void launch_row_attn_shared(const RowParams& p, bool f16, bool fp8, int d, int R, int64_t items, hipStream_t stream);

namespace {

constexpr int BS = 16;                 // tokens per block
constexpr float NEG_BIG = -1.0e30f;
constexpr float SLACK = 8.f;           // a weight is at most 2^8: exact in both formats' range

#define GLOBAL_PTR(p) ((const __attribute__((address_space(1))) void*)(p))
#define LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

// A sequence as the line of work sees it.
struct Seq {
    int begin, n, ctx, prior;          // ctx: 0 where its tokens are more than its context
    int row_tiles, key_tiles;
    __device__ __forceinline__ int64_t items(const RowParams& p) const { return (int64_t)p.hkv * row_tiles; }
};

// ROWS, KT: rows and keys of a tile
template <int ROWS, int KT> __device__ __forceinline__ Seq load_seq(const RowParams& p, int s) {
    Seq q;
    q.begin = p.cu_q_lens ? max(0, p.cu_q_lens[s]) : s;
    q.n = p.cu_q_lens ? min(min(p.cu_q_lens[s + 1], p.rows) - q.begin, p.max_q_len) : 1;
    q.n = max(0, q.n);
    q.ctx = min(p.context_lens[s], p.max_blocks * BS);
    q.prior = q.ctx - q.n;
    if (q.prior < 0) q.ctx = 0;
    q.row_tiles = (q.n * p.group + ROWS - 1) / ROWS;
    q.key_tiles = max(1, (q.ctx + KT - 1) / KT);
    return q;
}

// The line's length, over all threads of the workgroup; `mine`: the part of it before this thread's sequences, first .. last - 1.
template <int ROWS, int KT>
__device__ __forceinline__ int64_t line_of(const RowParams& p, int64_t* sums, int& first, int& last, int64_t& mine) {
    const int per = (p.num_seqs + 255) / 256, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    first = min((int)threadIdx.x * per, p.num_seqs);
    last = min(first + per, p.num_seqs);
    int64_t own = 0;
    for (int s = first; s < last; ++s) {
        const Seq q = load_seq<ROWS, KT>(p, s);
        own += q.items(p) * q.key_tiles;
    }
    int64_t up = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t x = __shfl_up((long long)up, o);
        if (lane >= o) up += x;
    }
    if (lane == 63) sums[w] = up;
    __syncthreads();
    mine = up - own;
    for (int i = 0; i < w; ++i) mine += sums[i];
    return sums[0] + sums[1] + sums[2] + sums[3];
}

__device__ __forceinline__ int64_t piece_of(const RowParams& p, int64_t line) {
    return max((int64_t)p.least, (line + p.workers - 1) / p.workers);
}

// Which of the 32 keys from `start` on a row sees.  Causal: those below `limit`; else by its mask words from key `prior` on.
__device__ __forceinline__ uint32_t window_of(const int64_t* words, int num_words, int start, int prior, int ctx, int limit) {
    auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
    if (words == nullptr) return below(limit - start);
    const int o = start - prior;                                   // bit of the first key
    auto bits = [&](int from) -> uint32_t {                        // from >= 0
        const int k = from >> 6, b = from & 63;
        const uint64_t lo = k < num_words ? (uint64_t)words[k] : 0, hi = b > 32 && k + 1 < num_words ? (uint64_t)words[k + 1] : 0;
        return (uint32_t)(lo >> b | (b > 32 ? hi << (64 - b) : 0));
    };
    const uint32_t w = o >= 0 ? bits(o) : o <= -32 ? ~0u : bits(0) << -o | below(-o);
    return w & below(ctx - start);
}

// Items that several workgroups had: out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i.  1024 / DV rows of an item to a workgroup.
template <typename E, int DV, int ROWS, int KT>
__global__ void __launch_bounds__(256)
row_join_kernel(RowParams p) {
    constexpr int PER = 1024 / DV, LPR = DV / 4;
    __shared__ int64_t sums[4];
    __shared__ int64_t before_seq;
    const int sub = blockIdx.x % (ROWS / PER), item_at = blockIdx.x / (ROWS / PER);
    const int rtile = item_at % p.row_tiles, kvh = item_at / p.row_tiles % p.hkv, seq = item_at / p.row_tiles / p.hkv;
    const Seq q = load_seq<ROWS, KT>(p, seq);
    const int nrows = q.n * p.group;
    if (rtile * ROWS + sub * PER >= nrows) return;                 // (the whole workgroup)
    int first, last;
    int64_t mine;
    const int64_t line = line_of<ROWS, KT>(p, sums, first, last, mine), piece = piece_of(p, line);
    for (int s = first; s < last; ++s) {
        if (s == seq) before_seq = mine;
        const Seq x = load_seq<ROWS, KT>(p, s);
        mine += x.items(p) * x.key_tiles;
    }
    __syncthreads();
    const int64_t begin = before_seq + ((int64_t)kvh * q.row_tiles + rtile) * q.key_tiles;
    const int a = (int)(begin / piece), b = (int)((begin + q.key_tiles - 1) / piece);
    if (a == b) return;                                            // (one workgroup had it whole)
    const int r = sub * PER + threadIdx.x / LPR, row = rtile * ROWS + r, col = threadIdx.x % LPR * 4;
    if (row >= nrows) return;
    auto slot_of = [&](int k) { return 2 * (int64_t)k + (k == a ? 1 : 0); };
    float top = NEG_BIG;
    for (int k = a; k <= b; ++k) top = fmaxf(top, p.ws_ml[slot_of(k) * ROWS + r].x);
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll 4
    for (int k = a; k <= b; ++k) {
        const float2 ml = p.ws_ml[slot_of(k) * ROWS + r];
        const f32x4_t x = *(const f32x4_t*)(p.ws_acc + (slot_of(k) * ROWS + r) * DV + col);
        const float f = __builtin_amdgcn_exp2f(ml.x - top);
        sum = fmaf(f, ml.y, sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = fmaf(f, x[i], o[i]);
    }
    const float inv = (p.v_scale != nullptr ? p.v_scale[kvh] : 1.f) / sum;
    o *= inv;
    if (sum == 0.f) o = f32x4_t{0.f, 0.f, 0.f, 0.f};
    uint16_t* dst = (uint16_t*)p.out + ((int64_t)(q.begin + row / p.group) * p.hq + kvh * p.group + row % p.group) * DV;
    *(uint2*)(dst + col) = make_uint2(E::pack(o[0], o[1]), E::pack(o[2], o[3]));
}

}  // namespace

}  // namespace aicomp
