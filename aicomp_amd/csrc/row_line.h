// The line of work of the matrix-core kernels of row_attn.h (row_attn_mfma.hip, row_attn_shared.hip, row_attn_latent.hip): which piece of
// it a workgroup has, what a row sees of a tile, and how the pieces of an item are joined.
//
// All (sequence, KV head, row tile, key tile) in this order are one line, of which every workgroup has a piece of equal length, whatever
// the sequences' lengths are.  Before an item's key tiles the line has `over` places more, in which nothing is done: what the start and
// the end of an item cost, in tiles, so that pieces of several items have fewer tiles.  An item (sequence, KV head, row tile) that one
// workgroup has whole is finished by it; of others each leaves (m, l, O) of its rows in the workspace: in its slot 0 where it does not have
// the item's first key tile, else in its slot 1.  Who has the first tile says who has the others.
//
// Where contexts are short, every workgroup has one item whole (`single`): nothing to join, and no line to find one's place on.
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
    int hq, hkv, group, num_blocks;
    int span, shift;                   // tokens of a table's row; a block has 16 << shift
    float mul;                         // scale * log2(e)
    const float* k_scale;
    const float* v_scale;
    int workers;                       // workgroups
    bool single;                       // one for each (sequence, KV head, row tile)
    int least;                         // places that a workgroup has at least
    int over;                          // places of an item before its key tiles
    int row_tiles;                     // of the longest sequence (the join's grid)
    float* ws_acc;                     // [2 workers][rows of a tile][DV]
    float2* ws_ml;                     // [2 workers][rows of a tile]
    int2* ws_items;                    // [num_seqs][hkv][row_tiles]: the first workgroup that has the item, and how many more do (NULL: one has all)
};

// d: head_dim; R: groups of 16 rows to a wave; items: of the join's grid
void launch_row_attn_shared(const RowParams& p, bool f16, bool fp8, int d, int R, int64_t items, hipStream_t stream);
void launch_row_attn_latent(const RowParams& p, bool f16, int64_t items, hipStream_t stream);

namespace {

constexpr int BS = 16;                 // tokens that are looked up together: a block, or a part of one
constexpr float NEG_BIG = -0x1.fffffep127f;                    // no score is below it: the first that a row sees moves its reference
constexpr float SLACK = 8.f;           // a weight is at most 2^8: exact in both formats' range
constexpr float FAR = 0x1p26f;         // a reference beyond which its own rounding, 2^2 there, is no longer small beside that

#define GLOBAL_PTR(p) ((const __attribute__((address_space(1))) void*)(p))
#define LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

// All waves of the workgroup meet, and what they wrote to LDS is there.  Unlike __syncthreads(), which waits for loads from memory too:
// those under way stay under way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A sequence as the line of work sees it.
struct Seq {
    int begin, n, ctx, prior;          // ctx: 0 where its tokens are more than its context
    int row_tiles, key_tiles;
    __device__ __forceinline__ int items(const RowParams& p) const { return p.hkv * row_tiles; }
    __device__ __forceinline__ int places(const RowParams& p) const { return items(p) * (key_tiles + p.over); }
};

// ROWS, KT: rows and keys of a tile
template <int ROWS, int KT> __device__ __forceinline__ Seq load_seq(const RowParams& p, int s) {
    Seq q;
    q.begin = p.cu_q_lens ? max(0, p.cu_q_lens[s]) : s;
    q.n = p.cu_q_lens ? min(min(p.cu_q_lens[s + 1], p.rows) - q.begin, p.max_q_len) : 1;
    q.n = max(0, q.n);
    q.ctx = min(p.context_lens[s], p.span);
    q.prior = q.ctx - q.n;
    if (q.prior < 0) q.ctx = 0;
    q.row_tiles = (q.n * p.group + ROWS - 1) / ROWS;
    q.key_tiles = max(1, (q.ctx + KT - 1) / KT);
    return q;
}

// Which entry of a table's row has the g-th 16 tokens, and where they are in the pool, in units of 16 rows.
__device__ __forceinline__ int entry_of(const RowParams& p, const Seq& q, int g) {
    return min(g >> p.shift, (q.ctx - 1) >> (4 + p.shift));    // (entries behind the last one are not this sequence's)
}
__device__ __forceinline__ int64_t place_of(const RowParams& p, int entry, int kvh, int g) {
    return (((int64_t)max(0, min(entry, p.num_blocks - 1)) * p.hkv + kvh) << p.shift) + (g & ((1 << p.shift) - 1));
}

// A workgroup's piece of the line: places at .. end - 1, the first of them place `off` of sequence `seq`, `q`.  (A line is less than 2^31
// places, which the host sees to: 64-bit divisions cost a microsecond each.)
struct Piece {
    int at, end, length, seq, off;     // length: of every workgroup's piece
    Seq q;
};
struct PieceScratch {
    int sums[8];
    int seq, off;
    Seq q;
};

template <int ROWS, int KT, int THREADS>
__device__ __forceinline__ bool piece_of(const RowParams& p, int worker, PieceScratch& sh, Piece& mine) {
    if (p.single) {
        const int of_seq = p.hkv * p.row_tiles;
        mine.seq = (unsigned)worker / (unsigned)of_seq;
        const int item = worker - mine.seq * of_seq, kvh = (unsigned)item / (unsigned)p.row_tiles, rtile = item - kvh * p.row_tiles;
        mine.q = load_seq<ROWS, KT>(p, mine.seq);
        mine.length = mine.end = mine.q.key_tiles;
        mine.at = 0;
        mine.off = (kvh * mine.q.row_tiles + rtile) * mine.q.key_tiles;
        return rtile < mine.q.row_tiles;
    }
    const int per = (p.num_seqs + THREADS - 1) / THREADS, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int first = min((int)threadIdx.x * per, p.num_seqs), last = min(first + per, p.num_seqs);
    Seq q;
    int own = 0;
    for (int s = first; s < last; ++s) {
        q = load_seq<ROWS, KT>(p, s);
        own += q.places(p);
    }
    int up = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(up, o);
        if (lane >= o) up += x;
    }
    if (lane == 63) sh.sums[w] = up;
    __syncthreads();
    int line = 0, before = up - own;                           // the line's length; the part of it before this thread's sequences
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) {
        if (i < w) before += sh.sums[i];
        line += sh.sums[i];
    }
    mine.length = max(p.least, (int)(((unsigned)line + p.workers - 1) / (unsigned)p.workers));
    mine.at = worker * mine.length;
    mine.end = min(line, mine.at + mine.length);
    if (mine.at >= mine.end) return false;
    if (mine.at >= before && mine.at < before + own) {
        for (int s = first; s < last; ++s) {
            if (per > 1) q = load_seq<ROWS, KT>(p, s);
            const int all = q.places(p);
            if (mine.at >= before && mine.at < before + all) { sh.seq = s; sh.off = mine.at - before; sh.q = q; }
            before += all;
        }
    }
    __syncthreads();
    mine.seq = __builtin_amdgcn_readfirstlane(sh.seq);
    mine.off = __builtin_amdgcn_readfirstlane(sh.off);
    mine.q.begin = __builtin_amdgcn_readfirstlane(sh.q.begin);
    mine.q.n = __builtin_amdgcn_readfirstlane(sh.q.n);
    mine.q.ctx = __builtin_amdgcn_readfirstlane(sh.q.ctx);
    mine.q.prior = __builtin_amdgcn_readfirstlane(sh.q.prior);
    mine.q.row_tiles = __builtin_amdgcn_readfirstlane(sh.q.row_tiles);
    mine.q.key_tiles = __builtin_amdgcn_readfirstlane(sh.q.key_tiles);
    return true;
}

// The next item of the piece: key tiles t0 .. t1 - 1 of row tile `rtile` of KV head `kvh`; false if what is left of the piece has none.
struct Item {
    int kvh, rtile, t0, t1;
    bool whole;
    int64_t slot;                      // of the workspace, unless whole
};
template <int ROWS, int KT> __device__ __forceinline__ bool next_item(const RowParams& p, int worker, Piece& mine, Item& it) {
    while (mine.at < mine.end) {
        if (mine.off >= mine.q.places(p)) {                    // (sequences without tokens have none)
            mine.off = 0;
            mine.q = load_seq<ROWS, KT>(p, ++mine.seq);
            continue;
        }
        const int places = mine.q.key_tiles + p.over, item = (unsigned)mine.off / (unsigned)places;
        const int from = mine.off - item * places, to = min(places, from + (mine.end - mine.at)), at = mine.at;
        mine.off += to - from;
        mine.at += to - from;
        if (to <= p.over) continue;                            // (its tiles are the next workgroup's)
        it.t0 = max(0, from - p.over);
        it.t1 = to - p.over;
        it.kvh = (unsigned)item / (unsigned)mine.q.row_tiles;
        it.rtile = item - it.kvh * mine.q.row_tiles;
        it.whole = it.t0 == 0 && it.t1 == mine.q.key_tiles;
        it.slot = 2 * (int64_t)worker + (it.t0 == 0 ? 1 : 0);
        // who has the item, for the join: from this workgroup on, as many more as its further tiles take
        if (it.t0 == 0 && threadIdx.x == 0 && p.ws_items != nullptr) {
            const int more = (unsigned)(at - from + places - 1) / (unsigned)mine.length - worker;
            p.ws_items[(mine.seq * p.hkv + it.kvh) * p.row_tiles + it.rtile] = make_int2(worker, more);
        }
        return true;
    }
    return false;
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
    const int sub = blockIdx.x % (ROWS / PER), item = blockIdx.x / (ROWS / PER);
    const int rtile = item % p.row_tiles, kvh = item / p.row_tiles % p.hkv, seq = item / p.row_tiles / p.hkv;
    const Seq q = load_seq<ROWS, KT>(p, seq);
    int2 who = p.ws_items[item];
    who.x = __builtin_amdgcn_readfirstlane(who.x);
    who.y = __builtin_amdgcn_readfirstlane(who.y);
    const int r = sub * PER + threadIdx.x / LPR, row = rtile * ROWS + r, col = threadIdx.x % LPR * 4;
    if (row >= q.n * p.group || who.y == 0) return;            // (no such row: its entry was not written)
    auto slot_of = [&](int k) { return 2 * (int64_t)(who.x + k) + (k == 0 ? 1 : 0); };
    // Pieces eight at a time, all their loads under way together (what they wait for is most of this kernel's time); a place behind the
    // last piece repeats that one's and is not added.
    constexpr int AT_ONCE = 8;
    float top = NEG_BIG, sum = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int first = 0; first <= who.y; first += AT_ONCE) {
        float2 ml[AT_ONCE];
        f32x4_t x[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int64_t at = slot_of(min(first + k, who.y)) * ROWS + r;
            ml[k] = p.ws_ml[at];
            x[k] = *(const f32x4_t*)(p.ws_acc + at * DV + col);
        }
        float m_new = top;
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) m_new = fmaxf(m_new, ml[k].x);
        const float alpha = __builtin_amdgcn_exp2f(top - m_new);
        top = m_new;
        sum *= alpha;
        o *= alpha;
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            if (first + k > who.y) break;                      // uniform
            const float f = __builtin_amdgcn_exp2f(ml[k].x - top);
            sum = fmaf(f, ml[k].y, sum);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = fmaf(f, x[k][i], o[i]);
        }
    }
    const float inv = (p.v_scale != nullptr ? p.v_scale[kvh] : 1.f) / sum;
    o *= inv;
    if (sum == 0.f) o = f32x4_t{0.f, 0.f, 0.f, 0.f};
    uint16_t* dst = (uint16_t*)p.out + ((int64_t)(q.begin + row / p.group) * p.hq + kvh * p.group + row % p.group) * DV;
    *(uint2*)(dst + col) = make_uint2(E::pack(o[0], o[1]), E::pack(o[2], o[3]));
}

}  // namespace

}  // namespace aicomp
