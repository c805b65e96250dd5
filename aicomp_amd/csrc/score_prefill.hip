// Rows of prompt chunks by a score rule (score.h) on gfx950 matrix cores.
//
// Mathematics: online softmax over tiles of 64 keys, one pass.  With a cap,
//   cap tanh(x / cap) = cap - 2 cap / (1 + e^(2 x / cap)):
// one exponential, one reciprocal and one multiply-add give the score in the exponent's units with the running maximum already
// subtracted; without a cap it is one multiply-add.  The bias by distance is one addition and one multiply-add more.
//
// Work split   one workgroup (4 waves) per (64 or 128 query rows, sequence, head group), or, with few rows, per one of the parts that
//              their keys are divided into (a second kernel joins the parts); a row is a (position, query head)
//              pair, the heads of a KV head packed side by side where the group divides 16, so that a K/V tile serves all of them.
//              Every row's visible keys are one interval [lo, hi): a workgroup walks the tiles between the smallest lo and the
//              largest hi of its rows, a wave computes those between its own, and only tiles that cross a row's
//              borders pay for the mask.
// K/V tiles    64 tokens, double-buffered in LDS, one barrier per tile.  16-bit pools: straight into LDS
//              (global_load_lds_dwordx4) one tile ahead, rows unpadded, 16-byte chunks swizzled by the row.  fp8 pools: through
//              registers, widened (exactly) to the query's type on the way.
// head_dim     64, 128 or 256 (its tiles are 128 KB of LDS, one workgroup to a CU).
// Per wave     16 or 32 rows.  S^T = K Q^T, rows as columns of the B operand; O^T += V^T P^T with V^T read by the transposing LDS
//              read, in the token order of the scores, so that P never leaves its lane.
// Rounding     The weights to the 16-bit format of the matrix cores; everything else in float32 until the one rounding of
//              the result.  (The scores' multiplier in Q would save an instruction per score, which no time shows, and round
//              Q once more: against float64 an error of 3.0e-3 where this has 2.1e-3, bf16, a prompt of 8192 under a cap.)
// Bound by     the issue of vector and matrix instructions, which overlap little: of a prompt of 8192, 32 / 8 heads of 128 under a cap,
//              the matrix cores hold 39 % of the cycles, vector instructions 56 % (8.5 a score, of which three, exponentials and
//              a reciprocal, take two slots each), and 9 % of them both; 600 us, 0.92 PFLOP/s (a large product reaches 1.26).  fp8
//              pools 724 us: the codes' widening and waits.  head_dim 64 the same 405 us: half the products for the same scores, vector
//              79 %.  4 x 512 with a window of 1024, 52 us (26 % and 46 %).  head_dim 256, 4096 tokens of 16 / 8 heads, 300 us:
//              19 % and 24 %, one wave to a SIMD has no other to run beside.
#include "score_prefill.h"

#include <algorithm>
#include <type_traits>

namespace aicomp {

namespace {

constexpr int KT = 64;                 // tokens per tile
constexpr int NB = KT / BS;            // blocks per tile

template <bool FP8> struct Stage;              // registers of one K and one V tile (fp8 pools)
template <> struct Stage<false> {};
template <> struct Stage<true> { uint2 k[8], v[8]; };

// E: 16-bit format of queries and output; R: column groups of 16 rows per wave; DH: head_dim
template <typename E, bool FP8, int R, int DH, bool CAP, bool BIAS>
__global__ void __launch_bounds__(256, DH == 256 ? 1 : DH == 64 ? 3 : 2)
score_prefill_kernel(ScorePrefillParams p) {
    constexpr int KROW = 2 * DH;               // bytes of an LDS row
    constexpr int NSL = DH / 32;               // k-slots of a row (QK^T MFMAs per 16 x 16 tile)
    constexpr int NJ = DH / 16;                // 16-element output tiles
    constexpr int CPR = DH / 8;                // 16-byte chunks per row
    constexpr int NH = KT / 16;
    constexpr int TILE_BYTES = KT * KROW;
    constexpr int WROWS = 16 * R;              // rows per wave
    constexpr int NS = 4 * NH;                 // scores per lane and column group
    const int part = R == 1 ? blockIdx.x / p.hgroups : 0, hgroup = R == 1 ? blockIdx.x % p.hgroups : blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g4 = lane >> 4;
    const int pos_per_wg = 4 * WROWS / p.gpack;

    __shared__ __attribute__((aligned(16))) unsigned char k0[TILE_BYTES];
    __shared__ __attribute__((aligned(16))) unsigned char v0[TILE_BYTES];
    __shared__ __attribute__((aligned(16))) unsigned char k1[TILE_BYTES];
    __shared__ __attribute__((aligned(16))) unsigned char v1[TILE_BYTES];
    __shared__ int span[2][4];

    int seq, qtile;
    place_of(p, seq, qtile);
    const int q_begin = p.cu_q_lens[seq];
    const int n = p.cu_q_lens[seq + 1] - q_begin;
    const int ctx = min(p.context_lens[seq], p.max_blocks * BS);
    const int prior = ctx - n;
    const int q0 = qtile * pos_per_wg;
    if (n <= 0 || q0 >= n) return;
    const int kvh = (hgroup * p.gpack) / p.group;

    // rows of this lane's columns (beyond the chunk's end: the last one's, computed and not stored)
    int head[R], pos[R], lo[R], hi[R];
    bool row_valid[R];
    int mine_lo = INT32_MAX, mine_hi = 0, all_lo = 0, all_hi = INT32_MAX;
#pragma unroll
    for (int c = 0; c < R; ++c) {
        const int row = WROWS * w + 16 * c + r16;
        const int qpos = q0 + row / p.gpack;
        head[c] = hgroup * p.gpack + row % p.gpack;
        row_valid[c] = qpos < n;
        const int i = min(qpos, n - 1);
        pos[c] = prior + i;
        lo[c] = hi[c] = 0;
        if (prior >= 0) visible_keys(p.rule, q_begin + i, seq, pos[c], ctx, lo[c], hi[c]);
        if (lo[c] < hi[c]) { mine_lo = min(mine_lo, lo[c]); mine_hi = max(mine_hi, hi[c]); }
        all_lo = max(all_lo, lo[c] < hi[c] ? lo[c] : INT32_MAX);
        all_hi = min(all_hi, hi[c]);
    }
    // keys that some row of the wave sees, [wave_lo, wave_hi), and those that all of them see, [full_lo, full_hi)
    const bool idle = q0 + (WROWS * w) / p.gpack >= n;         // wave-uniform: all rows beyond the chunk's end
    const int wave_lo = idle ? INT32_MAX : wave_min(mine_lo), wave_hi = idle ? 0 : -wave_min(-mine_hi);
    const int full_lo = -wave_min(-all_lo), full_hi = wave_min(all_hi);
    if (lane == 0) { span[0][w] = wave_lo; span[1][w] = wave_hi; }
    __syncthreads();
    int kv_lo = min(min(span[0][0], span[0][1]), min(span[0][2], span[0][3]));
    int kv_hi = max(max(span[1][0], span[1][1]), max(span[1][2], span[1][3]));
    kv_lo = __builtin_amdgcn_readfirstlane(kv_lo);
    kv_hi = __builtin_amdgcn_readfirstlane(kv_hi);
    int t_first = kv_lo / KT, t_end = (kv_hi + KT - 1) / KT;
    const bool divided = R == 1 && p.parts > 1;
    if (divided) {
        const int per = max((t_end - t_first + p.parts - 1) / p.parts, PART_KEYS / KT);
        t_end -= part * per;
        t_first = max(t_first, t_end - per);
    }
    if (kv_lo >= kv_hi || t_first >= t_end) {                  // nothing visible to any row: zero rows
        for (int i = tid; divided && i < 4 * WROWS; i += 256) {
            const int at = q0 + i / p.gpack;
            if (at < n) p.ws_ml[(part * p.rows + q_begin + at) * p.hq + hgroup * p.gpack + i % p.gpack] = make_float2(NEG_BIG, 0.f);
        }
        for (int i = tid; !divided && i < 4 * WROWS * CPR; i += 256) {
            const int row = i / CPR, at = q0 + row / p.gpack;
            if (at < n)
                *(uint4*)((uint16_t*)p.out + ((int64_t)(q_begin + at) * p.hq + hgroup * p.gpack + row % p.gpack) * DH + 8 * (i % CPR)) =
                    make_uint4(0, 0, 0, 0);
        }
        return;
    }

    // Q as the B operand: column = this lane's row, k-slots = dims 32 s + 8 g4 ..
    const float ks = FP8 ? p.k_scale[kvh] : 1.f;
    const float mul = CAP ? 2.f * LOG2E * p.rule.cap_mul * ks : p.rule.mul * ks;
    uint4 qf[R][NSL];
#pragma unroll
    for (int c = 0; c < R; ++c) {
        const uint16_t* qrow = (const uint16_t*)p.query + ((int64_t)(q_begin + pos[c] - prior) * p.hq + head[c]) * DH;
#pragma unroll
        for (int s = 0; s < NSL; ++s) {
            qf[c][s] = *(const uint4*)(qrow + 32 * s + 8 * g4);
        }
    }

    // m: the reference that exponents are taken against, in their units; 0 until the row has seen a key (fresh)
    float m[R], lsum[R], slope[R];
    bool fresh[R];
    f32x4_t O[R][NJ];
#pragma unroll
    for (int c = 0; c < R; ++c) {
        m[c] = 0.f; lsum[c] = 0.f; fresh[c] = true;
        slope[c] = BIAS ? p.rule.slopes[head[c]] * LOG2E : 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) O[c][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    const float cap = p.rule.cap_log2;

    typedef const __attribute__((address_space(4))) int32_t* const_i32_ptr;
    const_i32_ptr table = (const_i32_ptr)(p.block_table + (int64_t)seq * p.block_table_stride);

    // Chunk slot s of LDS row r holds chunk s ^ swz(r), fitted to how each operand is read (the LDS delivers its full width when
    // consecutive lanes share 64-byte segments that spread over a bank line; see prefill_mfma.hip for the measurements).
    auto swz_k = [](int row) {
        const int a = (row >> 2) & 3, b = row & 3;
        return DH >= 128 ? (a | (b << 2)) : (a | ((b >> 1) << 2));
    };
    auto swz_v = [](int row) {
        const int a = (row >> 2) & 3, b = row & 3;
        return DH >= 128 ? ((a | ((b & 1) << 2)) << 1) : (a << 1);
    };

    // --- 16-bit pools: tile t straight into LDS.  Wave w brings in block w of the tile, 1 KB per instruction.
    constexpr int RPI = 1024 / KROW, NQ = 16 / RPI;
    const uint32_t blk_stride = (uint32_t)p.hkv * (BS * DH * (FP8 ? 1 : 2));
    const char* kp = (const char*)p.k_pool + (int64_t)kvh * (BS * DH * (FP8 ? 1 : 2));
    const char* vp = (const char*)p.v_pool + (int64_t)kvh * (BS * DH * (FP8 ? 1 : 2));
    const int lrow = lane / CPR, lslot = lane % CPR;
    uint32_t offk[NQ], offv[NQ];               // pool offset of this lane's chunk, less the immediate
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        offk[q] = lrow * KROW + ((lslot ^ swz_k(RPI * q + lrow)) << 4);
        offv[q] = lrow * KROW + ((lslot ^ swz_v(RPI * q + lrow)) << 4);
    }
    auto fetch_dma = [&](int t, unsigned char* kb, unsigned char* vb) __attribute__((always_inline)) {
        const int first = NB * t;
        if (t * KT >= kv_lo && (t + 1) * KT <= kv_hi) {                // workgroup-uniform
            const uint32_t blk = min((uint32_t)max(table[first + w], 0), (uint32_t)(p.num_blocks - 1));
            const uint64_t base = (uint64_t)blk * blk_stride;
            // (opaque lane offsets: each address stays a uniform base plus a 32-bit offset; the instruction's own offset, up to
            // 3 KB, moves the pool's address and that in LDS together)
            uint32_t ok[NQ], ov[NQ];
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                ok[q] = offk[q]; ov[q] = offv[q];
                asm volatile("" : "+v"(ok[q]), "+v"(ov[q]));
            }
            const char* ka = kp + base;
            const char* va = vp + base;
#define AICOMP_DMA_ROWS(addr, o, buf, q)                                                                                   \
            if constexpr (q < NQ)                                                                                          \
                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(addr + (q / 4 * 4096) + o[q < NQ ? q : 0]),                    \
                                                 LDS_PTR(buf + 16 * w * KROW + q / 4 * 4096), 16, 1024 * (q % 4), 0);
            AICOMP_DMA_ROWS(ka, ok, kb, 0) AICOMP_DMA_ROWS(ka, ok, kb, 1) AICOMP_DMA_ROWS(ka, ok, kb, 2) AICOMP_DMA_ROWS(ka, ok, kb, 3)
            AICOMP_DMA_ROWS(ka, ok, kb, 4) AICOMP_DMA_ROWS(ka, ok, kb, 5) AICOMP_DMA_ROWS(ka, ok, kb, 6) AICOMP_DMA_ROWS(ka, ok, kb, 7)
            AICOMP_DMA_ROWS(va, ov, vb, 0) AICOMP_DMA_ROWS(va, ov, vb, 1) AICOMP_DMA_ROWS(va, ov, vb, 2) AICOMP_DMA_ROWS(va, ov, vb, 3)
            AICOMP_DMA_ROWS(va, ov, vb, 4) AICOMP_DMA_ROWS(va, ov, vb, 5) AICOMP_DMA_ROWS(va, ov, vb, 6) AICOMP_DMA_ROWS(va, ov, vb, 7)
#undef AICOMP_DMA_ROWS
        } else {
            // rows that nobody here sees take the nearest one that somebody does
            int l = lane;
            asm volatile("" : "+v"(l));                                // (nothing of this in registers across the loop)
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const int lslot = l % CPR, row = RPI * q + l / CPR;
                const int tok = max(kv_lo, min(BS * (first + w) + row, kv_hi - 1));
                const uint32_t blk = min((uint32_t)max(p.block_table[(int64_t)seq * p.block_table_stride + tok / BS], 0),
                                         (uint32_t)(p.num_blocks - 1));
                const uint64_t base = (uint64_t)blk * blk_stride + (tok % BS) * KROW;
                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(kp + base + ((lslot ^ swz_k(row)) << 4)),
                                                 LDS_PTR(kb + (16 * w + RPI * q) * KROW), 16, 0, 0);
                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(vp + base + ((lslot ^ swz_v(row)) << 4)),
                                                 LDS_PTR(vb + (16 * w + RPI * q) * KROW), 16, 0, 0);
            }
        }
    };
    // --- fp8 pools: tile t into registers, eight codes per lane and load; then widened into LDS
    constexpr int RPL = 256 / CPR, NL = KT / RPL;              // rows per load of the workgroup, loads per tile and pool
    auto fetch = [&](int t, Stage<FP8>& st) __attribute__((always_inline)) {
        if constexpr (FP8) {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int tok = max(kv_lo, min(KT * t + RPL * i + tid / CPR, kv_hi - 1));
                const int b = p.block_table[(int64_t)seq * p.block_table_stride + tok / BS];
                const uint32_t blk = min((uint32_t)max(b, 0), (uint32_t)(p.num_blocks - 1));
                const uint64_t at = (uint64_t)blk * blk_stride + (tok % BS) * DH + (tid % CPR) * 8;
                st.k[i] = *(const uint2*)(kp + at);
                st.v[i] = *(const uint2*)(vp + at);
            }
        }
    };
    auto stash = [&](const Stage<FP8>& st, unsigned char* kb, unsigned char* vb) __attribute__((always_inline)) {
        if constexpr (FP8) {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int row = RPL * i + tid / CPR, c = tid % CPR;
                *(uint4*)(kb + row * KROW + ((c ^ swz_k(row)) << 4)) = E::from_fp8(st.k[i]);
                *(uint4*)(vb + row * KROW + ((c ^ swz_v(row)) << 4)) = E::from_fp8(st.v[i]);
            }
        }
    };

    const int prow = 4 * (r16 & 3) + (r16 >> 2);               // permuted K row
    const int vrow = 4 * (r16 >> 2) + g4;

    // one tile out of LDS
    auto compute = [&](int t, const unsigned char* kb, const unsigned char* vb) __attribute__((always_inline)) {
        const int start = t * KT;
        if (start >= wave_hi || start + KT <= wave_lo) return;         // wave-uniform
        f32x4_t sa[NH][R];
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int c = 0; c < R; ++c) sa[h][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NSL; ++s) {
            uint4 a[NH];
#pragma unroll
            for (int h = 0; h < NH; ++h)
                a[h] = *(const uint4*)(kb + (16 * h + prow) * KROW + (((4 * s + g4) ^ swz_k(prow)) << 4));
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int c = 0; c < R; ++c) sa[h][c] = E::mfma(a[h], qf[c][s], sa[h][c]);
        }
        // issue order: the operand reads run two k-slots ahead of the matrix instructions that take them (and below, two output tiles)
        if constexpr (DH == 128 && R == 2 && !FP8) {
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * NH, 0);
#pragma unroll
            for (int s = 0; s < NSL; ++s) {
                __builtin_amdgcn_sched_group_barrier(0x008, NH * R, 0);
                if (s + 2 < NSL) __builtin_amdgcn_sched_group_barrier(0x100, NH, 0);
            }
        }
        uint4 pf[R][NH / 2];
        float alpha[R];
        bool grew[R];                                                  // wave-uniform
        auto softmax = [&](auto mask_tag) __attribute__((always_inline)) {
            constexpr bool MASK = decltype(mask_tag)::value;
#pragma unroll
            for (int c = 0; c < R; ++c) {
                float sc[NS];
                bool dead[NS];
                const float dist = (float)(start + g4 - pos[c]);       // score k is of key start + g4 + 16 (k / 4) + 4 (k % 4)
                const float top = (CAP ? cap : 0.f) - m[c];
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    const int r = 16 * (k >> 2) + 4 * (k & 3);
                    sc[k] = sa[k >> 2][c][k & 3];
                    const float base = BIAS ? fmaf(-slope[c], fabsf(dist + (float)r), top) : top;
                    if constexpr (CAP) sc[k] = fmaf(-2.f * cap, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(sc[k] * mul)), base);
                    else sc[k] = fmaf(sc[k], mul, base);
                    dead[k] = MASK && (uint32_t)(start + g4 - lo[c] + r) >= (uint32_t)(hi[c] - lo[c]);
                    if (MASK && dead[k]) sc[k] = NEG_BIG;
                }
                // Exponentials against the current reference; as long as a lane's sum stays at or below 2^8 every weight
                // is exact enough in the 16-bit format and neither the reference nor the accumulators move.
                uint32_t pk[NS / 2];
                float psum = 0.f;
                auto exps = [&]() {
                    psum = 0.f;
#pragma unroll
                    for (int k = 0; k < NS; k += 2) {
                        float p0 = __builtin_amdgcn_exp2f(sc[k]);
                        float p1 = __builtin_amdgcn_exp2f(sc[k + 1]);
                        if (MASK && dead[k]) p0 = 0.f;
                        if (MASK && dead[k + 1]) p1 = 0.f;
                        pk[k >> 1] = E::pack(p0, p1);
                        psum = E::pair_sum(pk[k >> 1], psum);
                    }
                };
                exps();
                // A row's scores sit in four lanes, which must share one reference: the wave takes the slow path together.
                // A row that has seen no key yet adopts the first maximum that it meets, whatever its sign.
                grew[c] = __any(fresh[c] || !(psum <= 256.f));
                if (grew[c]) {
                    float mx = sc[0];
#pragma unroll
                    for (int k = 1; k < NS; ++k) mx = fmaxf(mx, sc[k]);
                    mx = xor32_max(xor16_max(mx));
                    const bool live = mx > 0.5f * NEG_BIG;
                    const float shift = live && (fresh[c] || mx > 0.f) ? mx : 0.f;
                    alpha[c] = fresh[c] ? 0.f : __builtin_amdgcn_exp2f(-shift);
                    fresh[c] = fresh[c] && !live;
                    m[c] += shift;
                    lsum[c] *= alpha[c];
#pragma unroll
                    for (int k = 0; k < NS; ++k) sc[k] -= shift;
                    exps();
                }
                lsum[c] += psum;
#pragma unroll
                for (int hp = 0; hp < NH / 2; ++hp)
                    pf[c][hp] = make_uint4(pk[4 * hp], pk[4 * hp + 1], pk[4 * hp + 2], pk[4 * hp + 3]);
            }
        };
        if (start < full_lo || start + KT > full_hi) softmax(std::true_type{}); else softmax(std::false_type{});
#pragma unroll
        for (int c = 0; c < R; ++c) {
            if (grew[c]) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) O[c][j] *= alpha[c];
            }
        }
        // O^T += V^T P^T: two transposing reads (token slots 0..3, 4..7) make one operand, which feeds the R column groups
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            typedef short v4i16_t __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) v4i16_t* lds_v4i16_ptr;
            typedef short v8i16_t __attribute__((ext_vector_type(8)));
#pragma unroll
            for (int hp = 0; hp < NH / 2; ++hp) {
                const int voff = 32 * hp * KROW + vrow * KROW + (((2 * j + ((r16 >> 1) & 1)) ^ swz_v(vrow)) << 4) + (r16 & 1) * 8;
                const v4i16_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(vb + voff));
                const v4i16_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(vb + (voff + 16 * KROW)));
                const v8i16_t av = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
                for (int c = 0; c < R; ++c) O[c][j] = E::mfma(__builtin_bit_cast(uint4, av), pf[c][hp], O[c][j]);
            }
        }
        if constexpr (DH == 128 && R == 2 && !FP8) {
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * NH, 1);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                __builtin_amdgcn_sched_group_barrier(0x008, (NH / 2) * R, 1);
                if (j + 2 < NJ) __builtin_amdgcn_sched_group_barrier(0x100, NH, 1);
            }
        }
    };

    Stage<FP8> st;
    // Opens the step of tile t: it is in `kb` / `vb` afterwards for every wave, and the next one is on its way into the other pair.
    auto open = [&](int t, unsigned char* kb, unsigned char* vb, unsigned char* kn, unsigned char* vn) __attribute__((always_inline)) {
        if constexpr (FP8) {
            stash(st, kb, vb);                                     // (nobody reads this pair: its readers met at the tile between)
            __syncthreads();
            fetch(max(t - 1, t_first), st);
        } else {
            // every wave waits for its own direct-to-LDS loads and then meets the others
            __builtin_amdgcn_s_waitcnt(0x0F70);                    // vmcnt(0)
            __syncthreads();                                       // also: the tile before is no longer read by anyone
            if (t > t_first) fetch_dma(t - 1, kn, vn);
        }
    };
    // From the nearest keys to the farthest: with a bias the scores then fall from tile to tile, and the references, which the first
    // tiles set, stay (bias alone, a prompt of 8192, 32 / 8 heads: 660 us in the order of the keys).
    __syncthreads();
    if constexpr (FP8) fetch(t_end - 1, st); else fetch_dma(t_end - 1, k0, v0);
    for (int t = t_end - 1; t >= t_first; t -= 2) {
        open(t, k0, v0, k1, v1);
        compute(t, k0, v0);
        if (t > t_first) {
            open(t - 1, k1, v1, k0, v0);
            compute(t - 1, k1, v1);
        }
    }

    // lane (column r16 of column group c, g4) holds element 16 j + 4 g4 + i of its row in O[c][j][i]
#pragma unroll
    for (int c = 0; c < R; ++c) {
        float l = lsum[c];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        float worst = 0.f;                                             // (0 times a value that is not finite is not a number)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) worst = fmaf(0.f, O[c][j][i], worst);
        uint64_t again = __ballot(row_valid[c] && lo[c] < hi[c] && l - l == 0.f && !(worst == 0.f));
        again |= again >> 32;
        again = (again | (again >> 16)) & 0xffff;                      // rows, by column
        if (divided) {
            if (row_valid[c] && !((again >> r16) & 1)) {
                const int64_t slot = (part * p.rows + q_begin + pos[c] - prior) * p.hq + head[c];
                if (g4 == 0) p.ws_ml[slot] = make_float2(m[c], l);
                if (l != 0.f) {
#pragma unroll
                    for (int j = 0; j < NJ; ++j) *(f32x4_t*)(p.ws_acc + slot * DH + 16 * j + 4 * g4) = O[c][j];
                }
            }
            lo[c] = max(lo[c], t_first * KT);
            hi[c] = min(hi[c], t_end * KT);
        } else if (row_valid[c] && !((again >> r16) & 1)) {
            const bool none = l == 0.f;                                // (no visible key, or all of weight 0)
            const float inv = (FP8 ? p.v_scale[kvh] : 1.f) / l;
            uint16_t* o = (uint16_t*)p.out + ((int64_t)(q_begin + pos[c] - prior) * p.hq + head[c]) * DH + 4 * g4;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                *(uint2*)(o + 16 * j) = none ? make_uint2(0, 0) : make_uint2(E::pack(O[c][j][0] * inv, O[c][j][1] * inv),
                                                                             E::pack(O[c][j][2] * inv, O[c][j][3] * inv));
        }
        for (; again; again &= again - 1) {                            // wave-uniform
            const int r = __builtin_ctzll(again);
            const int at = __builtin_amdgcn_readlane(pos[c], r);
            score_row<E, FP8, DH, R == 1>(p, seq, q_begin + at - prior, __builtin_amdgcn_readlane(head[c], r), kvh, at,
                                  __builtin_amdgcn_readlane(lo[c], r), __builtin_amdgcn_readlane(hi[c], r), part, lane);
        }
    }
}

template <typename E, bool FP8, int R, int DH>
void launch_rule(const ScorePrefillParams& p, bool cap, bool bias, dim3 grid, hipStream_t stream) {
    if (cap && bias) hipLaunchKernelGGL((score_prefill_kernel<E, FP8, R, DH, true, true>), grid, dim3(256), 0, stream, p);
    else if (cap) hipLaunchKernelGGL((score_prefill_kernel<E, FP8, R, DH, true, false>), grid, dim3(256), 0, stream, p);
    else if (bias) hipLaunchKernelGGL((score_prefill_kernel<E, FP8, R, DH, false, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((score_prefill_kernel<E, FP8, R, DH, false, false>), grid, dim3(256), 0, stream, p);
}

template <typename E, bool FP8>
void launch_shape(const ScorePrefillParams& p, int R, int d, bool cap, bool bias, dim3 grid, hipStream_t stream) {
    if (d == 256) { if (R == 2) launch_rule<E, FP8, 2, 256>(p, cap, bias, grid, stream); else launch_rule<E, FP8, 1, 256>(p, cap, bias, grid, stream); }
    else if (d == 64) {
        if constexpr (!FP8) {              // (see score_chunk_plan)
            if (R == 2 && cap) { hipLaunchKernelGGL((score_prefill_kernel<E, FP8, 2, 64, true, false>), grid, dim3(256), 0, stream, p); return; }
            if (R == 2) { hipLaunchKernelGGL((score_prefill_kernel<E, FP8, 2, 64, false, false>), grid, dim3(256), 0, stream, p); return; }
        }
        launch_rule<E, FP8, 1, 64>(p, cap, bias, grid, stream);
    }
    else { if (R == 2) launch_rule<E, FP8, 2, 128>(p, cap, bias, grid, stream); else launch_rule<E, FP8, 1, 128>(p, cap, bias, grid, stream); }
}

}  // namespace

bool score_prefill_supported(const ScoreArgs& a) {
    if (a.bs != BS) return false;
    const int group = a.hq / a.hkv, gpack = 16 % group == 0 ? group : 1;
    const int64_t qtiles = ((int64_t)a.max_q_len * gpack + 63) / 64;
    return a.num_seqs <= 65535 && qtiles <= 65535 && a.num_blocks <= INT32_MAX && (int64_t)a.hkv * BS * a.d * 4 <= UINT32_MAX;
}

// 128 rows to a workgroup (R = 2) read a tile from LDS once for twice the rows, where they leave no CU without its workgroups; 64 rows
// in smaller calls, with fp8 pools or a bias at head_dim 64 too (there 128 take the registers of a second or third workgroup on a CU).
// us, 64 against 128 rows, 32 / 8 heads under a cap: prompts of 4 and 8 x 1024, head_dim 64: 41.4 against 41.3, 77 against 73 (fp8: 46
// against 59 for the first); 2048 and 2000 + 2048 tokens, head_dim 128: 64 against 64, 152 against 129; 512 after 2048: 54 against 72;
// head_dim 256, 16 / 8 heads: 2048 and 3000 tokens 110 against 119, 191 against 166; 64 with a bias alone, 8192 tokens: 347 against 351.
//
// Where even those are too few for two to a CU (head_dim 256: one), the keys are divided: i parts take the tiles' time / i and then a
// second kernel, which costs about 4 us, 0.6 us per part and the parts' sums at 3 TB/s both ways.  256 new tokens behind 2048, head_dim
// 128: 48 us in one part, 36 in 2 or 4, 41 in 8; 64 behind 4000: 79 in one, 28 in 8, 35 in 16; 512 from none: 16 in one, 25 in 2.
// float32, the same: 204, 115 in 2, 100 in 4; 356, 63 in 8.
ScoreChunkPlan score_chunk_plan(const ScoreArgs& a) {
    const int group = a.hq / a.hkv, gpack = 16 % group == 0 ? group : 1;
    const bool f32 = a.q_dtype == AICOMP_KV_F32, fp8 = a.kv_dtype == AICOMP_KV_FP8_E4M3;
    auto workgroups = [&](int rows) {
        const int64_t per = rows / gpack;
        return std::max<int64_t>(1, a.hq / gpack * std::min(a.num_seqs * ((a.max_q_len + per - 1) / per), a.rows / per + a.num_seqs));
    };
    if (!f32 && !(a.d == 64 && (fp8 || a.slopes != nullptr)) && workgroups(128) >= (a.d == 64 ? 1024 : a.d == 128 ? 512 : 320))
        return ScoreChunkPlan{2, 1};
    // (the bias decides nothing below here: the size of a workspace does not know of it)
    const double tile_us = (f32 ? 4.2 : 1.) * (a.d == 64 ? 0.9 : a.d == 128 ? 1.3 : 2.4), tiles = (double)((a.span + 63) / 64);
    const int64_t most = std::min({(a.d == 256 ? 256 : 512) / workgroups(64), (a.span + PART_KEYS - 1) / PART_KEYS, (int64_t)16});
    ScoreChunkPlan plan{1, 1};
    double best = tiles * tile_us;
    for (int i = 2; i <= (int)most; ++i) {
        const double us = tiles * tile_us / i + 4 + i * (0.6 + 8e-6 * a.rows * a.hq * a.d / 3);
        if (us < best) { best = us; plan.parts = i; }
    }
    return plan;
}

int launch_score_prefill(const ScoreArgs& a) {
    if (a.q_dtype == AICOMP_KV_F32) return launch_score_prefill_f32(a);
    const ScorePrefillParams p = chunk_params(a);
    const int R = score_chunk_plan(a).R;
    const int pos_per_wg = 64 * R / p.gpack;
    dim3 grid((unsigned)(p.hgroups * p.parts), (unsigned)a.num_seqs, (unsigned)((a.max_q_len + pos_per_wg - 1) / pos_per_wg));
    const bool fp8 = a.kv_dtype == AICOMP_KV_FP8_E4M3, cap = a.cap > 0.f, bias = a.slopes != nullptr;
    if (a.q_dtype == AICOMP_KV_F16) {
        if (fp8) launch_shape<F16Fmt, true>(p, R, a.d, cap, bias, grid, a.stream);
        else launch_shape<F16Fmt, false>(p, R, a.d, cap, bias, grid, a.stream);
    } else {
        if (fp8) launch_shape<Bf16Fmt, true>(p, R, a.d, cap, bias, grid, a.stream);
        else launch_shape<Bf16Fmt, false>(p, R, a.d, cap, bias, grid, a.stream);
    }
    if (p.parts > 1) { if (a.q_dtype == AICOMP_KV_F16) launch_join<F16Fmt>(p, a); else launch_join<Bf16Fmt>(p, a); }
    AICOMP_HIP_LAUNCH_CHECK();
    return AICOMP_KV_OK;
}

}  // namespace aicomp
