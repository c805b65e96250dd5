// Attention of query rows over cached rows (row_attn.h) on the matrix cores: latent rows of 512 + 64 elements, trees of drafts over K and
// V pools of head_dim 64, 128 and 256; 16-bit rows, and fp8 ones under them; blocks of 16, 32, 64 .. tokens.
//
// The rows of a sequence and KV head, (token, head) pairs one after the other, are cut into tiles of 16 R rows, and the keys into
// tiles of 32.  A workgroup has a row tile; its four waves take the key tiles in turn, each with its own piece of LDS, its own running
// reference m, sum l and output O, and nothing to wait for but its own loads:
//   S^T = K Q^T      16 x 16 x 32 products; a lane then has four keys of a row per 16, the order in which
//   O^T += V^T P^T   takes its weights from registers, V^T out of LDS by transposing reads
// The reference moves when a score passes it by 2^8, so most tiles leave O as it is.  Rows of a tile are swizzled in 16-byte chunks
// (chunk c of key k at c ^ f(k)), so that both reads spread over the banks.  Tiles come from the pool straight into LDS.
//
// How the work is divided: row_line.h.  Calls of more rows to a sequence and KV head are row_attn_latent.hip's (latent rows, above 16) and
// row_attn_shared.hip's (trees, above 32): there a key that one wave reads serves too few rows.
//
// Bound by latency in small calls (one row of 16 heads over 700 latent rows 15.3 us, of which 4.4 are the second launch) and by HBM in
// large ones: 64 rows of 16 heads over 512 .. 4096 latent rows 48 us, 3.6 TB/s of the 5.1 that a large copy reaches.
#include "row_line.h"

#include <algorithm>

namespace aicomp {

namespace {

constexpr int KT = 32;                 // keys per tile

// E: 16-bit format of queries and output; DK / DV: elements of a key / value row; R: groups of 16 rows; LATENT: a value is the
// first part of its key's row.  OCC: workgroups per CU.
template <typename E, bool FP8, int DK, int DV, bool LATENT, int R, int OCC>
__global__ void __launch_bounds__(256, OCC)
row_attn_kernel(RowParams p) {
    constexpr int ROWS = 16 * R;
    constexpr int KROW = 2 * DK, VROW = LATENT ? KROW : 2 * DV;    // bytes of a row in LDS
    constexpr int NS = DK / 32, NJ = DV / 16;
    constexpr int TILE = KT * KROW + (LATENT ? 0 : KT * VROW);     // bytes per wave
    constexpr int VBASE = LATENT ? 0 : KT * KROW;
    constexpr int CH = DV / R;                                     // columns that the waves' outputs are joined by at a time
    constexpr int PER8 = KROW / 128;                               // 1 KB loads per 8 keys
    constexpr bool WIDE = !LATENT && DV >= 128;                    // V rows of whole bank lines
    constexpr int NVA = WIDE ? 8 : 4;                              // V addresses that are no immediates of each other
    static_assert(4 * ROWS * (CH + 4) * 4 <= 4 * TILE, "the join takes the tiles' place");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[4 * TILE];
    __shared__ PieceScratch scratch;
    __shared__ float sm_m[4][ROWS], sm_l[4][ROWS];             // of each wave
    __shared__ float factor[4][ROWS];                          // of a wave's output in the whole

    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g4 = lane >> 4;
    // neighbours on the line, which share keys, on one XCD (workgroups go to the eight in turn)
    const int worker = (p.workers & 7) ? (int)blockIdx.x : ((int)blockIdx.x & 7) * (p.workers >> 3) + ((int)blockIdx.x >> 3);

    Piece mine;
    if (!piece_of<ROWS, KT, 256>(p, worker, scratch, mine)) return;

    auto fk = [](int key) { return key & 7; };
    auto fv = [](int key) { return LATENT ? key & 7 : WIDE ? 2 * (key & 7) : key & 6; };
    unsigned char* const tile = lds + w * TILE;
    // reads of a tile: chunk 4 s + g4 of key r16; column chunk 2 j + h of the keys 4 g4 + (r16 / 4)
    uint32_t ka[2], va[NVA];
    const int vkey = 4 * g4 + (r16 >> 2);
#pragma unroll
    for (int i = 0; i < 2; ++i) ka[i] = r16 * KROW + (((4 * i + g4) ^ fk(r16)) << 4);
#pragma unroll
    for (int i = 0; i < NVA; ++i) va[i] = VBASE + vkey * VROW + (((2 * i + ((r16 >> 1) & 1)) ^ fv(vkey)) << 4) + (r16 & 1) * 8;
    // loads of a tile: lane's 16 bytes of each 1 KB of eight keys
    uint32_t offk[FP8 ? 1 : PER8], offv[FP8 || LATENT ? 1 : PER8];
    if constexpr (!FP8) {
#pragma unroll
        for (int m = 0; m < PER8; ++m) {
            const int chunk = 64 * m + lane, key = chunk / (KROW / 16), slot = chunk % (KROW / 16);
            offk[m] = key * KROW + ((slot ^ fk(key)) << 4);
            if constexpr (!LATENT) offv[m] = key * KROW + ((slot ^ fv(key)) << 4);
        }
    }
    constexpr int PARTS = DK / 16, KPL = 64 / PARTS, NLD = KT / KPL;       // fp8: 16 codes to a lane, keys per load
    uint4 sk[FP8 ? NLD : 1], sv[FP8 ? NLD : 1];

    Item it;
    while (next_item<ROWS, KT>(p, worker, mine, it)) {
        const Seq q = mine.q;
        const int kvh = it.kvh, rtile = it.rtile, nrows = q.n * p.group;

        // keys that all rows here see, and that some may
        const int i_first = rtile * ROWS / p.group, i_last = (min(rtile * ROWS + ROWS, nrows) - 1) / p.group;
        const int full = p.masks ? q.prior : q.prior + i_first + 1;
        const int some = q.ctx == 0 ? 0 : p.masks ? q.ctx : q.prior + i_last + 1;
        const float mul = p.mul * (FP8 ? p.k_scale[kvh] : 1.f);

        typedef const __attribute__((address_space(4))) int32_t* const_i32_ptr;
        const const_i32_ptr table = (const_i32_ptr)(p.block_table + (int64_t)mine.seq * p.block_table_stride);
        auto block_base = [&](int t, int half) -> int64_t {                // element index of the first of the 16 rows
            const int g = 2 * t + half;
            return place_of(p, table[entry_of(p, q, g)], kvh, g) * (BS * DK);
        };
        auto fetch_dma = [&](int t) __attribute__((always_inline)) {
            if constexpr (!FP8) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int64_t base = block_base(t, half) * 2;
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const char* kp = (const char*)p.k_pool + base + g * 8 * KROW;
                        const char* vp = (const char*)p.v_pool + base + g * 8 * KROW;
                        unsigned char* to = tile + (2 * half + g) * 8 * KROW;
#pragma unroll
                        for (int m_ = 0; m_ < PER8; ++m_) {
                            __builtin_amdgcn_global_load_lds(GLOBAL_PTR(kp + offk[m_]), LDS_PTR(to + 1024 * m_), 16, 0, 0);
                            if constexpr (!LATENT)
                                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(vp + offv[m_]), LDS_PTR(to + VBASE + 1024 * m_), 16, 0, 0);
                        }
                    }
                }
            }
        };
        auto fetch = [&](int t) __attribute__((always_inline)) {
            if constexpr (FP8) {
#pragma unroll
                for (int i = 0; i < NLD; ++i) {
                    const int64_t from = block_base(t, KPL * i / BS) + (KPL * i % BS) * DK;
                    sk[i] = *(const uint4*)((const char*)p.k_pool + from + lane * 16);
                    sv[i] = *(const uint4*)((const char*)p.v_pool + from + lane * 16);
                }
            }
        };
        auto stash = [&]() __attribute__((always_inline)) {
            if constexpr (FP8) {
#pragma unroll
                for (int i = 0; i < NLD; ++i) {
                    const int key = KPL * i + lane / PARTS, c = 2 * (lane % PARTS);
                    *(uint4*)(tile + key * KROW + ((c ^ fk(key)) << 4)) = E::from_fp8(make_uint2(sk[i].x, sk[i].y));
                    *(uint4*)(tile + key * KROW + (((c + 1) ^ fk(key)) << 4)) = E::from_fp8(make_uint2(sk[i].z, sk[i].w));
                    *(uint4*)(tile + VBASE + key * VROW + ((c ^ fv(key)) << 4)) = E::from_fp8(make_uint2(sv[i].x, sv[i].y));
                    *(uint4*)(tile + VBASE + key * VROW + (((c + 1) ^ fv(key)) << 4)) = E::from_fp8(make_uint2(sv[i].z, sv[i].w));
                }
            }
        };

        // the first tile is on its way while the rows are read
        int t = it.t0 + w;
        const int t_end = min(it.t1, (some + KT - 1) / KT);
        if (t < t_end) {
            if constexpr (FP8) fetch(t); else fetch_dma(t);
        }
        // rows of this lane's columns (beyond the last: that one, computed and not stored)
        uint4 qf[R][NS];
        int limit[R];
        const int64_t* words[R];
#pragma unroll
        for (int c = 0; c < R; ++c) {
            const int row = min(rtile * ROWS + 16 * c + r16, nrows - 1), i = row / p.group;
            limit[c] = q.prior + i + 1;
            words[c] = p.masks ? p.masks + (int64_t)(q.begin + i) * p.mask_words : nullptr;
            const uint16_t* src = (const uint16_t*)p.query + ((int64_t)(q.begin + i) * p.hq + kvh * p.group + row % p.group) * DK;
#pragma unroll
            for (int s = 0; s < NS; ++s) qf[c][s] = *(const uint4*)(src + 32 * s + 8 * g4);
        }
        float m[R], l[R];
        f32x4_t O[R][NJ];
#pragma unroll
        for (int c = 0; c < R; ++c) {
            m[c] = NEG_BIG; l[c] = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) O[c][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }

        for (; t < t_end; t += 4) {
            if constexpr (FP8) {
                stash();
                if (t + 4 < t_end) fetch(t + 4);
            } else {
                __builtin_amdgcn_s_waitcnt(0x0F70);                        // vmcnt(0)
                asm volatile("" ::: "memory");
            }
            const int start = t * KT;
            const bool masked = start + KT > full;                         // wave-uniform
            if (masked) {
                // A weight of 0 times a value that is not finite is not 0: such a value becomes 0, and its key not a number, and with
                // it the score of the rows that see it (of a latent row, key and value in one, what is left is the key's part).  Two
                // lanes to a key.
                constexpr uint32_t EXP = E::DT == AICOMP_KV_F16 ? 0x7c007c00u : 0x7f807f80u;
                constexpr uint32_t ONE = E::DT == AICOMP_KV_F16 ? 0x04000400u : 0x00800080u;
                unsigned char* const mine_v = tile + VBASE + (lane >> 1) * VROW + (lane & 1) * DV;
                uint32_t acc = 0;
#pragma unroll 4
                for (int i = 0; i < DV / 16; ++i) {
                    const uint4 x = *(const uint4*)(mine_v + 16 * i);
                    acc |= ((x.x & EXP) + ONE) | ((x.y & EXP) + ONE) | ((x.z & EXP) + ONE) | ((x.w & EXP) + ONE);
                }
                const uint64_t bad = __ballot((acc & 0x80008000u) != 0);
                if (bad && ((bad >> (lane & ~1)) & 3)) {
                    for (int i = 0; i < DV / 16; ++i) *(uint4*)(mine_v + 16 * i) = make_uint4(0, 0, 0, 0);
                    *(uint4*)(tile + (lane >> 1) * KROW + (LATENT ? 2 * DV : 0)) = make_uint4(~0u, ~0u, ~0u, ~0u);
                }
            }

            f32x4_t sa[2][R];
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int c = 0; c < R; ++c) sa[a][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            // operands are read AHEAD steps before their products (one at a time, a step takes an LDS read's whole latency: 2500 cycles
            // for the scores of a tile of latent rows, whose products take 600)
            constexpr int AHEAD = NS < 4 ? NS : 4;
            uint4 key[AHEAD + 1][2];
            auto keys_of = [&](int s, uint4* to) __attribute__((always_inline)) {
                to[0] = *(const uint4*)(tile + ka[s & 1] + (s >> 1) * 128);
                to[1] = *(const uint4*)(tile + ka[s & 1] + (s >> 1) * 128 + 16 * KROW);
            };
#pragma unroll
            for (int s = 0; s < AHEAD; ++s) keys_of(s, key[s]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                if (s + AHEAD < NS) keys_of(s + AHEAD, key[(s + AHEAD) % (AHEAD + 1)]);
#pragma unroll
                for (int c = 0; c < R; ++c) {
                    sa[0][c] = E::mfma(key[s % (AHEAD + 1)][0], qf[c][s], sa[0][c]);
                    sa[1][c] = E::mfma(key[s % (AHEAD + 1)][1], qf[c][s], sa[1][c]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            uint4 pf[R];
#pragma unroll
            for (int c = 0; c < R; ++c) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = sa[e >> 2][c][e & 3] * mul;
                if (masked) {
                    const uint32_t win = window_of(words[c], p.mask_words, start, q.prior, q.ctx, limit[c]) >> (4 * g4);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int key = 16 * (e >> 2) + (e & 3);           // + 4 g4
                        if (!((win >> key) & 1)) x[e] = -INFINITY;
                    }
                }
                float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
                mx = xor32_max(xor16_max(mx));
                if (__ballot(mx > m[c] + SLACK)) {                         // wave-uniform
                    const float m_new = fmaxf(m[c], mx), alpha = __builtin_amdgcn_exp2f(m[c] - m_new);
                    m[c] = m_new;
                    l[c] *= alpha;
#pragma unroll
                    for (int j = 0; j < NJ; ++j) O[c][j] *= alpha;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __builtin_amdgcn_exp2f(x[e] - m[c]);
                pf[c] = make_uint4(E::pack(x[0], x[1]), E::pack(x[2], x[3]), E::pack(x[4], x[5]), E::pack(x[6], x[7]));
                l[c] = E::pair_sum(pf[c].x, E::pair_sum(pf[c].y, E::pair_sum(pf[c].z, E::pair_sum(pf[c].w, l[c]))));
            }
            typedef short v4i16_t __attribute__((ext_vector_type(4)));
            typedef short v8i16_t __attribute__((ext_vector_type(8)));
            typedef __attribute__((address_space(3))) v4i16_t* lds_v4i16_ptr;
            constexpr int VAHEAD = 3;
            v8i16_t val[VAHEAD + 1];
            auto value_of = [&](int j) __attribute__((always_inline)) {
                const uint32_t o = va[j % NVA] + j / NVA * (32 * NVA);
                const v4i16_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(tile + o));
                const v4i16_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(tile + o + 16 * VROW));
                return v8i16_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
            };
#pragma unroll
            for (int j = 0; j < VAHEAD; ++j) val[j] = value_of(j);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                if (j + VAHEAD < NJ) val[(j + VAHEAD) % (VAHEAD + 1)] = value_of(j + VAHEAD);
#pragma unroll
                for (int c = 0; c < R; ++c) O[c][j] = E::mfma(__builtin_bit_cast(uint4, val[j % (VAHEAD + 1)]), pf[c], O[c][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (!FP8) {
                if (t + 4 < t_end) {
                    __builtin_amdgcn_s_waitcnt(0xC07F);                    // lgkmcnt(0): the tile has been read
                    fetch_dma(t + 4);
                }
            }
        }

        // The four waves' outputs joined, through the tiles' LDS.
#pragma unroll
        for (int c = 0; c < R; ++c) {
            l[c] += __shfl_xor(l[c], 16);
            l[c] += __shfl_xor(l[c], 32);
            if (g4 == 0) { sm_m[w][16 * c + r16] = m[c]; sm_l[w][16 * c + r16] = l[c]; }
        }
        float* const joint = (float*)lds;
#pragma unroll
        for (int ch = 0; ch < DV / CH; ++ch) {
            __syncthreads();                                               // (the tiles, or the columns before, have been read)
#pragma unroll
            for (int c = 0; c < R; ++c)
#pragma unroll
                for (int j = 0; j < CH / 16; ++j)
                    *(f32x4_t*)(joint + (w * ROWS + 16 * c + r16) * (CH + 4) + 16 * j + 4 * g4) = O[c][ch * (CH / 16) + j];
            if (ch == 0 && tid < ROWS) {
                float top = sm_m[0][tid], sum = 0.f;
#pragma unroll
                for (int k = 1; k < 4; ++k) top = fmaxf(top, sm_m[k][tid]);
#pragma unroll
                for (int k = 0; k < 4; ++k) sum = fmaf(__builtin_amdgcn_exp2f(sm_m[k][tid] - top), sm_l[k][tid], sum);
                // (sum 0: nothing was seen, and O is 0)
                const float inv = !it.whole ? 1.f : sum == 0.f ? 0.f : (FP8 ? p.v_scale[kvh] : 1.f) / sum;
#pragma unroll
                for (int k = 0; k < 4; ++k) factor[k][tid] = __builtin_amdgcn_exp2f(sm_m[k][tid] - top) * inv;
                if (!it.whole) p.ws_ml[it.slot * ROWS + tid] = make_float2(top, sum);
            }
            __syncthreads();
            // (not unrolled: a call of one tile runs this once, and waits for its instructions)
#pragma unroll 1
            for (int i = tid; i < ROWS * (CH / 4); i += 256) {
                const int r = i / (CH / 4), col = i % (CH / 4) * 4, row = rtile * ROWS + r;
                if (row >= nrows) break;
                f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < 4; ++k) o += *(const f32x4_t*)(joint + (k * ROWS + r) * (CH + 4) + col) * factor[k][r];
                if (!it.whole) {
                    *(f32x4_t*)(p.ws_acc + (it.slot * ROWS + r) * DV + ch * CH + col) = o;
                } else {
                    uint16_t* dst = (uint16_t*)p.out + ((int64_t)(q.begin + row / p.group) * p.hq + kvh * p.group + row % p.group) * DV;
                    *(uint2*)(dst + ch * CH + col) = make_uint2(E::pack(o[0], o[1]), E::pack(o[2], o[3]));
                }
            }
        }
        __syncthreads();
    }
}

// How a call is laid out: rows and keys of a tile, workgroups, key tiles that one has at least.
struct RowPlan {
    bool shared;                       // row_attn_shared.hip
    int R, rows, keys;
    int workers, least, over, row_tiles;
    bool single;
};

RowPlan row_plan(const RowAttnArgs& a) {
    const bool latent = a.dk == 576;
    const int group = a.hq / a.hkv;
    const int64_t rows = (int64_t)a.max_q_len * group;
    RowPlan r;
    r.shared = rows > (latent ? 16 : 32);
    // (two groups to a wave at head_dim 256 too, where they spill: row_attn_shared.hip; here over fp8 pools 17 registers, 32 trees of 4 .. 8
    // drafts, 8 KV heads of 4, over 512 .. 4096 tokens 93 us, 3.3 TB/s)
    r.R = r.shared ? (latent || rows <= 64 ? 1 : 2) : rows <= 16 ? 1 : 2;
    r.rows = (r.shared ? 64 : 16) * r.R;
    r.keys = r.shared ? 64 : 32;
    // (8 skewed sequences of 2055 .. 6511 latent rows, 48 rows each: two tiles at least 37 us, three 29, four 34; trees of 36 .. 49 drafts over
    // 500 tokens two 17.7, three 22)
    r.least = !r.shared ? 4 : latent ? 3 : 2;
    r.row_tiles = (int)((rows + r.rows - 1) / r.rows);
    int64_t span = (int64_t)a.max_blocks * a.bs;
    if (a.longest_context > 0) span = std::min<int64_t>(span, a.longest_context);
    // (rows in all bound the row tiles too, where one long sequence is among many short ones)
    const int64_t items = a.hkv * std::min<int64_t>((int64_t)a.num_seqs * r.row_tiles, a.rows * group / r.rows + a.num_seqs);
    // What an item's start and end cost, in key tiles, counts where workgroups have several items (64 rows of 512 .. 4096 tokens, 16 heads:
    // 60 us without, 55 with); where items are divided, as many workgroups as there are tiles for are worth more (one row of 700 tokens:
    // 17 us without, 21 with).  32 rows of 128 heads over 512 .. 4096 latent rows: 54 us with one tile's worth, 49.5 with three, 47.2 with six,
    // 49 with ten; trees of 16 .. 64 drafts over as many tokens 117 with three, 119 with one, 117 with six.
    const int64_t tiles = (span + r.keys - 1) / r.keys, most = latent || a.dk == 256 ? 256 : 512;
    const bool many = items * 4 >= most;
    r.over = many ? (!r.shared ? 8 : latent ? 6 : 3) : 0;
    r.least += r.over;
    r.workers = (int)std::min<int64_t>(most, (items * (tiles + r.over) + r.least - 1) / r.least);
    // An item whole for every workgroup saves the second launch and the division, and costs what the longest item takes alone.  Measured
    // at equal lengths, divided and whole: one row of 16 heads, 256 tokens 15.4 and 12.7 us, 512 15.9 and 15.4, 768 16.8 and 18.6; 128
    // heads, 1 x 256 tokens 17.3 and 14.8, 1 x 512 17.5 and 20.9, 64 x 512 37.7 and 25.9, 64 x 768 42.7 and 32.3; trees of 9 drafts for
    // 8 KV heads of 4, 1 x 192 tokens 12.5 and 7.7, 1 x 384 11.7 and 10.5; of 2 drafts, 1 x 768 10.9 and 9.4, 8 x 768 14.4 and 11.3.
    // Many items even out whatever their lengths are (400 x 1024 tokens: 128 heads 234 and 193 us, trees of 9 drafts 356 and 317).
    const int64_t all = (int64_t)a.num_seqs * a.hkv * r.row_tiles, few = r.shared ? 256 : latent ? 384 : 768;
    r.single = span <= (items >= 2 * most ? 1024 : many ? 768 : few) && all <= 2 * items;       // (few workgroups for no rows)
    if (r.single) r.over = 0, r.workers = (int)std::min<int64_t>(all, INT32_MAX);
    return r;
}

template <typename E, bool FP8, int DK, int DV, bool LATENT, int R, int OCC>
void launch_variant(const RowParams& p, int64_t join_items, hipStream_t stream) {
    hipLaunchKernelGGL((row_attn_kernel<E, FP8, DK, DV, LATENT, R, OCC>), dim3((unsigned)p.workers), dim3(256), 0, stream, p);
    if (p.ws_items != nullptr)
        hipLaunchKernelGGL((row_join_kernel<E, DV, 16 * R, KT>), dim3((unsigned)(join_items * (16 * R * DV / 1024))), dim3(256), 0, stream, p);
}

template <typename E, bool FP8> void launch_tree(const RowParams& p, const RowPlan& r, int d, int64_t items, hipStream_t stream) {
    if (d == 64) { if (r.R == 1) launch_variant<E, FP8, 64, 64, false, 1, 2>(p, items, stream); else launch_variant<E, FP8, 64, 64, false, 2, 2>(p, items, stream); }
    else if (d == 128) { if (r.R == 1) launch_variant<E, FP8, 128, 128, false, 1, 2>(p, items, stream); else launch_variant<E, FP8, 128, 128, false, 2, 2>(p, items, stream); }
    else { if (r.R == 1) launch_variant<E, FP8, 256, 256, false, 1, 1>(p, items, stream); else launch_variant<E, FP8, 256, 256, false, 2, 1>(p, items, stream); }
}

}  // namespace

// (the join's grid holds less than 2^32 threads; a workgroup's place in a launch and a row are 32 bits)
bool row_attn_mfma_supported(const RowAttnArgs& a) {
    if (a.bs < BS || (a.bs & (a.bs - 1)) != 0 || !is_16bit_float(a.q_dtype) || a.num_blocks > INT32_MAX) return false;
    const bool latent = a.dk == 576 && a.dv == 512 && a.v_row == 576 && a.hkv == 1;
    if (!latent && (a.dk != a.dv || (a.dk != 64 && a.dk != 128 && a.dk != 256))) return false;
    const int64_t rows = (int64_t)a.max_q_len * (a.hq / a.hkv), wgs = (rows + 127) * a.hkv * a.num_seqs / 2;
    if (rows > INT32_MAX / 2 || a.rows > INT32_MAX || wgs >= ((int64_t)1 << 24) || (int64_t)a.num_seqs * a.hkv >= ((int64_t)1 << 24)) return false;
    const RowPlan r = row_plan(a);                             // (the whole line, contexts as long as the table)
    return (int64_t)a.num_seqs * a.hkv * r.row_tiles < ((int64_t)1 << 24) &&
           (int64_t)a.num_seqs * a.hkv * r.row_tiles * (((int64_t)a.max_blocks * a.bs + r.keys - 1) / r.keys + r.over) < ((int64_t)1 << 30);
}

size_t row_attn_mfma_workspace_bytes(const RowAttnArgs& a) {
    const RowPlan r = row_plan(a);
    return r.workers > 1 && !r.single ? (size_t)2 * r.workers * r.rows * (a.dv + 2) * sizeof(float) + (size_t)a.num_seqs * a.hkv * r.row_tiles * sizeof(int2) : 0;
}

int launch_row_attn_mfma(const RowAttnArgs& a) {
    const RowPlan r = row_plan(a);
    RowParams p;
    p.out = a.out; p.query = a.query; p.k_pool = a.k_pool; p.v_pool = a.v_pool; p.block_table = a.block_table;
    p.block_table_stride = a.block_table_stride; p.context_lens = a.context_lens; p.cu_q_lens = a.cu_q_lens; p.masks = a.masks;
    p.mask_words = a.mask_words; p.num_seqs = a.num_seqs; p.rows = (int)a.rows; p.max_q_len = a.max_q_len; p.hq = a.hq; p.hkv = a.hkv;
    p.group = a.hq / a.hkv; p.span = a.max_blocks * a.bs; p.shift = __builtin_ctz(a.bs / BS); p.num_blocks = (int)a.num_blocks; p.mul = a.scale * LOG2E; p.k_scale = a.k_scale;
    p.v_scale = a.v_scale; p.workers = r.workers; p.single = r.single; p.least = r.least; p.over = r.over; p.row_tiles = r.row_tiles;
    p.ws_acc = (float*)a.workspace;
    p.ws_ml = (float2*)(p.ws_acc + (size_t)2 * r.workers * r.rows * a.dv);
    p.ws_items = r.workers > 1 && !r.single ? (int2*)(p.ws_ml + (size_t)2 * r.workers * r.rows) : nullptr;
    const int64_t items = (int64_t)a.num_seqs * a.hkv * r.row_tiles;
    const bool fp8 = a.kv_dtype == AICOMP_KV_FP8_E4M3, f16 = a.q_dtype == AICOMP_KV_F16;
    if (r.shared && a.dk == 576) launch_row_attn_latent(p, f16, items, a.stream);
    else if (r.shared) launch_row_attn_shared(p, f16, fp8, a.dk, r.R, items, a.stream);
    else if (a.dk == 576 && f16) launch_variant<F16Fmt, false, 576, 512, true, 1, 1>(p, items, a.stream);
    else if (a.dk == 576) launch_variant<Bf16Fmt, false, 576, 512, true, 1, 1>(p, items, a.stream);
    else if (f16) { if (fp8) launch_tree<F16Fmt, true>(p, r, a.dk, items, a.stream); else launch_tree<F16Fmt, false>(p, r, a.dk, items, a.stream); }
    else { if (fp8) launch_tree<Bf16Fmt, true>(p, r, a.dk, items, a.stream); else launch_tree<Bf16Fmt, false>(p, r, a.dk, items, a.stream); }
    AICOMP_HIP_LAUNCH_CHECK();
    return AICOMP_KV_OK;
}

}  // namespace aicomp
