// Attention of many query rows over cached rows (row_attn.h) on the matrix cores: trees of drafts whose rows are more than two groups
// of 16 to a KV head, over K and V pools of head_dim 64, 128 and 256; blocks of 16, 32, 64 .. tokens.
//
// Where row_attn_mfma.hip has every wave stream keys of its own for all rows of the workgroup, here the four waves have rows of
// their own, 16 R each, and share the tiles of 64 keys, which are brought into LDS while the tile before is computed: a key is
// read from memory once for 64 R rows.  The products, the references and the marking of values that are not finite are those of
// prompt_attn.hip; the division of the work is that of row_line.h.
//
// Bound by LDS, which gives every key and value to four waves (1024 cycles of a tile of 128 rows and head_dim 128, its products 1024 too),
// and by the partial outputs: 32 trees of 16 .. 64 drafts, 8 KV heads of 4, over 512 .. 4096 tokens 112 us, 456 TFLOP/s, of which the
// second launch 15 (without loads 82, loads alone 84); over fp8 pools 105; head_dim 64 70, and 68 over fp8.  One tree of 24 drafts over 700
// tokens: 11 us, of which the second launch 4.5.
//
// Two groups of rows to a wave at head_dim 256 are more than its registers hold: 17 of them go by way of memory, 45 over fp8 pools (2 at head_dim
// 128).  They are right all the same in 16 bits, where a key serves twice the rows: the 32 trees 276 us, with one group 347 (back to back
// over two sets of pools; over fp8 pools 295 and 276).
#include "row_line.h"

namespace aicomp {

namespace {

constexpr int KT = 64;                 // keys per tile
constexpr int NH = KT / 16;

template <bool FP8, int N> struct Stage { uint4 k[N], v[N]; };  // an fp8 tile on its way, 16 codes to a lane and load
template <int N> struct Stage<false, N> {};

// E: 16-bit format of queries and output; D: head_dim; R: groups of 16 rows to a wave; OCC: workgroups per CU
template <typename E, bool FP8, int D, int R, int OCC>
__global__ void __launch_bounds__(256, OCC)
row_attn_shared_kernel(RowParams p) {
    constexpr int ROWS = 64 * R;
    constexpr int ROW = 2 * D;                                 // bytes of a row in LDS
    constexpr int NS = D / 32, NJ = D / 16;
    constexpr int RPI = 1024 / ROW, NQ = 16 / RPI;             // rows per 1 KB load, loads per block
    __shared__ __attribute__((aligned(1024))) unsigned char k0[KT * ROW];
    __shared__ __attribute__((aligned(1024))) unsigned char v0[KT * ROW];
    __shared__ __attribute__((aligned(1024))) unsigned char k1[KT * ROW];
    __shared__ __attribute__((aligned(1024))) unsigned char v1[KT * ROW];
    __shared__ PieceScratch scratch;

    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g4 = lane >> 4;
    // neighbours on the line, which share keys, on one XCD (workgroups go to the eight in turn)
    const int worker = (p.workers & 7) ? (int)blockIdx.x : ((int)blockIdx.x & 7) * (p.workers >> 3) + ((int)blockIdx.x >> 3);

    Piece mine;
    if (!piece_of<ROWS, KT, 256>(p, worker, scratch, mine)) return;

    // chunk c (16 bytes) of key k lies at c ^ f(k) (row_attn_mfma.hip)
    auto fk = [](int key) { return key & 7; };
    auto fv = [](int key) { return D >= 128 ? 2 * (key & 7) : key & 6; };
    const int vkey = 4 * g4 + (r16 >> 2);
    uint32_t offk[NQ], offv[NQ];                               // lane's 16 bytes of each 1 KB of a block
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int key = RPI * i + lane / (ROW / 16), c = lane % (ROW / 16);
        offk[i] = key * ROW + ((c ^ fk(key)) << 4);
        offv[i] = key * ROW + ((c ^ fv(key)) << 4);
    }
    constexpr int PARTS = D / 16, KPL = 64 / PARTS, NLD = 16 / KPL;        // fp8: lanes to a row, rows per load, loads of a wave's block

    Item it;
    while (next_item<ROWS, KT>(p, worker, mine, it)) {
        const Seq q = mine.q;
        const int kvh = it.kvh, rtile = it.rtile, t0 = it.t0;
        const int nrows = q.n * p.group, row0 = rtile * ROWS + 16 * R * w;             // of this wave

        // rows of this lane's columns (beyond the last: that one, computed and not stored)
        uint4 qf[R][NS];
        int limit[R];
        const int64_t* words[R];
#pragma unroll
        for (int c = 0; c < R; ++c) {
            const int row = min(row0 + 16 * c + r16, nrows - 1), i = row / p.group;
            limit[c] = q.prior + i + 1;
            words[c] = p.masks ? p.masks + (int64_t)(q.begin + i) * p.mask_words : nullptr;
            const uint16_t* src = (const uint16_t*)p.query + ((int64_t)(q.begin + i) * p.hq + kvh * p.group + row % p.group) * D;
#pragma unroll
            for (int s = 0; s < NS; ++s) qf[c][s] = *(const uint4*)(src + 32 * s + 8 * g4);
        }
        const int full = p.masks ? q.prior : q.prior + rtile * ROWS / p.group + 1;     // keys that all rows here see
        const int some = row0 >= nrows ? 0 : q.ctx;                                    // (a wave without rows only brings keys in)
        const float mul = p.mul * (FP8 ? p.k_scale[kvh] : 1.f);

        float m[R], l[R];
        f32x4_t O[R][NJ];
#pragma unroll
        for (int c = 0; c < R; ++c) {
            m[c] = NEG_BIG; l[c] = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) O[c][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }

        typedef const __attribute__((address_space(4))) int32_t* const_i32_ptr;
        const const_i32_ptr table = (const_i32_ptr)(p.block_table + (int64_t)mine.seq * p.block_table_stride);
        // wave w brings in block w of a tile
        auto block_base = [&](int t) -> int64_t {              // element index of its first row
            const int g = 4 * t + w;
            return place_of(p, table[entry_of(p, q, g)], kvh, g) * (BS * D);
        };
        auto fetch_dma = [&](int t, unsigned char* kb, unsigned char* vb) __attribute__((always_inline)) {
            const int64_t base = block_base(t) * 2;
            const char* ka = (const char*)p.k_pool + base;
            const char* va = (const char*)p.v_pool + base;
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(ka + offk[i]), LDS_PTR(kb + 16 * w * ROW + 1024 * i), 16, 0, 0);
                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(va + offv[i]), LDS_PTR(vb + 16 * w * ROW + 1024 * i), 16, 0, 0);
            }
        };
        Stage<FP8, NLD> st;
        auto fetch = [&](int t) __attribute__((always_inline)) {
            if constexpr (FP8) {
                const int64_t base = block_base(t) + lane * 16;
#pragma unroll
                for (int i = 0; i < NLD; ++i) {
                    st.k[i] = *(const uint4*)((const char*)p.k_pool + base + 1024 * i);
                    st.v[i] = *(const uint4*)((const char*)p.v_pool + base + 1024 * i);
                }
            }
        };
        auto stash = [&](unsigned char* kb, unsigned char* vb) __attribute__((always_inline)) {
            if constexpr (FP8) {
#pragma unroll
                for (int i = 0; i < NLD; ++i) {
                    const int key = 16 * w + KPL * i + lane / PARTS, c = 2 * (lane % PARTS);
                    *(uint4*)(kb + key * ROW + ((c ^ fk(key)) << 4)) = E::from_fp8(make_uint2(st.k[i].x, st.k[i].y));
                    *(uint4*)(kb + key * ROW + (((c + 1) ^ fk(key)) << 4)) = E::from_fp8(make_uint2(st.k[i].z, st.k[i].w));
                    *(uint4*)(vb + key * ROW + ((c ^ fv(key)) << 4)) = E::from_fp8(make_uint2(st.v[i].x, st.v[i].y));
                    *(uint4*)(vb + key * ROW + (((c + 1) ^ fv(key)) << 4)) = E::from_fp8(make_uint2(st.v[i].z, st.v[i].w));
                }
            }
        };
        // Values that are not finite become 0 and their keys not a number (prompt_attn.hip), in tiles that not all rows see whole: by the
        // wave that brought them in, before any other reads them.  Four lanes to a key.
        auto clean = [&](unsigned char* kb, unsigned char* vb) __attribute__((always_inline)) {
            constexpr uint32_t EXP = E::DT == AICOMP_KV_F16 ? 0x7c007c00u : 0x7f807f80u;
            constexpr uint32_t ONE = E::DT == AICOMP_KV_F16 ? 0x04000400u : 0x00800080u;
            const int k = 16 * w + (lane >> 2);
            uint4* const here = (uint4*)(vb + k * ROW + (lane & 3) * (D / 2));
            uint32_t acc = 0;
#pragma unroll 4
            for (int i = 0; i < D / 32; ++i) {
                const uint4 x = here[i];
                acc |= ((x.x & EXP) + ONE) | ((x.y & EXP) + ONE) | ((x.z & EXP) + ONE) | ((x.w & EXP) + ONE);
            }
            const uint64_t bad = __ballot((acc & 0x80008000u) != 0);
            if ((bad >> (lane & ~3)) & 15) {
                for (int i = 0; i < D / 32; ++i) here[i] = make_uint4(0, 0, 0, 0);
                *(uint4*)(kb + k * ROW) = make_uint4(~0u, ~0u, ~0u, ~0u);
            }
        };

        auto compute = [&](int t, const unsigned char* kb, const unsigned char* vb) __attribute__((always_inline)) {
            const int start = t * KT;
            if (start >= some) return;                         // wave-uniform
            const bool masked = start + KT > full;
            f32x4_t sa[NH][R];
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int c = 0; c < R; ++c) sa[h][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            // operands are read a step before their products (the order is kept by the barriers)
            uint4 a[2][NH];
            auto keys_of = [&](int s, uint4* to) __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < NH; ++h) to[h] = *(const uint4*)(kb + (16 * h + r16) * ROW + (((4 * s + g4) ^ fk(r16)) << 4));
            };
            keys_of(0, a[0]);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                if (s + 1 < NS) keys_of(s + 1, a[(s + 1) & 1]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int h = 0; h < NH; ++h)
#pragma unroll
                    for (int c = 0; c < R; ++c) sa[h][c] = E::mfma(a[s & 1][h], qf[c][s], sa[h][c]);
                __builtin_amdgcn_sched_barrier(0);
            }
            uint4 pf[R][NH / 2];
#pragma unroll
            for (int c = 0; c < R; ++c) {
                float x[4 * NH];
#pragma unroll
                for (int e = 0; e < 4 * NH; ++e) x[e] = sa[e >> 2][c][e & 3] * mul;
                if (masked) {
#pragma unroll
                    for (int hp = 0; hp < NH / 2; ++hp) {
                        const uint32_t win = window_of(words[c], p.mask_words, start + 32 * hp, q.prior, q.ctx, limit[c]) >> (4 * g4);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (!((win >> (16 * (e >> 2) + (e & 3))) & 1)) x[8 * hp + e] = -INFINITY;
                    }
                }
                float mx = x[0];
#pragma unroll
                for (int e = 1; e < 4 * NH; ++e) mx = fmaxf(mx, x[e]);
                mx = xor32_max(xor16_max(mx));
                if (__ballot(mx > m[c] + SLACK)) {             // wave-uniform
                    const float m_new = fmaxf(m[c], mx), alpha = __builtin_amdgcn_exp2f(m[c] - m_new);
                    m[c] = m_new;
                    l[c] *= alpha;
#pragma unroll
                    for (int j = 0; j < NJ; ++j) O[c][j] *= alpha;
                }
#pragma unroll
                for (int e = 0; e < 4 * NH; ++e) x[e] = __builtin_amdgcn_exp2f(x[e] - m[c]);
#pragma unroll
                for (int hp = 0; hp < NH / 2; ++hp) {
                    pf[c][hp] = make_uint4(E::pack(x[8 * hp], x[8 * hp + 1]), E::pack(x[8 * hp + 2], x[8 * hp + 3]),
                                           E::pack(x[8 * hp + 4], x[8 * hp + 5]), E::pack(x[8 * hp + 6], x[8 * hp + 7]));
                    l[c] = E::pair_sum(pf[c][hp].x, E::pair_sum(pf[c][hp].y, E::pair_sum(pf[c][hp].z, E::pair_sum(pf[c][hp].w, l[c]))));
                }
            }
            typedef short v4i16_t __attribute__((ext_vector_type(4)));
            typedef short v8i16_t __attribute__((ext_vector_type(8)));
            typedef __attribute__((address_space(3))) v4i16_t* lds_v4i16_ptr;
            constexpr int VAHEAD = FP8 ? 2 : 4;
            v8i16_t val[VAHEAD + 1];
            auto value_of = [&](int u) __attribute__((always_inline)) {            // 16 columns of 32 keys
                const int j = u >> 1, hp = u & 1;
                const int o = (32 * hp + vkey) * ROW + (((2 * j + ((r16 >> 1) & 1)) ^ fv(vkey)) << 4) + (r16 & 1) * 8;
                const v4i16_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(vb + o));
                const v4i16_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(vb + o + 16 * ROW));
                return v8i16_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
            };
#pragma unroll
            for (int u = 0; u < VAHEAD; ++u) val[u] = value_of(u);
#pragma unroll
            for (int u = 0; u < 2 * NJ; ++u) {
                if (u + VAHEAD < 2 * NJ) val[(u + VAHEAD) % (VAHEAD + 1)] = value_of(u + VAHEAD);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int c = 0; c < R; ++c) O[c][u >> 1] = E::mfma(__builtin_bit_cast(uint4, val[u % (VAHEAD + 1)]), pf[c][u & 1], O[c][u >> 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };

        // Opens the step of tile t: it is in LDS afterwards for every wave, and the next one is on its way.
        const int t_end = min(it.t1, (q.ctx + KT - 1) / KT);      // (0 tiles where the context is none)
        auto open = [&](int t, unsigned char* kb, unsigned char* vb, unsigned char* kn, unsigned char* vn) __attribute__((always_inline)) {
            if constexpr (FP8) {
                stash(kb, vb);                                 // (nobody reads this pair: its readers met at the tile between)
                if (t * KT + KT > full) clean(kb, vb);         // workgroup-uniform
                __syncthreads();
                fetch(max(t - 1, t0));
            } else {
                __builtin_amdgcn_s_waitcnt(0x0F70);            // vmcnt(0): this wave's part of the tile
                if (t * KT + KT > full) clean(kb, vb);
                __syncthreads();                               // also: the tile before is no longer read by anyone
                if (t > t0) fetch_dma(t - 1, kn, vn);
            }
        };
        if (t0 < t_end) {
            if constexpr (FP8) fetch(t_end - 1); else fetch_dma(t_end - 1, k0, v0);
        }
        for (int t = t_end - 1; t >= t0; t -= 2) {
            open(t, k0, v0, k1, v1);
            compute(t, k0, v0);
            if (t > t0) {
                open(t - 1, k1, v1, k0, v0);
                compute(t - 1, k1, v1);
            }
        }
        __syncthreads();                                       // (the buffers are free for the next item)

#pragma unroll
        for (int c = 0; c < R; ++c) {
            l[c] += __shfl_xor(l[c], 16);
            l[c] += __shfl_xor(l[c], 32);
            const int r = 16 * R * w + 16 * c + r16, row = rtile * ROWS + r;
            if (row >= nrows) continue;
            if (!it.whole) {
                if (g4 == 0) p.ws_ml[it.slot * ROWS + r] = make_float2(m[c], l[c]);
                float* dst = p.ws_acc + (it.slot * ROWS + r) * D + 4 * g4;
#pragma unroll
                for (int j = 0; j < NJ; ++j) *(f32x4_t*)(dst + 16 * j) = O[c][j];
            } else {
                const bool none = l[c] == 0.f;
                const float inv = (FP8 ? p.v_scale[kvh] : 1.f) / l[c];
                uint16_t* dst = (uint16_t*)p.out + ((int64_t)(q.begin + row / p.group) * p.hq + kvh * p.group + row % p.group) * D + 4 * g4;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    *(uint2*)(dst + 16 * j) = none ? make_uint2(0, 0) : make_uint2(E::pack(O[c][j][0] * inv, O[c][j][1] * inv),
                                                                                   E::pack(O[c][j][2] * inv, O[c][j][3] * inv));
            }
        }
    }
}

template <typename E, bool FP8, int D, int R, int OCC>
void launch_variant(const RowParams& p, int64_t join_items, hipStream_t stream) {
    hipLaunchKernelGGL((row_attn_shared_kernel<E, FP8, D, R, OCC>), dim3((unsigned)p.workers), dim3(256), 0, stream, p);
    if (p.ws_items != nullptr)
        hipLaunchKernelGGL((row_join_kernel<E, D, 64 * R, KT>), dim3((unsigned)(join_items * (64 * R * D / 1024))), dim3(256), 0, stream, p);
}

template <typename E, bool FP8> void launch_dim(const RowParams& p, int d, int R, int64_t items, hipStream_t stream) {
    if (d == 64) { if (R == 1) launch_variant<E, FP8, 64, 1, 2>(p, items, stream); else launch_variant<E, FP8, 64, 2, 2>(p, items, stream); }
    else if (d == 128) { if (R == 1) launch_variant<E, FP8, 128, 1, 2>(p, items, stream); else launch_variant<E, FP8, 128, 2, 2>(p, items, stream); }
    else { if (R == 1) launch_variant<E, FP8, 256, 1, 1>(p, items, stream); else launch_variant<E, FP8, 256, 2, 1>(p, items, stream); }
}

}  // namespace

void launch_row_attn_shared(const RowParams& p, bool f16, bool fp8, int d, int R, int64_t items, hipStream_t stream) {
    if (f16) { if (fp8) launch_dim<F16Fmt, true>(p, d, R, items, stream); else launch_dim<F16Fmt, false>(p, d, R, items, stream); }
    else { if (fp8) launch_dim<Bf16Fmt, true>(p, d, R, items, stream); else launch_dim<Bf16Fmt, false>(p, d, R, items, stream); }
}

}  // namespace aicomp
