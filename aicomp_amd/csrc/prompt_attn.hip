// Causal attention of prompts over expanded latent rows on the matrix cores: 16 bits, keys of 128 elements of a head and 64 that all
// heads share, values of 128.
//
// A workgroup has 128 queries of a head (64 in small calls), 32 (16) to a wave, and walks the keys in tiles of 64, from the nearest to the
// farthest, each brought straight into LDS while the one before is computed:
//   S^T = K Q^T      six steps of 32 elements, two of them over the shared part; a lane then has four keys of a query per 16
//   O^T += V^T P^T   weights from registers in that order, V^T out of LDS by transposing reads
// Two tiles of 40 KB are 80 KB, so that two workgroups share a CU and one's products run beside the other's exponentials.
// The reference of a query moves when a score passes it by 2^8 (row_attn_mfma.hip).
//
// Bound by the matrix cores: 8192 tokens of 16 heads 321 us, 1.07 PFLOP/s of the 1.27 that a large library product of the card reaches; 12
// prompts of 37 .. 1500 tokens behind 0 .. 2048, 16 heads, 203 us, 0.80 PFLOP/s (tiles that are partly masked, queries beyond the last).
#include "row_attn.h"

#include <algorithm>
#include <atomic>

namespace aicomp {

namespace {

constexpr int NOPE = 128, ROPE = 64, DV = 128;
constexpr int KT = 64;                 // keys per tile
constexpr int NS = (NOPE + ROPE) / 32, NJ = DV / 16, NH = KT / 16;
constexpr float NEG_BIG = -0x1.fffffep127f, SLACK = 8.f;         // (no score is below: the first that a row sees moves its reference)
constexpr float FAR = 0x1p26f;         // a reference beyond which its own rounding, 2^2 there, is no longer small beside SLACK

#define GLOBAL_PTR(p) ((const __attribute__((address_space(1))) void*)(p))
#define LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

struct PromptParams {
    void* out;
    const void* query;
    const char* key; const char* rope_key; const char* value;
    int64_t key_hs, value_hs;          // bytes
    uint32_t key_ts, rope_ts, value_ts;
    const int32_t* cu_q_lens;
    const int32_t* cu_k_lens;
    int heads, rows, keys;
    float mul;                         // |scale| log2(e), or 1 where the scale is 0
    uint32_t flip, keep;               // queries: sign bits to turn, bits to keep
    int num_cus;
};

// R: groups of 16 queries per wave
template <typename E, int R>
__global__ void __launch_bounds__(256, 2)
prompt_attn_kernel(PromptParams p) {
    constexpr int ROWS = 64 * R;
    __shared__ __attribute__((aligned(1024))) unsigned char k0[KT * 2 * NOPE];
    __shared__ __attribute__((aligned(1024))) unsigned char r0[KT * 2 * ROPE];
    __shared__ __attribute__((aligned(1024))) unsigned char v0[KT * 2 * DV];
    __shared__ __attribute__((aligned(1024))) unsigned char k1[KT * 2 * NOPE];
    __shared__ __attribute__((aligned(1024))) unsigned char r1[KT * 2 * ROPE];
    __shared__ __attribute__((aligned(1024))) unsigned char v1[KT * 2 * DV];

    const int head = blockIdx.x;
    int seq = blockIdx.y, qtile = prefill_tile_of_slice(blockIdx.z, gridDim.z, p.num_cus, gridDim.x * gridDim.y);
    const int tid = threadIdx.x, lane = tid & 63;
    // Ragged prompts: a tile costs the keys that its last query sees, which differ several-fold, and workgroups start in the order of
    // the grid.  So the one in place i takes the tile of rank i, the dearest first.  Every workgroup finds it for itself: a tile's rank
    // is how many tiles of each sequence are dearer, which follows from the sequence's lengths.  (12 prompts of 37 .. 1500 behind 0 ..
    // 2048, 16 heads: 254 us in the order of the grid, 223 so; 16 of 37 .. 300 behind 0 .. 300, 64 heads, 88 and 91.)  The table and the
    // tests are of 16 sequences.  More would gain as much (measured in a copy, 17 of 37 .. 1500: 316 and 287; 40 of 37 .. 700: 395 and 317;
    // 64 of 37 .. 124: 153 and 135) and take the order of the grid so far.
    const int nseq = gridDim.y, ntile = gridDim.z;
    if (nseq > 1 && nseq <= 16 && nseq * ntile <= 512) {                   // grid-uniform
        int* const tab = (int*)k0;                                         // [nseq][3]: context, prior, tiles; then the one found
        if (tid < nseq) {
            const int n = max(0, min(p.cu_q_lens[tid + 1], p.rows) - max(0, p.cu_q_lens[tid]));
            const int ctx = min(p.cu_k_lens[tid + 1], p.keys) - max(0, p.cu_k_lens[tid]);
            tab[3 * tid] = ctx;
            tab[3 * tid + 1] = ctx - n;
            tab[3 * tid + 2] = min(ntile, (n + ROWS - 1) / ROWS);
        }
        if (tid == 0) tab[48] = -1;
        __syncthreads();
        // tiles of a sequence that cost more than c
        auto dearer = [&](int s, int c) {
            const int ctx = tab[3 * s], prior = tab[3 * s + 1], tiles = tab[3 * s + 2];
            return ctx <= c ? 0 : max(0, tiles - (c < prior ? 0 : (c - prior) / ROWS));
        };
        const int place = blockIdx.y + nseq * blockIdx.z;
        for (int i = tid; i < nseq * ntile; i += 256) {
            const int s = i / ntile, t = i - s * ntile;
            if (t >= tab[3 * s + 2]) continue;
            const int c = min(tab[3 * s], tab[3 * s + 1] + (t + 1) * ROWS);
            int rank = 0;
            for (int o = 0; o < nseq; ++o) rank += o < s ? dearer(o, c - 1) : dearer(o, c);       // (of equal ones, the first sequence's)
            if (rank == place) { tab[48] = s; tab[49] = t; }
        }
        __syncthreads();
        seq = __builtin_amdgcn_readfirstlane(tab[48]);
        qtile = __builtin_amdgcn_readfirstlane(tab[49]);
        if (seq < 0) return;                                               // (more places than tiles)
        __syncthreads();
    }
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g4 = lane >> 4;
    const int q_begin = max(0, p.cu_q_lens[seq]), n = min(p.cu_q_lens[seq + 1], p.rows) - q_begin;
    const int k_begin = max(0, p.cu_k_lens[seq]), ctx = min(p.cu_k_lens[seq + 1], p.keys) - k_begin;
    const int prior = ctx - n, first = qtile * ROWS;               // position of the tile's first query, less `prior`
    if (first >= n) return;
    uint16_t* const out = (uint16_t*)p.out + ((int64_t)q_begin * p.heads + head) * DV;
    if (prior < 0) {                                               // more queries than keys: zero rows
        for (int i = tid; i < ROWS * (DV / 8); i += 256) {
            const int row = first + i / (DV / 8);
            if (row < n) *(uint4*)(out + (int64_t)row * p.heads * DV + 8 * (i % (DV / 8))) = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    const int row0 = first + 16 * R * w;                           // of this wave
    const int kv_end = min(ctx, prior + first + ROWS);             // keys that some query here sees
    const int wave_end = row0 >= n ? 0 : min(ctx, prior + row0 + 16 * R), wave_full = prior + row0 + 1;

    uint4 qf[R][NS];
    int pos[R];
#pragma unroll
    for (int c = 0; c < R; ++c) {
        const int row = min(row0 + 16 * c + r16, n - 1);           // (beyond the last: that one, computed and not stored)
        pos[c] = prior + row;
        const uint16_t* src = (const uint16_t*)p.query + ((int64_t)(q_begin + row) * p.heads + head) * (NOPE + ROPE);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            uint4 x = *(const uint4*)(src + 32 * s + 8 * g4);
            x.x = (x.x & p.keep) ^ p.flip; x.y = (x.y & p.keep) ^ p.flip; x.z = (x.z & p.keep) ^ p.flip; x.w = (x.w & p.keep) ^ p.flip;
            qf[c][s] = x;
        }
    }
    float m[R], l[R];
    f32x4_t O[R][NJ];
    uint32_t far = 0;                                              // bit c: some reference of group c is beyond FAR
#pragma unroll
    for (int c = 0; c < R; ++c) {
        m[c] = NEG_BIG; l[c] = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) O[c][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    // Chunk c (16 bytes) of key k lies at c ^ f(k): keys of eight lanes that read together, and the key quads of a transposing read,
    // then spread over the banks.
    auto fk = [](int key) { return key & 7; };
    auto fv = [](int key) { return 2 * (key & 7); };
    const char* const key = p.key + (int64_t)k_begin * p.key_ts + head * p.key_hs;
    const char* const rope = p.rope_key + (int64_t)k_begin * p.rope_ts;
    const char* const value = p.value + (int64_t)k_begin * p.value_ts + head * p.value_hs;
    // Wave w brings in keys 16 w .. 16 w + 15 of a tile.  Whole tiles: uniform bases and 32-bit offsets of the lane's row and chunk.
    uint32_t ok = (lane >> 4) * p.key_ts + (((lane & 15) ^ fk(lane >> 4)) << 4);
    uint32_t ov[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) ov[i] = (lane >> 4) * p.value_ts + (((lane & 15) ^ fv(4 * i + (lane >> 4))) << 4);
    const uint32_t orp = (lane >> 3) * p.rope_ts + (((lane & 7) ^ fk(lane >> 3)) << 4);
    const uint32_t ok1 = (lane >> 4) * p.key_ts + (((lane & 15) ^ fk(4 + (lane >> 4))) << 4);
    auto fetch = [&](int t, unsigned char* kb, unsigned char* rb, unsigned char* vb) __attribute__((always_inline)) {
        const int base = KT * t + 16 * w, last = ctx - 1 - base;
        const char* ka = key + (int64_t)base * p.key_ts;
        const char* ra = rope + (int64_t)base * p.rope_ts;
        const char* va = value + (int64_t)base * p.value_ts;
        if (last >= 15) {                                          // wave-uniform
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(ka + 4 * i * (int64_t)p.key_ts + (i & 1 ? ok1 : ok)),
                                                 LDS_PTR(kb + (16 * w + 4 * i) * 2 * NOPE), 16, 0, 0);
                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(va + 4 * i * (int64_t)p.value_ts + ov[i & 1]),
                                                 LDS_PTR(vb + (16 * w + 4 * i) * 2 * DV), 16, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(ra + 8 * i * (int64_t)p.rope_ts + orp),
                                                 LDS_PTR(rb + (16 * w + 8 * i) * 2 * ROPE), 16, 0, 0);
        } else {
            // keys beyond the last one, which are masked, take its row
            int x = lane;
            asm volatile("" : "+v"(x));                            // (nothing of this in registers across the loop)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = 4 * i + (x >> 4), from = min(k, last), c = x & 15;
                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(ka + (from * (int64_t)p.key_ts + ((c ^ fk(k)) << 4))),
                                                 LDS_PTR(kb + (16 * w + 4 * i) * 2 * NOPE), 16, 0, 0);
                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(va + (from * (int64_t)p.value_ts + ((c ^ fv(k)) << 4))),
                                                 LDS_PTR(vb + (16 * w + 4 * i) * 2 * DV), 16, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int k = 8 * i + (x >> 3), from = min(k, last), c = x & 7;
                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(ra + (from * (int64_t)p.rope_ts + ((c ^ fk(k)) << 4))),
                                                 LDS_PTR(rb + (16 * w + 8 * i) * 2 * ROPE), 16, 0, 0);
            }
        }
    };

    const int vkey = 4 * g4 + (r16 >> 2);
    auto compute = [&](int t, const unsigned char* kb, const unsigned char* rb, const unsigned char* vb) __attribute__((always_inline)) {
        const int start = t * KT;
        if (start >= wave_end) return;                             // wave-uniform
        const bool masked = start + KT > wave_full;
        f32x4_t sa[NH][R];
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int c = 0; c < R; ++c) sa[h][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        // operands are read a step before their products (the order is kept by the barriers)
        uint4 a[2][NH];
        auto keys_of = [&](int s, uint4* to) __attribute__((always_inline)) {
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                const int k = 16 * h + r16;
                to[h] = s < NOPE / 32 ? *(const uint4*)(kb + k * 2 * NOPE + (((4 * s + g4) ^ fk(r16)) << 4))
                                      : *(const uint4*)(rb + k * 2 * ROPE + (((4 * (s - NOPE / 32) + g4) ^ fk(r16)) << 4));
            }
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
            for (int e = 0; e < 4 * NH; ++e) x[e] = sa[e >> 2][c][e & 3];
            if (masked) {
                const int seen = pos[c] - start - 4 * g4;          // keys 16 (e / 4) + e % 4 up to that
#pragma unroll
                for (int e = 0; e < 4 * NH; ++e) {
                    const int k = 16 * (e >> 2) + (e & 3);
                    if (k > seen) x[e] = -INFINITY;
                }
            }
            float mx = x[0];
#pragma unroll
            for (int e = 1; e < 4 * NH; ++e) mx = fmaxf(mx, x[e]);
            mx = xor32_max(xor16_max(mx)) * p.mul;
            if (__ballot(mx > m[c] + SLACK)) {                     // wave-uniform
                const float m_new = fmaxf(m[c], mx), alpha = __builtin_amdgcn_exp2f(m[c] - m_new);
                m[c] = m_new;
                if (__ballot(fabsf(m_new) > FAR && m_new > NEG_BIG)) far |= 1u << c;
                l[c] *= alpha;
#pragma unroll
                for (int j = 0; j < NJ; ++j) O[c][j] *= alpha;
            }
            // The reference is a rounded product: against the exact ones of an fma, all weights of a row are off by its rounding.  Where that
            // would leave the range of 16 bits, the products are rounded too.
            float factor = p.mul, ref = m[c];
            if (far >> c & 1) {                                    // wave-uniform
#pragma clang fp contract(off)
                const bool mine = fabsf(m[c]) > FAR;               // (by row: another one keeps what it has in its other tiles)
#pragma unroll
                for (int e = 0; e < 4 * NH; ++e) {
                    const float s = x[e] * p.mul;
                    x[e] = mine ? s - m[c] : x[e];
                }
                factor = mine ? 1.f : p.mul;
                ref = mine ? 0.f : m[c];
            }
#pragma unroll
            for (int e = 0; e < 4 * NH; ++e) x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], factor, -ref));
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
        constexpr int VAHEAD = 5;
        v8i16_t val[VAHEAD + 1];
        auto value_of = [&](int u) __attribute__((always_inline)) {            // 16 columns of 32 keys
            const int j = u >> 1, hp = u & 1;
            const int o = (32 * hp + vkey) * 2 * DV + (((2 * j + ((r16 >> 1) & 1)) ^ fv(vkey)) << 4) + (r16 & 1) * 8;
            const v4i16_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(vb + o));
            const v4i16_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(vb + o + 16 * 2 * DV));
            return v8i16_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        };
#pragma unroll
        for (int u = 0; u < VAHEAD; ++u) val[u] = value_of(u);
        __builtin_amdgcn_s_setprio(2);                             // (before the other wave's softmax: 8192 tokens 333 and 321 us)
#pragma unroll
        for (int u = 0; u < 2 * NJ; ++u) {
            if (u + VAHEAD < 2 * NJ) val[(u + VAHEAD) % (VAHEAD + 1)] = value_of(u + VAHEAD);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < R; ++c) O[c][u >> 1] = E::mfma(__builtin_bit_cast(uint4, val[u % (VAHEAD + 1)]), pf[c][u & 1], O[c][u >> 1]);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
    };

    // A weight of 0 times a value that is not finite is not 0.  In tiles that not all queries here see whole, a wave looks through the
    // values that it brought in itself, before any other wave reads them: such a value becomes 0, and its key not a number, and with it
    // the score of the queries that see it.  Four lanes to a key.
    auto clean = [&](unsigned char* kb, unsigned char* vb) __attribute__((always_inline)) {
        constexpr uint32_t EXP = E::DT == AICOMP_KV_F16 ? 0x7c007c00u : 0x7f807f80u;
        constexpr uint32_t ONE = E::DT == AICOMP_KV_F16 ? 0x04000400u : 0x00800080u;
        const int k = 16 * w + (lane >> 2);
        uint4* const mine = (uint4*)(vb + k * 2 * DV + (lane & 3) * (DV / 2));
        uint32_t acc = 0;
#pragma unroll
        for (int i = 0; i < DV / 32; ++i) {
            const uint4 x = mine[i];
            acc |= ((x.x & EXP) + ONE) | ((x.y & EXP) + ONE) | ((x.z & EXP) + ONE) | ((x.w & EXP) + ONE);
        }
        const uint64_t bad = __ballot((acc & 0x80008000u) != 0);
        if ((bad >> (lane & ~3)) & 15) {
#pragma unroll
            for (int i = 0; i < DV / 32; ++i) mine[i] = make_uint4(0, 0, 0, 0);
            *(uint4*)(kb + k * 2 * NOPE) = make_uint4(~0u, ~0u, ~0u, ~0u);
        }
    };
    // Opens the step of tile t: it is in LDS afterwards for every wave, and the next one is on its way into the other buffers.
    auto open = [&](int t, unsigned char* kb, unsigned char* vb, unsigned char* kn, unsigned char* rn, unsigned char* vn)
        __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0x0F70);                        // vmcnt(0): this wave's part of the tile
        if (t * KT + KT > prior + first + 1) clean(kb, vb);        // workgroup-uniform
        __syncthreads();                                           // also: the tile before is no longer read by anyone
        if (t > 0) fetch(t - 1, kn, rn, vn);
    };
    const int tiles = (kv_end + KT - 1) / KT;
    fetch(tiles - 1, k0, r0, v0);
    for (int t = tiles - 1; t >= 0; t -= 2) {
        open(t, k0, v0, k1, r1, v1);
        compute(t, k0, r0, v0);
        if (t > 0) {
            open(t - 1, k1, v1, k0, r0, v0);
            compute(t - 1, k1, r1, v1);
        }
    }
#pragma unroll
    for (int c = 0; c < R; ++c) {
        l[c] += __shfl_xor(l[c], 16);
        l[c] += __shfl_xor(l[c], 32);
        const int row = row0 + 16 * c + r16;
        if (row >= n) continue;
        const float inv = 1.f / l[c];                              // (a query sees itself: at least 2^-8; not a number of a score that is not finite)
        uint16_t* o = out + (int64_t)row * p.heads * DV + 4 * g4;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
            *(uint2*)(o + 16 * j) = make_uint2(E::pack(O[c][j][0] * inv, O[c][j][1] * inv), E::pack(O[c][j][2] * inv, O[c][j][3] * inv));
    }
}

template <typename E, int R> void launch(const PromptParams& p, const PromptAttnArgs& a) {
    const dim3 grid((unsigned)a.heads, (unsigned)a.num_seqs, (unsigned)((a.max_q_len + 64 * R - 1) / (64 * R)));
    hipLaunchKernelGGL((prompt_attn_kernel<E, R>), grid, dim3(256), 0, a.stream, p);
}

}  // namespace

bool prompt_attn_mfma_supported(const PromptAttnArgs& a) {
    const int64_t step = (int64_t)1 << 26;                         // (token strides in bytes are 32 bits)
    return is_16bit_float(a.dtype) && a.nope == NOPE && a.rope == ROPE && a.dv == DV && a.num_seqs <= 65535 &&
           ((int64_t)a.max_q_len + 63) / 64 <= 65535 && a.key_ts < step && a.value_ts < step && a.rope_ts < step;
}

int launch_prompt_attn_mfma(const PromptAttnArgs& a) {
    PromptParams p;
    p.out = a.out; p.query = a.query; p.key = (const char*)a.key; p.rope_key = (const char*)a.rope_key; p.value = (const char*)a.value;
    p.key_hs = a.key_hs * 2; p.value_hs = a.value_hs * 2;
    p.key_ts = (uint32_t)a.key_ts * 2; p.rope_ts = (uint32_t)a.rope_ts * 2; p.value_ts = (uint32_t)a.value_ts * 2;
    p.cu_q_lens = a.cu_q_lens; p.cu_k_lens = a.cu_k_lens; p.heads = a.heads; p.rows = (int)a.rows; p.keys = (int)a.keys;
    // (weights e^(scale s) are e^(|scale| (-s)) for a negative scale, and alike for one that is 0 in float32)
    const float mul = a.scale * LOG2E, size = mul < 0.f ? -mul : mul;
    const bool none = !(size >= 1.2e-38f);
    p.mul = none ? 1.f : size;
    p.keep = none ? 0u : ~0u;
    p.flip = mul < 0.f && !none ? 0x80008000u : 0u;
    static std::atomic<int> cached_cus{-1};                        // (of the first device used: every GPU of a node is the same part)
    p.num_cus = cached_cus.load(std::memory_order_relaxed);
    if (p.num_cus < 0) {
        int dev = 0, cus = 0;
        if (hipGetDevice(&dev) != hipSuccess ||
            hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 0)
            cus = 0;
        p.num_cus = cus;
        cached_cus.store(cus, std::memory_order_relaxed);
    }
    // 128 queries to a workgroup read a tile once for twice the queries, where that leaves every CU its workgroups.  us, 64 against 128,
    // 16 heads: 2048 tokens 46 against 59, 3000 77 against 89, 4096 129 against 124, 8192 412 against 334; 12 prompts of 37 .. 1500
    // behind 0 .. 2048, 8 heads, 125 against 106
    const int64_t wgs = a.heads * std::min<int64_t>((int64_t)a.num_seqs * ((a.max_q_len + 127) / 128), a.rows / 128 + a.num_seqs);
    const bool f16 = a.dtype == AICOMP_KV_F16;
    if (wgs >= 448) { if (f16) launch<F16Fmt, 2>(p, a); else launch<Bf16Fmt, 2>(p, a); }
    else { if (f16) launch<F16Fmt, 1>(p, a); else launch<Bf16Fmt, 1>(p, a); }
    AICOMP_HIP_LAUNCH_CHECK();
    return AICOMP_KV_OK;
}

}  // namespace aicomp
