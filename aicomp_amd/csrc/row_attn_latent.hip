// Attention of many query rows over latent rows of 512 + 64 elements (row_attn.h) on the matrix cores: more than 16 (token, head) pairs
// to a sequence; 16 bits, blocks of 16, 32, 64 .. tokens.
//
// An output of 512 elements is too much of a wave's registers for more than 32 rows, and a row of 1152 bytes too much of LDS for every
// wave to have tiles of its own.  So four waves, one to a SIMD with all its registers, share 64 rows and tiles of 64 keys, two of those in
// LDS (147 KB), one on its way while the other is computed, and divide each product differently:
//   S^T = K Q^T      a wave has half of the rows and half of the keys; its queries stay in registers
//   O^T += V^T P^T   a wave has all the rows and 128 of the 512 columns: a value is read once, the weights go through LDS
// All of them need one reference for a row's weights.  They take the one they have, without asking each other: a wave that finds a score
// more than 2^8 above it says so in LDS, and then, as in an item's first tile, all of them meet once more, move the reference and write
// their weights anew.  So a tile costs two barriers.
//
// With one wave to a SIMD nothing hides what a wave waits for, or issues beside the products: products of 32 x 32 x 16, so that there are
// few of them and each covers the reads ahead and the next tile's loads, one of which goes out every other product or so (all eighteen
// at once hold the wave up for as long as the scores take).  395 of a wave's 512 registers are taken; what else might be begun beside a
// tile's softmax has room there.
//
// Causal chunks are taken like trees: an item has the keys of the whole context, those behind its last row too, which are masked.  2048 tokens
// of a new prompt, 16 heads: 199 us, about half of the products for nothing; 512 tokens behind 4096: 96 us, 0.80 PFLOP/s.
//
// The division of the work is that of row_line.h; values that are not finite are marked as in row_attn_mfma.hip.
//
// 32 rows of 128 heads over 512 .. 4096 latent rows: 46 us, 437 TFLOP/s, of which the second launch 9.  A tile takes 4600 cycles, its products
// 2200: the scores 1700 (LDS, which gives a key to two waves and takes in the next tile), weights 1150, the output 1300; an item's start
// and end some 7 us, its partial output in float32, 128 KB, among them.  Tiles of 48 rows by products of 16 x 16 x 32, a wave having all
// rows and 16 keys: 4550 cycles a tile, 59 us.
#include "row_line.h"

namespace aicomp {

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int DK = 576, DV = 512;
constexpr int ROWS = 64, KT = 64;      // rows and keys of a tile
constexpr int KROW = 2 * DK;           // bytes of a row
constexpr int BLOCK = 16 * KROW;       // bytes of 16 rows
constexpr int NS = DK / 16;            // steps of a score
constexpr int LOADS = BLOCK / 1024;    // a wave's, to a tile
constexpr int IN_S = 14;               // of these, between the scores' products; the others between the output's
constexpr int PROW = 2 * KT + 16;      // bytes of a row of weights (padded: sixteen rows start in different banks)

// D[32x32] += A[32x16] * B[16x32]
template <typename E> __device__ __forceinline__ f32x16_t mfma32(const uint4& a, const uint4& b, const f32x16_t& c) {
    if constexpr (E::DT == AICOMP_KV_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

template <typename E>
__global__ void __launch_bounds__(256, 1)
row_attn_latent_kernel(RowParams p) {
    __shared__ __attribute__((aligned(1024))) unsigned char buf0[KT * KROW];
    __shared__ __attribute__((aligned(1024))) unsigned char buf1[KT * KROW];
    __shared__ __attribute__((aligned(16))) unsigned char weights[ROWS * PROW];
    __shared__ float top[2][ROWS];                             // largest score of each half of the keys; then sums
    __shared__ int moved[2];                                   // by tile parity
    __shared__ PieceScratch scratch;

    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), kh = w & 1, rh = w >> 1;  // a wave's halves of the keys and of the rows
    const int n = lane & 31, h = lane >> 5, r16 = lane & 15;
    const int worker = (p.workers & 7) ? (int)blockIdx.x : ((int)blockIdx.x & 7) * (p.workers >> 3) + ((int)blockIdx.x >> 3);
    Piece mine;
    if (!piece_of<ROWS, KT, 256>(p, worker, scratch, mine)) return;

    // Sixteen rows lie in LDS by columns of 128 bytes: 1 KB for eight rows, which is what one load brings in, whole lines of memory.  In these,
    // chunk c (16 bytes) of row k is at c ^ f(k): of a key's chunk, eight rows and the eight even ones of sixteen lie in different banks;
    // of four neighbouring chunks of a value, four rows do.
    auto f = [](int k) { return (k >> 1 & 1) << 2 | ((k >> 2 ^ k) & 1) << 1 | ((k ^ k >> 3) & 1); };
    const int krow = lane & 15;                                // rows n of 32, in two blocks of 16
    const int vrow = 8 * h + (r16 >> 2);                       // the first of the two that a lane reads of a value; the other four behind
    uint32_t ka[4], va[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) ka[i] = (n >> 4) * BLOCK + (krow >> 3) * 1024 + (krow & 7) * 128 + (((2 * i + h) ^ f(krow)) << 4);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int row = vrow + 4 * b, c = 4 * i + 2 * (lane >> 4 & 1) + (r16 >> 1 & 1);
            va[i][b] = 2 * w * 2048 + (row >> 3) * 1024 + (row & 7) * 128 + ((c ^ f(row)) << 4) + (r16 & 1) * 8;
        }
    // what a lane loads: of eight rows, and of the eight behind them
    const int lrow = lane >> 3;
    const uint32_t lcol[2] = {(uint32_t)((lane & 7) ^ f(lrow)) << 4, (uint32_t)((lane & 7) ^ f(lrow + 8)) << 4};
    // a wave's weights: four neighbouring keys of a row at a time; all of them, eight
    const uint32_t p_to = (32 * rh + n) * PROW + (32 * kh + 4 * h) * 2, p_from = n * PROW + 16 * h;

    Item it;
    while (next_item<ROWS, KT>(p, worker, mine, it)) {
        const Seq q = mine.q;
        const int nrows = q.n * p.group, row0 = it.rtile * ROWS;
        const int full = p.masks ? q.prior : q.prior + it.rtile * ROWS / p.group + 1;  // keys that all rows of the item see

        typedef const __attribute__((address_space(4))) int32_t* const_i32_ptr;
        const const_i32_ptr table = (const_i32_ptr)(p.block_table + (int64_t)mine.seq * p.block_table_stride);
        // Wave w brings in 16 rows of a tile, by 18 loads.
        auto block = [&](int entry, int t) { return (const char*)p.k_pool + place_of(p, entry, 0, 4 * t + w) * BLOCK; };
        auto block_of = [&](int t) { return block(table[entry_of(p, q, 4 * t + w)], t); };
        // (a buffer of no bytes brings in nothing: the last tile's step has the same instructions as the others)
        auto buffer_of = [&](const char* from, bool there) {
            return __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, there ? BLOCK : 0, 0x00027000);
        };
        auto load = [&](__amdgpu_buffer_rsrc_t from, unsigned char* to, int i) __attribute__((always_inline)) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(from, LDS_PTR(to + w * BLOCK + 1024 * i), 16, lrow * KROW + lcol[i & 1],
                                                     (i & 1) * 8 * KROW + (i >> 1) * 128, 0, 0);
        };
        const int t_end = min(it.t1, (q.ctx + KT - 1) / KT);   // (0 tiles where the context is none)
        // The rows come by way of the second buffer, sixteen by each wave (rows beyond the last: that one, computed and not stored); before
        // the first tile, whose place in the table is still to arrive.
        const int entry = t_end > it.t0 ? table[entry_of(p, q, 4 * (t_end - 1) + w)] : 0;
        {
            const int here = min(row0 + 16 * w, nrows - 1);
            const char* from = (const char*)p.query + ((int64_t)q.begin * p.hq + here) * KROW;
            const uint32_t at[2] = {min(lrow, nrows - 1 - here) * KROW + lcol[0], min(lrow + 8, nrows - 1 - here) * KROW + lcol[1]};
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                __builtin_amdgcn_global_load_lds(GLOBAL_PTR(from + at[i & 1] + (i >> 1) * 128), LDS_PTR(buf1 + w * BLOCK + 1024 * i), 16, 0, 0);
        }
        if (it.t0 < t_end) {
            const auto from = buffer_of(block(entry, t_end - 1), true);
#pragma unroll
            for (int i = 0; i < LOADS; ++i) load(from, buf0, i);
        }
        if (tid < 2) moved[tid] = 0;
        __builtin_amdgcn_s_waitcnt(0x0F70);                    // vmcnt(0)
        __syncthreads();
        uint4 qf[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = *(const uint4*)(buf1 + 2 * rh * BLOCK + ka[s & 3] + (s >> 2) * 2048);
        __builtin_amdgcn_s_waitcnt(0xC07F);                    // lgkmcnt(0): the second buffer is free once all have met
        if (p.mul < 0.f) {                                     // (the sign of the scale: the largest product is then the largest score)
#pragma unroll
            for (int s = 0; s < NS; ++s) qf[s] = make_uint4(qf[s].x ^ E::SIGN_PAIR, qf[s].y ^ E::SIGN_PAIR, qf[s].z ^ E::SIGN_PAIR, qf[s].w ^ E::SIGN_PAIR);
        }
        const float mul = fabsf(p.mul);
        const int token = min(row0 + 32 * rh + n, nrows - 1) / p.group;

        // of rows n and 32 + n; l: of the wave's half of the rows and keys
        float m[2] = {NEG_BIG, NEG_BIG}, l = 0.f;
        bool far = false;                                      // some reference of the wave's half of the rows is beyond FAR
        f32x16_t O[4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int e = 0; e < 16; ++e) O[j][r][e] = 0.f;

        // Values that are not finite, among the wave's own keys, four lanes to each (row_attn_mfma.hip has the reason).
        auto clean = [&](unsigned char* kb) __attribute__((always_inline)) {
            constexpr uint32_t EXP = E::DT == AICOMP_KV_F16 ? 0x7c007c00u : 0x7f807f80u;
            constexpr uint32_t ONE = E::DT == AICOMP_KV_F16 ? 0x04000400u : 0x00800080u;
            const int key = lane >> 2;
            uint4* const at = (uint4*)(kb + w * BLOCK + (key >> 3) * 1024 + (key & 7) * 128) + (lane & 3);
            uint32_t acc = 0;
            for (int i = 0; i < DV / 32; ++i) {
                const uint4 x = at[128 * (i >> 1) + 4 * (i & 1)];
                acc |= ((x.x & EXP) + ONE) | ((x.y & EXP) + ONE) | ((x.z & EXP) + ONE) | ((x.w & EXP) + ONE);
            }
            const uint64_t bad = __ballot((acc & 0x80008000u) != 0);
            if ((bad >> (lane & ~3)) & 15) {
                for (int i = 0; i < DV / 32; ++i) at[128 * (i >> 1) + 4 * (i & 1)] = make_uint4(0, 0, 0, 0);
                at[128 * (DV / 64)] = make_uint4(~0u, ~0u, ~0u, ~0u);
            }
        };

        const int t_first = t_end - 1;
        auto step = [&](int t, unsigned char* kb, unsigned char* next) __attribute__((always_inline)) {
            const int start = t * KT;
            const bool masked = start + KT > full;             // workgroup-uniform
            __builtin_amdgcn_s_waitcnt(0x0F70);                // vmcnt(0): this wave's part of the tile
            if (masked) clean(kb);
            lds_barrier();                                     // also: the tile before and its weights are no longer read by anyone
            const auto from = buffer_of(block_of(max(t - 1, it.t0)), t > it.t0);
            if (tid == 0) moved[(t + 1) & 1] = 0;              // (read before this barrier, written after the next)
            // which of the wave's 32 keys this lane's row sees (made before the products: it takes registers that they need)
            uint32_t win = ~0u;
            if (masked) {
                const int64_t* words = p.masks ? p.masks + (int64_t)(q.begin + token) * p.mask_words : nullptr;
                win = window_of(words, p.mask_words, start + 32 * kh, q.prior, q.ctx, q.prior + token + 1) >> (4 * h);
                asm volatile("" : "+v"(win));
            }
            // The scores' products; keys are read four steps ahead.
            f32x16_t sa;
            uint4 ahead[5];
            auto key_of = [&](int s) { return *(const uint4*)(kb + 2 * kh * BLOCK + ka[s & 3] + (s >> 2) * 2048); };
#pragma unroll
            for (int e = 0; e < 16; ++e) sa[e] = 0.f;
#pragma unroll
            for (int s = 0; s < 4; ++s) ahead[s] = key_of(s);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                if (s + 4 < NS) ahead[(s + 4) % 5] = key_of(s + 4);
#pragma unroll
                for (int i = 0; i < IN_S; ++i)
                    if (i * NS / IN_S == s) load(from, next, i);
                sa = mfma32<E>(ahead[s % 5], qf[s], sa);
                __builtin_amdgcn_sched_barrier(0);
            }
            // element e: key 8 (e / 4) + 4 h + e % 4 of the wave's, row n
            float factor = mul;
            if (masked || far) {                               // (nothing is left to multiply: the factor may be 0)
                factor = 1.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) sa[e] = win >> (8 * (e >> 2) + (e & 3)) & 1 ? sa[e] * mul : -INFINITY;
            }
            float most = sa[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) most = fmaxf(most, sa[e]);
            most *= factor;
            // weights against the reference there is
            uint32_t pair[8];
            auto put = [&]() __attribute__((always_inline)) {
                const float ref = rh ? m[1] : m[0];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    pair[e] = E::pack(__builtin_amdgcn_exp2f(fmaf(sa[2 * e], factor, -ref)), __builtin_amdgcn_exp2f(fmaf(sa[2 * e + 1], factor, -ref)));
#pragma unroll
                for (int e = 0; e < 8; e += 2) *(uint2*)(weights + p_to + 8 * e) = make_uint2(pair[e], pair[e + 1]);
            };
            if (t != t_first) {
                if (__ballot(most > (rh ? m[1] : m[0]) + SLACK)) moved[t & 1] = 1;
                put();
                lds_barrier();
            }
            // the output's products, values three steps ahead
            typedef short v4i16_t __attribute__((ext_vector_type(4)));
            typedef short v8i16_t __attribute__((ext_vector_type(8)));
            typedef __attribute__((address_space(3))) v4i16_t* lds_v4i16_ptr;
            uint4 pf[2][2];
            v8i16_t val[4];
            auto value_of = [&](int u) {                       // 32 columns of 16 keys
                const uint32_t o = (u & 2) * 1024 + (u >> 2) * BLOCK;
                const v4i16_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(kb + va[u & 1][0] + o));
                const v4i16_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(kb + va[u & 1][1] + o));
                return v8i16_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
            };
            auto weights_of = [&](int b, int r) { return *(const uint4*)(weights + p_from + 32 * r * PROW + 32 * b); };
            const int beyond = moved[t & 1];
            pf[0][0] = weights_of(0, 0);
            pf[0][1] = weights_of(0, 1);
            if (t == t_first || beyond) {                      // workgroup-uniform; at first there is no reference
                const float mx = xor32_max(most);
                if (h == 0) top[kh][32 * rh + n] = mx;
                lds_barrier();
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float m_new = fmaxf(fmaxf(top[0][32 * r + n], top[1][32 * r + n]), m[r]);
                    const float alpha = __builtin_amdgcn_exp2f(m[r] - m_new);
                    m[r] = m_new;
                    if (r == rh) {
                        l *= alpha;
                        // The reference is a rounded product: against the exact ones of an fma, all weights of a row are off by its
                        // rounding.  Where that would leave the range of 16 bits, the products are rounded too.
                        if (!far && __ballot(fabsf(m_new) > FAR && m_new > NEG_BIG)) {     // (alike in the two waves of a row)
#pragma clang fp contract(off)
                            far = true;
#pragma unroll
                            for (int e = 0; e < 16; ++e) sa[e] *= factor;
                            factor = 1.f;
                        }
                    }
                    if (t == t_first) continue;                // (nothing to scale)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        // (each by itself from and to its accumulator registers: all at once they take the vector registers of the rest)
                        asm volatile("" : "+a"(O[j][r]));
                        O[j][r] *= alpha;
                        asm volatile("" : "+a"(O[j][r]));
                    }
                }
                put();
                lds_barrier();
                pf[0][0] = weights_of(0, 0);
                pf[0][1] = weights_of(0, 1);
            }
#pragma unroll
            for (int u = 0; u < 3; ++u) val[u] = value_of(u);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                if (u + 3 < 16) val[(u + 3) & 3] = value_of(u + 3);
                if ((u & 3) < 2 && u < 12) pf[(u >> 2) + 1 & 1][u & 1] = weights_of((u >> 2) + 1, u & 1);
                if (IN_S + u < LOADS) load(from, next, IN_S + u);
                if (u >= 8) l = E::pair_sum(pair[u - 8], l);   // (of the weights as rounded)
#pragma unroll
                for (int r = 0; r < 2; ++r) O[u & 3][r] = mfma32<E>(__builtin_bit_cast(uint4, val[u & 3]), pf[u >> 2 & 1][r], O[u & 3][r]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // from the nearest keys to the farthest
        for (int t = t_end - 1; t >= it.t0; t -= 2) {
            step(t, buf0, buf1);
            if (t > it.t0) step(t - 1, buf1, buf0);
        }
        lds_barrier();                                         // (buffers, weights and `top` are free)
        l += __shfl_xor(l, 32);
        if (h == 0) top[kh][32 * rh + n] = l;
        lds_barrier();
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = row0 + 32 * r + n;
            if (row >= nrows) continue;
            const float sum = top[0][32 * r + n] + top[1][32 * r + n];
            const int col = 128 * w + 4 * h;
            if (!it.whole) {
                if (h == 0 && w == 0) p.ws_ml[it.slot * ROWS + 32 * r + n] = make_float2(m[r], sum);
                float* dst = p.ws_acc + (it.slot * ROWS + 32 * r + n) * DV + col;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *(f32x4_t*)(dst + 32 * j + 2 * e) = f32x4_t{O[j][r][e], O[j][r][e + 1], O[j][r][e + 2], O[j][r][e + 3]};
            } else {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                uint16_t* dst = (uint16_t*)p.out + ((int64_t)(q.begin + row / p.group) * p.hq + row % p.group) * DV + col;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *(uint2*)(dst + 32 * j + 2 * e) = make_uint2(E::pack(O[j][r][e] * inv, O[j][r][e + 1] * inv),
                                                                     E::pack(O[j][r][e + 2] * inv, O[j][r][e + 3] * inv));
            }
        }
        lds_barrier();                                         // (`top` is free)
    }
}

template <typename E> void launch(const RowParams& p, int64_t items, hipStream_t stream) {
    hipLaunchKernelGGL((row_attn_latent_kernel<E>), dim3((unsigned)p.workers), dim3(256), 0, stream, p);
    if (p.ws_items != nullptr)
        hipLaunchKernelGGL((row_join_kernel<E, DV, ROWS, KT>), dim3((unsigned)(items * (ROWS * DV / 1024))), dim3(256), 0, stream, p);
}

}  // namespace

void launch_row_attn_latent(const RowParams& p, bool f16, int64_t items, hipStream_t stream) {
    if (f16) launch<F16Fmt>(p, items, stream); else launch<Bf16Fmt>(p, items, stream);
}

}  // namespace aicomp
