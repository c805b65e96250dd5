// Attention of many query rows over latent rows of 512 + 64 elements (row_attn.h) on the matrix cores: more than 16 (token, head) pairs
// to a sequence; 16 bits, blocks of 16 tokens.
//
// An output of 512 elements is too much of a wave's registers for more than 32 rows, and a row of 1152 bytes too much of LDS for every
// wave to have tiles of its own.  So four waves, one to a SIMD with all its registers, share up to 64 rows and tiles of 64 keys, two of
// those in LDS (147 KB), one on its way while the other is computed, and divide each product differently:
//   S^T = K Q^T      a wave has all the rows and 16 of the tile's keys: a key is read from LDS once, the queries stay in registers
//   O^T += V^T P^T   a wave has all the rows and 128 of the 512 columns: a value is read once, the weights go through LDS
// All of them need one reference for a row's weights.  They take the one they have, without asking each other: a wave that finds a score
// more than 2^8 above it says so in LDS, and then, as in an item's first tile, all of them meet once more, move the reference and write
// their weights anew.  So a tile costs two barriers.
//
// With one wave to a SIMD nothing hides what a wave waits for: operands are read some steps ahead of their products, and the next tile's
// loads go out between the products, one to a step (all eighteen at once hold the wave up for as long as the scores take).
//
// The division of the work is that of row_line.h; values that are not finite are marked as in row_attn_mfma.hip.
#include "row_line.h"

namespace aicomp {

namespace {

constexpr int DK = 576, DV = 512;
constexpr int KT = 64;                 // keys per tile
constexpr int KROW = 2 * DK;           // bytes of a row
constexpr int NS = DK / 32, NJ = 8;    // steps of a score; 16-column groups of a wave's quarter of the output
constexpr int PROW = 2 * KT + 16;      // bytes of a row of weights (padded: sixteen rows start in different banks)

// NC: groups of 16 rows
template <typename E, int NC>
__global__ void __launch_bounds__(256, 1)
row_attn_latent_kernel(RowParams p) {
    constexpr int ROWS = 16 * NC;
    __shared__ __attribute__((aligned(1024))) unsigned char buf0[KT * KROW];
    __shared__ __attribute__((aligned(1024))) unsigned char buf1[KT * KROW];
    __shared__ __attribute__((aligned(16))) unsigned char weights[ROWS * PROW];
    __shared__ float top[4][ROWS];                             // largest score of each quarter of the keys; then sums
    __shared__ int moved[2];                                   // by tile parity
    __shared__ __attribute__((aligned(16))) uint32_t offsets[64][12];                  // by lane: of its nine chunks of eight keys
    __shared__ PieceScratch scratch;

    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), quarter = w;
    const int r16 = lane & 15, g4 = lane >> 4;
    const int worker = (p.workers & 7) ? (int)blockIdx.x : ((int)blockIdx.x & 7) * (p.workers >> 3) + ((int)blockIdx.x >> 3);
    Piece mine;
    if (!piece_of<ROWS, KT, 256>(p, worker, scratch, mine)) return;

    auto fk = [](int key) { return key & 7; };                 // chunk c (16 bytes) of key k lies at c ^ f(k)
    uint32_t ka[2], va[4];
    const int vkey = 4 * g4 + (r16 >> 2);
#pragma unroll
    for (int i = 0; i < 2; ++i) ka[i] = r16 * KROW + (((4 * i + g4) ^ fk(r16)) << 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) va[i] = vkey * KROW + 256 * w + (((2 * i + ((r16 >> 1) & 1)) ^ fk(vkey)) << 4) + (r16 & 1) * 8;
    // a wave's weights: four keys of each of its rows; all of them, eight keys of a row at a time
    const uint32_t p_to = r16 * PROW + ((quarter >> 1) * 4 + g4) * 16 + (quarter & 1) * 8;
    const uint32_t p_from = r16 * PROW + g4 * 16;

    // eight rows of 1152 bytes in nine loads of 1 KB; `from` is uniform, `last` the last row that is there
    auto bring = [&](const char* from, int last, unsigned char* to) __attribute__((always_inline)) {
        int x = lane;
        asm volatile("" : "+v"(x));                            // (the offsets are made anew: nine registers less)
#pragma unroll
        for (int i = 0; i < 9; ++i) {
            const int chunk = 64 * i + x, row = chunk / 72, slot = chunk - row * 72;
            __builtin_amdgcn_global_load_lds(GLOBAL_PTR(from + (min(row, last) * KROW + ((slot ^ fk(row)) << 4))), LDS_PTR(to + 1024 * i), 16,
                                             0, 0);
        }
    };

    if (w == 0) {
#pragma unroll
        for (int i = 0; i < 9; ++i) {
            const int chunk = 64 * i + lane, row = chunk / 72, slot = chunk - row * 72;
            offsets[lane][i] = row * KROW + ((slot ^ fk(row)) << 4);
        }
    }
    __syncthreads();

    Item it;
    while (next_item<ROWS, KT>(p, worker, mine, it)) {
        const Seq q = mine.q;
        const int nrows = q.n * p.group, row0 = it.rtile * ROWS;
        const int full = p.masks ? q.prior : q.prior + it.rtile * ROWS / p.group + 1;  // keys that all rows of the item see

        typedef const __attribute__((address_space(4))) int32_t* const_i32_ptr;
        const const_i32_ptr table = (const_i32_ptr)(p.block_table + (int64_t)mine.seq * p.block_table_stride);
        const int last_block = (q.ctx - 1) / BS;               // (blocks behind it are not this sequence's)
        // Wave w brings in block w of a tile, 1 KB at a time: load i of 18.
        auto block_of = [&](int t) -> const char* {
            const int b = table[min(4 * t + w, last_block)];
            return (const char*)p.k_pool + (int64_t)max(0, min(b, p.num_blocks - 1)) * BS * KROW;
        };
        // (a buffer of no bytes brings in nothing: the last tile's step has the same instructions as the others)
        auto buffer_of = [&](const char* from, bool there) {
            return __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, there ? BS * KROW : 0, 0x00027000);
        };
        auto load = [&](__amdgpu_buffer_rsrc_t from, unsigned char* to, uint32_t off, int i) __attribute__((always_inline)) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(from, LDS_PTR(to + (16 * w + 8 * (i / 9)) * KROW + 1024 * (i % 9)), 16, off,
                                                     (i / 9) * 8 * KROW, 0, 0);
        };
        const int t_end = min(it.t1, (q.ctx + KT - 1) / KT);   // (0 tiles where the context is none)
        // The rows, which lie one after the other, come by way of the second buffer (rows beyond the last: that one, computed and not
        // stored).
        if (it.t0 < t_end) {
            const auto from = buffer_of(block_of(t_end - 1), true);
#pragma unroll
            for (int i = 0; i < 18; ++i) load(from, buf0, offsets[lane][i % 9], i);
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            if (16 * w + 8 * g >= ROWS) break;                 // wave-uniform
            const int here = min(row0 + 16 * w + 8 * g, nrows - 1);
            bring((const char*)p.query + ((int64_t)q.begin * p.hq + here) * KROW, nrows - 1 - here, buf1 + (16 * w + 8 * g) * KROW);
        }
        if (tid < 2) moved[tid] = 0;
        __builtin_amdgcn_s_waitcnt(0x0F70);                    // vmcnt(0)
        __syncthreads();
        uint4 qf[NC][NS];
        int token[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            token[c] = min(row0 + 16 * c + r16, nrows - 1) / p.group;
#pragma unroll
            for (int s = 0; s < NS; ++s) qf[c][s] = *(const uint4*)(buf1 + 16 * c * KROW + ka[s & 1] + (s >> 1) * 128);
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);                    // lgkmcnt(0): the second buffer is free once all have met

        float m[NC], l[NC];
        f32x4_t O[NC][NJ];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            m[c] = NEG_BIG; l[c] = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) O[c][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }

        // Values that are not finite, among the wave's own keys, four lanes to each (row_attn_mfma.hip has the reason).
        auto clean = [&](unsigned char* kb) __attribute__((always_inline)) {
            constexpr uint32_t EXP = E::DT == AICOMP_KV_F16 ? 0x7c007c00u : 0x7f807f80u;
            constexpr uint32_t ONE = E::DT == AICOMP_KV_F16 ? 0x04000400u : 0x00800080u;
            uint4* const at = (uint4*)(kb + (16 * w + (lane >> 2)) * KROW) + (lane & 3);
            uint32_t acc = 0;
            for (int i = 0; i < DV / 32; ++i) {
                const uint4 x = at[4 * i];
                acc |= ((x.x & EXP) + ONE) | ((x.y & EXP) + ONE) | ((x.z & EXP) + ONE) | ((x.w & EXP) + ONE);
            }
            const uint64_t bad = __ballot((acc & 0x80008000u) != 0);
            if ((bad >> (lane & ~3)) & 15) {
                for (int i = 0; i < DV / 32; ++i) at[4 * i] = make_uint4(0, 0, 0, 0);
                at[DV / 8] = make_uint4(~0u, ~0u, ~0u, ~0u);
            }
        };

        const int t_first = t_end - 1;
        auto step = [&](int t, unsigned char* kb, unsigned char* next) __attribute__((always_inline)) {
            const int start = t * KT;
            const bool masked = start + KT > full;             // workgroup-uniform
            __builtin_amdgcn_s_waitcnt(0x0F70);                // vmcnt(0): this wave's part of the tile
            if (masked) clean(kb);
            __syncthreads();                                   // also: the tile before and its weights are no longer read by anyone
            const auto from = buffer_of(block_of(max(t - 1, it.t0)), t > it.t0);
            if (tid == 0) moved[(t + 1) & 1] = 0;              // (read before this barrier, written after the next)
            // which of this lane's four keys its rows see (made before the products: it takes registers that they need)
            uint32_t win = ~0u;
            if (masked) {
                win = 0;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int64_t* words = p.masks ? p.masks + (int64_t)(q.begin + token[c]) * p.mask_words : nullptr;
                    win |= (window_of(words, p.mask_words, start + 16 * quarter, q.prior, q.ctx, q.prior + token[c] + 1) >> (4 * g4) & 15) << (4 * c);
                }
                asm volatile("" : "+v"(win));
            }
            // The scores' products.  The next tile's loads go out between them, one to a step (all at once they hold the wave up for longer
            // than the products take), keys are read three steps ahead.
            f32x4_t sa[NC];
            uint4 ahead[4];
            uint32_t off[4];
            auto key_of = [&](int s) { return *(const uint4*)(kb + 16 * quarter * KROW + ka[s & 1] + (s >> 1) * 128); };
#pragma unroll
            for (int c = 0; c < NC; ++c) sa[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < 3; ++s) { ahead[s] = key_of(s); off[s] = offsets[lane][s]; }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                if (s + 3 < NS) { ahead[(s + 3) & 3] = key_of(s + 3); off[(s + 3) & 3] = offsets[lane][(s + 3) % 9]; }
                load(from, next, off[s & 3], s);
#pragma unroll
                for (int c = 0; c < NC; ++c) sa[c] = E::mfma(ahead[s & 3], qf[c][s], sa[c]);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) sa[c] *= p.mul;
            if (masked) {
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!((win >> (4 * c + e)) & 1)) sa[c][e] = -INFINITY;
            }
            auto largest = [&](int c) { return fmaxf(fmaxf(sa[c][0], sa[c][1]), fmaxf(sa[c][2], sa[c][3])); };
            // weights against the reference there is
            float got[NC];
            auto put = [&]() __attribute__((always_inline)) {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const uint32_t lo = E::pack(__builtin_amdgcn_exp2f(sa[c][0] - m[c]), __builtin_amdgcn_exp2f(sa[c][1] - m[c]));
                    const uint32_t hi = E::pack(__builtin_amdgcn_exp2f(sa[c][2] - m[c]), __builtin_amdgcn_exp2f(sa[c][3] - m[c]));
                    *(uint2*)(weights + p_to + 16 * c * PROW) = make_uint2(lo, hi);
                    got[c] = E::pair_sum(lo, E::pair_sum(hi, 0.f));
                }
            };
            bool again = t == t_first;                         // workgroup-uniform: there is no reference yet
            if (!again) {
                bool beyond = false;
#pragma unroll
                for (int c = 0; c < NC; ++c) beyond |= largest(c) > m[c] + SLACK;
                if (__ballot(beyond)) moved[t & 1] = 1;
                put();
                __syncthreads();
                again = moved[t & 1];
            }
            if (again) {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const float mx = xor32_max(xor16_max(largest(c)));
                    if (g4 == 0) top[quarter][16 * c + r16] = mx;
                }
                __syncthreads();
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int r = 16 * c + r16;
                    const float m_new = fmaxf(fmaxf(fmaxf(top[0][r], top[1][r]), fmaxf(top[2][r], top[3][r])), m[c]);
                    const float alpha = __builtin_amdgcn_exp2f(m[c] - m_new);
                    m[c] = m_new;
                    l[c] *= alpha;
                    if (t == t_first) continue;                // (nothing to scale)
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        // (each by itself from and to its accumulator registers: all at once they take the vector registers of the rest)
                        asm volatile("" : "+a"(O[c][j]));
                        O[c][j] *= alpha;
                        asm volatile("" : "+a"(O[c][j]));
                    }
                }
                put();
                __syncthreads();
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) l[c] += got[c];
            // the output's products, values two steps ahead
            typedef short v4i16_t __attribute__((ext_vector_type(4)));
            typedef short v8i16_t __attribute__((ext_vector_type(8)));
            typedef __attribute__((address_space(3))) v4i16_t* lds_v4i16_ptr;
            uint4 pf[2][NC];
            v8i16_t val[3];
            auto value_of = [&](int u) {                       // 16 columns of 32 keys
                const uint32_t o = va[u & 3] + ((u >> 2) & 1) * 128 + (u >> 3) * 32 * KROW;
                const v4i16_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(kb + o));
                const v4i16_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(kb + o + 16 * KROW));
                return v8i16_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
            };
#pragma unroll
            for (int c = 0; c < NC; ++c) pf[0][c] = *(const uint4*)(weights + p_from + 16 * c * PROW);
            val[0] = value_of(0);
            val[1] = value_of(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < 2 * NJ; ++u) {
                if (u + 2 < 2 * NJ) val[(u + 2) % 3] = value_of(u + 2);
                if (u >= 2 && u < 2 + NC) pf[1][u - 2] = *(const uint4*)(weights + p_from + 64 + 16 * (u - 2) * PROW);
#pragma unroll
                for (int c = 0; c < NC; ++c) O[c][u % NJ] = E::mfma(__builtin_bit_cast(uint4, val[u % 3]), pf[u / NJ][c], O[c][u % NJ]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // from the nearest keys to the farthest
        for (int t = t_end - 1; t >= it.t0; t -= 2) {
            step(t, buf0, buf1);
            if (t > it.t0) step(t - 1, buf1, buf0);
        }
        __syncthreads();                                       // (buffers, weights and `top` are free)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            l[c] += __shfl_xor(l[c], 16);
            l[c] += __shfl_xor(l[c], 32);
            if (g4 == 0) top[quarter][16 * c + r16] = l[c];
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int r = 16 * c + r16, row = it.rtile * ROWS + r;
            if (row >= nrows) continue;
            const float sum = top[0][r] + top[1][r] + top[2][r] + top[3][r];
            const int col = 128 * w + 4 * g4;
            if (!it.whole) {
                if (g4 == 0 && w == 0) p.ws_ml[it.slot * ROWS + r] = make_float2(m[c], sum);
                float* dst = p.ws_acc + (it.slot * ROWS + r) * DV + col;
#pragma unroll
                for (int j = 0; j < NJ; ++j) *(f32x4_t*)(dst + 16 * j) = O[c][j];
            } else {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                uint16_t* dst = (uint16_t*)p.out + ((int64_t)(q.begin + row / p.group) * p.hq + row % p.group) * DV + col;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    *(uint2*)(dst + 16 * j) = make_uint2(E::pack(O[c][j][0] * inv, O[c][j][1] * inv), E::pack(O[c][j][2] * inv, O[c][j][3] * inv));
            }
        }
        __syncthreads();                                       // (`top` is free)
    }
}

template <typename E, int NC> void launch(const RowParams& p, int64_t items, hipStream_t stream) {
    hipLaunchKernelGGL((row_attn_latent_kernel<E, NC>), dim3((unsigned)p.workers), dim3(256), 0, stream, p);
    if (p.ws_items != nullptr)
        hipLaunchKernelGGL((row_join_kernel<E, DV, 16 * NC, KT>), dim3((unsigned)(items * (16 * NC * DV / 1024))), dim3(256), 0, stream, p);
}

template <typename E> void launch_groups(const RowParams& p, int groups, int64_t items, hipStream_t stream) {
    if (groups == 2) launch<E, 2>(p, items, stream);
    else if (groups == 3) launch<E, 3>(p, items, stream);
    else launch<E, 4>(p, items, stream);
}

}  // namespace

void launch_row_attn_latent(const RowParams& p, bool f16, int groups, int64_t items, hipStream_t stream) {
    if (f16) launch_groups<F16Fmt>(p, groups, items, stream); else launch_groups<Bf16Fmt>(p, groups, items, stream);
}

}  // namespace aicomp
