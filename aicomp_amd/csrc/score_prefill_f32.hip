// Rows of prompt chunks by a score rule (score.h) for float32 models, on gfx950's float32 matrix instruction: every product and
// sum stays float32.
//
// Mathematics, rows, visible intervals, order of the tiles, divided keys: as in score_prefill.hip; a cap takes the library's tanh, whose
// error is that of float32 also where it is multiplied by a large cap.
//
// Work split   one workgroup (4 waves of 16 rows) per (64 rows, sequence, head group[, part of the keys]).
// K/V tiles    32 tokens, double-buffered, straight into LDS (global_load_lds_dwordx4) one tile ahead, one barrier per tile.  K's 16-byte
//              chunks are swizzled by the row, so that four consecutive lanes of an operand read share a 64-byte segment and sixteen
//              a bank line; V's are read in the order they lie.
// S^T = K Q^T  v_mfma_f32_16x16x4_f32; the k index of MFMA 4 q + e in lane group g is dim 16 q + 4 g + e, so that one 16-byte LDS
//              read has the A operands of four.  O^T += V^T P^T: lane (r, g) reads dims 64 f + 4 r .. + 3 of token 4 g + e, and B is
//              the weight that the lane holds.
// Bound by     the float32 matrix instruction, beside which no vector instruction runs: 2048 new tokens, 32 / 8 heads of 128: it holds 71 %
//              of the cycles, the vector ALU 5 % (11 % under a cap) and both none; the rest are waits of two rounds of workgroups
//              unlike in length.  326 us under a cap, 322 without any term, 105 TFLOP/s, where a large product reaches 153 (on the vector
//              units 2880).  head_dim 64: a cap 198, a bias alone 180, neither 176; 65 % and 8 %.
#include "score_prefill.h"

namespace aicomp {

namespace {

constexpr int KT = 32;                 // tokens per tile

template <int DH, bool CAP, bool BIAS>
__global__ void __launch_bounds__(256, DH == 256 ? 1 : 2)
score_prefill_f32_kernel(ScorePrefillParams p) {
    constexpr int KROW = 4 * DH;               // bytes of an LDS row
    constexpr int NQ = DH / 16;                // 16-element chunks of a row
    constexpr int NF = DH / 64;
    constexpr int CPR = DH / 4;                // 16-byte chunks per row
    constexpr int TILE_BYTES = KT * KROW;
    const int part = blockIdx.x / p.hgroups, hgroup = blockIdx.x % p.hgroups;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g4 = lane >> 4;
    const int pos_per_wg = 64 / p.gpack;

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

    // this lane's row (beyond the chunk's end: the last one's, computed and not stored)
    const int row = 16 * w + r16, qpos = q0 + row / p.gpack, head = hgroup * p.gpack + row % p.gpack;
    const bool row_valid = qpos < n;
    const int pos = prior + min(qpos, n - 1);
    int lo = 0, hi = 0;
    if (prior >= 0) visible_keys(p.rule, q_begin + pos - prior, seq, pos, ctx, lo, hi);
    const bool sees = lo < hi;
    // keys that some row of the wave sees, [wave_lo, wave_hi), and those that all of them see, [full_lo, full_hi)
    const bool idle = q0 + (16 * w) / p.gpack >= n;            // wave-uniform: all rows beyond the chunk's end
    const int wave_lo = idle ? INT32_MAX : wave_min(sees ? lo : INT32_MAX), wave_hi = idle ? 0 : -wave_min(sees ? -hi : 0);
    const int full_lo = -wave_min(sees ? -lo : -INT32_MAX), full_hi = wave_min(hi);
    if (lane == 0) { span[0][w] = wave_lo; span[1][w] = wave_hi; }
    __syncthreads();
    int kv_lo = min(min(span[0][0], span[0][1]), min(span[0][2], span[0][3]));
    int kv_hi = max(max(span[1][0], span[1][1]), max(span[1][2], span[1][3]));
    kv_lo = __builtin_amdgcn_readfirstlane(kv_lo);
    kv_hi = __builtin_amdgcn_readfirstlane(kv_hi);
    int t_first = kv_lo / KT, t_end = (kv_hi + KT - 1) / KT;
    const bool divided = p.parts > 1;
    if (divided) {
        const int per = max((t_end - t_first + p.parts - 1) / p.parts, PART_KEYS / KT);
        t_end -= part * per;
        t_first = max(t_first, t_end - per);
    }
    if (kv_lo >= kv_hi || t_first >= t_end) {                  // nothing visible to any row: zero rows
        for (int i = tid; divided && i < 64; i += 256) {
            const int at = q0 + i / p.gpack;
            if (at < n) p.ws_ml[(part * p.rows + q_begin + at) * p.hq + hgroup * p.gpack + i % p.gpack] = make_float2(NEG_BIG, 0.f);
        }
        for (int i = tid; !divided && i < 64 * CPR; i += 256) {
            const int r = i / CPR, at = q0 + r / p.gpack;
            if (at < n)
                *(f32x4_t*)((float*)p.out + ((int64_t)(q_begin + at) * p.hq + hgroup * p.gpack + r % p.gpack) * DH + 4 * (i % CPR)) =
                    f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
        return;
    }

    // Q as the B operand: MFMA 4 q + e takes element 16 q + 4 g4 + e of this lane's row
    const float* qrow = (const float*)p.query + ((int64_t)(q_begin + pos - prior) * p.hq + head) * DH + 4 * g4;
    f32x4_t qf[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) qf[q] = *(const f32x4_t*)(qrow + 16 * q);
    const float mul = CAP ? p.rule.cap_mul : p.rule.mul, cap = p.rule.cap_log2;
    const float slope = BIAS ? p.rule.slopes[head] * LOG2E : 0.f;

    // m: the reference that exponents are taken against; 0 until the row has seen a key (fresh)
    float m = 0.f, lsum = 0.f;
    bool fresh = true;
    f32x4_t O[NQ];
#pragma unroll
    for (int j = 0; j < NQ; ++j) O[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    // Wave w brings in rows 8 w .. of a tile, 1 KB per instruction.  Slot s of K's row r holds chunk s ^ (r % 16).
    constexpr int RPI = 1024 / KROW, NI = 8 / RPI;
    const uint32_t blk_stride = (uint32_t)p.hkv * (BS * KROW);
    const char* kp = (const char*)p.k_pool + (int64_t)kvh * (BS * KROW);
    const char* vp = (const char*)p.v_pool + (int64_t)kvh * (BS * KROW);
    const int lrow = lane / CPR, lslot = lane % CPR;
    const int32_t* table = p.block_table + (int64_t)seq * p.block_table_stride;
    auto fetch = [&](int t, unsigned char* kb, unsigned char* vb) __attribute__((always_inline)) {
        const bool inside = t * KT >= kv_lo && (t + 1) * KT <= kv_hi;  // workgroup-uniform
        const int blk_of = inside ? table[(KT / BS) * t + (w >> 1)] : 0;
        const uint64_t block = (uint64_t)min((uint32_t)max(blk_of, 0), (uint32_t)(p.num_blocks - 1)) * blk_stride;
#pragma unroll
        for (int q = 0; q < NI; ++q) {
            const int r = 8 * (w & 1) + RPI * q + lrow;                // of its block
            uint64_t at = block + r * KROW;
            if (!inside) {                                             // rows that nobody here sees take the nearest one that somebody does
                const int tok = max(kv_lo, min(KT * t + 16 * (w >> 1) + r, kv_hi - 1));
                at = (uint64_t)min((uint32_t)max(table[tok / BS], 0), (uint32_t)(p.num_blocks - 1)) * blk_stride + (tok % BS) * KROW;
            }
            __builtin_amdgcn_global_load_lds(GLOBAL_PTR(kp + at + ((lslot ^ r) << 4)), LDS_PTR(kb + (8 * w + RPI * q) * KROW), 16, 0, 0);
            __builtin_amdgcn_global_load_lds(GLOBAL_PTR(vp + at + (lslot << 4)), LDS_PTR(vb + (8 * w + RPI * q) * KROW), 16, 0, 0);
        }
    };

    auto compute = [&](int t, const unsigned char* kb, const unsigned char* vb) __attribute__((always_inline)) {
        const int start = t * KT;
        if (start >= wave_hi || start + KT <= wave_lo) return;         // wave-uniform
        f32x4_t sa[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            f32x4_t ka[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) ka[h] = *(const f32x4_t*)(kb + (16 * h + r16) * KROW + (((4 * q + g4) ^ r16) << 4));
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int h = 0; h < 2; ++h) sa[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(ka[h][e], qf[q][e], sa[h], 0, 0, 0);
        }
        float pr[8], sc[8];
        float alpha = 1.f;
        bool grew;
        auto softmax = [&](auto mask_tag) __attribute__((always_inline)) {
            constexpr bool MASK = decltype(mask_tag)::value;
            bool dead[8];
            const float dist = (float)(start + 4 * g4 - pos);          // score k is of key start + 4 g4 + 16 (k / 4) + k % 4
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int r = 16 * (k >> 2) + (k & 3);
                float x = sa[k >> 2][k & 3] * mul;
                if constexpr (CAP) x = cap * tanhf(x);
                if constexpr (BIAS) x = fmaf(-slope, fabsf(dist + (float)r), x);
                dead[k] = MASK && (uint32_t)(start + 4 * g4 - lo + r) >= (uint32_t)(hi - lo);
                sc[k] = MASK && dead[k] ? NEG_BIG : x - m;
            }
            float psum = 0.f;
            auto exps = [&]() {
                psum = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    pr[k] = __builtin_amdgcn_exp2f(sc[k]);
                    if (MASK && dead[k]) pr[k] = 0.f;
                    psum += pr[k];
                }
            };
            exps();
            // the reference moves where a lane's sum outgrows 2^8, for the wave together; a fresh row takes its first maximum
            grew = __any(fresh || !(psum <= 256.f));
            if (grew) {
                float mx = sc[0];
#pragma unroll
                for (int k = 1; k < 8; ++k) mx = fmaxf(mx, sc[k]);
                mx = xor32_max(xor16_max(mx));
                const bool live = mx > 0.5f * NEG_BIG;
                const float shift = live && (fresh || mx > 0.f) ? mx : 0.f;
                alpha = fresh ? 0.f : __builtin_amdgcn_exp2f(-shift);
                fresh = fresh && !live;
                m += shift;
                lsum *= alpha;
#pragma unroll
                for (int k = 0; k < 8; ++k) sc[k] -= shift;
                exps();
            }
            lsum += psum;
        };
        if (start < full_lo || start + KT > full_hi) softmax(std::true_type{}); else softmax(std::false_type{});
        if (grew) {
#pragma unroll
            for (int j = 0; j < NQ; ++j) O[j] *= alpha;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            f32x4_t va[NF];
#pragma unroll
            for (int f = 0; f < NF; ++f)
                va[f] = *(const f32x4_t*)(vb + (16 * (k >> 2) + 4 * g4 + (k & 3)) * KROW + 256 * f + 16 * r16);
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int x = 0; x < 4; ++x) O[4 * f + x] = __builtin_amdgcn_mfma_f32_16x16x4f32(va[f][x], pr[k], O[4 * f + x], 0, 0, 0);
        }
    };

    // Opens the step of tile t: it is in LDS afterwards for every wave, and the next one is on its way into the other pair.
    auto open = [&](int t, unsigned char* kn, unsigned char* vn) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0x0F70);                    // vmcnt(0)
        __syncthreads();                                       // also: the tile before is no longer read by anyone
        if (t > t_first) fetch(t - 1, kn, vn);
    };
    __syncthreads();
    fetch(t_end - 1, k0, v0);
    for (int t = t_end - 1; t >= t_first; t -= 2) {
        open(t, k1, v1);
        compute(t, k0, v0);
        if (t > t_first) {
            open(t - 1, k0, v0);
            compute(t - 1, k1, v1);
        }
    }

    // lane (column r16, g4) holds element 64 f + 16 g4 + 4 i + x of its row in O[4 f + x][i]
    float l = lsum;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    float worst = 0.f;                                                 // (0 times a value that is not finite is not a number)
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) worst = fmaf(0.f, O[j][i], worst);
    uint64_t again = __ballot(row_valid && sees && l - l == 0.f && !(worst == 0.f));
    again |= again >> 32;
    again = (again | (again >> 16)) & 0xffff;                          // rows, by column
    if (row_valid && !((again >> r16) & 1)) {
        const int64_t at = (int64_t)(q_begin + pos - prior) * p.hq + head, slot = part * p.rows * p.hq + at;
        if (divided && g4 == 0) p.ws_ml[slot] = make_float2(m, l);
        float* o = divided ? p.ws_acc + slot * DH : (float*)p.out + at * DH;
        const bool none = l == 0.f;                                    // (no visible key, or all of weight 0)
        const float inv = divided ? 1.f : 1.f / l;
        if (!(divided && none)) {
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4_t x = {O[4 * f][i], O[4 * f + 1][i], O[4 * f + 2][i], O[4 * f + 3][i]};
                    *(f32x4_t*)(o + 64 * f + 16 * g4 + 4 * i) = none ? f32x4_t{0.f, 0.f, 0.f, 0.f} : x * inv;
                }
        }
    }
    if (divided) {
        lo = max(lo, t_first * KT);
        hi = min(hi, t_end * KT);
    }
    for (; again; again &= again - 1) {                                // wave-uniform
        const int r = __builtin_ctzll(again);
        const int at = __builtin_amdgcn_readlane(pos, r);
        score_row<F32Fmt, false, DH, true>(p, seq, q_begin + at - prior, __builtin_amdgcn_readlane(head, r), kvh, at,
                                           __builtin_amdgcn_readlane(lo, r), __builtin_amdgcn_readlane(hi, r), part, lane);
    }
}

template <int DH>
void launch_rule_f32(const ScorePrefillParams& p, bool cap, bool bias, dim3 grid, hipStream_t stream) {
    if (cap && bias) hipLaunchKernelGGL((score_prefill_f32_kernel<DH, true, true>), grid, dim3(256), 0, stream, p);
    else if (cap) hipLaunchKernelGGL((score_prefill_f32_kernel<DH, true, false>), grid, dim3(256), 0, stream, p);
    else if (bias) hipLaunchKernelGGL((score_prefill_f32_kernel<DH, false, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((score_prefill_f32_kernel<DH, false, false>), grid, dim3(256), 0, stream, p);
}

}  // namespace

int launch_score_prefill_f32(const ScoreArgs& a) {
    const ScorePrefillParams p = chunk_params(a);
    const int pos_per_wg = 64 / p.gpack;
    const dim3 grid((unsigned)(p.hgroups * p.parts), (unsigned)a.num_seqs, (unsigned)((a.max_q_len + pos_per_wg - 1) / pos_per_wg));
    const bool cap = a.cap > 0.f, bias = a.slopes != nullptr;
    if (a.d == 64) launch_rule_f32<64>(p, cap, bias, grid, a.stream);
    else if (a.d == 128) launch_rule_f32<128>(p, cap, bias, grid, a.stream);
    else launch_rule_f32<256>(p, cap, bias, grid, a.stream);
    if (p.parts > 1) launch_join<F32Fmt>(p, a);
    AICOMP_HIP_LAUNCH_CHECK();
    return AICOMP_KV_OK;
}

}  // namespace aicomp
