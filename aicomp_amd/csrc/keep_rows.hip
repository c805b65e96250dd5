// The cache rows of accepted drafts moved together, in every pool of every layer by one launch: in sequence s, the row of token
// first[s] + keep[i] becomes that of token first[s] + i, for the entries cu_keep[s] <= ... < cu_keep[s + 1], which ascend.
//
// keep ascends from 0 or more, so keep[i] >= i: the target of an entry lies below the sources of all later ones.  A thread that
// takes one 16-byte column of the rows through the entries in order therefore never overwrites what it still has to read, and no
// two threads touch a byte in common: no scratch, no barrier.  Four entries are read before the first of them is written, so that
// the chain of a sequence is a quarter of its entries.
//
// A copy of pieces of some hundred bytes: bound by the launch and by four dependent loads for one sequence, by them and the pieces' places
// all over HBM for many.  One sequence, 4 of 9 drafts in 64 pools: 5.3 us; 64 sequences, 8 of 32 in 32 pools: 18.8 us, 3.1 TB/s (one pool to
// a workgroup 20.9, two 19.9; eight entries at a time 20.8).
#include "row_attn.h"

#include <algorithm>

namespace aicomp {

namespace {

constexpr int MAX_POOLS = 128;             // per launch: 1 KB of arguments
constexpr int AHEAD = 4;
constexpr int TOGETHER = 4;                // pools of a workgroup, which looks the rows' places up once

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct KeepParams {
    void* pools[MAX_POOLS];
    const int32_t* block_table;
    int64_t block_table_stride, num_blocks, total;
    const int32_t* first;
    const int32_t* keep;
    const int32_t* cu_keep;
    int vecs;                              // vectors per row of one head
    int hkv, bs, max_blocks;
};

// Workgroup (sequence, four pools, slice of the row's vectors); V = the widest vector that the rows and the pools' alignment allow
template <typename V>
__global__ void __launch_bounds__(128)
keep_rows_kernel(KeepParams p) {
    const int seq = blockIdx.x;
    const int begin = max(0, p.cu_keep[seq]), end = (int)min((int64_t)p.cu_keep[seq + 1], p.total);
    const int col = blockIdx.z * 128 + threadIdx.x;
    if (col >= p.hkv * p.vecs) return;
    const int head = col / p.vecs, v = col - head * p.vecs;
    // (behind the last pool it is there again: the same thread then reads and writes the same twice)
    V* pool[TOGETHER];
#pragma unroll
    for (int j = 0; j < TOGETHER; ++j) pool[j] = (V*)p.pools[blockIdx.y * TOGETHER + j];
    const int32_t* table = p.block_table + seq * p.block_table_stride;
    const int64_t first = p.first[seq], limit = (int64_t)p.max_blocks * p.bs;
    // the vector of a token of this sequence, -1 where it has none
    auto at = [&](int64_t token) -> int64_t {
        if (token < 0 || token >= limit) return -1;
        const uint32_t entry = (uint32_t)token / (uint32_t)p.bs;            // (64-bit divisions: 3 of 21 us)
        const int64_t blk = table[entry];
        if (blk < 0 || blk >= p.num_blocks) return -1;
        return ((blk * p.hkv + head) * p.bs + ((uint32_t)token - entry * p.bs)) * p.vecs + v;
    };
    for (int i = begin; i < end; i += AHEAD) {
        int64_t from[AHEAD], to[AHEAD];
        V held[TOGETHER][AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            from[k] = i + k < end ? at(first + p.keep[i + k]) : -1;
            to[k] = i + k < end ? at(first + (i + k - begin)) : -1;
            if (from[k] >= 0) {
#pragma unroll
                for (int j = 0; j < TOGETHER; ++j) held[j][k] = pool[j][from[k]];
            }
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (from[k] >= 0 && to[k] >= 0 && from[k] != to[k]) {
#pragma unroll
                for (int j = 0; j < TOGETHER; ++j) pool[j][to[k]] = held[j][k];
            }
    }
}

}  // namespace

int launch_keep_rows(const KeepRowsArgs& a) {
    uintptr_t all = (uintptr_t)a.row_bytes;
    for (int i = 0; i < a.num_pools; ++i) all |= (uintptr_t)a.pools[i];
    const int width = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    const int64_t cols = a.row_bytes / width * a.hkv, slices = (cols + 127) / 128;
    AICOMP_REQUIRE(slices <= 65535, AICOMP_KV_EINVAL, "keep_rows: rows of %lld bytes in %d heads exceed one launch",
                   (long long)a.row_bytes, a.hkv);
    KeepParams p;
    p.block_table = a.block_table; p.block_table_stride = a.block_table_stride; p.num_blocks = a.num_blocks; p.total = a.total;
    p.first = a.first; p.keep = a.keep; p.cu_keep = a.cu_keep;
    p.vecs = (int)(a.row_bytes / width); p.hkv = a.hkv; p.bs = a.bs; p.max_blocks = a.max_blocks;
    for (int first = 0; first < a.num_pools; first += MAX_POOLS) {
        const int n = std::min(a.num_pools - first, MAX_POOLS);
        for (int i = 0; i < MAX_POOLS; ++i) p.pools[i] = a.pools[first + std::min(i, n - 1)];
        const dim3 grid((unsigned)a.num_seqs, (unsigned)((n + TOGETHER - 1) / TOGETHER), (unsigned)slices);
        if (width == 16) hipLaunchKernelGGL(keep_rows_kernel<u32x4>, grid, dim3(128), 0, a.stream, p);
        else if (width == 4) hipLaunchKernelGGL(keep_rows_kernel<uint32_t>, grid, dim3(128), 0, a.stream, p);
        else hipLaunchKernelGGL(keep_rows_kernel<uint8_t>, grid, dim3(128), 0, a.stream, p);
        AICOMP_HIP_LAUNCH_CHECK();
    }
    return AICOMP_KV_OK;
}

}  // namespace aicomp
