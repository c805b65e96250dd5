// Blocks of the paged pools copied, in every pool of every layer by one launch: pool[dst] = pool[src].
//
// What forking a sequence (its last, partly filled block; full ones are shared) and compacting a pool come to.  A block of
// one pool is one contiguous piece of Hkv * block_size * D elements, so the copy is bound by HBM, and for a fork, a
// piece of some KB per pool, by the launch: the pools' addresses travel in the kernel's arguments.
//
// One block in each of 64 pools (2 MB): 2.3 us on the device (10 with uint4 as the vector, whose array the compiler moves to LDS, the
// workgroup's shape being read from host memory for it).  500 pairs in each of 32 pools, 1.05 GB read and written: 188 us, 5.6 TB/s
// (198 without the nontemporal hint: nothing here is read again).
#include "common.h"

#include <algorithm>

namespace aicomp {

namespace {

constexpr int MAX_POOLS = 128;             // per launch: 1 KB of arguments
constexpr int UNROLL = 4;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct CopyParams {
    void* pools[MAX_POOLS];
    const int64_t* pairs;
    int64_t vecs;                          // vectors per block
    int64_t num_blocks;
    uint32_t pieces;                       // workgroups per block
};

// V = the widest vector that block_bytes and the pools' alignment allow
template <typename V>
__global__ void __launch_bounds__(256)
copy_blocks_kernel(CopyParams p) {
    const uint32_t pair = blockIdx.x / p.pieces, piece = blockIdx.x - pair * p.pieces;
    const int64_t src = p.pairs[2 * (int64_t)pair], dst = p.pairs[2 * (int64_t)pair + 1];
    if (src < 0 || src >= p.num_blocks || dst < 0 || dst >= p.num_blocks || src == dst) return;
    V* pool = (V*)p.pools[blockIdx.y];
    const V* from = pool + src * p.vecs;
    V* to = pool + dst * p.vecs;
    const int64_t i0 = (int64_t)piece * (256 * UNROLL) + threadIdx.x;
    if (i0 + 256 * (UNROLL - 1) < p.vecs) {
        V r[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) r[u] = __builtin_nontemporal_load(from + i0 + 256 * u);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) __builtin_nontemporal_store(r[u], to + i0 + 256 * u);
    } else {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (i0 + 256 * u < p.vecs) __builtin_nontemporal_store(__builtin_nontemporal_load(from + i0 + 256 * u), to + i0 + 256 * u);
    }
}

}  // namespace

int launch_copy_blocks(void* const* pools, int num_pools, int64_t block_bytes, int64_t num_blocks, const int64_t* pairs,
                       int64_t num_pairs, hipStream_t stream) {
    uintptr_t all = (uintptr_t)block_bytes;
    for (int i = 0; i < num_pools; ++i) all |= (uintptr_t)pools[i];
    const int width = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    CopyParams p;
    p.vecs = block_bytes / width;
    p.num_blocks = num_blocks;
    const int64_t pieces = (p.vecs + 256 * UNROLL - 1) / (256 * UNROLL);
    // (a launch dimension holds less than 2^32 lanes)
    const int64_t per_launch = ((int64_t)UINT32_MAX / 256) / pieces;
    AICOMP_REQUIRE(per_launch > 0, AICOMP_KV_EINVAL, "copy_blocks: blocks of %lld bytes exceed one launch", (long long)block_bytes);
    p.pieces = (uint32_t)pieces;
    for (int first = 0; first < num_pools; first += MAX_POOLS) {
        const int n = std::min(num_pools - first, MAX_POOLS);
        for (int i = 0; i < MAX_POOLS; ++i) p.pools[i] = pools[first + std::min(i, n - 1)];
        for (int64_t k = 0; k < num_pairs; k += per_launch) {
            p.pairs = pairs + 2 * k;
            dim3 grid((unsigned)(std::min(num_pairs - k, per_launch) * pieces), (unsigned)n);
            if (width == 16) hipLaunchKernelGGL(copy_blocks_kernel<u32x4>, grid, dim3(256), 0, stream, p);
            else if (width == 4) hipLaunchKernelGGL(copy_blocks_kernel<uint32_t>, grid, dim3(256), 0, stream, p);
            else hipLaunchKernelGGL(copy_blocks_kernel<uint8_t>, grid, dim3(256), 0, stream, p);
            AICOMP_HIP_LAUNCH_CHECK();
        }
    }
    return AICOMP_KV_OK;
}

}  // namespace aicomp
