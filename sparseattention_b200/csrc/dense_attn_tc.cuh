// Pieces shared by the tensor-core kernels of dense attention.
#pragma once

#include "dense_attn.cuh"
#include "tc5_common.cuh"
#include "tc_common.cuh"
#include "tma_common.cuh"

namespace hsa {

constexpr int kFlagTiles = 1024;                 // tiles whose mask state fits a block's table
constexpr int kTcThreads = 320;                  // eight warps for the element-wise part, one for copies, one for products

// Bit words of the keys [32 w, 32 w + 32) of a tile: those before `left` (keys of the sequence that remain)
__device__ __forceinline__ uint32_t tail_word(int left, int w) {
    const int c = left - 32 * w;
    return c >= 32 ? 0xffffffffu : c <= 0 ? 0u : (1u << c) - 1u;
}

// Zero the rows of a staged tile of 128 keys ([PLANES][128 rows][128 bytes]) that stand for keys which are not there: behind the
// sequence's length, or hidden from every query.  One whole warp; the tensor cores may read the tile afterwards.
template <int PLANES>
__device__ __forceinline__ void zero_hidden_rows(unsigned char *tile, int left, const uint32_t *seen, int lane) {
    uint32_t word[4];
    bool all = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        word[i] = tail_word(left, i);
        if (seen != nullptr) word[i] &= __ldg(seen + i);
        all = all && word[i] == 0xffffffffu;
    }
    if (all) return;
#pragma unroll 4
    for (int g = 0; g < 32; ++g) {
        const int r = g * 4 + (lane >> 3);
        const uint32_t w = g < 8 ? word[0] : g < 16 ? word[1] : g < 24 ? word[2] : word[3];
        if (!((w >> (r & 31)) & 1u)) {
#pragma unroll
            for (int p = 0; p < PLANES; ++p)
                *reinterpret_cast<uint4 *>(tile + p * 16384 + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
    }
    tc5::fence_async_smem();
    __syncwarp();
}

// Four 16-byte pieces (32 columns) of a row of a staged output tile ([planes][128 rows][128 bytes], 128-byte swizzle).
template <typename T>
__device__ __forceinline__ void stage_row32(unsigned char *tile, int row, int c32, const uint32_t (&v)[32], float scale) {
    unsigned char *line = tile + (c32 >> 1) * 16384 + row * 128;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            o[e] = pack2<T>(__uint_as_float(v[8 * j + 2 * e]) * scale, __uint_as_float(v[8 * j + 2 * e + 1]) * scale);
        *reinterpret_cast<uint4 *>(line + ((((c32 & 1) * 4 + j) ^ (row & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t mb) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(mb) : "memory");
}
__device__ __forceinline__ void bulk_store_done() {
    asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
    asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
}

}  // namespace hsa
