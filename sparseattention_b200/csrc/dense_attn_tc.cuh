// Pieces shared by the tensor-core kernels of dense attention.
#pragma once

#include "dense_attn_split.cuh"
#include "tc5_common.cuh"

namespace hsa {

constexpr int kFlagTiles = 768;                  // tiles whose mask state fits one of a block's two tables
// Two 32-bit numbers in a register pair: one instruction for both
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t pair_bits(uint32_t lo, uint32_t hi) { return pair(__uint_as_float(lo), __uint_as_float(hi)); }

// The largest of three; NaN if one of them is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// 2^x for both numbers of a pair without the special-function unit, x <= 15 (below -126: 2^-126).  x = n + f with n the nearest
// whole number (the addition of 1.5 * 2^23 leaves it in the low bits), |f| <= 1/2, 2^f by the degree-5 polynomial of least
// greatest relative error on that interval (found by exchange; 7.5e-8), and n goes into the exponent.  Off by at most 2^-22 in
// 32-bit arithmetic, as the special-function unit is.  NaN does not stay NaN (n added to its bits makes a finite number of them):
// callers take care of it.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
    x.x = fmaxf(x.x, -126.f);
    x.y = fmaxf(x.y, -126.f);
    const uint64_t x2 = pair(x.x, x.y);
    const uint64_t r = add2(x2, pair(12582912.f, 12582912.f));
    const uint64_t f = fma2(add2(r, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f), x2);
    uint64_t p = fma2(pair(0.00132764725f, 0.00132764725f), f, pair(0.00967554096f, 0.00967554096f));
    p = fma2(p, f, pair(0.0555071309f, 0.0555071309f));
    p = fma2(p, f, pair(0.240221202f, 0.240221202f));
    p = fma2(p, f, pair(0.693146944f, 0.693146944f));
    p = fma2(p, f, pair(1.00000012f, 1.00000012f));
    const float2 y = unpair(p), n = unpair(r);
    return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(n.x) << 23)),
                       __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(n.y) << 23)));
}

// The value of lane 0, which is every lane's: tells the compiler that what depends on it is the same in the whole warp.  The
// warps that issue products need that: with descriptors and loop state in uniform registers an issue takes 10 cycles, with
// per-lane ones 69 (and a commit 100), which bound all three kernels.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

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

// Every lane of a quad holds four 16-byte pieces of its own row; afterwards lane q holds piece q of the quad's four rows.  Four
// lanes then write 64 contiguous bytes of a row at a time, where a lane that writes its own row touches a line per lane (the
// output of a work item of 256 x 128 took 6300 cycles that way).
__device__ __forceinline__ void quad_pieces(uint4 (&p)[4], int quad) {
    uint32_t w[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) { w[0][t] = p[t].x; w[1][t] = p[t].y; w[2][t] = p[t].z; w[3][t] = p[t].w; }
#pragma unroll
    for (int e = 0; e < 4; ++e) quad_transpose4(w[e], quad);
#pragma unroll
    for (int t = 0; t < 4; ++t) p[t] = make_uint4(w[0][t], w[1][t], w[2][t], w[3][t]);
}
// A warp stores 32 consecutive columns of its 32 rows, as far as the head dim goes (a multiple of 8).  `row`: this lane's row,
// `below`: rows of the tensor from this one on (may be <= 0).
// REST: not the rounded values, but what rounding took from them.
template <typename T, bool REST = false>
__device__ __forceinline__ void store_rows32(T *row, int64_t row_stride, int below, int col, int D, const uint32_t (&v)[32], float scale) {
    const int quad = threadIdx.x & 3;
    uint4 p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x = __uint_as_float(v[8 * j + 2 * e]) * scale, y = __uint_as_float(v[8 * j + 2 * e + 1]) * scale;
            o[e] = REST ? pack2<T>(rounding_rest<T>(x), rounding_rest<T>(y)) : pack2<T>(x, y);
        }
        p[j] = make_uint4(o[0], o[1], o[2], o[3]);
    }
    quad_pieces(p, quad);
    if (col + 8 * quad >= D) return;
#pragma unroll
    for (int t = 0; t < 4; ++t)
        if (t - quad < below) *reinterpret_cast<uint4 *>(row + (t - quad) * row_stride + col + 8 * quad) = p[t];
}
__device__ __forceinline__ void scale_all(uint32_t (&v)[32], float by) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * by);
}
// The same for 32-bit rows.
__device__ __forceinline__ void store_rows32_f32(float *row, int64_t row_stride, int below, int col, int D, const uint32_t (&v)[32]) {
    const int quad = threadIdx.x & 3;
#pragma unroll
    for (int g = 0; g < 2; ++g) {                                        // 16 columns are four pieces
        uint4 p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = make_uint4(v[16 * g + 4 * j], v[16 * g + 4 * j + 1], v[16 * g + 4 * j + 2], v[16 * g + 4 * j + 3]);
        quad_pieces(p, quad);
        const int c = col + 16 * g + 4 * quad;
#pragma unroll
        for (int t = 0; t < 4; ++t)
            if (t - quad < below && c < D) *reinterpret_cast<uint4 *>(row + (t - quad) * row_stride + c) = p[t];
    }
}
template <typename T>
__device__ __forceinline__ void fill_row(T *row, int D, float value) {
    const uint32_t w = pack2<T>(value, value);
    for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4 *>(row + c) = make_uint4(w, w, w, w);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t mb) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(mb) : "memory");
}

// ------------------------------------------------------------------------------------------------------- work items
// The kernels are launched with one block per work item, but a running block takes over items whose block has not started
// (clusterlaunchcontrol.try_cancel): set-up is paid once per SM, copies and first products of the next item overlap the last
// softmax and the output of the current one, and items of unequal length balance themselves.  Only the copy warp asks; it
// hands the item's number (and the mask states of its tiles) to the other warps through two slots in shared memory.
__device__ __forceinline__ void take_over(uint32_t response, uint32_t mb) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n" ::"r"(response), "r"(mb) : "memory");
}
// The block number that was taken over, or -1
__device__ __forceinline__ int taken_over(uint32_t response) {
    int item;
    asm volatile("{\n.reg .pred p;\n.reg .b128 r;\nld.shared.b128 r, [%1];\n"
                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\nmov.b32 %0, -1;\n"
                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n}\n"
                 : "=r"(item) : "r"(response) : "memory");
    tc5::fence_async_smem();                          // read before the next answer lands
    return item;
}

// A wait of its own limit, for a block that has given up
__device__ __forceinline__ bool mbar_wait_limited(uint32_t mb, uint32_t parity, long long limit) {
    const long long start = clock64();
    while (!tc5::mbar_try(mb, parity))
        if (clock64() - start > limit) return false;
    return true;
}

// Shared-memory side of it; barriers: info_full[2], info_empty[2], answer.
struct ItemSlots {
    int item[2];
    int closed;                          // -1; in a block that has given up, how many items the copy warp has handed on
    int pad;
    uint4 answer;
    uint8_t flags[2][kFlagTiles];
};
constexpr int kItemBars = 5;

// In a block that has given up every item it holds must still be answered for, since a block number that was taken over runs
// nowhere else.  The element-wise warps void the one they could not finish and those that the copy warp had handed on
// already (`handed_on`, place k of the sequence); the copy warp hands on no more (`close_items`) and voids the one that is then
// still on its way (`item_on_its_way`: in its hand, or in an answer that it waits for).
constexpr long long kGiveUpCycles = 20000000;                    // each of these waits ends by itself in microseconds
__device__ __forceinline__ bool handed_on(ItemSlots &items, uint32_t mb, int k) {
    const volatile int *closed = &items.closed;
    const long long start = clock64();
    bool there;
    while (!(there = tc5::mbar_try(mb, (k >> 1) & 1))) {
        const int n = *closed;
        if ((n >= 0 && k >= n) || clock64() - start > kGiveUpCycles) break;
    }
    return __all_sync(0xffffffffu, there);
}
__device__ __forceinline__ void close_items(ItemSlots &items, int count, int lane) {
    __syncwarp();
    if (lane == 0) *const_cast<volatile int *>(&items.closed) = count;
    __syncwarp();
}
__device__ __forceinline__ int item_on_its_way(ItemSlots &items, bool asked, uint32_t answer, int k, int in_hand) {
    if (!asked) return in_hand;
    const bool there = __all_sync(0xffffffffu, mbar_wait_limited(answer, k & 1, kGiveUpCycles));
    return there ? taken_over(smem_u32(&items.answer)) : -1;
}

}  // namespace hsa
