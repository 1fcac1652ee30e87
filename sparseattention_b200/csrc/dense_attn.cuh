// Shared pieces of the dense attention kernels (queries of one sequence over the rows of another): launch arguments, the
// packed form of a mask, and which keys a batch entry has.
#pragma once

#include <math.h>

#include <atomic>

#include "hsa_common.cuh"

namespace hsa {

constexpr int kDenseTile = 128;          // keys and query rows per cell of the mask's tile table

// A mask [planes, rows, Lk] in bits.  One plane per (batch entry, head) that the mask tells apart, one row per query or one
// for all.  hsa_dense_mask_pack fills the arrays; their sizes follow from the mask's own sizes (dense_mask_layout).
struct DenseMask {
    const uint32_t *bits;                // [planes][rows][wk]: bit k of a row = the query may look at key k; bits >= Lk are 0
    const uint32_t *bits_t;              // [planes][Lk][wq]: the same, keys as rows (null when the mask has one row)
    const uint32_t *seen;                // [planes][wk]: keys that at least one query may look at
    const uint8_t *tiles;                // [planes][tq][tk] of 128 x 128 cells: 0 nothing allowed, 1 some, 2 everything
    int plane_b, plane_h;                // plane of (b, h) = b * plane_b + h * plane_h
    int rows;                            // 1 or Lq
    int wk, wq, tq, tk;
};

struct DenseMaskLayout {
    size_t bits, bits_t, seen, tiles, total;      // byte offsets
    int wk, wq, tq, tk;
};
inline DenseMaskLayout dense_mask_layout(long long planes, int rows, int Lk) {
    DenseMaskLayout l{};
    l.tk = (Lk + kDenseTile - 1) / kDenseTile;
    l.tq = (rows + kDenseTile - 1) / kDenseTile;
    l.wk = l.tk * 4;
    l.wq = rows > 1 ? l.tq * 4 : 0;
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    size_t at = 0;
    l.bits = at;
    at = up(at + (size_t)planes * rows * l.wk * 4);
    l.bits_t = at;
    if (rows > 1) at = up(at + (size_t)planes * Lk * l.wq * 4);
    l.seen = at;
    if (rows > 1) at = up(at + (size_t)planes * l.wk * 4); else l.seen = l.bits;
    l.tiles = at;
    at = up(at + (size_t)planes * l.tq * l.tk);
    l.total = at;
    return l;
}

inline DenseMask dense_mask_view(const void *packed, int Bm, int Hm, int rows, int Lk) {
    DenseMask m{};
    if (packed == nullptr) return m;
    const DenseMaskLayout l = dense_mask_layout((long long)Bm * Hm, rows, Lk);
    const char *p = (const char *)packed;
    m.bits = (const uint32_t *)(p + l.bits);
    m.bits_t = rows > 1 ? (const uint32_t *)(p + l.bits_t) : nullptr;
    m.seen = (const uint32_t *)(p + l.seen);
    m.tiles = (const uint8_t *)(p + l.tiles);
    m.plane_b = Bm > 1 ? Hm : 0;
    m.plane_h = Hm > 1 ? 1 : 0;
    m.rows = rows;
    m.wk = l.wk; m.wq = l.wq; m.tq = l.tq; m.tk = l.tk;
    return m;
}

struct DenseArgs {
    hsa_view q, k, v, out, dout, dq, dk, dv;
    float *lse;                          // forward: [B, Lq, H] natural log-sum-exp, or null
    void *out_lo;                        // [B, Lq, H, D] packed: what rounding took from the 16-bit output, in its type; or null
    const float *neg_lse2, *neg_delta;   // backward: [B, H, lq_pad] minus the log-sum-exp in base 2 (-inf: no key), minus the row sums of dout * out
    // backward on the tensor cores in f16 (kWeightShift is then part of neg_lse2): squared lengths of dout's rows [B, H, lq_pad], and the
    // largest of them and a bound on those of V's rows [B, Hkv, 2] as bit patterns
    const float *dout_sq;
    const unsigned int *top_sq;
    const int *key_lengths;              // [B] or null
    DenseMask mask;
    int B, Lq, Lk, H, Hkv, D, group;     // group = H / Hkv
    int lq_pad;                          // Lq rounded up to 128
    float scale, scale_log2;             // scale_log2 = scale * log2(e)
    float empty_value;                   // what the output row of a query without keys holds
    bool vec;                            // rows may be read four elements at a time
};

// float16 holds nothing between 0 and 2^-24, and full precision from 2^-14 only: weights near 1 / Lk, and score gradients, which are
// those times differences of the size of dout, would lose bits as operands or vanish while the sums over them do not.  So the
// backward's products take weights times 2^13 (the weights do not pass 1, but for the rounding of a large log-sum-exp), and score
// gradients times the power of two that a bound on them allows: ds_j = p_j sum_k p_k do.(v_j - v_k), so |ds_j| <= p_j (1 - p_j) 2 |do|
// max |v| <= |do| max |v| / 2.  What is multiplied by it does not pass 2^16 (and saturates there); the results are multiplied by the
// inverse, exactly.  (8192 keys, output gradients of 1e-3: dq off by 5.7e-3 of its size without this; 5.2e-4 is what rounding the
// result alone leaves.)  It costs a read of V next to the row sums and a clearing of the tops: backward of 3 x 515 x 1027, 12 on 4
// heads of 128, 98.6 us against 91.7; 2 x 4096 x 4096, 16 heads of 128, 799 against 792; most where few queries look at many keys, 2 x 33 x
// 30011, 16 heads of 128, 343 against 294.
constexpr int kWeightShift = 13;
__device__ __forceinline__ float grad_shift(float dout_sq, unsigned int v_sq_bits) {
    const float bound = 0.5f * sqrtf(dout_sq) * sqrtf(__uint_as_float(v_sq_bits));
    return bound > 0.f && bound < INFINITY ? (float)(15 - ilogbf(bound)) : 0.f;
}
// 2^e for whole e between -126 and 127
__device__ __forceinline__ float pow2(float e) { return __int_as_float(((int)e + 127) << 23); }

// Raise a kernel's shared-memory limit, once per device
template <auto Kernel>
cudaError_t allow_smem(int bytes) {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_release);
    return e;
}

// Strides of dimensions of one entry as a packed tensor would have them (nothing is addressed through them)
inline hsa_view dense_view(hsa_view v, int B, int rows, int H, int D) {
    if (rows == 1) v.row_stride = (int64_t)H * D;
    if (B == 1) v.batch_stride = (int64_t)rows * v.row_stride;
    return v;
}

inline int dense_sm_count() {
    int dev = 0, v = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) {
        (void)cudaGetLastError();
        return 148;
    }
    return v;
}

__device__ __forceinline__ int dense_keys(const DenseArgs &a, int b) {
    if (a.key_lengths == nullptr) return a.Lk;
    return max(0, min(a.Lk, __ldg(a.key_lengths + b)));      // lengths outside [0, Lk] mean the nearer end
}

}  // namespace hsa
