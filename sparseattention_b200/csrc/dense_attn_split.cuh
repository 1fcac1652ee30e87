// Ranges: an item whose loop is long, where there are few items, is cut into ranges that run as separate blocks and leave 32-bit
// partial results in a workspace; a second kernel joins them in their order.
#pragma once

#include "dense_attn.cuh"
#include "tc_common.cuh"
#include "tma_common.cuh"

namespace hsa {

struct DenseSplit {
    float *part_o, *part_ml;                     // [splits, B, Lq, H, D] and [splits, B, Lq, H, 2] (maximum in base 2, sum) when splits > 1
    int splits;
    unsigned int extra_tx;                       // test hook: bytes that the first copy is announced with and never brings
    long long wait_limit;
};
struct BwdSplit {
    float *part;                                 // [splits][B, rows, heads, D], dk before dv, when splits > 1
    int splits;
    unsigned int extra_tx;
    long long wait_limit;
};

// Ranges per work item when there are few items and each is long: the count that lets the slowest SM finish first.  `steps` tiles per
// item; an item costs `once` tiles' time besides, `once_split` as one of several ranges, whose partial results are then joined.
inline int range_count(long long items, int steps, double once, double once_split) {
    const int sms = dense_sm_count();
    if (items * 2 > sms || steps < 2) return 1;
    double best = 1e30;
    int best_s = 1;
    for (int s = 1; s <= 64 && s <= steps; ++s) {
        const double waves = (double)((items * s + sms - 1) / sms);
        const double t = waves * ((steps + s - 1) / s + (s > 1 ? once_split : once)) + (s > 1 ? once : 0.0);
        if (t < 0.95 * best) { best = t; best_s = s; }
    }
    const int per = (steps + best_s - 1) / best_s;
    return (steps + per - 1) / per;
}

inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }
inline size_t fwd_part_bytes(int splits, int B, int Lq, int H, int D) {
    return splits > 1 ? (size_t)splits * B * Lq * H * (D + 2) * sizeof(float) : 0;
}
inline size_t bwd_part_bytes(int sq, int sk, int B, int Lq, int Lk, int H, int Hkv, int D) {
    size_t n = 0;
    if (sq > 1) n += up256((size_t)sq * B * Lq * H * D * sizeof(float));
    if (sk > 1) n += up256((size_t)2 * sk * B * Lk * Hkv * D * sizeof(float));
    return n;
}
inline DenseSplit fwd_split(int splits, const DenseArgs &a, void *workspace) {
    DenseSplit sp{};
    sp.splits = splits;
    sp.part_o = (float *)workspace;
    if (splits > 1) sp.part_ml = sp.part_o + (size_t)splits * a.B * a.Lq * a.H * a.D;
    sp.wait_limit = wait_limit_cycles();
    sp.extra_tx = wait_extra_tx();
    return sp;
}
inline void bwd_splits(int nq, int nk, const DenseArgs &a, void *workspace, BwdSplit &sq, BwdSplit &sk) {
    sq.splits = nq;
    sk.splits = nk;
    sq.part = (float *)workspace;
    sk.part = (float *)((char *)workspace + (nq > 1 ? up256((size_t)nq * a.B * a.Lq * a.H * a.D * sizeof(float)) : 0));
    sq.wait_limit = sk.wait_limit = wait_limit_cycles();
    sq.extra_tx = sk.extra_tx = wait_extra_tx();
}

template <typename T>
__device__ __forceinline__ float rounding_rest(float x) { return x - Traits<T>::to_f(Traits<T>::from_f(x)); }

template <typename T>
__device__ __forceinline__ void store4(T *p, float x, float y, float z, float w, bool vec) {
    if constexpr (sizeof(T) == 4) {
        if (vec) { *reinterpret_cast<float4 *>(p) = make_float4(x, y, z, w); return; }
    } else {
        if (vec) { *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<T>(x, y), pack2<T>(z, w)); return; }
    }
    p[0] = Traits<T>::from_f(x); p[1] = Traits<T>::from_f(y); p[2] = Traits<T>::from_f(z); p[3] = Traits<T>::from_f(w);
}

// A query row per warp: out = sum 2^(m_s - M) o_s / sum 2^(m_s - M) l_s
template <typename T>
__global__ void __launch_bounds__(128) dense_join_kernel(const DenseArgs a, const DenseSplit sp) {
    const int64_t rows = (int64_t)a.B * a.Lq * a.H, row = blockIdx.x * 4LL + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= rows) return;
    float M = -INFINITY;
    for (int s = 0; s < sp.splits; ++s) M = fmaxf(M, sp.part_ml[2 * (s * rows + row)]);
    const float ref = M == -INFINITY ? 0.f : M;
    const int h = (int)(row % a.H), i = (int)(row / a.H % a.Lq);
    const int64_t b = row / a.H / a.Lq;
    T *out = (T *)a.out.ptr + b * a.out.batch_stride + (int64_t)i * a.out.row_stride + (int64_t)h * a.D;
    for (int c = lane * 4; c < a.D; c += 128) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float L = 0.f;
#pragma unroll 4
        for (int s = 0; s < sp.splits; ++s) {
            const int64_t at = s * rows + row;
            const float w = exp2f(sp.part_ml[2 * at] - ref);       // 0 for a range without keys
            L = fmaf(w, sp.part_ml[2 * at + 1], L);
            const float4 o = *reinterpret_cast<const float4 *>(sp.part_o + at * a.D + c);
            acc.x = fmaf(w, o.x, acc.x); acc.y = fmaf(w, o.y, acc.y); acc.z = fmaf(w, o.z, acc.z); acc.w = fmaf(w, o.w, acc.w);
        }
        const bool none = L == 0.f;
        const float inv = 1.f / L, e = a.empty_value;
        store4<T>(out + c, none ? e : acc.x * inv, none ? e : acc.y * inv, none ? e : acc.z * inv, none ? e : acc.w * inv, a.vec);
        if (a.out_lo != nullptr)                                   // packed, and D a multiple of four
            store4<T>((T *)a.out_lo + row * a.D + c, none ? 0.f : rounding_rest<T>(acc.x * inv), none ? 0.f : rounding_rest<T>(acc.y * inv),
                      none ? 0.f : rounding_rest<T>(acc.z * inv), none ? 0.f : rounding_rest<T>(acc.w * inv), true);
        if (a.lse != nullptr && c == 0) a.lse[row] = none ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
    }
}

// out = scale * sum over the ranges
template <typename T>
__global__ void __launch_bounds__(256) dense_grad_join_kernel(const float *__restrict__ part, int splits, int64_t slab, hsa_view out,
                                                             int rows, int row_elems, int64_t total, float scale, bool vec) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= total) return;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const float4 v = __ldg(reinterpret_cast<const float4 *>(part + s * slab + i));
        acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
    }
    const int64_t row = i / row_elems;
    T *o = (T *)out.ptr + (row / rows) * out.batch_stride + (row % rows) * out.row_stride + i % row_elems;
    store4<T>(o, acc.x * scale, acc.y * scale, acc.z * scale, acc.w * scale, vec);
}

template <typename T>
int join_forward(const DenseArgs &a, const DenseSplit &sp, cudaStream_t st) {
    const long long blocks = ((long long)a.B * a.Lq * a.H + 3) / 4;
    if (blocks > 0x7fffffffLL) return fail(HSA_ERR_ARG, "hsa_dense_attn_fwd: too many rows");
    dense_join_kernel<T><<<(unsigned)blocks, 128, 0, st>>>(a, sp);
    return launch_status("hsa_dense_attn_fwd(join)");
}
template <typename T>
int join_backward(const DenseArgs &a, const BwdSplit &sq, const BwdSplit &sk, cudaStream_t st) {
    auto join = [&](const float *part, int splits, int64_t elems, const hsa_view &out, int rows, int heads, float scale) -> int {
        const long long blocks = (elems / 4 + 255) / 256;
        if (blocks > 0x7fffffffLL) return fail(HSA_ERR_ARG, "hsa_dense_attn_bwd: too many rows");
        dense_grad_join_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(part, splits, elems, out, rows, heads * a.D, elems, scale, a.vec);
        return launch_status("hsa_dense_attn_bwd(join)");
    };
    const int64_t q_elems = (int64_t)a.B * a.Lq * a.H * a.D, k_elems = (int64_t)a.B * a.Lk * a.Hkv * a.D;
    if (sq.splits > 1 && a.dq.ptr != nullptr)
        if (int rc = join(sq.part, sq.splits, q_elems, a.dq, a.Lq, a.H, a.scale)) return rc;
    if (sk.splits > 1 && a.dk.ptr != nullptr) {
        if (int rc = join(sk.part, sk.splits, k_elems, a.dk, a.Lk, a.Hkv, a.scale)) return rc;
        return join(sk.part + sk.splits * k_elems, sk.splits, k_elems, a.dv, a.Lk, a.Hkv, 1.f);
    }
    return 0;
}

}  // namespace hsa
