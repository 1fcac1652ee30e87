// Dense attention on the CUDA cores: float32 inputs, head dims the tensor-core kernels do not take, unaligned rows.
//
//   p[i, j] = exp2(c q_i.k_j - m_i) / l_i,   out_i = sum_j p[i, j] v_j,     c = scale * log2(e)
//   dv_j = sum_i p[i, j] do_i,   ds[i, j] = p[i, j] (do_i.v_j - sum_d do_i out_i),   dq_i = scale sum_j ds[i, j] k_j,
//   dk_j = scale sum_i ds[i, j] q_i
//
// A block of 16 x 16 threads owns a tile of queries (forward, dq) or of keys (dk, dv) and walks over tiles of the other side,
// everything in float32 in shared memory.  A thread owns rows ty, ty + 16, ... of the score tile and columns tx, tx + 16, ...:
// the 16 lanes that share a row are half a warp, so row sums are shuffles and the weights pass between the two products with
// a warp barrier only.  Every operand row is padded by four floats, which makes the 16-byte reads free of bank conflicts.
// One writer per output row, fixed order of summation.  Keys behind a sequence's length, and keys that no query may look
// at, are stored as zeros: what lies there (NaN, infinities) cannot reach a result through 0 * x.
#include "dense_attn.cuh"

namespace hsa {

constexpr int kSimtThreads = 256;

// rows row0 .. row0 + ROWS - 1 of a [rows, D] matrix as float32 into dst[ROWS][DP + 4]; rows >= limit, rows whose bit in `seen`
// is clear and columns >= D are zeros
template <typename T, int ROWS, int DP>
__device__ __forceinline__ void load_rows(float *dst, const T *base, int64_t row_stride, int row0, int limit, int D, bool vec,
                                          const uint32_t *seen) {
    constexpr int C4 = DP / 4;
    for (int idx = threadIdx.x; idx < ROWS * C4; idx += kSimtThreads) {
        const int r = idx / C4, c = (idx % C4) * 4, row = row0 + r;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row < limit && c < D && (seen == nullptr || ((seen[row >> 5] >> (row & 31)) & 1u))) {
            const T *p = base + (int64_t)row * row_stride + c;
            if (vec) {
                if constexpr (sizeof(T) == 4) {
                    v = *reinterpret_cast<const float4 *>(p);
                } else {
                    const uint2 raw = *reinterpret_cast<const uint2 *>(p);
                    const T *e = reinterpret_cast<const T *>(&raw);
                    v = make_float4(Traits<T>::to_f(e[0]), Traits<T>::to_f(e[1]), Traits<T>::to_f(e[2]), Traits<T>::to_f(e[3]));
                }
            } else {
                v.x = Traits<T>::to_f(p[0]);
                if (c + 1 < D) v.y = Traits<T>::to_f(p[1]);
                if (c + 2 < D) v.z = Traits<T>::to_f(p[2]);
                if (c + 3 < D) v.w = Traits<T>::to_f(p[3]);
            }
        }
        *reinterpret_cast<float4 *>(dst + r * (DP + 4) + c) = v;
    }
}

__device__ __forceinline__ void fma4(float &acc, const float4 &a, const float4 &b) {
    acc = fmaf(a.x, b.x, acc); acc = fmaf(a.y, b.y, acc); acc = fmaf(a.z, b.z, acc); acc = fmaf(a.w, b.w, acc);
}

// s[i][j] = row (ty + 16 i) of A . row (tx + 16 j) of B
template <int RI, int RJ, int DP>
__device__ __forceinline__ void tile_dot(float (&s)[RI][RJ], const float *A, const float *B, int tx, int ty) {
#pragma unroll
    for (int i = 0; i < RI; ++i)
#pragma unroll
        for (int j = 0; j < RJ; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
        float4 av[RI], bv[RJ];
#pragma unroll
        for (int i = 0; i < RI; ++i) av[i] = *reinterpret_cast<const float4 *>(A + (ty + 16 * i) * (DP + 4) + d);
#pragma unroll
        for (int j = 0; j < RJ; ++j) bv[j] = *reinterpret_cast<const float4 *>(B + (tx + 16 * j) * (DP + 4) + d);
#pragma unroll
        for (int i = 0; i < RI; ++i)
#pragma unroll
            for (int j = 0; j < RJ; ++j) fma4(s[i][j], av[i], bv[j]);
    }
}

// o[i][c] += sum over k of W[ty + 16 i][k] * M[k][tx * 4 + 64 c ..]
template <int RI, int NC, int KT, int DP>
__device__ __forceinline__ void tile_acc(float4 (&o)[RI][NC], const float *W, const float *M, int tx, int ty) {
#pragma unroll 2
    for (int k = 0; k < KT; k += 4) {
        float4 w[RI];
#pragma unroll
        for (int i = 0; i < RI; ++i) w[i] = *reinterpret_cast<const float4 *>(W + (ty + 16 * i) * (KT + 4) + k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float4 m = *reinterpret_cast<const float4 *>(M + (k + kk) * (DP + 4) + tx * 4 + 64 * c);
#pragma unroll
                for (int i = 0; i < RI; ++i) {
                    const float x = kk == 0 ? w[i].x : kk == 1 ? w[i].y : kk == 2 ? w[i].z : w[i].w;
                    o[i][c].x = fmaf(x, m.x, o[i][c].x); o[i][c].y = fmaf(x, m.y, o[i][c].y);
                    o[i][c].z = fmaf(x, m.z, o[i][c].z); o[i][c].w = fmaf(x, m.w, o[i][c].w);
                }
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ void store4(T *p, const float4 &v, int c, int D, bool vec) {
    if (c >= D) return;
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4 *>(p) = v;
        } else {
            uint2 raw;
            T *e = reinterpret_cast<T *>(&raw);
            e[0] = Traits<T>::from_f(v.x); e[1] = Traits<T>::from_f(v.y); e[2] = Traits<T>::from_f(v.z); e[3] = Traits<T>::from_f(v.w);
            *reinterpret_cast<uint2 *>(p) = raw;
        }
        return;
    }
    p[0] = Traits<T>::from_f(v.x);
    if (c + 1 < D) p[1] = Traits<T>::from_f(v.y);
    if (c + 2 < D) p[2] = Traits<T>::from_f(v.z);
    if (c + 3 < D) p[3] = Traits<T>::from_f(v.w);
}

__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Whether query row i may look at key j (j < n checked by the caller)
__device__ __forceinline__ bool mask_allows(const DenseMask &m, const uint32_t *bits, int i, int j) {
    return (bits[(int64_t)(m.rows > 1 ? i : 0) * m.wk + (j >> 5)] >> (j & 31)) & 1u;
}

template <typename T, int DP, int BT>
__global__ void __launch_bounds__(kSimtThreads) dense_fwd_simt_kernel(const DenseArgs a) {
    constexpr int R = BT / 16, NC = DP / 64;
    extern __shared__ __align__(16) float sm[];
    float *Qs = sm, *Ks = Qs + BT * (DP + 4), *Vs = Ks + BT * (DP + 4), *Ps = Vs + BT * (DP + 4);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int qtiles = (a.Lq + BT - 1) / BT;
    const int h = (blockIdx.x / qtiles) % a.H, b = blockIdx.x / qtiles / a.H, q0 = (blockIdx.x % qtiles) * BT;
    const int hk = h / a.group;
    const T *Q = (const T *)a.q.ptr + b * a.q.batch_stride + (int64_t)h * a.D;
    const T *K = (const T *)a.k.ptr + b * a.k.batch_stride + (int64_t)hk * a.D;
    const T *V = (const T *)a.v.ptr + b * a.v.batch_stride + (int64_t)hk * a.D;
    T *O = (T *)a.out.ptr + b * a.out.batch_stride + (int64_t)h * a.D;
    const int n = dense_keys(a, b);
    const int64_t plane = (int64_t)b * a.mask.plane_b + (int64_t)h * a.mask.plane_h;
    const uint32_t *bits = a.mask.bits ? a.mask.bits + plane * a.mask.rows * a.mask.wk : nullptr;
    const uint32_t *seen = a.mask.bits ? a.mask.seen + plane * a.mask.wk : nullptr;

    load_rows<T, BT, DP>(Qs, Q, a.q.row_stride, q0, a.Lq, a.D, a.vec, nullptr);
    float4 o[R][NC];
    float m[R], l[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) o[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int k0 = 0; k0 < n; k0 += BT) {
        if (bits != nullptr) {
            const int qrow = a.mask.rows > 1 ? q0 / kDenseTile : 0;
            if (a.mask.tiles[(plane * a.mask.tq + qrow) * a.mask.tk + k0 / kDenseTile] == 0) continue;
        }
        __syncthreads();                                   // everybody is done with the previous tile
        load_rows<T, BT, DP>(Ks, K, a.k.row_stride, k0, n, a.D, a.vec, seen);
        load_rows<T, BT, DP>(Vs, V, a.v.row_stride, k0, n, a.D, a.vec, seen);
        __syncthreads();
        float s[R][R];
        tile_dot<R, R, DP>(s, Qs, Ks, tx, ty);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int qi = q0 + ty + 16 * i;
            float mx = m[i];
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const int kj = k0 + tx + 16 * j;
                const bool ok = kj < n && (bits == nullptr || (qi < a.Lq && mask_allows(a.mask, bits, qi, kj)));
                s[i][j] = ok ? s[i][j] * a.scale_log2 : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float base = mx == -INFINITY ? 0.f : mx;
            const float corr = exp2f(m[i] - base);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const float p = exp2f(s[i][j] - base);
                sum += p;
                Ps[(ty + 16 * i) * (BT + 4) + tx + 16 * j] = p;
            }
            l[i] = l[i] * corr + sum;
            m[i] = mx;
#pragma unroll
            for (int c = 0; c < NC; ++c) { o[i][c].x *= corr; o[i][c].y *= corr; o[i][c].z *= corr; o[i][c].w *= corr; }
        }
        __syncwarp();                                      // a row's weights come from its own half warp
        tile_acc<R, NC, BT, DP>(o, Ps, Vs, tx, ty);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int qi = q0 + ty + 16 * i;
        const float sum = half_warp_sum(l[i]);
        if (qi >= a.Lq) continue;
        const bool none = sum == 0.f;                      // not by the maximum: scores that are all NaN leave that at -inf
        const float inv = none ? 0.f : 1.f / sum;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float4 r = make_float4(o[i][c].x * inv, o[i][c].y * inv, o[i][c].z * inv, o[i][c].w * inv);
            if (none) r = make_float4(a.empty_value, a.empty_value, a.empty_value, a.empty_value);
            const int col = tx * 4 + 64 * c;
            store4<T>(O + (int64_t)qi * a.out.row_stride + col, r, col, a.D, a.vec);
        }
        if (a.lse != nullptr && tx == 0)
            a.lse[((int64_t)b * a.Lq + qi) * a.H + h] = none ? -INFINITY : (m[i] + log2f(sum)) * 0.6931471805599453f;
    }
}

template <typename T, int DP, int BT>
__global__ void __launch_bounds__(kSimtThreads) dense_dq_simt_kernel(const DenseArgs a) {
    constexpr int R = BT / 16, NC = DP / 64;
    extern __shared__ __align__(16) float sm[];
    float *Qs = sm, *Gs = Qs + BT * (DP + 4), *Ks = Gs + BT * (DP + 4), *Vs = Ks + BT * (DP + 4), *Ds = Vs + BT * (DP + 4);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int qtiles = (a.Lq + BT - 1) / BT;
    const int h = (blockIdx.x / qtiles) % a.H, b = blockIdx.x / qtiles / a.H, q0 = (blockIdx.x % qtiles) * BT;
    const int hk = h / a.group;
    const T *Q = (const T *)a.q.ptr + b * a.q.batch_stride + (int64_t)h * a.D;
    const T *G = (const T *)a.dout.ptr + b * a.dout.batch_stride + (int64_t)h * a.D;
    const T *K = (const T *)a.k.ptr + b * a.k.batch_stride + (int64_t)hk * a.D;
    const T *V = (const T *)a.v.ptr + b * a.v.batch_stride + (int64_t)hk * a.D;
    T *dQ = (T *)a.dq.ptr + b * a.dq.batch_stride + (int64_t)h * a.D;
    const int n = dense_keys(a, b);
    const int64_t plane = (int64_t)b * a.mask.plane_b + (int64_t)h * a.mask.plane_h;
    const uint32_t *bits = a.mask.bits ? a.mask.bits + plane * a.mask.rows * a.mask.wk : nullptr;
    const uint32_t *seen = a.mask.bits ? a.mask.seen + plane * a.mask.wk : nullptr;

    load_rows<T, BT, DP>(Qs, Q, a.q.row_stride, q0, a.Lq, a.D, a.vec, nullptr);
    load_rows<T, BT, DP>(Gs, G, a.dout.row_stride, q0, a.Lq, a.D, a.vec, nullptr);
    float4 o[R][NC];
    float lse2[R], delta[R];                                // both negated
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t at = ((int64_t)b * a.H + h) * a.lq_pad + q0 + ty + 16 * i;      // lq_pad covers whole tiles
        lse2[i] = a.neg_lse2[at];
        delta[i] = a.neg_delta[at];
#pragma unroll
        for (int c = 0; c < NC; ++c) o[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int k0 = 0; k0 < n; k0 += BT) {
        if (bits != nullptr) {
            const int qrow = a.mask.rows > 1 ? q0 / kDenseTile : 0;
            if (a.mask.tiles[(plane * a.mask.tq + qrow) * a.mask.tk + k0 / kDenseTile] == 0) continue;
        }
        __syncthreads();
        load_rows<T, BT, DP>(Ks, K, a.k.row_stride, k0, n, a.D, a.vec, seen);
        load_rows<T, BT, DP>(Vs, V, a.v.row_stride, k0, n, a.D, a.vec, seen);
        __syncthreads();
        float s[R][R], dp[R][R];
        tile_dot<R, R, DP>(s, Qs, Ks, tx, ty);
        tile_dot<R, R, DP>(dp, Gs, Vs, tx, ty);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int qi = q0 + ty + 16 * i;
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const int kj = k0 + tx + 16 * j;
                const bool ok = kj < n && lse2[i] != -INFINITY && (bits == nullptr || mask_allows(a.mask, bits, qi, kj));
                Ds[(ty + 16 * i) * (BT + 4) + tx + 16 * j] = ok ? exp2f(fmaf(s[i][j], a.scale_log2, lse2[i])) * (dp[i][j] + delta[i]) : 0.f;
            }
        }
        __syncwarp();
        tile_acc<R, NC, BT, DP>(o, Ds, Ks, tx, ty);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int qi = q0 + ty + 16 * i;
        if (qi >= a.Lq) continue;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float4 r = make_float4(o[i][c].x * a.scale, o[i][c].y * a.scale, o[i][c].z * a.scale, o[i][c].w * a.scale);
            const int col = tx * 4 + 64 * c;
            store4<T>(dQ + (int64_t)qi * a.dq.row_stride + col, r, col, a.D, a.vec);
        }
    }
}

template <typename T, int DP, int BT>
__global__ void __launch_bounds__(kSimtThreads) dense_dkdv_simt_kernel(const DenseArgs a) {
    constexpr int R = BT / 16, NC = DP / 64;
    extern __shared__ __align__(16) float sm[];
    float *Ks = sm, *Vs = Ks + BT * (DP + 4), *Qs = Vs + BT * (DP + 4), *Gs = Qs + BT * (DP + 4), *Ps = Gs + BT * (DP + 4),
          *Ds = Ps + BT * (BT + 4);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int ktiles = (a.Lk + BT - 1) / BT;
    const int hk = (blockIdx.x / ktiles) % a.Hkv, b = blockIdx.x / ktiles / a.Hkv, k0 = (blockIdx.x % ktiles) * BT;
    const T *K = (const T *)a.k.ptr + b * a.k.batch_stride + (int64_t)hk * a.D;
    const T *V = (const T *)a.v.ptr + b * a.v.batch_stride + (int64_t)hk * a.D;
    T *dK = (T *)a.dk.ptr + b * a.dk.batch_stride + (int64_t)hk * a.D;
    T *dV = (T *)a.dv.ptr + b * a.dv.batch_stride + (int64_t)hk * a.D;
    const int n = dense_keys(a, b);
    float4 ok4[R][NC], ov4[R][NC];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) { ok4[i][c] = make_float4(0.f, 0.f, 0.f, 0.f); ov4[i][c] = make_float4(0.f, 0.f, 0.f, 0.f); }
    if (k0 < n) {
        // K and V hold what they hold in keys that are masked: such rows only meet weights that are selected to zero, row by row
        load_rows<T, BT, DP>(Ks, K, a.k.row_stride, k0, n, a.D, a.vec, nullptr);
        load_rows<T, BT, DP>(Vs, V, a.v.row_stride, k0, n, a.D, a.vec, nullptr);
        for (int g = 0; g < a.group; ++g) {
            const int h = hk * a.group + g;
            const T *Q = (const T *)a.q.ptr + b * a.q.batch_stride + (int64_t)h * a.D;
            const T *G = (const T *)a.dout.ptr + b * a.dout.batch_stride + (int64_t)h * a.D;
            const int64_t plane = (int64_t)b * a.mask.plane_b + (int64_t)h * a.mask.plane_h;
            const uint32_t *bits = a.mask.bits ? a.mask.bits + plane * a.mask.rows * a.mask.wk : nullptr;
            for (int q0 = 0; q0 < a.Lq; q0 += BT) {
                if (bits != nullptr) {
                    const int qrow = a.mask.rows > 1 ? q0 / kDenseTile : 0;
                    if (a.mask.tiles[(plane * a.mask.tq + qrow) * a.mask.tk + k0 / kDenseTile] == 0) continue;
                }
                __syncthreads();
                load_rows<T, BT, DP>(Qs, Q, a.q.row_stride, q0, a.Lq, a.D, a.vec, nullptr);
                load_rows<T, BT, DP>(Gs, G, a.dout.row_stride, q0, a.Lq, a.D, a.vec, nullptr);
                __syncthreads();
                float s[R][R], dp[R][R];                      // rows: keys, columns: queries
                tile_dot<R, R, DP>(s, Ks, Qs, tx, ty);
                tile_dot<R, R, DP>(dp, Vs, Gs, tx, ty);
#pragma unroll
                for (int j = 0; j < R; ++j) {
                    const int qj = q0 + tx + 16 * j;
                    const int64_t at = ((int64_t)b * a.H + h) * a.lq_pad + qj;
                    const float lse2 = a.neg_lse2[at], delta = a.neg_delta[at];
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        const int ki = k0 + ty + 16 * i;
                        const bool ok = ki < n && lse2 != -INFINITY && (bits == nullptr || mask_allows(a.mask, bits, qj, ki));
                        const float p = ok ? exp2f(fmaf(s[i][j], a.scale_log2, lse2)) : 0.f;
                        Ps[(ty + 16 * i) * (BT + 4) + tx + 16 * j] = p;
                        Ds[(ty + 16 * i) * (BT + 4) + tx + 16 * j] = ok ? p * (dp[i][j] + delta) : 0.f;
                    }
                }
                __syncwarp();
                tile_acc<R, NC, BT, DP>(ov4, Ps, Gs, tx, ty);
                tile_acc<R, NC, BT, DP>(ok4, Ds, Qs, tx, ty);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int ki = k0 + ty + 16 * i;
        if (ki >= a.Lk) continue;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = tx * 4 + 64 * c;
            const float4 r = make_float4(ok4[i][c].x * a.scale, ok4[i][c].y * a.scale, ok4[i][c].z * a.scale, ok4[i][c].w * a.scale);
            store4<T>(dK + (int64_t)ki * a.dk.row_stride + col, r, col, a.D, a.vec);
            store4<T>(dV + (int64_t)ki * a.dv.row_stride + col, ov4[i][c], col, a.D, a.vec);
        }
    }
}

// 0 = forward, 1 = dq, 2 = dk and dv
template <typename T, int DP, int BT>
static int simt_launch(const DenseArgs &a, int what, cudaStream_t st) {
    const size_t rows = BT * (DP + 4) * sizeof(float), weights = BT * (BT + 4) * sizeof(float);
    const size_t smem = what == 0 ? 3 * rows + weights : what == 1 ? 4 * rows + weights : 4 * rows + 2 * weights;
    const long long blocks = what == 2 ? (long long)a.B * a.Hkv * ((a.Lk + BT - 1) / BT) : (long long)a.B * a.H * ((a.Lq + BT - 1) / BT);
    if (blocks > 0x7fffffffLL) return fail(HSA_ERR_ARG, "hsa_dense_attn: too many tiles");
    auto go = [&]<auto kernel>() -> int {
        const cudaError_t e = allow_smem<kernel>((int)smem);
        if (e != cudaSuccess) return fail((int)e, "hsa_dense_attn: shared memory %zu: %s", smem, cudaGetErrorString(e));
        kernel<<<(unsigned)blocks, kSimtThreads, smem, st>>>(a);
        return launch_status("hsa_dense_attn");
    };
    if (what == 0) return go.template operator()<dense_fwd_simt_kernel<T, DP, BT>>();
    if (what == 1) return go.template operator()<dense_dq_simt_kernel<T, DP, BT>>();
    return go.template operator()<dense_dkdv_simt_kernel<T, DP, BT>>();
}

// Tiles of 64 x 64 up to 128 head dims (70 to 170 KB of shared memory); 32 x 32 above, where 64 would not fit.
int dense_simt(const DenseArgs &a, int what, int dtype, cudaStream_t st) {
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        if (a.D <= 64) return simt_launch<T, 64, 64>(a, what, st);
        if (a.D <= 128) return simt_launch<T, 128, 64>(a, what, st);
        return simt_launch<T, 256, 32>(a, what, st);
    });
}

}  // namespace hsa
