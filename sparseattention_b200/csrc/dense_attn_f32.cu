// Dense attention in 32 bits: float32 inputs, head dims the tcgen05 kernels do not take, unaligned rows.
//
//   p[i, j] = exp2(c q_i.k_j - m_i) / l_i,   out_i = sum_j p[i, j] v_j,     c = scale * log2(e)
//   dv_j = sum_i p[i, j] do_i,   ds[i, j] = p[i, j] (do_i.v_j - sum_d do_i out_i),   dq_i = scale sum_j ds[i, j] k_j,
//   dk_j = scale sum_i ds[i, j] q_i
//
// A warp owns 16 rows (queries; keys in the dk/dv kernel) and walks over tiles of the other side, which lie in shared memory as
// float32.  Products run on the tensor cores in three passes: x = hi + lo with hi = x rounded to 11 bits (tf32) and lo the rest
// rounded to 11 bits, a b ~ hi hi + hi lo + lo hi, off by at most about 3 * 2^-22 |a b|, summed in 32 bits.  Bound by the rate of
// these warp-level products, measured at about 130 multiply-adds per cycle and SM, three for one here, and by the additions between them
// (mma_split): forward 2048 x 2048, 8 heads of 64: 399 us; forward and backward 2 x 1024 x 1024, 16 heads of 128: 3350 us.  That is no
// faster than 32-bit multiply-adds on the same tiles were: 420 and 314 us, and 3197 and 3594 us, with 8 x 4 and 4 x 4 of them per
// thread, either of which wins one of the two.  (With all sums left to the tensor cores, which cut off, it was 346 and 2734 us.)
// Weights pass from the first product to the second through shared memory, inside a warp.  Rows are padded so that fragment reads
// have no bank conflicts (two-way for the operands that are read along both axes).  One writer per output row, fixed order of
// summation.  Keys behind a sequence's length, and keys that no query may look at, are stored as zeros: what lies there (NaN,
// infinities) cannot reach a result through 0 * x.  Few items with long loops are cut into ranges, joined afterwards.
#include "dense_attn_split.cuh"

namespace hsa {

// Tile sizes by padded head dim: a block's own rows, the rows of a tile of the other side (32 where 64 would leave room for one block
// per SM only: 4686 -> 2734 us at 2 x 1024 x 1024, 16 heads of 128, forward and backward, with all sums in the tensor cores), and warps per 16 own rows (each with its
// share of the output columns)
template <int DP> struct F32Shape {
    static constexpr int kRows = DP <= 128 ? 64 : 32, kOther = DP <= 64 ? 64 : 32, kSplit = DP <= 128 ? 1 : 2;
    static constexpr int kThreads = kRows / 16 * kSplit * 32;
    static constexpr int kPitch = DP + 4;                    // floats between rows
    static constexpr int kWeights = kOther + 4;
};

__device__ __forceinline__ uint32_t to_tf32(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;\n" : "=r"(r) : "f"(x));
    return r;
}
struct Split { uint32_t hi, lo; };
__device__ __forceinline__ Split split(float x) {
    Split s;
    s.hi = to_tf32(x);
    s.lo = to_tf32(x - __uint_as_float(s.hi));
    return s;
}
__device__ __forceinline__ void mma1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d[n] += a b[n] for N tiles.  A pass runs over all tiles before the next one starts: back to back on one accumulator they would wait
// for each other.  Eight products at a time are summed by the tensor cores, whose additions cut off instead of rounding; the long
// sum over those is one of ordinary additions (2.7 times nearer to 64 bits).
template <int N, int NT>
__device__ __forceinline__ void mma_split(float (&d)[NT][4], int first, const Split (&a)[4], const Split (&b)[N][2]) {
    float t[N][4] = {};
#pragma unroll
    for (int n = 0; n < N; ++n) mma1688(t[n], a[0].lo, a[1].lo, a[2].lo, a[3].lo, b[n][0].hi, b[n][1].hi);
#pragma unroll
    for (int n = 0; n < N; ++n) mma1688(t[n], a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[n][0].lo, b[n][1].lo);
#pragma unroll
    for (int n = 0; n < N; ++n) mma1688(t[n], a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[n][0].hi, b[n][1].hi);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) d[first + n][e] += t[n][e];
}

// rows row0 .. row0 + ROWS - 1 of a [rows, D] matrix as float32 into dst[ROWS][DP + 4]; rows >= limit, rows whose bit in `seen`
// is clear and columns >= D are zeros
template <typename T, int ROWS, int DP, int THREADS>
__device__ __forceinline__ void load_rows(float *dst, const T *base, int64_t row_stride, int row0, int limit, int D, bool vec,
                                          const uint32_t *seen) {
    constexpr int C4 = DP / 4;
#pragma unroll 4
    for (int idx = threadIdx.x; idx < ROWS * C4; idx += THREADS) {
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

// s[n] = the warp's 16 rows of A times rows [8 n, 8 n + 8) of B, over DP columns
template <int NT, int DP>
__device__ __forceinline__ void rows_dot(float (&s)[NT][4], const float *A, const float *B, int g, int quad) {
    constexpr int P = DP + 4;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll 2
    for (int d = 0; d < DP; d += 8) {
        const Split a[4] = {split(A[g * P + d + quad]), split(A[(g + 8) * P + d + quad]), split(A[g * P + d + quad + 4]),
                            split(A[(g + 8) * P + d + quad + 4])};
        static_assert(NT % 4 == 0, "tiles come in fours");
#pragma unroll
        for (int n = 0; n < NT; n += 4) {
            Split b[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float *p = B + (8 * (n + j) + g) * P + d + quad;
                b[j][0] = split(p[0]); b[j][1] = split(p[4]);
            }
            mma_split<4>(s, n, a, b);
        }
    }
}
// o[n] += the warp's 16 rows of W [.., KT] times columns [8 n, 8 n + 8) of M [KT rows]
template <int NT, int KT, int DP>
__device__ __forceinline__ void rows_acc(float (&o)[NT][4], const float *W, const float *M, int g, int quad) {
    constexpr int P = DP + 4, PW = KT + 4;
#pragma unroll 2
    for (int k = 0; k < KT; k += 8) {
        const Split a[4] = {split(W[g * PW + k + quad]), split(W[(g + 8) * PW + k + quad]), split(W[g * PW + k + quad + 4]),
                            split(W[(g + 8) * PW + k + quad + 4])};
        static_assert(NT % 4 == 0, "tiles come in fours");
#pragma unroll
        for (int n = 0; n < NT; n += 4) {
            Split b[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float *p = M + (k + quad) * P + 8 * (n + j) + g;
                b[j][0] = split(p[0]); b[j][1] = split(p[4 * P]);
            }
            mma_split<4>(o, n, a, b);
        }
    }
}

template <typename T>
__device__ __forceinline__ void store2(T *p, float x, float y, int c, int D, bool vec) {
    if (vec && c < D) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float2 *>(p) = make_float2(x, y);
        else { T v[2] = {Traits<T>::from_f(x), Traits<T>::from_f(y)}; *reinterpret_cast<uint32_t *>(p) = *reinterpret_cast<uint32_t *>(v); }
        return;
    }
    if (c < D) p[0] = Traits<T>::from_f(x);
    if (c + 1 < D) p[1] = Traits<T>::from_f(y);
}

// Whether query row i may look at key j (j < n checked by the caller)
__device__ __forceinline__ bool mask_allows(const DenseMask &m, const uint32_t *bits, int i, int j) {
    return (bits[(int64_t)(m.rows > 1 ? i : 0) * m.wk + (j >> 5)] >> (j & 31)) & 1u;
}

template <typename T, int DP>
__global__ void __launch_bounds__(F32Shape<DP>::kThreads) dense_fwd_f32_kernel(const DenseArgs a, const DenseSplit sp) {
    using S = F32Shape<DP>;
    constexpr int BT = S::kRows, BO = S::kOther, NT = BO / 8, NO = DP / S::kSplit / 8;
    extern __shared__ __align__(16) float sm[];
    float *Qs = sm, *Ks = Qs + BT * S::kPitch, *Vs = Ks + BO * S::kPitch, *Ps = Vs + BO * S::kPitch;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, quad = lane & 3;
    const int wr = warp / S::kSplit, wc = warp % S::kSplit, col0 = wc * (DP / S::kSplit);
    const int qtiles = (a.Lq + BT - 1) / BT;
    int blk = blockIdx.x;
    const int q0 = blk % qtiles * BT; blk /= qtiles;
    const int h = blk % a.H; blk /= a.H;
    const int b = blk % a.B, range = blk / a.B, hk = h / a.group;
    const T *Q = (const T *)a.q.ptr + b * a.q.batch_stride + (int64_t)h * a.D;
    const T *K = (const T *)a.k.ptr + b * a.k.batch_stride + (int64_t)hk * a.D;
    const T *V = (const T *)a.v.ptr + b * a.v.batch_stride + (int64_t)hk * a.D;
    const int n = dense_keys(a, b), tiles = (n + BO - 1) / BO, per = (tiles + sp.splits - 1) / sp.splits;
    const int64_t plane = (int64_t)b * a.mask.plane_b + (int64_t)h * a.mask.plane_h;
    const uint32_t *bits = a.mask.bits ? a.mask.bits + plane * a.mask.rows * a.mask.wk : nullptr;
    const uint32_t *seen = a.mask.bits ? a.mask.seen + plane * a.mask.wk : nullptr;

    load_rows<T, BT, DP, S::kThreads>(Qs, Q, a.q.row_stride, q0, a.Lq, a.D, a.vec, nullptr);
    float o[NO][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    for (int t = range * per; t < min(tiles, (range + 1) * per); ++t) {
        const int k0 = t * BO;
        if (bits != nullptr) {
            const int cell = a.mask.rows > 1 ? q0 / kDenseTile : 0;
            if (a.mask.tiles[(plane * a.mask.tq + cell) * a.mask.tk + k0 / kDenseTile] == 0) continue;
        }
        __syncthreads();                                   // everybody is done with the previous tile
        load_rows<T, BO, DP, S::kThreads>(Ks, K, a.k.row_stride, k0, n, a.D, a.vec, seen);
        load_rows<T, BO, DP, S::kThreads>(Vs, V, a.v.row_stride, k0, n, a.D, a.vec, seen);
        __syncthreads();
        float s[NT][4];
        rows_dot<NT, DP>(s, Qs + wr * 16 * S::kPitch, Ks, g, quad);
        float top[2] = {m[0], m[1]};
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int qi = q0 + wr * 16 + g + 8 * (e >> 1), kj = k0 + 8 * i + 2 * quad + (e & 1);
                const bool ok = kj < n && (bits == nullptr || (qi < a.Lq && mask_allows(a.mask, bits, qi, kj)));
                s[i][e] = ok ? s[i][e] * a.scale_log2 : -INFINITY;
                top[e >> 1] = fmaxf(top[e >> 1], s[i][e]);
            }
        float base[2], corr[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
            base[r] = top[r] == -INFINITY ? 0.f : top[r];
            corr[r] = exp2f(m[r] - base[r]);
            m[r] = top[r];
            l[r] *= corr[r];
        }
        float *mine = Ps + (wr * S::kSplit + wc) * 16 * S::kWeights;     // this warp's own 16 rows of weights
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float p0 = exp2f(s[i][2 * r] - base[r]), p1 = exp2f(s[i][2 * r + 1] - base[r]);
                l[r] += p0 + p1;
                *reinterpret_cast<float2 *>(mine + (g + 8 * r) * S::kWeights + 8 * i + 2 * quad) = make_float2(p0, p1);
            }
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] *= corr[e >> 1];
        __syncwarp();
        rows_acc<NO, BO, DP>(o, mine, Vs + col0, g, quad);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        const int qi = q0 + wr * 16 + g + 8 * r;
        if (qi >= a.Lq) continue;
        const int64_t row = ((int64_t)b * a.Lq + qi) * a.H + h;
        if (sp.splits > 1) {
            const int64_t at = (int64_t)range * a.B * a.Lq * a.H + row;
#pragma unroll
            for (int i = 0; i < NO; ++i) {
                const int c = col0 + 8 * i + 2 * quad;
                if (c < a.D) *reinterpret_cast<float2 *>(sp.part_o + at * a.D + c) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
            }
            if (quad == 0 && wc == 0) *reinterpret_cast<float2 *>(sp.part_ml + 2 * at) = make_float2(m[r], l[r]);
            continue;
        }
        const bool none = l[r] == 0.f;                     // not by the maximum: scores that are all NaN leave that at -inf
        const float inv = none ? 0.f : 1.f / l[r];
        T *out = (T *)a.out.ptr + b * a.out.batch_stride + (int64_t)qi * a.out.row_stride + (int64_t)h * a.D;
#pragma unroll
        for (int i = 0; i < NO; ++i) {
            const int c = col0 + 8 * i + 2 * quad;
            store2<T>(out + c, none ? a.empty_value : o[i][2 * r] * inv, none ? a.empty_value : o[i][2 * r + 1] * inv, c, a.D, a.vec);
            if (a.out_lo != nullptr)
                store2<T>((T *)a.out_lo + row * a.D + c, none ? 0.f : rounding_rest<T>(o[i][2 * r] * inv),
                          none ? 0.f : rounding_rest<T>(o[i][2 * r + 1] * inv), c, a.D, a.D % 2 == 0);
        }
        if (a.lse != nullptr && quad == 0 && wc == 0) a.lse[row] = none ? -INFINITY : (m[r] + log2f(l[r])) * 0.6931471805599453f;
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(F32Shape<DP>::kThreads) dense_dq_f32_kernel(const DenseArgs a, const BwdSplit sp) {
    using S = F32Shape<DP>;
    constexpr int BT = S::kRows, BO = S::kOther, NT = BO / 8, NO = DP / S::kSplit / 8;
    extern __shared__ __align__(16) float sm[];
    float *Qs = sm, *Gs = Qs + BT * S::kPitch, *Ks = Gs + BT * S::kPitch, *Vs = Ks + BO * S::kPitch, *Ds = Vs + BO * S::kPitch;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, quad = lane & 3;
    const int wr = warp / S::kSplit, wc = warp % S::kSplit, col0 = wc * (DP / S::kSplit);
    const int qtiles = (a.Lq + BT - 1) / BT;
    int blk = blockIdx.x;
    const int q0 = blk % qtiles * BT; blk /= qtiles;
    const int h = blk % a.H; blk /= a.H;
    const int b = blk % a.B, range = blk / a.B, hk = h / a.group;
    const T *Q = (const T *)a.q.ptr + b * a.q.batch_stride + (int64_t)h * a.D;
    const T *G = (const T *)a.dout.ptr + b * a.dout.batch_stride + (int64_t)h * a.D;
    const T *K = (const T *)a.k.ptr + b * a.k.batch_stride + (int64_t)hk * a.D;
    const T *V = (const T *)a.v.ptr + b * a.v.batch_stride + (int64_t)hk * a.D;
    const int n = dense_keys(a, b), tiles = (n + BO - 1) / BO, per = (tiles + sp.splits - 1) / sp.splits;
    const int64_t plane = (int64_t)b * a.mask.plane_b + (int64_t)h * a.mask.plane_h;
    const uint32_t *bits = a.mask.bits ? a.mask.bits + plane * a.mask.rows * a.mask.wk : nullptr;
    const uint32_t *seen = a.mask.bits ? a.mask.seen + plane * a.mask.wk : nullptr;

    load_rows<T, BT, DP, S::kThreads>(Qs, Q, a.q.row_stride, q0, a.Lq, a.D, a.vec, nullptr);
    load_rows<T, BT, DP, S::kThreads>(Gs, G, a.dout.row_stride, q0, a.Lq, a.D, a.vec, nullptr);
    float o[NO][4], lse2[2], delta[2];                     // both negated
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int64_t at = ((int64_t)b * a.H + h) * a.lq_pad + q0 + wr * 16 + g + 8 * r;      // lq_pad covers whole tiles
        lse2[r] = a.neg_lse2[at];
        delta[r] = a.neg_delta[at];
    }
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    for (int t = range * per; t < min(tiles, (range + 1) * per); ++t) {
        const int k0 = t * BO;
        if (bits != nullptr) {
            const int cell = a.mask.rows > 1 ? q0 / kDenseTile : 0;
            if (a.mask.tiles[(plane * a.mask.tq + cell) * a.mask.tk + k0 / kDenseTile] == 0) continue;
        }
        __syncthreads();
        load_rows<T, BO, DP, S::kThreads>(Ks, K, a.k.row_stride, k0, n, a.D, a.vec, seen);
        load_rows<T, BO, DP, S::kThreads>(Vs, V, a.v.row_stride, k0, n, a.D, a.vec, seen);
        __syncthreads();
        float s[NT][4], dp[NT][4];
        rows_dot<NT, DP>(s, Qs + wr * 16 * S::kPitch, Ks, g, quad);
        rows_dot<NT, DP>(dp, Gs + wr * 16 * S::kPitch, Vs, g, quad);
        float *mine = Ds + (wr * S::kSplit + wc) * 16 * S::kWeights;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int qi = q0 + wr * 16 + g + 8 * r, kj = k0 + 8 * i + 2 * quad + e;
                    const bool ok = kj < n && lse2[r] != -INFINITY && (bits == nullptr || mask_allows(a.mask, bits, qi, kj));
                    x[e] = ok ? exp2f(fmaf(s[i][2 * r + e], a.scale_log2, lse2[r])) * (dp[i][2 * r + e] + delta[r]) : 0.f;
                }
                *reinterpret_cast<float2 *>(mine + (g + 8 * r) * S::kWeights + 8 * i + 2 * quad) = make_float2(x[0], x[1]);
            }
        __syncwarp();
        rows_acc<NO, BO, DP>(o, mine, Ks + col0, g, quad);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int qi = q0 + wr * 16 + g + 8 * r;
        if (qi >= a.Lq) continue;
        T *out = (T *)a.dq.ptr + b * a.dq.batch_stride + (int64_t)qi * a.dq.row_stride + (int64_t)h * a.D;
        float *part = sp.splits > 1 ? sp.part + ((((int64_t)range * a.B + b) * a.Lq + qi) * a.H + h) * a.D : nullptr;
#pragma unroll
        for (int i = 0; i < NO; ++i) {
            const int c = col0 + 8 * i + 2 * quad;
            if (part == nullptr) store2<T>(out + c, o[i][2 * r] * a.scale, o[i][2 * r + 1] * a.scale, c, a.D, a.vec);
            else if (c < a.D) *reinterpret_cast<float2 *>(part + c) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
        }
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(F32Shape<DP>::kThreads) dense_dkdv_f32_kernel(const DenseArgs a, const BwdSplit sp) {
    using S = F32Shape<DP>;
    constexpr int BT = S::kRows, BO = S::kOther, NT = BO / 8, NO = DP / S::kSplit / 8;
    extern __shared__ __align__(16) float sm[];
    float *Ks = sm, *Vs = Ks + BT * S::kPitch, *Qs = Vs + BT * S::kPitch, *Gs = Qs + BO * S::kPitch, *Ws = Gs + BO * S::kPitch;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, quad = lane & 3;
    const int wr = warp / S::kSplit, wc = warp % S::kSplit, col0 = wc * (DP / S::kSplit);
    const int ktiles = (a.Lk + BT - 1) / BT, qtiles = (a.Lq + BO - 1) / BO;
    int blk = blockIdx.x;
    const int k0 = blk % ktiles * BT; blk /= ktiles;
    const int hk = blk % a.Hkv; blk /= a.Hkv;
    const int b = blk % a.B, range = blk / a.B;
    const T *K = (const T *)a.k.ptr + b * a.k.batch_stride + (int64_t)hk * a.D;
    const T *V = (const T *)a.v.ptr + b * a.v.batch_stride + (int64_t)hk * a.D;
    const int n = dense_keys(a, b);
    const int units = k0 < n ? a.group * qtiles : 0, per = (units + sp.splits - 1) / sp.splits;
    float ok4[NO][4], ov4[NO][4];
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) { ok4[i][e] = 0.f; ov4[i][e] = 0.f; }
    // K and V hold what they hold in keys that are masked: such rows only meet weights that are selected to zero, row by row
    load_rows<T, BT, DP, S::kThreads>(Ks, K, a.k.row_stride, k0, n, a.D, a.vec, nullptr);
    load_rows<T, BT, DP, S::kThreads>(Vs, V, a.v.row_stride, k0, n, a.D, a.vec, nullptr);
    for (int u = range * per; u < min(units, (range + 1) * per); ++u) {
        const int h = hk * a.group + u / qtiles, q0 = u % qtiles * BO;
        const T *Q = (const T *)a.q.ptr + b * a.q.batch_stride + (int64_t)h * a.D;
        const T *G = (const T *)a.dout.ptr + b * a.dout.batch_stride + (int64_t)h * a.D;
        const int64_t plane = (int64_t)b * a.mask.plane_b + (int64_t)h * a.mask.plane_h;
        const uint32_t *bits = a.mask.bits ? a.mask.bits + plane * a.mask.rows * a.mask.wk : nullptr;
        if (bits != nullptr) {
            const int cell = a.mask.rows > 1 ? q0 / kDenseTile : 0;
            if (a.mask.tiles[(plane * a.mask.tq + cell) * a.mask.tk + k0 / kDenseTile] == 0) continue;
        }
        __syncthreads();
        load_rows<T, BO, DP, S::kThreads>(Qs, Q, a.q.row_stride, q0, a.Lq, a.D, a.vec, nullptr);
        load_rows<T, BO, DP, S::kThreads>(Gs, G, a.dout.row_stride, q0, a.Lq, a.D, a.vec, nullptr);
        __syncthreads();
        float s[NT][4], dp[NT][4];                            // rows: keys, columns: queries
        rows_dot<NT, DP>(s, Ks + wr * 16 * S::kPitch, Qs, g, quad);
        rows_dot<NT, DP>(dp, Vs + wr * 16 * S::kPitch, Gs, g, quad);
        const int64_t stats = ((int64_t)b * a.H + h) * a.lq_pad + q0;
        float *mine = Ws + (wr * S::kSplit + wc) * 16 * S::kWeights;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int c = 8 * i + 2 * quad;
            const float2 lse2 = *reinterpret_cast<const float2 *>(a.neg_lse2 + stats + c), delta = *reinterpret_cast<const float2 *>(a.neg_delta + stats + c);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float p[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int ki = k0 + wr * 16 + g + 8 * r, qj = q0 + c + e;
                    const float ls = e == 0 ? lse2.x : lse2.y;
                    const bool ok = ki < n && ls != -INFINITY && (bits == nullptr || mask_allows(a.mask, bits, qj, ki));
                    p[e] = ok ? exp2f(fmaf(s[i][2 * r + e], a.scale_log2, ls)) : 0.f;
                    dp[i][2 * r + e] = ok ? p[e] * (dp[i][2 * r + e] + (e == 0 ? delta.x : delta.y)) : 0.f;
                }
                *reinterpret_cast<float2 *>(mine + (g + 8 * r) * S::kWeights + c) = make_float2(p[0], p[1]);
            }
        }
        __syncwarp();
        rows_acc<NO, BO, DP>(ov4, mine, Gs + col0, g, quad);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r)
                *reinterpret_cast<float2 *>(mine + (g + 8 * r) * S::kWeights + 8 * i + 2 * quad) = make_float2(dp[i][2 * r], dp[i][2 * r + 1]);
        __syncwarp();
        rows_acc<NO, BO, DP>(ok4, mine, Qs + col0, g, quad);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int ki = k0 + wr * 16 + g + 8 * r;
        if (ki >= a.Lk) continue;
        T *dK = (T *)a.dk.ptr + b * a.dk.batch_stride + (int64_t)ki * a.dk.row_stride + (int64_t)hk * a.D;
        T *dV = (T *)a.dv.ptr + b * a.dv.batch_stride + (int64_t)ki * a.dv.row_stride + (int64_t)hk * a.D;
        float *part = sp.splits > 1 ? sp.part + ((((int64_t)range * a.B + b) * a.Lk + ki) * a.Hkv + hk) * a.D : nullptr;
        const int64_t dv_part = (int64_t)sp.splits * a.B * a.Lk * a.Hkv * a.D;
#pragma unroll
        for (int i = 0; i < NO; ++i) {
            const int c = col0 + 8 * i + 2 * quad;
            if (part == nullptr) {
                store2<T>(dK + c, ok4[i][2 * r] * a.scale, ok4[i][2 * r + 1] * a.scale, c, a.D, a.vec);
                store2<T>(dV + c, ov4[i][2 * r], ov4[i][2 * r + 1], c, a.D, a.vec);
            } else if (c < a.D) {
                *reinterpret_cast<float2 *>(part + c) = make_float2(ok4[i][2 * r], ok4[i][2 * r + 1]);
                *reinterpret_cast<float2 *>(part + dv_part + c) = make_float2(ov4[i][2 * r], ov4[i][2 * r + 1]);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------- launches
// Partial rows are read and written in pieces of four, and only as aligned as the head dim makes them
static bool f32_splittable(int D) { return D % 4 == 0; }
static int f32_rows(int D) { return D <= 128 ? 64 : 32; }
static int f32_other(int D) { return D <= 64 ? 64 : 32; }

// A block costs its tiles plus about one and a half tiles' time of set-up, three as one of several ranges.
static int f32_fwd_splits(int B, int Lq, int Lk, int H, int D) {
    const int bt = f32_rows(D);
    return f32_splittable(D) ? range_count((long long)B * H * ((Lq + bt - 1) / bt), (Lk + f32_other(D) - 1) / f32_other(D), 1.5, 3.0) : 1;
}
static int f32_dkdv_splits(int B, int Lq, int Lk, int H, int Hkv, int D) {
    const int bt = f32_rows(D);
    return f32_splittable(D) ? range_count((long long)B * Hkv * ((Lk + bt - 1) / bt), H / Hkv * ((Lq + f32_other(D) - 1) / f32_other(D)), 1.5, 3.0) : 1;
}

size_t dense_fwd_f32_workspace(int B, int Lq, int Lk, int H, int D) { return fwd_part_bytes(f32_fwd_splits(B, Lq, Lk, H, D), B, Lq, H, D); }
size_t dense_bwd_f32_workspace(int B, int Lq, int Lk, int H, int Hkv, int D) {
    return bwd_part_bytes(f32_fwd_splits(B, Lq, Lk, H, D), f32_dkdv_splits(B, Lq, Lk, H, Hkv, D), B, Lq, Lk, H, Hkv, D);
}

template <typename T, int DP>
static int f32_fwd(const DenseArgs &a, void *workspace, cudaStream_t st) {
    using S = F32Shape<DP>;
    constexpr int smem = ((S::kRows + 2 * S::kOther) * S::kPitch + S::kThreads / 32 * 16 * S::kWeights) * (int)sizeof(float);
    DenseSplit sp = fwd_split(f32_fwd_splits(a.B, a.Lq, a.Lk, a.H, a.D), a, workspace);
    const long long blocks = (long long)a.B * a.H * ((a.Lq + S::kRows - 1) / S::kRows) * sp.splits;
    if (blocks > 0x7fffffffLL) return fail(HSA_ERR_ARG, "hsa_dense_attn_fwd: too many tiles");
    const cudaError_t e = allow_smem<dense_fwd_f32_kernel<T, DP>>(smem);
    if (e != cudaSuccess) return fail((int)e, "hsa_dense_attn_fwd: shared memory %d: %s", smem, cudaGetErrorString(e));
    dense_fwd_f32_kernel<T, DP><<<(unsigned)blocks, S::kThreads, smem, st>>>(a, sp);
    if (int rc = launch_status("hsa_dense_attn_fwd")) return rc;
    return sp.splits > 1 ? join_forward<T>(a, sp, st) : 0;
}

template <typename T, int DP>
static int f32_bwd(const DenseArgs &a, void *workspace, cudaStream_t st) {
    using S = F32Shape<DP>;
    constexpr int smem = (2 * (S::kRows + S::kOther) * S::kPitch + S::kThreads / 32 * 16 * S::kWeights) * (int)sizeof(float);
    BwdSplit sq, sk;
    bwd_splits(f32_fwd_splits(a.B, a.Lq, a.Lk, a.H, a.D), f32_dkdv_splits(a.B, a.Lq, a.Lk, a.H, a.Hkv, a.D), a, workspace, sq, sk);
    const long long q_blocks = (long long)a.B * a.H * ((a.Lq + S::kRows - 1) / S::kRows) * sq.splits;
    const long long k_blocks = (long long)a.B * a.Hkv * ((a.Lk + S::kRows - 1) / S::kRows) * sk.splits;
    if (q_blocks > 0x7fffffffLL || k_blocks > 0x7fffffffLL) return fail(HSA_ERR_ARG, "hsa_dense_attn_bwd: too many tiles");
    cudaError_t e = allow_smem<dense_dq_f32_kernel<T, DP>>(smem);
    if (e == cudaSuccess) e = allow_smem<dense_dkdv_f32_kernel<T, DP>>(smem);
    if (e != cudaSuccess) return fail((int)e, "hsa_dense_attn_bwd: shared memory %d: %s", smem, cudaGetErrorString(e));
    if (a.dk.ptr != nullptr) {
        dense_dkdv_f32_kernel<T, DP><<<(unsigned)k_blocks, S::kThreads, smem, st>>>(a, sk);
        if (int rc = launch_status("hsa_dense_attn_bwd(dk, dv)")) return rc;
    }
    if (a.dq.ptr != nullptr) {
        dense_dq_f32_kernel<T, DP><<<(unsigned)q_blocks, S::kThreads, smem, st>>>(a, sq);
        if (int rc = launch_status("hsa_dense_attn_bwd(dq)")) return rc;
    }
    return join_backward<T>(a, sq, sk, st);
}

int dense_fwd_f32(const DenseArgs &a, void *workspace, int dtype, cudaStream_t st) {
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        if (a.D <= 32) return f32_fwd<T, 32>(a, workspace, st);
        if (a.D <= 64) return f32_fwd<T, 64>(a, workspace, st);
        if (a.D <= 128) return f32_fwd<T, 128>(a, workspace, st);
        return f32_fwd<T, 256>(a, workspace, st);
    });
}
int dense_bwd_f32(const DenseArgs &a, void *workspace, int dtype, cudaStream_t st) {
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        if (a.D <= 32) return f32_bwd<T, 32>(a, workspace, st);
        if (a.D <= 64) return f32_bwd<T, 64>(a, workspace, st);
        if (a.D <= 128) return f32_bwd<T, 128>(a, workspace, st);
        return f32_bwd<T, 256>(a, workspace, st);
    });
}

}  // namespace hsa
