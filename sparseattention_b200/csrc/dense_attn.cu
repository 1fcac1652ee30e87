// Entry points of dense attention, the packing of its masks, and the row sums its backward starts from.
#include "dense_attn.cuh"

namespace hsa {

int dense_fwd_f32(const DenseArgs &a, void *workspace, int dtype, cudaStream_t st);
int dense_bwd_f32(const DenseArgs &a, void *workspace, int dtype, cudaStream_t st);
size_t dense_fwd_f32_workspace(int B, int Lq, int Lk, int H, int D);
size_t dense_bwd_f32_workspace(int B, int Lq, int Lk, int H, int Hkv, int D);
bool dense_tc_ok(const DenseArgs &a, int dtype, bool backward);
size_t dense_fwd_tc_workspace(int B, int Lq, int Lk, int H, int D);
bool dense_bwd_tables_ok(const DenseArgs &a);
size_t dense_bwd_tc_workspace(int B, int Lq, int Lk, int H, int Hkv, int D);
int dense_bwd_tc(const DenseArgs &a, void *workspace, int dtype, cudaStream_t st);
int dense_fwd_tc(const DenseArgs &a, void *workspace, int dtype, cudaStream_t st);

// ------------------------------------------------------------------------------------------------------------ mask
// One block per 128 x 128 cell of a plane, a warp per 32 x 32 piece: 32 coalesced row reads turn into words by ballot, 32 more
// ballots transpose them.  The whole mask is read once (a byte per entry) and comes out at an eighth (two eighths with the
// transposed copy) of its size; the attention kernels then read 16 bytes per query row and 128 keys.
__global__ void __launch_bounds__(512)
dense_mask_pack_kernel(const uint8_t *__restrict__ mask, int64_t sb, int64_t sh, int64_t sq, int64_t sk, int Hm, int rows, int Lk,
                       uint32_t *__restrict__ bits, uint32_t *__restrict__ bits_t, uint32_t *__restrict__ seen,
                       uint8_t *__restrict__ tiles, int wk, int wq, int tq, int tk) {
    const long long cell = blockIdx.x;
    const int ct = (int)(cell % tk), rt = (int)(cell / tk % tq);
    const long long plane = cell / tk / tq;
    const uint8_t *M = mask + (plane / Hm) * sb + (plane % Hm) * sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r0 = rt * kDenseTile + (warp >> 2) * 32, c0 = ct * kDenseTile + (warp & 3) * 32;
    const int key = c0 + lane;
    const int nrows = max(0, min(32, rows - r0)), ncols = max(0, min(32, Lk - c0));
    uint32_t mine = 0, any = 0, all = 0xffffffffu;
    const uint32_t full = ncols == 32 ? 0xffffffffu : (1u << ncols) - 1u;
#pragma unroll 8
    for (int r = 0; r < nrows; ++r) {
        const bool on = key < Lk && M[(int64_t)(r0 + r) * sq + (int64_t)key * sk] != 0;
        const uint32_t w = __ballot_sync(0xffffffffu, on);
        if (r == lane) mine = w;
        any |= w;
        all &= w;
    }
    const int word = c0 >> 5;
    if (lane < nrows) bits[((int64_t)plane * rows + r0 + lane) * wk + word] = mine;
    if (bits_t != nullptr) {
        uint32_t col = 0;
#pragma unroll 8
        for (int j = 0; j < 32; ++j) {
            const uint32_t w = __ballot_sync(0xffffffffu, (mine >> j) & 1u);
            if (j == lane) col = w;
        }
        if (lane < ncols) bits_t[((int64_t)plane * Lk + key) * wq + (r0 >> 5)] = col;
        if (lane == 0 && any != 0) atomicOr(seen + (int64_t)plane * wk + word, any);
    }
    const int some = __syncthreads_or(any != 0);
    const int every = __syncthreads_and(nrows == 0 || (all & full) == full);
    if (threadIdx.x == 0) tiles[((int64_t)plane * tq + rt) * tk + ct] = every ? 2 : some ? 1 : 0;
}

// ------------------------------------------------------------------------------------------------ backward's row sums
// -sum_d dout * out and minus the row's log-sum-exp in base 2 (the kernels add both), padded with rows that give weight zero.  A
// query without keys gets -inf and 0 whatever its output row holds.
template <typename T, int VEC, int LPR, int CPL>
__device__ __forceinline__ float delta_row(const DenseArgs &a, int64_t b, int i, int h, int g, float *neg_lse2, float *neg_delta, float shift) {
    const int64_t at = (b * a.H + h) * a.lq_pad + i;
    if (i >= a.Lq) {
        if (g == 0) { neg_lse2[at] = -INFINITY; neg_delta[at] = 0.f; }
        return 0.f;
    }
    RowFrag<T, VEC, LPR, CPL> x, y;
    x.load((const T *)a.out.ptr + b * a.out.batch_stride + (int64_t)i * a.out.row_stride + (int64_t)h * a.D, g, a.D / VEC);
    y.load((const T *)a.dout.ptr + b * a.dout.batch_stride + (int64_t)i * a.dout.row_stride + (int64_t)h * a.D, g, a.D / VEC);
    float part = x.dot_partial(y);
    if (a.out_lo != nullptr) {
        // what rounding took from the output: without it a sum over few keys, whose differences are small, is off by more than
        // the rest of the backward (2.9e-3 against 2.4e-3 in bfloat16)
        x.load((const T *)a.out_lo + ((b * a.Lq + i) * a.H + h) * a.D, g, a.D / VEC);
        part += x.dot_partial(y);
    }
    const float s = group_sum<LPR>(part);
    if (g == 0) {
        const float l = a.lse[(b * a.Lq + i) * a.H + h];
        const bool none = l == -INFINITY;
        neg_lse2[at] = none ? -INFINITY : l * -1.4426950408889634f + shift;
        neg_delta[at] = none ? 0.f : -s;
    }
    return y.dot_partial(y);                              // this lane's part of dout's squared length
}
template <typename T, int VEC, int LPR, int CPL>
__global__ void __launch_bounds__(256) dense_delta_kernel(const DenseArgs a, float *__restrict__ neg_lse2, float *__restrict__ neg_delta) {
    const long long row = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    const int h = (int)(row % a.H), i = (int)(row / a.H % a.lq_pad);
    const long long b = row / a.H / a.lq_pad;
    if (b >= a.B) return;
    delta_row<T, VEC, LPR, CPL>(a, b, i, h, threadIdx.x % LPR, neg_lse2, neg_delta, 0.f);
}

// The same for float16 on the tensor cores, with the squared lengths of dout's rows, the largest of those per (batch entry, key/value
// head), and a bound on those of V's rows: D times the square of the largest entry.  A block takes a stretch of the query rows of all
// heads of a group, or of V's rows (those that may be looked at: the others may hold anything).  V's part is bound by HBM, so a thread
// asks for eight pieces before it looks at one, and takes entries instead of lengths of rows, whose sums would stand between the loads.
constexpr int kStretch = 4;                               // times 256 / LPR query rows
constexpr int kValueRows = 128;
template <int VEC, int LPR, int CPL>
__global__ void __launch_bounds__(256)
dense_delta_f16_kernel(const DenseArgs a, float *__restrict__ neg_lse2, float *__restrict__ neg_delta, float *__restrict__ dout_sq,
                       unsigned int *__restrict__ top_sq, int q_blocks, int v_blocks) {
    using T = __half;
    constexpr int RPB = 256 / LPR;
    const int at = blockIdx.x % (q_blocks + v_blocks);
    const int bh = blockIdx.x / (q_blocks + v_blocks), hk = bh % a.Hkv;
    const int64_t b = bh / a.Hkv;
    const bool values = at < v_blocks;
    float top = 0.f;
    if (!values) {
        const int g = threadIdx.x % LPR, unit = threadIdx.x / LPR, rows = a.group * a.lq_pad;
        for (int s = 0; s < kStretch; ++s) {
            const int r = ((at - v_blocks) * kStretch + s) * RPB + unit, h = hk * a.group + r / a.lq_pad, i = r % a.lq_pad;
            if (r >= rows) break;
            const float sq = group_sum<LPR>(delta_row<T, VEC, LPR, CPL>(a, b, i, h, g, neg_lse2, neg_delta, (float)kWeightShift));
            if (g == 0) dout_sq[(b * a.H + h) * a.lq_pad + i] = sq;
            top = sq > top || sq != sq ? sq : top;
        }
    } else {
        const int n = dense_keys(a, (int)b), chunks = a.D / 8, j0 = at * kValueRows, pieces = min(kValueRows, n - j0) * chunks;
        const T *V = (const T *)a.v.ptr + b * a.v.batch_stride + (int64_t)j0 * a.v.row_stride + (int64_t)hk * a.D;
        __half2 most = __float2half2_rn(0.f);
        for (int first = threadIdx.x; first < pieces; first += 8 * 256) {
            uint4 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int idx = first + u * 256, r = idx / chunks;
                bool take = idx < pieces;
                if (take && a.mask.bits != nullptr) {
                    take = false;
                    for (int h = hk * a.group; !take && h < (hk + 1) * a.group; ++h) {
                        const int64_t plane = b * a.mask.plane_b + (int64_t)h * a.mask.plane_h;
                        take = (a.mask.seen[plane * a.mask.wk + ((j0 + r) >> 5)] >> ((j0 + r) & 31)) & 1u;
                    }
                }
                x[u] = take ? __ldg(reinterpret_cast<const uint4 *>(V + (int64_t)r * a.v.row_stride + (idx - r * chunks) * 8)) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = e == 0 ? x[u].x : e == 1 ? x[u].y : e == 2 ? x[u].z : x[u].w;
                    most = __hmax2(most, __habs2(*reinterpret_cast<const __half2 *>(&w)));
                }
        }
        const float m = fmaxf(__low2float(most), __high2float(most));
        top = (float)a.D * m * m;
    }
    __shared__ unsigned int warp_top[8];
    // bit patterns of numbers that are not negative are in the numbers' order, NaN last
    const unsigned int bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7fffffffu);
    if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = bits;
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned int all = warp_top[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) all = max(all, warp_top[w]);
        if (all != 0) atomicMax(top_sq + 2 * bh + values, all);
    }
}

static int dense_delta(const DenseArgs &a, float *neg_lse2, float *neg_delta, int dtype, bool vec, cudaStream_t st) {
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        int rc = 0;
        const bool ok = dispatch_row_shape<T>(a.D, vec, [&]<typename T2, int VEC, int LPR, int CPL>() {
            const long long rows = (long long)a.B * a.lq_pad * a.H, blocks = (rows + 256 / LPR - 1) / (256 / LPR);
            if (blocks > 0x7fffffffLL) { rc = fail(HSA_ERR_ARG, "hsa_dense_attn_bwd: too many rows"); return; }
            dense_delta_kernel<T2, VEC, LPR, CPL><<<(unsigned)blocks, 256, 0, st>>>(a, neg_lse2, neg_delta);
            rc = launch_status("hsa_dense_attn_bwd(row sums)");
        });
        return ok ? rc : fail(HSA_ERR_ARG, "hsa_dense_attn_bwd: head dim %d not supported", a.D);
    });
}
static int dense_delta_f16(const DenseArgs &a, float *neg_lse2, float *neg_delta, float *dout_sq, unsigned int *top_sq, bool vec, cudaStream_t st) {
    const cudaError_t e = cudaMemsetAsync(top_sq, 0, (size_t)2 * a.B * a.Hkv * sizeof(unsigned int), st);
    if (e != cudaSuccess) return fail((int)e, "hsa_dense_attn_bwd: %s", cudaGetErrorString(e));
    int rc = 0;
    const bool ok = dispatch_row_shape<__half>(a.D, vec, [&]<typename T, int VEC, int LPR, int CPL>() {
        constexpr int per = kStretch * (256 / LPR);
        const long long q_blocks = ((long long)a.group * a.lq_pad + per - 1) / per, v_blocks = (a.Lk + kValueRows - 1) / kValueRows;
        const long long blocks = (q_blocks + v_blocks) * a.B * a.Hkv;
        if (blocks > 0x7fffffffLL || (long long)a.group * a.lq_pad > 0x7fffffffLL) { rc = fail(HSA_ERR_ARG, "hsa_dense_attn_bwd: too many rows"); return; }
        dense_delta_f16_kernel<VEC, LPR, CPL><<<(unsigned)blocks, 256, 0, st>>>(a, neg_lse2, neg_delta, dout_sq, top_sq, (int)q_blocks, (int)v_blocks);
        rc = launch_status("hsa_dense_attn_bwd(row sums)");
    });
    return ok ? rc : fail(HSA_ERR_ARG, "hsa_dense_attn_bwd: head dim %d not supported", a.D);
}

static bool rows_in_fours(const hsa_view &v, int esize) {
    return (reinterpret_cast<uintptr_t>(v.ptr) % (4 * esize)) == 0 && v.batch_stride % 4 == 0 && v.row_stride % 4 == 0;
}

static int check_shape(const char *who, int B, int Lq, int Lk, int H, int Hkv, int D, float scale, int dtype, int algo) {
    HSA_CHECK_ARG(B >= 1 && Lq >= 1 && Lk >= 1 && H >= 1 && Hkv >= 1, "%s: bad shape B=%d Lq=%d Lk=%d H=%d Hkv=%d", who, B, Lq, Lk, H, Hkv);
    HSA_CHECK_ARG(H % Hkv == 0, "%s: %d query heads are not a multiple of %d key/value heads", who, H, Hkv);
    HSA_CHECK_ARG(D >= 1 && D <= 256, "%s: head dim %d outside 1..256", who, D);
    HSA_CHECK_ARG(Lq <= (1 << 30) && Lk <= (1 << 30), "%s: more than 2^30 rows", who);
    HSA_CHECK_ARG((long long)(H / Hkv) * Lq <= (1LL << 30), "%s: more than 2^30 query rows per key/value head", who);
    HSA_CHECK_ARG(scale > 0.f && scale < INFINITY, "%s: the scale must be positive and finite", who);
    HSA_CHECK_ARG(algo >= 0 && algo <= 2, "%s: unknown algo %d", who, algo);
    if (dtype != HSA_F32 && dtype != HSA_BF16 && dtype != HSA_F16) return fail(HSA_ERR_DTYPE, "unknown dtype code %d", dtype);
    return 0;
}

static int check_mask(const char *who, const void *packed, int mb, int mh, int mr, int B, int H, int Lq) {
    if (packed == nullptr) return 0;
    HSA_CHECK_ARG((mb == 1 || mb == B) && (mh == 1 || mh == H) && (mr == 1 || mr == Lq),
                  "%s: the mask's sizes (%d, %d, %d) do not broadcast to (%d, %d, %d)", who, mb, mh, mr, B, H, Lq);
    return 0;
}

}  // namespace hsa

using namespace hsa;

extern "C" size_t hsa_dense_mask_bytes(int batches, int heads, int rows, int Lk) {
    if (batches < 1 || heads < 1 || rows < 1 || Lk < 1) return 0;
    return dense_mask_layout((long long)batches * heads, rows, Lk).total;
}

extern "C" int hsa_dense_mask_pack(const void *mask, int64_t stride_b, int64_t stride_h, int64_t stride_q, int64_t stride_k,
                                   int batches, int heads, int rows, int Lk, void *packed, size_t packed_bytes, void *stream) {
    HSA_CHECK_ARG(mask && packed, "hsa_dense_mask_pack: null pointer");
    HSA_CHECK_ARG(batches >= 1 && heads >= 1 && rows >= 1 && Lk >= 1 && rows <= (1 << 30) && Lk <= (1 << 30),
                  "hsa_dense_mask_pack: bad shape (%d, %d, %d, %d)", batches, heads, rows, Lk);
    const long long planes = (long long)batches * heads;
    const DenseMaskLayout l = dense_mask_layout(planes, rows, Lk);
    if (packed_bytes < l.total) return fail(HSA_ERR_WORKSPACE, "hsa_dense_mask_pack: %zu bytes needed, %zu given", l.total, packed_bytes);
    if (reinterpret_cast<uintptr_t>(packed) & 255u) return fail(HSA_ERR_ALIGN, "hsa_dense_mask_pack: the packed mask must be 256-byte aligned");
    const long long cells = planes * l.tq * l.tk;
    HSA_CHECK_ARG(cells <= 0x7fffffffLL, "hsa_dense_mask_pack: too many cells");
    char *p = (char *)packed;
    if (rows > 1) {
        const cudaError_t e = cudaMemsetAsync(p + l.seen, 0, (size_t)planes * l.wk * 4, (cudaStream_t)stream);
        if (e != cudaSuccess) return fail((int)e, "hsa_dense_mask_pack: %s", cudaGetErrorString(e));
    }
    dense_mask_pack_kernel<<<(unsigned)cells, 512, 0, (cudaStream_t)stream>>>(
        (const uint8_t *)mask, stride_b, stride_h, stride_q, stride_k, heads, rows, Lk, (uint32_t *)(p + l.bits),
        rows > 1 ? (uint32_t *)(p + l.bits_t) : nullptr, (uint32_t *)(p + l.seen), (uint8_t *)(p + l.tiles), l.wk, l.wq, l.tq, l.tk);
    return launch_status("hsa_dense_mask_pack");
}

// The tcgen05 kernels may turn inputs down for their alignment as well, so the room is that of whichever kernels need more.
static bool tc_shape(int D, int dtype, int algo) { return D <= 128 && D % 8 == 0 && algo != 1 && dtype != HSA_F32; }

extern "C" size_t hsa_dense_attn_fwd_workspace_bytes(int B, int Lq, int Lk, int H, int Hkv, int D, int dtype, int algo) {
    if (B < 1 || Lq < 1 || Lk < 1 || H < 1 || Hkv < 1 || D < 1) return 0;
    const size_t f32 = algo != 2 ? dense_fwd_f32_workspace(B, Lq, Lk, H, D) : 0;
    const size_t tc = tc_shape(D, dtype, algo) ? dense_fwd_tc_workspace(B, Lq, Lk, H, D) : 0;
    return f32 > tc ? f32 : tc;
}

extern "C" int hsa_dense_attn_fwd(hsa_view Q, hsa_view K, hsa_view V, hsa_view Out, void *out_rest, float *LSE, const int *key_lengths,
                                  const void *packed_mask, int mask_batches, int mask_heads, int mask_rows, void *workspace,
                                  size_t workspace_bytes, int B, int Lq, int Lk, int H, int Hkv, int D, float scale,
                                  float empty_value, int dtype, int algo, void *stream) {
    HSA_CHECK_ARG(Q.ptr && K.ptr && V.ptr && Out.ptr, "hsa_dense_attn_fwd: null pointer");
    if (int rc = check_shape("hsa_dense_attn_fwd", B, Lq, Lk, H, Hkv, D, scale, dtype, algo)) return rc;
    if (int rc = check_mask("hsa_dense_attn_fwd", packed_mask, mask_batches, mask_heads, mask_rows, B, H, Lq)) return rc;
    DenseArgs a{};
    Q = dense_view(Q, B, Lq, H, D); Out = dense_view(Out, B, Lq, H, D);
    K = dense_view(K, B, Lk, Hkv, D); V = dense_view(V, B, Lk, Hkv, D);
    HSA_CHECK_ARG(out_rest == nullptr || dtype != HSA_F32, "hsa_dense_attn_fwd: a float32 output has no rounding rest");
    if (!aligned16(out_rest)) return fail(HSA_ERR_ALIGN, "hsa_dense_attn_fwd: the rounding rest must be 16-byte aligned");
    a.q = Q; a.k = K; a.v = V; a.out = Out; a.out_lo = out_rest; a.lse = LSE;
    a.key_lengths = key_lengths;
    a.mask = dense_mask_view(packed_mask, mask_batches, mask_heads, mask_rows, Lk);
    a.B = B; a.Lq = Lq; a.Lk = Lk; a.H = H; a.Hkv = Hkv; a.D = D; a.group = H / Hkv;
    a.lq_pad = (Lq + 127) / 128 * 128;
    a.scale = scale; a.scale_log2 = scale * 1.4426950408889634f; a.empty_value = empty_value;
    const int es = dtype_size(dtype);
    a.vec = D % 4 == 0;
    for (const hsa_view &v : {Q, K, V, Out}) a.vec = a.vec && rows_in_fours(v, es);
    // The tcgen05 kernel wherever its layout rules allow it: from the smallest call on it is not behind the 32-bit kernel (16 x 77,
    // 8 heads of 64: both are bound by the launch), and at 4096 x 4096 it is 40 times as fast.
    const size_t need = hsa_dense_attn_fwd_workspace_bytes(B, Lq, Lk, H, Hkv, D, dtype, algo);
    if (need && (workspace == nullptr || workspace_bytes < need))
        return fail(HSA_ERR_WORKSPACE, "hsa_dense_attn_fwd: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return fail(HSA_ERR_ALIGN, "hsa_dense_attn_fwd: workspace must be 256-byte aligned");
    if (algo != 1 && dense_tc_ok(a, dtype, false)) return dense_fwd_tc(a, workspace, dtype, (cudaStream_t)stream);
    HSA_CHECK_ARG(algo != 2, "hsa_dense_attn_fwd: no tensor-core kernel for these inputs");
    return dense_fwd_f32(a, workspace, dtype, (cudaStream_t)stream);
}

// Row sums and log-sum-exps of the padded rows, in float16 with what the shift of score gradients follows from, then what the kernels
// keep of partial gradients
static size_t bwd_stats_bytes(int B, int Lq, int H, int Hkv, bool f16) {
    const size_t row = (size_t)B * H * ((Lq + 127) / 128 * 128) * sizeof(float);
    return f16 ? 3 * row + ((size_t)2 * B * Hkv * sizeof(unsigned int) + 255) / 256 * 256 : 2 * row;
}

extern "C" size_t hsa_dense_attn_bwd_workspace_bytes(int B, int Lq, int Lk, int H, int Hkv, int D, int dtype, int algo) {
    if (B < 1 || Lq < 1 || Lk < 1 || H < 1 || Hkv < 1 || H % Hkv != 0 || D < 1) return 0;
    const size_t f32 = algo != 2 ? dense_bwd_f32_workspace(B, Lq, Lk, H, Hkv, D) : 0;
    const size_t tc = tc_shape(D, dtype, algo) ? dense_bwd_tc_workspace(B, Lq, Lk, H, Hkv, D) : 0;
    return bwd_stats_bytes(B, Lq, H, Hkv, dtype == HSA_F16 && tc_shape(D, dtype, algo)) + (f32 > tc ? f32 : tc);
}

extern "C" int hsa_dense_attn_bwd(hsa_view Q, hsa_view K, hsa_view V, hsa_view Out, const void *out_rest, const float *LSE, hsa_view dOut, hsa_view dQ,
                                  hsa_view dK, hsa_view dV, const int *key_lengths, const void *packed_mask, int mask_batches,
                                  int mask_heads, int mask_rows, void *workspace, size_t workspace_bytes, int B, int Lq, int Lk,
                                  int H, int Hkv, int D, float scale, int dtype, int algo, void *stream) {
    HSA_CHECK_ARG(Q.ptr && K.ptr && V.ptr && Out.ptr && LSE && dOut.ptr && (dQ.ptr || dK.ptr), "hsa_dense_attn_bwd: null pointer");
    HSA_CHECK_ARG((dK.ptr == nullptr) == (dV.ptr == nullptr), "hsa_dense_attn_bwd: dK and dV are wanted together or not at all");
    if (int rc = check_shape("hsa_dense_attn_bwd", B, Lq, Lk, H, Hkv, D, scale, dtype, algo)) return rc;
    if (int rc = check_mask("hsa_dense_attn_bwd", packed_mask, mask_batches, mask_heads, mask_rows, B, H, Lq)) return rc;
    const size_t need = hsa_dense_attn_bwd_workspace_bytes(B, Lq, Lk, H, Hkv, D, dtype, algo);
    if (workspace == nullptr || workspace_bytes < need)
        return fail(HSA_ERR_WORKSPACE, "hsa_dense_attn_bwd: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return fail(HSA_ERR_ALIGN, "hsa_dense_attn_bwd: workspace must be 256-byte aligned");
    DenseArgs a{};
    for (hsa_view *v : {&Q, &Out, &dOut, &dQ}) *v = dense_view(*v, B, Lq, H, D);
    for (hsa_view *v : {&K, &V, &dK, &dV}) *v = dense_view(*v, B, Lk, Hkv, D);
    HSA_CHECK_ARG(out_rest == nullptr || dtype != HSA_F32, "hsa_dense_attn_bwd: a float32 output has no rounding rest");
    if (!aligned16(out_rest)) return fail(HSA_ERR_ALIGN, "hsa_dense_attn_bwd: the rounding rest must be 16-byte aligned");
    a.q = Q; a.k = K; a.v = V; a.out = Out; a.out_lo = const_cast<void *>(out_rest); a.dout = dOut; a.dq = dQ; a.dk = dK; a.dv = dV;
    a.lse = const_cast<float *>(LSE);
    a.key_lengths = key_lengths;
    a.mask = dense_mask_view(packed_mask, mask_batches, mask_heads, mask_rows, Lk);
    a.B = B; a.Lq = Lq; a.Lk = Lk; a.H = H; a.Hkv = Hkv; a.D = D; a.group = H / Hkv;
    a.lq_pad = (Lq + 127) / 128 * 128;
    a.scale = scale; a.scale_log2 = scale * 1.4426950408889634f;
    float *neg_lse2 = (float *)workspace, *neg_delta = neg_lse2 + (size_t)B * H * a.lq_pad;
    a.neg_lse2 = neg_lse2; a.neg_delta = neg_delta;
    const int es = dtype_size(dtype);
    a.vec = D % 4 == 0;
    for (const hsa_view &v : {Q, K, V, dOut, dQ, dK, dV}) a.vec = a.vec && (v.ptr == nullptr || rows_in_fours(v, es));
    const bool tc = algo != 1 && dense_tc_ok(a, dtype, true) && dense_bwd_tables_ok(a);
    HSA_CHECK_ARG(algo != 2 || tc, "hsa_dense_attn_bwd: no tensor-core kernel for these inputs");
    cudaStream_t st = (cudaStream_t)stream;
    const bool f16 = dtype == HSA_F16 && tc_shape(D, dtype, algo), vec = D % (16 / es) == 0 && view_vec_ok(Out, es) && view_vec_ok(dOut, es);
    if (f16 && tc) {
        float *dout_sq = neg_delta + (size_t)B * H * a.lq_pad;
        unsigned int *top_sq = (unsigned int *)(dout_sq + (size_t)B * H * a.lq_pad);
        a.dout_sq = dout_sq; a.top_sq = top_sq;
        if (int rc = dense_delta_f16(a, neg_lse2, neg_delta, dout_sq, top_sq, vec, st)) return rc;
    } else if (int rc = dense_delta(a, neg_lse2, neg_delta, dtype, vec, st)) {
        return rc;
    }
    void *rest = (char *)workspace + bwd_stats_bytes(B, Lq, H, Hkv, f16);
    return tc ? dense_bwd_tc(a, rest, dtype, st) : dense_bwd_f32(a, rest, dtype, st);
}
