// Attention of one new token per sequence over a key/value cache that lives in pages.
//
//   out[b, h] = sum over j < length[b] of softmax_j(scale q[b, h].k_j) v_j,   key j in page table[b, j / page], slot j % page
//
// Bound by HBM: every key and value row is read once, for all query heads that share it.  A sequence's keys are cut into
// `splits` ranges that run as separate blocks (there are few rows and a long axis); each range keeps its running maximum m,
// sum l and weighted sum o in float32, and a second kernel joins them: M = max m, out = sum e^(m-M) o / sum e^(m-M) l.
// With one split the block writes the output itself.
//
// Measured, bf16: 2 x 131072 keys, 32 query heads on 4 key/value heads of 128, 537 MB: 88.6 us = 6.06 TB/s, 0.94 of the measured
// copy bandwidth; 32 sequences of ragged length up to 4096, 16 heads of 128, 524 MB: 89.6 us = 0.90 of it (112 before the longest
// sequences started first).
//
// A page number outside [0, num_pages), or a length outside [0, max_pages * page], is not followed: the sequence's output
// is NaN.  Rows behind a sequence's length are not read.
#include <climits>

#include "dense_attn.cuh"
#include "tc_common.cuh"

namespace hsa {

struct PagedArgs {
    hsa_view q, k, v, out;               // k, v: batch_stride = elements between pages, row_stride = between slots of a page
    const int *table;                    // [B, max_pages]
    int64_t table_stride;
    const int *lengths;                  // [B]
    float *part_o, *part_ml;             // [splits, B, H, D] weighted sums; [splits, B, H, 2] maximum (base 2) and sum
    int B, H, Hkv, D, group;
    int page, page_shift;                // page_shift >= 0 when the page size is a power of two
    int num_pages, max_pages, splits;
    float scale_log2;
};

constexpr int kPagedWarps = 4;

// The keys [k0, k1) of a split: equal shares of the sequence's own length, in whole steps of 64 keys.  Returns false for a
// length that the table cannot hold.
__device__ __forceinline__ bool split_range(const PagedArgs &a, int b, int split, int &k0, int &k1) {
    const int n = __ldg(a.lengths + b);
    const bool ok = n >= 0 && (long long)n <= (long long)a.max_pages * a.page;
    const int len = ok ? n : 0;
    const int steps = (len + 63) / 64, per = (steps + a.splits - 1) / a.splits;
    k0 = (int)min((long long)len, (long long)split * per * 64);
    k1 = (int)min((long long)len, (long long)(split + 1) * per * 64);
    return ok;
}

__device__ __forceinline__ void split_page(const PagedArgs &a, int key, int &index, int &slot) {
    if (a.page_shift >= 0) {
        index = key >> a.page_shift;
        slot = key & (a.page - 1);
    } else {
        index = key / a.page;
        slot = key - index * a.page;
    }
}

// ------------------------------------------------------------------------------------------------- any type, CUDA cores
// A warp takes 32 / LPK keys at a time, LPK lanes per key, four elements (NV pieces of four) per lane; GM query heads share
// every row that is loaded.
template <typename T, int LPK, int NV, int GM>
__global__ void __launch_bounds__(kPagedWarps * 32) paged_decode_simt_kernel(const PagedArgs a) {
    constexpr int KPW = 32 / LPK, UNITS = kPagedWarps * KPW, DP = LPK * NV * 4, U = NV == 1 ? 4 : 2;
    __shared__ __align__(16) float so[UNITS][GM][DP];
    __shared__ float sm[UNITS][GM], sl[UNITS][GM];
    const int chunks = (a.group + GM - 1) / GM;
    const int split = blockIdx.x % a.splits, gc = blockIdx.x / a.splits % chunks;
    const int hk = blockIdx.x / a.splits / chunks % a.Hkv, b = blockIdx.x / a.splits / chunks / a.Hkv;
    const int h0 = hk * a.group + gc * GM, heads = min(GM, a.group - gc * GM);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LPK, g = lane % LPK;
    int k0, k1;
    bool bad = !split_range(a, b, split, k0, k1);

    auto load = [&](const T *row, float (&x)[NV * 4]) {
#pragma unroll
        for (int p = 0; p < NV; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = (p * LPK + g) * 4 + e;
                x[p * 4 + e] = (row != nullptr && c < a.D) ? Traits<T>::to_f(row[c]) : 0.f;
            }
    };
    auto load_fast = [&](const T *row, float (&x)[NV * 4]) {      // D a multiple of four, rows aligned to four elements
#pragma unroll
        for (int p = 0; p < NV; ++p) {
            const int c = (p * LPK + g) * 4;
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row != nullptr && c < a.D) {
                if constexpr (sizeof(T) == 4) {
                    f = __ldg(reinterpret_cast<const float4 *>(row + c));
                } else {
                    const uint2 raw = __ldg(reinterpret_cast<const uint2 *>(row + c));
                    const T *t = reinterpret_cast<const T *>(&raw);
                    f = make_float4(Traits<T>::to_f(t[0]), Traits<T>::to_f(t[1]), Traits<T>::to_f(t[2]), Traits<T>::to_f(t[3]));
                }
            }
            x[p * 4] = f.x; x[p * 4 + 1] = f.y; x[p * 4 + 2] = f.z; x[p * 4 + 3] = f.w;
        }
    };
    const bool fast = a.D % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.k.ptr) | reinterpret_cast<uintptr_t>(a.v.ptr)) % (4 * sizeof(T))) == 0 &&
                      ((a.k.batch_stride | a.k.row_stride | a.v.batch_stride | a.v.row_stride) & 3) == 0;

    float q[GM][NV * 4], o[GM][NV * 4], m[GM], l[GM];
#pragma unroll
    for (int i = 0; i < GM; ++i) {
        load(i < heads ? (const T *)a.q.ptr + b * a.q.batch_stride + (int64_t)(h0 + i) * a.D : nullptr, q[i]);
        m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < NV * 4; ++e) { q[i][e] *= a.scale_log2; o[i][e] = 0.f; }
    }
    const unsigned mask = group_mask<LPK>();
    for (int base = k0 + warp * KPW; base < k1; base += UNITS * U) {
        float kx[U][NV * 4], vx[U][NV * 4];
        bool have[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = base + u * UNITS + sub;
            const T *kr = nullptr, *vr = nullptr;
            have[u] = key < k1;
            if (have[u]) {
                int index, slot;
                split_page(a, key, index, slot);
                const int page = __ldg(a.table + b * a.table_stride + index);
                if (page < 0 || page >= a.num_pages) {
                    bad = true;
                } else {
                    kr = (const T *)a.k.ptr + (int64_t)page * a.k.batch_stride + (int64_t)slot * a.k.row_stride + (int64_t)hk * a.D;
                    vr = (const T *)a.v.ptr + (int64_t)page * a.v.batch_stride + (int64_t)slot * a.v.row_stride + (int64_t)hk * a.D;
                }
            }
            if (fast) { load_fast(kr, kx[u]); load_fast(vr, vx[u]); } else { load(kr, kx[u]); load(vr, vx[u]); }
        }
#pragma unroll
        for (int i = 0; i < GM; ++i) {
            float s[U], top = m[i];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float d = 0.f;
#pragma unroll
                for (int e = 0; e < NV * 4; ++e) d = fmaf(q[i][e], kx[u][e], d);
                d = group_sum<LPK>(d, mask);
                s[u] = have[u] ? d : -INFINITY;
                top = fmaxf(top, s[u]);
            }
            const float ref = top == -INFINITY ? 0.f : top;
            const float corr = exp2f(m[i] - ref);
            m[i] = top;
            l[i] *= corr;
#pragma unroll
            for (int e = 0; e < NV * 4; ++e) o[i][e] *= corr;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float p = exp2f(s[u] - ref);
                l[i] += p;
#pragma unroll
                for (int e = 0; e < NV * 4; ++e) o[i][e] = fmaf(p, vx[u][e], o[i][e]);
            }
        }
    }
    const int unit = warp * KPW + sub;
#pragma unroll
    for (int i = 0; i < GM; ++i) {
        if (g == 0) { sm[unit][i] = m[i]; sl[unit][i] = l[i]; }
#pragma unroll
        for (int p = 0; p < NV; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) so[unit][i][(p * LPK + g) * 4 + e] = o[i][p * 4 + e];
    }
    const bool any_bad = __syncthreads_or(bad);
    for (int idx = threadIdx.x; idx < heads * DP; idx += kPagedWarps * 32) {
        const int i = idx / DP, c = idx % DP;
        float M = -INFINITY;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) M = fmaxf(M, sm[u][i]);
        const float ref = M == -INFINITY ? 0.f : M;
        float L = 0.f, acc = 0.f;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const float w = exp2f(sm[u][i] - ref);
            L = fmaf(w, sl[u][i], L);
            acc = fmaf(w, so[u][i][c], acc);
        }
        if (any_bad) { L = NAN; M = 0.f; acc = NAN; }
        if (c >= a.D) continue;
        if (a.splits == 1) {
            T *out = (T *)a.out.ptr + b * a.out.batch_stride + (int64_t)(h0 + i) * a.D;
            out[c] = Traits<T>::from_f(L == 0.f ? 0.f : acc / L);
        } else {
            const int64_t row = ((int64_t)split * a.B + b) * a.H + h0 + i;
            a.part_o[row * a.D + c] = acc;
            if (c == 0) { a.part_ml[2 * row] = M; a.part_ml[2 * row + 1] = L; }
        }
    }
}

// ------------------------------------------------------------------------------- bf16 / f16, 16 query heads at a time
// A warp takes 16 keys at a time through its own ring of cp.async stages (no barrier in the loop): scores and weighted sums are
// m16n8k16 products whose 16 rows are the query heads that share the key head (rows behind them are zeros).  Half-empty tiles
// cost nothing here: a 4 KB step of K takes 16 products, far less than HBM needs to deliver it.  Rows are 16-byte pieces
// swizzled by the row number, which keeps ldmatrix free of bank conflicts.  The running maximum is raised, and the sums
// rescaled, only when a score exceeds it by 2^8.  Weights are rounded to the type for the second product; their sum is not.  In
// float16 they are 2^7 times as large, so that many small ones next to a large one keep their bits (they stay below 2^15).
template <int DP> struct PagedShape {
    // Three stages: at head dims up to 64 four blocks then share an SM, and one block's first loads pass under another's loop (six
    // stages and two blocks, the same bytes in flight: 20 sequences of 8192 keys, 16 heads of 64, 166 us against 115; 100 of 512, 71
    // against 45).  Two stages and three blocks at head dim 128: 92.9 us against 87.5 for 2 x 131072 keys.
    static constexpr int kStages = 3;
    static constexpr int kStage = 2 * 16 * DP * 2;                               // 16 rows of K and of V
    static constexpr int kSmem = kPagedWarps * kStages * kStage + 2 * kPagedWarps * 16 * 4;
};

// The batch entry that comes at place `at` when longer sequences come first (equal ones in their order).  All threads of a block call
// it; B <= threads.
__device__ __forceinline__ int by_length(const PagedArgs &a, int at) {
    __shared__ int found;
    __shared__ __align__(16) int lengths[kPagedWarps * 32];
    const int i = threadIdx.x, mine = i < a.B ? __ldg(a.lengths + i) : INT_MIN;
    lengths[i] = mine;
    __syncthreads();
    int rank = 0;
    for (int j = 0; j < a.B; j += 4) {
        const int4 x = *reinterpret_cast<const int4 *>(lengths + j);
        rank += (x.x > mine || (x.x == mine && j < i)) + (x.y > mine || (x.y == mine && j + 1 < i)) +
                (x.z > mine || (x.z == mine && j + 2 < i)) + (x.w > mine || (x.w == mine && j + 3 < i));
    }
    if (rank == at) found = i;
    __syncthreads();
    return found;
}

template <typename T, int DP, bool SORTED>
__global__ void __launch_bounds__(kPagedWarps * 32) paged_decode_mma_kernel(const PagedArgs a) {
    using Shape = PagedShape<DP>;
    constexpr float SHIFT = std::is_same<T, __half>::value ? 7.f : 0.f;
    constexpr int ST = Shape::kStages, CPR = DP / 8, PIECES = 16 * CPR / 32;
    extern __shared__ __align__(128) unsigned char smem[];
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int chunks = (a.group + 15) / 16;
    const int split = blockIdx.x % a.splits, gc = blockIdx.x / a.splits % chunks;
    const int hk = blockIdx.x / a.splits / chunks % a.Hkv, at = blockIdx.x / a.splits / chunks / a.Hkv;
    const int b = SORTED ? by_length(a, at) : at;
    const int h0 = hk * a.group + gc * 16, heads = min(16, a.group - gc * 16);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, grow = lane >> 2;
    unsigned char *ring = smem + warp * ST * Shape::kStage;
    float *ml = reinterpret_cast<float *>(smem + kPagedWarps * ST * Shape::kStage);       // [warps][2][16]
    int k0, k1;
    bool bad = !split_range(a, b, split, k0, k1);
    const int steps = (k1 - k0 + 63) / 64;                       // of 16 keys per warp

    // where the row that this lane looks up (lane & 15) of step t lies; page < 0: no such key
    auto look_up = [&](int t, int &page, int &slot) {
        const int key = k0 + (t * kPagedWarps + warp) * 16 + (lane & 15);
        page = -1; slot = 0;
        if (t < steps && key < k1) {
            int index;
            split_page(a, key, index, slot);
            page = __ldg(a.table + b * a.table_stride + index);
            if (page < 0 || page >= a.num_pages) { bad = true; page = -1; }
        }
    };
    const T *kb = (const T *)a.k.ptr + (int64_t)hk * a.D, *vb = (const T *)a.v.ptr + (int64_t)hk * a.D;
    auto stage_in = [&](int st, int page, int slot) {
        const uint32_t dst = smem_u32(ring + st * Shape::kStage);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int c = i * 32 + lane, r = c / CPR, ch = c % CPR;
            const int pg = __shfl_sync(0xffffffffu, page, r), sl = __shfl_sync(0xffffffffu, slot, r);
            const bool there = pg >= 0 && ch * 8 < a.D;
            const int64_t ko = there ? (int64_t)pg * a.k.batch_stride + (int64_t)sl * a.k.row_stride + ch * 8 : 0;
            const int64_t vo = there ? (int64_t)pg * a.v.batch_stride + (int64_t)sl * a.v.row_stride + ch * 8 : 0;
            const uint32_t at = dst + r * (DP * 2) + ((ch ^ (r & 7)) << 4);
            cp_async16(at, kb + ko, there);
            cp_async16(at + 16 * DP * 2, vb + vo, there);
        }
    };
    int page, slot;
#pragma unroll
    for (int t = 0; t < ST - 1; ++t) {
        look_up(t, page, slot);
        stage_in(t, page, slot);
        cp_async_commit();
    }
    look_up(ST - 1, page, slot);                                 // one step ahead of its copies: the table's latency is hidden

    uint32_t q[DP / 16][4];
    {
        const T *Q = (const T *)a.q.ptr + b * a.q.batch_stride + (int64_t)h0 * a.D;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = grow + (e & 1) * 8, col = k * 16 + (e >> 1) * 8 + quad * 2;
                q[k][e] = row < heads && col < a.D ? ldg32(Q + (int64_t)row * a.D + col) : 0u;
            }
    }
    float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

    int st = 0, st_in = ST - 1;
    for (int t = 0; t < steps; ++t) {
        cp_async_wait<ST - 2>();
        __syncwarp();                                            // everybody's pieces of this step, and nobody reads the next target any more
        stage_in(st_in, page, slot);
        cp_async_commit();
        look_up(t + ST, page, slot);
        const uint32_t kt = smem_u32(ring + st * Shape::kStage), vt = kt + 16 * DP * 2;
        if (++st == ST) st = 0;
        if (++st_in == ST) st_in = 0;
        const int base = k0 + (t * kPagedWarps + warp) * 16;
        if (base >= k1) continue;                                // the last step has keys for some of the warps only
        float s[2][4] = {};
        const int mi = lane >> 3, mr = lane & 7;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            uint32_t f[4];
            ldmatrix_x4(f, kt + ((mi >> 1) * 8 + mr) * (DP * 2) + (((k * 2 + (mi & 1)) ^ mr) << 4));
            mma16816<T>(s[0], q[k], f[0], f[1]);
            mma16816<T>(s[1], q[k], f[2], f[3]);
        }
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = base + n * 8 + quad * 2 + (e & 1);
                s[n][e] = key < k1 ? s[n][e] * a.scale_log2 : -INFINITY;
                top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
            }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] + 8.f || top[1] > m[1] + 8.f)) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float up = fmaxf(m[r], top[r]), corr = up == -INFINITY ? 1.f : fast_exp2(m[r] - up);
                m[r] = up;
                l[r] *= corr;
#pragma unroll
                for (int i = 0; i < DP / 8; ++i) { o[i][2 * r] *= corr; o[i][2 * r + 1] *= corr; }
            }
        }
        const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0] - SHIFT, m[1] == -INFINITY ? 0.f : m[1] - SHIFT};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] = fast_exp2(s[n][e] - ref[e >> 1]);
                l[e >> 1] += s[n][e];
            }
        const uint32_t p[4] = {pack2_finite<T>(s[0][0], s[0][1]), pack2_finite<T>(s[0][2], s[0][3]), pack2_finite<T>(s[1][0], s[1][1]), pack2_finite<T>(s[1][2], s[1][3])};
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
            uint32_t f[4];
            ldmatrix_x4_trans(f, vt + ((mi & 1) * 8 + mr) * (DP * 2) + (((d * 2 + (mi >> 1)) ^ mr) << 4));
            mma16816<T>(o[2 * d], p, f[0], f[1]);
            mma16816<T>(o[2 * d + 1], p, f[2], f[3]);
        }
    }
    cp_async_wait<0>();
    __syncwarp();
    // the warps' sums meet in the room of their rings
    float *mine = reinterpret_cast<float *>(ring);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (quad == 0) { ml[warp * 32 + grow + 8 * r] = m[r]; ml[warp * 32 + 16 + grow + 8 * r] = l[r]; }
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
            *reinterpret_cast<float2 *>(mine + (grow + 8 * r) * DP + i * 8 + quad * 2) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
    }
    const bool any_bad = __syncthreads_or(bad);
    const int fours = a.D / 4;
    for (int idx = threadIdx.x; idx < heads * fours; idx += kPagedWarps * 32) {
        const int i = idx / fours, c = idx % fours * 4;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kPagedWarps; ++w) M = fmaxf(M, ml[w * 32 + i]);
        const float ref = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kPagedWarps; ++w) {
            const float f = fast_exp2(ml[w * 32 + i] - ref);
            const float4 x = *reinterpret_cast<const float4 *>(reinterpret_cast<float *>(smem + w * ST * Shape::kStage) + i * DP + c);
            L = fmaf(f, ml[w * 32 + 16 + i], L);
            acc.x = fmaf(f, x.x, acc.x); acc.y = fmaf(f, x.y, acc.y); acc.z = fmaf(f, x.z, acc.z); acc.w = fmaf(f, x.w, acc.w);
        }
        if (any_bad) { L = NAN; M = 0.f; acc = make_float4(NAN, NAN, NAN, NAN); }
        if (a.splits == 1) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            *reinterpret_cast<uint2 *>((T *)a.out.ptr + b * a.out.batch_stride + (int64_t)(h0 + i) * a.D + c) =
                make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
        } else {
            const int64_t row = ((int64_t)split * a.B + b) * a.H + h0 + i;
            *reinterpret_cast<float4 *>(a.part_o + row * a.D + c) = acc;
            if (c == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * row) = make_float2(M, L);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ join
// A block per output row; its eight warps take every eighth range and meet in shared memory.
constexpr int kJoinWarps = 8;
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const PagedArgs a) {
    __shared__ float so[kJoinWarps][256], sm[kJoinWarps], sl[kJoinWarps];
    asm volatile("griddepcontrol.wait;\n" ::: "memory");       // launched while the ranges still run: their sums come first
    const int64_t bh = blockIdx.x, rows = (int64_t)a.B * a.H;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float M = -INFINITY;
    for (int s = warp + lane * kJoinWarps; s < a.splits; s += 32 * kJoinWarps) M = fmaxf(M, a.part_ml[2 * (s * rows + bh)]);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc[8] = {};
#pragma unroll 4
    for (int s = warp; s < a.splits; s += kJoinWarps) {
        const int64_t row = s * rows + bh;
        const float w = exp2f(a.part_ml[2 * row] - ref);        // 0 for a range without keys
        L = fmaf(w, a.part_ml[2 * row + 1], L);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j * 32 + lane < a.D) acc[j] = fmaf(w, a.part_o[row * a.D + j * 32 + lane], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) so[warp][j * 32 + lane] = acc[j];
    if (lane == 0) { sm[warp] = M; sl[warp] = L; }
    __syncthreads();
    M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) M = fmaxf(M, sm[w]);
    const float base = M == -INFINITY ? 0.f : M;
    for (int c = threadIdx.x; c < a.D; c += kJoinWarps * 32) {
        float total = 0.f, x = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) {
            const float f = exp2f(sm[w] - base);
            total = fmaf(f, sl[w], total);
            x = fmaf(f, so[w][c], x);
        }
        T *out = (T *)a.out.ptr + (bh / a.H) * a.out.batch_stride + (bh % a.H) * a.D;
        out[c] = Traits<T>::from_f(total == 0.f ? 0.f : x / total);
    }
}

template <typename T>
static int paged_mma(const PagedArgs &a, bool sorted, cudaStream_t st) {
    const long long blocks = (long long)a.B * a.Hkv * ((a.group + 15) / 16) * a.splits;
    if (blocks > 0x7fffffffLL) return fail(HSA_ERR_ARG, "hsa_paged_attn_decode: too many blocks");
    auto go = [&]<int DP, bool SORTED>() -> int {
        constexpr auto kernel = paged_decode_mma_kernel<T, DP, SORTED>;
        constexpr int smem = PagedShape<DP>::kSmem;
        const cudaError_t e = allow_smem<kernel>(smem);
        if (e != cudaSuccess) return fail((int)e, "hsa_paged_attn_decode: shared memory %d: %s", smem, cudaGetErrorString(e));
        kernel<<<(unsigned)blocks, kPagedWarps * 32, smem, st>>>(a);
        return launch_status("hsa_paged_attn_decode");
    };
    if (a.D <= 64) return sorted ? go.template operator()<64, true>() : go.template operator()<64, false>();
    if (a.D <= 128) return sorted ? go.template operator()<128, true>() : go.template operator()<128, false>();
    return sorted ? go.template operator()<256, true>() : go.template operator()<256, false>();
}

template <typename T>
static int paged_simt(const PagedArgs &a, cudaStream_t st) {
    auto go = [&]<int LPK, int NV, int GM>() -> int {
        const long long blocks = (long long)a.B * a.Hkv * ((a.group + GM - 1) / GM) * a.splits;
        if (blocks > 0x7fffffffLL) return fail(HSA_ERR_ARG, "hsa_paged_attn_decode: too many blocks");
        paged_decode_simt_kernel<T, LPK, NV, GM><<<(unsigned)blocks, kPagedWarps * 32, 0, st>>>(a);
        return launch_status("hsa_paged_attn_decode");
    };
    auto heads = [&]<int LPK, int NV>() -> int {
        if (a.group == 1) return go.template operator()<LPK, NV, 1>();
        if (a.group <= 4) return go.template operator()<LPK, NV, 4>();
        return go.template operator()<LPK, NV, 8>();
    };
    if (a.D <= 32) return heads.template operator()<8, 1>();
    if (a.D <= 64) return heads.template operator()<16, 1>();
    if (a.D <= 128) return heads.template operator()<32, 1>();
    return heads.template operator()<32, 2>();
}

}  // namespace hsa

using namespace hsa;

// Whether blocks start in the order of their sequences' lengths, the longest first: where more blocks are launched than run at
// once, so that the last ones to start are short, and where sequences may be long enough to pay for every block's look at all
// lengths (64 sequences of up to 2000 keys on 8 heads of 64 in one range: 41.2 us unsorted and 38.3 sorted when ragged, 50.7 and 51.7
// when all are full; 100 of up to 512 on 16 heads would go from 32.2 to 33.6 and from 44.8 to 47.8, and stay unsorted).
static bool paged_sorted(int B, int H, int Hkv, int page_size, int max_pages, int splits) {
    const long long blocks = (long long)B * Hkv * ((H / Hkv + 15) / 16) * splits;
    const long long room = (long long)max_pages * page_size;
    return B > 1 && B <= kPagedWarps * 32 && blocks > 2LL * dense_sm_count() && room >= (long long)splits * (B > 64 ? 8 * B : 512);
}

// Ranges per sequence.  Two blocks fit an SM at head dims from 72 to 128; a block costs its steps of 64 keys plus about two and a
// half steps' time, and the join about one.  The count with the least (rounds of blocks) x (cost of a block): one full round where
// that fits (2 sequences of 131072 keys on 4 key/value heads of 128: 88.7 us in 37 ranges, 96.6 in 74, 144 in 16).  With more sequences
// than blocks fit at once, where lengths may differ: the coarsest cut that costs no more than a tenth if the longest come first (32
// sequences of up to 4096 keys on 16 heads of 128: 89.2 us ragged and 186 full in one range, 110 and 188 in four), else the finest
// that costs no more than a twentieth (the same unsorted: 121 us ragged in one range, 112 in four).  The table's room stands in for
// the lengths, which are on the device.
// The head dim has no part in it, though four blocks fit an SM up to 64 and one above 128: at 64 the count is the best or near it for
// some sizes (20 sequences of up to 8192 keys on 16 heads: three ranges, 57.1 us ragged and 115 full; 100 of 512: one, 44.8) and far
// from it for others (16 of up to 4096 on 16 heads: 54.5 and 60.2 us in its one range, 29.3 and 51.4 in four).
extern "C" int hsa_paged_attn_choose_splits(int B, int H, int Hkv, int page_size, int max_pages) {
    if (B < 1 || H < 1 || Hkv < 1 || page_size < 1 || max_pages < 1) return 1;
    const long long units = (long long)B * Hkv * ((H / Hkv + 15) / 16), room = (long long)max_pages * page_size;
    const long long slots = 2LL * dense_sm_count(), steps = (room + 63) / 64;
    const bool sorted = paged_sorted(B, H, Hkv, page_size, max_pages, 1);
    const bool finer = !sorted && units > slots && units < 8 * slots;
    const int most = (int)(steps < 148 ? steps : 148);
    auto cost = [&](int s) { return (double)((units * s + slots - 1) / slots) * ((double)((steps + s - 1) / s) + 2.5) + (s > 1 ? 1.0 : 0.0); };
    double best = 1e30;
    int best_s = 1;
    for (int s = 1; s <= most; ++s) {
        const double t = cost(s);
        if (t < (finer ? 1.05 : 0.999) * best) {
            if (t < best) best = t;
            best_s = s;
        }
    }
    if (sorted)
        for (int s = 1; s < best_s; ++s)
            if (cost(s) <= 1.1 * best) return s;
    return best_s;
}

extern "C" size_t hsa_paged_attn_workspace_bytes(int B, int H, int D, int splits) {
    if (B < 1 || H < 1 || D < 1 || splits <= 1) return 0;
    return (size_t)splits * B * H * (D + 2) * sizeof(float);
}

extern "C" int hsa_paged_attn_decode(hsa_view q, hsa_view k_pages, hsa_view v_pages, hsa_view out, const int *page_table,
                                     int64_t table_stride, const int *lengths, void *workspace, size_t workspace_bytes, int B, int H,
                                     int Hkv, int D, int page_size, int num_pages, int max_pages, float scale, int dtype, int splits,
                                     int algo, void *stream) {
    HSA_CHECK_ARG(q.ptr && k_pages.ptr && v_pages.ptr && out.ptr && page_table && lengths, "hsa_paged_attn_decode: null pointer");
    HSA_CHECK_ARG(B >= 1 && H >= 1 && Hkv >= 1, "hsa_paged_attn_decode: bad shape B=%d H=%d Hkv=%d", B, H, Hkv);
    HSA_CHECK_ARG(H % Hkv == 0, "hsa_paged_attn_decode: %d query heads are not a multiple of %d key/value heads", H, Hkv);
    HSA_CHECK_ARG(D >= 1 && D <= 256, "hsa_paged_attn_decode: head dim %d outside 1..256", D);
    HSA_CHECK_ARG(page_size >= 1 && num_pages >= 1 && max_pages >= 1, "hsa_paged_attn_decode: bad pages (size %d, %d pages, %d per sequence)",
                  page_size, num_pages, max_pages);
    HSA_CHECK_ARG((long long)max_pages * page_size <= (1LL << 30), "hsa_paged_attn_decode: more than 2^30 keys per sequence");
    HSA_CHECK_ARG(scale > 0.f && scale < INFINITY, "hsa_paged_attn_decode: the scale must be positive and finite");
    HSA_CHECK_ARG(splits >= 1 && splits <= 1024, "hsa_paged_attn_decode: splits out of range");
    HSA_CHECK_ARG(algo >= 0 && algo <= 2, "hsa_paged_attn_decode: unknown algo %d", algo);
    if (dtype != HSA_F32 && dtype != HSA_BF16 && dtype != HSA_F16) return fail(HSA_ERR_DTYPE, "unknown dtype code %d", dtype);
    const size_t need = hsa_paged_attn_workspace_bytes(B, H, D, splits);
    if (need && (workspace == nullptr || workspace_bytes < need))
        return fail(HSA_ERR_WORKSPACE, "hsa_paged_attn_decode: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return fail(HSA_ERR_ALIGN, "hsa_paged_attn_decode: workspace must be 256-byte aligned");
    PagedArgs a{};
    a.q = q; a.k = k_pages; a.v = v_pages; a.out = out;
    a.table = page_table; a.table_stride = table_stride; a.lengths = lengths;
    a.part_o = (float *)workspace;
    a.part_ml = a.part_o ? a.part_o + (size_t)splits * B * H * D : nullptr;
    a.B = B; a.H = H; a.Hkv = Hkv; a.D = D; a.group = H / Hkv;
    a.page = page_size; a.page_shift = (page_size & (page_size - 1)) == 0 ? ilog2((unsigned)page_size) : -1;
    a.num_pages = num_pages; a.max_pages = max_pages; a.splits = splits;
    a.scale_log2 = scale * 1.4426950408889634f;
    const bool sorted = paged_sorted(B, H, Hkv, page_size, max_pages, splits);
    // Whole 16-byte pieces everywhere: the tensor-core kernel
    const bool mma = algo != 1 && dtype != HSA_F32 && D % 8 == 0 && view_vec_ok(k_pages, 2) && view_vec_ok(v_pages, 2) &&
                     view_vec_ok(hsa_view{q.ptr, q.batch_stride, 0}, 2) && view_vec_ok(hsa_view{out.ptr, out.batch_stride, 0}, 2);
    HSA_CHECK_ARG(algo != 2 || mma, "hsa_paged_attn_decode: no tensor-core kernel for these inputs");
    cudaStream_t st = (cudaStream_t)stream;
    int rc;
    if (mma) rc = dtype == HSA_BF16 ? paged_mma<__nv_bfloat16>(a, sorted, st) : paged_mma<__half>(a, sorted, st);
    else rc = dispatch_dtype(dtype, [&]<typename T>() -> int { return paged_simt<T>(a, st); });
    if (rc != 0 || splits == 1) return rc;
    const long long rows = (long long)B * H;
    HSA_CHECK_ARG(rows <= 0x7fffffffLL, "hsa_paged_attn_decode: too many rows");
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)rows);
        cfg.blockDim = dim3(kJoinWarps * 32);
        cfg.stream = st;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_join_kernel<T>, a);
        if (e != cudaSuccess) return fail((int)e, "hsa_paged_attn_decode(join): %s", cudaGetErrorString(e));
        return launch_status("hsa_paged_attn_decode(join)");
    });
}
