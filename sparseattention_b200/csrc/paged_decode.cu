// Attention of one new token per sequence over a key/value cache that lives in pages.
//
//   out[b, h] = sum over j < length[b] of softmax_j(scale q[b, h].k_j) v_j,   key j in page table[b, j / page], slot j % page
//
// Bound by HBM: every key and value row is read once, for all query heads that share it.  A sequence's keys are cut into
// `splits` ranges that run as separate blocks (there are few rows and a long axis); each range keeps its running maximum m,
// sum l and weighted sum o in float32, and a second kernel joins them: M = max m, out = sum e^(m-M) o / sum e^(m-M) l.
// With one split the block writes the output itself.
//
// A page number outside [0, num_pages), or a length outside [0, max_pages * page], is not followed: the sequence's output
// is NaN.  Rows behind a sequence's length are not read.
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

// ------------------------------------------------------------------------------------------------------------ join
template <typename T>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedArgs a) {
    asm volatile("griddepcontrol.wait;\n" ::: "memory");       // launched while the ranges still run: their sums come first
    const int64_t bh = blockIdx.x;
    const int b = (int)(bh / a.H), h = (int)(bh % a.H);
    const int64_t rows = (int64_t)a.B * a.H;
    float M = -INFINITY;
    for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.part_ml[2 * (s * rows + bh)]);
    const float ref = M == -INFINITY ? 0.f : M;
    for (int c = threadIdx.x; c < a.D; c += 128) {
        float L = 0.f, acc = 0.f;
        for (int s = 0; s < a.splits; ++s) {
            const int64_t row = s * rows + bh;
            const float w = exp2f(a.part_ml[2 * row] - ref);    // 0 for a range without keys
            L = fmaf(w, a.part_ml[2 * row + 1], L);
            acc = fmaf(w, a.part_o[row * a.D + c], acc);
        }
        T *out = (T *)a.out.ptr + b * a.out.batch_stride + (int64_t)h * a.D;
        out[c] = Traits<T>::from_f(L == 0.f ? 0.f : acc / L);
    }
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

// Ranges per sequence: enough blocks for four rounds over the GPU, each range at least 256 keys of what the table can hold.
extern "C" int hsa_paged_attn_choose_splits(int B, int H, int Hkv, int page_size, int max_pages) {
    if (B < 1 || H < 1 || Hkv < 1 || page_size < 1 || max_pages < 1) return 1;
    const long long units = (long long)B * Hkv, room = (long long)max_pages * page_size;
    const long long want = (4LL * dense_sm_count() + units - 1) / units, most = (room + 255) / 256;
    const long long s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s > 128 ? 128 : s);
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
    HSA_CHECK_ARG(algo != 2, "hsa_paged_attn_decode: no tensor-core kernel for these inputs");
    cudaStream_t st = (cudaStream_t)stream;
    const int rc = dispatch_dtype(dtype, [&]<typename T>() -> int { return paged_simt<T>(a, st); });
    if (rc != 0 || splits == 1) return rc;
    const long long rows = (long long)B * H;
    HSA_CHECK_ARG(rows <= 0x7fffffffLL, "hsa_paged_attn_decode: too many rows");
    return dispatch_dtype(dtype, [&]<typename T>() -> int {
        paged_join_kernel<T><<<(unsigned)rows, 128, 0, st>>>(a);
        return launch_status("hsa_paged_attn_decode(join)");
    });
}
