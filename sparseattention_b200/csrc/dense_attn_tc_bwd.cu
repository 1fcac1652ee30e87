// Dense attention backward on the 5th-generation tensor cores (bf16 / f16, head dims up to 128).
//
//   p_ij = exp2(c q_i.k_j - lse2_i),  ds_ij = p_ij (do_i.v_j - delta_i),  delta_i = do_i.out_i
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij do_i
//
// Two kernels, one per side, each of which recomputes the scores: seven products instead of the five that one kernel would need,
// but every gradient row has one writer and a fixed order of summation, and no 32-bit partial gradients cross HBM.
//   dq:    a work item is 128 queries against tiles of 128 keys, in halves of 64.  Tensor memory: two buffers of S and dP (64
//          columns each) and dq (DP columns).  dS replaces S in place, as the first operand of dq += dS k.
//   dk/dv: a work item is 128 keys of a key/value head against tiles of 64 queries of all its query heads, with everything
//          transposed (S^T = K Q^T), so that P^T and dS^T can stay in tensor memory, in place of the scores they came from, as
//          the first operands of dv += P^T do and dk += dS^T q.  Two buffers of S^T and dP^T; with dv and dk all 512 columns are
//          in use at DP = 128.
// Eight element-wise warps (two per 32 rows, half of the columns each), one for copies, two for products (scores, gradients).
// While the element-wise warps work on one buffer, the products fill the other.
// Measured at 4096 x 4096, batch 2, 16 heads of 128, bf16: dk/dv 392 to 413 us = 1.33 to 1.40 PFLOP/s, dq 320 to 341 us = 1.21 to
// 1.29 PFLOP/s, tensor pipe 79 and 78 % busy (products with 64 rows on one side read shared memory at its full rate for two
// thirds of the tensor cores').  On the way there: a warpgroup per buffer instead of both on one 738 us and 128 columns in one buffer 436 us;
// products issued from uniform registers 492 and 427 us; scores and gradients issued by a warp each 445 and 350 us; output rows
// through quad transposes 430 and 341 us.
// Rounding: p and ds are rounded to the inputs' type once, as operands; all sums are 32-bit.  In float16 both are moved into the middle
// of the type's range first (grad_shift): p by 2^13, ds by a power of two per query row for dq, per key/value head for dk.  Weights
// come back from the saved log-sum-exp, whose 32 bits hold a score of 1e5 to 1e-2: beyond that gradients follow its rounding.
#include "dense_attn_tc.cuh"

namespace hsa {

constexpr int kBwdThreads = 352;                 // eight element-wise warps, copies, score products, gradient products

__device__ unsigned int g_dense_bwd_aborts = 0;

// ------------------------------------------------------------------------------------------------------------------ dq
template <int DP>
struct DqShape {
    static constexpr int kTile = 128 * DP * 2, kKSlots = 3, kVSlots = 2;
    static constexpr int kBars = 11 + 2 * (kKSlots + kVSlots) + kItemBars;
    static constexpr int kSmem = 1024 + (2 + kKSlots + kVSlots) * kTile + (int)sizeof(ItemSlots) + kBars * 8 + 8;
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

// A work item: 128 query rows of a (batch entry, head) against one range of its keys
struct DqItem {
    int q0, h, hk, b, split, n, kt0, kt1;
    int64_t plane;
    __device__ __forceinline__ DqItem(const DenseArgs &a, int splits, int item) {
        const int qblocks = (a.Lq + 127) / 128;
        q0 = item % qblocks * 128; item /= qblocks;
        h = item % a.H; item /= a.H;
        b = item % a.B; split = item / a.B;
        hk = h / a.group;
        n = dense_keys(a, b);
        const int tiles = (n + 127) / 128, per = (tiles + splits - 1) / splits;
        kt0 = min(tiles, split * per);
        kt1 = min(tiles, kt0 + per);
        plane = (int64_t)b * a.mask.plane_b + (int64_t)h * a.mask.plane_h;
    }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kBwdThreads, 1)
dense_dq_tc5_kernel(const DenseArgs a, const BwdSplit sp, const __grid_constant__ CUtensorMap map_q,
                    const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ CUtensorMap map_g) {
    using namespace tc5;
    using Shape = DqShape<DP>;
    constexpr int TILE = Shape::kTile, KS = Shape::kKSlots, VS = Shape::kVSlots, PLANES = DP / 64, PLANE = 16384;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    constexpr uint32_t IDESC_S = instr_desc(128, 64, BF, false, false), IDESC_O = instr_desc(128, DP, BF, false, true);
    constexpr uint32_t COL_Q = 256;                          // below: two buffers of S and dP, 64 columns each

    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    unsigned char *q_s = smem, *g_s = q_s + TILE, *k_s = g_s + TILE, *v_s = k_s + KS * TILE;
    ItemSlots &items = *reinterpret_cast<ItemSlots *>(v_s + VS * TILE);
    unsigned long long *bars = reinterpret_cast<unsigned long long *>(&items + 1);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + Shape::kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const uint32_t bar0 = smem_addr(bars);
    const uint32_t qg_full = bar0, qg_empty = bar0 + 8, q_done = bar0 + 16, answer = bar0 + 24;
    auto s_full = [&](uint32_t x) { return bar0 + 8u * (5 + x); };
    auto d_full = [&](uint32_t x) { return bar0 + 8u * (7 + x); };
    auto s_free = [&](uint32_t x) { return bar0 + 8u * (9 + x); };
    auto k_full = [&](int s) { return bar0 + 8u * (11 + s); };
    auto k_empty = [&](int s) { return bar0 + 8u * (11 + KS + s); };
    auto v_full = [&](int s) { return bar0 + 8u * (11 + 2 * KS + s); };
    auto v_empty = [&](int s) { return bar0 + 8u * (11 + 2 * KS + VS + s); };
    auto info_full = [&](int s) { return bar0 + 8u * (11 + 2 * KS + 2 * VS + s); };
    auto info_empty = [&](int s) { return bar0 + 8u * (13 + 2 * KS + 2 * VS + s); };

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const bool masked = a.mask.bits != nullptr;
    if (threadIdx.x == 0) {
        mbar_init(qg_full, 1); mbar_init(qg_empty, 1); mbar_init(q_done, 1); mbar_init(answer, 1);
        for (int s = 0; s < KS; ++s) { mbar_init(k_full(s), 1); mbar_init(k_empty(s), 1); }
        for (int s = 0; s < VS; ++s) { mbar_init(v_full(s), 1); mbar_init(v_empty(s), 1); }
        for (int x = 0; x < 2; ++x) { mbar_init(s_full(x), 1); mbar_init(d_full(x), 8); mbar_init(s_free(x), 1); mbar_init(info_full(x), 1); mbar_init(info_empty(x), 10); }
        *abort_flag = 0;
        items.closed = -1;
        mbar_fence_init();
        prefetch_map(&map_q); prefetch_map(&map_k); prefetch_map(&map_v); prefetch_map(&map_g);
    }
    if (warp == 9) tmem_alloc(smem_addr(tmem_slot), 512);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    auto wait = [&](uint32_t bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, sp.wait_limit, abort_flag)); };
    // Gave up: a row of an item that will not be computed reads NaN
    auto void_row = [&](const DqItem &it, int qi) {
        if (qi >= a.Lq) return;
        const float nan = __int_as_float(0x7fffffff);
        if (sp.splits > 1)
            for (int d = 0; d < a.D; ++d) sp.part[((((int64_t)it.split * a.B + it.b) * a.Lq + qi) * a.H + it.h) * a.D + d] = nan;
        else
            fill_row<T>((T *)a.dq.ptr + it.b * a.dq.batch_stride + (int64_t)qi * a.dq.row_stride + (int64_t)it.h * a.D, a.D, nan);
    };

    if (warp == 8) {
        bool ok = true;
        int ks = 0, vs = 0; uint32_t kp = 0, vp = 0, qc = 0;
        auto load = [&](uint32_t bar, const CUtensorMap *map, unsigned char *dst, int head, int row, int b) {
#pragma unroll
            for (int p = 0; p < PLANES; ++p) tma_load_4d(smem_addr(dst + p * PLANE), map, p * 64, head, row, b, bar);
        };
        int item = blockIdx.x, k = 0, handed = 0;
        bool asked = false;
        for (; ok; ++k) {
            const int is = k & 1;
            if (!(ok = wait(info_empty(is), ((k >> 1) & 1) ^ 1))) break;
            if (item >= 0 && masked) {
                const DqItem it(a, sp.splits, item);
                const int cell = a.mask.rows > 1 ? it.q0 / kDenseTile : 0;
                for (int t = it.kt0 + lane; t < it.kt1; t += 32) items.flags[is][t - it.kt0] = a.mask.tiles[(it.plane * a.mask.tq + cell) * a.mask.tk + t];
            }
            if (lane == 0) items.item[is] = item;
            __syncwarp();
            if (lane == 0) mbar_arrive(info_full(is));
            ++handed;
            if (item < 0) break;
            // The next item is asked for when this one's last copies are due: an item taken over earlier would wait here while
            // other SMs run dry.
            auto ask = [&]() {
                if (!asked && lane == 0) {
                    mbar_expect_tx(answer, 16);
                    take_over(smem_addr(&items.answer), answer);
                }
                asked = true;
                __syncwarp();
            };
            const DqItem it(a, sp.splits, item);
            bool first = true;
            for (int t = it.kt0; t < it.kt1 && ok; ++t) {
                if (t + 2 >= it.kt1) ask();
                if (masked && items.flags[is][t - it.kt0] == 0) continue;
                if (!(ok = wait(k_empty(ks), kp ^ 1))) break;
                if (lane == 0) {
                    mbar_expect_tx(k_full(ks), TILE);
                    load(k_full(ks), &map_k, k_s + ks * TILE, it.hk, t * 128, it.b);
                }
                __syncwarp();
                if (++ks == KS) { ks = 0; kp ^= 1; }
                if (first) {
                    if (!(ok = wait(qg_empty, (qc & 1) ^ 1))) break;
                    ++qc;
                    if (lane == 0) {
                        mbar_expect_tx(qg_full, 2 * TILE + sp.extra_tx);
                        load(qg_full, &map_q, q_s, it.h, it.q0, it.b);
                        load(qg_full, &map_g, g_s, it.h, it.q0, it.b);
                    }
                    __syncwarp();
                    first = false;
                }
                if (!(ok = wait(v_empty(vs), vp ^ 1))) break;
                if (lane == 0) {
                    mbar_expect_tx(v_full(vs), TILE);
                    load(v_full(vs), &map_v, v_s + vs * TILE, it.hk, t * 128, it.b);
                }
                __syncwarp();
                if (++vs == VS) { vs = 0; vp ^= 1; }
            }
            if (!ok) break;
            ask();
            if (!(ok = wait(answer, k & 1))) break;
            item = taken_over(smem_addr(&items.answer));
            asked = false;
        }
        if (!ok) {
            close_items(items, handed, lane);
            const int lost = item_on_its_way(items, asked, answer, k, handed > k ? -1 : item);
            if (lost >= 0) {
                const DqItem it(a, sp.splits, lost);
                for (int row = lane; row < 128; row += 32) void_row(it, it.q0 + row);
            }
            // let copies already issued land before the block goes
            const long long start = clock64();
            while (clock64() - start < 200000) {}
        }
    } else if (warp == 9) {
        // S and dP: half tile j into buffer j & 1, once dq has taken half tile j - 2 from there
        bool ok = true;
        int ks = 0, vs = 0; uint32_t kp = 0, vp = 0, qc = 0, i = 0;
        const uint64_t q_desc = smem_desc(smem_addr(q_s), 16, 1024), g_desc = smem_desc(smem_addr(g_s), 16, 1024);
        const uint64_t k_desc = smem_desc(smem_addr(k_s), 16, 1024), v_desc = smem_desc(smem_addr(v_s), 16, 1024);
        for (int k = 0; ok; ++k) {
            const int is = k & 1;
            if (!(ok = wait(info_full(is), (k >> 1) & 1))) break;
            const int item = uniform(items.item[is]);
            if (item < 0) break;
            DqItem it(a, sp.splits, item);
            it.n = uniform(it.n); it.kt0 = uniform(it.kt0); it.kt1 = uniform(it.kt1);
            auto next_tile = [&](int t) {
                if (masked) { while (t < it.kt1 && items.flags[is][t - it.kt0] == 0) ++t; t = uniform(t); }
                return t;
            };
            int t = next_tile(it.kt0);
            if (t < it.kt1) { ok = wait(qg_full, qc & 1); ++qc; }
            while (ok && t < it.kt1) {
                if (!(ok = wait(k_full(ks), kp))) break;
                if (it.n - t * 128 < 128 || masked)
                    zero_hidden_rows<PLANES>(k_s + ks * TILE, it.n - t * 128, masked ? a.mask.seen + it.plane * a.mask.wk + t * 4 : nullptr, lane);
                if (!(ok = wait(v_full(vs), vp))) break;
                const int halves = it.n - t * 128 > 64 ? 2 : 1, tn = next_tile(t + 1);
                for (int half = 0; half < halves; ++half, ++i) {
                    if (!(ok = wait(s_free(i & 1), (i >> 1 & 1) ^ 1))) break;
                    fence_after_sync();
                    if (elect_one()) {
                        const uint32_t d = tmem + (i & 1) * 128;
                        const uint64_t kd = k_desc + (ks * (TILE >> 4) + half * (8192 >> 4)), vd = v_desc + (vs * (TILE >> 4) + half * (8192 >> 4));
#pragma unroll
                        for (int j = 0; j < DP / 16; ++j) {
                            const uint32_t off = (j >> 2) * (PLANE >> 4) + (j & 3) * 2;
                            mma_f16(d, q_desc + off, kd + off, IDESC_S, j > 0);
                        }
#pragma unroll
                        for (int j = 0; j < DP / 16; ++j) {
                            const uint32_t off = (j >> 2) * (PLANE >> 4) + (j & 3) * 2;
                            mma_f16(d + 64, g_desc + off, vd + off, IDESC_S, j > 0);
                        }
                        mma_commit(s_full(i & 1));
                        if (half + 1 == halves) {
                            mma_commit(v_empty(vs));
                            if (tn >= it.kt1) mma_commit(qg_empty);
                        }
                    }
                    __syncwarp();
                }
                if (++ks == KS) { ks = 0; kp ^= 1; }
                if (++vs == VS) { vs = 0; vp ^= 1; }
                t = tn;
            }
            if (ok && lane == 0) mbar_arrive(info_empty(is));
            __syncwarp();
        }
    } else if (warp == 10) {
        // dq += dS K
        bool ok = true;
        int ks = 0; uint32_t i = 0;
        const uint64_t k_desc = smem_desc(smem_addr(k_s), PLANE, 1024);
        for (int k = 0; ok; ++k) {
            const int is = k & 1;
            if (!(ok = wait(info_full(is), (k >> 1) & 1))) break;
            const int item = uniform(items.item[is]);
            if (item < 0) break;
            DqItem it(a, sp.splits, item);
            it.n = uniform(it.n); it.kt0 = uniform(it.kt0); it.kt1 = uniform(it.kt1);
            auto next_tile = [&](int t) {
                if (masked) { while (t < it.kt1 && items.flags[is][t - it.kt0] == 0) ++t; t = uniform(t); }
                return t;
            };
            bool fresh = true;
            int t = next_tile(it.kt0);
            while (ok && t < it.kt1) {
                const int halves = it.n - t * 128 > 64 ? 2 : 1, tn = next_tile(t + 1);
                for (int half = 0; half < halves; ++half, ++i) {
                    if (!(ok = wait(d_full(i & 1), i >> 1 & 1))) break;
                    fence_after_sync();
                    if (elect_one()) {
                        const uint64_t kd = k_desc + (ks * (TILE >> 4) + half * (8192 >> 4));
                        const uint32_t d = tmem + (i & 1) * 128;
#pragma unroll
                        for (int j = 0; j < 4; ++j)          // either warpgroup's 32 keys lie where its scores were
                            mma_f16_ta(tmem + COL_Q, d + (j >> 1) * 32 + (j & 1) * 8, kd + j * 128, IDESC_O, (!fresh || j > 0) ? 1u : 0u);
                        mma_commit(s_free(i & 1));
                        if (half + 1 == halves) {
                            mma_commit(k_empty(ks));
                            if (tn >= it.kt1) mma_commit(q_done);      // last: the block may end after it
                        }
                    }
                    __syncwarp();
                    fresh = false;
                }
                if (++ks == KS) ks = 0;
                t = tn;
            }
            if (ok && lane == 0) mbar_arrive(info_empty(is));
            __syncwarp();
        }
    } else {
        const int x = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;      // warpgroup x: keys [32 x, 32 x + 32) of a half tile
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        bool ok = true;
        uint32_t i = 0, qc = 0;                              // half tiles, and items that had any
        int k = 0, item = -1;
        for (; ok; ++k) {
            const int is = k & 1;
            item = -1;
            if (!(ok = wait(info_full(is), (k >> 1) & 1))) break;
            item = items.item[is];
            if (item < 0) break;
            const DqItem it(a, sp.splits, item);
            const int qi = it.q0 + row;
            const int64_t at = ((int64_t)it.b * a.H + it.h) * a.lq_pad + qi;
            float neg_lse2 = a.neg_lse2[at], neg_delta = a.neg_delta[at], unshift = 1.f;
            if constexpr (!BF) {
                const float e = grad_shift(a.dout_sq[at], a.top_sq[2 * (it.b * a.Hkv + it.hk) + 1]);
                neg_lse2 += e - (float)kWeightShift;
                unshift = pow2(-e);
            }
            const uint64_t c2 = pair(a.scale_log2, a.scale_log2), lse22 = pair(neg_lse2, neg_lse2), delta2 = pair(neg_delta, neg_delta);
            const uint32_t *bits = masked ? a.mask.bits + (it.plane * a.mask.rows + (a.mask.rows > 1 ? min(qi, a.Lq - 1) : 0)) * a.mask.wk : nullptr;
            bool any = false;
            for (int t = it.kt0; t < it.kt1 && ok; ++t) {
                const uint32_t flag = masked ? items.flags[is][t - it.kt0] : 2u;
                if (flag == 0) continue;
                const int left = it.n - t * 128;
                const bool partial = left < 128 || flag != 2;
                for (int half = 0; half < (left > 64 ? 2 : 1); ++half) {
                    uint32_t keep = 0xffffffffu;
                    if (partial) {
                        keep = tail_word(left, 2 * half + x);
                        if (masked) keep &= __ldg(bits + t * 4 + 2 * half + x);
                    }
                    if (!(ok = wait(s_full(i & 1), i >> 1 & 1))) break;
                    fence_after_sync();
                    const uint32_t ts = tmem + lanes + (i & 1) * 128 + 32 * x;
                    uint32_t r[32], g[32], d[16];
                    tmem_ld32(ts, r);
                    tmem_ld32(ts + 64, g);
                    tmem_ld_wait();
                    auto gradients = [&](auto whole) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float2 e = unpair(fma2(pair_bits(r[2 * j], r[2 * j + 1]), c2, lse22));
                            float2 y = unpair(mul2(pair(fast_exp2(e.x), fast_exp2(e.y)), add2(pair_bits(g[2 * j], g[2 * j + 1]), delta2)));
                            if (!decltype(whole)::value) {   // not through p = 0: what a hidden row holds may be NaN
                                if (!((keep >> (2 * j)) & 1u)) y.x = 0.f;
                                if (!((keep >> (2 * j + 1)) & 1u)) y.y = 0.f;
                            }
                            d[j] = pack2_finite<T>(y.x, y.y);
                        }
                    };
                    if (partial) gradients(std::false_type{}); else gradients(std::true_type{});
                    tmem_st16(ts, d);
                    tmem_st_wait();
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(d_full(i & 1));
                    ++i;
                    any = true;
                }
            }
            if (ok && any) { ok = wait(q_done, qc & 1); ++qc; }
            if (!ok) break;                                  // with k and item of the unfinished one
            fence_after_sync();
            T *out = (T *)a.dq.ptr + it.b * a.dq.batch_stride + (int64_t)qi * a.dq.row_stride + (int64_t)it.h * a.D;
#pragma unroll 1
            for (int c = x * (DP / 64); c < (x + 1) * (DP / 64); ++c) {        // 32 columns at a time
                uint32_t o[32];
                if (any) {
                    tmem_ld32(tmem + COL_Q + lanes + 32 * c, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = 0u;
                }
                if (sp.splits > 1) {
                    if constexpr (!BF) scale_all(o, unshift);
                    store_rows32_f32(sp.part + ((((int64_t)it.split * a.B + it.b) * a.Lq + qi) * a.H + it.h) * a.D, (int64_t)a.H * a.D, a.Lq - qi,
                                     32 * c, a.D, o);
                } else {
                    store_rows32<T>(out, a.dq.row_stride, a.Lq - qi, 32 * c, a.D, o, a.scale * unshift);
                }
            }
            fence_before_sync();                             // the accumulator may be written again
            __syncwarp();
            if (lane == 0) mbar_arrive(info_empty(is));
        }
        if (!ok) {                                           // gave up: this item, and any handed on already
            for (;; ++k) {
                if (item < 0) {
                    if (!handed_on(items, info_full(k & 1), k)) break;
                    item = items.item[k & 1];
                    if (item < 0) break;
                }
                const DqItem it(a, sp.splits, item);
                void_row(it, it.q0 + row);
                item = -1;
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (warp == 9) tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0 && *abort_flag) atomicAdd(&g_dense_bwd_aborts, 1u);
}

// --------------------------------------------------------------------------------------------------------------- dk, dv
template <int DP>
struct DkvShape {
    static constexpr int kTile = 128 * DP * 2, kHalf = 64 * DP * 2, kStages = 4;
    static constexpr int kStage = 2 * kHalf;                                      // a query tile and its output gradients
    static constexpr int kBars = 11 + 2 * kStages + kItemBars;
    static constexpr int kSmem = 1024 + 2 * kTile + kStages * (kStage + 512) + (int)sizeof(ItemSlots) + kBars * 8 + 8;
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

// A work item: 128 keys of a (batch entry, key/value head) against one range of the units (query head of the group, tile of 64
// queries), in this order
struct DkvItem {
    int kt, k0, hk, b, split, n, u0, u1;
    __device__ __forceinline__ DkvItem(const DenseArgs &a, int splits, int item, int qtiles) {
        const int ktiles = (a.Lk + 127) / 128;
        kt = item % ktiles; k0 = kt * 128; item /= ktiles;
        hk = item % a.Hkv; item /= a.Hkv;
        b = item % a.B; split = item / a.B;
        n = dense_keys(a, b);
        const int total = k0 < n ? a.group * qtiles : 0, per = (total + splits - 1) / splits;
        u0 = min(total, split * per);
        u1 = min(total, u0 + per);
    }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kBwdThreads, 1)
dense_dkdv_tc5_kernel(const DenseArgs a, const BwdSplit sp, const __grid_constant__ CUtensorMap map_q,
                      const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ CUtensorMap map_g) {
    using namespace tc5;
    using Shape = DkvShape<DP>;
    constexpr int TILE = Shape::kTile, HALF = Shape::kHalf, ST = Shape::kStages, PLANES = DP / 64, PLANE = 16384, HPLANE = 8192;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    constexpr uint32_t IDESC_S = instr_desc(128, 64, BF, false, false), IDESC_O = instr_desc(128, DP, BF, false, true);
    constexpr uint32_t COL_V = 256, COL_K = 256 + DP;

    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    unsigned char *k_s = smem, *v_s = k_s + TILE, *ring = v_s + TILE;
    float *stats = reinterpret_cast<float *>(ring + ST * Shape::kStage);          // per stage: 64 log-sum-exps, 64 row sums, both negated
    ItemSlots &items = *reinterpret_cast<ItemSlots *>(stats + ST * 128);
    unsigned long long *bars = reinterpret_cast<unsigned long long *>(&items + 1);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + Shape::kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const uint32_t bar0 = smem_addr(bars);
    const uint32_t kv_full = bar0, kv_empty = bar0 + 8, done = bar0 + 16, answer = bar0 + 24;
    auto s_full = [&](uint32_t x) { return bar0 + 8u * (5 + x); };
    auto d_full = [&](uint32_t x) { return bar0 + 8u * (7 + x); };
    auto s_free = [&](uint32_t x) { return bar0 + 8u * (9 + x); };
    auto full = [&](int s) { return bar0 + 8u * (11 + s); };
    auto empty = [&](int s) { return bar0 + 8u * (11 + ST + s); };
    auto info_full = [&](int s) { return bar0 + 8u * (11 + 2 * ST + s); };
    auto info_empty = [&](int s) { return bar0 + 8u * (13 + 2 * ST + s); };

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int qtiles = (a.Lq + 63) / 64;
    const bool masked = a.mask.bits != nullptr;
    const int cells = masked ? a.mask.tq : 0;

    if (threadIdx.x == 0) {
        mbar_init(kv_full, 1); mbar_init(kv_empty, 1); mbar_init(done, 1); mbar_init(answer, 1);
        for (int x = 0; x < 2; ++x) { mbar_init(s_full(x), 1); mbar_init(d_full(x), 8); mbar_init(s_free(x), 1); mbar_init(info_full(x), 1); mbar_init(info_empty(x), 10); }
        for (int s = 0; s < ST; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        *abort_flag = 0;
        items.closed = -1;
        mbar_fence_init();
        prefetch_map(&map_q); prefetch_map(&map_k); prefetch_map(&map_v); prefetch_map(&map_g);
    }
    if (warp == 9) tmem_alloc(smem_addr(tmem_slot), 512);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    auto wait = [&](uint32_t bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, sp.wait_limit, abort_flag)); };
    auto part_row = [&](const DkvItem &it, int x, int key) {
        return sp.part + (((((int64_t)(x == 0 ? sp.splits : 0) + it.split) * a.B + it.b) * a.Lk + key) * a.Hkv + it.hk) * a.D;
    };
    // Gave up: a row (x = 0: of dv, 1: of dk) of an item that will not be computed reads NaN
    auto void_row = [&](const DkvItem &it, int x, int key) {
        if (key >= a.Lk) return;
        const float nan = __int_as_float(0x7fffffff);
        const hsa_view &g = x == 0 ? a.dv : a.dk;
        if (sp.splits > 1)
            for (int d = 0; d < a.D; ++d) part_row(it, x, key)[d] = nan;
        else
            fill_row<T>((T *)g.ptr + it.b * g.batch_stride + (int64_t)key * g.row_stride + (int64_t)it.hk * a.D, a.D, nan);
    };
    auto plane_of = [&](int b, int h) { return (int64_t)b * a.mask.plane_b + (int64_t)h * a.mask.plane_h; };
    auto flag_of = [&](int is, int u) { return items.flags[is][u / qtiles * cells + (a.mask.rows > 1 ? (u % qtiles) >> 1 : 0)]; };
    auto next_unit = [&](int is, int u, int total) {
        if (masked) { while (u < total && flag_of(is, u) == 0) ++u; u = uniform(u); }
        return u;
    };

    if (warp == 8) {
        bool ok = true;
        int s = 0; uint32_t ph = 0, kc = 0;
        int item = blockIdx.x, k = 0, handed = 0;
        bool asked = false;
        for (; ok; ++k) {
            const int is = k & 1;
            if (!(ok = wait(info_empty(is), ((k >> 1) & 1) ^ 1))) break;
            if (item >= 0 && masked) {
                const DkvItem it(a, sp.splits, item, qtiles);
                if (it.u0 < it.u1)
                    for (int c = lane; c < a.group * cells; c += 32)
                        items.flags[is][c] = a.mask.tiles[(plane_of(it.b, it.hk * a.group + c / cells) * cells + c % cells) * a.mask.tk + it.kt];
            }
            if (lane == 0) items.item[is] = item;
            __syncwarp();
            if (lane == 0) mbar_arrive(info_full(is));
            ++handed;
            if (item < 0) break;
            // The next item is asked for when this one's last copies are due: an item taken over earlier would wait here while
            // other SMs run dry.
            auto ask = [&]() {
                if (!asked && lane == 0) {
                    mbar_expect_tx(answer, 16);
                    take_over(smem_addr(&items.answer), answer);
                }
                asked = true;
                __syncwarp();
            };
            const DkvItem it(a, sp.splits, item, qtiles);
            int u = next_unit(is, it.u0, it.u1);
            if (u < it.u1) {
                if (!(ok = wait(kv_empty, (kc & 1) ^ 1))) break;
                ++kc;
                if (lane == 0) {
                    mbar_expect_tx(kv_full, 2 * TILE + sp.extra_tx);
#pragma unroll
                    for (int p = 0; p < PLANES; ++p) {
                        tma_load_4d(smem_addr(k_s + p * PLANE), &map_k, p * 64, it.hk, it.k0, it.b, kv_full);
                        tma_load_4d(smem_addr(v_s + p * PLANE), &map_v, p * 64, it.hk, it.k0, it.b, kv_full);
                    }
                }
                __syncwarp();
            }
            for (; u < it.u1; u = next_unit(is, u + 1, it.u1)) {
                const int h = it.hk * a.group + u / qtiles, q0 = u % qtiles * 64;
                if (u + 4 >= it.u1) ask();
                if (!(ok = wait(empty(s), ph ^ 1))) break;
                if (lane == 0) {
                    mbar_expect_tx(full(s), 2 * HALF + 512);
                    const uint32_t qs = smem_addr(ring + s * Shape::kStage), gs = qs + HALF, fs = smem_addr(stats + s * 128);
                    const int64_t at = ((int64_t)it.b * a.H + h) * a.lq_pad + q0;
#pragma unroll
                    for (int p = 0; p < PLANES; ++p) tma_load_4d(qs + p * HPLANE, &map_q, p * 64, h, q0, it.b, full(s));
                    bulk_load(fs, a.neg_lse2 + at, 256, full(s));
#pragma unroll
                    for (int p = 0; p < PLANES; ++p) tma_load_4d(gs + p * HPLANE, &map_g, p * 64, h, q0, it.b, full(s));
                    bulk_load(fs + 256, a.neg_delta + at, 256, full(s));
                }
                __syncwarp();
                if (++s == ST) { s = 0; ph ^= 1; }
            }
            if (!ok) break;
            ask();
            if (!(ok = wait(answer, k & 1))) break;
            item = taken_over(smem_addr(&items.answer));
            asked = false;
        }
        if (!ok) {
            close_items(items, handed, lane);
            const int lost = item_on_its_way(items, asked, answer, k, handed > k ? -1 : item);
            if (lost >= 0) {
                const DkvItem it(a, sp.splits, lost, qtiles);
                for (int row = lane; row < 128; row += 32) {
                    void_row(it, 0, it.k0 + row);
                    void_row(it, 1, it.k0 + row);
                }
            }
            // let copies already issued land before the block goes
            const long long start = clock64();
            while (clock64() - start < 200000) {}
        }
    } else if (warp == 9) {
        // S^T and dP^T: tile j into buffer j & 1, once the gradients have taken tile j - 2 from there
        bool ok = true;
        int s = 0; uint32_t ph = 0, kc = 0, i = 0;
        const uint64_t k_desc = smem_desc(smem_addr(k_s), 16, 1024), v_desc = smem_desc(smem_addr(v_s), 16, 1024);
        const uint64_t ring_desc = smem_desc(smem_addr(ring), 16, 1024);
        for (int k = 0; ok; ++k) {
            const int is = k & 1;
            if (!(ok = wait(info_full(is), (k >> 1) & 1))) break;
            const int item = uniform(items.item[is]);
            if (item < 0) break;
            const DkvItem it(a, sp.splits, item, qtiles);
            const int u0 = uniform(it.u0), u1 = uniform(it.u1);
            int u = next_unit(is, u0, u1);
            if (u < u1) { ok = wait(kv_full, kc & 1); ++kc; }
            while (ok && u < u1) {
                const int un = next_unit(is, u + 1, u1);
                if (!(ok = wait(full(s), ph) && wait(s_free(i & 1), (i >> 1 & 1) ^ 1))) break;
                fence_after_sync();
                if (elect_one()) {
                    const uint32_t col = tmem + (i & 1) * 128;
                    const uint64_t qd = ring_desc + s * (Shape::kStage >> 4), gd = qd + (HALF >> 4);
#pragma unroll
                    for (int j = 0; j < DP / 16; ++j)
                        mma_f16(col, k_desc + (j >> 2) * (PLANE >> 4) + (j & 3) * 2, qd + (j >> 2) * (HPLANE >> 4) + (j & 3) * 2, IDESC_S, j > 0);
#pragma unroll
                    for (int j = 0; j < DP / 16; ++j)
                        mma_f16(col + 64, v_desc + (j >> 2) * (PLANE >> 4) + (j & 3) * 2, gd + (j >> 2) * (HPLANE >> 4) + (j & 3) * 2, IDESC_S, j > 0);
                    mma_commit(s_full(i & 1));
                    if (un >= u1) mma_commit(kv_empty);
                }
                __syncwarp();
                if (++s == ST) { s = 0; ph ^= 1; }
                ++i;
                u = un;
            }
            if (ok && lane == 0) mbar_arrive(info_empty(is));
            __syncwarp();
        }
    } else if (warp == 10) {
        // dv += P^T do, dk += dS^T q
        bool ok = true;
        int s = 0; uint32_t i = 0;
        const uint64_t ring_desc = smem_desc(smem_addr(ring), HPLANE, 1024);
        for (int k = 0; ok; ++k) {
            const int is = k & 1;
            if (!(ok = wait(info_full(is), (k >> 1) & 1))) break;
            const int item = uniform(items.item[is]);
            if (item < 0) break;
            const DkvItem it(a, sp.splits, item, qtiles);
            const int u0 = uniform(it.u0), u1 = uniform(it.u1);
            bool fresh = true;
            int u = next_unit(is, u0, u1);
            while (ok && u < u1) {
                const int un = next_unit(is, u + 1, u1);
                if (!(ok = wait(d_full(i & 1), i >> 1 & 1))) break;
                fence_after_sync();
                if (elect_one()) {
                    const uint32_t col = tmem + (i & 1) * 128;
                    const uint64_t qd = ring_desc + s * (Shape::kStage >> 4), gd = qd + (HALF >> 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j)              // either warpgroup's 32 queries lie where its scores were
                        mma_f16_ta(tmem + COL_V, col + (j >> 1) * 32 + (j & 1) * 8, gd + j * 128, IDESC_O, (!fresh || j > 0) ? 1u : 0u);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_f16_ta(tmem + COL_K, col + 64 + (j >> 1) * 32 + (j & 1) * 8, qd + j * 128, IDESC_O, (!fresh || j > 0) ? 1u : 0u);
                    mma_commit(s_free(i & 1));
                    mma_commit(empty(s));
                    if (un >= u1) mma_commit(done);       // last: the block may end after it
                }
                __syncwarp();
                if (++s == ST) s = 0;
                ++i;
                fresh = false;
                u = un;
            }
            if (ok && lane == 0) mbar_arrive(info_empty(is));
            __syncwarp();
        }
    } else {
        const int x = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;      // warpgroup x: queries [32 x, 32 x + 32) of a tile
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint64_t c2 = pair(a.scale_log2, a.scale_log2);
        bool ok = true;
        uint32_t i = 0, kc = 0;                              // tiles, and items that had any
        int s = 0, k = 0, item = -1; uint32_t ph = 0;
        for (; ok; ++k) {
            const int is = k & 1;
            item = -1;
            if (!(ok = wait(info_full(is), (k >> 1) & 1))) break;
            item = items.item[is];
            if (item < 0) break;
            const DkvItem it(a, sp.splits, item, qtiles);
            const int key = it.k0 + row;
            const bool tail = it.n - it.k0 < 128;
            bool any = false;
            float ds_shift = 0.f;
            if constexpr (!BF) {
                const unsigned int *tops = a.top_sq + 2 * (it.b * a.Hkv + it.hk);
                ds_shift = grad_shift(__uint_as_float(tops[0]), tops[1]);
            }
            const float ds_factor = pow2(ds_shift - (float)kWeightShift), unshift = BF ? 1.f : pow2(x == 0 ? -(float)kWeightShift : -ds_shift);
            const uint64_t ds_factor2 = pair(ds_factor, ds_factor);
            for (int u = next_unit(is, it.u0, it.u1); u < it.u1; u = next_unit(is, u + 1, it.u1)) {
                uint32_t keep = 0xffffffffu;
                bool partial = tail;
                if (masked && flag_of(is, u) != 2) {
                    partial = true;
                    const int64_t plane = plane_of(it.b, it.hk * a.group + u / qtiles);
                    if (key < a.Lk) {
                        if (a.mask.rows > 1) keep = __ldg(a.mask.bits_t + (plane * a.Lk + key) * a.mask.wq + u % qtiles * 2 + x);
                        else if (!((__ldg(a.mask.bits + plane * a.mask.wk + (key >> 5)) >> (key & 31)) & 1u)) keep = 0u;
                    }
                }
                if (key >= it.n) keep = 0u;
                if (!(ok = wait(full(s), ph) && wait(s_full(i & 1), i >> 1 & 1))) break;
                fence_after_sync();
                const float *st = stats + s * 128 + 32 * x;
                const uint32_t ts = tmem + lanes + (i & 1) * 128 + 32 * x;
                uint32_t r[32], g[32], pk[16], dk[16];
                tmem_ld32(ts, r);
                tmem_ld32(ts + 64, g);
                tmem_ld_wait();
                auto gradients = [&](auto whole) {
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const float4 lse = *reinterpret_cast<const float4 *>(st + 2 * j), dl = *reinterpret_cast<const float4 *>(st + 64 + 2 * j);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int c = j + e;
                            const float2 z = unpair(fma2(pair_bits(r[2 * c], r[2 * c + 1]), c2, e == 0 ? pair(lse.x, lse.y) : pair(lse.z, lse.w)));
                            float2 p = make_float2(fast_exp2(z.x), fast_exp2(z.y));
                            float2 y = unpair(mul2(pair(p.x, p.y), add2(pair_bits(g[2 * c], g[2 * c + 1]), e == 0 ? pair(dl.x, dl.y) : pair(dl.z, dl.w))));
                            if (!decltype(whole)::value) {       // not through p = 0: what a hidden row holds may be NaN
                                if (!((keep >> (2 * c)) & 1u)) p.x = y.x = 0.f;
                                if (!((keep >> (2 * c + 1)) & 1u)) p.y = y.y = 0.f;
                            }
                            if constexpr (!BF) y = unpair(mul2(pair(y.x, y.y), ds_factor2));
                            pk[c] = pack2_finite<T>(p.x, p.y);
                            dk[c] = pack2_finite<T>(y.x, y.y);
                        }
                    }
                };
                if (partial) gradients(std::false_type{}); else gradients(std::true_type{});
                tmem_st16(ts, pk);
                tmem_st16(ts + 64, dk);
                tmem_st_wait();
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(d_full(i & 1));
                if (++s == ST) { s = 0; ph ^= 1; }
                ++i;
                any = true;
            }
            if (ok && any) { ok = wait(done, kc & 1); ++kc; }
            if (!ok) break;                                      // with k and item of the unfinished one
            fence_after_sync();
            // dv by the first warpgroup, dk by the second
            const hsa_view &g = x == 0 ? a.dv : a.dk;
            T *out = (T *)g.ptr + it.b * g.batch_stride + (int64_t)key * g.row_stride + (int64_t)it.hk * a.D;
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
                uint32_t o[32];
                if (any) {
                    tmem_ld32(tmem + lanes + (x == 0 ? COL_V : COL_K) + 32 * c, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = 0u;
                }
                if (sp.splits > 1) {
                    if constexpr (!BF) scale_all(o, unshift);
                    store_rows32_f32(part_row(it, x, key), (int64_t)a.Hkv * a.D, a.Lk - key, 32 * c, a.D, o);
                } else {
                    store_rows32<T>(out, g.row_stride, a.Lk - key, 32 * c, a.D, o, (x == 0 ? 1.f : a.scale) * unshift);
                }
            }
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(info_empty(is));
        }
        if (!ok) {                                           // gave up: this item, and any handed on already
            for (;; ++k) {
                if (item < 0) {
                    if (!handed_on(items, info_full(k & 1), k)) break;
                    item = items.item[k & 1];
                    if (item < 0) break;
                }
                const DkvItem it(a, sp.splits, item, qtiles);
                void_row(it, x, it.k0 + row);
                item = -1;
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (warp == 9) tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0 && *abort_flag) atomicAdd(&g_dense_bwd_aborts, 1u);
}

// Few queries over many keys cut the keys of a dq item; few keys under many queries cut the queries of a dk/dv item.  A dq item costs
// about three key tiles' time besides its own (seven as a partial one), a dk/dv item about six query tiles' (twelve).
static int dq_splits(int B, int Lq, int Lk, int H) { return range_count((long long)B * H * ((Lq + 127) / 128), (Lk + 127) / 128, 3.0, 7.0); }
static int dkdv_splits(int B, int Lq, int Lk, int H, int Hkv) {
    const long long units = (long long)(H / Hkv) * ((Lq + 63) / 64);
    return units > (1 << 30) ? 1 : range_count((long long)B * Hkv * ((Lk + 127) / 128), (int)units, 6.0, 12.0);
}

size_t dense_bwd_tc_workspace(int B, int Lq, int Lk, int H, int Hkv, int D) {
    return bwd_part_bytes(dq_splits(B, Lq, Lk, H), dkdv_splits(B, Lq, Lk, H, Hkv), B, Lq, Lk, H, Hkv, D);
}

template <typename T, int DP>
static int bwd_launch(const DenseArgs &a, void *workspace, cudaStream_t st) {
    CUtensorMap mq, mq64, mk, mv, mg, mg64;
    if (!make_map(&mq, a.q, a.B, a.Lq, a.H, a.D, 1, 128) || !make_map(&mq64, a.q, a.B, a.Lq, a.H, a.D, 1, 64) ||
        !make_map(&mk, a.k, a.B, a.Lk, a.Hkv, a.D, 1, 128) || !make_map(&mv, a.v, a.B, a.Lk, a.Hkv, a.D, 1, 128) ||
        !make_map(&mg, a.dout, a.B, a.Lq, a.H, a.D, 1, 128) || !make_map(&mg64, a.dout, a.B, a.Lq, a.H, a.D, 1, 64))
        return fail(HSA_ERR_ARG, "hsa_dense_attn_bwd: the driver refused a tensor map");
    BwdSplit sq, sk;
    bwd_splits(dq_splits(a.B, a.Lq, a.Lk, a.H), dkdv_splits(a.B, a.Lq, a.Lk, a.H, a.Hkv), a, workspace, sq, sk);
    const long long dq_blocks = (long long)a.B * a.H * ((a.Lq + 127) / 128) * sq.splits;
    const long long kv_blocks = (long long)a.B * a.Hkv * ((a.Lk + 127) / 128) * sk.splits;
    if (dq_blocks > 0x7fffffffLL || kv_blocks > 0x7fffffffLL) return fail(HSA_ERR_ARG, "hsa_dense_attn_bwd: too many tiles");
    constexpr auto kdq = dense_dq_tc5_kernel<T, DP>;
    constexpr auto kkv = dense_dkdv_tc5_kernel<T, DP>;
    constexpr int smem_dq = DqShape<DP>::kSmem, smem_kv = DkvShape<DP>::kSmem;
    cudaError_t e = allow_smem<kdq>(smem_dq);
    if (e == cudaSuccess) e = allow_smem<kkv>(smem_kv);
    if (e != cudaSuccess) return fail((int)e, "hsa_dense_attn_bwd: shared memory %d / %d: %s", smem_dq, smem_kv, cudaGetErrorString(e));
    if (a.dk.ptr != nullptr) {
        kkv<<<(unsigned)kv_blocks, kBwdThreads, smem_kv, st>>>(a, sk, mq64, mk, mv, mg64);
        if (int rc = launch_status("hsa_dense_attn_bwd(dk, dv)")) return rc;
    }
    if (a.dq.ptr != nullptr) {
        kdq<<<(unsigned)dq_blocks, kBwdThreads, smem_dq, st>>>(a, sq, mq, mk, mv, mg);
        if (int rc = launch_status("hsa_dense_attn_bwd(dq)")) return rc;
    }
    return join_backward<T>(a, sq, sk, st);
}

// Whether the mask's tile states fit a block's table on both sides.
bool dense_bwd_tables_ok(const DenseArgs &a) {
    return a.mask.bits == nullptr || (a.mask.tk <= kFlagTiles && (long long)a.group * a.mask.tq <= kFlagTiles);
}

int dense_bwd_tc(const DenseArgs &a, void *workspace, int dtype, cudaStream_t st) {
    if (dtype == HSA_BF16) return a.D <= 64 ? bwd_launch<__nv_bfloat16, 64>(a, workspace, st) : bwd_launch<__nv_bfloat16, 128>(a, workspace, st);
    return a.D <= 64 ? bwd_launch<__half, 64>(a, workspace, st) : bwd_launch<__half, 128>(a, workspace, st);
}

cudaError_t dense_bwd_aborts(unsigned int *count) { return cudaMemcpyFromSymbol(count, g_dense_bwd_aborts, sizeof(unsigned int)); }

}  // namespace hsa
