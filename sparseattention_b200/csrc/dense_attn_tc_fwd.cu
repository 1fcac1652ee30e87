// Dense attention forward on the 5th-generation tensor cores (bf16 / f16, head dims up to 128).
//
//   out_i = sum_j exp2(c s_ij - m_i) v_j / sum_j exp2(c s_ij - m_i),   s_ij = q_i.k_j,  c = scale log2(e)
//
// One pass over the keys with a running maximum and sum.  A work item is 256 query rows of one (batch entry, head), two tiles of
// 128, against tiles of 128 keys in halves of 64; 11 warps with fixed roles:
//   warp 8     copies K and V tiles into a ring (TMA boxes of [128 rows][128 bytes], 128-byte swizzle)
//   warps 9, 10  issue S = Q K^T (both operands in shared memory) and O += P V (P in tensor memory, V as an MN-major operand),
//              each for one query tile
//   warps 0-3  and 4-7: the softmax of the first and of the second query tile, a thread per row
// Tensor memory (512 columns): two half tiles of S for either query tile (64 columns each), O of both (DP each).  P replaces the
// S it came from as 16-bit numbers, so it never passes through shared memory, and the other half tile's scores are computed
// meanwhile.
// Measured at 4096 x 4096, batch 4, 16 heads of 128, bf16: 459 to 464 us = 1.19 PFLOP/s, tensor pipe 65 % busy; what is left is the
// softmax, two warps per scheduler that overlap each other only in part (459 with the treatment of NaN and large scores).  On the way there: scores in one piece of 128 columns,
// which wait for the product that consumes P, 594 us; half tiles with products issued from per-lane registers slower still, from
// uniform ones and by a warp per query tile 524 us; a quarter of the exponentials in multiply-adds 514 us; registers enough to
// keep the softmax out of local memory (most of L1 is shared memory here, a spill goes to L2) 464 us.
// Tried and slower: fetching the next scores before this half tile's weights are handed over (497), taking turns with the
// exponentials (554), four softmax warps per 32 rows of which pairs exchange maxima (registers).
// The output is rescaled only when a row's maximum has grown by more than 2^8 since the last time (the weights then lie below
// 2^8, which changes nothing in their relative precision), so almost every tile leaves O alone.
// Rounding: weights are rounded to the inputs' type for the second product (what the tensor cores take); their sum is taken
// from the unrounded 32-bit values, and the division by it comes last, in 32 bits.  In float16 all weights of a row are 2^7 times as
// large: the largest then still fits (2^15), and what a weight loses below the type's smallest step is 2^-32 of the row's largest
// instead of 2^-25, which many small weights next to a large one would show (100000 keys 17.6 below one: all of their part).
// Keys behind a sequence's length and keys that no query may look at: the scores are replaced, and their V rows are zeroed in
// shared memory, so that NaN there cannot come back as 0 * NaN.
#include "dense_attn_tc.cuh"

namespace hsa {

__device__ unsigned int g_dense_aborts = 0;

// Softmax of two query tiles, copies, a warp of products for either tile, and an idle warp that completes the last warpgroup:
// its registers go to the softmax (2 x 128 x 200 + 128 x 104 = 384 x 168, what the block is launched with).
constexpr int kFwdThreads = 384;
constexpr float kLargeScore = 1048576.f;         // in base 2

template <int DP>
struct FwdShape {
    static constexpr int kTile = 128 * DP * 2;                       // bytes of a tile of 128 rows
    static constexpr int kSlots = DP == 128 ? 5 : 8;                 // K and V tiles in flight
    static constexpr int kSmem = 1024 + 2 * kTile + kSlots * kTile + (int)sizeof(ItemSlots) + (16 + 2 * kSlots + kItemBars) * 8 + 8;
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

// A work item: 256 query rows of a (batch entry, head) against one range of its keys
struct FwdItem {
    int q0, h, b, split, hk, nw, n, kt0, kt1;
    int64_t plane;
    __device__ __forceinline__ FwdItem(const DenseArgs &a, int splits, int item) {
        const int qblocks = (a.Lq + 255) / 256;
        q0 = item % qblocks * 256; item /= qblocks;
        h = item % a.H; item /= a.H;
        b = item % a.B; split = item / a.B;
        hk = h / a.group;
        nw = a.Lq - q0 > 128 ? 2 : 1;                    // query tiles
        n = dense_keys(a, b);
        const int tiles = (n + 127) / 128, per = (tiles + splits - 1) / splits;
        kt0 = min(tiles, split * per);
        kt1 = min(tiles, kt0 + per);
        plane = (int64_t)b * a.mask.plane_b + (int64_t)h * a.mask.plane_h;
    }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kFwdThreads, 1)
dense_fwd_tc5_kernel(const DenseArgs a, const DenseSplit sp, const __grid_constant__ CUtensorMap map_q,
                     const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using namespace tc5;
    using Shape = FwdShape<DP>;
    constexpr int TILE = Shape::kTile, SLOTS = Shape::kSlots, PLANES = DP / 64, PLANE = 128 * 128;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    constexpr uint32_t IDESC_S = instr_desc(128, 64, BF, false, false), IDESC_O = instr_desc(128, DP, BF, false, true);
    constexpr uint32_t COL_S = 0, COL_O = 256;
    constexpr float SHIFT = BF ? 0.f : 7.f;                          // weights are taken times 2^SHIFT

    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    unsigned char *q_s = smem, *ring = smem + 2 * TILE;
    ItemSlots &items = *reinterpret_cast<ItemSlots *>(ring + (size_t)SLOTS * TILE);
    unsigned long long *bars = reinterpret_cast<unsigned long long *>(&items + 1);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 16 + 2 * SLOTS + kItemBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const uint32_t bar0 = smem_addr(bars);
    auto q_full = [&](int w) { return bar0 + 8u * w; };
    auto q_empty = [&](int w) { return bar0 + 8u * (2 + w); };
    auto o_full = [&](int w) { return bar0 + 8u * (4 + w); };
    auto s_full = [&](int w, uint32_t x) { return bar0 + 8u * (6 + 2 * w + x); };
    auto p_full = [&](int w, uint32_t x) { return bar0 + 8u * (10 + 2 * w + x); };
    auto o_done = [&](int w) { return bar0 + 8u * (14 + w); };
    auto kv_full = [&](int s) { return bar0 + 8u * (16 + s); };
    auto kv_empty = [&](int s) { return bar0 + 8u * (16 + SLOTS + s); };
    auto info_full = [&](int s) { return bar0 + 8u * (16 + 2 * SLOTS + s); };
    auto info_empty = [&](int s) { return bar0 + 8u * (18 + 2 * SLOTS + s); };
    const uint32_t answer = bar0 + 8u * (20 + 2 * SLOTS);

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const bool masked = a.mask.bits != nullptr;
    if (threadIdx.x == 0) {
        for (int w = 0; w < 2; ++w) {
            mbar_init(q_full(w), 1); mbar_init(q_empty(w), 1); mbar_init(o_full(w), 1); mbar_init(o_done(w), 1);
            for (int x = 0; x < 2; ++x) { mbar_init(s_full(w, x), 1); mbar_init(p_full(w, x), 4); }
            mbar_init(info_full(w), 1); mbar_init(info_empty(w), 10);
        }
        for (int s = 0; s < SLOTS; ++s) { mbar_init(kv_full(s), 1); mbar_init(kv_empty(s), 2); }
        mbar_init(answer, 1);
        *abort_flag = 0;
        items.closed = -1;
        mbar_fence_init();
        prefetch_map(&map_q); prefetch_map(&map_k); prefetch_map(&map_v);
    }
    if (warp == 9) tmem_alloc(smem_addr(tmem_slot), 512);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    // a whole warp waits, and goes on or gives up as one
    auto wait = [&](uint32_t bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, sp.wait_limit, abort_flag)); };
    // Gave up: a row of an item that will not be computed reads NaN
    auto void_row = [&](const FwdItem &it, int qi) {
        if (qi >= a.Lq) return;
        const float nan = __int_as_float(0x7fffffff);
        const int64_t at = (((int64_t)it.split * a.B + it.b) * a.Lq + qi) * a.H + it.h;
        if (sp.splits > 1) { *reinterpret_cast<float2 *>(sp.part_ml + 2 * at) = make_float2(0.f, nan); return; }
        fill_row<T>((T *)a.out.ptr + it.b * a.out.batch_stride + (int64_t)qi * a.out.row_stride + (int64_t)it.h * a.D, a.D, nan);
        if (a.out_lo != nullptr) fill_row<T>((T *)a.out_lo + at * a.D, a.D, nan);
        if (a.lse != nullptr) a.lse[at] = nan;
    };

    if (warp == 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;\n");
        // ------------------------------------------------------------------------------------------------- copies
        bool ok = true;
        int slot = 0; uint32_t ph = 0, qc[2] = {0, 0};
        auto push = [&](const CUtensorMap *map, int hk, int row, int b) {
            if (!(ok = wait(kv_empty(slot), ph ^ 1))) return;
            if (lane == 0) {
                mbar_expect_tx(kv_full(slot), TILE);
                const uint32_t dst = smem_addr(ring + (size_t)slot * TILE);
#pragma unroll
                for (int p = 0; p < PLANES; ++p) tma_load_4d(dst + p * PLANE, map, p * 64, hk, row, b, kv_full(slot));
            }
            __syncwarp();
            if (++slot == SLOTS) { slot = 0; ph ^= 1; }
        };
        int item = blockIdx.x, k = 0, handed = 0;
        bool asked = false;
        for (; ok; ++k) {
            const int is = k & 1;
            if (!(ok = wait(info_empty(is), ((k >> 1) & 1) ^ 1))) break;
            if (item >= 0 && masked) {
                // mask states of the item's key tiles: two bits per query tile
                const FwdItem it(a, sp.splits, item);
                for (int t = it.kt0 + lane; t < it.kt1; t += 32) {
                    uint8_t f = 0;
                    for (int w = 0; w < it.nw; ++w) {
                        const int row = a.mask.rows > 1 ? it.q0 / kDenseTile + w : 0;
                        f |= a.mask.tiles[(it.plane * a.mask.tq + row) * a.mask.tk + t] << (2 * w);
                    }
                    items.flags[is][t - it.kt0] = f;
                }
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
            const FwdItem it(a, sp.splits, item);
            bool first = true;
            for (int t = it.kt0; t < it.kt1 && ok; ++t) {
                if (t + 2 >= it.kt1) ask();
                if (masked && items.flags[is][t - it.kt0] == 0) continue;
                push(&map_k, it.hk, t * 128, it.b);
                if (first) {
                    for (int w = 0; w < it.nw && ok; ++w) {
                        if (!(ok = wait(q_empty(w), (qc[w] & 1) ^ 1))) break;
                        ++qc[w];
                        if (lane == 0) {
                            mbar_expect_tx(q_full(w), TILE + sp.extra_tx);
#pragma unroll
                            for (int p = 0; p < PLANES; ++p)
                                tma_load_4d(smem_addr(q_s + w * TILE + p * PLANE), &map_q, p * 64, it.h, it.q0 + 128 * w, it.b, q_full(w));
                        }
                        __syncwarp();
                    }
                    first = false;
                }
                if (ok) push(&map_v, it.hk, t * 128, it.b);
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
                const FwdItem it(a, sp.splits, lost);
                for (int row = lane; row < 128 * it.nw; row += 32) void_row(it, it.q0 + row);
            }
            // let copies already issued land before the block goes
            const long long start = clock64();
            while (clock64() - start < 200000) {}
        }
    } else if (warp == 9 || warp == 10) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;\n");
        // -------------------------------------------------------------------------------------------- matrix products
        // Half tiles of 64 keys: S of half tile j + 2 follows the product that has consumed the weights of half tile j, whose
        // columns it takes, so that the softmax always finds the next scores ready.  One warp for either query tile: with one
        // for both, issuing took as long as the products.
        const int w = warp - 9;
        bool ok = true;
        uint32_t qc = 0, sn = 0, pn = 0;                               // items, half tiles scored, half tiles summed
        uint32_t ks_tile = 0, pv_tile = 0;                             // tiles so far on either side; tile m: ring places 2 m (K), 2 m + 1 (V)
        const uint64_t q_desc = smem_desc(smem_addr(q_s + w * TILE), 16, 1024);
        // a descriptor's start address counts in 16 bytes, and no sum of these leaves its field
        const uint64_t k_desc = smem_desc(smem_addr(ring), 16, 1024), v_desc = smem_desc(smem_addr(ring), PLANE, 1024);
        const uint32_t s_col = tmem + COL_S + w * 128, o_col = tmem + COL_O + w * DP;
        for (int k = 0; ok; ++k) {
            const int is = k & 1;
            if (!(ok = wait(info_full(is), (k >> 1) & 1))) break;
            const int item = uniform(items.item[is]);
            if (item < 0) break;
            FwdItem it(a, sp.splits, item);
            it.n = uniform(it.n); it.kt0 = uniform(it.kt0); it.kt1 = uniform(it.kt1);
            auto next_tile = [&](int t) {
                if (masked) { while (t < it.kt1 && items.flags[is][t - it.kt0] == 0) ++t; t = uniform(t); }
                return t;
            };
            auto halves = [&](int t) { return it.n - t * 128 > 64 ? 2 : 1; };
            int ts = next_tile(it.kt0), hs = 0, tp = ts, hp = 0;        // next half tile to score, next to sum
            if (w >= it.nw) {                                           // no such query tile: let the key tiles go
                for (; tp < it.kt1 && ok; tp = next_tile(tp + 1), ++ks_tile, ++pv_tile)
                    for (uint32_t place = 2 * pv_tile; place < 2 * pv_tile + 2 && ok; ++place) {
                        ok = wait(kv_full(place % SLOTS), place / SLOTS & 1);
                        if (ok && lane == 0) mbar_arrive(kv_empty(place % SLOTS));
                        __syncwarp();
                    }
                if (ok && lane == 0) mbar_arrive(info_empty(is));
                __syncwarp();
                continue;
            }
            auto score = [&]() -> bool {                                // S of (ts, hs)
                const uint32_t place = 2 * ks_tile, slot = place % SLOTS;
                if (hs == 0 && !wait(kv_full(slot), place / SLOTS & 1)) return false;
                fence_after_sync();
                const bool half_last = hs + 1 == halves(ts);
                const int tn = half_last ? next_tile(ts + 1) : ts;
                if (elect_one()) {
                    const uint64_t kd = k_desc + (slot * (TILE >> 4) + hs * (8192 >> 4));
                    const uint32_t d = s_col + (sn & 1) * 64;
#pragma unroll
                    for (int j = 0; j < DP / 16; ++j) {
                        const uint32_t off = (j >> 2) * (PLANE >> 4) + (j & 3) * 2;
                        mma_f16(d, q_desc + off, kd + off, IDESC_S, j > 0);
                    }
                    mma_commit(s_full(w, sn & 1));
                    if (half_last) mma_commit(kv_empty(slot));
                    if (tn >= it.kt1) mma_commit(q_empty(w));
                }
                __syncwarp();
                ++sn;
                if (half_last) ++ks_tile;
                hs = half_last ? 0 : 1;
                ts = tn;
                return true;
            };
            if (ts < it.kt1) {
                ok = wait(q_full(w), qc & 1) && score();
                ++qc;
                if (ok && ts < it.kt1) ok = score();
            }
            bool fresh = true;
            while (ok && tp < it.kt1) {
                const uint32_t place = 2 * pv_tile + 1, slot = place % SLOTS;
                if (hp == 0) {
                    if (!(ok = wait(kv_full(slot), place / SLOTS & 1))) break;
                    if (it.n - tp * 128 < 128 || masked)             // (both warps write the same zeros)
                        zero_hidden_rows<PLANES>(ring + slot * TILE, it.n - tp * 128,
                                                 masked ? a.mask.seen + it.plane * a.mask.wk + tp * 4 : nullptr, lane);
                }
                const bool half_last = hp + 1 == halves(tp);
                const int tn = half_last ? next_tile(tp + 1) : tp;
                if (!(ok = wait(p_full(w, pn & 1), pn >> 1 & 1))) break;
                fence_after_sync();
                if (elect_one()) {
                    const uint64_t vd = v_desc + (slot * (TILE >> 4) + hp * (8192 >> 4));
                    const uint32_t p = s_col + (pn & 1) * 64;
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma_f16_ta(o_col, p + j * 8, vd + j * 128, IDESC_O, (!fresh || j > 0) ? 1u : 0u);
                    mma_commit(o_full(w));
                    if (half_last) mma_commit(kv_empty(slot));
                    if (tn >= it.kt1) mma_commit(o_done(w));         // last: the block may end after it
                }
                __syncwarp();
                ++pn;
                if (ts < it.kt1) ok = score();
                fresh = false;
                if (half_last) ++pv_tile;
                hp = half_last ? 0 : 1;
                tp = tn;
            }
            if (ok && lane == 0) mbar_arrive(info_empty(is));
            __syncwarp();
        }
    } else if (warp == 11) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;\n");
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;\n");
        // -------------------------------------------------------------------------------------------------- softmax
        const int w = warp >> 2, quarter = warp & 3;
        const int row = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t ts = tmem + COL_S + w * 128 + lanes, to = tmem + COL_O + w * DP + lanes;
        bool ok = true;
        uint32_t sc = 0, oc = 0;                             // half tiles, and items with any, done so far
        int k = 0, item = -1;
        for (; ok; ++k) {
            const int is = k & 1;
            item = -1;
            if (!(ok = wait(info_full(is), (k >> 1) & 1))) break;
            item = items.item[is];
            if (item < 0) break;
            const FwdItem it(a, sp.splits, item);
            const int qi = it.q0 + 128 * w + row;
            if (w < it.nw) {
                const uint32_t *bits = masked ? a.mask.bits + (it.plane * a.mask.rows + (a.mask.rows > 1 ? min(qi, a.Lq - 1) : 0)) * a.mask.wk : nullptr;
                float m = -INFINITY, l = 0.f;
                bool any = false;
                for (int t = it.kt0; t < it.kt1 && ok; ++t) {
                    uint32_t flag = 2;
                    if (masked) {
                        flag = items.flags[is][t - it.kt0];
                        if (flag == 0) continue;
                        flag = (flag >> (2 * w)) & 3;
                    }
                    const int left = it.n - t * 128;
                    const bool partial = left < 128 || flag != 2;
                    uint32_t words[4] = {~0u, ~0u, ~0u, ~0u};
                    if (partial) {
                        if (masked) {
                            const uint4 m4 = __ldg(reinterpret_cast<const uint4 *>(bits + t * 4));
                            words[0] = m4.x; words[1] = m4.y; words[2] = m4.z; words[3] = m4.w;
                        }
#pragma unroll
                        for (int c = 0; c < 4; ++c) words[c] &= tail_word(left, c);
                    }
                    for (int half = 0; half < (left > 64 ? 2 : 1); ++half) {
                        const uint32_t x = sc & 1, tsx = ts + x * 64;
                        if (!(ok = wait(s_full(w, x), sc >> 1 & 1))) break;
                        fence_after_sync();
                        uint32_t r[2][32];
                        tmem_ld32(tsx, r[0]);
                        tmem_ld32(tsx + 32, r[1]);
                        tmem_ld_wait();
                        if (partial) {
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const uint32_t keep = half == 0 ? words[c] : words[2 + c];
#pragma unroll
                                for (int j = 0; j < 32; ++j)
                                    if (!((keep >> j) & 1u)) r[c][j] = 0xff800000u;
                            }
                        }
                        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int j = 0; j < 64; j += 2)
                            tops[j >> 1 & 3] = max3_nan(tops[j >> 1 & 3], __uint_as_float(r[j >> 5][j & 31]), __uint_as_float(r[j >> 5][(j + 1) & 31]));
                        const float top = max3_nan(max3_nan(tops[0], tops[1], tops[2]), tops[3], tops[3]);
                        float ref = m * a.scale_log2;
                        const bool grow = top * a.scale_log2 > ref + 8.f;       // also the first finite maximum (m = -inf)
                        if (__any_sync(0xffffffffu, grow || (fabsf(ref) > kLargeScore && m != -INFINITY))) {
                            const float m_new = grow ? top : m;
                            const float corr = grow ? fast_exp2((m - m_new) * a.scale_log2) : 1.f;
                            if (any) {
                                if (!(ok = wait(o_full(w), (sc - 1) & 1))) break;      // these scores follow the product before that one
                                fence_after_sync();
#pragma unroll
                                for (int c = 0; c < DP / 32; ++c) {
                                    uint32_t o[32];
                                    tmem_ld32(to + 32 * c, o);
                                    tmem_ld_wait();
#pragma unroll
                                    for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
                                    tmem_st32(to + 32 * c, o);
                                }
                                l *= corr;
                            }
                            m = m_new;
                            ref = m * a.scale_log2;
                            // c s - c m, one rounding of c m apart, is off by that rounding: a common factor of the row's weights, but
                            // beyond 2^24 one that leaves their range.  Such rows take the difference first.
                            const bool large = fabsf(ref) > kLargeScore && m != -INFINITY;
                            if (__any_sync(0xffffffffu, large)) {
                                const float base = large ? m : 0.f;
#pragma unroll
                                for (int j = 0; j < 64; ++j) r[j >> 5][j & 31] = __float_as_uint(__uint_as_float(r[j >> 5][j & 31]) - base);
                                if (large) ref = 0.f;
                            }
                        }
                        // a NaN score, or one of plus infinity, makes NaN of all weights of its row here, and so of its sum and result
                        ref = !(top < INFINITY) ? NAN : ref == -INFINITY ? 0.f : ref - SHIFT;
                        const uint64_t c2 = pair(a.scale_log2, a.scale_log2), ref2 = pair(-ref, -ref);
                        uint64_t sum[2] = {0, 0};                    // two pairs of zeros
                        uint32_t pk[32];
                        auto weights = [&](auto mixed) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                const float2 e = unpair(fma2(pair_bits(r[j >> 4][(2 * j) & 31], r[j >> 4][(2 * j + 1) & 31]), c2, ref2));
                                float2 p;
                                if (decltype(mixed)::value && j % 3 == 0) p = exp2_poly(e);
                                else p = make_float2(fast_exp2(e.x), fast_exp2(e.y));
                                sum[j & 1] = add2(sum[j & 1], pair(p.x, p.y));
                                pk[j] = pack2_finite<T>(p.x, p.y);
                            }
                        };
                        // A third of the exponentials goes to the multiply-add units: with fewer the special-function unit, with
                        // half of them those units are the busier (none 469 us, a quarter 464, a third 459 at 4096 x 4096, batch 4,
                        // 16 heads of 128).  Hidden scores (-inf) have to give 0, which the polynomial does not.
                        if (partial) weights(std::false_type{}); else weights(std::true_type{});
                        tmem_st32(tsx, pk);
                        const float2 total = unpair(add2(sum[0], sum[1]));
                        l += total.x + total.y;
                        tmem_st_wait();
                        fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_full(w, x));
                        ++sc;
                        any = true;
                    }
                }
                // ------------------------------------------------------------------------------------------ results
                if (ok && any) { ok = wait(o_done(w), oc & 1); ++oc; }
                if (!ok) break;                                  // with k and item of the unfinished one
                fence_after_sync();
                const bool none = l == 0.f;
                const float inv = none ? 0.f : 1.f / l;
                const int64_t at = (((int64_t)it.split * a.B + it.b) * a.Lq + qi) * a.H + it.h;
                T *orow = (T *)a.out.ptr + it.b * a.out.batch_stride + (int64_t)qi * a.out.row_stride + (int64_t)it.h * a.D;
#pragma unroll 1
                for (int c = 0; c < DP / 32; ++c) {
                    uint32_t o[32];
                    if (any) {
                        tmem_ld32(to + 32 * c, o);
                        tmem_ld_wait();
                    }
                    if (none) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = 0u;
                    }
                    if (sp.splits > 1) {
                        store_rows32_f32(sp.part_o + at * a.D, (int64_t)a.H * a.D, a.Lq - qi, 32 * c, a.D, o);
                    } else {
                        store_rows32<T>(orow, a.out.row_stride, a.Lq - qi, 32 * c, a.D, o, inv);
                        if (a.out_lo != nullptr)
                            store_rows32<T, true>((T *)a.out_lo + at * a.D, (int64_t)a.H * a.D, a.Lq - qi, 32 * c, a.D, o, inv);
                    }
                }
                if (qi < a.Lq) {
                    if (sp.splits > 1) *reinterpret_cast<float2 *>(sp.part_ml + 2 * at) = make_float2(m * a.scale_log2 - SHIFT, l);
                    if (sp.splits == 1 && a.lse != nullptr) a.lse[at] = none ? -INFINITY : (m * a.scale_log2 - SHIFT + log2f(l)) * 0.6931471805599453f;
                }
                if (sp.splits == 1 && a.empty_value != 0.f) {        // other lanes wrote the row's zeros: they come first
                    __syncwarp();
                    if (qi < a.Lq && none) fill_row<T>(orow, a.D, a.empty_value);
                }
                fence_before_sync();                             // the accumulator may be written again
            }
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
                const FwdItem it(a, sp.splits, item);
                void_row(it, it.q0 + 128 * w + row);
                item = -1;
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (warp == 9) tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0 && *abort_flag) atomicAdd(&g_dense_aborts, 1u);
}

// A block of queries costs its key tiles plus about four tiles' time of set-up and result, twice that when the result is partial.
static int dense_fwd_splits(int B, int Lq, int Lk, int H) {
    return range_count((long long)B * H * ((Lq + 255) / 256), (Lk + 127) / 128, 4.0, 8.0);
}

size_t dense_fwd_tc_workspace(int B, int Lq, int Lk, int H, int D) { return fwd_part_bytes(dense_fwd_splits(B, Lq, Lk, H), B, Lq, H, D); }

static bool tc_view(const hsa_view &v, int B, int rows, int H, int D) { return view_vec_ok(v, 2) && map_ok(v, B, rows, H, D); }

// bf16 / f16 with head dims in whole 16-byte pieces up to 128, rows a tensor map can describe, and a mask whose tile states
// fit the block's table.
bool dense_tc_ok(const DenseArgs &a, int dtype, bool backward) {
    if ((dtype != HSA_BF16 && dtype != HSA_F16) || a.D % 8 != 0 || a.D > 128) return false;
    if (a.mask.bits != nullptr && a.mask.tk > kFlagTiles) return false;
    if (!tc_view(a.q, a.B, a.Lq, a.H, a.D) || !tc_view(a.k, a.B, a.Lk, a.Hkv, a.D) || !tc_view(a.v, a.B, a.Lk, a.Hkv, a.D)) return false;
    if (!backward) return tc_view(a.out, a.B, a.Lq, a.H, a.D);
    return tc_view(a.dout, a.B, a.Lq, a.H, a.D) && (a.dq.ptr == nullptr || tc_view(a.dq, a.B, a.Lq, a.H, a.D)) &&
           (a.dk.ptr == nullptr || (tc_view(a.dk, a.B, a.Lk, a.Hkv, a.D) && tc_view(a.dv, a.B, a.Lk, a.Hkv, a.D)));
}

template <typename T, int DP>
static int fwd_launch(const DenseArgs &a, DenseSplit sp, cudaStream_t st) {
    CUtensorMap mq, mk, mv;
    if (!make_map(&mq, a.q, a.B, a.Lq, a.H, a.D, 1, 128) || !make_map(&mk, a.k, a.B, a.Lk, a.Hkv, a.D, 1, 128) ||
        !make_map(&mv, a.v, a.B, a.Lk, a.Hkv, a.D, 1, 128))
        return fail(HSA_ERR_ARG, "hsa_dense_attn_fwd: the driver refused a tensor map");
    const long long blocks = (long long)a.B * a.H * ((a.Lq + 255) / 256) * sp.splits;
    if (blocks > 0x7fffffffLL) return fail(HSA_ERR_ARG, "hsa_dense_attn_fwd: too many tiles");
    constexpr auto kernel = dense_fwd_tc5_kernel<T, DP>;
    constexpr int smem = FwdShape<DP>::kSmem;
    const cudaError_t e = allow_smem<kernel>(smem);
    if (e != cudaSuccess) return fail((int)e, "hsa_dense_attn_fwd: shared memory %d: %s", smem, cudaGetErrorString(e));
    kernel<<<(unsigned)blocks, kFwdThreads, smem, st>>>(a, sp, mq, mk, mv);
    if (int rc = launch_status("hsa_dense_attn_fwd")) return rc;
    return sp.splits > 1 ? join_forward<T>(a, sp, st) : 0;
}

int dense_fwd_tc(const DenseArgs &a, void *workspace, int dtype, cudaStream_t st) {
    const DenseSplit sp = fwd_split(dense_fwd_splits(a.B, a.Lq, a.Lk, a.H), a, workspace);
    if (dtype == HSA_BF16)
        return a.D <= 64 ? fwd_launch<__nv_bfloat16, 64>(a, sp, st) : fwd_launch<__nv_bfloat16, 128>(a, sp, st);
    return a.D <= 64 ? fwd_launch<__half, 64>(a, sp, st) : fwd_launch<__half, 128>(a, sp, st);
}

}  // namespace hsa

namespace hsa { cudaError_t dense_bwd_aborts(unsigned int *count); }

extern "C" int hsa_dense_attn_aborts(unsigned int *count) {
    if (count == nullptr) return hsa::fail(HSA_ERR_ARG, "hsa_dense_attn_aborts: null pointer");
    unsigned int bwd = 0;
    cudaError_t e = cudaDeviceSynchronize();                 // the copy alone does not wait for streams that do not wait for the default one
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(count, hsa::g_dense_aborts, sizeof(unsigned int));
    if (e == cudaSuccess) e = hsa::dense_bwd_aborts(&bwd);
    if (e == cudaSuccess) *count += bwd;
    return e == cudaSuccess ? 0 : hsa::fail((int)e, "hsa_dense_attn_aborts: %s", cudaGetErrorString(e));
}
