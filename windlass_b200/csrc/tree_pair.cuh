// tree_pair.cuh — attention of drafted trees, two nodes of a request at a time, by
// pairs of CTAs (the same mathematics as tree_attn.cuh, every key a node sees).
//
// An MMA with M = 64 costs as many cycles as one with M = 128 (measured: N = 64,
// K = 16: 32; N = 256: 128), so 128 rows (two nodes x 64 heads) double the rate.
// Their O [128 x 512] fp32 fills an SM's tensor memory alone, which leaves no
// room for scores: a cluster of two CTAs splits the work by operation. Per tile
// of 64 keys:
//   score CTA  S = Q K^T (A = the queries in tensor memory, 288 columns; S twice
//              64 columns): 36 MMAs M = 128, N = 64: 1,152 cycles. Its softmax
//              warps keep the running maximum and sum, one row a thread; each
//              sends its rows' P (bf16, 4 KB) and rescale factors by a bulk copy
//              into the value CTA's shared memory, four tiles deep (stores of
//              16 bytes to the other SM took 4,700 cycles a tile).
//   value CTA  O += P V: 8 MMAs M = 128, N = 256: 1,024 cycles. Four warps rescale
//              O when a factor is not 1 (rare: the maximum moves only by more than
//              2^8), and write O / l at the end of an item.
// So both SMs work on the same 64 keys of two nodes, in 1,434 to 1,484 cycles, where
// two SMs of tree_attn_kernel take 2,176 for one node each. Each key row is read by
// both CTAs (from L2 once more), 50 bytes a cycle and SM.
// Bound: shared-memory bandwidth. A score SM writes 72 KB of keys, reads them for the MMAs and
// writes and sends 16 KB of P, a value SM likewise: 1,410 cycles at 128 bytes; 1,434
// (1 request x 64 nodes x 30K) and 1,484 (9 x 16 x 16K) measured.
// Under lasting load the power cap brings the clock down: 394 nodes of 16 requests x 32K keys
// 1,240 us (1.14 PFLOP/s), 92 nodes of 8 x 16K 173 us; in the first calls after a rest 1,090 and 155 us.
// Two nodes share V in one MMA: a drafted row that not both see, and that holds
// a NaN or an infinity, would reach the other through 0 x NaN. In tiles with
// drafted rows the value CTA therefore clears rows that neither sees and the
// non-finite elements of rows that one sees. Whatever the weight p is (0, or NaN),
// p x NaN and p x infinity are NaN there: the value CTA notes these columns for the
// node that sees the row and writes NaN into them. Scores are per row; unseen ones are masked.
#pragma once
#include "tree_attn.cuh"

namespace wl {

// Warps 0-7 rows (score: four for even and four for odd tiles; value: 0-3), 8 and 9 loads of even and odd tiles,
// 10 and 11 MMAs (score: of even and odd tiles; value: 10). One warp for each took 1,500 to 1,700 cycles a tile.
constexpr int TP_THREADS = 384;
constexpr int TP_LOAD_WARP = 8, TP_MMA_WARP = 10;
// Even and odd tiles have their own space, loader, MMA warp and softmax warps throughout, so that each barrier's
// phases are waited for one after the other by the same threads (a wait that skipped a phase could take an older
// one for it):
constexpr int TP_UNITS = 6;   // score CTA: [even, odd][3] thirds of a tile (64 keys x 192 columns), the queries' way in
constexpr int TP_HALVES = 4;  // value CTA: [even, odd][2] halves of a tile (64 keys x 256 columns)
constexpr int TP_P = 4;       // value CTA: tiles of P (score CTA: on their way), tile & 3
constexpr uint32_t TP_TM_S = 384;  // score columns in tensor memory (the queries take [0, 288))
// (0.8 us a tile; see TA_PRICE. From a rest, at these and at (6, .12, .2): 9 requests, 109 nodes x 9K 126 / 144 us, 12, 74 x 13K
// 121 / 128, 8, 92 x 16K 166 / 169; 20, 235 x 3K 95 / 92.)
constexpr TreePrice TP_PRICE = {6.f, 0.03f, 0.06f};

struct TpLayout {
    static constexpr uint32_t CHUNK = TA_TILE * 128;          // 8 KB: 64 keys x 64 columns
    static constexpr uint32_t UNIT = 3 * CHUNK, HALF = 4 * CHUNK;
    static constexpr uint32_t P = 128 * 128;                  // 128 rows x 64 keys bf16
    static constexpr uint32_t OFF_P = TP_HALVES * HALF;       // value CTA
    static constexpr uint32_t OFF_PS = TP_UNITS * UNIT;       // score CTA: P on its way
    // Both: the schedule's sums and table. The score CTA's first copies of P may reach a value CTA that is still at its
    // schedule (nothing waits for it before), so the scratch is behind P there; in the score CTA it is the place of
    // the fourth tile of P, which only that CTA writes, after its schedule.
    static constexpr uint32_t OFF_SCHED = OFF_P + TP_P * P;
    static constexpr uint32_t OFF_ALPHA = OFF_PS + TP_P * P;  // both: rescale factors [TP_P][128]
    static constexpr uint32_t OFF_FIN = OFF_ALPHA + TP_P * 512;  // value CTA: 1 / l of the item's rows [128]
    static constexpr uint32_t OFF_MAX = OFF_FIN + 512;        // score CTA: rows' maxima after even and odd tiles [2][128]
    static constexpr uint32_t OFF_SUM = OFF_MAX + 1024;       // score CTA: one half's (sum, maximum) at an item's end [128]
    static constexpr uint32_t OFF_ITEM = OFF_SUM + 1024;      // item descriptors [2]
    static constexpr uint32_t OFF_LOST = OFF_ITEM + 128;      // keys lost to bad pages, per tile [8]
    static constexpr uint32_t OFF_NAN = OFF_LOST + 64;        // value CTA: columns that are NaN, by item & 1 and node [2][2][512 bits]
    static constexpr uint32_t OFF_BAR = OFF_NAN + 256;
    static constexpr int N_BARS = 34;
    static constexpr uint32_t OFF_MISC = OFF_BAR + N_BARS * 8;  // tensor-memory slot, longest, out count, slots [2][8]
    static constexpr uint32_t BYTES = OFF_MISC + 80 + 1024;
    static constexpr uint32_t IDESC_QK = idesc_bf16(128, TA_TILE, 0, 0);
    static constexpr uint32_t IDESC_PV = idesc_bf16(128, 256, 0, 1);
};
static_assert(TpLayout::BYTES <= 232448, "one CTA per SM");
static_assert(TP_P == 4 && TpLayout::OFF_SCHED + sizeof(TreeCost) + 32 * sizeof(int2) <= TpLayout::OFF_ALPHA, "value CTA's layout");
static_assert(TpLayout::OFF_SCHED >= TpLayout::OFF_PS, "score CTA's layout: no key tile over the schedule");

struct TpItem {  // what the roles of a CTA need of an item
    int rows, row0;        // nodes (1 or 2; 0: no more), first row
    int tiles, pos0, ctx;  // key tiles, position of the first key
    int part, runs;        // first node's partial (-1: written directly); the second node's is `runs` on
    int pad;
    unsigned long long see[2];
};
static_assert(sizeof(TpItem) == 48, "descriptor");

// e^(x ln 2); denormal results flush to zero.
__device__ __forceinline__ float exp2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// N column chunks from C0 on of a key tile in NB boxes, by one thread (see tree_boxes).
template <int NB, int C0, int N>
__device__ __forceinline__ void pair_boxes(const TreeMaps& tm, uint32_t dst, const volatile int* rows, uint64_t* bar) {
    constexpr uint32_t CHUNK = TA_TILE * 128, BOX = CHUNK / NB;
    constexpr int M = C0 + N > 8 ? 8 - C0 : N;  // latent chunks; the ninth is the roped one
    int y[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) y[j] = rows[j];
#pragma unroll(NB <= 2 ? 4 : 1)
    for (int c = 0; c < M; ++c) {
#pragma unroll
        for (int j = 0; j < NB; ++j) tma_load2d(dst + c * CHUNK + j * BOX, &tm.ckv, (C0 + c) * 64, y[j], bar);
    }
    if (M < N) {
#pragma unroll
        for (int j = 0; j < NB; ++j) tma_load2d(dst + M * CHUNK + j * BOX, &tm.krot, 0, y[j], bar);
    }
}
template <int C0, int N>
__device__ __forceinline__ void pair_load(const TreeMaps& tm, uint32_t dst, int nbox, const volatile int* rows, uint64_t* bar) {
    if (elect_one()) {
        mbar_expect_tx(bar, (uint32_t)N * TpLayout::CHUNK);
        if (nbox == 1) pair_boxes<1, C0, N>(tm, dst, rows, bar);
        else if (nbox == 2) pair_boxes<2, C0, N>(tm, dst, rows, bar);
        else if (nbox == 4) pair_boxes<4, C0, N>(tm, dst, rows, bar);
        else pair_boxes<8, C0, N>(tm, dst, rows, bar);
    }
    __syncwarp();
}

__device__ __forceinline__ unsigned nonfinite(uint32_t w) {  // which of two bf16
    return ((w & 0x7f80u) == 0x7f80u ? 1u : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 2u : 0u);
}
__device__ __forceinline__ uint32_t clear_nonfinite(uint32_t w) {
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
    return w;
}

__global__ void __launch_bounds__(TP_THREADS, 1) tree_pair_kernel(const TreeParams p, const __grid_constant__ TreeMaps tm) {
    using L = TpLayout;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t base = smem_u32(smem);
    float* alpha_sh = reinterpret_cast<float*>(smem + L::OFF_ALPHA);
    float* fin_sh = reinterpret_cast<float*>(smem + L::OFF_FIN);
    float* max_sh = reinterpret_cast<float*>(smem + L::OFF_MAX);
    float2* sum_sh = reinterpret_cast<float2*>(smem + L::OFF_SUM);
    TpItem* item_sh = reinterpret_cast<TpItem*>(smem + L::OFF_ITEM);
    unsigned long long* lost_sh = reinterpret_cast<unsigned long long*>(smem + L::OFF_LOST);
    unsigned* nan_sh = reinterpret_cast<unsigned*>(smem + L::OFF_NAN);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
    uint64_t *ifull = bars, *ifree = bars + 2;  // item descriptors
    // score CTA
    uint64_t *ufull = bars + 4, *ufree = bars + 10, *qtmem = bars + 16, *sfull = bars + 17, *sfree = bars + 19, *pfree = bars + 21,
             *finfree = bars + 25, *mready = bars + 26, *lready = bars + 28, *ldone = bars + 29;
    // value CTA (pfree's places are not used here: the commit that frees P names them in the score CTA)
    uint64_t *vfull = bars + 4, *vfree = bars + 8, *pfull = bars + 12, *pok = bars + 16, *pvdone = bars + 26, *finfull = bars + 30;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
    int* longest_sh = reinterpret_cast<int*>(tmem_slot + 1);
    int* out_done = reinterpret_cast<int*>(tmem_slot + 2);
    volatile int* slots_sh = reinterpret_cast<volatile int*>(tmem_slot + 4);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const bool score = rank == 0;
    const int me = blockIdx.x / 2, G = gridDim.x / 2;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(ifull + i, 1);
            mbar_init(ifree + i, score ? 10 : 5);  // a lane of each consumer warp
        }
        if (score) {
            for (int i = 0; i < TP_UNITS; ++i) {
                mbar_init(ufull + i, 1);
                mbar_init(ufree + i, 1);
            }
            mbar_init(qtmem, 256);
            for (int i = 0; i < 2; ++i) {
                mbar_init(sfull + i, 1);
                mbar_init(sfree + i, 128);
                mbar_init(mready + i, 128);
            }
            mbar_init(lready, 128);
            mbar_init(ldone, 128);
            for (int i = 0; i < TP_P; ++i) mbar_init(pfree + i, 1);
            mbar_init(finfree, 4);
        } else {
            for (int i = 0; i < TP_HALVES; ++i) {
                mbar_init(vfull + i, 1);
                mbar_init(vfree + i, 1);
            }
            for (int i = 0; i < TP_P; ++i) {
                mbar_init(pfull + i, 1);
                mbar_init(pok + i, 128);
                mbar_init(pvdone + i, 1);
            }
            mbar_init(finfull, 128);
            *out_done = 0;
        }
        fence_mbar_init();
        if (!score)
            for (int i = 0; i < TP_P; ++i) mbar_expect_tx(pfull + i, L::P + 512);
    }
    if (tid < 64) nan_sh[tid] = 0;
    if (warp == TP_MMA_WARP) tmem_alloc(tmem_slot, 512);
    if (warp == TP_LOAD_WARP && lane < 3)
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane == 0 ? &tm.q : lane == 1 ? &tm.ckv : &tm.krot)) : "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    cluster_sync_all();  // both CTAs' barriers exist before either reaches into the other
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_trigger();
    TreeCost* cost = reinterpret_cast<TreeCost*>(smem + L::OFF_SCHED);
    const bool many = p.batch > 32;
    int2* tab = reinterpret_cast<int2*>(many ? smem : smem + L::OFF_SCHED + sizeof(TreeCost));
    TreeWalk<false, 2> walk;
    if (many) {
        if (tid == 0) *longest_sh = 0;
        __syncthreads();
        int longest = 0;
        for (int b = tid; b < p.batch; b += TP_THREADS) {
            const TreeSeq q = tree_seq(p, b);
            const int t = q.n > 0 ? tree_tiles<false>(p, q) : 0;
            tab[b] = make_int2(q.n, t);
            longest = max(longest, t);
        }
        if (longest > 0) atomicMax(longest_sh, longest);
    }
    const bool loads = warp == TP_LOAD_WARP || warp == TP_LOAD_WARP + 1;
    if (loads) {
        walk.b0 = walk.item0 = walk.part0 = 0;
        walk.load(p);
        if (!many) {
            if (p.batch > 1) walk.sort(walk.tiles);
            if (warp == TP_LOAD_WARP && lane < p.batch) tab[lane] = make_int2(walk.n, walk.tiles);
            if (warp == TP_LOAD_WARP && lane == 0) *longest_sh = walk.tiles;
        }
    }
    __syncthreads();
    const int chosen = tree_schedule<2>(p, tab, *longest_sh, cost, G, TP_PRICE, TP_LOAD_WARP);
    if (warp == TP_LOAD_WARP && lane == 0) *longest_sh = chosen;
    fence_proxy_async_smem();  // the scratch becomes key tiles and P: its generic accesses come before async writes
    __syncthreads();
    walk.C = *longest_sh;

    bool ok = true;
    // the consumers' view of item k
    auto take = [&](int k, TpItem& t) -> bool {
        const int x = k & 1;
        if (!mbar_wait_fast(ifull + x, (uint32_t)(k >> 1) & 1u, 70)) return false;
        t = item_sh[x];
        __syncwarp();
        if (lane == 0) mbar_arrive(ifree + x);
        return true;
    };
    if (loads) {
        // ---------------- loads: even or odd tiles ----------------
        if (p.batch > 1 && !many) walk.sort(walk.run_len());
        walk.count();
        const int which = warp - TP_LOAD_WARP;
        if (score && me == G - 1 && which == 0) tree_table(p, walk);
        const int steps = score ? 3 : 2;          // pieces of a tile
        const int first = which * steps;          // this loader's barriers
        int use = 0, gt = 0;                      // times its space was filled; the CTA's tiles so far
        uint64_t *full = (score ? ufull : vfull) + first, *free_ = (score ? ufree : vfree) + first;
        volatile int* slots = slots_sh + 8 * which;
        const uint32_t space = base + (uint32_t)first * (score ? L::UNIT : L::HALF);
        auto acquire = [&](int j) -> bool { return use == 0 || mbar_wait_fast(free_ + j, (uint32_t)(use - 1) & 1u, 71); };
        for (int k = 0; ok; ++k) {
            TreeItem t{};
            const bool more = tree_item(p, walk, item_of(k, me, G), t);
            const int rows = more ? min(2, t.n - t.node) : 0;
            if (score && more) {
                // the query of the first node by the one loader, of the second (a lone node's again) by the other
                for (int j = 0; j < 3; ++j) {
                    if (!(ok = acquire(j))) break;
                    const int y = (t.r0 + t.node + min(which, rows - 1)) * AT_H;
                    if (elect_one()) {
                        mbar_expect_tx(full + j, L::UNIT);
                        for (int c = 0; c < 3; ++c) tma_load2d(space + j * L::UNIT + c * L::CHUNK, &tm.q, (3 * j + c) * 64, y, full + j);
                    }
                    __syncwarp();
                }
                if (!ok) break;
                ++use;
            }
            const int own = (gt & 1) == which ? 0 : 1;  // this loader's first tile
            TreePages<2> pages;
            if (more) pages.start(p, t, own);
            if (which == 0) {
                if (k >= 2 && !(ok = mbar_wait_fast(ifree + (k & 1), (uint32_t)((k >> 1) - 1) & 1u, 72))) break;
                TpItem d{};
                if (more) {
                    d.see[0] = tree_mask_of(p, t.r0, t.n, t.node);
                    d.see[1] = rows > 1 ? tree_mask_of(p, t.r0, t.n, t.node + 1) : d.see[0];
                    d.rows = rows;
                    d.row0 = t.r0 + t.node;
                    d.tiles = t.tiles;
                    d.pos0 = t.tile0 * TA_TILE;
                    d.ctx = t.ctx;
                    d.part = t.part;
                    d.runs = t.runs;
                }
                if (lane == 0) {
                    item_sh[k & 1] = d;
                    mbar_arrive(ifull + (k & 1));
                }
                __syncwarp();
            }
            if (!more) break;
            for (int i = own; i < t.tiles; i += 2) {
                unsigned long long lost;
                const int slot = pages.next(i + 2 < t.tiles, lost);
                if (lane < 8) slots[lane] = slot;
                if (lane == 0) lost_sh[(gt + i) & 7] = lost;
                __syncwarp();
                if (score) {
                    if (!(ok = acquire(0))) break;
                    pair_load<0, 3>(tm, space, pages.nbox, slots, full);
                    if (!(ok = acquire(1))) break;
                    pair_load<3, 3>(tm, space + L::UNIT, pages.nbox, slots, full + 1);
                    if (!(ok = acquire(2))) break;
                    pair_load<6, 3>(tm, space + 2 * L::UNIT, pages.nbox, slots, full + 2);
                } else {
                    if (!(ok = acquire(0))) break;
                    pair_load<0, 4>(tm, space, pages.nbox, slots, full);
                    if (!(ok = acquire(1))) break;
                    pair_load<4, 4>(tm, space + L::HALF, pages.nbox, slots, full + 1);
                }
                ++use;
            }
            gt += t.tiles;
        }
        if (!ok && use > 0)  // copies in flight must land before the CTA leaves
            for (int j = 0; j < steps; ++j) mbar_wait_fast(full + j, (uint32_t)(use - 1) & 1u, 73);
    } else if (score && warp >= TP_MMA_WARP) {
        // ---------------- score CTA: Q K^T of even or odd tiles ----------------
        // (two warps, so that the waits of one tile pass under the MMAs of the other)
        const int s = warp - TP_MMA_WARP;
        const uint32_t d = tmem + TP_TM_S + (uint32_t)(s * TA_TILE);
        uint64_t *full = ufull + 3 * s, *free_ = ufree + 3 * s;
        const uint64_t k0 = desc_sw128(base + (uint32_t)(3 * s) * L::UNIT, 16, 1024);
        int use = 0, gt = 0;
        for (int k = 0; ok; ++k) {
            TpItem t;
            if (!(ok = take(k, t)) || t.rows == 0) break;
            if (!(ok = mbar_wait_fast(qtmem, (uint32_t)k & 1u, 74))) break;  // the queries are in tensor memory
            if (elect_one())
                for (int j = 0; j < 3; ++j) mbar_arrive(free_ + j);
            __syncwarp();
            ++use;
            for (int i = 0; i < t.tiles && ok; ++i, ++gt) {
                if ((gt & 1) != s) continue;
                if (gt >= 2 && !(ok = mbar_wait_fast(sfree + s, (uint32_t)((gt >> 1) - 1) & 1u, 75))) break;
#pragma unroll
                for (int j = 0; j < 3; ++j) {
                    if (!(ok = mbar_wait_fast(full + j, (uint32_t)use & 1u, 76))) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int c = 0; c < 3; ++c)
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                mma_bf16_ts(d, tmem + (uint32_t)((3 * j + c) * 32 + kk * 8), k0 + (((3 * j + c) * L::CHUNK + kk * 32) >> 4),
                                            L::IDESC_QK, (j | c | kk) != 0 ? 1u : 0u);
                        mma_commit(free_ + j);
                        if (j == 2) mma_commit(sfull + s);
                    }
                    __syncwarp();
                }
                ++use;
            }
        }
    } else if (score) {
        // ---------------- score CTA: softmax of even (warps 0-3) or odd tiles (4-7), one row a thread ----------------
        const int r = tid & 127, half = r >> 6, s = tid >> 7, quarter = warp & 3;
        const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
        int gt = 0, tiles_of[2] = {0, 0};  // the CTA's tiles so far, even and odd
        // scores are scaled inside the exponent's multiply-add, so maxima are of raw scores: a negative scale
        // flips them once, and none at all (every key alike) is as good as a tiny one
        const bool flip = p.scale_log2 < 0.f;
        const float scale = fmaxf(fabsf(p.scale_log2), 1e-30f);
        const uint32_t p_here = base + L::OFF_PS + (uint32_t)r * 128u;
        for (int k = 0; ok; ++k) {
            TpItem t;
            if (!(ok = take(k, t)) || t.rows == 0) break;
            // this row's query into tensor memory, two thirds by warps 0-3, one by 4-7 (every QK of the item
            // before is done: its last scores were read)
            const uint32_t qph = (uint32_t)(k + tiles_of[half]) & 1u;  // the space of the node's query was filled that often
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                if ((j == 2) != (s == 1)) continue;
                if (!(ok = mbar_wait_fast(ufull + 3 * half + j, qph, 78))) break;
                const uint32_t src = base + (uint32_t)(3 * half + j) * L::UNIT + (uint32_t)(r & 63) * 128u;
#pragma unroll
                for (int c = 0; c < 3; ++c) {
                    uint32_t v[32];
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const uint4 w = lds_v4(src + c * L::CHUNK + (uint32_t)((x ^ r) & 7) * 16u);
                        v[4 * x] = w.x;
                        v[4 * x + 1] = w.y;
                        v[4 * x + 2] = w.z;
                        v[4 * x + 3] = w.w;
                    }
                    tmem_st32(tmem + lanes + (uint32_t)((3 * j + c) * 32), v);
                }
            }
            if (!ok) break;
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(qtmem);
            tiles_of[gt & 1] += (t.tiles + 1) / 2;
            tiles_of[(gt & 1) ^ 1] += t.tiles / 2;
            const unsigned long long see = t.see[half];
            float m_mine = -INFINITY, l_run = 0.f;  // this half's sum, and the maximum that it is relative to
            for (int i = 0; i < t.tiles; ++i, ++gt) {
                if ((gt & 1) != s) continue;
                const int pb = gt & 3;
                if (!(ok = mbar_wait_fast(sfull + s, (uint32_t)(gt >> 1) & 1u, 79))) break;
                tc_fence_after();
                float sv[64];
                tmem_ld64(tmem + lanes + TP_TM_S + (uint32_t)(s * TA_TILE), sv);
                tc_fence_before();
                mbar_arrive(sfree + s);
                const unsigned long long lost = lost_sh[gt & 7];
                const unsigned long long bits = tree_tile_mask(see, t.pos0 + i * TA_TILE, t.ctx) & ~lost;
                if (flip) {
#pragma unroll
                    for (int j = 0; j < 64; ++j) sv[j] = -sv[j];
                }
                if (bits != ~0ull) {
#pragma unroll
                    for (int j = 0; j < 64; ++j) sv[j] = (bits >> j) & 1 ? sv[j] : -INFINITY;
                }
                float top[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
                for (int j = 4; j < 64; ++j) top[j & 3] = fmaxf(top[j & 3], sv[j]);
                const float tmax = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
                // the row's maximum runs through all tiles: from the other half's tile before to its next
                if (gt > 0 && !(ok = mbar_wait_fast(mready + (s ^ 1), (uint32_t)((gt - 1) >> 1) & 1u, 90))) break;
                const float m_run = i == 0 ? -INFINITY : max_sh[128 * (s ^ 1) + r];
                const float m_new = (m_run == -INFINITY || tmax > m_run + PF_RESCALE_LOG2) ? tmax : m_run;
                max_sh[128 * s + r] = m_new;
                mbar_arrive(mready + s);
                const float m_use = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = m_run == -INFINITY ? 0.f : exp2_ftz(m_run - m_new);
                // P's place, here and there: the P.V of four tiles before has read it
                if (gt >= 4 && !(ok = mbar_wait_cluster(pfree + pb, (uint32_t)((gt >> 2) - 1) & 1u, 80))) break;
                const uint32_t prow = p_here + (uint32_t)pb * L::P;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t w[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float e0 = exp2_ftz(fmaf(sv[8 * c + 2 * x], scale, -m_use)), e1 = exp2_ftz(fmaf(sv[8 * c + 2 * x + 1], scale, -m_use));
                        const __nv_bfloat162 b2 = __floats2bfloat162_rn(e0, e1);
                        w[x] = *reinterpret_cast<const uint32_t*>(&b2);
                        sum[x] += e0 + e1;
                    }
                    sts_v4(prow + (uint32_t)((c ^ r) & 7) * 16u, make_uint4(w[0], w[1], w[2], w[3]));
                }
                // O moves to the new maximum only after the item's first tile; the sign tells of keys lost to bad pages
                const float factor = i == 0 || m_new == m_run ? 1.f : alpha;
                alpha_sh[128 * pb + r] = lost != 0 ? -factor : factor;
                l_run = l_run * (m_mine == -INFINITY ? 0.f : exp2_ftz(m_mine - m_new)) + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
                m_mine = m_new;
                fence_proxy_async_smem();  // the copies read this warp's writes
                __syncwarp();
                if (elect_one()) {
                    const uint32_t bar = dsmem_addr(pfull + pb, 1), row0 = 32u * quarter;
                    bulk_s2s(dsmem_addr(smem + L::OFF_P + pb * L::P + row0 * 128u, 1), base + L::OFF_PS + pb * L::P + row0 * 128u, 4096, bar);
                    bulk_s2s(dsmem_addr(alpha_sh + 128 * pb + row0, 1), smem_u32(alpha_sh + 128 * pb + row0), 128, bar);
                }
                __syncwarp();
            }
            if (!ok) break;
            // the half without the item's last tile hands its sum to the other
            if (((gt - 1) & 1) != s) {
                sum_sh[r] = make_float2(l_run, m_mine);
                mbar_arrive(lready);
                if (!(ok = mbar_wait_fast(ldone, (uint32_t)k & 1u, 91))) break;
                continue;  // every QK of the item is done
            }
            if (!(ok = mbar_wait_fast(lready, (uint32_t)k & 1u, 92))) break;
            const float2 other = sum_sh[r];
            l_run += other.x * (other.y == -INFINITY ? 1.f : exp2_ftz(other.y - m_mine));  // (its sum is then 0, or NaN)
            const bool any = l_run != 0.f;  // (NaN counts: it reaches the result)
            if (half < t.rows) {
                const float lse = any ? (m_mine + log2f(l_run)) * 0.69314718055994531f : -INFINITY;
                const int h = r & 63;
                if (t.part >= 0) p.lse_part[(long long)(t.part + half * t.runs) * AT_H + h] = lse;
                else if (p.lse) p.lse[(long long)(t.row0 + half) * AT_H + h] = lse;
            }
            if (k >= 1 && !(ok = mbar_wait_cluster(finfree, (uint32_t)(k - 1) & 1u, 81))) break;
            dsmem_st_f32(dsmem_addr(fin_sh + r, 1), any ? 1.f / l_run : 0.f);
            mbar_arrive_remote(dsmem_addr(finfull, 1));
            mbar_arrive(ldone);
            if (!(ok = mbar_wait_fast(ldone, (uint32_t)k & 1u, 91))) break;  // all of its threads are this far
        }
        // The last tiles of P: the value CTA's word that their places are free must be here before this CTA leaves.
        for (int pb = s; ok && pb < TP_P && pb < gt; pb += 2) ok = mbar_wait_cluster(pfree + pb, (uint32_t)((gt - 1 - pb) >> 2) & 1u, 80);
    } else if (warp == TP_MMA_WARP) {
        // ---------------- value CTA: P V ----------------
        int gt = 0;
        for (int k = 0; ok; ++k) {
            TpItem t;
            if (!(ok = take(k, t)) || t.rows == 0) break;
            for (int i = 0; i < t.tiles && ok; ++i, ++gt) {
                const int pb = gt & 3, v = 2 * (gt & 1);
                if (!(ok = mbar_wait_fast(pok + pb, (uint32_t)(gt >> 2) & 1u, 82))) break;  // P is here, O at its maximum
                const uint64_t p0 = desc_sw128(base + L::OFF_P + pb * L::P, 16, 1024);
                const uint64_t v0 = desc_sw128(base + v * L::HALF, L::CHUNK, 1024);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (!(ok = mbar_wait_fast(vfull + v + half, (uint32_t)(gt >> 1) & 1u, 83))) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < TA_TILE / 16; ++ks)
                            mma_bf16(tmem + (uint32_t)(half * 256), p0 + ks * 2, v0 + ((half * L::HALF + ks * 2048) >> 4), L::IDESC_PV,
                                     (i > 0 || ks > 0) ? 1u : 0u);
                        if (i + 1 < t.tiles) mma_commit(vfree + v + half);  // the item's last tile: its output goes through this space
                        if (half == 1) {
                            mma_commit(pvdone + pb);
                            mma_commit_cluster(pfree + pb, 1);  // P's place is free, to the score CTA
                        }
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp < 4) {
        // ---------------- value CTA: rescale and output, one row a thread (warps 0-3) ----------------
        const int r = tid, half = r >> 6;
        const uint32_t lanes = (uint32_t)(32 * warp) << 16;
        int gt = 0;
        auto pv_done = [&](int tile, unsigned site) -> bool { return mbar_wait_fast(pvdone + (tile & 3), (uint32_t)(tile >> 2) & 1u, site); };
        for (int k = 0; ok; ++k) {
            TpItem t;
            if (!(ok = take(k, t)) || t.rows == 0) break;
            for (int i = 0; i < t.tiles; ++i, ++gt) {
                const int pos = t.pos0 + i * TA_TILE;
                const int pb = gt & 3, v = 2 * (gt & 1);
                if (!(ok = mbar_wait_fast(pfull + pb, (uint32_t)(gt >> 2) & 1u, 85))) break;
                if (tid == 0) mbar_expect_tx(pfull + pb, L::P + 512);  // for the P of four tiles on
                const float alpha = fabsf(alpha_sh[128 * pb + r]);
                if (pos + TA_TILE > t.ctx || signbit(alpha_sh[128 * pb + r])) {  // rows that not both nodes see
                    // These warps run ahead of the values (waiting for them in every tile cost 2 to 4 %), so
                    // the space's use before comes first: its barrier's phase could be taken for this one's. The
                    // loader's word on the tile is read once its keys are here.
                    if (gt >= 2 && !(ok = pv_done(gt - 2, 84))) break;
                    if (!(ok = mbar_wait_fast(vfull + v, (uint32_t)(gt >> 1) & 1u, 86) && mbar_wait_fast(vfull + v + 1, (uint32_t)(gt >> 1) & 1u, 86))) break;
                    const unsigned long long lost = lost_sh[gt & 7];
                    const unsigned long long m0 = tree_tile_mask(t.see[0], pos, t.ctx) & ~lost, m1 = tree_tile_mask(t.see[1], pos, t.ctx) & ~lost;
                    for (int j = warp; j < TA_TILE; j += 4) {
                        if (((m0 & m1) >> j) & 1) continue;
                        const bool one = ((m0 | m1) >> j) & 1;
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const uint32_t at = base + (uint32_t)(v + x) * L::HALF + (uint32_t)(lane >> 3) * L::CHUNK + (uint32_t)j * 128u + (uint32_t)(lane & 7) * 16u;
                            uint4 w = make_uint4(0, 0, 0, 0);
                            if (one) {
                                w = lds_v4(at);
                                const unsigned gone = nonfinite(w.x) | nonfinite(w.y) << 2 | nonfinite(w.z) << 4 | nonfinite(w.w) << 6;
                                if (gone) {  // columns 8 seg + .. of this chunk of 64 (128B swizzle)
                                    const int seg = (lane ^ j) & 7, node = (m0 >> j) & 1 ? 0 : 1;
                                    atomicOr(nan_sh + 32 * (k & 1) + 16 * node + 8 * x + 2 * (lane >> 3) + (seg >> 2), gone << (8 * (seg & 3)));
                                    w = make_uint4(clear_nonfinite(w.x), clear_nonfinite(w.y), clear_nonfinite(w.z), clear_nonfinite(w.w));
                                }
                            }
                            sts_v4(at, w);
                        }
                    }
                }
                if (__any_sync(0xffffffffu, alpha != 1.f)) {  // never at an item's first tile
                    if (!(ok = pv_done(gt - 1, 87))) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < AT_DV; c += 32) {
                        float o[32];
                        tmem_ld32(tmem + lanes + (uint32_t)c, o);
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] *= alpha;
                        tmem_st32(tmem + lanes + (uint32_t)c, reinterpret_cast<const uint32_t*>(o));
                    }
                    tmem_wait_st();
                }
                fence_proxy_async_smem();  // cleared rows are read by the tensor cores
                tc_fence_before();
                mbar_arrive(pok + pb);
            }
            if (!ok) break;
            if (!(ok = pv_done(gt - 1, 88) && mbar_wait_cluster(finfull, (uint32_t)k & 1u, 89))) break;
            if (!(ok = mbar_wait_fast(pok + ((gt - 1) & 3), (uint32_t)((gt - 1) >> 2) & 1u, 93))) break;  // all four warps' nan_sh
            tc_fence_after();
            const float inv = fin_sh[r];
            const bool none = inv == 0.f && t.part < 0;  // a sum of zero: nothing seen (a partial keeps its NaN)
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(dsmem_addr(finfree, 0));
            // O / l through the last tile's space, 128-byte pieces of this warp's 32 rows in four boxes of 4 KB
            const bool narrow = t.part < 0 && p.ctx_bf16, there = half < t.rows;
            const int y = (t.part >= 0 ? t.part + half * t.runs : t.row0 + half) * AT_H + 32 * (warp & 1);
            const int v = 2 * ((gt - 1) & 1);
            const uint32_t space = base + (uint32_t)v * L::HALF + warp * 16384u, mine = space + (uint32_t)lane * 128u;
            auto piece = [&](int box, int seg, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
                sts_v4(mine + (uint32_t)box * 4096u + (uint32_t)((seg ^ lane) & 7) * 16u, make_uint4(a, b, c, d));
            };
#pragma unroll 1
            for (int c = 0; c < AT_DV / 64; ++c) {
                float o[64];
                tmem_ld64(tmem + lanes + (uint32_t)(64 * c), o);
                if (c >= (narrow ? 4 : 2)) {  // the boxes come round again: their last stores have been read
                    if (elect_one()) {
                        if (narrow) asm volatile("cp.async.bulk.wait_group.read 3;" ::: "memory");
                        else asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                    }
                    __syncwarp();
                }
                const unsigned n0 = nan_sh[32 * (k & 1) + 16 * half + 2 * c], n1 = nan_sh[32 * (k & 1) + 16 * half + 2 * c + 1];
                if (n0 | n1) {
#pragma unroll
                    for (int x = 0; x < 64; ++x) o[x] = ((x < 32 ? n0 : n1) >> (x & 31)) & 1 ? __int_as_float(0x7fffffff) : o[x];
                }
#pragma unroll
                for (int x = 0; x < 64; ++x) o[x] = none ? 0.f : o[x] * inv;
                if (narrow) {
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        uint32_t w[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const __nv_bfloat162 b2 = __floats2bfloat162_rn(o[8 * s + 2 * x], o[8 * s + 2 * x + 1]);
                            w[x] = *reinterpret_cast<const uint32_t*>(&b2);
                        }
                        piece(c & 3, s, w[0], w[1], w[2], w[3]);
                    }
                } else {
#pragma unroll
                    for (int s = 0; s < 16; ++s)
                        piece((2 * c + (s >> 3)) & 3, s & 7, __float_as_uint(o[4 * s]), __float_as_uint(o[4 * s + 1]), __float_as_uint(o[4 * s + 2]),
                              __float_as_uint(o[4 * s + 3]));
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (elect_one()) {
                    if (there && narrow) {
                        tma_store2d(&tm.out, 64 * c, y, space + (c & 3) * 4096u);
                    } else if (there) {
                        const CUtensorMap* m = t.part >= 0 ? &tm.part : &tm.out;
                        tma_store2d(m, 64 * c, y, space + ((2 * c) & 3) * 4096u);
                        tma_store2d(m, 64 * c + 32, y, space + ((2 * c + 1) & 3) * 4096u);
                    }
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            }
            tc_fence_before();  // these reads come before the next item's P.V (ordered by pok)
            if (elect_one()) {
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __threadfence_block();
                if (atomicAdd(out_done, 1) == 3) {  // the last of the four warps gives the space back
                    *out_done = 0;
                    for (int x = 0; x < 32; ++x) nan_sh[32 * (k & 1) + x] = 0;  // next used two items on
                    mbar_arrive(vfree + v);
                    mbar_arrive(vfree + v + 1);
                }
            }
            __syncwarp();
        }
    }
    if (!ok) {  // a wait ran out: let copies between the two CTAs land before either leaves
        const long long t0 = clock64();
        while (clock64() - t0 < 200000) {
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // the other CTA may still arrive on this one's barriers
    if (warp == TP_MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace wl
