// tree_attn.cuh — absorbed-MLA attention of drafted trees over a paged latent cache.
//
// Row r = node i of request b sees the positions t < ctx_b and the nodes of its
// own ancestor mask (position ctx_b + j):
//     s[h,t] = (q_abs[r,h] . [c_kv | k_rot][slot(b,t)]) * softmax_scale
//     ctx[r,h] = sum_t softmax_t(s[h,t]) c_kv[slot(b,t)],  lse[r,h] = log sum_t e^s[h,t]
// or only those of them that its selection list names.
//
// One CTA works on one node at a time: its 64 heads are the M of the MMAs, 64
// keys a tile, so a key row that a node does not see never shares an MMA with a
// node that does, and masks stay per node. Work is cut into items (node, run of
// C key tiles); the CTAs of the grid (one per SM) take items in turn. C is
// chosen on the device from the actual lengths (tree_schedule). An item that
// holds all of its node's keys writes the result itself; the others write
// (o, lse) partials that tree_merge_kernel joins. Items of one run of keys and
// neighbouring nodes are next to each other, so a request's rows are read from
// HBM once and by its other nodes from L2.
//
// Pipeline of a CTA (mbarriers between the roles; a ring of three 72 KB tiles):
//   producer  the item's query (one ring entry), then its key tiles. Dense: one
//             warp issues TMA boxes, one per page part and 64 columns, so the
//             128B-swizzled tile needs no threads. Lists: 8 warps gather rows
//             with 16-byte cp.async, two tiles in flight.
//   MMA       QK of tile i + 1 (A = the query in tensor memory), then P.V of
//             tile i: the softmax of tile i runs under QK of tile i + 1.
//   softmax   4 warps, two threads a head: query into tensor memory, mask,
//             running maximum and sum, P (bf16) to shared memory, lazy rescale
//             of O, and the item's output, written while the MMA warp is
//             already at QK of the next item.
// Tensor memory as in mla_attn64.cuh: O in lanes 0-15 of each quarter, S tiles
// and the query in lanes 16-31.
// Roundings: scores, maxima, sums and O are fp32; only P enters P.V in bf16 (the
// tensor core's operand type: the cache is bf16); l sums P before that rounding.
#pragma once
#include "mla_attn64.cuh"
#include "paged.cuh"

namespace wl {

struct TreeParams {
    int batch, n_nodes;
    const int* ctx_len;
    const int* cu;
    const unsigned long long* mask;
    const int* parent;
    const int* table;
    long long table_stride;
    int max_pages, page_size, n_pages, T_max;
    const __nv_bfloat16* c_kv;
    const __nv_bfloat16* k_rot;
    long long ckv_row, krot_row;
    const __nv_bfloat16* q;  // [n_nodes][64][576]
    const int* sel;          // null: every key
    long long sel_stride;
    const int* sel_n_dev;
    int sel_n;
    float scale_log2;
    void* ctx;
    int ctx_bf16;
    float* lse;  // may be null
    int box_rows;      // rows of a TMA box: gcd(page_size, 64)
    float* o_part;     // [parts_max][64][512]
    float* lse_part;   // [parts_max][64]
    int2* node_tab;    // [n_nodes]: (first part, parts); parts <= 1: written directly, or not at all
    int parts_max;
};
struct TreeMaps {
    CUtensorMap q;     // {576, 64 n_nodes}, box {64, 64}
    CUtensorMap ckv;   // {512, slots}, box {64, box_rows}
    CUtensorMap krot;  // {64, slots}, box {64, box_rows}
};

// A request's rows and context; n = 0 (and the error word) when they are out of range.
struct TreeSeq {
    int r0, n, ctx;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& p, int b) {
    TreeSeq s;
    const int r1 = p.cu[b + 1];
    s.r0 = p.cu[b];
    s.ctx = p.ctx_len[b];
    s.n = r1 - s.r0;
    const long long end = (long long)s.ctx + s.n;
    if (s.r0 < 0 || r1 > p.n_nodes || s.n < 0 || s.n > TREE_MAX || s.ctx < 0 || end > p.T_max ||
        end > (long long)p.max_pages * p.page_size) {
        set_error(ERRC_BOUNDS, 44);
        s.n = 0;
    }
    return s;
}

// The nodes that node j of a request sees (bits past the request's nodes
// cleared), by a whole warp: the parents of all its nodes, two a lane, are
// walked by shuffles (one load deep instead of one per ancestor).
__device__ __forceinline__ unsigned long long tree_mask_of(const TreeParams& p, int r0, int n, int j) {
    const unsigned long long all = n >= 64 ? ~0ull : (1ull << n) - 1;
    if (p.mask) return p.mask[r0 + j] & all;
    if (!p.parent) return all & (j >= 63 ? ~0ull : (2ull << j) - 1);
    const int lane = threadIdx.x & 31;
    const int p0 = lane < n ? p.parent[r0 + lane] : -1, p1 = lane + 32 < n ? p.parent[r0 + lane + 32] : -1;
    unsigned long long m = 0;
    for (int at = j; at >= 0;) {
        m |= 1ull << at;
        const int u0 = __shfl_sync(0xffffffffu, p0, at & 31), u1 = __shfl_sync(0xffffffffu, p1, at & 31);
        const int up = at < 32 ? u0 : u1;
        if (up >= at) {  // not an earlier node
            if (lane == 0) set_error(ERRC_BOUNDS, 45);
            break;
        }
        at = up;
    }
    return m;
}

constexpr int TA_TILE = 64;
constexpr int TA_NBUF = 3;
constexpr int TA_GATHER_WARPS = 8;
constexpr int TA_MAX_BATCH = 16384;   // the schedule's table of a CTA (8 bytes a request) fits the key tiles' space
constexpr int TA_CANDS = 64;          // candidate splits: 1..32, then 36, 40, .. 160
constexpr int TA_MAX_SPLIT = 160;
constexpr float TA_ITEM_COST = 3.f;   // an item's fixed cost (query in, output out, pipeline fill), in key tiles
constexpr float TA_PART_COST = 0.04f; // a partial written and joined, in key tiles of one CTA

template <bool SEL>
struct TaLayout {
    static constexpr int LOADERS = SEL ? 32 * TA_GATHER_WARPS : 32;
    static constexpr int THREADS = 128 + LOADERS + 32;
    static constexpr int MMA_WARP = (128 + LOADERS) / 32;
    static constexpr uint32_t CHUNK = TA_TILE * 128;
    static constexpr uint32_t TILE = AT_CHUNKS * CHUNK;
    static constexpr uint32_t OFF_P = TA_NBUF * TILE;
    static constexpr uint32_t OFF_ITEM = OFF_P + AT_H * 128;           // int4 per ring entry
    static constexpr uint32_t OFF_SEE = OFF_ITEM + TA_NBUF * 16;       // valid-key bits per ring entry
    static constexpr uint32_t OFF_ROWS = OFF_SEE + TA_NBUF * 8 + 8;    // gathered rows (lists only)
    static constexpr uint32_t OFF_BAR = OFF_ROWS + (SEL ? TA_NBUF * TA_TILE * 4 : 0);
    static constexpr int N_BARS = 2 * TA_NBUF + 4 + 3;  // kfull, kfree, sfull[2], sfree[2], pready, pvdone, qtmem
    static constexpr uint32_t OFF_MISC = OFF_BAR + N_BARS * 8;         // tensor-memory slot, go flag, chosen C, node info
    static constexpr uint32_t BYTES = OFF_MISC + 64 + 1024;
    static constexpr uint32_t IDESC_QK = idesc_bf16(64, TA_TILE, 0, 0);
    static constexpr uint32_t IDESC_PV = idesc_bf16(64, 256, 0, 1);
};
static_assert(TaLayout<true>::BYTES <= 232448 && TaLayout<false>::BYTES <= 232448, "one CTA per SM");
static_assert(TA_MAX_BATCH * 8 + 1024 <= TA_NBUF * 73728, "schedule table");

// Keys of a row's list (clamped to the list's room).
__device__ __forceinline__ int tree_list_n(const TreeParams& p, int r) {
    const int n = p.sel_n_dev ? __ldg(p.sel_n_dev + r) : p.sel_n;
    return (int)min((long long)max(n, 0), p.sel_stride);
}
// Key tiles of a request's nodes (at least one).
template <bool SEL>
__device__ __forceinline__ int tree_tiles(const TreeParams& p, const TreeSeq& s) {
    if (!SEL) return (s.ctx + s.n + TA_TILE - 1) / TA_TILE;
    int m = 1;
    for (int j = 0; j < s.n; ++j) m = max(m, tree_list_n(p, s.r0 + j));
    return (m + TA_TILE - 1) / TA_TILE;
}

// Cost of a candidate in key tiles of one CTA; too large when its partials do not fit.
__device__ __forceinline__ float tree_cost(const TreeParams& p, int items, int parts, int C) {
    const float cost = (float)((items + gridDim.x - 1) / gridDim.x) * ((float)C + TA_ITEM_COST) + (float)parts * TA_PART_COST;
    return parts <= p.parts_max ? cost : 3e38f;
}
// C of the warp's cheapest candidate (the fewest runs among equals).
__device__ __forceinline__ int tree_cheapest(float best, int best_s, int longest) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float c = __shfl_xor_sync(0xffffffffu, best, o);
        const int s = __shfl_xor_sync(0xffffffffu, best_s, o);
        if (c < best || (c == best && s < best_s)) {
            best = c;
            best_s = s;
        }
    }
    return max(1, (longest + best_s - 1) / best_s);
}

// Tiles per item, from the lengths: with a request's nodes cut into runs of C
// tiles, all items run in ceil(items / CTAs) rounds of about C + TA_ITEM_COST
// tiles each, and every partial costs a write and a read. C = ceil(longest / s)
// for 64 values of s; the cheapest that fits the workspace is taken, the fewest
// parts among equals. Every CTA computes the same choice (no launch of its own).
template <bool SEL>
__device__ int tree_schedule(const TreeParams& p, uint8_t* scratch, int* out) {
    int* acc = reinterpret_cast<int*>(scratch);  // [64] items, [64] parts, longest
    int2* tab = reinterpret_cast<int2*>(scratch + 1024);
    const int tid = threadIdx.x, nthr = TaLayout<SEL>::THREADS;
    for (int i = tid; i < 2 * TA_CANDS + 1; i += nthr) acc[i] = 0;
    __syncthreads();
    int longest = 0;
    for (int b = tid; b < p.batch; b += nthr) {
        const TreeSeq s = tree_seq(p, b);
        const int t = s.n > 0 ? tree_tiles<SEL>(p, s) : 0;
        tab[b] = make_int2(s.n, t);
        longest = max(longest, t);
    }
    if (longest > 0) atomicMax(acc + 2 * TA_CANDS, longest);
    __syncthreads();
    longest = acc[2 * TA_CANDS];
    const int cand = tid % TA_CANDS, grp = tid / TA_CANDS, ngrp = nthr / TA_CANDS;
    if (grp < ngrp && longest > 0) {
        const int s = cand < 32 ? cand + 1 : 32 + 4 * (cand - 31);
        const int C = (longest + s - 1) / s;
        int items = 0, parts = 0;
        for (int b = grp; b < p.batch; b += ngrp) {
            const int2 v = tab[b];
            const int runs = (v.y + C - 1) / C;
            items += v.x * runs;
            parts += runs > 1 ? v.x * runs : 0;
        }
        atomicAdd(acc + cand, items);
        atomicAdd(acc + TA_CANDS + cand, parts);
    }
    __syncthreads();
    if (tid < 32) {
        float best = 3e38f;
        int best_s = 1;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int s = k == 0 ? tid + 1 : 32 + 4 * (tid + 1);
            const int C = max(1, (longest + s - 1) / s), i = tid + 32 * k;
            const float cost = tree_cost(p, acc[i], acc[TA_CANDS + i], C);
            if (cost < best) {
                best = cost;
                best_s = s;
            }
        }
        const int c = tree_cheapest(best, best_s, longest);
        if (tid == 0) *out = c;
    }
    __syncthreads();
    return *out;
}

// x / c for a quotient far below 2^22, by a reciprocal and one correction.
__device__ __forceinline__ int div_near(int x, int c, float inv) {
    int q = (int)((float)x * inv);
    const int r = x - q * c;
    q += r >= c ? 1 : 0;
    return r < 0 ? q - 1 : q;
}
// The same choice for at most 32 requests, one a lane, by one warp: no shared
// memory and no block barriers, so the other roles need not wait for it.
__device__ __forceinline__ int tree_schedule_warp(const TreeParams& p, int n, int tiles) {
    const int lane = threadIdx.x & 31;
    int longest = tiles;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
    const int s0 = lane + 1, s1 = 32 + 4 * (lane + 1);
    const int C0 = max(1, (longest + s0 - 1) / s0), C1 = max(1, (longest + s1 - 1) / s1);
    const float i0 = 1.f / (float)C0, i1 = 1.f / (float)C1;
    int items0 = 0, parts0 = 0, items1 = 0, parts1 = 0;
    for (int b = 0; b < p.batch; ++b) {
        const int nb = __shfl_sync(0xffffffffu, n, b), tb = __shfl_sync(0xffffffffu, tiles, b);
        const int r0 = div_near(tb + C0 - 1, C0, i0), r1 = div_near(tb + C1 - 1, C1, i1);
        items0 += nb * r0;
        parts0 += r0 > 1 ? nb * r0 : 0;
        items1 += nb * r1;
        parts1 += r1 > 1 ? nb * r1 : 0;
    }
    float best = tree_cost(p, items0, parts0, C0);
    int best_s = s0;
    const float c1 = tree_cost(p, items1, parts1, C1);
    if (c1 < best) {
        best = c1;
        best_s = s1;
    }
    return tree_cheapest(best, best_s, longest);
}

// Walks the requests with a warp, 32 at a time, and finds the item with a given
// number (ascending from call to call).
template <bool SEL>
struct TreeWalk {
    int C, b0, item0, part0;         // block of 32 requests: its first, and the items and parts before it
    int items, parts;                // of the block
    int r0, n, ctx, tiles, runs;     // this lane's request
    int excl_item, excl_part;
    __device__ void load(const TreeParams& p) {
        const int b = b0 + (threadIdx.x & 31);
        r0 = n = ctx = tiles = 0;
        if (b < p.batch) {
            const TreeSeq s = tree_seq(p, b);
            r0 = s.r0;
            n = s.n;
            ctx = s.ctx;
            tiles = n > 0 ? tree_tiles<SEL>(p, s) : 0;
        }
    }
    __device__ void count() {  // items and parts of the loaded block
        runs = (tiles + C - 1) / C;
        const int it = n * runs, pt = runs > 1 ? it : 0;
        int si = it, sp = pt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, si, o), y = __shfl_up_sync(0xffffffffu, sp, o);
            if ((threadIdx.x & 31) >= o) {
                si += x;
                sp += y;
            }
        }
        excl_item = si - it;
        excl_part = sp - pt;
        items = __shfl_sync(0xffffffffu, si, 31);
        parts = __shfl_sync(0xffffffffu, sp, 31);
    }
    __device__ void start(const TreeParams& p) {
        b0 = item0 = part0 = 0;
        load(p);
    }
    __device__ bool next_block(const TreeParams& p) {
        item0 += items;
        part0 += parts;
        b0 += 32;
        if (b0 >= p.batch) return false;
        load(p);
        count();
        return true;
    }
};
struct TreeItem {
    int b, r0, n, ctx, node, tile0, tiles;  // tiles of this item
    int part;                               // -1: the node's only item
};
template <bool SEL>
__device__ bool tree_item(const TreeParams& p, TreeWalk<SEL>& w, int item, TreeItem& t) {
    while (item >= w.item0 + w.items)
        if (!w.next_block(p)) return false;
    const unsigned here = __ballot_sync(0xffffffffu, w.item0 + w.excl_item <= item && w.n * w.runs > 0);
    const int l = 31 - __clz((int)here);  // the last request that starts at or before the item
    const int local = item - (w.item0 + __shfl_sync(0xffffffffu, w.excl_item, l));
    t.b = w.b0 + l;
    t.r0 = __shfl_sync(0xffffffffu, w.r0, l);
    t.n = __shfl_sync(0xffffffffu, w.n, l);
    t.ctx = __shfl_sync(0xffffffffu, w.ctx, l);
    const int all = __shfl_sync(0xffffffffu, w.tiles, l), runs = __shfl_sync(0xffffffffu, w.runs, l);
    const int run = local / t.n;  // the request's nodes side by side on one run of keys
    t.node = local - run * t.n;
    t.tile0 = run * w.C;
    t.tiles = min(w.C, all - t.tile0);
    t.part = runs > 1 ? w.part0 + __shfl_sync(0xffffffffu, w.excl_part, l) + t.node * runs + run : -1;
    return true;
}

template <bool SEL>
__global__ void __launch_bounds__(TaLayout<SEL>::THREADS, 1)
    tree_attn_kernel(const TreeParams p, const __grid_constant__ TreeMaps tm) {
    using L = TaLayout<SEL>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sK = smem_u32(smem), sP = smem_u32(smem + L::OFF_P);
    int4* items = reinterpret_cast<int4*>(smem + L::OFF_ITEM);  // (row or -1 = no more, tiles, part, unused)
    unsigned long long* see_sh = reinterpret_cast<unsigned long long*>(smem + L::OFF_SEE);
    int* rows_sh = reinterpret_cast<int*>(smem + L::OFF_ROWS);
    uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
    uint64_t* kfree = kfull + TA_NBUF;
    uint64_t* sfull = kfree + TA_NBUF;
    uint64_t* sfree = sfull + 2;
    uint64_t* pready = sfree + 2;
    uint64_t* pvdone = pready + 1;
    uint64_t* qtmem = pvdone + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
    volatile int* go = reinterpret_cast<volatile int*>(tmem_slot + 1);  // [2], by ring entry parity
    int* chosen = reinterpret_cast<int*>(tmem_slot + 3);
    volatile int* info = reinterpret_cast<volatile int*>(tmem_slot + 4);  // lists: the item, for all gather threads

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int b = 0; b < TA_NBUF; ++b) {
            mbar_init(kfull + b, SEL ? L::LOADERS : 1);
            mbar_init(kfree + b, 1);  // the P.V commit; the MMA warp for a query entry
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(sfull + b, 1);
            mbar_init(sfree + b, 128);
        }
        mbar_init(pready, 128);
        mbar_init(pvdone, 1);
        mbar_init(qtmem, 128);
        fence_mbar_init();
    }
    if (warp == L::MMA_WARP) tmem_alloc(tmem_slot, 512);
    if (warp == 4 && lane < (SEL ? 1 : 3))
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane == 0 ? &tm.q : lane == 1 ? &tm.ckv : &tm.krot)) : "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_trigger();
    if (p.batch > 32) {
        tree_schedule<SEL>(p, smem, chosen);
        // the schedule's scratch becomes key tiles: order its generic accesses before TMA writes
        fence_proxy_async_smem();
        __syncthreads();
    }

    if (warp >= 4 && warp < L::MMA_WARP) {
        // ---------------- producer ----------------
        const int g = tid - 128;
        TreeWalk<SEL> walk;
        if (warp == 4) {
            walk.start(p);
            walk.C = p.batch > 32 ? *chosen : tree_schedule_warp(p, walk.n, walk.tiles);
            walk.count();
            if (blockIdx.x == gridDim.x - 1) {  // the parts of every node, for the merge
                for (int r = lane; r < p.n_nodes; r += 32) p.node_tab[r] = make_int2(0, 0);
                __syncwarp();
                TreeWalk<SEL> w = walk;
                do {
                    if (w.runs > 1)
                        for (int j = 0; j < w.n; ++j) p.node_tab[w.r0 + j] = make_int2(w.part0 + w.excl_part + j * w.runs, w.runs);
                } while (w.next_block(p));
            }
        }
        int e = 0;  // ring entries issued
        bool ok = true;
        // Waits for ring entry e's space; all loader threads get the same answer.
        auto acquire = [&]() -> bool {
            const int b = e % TA_NBUF;
            if constexpr (SEL) {
                if (g == 0) go[e & 1] = e < TA_NBUF || mbar_wait_fast(kfree + b, (uint32_t)(e / TA_NBUF - 1) & 1u, 50) ? 1 : 0;
                asm volatile("bar.sync 2, %0;" ::"n"(L::LOADERS) : "memory");
                return go[e & 1] != 0;  // rewritten two entries on, behind the barrier in between
            } else {
                return e < TA_NBUF || mbar_wait_fast(kfree + b, (uint32_t)(e / TA_NBUF - 1) & 1u, 50);
            }
        };
        int pend = -1;  // lists: the tile whose copies are in flight
        auto flush = [&]() {
            if constexpr (SEL) {
                if (pend >= 0) {
                    cp_async_wait<0>();
                    fence_proxy_async_smem();
                    mbar_arrive(kfull + pend);
                    pend = -1;
                }
            }
        };
        for (int item = blockIdx.x;; item += gridDim.x) {
            TreeItem t;
            bool more = true;
            if (warp == 4) more = tree_item<SEL>(p, walk, item, t);
            if constexpr (SEL) {
                flush();
                if (warp == 4 && lane == 0) {
                    info[0] = more ? 1 : 0;
                    if (more) {
                        const int left = tree_list_n(p, t.r0 + t.node) - t.tile0 * TA_TILE;  // of the list, from this item on
                        info[1] = t.b;
                        info[2] = t.r0 + t.node;
                        info[3] = t.ctx;
                        info[4] = t.n;
                        info[5] = t.tile0 * TA_TILE;
                        info[6] = max(0, min(left, t.tiles * TA_TILE));
                    }
                }
            }
            if (!(ok = acquire())) break;  // also orders info[] for the gather threads
            const int b = e % TA_NBUF;
            if constexpr (SEL) more = info[0] != 0;
            const int row = SEL ? info[2] : t.r0 + t.node;
            const int n_keys = SEL ? info[6] : 0;
            const int n_tiles = SEL ? (n_keys + TA_TILE - 1) / TA_TILE : t.tiles;
            if (g == 0) items[b] = make_int4(more ? row : -1, n_tiles, t.part, 0);
            if (!more) {
                if (SEL || lane == 0) mbar_arrive(kfull + b);
                ++e;
                break;
            }
            // the query, 64 heads x 576: nine boxes
            if (g == 0) {
                mbar_expect_tx(kfull + b, L::TILE);
                for (int c = 0; c < AT_CHUNKS; ++c)
                    tma_load2d(sK + b * L::TILE + c * L::CHUNK, &tm.q, c * 64, row * AT_H, kfull + b);
            } else if (SEL) {
                mbar_arrive(kfull + b);
            }
            ++e;
            if constexpr (!SEL) {
                const int R = p.box_rows, nbox = TA_TILE / R;
                const int* table = p.table + (long long)t.b * p.table_stride;
                // this lane's box of a tile: its page, loaded a tile ahead
                int pos = t.tile0 * TA_TILE + lane * R, page = 0;
                if (lane < nbox && pos < t.ctx + t.n) page = __ldg(table + pos / p.page_size);
                const unsigned long long see = tree_mask_of(p, t.r0, t.n, t.node);
                for (int i = 0; i < n_tiles; ++i, ++e) {
                    const int pos0 = (t.tile0 + i) * TA_TILE, bb = e % TA_NBUF;
                    // its first slot, -1 past the request's rows or outside the pool
                    int slot = -1;
                    bool bad = false;
                    if (lane < nbox && pos < t.ctx + t.n) {
                        bad = page < 0 || page >= p.n_pages;
                        if (bad) set_error(ERRC_BOUNDS, 46);
                        else slot = page * p.page_size + pos % p.page_size;
                    }
                    pos += TA_TILE;
                    if (lane < nbox && pos < t.ctx + t.n && i + 1 < n_tiles) page = __ldg(table + pos / p.page_size);
                    const int have = __popc(__ballot_sync(0xffffffffu, slot >= 0));
                    const unsigned lost = __ballot_sync(0xffffffffu, bad);
                    if (!(ok = acquire())) break;
                    if (lane == 0) {
                        const int k = pos0 - t.ctx;  // first key as a node number
                        unsigned long long v = k >= 64 ? 0ull : k >= 0 ? see >> k : k <= -64 ? ~0ull : (see << -k) | ((1ull << -k) - 1);
                        if (lost)
                            for (int j = 0; j < nbox; ++j)
                                if ((lost >> j) & 1) v &= ~((R >= 64 ? ~0ull : (1ull << R) - 1) << (j * R));
                        see_sh[bb] = v;
                        if (have > 0) mbar_expect_tx(kfull + bb, (uint32_t)have * R * 128 * AT_CHUNKS);
                        else mbar_arrive(kfull + bb);
                    }
                    __syncwarp();
                    const uint32_t tile = sK + bb * L::TILE;
                    for (int x0 = 0; x0 < nbox * AT_CHUNKS; x0 += 32) {
                        const int x = x0 + lane, j = x / AT_CHUNKS, c = x - j * AT_CHUNKS;
                        const int y = __shfl_sync(0xffffffffu, slot, j & 31);
                        if (x < nbox * AT_CHUNKS && y >= 0)
                            tma_load2d(tile + c * L::CHUNK + j * R * 128, c < 8 ? &tm.ckv : &tm.krot, c < 8 ? c * 64 : 0, y, kfull + bb);
                    }
                }
            } else {
                const int qb = info[1], ctx = info[3], n = info[4];
                if (warp == 4) {
                    const unsigned long long see = tree_mask_of(p, t.r0, t.n, t.node);
                    if (lane == 0) {
                        info[7] = (int)(unsigned)see;
                        info[8] = (int)(unsigned)(see >> 32);
                    }
                }
                const int* list = p.sel + (long long)row * p.sel_stride + info[5];
                const int* table = p.table + (long long)qb * p.table_stride;
                // the slot of this thread's key of tile i (threads 0-63), -1 when the row does not see it
                asm volatile("bar.sync 2, %0;" ::"n"(L::LOADERS) : "memory");  // info[0..6] is read, info[7..8] written
                const unsigned long long mine = (unsigned)info[7] | ((unsigned long long)(unsigned)info[8] << 32);
                auto slot_of = [&](int i) -> int {
                    const int k = i * TA_TILE + g;
                    if (g >= TA_TILE || k >= n_keys) return -1;
                    const int pos = __ldg(list + k);
                    if (pos < 0 || pos >= ctx + n || (pos >= ctx && !((mine >> (pos - ctx)) & 1))) return -1;
                    return page_slot(table, p.page_size, p.n_pages, pos, 46);
                };
                int next = slot_of(0);
                for (int i = 0; i < n_tiles; ++i, ++e) {
                    const int bb = e % TA_NBUF;
                    if (g < TA_TILE) {
                        // rows_sh and see_sh of this entry were last read three entries ago, behind acquire's barrier
                        const unsigned bits = __ballot_sync(0xffffffffu, next >= 0);
                        rows_sh[bb * TA_TILE + g] = next;
                        next = slot_of(i + 1);
                        if (!(ok = acquire())) break;
                        if (lane == 0) reinterpret_cast<volatile unsigned*>(see_sh + bb)[g >> 5] = bits;
                    } else if (!(ok = acquire())) {
                        break;
                    }
                    const uint32_t tile = sK + bb * L::TILE;
#pragma unroll 3
                    for (int k2 = 0; k2 < AT_CHUNKS * TA_TILE * 8 / L::LOADERS; ++k2) {  // 18 pieces of 16 B a thread
                        const int pid = k2 * L::LOADERS + g;
                        const int c = pid / (TA_TILE * 8), rem = pid % (TA_TILE * 8);
                        const int j = rem >> 3, seg = rem & 7;
                        const int sl = rows_sh[bb * TA_TILE + j];
                        const __nv_bfloat16* src = c < 8 ? p.c_kv + (long long)max(sl, 0) * p.ckv_row + c * 64 + seg * 8
                                                         : p.k_rot + (long long)max(sl, 0) * p.krot_row + seg * 8;
                        cp_async16(tile + c * L::CHUNK + sw128_off(j, seg), src, sl < 0 ? 0u : 16u);
                    }
                    cp_async_commit();
                    if (pend >= 0) {
                        cp_async_wait<1>();
                        fence_proxy_async_smem();
                        mbar_arrive(kfull + pend);
                    }
                    pend = bb;
                }
            }
            if (!ok) break;
        }
        if (SEL) {
            cp_async_wait<0>();
            if (ok) flush();
        }
        if (!ok && g == 0)  // copies in flight must land before the CTA leaves
            for (int k = max(0, e - TA_NBUF); k < e; ++k) mbar_wait_fast(kfull + k % TA_NBUF, (uint32_t)(k / TA_NBUF) & 1u, 51);
    } else if (warp == L::MMA_WARP) {
        // ---------------- MMA ----------------
        const uint32_t tq = tmem + (16u << 16) + PF_TM_Q;
        int e = 0, gt = 0;  // ring entries and key tiles taken
        auto issue_qk = [&](int entry, int g_) -> bool {
            const int b = entry % TA_NBUF, s = g_ & 1;
            if (!mbar_wait_fast(kfull + b, (uint32_t)(entry / TA_NBUF) & 1u, 52)) return false;
            if (g_ >= 2 && !mbar_wait_fast(sfree + s, (uint32_t)((g_ >> 1) - 1) & 1u, 53)) return false;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t d = tmem + (16u << 16) + (uint32_t)(s * TA_TILE);
                const uint64_t k0 = desc_sw128(sK + b * L::TILE, 16, 1024);
#pragma unroll
                for (int c = 0; c < AT_CHUNKS; ++c) {
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)  // descriptors step in 16-byte units
                        mma_bf16_ts(d, tq + (uint32_t)(c * 32 + kk * 8), k0 + ((c * L::CHUNK + kk * 32) >> 4), L::IDESC_QK,
                                    (c | kk) != 0 ? 1u : 0u);
                }
                mma_commit(sfull + s);
            }
            __syncwarp();
            return true;
        };
        auto issue_pv = [&](int entry, int g_, bool first) -> bool {
            const int b = entry % TA_NBUF;
            if (!mbar_wait_fast(pready, (uint32_t)g_ & 1u, 54)) return false;
            tc_fence_after();
            if (elect_one()) {
                const uint64_t p0 = desc_sw128(sP, 16, 1024), v0 = desc_sw128(sK + b * L::TILE, L::CHUNK, 1024);
#pragma unroll
                for (int ks = 0; ks < TA_TILE / 16; ++ks) {
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                        mma_bf16(tmem + (uint32_t)(half * 256), p0 + ks * 2, v0 + ((4 * half * L::CHUNK + ks * 2048) >> 4),
                                 L::IDESC_PV, (!first || ks > 0) ? 1u : 0u);
                }
                mma_commit(kfree + b);
                mma_commit(pvdone);
            }
            __syncwarp();
            return true;
        };
        bool ok = true;
        for (int it = 0; ok; ++it) {
            const int qb = e % TA_NBUF;
            if (!(ok = mbar_wait_fast(kfull + qb, (uint32_t)(e / TA_NBUF) & 1u, 55))) break;
            const int4 t = items[qb];
            if (t.x < 0) break;
            if (!(ok = mbar_wait_fast(qtmem, (uint32_t)it & 1u, 56))) break;  // the query is in tensor memory
            if (elect_one()) mbar_arrive(kfree + qb);
            ++e;
            const int n = t.y;
            if (n > 0) ok = issue_qk(e, gt);
            for (int i = 0; ok && i < n; ++i) {
                if (i + 1 < n) ok = issue_qk(e + i + 1, gt + i + 1);
                if (ok) ok = issue_pv(e + i, gt + i, i == 0);
            }
            e += n;
            gt += n;
        }
    } else {
        // ---------------- softmax and output (warps 0-3) ----------------
        const int h = 16 * warp + (lane & 15);
        const bool hi_half = lane >= 16;
        const uint32_t lane_o = (uint32_t)(32 * warp) << 16, lane_s = (uint32_t)(32 * warp + 16) << 16;
        int e = 0, gt = 0;
        int out_row = -1, out_part = -1;  // the item whose output is still in tensor memory
        float m_run = -INFINITY, l_run = 0.f;
        bool ok = true;
        while (ok) {
            const int qb = e % TA_NBUF;
            if (!(ok = mbar_wait_fast(kfull + qb, (uint32_t)(e / TA_NBUF) & 1u, 57))) break;
            const int4 t = items[qb];
            if (t.x >= 0) {
                // The next query into tensor memory: every QK of the item before is done (its scores were read).
                const uint32_t src0 = sK + qb * L::TILE + (uint32_t)h * 128u;
#pragma unroll 3
                for (int k = 0; k < 9; ++k) {
                    const int e0 = 32 * k + (hi_half ? 288 : 0);
                    const uint32_t src = src0 + (uint32_t)(e0 >> 6) * L::CHUNK;
                    const int seg0 = (e0 & 63) >> 3;
                    uint32_t v[16];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const uint4 x = lds_v4(src + ((((uint32_t)(seg0 + q)) ^ (uint32_t)h) & 7u) * 16u);
                        v[4 * q] = x.x;
                        v[4 * q + 1] = x.y;
                        v[4 * q + 2] = x.z;
                        v[4 * q + 3] = x.w;
                    }
                    tmem_st16x2_16u<144>(tmem + lane_s + PF_TM_Q + (uint32_t)(16 * k), v);
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(qtmem);
            }
            ++e;
            if (out_row >= 0) {
                // Output of the item before: O / l, under the next item's first QK.
                if (gt > 0 && !(ok = mbar_wait_fast(pvdone, (uint32_t)(gt - 1) & 1u, 58))) break;
                tc_fence_after();
                const bool any = l_run != 0.f;  // (NaN counts: it reaches the result)
                const float inv = any ? 1.f / l_run : 0.f;
                const float lse = any ? (m_run + log2f(l_run)) * 0.69314718055994531f : -INFINITY;
                if (!hi_half) {
                    if (out_part >= 0) p.lse_part[(long long)out_part * AT_H + h] = lse;
                    else if (p.lse) p.lse[(long long)out_row * AT_H + h] = lse;
                }
                // A warp's 16 heads pass through its own 2 KB of P's space (P.V is done with it), 128 bytes
                // a head at a time, so that each store instruction writes four whole 128-byte lines: an item's
                // output takes about 2,500 cycles instead of 11,000 with every thread storing its own columns.
                const long long at = (out_part >= 0 ? (long long)out_part : (long long)out_row) * AT_H + 16 * warp;
                const uint32_t mine = sP + (uint32_t)h * 128u, base = sP + (uint32_t)(16 * warp) * 128u;
                const bool narrow = out_part < 0 && p.ctx_bf16;
                char* out = narrow ? reinterpret_cast<char*>(static_cast<__nv_bfloat16*>(p.ctx) + at * AT_DV)
                                   : reinterpret_cast<char*>((out_part >= 0 ? p.o_part : static_cast<float*>(p.ctx)) + at * AT_DV);
                const int row_bytes = narrow ? AT_DV * 2 : AT_DV * 4;
                auto store = [&](int byte0) {  // the staged 16 x 128 bytes to columns from byte0 on
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int r = 4 * k + (lane >> 3), seg = lane & 7;
                        const uint4 x = lds_v4(base + (uint32_t)r * 128u + (uint32_t)((seg ^ r) & 7) * 16u);
                        *reinterpret_cast<uint4*>(out + (long long)r * row_bytes + byte0 + seg * 16) = x;
                    }
                    __syncwarp();
                };
                if (narrow) {
#pragma unroll 1
                    for (int c = 0; c < AT_DV; c += 64) {
                        float ov[32];
                        tmem_ld16x2_32<32>(tmem + lane_o + (uint32_t)c, ov);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t w[4];
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const float a = ov[8 * k + 2 * x], b = ov[8 * k + 2 * x + 1];
                                const __nv_bfloat162 b2 = __floats2bfloat162_rn(any ? a * inv : 0.f, any ? b * inv : 0.f);
                                w[x] = *reinterpret_cast<const uint32_t*>(&b2);
                            }
                            sts_v4(mine + (uint32_t)(((hi_half ? 4 : 0) + k) ^ (h & 7)) * 16u, make_uint4(w[0], w[1], w[2], w[3]));
                        }
                        store(c * 2);
                    }
                } else {
#pragma unroll 1
                    for (int c = 0; c < AT_DV; c += 32) {
                        float ov[16];
                        tmem_ld16x2_16<16>(tmem + lane_o + (uint32_t)c, ov);
#pragma unroll
                        for (int k = 0; k < 16; ++k) ov[k] = any ? ov[k] * inv : 0.f;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            sts_v4(mine + (uint32_t)(((hi_half ? 4 : 0) + k) ^ (h & 7)) * 16u,
                                   make_uint4(__float_as_uint(ov[4 * k]), __float_as_uint(ov[4 * k + 1]),
                                              __float_as_uint(ov[4 * k + 2]), __float_as_uint(ov[4 * k + 3])));
                        store(c * 4);
                    }
                }
                tc_fence_before();  // these reads come before the next P.V (ordered by pready)
            }
            if (t.x < 0) break;
            out_row = t.x;
            out_part = t.z;
            m_run = -INFINITY;
            l_run = 0.f;
            for (int i = 0; i < t.y && ok; ++i, ++e, ++gt) {
                const int s = gt & 1, b = e % TA_NBUF;
                if (!(ok = mbar_wait_fast(kfull + b, (uint32_t)(e / TA_NBUF) & 1u, 59))) break;  // orders see_sh
                const unsigned long long see = see_sh[b];
                if (!(ok = mbar_wait_fast(sfull + s, (uint32_t)(gt >> 1) & 1u, 60))) break;
                tc_fence_after();
                float sv[32];
                tmem_ld16x2_32<32>(tmem + lane_s + (uint32_t)(s * TA_TILE), sv);
                tc_fence_before();
                mbar_arrive(sfree + s);
                float tmax = -INFINITY;
                if (see == ~0ull) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        sv[j] *= p.scale_log2;
                        tmax = fmaxf(tmax, sv[j]);
                    }
                } else {
                    const unsigned bits = (unsigned)(see >> (hi_half ? 32 : 0));
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        sv[j] = (bits >> j) & 1u ? sv[j] * p.scale_log2 : -INFINITY;
                        tmax = fmaxf(tmax, sv[j]);
                    }
                    if constexpr (!SEL) {
                        // An unseen row may hold anything (0 x NaN is NaN): its values become zeros
                        // before P.V reads them. Lists load zeros for such rows.
                        for (int j = warp; j < TA_TILE; j += 4) {
                            if ((see >> j) & 1) continue;
                            const uint32_t dst = sK + b * L::TILE + (uint32_t)(lane >> 3) * L::CHUNK + (uint32_t)j * 128u + (uint32_t)(lane & 7) * 16u;
                            sts_v4(dst, make_uint4(0, 0, 0, 0));
                            sts_v4(dst + 4 * L::CHUNK, make_uint4(0, 0, 0, 0));
                        }
                    }
                }
                tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, 16));
                const float m_new = (m_run == -INFINITY || tmax > m_run + PF_RESCALE_LOG2) ? tmax : m_run;
                const float m_use = m_new == -INFINITY ? 0.f : m_new;  // nothing seen yet: every e^s is 0
                const float alpha = m_run == -INFINITY ? 0.f : exp2f(m_run - m_new);
                if (gt >= 1 && !(ok = mbar_wait_fast(pvdone, (uint32_t)(gt - 1) & 1u, 61))) break;
                tc_fence_after();
                float sum = 0.f;
                const uint32_t prow = sP + (uint32_t)h * 128u;
#pragma unroll
                for (int c4 = 0; c4 < 4; ++c4) {
                    uint32_t w4[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int j = c4 * 8 + x * 2;
                        const float e0 = exp2f(sv[j] - m_use), e1 = exp2f(sv[j + 1] - m_use);
                        const __nv_bfloat162 b2 = __floats2bfloat162_rn(e0, e1);
                        w4[x] = *reinterpret_cast<const uint32_t*>(&b2);
                        sum += e0 + e1;
                    }
                    const uint32_t chunk = (uint32_t)((hi_half ? 4 : 0) + c4);
                    sts_v4(prow + (((chunk ^ (uint32_t)h) & 7u) << 4), make_uint4(w4[0], w4[1], w4[2], w4[3]));
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                l_run = l_run * alpha + sum;
                const bool resc = i > 0 && m_new != m_run;
                m_run = m_new;
                if (__any_sync(0xffffffffu, resc)) {
#pragma unroll 1
                    for (int c = 0; c < 256; c += 32) {
                        float ov[32];
                        tmem_ld16x2_32<256>(tmem + lane_o + (uint32_t)c, ov);
                        const float f = resc ? alpha : 1.f;
#pragma unroll
                        for (int x = 0; x < 32; ++x) ov[x] *= f;
                        tmem_st16x2_32<256>(tmem + lane_o + (uint32_t)c, ov);
                    }
                    tmem_wait_st();
                }
                fence_proxy_async_smem();  // P (and zeroed rows) are read by the tensor cores
                tc_fence_before();
                mbar_arrive(pready);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == L::MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the partials of the nodes that were cut: ctx = sum_s e^(lse_s - L) o_s,
// L = log sum_s e^lse_s. A block owns one (head, 128 columns) of every k-th node;
// its four warps take the parts in turn, eight loads in flight each, and add
// their sums in warp order.
constexpr int TM_UNITS = AT_H * (AT_DV / 128);
__global__ void __launch_bounds__(128) tree_merge_kernel(const TreeParams p) {
    pdl_wait();
    pdl_trigger();
    __shared__ float w_sh[TA_MAX_SPLIT];
    __shared__ float4 part_sh[3][32];
    const int lane = threadIdx.x & 31, wi = threadIdx.x >> 5;
    const int h = (blockIdx.x % TM_UNITS) >> 2, q = blockIdx.x & 3, step = gridDim.x / TM_UNITS;
    for (int r0 = blockIdx.x / TM_UNITS; r0 < p.n_nodes; r0 += 32 * step) {
        const int rl = r0 + lane * step;
        const int2 mine = rl < p.n_nodes ? p.node_tab[rl] : make_int2(0, 0);
        for (unsigned cut = __ballot_sync(0xffffffffu, mine.y > 1); cut; cut &= cut - 1) {
            const int l = __ffs(cut) - 1, r = r0 + l * step;
            const int part0 = __shfl_sync(0xffffffffu, mine.x, l), n = __shfl_sync(0xffffffffu, mine.y, l);
            // the first round of partials is under way while the weights are worked out
            const float* src = p.o_part + ((long long)part0 * AT_H + h) * AT_DV + q * 128 + lane * 4;
            float4 v[8];
            auto fetch = [&](int s0) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (s0 + 4 * k < n) v[k] = *reinterpret_cast<const float4*>(src + (long long)(s0 + 4 * k) * (AT_H * AT_DV));
            };
            fetch(wi);
            float ls[TA_MAX_SPLIT / 32], M = -INFINITY, W = 0.f;
#pragma unroll
            for (int k = 0; k < TA_MAX_SPLIT / 32; ++k) {
                const int s = lane + 32 * k;
                ls[k] = s < n ? p.lse_part[(long long)(part0 + s) * AT_H + h] : -INFINITY;
                M = fmaxf(M, ls[k]);
            }
            for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
            const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int k = 0; k < TA_MAX_SPLIT / 32; ++k) {
                ls[k] = exp2f((ls[k] - Mu) * 1.4426950408889634f);
                W += ls[k];
            }
            for (int o = 16; o > 0; o >>= 1) W += __shfl_xor_sync(0xffffffffu, W, o);
            const float inv = W != 0.f ? 1.f / W : 0.f;
            if (wi == 0) {
#pragma unroll
                for (int k = 0; k < TA_MAX_SPLIT / 32; ++k)
                    if (lane + 32 * k < n) w_sh[lane + 32 * k] = ls[k] * inv;
            }
            __syncthreads();
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int s0 = wi; s0 < n; s0 += 32) {
                if (s0 > wi) fetch(s0);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (s0 + 4 * k >= n) continue;
                    const float w = w_sh[s0 + 4 * k];
                    acc.x = fmaf(w, v[k].x, acc.x);
                    acc.y = fmaf(w, v[k].y, acc.y);
                    acc.z = fmaf(w, v[k].z, acc.z);
                    acc.w = fmaf(w, v[k].w, acc.w);
                }
            }
            if (wi > 0) part_sh[wi - 1][lane] = acc;
            __syncthreads();
            if (wi == 0) {
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    const float4 o = part_sh[k][lane];
                    acc.x += o.x;
                    acc.y += o.y;
                    acc.z += o.z;
                    acc.w += o.w;
                }
                const long long at = ((long long)r * AT_H + h) * AT_DV + q * 128 + lane * 4;
                if (p.ctx_bf16) {
                    const __nv_bfloat162 a = __floats2bfloat162_rn(acc.x, acc.y), c = __floats2bfloat162_rn(acc.z, acc.w);
                    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.ctx) + at) =
                        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&c));
                } else {
                    *reinterpret_cast<float4*>(static_cast<float*>(p.ctx) + at) = acc;
                }
                if (q == 0 && lane == 0 && p.lse) p.lse[(long long)r * AT_H + h] = W != 0.f ? M + logf(W) : -INFINITY;
            }
            __syncthreads();  // shared arrays are reused
        }
    }
}

}  // namespace wl
