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
//   loaders   the item's query (one ring entry), then its key tiles. Dense: one
//             warp issues TMA boxes, one per page part and 64 columns, so the
//             128B-swizzled tile needs no threads. Lists: 8 warps gather rows with
//             16-byte cp.async (80 bytes a cycle and SM from L2; TMA gather4 of four
//             rows x 64 columns at best 35), each half of a tile reported by
//             its copies' own arrival. A tile comes and goes in two
//             halves (columns 0-255 and the roped ones; columns 256-511): QK
//             starts on the first while the second is on its way, and P.V gives
//             the first back while it reads the second.
//   MMA       QK of tile i + 1 (A = the query in tensor memory), then P.V of
//             tile i: the softmax of tile i runs under QK of tile i + 1.
//   softmax   4 warps, two threads a head: query into tensor memory, mask,
//             running maximum and sum, P (bf16) to shared memory, lazy rescale
//             of O, and the item's output, written while the MMA warp is
//             already at QK of the next item.
// Tensor memory as in mla_attn64.cuh: O in lanes 0-15 of each quarter, S tiles
// and the query in lanes 16-31.
// Bound: with one node a request by HBM (148 requests x 8K keys 229 us, 6.1 TB/s; 6.7 in the
// middle, 1.63 us a tile), with more nodes by the MMAs, which with M = 64 run at half rate
// (2,176 cycles a tile), and in small calls by latency: 1 node x 1K keys 13.5 us, of
// which the schedule 1.1, query and first tile 2.5, output 3, join 2.5.
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
    int sel_n;  // entries of a list, or with sel_n_dev at most
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
    CUtensorMap wide;  // tiles inside a page: the latent rows as {64, slots, 8 column chunks}, box {64, 64, 4}
    CUtensorMap part;  // the partials {512, 64 parts} fp32, box {32, 16}
    CUtensorMap out;   // ctx {512, 64 n_nodes}, box of 128 bytes x 16 rows
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
constexpr int TA_LOAD_WARP = 4;       // warps 0-3 softmax, then the loaders (dense 1 warp, lists 8), then MMA
constexpr int TA_SCHED_THREADS = 192;
constexpr int TA_MAX_BATCH = 16384;   // the schedule's table of a CTA (8 bytes a request) fits the key tiles' space
constexpr int TA_CANDS = 64;          // candidate splits: 1, 1.25, .. 8.75, 9 .. 24, then 32.5, 41, .. 160 (3 x TA_CANDS threads sum up)
constexpr int TA_MAX_SPLIT = 160;
// Costs in key tiles of one CTA (1.25 us): an item's query, output and pipeline fill; a partial written and
// joined, and one beyond a round of the CTAs. Fitted on 35 workloads of 1 to 230 nodes, within 2 % over a wide
// range of prices for most. Where it shows, at these and at (4, .04, .08): 3 x 3 nodes x 2K keys 17.4 / 19.1 us,
// 64 x 2 x 4K 81.8 / 85.4, lists 1 x 16 x 2048 22.5 / 24.0; lower ones cut too much (1 x 1 x 8K 17.6, 20.4 at .01).
struct TreePrice {
    float item, part, more;
};
constexpr TreePrice TA_PRICE = {4.f, 0.02f, 0.06f};

template <bool SEL>
struct TaLayout {
    static constexpr int LOADERS = SEL ? 256 : 32;
    static constexpr int THREADS = 128 + LOADERS + 32;
    static constexpr int MMA_WARP = (128 + LOADERS) / 32;
    static constexpr uint32_t CHUNK = TA_TILE * 128;
    static constexpr uint32_t TILE = AT_CHUNKS * CHUNK;
    static constexpr uint32_t OFF_P = TA_NBUF * TILE;
    static constexpr uint32_t OFF_ITEM = OFF_P + AT_H * 128;           // int4 per ring entry
    static constexpr uint32_t OFF_SEE = OFF_ITEM + TA_NBUF * 16;       // valid-key bits per ring entry
    static constexpr uint32_t OFF_ROWS = OFF_SEE + TA_NBUF * 8 + 8;    // gathered slots (lists only)
    static constexpr uint32_t OFF_BAR = OFF_ROWS + (SEL ? TA_NBUF * TA_TILE * 4 : 0);
    static constexpr int N_BARS = 4 * TA_NBUF + 2 + 3;  // kfull[3][2], kfree[3][2], sfull[2], pready, pvdone, qtmem
    static constexpr uint32_t OFF_MISC = OFF_BAR + N_BARS * 8;         // tensor-memory slot, longest request, go flags, item
    static constexpr uint32_t BYTES = OFF_MISC + 64 + 1024;
    static constexpr uint32_t IDESC_QK = idesc_bf16(64, TA_TILE, 0, 0);
    static constexpr uint32_t IDESC_PV = idesc_bf16(64, 256, 0, 1);
};
static_assert(TaLayout<true>::BYTES <= 232448 && TaLayout<false>::BYTES <= 232448, "one CTA per SM");
static_assert(TA_MAX_BATCH * 8 <= TaLayout<false>::OFF_P, "schedule table");

// Keys of a row's list (clamped to the list's room).
__device__ __forceinline__ int tree_list_n(const TreeParams& p, int r) {
    return p.sel_n_dev ? max(0, min(__ldg(p.sel_n_dev + r), p.sel_n)) : p.sel_n;
}
// Key tiles of a request's nodes (at least one).
template <bool SEL>
__device__ __forceinline__ int tree_tiles(const TreeParams& p, const TreeSeq& s) {
    if (!SEL) return (s.ctx + s.n + TA_TILE - 1) / TA_TILE;
    int m = 1;
    for (int j = 0; j < s.n; ++j) m = max(m, tree_list_n(p, s.r0 + j));
    return (m + TA_TILE - 1) / TA_TILE;
}

// x / c for a quotient far below 2^22, by a reciprocal and one correction.
__device__ __forceinline__ int div_near(int x, int c, float inv) {
    int q = (int)((float)x * inv);
    const int r = x - q * c;
    q += r >= c ? 1 : 0;
    return r < 0 ? q - 1 : q;
}

// Tiles per item, from the lengths: a request's nodes are cut into the fewest
// equal runs of at most C tiles, with C = ceil(longest / s) for 64 values of s.
// The CTAs take the items in order, forth and back (item_of); with the longest
// runs first (up to 32 requests are sorted, by their tiles for the choice and by
// their runs' for the walk: 4 requests, 177 nodes x 10K 244 -> 201 us, 25, 512 x 1.5K
// 131 -> 116) full rounds balance out, so a choice costs the mean of its full
// rounds plus the longest item of the last one, plus a write and a read per
// partial: within 5 % of the best of all choices on 26 drawn workloads. The cheapest that fits the workspace is taken, the fewest
// runs among equals. Every CTA computes the same choice, all its threads sharing
// the sums (64 candidates x 3 thirds of the requests); the producer warp, which
// alone needs it, ends with C. tab: (nodes, tiles) of each request; acc: 4 x 3 x 64.
struct TreeCost {
    int items[3][TA_CANDS], parts[3][TA_CANDS];
    float sum[3][TA_CANDS], last[3][TA_CANDS];
};
// Runs of the longest request, and from them the tiles a run has at most. (Fractions: requests of other lengths
// then find a C between the whole parts of the longest; 32 requests of 4-8K: 130 runs of 26 tiles become 142 of 23.)
__device__ __forceinline__ float tree_candidate(int c) {
    return c < 32 ? 1.f + 0.25f * c : c < 48 ? 9.f + (c - 32) : 24.f + 8.5f * (c - 47);
}
// The tiles a run then has at most. Of eight and more requests none is cut into more than 24 runs with profit: there
// the lengths of the first 16 take the place of the last candidates, so that all longer ones are cut and no other
// (8 requests, 92 nodes x 16K 176 -> 167 us; 12, 479 x 17K 751 -> 725; 23, 311 x 6K 204 -> 197).
__device__ __forceinline__ int tree_run_tiles(int c, int longest, const int2* tab, int batch) {
    if (c >= 48 && batch >= 8)
        return max(max(1, tab[min(c - 48, batch - 1)].y), (longest + TA_MAX_SPLIT - 1) / TA_MAX_SPLIT);
    return max(1, (int)ceilf(__fdividef((float)longest, tree_candidate(c))));
}

template <int PER>  // nodes an item takes
__device__ __forceinline__ int tree_schedule(const TreeParams& p, const int2* tab, int longest, TreeCost* acc, int G, TreePrice price,
                                             int last_warp = TA_LOAD_WARP) {
    const int cand = threadIdx.x % TA_CANDS, grp = threadIdx.x / TA_CANDS;
    const int per = (p.batch + 2) / 3, b0 = min(grp * per, p.batch), b1 = min(b0 + per, p.batch);
    const int C = tree_run_tiles(cand, longest, tab, p.batch);
    const float inv = __fdividef(1.f, (float)C);
    const bool mine = threadIdx.x < TA_SCHED_THREADS;
    if (mine) {
        int items = 0, parts = 0;
#pragma unroll 2
        for (int b = b0; b < b1; ++b) {
            const int2 v = tab[b];
            const int r = div_near(v.y + C - 1, C, inv);
            items += (v.x + PER - 1) / PER * r;
            parts += r > 1 ? v.x * r : 0;
        }
        acc->items[grp][cand] = items;
        acc->parts[grp][cand] = parts;
    }
    __syncthreads();
    if (mine) {
        const int all = acc->items[0][cand] + acc->items[1][cand] + acc->items[2][cand], full = all / G * G;
        int seen = (grp > 0 ? acc->items[0][cand] : 0) + (grp > 1 ? acc->items[1][cand] : 0);
        float sum = 0.f, last = 0.f;
#pragma unroll 2
        for (int b = b0; b < b1; ++b) {
            const int2 v = tab[b];
            const int r = div_near(v.y + C - 1, C, inv), it = (v.x + PER - 1) / PER * r;
            if (it == 0) continue;
            const float len = __fdividef((float)v.y, (float)r) + price.item;
            sum += (float)max(0, min(it, full - seen)) * len;
            seen += it;
            if (seen > full) last = fmaxf(last, len);
        }
        acc->sum[grp][cand] = sum;
        acc->last[grp][cand] = last;
    }
    __syncthreads();
    if ((int)threadIdx.x / 32 != last_warp) return 0;
    const int lane = threadIdx.x & 31;
    float best = 3e38f;
    int best_c = max(1, longest);
    const float inv_g = __fdividef(1.f, (float)G);
#pragma unroll
    for (int c = lane; c < TA_CANDS; c += 32) {
        const int n_parts = acc->parts[0][c] + acc->parts[1][c] + acc->parts[2][c];
        const float cost = (acc->sum[0][c] + acc->sum[1][c] + acc->sum[2][c]) * inv_g +
                           fmaxf(fmaxf(acc->last[0][c], acc->last[1][c]), acc->last[2][c]) + (float)n_parts * price.part +
                           (float)max(0, n_parts - G * PER) * (price.more - price.part);
        if (n_parts <= p.parts_max && cost < best) {
            best = cost;
            best_c = tree_run_tiles(c, longest, tab, p.batch);
        }
    }
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) {
        const float c = __shfl_xor_sync(0xffffffffu, best, o);
        const int t = __shfl_xor_sync(0xffffffffu, best_c, o);
        if (c < best || (c == best && t > best_c)) {
            best = c;
            best_c = t;
        }
    }
    return best_c;
}
// Worker me's item of round k: the G workers take them forth and back.
__device__ __forceinline__ int item_of(int k, int me, int G) { return k * G + ((k & 1) ? G - 1 - me : me); }


// Walks the requests with a warp, 32 at a time, and finds the item with a given
// number (ascending from call to call).
template <bool SEL, int PER = 1>
struct TreeWalk {
    int C, b0, item0, part0;             // block of 32 requests: its first, and the items and parts before it
    int items, parts;                    // of the block
    int id, r0, n, ctx, tiles, len, runs;  // this lane's request
    int excl_item, excl_part;
    __device__ void load(const TreeParams& p) {
        id = b0 + (threadIdx.x & 31);
        r0 = n = ctx = tiles = 0;
        if (id < p.batch) {
            const TreeSeq s = tree_seq(p, id);
            r0 = s.r0;
            n = s.n;
            ctx = s.ctx;
            tiles = n > 0 ? tree_tiles<SEL>(p, s) : 0;
        }
    }
    __device__ void sort(int by) {  // largest first (a single block only), by a bitonic network
        const int lane = threadIdx.x & 31;
        unsigned key = (unsigned)by * 32u + (unsigned)(31 - lane);  // by < 2^26
#pragma unroll 1
        for (int k = 2; k <= 32; k <<= 1)
#pragma unroll 1
            for (int j = k >> 1; j > 0; j >>= 1) {
                const unsigned other = __shfl_xor_sync(0xffffffffu, key, j);
                const bool high = ((lane & j) == 0) == ((lane & k) == 0);  // keeps the larger
                key = high ? max(key, other) : min(key, other);
            }
        const int from = 31 - (int)(key & 31);
        id = __shfl_sync(0xffffffffu, id, from);
        r0 = __shfl_sync(0xffffffffu, r0, from);
        n = __shfl_sync(0xffffffffu, n, from);
        ctx = __shfl_sync(0xffffffffu, ctx, from);
        tiles = __shfl_sync(0xffffffffu, tiles, from);
    }
    __device__ int run_len() const {
        const int r = div_near(tiles + C - 1, C, __fdividef(1.f, (float)C));
        return r > 1 ? div_near(tiles + r - 1, r, __fdividef(1.f, (float)r)) : max(tiles, 1);
    }
    __device__ void count() {  // items and parts of the loaded block
        len = run_len();
        runs = div_near(tiles + len - 1, len, __fdividef(1.f, (float)len));  // <= r: no run is empty
        const int it = (n + PER - 1) / PER * runs, pt = runs > 1 ? n * runs : 0;
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
// The parts of every node, for the merge; by a warp.
template <bool SEL, int PER>
__device__ void tree_table(const TreeParams& p, TreeWalk<SEL, PER> w) {
    for (int r = threadIdx.x & 31; r < p.n_nodes; r += 32) p.node_tab[r] = make_int2(0, 0);
    __syncwarp();
    do {
        if (w.runs > 1)
            for (int j = 0; j < w.n; ++j) p.node_tab[w.r0 + j] = make_int2(w.part0 + w.excl_part + j * w.runs, w.runs);
    } while (w.next_block(p));
}
struct TreeItem {
    int b, r0, n, ctx, node, tile0, tiles;  // tiles of this item
    int part;                               // -1: the node's only item
    int runs;
};
template <bool SEL, int PER>
__device__ bool tree_item(const TreeParams& p, TreeWalk<SEL, PER>& w, int item, TreeItem& t) {
    while (item >= w.item0 + w.items)
        if (!w.next_block(p)) return false;
    const unsigned here = __ballot_sync(0xffffffffu, w.item0 + w.excl_item <= item && w.n * w.runs > 0);
    const int l = 31 - __clz((int)here);  // the last request that starts at or before the item
    const int local = item - (w.item0 + __shfl_sync(0xffffffffu, w.excl_item, l));
    t.b = __shfl_sync(0xffffffffu, w.id, l);
    t.r0 = __shfl_sync(0xffffffffu, w.r0, l);
    t.n = __shfl_sync(0xffffffffu, w.n, l);
    t.ctx = __shfl_sync(0xffffffffu, w.ctx, l);
    const int all = __shfl_sync(0xffffffffu, w.tiles, l), runs = __shfl_sync(0xffffffffu, w.runs, l);
    const int len = __shfl_sync(0xffffffffu, w.len, l);
    const int per = (t.n + PER - 1) / PER;
    const int run = local / per;  // the request's nodes side by side on one run of keys
    t.node = (local - run * per) * PER;
    t.tile0 = run * len;
    t.tiles = min(len, all - t.tile0);
    t.runs = runs;
    t.part = runs > 1 ? w.part0 + __shfl_sync(0xffffffffu, w.excl_part, l) + t.node * runs + run : -1;
    return true;
}

// The keys of the tile at position pos0 that a node with mask `see` sees.
__device__ __forceinline__ unsigned long long tree_tile_mask(unsigned long long see, int pos0, int ctx) {
    if (pos0 + TA_TILE <= ctx) return ~0ull;
    const int first = pos0 - ctx;  // the tile's first key as a node number
    return first >= 64 ? 0ull : first >= 0 ? see >> first : (see << -first) | ((1ull << -first) - 1);
}
// This lane's box of every STEP-th tile of a run of key tiles (a warp holds the nbox boxes of a tile): its page,
// loaded a step ahead, and its first row there; a step on is `hop` pages and `rest` rows on.
template <int STEP = 1>
struct TreePages {
    const int* table;
    int nbox, page_size, n_pages, end, hop, rest;
    int pos, at, off, page;
    bool mine;
    __device__ void start(const TreeParams& p, const TreeItem& t, int first = 0) {
        const int lane = threadIdx.x & 31, R = p.box_rows;
        table = p.table + (long long)t.b * p.table_stride;
        nbox = TA_TILE / R;
        page_size = p.page_size;
        n_pages = p.n_pages;
        end = t.ctx + t.n;
        hop = STEP * TA_TILE / page_size;
        rest = STEP * TA_TILE % page_size;
        pos = (t.tile0 + first) * TA_TILE + lane * R;
        at = pos / page_size;
        off = pos - at * page_size;
        mine = lane < nbox && pos < end;
        page = mine ? __ldg(table + at) : 0;
    }
    // First slot of this lane's box of the current tile, behind the pool (read as zeros) past the request's rows
    // or for a page outside the pool (the error word, and `lost` then holds the tile's keys there), then a step on.
    __device__ int next(bool more, unsigned long long& lost) {
        const bool bad = mine && (page < 0 || page >= n_pages);
        if (bad) set_error(ERRC_BOUNDS, 46);
        const int slot = mine && !bad ? page * page_size + off : n_pages * page_size;
        pos += STEP * TA_TILE;
        at += hop;
        off += rest;
        if (off >= page_size) {
            off -= page_size;
            ++at;
        }
        mine = (int)(threadIdx.x & 31) < nbox && pos < end;
        if (mine && more) page = __ldg(table + at);
        lost = 0;
        const unsigned out = __ballot_sync(0xffffffffu, bad);
        if (out) {
            const int R = TA_TILE / nbox;
            for (int j = 0; j < nbox; ++j)
                if ((out >> j) & 1) lost |= (R >= 64 ? ~0ull : (1ull << R) - 1) << (j * R);
        }
        return slot;
    }
};

// One half of a key tile (columns 0-255 and the roped ones, or 256-511) in NB
// boxes, by one thread: column by column, the boxes' rows in registers. A TMA
// instruction takes its coordinates from uniform registers; with lanes issuing a
// box each, or a branch and a shared-memory read per box, an instruction takes
// 75 and 42 cycles, like this 17 to 30.
template <int NB>
__device__ __forceinline__ void tree_boxes(const TreeMaps& tm, uint32_t dst, int half, const volatile int* rows, uint64_t* bar) {
    constexpr uint32_t CHUNK = TA_TILE * 128, BOX = CHUNK / NB;
    int y[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) y[j] = rows[j];
    if constexpr (NB == 1) {  // a tile inside a page: its four column chunks at once (1 node x 1K 14.2 -> 13.7 us; pairs 1 % slower)
        tma_load3d(dst + 4 * half * CHUNK, &tm.wide, 0, y[0], 4 * half, bar);
    } else {
#pragma unroll(NB <= 2 ? 4 : 1)
        for (int c = 4 * half; c < 4 * half + 4; ++c) {
#pragma unroll
            for (int j = 0; j < NB; ++j) tma_load2d(dst + c * CHUNK + j * BOX, &tm.ckv, c * 64, y[j], bar);
        }
    }
    if (half == 0) {
#pragma unroll
        for (int j = 0; j < NB; ++j) tma_load2d(dst + 8 * CHUNK + j * BOX, &tm.krot, 0, y[j], bar);
    }
}

template <bool SEL>
__global__ void __launch_bounds__(TaLayout<SEL>::THREADS, 1) tree_attn_kernel(const TreeParams p, const __grid_constant__ TreeMaps tm) {
    using L = TaLayout<SEL>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sK = smem_u32(smem), sP = smem_u32(smem + L::OFF_P);
    int4* items = reinterpret_cast<int4*>(smem + L::OFF_ITEM);  // (row or -1 = no more, tiles, part, unused)
    unsigned long long* see_sh = reinterpret_cast<unsigned long long*>(smem + L::OFF_SEE);
    uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);  // [entry][half]
    uint64_t* kfree = kfull + 2 * TA_NBUF;
    uint64_t* sfull = kfree + 2 * TA_NBUF;
    uint64_t* pready = sfull + 2;
    uint64_t* pvdone = pready + 1;
    uint64_t* qtmem = pvdone + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
    int* longest_sh = reinterpret_cast<int*>(tmem_slot + 1);
    volatile int* go = reinterpret_cast<volatile int*>(tmem_slot + 2);    // lists: [2], by the parity of the wait
    volatile int* info = reinterpret_cast<volatile int*>(tmem_slot + 4);  // lists: the item, for all gather threads
    int* out_done = reinterpret_cast<int*>(tmem_slot + 12);  // softmax warps through with an item's output
    int* rows_sh = reinterpret_cast<int*>(smem + L::OFF_ROWS);
    volatile int* slots_sh = info;  // dense: first slots of a tile's boxes

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int b = 0; b < 2 * TA_NBUF; ++b) {
            mbar_init(kfull + b, !SEL ? 1 : L::LOADERS + (b & 1 ? 0 : 2));  // lists: and two for see_sh, with the first half
            mbar_init(kfree + b, 1);  // the P.V commit of that half; the MMA warp for a query
                                      // entry, the softmax warps for an item's last tile
        }
        mbar_init(sfull, 1);
        mbar_init(sfull + 1, 1);
        mbar_init(pready, 128);
        mbar_init(pvdone, 1);
        mbar_init(qtmem, 128);
        *out_done = 0;
        fence_mbar_init();
    }
    if (warp == L::MMA_WARP) tmem_alloc(tmem_slot, 512);
    if (warp == TA_LOAD_WARP && lane < (SEL ? 1 : 3))
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane == 0 ? &tm.q : lane == 1 ? &tm.ckv : &tm.krot)) : "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_trigger();
    // The schedule: (nodes, tiles) of the requests, up to 32 by the producer warp, which keeps them sorted
    // in registers; more by all threads, in the key tiles' space.
    TreeCost* cost = reinterpret_cast<TreeCost*>(smem + L::OFF_P);
    const bool many = p.batch > 32;
    int2* tab = reinterpret_cast<int2*>(many ? smem : smem + L::OFF_P + sizeof(TreeCost));
    TreeWalk<SEL> walk;
    if (many) {
        if (tid == 0) *longest_sh = 0;
        __syncthreads();
        int longest = 0;
        for (int b = tid; b < p.batch; b += L::THREADS) {
            const TreeSeq q = tree_seq(p, b);
            const int t = q.n > 0 ? tree_tiles<SEL>(p, q) : 0;
            tab[b] = make_int2(q.n, t);
            longest = max(longest, t);
        }
        if (longest > 0) atomicMax(longest_sh, longest);
    }
    if (warp == TA_LOAD_WARP) {
        walk.b0 = walk.item0 = walk.part0 = 0;
        walk.load(p);
        if (!many) {
            if (p.batch > 1) walk.sort(walk.tiles);
            if (lane < p.batch) tab[lane] = make_int2(walk.n, walk.tiles);
            if (lane == 0) *longest_sh = walk.tiles;
        }
    }
    __syncthreads();
    walk.C = tree_schedule<1>(p, tab, *longest_sh, cost, gridDim.x, TA_PRICE);
    if (many) {
        fence_proxy_async_smem();  // the table becomes key tiles: its generic accesses come before TMA writes
        __syncthreads();
    }

    if (warp == TA_LOAD_WARP) {  // the producer, or the first gather warp
        if (p.batch > 1 && !many) walk.sort(walk.run_len());
        walk.count();
        if (blockIdx.x == gridDim.x - 1) tree_table(p, walk);
    }

    if (warp >= TA_LOAD_WARP && warp < L::MMA_WARP) {
        if constexpr (!SEL) {
            // ---------------- producer (every key): one warp ----------------
            int e = 0;  // ring entries issued
            bool ok = true;
            // A ring entry's half is free: its third-last use was consumed.
            auto acquire = [&](int half) -> bool {
                return e < TA_NBUF || mbar_wait_fast(kfree + 2 * (e % TA_NBUF) + half, (uint32_t)(e / TA_NBUF - 1) & 1u, 50);
            };
            for (int k = 0; ok; ++k) {
                TreeItem t{};
                const bool more = tree_item(p, walk, item_of(k, blockIdx.x, gridDim.x), t);
                const int row = t.r0 + t.node, n_tiles = t.tiles;
                if (!(ok = acquire(0) && acquire(1))) break;
                {
                    const int b = e % TA_NBUF;
                    if (lane == 0) items[b] = make_int4(more ? row : -1, n_tiles, t.part, 0);
                    __syncwarp();
                    if (elect_one()) {
                        if (more) {  // the query, 64 heads x 576: nine boxes
                            mbar_expect_tx(kfull + 2 * b, 5 * L::CHUNK);
                            mbar_expect_tx(kfull + 2 * b + 1, 4 * L::CHUNK);
#pragma unroll
                            for (int c = 0; c < AT_CHUNKS; ++c)
                                tma_load2d(sK + b * L::TILE + c * L::CHUNK, &tm.q, c * 64, row * AT_H,
                                           kfull + 2 * b + (c >= 4 && c < 8 ? 1 : 0));
                        } else {
                            mbar_arrive(kfull + 2 * b);
                        }
                    }
                    __syncwarp();
                    if (!more) break;
                    ++e;
                }
                TreePages<> pages;
                pages.start(p, t);
                const int nbox = pages.nbox;
                const unsigned long long see = tree_mask_of(p, t.r0, t.n, t.node);
                for (int i = 0; i < n_tiles && ok; ++i) {
                    const int b = e % TA_NBUF;
                    unsigned long long lost;
                    const int slot = pages.next(i + 1 < n_tiles, lost);
                    const unsigned long long v = tree_tile_mask(see, (t.tile0 + i) * TA_TILE, t.ctx) & ~lost;
                    if (lane < 8) slots_sh[lane] = slot;
                    if (!(ok = acquire(0))) break;
                    if (lane == 0) see_sh[b] = v;
                    __syncwarp();
                    // columns 0-255 and the roped ones, then 256-511
                    auto boxes = [&](int half) {
                        if (elect_one()) {
                            uint64_t* bar = kfull + 2 * b + half;
                            mbar_expect_tx(bar, (uint32_t)((5 - half) * L::CHUNK));
                            const uint32_t dst = sK + b * L::TILE;
                            if (nbox == 1) tree_boxes<1>(tm, dst, half, slots_sh, bar);
                            else if (nbox == 2) tree_boxes<2>(tm, dst, half, slots_sh, bar);
                            else if (nbox == 4) tree_boxes<4>(tm, dst, half, slots_sh, bar);
                            else tree_boxes<8>(tm, dst, half, slots_sh, bar);
                        }
                        __syncwarp();
                    };
                    boxes(0);
                    if (!(ok = acquire(1))) break;
                    boxes(1);
                    ++e;
                }
            }
            if (!ok)  // copies in flight must land before the CTA leaves
                for (int k = max(0, e - TA_NBUF); k <= e; ++k)
                    for (int half = 0; half < 2; ++half) mbar_wait_fast(kfull + 2 * (k % TA_NBUF) + half, (uint32_t)(k / TA_NBUF) & 1u, 51);
        } else {
            // ---------------- gather (lists): all 8 warps ----------------
            const int g = tid - 128;
            int e = 0, waits = 0;  // ring entries issued, acquire calls
            bool ok = true;
            // A ring entry's half is free. One thread waits; all gather threads get the same answer.
            auto acquire = [&](int half) -> bool {
                const int x = waits++ & 1;
                if (g == 0)
                    go[x] = e < TA_NBUF || mbar_wait_fast(kfree + 2 * (e % TA_NBUF) + half, (uint32_t)(e / TA_NBUF - 1) & 1u, 50) ? 1 : 0;
                asm volatile("bar.sync 2, %0;" ::"n"(L::LOADERS) : "memory");
                return go[x] != 0;  // rewritten two calls on, behind the barrier in between
            };
            // The first half's two further arrivals: the threads that write see_sh.
            const bool marks = g == 0 || g == 32;
            const int r8 = g >> 3, seg = g & 7;  // this thread's 16 bytes of rows r8 and r8 + 32 of a tile
            for (int k = 0; ok; ++k) {
                TreeItem t{};
                if (warp == TA_LOAD_WARP) {
                    const bool more = tree_item(p, walk, item_of(k, blockIdx.x, gridDim.x), t);
                    unsigned long long see = 0;
                    int left = 0;  // entries of this item
                    if (more) {
                        left = max(0, min(tree_list_n(p, t.r0 + t.node) - t.tile0 * TA_TILE, t.tiles * TA_TILE));
                        see = tree_mask_of(p, t.r0, t.n, t.node);
                    }
                    if (lane == 0) {
                        info[0] = more ? t.r0 + t.node : -1;
                        info[1] = t.b;
                        info[2] = t.ctx;
                        info[3] = t.n;
                        info[4] = t.tile0 * TA_TILE;
                        info[5] = left;
                        info[6] = (int)(unsigned)see;
                        info[7] = (int)(unsigned)(see >> 32);
                    }
                }
                if (!(ok = acquire(0))) break;  // also orders info[]
                const int row = info[0], left = info[5], n_tiles = (left + TA_TILE - 1) / TA_TILE, ctx = info[2], n = info[3];
                const unsigned long long see = (unsigned)info[6] | ((unsigned long long)(unsigned)info[7] << 32);
                const int* table = p.table + (long long)info[1] * p.table_stride;
                const int* list = p.sel + (long long)max(row, 0) * p.sel_stride + info[4];
                if (!(ok = acquire(1))) break;  // and info[] is read before the next item's
                const int qb = e % TA_NBUF;
                if (g == 0) items[qb] = make_int4(row, n_tiles, t.part, 0);
                if (marks) mbar_arrive(kfull + 2 * qb);
                if (row < 0) {
                    mbar_arrive(kfull + 2 * qb);
                    break;
                }
                if (g == 0) {  // the query, 64 heads x 576: nine boxes
                    mbar_expect_tx(kfull + 2 * qb, 5 * L::CHUNK);
                    mbar_expect_tx(kfull + 2 * qb + 1, 4 * L::CHUNK);
                    for (int c = 0; c < AT_CHUNKS; ++c)
                        tma_load2d(sK + qb * L::TILE + c * L::CHUNK, &tm.q, c * 64, row * AT_H, kfull + 2 * qb + (c >= 4 && c < 8 ? 1 : 0));
                } else {
                    mbar_arrive(kfull + 2 * qb);
                    mbar_arrive(kfull + 2 * qb + 1);
                }
                ++e;
                // threads 0-63: the slot of a tile's key, -1 when the row does not see it; positions are loaded two
                // tiles ahead, pages one
                auto entry = [&](int j) -> int { return g < TA_TILE && j < left ? __ldg(list + j) : -1; };
                auto page_of = [&](int& pos) -> int {
                    const bool is = pos >= 0 && pos < ctx + n && (pos < ctx || ((see >> (pos - ctx)) & 1));
                    if (!is) pos = -1;
                    return is ? __ldg(table + pos / p.page_size) : 0;
                };
                int pos = entry(g), nxt = entry(g + TA_TILE), page = page_of(pos);
                for (int i = 0; i < n_tiles; ++i) {
                    const int b = e % TA_NBUF;
                    if (g < TA_TILE) {
                        int slot = -1;
                        if (pos >= 0) {
                            if (page < 0 || page >= p.n_pages) set_error(ERRC_BOUNDS, 46);
                            else slot = page * p.page_size + pos % p.page_size;
                        }
                        // rows_sh and see_sh of this slot were last read three entries ago, behind acquire's barriers
                        rows_sh[b * TA_TILE + g] = slot;
                        const unsigned bits = __ballot_sync(0xffffffffu, slot >= 0);
                        pos = nxt;
                        page = page_of(pos);
                        nxt = entry((i + 2) * TA_TILE + g);
                        if (!(ok = acquire(0))) break;
                        if (marks) {
                            reinterpret_cast<volatile unsigned*>(see_sh + b)[g >> 5] = bits;
                            mbar_arrive(kfull + 2 * b);
                        }
                    } else if (!(ok = acquire(0))) {
                        break;
                    }
                    const uint32_t dst = sK + b * L::TILE + sw128_off(r8, seg);  // row r8 + 32 swizzles alike
                    const int sl0 = rows_sh[b * TA_TILE + r8], sl1 = rows_sh[b * TA_TILE + r8 + 32];
                    const uint32_t by0 = sl0 < 0 ? 0u : 16u, by1 = sl1 < 0 ? 0u : 16u;
                    const __nv_bfloat16* src0 = p.c_kv + (long long)max(sl0, 0) * p.ckv_row + seg * 8;
                    const __nv_bfloat16* src1 = p.c_kv + (long long)max(sl1, 0) * p.ckv_row + seg * 8;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        cp_async16(dst + c * L::CHUNK, src0 + c * 64, by0);
                        cp_async16(dst + c * L::CHUNK + 32 * 128, src1 + c * 64, by1);
                    }
                    cp_async16(dst + 8 * L::CHUNK, p.k_rot + (long long)max(sl0, 0) * p.krot_row + seg * 8, by0);
                    cp_async16(dst + 8 * L::CHUNK + 32 * 128, p.k_rot + (long long)max(sl1, 0) * p.krot_row + seg * 8, by1);
                    cp_async_arrive(kfull + 2 * b);
                    if (!(ok = acquire(1))) break;
#pragma unroll
                    for (int c = 4; c < 8; ++c) {
                        cp_async16(dst + c * L::CHUNK, src0 + c * 64, by0);
                        cp_async16(dst + c * L::CHUNK + 32 * 128, src1 + c * 64, by1);
                    }
                    cp_async_arrive(kfull + 2 * b + 1);
                    ++e;
                }
            }
            cp_async_wait_all();
            if (!ok && g == 0) {  // a query in flight must land before the CTA leaves
                for (int k = 0; k < 2 * TA_NBUF; ++k) mbar_wait_fast(kfull + k, 0, 51);
            }
        }
    } else if (warp == L::MMA_WARP) {
        // ---------------- MMA ----------------
        const uint32_t tq = tmem + (16u << 16) + PF_TM_Q;
        int e = 0, gt = 0;  // ring entries and key tiles taken
        // Tile g's scores go to S buffer g & 1: its reader of two tiles before is done (that tile's P.V was issued).
        auto issue_qk = [&](int entry, int g_) -> bool {
            const int b = entry % TA_NBUF, s = g_ & 1;
            const uint32_t d = tmem + (16u << 16) + (uint32_t)(s * TA_TILE);
            const uint64_t k0 = desc_sw128(sK + b * L::TILE, 16, 1024);
            auto chunk = [&](int c) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)  // descriptors step in 16-byte units
                    mma_bf16_ts(d, tq + (uint32_t)(c * 32 + kk * 8), k0 + ((c * L::CHUNK + kk * 32) >> 4), L::IDESC_QK,
                                (c | kk) != 0 ? 1u : 0u);
            };
            if (!mbar_wait_fast(kfull + 2 * b, (uint32_t)(entry / TA_NBUF) & 1u, 52)) return false;
            if (SEL) fence_proxy_async_smem();  // gathered rows (cp.async) -> tensor cores
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int c = 0; c < 4; ++c) chunk(c);
                chunk(8);
            }
            if (!mbar_wait_fast(kfull + 2 * b + 1, (uint32_t)(entry / TA_NBUF) & 1u, 53)) return false;
            if (SEL) fence_proxy_async_smem();
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int c = 4; c < 8; ++c) chunk(c);
                mma_commit(sfull + s);
            }
            __syncwarp();
            return true;
        };
        auto issue_pv = [&](int entry, int g_, bool first, bool last) -> bool {
            const int b = entry % TA_NBUF;
            if (!mbar_wait_fast(pready, (uint32_t)g_ & 1u, 54)) return false;
            tc_fence_after();
            if (elect_one()) {
                const uint64_t p0 = desc_sw128(sP, 16, 1024), v0 = desc_sw128(sK + b * L::TILE, L::CHUNK, 1024);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int ks = 0; ks < TA_TILE / 16; ++ks)
                        mma_bf16(tmem + (uint32_t)(half * 256), p0 + ks * 2, v0 + ((4 * half * L::CHUNK + ks * 2048) >> 4),
                                 L::IDESC_PV, (!first || ks > 0) ? 1u : 0u);
                    if (!last) mma_commit(kfree + 2 * b + half);  // the item's last: its output goes through this space
                }
                mma_commit(pvdone);
            }
            __syncwarp();
            return true;
        };
        bool ok = true;
        for (int it = 0; ok; ++it) {
            const int qb = e % TA_NBUF;
            if (!(ok = mbar_wait_fast(kfull + 2 * qb, (uint32_t)(e / TA_NBUF) & 1u, 55))) break;
            const int4 t = items[qb];
            if (t.x < 0) break;
            if (!(ok = mbar_wait_fast(qtmem, (uint32_t)it & 1u, 56))) break;  // the query is in tensor memory
            if (elect_one()) {
                mbar_arrive(kfree + 2 * qb);
                mbar_arrive(kfree + 2 * qb + 1);
            }
            ++e;
            const int n = t.y;
            if (n > 0) ok = issue_qk(e, gt);
            for (int i = 0; ok && i < n; ++i) {
                if (i + 1 < n) ok = issue_qk(e + i + 1, gt + i + 1);
                if (ok) ok = issue_pv(e + i, gt + i, i == 0, i + 1 == n);
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
        int out_row = -1, out_part = -1, out_slot = -1;  // the item whose output is still in tensor memory, its last tile
        float m_run = -INFINITY, l_run = 0.f;
        bool ok = true;
        while (ok) {
            const int qb = e % TA_NBUF;
            if (!(ok = mbar_wait_fast(kfull + 2 * qb, (uint32_t)(e / TA_NBUF) & 1u, 57))) break;
            const int4 t = items[qb];
            if (t.x >= 0) {
                if (!(ok = mbar_wait_fast(kfull + 2 * qb + 1, (uint32_t)(e / TA_NBUF) & 1u, 57))) break;
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
                const bool none = !any && out_part < 0;  // (a partial keeps the NaN of 0 x infinity)
                const float lse = any ? (m_run + log2f(l_run)) * 0.69314718055994531f : -INFINITY;
                if (!hi_half) {
                    if (out_part >= 0) p.lse_part[(long long)out_part * AT_H + h] = lse;
                    else if (p.lse) p.lse[(long long)out_row * AT_H + h] = lse;
                }
                if (out_slot >= 0) {
                    // O leaves through the space of the item's last tile (its P.V is done; the MMA warp leaves it
                    // to this role to give back), a warp's 16 heads in boxes of 128 bytes a head, by TMA stores:
                    // nothing waits until the eighth box (stores of single threads took 6,000 to 11,000 cycles).
                    const bool narrow = out_part < 0 && p.ctx_bf16;
                    const int y = (out_part >= 0 ? out_part : out_row) * AT_H + 16 * warp;
                    const uint32_t base = sK + out_slot * L::TILE + warp * 16384u, mine = base + (uint32_t)(lane & 15) * 128u;
                    auto piece = [&](uint32_t box, int seg, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
                        sts_v4(mine + box * 2048u + (uint32_t)((seg ^ lane) & 7) * 16u, make_uint4(a, b, c, d));
                    };
#pragma unroll 1
                    for (int c = 0; c < AT_DV / 64; ++c) {
                        float ov[32];
                        tmem_ld16x2_32<32>(tmem + lane_o + (uint32_t)(64 * c), ov);
#pragma unroll
                        for (int x = 0; x < 32; ++x) ov[x] = none ? 0.f : ov[x] * inv;
                        if (narrow) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                uint32_t w[4];
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    const __nv_bfloat162 b2 = __floats2bfloat162_rn(ov[8 * k + 2 * x], ov[8 * k + 2 * x + 1]);
                                    w[x] = *reinterpret_cast<const uint32_t*>(&b2);
                                }
                                piece(c, (hi_half ? 4 : 0) + k, w[0], w[1], w[2], w[3]);
                            }
                        } else {
                            if (c >= 4) {  // the eight boxes come round again: their last stores have been read
                                if (elect_one()) asm volatile("cp.async.bulk.wait_group.read 3;" ::: "memory");
                                __syncwarp();
                            }
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                piece((2 * c + (hi_half ? 1 : 0)) & 7, k, __float_as_uint(ov[4 * k]), __float_as_uint(ov[4 * k + 1]),
                                      __float_as_uint(ov[4 * k + 2]), __float_as_uint(ov[4 * k + 3]));
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (elect_one()) {
                            if (narrow) {
                                tma_store2d(&tm.out, 64 * c, y, base + c * 2048u);
                            } else {
                                const CUtensorMap* m = out_part >= 0 ? &tm.part : &tm.out;
                                tma_store2d(m, 64 * c, y, base + ((2 * c) & 7) * 2048u);
                                tma_store2d(m, 64 * c + 32, y, base + ((2 * c + 1) & 7) * 2048u);
                            }
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                    }
                    if (elect_one()) {
                        // the copies have read the space; the writes themselves complete with the grid
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        __threadfence_block();
                        if (atomicAdd(out_done, 1) == 3) {  // the last of the four warps gives the space back
                            *out_done = 0;
                            mbar_arrive(kfree + 2 * out_slot);
                            mbar_arrive(kfree + 2 * out_slot + 1);
                        }
                    }
                    __syncwarp();
                } else {
                    // an item without a tile: a row that sees nothing, or a run behind a short list's end
                    const long long at = (out_part >= 0 ? (long long)out_part : (long long)out_row) * AT_H + h;
                    const bool narrow = out_part < 0 && p.ctx_bf16;
                    const int n4 = narrow ? AT_DV / 16 : AT_DV / 8;  // 16-byte pieces of half a row
                    uint4* z = narrow ? reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.ctx) + at * AT_DV)
                                      : reinterpret_cast<uint4*>((out_part >= 0 ? p.o_part : static_cast<float*>(p.ctx)) + at * AT_DV);
                    for (int x = 0; x < n4; ++x) z[x + (hi_half ? n4 : 0)] = make_uint4(0, 0, 0, 0);
                }
                tc_fence_before();  // these reads come before the next P.V (ordered by pready)
            }
            if (t.x < 0) break;
            out_row = t.x;
            out_part = t.z;
            out_slot = t.y > 0 ? (e + t.y - 1) % TA_NBUF : -1;
            m_run = -INFINITY;
            l_run = 0.f;
            for (int i = 0; i < t.y && ok; ++i, ++e, ++gt) {
                const int s = gt & 1, b = e % TA_NBUF;
                if (!(ok = mbar_wait_fast(kfull + 2 * b, (uint32_t)(e / TA_NBUF) & 1u, 59))) break;  // orders see_sh
                const unsigned long long see = see_sh[b];
                if (!(ok = mbar_wait_fast(sfull + s, (uint32_t)(gt >> 1) & 1u, 60))) break;
                tc_fence_after();
                float sv[32];
                tmem_ld16x2_32<32>(tmem + lane_s + (uint32_t)(s * TA_TILE), sv);
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
                    // An unseen row may hold anything (0 x NaN is NaN): its values become zeros
                    // before P.V reads them.
                    for (int j = warp; j < TA_TILE; j += 4) {
                        if ((see >> j) & 1) continue;
                        const uint32_t dst = sK + b * L::TILE + (uint32_t)(lane >> 3) * L::CHUNK + (uint32_t)j * 128u + (uint32_t)(lane & 7) * 16u;
                        sts_v4(dst, make_uint4(0, 0, 0, 0));
                        sts_v4(dst + 4 * L::CHUNK, make_uint4(0, 0, 0, 0));
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
// L = log sum_s e^lse_s. A block owns one (head, 128 columns) of every k-th node.
// A node of up to TM_SOLO parts is joined by one warp, four nodes at a time; a
// longer one by the four warps together, their sums added in warp order. Bound by
// the latency of dependent loads: a warp reads TM_DEPTH partials and their lse
// at once, and every lane works out the weights itself, with a running maximum.
constexpr int TM_UNITS = AT_H * (AT_DV / 128), TM_WARPS = 4, TM_DEPTH = 4, TM_SOLO = 8;
__global__ void __launch_bounds__(TM_WARPS * 32) tree_merge_kernel(const TreeParams p) {
    pdl_wait();
    pdl_trigger();
    __shared__ float4 part_sh[TM_WARPS - 1][32];
    __shared__ float2 stat_sh[TM_WARPS - 1];
    constexpr float LOG2E = 1.4426950408889634f;
    const int lane = threadIdx.x & 31, wi = threadIdx.x >> 5;
    const int h = (blockIdx.x % TM_UNITS) >> 2, q = blockIdx.x & 3, step = gridDim.x / TM_UNITS;
    int turn = 0;  // of the warps at the short nodes
    for (int r0 = blockIdx.x / TM_UNITS; r0 < p.n_nodes; r0 += 32 * step) {
        const int rl = r0 + lane * step;
        const int2 mine = rl < p.n_nodes ? p.node_tab[rl] : make_int2(0, 0);
        for (unsigned cut = __ballot_sync(0xffffffffu, mine.y > 1); cut; cut &= cut - 1) {
            const int l = __ffs(cut) - 1, r = r0 + l * step;
            const int part0 = __shfl_sync(0xffffffffu, mine.x, l), n = __shfl_sync(0xffffffffu, mine.y, l);
            const bool solo = n <= TM_SOLO;
            if (solo && (turn++ & (TM_WARPS - 1)) != wi) continue;
            const int by = solo ? 1 : TM_WARPS;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float M = -INFINITY, W = 0.f;
            // (M, W, acc) times e^(M - what) and more: the sums of two sets of parts by one maximum
            auto scale_to = [&](float m_new) {
                const float a = exp2f((M - (m_new == -INFINITY ? 0.f : m_new)) * LOG2E);
                M = m_new;
                W *= a;
                acc.x *= a;
                acc.y *= a;
                acc.z *= a;
                acc.w *= a;
            };
#pragma unroll 1
            for (int s0 = solo ? 0 : wi; s0 < n; s0 += TM_DEPTH * by) {
                const long long at0 = (long long)(part0 + s0) * AT_H + h, hop = (long long)by * AT_H;
                float4 v[TM_DEPTH];
                float ls[TM_DEPTH], m_new = M;
#pragma unroll
                for (int k = 0; k < TM_DEPTH; ++k) {
                    const bool is = s0 + by * k < n;
                    ls[k] = is ? p.lse_part[at0 + k * hop] : -INFINITY;
                    v[k] = is ? *reinterpret_cast<const float4*>(p.o_part + (at0 + k * hop) * AT_DV + q * 128 + lane * 4)
                              : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int k = 0; k < TM_DEPTH; ++k) m_new = fmaxf(m_new, ls[k]);
                scale_to(m_new);
                const float m_use = m_new == -INFINITY ? 0.f : m_new;
#pragma unroll
                for (int k = 0; k < TM_DEPTH; ++k) {
                    const float w = exp2f((ls[k] - m_use) * LOG2E);
                    W += w;
                    acc.x = fmaf(w, v[k].x, acc.x);
                    acc.y = fmaf(w, v[k].y, acc.y);
                    acc.z = fmaf(w, v[k].z, acc.z);
                    acc.w = fmaf(w, v[k].w, acc.w);
                }
            }
            if (!solo) {
                if (wi > 0) {
                    part_sh[wi - 1][lane] = acc;
                    if (lane == 0) stat_sh[wi - 1] = make_float2(M, W);
                }
                __syncthreads();
                if (wi == 0) {
                    float m_new = M;
#pragma unroll
                    for (int k = 0; k < TM_WARPS - 1; ++k) m_new = fmaxf(m_new, stat_sh[k].x);
                    scale_to(m_new);
                    const float m_use = m_new == -INFINITY ? 0.f : m_new;
#pragma unroll
                    for (int k = 0; k < TM_WARPS - 1; ++k) {
                        const float4 o = part_sh[k][lane];
                        const float w = exp2f((stat_sh[k].x - m_use) * LOG2E);
                        W = fmaf(w, stat_sh[k].y, W);
                        acc.x = fmaf(w, o.x, acc.x);
                        acc.y = fmaf(w, o.y, acc.y);
                        acc.z = fmaf(w, o.z, acc.z);
                        acc.w = fmaf(w, o.w, acc.w);
                    }
                }
                __syncthreads();  // the shared arrays are reused
                if (wi > 0) continue;
            }
            const float inv = 1.f / W;
            acc.x *= inv;
            acc.y *= inv;
            acc.z *= inv;
            acc.w *= inv;
            if (W == 0.f) acc = make_float4(0.f, 0.f, 0.f, 0.f);  // (NaN does not count as none: it reaches the result)
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
    }
}

}  // namespace wl
