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
//              warps keep the running maximum and sum, one row a thread, and a
//              bulk copy takes P (bf16, 16 KB) and the rows' rescale factors to
//              the value CTA's shared memory.
//   value CTA  O += P V: 8 MMAs M = 128, N = 256: 1,024 cycles. Four warps rescale
//              O when a factor is not 1 (rare: the maximum moves only by more than
//              2^8), and write O / l at the end of an item.
// So both tensor cores work all the time, on 64 keys of two nodes in about 1,152
// cycles, where tree_attn_kernel's two SMs take 2 x 2,176 for the same. Each key
// row is read by both CTAs (from L2 once more), 64 bytes a cycle and SM.
// Two nodes share V in one MMA: a drafted row that not both see, and that holds
// a NaN or an infinity, would reach the other through 0 x NaN. In tiles with
// drafted rows the value CTA therefore clears rows that neither sees and the
// non-finite elements of rows that one sees (that node's own result is NaN
// through its scores). Scores are per row; unseen ones are masked.
#pragma once
#include "tree_attn.cuh"

namespace wl {

constexpr int TP_THREADS = 224;  // warps 0-3 rows, 4 loads, 5 MMA, 6 copies P over (score) / tells of freed P (value)
constexpr int TP_UNITS = 7;      // score CTA's ring: units of 64 keys x 192 columns (a third of a tile)
constexpr int TP_VBUF = 3;       // value CTA's ring: tiles of 64 keys x 512 columns, in halves
constexpr uint32_t TP_TM_S = 384;  // score columns in tensor memory (the queries take [0, 288))
constexpr TreePrice TP_PRICE = {9.f, 0.08f, 0.16f};

struct TpLayout {
    static constexpr uint32_t CHUNK = TA_TILE * 128;          // 8 KB: 64 keys x 64 columns
    static constexpr uint32_t UNIT = 3 * CHUNK, HALF = 4 * CHUNK, VTILE = 2 * HALF;
    static constexpr uint32_t P = 128 * 128;                  // 128 rows x 64 keys bf16
    static constexpr uint32_t OFF_PS = TP_UNITS * UNIT;       // score CTA: P on its way (two)
    static constexpr uint32_t OFF_P = TP_VBUF * VTILE;        // value CTA: P arrived (two)
    static constexpr uint32_t OFF_ALPHA = OFF_P + 2 * P;      // both: rescale factors [2][128]
    static constexpr uint32_t OFF_FIN = OFF_ALPHA + 1024;     // value CTA: 1 / l of the item's rows [128]
    static constexpr uint32_t OFF_ITEM = OFF_FIN + 512;       // item descriptors [2]
    static constexpr uint32_t OFF_LOST = OFF_ITEM + 128;      // keys lost to bad pages, per tile [8]
    static constexpr uint32_t OFF_BAR = OFF_LOST + 64;
    static constexpr int N_BARS = 28;
    static constexpr uint32_t OFF_MISC = OFF_BAR + N_BARS * 8;  // tensor-memory slot, longest, out count, slots [8]
    static constexpr uint32_t BYTES = OFF_MISC + 48 + 1024;
    static constexpr uint32_t IDESC_QK = idesc_bf16(128, TA_TILE, 0, 0);
    static constexpr uint32_t IDESC_PV = idesc_bf16(128, 256, 0, 1);
    static constexpr uint32_t COPY = P + 512;
};
static_assert(TpLayout::BYTES <= 232448, "one CTA per SM");
static_assert(TpLayout::OFF_PS + 2 * TpLayout::P <= TpLayout::OFF_ALPHA, "score CTA's layout");

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

// `count` column chunks from c0 on of a key tile in NB boxes (see tree_boxes).
template <int NB>
__device__ __forceinline__ void pair_boxes(const TreeMaps& tm, uint32_t dst, int c0, int count, const volatile int* rows, uint64_t* bar) {
    constexpr uint32_t CHUNK = TA_TILE * 128, BOX = CHUNK / NB;
    int y[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) y[j] = rows[j];
#pragma unroll 1
    for (int c = c0; c < c0 + count; ++c, dst += CHUNK) {
        const CUtensorMap* m = c < 8 ? &tm.ckv : &tm.krot;
        const int x = c < 8 ? c * 64 : 0;
#pragma unroll
        for (int j = 0; j < NB; ++j) tma_load2d(dst + j * BOX, m, x, y[j], bar);
    }
}
__device__ __forceinline__ void pair_load(const TreeMaps& tm, uint32_t dst, int c0, int count, int nbox, const volatile int* rows, uint64_t* bar) {
    if (elect_one()) {
        mbar_expect_tx(bar, (uint32_t)count * TpLayout::CHUNK);
        if (nbox == 1) pair_boxes<1>(tm, dst, c0, count, rows, bar);
        else if (nbox == 2) pair_boxes<2>(tm, dst, c0, count, rows, bar);
        else if (nbox == 4) pair_boxes<4>(tm, dst, c0, count, rows, bar);
        else pair_boxes<8>(tm, dst, c0, count, rows, bar);
    }
    __syncwarp();
}

__device__ __forceinline__ uint32_t clear_nonfinite(uint32_t w) {  // two bf16
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
    TpItem* item_sh = reinterpret_cast<TpItem*>(smem + L::OFF_ITEM);
    unsigned long long* lost_sh = reinterpret_cast<unsigned long long*>(smem + L::OFF_LOST);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
    uint64_t *ifull = bars, *ifree = bars + 2;  // item descriptors
    // score CTA
    uint64_t *ufull = bars + 4, *ufree = bars + 11, *qtmem = bars + 18, *sfull = bars + 19, *sfree = bars + 21, *pstaged = bars + 23,
             *pfree = bars + 25, *finfree = bars + 27;
    // value CTA
    uint64_t *vfull = bars + 4, *vfree = bars + 10, *pfull = bars + 16, *pok = bars + 18, *pvdone = bars + 19, *finfull = bars + 21;
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
            mbar_init(ifree + i, 6);  // a lane of each consumer warp
        }
        if (score) {
            for (int i = 0; i < TP_UNITS; ++i) {
                mbar_init(ufull + i, 1);
                mbar_init(ufree + i, 1);
            }
            mbar_init(qtmem, 128);
            for (int i = 0; i < 2; ++i) {
                mbar_init(sfull + i, 1);
                mbar_init(sfree + i, 128);
                mbar_init(pstaged + i, 128);
                mbar_init(pfree + i, 1);
            }
            mbar_init(finfree, 4);
        } else {
            for (int i = 0; i < 2 * TP_VBUF; ++i) {
                mbar_init(vfull + i, 1);
                mbar_init(vfree + i, 1);
            }
            mbar_init(pfull, 1);
            mbar_init(pfull + 1, 1);
            mbar_init(pok, 128);
            mbar_init(pvdone, 1);
            mbar_init(pvdone + 1, 1);
            mbar_init(finfull, 128);
            *out_done = 0;
        }
        fence_mbar_init();
        if (!score)
            for (int i = 0; i < 2; ++i) mbar_expect_tx(pfull + i, L::COPY);
    }
    if (warp == 5) tmem_alloc(tmem_slot, 512);
    if (warp == 4 && lane < 3)
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane == 0 ? &tm.q : lane == 1 ? &tm.ckv : &tm.krot)) : "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    cluster_sync_all();  // both CTAs' barriers exist before either reaches into the other
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_trigger();
    TreeCost* cost = reinterpret_cast<TreeCost*>(smem + L::OFF_P);
    const bool many = p.batch > 32;
    int2* tab = reinterpret_cast<int2*>(many ? smem : smem + L::OFF_P + sizeof(TreeCost));
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
    if (warp == TA_LOAD_WARP) {
        walk.b0 = walk.item0 = walk.part0 = 0;
        walk.load(p);
        if (!many) {
            if (p.batch > 1) walk.sort();
            if (lane < p.batch) tab[lane] = make_int2(walk.n, walk.tiles);
            if (lane == 0) *longest_sh = walk.tiles;
        }
    }
    __syncthreads();
    walk.C = tree_schedule<2>(p, tab, *longest_sh, cost, G, TP_PRICE);
    fence_proxy_async_smem();  // the scratch becomes key tiles and P: its generic accesses come before async writes
    __syncthreads();

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
    if (warp == 4) {
        // ---------------- loads ----------------
        walk.count();
        if (score && me == G - 1) tree_table(p, walk);
        int u = 0, round = 0, gt = 0;  // ring unit (score: a third of a tile, value: half) and how often it went round
        const int ring = score ? TP_UNITS : 2 * TP_VBUF;
        uint64_t *full = score ? ufull : vfull, *free_ = score ? ufree : vfree;
        const uint32_t unit = score ? L::UNIT : L::HALF;
        auto acquire = [&]() -> bool { return round == 0 || mbar_wait_fast(free_ + u, (uint32_t)(round - 1) & 1u, 71); };
        auto advance = [&]() {
            if (++u == ring) {
                u = 0;
                ++round;
            }
        };
        for (int k = 0; ok; ++k) {
            TreeItem t{};
            const bool more = tree_item(p, walk, item_of(k, me, G), t);
            const int rows = more ? min(2, t.n - t.node) : 0;
            if (score && more) {
                // the queries: two nodes x three units (a lone node's twice)
                for (int q = 0; q < 6 && ok; ++q) {
                    if (!(ok = acquire())) break;
                    const int y = (t.r0 + t.node + min(q / 3, rows - 1)) * AT_H;
                    if (elect_one()) {
                        mbar_expect_tx(ufull + u, L::UNIT);
                        for (int c = 0; c < 3; ++c)
                            tma_load2d(base + u * L::UNIT + c * L::CHUNK, &tm.q, (3 * (q % 3) + c) * 64, y, ufull + u);
                    }
                    __syncwarp();
                    advance();
                }
                if (!ok) break;
            }
            if (k >= 2 && !(ok = mbar_wait_fast(ifree + (k & 1), (uint32_t)((k >> 1) - 1) & 1u, 72))) break;
            TpItem d{};
            TreePages pages;
            if (more) {
                pages.start(p, t);
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
            if (!more) break;
            for (int i = 0; i < t.tiles && ok; ++i, ++gt) {
                unsigned long long lost;
                const int slot = pages.next(i + 1 < t.tiles, lost);
                if (lane < 8) slots_sh[lane] = slot;
                if (lane == 0) lost_sh[gt & 7] = lost;
                __syncwarp();
                const int steps = score ? 3 : 2, width = score ? 3 : 4;
                for (int j = 0; j < steps; ++j) {
                    if (!(ok = acquire())) break;
                    pair_load(tm, base + u * unit, j * width, width, pages.nbox, slots_sh, full + u);
                    advance();
                }
            }
        }
        if (!ok)  // copies in flight must land before the CTA leaves
            for (int i = 0; i < ring; ++i)
                if (i < u || round > 0) mbar_wait_fast(full + i, (uint32_t)(i < u ? round : round - 1) & 1u, 73);
    } else if (score && warp == 5) {
        // ---------------- score CTA: Q K^T ----------------
        int u = 0, uph = 0, gt = 0;
        auto advance = [&]() {
            if (++u == TP_UNITS) {
                u = 0;
                uph ^= 1;
            }
        };
        for (int k = 0; ok; ++k) {
            TpItem t;
            if (!(ok = take(k, t)) || t.rows == 0) break;
            if (!(ok = mbar_wait_fast(qtmem, (uint32_t)k & 1u, 74))) break;  // the queries are in tensor memory
            for (int q = 0; q < 6; ++q) {
                if (elect_one()) mbar_arrive(ufree + u);
                advance();
            }
            for (int i = 0; i < t.tiles && ok; ++i, ++gt) {
                const int s = gt & 1;
                if (gt >= 2 && !(ok = mbar_wait_fast(sfree + s, (uint32_t)((gt >> 1) - 1) & 1u, 75))) break;
                const uint32_t d = tmem + TP_TM_S + (uint32_t)(s * TA_TILE);
#pragma unroll
                for (int j = 0; j < 3; ++j) {
                    if (!(ok = mbar_wait_fast(ufull + u, (uint32_t)uph, 76))) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t k0 = desc_sw128(base + u * L::UNIT, 16, 1024);
#pragma unroll
                        for (int c = 0; c < 3; ++c)
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                mma_bf16_ts(d, tmem + (uint32_t)((3 * j + c) * 32 + kk * 8), k0 + ((c * L::CHUNK + kk * 32) >> 4), L::IDESC_QK,
                                            (j | c | kk) != 0 ? 1u : 0u);
                        mma_commit(ufree + u);
                        if (j == 2) mma_commit(sfull + s);
                    }
                    __syncwarp();
                    advance();
                }
            }
        }
    } else if (score && warp == 6) {
        // ---------------- score CTA: P to the value CTA ----------------
        int gt = 0;
        for (int k = 0; ok; ++k) {
            TpItem t;
            if (!(ok = take(k, t)) || t.rows == 0) break;
            for (int i = 0; i < t.tiles; ++i, ++gt) {
                const int b = gt & 1;
                if (!(ok = mbar_wait_fast(pstaged + b, (uint32_t)(gt >> 1) & 1u, 77))) break;
                if (elect_one()) {  // its space there is free: the rows waited for that before they wrote
                    const uint32_t bar = dsmem_addr(pfull + b, 1);
                    bulk_s2s(dsmem_addr(smem + L::OFF_P + b * L::P, 1), base + L::OFF_PS + b * L::P, L::P, bar);
                    bulk_s2s(dsmem_addr(alpha_sh + 128 * b, 1), smem_u32(alpha_sh + 128 * b), 512, bar);
                }
                __syncwarp();
            }
        }
    } else if (score) {
        // ---------------- score CTA: softmax, one row a thread (warps 0-3) ----------------
        const int r = tid, half = r >> 6;
        const uint32_t lanes = (uint32_t)(32 * warp) << 16;
        int u = 0, uph = 0, gt = 0;  // ring position of the item's first unit
        for (int k = 0; ok; ++k) {
            TpItem t;
            if (!(ok = take(k, t)) || t.rows == 0) break;
            // this row's query into tensor memory (every QK of the item before is done: its scores were read)
            int qu = u, qph = uph;
            for (int j = 0; j < 3 * half; ++j)
                if (++qu == TP_UNITS) {
                    qu = 0;
                    qph ^= 1;
                }
            for (int j = 0; j < 3 && ok; ++j) {
                if (!(ok = mbar_wait_fast(ufull + qu, (uint32_t)qph, 78))) break;
                const uint32_t src = base + qu * L::UNIT + (uint32_t)(r & 63) * 128u;
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
                if (++qu == TP_UNITS) {
                    qu = 0;
                    qph ^= 1;
                }
            }
            if (!ok) break;
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(qtmem);
            {  // on to the next item's first unit
                const int n = u + 6 + 3 * t.tiles;
                uph ^= (n / TP_UNITS) & 1;
                u = n % TP_UNITS;
            }
            const unsigned long long see = t.see[half];
            float m_run = -INFINITY, l_run = 0.f;
            for (int i = 0; i < t.tiles; ++i, ++gt) {
                const int s = gt & 1;
                if (!(ok = mbar_wait_fast(sfull + s, (uint32_t)(gt >> 1) & 1u, 79))) break;
                tc_fence_after();
                float sv[64];
                tmem_ld64(tmem + lanes + TP_TM_S + (uint32_t)(s * TA_TILE), sv);
                tc_fence_before();
                mbar_arrive(sfree + s);
                const unsigned long long bits = tree_tile_mask(see, t.pos0 + i * TA_TILE, t.ctx) & ~lost_sh[gt & 7];
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (bits == ~0ull) {
#pragma unroll
                    for (int j = 0; j < 64; ++j) {
                        sv[j] *= p.scale_log2;
                        top[j & 3] = fmaxf(top[j & 3], sv[j]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 64; ++j) {
                        sv[j] = (bits >> j) & 1 ? sv[j] * p.scale_log2 : -INFINITY;
                        top[j & 3] = fmaxf(top[j & 3], sv[j]);
                    }
                }
                const float tmax = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                const float m_new = (m_run == -INFINITY || tmax > m_run + PF_RESCALE_LOG2) ? tmax : m_run;
                const float m_use = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = m_run == -INFINITY ? 0.f : exp2_ftz(m_run - m_new);
                // P's place here and there: the P.V of two tiles before has read it
                if (gt >= 2 && !(ok = mbar_wait_cluster(pfree + s, (uint32_t)((gt >> 1) - 1) & 1u, 80))) break;
                const uint32_t prow = base + L::OFF_PS + s * L::P + (uint32_t)r * 128u;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t w[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float e0 = exp2_ftz(sv[8 * c + 2 * x] - m_use), e1 = exp2_ftz(sv[8 * c + 2 * x + 1] - m_use);
                        const __nv_bfloat162 b2 = __floats2bfloat162_rn(e0, e1);
                        w[x] = *reinterpret_cast<const uint32_t*>(&b2);
                        sum[x] += e0 + e1;
                    }
                    sts_v4(prow + (uint32_t)((c ^ r) & 7) * 16u, make_uint4(w[0], w[1], w[2], w[3]));
                }
                // O moves to the new maximum only after the item's first tile
                alpha_sh[128 * s + r] = i == 0 || m_new == m_run ? 1.f : alpha;
                l_run = l_run * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
                m_run = m_new;
                fence_proxy_async_smem();  // P and the factors leave by an async copy
                mbar_arrive(pstaged + s);
            }
            if (!ok) break;
            const bool any = l_run != 0.f;  // (NaN counts: it reaches the result)
            if (half < t.rows) {
                const float lse = any ? (m_run + log2f(l_run)) * 0.69314718055994531f : -INFINITY;
                const int h = r & 63;
                if (t.part >= 0) p.lse_part[(long long)(t.part + half * t.runs) * AT_H + h] = lse;
                else if (p.lse) p.lse[(long long)(t.row0 + half) * AT_H + h] = lse;
            }
            if (k >= 1 && !(ok = mbar_wait_cluster(finfree, (uint32_t)(k - 1) & 1u, 81))) break;
            dsmem_st_f32(dsmem_addr(fin_sh + r, 1), any ? 1.f / l_run : 0.f);
            mbar_arrive_remote(dsmem_addr(finfull, 1));
        }
    } else if (warp == 5) {
        // ---------------- value CTA: P V ----------------
        int v = 0, vph = 0, gt = 0;
        for (int k = 0; ok; ++k) {
            TpItem t;
            if (!(ok = take(k, t)) || t.rows == 0) break;
            for (int i = 0; i < t.tiles && ok; ++i, ++gt) {
                const int b = gt & 1;
                if (!(ok = mbar_wait_fast(pok, (uint32_t)gt & 1u, 82) && mbar_wait_fast(pfull + b, (uint32_t)(gt >> 1) & 1u, 82))) break;
                const uint64_t p0 = desc_sw128(base + L::OFF_P + b * L::P, 16, 1024);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (!(ok = mbar_wait_fast(vfull + 2 * v + half, (uint32_t)vph, 83))) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t v0 = desc_sw128(base + v * L::VTILE + half * L::HALF, L::CHUNK, 1024);
#pragma unroll
                        for (int ks = 0; ks < TA_TILE / 16; ++ks)
                            mma_bf16(tmem + (uint32_t)(half * 256), p0 + ks * 2, v0 + ((ks * 2048) >> 4), L::IDESC_PV, (i > 0 || ks > 0) ? 1u : 0u);
                        if (i + 1 < t.tiles) mma_commit(vfree + 2 * v + half);  // the item's last: its output goes through this space
                        if (half == 1) mma_commit(pvdone + b);
                    }
                    __syncwarp();
                }
                if (++v == TP_VBUF) {
                    v = 0;
                    vph ^= 1;
                }
            }
        }
    } else if (warp == 6) {
        // ---------------- value CTA: P's space is free again ----------------
        int gt = 0;
        for (int k = 0; ok; ++k) {
            TpItem t;
            if (!(ok = take(k, t)) || t.rows == 0) break;
            for (int i = 0; i < t.tiles; ++i, ++gt) {
                if (!(ok = mbar_wait_fast(pvdone + (gt & 1), (uint32_t)(gt >> 1) & 1u, 84))) break;
                if (elect_one()) mbar_arrive_remote(dsmem_addr(pfree + (gt & 1), 0));
                __syncwarp();
            }
        }
    } else {
        // ---------------- value CTA: rescale and output, one row a thread (warps 0-3) ----------------
        const int r = tid, half = r >> 6;
        const uint32_t lanes = (uint32_t)(32 * warp) << 16;
        int v = 0, vph = 0, gt = 0;
        for (int k = 0; ok; ++k) {
            TpItem t;
            if (!(ok = take(k, t)) || t.rows == 0) break;
            int last_v = 0;
            for (int i = 0; i < t.tiles; ++i, ++gt) {
                const int b = gt & 1, pos = t.pos0 + i * TA_TILE;
                if (!(ok = mbar_wait_fast(pfull + b, (uint32_t)(gt >> 1) & 1u, 85))) break;
                if (tid == 0) mbar_expect_tx(pfull + b, L::COPY);  // for the P of two tiles on
                const float alpha = alpha_sh[128 * b + r];
                const unsigned long long lost = lost_sh[gt & 7];
                if (pos + TA_TILE > t.ctx || lost != 0) {  // rows that not both nodes see
                    if (!(ok = mbar_wait_fast(vfull + 2 * v, (uint32_t)vph, 86) && mbar_wait_fast(vfull + 2 * v + 1, (uint32_t)vph, 86))) break;
                    const unsigned long long m0 = tree_tile_mask(t.see[0], pos, t.ctx) & ~lost, m1 = tree_tile_mask(t.see[1], pos, t.ctx) & ~lost;
                    for (int j = warp; j < TA_TILE; j += 4) {
                        if (((m0 & m1) >> j) & 1) continue;
                        const bool one = ((m0 | m1) >> j) & 1;
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const uint32_t at = base + v * L::VTILE + (uint32_t)((lane >> 3) + 4 * x) * L::CHUNK + (uint32_t)j * 128u + (uint32_t)(lane & 7) * 16u;
                            uint4 w = make_uint4(0, 0, 0, 0);
                            if (one) {
                                w = lds_v4(at);
                                w = make_uint4(clear_nonfinite(w.x), clear_nonfinite(w.y), clear_nonfinite(w.z), clear_nonfinite(w.w));
                            }
                            sts_v4(at, w);
                        }
                    }
                    fence_proxy_async_smem();
                }
                if (__any_sync(0xffffffffu, alpha != 1.f)) {
                    if (gt >= 1 && !(ok = mbar_wait_fast(pvdone + (b ^ 1), (uint32_t)((gt - 1) >> 1) & 1u, 87))) break;
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
                tc_fence_before();
                mbar_arrive(pok);
                last_v = v;
                if (++v == TP_VBUF) {
                    v = 0;
                    vph ^= 1;
                }
            }
            if (!ok) break;
            if (!(ok = mbar_wait_fast(pvdone + ((gt - 1) & 1), (uint32_t)((gt - 1) >> 1) & 1u, 88) && mbar_wait_cluster(finfull, (uint32_t)k & 1u, 89))) break;
            tc_fence_after();
            const float inv = fin_sh[r];
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(dsmem_addr(finfree, 0));
            // O / l through the last tile's space, 128-byte pieces of this warp's 32 rows in four boxes of 4 KB
            const bool narrow = t.part < 0 && p.ctx_bf16, there = half < t.rows;
            const int y = (t.part >= 0 ? t.part + half * t.runs : t.row0 + half) * AT_H + 32 * (warp & 1);
            const uint32_t space = base + last_v * L::VTILE + warp * 16384u, mine = space + (uint32_t)lane * 128u;
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
#pragma unroll
                for (int x = 0; x < 64; ++x) o[x] *= inv;
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
                    mbar_arrive(vfree + 2 * last_v);
                    mbar_arrive(vfree + 2 * last_v + 1);
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
    if (warp == 5) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace wl
