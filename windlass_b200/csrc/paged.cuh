// paged.cuh — the bookkeeping of a paged cache and of drafted trees: block
// tables and slot maps from request lengths, pages given back, and the commit
// of an accepted path.
//
// All of it moves a few kilobytes, so it is bound by latency: chains of
// dependent loads and launches. Each operator is one launch (a plan with many
// tokens two), its sums run in shared memory, and every result is a fixed
// function of the inputs (no atomics decide an order). Measured: a plan of 64
// requests with 795 tokens 4.9 us (with their trees by parents 5.4, by masks 5.0),
// of 24 prompts with 73K tokens 8.2 us; 8,192 pages of 64 requests given back 7.3
// us; a commit of 8 requests in 78 layers 3.3 us, of 64 in one owner layer 4.9 us.
#pragma once
#include "ptx.cuh"

namespace wl {

constexpr int TREE_MAX = 64;      // drafted nodes of one request (one bit each in a 64-bit mask)
constexpr int PLAN_THREADS = 1024;

struct PlanParams {
    int batch, n_tokens, page_size, n_pages;
    const int* ctx_len;
    const int* n_new;
    int* table;
    long long table_stride;
    int max_pages;
    const int* held;
    int* held_out;
    const int* free_list;
    const int* n_free;
    int* n_free_out;
    int* cu;
    int* lack;
    int* slot;
    int* pos;
    int* seq;
    const int* parent;               // with one of these, pos counts a drafted token's ancestors, not its predecessors
    const unsigned long long* mask;
    int own_tokens;  // the plan kernel writes the token rows too
};

// Inclusive sum over the block of a pair of values (PLAN_THREADS threads).
__device__ __forceinline__ longlong2 block_scan2(longlong2 v, longlong2* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, v.x, o), y = __shfl_up_sync(0xffffffffu, v.y, o);
        if (lane >= o) {
            v.x += x;
            v.y += y;
        }
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
        longlong2 w = lane < PLAN_THREADS / 32 ? warp_sums[lane] : make_longlong2(0, 0);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, w.x, o), y = __shfl_up_sync(0xffffffffu, w.y, o);
            if (lane >= o) {
                w.x += x;
                w.y += y;
            }
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    if (warp > 0) {
        v.x += warp_sums[warp - 1].x;
        v.y += warp_sums[warp - 1].y;
    }
    __syncthreads();  // warp_sums is reused
    return v;
}

// Last index b of [lo, hi) with a[b] <= x (a ascending, a[lo] <= x).
__device__ __forceinline__ int last_le(const int* a, int lo, int hi, int x) {
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Slot of position `pos` by a table row; -1 (and the error word) for an entry outside the pool.
__device__ __forceinline__ int page_slot(const int* row, int page_size, int n_pages, int pos, unsigned site) {
    const int page = row[pos / page_size];
    if (page < 0 || page >= n_pages) {
        set_error(ERRC_BOUNDS, site);
        return -1;
    }
    return page * page_size + pos % page_size;
}

// Depth of node j of a request's tree (`parent` from its first row on): the number of its ancestors, which stand
// before it. A parent that does not sets the error word and counts as none, as in the attention's masks. (A load an
// ancestor, from L1 after the first: 8 requests with chains of up to 64 7.8 us a plan, with trees 5.6, without 4.2.)
__device__ __forceinline__ int plan_depth(const int* parent, int j) {
    int d = 0;
    for (int at = j;;) {
        const int up = __ldg(parent + at);
        if (up < 0) return d;
        if (up >= at) {
            set_error(ERRC_BOUNDS, 45);
            return d;
        }
        at = up;
        ++d;
    }
}

// One token row (shared by the plan kernel and plan_tokens_kernel): token i, of n that request b has from row
// `first` on. Its cache row goes by its number in the request; its position in the text is that of a branch, so
// siblings share one (a request of more than TREE_MAX tokens is a prompt: a line).
__device__ __forceinline__ void plan_token(const PlanParams& p, int i, int b, int first, int n, int lack, int ctx) {
    const int j = i - first, pos = ctx + j;
    int deep = j;
    if (n <= TREE_MAX) {
        if (p.parent) deep = plan_depth(p.parent + first, j);
        else if (p.mask) deep = __popcll(p.mask[i] & (n >= 64 ? ~0ull : (1ull << n) - 1) & ~(1ull << j));
    }
    p.slot[i] = lack != 0 ? -1 : page_slot(p.table + (long long)b * p.table_stride, p.page_size, p.n_pages, pos, 41);
    p.pos[i] = ctx + deep;
    p.seq[i] = b;
}

// The whole plan in one CTA: per request its missing pages and tokens, two
// running sums over the requests (PLAN_THREADS at a time), then the pages and,
// for small plans, the token rows, spread over the threads by binary search.
__global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(PlanParams p) {
    pdl_wait();
    pdl_trigger();
    __shared__ longlong2 warp_sums[32];
    __shared__ int sh_page[PLAN_THREADS + 1];  // first new page of each request of the block (call-wide numbering)
    __shared__ int sh_tok[PLAN_THREADS + 1];   // first token
    __shared__ int sh_lack[PLAN_THREADS];
    __shared__ int sh_held[PLAN_THREADS];
    __shared__ int sh_total[PLAN_THREADS];     // table entries a request without its pages loses
    __shared__ int sh_ctx[PLAN_THREADS];
    __shared__ int sh_last[2];                 // new pages and tokens served so far
    const int tid = threadIdx.x;
    int n_free = p.n_free[0];
    if (n_free < 0 || n_free > p.n_pages) {
        if (tid == 0) set_error(ERRC_BOUNDS, 41);
        n_free = n_free < 0 ? 0 : p.n_pages;
    }
    long long carry_page = 0, carry_tok = 0;
    if (tid == 0) sh_last[0] = 0;
    for (int b0 = 0; b0 < p.batch; b0 += PLAN_THREADS) {
        const int b = b0 + tid, nb = min(PLAN_THREADS, p.batch - b0);
        long long need = 0, total = 0;
        int lack = 0, held = 0, ctx = 0, fresh = 0;
        if (b < p.batch) {
            ctx = p.ctx_len[b];
            fresh = p.n_new[b];
            held = p.held[b];
            if (ctx < 0 || fresh < 0 || held < 0 || held > p.max_pages || (long long)ctx + fresh > 0x7fffffff) {
                set_error(ERRC_BOUNDS, 41);
                lack = -1;
                fresh = 0;
            } else {
                total = ((long long)ctx + fresh + p.page_size - 1) / p.page_size;
                need = total > held ? total - held : 0;
                if (total > p.max_pages) {  // the table row is too narrow: takes nothing from the pool
                    lack = (int)min(need, (long long)0x7fffffff);
                    need = 0;
                }
            }
        }
        const longlong2 s = block_scan2(make_longlong2(need, fresh), warp_sums);
        const long long page0 = carry_page + s.x - need, tok0 = carry_tok + s.y - fresh;
        if (lack == 0 && need > 0 && page0 + need > n_free) lack = (int)need;
        const int got = lack == 0 ? (int)need : 0;
        // served requests are a prefix of those that need pages, so their page
        // numbers are dense and every later start is clamped to their end
        sh_page[tid] = (int)min(page0, (long long)0x7fffffff);
        sh_tok[tid] = (int)min(tok0, (long long)0x7fffffff);
        sh_lack[tid] = lack;
        sh_held[tid] = held;
        sh_total[tid] = lack > 0 ? (int)min(total, (long long)p.max_pages) : 0;
        sh_ctx[tid] = ctx;
        if (tid == nb - 1) {
            sh_page[nb] = (int)min(page0 + need, (long long)0x7fffffff);
            sh_tok[nb] = (int)min(tok0 + fresh, (long long)0x7fffffff);
        }
        if (b < p.batch) {
            p.cu[b] = (int)min(tok0, (long long)0x7fffffff);
            p.lack[b] = lack;
            if (got > 0) atomicMax(&sh_last[0], (int)(page0 + need));
            p.held_out[b] = held + got;  // after this thread's own read of held[b]
        }
        carry_page += warp_sums[31].x;
        carry_tok += warp_sums[31].y;
        __syncthreads();
        // new pages [sh_page[0], end of the last served request)
        const int k1 = min(sh_page[nb], sh_last[0]);
        for (int k = sh_page[0] + tid; k < k1; k += PLAN_THREADS) {
            const int j = last_le(sh_page, 0, nb, k);
            const int page = p.free_list[n_free - 1 - k];
            p.table[(long long)(b0 + j) * p.table_stride + sh_held[j] + (k - sh_page[j])] = page;
        }
        // a request that went without: nothing may be read or moved through entries that an earlier owner left
        for (int j = tid >> 5; j < nb; j += PLAN_THREADS / 32)
            for (int k = sh_held[j] + (tid & 31); k < sh_total[j]; k += 32) p.table[(long long)(b0 + j) * p.table_stride + k] = -1;
        if (p.own_tokens) {
            __syncthreads();  // the tokens read the table rows written above
            const int t1 = min(sh_tok[nb], p.n_tokens);
            for (int i = sh_tok[0] + tid; i < t1; i += PLAN_THREADS) {
                const int j = last_le(sh_tok, 0, nb, i);
                plan_token(p, i, b0 + j, sh_tok[j], sh_tok[j + 1] - sh_tok[j], sh_lack[j], sh_ctx[j]);
            }
        }
        __syncthreads();  // shared arrays are reused
    }
    if (tid == 0) {
        p.cu[p.batch] = (int)min(carry_tok, (long long)0x7fffffff);
        p.n_free_out[0] = n_free - sh_last[0];
        if (carry_tok > p.n_tokens) set_error(ERRC_BOUNDS, 41);
    }
    if (p.own_tokens)
        for (long long i = carry_tok + tid; i < p.n_tokens; i += PLAN_THREADS) p.slot[i] = p.pos[i] = p.seq[i] = -1;
}

// Token rows of a large plan: one thread a row, its request by binary search in cu.
__global__ void __launch_bounds__(256) plan_tokens_kernel(PlanParams p) {
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= p.n_tokens) return;
    if (i >= p.cu[p.batch]) {
        p.slot[i] = p.pos[i] = p.seq[i] = -1;
        return;
    }
    const int b = last_le(p.cu, 0, p.batch, i);
    plan_token(p, i, b, p.cu[b], p.cu[b + 1] - p.cu[b], p.lack[b], p.ctx_len[b]);
}

struct ReleaseParams {
    int batch;
    const int* done;
    const int* table;
    long long table_stride;
    int max_pages;
    int* held;
    int* free_list;
    int n_pages;
    int* n_free;
};

__global__ void __launch_bounds__(PLAN_THREADS) page_release_kernel(ReleaseParams p) {
    pdl_wait();
    pdl_trigger();
    __shared__ longlong2 warp_sums[32];
    __shared__ int sh_page[PLAN_THREADS + 1];
    const int tid = threadIdx.x;
    long long base = p.n_free[0];
    if (base < 0 || base > p.n_pages) {
        if (tid == 0) set_error(ERRC_BOUNDS, 42);
        base = base < 0 ? 0 : p.n_pages;
    }
    for (int b0 = 0; b0 < p.batch; b0 += PLAN_THREADS) {
        const int b = b0 + tid, nb = min(PLAN_THREADS, p.batch - b0);
        int n = 0;
        if (b < p.batch && p.done[b] != 0) {
            n = p.held[b];
            if (n < 0 || n > p.max_pages) {
                set_error(ERRC_BOUNDS, 42);
                n = 0;
            }
            p.held[b] = 0;
        }
        const longlong2 s = block_scan2(make_longlong2(n, 0), warp_sums);
        sh_page[tid] = (int)min(s.x - n, (long long)0x7fffffff);
        if (tid == nb - 1) sh_page[nb] = (int)min(s.x, (long long)0x7fffffff);
        const long long all = warp_sums[31].x;
        __syncthreads();
        for (int k = tid; k < sh_page[nb]; k += PLAN_THREADS) {
            const int j = last_le(sh_page, 0, nb, k);
            if (base + k < p.n_pages) p.free_list[base + k] = p.table[(long long)(b0 + j) * p.table_stride + (k - sh_page[j])];
            else set_error(ERRC_BOUNDS, 42);
        }
        base += all;
        __syncthreads();
    }
    if (tid == 0) p.n_free[0] = (int)(base < p.n_pages ? base : p.n_pages);
}

// ---- the commit of an accepted path ----------------------------------------------------
constexpr int COMMIT_LAYERS = 80;   // layers of one launch (their pointers travel as a kernel argument of 4 KB at most)
constexpr int COMMIT_THREADS = 96;  // one 16-byte piece of a layer's rows each: 64 c_kv, 8 k_rot, 8 key, 1 scale

struct CommitLayer {
    __nv_bfloat16* c_kv;
    __nv_bfloat16* k_rot;
    uint8_t* keys;  // null: the layer owns no indexer
    float* scale;
    long long ckv_row, krot_row;
};
struct CommitParams {
    int n_nodes;
    const int* ctx_len;
    const int* cu;
    const int* parent;
    const int* draft;
    const int* target;
    int page_size, n_pages;
    const int* table;
    long long table_stride;
    int max_pages;
    int* n_accept;
    int* path;
    int* next;
    int* ctx_out;
    int first;     // this launch writes the outputs (the walk is the same in every launch)
    int n_layers;  // layers of this launch
    CommitLayer layer[COMMIT_LAYERS];
};
static_assert(sizeof(CommitParams) <= 4096, "kernel arguments");

// grid (layers or 1, batch). Warp 0 walks the request's tree in registers (two
// nodes a lane, one ballot a step); every thread then owns one 16-byte column
// of the layer's rows and moves it along the path in ascending order, eight
// rows read before eight are written: the d-th node of the path has an index
// >= d, so a row is written only after it has been read as a source.
__global__ void __launch_bounds__(COMMIT_THREADS) tree_commit_kernel(const __grid_constant__ CommitParams p) {
    pdl_wait();
    pdl_trigger();
    __shared__ int src_sh[TREE_MAX], dst_sh[TREE_MAX];  // slots, -1 past the path
    __shared__ int n_sh;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    if (tid < 32) {
        const int r0 = p.cu[b], r1 = p.cu[b + 1], ctx = p.ctx_len[b];
        int n = r1 - r0;
        if (r0 < 0 || r1 > p.n_nodes || n < 0 || n > TREE_MAX || ctx < 0 ||
            (long long)ctx + n > min((long long)p.max_pages * p.page_size, 0x7fffffffll)) {
            if (lane == 0) set_error(ERRC_BOUNDS, 43);
            n = 0;
        }
        // The cache row of every drafted node, before the walk: a request without a page under one of them (a plan with too
        // few pages leaves such) wrote nothing, so nothing of it is committed.
        const int* row = p.table + (long long)b * p.table_stride;
        int par[2], tok[2], tgt[2], slot[2];
        bool bad = false;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int j = lane + 32 * k;
            par[k] = j < n ? p.parent[r0 + j] : -2;
            tok[k] = j < n ? p.draft[r0 + j] : 0;
            tgt[k] = j < n ? p.target[r0 + j] : 0;
            slot[k] = j < n ? page_slot(row, p.page_size, p.n_pages, ctx + j, 43) : 0;
            bad |= slot[k] < 0;
        }
        if (__any_sync(0xffffffffu, bad)) n = 0;
        int cur = 0, cnt = 0, want = -1, mine[2] = {-1, -1};
        while (cnt < n) {
            if (lane == (cnt & 31)) mine[cnt >> 5] = cur;
            ++cnt;
            const int t0 = __shfl_sync(0xffffffffu, tgt[0], cur & 31), t1 = __shfl_sync(0xffffffffu, tgt[1], cur & 31);
            want = cur < 32 ? t0 : t1;
            const unsigned m0 = __ballot_sync(0xffffffffu, par[0] == cur && tok[0] == want && lane > cur);
            const unsigned m1 = __ballot_sync(0xffffffffu, par[1] == cur && tok[1] == want && lane + 32 > cur);
            if (!(m0 | m1)) break;
            cur = m0 ? __ffs(m0) - 1 : 31 + __ffs(m1);
        }
        const bool write = p.first && blockIdx.x == 0;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int d = lane + 32 * k;
            const int from = mine[k] < 0 ? 0 : mine[k];
            const int s0 = __shfl_sync(0xffffffffu, slot[0], from & 31), s1 = __shfl_sync(0xffffffffu, slot[1], from & 31);
            // a node already in place does not move
            const int s = mine[k] > d ? (from < 32 ? s0 : s1) : -1, t = slot[k];
            src_sh[d] = s;
            dst_sh[d] = t;
            if (write) p.path[(long long)b * TREE_MAX + d] = mine[k];
        }
        if (lane == 0) {
            n_sh = cnt;
            if (write) {
                p.n_accept[b] = cnt;
                p.next[b] = n > 0 ? want : -1;
                p.ctx_out[b] = ctx + cnt;
            }
        }
    }
    if (p.n_layers == 0) return;
    __syncthreads();
    const CommitLayer& c = p.layer[blockIdx.x];
    const int n = n_sh;
    if (tid < 80) {
        char* base;
        long long stride;  // bytes
        if (tid < 64) {
            base = reinterpret_cast<char*>(c.c_kv) + tid * 16;
            stride = c.ckv_row * 2;
        } else if (tid < 72) {
            base = reinterpret_cast<char*>(c.k_rot) + (tid - 64) * 16;
            stride = c.krot_row * 2;
        } else {
            if (!c.keys) return;
            base = reinterpret_cast<char*>(c.keys) + (tid - 72) * 16;
            stride = 128;
        }
        for (int d0 = 0; d0 < n; d0 += 8) {
            uint4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (d0 + k < n && src_sh[d0 + k] >= 0) v[k] = *reinterpret_cast<const uint4*>(base + src_sh[d0 + k] * stride);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (d0 + k < n && src_sh[d0 + k] >= 0) *reinterpret_cast<uint4*>(base + dst_sh[d0 + k] * stride) = v[k];
        }
    } else if (tid == 80 && c.keys) {
        for (int d = 0; d < n; ++d)
            if (src_sh[d] >= 0) c.scale[dst_sh[d]] = c.scale[src_sh[d]];
    }
}

}  // namespace wl
