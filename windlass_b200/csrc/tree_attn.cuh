// tree_attn.cuh — absorbed-MLA attention of drafted trees over a paged latent cache.
//
// Row r = node i of request b sees the positions t < ctx_b and the nodes of its
// own ancestor mask (position ctx_b + j):
//     s[h,t] = (q_abs[r,h] . [c_kv | k_rot][slot(b,t)]) * softmax_scale
//     ctx[r,h] = sum_t softmax_t(s[h,t]) c_kv[slot(b,t)],  lse[r,h] = log sum_t e^s[h,t]
// or only those of them that its selection list names.
#pragma once
#include "mla_attn.cuh"
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

// The nodes that node j of a request sees (bits past the request's nodes cleared).
__device__ __forceinline__ unsigned long long tree_mask_of(const TreeParams& p, const TreeSeq& s, int j) {
    const unsigned long long all = s.n >= 64 ? ~0ull : (1ull << s.n) - 1;
    if (p.mask) return p.mask[s.r0 + j] & all;
    if (!p.parent) return all & (j >= 63 ? ~0ull : (2ull << j) - 1);
    unsigned long long m = 1ull << j;
    int at = j;
    while (true) {
        const int up = p.parent[s.r0 + at];
        if (up < 0) break;
        if (up >= at) {  // not an earlier node
            set_error(ERRC_BOUNDS, 45);
            break;
        }
        m |= 1ull << up;
        at = up;
    }
    return m;
}

// The plain kernel: grid (n_nodes, 8), a warp per head, the keys one after the
// other with a running maximum and sum; lane l holds columns l + 32 k.
__global__ void __launch_bounds__(256) tree_attn_simple_kernel(TreeParams p) {
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.x, h = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= p.cu[p.batch]) return;
    const int b = last_le(p.cu, 0, p.batch, r);
    const TreeSeq s = tree_seq(p, b);
    const int i = r - s.r0;
    if (i < 0 || i >= s.n) return;
    const unsigned long long see = tree_mask_of(p, s, i);
    float q[18], o[16];
    const __nv_bfloat16* qr = p.q + ((long long)r * AT_H + h) * AT_D;
#pragma unroll
    for (int k = 0; k < 18; ++k) q[k] = __bfloat162float(qr[lane + 32 * k]) * p.scale_log2;
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = 0.f;
    float m = -INFINITY, l = 0.f;
    const int* row = p.table + (long long)b * p.table_stride;
    const int count = p.sel ? (p.sel_n_dev ? p.sel_n_dev[r] : p.sel_n) : s.ctx + s.n;
    for (int e = 0; e < count; ++e) {
        const int t = p.sel ? p.sel[(long long)r * p.sel_stride + e] : e;
        if (t < 0 || t >= s.ctx + s.n || (t >= s.ctx && !((see >> (t - s.ctx)) & 1))) continue;
        const int slot = page_slot(row, p.page_size, p.n_pages, t, 46);
        if (slot < 0) continue;
        float k[18], dot = 0.f;
#pragma unroll
        for (int c = 0; c < 18; ++c) {
            k[c] = __bfloat162float(c < 16 ? p.c_kv[slot * p.ckv_row + lane + 32 * c] : p.k_rot[slot * p.krot_row + lane + 32 * (c - 16)]);
            dot = fmaf(q[c], k[c], dot);
        }
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, w);
        const float m_new = fmaxf(m, dot), f = exp2f(m - m_new), w = exp2f(dot - m_new);
        m = m_new;
        l = l * f + w;
#pragma unroll
        for (int c = 0; c < 16; ++c) o[c] = fmaf(w, k[c], o[c] * f);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int c = 0; c < 16; ++c) {
        const long long at = ((long long)r * AT_H + h) * AT_DV + lane + 32 * c;
        if (p.ctx_bf16) static_cast<__nv_bfloat16*>(p.ctx)[at] = __float2bfloat16_rn(o[c] * inv);
        else static_cast<float*>(p.ctx)[at] = o[c] * inv;
    }
    if (p.lse && lane == 0) p.lse[(long long)r * AT_H + h] = l > 0.f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
}

}  // namespace wl
