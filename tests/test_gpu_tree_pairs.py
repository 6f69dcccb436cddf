"""Attention of drafted trees where its schedule works on more than 32 requests, on long contexts and on large pools, for
the kernels that take one node, two nodes and lists, against 64 bits (tolerances as in test_gpu_paged)."""
import numpy as np
import pytest
import torch

from test_gpu_paged import T_MAX, Trees, clean_device_error, i32  # noqa: F401
from windlass_b200 import attn as A
from windlass_b200 import paged as P

pytestmark = pytest.mark.gpu


def pairs(t):
    """The call goes to pairs of CTAs (enough nodes, nodes a request, and keys as the table's width bounds them)."""
    assert t.n >= 12 and t.n >= 6 * len(t.ctx) and t.n * (20480 + t.page) >= 160 * 1024


@pytest.mark.parametrize("B,long_at", [(33, 32), (33, 0), (64, 40), (65, 63), (100, 97), (130, 64)])
@pytest.mark.parametrize("page", [16, 64])
def test_pairs_over_more_than_32_requests(B, long_at, page):
    """Requests without nodes, odd trees, and one that is cut into parts, in every block of 32 requests."""
    rng = np.random.default_rng(B + long_at)
    ctx, nodes = rng.integers(0, 300, B), rng.integers(6, 14, B)
    nodes[rng.random(B) < 0.1] = 0
    ctx[long_at], nodes[long_at] = 6000, 17
    ctx[(long_at + 7) % B], nodes[(long_at + 7) % B] = 3500, 64
    t = Trees(ctx.tolist(), nodes.tolist(), page, seed=B)
    pairs(t)
    got = t.call(out_dtype=torch.bfloat16 if page == 64 else torch.float32)
    t.check(got)
    for _ in range(5):
        again = t.call(out_dtype=got["ctx"].dtype)
        assert torch.equal(again["ctx"], got["ctx"]) and torch.equal(again["lse"], got["lse"])


def test_the_most_requests():
    """The schedule's table at its full size in the key tiles' space (one node at a time): most requests have nothing to do."""
    B = 16384
    nodes, ctx = np.zeros(B, np.int64), np.zeros(B, np.int64)
    nodes[[5, 31, 32, 9000, B - 1]], ctx[[5, 31, 32, 9000, B - 1]] = [64, 13, 1, 30, 7], [100, 2000, 0, 64, 333]
    t = Trees(ctx.tolist(), nodes.tolist(), 16, seed=2)
    t.wide = False
    t.check(t.call())


@pytest.mark.parametrize("B", [33, 70, 160])
def test_lists_of_more_than_32_requests(B):
    rng = np.random.default_rng(B)
    ctx, nodes = rng.integers(0, 900, B), rng.integers(0, 4, B)
    ctx[B - 1], nodes[B - 1] = 5000, 3
    t = Trees(ctx.tolist(), nodes.tolist(), 16, seed=B)
    sel = [rng.permutation(ctx[b] + nodes[b])[:rng.integers(0, 700)] for b in range(B) for _ in range(nodes[b])]
    sel[-1], sel[0] = rng.permutation(5003)[:4100], np.zeros(0, np.int64)
    lst = np.full((t.n, 4100), -1, np.int32)
    for r, x in enumerate(sel):
        lst[r, :len(x)] = x
    counts = i32([len(x) for x in sel])
    got = t.call(sel_in=i32(lst), sel_n_in=counts)
    t.check(got, sel=sel)
    again = t.call(sel_in=i32(lst), sel_n_in=counts)
    assert torch.equal(again["ctx"], got["ctx"]) and torch.equal(again["lse"], got["lse"])


@pytest.mark.parametrize("ctx,nodes,page", [([20011], [15], 64), ([9001, 30, 16384], [13, 6, 24], 48)])
def test_pairs_over_long_contexts(ctx, nodes, page):
    t = Trees(ctx, nodes, page, seed=5)
    pairs(t)
    t.check(t.call(out_dtype=torch.bfloat16))


def test_pairs_past_32_bits():
    """The last pages of a pool of more than 2^32 elements, two nodes at a time and as lists."""
    t = Trees([300], [13], 64, seed=12, pages=120000)
    t.table[0, :5] = [119999, 0, 119998, 117000, 119990]
    pairs(t)
    got, pos = t.call(out_dtype=torch.bfloat16), np.arange(313)
    slots = torch.from_numpy(t.table[0][pos // 64].astype(np.int64) * 64 + pos % 64).cuda()
    small = torch.zeros(40 * 8, 576, device="cuda", dtype=torch.bfloat16)
    small[:313] = torch.cat([t.c_kv[slots], t.k_rot[slots]], 1)
    t.c_kv, t.k_rot, t.table, t.page = small[:, :512], small[:, 512:], np.arange(40, dtype=np.int32)[None], 8
    t.check(got)


def test_graphs_of_pairs_replayed_on_two_streams_at_once():
    t = Trees([900, 300, 20], [14, 13, 9], 16, seed=17)
    pairs(t)
    cfg, kv = A.glm52_cfg(T_MAX), t.kv()
    ctx_len, cu, par = i32(t.ctx), i32(t.cu), i32(t.parent)
    call = lambda: P.mla_tree_attn(cfg, kv, t.q, ctx_len, cu, parent=par)  # noqa: E731
    call()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for lengths in ([900, 300, 20], [64, 1, 0], [0, 299, 19]):
        ctx_len.copy_(i32(lengths))
        t.ctx = lengths
        torch.cuda.synchronize()
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        for _ in range(5):
            with torch.cuda.stream(s1):
                graphs[0].replay()
            with torch.cuda.stream(s2):
                graphs[1].replay()
        torch.cuda.synchronize()
        t.check(outs[0])
        assert torch.equal(outs[0]["ctx"], outs[1]["ctx"]) and torch.equal(outs[0]["lse"], outs[1]["lse"])
