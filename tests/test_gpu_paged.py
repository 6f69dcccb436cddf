"""The paged cache and drafted trees on the GPU, against the 64-bit restatement in
oracle/paged_ref.py.

Whole numbers (plans, paths, moved rows) are exact. Attention tolerances count roundings:
P enters the P.V product in bf16 (half a step, 2^-8 of each p), scores and sums are fp32.
A score is a sum of 576 products in at most 36 + 16 roundings of 2^-23 of the running
magnitude (the tensor core adds 16 products at a time), so it is off by at most
DS = 64 * 2^-23 * scale * sum|q k|; e^s and the sums add less than 2^-20. With
A = sum_t p_t |v_t| that bounds |ctx - ref| by (2^-8 + 2 DS + 2^-18) A, plus 2^-8 |ref| for
a bf16 output, and |lse - ref| by DS + 2^-20 (1 + |lse|).
"""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import paged_ref as R
from windlass_b200 import _lib
from windlass_b200 import attn as A
from windlass_b200 import paged as P

pytestmark = pytest.mark.gpu

SCALE = 1 / 16
T_MAX = 1 << 18


@pytest.fixture(autouse=True)
def clean_device_error():
    A.device_error(clear=True)
    yield
    st, word = A.device_error(clear=True)
    assert st == _lib.WL_OK, f"device error word 0x{word:08x}"


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def cpu(t):
    return t.detach().cpu().numpy()


def bad_word():
    st, word = A.device_error(clear=True)
    assert st == _lib.WL_ERR_DEVICE, (st, hex(word))


# ---- plans -----------------------------------------------------------------------------------

def make_plan(rng, B, ctx_max, new_max, page, spare, width=None):
    ctx, new = rng.integers(0, ctx_max + 1, B), rng.integers(0, new_max + 1, B)
    # some requests already hold a page more than their context needs
    held = -(-ctx // page) + (rng.random(B) < 0.3) * (-(-(ctx + new) // page) > -(-ctx // page))
    most = -(-(ctx + new) // page)
    width = int(max(most.max(), held.max(), 1)) if width is None else width
    need = np.maximum(0, most - held).sum()
    n_pages = int(held.sum() + need + 7)
    perm = rng.permutation(n_pages)
    table, at = np.full((B, width), -1, np.int32), 0
    for b in range(B):
        table[b, :held[b]] = perm[at:at + held[b]]
        at += held[b]
    n_free = max(0, int(need) + spare)
    free = np.full(n_pages, -1, np.int32)
    free[:min(n_free, n_pages - at)] = perm[at:at + n_free]
    n_free = min(n_free, n_pages - at)
    return ctx, new, held, table, free, n_free, n_pages


def check_plan(args, page, n_tokens, in_place=False):
    ctx, new, held, table, free, n_free, n_pages = args
    ref = R.page_plan(ctx.tolist(), new.tolist(), held.tolist(), table, free, n_free, page, n_pages, n_tokens)
    t, h, f = i32(table), i32(held), i32([n_free])
    got = P.page_plan(i32(ctx), i32(new), t, h, i32(free), f, page, n_tokens, in_place=in_place)
    for k in ("slot", "pos", "seq", "cu", "short", "n_held"):
        assert np.array_equal(cpu(got[k]), ref[k]), k
    assert int(got["n_free"]) == ref["n_free"]
    assert np.array_equal(cpu(t), ref["table"])
    assert (got["n_held"] is h and got["n_free"] is f) == in_place
    if not in_place:
        assert np.array_equal(cpu(h), held) and int(f) == n_free
    return ref


@pytest.mark.parametrize("B,ctx_max,new_max,page", [(1, 0, 1, 8), (1, 1, 0, 16), (5, 100, 1, 1), (64, 5000, 16, 64),
                                                    (33, 300, 70, 7), (1025, 40, 5, 16), (2500, 9, 3, 4)])
def test_plan_matches_the_restatement(B, ctx_max, new_max, page):
    rng = np.random.default_rng(B + page)
    args = make_plan(rng, B, ctx_max, new_max, page, spare=3)
    total = int(args[1].sum())
    check_plan(args, page, total)
    check_plan(args, page, total + 13, in_place=True)  # a padded batch


@pytest.mark.parametrize("n_tokens", [2048, 2049, 4096, 4097, 9001])
def test_plan_on_both_sides_of_the_second_launch(n_tokens):
    rng = np.random.default_rng(n_tokens)
    B = 11
    args = list(make_plan(rng, B, 500, 10, 16, spare=0))
    new = rng.multinomial(n_tokens, np.ones(B) / B)
    ctx, held = args[0], -(-args[0] // 16)
    most = -(-(ctx + new) // 16)
    n_pages = int(most.sum()) + 2
    perm, table, at = rng.permutation(n_pages), np.zeros((B, int(most.max())), np.int32), 0
    for b in range(B):
        table[b, :held[b]] = perm[at:at + held[b]]
        at += held[b]
    free = np.zeros(n_pages, np.int32)
    free[:n_pages - at] = perm[at:]
    check_plan((ctx, new, held, table, free, n_pages - at, n_pages), 16, n_tokens)


@pytest.mark.parametrize("spare", [-1, -4, -1000])
def test_plan_with_too_few_pages_serves_a_prefix(spare):
    args = make_plan(np.random.default_rng(7), 40, 200, 30, 8, spare)
    ref = check_plan(args, 8, int(args[1].sum()))
    assert (ref["short"] > 0).any()


def test_plan_with_a_narrow_table_leaves_that_request_out():
    rng = np.random.default_rng(8)
    args = list(make_plan(rng, 12, 60, 30, 8, 5, width=20))
    args[1][3] = 200  # more than its table row can hold
    ref = check_plan(tuple(args), 8, int(args[1].sum()))
    assert ref["short"][3] > 0 and (ref["short"] > 0).sum() == 1


def test_plan_flags_bad_lengths_and_overflowing_rows():
    t, f = i32(np.zeros((2, 4))), i32(np.arange(4))
    got = P.page_plan(i32([-1, 3]), i32([2, 2]), t, i32([0, 1]), f, i32([4]), 8, 4)
    assert cpu(got["short"]).tolist() == [-1, 0] and cpu(got["cu"]).tolist() == [0, 0, 2]
    assert cpu(got["slot"]).tolist() == [3, 4, -1, -1]
    bad_word()
    got = P.page_plan(i32([0, 0]), i32([3, 2]), t, i32([0, 0]), f, i32([4]), 8, 4)  # five tokens, four rows
    assert cpu(got["seq"]).tolist() == [0, 0, 0, 1]
    bad_word()


def test_plan_of_a_table_without_rows():
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    got = P.page_plan(e, e, torch.zeros(0, 3, dtype=torch.int32, device="cuda"), e, i32([0, 1]), i32([2]), 8, 3)
    assert cpu(got["cu"]).tolist() == [0] and cpu(got["slot"]).tolist() == [-1] * 3


def test_plan_of_no_requests():
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    got = P.page_plan(e, e, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), e, i32([0, 1]), i32([2]), 8, 3)
    assert cpu(got["cu"]).tolist() == [0] and int(got["n_free"]) == 2 and cpu(got["slot"]).tolist() == [-1] * 3


@pytest.mark.parametrize("B", [1, 7, 1024, 1500])
def test_release_then_plan_hands_the_pages_out_again(B):
    rng = np.random.default_rng(B)
    held = rng.integers(0, 5, B)
    n_pages = int(held.sum()) + 3
    perm, table, at = rng.permutation(n_pages), np.full((B, 5), -1, np.int32), 0
    for b in range(B):
        table[b, :held[b]] = perm[at:at + held[b]]
        at += held[b]
    free = np.full(n_pages, -1, np.int32)
    free[:3] = perm[at:]
    done = (rng.random(B) < 0.5).astype(np.int32)
    h, f, n = i32(held), i32(free), i32([3])
    P.page_release(i32(done), i32(table), h, f, n)
    want = perm[at:].tolist() + [int(p) for b in range(B) if done[b] for p in table[b, :held[b]]]
    assert int(n) == len(want) and cpu(f)[:len(want)].tolist() == want
    assert np.array_equal(cpu(h), np.where(done, 0, held))


# ---- attention -------------------------------------------------------------------------------

class Trees:
    """A pool, block tables and trees of given context lengths and node counts. ``wide``: the table has room for
    long requests, with which trees of many nodes are worked on by pairs of CTAs whatever their lengths."""
    wide = True

    def __init__(self, ctx, nodes, page, seed=0, row=576, split=False, spread=1.0, spare_rows=0, pages=None):
        rng = np.random.default_rng(seed)
        self.ctx, self.nodes, self.page = list(ctx), list(nodes), page
        B = len(self.ctx)
        most = [-(-(c + n) // page) for c, n in zip(ctx, nodes)]
        self.n_pages = sum(most) + 3 if pages is None else pages
        perm = rng.permutation(self.n_pages)[:sum(most)]
        self.table, at = np.zeros((B, max(max(most), 1)), np.int32), 0
        for b in range(B):
            self.table[b, :most[b]] = perm[at:at + most[b]]
            at += most[b]
        self.cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
        self.n = int(self.cu[-1]) + spare_rows
        g = torch.Generator(device="cuda").manual_seed(seed)
        slots = self.n_pages * page
        if split:
            self.c_kv = torch.randn(slots, 512 + row - 576, generator=g, device="cuda", dtype=torch.bfloat16)[:, :512]
            self.k_rot = torch.randn(slots, 64 + 8, generator=g, device="cuda", dtype=torch.bfloat16)[:, :64]
        else:
            kv = torch.randn(slots, row, generator=g, device="cuda", dtype=torch.bfloat16)
            self.c_kv, self.k_rot = kv[:, :512], kv[:, 512:576]
        self.q = (torch.randn(self.n, 64, 576, generator=g, device="cuda") * spread).to(torch.bfloat16)
        self.parent = np.concatenate([[-1] + [rng.integers(max(0, j - 3), j) for j in range(1, n)] if n else []
                                      for n in nodes] + [[0] * spare_rows]).astype(np.int32)
        self.masks = R.tree_masks(self.parent, self.cu)

    def kv(self):
        room = 20480 // self.page + 1 if self.wide else 0
        return P.PagedKV(self.c_kv, self.k_rot, self.page, i32(np.pad(self.table, ((0, 0), (0, room)), constant_values=-7)))

    def call(self, **kw):
        kw.setdefault("parent", i32(self.parent))
        return P.mla_tree_attn(A.glm52_cfg(T_MAX), self.kv(), self.q, i32(self.ctx), i32(self.cu), **kw)

    def rows(self):
        return torch.cat([self.c_kv, self.k_rot], 1).float().cpu().numpy()

    def check(self, got, sel=None, masks=None):
        n = int(self.cu[-1])
        q, rows = self.q.float().cpu().numpy()[:n], self.rows()
        ref, lse, spread = R.tree_attn(q, rows, self.ctx, self.cu, masks or self.masks, self.table, self.page, SCALE, sel)
        # the largest sum of |q k|: over some rows of the pool, with half as much again for the others
        fin = np.where(np.abs(rows) < 1e30, np.abs(rows), 0)
        top = (np.abs(q).reshape(-1, 576) @ fin[:256].T).max() * 1.5
        ds = 64 * 2.0 ** -23 * SCALE * top
        o = got["ctx"].float().cpu().numpy()[:n]
        tol = (2.0 ** -8 + 2 * ds + 2.0 ** -18) * spread + (2.0 ** -8 * np.abs(ref) if got["ctx"].dtype == torch.bfloat16 else 0)
        assert np.isfinite(o).all()
        worst = np.max(np.abs(o - ref) - tol)
        assert worst <= 0, worst
        z, w = cpu(got["lse"])[:n], lse
        assert np.array_equal(np.isneginf(z), np.isneginf(w))
        f = np.isfinite(w)
        assert np.all(np.abs(z[f] - w[f]) <= ds + 2.0 ** -20 * (1 + np.abs(w[f])))


CASES = [
    # ctx, nodes, page
    ([0], [1], 8), ([1], [1], 16), ([62], [1], 64), ([63], [1], 64), ([64], [2], 64), ([127], [3], 16),
    ([128], [64], 64), ([0], [64], 8), ([1000], [1], 64), ([515], [9], 48), ([777], [33], 256), ([90], [5], 24),
    ([0, 65, 3, 700], [3, 0, 17, 1], 16), ([40, 0, 0, 129], [0, 0, 5, 2], 8), ([3000], [4], 32),
    ([5, 260, 1031, 64, 0, 2, 77], [1, 2, 3, 4, 5, 6, 7], 40),
    # trees of many nodes: odd ones, requests without any, tiles that are all drafts
    ([0, 65, 3, 700], [13, 0, 27, 1], 16), ([63, 0], [12, 0], 64), ([0], [63], 8), ([1, 129, 4100], [17, 16, 15], 48),
]


@pytest.mark.parametrize("ctx,nodes,page", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("wide", [True, False])
def test_tree_attention_matches_64_bits(ctx, nodes, page, dtype, wide):
    t = Trees(ctx, nodes, page, seed=len(ctx) + page)
    t.wide = wide
    t.check(t.call(out_dtype=dtype))


@pytest.mark.parametrize("row,split", [(576, True), (640, False), (704, True)])
def test_row_strides(row, split):
    t = Trees([200, 31], [5, 2], 16, seed=row, row=row, split=split)
    t.check(t.call())


@pytest.mark.parametrize("spread", [0.01, 6.0])
@pytest.mark.parametrize("nodes", [[6, 1], [21, 4]])
def test_flat_and_peaked_scores(spread, nodes):
    t = Trees([900, 3], nodes, 16, seed=5, spread=spread)
    t.check(t.call())


@pytest.mark.parametrize("nodes", [[2], [13]])
def test_the_maximum_that_grows_tile_by_tile(nodes):
    """Keys of growing size, so that O is rescaled again and again, in every split."""
    t = Trees([1500], nodes, 64, seed=23)
    pos = np.arange(1500 + nodes[0])
    slots = torch.from_numpy(t.table[0][pos // 64].astype(np.int64) * 64 + pos % 64).cuda()
    grow = torch.linspace(0.05, 6, len(pos), device="cuda")[:, None]
    for pool in (t.c_kv, t.k_rot):
        pool[slots] = (pool[slots].float() * grow).to(torch.bfloat16)
    t.check(t.call())


@pytest.mark.parametrize("scale", [-0.0625, 0.0, 0.3])
@pytest.mark.parametrize("nodes", [[2], [13]])
def test_other_softmax_scales(scale, nodes):
    t = Trees([300], nodes, 16, seed=24, spread=0.3)
    cfg = A.glm52_cfg(T_MAX)
    cfg.softmax_scale = scale
    got = P.mla_tree_attn(cfg, t.kv(), t.q, i32(t.ctx), i32(t.cu), parent=i32(t.parent))
    q, rows = t.q.float().cpu().numpy(), t.rows()
    ref, lse, a = R.tree_attn(q, rows, t.ctx, t.cu, t.masks, t.table, t.page, scale)
    assert np.all(np.abs(cpu(got["ctx"]) - ref) <= (2.0 ** -8 + 1e-3) * a)
    assert np.abs(cpu(got["lse"]) - lse).max() < 1e-3


def test_many_requests_and_long_contexts():
    rng = np.random.default_rng(3)
    t = Trees(rng.integers(0, 400, 90).tolist(), rng.integers(0, 4, 90).tolist(), 16, seed=3)
    t.check(t.call(out_dtype=torch.bfloat16))
    t = Trees([20011, 5], [2, 1], 64, seed=4)
    t.check(t.call())


@pytest.mark.parametrize("B,lo,hi", [(30, 8, 12), (60, 2, 4), (61, 1, 9), (200, 1, 3)])
@pytest.mark.parametrize("wide", [True, False])
def test_more_work_than_a_round_of_the_gpu(B, lo, hi, wide):
    """Every CTA (pair) takes several pieces of work one after the other, of all lengths."""
    rng = np.random.default_rng(B)
    t = Trees(rng.integers(0, 400, B).tolist(), rng.integers(lo, hi, B).tolist(), 16 if B % 2 else 64, seed=B)
    t.wide = wide
    got = t.call()
    t.check(got)
    for _ in range(5):
        again = t.call()
        assert torch.equal(again["ctx"], got["ctx"]) and torch.equal(again["lse"], got["lse"])


def test_a_node_may_see_other_than_its_ancestors_or_nothing():
    t = Trees([0, 70], [6, 4], 16, seed=6)
    masks = [0, 0b10, 0b111111, 0b000001, 0b100000, 0, 0, 0b1000, 0b1111, 0b0101]
    got = t.call(parent=None, mask=torch.tensor(masks, dtype=torch.int64, device="cuda"))
    t.check(got, masks=masks)
    assert (cpu(got["ctx"])[[0, 5]] == 0).all() and np.isneginf(cpu(got["lse"])[[0, 5]]).all()


def test_all_64_bits_of_a_mask():
    t = Trees([10], [64], 16, seed=7)
    masks = [(1 << 64) - 1 - (1 << (j * 7 % 64)) for j in range(64)]
    signed = [m - (1 << 64) if m >= 1 << 63 else m for m in masks]
    t.check(t.call(parent=None, mask=torch.tensor(signed, dtype=torch.int64, device="cuda")), masks=masks)


@pytest.mark.parametrize("nodes", [[13, 64], [64, 1]])
@pytest.mark.parametrize("wide", [True, False])
def test_masks_of_many_nodes(nodes, wide):
    t = Trees([0, 70], nodes, 16, seed=21)
    t.wide = wide
    rng = np.random.default_rng(21)
    masks = [int(rng.integers(0, 1 << 62)) & int(rng.integers(0, 1 << 62)) | int(rng.integers(0, 4)) << 62 for _ in range(t.n)]
    masks[0] = masks[3] = 0  # request 0 has no context: these rows see nothing
    masks = [m & ((1 << nodes[0 if r < nodes[0] else 1]) - 1) for r, m in enumerate(masks)]
    junk = [m | (1 << 40 if n < 40 else 0) for m, n in zip(masks, [nodes[0]] * nodes[0] + [nodes[1]] * nodes[1])]  # bits of no node
    signed = [m - (1 << 64) if m >= 1 << 63 else m for m in junk]
    got = t.call(parent=None, mask=torch.tensor(signed, dtype=torch.int64, device="cuda"))
    t.check(got, masks=masks)
    assert (cpu(got["ctx"])[[0, 3]] == 0).all() and np.isneginf(cpu(got["lse"])[[0, 3]]).all()


def test_chain_is_the_default():
    t = Trees([33, 0], [7, 64], 8, seed=8)
    chain = [(2 << i) - 1 for n in t.nodes for i in range(n)]
    t.check(t.call(parent=None), masks=chain)


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("with_sel", [False, True])
def test_unseen_rows_never_reach_a_result(junk, with_sel):
    """Junk in unused slots, in slots behind a request, and in a node that another node does see."""
    t = Trees([70, 5], [5, 3], 16, seed=9)
    used = np.zeros(t.n_pages * 16, bool)
    for b in range(2):
        p = np.arange(t.ctx[b] + t.nodes[b])
        used[t.table[b][p // 16] * 16 + p % 16] = True
    gone = torch.from_numpy(np.flatnonzero(~used)).cuda()
    masks = [1, 0b11, 0b101, 0b1011, 0b10001, 1, 0b11, 0b100]  # node 1 of request 0 is seen by nodes 1 and 3
    slot = int(t.table[0][71 // 16] * 16 + 71 % 16)
    clean = t.c_kv[slot].clone(), t.k_rot[slot].clone()
    for pool in (t.c_kv, t.k_rot):
        pool[gone] = junk
    m = torch.tensor(masks, dtype=torch.int64, device="cuda")
    kw, sel = dict(parent=None, mask=m), None
    if with_sel:
        lst = np.full((8, 80), 10 ** 6, np.int32)
        sel = []
        for r in range(8):
            b = 0 if r < 5 else 1
            sel.append(np.arange(t.ctx[b] + t.nodes[b])[::2 if r % 2 else 1])
            lst[r, :len(sel[-1])] = sel[-1]
        kw.update(sel_in=i32(lst), sel_n_in=i32([len(x) for x in sel]))
    t.check(t.call(**kw), masks=masks, sel=sel)
    want = t.call(**kw)
    for pool in (t.c_kv, t.k_rot):
        pool[slot] = junk
    got = t.call(**kw)
    same = [0, 2, 4, 5, 6, 7]  # rows that do not see it
    assert torch.equal(got["ctx"][same], want["ctx"][same]) and torch.equal(got["lse"][same], want["lse"][same])
    t.c_kv[slot], t.k_rot[slot] = clean


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min])
def test_unseen_rows_of_many_nodes(junk):
    """As above for trees whose nodes are worked on two at a time: a junk row may be seen by one of the two."""
    ctx, nodes = [70, 5], [15, 10]
    t = Trees(ctx, nodes, 16, seed=22)
    used = np.zeros(t.n_pages * 16, bool)
    for b in range(2):
        p = np.arange(ctx[b] + nodes[b])
        used[t.table[b][p // 16] * 16 + p % 16] = True
    gone = torch.from_numpy(np.flatnonzero(~used)).cuda()
    for pool in (t.c_kv, t.k_rot):
        pool[gone] = junk
    masks = [1 << (r if r < 15 else r - 15) for r in range(25)]  # each node itself
    seers = {4: [4, 7, 8, 9], 11: [2, 11]}  # junk drafts of request 0, and who sees them: one or both of a pair
    for j, rows in seers.items():
        for r in rows:
            masks[r] |= 1 << j
    kw = dict(parent=None, mask=torch.tensor(masks, dtype=torch.int64, device="cuda"))
    want = t.call(**kw)
    t.check(want, masks=masks)
    for j in seers:
        slot = int(t.table[0][(70 + j) // 16] * 16 + (70 + j) % 16)
        t.c_kv[slot], t.k_rot[slot] = junk, junk
    got = t.call(**kw)
    same = [r for r in range(25) if not any(r in rows for rows in seers.values())]
    assert torch.equal(got["ctx"][same], want["ctx"][same]) and torch.equal(got["lse"][same], want["lse"][same])
    if junk != junk:
        seen = sorted(set(sum(seers.values(), [])))
        assert torch.isnan(got["ctx"][seen]).all() and torch.isnan(got["lse"][seen]).all()


@pytest.mark.parametrize("nodes", [[3, 2], [20, 9]])
def test_rows_behind_the_last_request_stay(nodes):
    t = Trees([50, 20], nodes, 16, seed=10, spare_rows=4)
    ctx = torch.full((t.n, 64, 512), 7.0, device="cuda")
    lse = torch.full((t.n, 64), 9.0, device="cuda")
    t.check(t.call(ctx=ctx, lse=lse))
    assert (ctx[sum(nodes):] == 7).all() and (lse[sum(nodes):] == 9).all()


SEL_CASES = [([300], [4], 16, 64), ([300], [4], 16, 65), ([2000, 40, 0], [3, 0, 9], 64, 256), ([5], [2], 8, 1),
             ([4000], [1], 32, 2048), ([900, 901], [16, 2], 48, 333), ([0], [5], 8, 7)]


@pytest.mark.parametrize("ctx,nodes,page,k", SEL_CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_selected_keys(ctx, nodes, page, k, dtype):
    t = Trees(ctx, nodes, page, seed=k)
    rng = np.random.default_rng(k)
    lst, sel = np.full((t.n, k), -5, np.int32), []
    for b in range(len(ctx)):
        for _ in range(nodes[b]):
            room = ctx[b] + nodes[b] + 3  # some entries point behind the request
            x = rng.permutation(room)[:rng.integers(0, min(k, room) + 1)]  # any order, counts from zero
            lst[len(sel), :len(x)] = x
            sel.append(x)
    got = t.call(sel_in=i32(lst), sel_n_in=i32([len(x) for x in sel]), out_dtype=dtype)
    t.check(got, sel=sel)
    lst[lst < 0] = 10 ** 9  # entries outside every range are dropped, whatever the count says
    got = t.call(sel_in=i32(lst), out_dtype=dtype)
    t.check(got, sel=sel)


def test_lists_end_at_the_slice_that_holds_them():
    """A list tensor that is a slice of a wider one: counts above its width do not reach the columns behind it."""
    t = Trees([400, 90], [3, 2], 16, seed=21)
    rng = np.random.default_rng(21)
    wide = np.stack([rng.permutation(90)[:60] for _ in range(5)]).astype(np.int32)
    got = t.call(sel_in=i32(wide)[:, 10:37], sel_n_in=i32([27, 28, 60, 10 ** 9, 5]))
    t.check(got, sel=[wide[r, 10:10 + min(27, c)] for r, c in enumerate([27, 28, 60, 10 ** 9, 5])])


def test_a_position_named_twice_counts_twice():
    t = Trees([50], [2], 16, seed=25)
    got = t.call(sel_in=i32([[7, 9, 7], [49, 3, 3]]))
    q, rows = t.q.float().cpu().numpy().astype(np.float64), t.rows().astype(np.float64)
    for r, x in enumerate(([7, 9, 7], [49, 3, 3])):
        k = rows[[t.table[0, p // 16] * 16 + p % 16 for p in x]]
        e = np.exp(q[r] @ k.T * SCALE)
        p = e / e.sum(1, keepdims=True)
        ref, spread = p @ k[:, :512], p @ np.abs(k[:, :512])
        # P to bf16 and 2 DS of unit-size q and k, as above
        assert np.all(np.abs(cpu(got["ctx"])[r] - ref) <= (2.0 ** -8 + 4e-4) * spread)
        assert np.abs(cpu(got["lse"])[r] - np.log(e.sum(1))).max() < 4e-4


def test_selecting_everything_is_the_dense_result():
    t = Trees([500, 64], [5, 2], 16, seed=11)
    every = np.tile(np.arange(505, dtype=np.int32), (7, 1))
    got, want = t.call(sel_in=i32(every)), t.call()
    t.check(got)
    assert (got["lse"] - want["lse"]).abs().max() < 1e-5


def test_offsets_past_32_bits():
    """The last pages of a pool of more than 2^32 elements."""
    t = Trees([300], [3], 64, seed=12, pages=120000)
    t.table[0, :5] = [119999, 0, 119998, 117000, 119990]
    got, sel = t.call(), np.arange(303)
    rows = np.zeros((0, 576), np.float32)
    pos = np.arange(303)
    slots = torch.from_numpy(t.table[0][pos // 64].astype(np.int64) * 64 + pos % 64).cuda()
    small = torch.cat([t.c_kv[slots], t.k_rot[slots]], 1)
    got2 = t.call(sel_in=i32(np.tile(sel, (3, 1))))
    t.c_kv, t.k_rot, t.table, t.page = small[:, :512], small[:, 512:], np.arange(38, dtype=np.int32)[None], 8
    t.check(got)
    t.check(got2)
    del rows


def test_same_call_twice_is_bit_identical():
    t = Trees([3000, 700, 20], [9, 3, 64], 64, seed=13)
    a, b = t.call(), t.call()
    assert torch.equal(a["ctx"], b["ctx"]) and torch.equal(a["lse"], b["lse"])


def test_bad_numbers_are_flagged_and_skipped():
    t = Trees([50, 20, 30], [3, 2, 1], 16, seed=14)
    ctx = torch.full((t.n, 64, 512), 7.0, device="cuda")
    good = t.ctx[1]
    t.ctx[1] = -4
    got = t.call(ctx=ctx)
    bad_word()
    assert (ctx[3:5] == 7).all() and torch.isfinite(got["ctx"]).all() and not (ctx[:3] == 7).all()
    t.ctx[1] = 10 ** 6  # past its table row
    t.call(ctx=ctx.fill_(7.0))
    bad_word()
    assert (ctx[3:5] == 7).all()
    t.ctx[1] = good
    kw = dict(parent=None)
    t2 = Trees([5], [70], 16, seed=15)  # more than 64 nodes
    ctx = torch.full((70, 64, 512), 7.0, device="cuda")
    t2.call(ctx=ctx, **kw)
    bad_word()
    assert (ctx == 7).all()


@pytest.mark.parametrize("n", [2, 14])
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
def test_a_page_outside_the_pool_is_flagged_and_left_out(n, bad):
    t = Trees([100], [n], 16, seed=16)
    keep = np.r_[np.arange(32), np.arange(48, 100 + n)]  # page 2 of the request is bad
    t.table[0, 2] = bad
    got = t.call()
    bad_word()
    sel = t.call(sel_in=i32(np.tile(np.arange(100 + n), (n, 1))))
    bad_word()
    t.table[0, 2] = 0
    t.check(got, sel=[keep] * n)
    t.check(sel, sel=[keep] * n)


def test_graph_replays_follow_the_lengths_and_streams_do_not_mix():
    t = Trees([900, 300], [4, 3], 16, seed=17)
    cfg, kv = A.glm52_cfg(T_MAX), t.kv()
    ctx_len, cu, par = i32(t.ctx), i32(t.cu), i32(t.parent)
    call = lambda: P.mla_tree_attn(cfg, kv, t.q, ctx_len, cu, parent=par)  # noqa: E731
    call()
    graphs, outs = [], []
    for _ in range(2):  # two graphs, replayed on two streams at once
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for lengths in ([900, 300], [64, 1], [0, 299]):
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


# ---- the commit ------------------------------------------------------------------------------

@pytest.mark.parametrize("B,layers,index", [(1, 1, False), (5, 3, True), (40, 2, True), (3, 78, False), (2, 130, True)])
def test_commit_moves_the_accepted_rows(B, layers, index):
    rng = np.random.default_rng(B + layers)
    page = 16
    nodes = rng.integers(0, 65, B)
    ctx = rng.integers(0, 100, B)
    most = -(-(ctx + nodes) // page)
    n_pages = int(most.sum()) + 2
    perm, table, at = rng.permutation(n_pages), np.zeros((B, max(int(most.max()), 1)), np.int32), 0
    for b in range(B):
        table[b, :most[b]] = perm[at:at + most[b]]
        at += most[b]
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    n = int(cu[-1])
    parent = np.concatenate([[-1] + [rng.integers(max(0, j - 4), j) for j in range(1, k)] if k else [] for k in nodes]).astype(np.int32)
    draft, target = rng.integers(0, 3, n).astype(np.int32), rng.integers(0, 3, n).astype(np.int32)  # siblings collide
    kv = [torch.randn(n_pages * page, 576, device="cuda", dtype=torch.bfloat16) for _ in range(layers)]
    keys = None
    if index:
        keys = [A.IndexKeys(torch.randint(0, 255, (n_pages * page, 128), device="cuda", dtype=torch.uint8),
                            torch.rand(n_pages * page, device="cuda")) if i % 2 == 0 else None for i in range(layers)]
    before = [x.clone() for x in kv]
    kbefore = [(k.keys.clone(), k.scale.clone()) if k else None for k in keys] if index else None
    t = i32(table)
    caches = P.LayerCaches([P.PagedKV.packed(x, page, t) for x in kv], keys)
    ctx_len = i32(ctx)
    got = P.tree_commit(caches, ctx_len, i32(cu), i32(parent), i32(draft), i32(target))
    src, dst = np.arange(n_pages * page), np.arange(n_pages * page)
    for b in range(B):
        sl = slice(cu[b], cu[b + 1])
        path, nxt = R.tree_walk(parent[sl], draft[sl], target[sl])
        assert cpu(got["path"])[b].tolist() == path + [-1] * (64 - len(path))
        assert int(got["n_accept"][b]) == len(path) and int(got["next"][b]) == nxt
        for d, j in enumerate(path):
            p, s = ctx[b] + d, ctx[b] + j
            src[table[b][p // page] * page + p % page] = table[b][s // page] * page + s % page
    assert np.array_equal(cpu(got["ctx_len"]), ctx + cpu(got["n_accept"])) and np.array_equal(cpu(ctx_len), ctx)
    src = torch.from_numpy(src).cuda()
    for i in range(layers):
        assert torch.equal(kv[i], before[i][src])
        if index and keys[i] is not None:
            assert torch.equal(keys[i].keys, kbefore[i][0][src]) and torch.equal(keys[i].scale, kbefore[i][1][src])
    del dst


def test_commit_never_follows_a_later_parent_and_flags_bad_requests():
    kv = torch.randn(64, 576, device="cuda", dtype=torch.bfloat16)
    was = kv.clone()
    caches = P.LayerCaches([P.PagedKV.packed(kv, 16, i32([[0, 1], [2, 3]]))])
    # a node that names itself, one that names a later node, and one with no root above it
    got = P.tree_commit(caches, i32([0, 3]), i32([0, 4, 6]), i32([-1, 1, 3, 7, -1, 0]), i32([1, 1, 1, 1, 1, 2]), i32([1] * 6))
    assert cpu(got["n_accept"]).tolist() == [1, 1] and torch.equal(kv, was)
    got = P.tree_commit(caches, i32([0, 30]), i32([0, 4, 8]), i32([-1, 0, 0, 0] * 2), i32([1] * 8), i32([1] * 8))
    bad_word()  # 30 + 4 positions do not fit request 1's two pages
    assert cpu(got["n_accept"]).tolist() == [2, 0] and cpu(got["next"]).tolist() == [1, -1]
    assert torch.equal(kv, was)


# ---- the step together -----------------------------------------------------------------------

def test_plan_append_attend_commit_follow_a_plain_sequence():
    """Two requests, three drafting steps over pages of 8: after every commit the pool holds, position
    for position, what appending the accepted tokens one by one would hold, and the attention of the
    drafts equals the 64-bit result over it. The steps are captured once and replayed."""
    page, B, L, N = 8, 2, 2, 10
    rng = np.random.default_rng(20)
    cfg = A.glm52_cfg(T_MAX)
    pool = [torch.full((40 * page, 576), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(L)]
    ikeys = A.IndexKeys(torch.zeros(40 * page, 128, dtype=torch.uint8, device="cuda"), torch.zeros(40 * page, device="cuda"))
    table, held, free = i32(np.zeros((B, 12))), i32([0] * B), i32(rng.permutation(40))
    n_free, ctx_len, n_new = i32([40]), i32([0] * B), i32([5, 4])
    kvs = [P.PagedKV.packed(x, page, table) for x in pool]
    caches = P.LayerCaches(kvs, [ikeys, None])
    norm = torch.ones(512, device="cuda", dtype=torch.bfloat16)
    kn = torch.ones(128, device="cuda", dtype=torch.bfloat16)
    raw = torch.zeros(L, N, 576, device="cuda")
    kraw = torch.zeros(N, 128, device="cuda")
    cos, sin = torch.ones(N, 32, device="cuda"), torch.zeros(N, 32, device="cuda")
    q = torch.randn(N, 64, 576, device="cuda").to(torch.bfloat16)
    parent, draft, target = i32([0] * N), i32([0] * N), i32([0] * N)

    def step():
        plan = P.page_plan(ctx_len, n_new, table, held, free, n_free, page, N, in_place=True)
        outs = []
        for i in range(L):
            P.cache_append_paged(cfg, plan["slot"], cos, sin, kv=kvs[i], kv_raw=raw[i], kv_norm_w=norm,
                                 **(dict(keys=ikeys, k_raw=kraw, k_norm_w=kn, k_norm_b=kn) if i == 0 else {}))
            outs.append(P.mla_tree_attn(cfg, kvs[i], q, ctx_len, plan["cu"], parent=parent))
        done = P.tree_commit(caches, ctx_len, plan["cu"], parent, draft, target)
        return plan, outs, done

    n_new.zero_()
    step()  # nothing to do: loads the kernels
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan, outs, done = step()
    kept = [[[] for _ in range(B)] for _ in range(L)]
    for it, sizes in enumerate(([5, 4], [3, 6], [9, 0])):
        n_new.copy_(i32(sizes))
        par = np.concatenate([[-1] + [rng.integers(0, j) for j in range(1, n)] if n else [] for n in sizes] + [[0] * (N - sum(sizes))])
        dr, tg = rng.integers(0, 2, N), rng.integers(0, 2, N)
        parent.copy_(i32(par)), draft.copy_(i32(dr)), target.copy_(i32(tg))
        raw.copy_(torch.randn(L, N, 576, device="cuda")), kraw.copy_(torch.randn(N, 128, device="cuda"))
        ctx = cpu(ctx_len).tolist()
        g.replay()
        torch.cuda.synchronize()
        cu = np.concatenate([[0], np.cumsum(sizes)])
        assert cpu(plan["cu"]).tolist() == cu.tolist() and (cpu(plan["short"]) == 0).all()
        flat_kv = torch.zeros(L, N, 576, device="cuda", dtype=torch.bfloat16)  # the same rows by the plain append
        for i in range(L):
            A.cache_append(cfg, i32(np.arange(N)), cos, sin, kv=A.LatentKV.packed(flat_kv[i]), kv_raw=raw[i], kv_norm_w=norm)
        fresh = flat_kv.float().cpu().numpy()
        masks = R.tree_masks(par, cu)
        tab = cpu(table)
        for i in range(L):
            # the attention saw kept rows and all drafts; compare on a flat copy of what was there
            rows = np.zeros((B * 64, 576), np.float32)
            for b in range(B):
                seen = kept[i][b] + list(fresh[i, cu[b]:cu[b + 1]])
                rows[b * 64:b * 64 + len(seen)] = seen if seen else np.zeros((0, 576))
            flat = np.arange(B * 8, dtype=np.int32).reshape(B, 8)
            ref, lse, a = R.tree_attn(q.float().cpu().numpy()[:cu[-1]], rows, ctx, cu, masks, flat, 8, SCALE)
            o = cpu(outs[i]["ctx"])[:cu[-1]]
            assert np.all(np.abs(o - ref) <= (2.0 ** -8 + 4e-4) * a)  # 2 DS of q and k of unit size is below 4e-4
        for b in range(B):
            path, _ = R.tree_walk(par[cu[b]:cu[b + 1]], dr[cu[b]:cu[b + 1]], tg[cu[b]:cu[b + 1]])
            assert int(done["n_accept"][b]) == len(path)
            for i in range(L):
                kept[i][b] += [fresh[i, cu[b] + j] for j in path]
                pos = np.arange(len(kept[i][b]))
                have = pool[i].float().cpu().numpy()[tab[b][pos // page] * page + pos % page]
                if len(pos):
                    assert np.array_equal(have, np.array(kept[i][b]))
        ctx_len.copy_(done["ctx_len"])
    free_now = int(n_free)
    P.page_release(i32([1, 1]), table, held, free, n_free)
    assert int(n_free) == 40 and free_now < 40 and sorted(cpu(free).tolist()) == list(range(40))


def test_append_skips_padding_and_flags_slots_outside_the_pool():
    kv = torch.zeros(32, 576, device="cuda", dtype=torch.bfloat16)
    k = P.PagedKV.packed(kv, 16, i32([[0, 1]]))
    cfg, norm = A.glm52_cfg(8), torch.ones(512, device="cuda", dtype=torch.bfloat16)  # T_max plays no part
    one, zero = torch.ones(3, 32, device="cuda"), torch.zeros(3, 32, device="cuda")
    raw = torch.ones(3, 576, device="cuda")
    P.cache_append_paged(cfg, i32([31, -1, 9]), one, zero, kv=k, kv_raw=raw, kv_norm_w=norm)
    torch.cuda.synchronize()
    assert sorted(torch.nonzero(kv.abs().sum(1)).flatten().tolist()) == [9, 31]
    P.cache_append_paged(cfg, i32([32, -2, 3]), one, zero, kv=k, kv_raw=raw, kv_norm_w=norm)
    bad_word()
    assert sorted(torch.nonzero(kv.abs().sum(1)).flatten().tolist()) == [3, 9, 31]


def test_a_request_without_pages_neither_reads_nor_moves_others_rows():
    """Stale table entries of a request that got no pages lead nowhere: its drafts are left out and its commit
    moves nothing, in whatever pages the entries named before."""
    page = 16
    pool = torch.randn(4 * page, 576, device="cuda", dtype=torch.bfloat16)
    was = pool.clone()
    table, held = i32([[0, 1], [2, 1]]), i32([2, 1])  # request 1's second entry names request 0's page
    plan = P.page_plan(i32([20, 14]), i32([4, 6]), table, held, i32([3, 3, 3, 3]), i32([0]), page, 10)
    assert cpu(plan["short"]).tolist() == [0, 1] and cpu(table).tolist() == [[0, 1], [2, -1]]
    assert (cpu(plan["slot"])[4:] == -1).all() and int(plan["n_free"]) == 0
    kv = P.PagedKV.packed(pool, page, table)
    q = torch.randn(10, 64, 576, device="cuda").to(torch.bfloat16)
    par = i32([-1, 0, 0, 0, -1, 0, 0, 0, 0, 0])
    out = P.mla_tree_attn(A.glm52_cfg(64), kv, q, i32([20, 14]), plan["cu"], parent=par)
    bad_word()
    assert torch.isfinite(out["ctx"]).all()
    tok, tgt = i32([0, 1, 2, 3, 0, 9, 9, 9, 5, 9]), i32([7, 7, 7, 7, 5, 0, 0, 0, 0, 0])  # request 1 accepts its node 4
    P.tree_commit(P.LayerCaches([kv]), i32([20, 14]), plan["cu"], par, tok, tgt)
    bad_word()
    assert torch.equal(pool, was)


def test_layers_of_one_commit_share_the_whole_table():
    kv = torch.zeros(32, 576, dtype=torch.bfloat16, device="cuda")
    wide = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    a, b = (P.PagedKV.packed(kv, 8, t) for t in (wide[:, :2], wide))
    with pytest.raises(ValueError, match="share one block table"):
        P.LayerCaches([a, b])


def test_append_stays_inside_the_smallest_pool():
    """Keys with fewer scales than rows: the slots behind the scales are flagged, and neither is written."""
    keys = A.IndexKeys(torch.zeros(32, 128, dtype=torch.uint8, device="cuda"), torch.zeros(32, device="cuda")[:16])
    one, zero = torch.ones(2, 32, device="cuda"), torch.zeros(2, 32, device="cuda")
    kn = torch.ones(128, device="cuda", dtype=torch.bfloat16)
    raw = torch.randn(2, 128, device="cuda")
    P.cache_append_paged(A.glm52_cfg(8), i32([3, 20]), one, zero, keys=keys, k_raw=raw, k_norm_w=kn, k_norm_b=kn)
    bad_word()
    assert torch.nonzero(keys.scale).flatten().tolist() == [3]
    assert torch.nonzero(keys.keys.sum(1)).flatten().tolist() == [3]
