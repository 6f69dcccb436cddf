"""Positions of drafted trees in a plan, and whole steps with rotated keys, on the GPU. Everything here is
compared bit for bit: whole numbers, and rows that the plain append writes at the same positions."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import paged_ref as R
from test_gpu_paged import SCALE, T_MAX, Trees, bad_word, clean_device_error, cpu, i32  # noqa: F401
from windlass_b200 import _lib
from windlass_b200 import attn as A
from windlass_b200 import paged as P

pytestmark = pytest.mark.gpu


def signed(masks):
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64, device="cuda")


def random_trees(rng, sizes, back=4):
    return np.concatenate([[-1] + [rng.integers(max(0, j - back), j) for j in range(1, n)] if n else [] for n in sizes]).astype(np.int32)


def plan_of(ctx, new, page, n_tokens, **kw):
    """A plan for requests that hold what their contexts need, with pages enough."""
    ctx, new = np.asarray(ctx), np.asarray(new)
    held, most = -(-ctx // page), -(-(ctx + new) // page)
    n_pages = int(most.sum()) + 1
    table, at = np.zeros((len(ctx), max(int(most.max()), 1)), np.int32), 0
    for b, h in enumerate(held):
        table[b, :h] = np.arange(at, at + h)
        at += h
    free = np.zeros(n_pages, np.int32)
    free[:n_pages - at] = np.arange(at, n_pages)
    return P.page_plan(i32(ctx), i32(new), i32(table), i32(held), i32(free), i32([n_pages - at]), page, n_tokens, **kw)


# one launch and two, padded and not
@pytest.mark.parametrize("B,most,spare", [(1, 1, 0), (1, 64, 0), (9, 16, 5), (70, 64, 0), (1100, 3, 2), (40, 64, 1000)])
def test_positions_of_trees_count_ancestors(B, most, spare):
    rng = np.random.default_rng(B + most)
    ctx, new = rng.integers(0, 500, B), rng.integers(0, most + 1, B)
    new[0] = most
    total = int(new.sum())
    parent = random_trees(rng, new)
    cu = np.concatenate([[0], np.cumsum(new)])
    masks = R.tree_masks(parent, cu)
    seq = np.repeat(np.arange(B), new)
    want = ctx[seq] + [bin(m).count("1") - 1 for m in masks]
    line = plan_of(ctx, new, 16, total + spare)
    for kw in (dict(parent=i32(np.pad(parent, (0, spare)))), dict(mask=signed(masks + [0] * spare))):
        got = plan_of(ctx, new, 16, total + spare, **kw)
        assert np.array_equal(cpu(got["pos"]), np.pad(want, (0, spare), constant_values=-1))
        for k in ("slot", "seq", "cu", "short", "n_held", "n_free"):
            assert torch.equal(got[k], line[k]), k
    assert np.array_equal(cpu(line["pos"])[:total], ctx[seq] + np.arange(total) - cu[seq])


def test_positions_of_prompts_roots_and_bad_parents():
    parent = i32([-1, 0, 0, -1, 3, 1] + [0] * 65)  # two roots in the first request, a prompt of 65 tokens behind it
    got = plan_of([10, 7], [6, 65], 8, 71, parent=parent)
    assert cpu(got["pos"])[:6].tolist() == [10, 11, 11, 10, 11, 12]
    assert cpu(got["pos"])[6:].tolist() == list(range(7, 72))
    got = plan_of([3], [4], 8, 4, parent=i32([-1, 1, 3, 2]))  # itself, and a later node
    bad_word()
    assert cpu(got["pos"]).tolist() == [3, 3, 3, 4]
    got = plan_of([3], [3], 8, 3, mask=signed([(1 << 64) - 1, 0, 0b1000]))  # later nodes and itself, none, no node of the request
    assert cpu(got["pos"]).tolist() == [5, 3, 3]


@pytest.mark.parametrize("by", ["parent", "mask"])
def test_branched_steps_leave_what_appending_the_accepted_tokens_leaves(by):
    """Drafted trees with a real RoPE table, three steps, captured once: after every commit the pools of latent rows, index
    keys and scales hold, bit for bit, what appending the accepted tokens one by one at their positions leaves, and the
    attention of every node saw the keys of its branch, rotated by their places on it."""
    page, B, L, N = 8, 2, 2, 12
    rng = np.random.default_rng(31)
    cfg = A.glm52_cfg(T_MAX)
    angle = np.arange(80)[:, None] / 10000 ** (np.arange(32) / 32)
    cos_t, sin_t = (torch.tensor(f(angle), dtype=torch.float32, device="cuda") for f in (np.cos, np.sin))
    pool = [torch.zeros(24 * page, 576, device="cuda", dtype=torch.bfloat16) for _ in range(L)]
    ikeys = A.IndexKeys(torch.zeros(24 * page, 128, dtype=torch.uint8, device="cuda"), torch.zeros(24 * page, device="cuda"))
    table, held, free = i32(np.zeros((B, 8))), i32([0] * B), i32(rng.permutation(24))
    n_free, ctx_len, n_new = i32([24]), i32([0] * B), i32([0] * B)
    kvs = [P.PagedKV.packed(x, page, table) for x in pool]
    caches = P.LayerCaches(kvs, [ikeys, None])
    g = torch.Generator(device="cuda").manual_seed(3)
    norm = torch.rand(512, generator=g, device="cuda").to(torch.bfloat16)
    kw_, kb_ = (torch.rand(128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    raw, kraw = torch.zeros(L, N, 576, device="cuda"), torch.zeros(N, 128, device="cuda")
    q = torch.randn(N, 64, 576, generator=g, device="cuda").to(torch.bfloat16)
    parent, draft, target = i32([0] * N), i32([0] * N), i32([0] * N)
    mask = torch.zeros(N, dtype=torch.int64, device="cuda")
    trees = dict(parent=parent) if by == "parent" else dict(mask=mask)

    def step():
        plan = P.page_plan(ctx_len, n_new, table, held, free, n_free, page, N, in_place=True, **trees)
        cos, sin = cos_t[plan["pos"]], sin_t[plan["pos"]]
        outs = []
        for i in range(L):
            P.cache_append_paged(cfg, plan["slot"], cos, sin, kv=kvs[i], kv_raw=raw[i], kv_norm_w=norm,
                                 **(dict(keys=ikeys, k_raw=kraw, k_norm_w=kw_, k_norm_b=kb_) if i == 0 else {}))
            outs.append(P.mla_tree_attn(cfg, kvs[i], q, ctx_len, plan["cu"], **trees))
        return plan, outs, P.tree_commit(caches, ctx_len, plan["cu"], parent, draft, target)

    step()  # nothing to do: loads the kernels
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, outs, done = step()

    # the plain sequences: one contiguous cache per request and layer, appended token by token
    flat = [[torch.zeros(1, 64, 576, device="cuda", dtype=torch.bfloat16) for _ in range(B)] for _ in range(L)]
    fkeys = [A.IndexKeys(torch.zeros(1, 64, 128, dtype=torch.uint8, device="cuda"), torch.zeros(1, 64, device="cuda")) for _ in range(B)]

    def append(b, row, pos):
        at = i32([pos])
        for i in range(L):
            A.cache_append(cfg, at, cos_t[pos:pos + 1], sin_t[pos:pos + 1], kv=A.LatentKV.packed(flat[i][b]), kv_raw=raw[i, row:row + 1],
                           kv_norm_w=norm, **(dict(keys=fkeys[b], k_raw=kraw[row:row + 1], k_norm_w=kw_, k_norm_b=kb_) if i == 0 else {}))

    jumped = 0
    for sizes in ([6, 6], [7, 5], [9, 3], [0, 12]):
        n_new.copy_(i32(sizes))
        par = np.concatenate([random_trees(rng, sizes), np.zeros(N - sum(sizes))]).astype(np.int32)
        dr, tg = rng.integers(0, 2, N), rng.integers(0, 2, N)
        cu = np.concatenate([[0], np.cumsum(sizes)])
        masks = R.tree_masks(par, cu)
        parent.copy_(i32(par)), draft.copy_(i32(dr)), target.copy_(i32(tg)), mask.copy_(signed(masks + [0] * (N - len(masks))))
        raw.copy_(torch.randn(L, N, 576, generator=g, device="cuda")), kraw.copy_(torch.randn(N, 128, generator=g, device="cuda"))
        ctx = cpu(ctx_len).tolist()
        graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            for j in range(sizes[b]):  # every node alone on its branch
                r = cu[b] + j
                for d, a in enumerate([a for a in range(j + 1) if masks[r] >> a & 1]):
                    append(b, cu[b] + a, ctx[b] + d)
                depth = bin(masks[r]).count("1")
                for i in range(L):
                    rows = flat[i][b][0].float().cpu().numpy()
                    ref, lse, spread = R.tree_attn(q[r:r + 1].float().cpu().numpy(), rows, [ctx[b] + depth - 1], [0, 1], [1],
                                                   np.arange(8, dtype=np.int32)[None], 8, SCALE)
                    # P in bf16, 2 DS of q and k of unit size below 4e-4 (k: at most 1 after the norm's weights below 1)
                    assert np.all(np.abs(cpu(outs[i]["ctx"])[r:r + 1] - ref) <= (2.0 ** -8 + 4e-4) * spread)
                    assert np.abs(cpu(outs[i]["lse"])[r:r + 1] - lse).max() < 4e-4
            path, _ = R.tree_walk(par[cu[b]:cu[b + 1]], dr[cu[b]:cu[b + 1]], tg[cu[b]:cu[b + 1]])
            jumped += path != list(range(len(path)))
            for d, j in enumerate(path):
                append(b, cu[b] + j, ctx[b] + d)
            assert int(done["n_accept"][b]) == len(path)
            pos = np.arange(ctx[b] + len(path))
            slots = torch.from_numpy(cpu(table)[b][pos // page].astype(np.int64) * page + pos % page).cuda()
            for i in range(L):
                assert torch.equal(pool[i][slots], flat[i][b][0, :len(pos)])
            assert torch.equal(ikeys.keys[slots], fkeys[b].keys[0, :len(pos)])
            assert torch.equal(ikeys.scale[slots], fkeys[b].scale[0, :len(pos)])
        ctx_len.copy_(done["ctx_len"])
    assert jumped >= 2  # the paths left the line


@pytest.mark.parametrize("layers", [0, 1])
def test_nothing_of_a_request_without_pages_is_committed(layers):
    """Chains, whose accepted nodes stand where they belong already, and a jumping path. Request 0 has its pages; 1 lacks its
    second page, 2 all of them, and 3's table row is too narrow; the drafts of 1 begin in a page that it holds."""
    page = 8
    pool = torch.randn(8 * page, 576, device="cuda", dtype=torch.bfloat16)
    was = pool.clone()
    ctx, new = [6, 5, 8, 20], [2, 5, 4, 6]
    table, held = i32([[0, 9, 9], [1, 0, 0], [2, 0, 0], [3, 4, 5]]), i32([1, 1, 1, 3])
    plan = P.page_plan(i32(ctx), i32(new), table, held, i32([7] * 8), i32([0]), page, 17)
    assert cpu(plan["short"]).tolist() == [0, 1, 1, 1]
    parent = i32([-1, 0] + [-1, 0, 0, 0, 2] + [-1, 0, 1, 2] + [-1, 0, 1, 2, 3, 4])
    draft, target = i32([1] * 17), i32([1] * 17)
    draft[3], draft[4] = 2, 1  # request 1 jumps from node 0 to node 2
    ctx_len = i32(ctx)
    if layers:
        got = P.tree_commit(P.LayerCaches([P.PagedKV.packed(pool, page, table)]), ctx_len, plan["cu"], parent, draft, target)
    else:  # the walk alone
        out = {k: torch.full(s, 77, dtype=torch.int32, device="cuda") for k, s in
               dict(n_accept=(4,), path=(4, 64), next=(4,), ctx_len=(4,)).items()}
        io = _lib.TreeCommitIO(4, 17, ctx_len.data_ptr(), plan["cu"].data_ptr(), parent.data_ptr(), draft.data_ptr(), target.data_ptr(),
                               page, 8, table.data_ptr(), 3, 3, 0, None, None, out["n_accept"].data_ptr(), out["path"].data_ptr(),
                               out["next"].data_ptr(), out["ctx_len"].data_ptr())
        assert _lib.lib().wl_tree_commit(C.byref(A.glm52_cfg(64)), C.byref(io), torch.cuda.current_stream().cuda_stream) == _lib.WL_OK
        got = out
    bad_word()
    assert cpu(got["n_accept"]).tolist() == [2, 0, 0, 0] and cpu(got["next"]).tolist() == [1, -1, -1, -1]
    assert cpu(got["ctx_len"]).tolist() == [8, 5, 8, 20]
    assert cpu(got["path"])[:, 0].tolist() == [0, -1, -1, -1] and torch.equal(pool, was)


@pytest.mark.parametrize("ctx,nodes", [([70], [5]), ([70], [15]), ([0], [14]), ([64], [13]), ([3000, 5], [13, 12]), ([4096], [3]), ([4096], [13])])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_of_seen_rows_give_what_the_formula_gives(ctx, nodes, dtype):
    """Drafted rows with an infinity in a latent column, or in a roped one, seen by some nodes: NaN where the formula has it,
    whichever nodes share the work and however the keys are cut. (A row whose scores are all -infinity gives zeros.)"""
    t = Trees(ctx, nodes, 16, seed=41)
    rng = np.random.default_rng(41)
    masks = []
    for n in nodes:
        for i in range(n):
            masks.append(1 << i | int(rng.integers(0, 1 << n)) & int(rng.integers(0, 1 << n)))
    for j, (col, v) in {1: (0, np.inf), 2: (77, -np.inf), 3: (300, np.inf), 4: (511, -np.inf)}.items():
        p = t.ctx[0] + j
        t.c_kv[int(t.table[0][p // 16]) * 16 + p % 16, col] = v
    if nodes[0] > 6:
        p = t.ctx[0] + 6
        slot = int(t.table[0][p // 16]) * 16 + p % 16
        t.k_rot[slot, 3], t.c_kv[slot, 200] = np.inf, np.inf  # two that may meet as infinity - infinity
    got = t.call(parent=None, mask=signed(masks), out_dtype=dtype)
    with np.errstate(invalid="ignore"):
        ref, lse, spread = R.tree_attn(t.q.float().cpu().numpy(), t.rows(), t.ctx, t.cu, masks, t.table, 16, SCALE)
        keys = [np.r_[:t.ctx[b], [t.ctx[b] + j for j in range(n) if masks[t.cu[b] + i] >> j & 1]].astype(int) for b, n in enumerate(nodes) for i in range(n)]
    rows = t.rows().astype(np.float64)
    for r, k in enumerate(keys):
        b = int(np.searchsorted(t.cu, r, "right")) - 1
        with np.errstate(invalid="ignore"):
            z = t.q[r].double().cpu().numpy() @ rows[t.table[b][k // 16].astype(int) * 16 + k % 16].T
        none = (z == -np.inf).all(1)
        ref[r][none], lse[r][none], spread[r][none] = 0, -np.inf, 0
    o, z = got["ctx"].double().cpu().numpy(), got["lse"].double().cpu().numpy()
    assert np.isnan(ref).any() and np.array_equal(np.isnan(o), np.isnan(ref))
    assert np.array_equal(np.isnan(z), np.isnan(lse)) and np.array_equal(np.isneginf(z), np.isneginf(lse))
    f, g = np.isfinite(ref), np.isfinite(lse)
    spread = np.where(np.isfinite(spread), spread, 0)
    tol = (2.0 ** -8 + 4e-4) * spread + (2.0 ** -8 * np.abs(ref) if dtype == torch.bfloat16 else 0)
    assert np.all(np.abs(o - ref)[f] <= tol[f]) and np.abs(z - lse)[g].max(initial=0) < 4e-4


def test_the_fields_of_a_paged_cache_do_not_change():
    """Its addresses are taken once: a field that could be replaced would leave them behind."""
    kv = P.PagedKV.packed(torch.zeros(32, 576, dtype=torch.bfloat16, device="cuda"), 16, i32([[0, 1]]))
    for name in ("c_kv", "k_rot", "page_size", "block_table", "n_pages"):
        with pytest.raises(AttributeError):
            setattr(kv, name, getattr(kv, name))
    assert kv.n_pages == 2 and kv.c().max_pages == 2


def test_layers_of_one_commit_have_pools_of_their_own():
    t = i32([[0, 1]])
    a, b = (torch.zeros(16, 576, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    keys = A.IndexKeys(torch.zeros(16, 128, dtype=torch.uint8, device="cuda"), torch.zeros(16, device="cuda"))
    ka, kb = P.PagedKV.packed(a, 8, t), P.PagedKV.packed(b, 8, t)
    P.LayerCaches([ka, kb], [keys, None])
    with pytest.raises(ValueError, match="share one latent pool"):
        P.LayerCaches([ka, ka])
    with pytest.raises(ValueError, match="share one index pool"):
        P.LayerCaches([ka, kb], [keys, keys])


def test_lists_that_share_memory_are_refused():
    """Rows that overlap (one list for all nodes, a window that slides): with counts, the lists ended at the row stride."""
    t = Trees([50], [3], 16, seed=51)
    one = i32([list(range(20))])
    slide = torch.as_strided(i32(range(40)), (3, 20), (5, 1))
    for lst in (one.expand(3, 20), slide):
        for kw in (dict(), dict(sel_n_in=i32([20, 20, 20]))):
            with pytest.raises(ValueError, match="must not overlap"):
                t.call(sel_in=lst, **kw)
    got = t.call(sel_in=one.expand(3, 20).contiguous())
    t.check(got, sel=[np.arange(20)] * 3)


def test_lengths_that_pass_31_bits_are_flagged():
    """A table that could hold them, of one large page over and over."""
    page, wide, end = 1 << 20, 2100, (1 << 31) - 3
    pool = torch.zeros(page, 576, device="cuda", dtype=torch.bfloat16)
    table = torch.zeros(1, wide, dtype=torch.int32, device="cuda")
    plan = P.page_plan(i32([end]), i32([10]), table, i32([2047]), i32([0] * 8), i32([8]), page, 10)
    bad_word()
    assert cpu(plan["short"]).tolist() == [-1] and cpu(plan["cu"]).tolist() == [0, 0] and (cpu(plan["slot"]) == -1).all()
    kv = P.PagedKV.packed(pool, page, table)
    cu, parent, tok = i32([0, 10]), i32([-1] + [0] * 9), i32([1] * 10)
    done = P.tree_commit(P.LayerCaches([kv]), i32([end]), cu, parent, tok, tok)
    bad_word()
    assert cpu(done["n_accept"]).tolist() == [0] and cpu(done["ctx_len"]).tolist() == [end]
    for nodes in (10, 13):
        ctx = torch.full((nodes, 64, 512), 7.0, device="cuda")
        P.mla_tree_attn(A.glm52_cfg((1 << 31) - 1), kv, torch.zeros(nodes, 64, 576, device="cuda", dtype=torch.bfloat16),
                        i32([end - nodes]), i32([0, nodes]), ctx=ctx)
        bad_word()
        assert (ctx == 7).all()
