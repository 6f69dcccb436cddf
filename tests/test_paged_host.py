"""Refusals of the paged-cache and drafted-tree entry points (argument checks run before
any launch, so no GPU is needed), and the restatement's own consistency."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

from oracle import paged_ref as R
from windlass_b200 import _lib
from windlass_b200 import attn as A
from windlass_b200 import paged as P
from windlass_b200._lib import IndexCache, LatentCache, PagedKVC, lib

OK, ARG, UNS, WS = _lib.WL_OK, _lib.WL_ERR_ARG, _lib.WL_ERR_UNSUPPORTED, _lib.WL_ERR_WORKSPACE
FAKE = 0x10000  # 16-byte aligned, never read


def cfg(T=4096):
    c = _lib.AttnCfg()
    lib().wl_attn_cfg_glm52(C.byref(c), T)
    return c


def pool(**kw):
    f = dict(c_kv=FAKE, c_kv_row_stride=576, c_kv_seq_stride=0, k_rot=FAKE + 1024, k_rot_row_stride=576, k_rot_seq_stride=0)
    f.update(kw)
    return LatentCache(**f)


def attn_io(**kw):
    kv = PagedKVC(kw.pop("latent", pool()), kw.pop("page_size", 64), kw.pop("n_pages", 100), kw.pop("block_table", FAKE),
                  kw.pop("table_stride", 20), kw.pop("max_pages", 20))
    f = dict(batch=2, n_nodes=4, ctx_len=FAKE, cu_nodes=FAKE, kv=kv, q_abs=FAKE, mode=_lib.WL_MODE_DENSE, ctx_type=0, ctx=FAKE)
    f.update(kw)
    return _lib.TreeAttnIO(**f)


def attn(io, c=None, ws=FAKE, nbytes=1 << 40):
    return lib().wl_mla_tree_attn(C.byref(c or cfg()), C.byref(io), ws, nbytes, None)


BAD_ATTN = [dict(n_nodes=-1), dict(batch=-1), dict(ctx_len=None), dict(cu_nodes=None), dict(block_table=None),
            dict(page_size=0), dict(page_size=12), dict(page_size=-8), dict(n_pages=0), dict(n_pages=1 << 26),
            dict(table_stride=19), dict(max_pages=0), dict(tree_mask=FAKE, parent=FAKE), dict(mode=_lib.WL_MODE_OWNER),
            dict(ctx_type=2), dict(mode=_lib.WL_MODE_CONSUMER), dict(mode=_lib.WL_MODE_CONSUMER, sel_in=FAKE),
            dict(mode=_lib.WL_MODE_CONSUMER, sel_in=FAKE, sel_stride=8, sel_n=9),
            dict(mode=_lib.WL_MODE_CONSUMER, sel_in=FAKE, sel_stride=8, sel_n=-1),
            dict(latent=pool(c_kv=None)), dict(latent=pool(k_rot=None)), dict(latent=pool(c_kv=FAKE + 8)),
            dict(latent=pool(c_kv_row_stride=516)), dict(latent=pool(c_kv_row_stride=504)),
            dict(latent=pool(k_rot_row_stride=56)), dict(latent=pool(k_rot_row_stride=68))]


@pytest.mark.parametrize("kw", BAD_ATTN)
def test_tree_attention_refuses(kw):
    assert attn(attn_io(**kw)) == ARG


def test_tree_attention_accepts_nothing_to_do_and_refuses_what_it_would_read():
    assert attn(attn_io(batch=0, ctx_len=None, cu_nodes=None)) == OK  # no requests
    assert attn(attn_io(n_nodes=0)) == OK
    assert attn(attn_io(batch=0, ctx_len=None, block_table=None)) == OK
    assert attn(attn_io(batch=2, q_abs=None)) == ARG
    assert attn(attn_io(batch=2, q_abs=FAKE + 2)) == ARG
    assert attn(attn_io(batch=2, ctx=None)) == ARG
    assert attn(attn_io(batch=2), ws=None) == WS
    assert attn(attn_io(batch=2), nbytes=10) == WS
    c = cfg()
    c.n_heads = 32
    assert attn(attn_io(), c) == UNS
    assert lib().wl_mla_tree_attn(None, C.byref(attn_io()), FAKE, 1 << 40, None) == ARG
    assert lib().wl_mla_tree_attn(C.byref(cfg()), None, FAKE, 1 << 40, None) == ARG
    assert lib().wl_tree_attn_workspace_bytes(None, 1, 1) == 0 and lib().wl_tree_attn_workspace_bytes(C.byref(cfg()), 0, 1) == 0


def plan_io(**kw):
    f = dict(batch=2, n_tokens=4, page_size=16, n_pages=10, table_stride=4, max_pages=4)
    for k in ("ctx_len", "n_new", "block_table", "n_held", "n_held_out", "free_list", "n_free", "n_free_out", "cu_new",
              "short_out", "slot", "pos", "seq"):
        f[k] = FAKE
    f.update(kw)
    return _lib.PagePlanIO(**f)


@pytest.mark.parametrize("kw", [dict(batch=-1), dict(n_tokens=-1), dict(page_size=0), dict(n_pages=0), dict(max_pages=0),
                                dict(table_stride=3), dict(page_size=1 << 20, n_pages=1 << 11)] +
                         [{k: None} for k in ("ctx_len", "n_new", "block_table", "n_held", "n_held_out", "free_list", "n_free",
                                              "n_free_out", "cu_new", "short_out", "slot", "pos", "seq")])
def test_page_plan_refuses(kw):
    assert lib().wl_page_plan(C.byref(plan_io(**kw)), None) == ARG


def test_page_release_refuses():
    good = [2, FAKE, FAKE, 4, 4, FAKE, FAKE, 10, FAKE]
    for i, bad in ((0, -1), (1, None), (2, None), (3, 3), (4, 0), (5, None), (6, None), (7, 0), (8, None)):
        a = list(good)
        a[i] = bad
        assert lib().wl_page_release(*a, None) == ARG, i
    assert lib().wl_page_release(0, *good[1:], None) == OK
    assert lib().wl_page_release(0, None, None, 4, 4, None, None, 10, None, None) == OK  # no requests, no table


def commit_io(**kw):
    f = dict(batch=2, n_nodes=3, page_size=16, n_pages=10, table_stride=4, max_pages=4, n_layers=1,
             latent=(LatentCache * 1)(pool()))
    for i, k in enumerate(("ctx_len", "cu_nodes", "parent", "draft", "target", "block_table", "n_accept", "path", "next", "ctx_out")):
        f[k] = FAKE + 4096 * i
    f.update(kw)
    return _lib.TreeCommitIO(**f)


@pytest.mark.parametrize("kw", [dict(batch=-1), dict(batch=65536), dict(n_nodes=-1), dict(n_layers=-1), dict(latent=None),
                                dict(page_size=0), dict(n_pages=0), dict(max_pages=5), dict(ctx_out=FAKE),
                                dict(latent=(LatentCache * 1)(pool(c_kv_row_stride=100))),
                                dict(latent=(LatentCache * 1)(pool(k_rot=FAKE + 2))),
                                dict(index=(IndexCache * 1)(IndexCache(FAKE, 0, None, 0))),
                                dict(index=(IndexCache * 1)(IndexCache(FAKE + 4, 0, FAKE, 0)))] +
                         [{k: None} for k in ("ctx_len", "cu_nodes", "parent", "draft", "target", "block_table", "n_accept",
                                              "path", "next", "ctx_out")])
def test_tree_commit_refuses(kw):
    assert lib().wl_tree_commit(C.byref(cfg()), C.byref(commit_io(**kw)), None) == ARG


def test_tree_commit_of_no_requests():
    assert lib().wl_tree_commit(C.byref(cfg()), C.byref(commit_io(batch=0, ctx_len=None)), None) == OK
    assert lib().wl_tree_commit(None, C.byref(commit_io()), None) == ARG


def test_cache_append_paged_refuses():
    io = _lib.CacheAppendIO(n=0, n_seq=1)
    f = lib().wl_cache_append_paged
    assert f(C.byref(cfg()), C.byref(io), 10, None) == OK
    assert f(C.byref(cfg()), C.byref(io), 0, None) == ARG
    assert f(C.byref(cfg()), None, 10, None) == ARG
    io.seq = FAKE
    assert f(C.byref(cfg()), C.byref(io), 10, None) == ARG
    io.seq, io.n_seq = None, 2
    assert f(C.byref(cfg()), C.byref(io), 10, None) == ARG


def test_python_checks_run_before_any_launch():
    z = torch.zeros(4, dtype=torch.int32)
    kv = torch.zeros(32, 576, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        P.page_plan(z, z, z.view(4, 1), z, z, z, 8, 4)
    with pytest.raises(ValueError, match="int32"):
        P.page_plan(z, z.long(), z.view(4, 1), z, z, z, 8, 4)
    with pytest.raises(ValueError, match="2 elements"):
        P.page_plan(z[:2], z[:1], z.view(4, 1), z, z, z, 8, 4)
    with pytest.raises(ValueError, match="CUDA"):
        P.page_release(z, z.view(4, 1), z, z, z)
    for bad in (dict(page_size=12), dict(page_size=0), dict(page_size=64), dict(c_kv=kv[:, :500])):
        f = dict(c_kv=kv[:, :512], k_rot=kv[:, 512:], page_size=16, block_table=z.view(2, 2))
        f.update(bad)
        with pytest.raises(ValueError):
            P.PagedKV(**f)
    with pytest.raises(ValueError):
        P.LayerCaches([])


def layout(name, **known):
    """The uint32_t constants of a shared-memory layout in tree_pair.cuh."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "windlass_b200", "csrc", "tree_pair.cuh")
    with open(path) as f:
        src = f.read()
    vals = {k: int(v) for k, v in re.findall(r"constexpr int (TP_\w+) = (\d+);", src)}
    vals.update(known)
    for k, v in re.findall(r"static constexpr \w+ (\w+) = (.*?);", src[src.index("struct " + name):]):
        if "idesc" not in v:
            for part in [x.split("=") for x in (k + "=" + v).split(", ")]:
                vals[part[0].strip()] = eval(part[1], {}, vals)
    return vals, src


def test_no_copy_of_the_other_cta_lands_on_the_schedule():
    """The score CTA sends P, rescale factors and 1 / l into the value CTA's shared memory as soon as it has them: the value
    CTA's schedule, which nothing holds them back for, lies elsewhere."""
    v, src = layout("TpLayout", TA_TILE=64)
    assert re.search(r"cost = reinterpret_cast<TreeCost\*>\(smem \+ L::OFF_SCHED\)", src)
    assert re.search(r"tab = reinterpret_cast<int2\*>\(many \? smem : smem \+ L::OFF_SCHED \+ sizeof\(TreeCost\)\)", src)
    cost = 4 * 3 * 64 * 4 + 32 * 8  # four sums for three thirds of the requests and 64 choices; (nodes, tiles) of 32 requests
    sched = (v["OFF_SCHED"], v["OFF_SCHED"] + cost)
    many = (0, 16384 * 8)  # the table of more requests
    for first, size in ((v["OFF_P"], v["TP_P"] * v["P"]), (v["OFF_ALPHA"], v["TP_P"] * 512), (v["OFF_FIN"], 512),
                        (v["OFF_BAR"], 8 * v["N_BARS"])):
        for a, b in (sched, many):
            assert b <= first or first + size <= a


def test_page_plan_takes_the_trees_in_one_form():
    assert lib().wl_page_plan(C.byref(plan_io(parent=FAKE, tree_mask=FAKE)), None) == ARG
    z = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="not both"):
        P.page_plan(z, z, z.view(4, 1), z, z, z, 8, 4, parent=z, mask=z.long())
    with pytest.raises(ValueError, match="parent must hold 4"):
        P.page_plan(z, z, z.view(4, 1), z, z, z, 8, 4, parent=z[:3])
    with pytest.raises(ValueError, match="int32"):
        P.page_plan(z, z, z.view(4, 1), z, z, z, 8, 4, parent=z.long())
    with pytest.raises(ValueError, match="int64"):
        P.page_plan(z, z, z.view(4, 1), z, z, z, 8, 4, mask=z)


def test_tree_commit_refuses_a_pool_named_twice():
    two = dict(n_layers=2, batch=0, ctx_len=None)
    commit = lambda **kw: lib().wl_tree_commit(C.byref(cfg()), C.byref(commit_io(**two, **kw)), None)  # noqa: E731
    pools = (LatentCache * 2)(pool(), pool(c_kv=FAKE + 4096, k_rot=FAKE + 5120))
    assert commit(latent=pools) == OK
    assert commit(latent=(LatentCache * 2)(pool(), pool())) == ARG
    keys = [IndexCache(FAKE + 8192 * i, 0, FAKE, 0) for i in (1, 2)]
    assert commit(latent=pools, index=(IndexCache * 2)(*keys)) == OK
    assert commit(latent=pools, index=(IndexCache * 2)(keys[0], IndexCache())) == OK
    assert commit(latent=pools, index=(IndexCache * 2)(IndexCache(), IndexCache())) == OK
    assert commit(latent=pools, index=(IndexCache * 2)(keys[0], keys[0])) == ARG
    for n in (78, 512, 700):
        many = [pool(c_kv=FAKE + 4096 * i) for i in range(n)]
        io = commit_io(n_layers=n, batch=0, ctx_len=None, latent=(LatentCache * n)(*many))
        assert lib().wl_tree_commit(C.byref(cfg()), C.byref(io), None) == OK
        io.latent[n - 1] = many[n // 3]
        assert lib().wl_tree_commit(C.byref(cfg()), C.byref(io), None) == ARG


def test_paged_append_refuses_what_it_would_read_past():
    """Sizes and devices are looked at before anything else (no CUDA tensor is needed to see them)."""
    keys = A.IndexKeys(torch.zeros(16, 128, dtype=torch.uint8), torch.zeros(16))
    good = dict(slot=torch.zeros(3, dtype=torch.int32), cos=torch.zeros(3, 32), sin=torch.zeros(3, 32), k_raw=torch.zeros(3, 128),
                k_norm_w=torch.zeros(128, dtype=torch.bfloat16), k_norm_b=torch.zeros(128, dtype=torch.bfloat16))
    call = lambda **kw: P.cache_append_paged(cfg(), keys=keys, **{**good, **kw})  # noqa: E731
    with pytest.raises(ValueError, match="CUDA"):
        call()
    for name, t in good.items():
        if name == "slot":
            continue
        with pytest.raises(ValueError, match=f"{name} must hold {t.numel()}"):
            call(**{name: t[:-1]})
    with pytest.raises(ValueError, match="kv_raw must hold 1728"):
        call(kv_raw=torch.zeros(2, 576))
    with pytest.raises(ValueError, match="kv_norm_w must hold 512"):
        call(kv_norm_w=torch.zeros(511, dtype=torch.bfloat16))
    for name, t in good.items():
        with pytest.raises(ValueError, match=f"{name} must be on cpu"):
            call(**{name: t.to("meta")})
    keys.scale = keys.scale.to("meta")
    with pytest.raises(ValueError, match="one device"):
        call()


# ---- the restatement -------------------------------------------------------------------------

def test_restated_plan_gives_every_position_its_own_slot():
    rng = np.random.default_rng(1)
    ctx, new, page = [5, 0, 17, 8], [4, 9, 0, 1], 8
    held = [1, 0, 3, 1]
    table = np.full((4, 4), -1)
    perm = rng.permutation(12)
    table[0, 0], table[2, :3], table[3, 0] = perm[0], perm[1:4], perm[4]
    r = R.page_plan(ctx, new, held, table, perm[5:], 7, page, 12, sum(new))
    assert (r["short"] == 0).all() and r["n_held"].tolist() == [2, 2, 3, 2] and r["n_free"] == 3
    slots = [int(r["table"][b, p // page]) * page + p % page for b in range(4) for p in range(ctx[b] + new[b])]
    assert len(set(slots)) == len(slots)
    assert set(r["slot"].tolist()) <= set(slots)


def test_restated_tree_attention_is_the_decode_of_each_branch():
    """A node's result equals plain attention over the context and its branch laid out in a row."""
    rng = np.random.default_rng(2)
    rows, q = rng.standard_normal((40, 576)), rng.standard_normal((4, 2, 576))
    parent, cu = [-1, 0, 0, 2], [0, 4]
    m = R.tree_masks(parent, cu)
    assert m == [0b1, 0b11, 0b101, 0b1101]
    table = np.array([[3, 1, 0, 2]])
    o, lse, _ = R.tree_attn(q, rows, [9], cu, m, table, 8, 1 / 16)
    line = [3 * 8 + i for i in range(8)] + [8] + [9, 11, 12]  # nodes 0, 2, 3 behind the context
    z = q[3] @ rows[line].T / 16
    p = np.exp(z - z.max(1, keepdims=True))
    assert np.allclose(o[3], p @ rows[line][:, :512] / p.sum(1, keepdims=True), atol=1e-12)


def test_restated_walk_takes_the_lowest_agreeing_child():
    assert R.tree_walk([-1, 0, 0, 2, 2], [0, 7, 7, 9, 4], [7, 1, 4, 5, 6]) == ([0, 1], 1)
    assert R.tree_walk([-1, 0, 0, 2, 2], [0, 8, 7, 9, 4], [7, 1, 4, 5, 6]) == ([0, 2, 4], 6)
    assert R.tree_walk([], [], []) == ([], -1)
