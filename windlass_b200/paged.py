"""A paged latent cache and drafted trees: the serving step around speculative decoding.

One pool of cache rows serves requests of different lengths: a page is ``page_size``
consecutive rows ("slots") and a request's block table lists its pages in position
order. A step with drafted tokens is::

    plan = page_plan(ctx_len, n_new, table, n_held, free_list, n_free, page_size, n_tokens, parent=parent)
    cos, sin = cos_table[plan["pos"]], sin_table[plan["pos"]]                   # of the queries too
    cache_append_paged(cfg, plan["slot"], cos, sin, kv=kv, kv_raw=..., ...)     # each layer
    out = mla_tree_attn(cfg, kv, q_abs, ctx_len, plan["cu"], parent=parent)     # each layer
    done = tree_commit(layers, ctx_len, plan["cu"], parent, draft, target)

Everything that changes from step to step lives in device tensors, nothing
synchronises, and each call runs on the current stream of its tensors' device, so a
step can be captured into a CUDA graph. Outputs and workspaces are allocated per call
from torch's caching allocator (two streams or two graphs never share one). The C ABI
behind these calls is in ``include/wl_attn.h``; the reference has no counterpart (it
decodes one sequence, one token at a time, greedily).
"""
from __future__ import annotations

import ctypes as C
import functools
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import AttnCfg, IndexCache, LatentCache, PagedKVC, check, lib
from .attn import D_QK, KV_LORA, N_HEADS, IndexKeys, LatentKV, cache_append_io

TREE_MAX = _lib.WL_TREE_MAX
_I32 = torch.int32


def _i32(t: torch.Tensor, name: str, dev: torch.device, numel: int | None = None) -> int:
    """Address of a contiguous int32 tensor on ``dev`` with at least ``numel`` elements."""
    if t.dtype != _I32:
        raise ValueError(f"{name} must be {_I32}, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{name} must be on {dev}, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if numel is not None and t.numel() < numel:
        raise ValueError(f"{name} must hold {numel} elements, got {t.numel()}")
    return t.data_ptr()


def _table(t: torch.Tensor, batch: int, dev: torch.device) -> tuple[int, int, int]:
    """(address, row stride, entries a row) of a block table of at least ``batch`` rows."""
    if t.dtype != _I32 or t.dim() != 2 or t.device != dev:
        raise ValueError(f"block_table must be a 2-D int32 tensor on {dev}")
    rows, width = t.shape
    row, col = t.stride()
    if rows < batch or (width > 1 and col != 1) or (batch > 1 and row < width):
        raise ValueError(f"block_table must have {batch} rows of consecutive entries")
    return t.data_ptr(), row if batch > 1 else max(width, 1), width


def _trees(parent: torch.Tensor | None, mask: torch.Tensor | None, n: int, dev: torch.device) -> tuple:
    """Addresses of the trees of ``n`` rows: parents (int32) or masks (int64), the other None."""
    if parent is not None and mask is not None:
        raise ValueError("give parent or mask, not both")
    if mask is None:
        return None if parent is None else _i32(parent, "parent", dev, n), None
    if mask.dtype != torch.int64 or mask.device != dev or not mask.is_contiguous() or mask.numel() < n:
        raise ValueError(f"mask must be a contiguous int64 tensor of {n} elements on {dev}")
    return None, mask.data_ptr()


def _call(dev: torch.device, fn, *args) -> int:
    """``fn(*args, stream)`` on the current stream of ``dev``, with that device current (as torch's
    own operators do)."""
    if dev.type != "cuda":
        raise ValueError(f"tensors must be CUDA tensors, got {dev}")
    if torch._C._cuda_getDevice() == dev.index:
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    with torch.cuda.device(dev):
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))


@dataclass(frozen=True, eq=False)
class PagedKV:
    """One layer's latent pool: c_kv [slots, 512] and k_rot [slots, 64] bf16 (rows of any
    stride that keeps them 16-byte aligned), pages of ``page_size`` rows (a multiple of
    8), ``block_table`` [batch, max_pages] int32. Slots past the last whole page are
    not used. ``packed(kv)`` splits a [slots, 576] tensor. The tensors' contents, the table's
    included, may change freely, the tensors themselves not (other ones: a new object). A table no
    wider than the requests need lets ``mla_tree_attn`` choose its kernel well."""
    c_kv: torch.Tensor
    k_rot: torch.Tensor
    page_size: int
    block_table: torch.Tensor

    @staticmethod
    def packed(kv: torch.Tensor, page_size: int, block_table: torch.Tensor) -> "PagedKV":
        return PagedKV(kv[:, :KV_LORA], kv[:, KV_LORA:], page_size, block_table)

    def __post_init__(self):
        ckv, krt, t = self.c_kv, self.k_rot, self.block_table
        if ckv.dim() != 2 or krt.dim() != 2 or ckv.shape[0] != krt.shape[0]:
            raise ValueError("c_kv and k_rot must be [slots, 512] and [slots, 64]")
        if ckv.shape[1] != KV_LORA or krt.shape[1] != D_QK - KV_LORA:
            raise ValueError("c_kv and k_rot must be [slots, 512] and [slots, 64]")
        if krt.device != ckv.device:
            raise ValueError(f"k_rot must be on {ckv.device}, got {krt.device}")
        n_pages = ckv.shape[0] // self.page_size if self.page_size > 0 else 0
        if self.page_size <= 0 or self.page_size % 8 or n_pages <= 0:
            raise ValueError("page_size must be a multiple of 8 that the pool holds at least once")
        lat = LatentKV(ckv.unsqueeze(0), krt.unsqueeze(0)).c()
        # the addresses are taken here, so the fields are frozen
        object.__setattr__(self, "n_pages", n_pages)
        object.__setattr__(self, "_c", PagedKVC(lat, self.page_size, n_pages, *_table(t, t.shape[0], ckv.device)))

    def c(self) -> PagedKVC:
        return self._c

    def latent(self) -> LatentKV:
        """The pool as a cache of one sequence."""
        return LatentKV(self.c_kv.unsqueeze(0), self.k_rot.unsqueeze(0))


# ---- block tables and slot maps ------------------------------------------------------------------

def page_plan(ctx_len: torch.Tensor, n_new: torch.Tensor, block_table: torch.Tensor, n_held: torch.Tensor,
              free_list: torch.Tensor, n_free: torch.Tensor, page_size: int, n_tokens: int, *,
              in_place: bool = False, parent: torch.Tensor | None = None, mask: torch.Tensor | None = None) -> dict:
    """Pages and slots for ``n_new[b]`` tokens behind ``ctx_len[b]`` cached ones
    (``wl_page_plan``). New pages come from the top of the stack ``free_list[:n_free]`` in
    request order and are written into ``block_table``. Returns slot, pos, seq
    [n_tokens] (rows behind the last token: -1), cu [batch + 1], short [batch] (pages a
    request lacks; such a request gets none, and slots and table entries of -1), n_held [batch] and
    n_free [1] after the call: new tensors, or the given ones with ``in_place``.

    ``pos`` is what a token's query and keys are rotated by: ``ctx_len`` + its number in the
    request, or, with the trees that ``mla_tree_attn`` gets (``parent`` or ``mask``, at least
    [n_tokens]), ``ctx_len`` + the number of its ancestors (the other nodes of its mask), so
    that siblings share a position. Slots are one a token either way. A request of more than 64 tokens is a
    prompt: its positions run on."""
    dev = ctx_len.device
    B, T = ctx_len.numel(), int(n_tokens)
    c, n, held, nf = (_i32(ctx_len, "ctx_len", dev), _i32(n_new, "n_new", dev, B), _i32(n_held, "n_held", dev, B),
                      _i32(n_free, "n_free", dev, 1))
    table, stride, width = _table(block_table, B, dev)
    free = _i32(free_list, "free_list", dev)
    if T < 0:
        raise ValueError("n_tokens must not be negative")
    par, m = _trees(parent, mask, T, dev)
    # one allocation: slot, pos, seq [T], cu [B + 1], short [B] and, unless in place, n_held [B] and n_free [1]
    sizes = [T, T, T, B + 1, B] if in_place else [T, T, T, B + 1, B, B, 1]
    out = torch.empty(sum(sizes), dtype=_I32, device=dev)
    o = out.data_ptr()
    short = o + 4 * (3 * T + B + 1)
    io = _lib.PagePlanIO(B, T, page_size, free_list.numel(), c, n, table, stride, width, held,
                         held if in_place else short + 4 * B, free, nf, nf if in_place else short + 8 * B, o + 12 * T,
                         short, o, o + 4 * T, o + 8 * T, par, m)
    check(_call(dev, lib().wl_page_plan, C.byref(io)), "wl_page_plan")
    parts = torch.unsafe_split_with_sizes(out, sizes)  # (integers: no gradient to track, and `out` ends here)
    return dict(slot=parts[0], pos=parts[1], seq=parts[2], cu=parts[3], short=parts[4],
                n_held=n_held if in_place else parts[5], n_free=n_free if in_place else parts[6])


def page_release(done: torch.Tensor, block_table: torch.Tensor, n_held: torch.Tensor, free_list: torch.Tensor,
                 n_free: torch.Tensor) -> None:
    """Push the pages of the requests with ``done[b] != 0`` back on the free stack, in
    place (``wl_page_release``)."""
    dev = done.device
    B = done.numel()
    args = (B, _i32(done, "done", dev), *_table(block_table, B, dev), _i32(n_held, "n_held", dev, B), _i32(free_list, "free_list", dev), free_list.numel(),
            _i32(n_free, "n_free", dev, 1))
    check(_call(dev, lib().wl_page_release, *args), "wl_page_release")


# ``cache_append``'s tensors: elements a token, or in all
_APPEND = (("k_raw", 128, 0), ("k_norm_w", 0, 128), ("k_norm_b", 0, 128), ("kv_raw", D_QK, 0), ("kv_norm_w", 0, KV_LORA))


def cache_append_paged(cfg: AttnCfg, slot: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                       kv: PagedKV | None = None, keys: IndexKeys | None = None, **kw) -> None:
    """``cache_append`` into pools: token i goes to row ``slot[i]`` (``page_plan``'s slots), -1
    is skipped. ``keys`` is the owner layer's index pool (keys [slots, 128], scale
    [slots]); the other arguments are ``cache_append``'s, for every token of ``slot``, and all
    are on the pools' device."""
    pools = ([kv.c_kv] if kv is not None else []) + ([keys.keys, keys.scale] if keys is not None else [])
    if not pools:
        raise ValueError("cache_append_paged needs kv or keys")
    if keys is not None and (keys.keys.dim() != 2 or keys.scale.dim() != 1):
        raise ValueError("index pools must be [slots, 128] with scales [slots]")
    dev, n = pools[0].device, slot.numel()
    for t in pools:
        if t.device != dev:
            raise ValueError(f"the pools must be on one device, got {dev} and {t.device}")
    for name, t, numel in (("slot", slot, n), ("cos", cos, 32 * n), ("sin", sin, 32 * n),
                           *((k, kw[k], w * n if w else m) for k, w, m in _APPEND if kw.get(k) is not None)):
        if t.device != dev:
            raise ValueError(f"{name} must be on {dev}, got {t.device}")
        if t.numel() < numel:
            raise ValueError(f"{name} must hold {numel} elements, got {t.numel()}")
    io, hold = cache_append_io(slot, cos, sin, kv=None if kv is None else kv.latent(), keys=keys, **kw)
    n_slots = min(t.shape[0] for t in pools)
    check(_call(dev, lib().wl_cache_append_paged, C.byref(cfg), C.byref(io), n_slots), "wl_cache_append_paged")


# ---- attention of drafted trees ------------------------------------------------------------------

def mla_tree_attn(cfg: AttnCfg, kv: PagedKV, q_abs: torch.Tensor, ctx_len: torch.Tensor, cu_nodes: torch.Tensor, *,
                  parent: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                  sel_in: torch.Tensor | None = None, sel_n_in: torch.Tensor | None = None,
                  out_dtype: torch.dtype = torch.float32, ctx: torch.Tensor | None = None,
                  lse: torch.Tensor | None = None) -> dict:
    """Absorbed-MLA attention of every request's drafted nodes (``wl_mla_tree_attn``).

    q_abs bf16 [n, 64, 576]; request b's rows are ``cu_nodes[b]:cu_nodes[b + 1]`` and its
    node i's cache row is that of position ``ctx_len[b] + i`` (``page_plan``'s slot; rotated by its ``pos``). A row sees the context and its
    ancestors by ``parent`` [n] (int32, index within the request, -1 for a root), or the
    nodes of ``mask`` [n] (int64 bit masks), or nodes 0..i (neither given: a chain; one node
    is plain decode). ``sel_in`` [n, k] int32 (with counts ``sel_n_in`` [n]) narrows each
    row to its own list of unique positions, in any order (counts above k end there). Returns ctx [n, 64, 512] of
    ``out_dtype`` (float32 or bfloat16) and lse [n, 64] fp32 — the given tensors, where
    given; rows behind the last request are not written."""
    dev = q_abs.device
    shape, B = q_abs.shape, ctx_len.numel()
    n = shape[0] if shape else 0
    if q_abs.dtype != torch.bfloat16 or len(shape) != 3 or shape[1] != N_HEADS or shape[2] != D_QK:
        raise ValueError("q_abs must be bf16 [n, 64, 576]")
    if kv.c_kv.device != dev:
        raise ValueError(f"the pool must be on {dev}, got {kv.c_kv.device}")
    if kv.block_table.shape[0] < B:
        raise ValueError(f"block_table must have {B} rows")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("out_dtype must be float32 or bfloat16")
    if sel_in is None and sel_n_in is not None:
        raise ValueError("sel_n_in needs sel_in")
    q_abs = q_abs.contiguous()
    par, m = _trees(parent, mask, n, dev)
    mode, sel, seln, stride, k = _lib.WL_MODE_DENSE, None, None, 0, 0
    if sel_in is not None:
        if sel_in.dim() != 2 or sel_in.shape[0] < n or sel_in.shape[1] < 1 or (sel_in.shape[1] > 1 and sel_in.stride(1) != 1):
            raise ValueError(f"sel_in must be [{n}, k] with consecutive entries")
        if sel_in.dtype != _I32 or sel_in.device != dev:
            raise ValueError(f"sel_in must be {_I32} on {dev}")
        if sel_in.shape[0] > 1 and sel_in.stride(0) < sel_in.shape[1]:
            raise ValueError("the rows of sel_in must not overlap (an expanded list: one contiguous row a node)")
        mode, sel, k = _lib.WL_MODE_CONSUMER, sel_in.data_ptr(), sel_in.shape[1]
        stride = sel_in.stride(0) if sel_in.shape[0] > 1 else k
        seln = None if sel_n_in is None else _i32(sel_n_in, "sel_n_in", dev, n)
    if ctx is None:
        ctx = torch.empty(n, N_HEADS, KV_LORA, dtype=out_dtype, device=dev)
    elif ctx.dtype != out_dtype or ctx.device != dev or not ctx.is_contiguous() or ctx.numel() != n * N_HEADS * KV_LORA:
        raise ValueError(f"ctx must be a contiguous {out_dtype} tensor [{n}, 64, 512] on {dev}")
    if lse is None:
        lse = torch.empty(n, N_HEADS, dtype=torch.float32, device=dev)
    elif lse.dtype != torch.float32 or lse.device != dev or not lse.is_contiguous() or lse.numel() != n * N_HEADS:
        raise ValueError(f"lse must be a contiguous float32 tensor [{n}, 64] on {dev}")
    io = _lib.TreeAttnIO(B, n, _i32(ctx_len, "ctx_len", dev), _i32(cu_nodes, "cu_nodes", dev, B + 1), m, par, kv.c(),
                         q_abs.data_ptr(), mode, _lib.WL_BF16 if out_dtype == torch.bfloat16 else _lib.WL_F32, sel, seln,
                         k, stride, ctx.data_ptr(), lse.data_ptr())
    L, nbytes = lib(), _tree_workspace(B, n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    check(_call(dev, L.wl_mla_tree_attn, C.byref(cfg), C.byref(io), ws.data_ptr(), nbytes), "wl_mla_tree_attn")
    return dict(ctx=ctx, lse=lse)


@functools.lru_cache(maxsize=1024)
def _tree_workspace(batch: int, n: int) -> int:
    return max(1, lib().wl_tree_attn_workspace_bytes(C.byref(_default_cfg()), batch, n))


# ---- the commit ----------------------------------------------------------------------------------

class LayerCaches:
    """The pools that ``tree_commit`` moves rows in: ``kvs`` one ``PagedKV`` per layer, ``keys``
    None or one ``IndexKeys`` (pools [slots, 128] / [slots]) or None per layer. All layers
    share one block table and page size, and no two a pool (keys that several layers read are
    named once, at their owner)."""

    def __init__(self, kvs: list[PagedKV], keys: list[IndexKeys | None] | None = None):
        if not kvs:
            raise ValueError("LayerCaches needs at least one layer")
        if keys is not None and len(keys) != len(kvs):
            raise ValueError(f"{len(kvs)} latent pools, {len(keys)} index pools")
        first = kvs[0]
        rows = first.c_kv.shape[0]
        for kv in kvs:
            t, u = kv.block_table, first.block_table
            if kv.page_size != first.page_size or t.data_ptr() != u.data_ptr() or t.shape != u.shape or t.stride() != u.stride():
                raise ValueError("the layers must share one block table and page size")
            if kv.c_kv.device != first.c_kv.device:
                raise ValueError("the layers must be on one device")
            rows = min(rows, kv.c_kv.shape[0])
        self.kvs, self.keys = list(kvs), None if keys is None else list(keys)
        self._latent = (LatentCache * len(kvs))(*[kv.c().latent for kv in kvs])
        self._index = None
        if keys is not None:
            self._index = (IndexCache * len(kvs))()
            for i, k in enumerate(keys):
                if k is None:
                    continue
                if k.keys.dim() != 2 or k.scale.dim() != 1 or k.keys.device != first.c_kv.device or \
                        k.scale.device != first.c_kv.device:
                    raise ValueError("index pools must be [slots, 128] with scales [slots], on the layers' device")
                rows = min(rows, k.keys.shape[0], k.scale.shape[0])
                self._index[i] = k.c()
        for what, at in (("latent", [kv.c_kv.data_ptr() for kv in kvs]), ("index", [k.keys.data_ptr() for k in keys or () if k is not None])):
            if len(set(at)) < len(at):
                raise ValueError(f"two layers share one {what} pool: its rows would move twice")
        self.n_pages = rows // first.page_size
        if self.n_pages <= 0:
            raise ValueError("a pool holds less than one page")


def tree_commit(layers: LayerCaches, ctx_len: torch.Tensor, cu_nodes: torch.Tensor, parent: torch.Tensor,
                draft: torch.Tensor, target: torch.Tensor, cfg: AttnCfg | None = None) -> dict:
    """Greedy verification and commit (``wl_tree_commit``): from node 0 the path goes to the
    lowest child whose ``draft`` token is the current node's ``target`` token; its cache
    rows move to positions ctx_len + d in every layer. Returns n_accept [batch], path
    [batch, 64] (-1 behind the path), next [batch] (the target of the last node) and
    ctx_len [batch] after the commit. Nothing of a request that lacks a page is committed."""
    dev = ctx_len.device
    B, n = ctx_len.numel(), parent.numel()
    first = layers.kvs[0]
    kv = first.c()
    if first.c_kv.device != dev:
        raise ValueError(f"ctx_len must be on {first.c_kv.device}, got {dev}")
    if first.block_table.shape[0] < B:
        raise ValueError(f"block_table must have {B} rows")
    sizes = [TREE_MAX * B, B, B, B]
    out = torch.empty((TREE_MAX + 3) * B, dtype=_I32, device=dev)
    path = out.data_ptr()
    acc = path + 4 * TREE_MAX * B
    io = _lib.TreeCommitIO(B, n, _i32(ctx_len, "ctx_len", dev), _i32(cu_nodes, "cu_nodes", dev, B + 1),
                           _i32(parent, "parent", dev), _i32(draft, "draft", dev, n), _i32(target, "target", dev, n),
                           kv.page_size, layers.n_pages, kv.block_table, kv.table_stride, kv.max_pages,
                           len(layers.kvs), layers._latent, layers._index, acc, path, acc + 4 * B, acc + 8 * B)
    check(_call(dev, lib().wl_tree_commit, C.byref(cfg if cfg is not None else _default_cfg()), C.byref(io)), "wl_tree_commit")
    parts = torch.unsafe_split_with_sizes(out, sizes)
    return dict(n_accept=parts[1], path=parts[0].view(B, TREE_MAX), next=parts[2], ctx_len=parts[3])


_cfg: AttnCfg | None = None


def _default_cfg() -> AttnCfg:
    global _cfg
    if _cfg is None:
        c = AttnCfg()
        lib().wl_attn_cfg_glm52(C.byref(c), 1)
        _cfg = c
    return _cfg
