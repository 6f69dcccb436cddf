"""Cases and plain forms of the paged-cache and drafted-tree operators.

Three operators of one serving step: the page plan (block tables and slot maps from request
lengths), absorbed-MLA attention of drafted trees over the paged latent cache (every key, or a
selection per node), and the commit (greedy walk of the tree, accepted rows moved up in every
layer's cache). ``run`` with ``own`` false computes them from elementary torch operations;
with ``own`` true through ``windlass_b200.paged``. ``exact`` restates them in 64 bits.
"""
import math
import random

import torch

own = False

H, LORA, D = 64, 512, 576  # heads, latent columns, latent + roped columns of a cache row
SCALE = 1.0 / 16.0


# ---- cases ---------------------------------------------------------------------------------------

def listed():
    return [
        # pages and slots of one decode step: 64 requests, a tree of up to 16 drafted tokens each
        dict(name="plan_decode", op="plan", batch=64, ctx=8192, new=16, page=64, lens=1),
        # a prefill step: 24 ragged prompts, tens of thousands of tokens in small pages
        dict(name="plan_prefill", op="plan", batch=24, ctx=0, new=4001, page=16, lens=2),
        # one request, one token, a short context: latency alone
        dict(name="tree_single", op="tree", batch=1, nodes=1, ctx=1000, page=64, lens=3),
        # four requests with small ragged trees, pages that end inside a key tile
        dict(name="tree_small", op="tree", batch=4, nodes=7, ctx=4099, page=16, lens=4),
        # plain batched decode: 32 requests of very different lengths, one token each
        dict(name="tree_decode32", op="tree", batch=32, nodes=1, ctx=8192, page=64, lens=5),
        # one request at the longest context of the benchmark, a short chain of drafts
        dict(name="tree_long", op="tree", batch=1, nodes=3, ctx=131069, page=64, lens=6),
        # a serving batch: 8 requests x trees of up to 16 nodes
        dict(name="tree_serve", op="tree", batch=8, nodes=16, ctx=16384, page=64, lens=7),
        # the largest: 16 requests x trees of up to 32 nodes at 32K keys
        dict(name="tree_large", op="tree", batch=16, nodes=32, ctx=32768, page=64, lens=8),
        # a sparse layer, one request: 2048 selected keys for each of 4 nodes
        dict(name="sel_small", op="sel", batch=1, nodes=4, ctx=8192, page=16, topk=2048, lens=9),
        # a sparse layer of the serving batch
        dict(name="sel_serve", op="sel", batch=8, nodes=16, ctx=32768, page=64, topk=2048, lens=10),
        # commit of 8 requests over every layer of the model (latent rows)
        dict(name="commit_layers", op="commit", batch=8, branches=4, depth=5, ctx=100, page=64, layers=78,
             index=False, lens=11),
        # commit of a large batch into one owner layer (latent rows and indexer keys)
        dict(name="commit_batch", op="commit", batch=64, branches=3, depth=9, ctx=300, page=16, layers=1,
             index=True, lens=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "tree", "tree", "tree", "sel", "commit"])
    page = rng.choice([8, 16, 32, 48, 64, 128, 256])
    lens = rng.randrange(1 << 30)
    if op == "plan":
        return dict(op=op, batch=_log(rng, 1, 512), ctx=_log(rng, 1, 32768), new=_log(rng, 1, 120), page=page,
                    lens=lens)
    if op == "tree":
        batch, nodes = _log(rng, 1, 32), _log(rng, 1, 64)
        ctx = _log(rng, 1, min(131072, 2 ** 21 // batch, 2 ** 24 // (batch * nodes)))
        return dict(op=op, batch=batch, nodes=nodes, ctx=ctx, page=page, lens=lens)
    if op == "sel":
        return dict(op=op, batch=_log(rng, 1, 8), nodes=_log(rng, 1, 16), ctx=_log(rng, 1, 32768), page=page,
                    topk=_log(rng, 1, 2048), lens=lens)
    return dict(op=op, batch=_log(rng, 1, 64), branches=rng.randint(1, 4), depth=rng.randint(1, 15),
                ctx=_log(rng, 1, 300), page=page, layers=_log(rng, 1, 16), index=rng.random() < 0.5, lens=lens)


def _lens(case):
    """Context lengths and token counts of the case's requests (plain lists)."""
    r = random.Random(case["lens"])
    B = case["batch"]
    ctx = [r.randint(case["ctx"] // 2, case["ctx"]) for _ in range(B)]
    most = case.get("new", case.get("nodes"))
    if most is None:
        most = 1 + case["branches"] * case["depth"]
        return ctx, [most] * B
    new = [r.randint((most + 1) // 2, most) for _ in range(B)]
    ctx[0], new[0] = case["ctx"], most
    return ctx, new


# ---- inputs --------------------------------------------------------------------------------------

def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pages(case, ctx, new, gen, filled):
    """A pool with every request's pages in random order: (table, pages held, free list, free count, pool pages).
    ``filled``: pages for the new tokens are in the table already."""
    P = case["page"]
    held = [(c + (n if filled else 0) + P - 1) // P for c, n in zip(ctx, new)]
    most = [(c + n + P - 1) // P for c, n in zip(ctx, new)]
    n_pages = sum(most) + 5
    perm = torch.randperm(n_pages, generator=gen, device="cuda", dtype=torch.int32)
    width = max(max(most), 1)
    start = torch.tensor([sum(held[:i]) for i in range(len(held))], device="cuda")[:, None]
    col = torch.arange(width, device="cuda")[None]
    h = torch.tensor(held, device="cuda")[:, None]
    table = torch.where(col < h, perm[(start + col).clamp(max=n_pages - 1)], torch.zeros_like(perm[:1]))
    free = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    n_free = n_pages - sum(held)
    free[:n_free] = perm[sum(held):]
    return table.contiguous(), _i32(held), free, _i32([n_free]), n_pages


def _parents(new, rng):
    """A tree per request: node 0 is the root, later nodes hang from one of the four before them."""
    out = []
    for n in new:
        out += [-1] + [rng.randint(max(0, j - 4), j - 1) for j in range(1, n)] if n else []
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    ctx, new = _lens(case)
    B, P, op = case["batch"], case["page"], case["op"]
    s = dict(case=case, op=op, ctx_len=_i32(ctx), most=max(new), n_rows=sum(new), L=max(c + n for c, n in zip(ctx, new)))
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s["cu"] = _i32(cu)
    if op == "plan":
        s["n_new"] = _i32(new)
        s["table"], s["held"], s["free"], s["n_free"], s["n_pages"] = _pages(case, ctx, new, gen, False)
        return s
    table, _, _, _, n_pages = _pages(case, ctx, new, gen, True)
    s["table"] = table
    rows = n_pages * P
    if op in ("tree", "sel"):
        s["kv"] = torch.randn(rows, D, generator=gen, device="cuda", dtype=torch.bfloat16)
        s["q"] = torch.randn(sum(new), H, D, generator=gen, device="cuda", dtype=torch.bfloat16)
        s["parent"] = _i32(_parents(new, rng))
        if op == "sel":  # the node's best keys among the prefix, and its ancestors where they are among them
            k = case["topk"]
            seq = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(new, device="cuda"))
            full = s["ctx_len"].long()[seq] + 1 + torch.arange(sum(new), device="cuda") - s["cu"].long()[seq]
            score = torch.rand(sum(new), s["L"], generator=gen, device="cuda")
            score = torch.where(torch.arange(s["L"], device="cuda")[None] < full[:, None], score, -1.0)
            kk = min(k, s["L"])
            top = score.topk(kk, dim=1).indices
            cnt = full.clamp(max=kk)
            top = torch.where(torch.arange(kk, device="cuda")[None] < cnt[:, None], top, s["L"])
            s["sel"] = top.sort(dim=1).values.to(torch.int32).contiguous()
            s["sel_n"] = cnt.to(torch.int32)
    else:
        L = case["layers"]
        s["kv"] = torch.randn(L, rows, D, generator=gen, device="cuda", dtype=torch.bfloat16)
        if case["index"]:
            s["keys"] = torch.randint(0, 120, (L, rows, 128), generator=gen, device="cuda", dtype=torch.uint8)
            s["scale"] = torch.rand(L, rows, generator=gen, device="cuda") + 0.5
        # a root with `branches` chains of `depth` drafts each; one chain agrees with the model for some steps
        par, draft, target = [], [], []
        for _ in range(B):
            nb, dp = case["branches"], case["depth"]
            first = rng.randrange(1000)
            p, d = [-1], [first]
            for j in range(nb):
                for i in range(dp):
                    p.append(0 if i == 0 else len(p) - 1)
                    d.append(1000 * (i + 1) + 7 * j + rng.randrange(7))
            t = [50000 + rng.randrange(100) for _ in p]
            good, upto, cur = rng.randrange(nb), rng.randint(0, dp), 0
            for i in range(upto):
                nxt = 1 + good * dp + i
                t[cur], cur = d[nxt], nxt
            par += p
            draft += d
            target += t
        s["parent"], s["draft"], s["target"] = _i32(par), _i32(draft), _i32(target)
    if own:
        from windlass_b200 import attn, paged
        if op == "commit":
            kvs = [paged.PagedKV.packed(s["kv"][i], P, table) for i in range(case["layers"])]
            keys = [attn.IndexKeys(s["keys"][i], s["scale"][i]) for i in range(case["layers"])] if case["index"] else None
            s["layers"] = paged.LayerCaches(kvs, keys)
        else:
            s["cfg"] = attn.glm52_cfg(262144)
            s["paged"] = paged.PagedKV.packed(s["kv"], P, table)
    return s


# ---- the operators in their plain form -----------------------------------------------------------

def _plan(s):
    P = s["case"]["page"]
    ctx, new, held, free = s["ctx_len"].long(), s["n_new"].long(), s["held"].long(), s["free"].long()
    n_free = s["n_free"].long()
    B, width = s["table"].shape
    need = ((ctx + new + P - 1) // P - held).clamp(min=0)
    before = need.cumsum(0) - need
    served = (need == 0) | (before + need <= n_free)
    got = torch.where(served, need, 0)
    col = torch.arange(width, device="cuda")[None]
    k = col - held[:, None]
    fresh = (k >= 0) & (k < got[:, None])
    at = (n_free - 1 - (before[:, None] + k)).clamp(0, free.numel() - 1)
    s["table"].copy_(torch.where(fresh, free[at], s["table"].long()))
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    i = torch.arange(s["n_rows"], device="cuda")
    seq = (i[:, None] >= cu[None, 1:]).sum(1)
    pos = ctx[seq] + i - cu[seq]
    slot = s["table"].long()[seq, pos // P] * P + pos % P
    slot = torch.where(served[seq], slot, -1)
    t = torch.int32
    return dict(slot=slot.to(t), pos=pos.to(t), seq=seq.to(t), cu=cu.to(t), short=torch.where(served, 0, need).to(t),
                n_held=(held + got).to(t), n_free=(n_free - got.sum()).to(t), table=s["table"])


def _ancestors(s):
    """[batch, most, most] truth values: node j is node i or above it."""
    cu, m = s["cu"].long(), s["most"]
    i = torch.arange(m, device="cuda")
    there = i[None] < (cu[1:] - cu[:-1])[:, None]
    par = s["parent"].long()[(cu[:-1, None] + i[None]).clamp(max=s["n_rows"] - 1)]
    step = ((par[:, :, None] == i[None, None, :]) & there[:, :, None]).float()
    reach = torch.matrix_power(torch.eye(m, device="cuda") + step, 64) > 0
    return reach & there[:, :, None] & there[:, None, :]


def _tree(s):
    P = s["case"]["page"]
    cu, ctx, m, L = s["cu"].long(), s["ctx_len"].long(), s["most"], s["L"]
    B = ctx.numel()
    i, t = torch.arange(m, device="cuda"), torch.arange(L, device="cuda")
    n = cu[1:] - cu[:-1]
    slot = s["table"].long()[:, t // P] * P + t % P
    here = t[None] < (ctx + n)[:, None]
    k = torch.where(here[:, :, None], s["kv"][slot].float(), 0.0)
    q = s["q"][(cu[:-1, None] + i[None]).clamp(max=s["n_rows"] - 1)].float().reshape(B, m * H, D)
    j = (t[None] - ctx[:, None])
    up = torch.gather(_ancestors(s), 2, j.clamp(0, m - 1)[:, None, :].expand(B, m, L))
    see = (j < 0)[:, None, :] | (up & (j >= 0)[:, None, :] & (j < m)[:, None, :])
    sc = torch.bmm(q, k.transpose(1, 2)).mul_(SCALE).reshape(B, m, H, L)
    sc.masked_fill_(~see[:, :, None, :], -math.inf)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    e = sc.sub_(top).exp_()
    tot = e.sum(-1)
    o = torch.bmm(e.reshape(B, m * H, L), k[:, :, :LORA]).reshape(B, m, H, LORA)
    o = torch.where(tot[..., None] > 0, o / tot[..., None], 0.0)
    lse = top[..., 0] + tot.log()
    r = torch.arange(s["n_rows"], device="cuda")
    seq = (r[:, None] >= cu[None, 1:]).sum(1)
    at = r - cu[seq]
    return dict(ctx=o[seq, at].to(torch.bfloat16), lse=lse[seq, at])


def _sel(s):
    P = s["case"]["page"]
    cu, ctx = s["cu"].long(), s["ctx_len"].long()
    r = torch.arange(s["n_rows"], device="cuda")
    seq = (r[:, None] >= cu[None, 1:]).sum(1)
    key = s["sel"].long()
    there = torch.arange(key.shape[1], device="cuda")[None] < s["sel_n"].long()[:, None]
    j = key - ctx[seq][:, None]
    up = torch.gather(_ancestors(s)[seq, r - cu[seq]], 1, j.clamp(0, s["most"] - 1))
    see = there & ((j < 0) | (up & (j < s["most"])))
    pos = torch.where(see, key, 0)
    k = s["kv"][s["table"].long()[seq[:, None], pos // P] * P + pos % P].float()
    sc = torch.bmm(s["q"].float(), k.transpose(1, 2)) * SCALE
    sc = sc.masked_fill(~see[:, None, :], -math.inf)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    e = (sc - top).exp()
    tot = e.sum(-1)
    o = torch.bmm(e, k[:, :, :LORA])
    return dict(ctx=torch.where(tot[..., None] > 0, o / tot[..., None], 0.0).to(torch.bfloat16), lse=top[..., 0] + tot.log())


def _commit(s):
    P = s["case"]["page"]
    cu, ctx, m = s["cu"].long(), s["ctx_len"].long(), s["most"]
    B = ctx.numel()
    i = torch.arange(m, device="cuda")
    there = i[None] < (cu[1:] - cu[:-1])[:, None]
    at = (cu[:-1, None] + i[None]).clamp(max=s["n_rows"] - 1)
    par, draft, target = s["parent"].long()[at], s["draft"].long()[at], s["target"].long()[at]
    fits = there & (par >= 0) & (draft == torch.gather(target, 1, par.clamp(min=0)))
    rival = fits[:, None, :] & (par[:, None, :] == par[:, :, None]) & (i[None, None, :] < i[None, :, None])
    taken = (fits & ~rival.any(2)) | ((i == 0)[None] & there)
    off = _ancestors(s) & ~taken[:, None, :]
    acc = there & ~off.any(2)
    count = acc.sum(1)
    path = torch.where(acc, i[None], 64).sort(1).values
    last = torch.gather(path, 1, (count - 1).clamp(min=0)[:, None]).clamp(max=m - 1)
    nxt = torch.where(count > 0, torch.gather(target, 1, last)[:, 0], -1)
    src, dst = ctx[:, None] + path.clamp(max=m - 1), ctx[:, None] + i[None]
    moved = i[None] < count[:, None]
    src, dst = torch.where(moved, src, ctx[:, None]), torch.where(moved, dst, ctx[:, None])
    rows = torch.arange(B, device="cuda")[:, None]
    src = (s["table"].long()[rows, src // P] * P + src % P).reshape(-1)
    dst = (s["table"].long()[rows, dst // P] * P + dst % P).reshape(-1)
    s["kv"][:, dst] = s["kv"][:, src]
    t = torch.int32
    full = torch.full((B, 64), -1, dtype=t, device="cuda")
    full[:, :m] = torch.where(moved, path, -1).to(t)
    out = dict(n_accept=count.to(t), path=full, next=nxt.to(t), ctx_len=(ctx + count).to(t), kv=s["kv"])
    if "keys" in s:
        s["keys"][:, dst] = s["keys"][:, src]
        s["scale"][:, dst] = s["scale"][:, src]
        out.update(keys=s["keys"], scale=s["scale"])
    return out


def run(s):
    op = s["op"]
    if not own:
        return dict(plan=_plan, tree=_tree, sel=_sel, commit=_commit)[op](s)
    from windlass_b200 import paged
    if op == "plan":
        r = paged.page_plan(s["ctx_len"], s["n_new"], s["table"], s["held"], s["free"], s["n_free"], s["case"]["page"],
                            s["n_rows"])
        return dict(slot=r["slot"], pos=r["pos"], seq=r["seq"], cu=r["cu"], short=r["short"], n_held=r["n_held"],
                    n_free=r["n_free"], table=s["table"])
    if op == "tree":
        r = paged.mla_tree_attn(s["cfg"], s["paged"], s["q"], s["ctx_len"], s["cu"], parent=s["parent"],
                                out_dtype=torch.bfloat16)
        return dict(ctx=r["ctx"], lse=r["lse"])
    if op == "sel":
        r = paged.mla_tree_attn(s["cfg"], s["paged"], s["q"], s["ctx_len"], s["cu"], parent=s["parent"],
                                sel_in=s["sel"], sel_n_in=s["sel_n"], out_dtype=torch.bfloat16)
        return dict(ctx=r["ctx"], lse=r["lse"])
    r = paged.tree_commit(s["layers"], s["ctx_len"], s["cu"], s["parent"], s["draft"], s["target"])
    out = dict(n_accept=r["n_accept"], path=r["path"], next=r["next"], ctx_len=r["ctx_len"], kv=s["kv"])
    if "keys" in s:
        out.update(keys=s["keys"], scale=s["scale"])
    return out


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    ctx, new = _lens(case)
    n, P = sum(new), case["page"]
    if case["op"] == "plan":
        pages = sum(max(0, (c + k + P - 1) // P - (c + P - 1) // P) for c, k in zip(ctx, new))
        # lengths, counts and pages held read; the slot, position and request of each token, a page twice, totals
        return dict(bytes=4 * (3 * case["batch"] + 3 * n + 2 * pages + 3 * case["batch"] + 2), flops=0)
    if case["op"] == "commit":
        row = 2 * D + (132 if case["index"] else 0)
        moves = case["batch"] * case["depth"] / 2 * (case["branches"] - 1) / case["branches"]  # on average
        return dict(bytes=2 * row * moves * case["layers"] + 12 * n + 4 * case["batch"] * 68, flops=0)
    io = n * H * (D * 2 + LORA * 2 + 4)
    if case["op"] == "sel":
        k = case["topk"]
        keys = [min(k, c + (j + 1)) for c, m in zip(ctx, new) for j in range(m)]
        # nodes of a request share keys: no more rows than the request has, no fewer than one list needs
        rows = sum(min(c + m, m * k) for c, m in zip(ctx, new))
        return dict(bytes=rows * D * 2 + io + 4 * sum(keys), flops=sum(keys) * H * 2 * (D + LORA))
    keys = sum((c + m) for c, m in zip(ctx, new))
    return dict(bytes=keys * D * 2 + io, flops=sum(m * c + m * (m + 1) // 4 for c, m in zip(ctx, new)) * H * 2 * (D + LORA))


# ---- 64 bits, from the definitions ---------------------------------------------------------------

def exact(case, seed):
    if case["op"] not in ("tree", "sel"):
        return None  # whole numbers and rows moved bit for bit
    s = prepare(case, seed)
    ctx, new = _lens(case)
    P, parent = case["page"], s["parent"].tolist()
    out, lses, r = [], [], 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        pos = torch.arange(c + n, device="cuda")
        rows = s["kv"][s["table"][b].long()[torch.div(pos, P, rounding_mode="floor")] * P + pos.remainder(P)].double()
        line = []
        for j in range(n):
            line.append({j} | (line[parent[r + j]] if parent[r + j] >= 0 else set()))
        for j in range(n):
            if case["op"] == "tree":
                use = torch.cat([pos[:c], torch.tensor(sorted(c + a for a in line[j]), device="cuda")])
            else:
                lst = s["sel"][r + j, : int(s["sel_n"][r + j])].tolist()
                use = torch.tensor([x for x in lst if 0 <= x < c or x - c in line[j]], device="cuda", dtype=torch.long)
            k = rows[use]
            z = k @ s["q"][r + j].double().t() / 16.0  # [keys, heads]
            lses.append(torch.logsumexp(z, 0))
            out.append(torch.softmax(z, 0).t() @ k[:, :LORA])
        r += n
    return dict(ctx=torch.stack(out), lse=torch.stack(lses))
