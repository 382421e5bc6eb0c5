"""The paged KV cache and the attentions that read it, as a serving program calls them.

K and V live in pools [layer][page][kv head][offset in page][head dim]; page_table row s names the pages of sequence
s in order, -1 where there is none.  Three operators and the calls that keep their cache:

  tree     drafted tokens (a tree, or a chain) of several sequences attend to their cached contexts and, among
           themselves, to what a bit mask lets them see;
  sparse   one token per sequence attends to those pages of its context that a score picks, the bounds of the page
           that it was written to being brought up to date first;
  fork     sequences are forked (pages shared) and the forks grown, which copies a shared last page in all layers;
  write    new K / V rows go to their places in the pages of one layer;
  compact  the accepted rows of a draft move up behind their context, in all layers.

Where `own` is false, run() computes them by elementary torch operations; where it is true, it makes the calls of
lokal_amd.kernels.  Heads are those of lokal_amd/config.py (9/3, 14/2, 32/4 of 64) and of wider models.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

own = False

LAYERS = 4     # layers of the attention cases' pools: a call reads one of them
NO_PAGE = -1   # 0xFFFFFFFF


def listed():
    return [
        # One token of one short conversation over small pages: latency is all of it.
        {"name": "tree-1x1-ctx300", "op": "tree", "n": 1, "draft": 1, "tree": True, "heads": 9, "kv_heads": 3,
         "dim": 64, "page": 16, "ctx": 300, "f32": False},
        # A few conversations, each with a tree of 16 drafted tokens.
        {"name": "tree-4x16-ctx4096", "op": "tree", "n": 4, "draft": 16, "tree": True, "heads": 14, "kv_heads": 2,
         "dim": 64, "page": 64, "ctx": 4096, "f32": False},
        # Chains of drafted tokens over an f32 cache, odd in everything.
        {"name": "chain-3x23-ctx5000-f32", "op": "tree", "n": 3, "draft": 23, "tree": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "ctx": 5000, "f32": True},
        # A serving batch verifying small trees.
        {"name": "tree-24x12-ctx2048", "op": "tree", "n": 24, "draft": 12, "tree": True, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "ctx": 2048, "f32": False},
        # Long documents and large trees: the most work there is.
        {"name": "tree-8x64-ctx32768", "op": "tree", "n": 8, "draft": 64, "tree": True, "heads": 32, "kv_heads": 4,
         "dim": 64, "page": 64, "ctx": 32768, "f32": False},
        # One conversation of middle length, 16 small pages of it.
        {"name": "sparse-1-ctx2000", "op": "sparse", "n": 1, "heads": 9, "kv_heads": 3, "dim": 64, "page": 16,
         "ctx": 2000, "take": 16, "f32": False},
        # A few long conversations, an eighth of their pages.
        {"name": "sparse-4-ctx32768", "op": "sparse", "n": 4, "heads": 14, "kv_heads": 2, "dim": 64, "page": 64,
         "ctx": 32768, "take": 64, "f32": False},
        # A serving batch of long contexts over small pages.
        {"name": "sparse-32-ctx16384", "op": "sparse", "n": 32, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "ctx": 16384, "take": 48, "f32": False},
        # Two more answers to one short prompt.
        {"name": "fork-2-ctx40", "op": "fork", "n": 2, "grow": 1, "layers": 24, "kv_heads": 2, "dim": 64, "page": 16,
         "ctx": 40, "f32": False},
        # A batch forked at once, with pages to copy in 22 layers.
        {"name": "fork-48-ctx600", "op": "fork", "n": 48, "grow": 70, "layers": 22, "kv_heads": 4, "dim": 64,
         "page": 64, "ctx": 600, "f32": False},
        # The K / V rows of prompts of up to 512 tokens.
        {"name": "write-8x512", "op": "write", "n": 8, "rows": 512, "kv_heads": 8, "dim": 128, "page": 32,
         "ctx": 1000, "f32": False},
        # The accepted tokens of a batch's trees, in all layers.
        {"name": "compact-64x16", "op": "compact", "n": 64, "draft": 16, "layers": 24, "kv_heads": 2, "dim": 64,
         "page": 16, "ctx": 500, "f32": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "sparse", "sparse", "fork", "write", "compact"])
    heads, kv = rng.choice([(9, 3), (14, 2), (32, 4), (32, 8), (8, 8), (16, 1)])
    dim, page, f32 = rng.choice([64, 64, 128]), rng.choice([16, 32, 64, 128, 256]), rng.random() < 0.25
    size = kv * dim * (2 if f32 else 1)  # of a position, in 4 bytes (K and V)
    if op == "tree":
        draft = _log(rng, 1, 64)
        ctx = _log(rng, 16, 32768)
        n = max(1, min(_log(rng, 1, 32), 8 * 32768 * 256 // (size * ctx), 8 * 64 * 32 * 64 * 32768 // (draft * heads * dim * ctx)))
        return {"op": op, "n": n, "draft": draft, "tree": rng.random() < 0.7, "heads": heads, "kv_heads": kv,
                "dim": dim, "page": page, "ctx": ctx, "f32": f32}
    if op == "sparse":
        ctx = _log(rng, 64, 32768)
        n = max(1, min(_log(rng, 1, 64), 32 * 16384 * 1024 // (size * ctx)))
        return {"op": op, "n": n, "heads": heads, "kv_heads": kv, "dim": dim, "page": page, "ctx": ctx,
                "take": max(4, min(_log(rng, 4, 128), 8192 // page)), "f32": f32}
    layers = rng.randint(1, 24)
    if op == "write":
        rows = _log(rng, 1, 512)
        return {"op": op, "n": max(1, min(_log(rng, 1, 64), 4096 // rows)), "rows": rows, "kv_heads": kv, "dim": dim,
                "page": page, "ctx": _log(rng, 1, 1000), "f32": f32}
    ctx = _log(rng, 8, 600)
    most = 48 * 700 * 22 * 256 // (size * layers * (ctx + 2 * page))
    n = max(1, min(_log(rng, 1, 64), most))
    if op == "fork":
        return {"op": op, "n": n, "grow": _log(rng, 1, 100), "layers": layers, "kv_heads": kv, "dim": dim,
                "page": page, "ctx": ctx, "f32": f32}
    return {"op": op, "n": n, "draft": rng.randint(2, 64), "layers": layers, "kv_heads": kv, "dim": dim,
            "page": page, "ctx": ctx, "f32": f32}


# ------------------------------------------------------------------ inputs

class _Dev:
    """A torch tensor as the device buffer that the kernel-level calls take."""

    def __init__(self, t):
        self.t = t
        self.ptr = ctypes.c_void_p(t.data_ptr())


class _State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def _pages_for(length, page):
    return (length + page - 1) // page


def _pool(g, layers, pages, case):
    """K and V of about unit scale."""
    shape = (layers, pages, case["kv_heads"], case["page"], case["dim"])
    t = torch.float32 if case["f32"] else torch.float16
    return [torch.randn(shape, generator=g, device="cuda", dtype=t) for _ in range(2)]


def _whole(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda")


def _table(g, length, width, pages):
    """[n][width] page ids in no order for sequences of `length` positions' pages, -1 behind them."""
    n = length.numel()
    ids = torch.randperm(pages, generator=g, device="cuda")[:n * width].view(n, width).int()
    return torch.where(torch.arange(width, device="cuda") < length[:, None], ids, NO_PAGE).int()


def _words(bits):
    """[..., T] truth values as [..., ceil(T / 32)] int32 words, bit j of the row in word j / 32."""
    t = bits.shape[-1]
    b = torch.nn.functional.pad(bits.long(), (0, -t % 32)).unflatten(-1, (-1, 32))
    v = (b << torch.arange(32, device="cuda")).sum(-1)
    return torch.where(v >= 1 << 31, v - (1 << 32), v).int()


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1013 + 5)
    op, n, page = case["op"], case["n"], case["page"]
    s = _State(case=case, op=op)
    hi = case["ctx"]
    s.ctx = _whole(g, max(1, hi // 4), hi + 1, n).int()
    s.ctx[0] = hi
    s.slots = torch.arange(n, device="cuda").int()
    if op == "tree":
        t = case["draft"]
        s.nd = _whole(g, 1, t + 1, n).int()
        s.nd[0] = t
        width = _pages_for(hi + t, page)
        s.k, s.v = _pool(g, LAYERS, n * width + 3, case)
        s.table = _table(g, _pages_for(s.ctx + s.nd, page), width, n * width + 3)
        s.q = torch.randn(n, t, case["heads"] * case["dim"], generator=g, device="cuda") * 2
        s.mask = None
        if case["tree"]:  # token j hangs on an earlier one and sees its ancestors and itself
            sees = torch.eye(t, device="cuda", dtype=torch.bool).repeat(n, 1, 1)
            for j in range(1, t):
                sees[:, j] |= sees[s.slots.long(), _whole(g, 0, j, n)]
            s.mask = _words(sees)
        s.out = torch.zeros_like(s.q)
        s.layer = 1
    elif op == "sparse":
        width = _pages_for(hi, page)
        pages = n * width + 3
        s.k, s.v = _pool(g, 1, pages, case)
        # what a page holds belongs together: its keys have a part in common
        s.k += torch.randn(1, pages, case["kv_heads"], 1, case["dim"], generator=g, device="cuda").to(s.k.dtype) / 2
        s.table = _table(g, _pages_for(s.ctx, page), width, pages)
        s.q = torch.randn(n, case["heads"] * case["dim"], generator=g, device="cuda") * 2
        s.bounds = torch.stack([s.k[0].amin(2), s.k[0].amax(2)], 2)  # [page][kv head][min, max][dim]
        s.out = torch.zeros_like(s.q)
        s.taken = torch.zeros(n, case["kv_heads"], case["take"], device="cuda", dtype=torch.int32)
        s.before = s.ctx - 1
        s.layer = 0
    elif op == "fork":
        # sequences 0..n-1 hold contexts, n..2n-1 are free
        width = _pages_for(hi + case["grow"], page)
        pages = 2 * n * width + 2
        s.k, s.v = _pool(g, case["layers"], pages, case)
        s.table = torch.cat([_table(g, _pages_for(s.ctx, page), width, pages),
                             torch.full((n, width), NO_PAGE, device="cuda", dtype=torch.int32)])
        s.length = torch.cat([s.ctx, torch.zeros_like(s.ctx)])
        s.refs = torch.zeros(pages + 1, device="cuda", dtype=torch.int32)
        s.refs.scatter_(0, torch.where(s.table < 0, pages, s.table).long().flatten(), 1)
        s.refs = s.refs[:pages].contiguous()
        s.forks = s.slots + n
        s.none = torch.zeros_like(s.slots)
        s.add = torch.full_like(s.slots, case["grow"])
        s.ok = torch.zeros(2, n, device="cuda", dtype=torch.int32)
        s.copied = torch.zeros(n, 2, device="cuda", dtype=torch.int32)
    else:
        m = case["rows"] if op == "write" else case["draft"]
        width = _pages_for(hi + m, page)
        s.k, s.v = _pool(g, LAYERS if op == "write" else case["layers"], n * width + 3, case)
        s.table = _table(g, _pages_for(s.ctx + m, page), width, n * width + 3)
        if op == "write":
            s.layer = 2
            s.row_slot = s.slots.repeat_interleave(m)
            s.row_pos = (s.ctx[:, None] + torch.arange(m, device="cuda").int()).flatten().contiguous()
            s.rows = [torch.randn(n * m, case["kv_heads"] * case["dim"], generator=g, device="cuda") for _ in range(2)]
        else:
            s.n_path = _whole(g, 1, m // 2 + 1, n).int()
            # increasing draft places, the first of them the root
            order = torch.rand(n, m, generator=g, device="cuda")
            order[:, 0] = -1
            path = order.argsort(1)[:, :m // 2 + 1]
            path = torch.where(torch.arange(path.shape[1], device="cuda") < s.n_path[:, None], path, m)
            s.path = path.sort(1)[0].int().contiguous()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the descriptors and the workspace that a program keeps with its cache
        _keep(s)
    torch.cuda.synchronize()
    return s


def _keep(s):
    from lokal_amd import kernels
    c, d = s.case, {}
    for name, t in s.__dict__.items():
        if isinstance(t, torch.Tensor):
            d[name] = _Dev(t)
    s.d = d
    layers, pages = s.k.shape[:2]
    s.pages = kernels.KvPages(d["k"], d["v"], kernels.F32 if c["f32"] else kernels.F16, layers, pages, c["kv_heads"],
                              c["page"], c["dim"])
    s.seqs = kernels.PageTable(d["table"], d.get("length"), d.get("refs"), *s.table.shape)
    if s.op == "tree":
        size = kernels.tree_attn_workspace(s.pages, s.seqs, c["n"], c["draft"], c["heads"])
    elif s.op == "sparse":
        size = kernels.sparse_attn_workspace(s.pages, s.seqs, c["n"], c["heads"], c["take"])
    else:
        size = 0
    if s.op == "fork":
        s.d["ok0"], s.d["ok1"] = _Dev(s.ok[0]), _Dev(s.ok[1])
    if s.op == "write":
        s.d["k_rows"], s.d["v_rows"] = (_Dev(t) for t in s.rows)
    s.ws = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")
    s.d["ws"] = _Dev(s.ws)
    s.kernels = kernels


# ---------------------------------------------------------------------- run

def run(s):
    if own:
        return _run_own(s)
    return {"tree": _plain_tree, "sparse": _plain_sparse, "fork": _plain_fork, "write": _plain_write,
            "compact": _plain_compact}[s.op](s)


def _run_own(s):
    kernels, c, d, n = s.kernels, s.case, s.d, s.case["n"]
    if s.op == "tree":
        kernels.tree_attn(s.pages, s.seqs, s.layer, d["q"], d["ctx"], d["nd"], d.get("mask"), n, c["draft"],
                          c["heads"], d["ws"], s.ws.numel(), d["out"])
        return [s.out]
    if s.op == "sparse":
        kernels.page_bounds(s.pages, s.seqs, s.layer, d["before"], d["ctx"], n, d["bounds"])
        kernels.sparse_attn(s.pages, s.seqs, s.layer, d["q"], d["ctx"], d["bounds"], n, c["heads"], c["take"], 1, 1,
                            d["taken"], d["ws"], s.ws.numel(), d["out"])
        return [s.out, s.taken, s.bounds]
    if s.op == "fork":
        kernels.pages_trim(s.pages, s.seqs, d["forks"], d["none"], n)
        kernels.pages_fork(s.pages, s.seqs, d["slots"], d["forks"], n, d["ok0"])
        kernels.pages_grow(s.pages, s.seqs, d["forks"], d["add"], n, d["ok1"], d["copied"])
        return [s.k, s.v, s.table, s.length, s.refs, s.ok, s.copied]
    if s.op == "write":
        kernels.pages_write(s.pages, s.seqs, s.layer, d["k_rows"], d["v_rows"], d["row_slot"], d["row_pos"],
                            n * c["rows"])
    else:
        kernels.pages_compact(s.pages, s.seqs, d["slots"], d["ctx"], d["path"], d["n_path"], n, s.path.shape[1])
    return [s.k, s.v]


def _attend(q, k, v, sees):
    """softmax(q k^T / sqrt(dim)) v over what `sees` lets through, in 32 bits; zeros where that is nothing."""
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(q.shape[-1])
    x = x.masked_fill(~sees, -torch.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -torch.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, 1, total)


def _rows_of(pool, ids):
    """[n][m] pages of [page][kv head][offset][dim] as [n][kv head][m * page][dim] in 32 bits."""
    x = pool[ids.clamp(min=0).long()].float()
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3).contiguous()


def _plain_tree(s):
    c, n, t = s.case, s.case["n"], s.case["draft"]
    kv, dim = c["kv_heads"], c["dim"]
    k, v = (_rows_of(pool[s.layer], s.table) for pool in (s.k, s.v))
    pos = torch.arange(k.shape[2], device="cuda")
    j = pos - s.ctx[:, None, None]  # place in the draft
    if s.mask is None:
        sees = j <= torch.arange(t, device="cuda")[:, None]
    else:
        at = j.clamp(0, t - 1).expand(n, t, -1).long()
        sees = (s.mask.gather(2, at >> 5) >> (at & 31)) & 1 != 0
    sees = (j < 0) | (sees & (j < s.nd[:, None, None]))
    q = s.q.view(n, t, kv, -1, dim).permute(0, 2, 1, 3, 4)  # [n][kv head][token][head of the group][dim]
    group = q.shape[3]
    sees = sees[:, None, :, None].expand(n, 1, t, group, -1).flatten(2, 3)
    o = _attend(q.flatten(2, 3).contiguous(), k, v, sees).view(n, kv, t, group, dim).permute(0, 2, 1, 3, 4)
    live = torch.arange(t, device="cuda") < s.nd[:, None]
    return [torch.where(live[..., None], o.reshape(n, t, -1), s.out)]


def _plain_sparse(s):
    c, n, page = s.case, s.case["n"], s.case["page"]
    kv, dim, take = c["kv_heads"], c["dim"], c["take"]
    # the bounds of the page that the newest position lies in
    at = s.table.gather(1, (s.before // page).long()[:, None])[:, 0].long()
    live = (torch.arange(page, device="cuda") < (s.before % page + 1)[:, None])[:, None, :, None]
    rows = s.k[s.layer][at]
    s.bounds[at] = torch.stack([rows.masked_fill(~live, torch.inf).amin(2), rows.masked_fill(~live, -torch.inf).amax(2)], 2)
    # an upper bound of every score of a page, and with it the pages: in 64 bits, as two may be close
    q = s.q.view(n, kv, -1, dim)
    b = s.bounds[s.table.clamp(min=0).long()].double()  # [n][page][kv head][2][dim]
    lo, hi = (b[:, :, :, i].permute(0, 2, 3, 1).contiguous() for i in (0, 1))
    score = (torch.matmul(q.double().clamp(min=0), hi) + torch.matmul(q.double().clamp(max=0), lo)).amax(2)
    number = torch.arange(s.table.shape[1], device="cuda")
    held = _pages_for(s.ctx, page)[:, None, None]
    score = score.masked_fill((number < 1) | (number >= held - 1), torch.inf).masked_fill(number >= held, -torch.inf)
    order = torch.argsort(score, dim=-1, descending=True, stable=True)[..., :take]
    order = torch.where(order < held, order, 1 << 30).sort(-1)[0]
    width = min(take, order.shape[-1])
    taken = torch.full_like(s.taken, NO_PAGE)
    taken[..., :width] = torch.where(order < held, order, NO_PAGE).int()
    # attention over these
    ids = s.table[:, None].expand(n, kv, -1).gather(2, taken.clamp(min=0).long()).long()
    head = torch.arange(kv, device="cuda")[:, None]
    k, v = (pool[s.layer][ids, head].float().flatten(2, 3) for pool in (s.k, s.v))
    pos = (taken[..., None] * page + torch.arange(page, device="cuda")).flatten(2)
    sees = (pos < s.ctx[:, None, None]) & (taken >= 0).repeat_interleave(page, 2)
    return [_attend(q, k, v, sees[:, :, None]).reshape(n, -1), taken, s.bounds]


def _add_refs(s, ids, by):
    s.refs.scatter_add_(0, ids.clamp(min=0).flatten().long(), torch.where(ids >= 0, by, 0).int().flatten())


def _plain_fork(s):
    c, n, page = s.case, s.case["n"], s.case["page"]
    number = torch.arange(s.table.shape[1], device="cuda")
    forks = s.forks.long()
    # free what the forks hold
    _add_refs(s, s.table[forks], -1)
    s.table[forks] = NO_PAGE
    # share their sources' pages
    mine = s.table[s.slots.long()]
    _add_refs(s, mine, 1)
    s.table[forks] = mine
    length = s.length[s.slots.long()]
    s.ok[0] = 1
    # grow: a shared last page that is not full is replaced by a copy, new pages follow; lowest free pages first
    held, want = _pages_for(length, page), _pages_for(length + s.add, page)
    last = mine.gather(1, (length // page).clamp(max=mine.shape[1] - 1).long()[:, None])[:, 0]
    copies = (length % page != 0) & (s.refs[last.clamp(min=0).long()] > 1)
    first = held - copies.int()
    need = (want - first).cumsum(0)
    s.ok[1] = need <= (s.refs == 0).sum()
    grows = s.ok[1] != 0
    free = torch.argsort((s.refs != 0).int(), stable=True).int()
    at = (need - (want - first))[:, None] + number - first[:, None]
    new = (number >= first[:, None]) & (number < want[:, None]) & grows[:, None]
    row = torch.where(new, free[at.clamp(0, free.numel() - 1).long()], mine)
    copies &= grows
    s.table[forks] = row
    s.refs.scatter_(0, torch.where(new, row, free[-1]).flatten().long(),
                    torch.where(new, 1, s.refs[free[-1].long()]).int().flatten())
    _add_refs(s, torch.where(copies, last, NO_PAGE), -1)
    s.length[forks] = torch.where(grows, length + s.add, length)
    to = row.gather(1, (length // page).clamp(max=mine.shape[1] - 1).long()[:, None])[:, 0]
    s.copied[:, 0], s.copied[:, 1] = torch.where(copies, last, NO_PAGE), torch.where(copies, to, NO_PAGE)
    src, dst = last[copies].long(), to[copies].long()
    old = (torch.arange(page, device="cuda") < (length % page)[copies][:, None])[:, None, :, None]
    for pool in (s.k, s.v):
        pool[:, dst] = torch.where(old, pool[:, src], pool[:, dst])
    return [s.k, s.v, s.table, s.length, s.refs, s.ok, s.copied]


def _plain_write(s):
    c, page = s.case, s.case["page"]
    ids = s.table[s.row_slot.long(), (s.row_pos // page).long()].long()
    for pool, rows in zip((s.k, s.v), s.rows):
        pool[s.layer][ids, :, (s.row_pos % page).long()] = rows.view(-1, c["kv_heads"], c["dim"]).to(pool.dtype)
    return [s.k, s.v]


def _plain_compact(s):
    page, m = s.case["page"], s.path.shape[1]
    i = torch.arange(m, device="cuda")
    live = i < s.n_path[:, None]
    to = s.ctx[:, None] + i
    at = torch.where(live, s.ctx[:, None] + s.path, to)
    page_of = lambda x: s.table.gather(1, (x // page).long())[live].long()  # noqa: E731
    src, dst, a, b = page_of(at), page_of(to), (at % page)[live].long(), (to % page)[live].long()
    for pool in (s.k, s.v):
        pool[:, dst, :, b] = pool[:, src, :, a].clone()
    return [s.k, s.v]


# ------------------------------------------------------ what a pass has to do

def work(case):
    n, kv, dim = case["n"], case["kv_heads"], case["dim"]
    row = kv * dim * 2 * (4 if case["f32"] else 2)  # K and V of a position
    ctx = case["ctx"] * 5 / 8  # of a drawn sequence, in the mean
    if case["op"] == "tree":
        draft, heads = (case["draft"] + 1) / 2, case["heads"]
        return {"bytes": n * ((ctx + draft) * row + draft * heads * dim * 8),
                "flops": 4 * n * draft * heads * dim * (ctx + draft / 2)}
    if case["op"] == "sparse":
        pages = ctx / case["page"]
        taken = min(case["take"], pages) * case["page"]
        return {"bytes": n * (pages * row + taken * row + case["heads"] * dim * 8),
                "flops": 4 * n * case["heads"] * dim * (pages + taken)}
    if case["op"] == "fork":
        return {"bytes": n * (case["page"] / 2 * row * 2 * case["layers"] + 16 * ctx / case["page"]), "flops": 0}
    if case["op"] == "write":
        return {"bytes": n * case["rows"] * (row + kv * dim * 8), "flops": 0}
    return {"bytes": n * (case["draft"] // 2 + 1) / 2 * row * 2 * case["layers"], "flops": 0}


# ----------------------------------------------------------- in 64 bits, plainly

def _one64(q, k, v, sees):
    """One sequence and kv head: rows q over keys k, values v, all in 64 bits."""
    x = (q @ k.T) * dim_scale(q)
    w = torch.where(sees, torch.exp(x - x.masked_fill(~sees, -1e300).max(1, keepdim=True)[0]), 0.0)
    t = w.sum(1, keepdim=True)
    return torch.where(t > 0, (w @ v) / t, 0.0)


def dim_scale(q):
    return q.shape[1] ** -0.5


def _cached64(pool, layer, ids, kv, length):
    """The first `length` rows of a sequence with pages `ids`, kv head by kv head."""
    return pool[layer, ids.long()].transpose(0, 1).reshape(kv, -1, pool.shape[-1])[:, :length].double()


def _exact_tree(s):
    c = s.case
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    group, dim = c["heads"] // c["kv_heads"], c["dim"]
    for i, (ctx, nd) in enumerate(zip(s.ctx.tolist(), s.nd.tolist())):
        ids = s.table[i][:_pages_for(ctx + nd, c["page"])]
        k, v = (_cached64(p, s.layer, ids, c["kv_heads"], ctx + nd) for p in (s.k, s.v))
        sees = torch.ones(nd, ctx + nd, dtype=torch.bool, device="cuda")
        if s.mask is None:
            sees[:, ctx:] = torch.ones(nd, nd, dtype=torch.bool, device="cuda").tril()
        else:
            words = s.mask[i, :nd].cpu().numpy().view(np.uint8)
            bits = np.unpackbits(words, axis=1, bitorder="little")[:, :nd]
            sees[:, ctx:] = torch.from_numpy(bits.astype(bool)).cuda()
        q = s.q[i, :nd].double().view(nd, c["kv_heads"], group, dim)
        for h in range(c["kv_heads"]):
            o = _one64(q[:, h].reshape(-1, dim), k[h], v[h], sees.repeat_interleave(group, 0))
            out[i, :nd].view(nd, c["kv_heads"], group, dim)[:, h] = o.view(nd, group, dim)
    return [out]


def _exact_sparse(s):
    c, page = s.case, s.case["page"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    bounds = s.bounds.double()
    group, dim, take = c["heads"] // c["kv_heads"], c["dim"], c["take"]
    for i, ctx in enumerate(s.ctx.tolist()):
        m = _pages_for(ctx, page)
        ids = s.table[i][:m].long()
        k, v = (_cached64(p, s.layer, ids, c["kv_heads"], ctx) for p in (s.k, s.v))
        newest = k[:, (m - 1) * page:]
        bounds[ids[-1]] = torch.stack([newest.min(1)[0], newest.max(1)[0]], 1)
        for h in range(c["kv_heads"]):
            q = s.q[i].double().view(c["kv_heads"], group, dim)[h]
            b = bounds[ids, h]
            best = torch.maximum(q[:, None] * b[:, 0], q[:, None] * b[:, 1]).sum(2).max(0)[0].tolist()
            keep = {0, m - 1}
            rest = sorted((p for p in range(m) if p not in keep), key=lambda p: (-best[p], p))
            keep = sorted(sorted(keep) + rest[:max(0, take - len(keep))])[:m]
            sees = torch.zeros(m, dtype=torch.bool, device="cuda")
            sees[keep] = True
            sees = sees.repeat_interleave(page)[:ctx]
            out[i].view(c["kv_heads"], group, dim)[h] = _one64(q, k[h][sees], v[h][sees], torch.ones(1, 1, dtype=torch.bool, device="cuda"))
    return [out, None, bounds]


def _exact_fork(s):
    c, page, n = s.case, s.case["page"], s.case["n"]
    k, v = s.k.double(), s.v.double()
    refs, table = s.refs.tolist(), s.table.tolist()
    for i in range(n):
        table[n + i] = list(table[i])
        for p in table[i]:
            if p >= 0:
                refs[p] += 1
    free = [p for p, r in enumerate(refs) if r == 0]
    for i, ctx in enumerate(s.ctx.tolist()):
        copies = ctx % page != 0 and refs[table[i][ctx // page]] > 1
        need = _pages_for(ctx + c["grow"], page) - _pages_for(ctx, page) + copies
        if need > len(free):
            break
        if copies:
            a, b = table[i][ctx // page], free[0]
            k[:, b, :, :ctx % page], v[:, b, :, :ctx % page] = k[:, a, :, :ctx % page], v[:, a, :, :ctx % page]
        free = free[need:]
    return [k, v, None, None, None, None, None]


def _exact_write(s):
    c, page = s.case, s.case["page"]
    out = []
    for pool, rows in zip((s.k, s.v), s.rows):
        o = pool.double()
        r = rows.to(pool.dtype).double().view(c["n"], c["rows"], c["kv_heads"], c["dim"])
        for i, ctx in enumerate(s.ctx.tolist()):
            for p in range(ctx // page, (ctx + c["rows"] - 1) // page + 1):
                a, b = max(ctx, p * page), min(ctx + c["rows"], (p + 1) * page)
                o[s.layer, s.table[i, p], :, a - p * page:b - p * page] = r[i, a - ctx:b - ctx].transpose(0, 1)
        out.append(o)
    return out


def _exact_compact(s):
    page = s.case["page"]
    out = []
    table, ctxs, paths, counts = s.table.tolist(), s.ctx.tolist(), s.path.tolist(), s.n_path.tolist()
    for pool in (s.k, s.v):
        o = pool.double()
        for i, ctx in enumerate(ctxs):
            for j in range(counts[i]):  # a row moves up: none is needed after it is written over
                a, b = ctx + paths[i][j], ctx + j
                o[:, table[i][b // page], :, b % page] = o[:, table[i][a // page], :, a % page]
        out.append(o)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return {"tree": _exact_tree, "sparse": _exact_sparse, "fork": _exact_fork, "write": _exact_write,
            "compact": _exact_compact}[s.op](s)
