"""The paged KV cache and its attentions against numpy in 64 bits.  What no row may see is NaN in every cache here.
Tolerances: ref_paged.attn_tol for attention (relative to the largest value); page contents, bounds, choices, tables
and counts are exact."""
import ctypes as C

import numpy as np
import pytest

from lokal_amd import kernels as K

from . import ref_paged as R

pytestmark = pytest.mark.gpu
NO = K.NO_PAGE
u32 = np.uint32


def dev(a, t=None):
    return K.DeviceArray.from_numpy(np.asarray(a, t))


def close(got, want, tol, v):
    top = np.abs(v[np.isfinite(v)].astype(np.float64)).max()
    off = np.abs(got.astype(np.float64) - want).max()
    assert np.isfinite(got).all() and off <= tol * top, (off / top, tol)


def run_tree(c, layer, q, ctx, nd, mask, heads, slots=None, fill=7.5):
    n, T = q.shape[:2]
    out = dev(np.full(q.shape, fill, np.float32))
    size = K.tree_attn_workspace(c.pages, c.seqs, n, T, heads)
    ws = dev(np.full(max(size, 4), 255, np.uint8)) if size else None
    K.tree_attn(c.pages, c.seqs, layer, dev(q), dev(ctx, u32), None if nd is None else dev(nd, u32),
                None if mask is None else dev(mask), n, T, heads, ws, size, out,
                slots=None if slots is None else dev(slots, u32))
    return out.numpy()


TREE = [
    # kv type, hd, page, heads, kv heads, tokens, contexts, tree
    ("f16", 64, 16, 3, 3, 1, [0, 1, 15, 16, 17, 63, 64, 65], False),
    ("f16", 64, 64, 14, 2, 5, [300, 0, 127], True),
    ("f16", 64, 32, 9, 3, 16, [1000, 31], True),
    ("f16", 64, 256, 32, 4, 23, [700, 255, 256, 1], False),
    ("f16", 64, 16, 16, 1, 37, [400], True),
    ("f16", 64, 64, 8, 1, 70, [100, 2], True),
    ("f16", 128, 16, 32, 8, 12, [500, 33], True),
    ("f16", 128, 128, 4, 4, 3, [129], True),
    ("f16", 128, 64, 20, 2, 33, [200], False),
    ("f32", 64, 16, 6, 2, 4, [77, 0], True),
    ("f32", 128, 32, 32, 8, 23, [333], False),
    ("f32", 128, 64, 3, 3, 1, [1000], True),
    ("f32", 64, 128, 7, 1, 40, [90], True),
]


@pytest.mark.parametrize("case", TREE, ids=lambda c: "-".join(map(str, c[:6])))
def test_tree_attn(case):
    t, hd, page, heads, kv, T, ctxs, tree = case
    rng = np.random.default_rng(T * 7 + hd + page)
    n = len(ctxs)
    nd = [T] + [int(x) for x in rng.integers(1, T + 1, n - 1)]
    if n > 2:
        nd[1] = 0
    c = R.Cache(rng, [x + d for x, d in zip(ctxs, nd)], kv=kv, hd=hd, page=page, f32=t == "f32", layers=2).up()
    q = rng.standard_normal((n, T, heads * hd)).astype(np.float32) * 2
    mask = R.words(np.stack([R.ancestors(rng, T) for _ in range(n)])) if tree else None
    got = run_tree(c, 1, q, ctxs, nd, mask, heads)
    want = R.tree_rows(c, 1, q, ctxs, nd, mask, heads, np.full(q.shape, 7.5))
    for i in range(n):
        assert (got[i, nd[i]:] == 7.5).all()  # rows behind the draft are left
    close(got, want, R.attn_tol(hd, max(c.len), q, c.k), c.v)


@pytest.mark.parametrize("t", ["f16", "f32"])
def test_long_context_in_many_chunks(t):
    rng = np.random.default_rng(3)
    c = R.Cache(rng, [9000, 130], kv=1, hd=64, page=64, f32=t == "f32").up()
    q = rng.standard_normal((2, 2, 7 * 64)).astype(np.float32) * 2
    ctx = [8998, 128]
    got = run_tree(c, 0, q, ctx, [2, 2], None, 7)
    close(got, R.tree_rows(c, 0, q, ctx, [2, 2], None, 7, np.zeros(q.shape)), R.attn_tol(64, 9000, q, c.k), c.v)


@pytest.mark.parametrize("t,heads", [("f16", 4), ("f16", 32), ("f32", 4), ("f32", 32)])
@pytest.mark.parametrize("scale", [1e-30, 1e-6, 300.0, 1e20])
def test_queries_of_any_size(scale, t, heads):
    """Tiny queries see everything alike, huge ones one position; neither leaves what two f16 parts hold."""
    rng = np.random.default_rng(5)
    c = R.Cache(rng, [100], kv=2, hd=64, f32=t == "f32").up()
    q = (rng.standard_normal((1, 3, heads * 64)) * scale).astype(np.float32)
    got = run_tree(c, 0, q, [97], [3], None, heads)
    want = R.tree_rows(c, 0, q, [97], [3], None, heads, np.zeros(q.shape))
    if scale <= 300:
        close(got, want, R.attn_tol(64, 100, q, c.k), c.v)
    else:  # scores of 1e20: the best position alone; no other comes within an f32 step of it here
        close(got, want, 2.0 ** -20, c.v)


@pytest.mark.parametrize("heads", [6, 16, 32])
@pytest.mark.parametrize("t,hd", [("f16", 64), ("f16", 128), ("f32", 64), ("f32", 128)])
def test_what_a_row_does_not_see_does_not_reach_it(t, hd, heads):
    """Draft tokens with NaN and infinite K / V, seen by some rows alone; masks that leave rows empty."""
    rng = np.random.default_rng(6)
    T, kv = 9, 2
    for ctx in (0, 5, 60, 130):
        c = R.Cache(rng, [ctx + T], kv=kv, hd=hd, f32=t == "f32")
        bad = {2: np.nan, 4: np.inf, 7: -np.inf}
        for j, x in bad.items():
            at = (0, c.table[0, (ctx + j) // c.page], slice(None), (ctx + j) % c.page)
            c.v[at][:, ::3] = x
            c.k[at][:, 1] = x
        c.up()
        sees = np.eye(T, dtype=bool)
        sees[5, [0, 1, 3]] = True
        sees[6, 2] = sees[8, 7] = True
        sees[0] = False  # nothing of the draft
        q = rng.standard_normal((1, T, heads * hd)).astype(np.float32)
        got = run_tree(c, 0, q, [ctx], [T], R.words(sees[None]), heads)
        want = R.tree_rows(c, 0, q, [ctx], [T], R.words(sees[None]), heads, np.zeros(q.shape))
        clean = [i for i in range(T) if i not in (2, 4, 6, 7, 8)]
        close(got[:, clean], want[:, clean], R.attn_tol(hd, ctx + T, q, c.k), c.v)
        for i in (2, 6):  # a NaN key: all of the row
            assert not np.isfinite(got[0, i]).any()
        for i in (4, 7, 8):  # a value that is not finite: at least its dims
            assert not np.isfinite(got[0, i].reshape(heads, hd)[:, ::3]).any()
        if ctx == 0:
            assert (got[0, 0] == 0).all()


@pytest.mark.parametrize("heads", [2, 10, 25])
@pytest.mark.parametrize("t,hd", [("f16", 64), ("f16", 128), ("f32", 64), ("f32", 128)])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(t, hd, heads):
    rng = np.random.default_rng(16)
    T, kv, ctx = 5, 1, 20
    c = R.Cache(rng, [ctx + T], kv=kv, hd=hd, f32=t == "f32")
    c.v[0, c.table[0, (ctx + 1) // c.page], 0, (ctx + 1) % c.page, 5] = np.nan
    c.up()
    sees = np.tril(np.ones((T, T), bool))
    sees[3, 1] = False
    q = rng.standard_normal((1, T, heads * hd)).astype(np.float32)
    got = run_tree(c, 0, q, [ctx], [T], R.words(sees[None]), heads)[0].reshape(T, heads, hd)
    want = R.tree_rows(c, 0, q, [ctx], [T], R.words(sees[None]), heads, np.zeros(q.shape))[0].reshape(T, heads, hd)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.isnan(got[[1, 2, 4], :, 5]).all() and np.isnan(got).sum() == 3 * heads
    fine = ~np.isnan(want)
    close(got[fine], want[fine], R.attn_tol(hd, ctx + T, q, c.k), c.v)


def test_scores_that_are_not_finite():
    """A key of +inf that a row sees makes it NaN, all keys -inf-scored count as nothing seen."""
    rng = np.random.default_rng(7)
    c = R.Cache(rng, [40], kv=1, hd=64)
    c.k[0, c.table[0, 1], 0, 3] = np.inf
    c.up()
    q = np.abs(rng.standard_normal((1, 2, 64)).astype(np.float32))
    got = run_tree(c, 0, q, [38], [2], None, 1)
    assert not np.isfinite(got).any()
    q[0, 0, 0] = np.nan  # a query's own row, no other
    c = R.Cache(rng, [40], kv=1, hd=64).up()
    got = run_tree(c, 0, q, [38], [2], None, 1)
    assert np.isnan(got[0, 0]).all() and np.isfinite(got[0, 1]).all()


def test_tables_with_holes_slots_and_lengths_past_their_capacity():
    rng = np.random.default_rng(8)
    c = R.Cache(rng, [100, 64, 47], kv=2, hd=64)
    c.table[0, 2], c.table[1, 0] = NO, c.n_pages + 5
    c.up()
    heads, T = 4, 4
    q = rng.standard_normal((5, T, heads * 64)).astype(np.float32)
    slots = [2, 0, 3, 1, 0xFFFFFFFF]  # 3 and the last do not exist
    ctx = [43, 96, 10, 200, 5]       # 200: more than the table holds
    nd = [4, 9, 2, 2, 1]             # 9: more than the call's T
    got = run_tree(c, 0, q, ctx, nd, None, heads, slots)
    want = R.tree_rows(c, 0, q, ctx, nd, None, heads, np.full(q.shape, 7.5), slots)
    assert (got[2] == 7.5).all() and (got[4] == 7.5).all() and (got[3, 2:] == 7.5).all()
    keep = [0, 1]
    close(got[keep], want[keep], R.attn_tol(64, 100, q, c.k), c.v)
    # sequence 1's pages end before its table does: all behind them are holes
    assert np.isfinite(got[3, :2]).all()
    close(got[3, :2], want[3, :2], R.attn_tol(64, 112, q, c.k), c.v)
    # all of them holes: nothing to see
    c.table[:] = NO
    c.up()
    got = run_tree(c, 0, q[:3], [50, 0, 12], None, None, heads)
    assert (got == 0).all()


@pytest.mark.parametrize("kv_type", ["f16", "f32"])
def test_a_slot_cache_is_a_paged_one(kv_type):
    """[slot][kv head][max_seq][64] through strides; one token is what attn_decode computes."""
    rng = np.random.default_rng(9)
    n, kv, heads, most, page = 3, 2, 14, 256, 32
    t = np.float16 if kv_type == "f16" else np.float32
    k, v = (rng.standard_normal((n, kv, most, 64)).astype(t) for _ in range(2))
    q = rng.standard_normal((n, heads * 64)).astype(np.float32)
    ctx = np.array([200, 33, 256], u32)
    per = most // page
    pages = K.KvPages(dev(k), dev(v), K.F16 if kv_type == "f16" else K.F32, 1, (n - 1) * kv * per + per, kv, page, 64,
                      page_stride=page * 64, head_stride=most * 64)
    ids = (np.arange(n)[:, None] * kv * per + np.arange(per)).astype(u32)
    seqs = K.PageTable(dev(ids), None, None, n, per)
    size = K.tree_attn_workspace(pages, seqs, n, 1, heads)
    out, ref = K.DeviceArray((n, heads * 64)), K.DeviceArray((n, heads * 64))
    K.tree_attn(pages, seqs, 0, dev(q), dev(ctx - 1), None, None, n, 1, heads, K.DeviceArray(max(size, 4), np.uint8),
                size, out)
    got = out.numpy()
    for s in range(n):
        for h in range(heads):
            a = slice(h * 64, h * 64 + 64)
            kk, vv = (x[s, h // 7, :ctx[s]].astype(np.float64) for x in (k, v))
            want = R.softmax_rows(q[s:s + 1, a].astype(np.float64), kk, vv, np.ones((1, ctx[s]), bool))[0]
            close(got[s, a], want, R.attn_tol(64, 256, q, k), v)
    if kv_type == "f16":
        K.attn_decode(dev(q), dev(k.view(np.uint16)), dev(v.view(np.uint16)), dev(ctx), n, heads, kv, 64, most, ref)
        close(got, ref.numpy().astype(np.float64), 2 * R.attn_tol(64, 256, q, k), v)


@pytest.mark.parametrize("kv_type", ["f16", "f32"])
def test_pages_past_32_bit_offsets(kv_type):
    """Three pages 2^31 - 64 elements apart: the last is past 2^32 elements."""
    rng = np.random.default_rng(10)
    page, hd, kv, stride = 16, 64, 2, (1 << 31) - 64
    t = np.float16 if kv_type == "f16" else np.float32
    k, v = (K.DeviceArray(2 * stride + kv * page * hd, t) for _ in range(2))
    pages = K.KvPages(k, v, K.F16 if kv_type == "f16" else K.F32, 1, 3, kv, page, hd, page_stride=stride)
    seqs = K.PageTable(dev([[2, 0, 1]], u32), dev([0], u32), dev([1, 1, 1], u32), 1, 3)
    n = 40
    kr, vr = (rng.standard_normal((n, kv * hd)).astype(np.float32) for _ in range(2))
    K.pages_write(pages, seqs, 0, dev(kr), dev(vr), dev(np.zeros(n), u32), dev(np.arange(n), u32), n)
    c = R.Cache(rng, [n], kv=kv, hd=hd, page=page, f32=kv_type == "f32")
    c.table[0, :3] = [2, 0, 1]
    for x in range(n):
        at = (0, c.table[0, x // page], slice(None), x % page)
        c.k[at], c.v[at] = kr[x].reshape(kv, hd).astype(t), vr[x].reshape(kv, hd).astype(t)
    q = rng.standard_normal((1, 4, 4 * hd)).astype(np.float32)
    size = K.tree_attn_workspace(pages, seqs, 1, 4, 4)
    out = K.DeviceArray(q.shape)
    K.tree_attn(pages, seqs, 0, dev(q), dev([36], u32), None, None, 1, 4, 4, K.DeviceArray(max(size, 4), np.uint8),
                size, out)
    close(out.numpy(), R.tree_rows(c, 0, q, [36], [4], None, 4, np.zeros(q.shape)), R.attn_tol(hd, n, q, c.k), c.v)
    bounds = K.DeviceArray((3, kv, 2, hd), t)
    bounds.zero()
    K.page_bounds(pages, seqs, 0, dev([0], u32), dev([n], u32), 1, bounds)
    want = np.zeros((3, kv, 2, hd), t)
    R.bounds_of(c, 0, 0, 0, n, want)
    assert np.array_equal(bounds.numpy(), want)


@pytest.mark.parametrize("heads", [2, 24])
def test_f32_values_of_any_size(heads):
    """Keys and values whose size changes from page to page by many powers of ten, either way, among them nothing but
    zeros; and all of one size, far from 1."""
    rng = np.random.default_rng(25)
    T, hd, sizes = 3, 64, [1e-12, 1.0, 0.0, 1e9, 1e-3, 1e30, 1e-30]
    for order in (sizes, sizes[::-1]):
        c = R.Cache(rng, [32 * len(order) + T], kv=1, hd=hd, page=32, f32=True)
        for x, size in enumerate(order):
            c.v[0, c.table[0, x]] *= np.float32(size)
        for x in range(0, len(order), 2):
            c.k[0, c.table[0, x]] *= np.float32(1e-20)
        c.up()
        q = rng.standard_normal((1, T, heads * hd)).astype(np.float32)
        ctx = 32 * len(order)
        got = run_tree(c, 0, q, [ctx], [T], None, heads)
        want = R.tree_rows(c, 0, q, [ctx], [T], None, heads, np.zeros(q.shape))
        close(got, want, R.attn_tol(hd, ctx + T, q, c.k), c.v)
    # one size at a time
    for size in (1e-30, 1e-9, 1e25):
        c = R.Cache(rng, [40 + T], kv=1, hd=hd, f32=True)
        c.v *= np.float32(size)
        c.k *= np.float32(1 / size if size < 1 else 1)
        c.up()
        q = (rng.standard_normal((1, T, heads * hd)) * min(size, 1)).astype(np.float32)
        got = run_tree(c, 0, q, [40], [T], None, heads)
        want = R.tree_rows(c, 0, q, [40], [T], None, heads, np.zeros(q.shape))
        close(got, want, R.attn_tol(hd, 40 + T, q * (1 / min(size, 1)), c.k * min(size, 1)), c.v)


def ragged(rng, n, most, T):
    """Lengths of a batch: short ones, a few long, some without a draft."""
    ctx = [int(x) for x in rng.integers(0, 60, n)]
    for i in rng.integers(0, n, 5):
        ctx[i] = int(rng.integers(most // 2, most))
    nd = [int(x) for x in rng.integers(0, T + 1, n)]
    return ctx, nd


@pytest.mark.parametrize("t,hd,heads,kv,T,n", [("f16", 64, 8, 1, 16, 300), ("f16", 64, 16, 2, 20, 7), ("f16", 128, 6, 1, 8, 160),
                                               ("f16", 128, 16, 2, 30, 5), ("f32", 64, 16, 2, 12, 9), ("f32", 128, 5, 1, 9, 6)])
def test_long_tables_over_runs_of_steps(t, hd, heads, kv, T, n):
    """Tables long enough that the work is counted on the device and dealt out in equal runs: many short sequences, a few
    long ones, some with nothing to do, one without a slot, more of them than a workgroup has threads."""
    rng = np.random.default_rng(n + hd)
    ctx, nd = ragged(rng, n, 1500 if n > 100 else 4000, T)
    ctx[0] = 1500
    c = R.Cache(rng, [x + d for x, d in zip(ctx, nd)], kv=kv, hd=hd, f32=t == "f32", width=1 << 12).up()
    q = rng.standard_normal((n, T, heads * hd)).astype(np.float32) * 2
    mask = R.words(np.stack([R.ancestors(rng, T) for _ in range(n)]))
    slots = rng.permutation(n)
    slots[-1] = n + 3
    pick = lambda a: [a[i] if i < n else 5 for i in slots]  # noqa: E731
    got = run_tree(c, 0, q, pick(ctx), pick(nd), mask, heads, slots)
    want = R.tree_rows(c, 0, q, pick(ctx), pick(nd), mask, heads, np.full(q.shape, 7.5), slots)
    for i in range(n - 1):
        assert (got[i, pick(nd)[i]:] == 7.5).all()
    assert (got[-1] == 7.5).all()
    close(got, want, R.attn_tol(hd, 4100, q, c.k), c.v[np.isfinite(c.v)])
    again = run_tree(c, 0, q, pick(ctx), pick(nd), mask, heads, slots)
    assert np.array_equal(got, again)


@pytest.mark.parametrize("heads", [3, 20, 60])
@pytest.mark.parametrize("t,hd", [("f16", 64), ("f16", 128), ("f32", 64), ("f32", 128)])
def test_short_sequences_in_a_long_table(t, hd, heads):
    """Chunks follow a sequence's own length: none, one position, about a chunk, the table's whole capacity."""
    rng = np.random.default_rng(hd + heads)
    T, ctx = 2, [0, 1, 126, 127, 128, 254, 255, 256, 600, 3000, 4094]
    c = R.Cache(rng, [x + T for x in ctx], kv=1, hd=hd, f32=t == "f32", width=256).up()
    q = rng.standard_normal((len(ctx), T, heads * hd)).astype(np.float32)
    got = run_tree(c, 0, q, ctx, None, None, heads)
    want = R.tree_rows(c, 0, q, ctx, [T] * len(ctx), None, heads, np.full(q.shape, 7.5))
    close(got, want, R.attn_tol(hd, 4096, q, c.k), c.v)


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("heads", [1, 40])
def test_many_small_weights_beside_a_large_one(t, heads):
    """One position of weight 1 and V 0, the others of 2^-17 (1 + 2^-8) and V 1: many weights that all round alike.

    So many sequences (of the same pages) that a wave's share is long, 4096 positions (heads 1).  A rounding of a sum
    for each product of 32 positions and part, 2^-24 each, were one wave to take all.  The large score is off by 4 + 1
    steps of its 17, times ln 2 on a weight; the small scores are exact, their weights off by 4 steps; 64 for the rest."""
    n, length = 1024 if heads == 1 else 64, 16384
    rng = np.random.default_rng(3)
    c = R.Cache(rng, [length], kv=1, hd=64, page=256, f32=t == "f32")
    c.k[...] = 0
    c.v[...] = 1
    c.k[0, c.table[0, 1], 0, 2, 0] = 1
    c.v[0, c.table[0, 1], 0, 2] = 0
    c.up()
    low = 17 - np.log2(1 + 2.0 ** -8)
    q = np.zeros((n, 1, heads * 64), np.float32)
    q[:, :, ::64] = low * 8 / np.log2(np.e)
    got = run_tree(c, 0, q, [length - 1] * n, None, None, heads, np.zeros(n, np.uint32))
    w = (length - 1) * np.exp(-q[0, 0, 0].astype(np.float64) / 8)
    tol = 2.0 ** -24 * (2 * length // 32 + 17 * 5 + 4 + 64)
    assert np.abs(got - w / (1 + w)).max() <= tol * w / (1 + w)


@pytest.mark.parametrize("t,hd,heads", [("f16", 128, 9), ("f16", 64, 17), ("f32", 64, 5), ("f32", 128, 8)])
def test_sparse_of_many_heads_over_long_tables(t, hd, heads):
    rng = np.random.default_rng(hd * heads)
    ctx = [16 * 500 - 1, 16 * 300, 40]
    c = R.Cache(rng, ctx, kv=1, hd=hd, f32=t == "f32").up()
    q = rng.standard_normal((3, heads * hd)).astype(np.float32)
    b = all_bounds(c, 0)
    got, taken = run_sparse(c, 0, q, ctx, b, heads, 20, 1, 2)
    for s in range(3):
        assert np.array_equal(taken[s], R.choose(c, s, q[s], ctx[s], b, heads, 20, 1, 2)), s
        close(got[s], R.sparse_rows(c, 0, s, q[s], ctx[s], taken[s], heads), R.attn_tol(hd, 320, q, c.k), c.v)


def test_nothing_to_do_in_a_long_table():
    rng = np.random.default_rng(26)
    c = R.Cache(rng, [5, 0], kv=2, hd=64, width=1 << 14).up()
    q = rng.standard_normal((2, 40, 8 * 64)).astype(np.float32)
    assert (run_tree(c, 0, q, [5, 0], [0, 0], None, 8) == 7.5).all()


def test_drafts_longer_than_a_step():
    """300 tokens: masks of ten words, windows that begin inside a word; and a chain of them."""
    rng = np.random.default_rng(27)
    T = 300
    c = R.Cache(rng, [77 + T], kv=1, hd=64).up()
    q = rng.standard_normal((1, T, 64)).astype(np.float32) * 2
    for mask in (R.words(R.ancestors(rng, T)[None]), None):
        got = run_tree(c, 0, q, [77], [T], mask, 1)
        close(got, R.tree_rows(c, 0, q, [77], [T], mask, 1, np.zeros(q.shape)), R.attn_tol(64, 77 + T, q, c.k), c.v)


def test_compact_of_long_paths():
    """More rows than a block finds at once, over page borders, every place a source of a later one."""
    rng = np.random.default_rng(28)
    T = 260
    c = R.Cache(rng, [30 + T, 5 + T], kv=2, hd=64, layers=2).up()
    path = np.stack([np.sort(rng.choice(T, 200, replace=False)) for _ in range(2)]).astype(u32)
    path[0, 150:] = path[0, 149]  # ends here
    start = [30, 5]
    K.pages_compact(c.pages, c.seqs, dev([0, 1], u32), dev(start, u32), dev(path), dev([200, 193], u32), 2, 200)
    for s, n in ((0, 150), (1, 193)):
        for j in range(n):
            a, b = start[s] + int(path[s, j]), start[s] + j
            for pool in (c.k, c.v):
                pool[:, c.table[s, b // 16], :, b % 16] = pool[:, c.table[s, a // 16], :, a % 16]
    assert np.array_equal(c.dk.numpy(), c.k, equal_nan=True) and np.array_equal(c.dv.numpy(), c.v, equal_nan=True)


def test_sparse_over_thousands_of_pages():
    rng = np.random.default_rng(29)
    c = R.Cache(rng, [16 * 2600 - 3, 100], kv=1, hd=64).up()
    q = rng.standard_normal((2, 2 * 64)).astype(np.float32)
    b = all_bounds(c, 0)
    b[c.table[0, 1000], 0, 1, 5] = np.inf
    ctx = [int(x) for x in c.len]
    for take in (1, 40, 2599):
        got, taken = run_sparse(c, 0, q, ctx, b, 2, take, 0, min(1, take - 1))
        for s in range(2):
            assert np.array_equal(taken[s], R.choose(c, s, q[s], ctx[s], b, 2, take, 0, min(1, take - 1))), (take, s)
        assert 1000 in taken[0]
        close(got[0], R.sparse_rows(c, 0, 0, q[0], ctx[0], taken[0], 2), R.attn_tol(64, take * 16, q, c.k), c.v)


# ------------------------------------------------------------------- pages

def same_book(c, b):
    assert np.array_equal(c.dt.numpy(), b.table())
    assert c.dl.numpy().tolist() == b.len and c.dr.numpy().tolist() == b.refs


def grow(c, b, slots, add):
    ok, copied = dev(np.full(len(slots), 9), u32), dev(np.full((len(slots), 2), 9), u32)
    K.pages_grow(c.pages, c.seqs, dev(slots, u32), dev(add, u32), len(slots), ok, copied)
    want = b.grow(slots, add)
    assert ok.numpy().tolist() == want[0] and [tuple(x) for x in copied.numpy().tolist()] == want[1]
    same_book(c, b)
    return want


def fork(c, b, src, dst):
    ok = dev(np.full(len(src), 9), u32)
    K.pages_fork(c.pages, c.seqs, dev(src, u32), dev(dst, u32), len(src), ok)
    assert ok.numpy().tolist() == b.fork(src, dst)
    same_book(c, b)


def trim(c, b, slots, keep):
    K.pages_trim(c.pages, c.seqs, dev(slots, u32), dev(keep, u32), len(slots))
    b.trim(slots, keep)
    same_book(c, b)


@pytest.mark.parametrize("page,f32", [(16, False), (64, True)])
def test_fork_grow_trim_as_a_book_does(page, f32):
    rng = np.random.default_rng(11)
    c = R.Cache(rng, [37, 0, page, 0, 2 * page + 1, 0], page=page, f32=f32, layers=3, spare=7, width=6).up()
    b = R.Book(c)
    k0, v0 = c.k.copy(), c.v.copy()
    fork(c, b, [0, 4, 1, 0], [1, 3, 5, 1])          # 1 is a destination, and named twice: refused
    ok, copied = grow(c, b, [1, 3, 0, 2], [1, page, 0, 5])
    for i, s in enumerate([1, 3]):                   # their shared last pages were copied, in all layers
        old, new = copied[i]
        assert old != NO and new != NO
        rows = [37, 2 * page + 1][i] % page
        k0[:, new, :, :rows], v0[:, new, :, :rows] = k0[:, old, :, :rows], v0[:, old, :, :rows]
    assert np.array_equal(c.dk.numpy(), k0, equal_nan=True) and np.array_equal(c.dv.numpy(), v0, equal_nan=True)
    grow(c, b, [1, 2, 6, 2, 0], [3, 1, 1, 1, 60000])  # no such slot, twice, too long
    trim(c, b, [1, 9, 3, 1], [page + 1, 0, 0, 0])
    grow(c, b, [5, 0], [5 * page, 1])                 # an empty one grows
    grow(c, b, [2, 4, 3, 0], [4 * page, 3 * page, 4 * page, 0])  # the pages run out
    trim(c, b, [0, 1, 2, 3, 4, 5], [0] * 6)
    assert sum(b.refs) == 0


def test_two_forks_of_one_page_grow_at_once():
    """Both copy it; the page itself is free afterwards where nobody else holds it."""
    rng = np.random.default_rng(12)
    c = R.Cache(rng, [20, 0, 0], spare=6, width=4).up()
    b = R.Book(c)
    fork(c, b, [0, 0], [1, 2])
    _, copied = grow(c, b, [0, 1, 2], [1, 1, 1])
    assert len({x[1] for x in copied}) == 3 and b.refs[copied[0][0]] == 0
    k = c.dk.numpy()
    for s in range(3):
        assert np.array_equal(k[:, b.held[s][1], :, :4], c.k[:, c.table[0, 1], :, :4])


def test_trimmed_into_a_shared_page():
    rng = np.random.default_rng(13)
    c = R.Cache(rng, [64, 0], spare=3, width=6).up()
    b = R.Book(c)
    fork(c, b, [0], [1])
    trim(c, b, [1], [40])
    _, copied = grow(c, b, [1], [30])
    assert copied[0][0] == c.table[0, 2]
    fork(c, b, [0], [0])


def test_books_of_many_sequences():
    rng = np.random.default_rng(14)
    n = 300
    lengths = [int(x) for x in rng.integers(0, 200, n)] + [0] * n
    c = R.Cache(rng, lengths, kv=1, spare=6000, width=32).up()
    b = R.Book(c)
    for _ in range(4):
        src, dst = rng.integers(0, 2 * n + 3, n).tolist(), rng.integers(0, 2 * n + 3, n).tolist()
        fork(c, b, src, dst)
        slots = rng.integers(0, 2 * n, 700).tolist()
        grow(c, b, slots, rng.integers(0, 120, 700).tolist())
        slots = rng.integers(0, 2 * n, 500).tolist()
        trim(c, b, slots, rng.integers(0, 150, 500).tolist())
    grow(c, b, list(range(2 * n)), [500] * (2 * n))  # more than there is


@pytest.mark.parametrize("f32,hd,kv", [(False, 64, 2), (False, 128, 3), (True, 64, 1), (True, 128, 2)])
def test_write(f32, hd, kv):
    rng = np.random.default_rng(15)
    c = R.Cache(rng, [50, 33], kv=kv, hd=hd, f32=f32, layers=2, page=32, width=3)
    c.table[1, 1] = NO
    c.up()
    slots = [0, 0, 1, 1, 0, 2, 1, 0]
    pos = [49, 32, 0, 40, 63, 0, 95, 0xFFFFFFFF]  # a hole, a place behind the table, no such slot
    n, ld = len(slots), kv * hd + 12
    k, v = (rng.standard_normal((n, ld)).astype(np.float32) for _ in range(2))
    k[0, :4] = [65504, 65520, 1e-9, -2.0 ** -25]
    v[2, 0] = np.nan
    K.pages_write(c.pages, c.seqs, 1, dev(k), dev(v), dev(slots, u32), dev(pos, u32), n, ld=ld)
    with np.errstate(over="ignore"):
        for r, (s, x) in enumerate(zip(slots, pos)):
            if s < c.n and x // 32 < 3 and c.table[s, x // 32] < c.n_pages:
                at = (1, c.table[s, x // 32], slice(None), x % 32)
                c.k[at], c.v[at] = (a[r, :kv * hd].reshape(kv, hd).astype(c.k.dtype) for a in (k, v))
    assert np.array_equal(c.dk.numpy(), c.k, equal_nan=True) and np.array_equal(c.dv.numpy(), c.v, equal_nan=True)


@pytest.mark.parametrize("f32,hd", [(False, 64), (False, 128), (True, 64)])
def test_compact(f32, hd):
    rng = np.random.default_rng(17)
    T = 21
    c = R.Cache(rng, [40 + T, T, 15 + T, 100 + T, 30], kv=2, hd=hd, f32=f32, layers=3)
    c.table[3, 6] = NO
    c.up()
    slots = [0, 2, 3, 0, 7, 1, 4]
    start = [40, 15, 100, 40, 0, 0, 28]
    paths = [[0, 2, 3, 9, 10, 11, 12, 13, 14, 15, 20], [5], [1, 2, 20], [4, 5], [1], [0, 1, 5, 4, 9], [0, 1, 100, 1 << 31]]
    n_path = [11, 1, 3, 2, 1, 5, 999]
    path = np.full((len(slots), 12), 3, u32)
    for i, p in enumerate(paths):
        path[i, :len(p)] = p
    K.pages_compact(c.pages, c.seqs, dev(slots, u32), dev(start, u32), dev(path), dev(n_path, u32), len(slots), 12)
    for i, s in enumerate(slots):
        if s >= c.n or s in slots[:i]:
            continue
        before = -1
        for j in range(min(n_path[i], 12)):
            a, b = int(path[i, j]), start[i] + j
            if a <= before:
                break
            before = a
            a += start[i]
            if a // 16 >= c.width or c.table[s, a // 16] >= c.n_pages or c.table[s, b // 16] >= c.n_pages:
                continue
            for pool in (c.k, c.v):
                pool[:, c.table[s, b // 16], :, b % 16] = pool[:, c.table[s, a // 16], :, a % 16]
    assert np.array_equal(c.dk.numpy(), c.k, equal_nan=True) and np.array_equal(c.dv.numpy(), c.v, equal_nan=True)


# ------------------------------------------------------------------ sparse

@pytest.mark.parametrize("f32,hd,page", [(False, 64, 16), (False, 128, 32), (True, 64, 256), (True, 128, 64)])
def test_page_bounds(f32, hd, page):
    rng = np.random.default_rng(18)
    c = R.Cache(rng, [3 * page + 5, page, 0, 2 * page], kv=3, hd=hd, page=page, f32=f32, layers=2)
    c.k[:, c.table[3, 1], 1, page - 1, 7] = np.nan
    c.table[0, 1] = NO
    c.up()
    t = c.k.dtype
    want = rng.standard_normal((c.n_pages, 3, 2, hd)).astype(t)
    bounds = dev(want)
    slots, start, end = [0, 1, 2, 3, 9], [0, page - 1, 0, page, 0], [3 * page + 5, page, 0, 2 * page, 4]
    K.page_bounds(c.pages, c.seqs, 1, dev(start, u32), dev(end, u32), 5, bounds, slots=dev(slots, u32))
    for s, a, b in zip(slots, start, end):
        if s < c.n:
            R.bounds_of(c, 1, s, a, b, want)
    assert np.array_equal(bounds.numpy(), want, equal_nan=True)


def run_sparse(c, layer, q, ctx, bounds, heads, take, first, last, slots=None):
    n = len(q)
    out, taken = dev(np.full(q.shape, 7.5, np.float32)), dev(np.full((n, c.kv, take), 5), u32)
    size = K.sparse_attn_workspace(c.pages, c.seqs, n, heads, take)
    ws = dev(np.full(size, 255, np.uint8))
    K.sparse_attn(c.pages, c.seqs, layer, dev(q), dev(ctx, u32), dev(bounds), n, heads, take, first, last, taken, ws,
                  size, out, slots=None if slots is None else dev(slots, u32))
    return out.numpy(), taken.numpy()


def all_bounds(c, layer):
    b = np.zeros((c.n_pages, c.kv, 2, c.hd), c.k.dtype)
    for s in range(c.n):
        R.bounds_of(c, layer, s, 0, int(c.len[s]), b)
    return b


SPARSE = [
    # kv type, hd, page, heads, kv heads, contexts, take, first, last
    ("f16", 64, 16, 9, 3, [2000, 100, 0, 1, 129], 8, 1, 1),
    ("f16", 64, 64, 14, 2, [3000, 513], 7, 1, 2),
    ("f16", 128, 32, 32, 8, [1500], 5, 0, 0),
    ("f16", 64, 256, 16, 1, [5000, 1025], 4, 2, 2),
    ("f16", 128, 16, 20, 1, [600], 30, 0, 3),
    ("f32", 64, 16, 4, 4, [700, 17], 3, 0, 1),
    ("f32", 128, 64, 8, 2, [900], 6, 1, 1),
    ("f16", 64, 16, 3, 1, [9000], 300, 1, 1),
]


@pytest.mark.parametrize("case", SPARSE, ids=lambda c: "-".join(map(str, c[:5])))
def test_sparse_attn(case):
    t, hd, page, heads, kv, ctxs, take, first, last = case
    rng = np.random.default_rng(hd + page + heads)
    c = R.Cache(rng, ctxs, kv=kv, hd=hd, page=page, f32=t == "f32", layers=2).up()
    q = rng.standard_normal((len(ctxs), heads * hd)).astype(np.float32) * 2
    b = all_bounds(c, 1)
    got, taken = run_sparse(c, 1, q, ctxs, b, heads, take, first, last)
    for s, x in enumerate(ctxs):
        want = R.choose(c, s, q[s], x, b, heads, take, first, last)
        assert np.array_equal(taken[s], want), s
        close(got[s], R.sparse_rows(c, 1, s, q[s], x, want, heads), R.attn_tol(hd, take * page, q, c.k), c.v)
        if x == 0:
            assert (got[s] == 0).all()


def test_sparse_ties_nans_and_holes():
    """Pages of one content have one score: the lowest are taken; a NaN bound is taken first; a hole last."""
    rng = np.random.default_rng(19)
    c = R.Cache(rng, [16 * 40, 16 * 30], kv=2, hd=64)
    same = c.k[0, c.table[0, 3]].copy()
    for x in range(2, 30):
        c.k[0, c.table[0, x]] = same
    c.k[0, c.table[0, 33], 1, 4, 9] = np.nan
    c.table[1, [4, 5, 6]] = [NO, c.n_pages, 1 << 31]
    c.up()
    q = rng.standard_normal((2, 4 * 64)).astype(np.float32)
    c.len[1] = 16 * 30
    b = np.zeros((c.n_pages, 2, 2, 64), np.float16)
    for s in range(2):
        R.bounds_of(c, 0, s, 0, int(c.len[s]), b)
    for take in (5, 12, 28, 39):
        got, taken = run_sparse(c, 0, q, c.len, b, 4, take, 1, 1)
        for s in range(2):
            want = R.choose(c, s, q[s], int(c.len[s]), b, 4, take, 1, 1)
            assert np.array_equal(taken[s], want), (take, s)
        assert 33 in taken[0, 1]
        # sequence 1 reads around its holes
        close(got[1], R.sparse_rows(c, 0, 1, q[1], 480, taken[1], 4), R.attn_tol(64, 640, q, c.k[np.isfinite(c.k)]), c.v)


def test_sparse_of_everything_is_all_of_it():
    rng = np.random.default_rng(20)
    ctx = [333, 64, 1]
    c = R.Cache(rng, ctx, kv=2, hd=64).up()
    q = rng.standard_normal((3, 14 * 64)).astype(np.float32)
    got, taken = run_sparse(c, 0, q, ctx, all_bounds(c, 0), 14, 64, 0, 0)
    one = run_tree(c, 0, q[:, None], [x - 1 for x in ctx], None, None, 14)[:, 0]
    close(got, one.astype(np.float64), 2 * R.attn_tol(64, 333, q, c.k), c.v)
    assert (taken[2, :, 0] == 0).all() and (taken[2, :, 1:] == NO).all()


def test_sparse_slots():
    rng = np.random.default_rng(21)
    c = R.Cache(rng, [300, 500], kv=1, hd=64).up()
    q = rng.standard_normal((3, 2 * 64)).astype(np.float32)
    slots, ctx = [1, 2, 0], [500, 30, 299]
    b = all_bounds(c, 0)
    got, taken = run_sparse(c, 0, q, ctx, b, 2, 6, 1, 1, slots=slots)
    assert (got[1] == 7.5).all() and (taken[1] == NO).all()
    for i in (0, 2):
        want = R.choose(c, slots[i], q[i], ctx[i], b, 2, 6, 1, 1)
        assert np.array_equal(taken[i], want)
        close(got[i], R.sparse_rows(c, 0, slots[i], q[i], ctx[i], want, 2), R.attn_tol(64, 500, q, c.k), c.v)


# ------------------------------------------------------------ all together

@pytest.mark.parametrize("f32", [False, True])
def test_drafting_over_forked_sequences(f32):
    """Prompts are written, one is forked, both draft trees, verify them, keep a path each and go on with one token,
    over few pages; checked against caches kept as plain arrays."""
    rng = np.random.default_rng(22)
    kv, hd, heads, page, layers, T = 2, 64, 6, 16, 2, 6
    c = R.Cache(rng, [0, 0, 0], kv=kv, hd=hd, page=page, f32=f32, layers=layers, spare=14, width=5).up()
    b = R.Book(c)
    t = c.k.dtype
    plain = [[np.zeros((2, 0, kv, hd)) for _ in range(layers)] for _ in range(3)]  # [slot][layer] K, V rows

    def write(slots, pos):
        for layer in range(layers):
            k, v = (rng.standard_normal((len(slots), kv * hd)).astype(np.float32) for _ in range(2))
            K.pages_write(c.pages, c.seqs, layer, dev(k), dev(v), dev(slots, u32), dev(pos, u32), len(slots))
            for r, (s, x) in enumerate(zip(slots, pos)):
                assert x == plain[s][layer].shape[1]
                row = np.stack([a[r].astype(t).reshape(1, kv, hd) for a in (k, v)]).astype(np.float64)
                plain[s][layer] = np.concatenate([plain[s][layer], row], 1)

    def attend(layer, slots, ctx, nd, mask):
        q = rng.standard_normal((len(slots), T, heads * hd)).astype(np.float32)
        got = run_tree(c, layer, q, ctx, nd, mask, heads, slots)
        for i, s in enumerate(slots):
            kk, vv = plain[s][layer]
            for r in range(nd[i]):
                sees = np.arange(len(kk)) < ctx[i]
                for j in range(nd[i]):
                    sees[ctx[i] + j] = mask[i, r, 0] >> j & 1
                for h in range(heads):
                    a = slice(h * hd, h * hd + hd)
                    want = R.softmax_rows(q[i, r:r + 1, a].astype(np.float64), kk[:, h // 3], vv[:, h // 3], sees[None])
                    close(got[i, r, a], want[0], R.attn_tol(hd, 80, q, kk), vv)

    grow(c, b, [0, 2], [21, 9])
    write([0] * 21 + [2] * 9, list(range(21)) + list(range(9)))
    fork(c, b, [0], [1])
    plain[1] = [x.copy() for x in plain[0]]
    for turn in range(3):
        slots, ctx = [1, 0, 2], [b.len[1], b.len[0], b.len[2]]
        nd = [6, 4, 1 + turn]
        ok, _ = grow(c, b, slots, nd)
        assert ok == [1, 1, 1]
        write([s for s, m in zip(slots, nd) for _ in range(m)], [x + j for x, m in zip(ctx, nd) for j in range(m)])
        mask = R.words(np.stack([R.ancestors(rng, T) for _ in slots]))
        for layer in range(layers):
            attend(layer, slots, ctx, nd, mask)
        paths = [[0, 2, 5], [0, 3], [0]]
        path = np.zeros((3, 3), u32)
        for i, p in enumerate(paths):
            path[i, :len(p)] = p
        K.pages_compact(c.pages, c.seqs, dev(slots, u32), dev(ctx, u32), dev(path), dev([3, 2, 1], u32), 3, 3)
        trim(c, b, slots, [x + len(p) for x, p in zip(ctx, paths)])
        for i, s in enumerate(slots):
            for layer in range(layers):
                at = list(range(ctx[i])) + [ctx[i] + j for j in paths[i]]
                plain[s][layer] = plain[s][layer][:, at]
    # and one token each over pages chosen by their bounds
    n = [b.len[s] for s in range(3)]
    bounds = dev(np.zeros((c.n_pages, kv, 2, hd), t))
    K.page_bounds(c.pages, c.seqs, 1, dev([0, 0, 0], u32), dev(n, u32), 3, bounds)
    q = rng.standard_normal((3, heads * hd)).astype(np.float32)
    got, taken = run_sparse(c, 1, q, n, bounds.numpy(), heads, 2, 0, 1)
    c.k, c.v, c.table = c.dk.numpy(), c.dv.numpy(), c.dt.numpy()
    for s in range(3):
        kk, vv = plain[s][1]
        assert np.array_equal(c.rows(c.k, 1, s, n[s]).transpose(1, 0, 2), kk)
        want = R.choose(c, s, q[s], n[s], bounds.numpy(), heads, 2, 0, 1)
        assert np.array_equal(taken[s], want)
        close(got[s], R.sparse_rows(c, 1, s, q[s], n[s], want, heads), R.attn_tol(hd, 80, q, kk), vv)


def test_results_do_not_depend_on_the_run():
    rng = np.random.default_rng(23)
    c = R.Cache(rng, [4000, 700], kv=2, hd=64).up()
    q = rng.standard_normal((2, 20, 14 * 64)).astype(np.float32)
    mask = R.words(np.stack([R.ancestors(rng, 20) for _ in range(2)]))
    a = [run_tree(c, 0, q, [3980, 680], [20, 20], mask, 14) for _ in range(3)]
    assert all(np.array_equal(x, a[0]) for x in a)
    b = all_bounds(c, 0)
    s = [run_sparse(c, 0, q[:, 0], [4000, 700], b, 14, 9, 1, 1) for _ in range(3)]
    assert all(np.array_equal(x[0], s[0][0]) and np.array_equal(x[1], s[0][1]) for x in s)


def test_streams_and_two_captured_graphs():
    """The calls on a caller's stream, and a step of them captured twice, each with its workspace, replayed in turn
    with eager calls between."""
    hip = C.CDLL("libamdhip64.so")
    hip.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    hip.hipStreamEndCapture.argtypes = [C.c_void_p, C.c_void_p]
    hip.hipGraphInstantiate.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    hip.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    hip.hipGraphExecDestroy.argtypes = hip.hipGraphDestroy.argtypes = [C.c_void_p]
    rng = np.random.default_rng(24)
    kv, hd, heads, T = 2, 64, 6, 4
    c = R.Cache(rng, [600, 90], kv=kv, hd=hd, layers=1, spare=8, width=48).up()
    ctx = [596, 86]
    mask = dev(R.words(np.stack([R.ancestors(rng, T) for _ in range(2)])))
    q = rng.standard_normal((2, T, heads * hd)).astype(np.float32)
    size = K.tree_attn_workspace(c.pages, c.seqs, 2, T, heads)
    size2 = K.sparse_attn_workspace(c.pages, c.seqs, 2, heads, 4)
    dctx, dend, dnd, dq1 = dev(ctx, u32), dev([600, 90], u32), dev([T, T - 1], u32), dev(q[:, 0])
    bounds = dev(np.zeros((c.n_pages, kv, 2, hd), np.float16))
    zero = dev([0, 0], u32)
    dslots, dadd, dkeep = dev([0, 1], u32), dev([3, 40], u32), dev([600, 90], u32)

    def buffers():
        return dict(q=dev(q), out=dev(np.zeros(q.shape, np.float32)), sout=dev(np.zeros((2, heads * hd), np.float32)),
                    taken=dev(np.zeros((2, kv, 4), u32)), ws=K.DeviceArray(max(size, 4), np.uint8),
                    ws2=K.DeviceArray(size2, np.uint8), ok=dev([9, 9], u32), copied=dev(np.full((2, 2), 9), u32))

    def step(d, stream):
        K.pages_grow(c.pages, c.seqs, dslots, dadd, 2, d["ok"], d["copied"], stream=stream)
        K.tree_attn(c.pages, c.seqs, 0, d["q"], dctx, dnd, mask, 2, T, heads, d["ws"], size, d["out"], stream=stream)
        K.pages_trim(c.pages, c.seqs, dslots, dkeep, 2, stream=stream)
        K.page_bounds(c.pages, c.seqs, 0, zero, dend, 2, bounds, stream=stream)
        K.sparse_attn(c.pages, c.seqs, 0, dq1, dend, bounds, 2, heads, 4, 1, 1, d["taken"], d["ws2"], size2, d["sout"],
                      stream=stream)

    def result(d):
        return d["out"].numpy(), d["sout"].numpy(), d["taken"].numpy(), d["ok"].numpy()

    eager, mine = buffers(), buffers()
    step(eager, None)
    want = result(eager)
    assert want[3].tolist() == [1, 1]
    st = K.Stream()
    step(mine, st.ptr)
    st.synchronize()
    assert all(np.array_equal(a, b) for a, b in zip(result(mine), want))
    graphs = []
    for _ in range(2):
        d, graph, ex = buffers(), C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(st.ptr, 0) == 0
        step(d, st.ptr)
        assert hip.hipStreamEndCapture(st.ptr, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
        graphs.append((d, graph, ex))
    for _ in range(4):
        for d, _, ex in graphs:
            K.memset(d["out"], 0)
            K.memset(d["taken"], 0)
            K.synchronize()
            assert hip.hipGraphLaunch(ex, st.ptr) == 0
            st.synchronize()
            assert all(np.array_equal(a, b) for a, b in zip(result(d), want))
        step(eager, None)
        assert all(np.array_equal(a, b) for a, b in zip(result(eager), want))
    for _, graph, ex in graphs:
        assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0
    st.close()
    same = R.Book(c)
    same_book(c, same)
