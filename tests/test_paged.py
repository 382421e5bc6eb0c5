"""The paged KV cache's refusals, before any device work (no GPU needed), and what its workspaces ask for."""
import ctypes as C

import pytest

from lokal_amd import _lib
from lokal_amd import kernels as K


class Ptr:
    """A buffer that no call here may touch: the address alone."""

    def __init__(self, at=0x10000):
        self.ptr = C.c_void_p(at)


B = Ptr()


def pages(**kw):
    d = dict(kv_type=K.F16, n_layers=2, n_pages=8, n_kv_heads=2, page_size=16, head_dim=64)
    at = {n: kw.pop(n, B) for n in ("k", "v")}
    d.update(kw)
    return K.KvPages(at["k"], at["v"], **d)


def table(n_seq=4, max_pages=8, **kw):
    return K.PageTable(kw.get("table", B), kw.get("length", B), kw.get("refs", B), n_seq, max_pages)


def calls(p, t, n=2):
    """Every entry point on one cache."""
    return {
        "fork": lambda: K.pages_fork(p, t, B, B, n, B),
        "grow": lambda: K.pages_grow(p, t, B, B, n, B, B),
        "trim": lambda: K.pages_trim(p, t, B, B, n),
        "write": lambda: K.pages_write(p, t, 0, B, B, B, B, n),
        "compact": lambda: K.pages_compact(p, t, B, B, B, B, n, 4),
        "bounds": lambda: K.page_bounds(p, t, 0, B, B, n, B),
        "tree": lambda: K.tree_attn(p, t, 0, B, B, B, B, n, 4, 6, B, 1 << 40, B),
        "sparse": lambda: K.sparse_attn(p, t, 0, B, B, B, n, 6, 4, 1, 1, B, B, 1 << 40, B),
        "tree_ws": lambda: K.tree_attn_workspace(p, t, n, 4, 6),
        "sparse_ws": lambda: K.sparse_attn_workspace(p, t, n, 6, 4),
    }


NAMES = sorted(calls(pages(), table()))


def refused(f, match, code=-1):
    with pytest.raises(_lib.LokalHipError, match=match) as e:
        f()
    assert e.value.code == code and "\n" not in str(e.value)


@pytest.mark.parametrize("name", NAMES)
def test_caches_that_do_not_run(name):
    def call(**kw):
        return calls(pages(**kw), table())[name]
    refused(call(k=Ptr(0)), "null argument")
    refused(call(v=Ptr(0)), "null argument")
    refused(call(kv_type=8), "F16 or F32", -2)
    for hd in (0, 32, 80, 96, 256):
        refused(call(head_dim=hd), "64 or 128", -2)
    for size in (0, 1, 8, 24, 48, 512):
        refused(call(page_size=size), "16, 32, 64, 128 or 256", -2)
    refused(call(n_kv_heads=0), "kv heads")
    refused(call(n_kv_heads=1025), "kv heads")
    refused(call(n_layers=0), "layers")
    refused(call(n_pages=0), "number of pages")
    refused(call(n_pages=1 << 31), "number of pages")
    refused(call(k=Ptr(0x10008)), "16-byte aligned")
    refused(call(v=Ptr(0x10002)), "16-byte aligned")
    refused(call(page_stride=2 * 16 * 64 + 4), "page_stride")
    refused(call(kv_type=K.F32, page_stride=2 * 16 * 64 + 2), "page_stride")
    refused(call(page_stride=16 * 64 - 8), "page_stride")
    refused(call(head_stride=512), "head_stride")
    refused(call(layer_stride=0), "layer_stride")
    refused(call(page_stride=1 << 62), "2\\^60")
    refused(call(layer_stride=(1 << 64) - 8, n_layers=4), "2\\^60")


@pytest.mark.parametrize("name", NAMES)
def test_tables_that_do_not_run(name):
    def call(**kw):
        return calls(pages(), table(**kw))[name]
    refused(call(table=Ptr(0)), "null argument")
    refused(call(n_seq=0), "at least one")
    refused(call(max_pages=0), "at least one")
    refused(call(max_pages=1 << 27), "2\\^31 positions")
    if name in ("fork", "grow", "trim"):
        refused(call(length=None), "null argument")
        refused(call(refs=None), "null argument")
        refused(calls(pages(), table(), 1025)[name], "at most 1024")


def test_strides_whose_count_is_one_do_not_matter():
    p = pages(n_layers=1, n_pages=1, n_kv_heads=1, page_stride=0, head_stride=3, layer_stride=1)
    assert K.tree_attn_workspace(p, table(max_pages=1), 1, 1, 1) >= 0


@pytest.mark.parametrize("name", NAMES)
def test_nothing_to_do_needs_no_device(name):
    calls(pages(), table(), 0)[name]()


def test_null_arguments():
    p, t, no = pages(), table(), Ptr(0)
    lists = [lambda x: K.pages_fork(p, t, *x[:2], 1, x[2]), lambda x: K.pages_grow(p, t, *x[:2], 1, *x[2:4]),
             lambda x: K.pages_trim(p, t, *x[:2], 1), lambda x: K.pages_write(p, t, 0, *x[:4], 1),
             lambda x: K.pages_compact(p, t, *x[:4], 1, 4), lambda x: K.page_bounds(p, t, 0, *x[:2], 1, x[2]),
             lambda x: K.tree_attn(p, t, 0, *x[:2], B, B, 1, 4, 6, B, 1 << 40, x[2]),
             lambda x: K.sparse_attn(p, t, 0, *x[:3], 1, 6, 4, 1, 1, x[3], B, 1 << 40, x[4])]
    counts = [3, 4, 2, 4, 4, 3, 3, 5]
    for f, m in zip(lists, counts):
        for i in range(m):
            refused(lambda: f([no if j == i else B for j in range(m)]), "null argument")


@pytest.mark.parametrize("layer", [2, 4294967295])
def test_layers_outside_the_cache(layer):
    p, t = pages(), table()
    refused(lambda: K.pages_write(p, t, layer, B, B, B, B, 1), "layer")
    refused(lambda: K.page_bounds(p, t, layer, B, B, 1, B), "layer")
    refused(lambda: K.tree_attn(p, t, layer, B, B, B, B, 1, 4, 6, B, 1 << 40, B), "layer")
    refused(lambda: K.sparse_attn(p, t, layer, B, B, B, 1, 6, 4, 1, 1, B, B, 1 << 40, B), "layer")


def test_write_rows():
    p, t = pages(), table()
    for ld in (124, 130, 1 << 31):
        refused(lambda: K.pages_write(p, t, 0, B, B, B, B, 1, ld=ld), "ld must be")
    refused(lambda: K.pages_write(p, t, 0, Ptr(0x10004), B, B, B, 1), "16-byte")
    refused(lambda: K.pages_write(p, t, 0, B, Ptr(0x10004), B, B, 1), "16-byte")
    refused(lambda: K.pages_write(p, t, 0, B, B, B, B, 1 << 28), "too many")


def test_attention_shapes():
    p, t = pages(), table()
    for heads in (0, 3, 4098):
        refused(lambda: K.tree_attn(p, t, 0, B, B, B, B, 1, 4, heads, B, 1 << 40, B), "query heads", -2)
        refused(lambda: K.tree_attn_workspace(p, t, 1, 4, heads), "query heads", -2)
        refused(lambda: K.sparse_attn(p, t, 0, B, B, B, 1, heads, 4, 1, 1, B, B, 1 << 40, B), "query heads", -2)
    refused(lambda: K.tree_attn(p, t, 0, B, B, B, B, 1, 1025, 6, B, 1 << 40, B), "at most 1024", -2)
    one = pages(n_kv_heads=1)
    refused(lambda: K.tree_attn(one, t, 0, B, B, B, B, 1, 1024, 65, B, 1 << 40, B), "at most 65536 rows", -2)
    assert K.tree_attn_workspace(one, t, 1, 1024, 64) >= 0
    many = pages(n_kv_heads=1024, n_pages=4)
    refused(lambda: K.tree_attn_workspace(many, t, 0xFFFF, 1, 1024), "too many for one call")
    refused(lambda: K.tree_attn_workspace(one, table(max_pages=(1 << 27) - 1), 1024, 1024, 8), "too many for one call")
    refused(lambda: K.tree_attn(p, t, 0, B, B, B, B, 1 << 16, 1, 6, B, 1 << 40, B), "at most 65535")
    refused(lambda: K.page_bounds(p, t, 0, B, B, 1 << 16, B), "at most 65535")
    refused(lambda: K.tree_attn(p, t, 0, Ptr(0x10004), B, B, B, 1, 4, 6, B, 1 << 40, B), "16-byte")
    refused(lambda: K.tree_attn(p, t, 0, B, B, B, B, 1, 4, 6, B, 1 << 40, Ptr(0x10008)), "16-byte")
    refused(lambda: K.sparse_attn(p, t, 0, B, B, Ptr(0x10002), 1, 6, 4, 1, 1, B, B, 1 << 40, B), "16-byte")
    for take, first, last in ((0, 0, 0), (4, 5, 0), (4, 0, 5), (4, 3, 2), (1 << 31, 0, 0), (4, (1 << 64) - 1, 2)):
        refused(lambda: K.sparse_attn(p, t, 0, B, B, B, 1, 6, take, first, last, B, B, 1 << 40, B), "first and")


def test_workspaces_are_checked():
    p, t = pages(n_pages=4096), table(max_pages=2048)
    need = K.tree_attn_workspace(p, t, 2, 8, 14)
    assert need > 0
    for ws, have in ((B, need - 1), (None, need), (Ptr(0x10008), need)):
        refused(lambda: K.tree_attn(p, t, 0, B, B, B, B, 2, 8, 14, ws, have, B), f"workspace of {need} bytes")
    need = K.sparse_attn_workspace(p, t, 2, 14, 16)
    assert need >= 2 * 2 * 2048 * 8
    refused(lambda: K.sparse_attn(p, t, 0, B, B, B, 2, 14, 16, 1, 1, B, B, need - 1, B), f"workspace of {need} bytes")


def test_workspaces_do_not_grow_with_what_a_sequence_holds():
    """They follow the table's capacity: what is known when a program makes them."""
    t = table(max_pages=2048)
    a = K.tree_attn_workspace(pages(n_pages=64), t, 4, 16, 14)
    assert a == K.tree_attn_workspace(pages(n_pages=8192), t, 4, 16, 14)
    assert K.tree_attn_workspace(pages(), t, 0, 16, 14) == 0 == K.tree_attn_workspace(pages(), t, 4, 0, 14)


def test_q_and_out_are_apart():
    rows = 2 * 4 * 6 * 64 * 4  # bytes of q, and of out
    for at in (0, 16, rows - 16, -16, 16 - rows):
        out = Ptr(0x100000 + at)
        refused(lambda: K.tree_attn(pages(), table(), 0, Ptr(0x100000), B, B, B, 2, 4, 6, B, 1 << 40, out), "overlap")
        if abs(at) < rows // 4:
            refused(lambda: K.sparse_attn(pages(), table(), 0, Ptr(0x100000), B, B, 2, 6, 4, 1, 1, B, B, 1 << 40, out), "overlap")
