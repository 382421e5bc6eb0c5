// paged_api.hip -- the entry points of the paged KV cache (include/lokal_hip.h):
// what the host can check of a call, the launches' plans and workspaces.
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/lokal_hip.h"
#include "lkhip_common.h"
#include "pages.h"

static int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return lk_fail(code, buf);
}
static int launched(hipError_t e, const char* who) {
    return e == hipSuccess ? LKHIP_OK : fail(LKHIP_E_HIP, "%s: kernel launch failed: %s", who, hipGetErrorString(e));
}

static bool aligned(const void* p, size_t to) { return (uintptr_t)p % to == 0; }

// layer < 0: all layers.
static int pages_of(const lkhip_kv_pages* c, int64_t layer, const char* who, LkPages& out) {
    if (!c || !c->k || !c->v) return fail(LKHIP_E_INVALID, "%s: null argument", who);
    if (c->kv_type != LKHIP_F16 && c->kv_type != LKHIP_F32)
        return fail(LKHIP_E_UNSUPPORTED, "%s: the KV cache is F16 or F32, not type %u", who, c->kv_type);
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(LKHIP_E_UNSUPPORTED, "%s: head_dim %u — 64 or 128", who, c->head_dim);
    uint32_t shift = 4;
    while (shift < 8 && (1u << shift) != c->page_size) shift++;
    if ((1u << shift) != c->page_size)
        return fail(LKHIP_E_UNSUPPORTED, "%s: pages of %u positions — 16, 32, 64, 128 or 256", who, c->page_size);
    if (c->n_kv_heads == 0 || c->n_kv_heads > 1024 || c->n_layers == 0 || c->n_layers > 4096)
        return fail(LKHIP_E_INVALID, "%s: %u kv heads (1..1024), %u layers (1..4096)", who, c->n_kv_heads, c->n_layers);
    if (c->n_pages == 0 || c->n_pages > 0x7FFFFFFF)
        return fail(LKHIP_E_INVALID, "%s: the number of pages must be in 1..2^31-1", who);
    const uint64_t es = c->kv_type == LKHIP_F32 ? 4 : 2, unit = 16 / es, rows = (uint64_t)c->page_size * c->head_dim;
    if (!aligned(c->k, 16) || !aligned(c->v, 16))
        return fail(LKHIP_E_INVALID, "%s: k and v must be 16-byte aligned", who);
    const struct {
        uint64_t stride, count;
        const char* name;
    } dims[3] = {{c->page_stride, c->n_pages, "page_stride"},
                 {c->head_stride, c->n_kv_heads, "head_stride"},
                 {c->layer_stride, c->n_layers, "layer_stride"}};
    uint64_t last = rows;
    for (const auto& d : dims) {
        if (d.count == 1) continue;
        uint64_t far;
        if (d.stride < rows || d.stride % unit)
            return fail(LKHIP_E_INVALID, "%s: %s (%llu) must be a multiple of %llu and at least a page's %llu elements",
                        who, d.name, (unsigned long long)d.stride, (unsigned long long)unit, (unsigned long long)rows);
        if (__builtin_mul_overflow(d.stride, d.count - 1, &far) || __builtin_add_overflow(far, last, &last) ||
            last > (1ull << 60))
            return fail(LKHIP_E_INVALID, "%s: the cache's strides pass 2^60 elements", who);
    }
    if (layer >= (int64_t)c->n_layers)
        return fail(LKHIP_E_INVALID, "%s: layer %lld of %u", who, (long long)layer, c->n_layers);
    const uint64_t at = layer > 0 ? (uint64_t)layer * c->layer_stride * es : 0;
    out = LkPages{(char*)c->k + at, (char*)c->v + at, c->kv_type == LKHIP_F32, c->head_dim, c->n_kv_heads, shift,
                  c->n_layers,      (uint32_t)c->n_pages, c->n_pages > 1 ? c->page_stride : 0,
                  c->n_kv_heads > 1 ? c->head_stride : 0, c->n_layers > 1 ? c->layer_stride : 0};
    return LKHIP_OK;
}

enum { NEED_LEN = 1, NEED_REFS = 2 };
static int table_of(const lkhip_page_table* t, const LkPages& p, int need, const char* who, LkTable& out) {
    if (!t || !t->table || ((need & NEED_LEN) && !t->len) || ((need & NEED_REFS) && !t->refs))
        return fail(LKHIP_E_INVALID, "%s: null argument", who);
    if (t->n_seq == 0 || t->n_seq > 0x7FFFFFFF || t->max_pages == 0 ||
        (uint64_t)t->max_pages << p.pshift > 0x7FFFFFFF)
        return fail(LKHIP_E_INVALID, "%s: a table of %u sequences x %u pages — at least one each, and below 2^31 positions",
                    who, t->n_seq, t->max_pages);
    out = LkTable{t->table, t->len, t->refs, t->n_seq, t->max_pages};
    return LKHIP_OK;
}

static int list_check(size_t n, const char* who) {
    if (n > LK_PAGES_LIST_MAX)
        return fail(LKHIP_E_INVALID, "%s: %zu sequences — one call takes at most %u", who, n, LK_PAGES_LIST_MAX);
    return LKHIP_OK;
}

#define CHECK(expr)            \
    do {                       \
        const int _rc = (expr); \
        if (_rc) return _rc;   \
    } while (0)

extern "C" int lkhip_pages_fork(const lkhip_kv_pages* pages, const lkhip_page_table* table, const uint32_t* src,
                                const uint32_t* dst, size_t n, uint32_t* ok, void* stream) {
    const char* who = "pages_fork";
    LkPages p;
    LkTable t;
    CHECK(pages_of(pages, -1, who, p));
    CHECK(table_of(table, p, NEED_LEN | NEED_REFS, who, t));
    CHECK(list_check(n, who));
    if (n == 0) return LKHIP_OK;
    if (!src || !dst || !ok) return fail(LKHIP_E_INVALID, "%s: null argument", who);
    return launched(lk_pages_fork_launch(p, t, src, dst, (uint32_t)n, ok, (hipStream_t)stream), who);
}

extern "C" int lkhip_pages_grow(const lkhip_kv_pages* pages, const lkhip_page_table* table, const uint32_t* slots,
                                const uint32_t* add, size_t n, uint32_t* ok, uint32_t* copied, void* stream) {
    const char* who = "pages_grow";
    LkPages p;
    LkTable t;
    CHECK(pages_of(pages, -1, who, p));
    CHECK(table_of(table, p, NEED_LEN | NEED_REFS, who, t));
    CHECK(list_check(n, who));
    if (n == 0) return LKHIP_OK;
    if (!slots || !add || !ok || !copied) return fail(LKHIP_E_INVALID, "%s: null argument", who);
    return launched(lk_pages_grow_launch(p, t, slots, add, (uint32_t)n, ok, copied, (hipStream_t)stream), who);
}

extern "C" int lkhip_pages_trim(const lkhip_kv_pages* pages, const lkhip_page_table* table, const uint32_t* slots,
                                const uint32_t* keep, size_t n, void* stream) {
    const char* who = "pages_trim";
    LkPages p;
    LkTable t;
    CHECK(pages_of(pages, -1, who, p));
    CHECK(table_of(table, p, NEED_LEN | NEED_REFS, who, t));
    CHECK(list_check(n, who));
    if (n == 0) return LKHIP_OK;
    if (!slots || !keep) return fail(LKHIP_E_INVALID, "%s: null argument", who);
    return launched(lk_pages_trim_launch(p, t, slots, keep, (uint32_t)n, (hipStream_t)stream), who);
}

extern "C" int lkhip_pages_write(const lkhip_kv_pages* pages, const lkhip_page_table* table, uint32_t layer,
                                 const float* k, const float* v, size_t ld, const uint32_t* slots, const uint32_t* pos,
                                 size_t n_rows, void* stream) {
    const char* who = "pages_write";
    LkPages p;
    LkTable t;
    CHECK(pages_of(pages, layer, who, p));
    CHECK(table_of(table, p, 0, who, t));
    if (n_rows == 0) return LKHIP_OK;
    if (!k || !v || !slots || !pos) return fail(LKHIP_E_INVALID, "%s: null argument", who);
    const size_t width = (size_t)p.n_kv * p.hd;
    if (ld < width || ld % 4 || ld > 0x7FFFFFFF || !aligned(k, 16) || !aligned(v, 16))
        return fail(LKHIP_E_INVALID, "%s: ld must be >= %zu (kv heads x head_dim) and a multiple of 4, k and v 16-byte aligned",
                    who, width);
    if (n_rows > 0x7FFFFFFF / (width / 8))
        return fail(LKHIP_E_INVALID, "%s: %zu rows of %zu values are too many for one call", who, n_rows, width);
    return launched(lk_pages_write_launch(p, t, k, v, (uint32_t)ld, slots, pos, (uint32_t)n_rows, (hipStream_t)stream),
                    who);
}

extern "C" int lkhip_pages_compact(const lkhip_kv_pages* pages, const lkhip_page_table* table, const uint32_t* slots,
                                   const uint32_t* from, const uint32_t* path, size_t ld_path, const uint32_t* n_path,
                                   size_t n, void* stream) {
    const char* who = "pages_compact";
    LkPages p;
    LkTable t;
    CHECK(pages_of(pages, -1, who, p));
    CHECK(table_of(table, p, 0, who, t));
    CHECK(list_check(n, who));
    if (n == 0 || ld_path == 0) return LKHIP_OK;
    if (!slots || !from || !path || !n_path) return fail(LKHIP_E_INVALID, "%s: null argument", who);
    if (ld_path > 0x7FFFFFFF) return fail(LKHIP_E_INVALID, "%s: paths of %zu entries", who, ld_path);
    return launched(lk_pages_compact_launch(p, t, slots, from, path, (uint32_t)ld_path, n_path, (uint32_t)n,
                                            (hipStream_t)stream),
                    who);
}

extern "C" int lkhip_page_bounds(const lkhip_kv_pages* pages, const lkhip_page_table* table, uint32_t layer,
                                 const uint32_t* slots, const uint32_t* from, const uint32_t* to, size_t n,
                                 void* bounds, void* stream) {
    const char* who = "page_bounds";
    LkPages p;
    LkTable t;
    CHECK(pages_of(pages, layer, who, p));
    CHECK(table_of(table, p, 0, who, t));
    if (n > 0xFFFF) return fail(LKHIP_E_INVALID, "%s: at most 65535 sequences per call", who);
    if (n == 0) return LKHIP_OK;
    if (!from || !to || !bounds) return fail(LKHIP_E_INVALID, "%s: null argument", who);
    return launched(lk_page_bounds_launch(p, t, slots, from, to, (uint32_t)n, bounds, (hipStream_t)stream), who);
}

// Shape checks that both attentions and their workspace sizes share; tokens > 0.
static int attn_shape(const LkPages& p, size_t n, size_t tokens, size_t n_heads, const char* who) {
    if (n > 0xFFFF) return fail(LKHIP_E_INVALID, "%s: at most 65535 sequences per call", who);
    if (n_heads == 0 || n_heads % p.n_kv || n_heads > 4096)
        return fail(LKHIP_E_UNSUPPORTED, "%s: %zu query heads over %u kv heads — a multiple of them, at most 4096", who,
                    n_heads, p.n_kv);
    if (tokens > 1024) return fail(LKHIP_E_UNSUPPORTED, "%s: %zu drafted tokens — at most 1024", who, tokens);
    if (tokens * (n_heads / p.n_kv) > 0x10000)
        return fail(LKHIP_E_UNSUPPORTED, "%s: %zu drafted tokens x %zu query heads of a kv head — at most 65536 rows", who,
                    tokens, n_heads / p.n_kv);
    return LKHIP_OK;
}
static int plan_of(const LkPages& p, const LkTable& t, size_t n, size_t tokens, size_t n_heads, size_t take,
                   const char* who, LkPagedPlan& plan, size_t& keys, size_t& bytes) {
    CHECK(attn_shape(p, n, tokens, n_heads, who));
    const uint64_t cap = (uint64_t)t.max_pages << p.pshift, taken = (uint64_t)take << p.pshift;
    plan = lk_paged_plan(p.hd, p.f32, take != 0, (uint32_t)n, p.n_kv, (uint32_t)(tokens * (n_heads / p.n_kv)),
                         take && taken < cap ? taken : cap);
    keys = take ? (size_t)n * p.n_kv * t.max_pages * 8 : 0;
    keys = (keys + 255) / 256 * 256;
    bytes = keys + plan.part_bytes;
    // grids of 256 threads a block, below 2^32 threads; steps are counted in 32 bits
    if (plan.blocks > 0xFFFFFF || (uint64_t)n * p.n_kv * (plan.n_chunks + 1) > 0xFFFFFF || plan.steps > 0xFFFFFFFF)
        return fail(LKHIP_E_INVALID, "%s: %zu sequences x %zu tokens x %zu heads over %llu positions are too many for one call",
                    who, n, tokens, n_heads, (unsigned long long)cap);
    return LKHIP_OK;
}
static int apart(const float* q, const float* out, size_t count, const char* who) {
    if ((uintptr_t)q < (uintptr_t)(out + count) && (uintptr_t)out < (uintptr_t)(q + count))
        return fail(LKHIP_E_INVALID, "%s: q and out overlap", who);
    return LKHIP_OK;
}
static int ws_check(const void* ws, size_t have, size_t need, const char* who) {
    if (need && (!ws || have < need || !aligned(ws, 16)))
        return fail(LKHIP_E_INVALID, "%s: needs a 16-byte aligned workspace of %zu bytes (got %zu)", who, need,
                    ws ? have : (size_t)0);
    return LKHIP_OK;
}

extern "C" int lkhip_tree_attn_workspace(const lkhip_kv_pages* pages, const lkhip_page_table* table, size_t n,
                                         size_t max_draft, size_t n_heads, size_t* bytes) {
    const char* who = "tree_attn_workspace";
    LkPages p;
    LkTable t;
    LkPagedPlan plan;
    size_t keys;
    if (!bytes) return fail(LKHIP_E_INVALID, "%s: null argument", who);
    *bytes = 0;
    CHECK(pages_of(pages, -1, who, p));
    CHECK(table_of(table, p, 0, who, t));
    if (n == 0 || max_draft == 0) return LKHIP_OK;
    return plan_of(p, t, n, max_draft, n_heads, 0, who, plan, keys, *bytes);
}

extern "C" int lkhip_tree_attn(const lkhip_kv_pages* pages, const lkhip_page_table* table, uint32_t layer,
                               const float* q, const uint32_t* slots, const uint32_t* ctx_len, const uint32_t* n_draft,
                               const uint32_t* mask, size_t n, size_t max_draft, size_t n_heads, void* ws,
                               size_t ws_bytes, float* out, void* stream) {
    const char* who = "tree_attn";
    LkPages p;
    LkTable t;
    LkPagedPlan plan;
    size_t keys, bytes;
    CHECK(pages_of(pages, layer, who, p));
    CHECK(table_of(table, p, 0, who, t));
    if (n == 0 || max_draft == 0) return LKHIP_OK;
    if (!q || !ctx_len || !out) return fail(LKHIP_E_INVALID, "%s: null argument", who);
    if (!aligned(q, 16) || !aligned(out, 16)) return fail(LKHIP_E_INVALID, "%s: q and out must be 16-byte aligned", who);
    CHECK(plan_of(p, t, n, max_draft, n_heads, 0, who, plan, keys, bytes));
    CHECK(ws_check(ws, ws_bytes, bytes, who));
    CHECK(apart(q, out, n * max_draft * n_heads * p.hd, who));
    LkPagedAttn a{};
    a.p = p;
    a.t = t;
    a.q = q;
    a.out = out;
    a.slots = slots;
    a.ctx = ctx_len;
    a.draft = n_draft;
    a.mask = mask;
    a.n = (uint32_t)n;
    a.tokens = (uint32_t)max_draft;
    a.n_heads = (uint32_t)n_heads;
    a.G = (uint32_t)(n_heads / p.n_kv);
    return launched(lk_paged_attn_launch(a, plan, ws, (hipStream_t)stream), who);
}

static int sparse_check(const LkPages& p, size_t take, size_t first, size_t last, const char* who) {
    if (take == 0 || take > 0x7FFFFFFF || first > take || last > take - first)
        return fail(LKHIP_E_INVALID, "%s: %zu first and %zu last pages of %zu taken ones", who, first, last, take);
    return LKHIP_OK;
}

extern "C" int lkhip_sparse_attn_workspace(const lkhip_kv_pages* pages, const lkhip_page_table* table, size_t n,
                                           size_t n_heads, size_t n_take, size_t* bytes) {
    const char* who = "sparse_attn_workspace";
    LkPages p;
    LkTable t;
    LkPagedPlan plan;
    size_t keys;
    if (!bytes) return fail(LKHIP_E_INVALID, "%s: null argument", who);
    *bytes = 0;
    CHECK(pages_of(pages, -1, who, p));
    CHECK(table_of(table, p, 0, who, t));
    CHECK(sparse_check(p, n_take, 0, 0, who));
    if (n == 0) return LKHIP_OK;
    return plan_of(p, t, n, 1, n_heads, n_take, who, plan, keys, *bytes);
}

extern "C" int lkhip_sparse_attn(const lkhip_kv_pages* pages, const lkhip_page_table* table, uint32_t layer,
                                 const float* q, const uint32_t* slots, const uint32_t* ctx_len, const void* bounds,
                                 size_t n, size_t n_heads, size_t n_take, size_t n_first, size_t n_last,
                                 uint32_t* taken, void* ws, size_t ws_bytes, float* out, void* stream) {
    const char* who = "sparse_attn";
    LkPages p;
    LkTable t;
    LkPagedPlan plan;
    size_t keys, bytes;
    CHECK(pages_of(pages, layer, who, p));
    CHECK(table_of(table, p, 0, who, t));
    CHECK(sparse_check(p, n_take, n_first, n_last, who));
    if (n == 0) return LKHIP_OK;
    if (!q || !ctx_len || !bounds || !taken || !out) return fail(LKHIP_E_INVALID, "%s: null argument", who);
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(bounds, 16))
        return fail(LKHIP_E_INVALID, "%s: q, bounds and out must be 16-byte aligned", who);
    CHECK(plan_of(p, t, n, 1, n_heads, n_take, who, plan, keys, bytes));
    CHECK(ws_check(ws, ws_bytes, bytes, who));
    CHECK(apart(q, out, n * n_heads * p.hd, who));
    LkSparse c{};
    c.p = p;
    c.t = t;
    c.q = q;
    c.slots = slots;
    c.ctx = ctx_len;
    c.bounds = bounds;
    c.n = (uint32_t)n;
    c.n_heads = (uint32_t)n_heads;
    c.G = (uint32_t)(n_heads / p.n_kv);
    c.take = (uint32_t)n_take;
    c.first = (uint32_t)n_first;
    c.last = (uint32_t)n_last;
    c.sel = taken;
    c.keys = (uint64_t*)ws;
    CHECK(launched(lk_sparse_select_launch(c, (hipStream_t)stream), who));
    LkPagedAttn a{};
    a.p = p;
    a.t = t;
    a.q = q;
    a.out = out;
    a.slots = slots;
    a.ctx = ctx_len;
    a.n = (uint32_t)n;
    a.tokens = 1;
    a.n_heads = (uint32_t)n_heads;
    a.G = c.G;
    a.sel = taken;
    a.take = c.take;
    return launched(lk_paged_attn_launch(a, plan, (char*)ws + keys, (hipStream_t)stream), who);
}
