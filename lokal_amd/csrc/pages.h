// pages.h -- the paged KV cache as the kernels see it, and their launches
// (pages.hip: keeping the pages; paged_attn.hip: the attentions that read
// them).  The lkhip_pages_* / lkhip_*_attn entry points (paged_api.hip) check
// what the host can see; what lies in device memory (page ids, lengths,
// slots) is checked by the kernels: an id that names no page is a hole.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

// One layer's view, or (layer_stride, n_layers) all of them.  Row o of page p
// and kv head h starts at element p * page_stride + h * head_stride + o * hd.
struct LkPages {
    void *k, *v;
    uint32_t f32;        // element type: 1 f32, 0 f16
    uint32_t hd;         // 64 or 128
    uint32_t n_kv;
    uint32_t pshift;     // page size 1 << pshift: 16..256 positions
    uint32_t n_layers, n_pages;
    uint64_t page_stride, head_stride, layer_stride;
};
#define LK_NO_PAGE 0xFFFFFFFFu
struct LkTable {
    uint32_t* table;     // [n_seq][max_pages] page ids
    uint32_t* len;       // [n_seq] positions held
    uint32_t* refs;      // [n_pages] tables that hold the page
    uint32_t n_seq, max_pages;
};
// Entries of one fork / grow / trim / compact call: grow's single workgroup
// gives each a thread.
#define LK_PAGES_LIST_MAX 1024u

hipError_t lk_pages_fork_launch(const LkPages& p, const LkTable& t, const uint32_t* src, const uint32_t* dst,
                                uint32_t n, uint32_t* ok, hipStream_t st);
hipError_t lk_pages_grow_launch(const LkPages& p, const LkTable& t, const uint32_t* slots, const uint32_t* add,
                                uint32_t n, uint32_t* ok, uint32_t* copied, hipStream_t st);
hipError_t lk_pages_trim_launch(const LkPages& p, const LkTable& t, const uint32_t* slots, const uint32_t* keep,
                                uint32_t n, hipStream_t st);
hipError_t lk_pages_write_launch(const LkPages& p, const LkTable& t, const float* k, const float* v, uint32_t ld,
                                 const uint32_t* slots, const uint32_t* pos, uint32_t n_rows, hipStream_t st);
hipError_t lk_pages_compact_launch(const LkPages& p, const LkTable& t, const uint32_t* slots, const uint32_t* from,
                                   const uint32_t* path, uint32_t ld_path, const uint32_t* n_path, uint32_t n,
                                   hipStream_t st);
hipError_t lk_page_bounds_launch(const LkPages& p, const LkTable& t, const uint32_t* slots, const uint32_t* from,
                                 const uint32_t* to, uint32_t n, void* bounds, hipStream_t st);

// Attention over pages.  Rows of one (sequence, kv head): token-major, row
// r = token r / G, query head kvh * G + r % G.
struct LkPagedAttn {
    LkPages p;             // k / v: the layer's
    LkTable t;
    const float* q;        // [n][tokens][n_heads * hd]
    float* out;            // like q
    const uint32_t* slots; // [n] table rows, null: 0..n-1
    const uint32_t* ctx;   // [n] cached positions before the tokens
    const uint32_t* draft; // [n] tokens of each sequence; null: `tokens`
    const uint32_t* mask;  // [n][tokens][words]: bit j of a token's row: it sees token j; null: j <= its own
    uint32_t n, tokens, n_heads, G;
    // sparse: the pages read, [n][n_kv][take] page numbers of the sequence, ascending, LK_NO_PAGE behind
    const uint32_t* sel;
    uint32_t take;
    // set by the launch
    float *part_ml, *part_o;
    uint64_t* place;       // wide: steps of a run, then where each sequence's steps begin
    uint32_t chunk, unit;  // positions of a chunk: at least, and log2 of what they are a multiple of
    uint32_t n_chunks, n_rg, rows_pad;
    float scale;           // log2(e) / sqrt(hd)
};
struct LkPagedPlan {
    bool narrow;           // waves take positions in turn; else they lie side by side in rows
    uint32_t tiles, waves; // 16-row tiles of a wave, waves of a workgroup
    uint32_t chunk, unit, n_chunks, n_rg, rows_pad;
    uint64_t blocks, steps;  // steps: of all items at the table's capacity
    uint64_t place_bytes, part_rows, part_bytes;
};
// positions: the most that a sequence can show (its table's capacity; sparse: take pages)
LkPagedPlan lk_paged_plan(uint32_t hd, bool f32, bool sparse, uint32_t n, uint32_t n_kv, uint32_t rows, uint64_t positions);
hipError_t lk_paged_attn_launch(LkPagedAttn a, const LkPagedPlan& plan, void* ws, hipStream_t st);

// The pages that a sparse attention reads: scores (64-bit keys) into `keys`
// [n][n_kv][max_pages], then the choice into sel.
struct LkSparse {
    LkPages p;
    LkTable t;
    const float* q;        // [n][n_heads * hd]
    const uint32_t* slots;
    const uint32_t* ctx;
    const void* bounds;    // [n_pages][n_kv][2][hd], the cache's type
    uint32_t n, n_heads, G, take, first, last;
    uint32_t* sel;
    uint64_t* keys;
};
hipError_t lk_sparse_select_launch(const LkSparse& a, hipStream_t st);
