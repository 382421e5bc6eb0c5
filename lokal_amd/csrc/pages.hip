// pages.hip -- keeping the pages of a paged KV cache (pages.h): sharing,
// taking, giving back, filling and compacting them, and the bounds of their
// keys.  Everything that decides lies in device memory (tables, lengths,
// reference counts), so a serving loop needs no host round trip and can be
// captured; the host sees only the calls' own arguments.  Results do not
// depend on the order in which workgroups run: free pages are taken lowest
// index first, in list order; counts change by integer atomics only; a slot
// named twice in one list is taken once, at its first place.
#include "lkhip_common.h"
#include "pages.h"

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t pages_of(uint64_t positions, uint32_t pshift) {
    return (uint32_t)((positions + (1u << pshift) - 1) >> pshift);
}

// Whether list[j] == x for some j in [0, n) other than `but`: uniform over the block.
__device__ __forceinline__ bool in_list(const uint32_t* list, uint32_t n, uint32_t x, uint32_t but) {
    bool hit = false;
    for (uint32_t j = threadIdx.x; j < n; j += blockDim.x) hit |= j != but && list[j] == x;
    return __syncthreads_or(hit) != 0;
}

// ------------------------------------------------------------ fork, trim

// Bound by launch and a chain of four dependent reads: 3-4 us for 2 or 48 pairs, and
// as much for trim.  One block per pair.  A pair is refused where its rows do not exist, its
// destination holds something or appears before in the list, or its source is
// a destination of the call: every row read is one that no block writes.
__global__ __launch_bounds__(256) void pages_fork_kernel(LkPages p, LkTable t, const uint32_t* src,
                                                         const uint32_t* dst, uint32_t n, uint32_t* ok) {
    const uint32_t i = blockIdx.x, s = src[i], d = dst[i];
    const bool bad = in_list(dst, i, d, n) || in_list(dst, n, s, n);
    if (bad || s >= t.n_seq || d >= t.n_seq || t.len[d] != 0) {  // uniform
        if (threadIdx.x == 0) ok[i] = 0;
        return;
    }
    const uint32_t len = t.len[s];
    uint32_t held = pages_of(len, p.pshift);
    held = held < t.max_pages ? held : t.max_pages;
    const uint32_t* from = t.table + (size_t)s * t.max_pages;
    uint32_t* to = t.table + (size_t)d * t.max_pages;
    for (uint32_t x = threadIdx.x; x < t.max_pages; x += blockDim.x) {
        uint32_t id = LK_NO_PAGE;
        if (x < held) {
            id = from[x];
            if (id < p.n_pages) atomicAdd(t.refs + id, 1u);
        }
        to[x] = id;
    }
    __syncthreads();  // every thread has read len[d]
    if (threadIdx.x == 0) {
        t.len[d] = len;
        ok[i] = 1;
    }
}

__global__ __launch_bounds__(256) void pages_trim_kernel(LkPages p, LkTable t, const uint32_t* slots,
                                                         const uint32_t* keep, uint32_t n) {
    const uint32_t i = blockIdx.x, s = slots[i];
    if (s >= t.n_seq || in_list(slots, i, s, n)) return;  // uniform
    const uint32_t len = t.len[s], left = keep[i] < len ? keep[i] : len;
    uint32_t* row = t.table + (size_t)s * t.max_pages;
    for (uint32_t x = pages_of(left, p.pshift) + threadIdx.x; x < t.max_pages; x += blockDim.x) {
        const uint32_t id = row[x];
        if (id == LK_NO_PAGE) continue;
        if (id < p.n_pages) atomicSub(t.refs + id, 1u);
        row[x] = LK_NO_PAGE;
    }
    __syncthreads();  // every thread has read len[s]
    if (threadIdx.x == 0) t.len[s] = left;
}

// ------------------------------------------------------------------ grow

constexpr uint32_t kScan = 4;

// Exclusive sum of v over the block's threads, and the total.  part: one word per wave.
__device__ __forceinline__ uint32_t block_exclusive(uint32_t v, uint32_t* part, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6, x = lk_wave_scan(v);
    __syncthreads();  // part is free
    if (lane == 63) part[w] = x;
    __syncthreads();
    // the waves before this one: a lane each
    const uint32_t y = lk_wave_scan(lane < nw ? part[lane] : 0);
    total = __builtin_amdgcn_readlane(y, 63);
    return (w ? __builtin_amdgcn_readlane(y, w - 1) : 0) + x - v;
}

// One workgroup, entry i on thread i: what each entry needs, an exclusive sum
// over the list, then a walk over refs whose r-th free page goes to the entry
// that owns rank r.  An entry is refused (and changes nothing) where its row
// does not exist, came before, has no room, or where the free pages end
// before its last one; entries that need none are never refused for that.
// T: threads, at least n; kScan refs a thread looks at in one go.  Bound by its chain
// of reads and barriers: 6.0 us for 2 entries and a page, 8.4 for 48 and two pages each.
// One workgroup, as the order of the list decides who gets a page.
template <uint32_t T>
__global__ __launch_bounds__(T) void pages_grow_kernel(LkPages p, LkTable t, const uint32_t* slots,
                                                       const uint32_t* add, uint32_t n, uint32_t* ok,
                                                       uint32_t* copied) {
    __shared__ __align__(16) uint32_t s_slot[T];
    __shared__ uint32_t s_first[T], s_to[T], s_off[T], s_part[T / 64], s_end[T / 64];
    const uint32_t i = threadIdx.x;
    const uint32_t page = 1u << p.pshift;
    const uint32_t slot = i < n ? slots[i] : LK_NO_PAGE;
    const uint32_t more = i < n ? add[i] : 0;
    s_slot[i] = slot;
    s_to[i] = LK_NO_PAGE;
    __syncthreads();
    bool valid = slot < t.n_seq;
    for (uint32_t j = 0; j < n; j += 4) {  // no way out early: reads follow each other
        const u4 x = *(const u4*)(s_slot + j);
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) valid &= x[e] != slot || j + e >= i;
    }
    uint32_t old = LK_NO_PAGE, need = 0;
    uint64_t now = 0;
    if (valid) {
        const uint32_t len = t.len[slot];
        now = (uint64_t)len + more;
        const uint64_t want = (now + page - 1) >> p.pshift;
        const uint32_t held = pages_of(len, p.pshift);
        valid = now <= 0xFFFFFFFFull && want <= t.max_pages;
        if (valid) {
            if (more && (len & (page - 1))) {  // the last page is written on: its own copy, if it is shared
                const uint32_t id = t.table[(size_t)slot * t.max_pages + held - 1];
                if (id < p.n_pages && t.refs[id] > 1) old = id;
            }
            const uint32_t first = held - (old != LK_NO_PAGE);
            s_first[i] = first;
            need = want > first ? (uint32_t)want - first : 0;
        }
    }
    // The sum in two halves of 32 bits, as a need is below 2^27 + 1; what passes 32 bits together is more than there can
    // be free.
    uint32_t total_lo, total_hi;
    const uint32_t off_lo = block_exclusive(need & 0xFFFF, s_part, total_lo), off_hi = block_exclusive(need >> 16, s_part, total_hi);
    auto whole = [](uint32_t hi, uint32_t lo) {
        const uint64_t x = ((uint64_t)hi << 16) + lo;
        return x < 0xFFFFFFFFull ? (uint32_t)x : 0xFFFFFFFFu;
    };
    const uint32_t off = whole(off_hi, off_lo), total = whole(total_hi, total_lo);
    s_off[i] = off;
    // how many of the `total` pages there are
    uint32_t n_free = 0;
    for (uint32_t x0 = 0; x0 < p.n_pages && n_free < total; x0 += T * kScan) {  // below 2^31 + T * kScan
        uint32_t c = 0, all;
#pragma unroll
        for (uint32_t k = 0; k < kScan; k++) {
            const uint32_t x = x0 + i * kScan + k;
            c += x < p.n_pages && t.refs[x] == 0;
        }
        (void)block_exclusive(c, s_part, all);
        n_free += all;
    }
    const bool grows = valid && (need == 0 || (uint64_t)off + need <= n_free);
    // the ranks that are given out end with the last entry that takes any
    uint32_t end = grows && need ? off + need : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t y = __shfl_xor(end, d, 64);
        end = y > end ? y : end;
    }
    if ((i & 63) == 0) s_end[i >> 6] = end;
    __syncthreads();
    for (uint32_t k = 0; k < T / 64; k++) end = s_end[k] > end ? s_end[k] : end;
    uint32_t rank = 0;
    for (uint32_t x0 = 0; x0 < p.n_pages && rank < end; x0 += T * kScan) {
        uint32_t c = 0, all;
        bool is_free[kScan];
#pragma unroll
        for (uint32_t k = 0; k < kScan; k++) {
            const uint32_t x = x0 + i * kScan + k;
            is_free[k] = x < p.n_pages && t.refs[x] == 0;
            c += is_free[k];
        }
        uint32_t r = rank + block_exclusive(c, s_part, all);
#pragma unroll
        for (uint32_t k = 0; k < kScan; k++) {
            if (!is_free[k]) continue;
            if (r < end) {
                // the entry e with off[e] <= r < off[e + 1]: the last one with off <= r, as entries that need none share
                // their offset with the one behind them
                uint32_t lo = 0, hi = T;
                while (hi - lo > 1) {
                    const uint32_t mid = (lo + hi) / 2;
                    if (s_off[mid] <= r) lo = mid;
                    else hi = mid;
                }
                const uint32_t id = x0 + i * kScan + k, k0 = r - s_off[lo];
                t.table[(size_t)s_slot[lo] * t.max_pages + s_first[lo] + k0] = id;
                t.refs[id] = 1;  // read by this thread alone in this walk
                if (k0 == 0) s_to[lo] = id;
            }
            r++;
        }
        rank += all;
    }
    __syncthreads();
    if (i >= n) return;
    ok[i] = grows;
    const bool copies = grows && old != LK_NO_PAGE;
    copied[2 * i] = copies ? old : LK_NO_PAGE;
    copied[2 * i + 1] = copies ? s_to[i] : LK_NO_PAGE;
    if (grows) t.len[slot] = (uint32_t)now;
    if (copies) atomicSub(t.refs + old, 1u);
}

// The rows that a copied last page held, in every layer: block = (entry, layer, kv head and K or V).  Bound by memory:
// 48 pages of up to 64 rows in 22 layers (69 MB read and written) 16.4 us, 4.2 TB/s.
__global__ __launch_bounds__(256) void pages_copy_kernel(LkPages p, LkTable t, const uint32_t* slots,
                                                         const uint32_t* add, const uint32_t* copied) {
    const uint32_t i = blockIdx.x, src = copied[2 * i], dst = copied[2 * i + 1];
    if (src >= p.n_pages || dst >= p.n_pages) return;  // nothing to copy
    const uint32_t rows = (t.len[slots[i]] - add[i]) & ((1u << p.pshift) - 1);
    const uint64_t base = blockIdx.y * p.layer_stride + (blockIdx.z >> 1) * p.head_stride;
    const uint32_t es = p.f32 ? 4 : 2;
    char* pool = (char*)(blockIdx.z & 1 ? p.v : p.k);
    const uint4* from = (const uint4*)(pool + (base + src * p.page_stride) * es);
    uint4* to = (uint4*)(pool + (base + dst * p.page_stride) * es);
    const uint32_t words = rows * p.hd * es / 16;
    for (uint32_t x = threadIdx.x; x < words; x += 256) to[x] = from[x];
}

// ----------------------------------------------------------------- write

// A thread takes 8 values of a row: 32 bytes in, 16 (f16) or 32 (f32) out.  Bound by memory: 4096 rows of 1024 to f16
// (50 MB) 9.8 us, 5.1 TB/s.
__global__ __launch_bounds__(256) void pages_write_kernel(LkPages p, LkTable t, const float* k, const float* v,
                                                          uint32_t ld, const uint32_t* slots, const uint32_t* pos,
                                                          uint32_t n_rows) {
    const uint32_t per = p.n_kv * p.hd / 8;
    const uint32_t u = blockIdx.x * 256 + threadIdx.x;  // the host keeps n_rows * per below 2^31
    const uint32_t r = u / per, c = u % per * 8;
    if (r >= n_rows) return;
    const uint32_t s = slots[r], x = pos[r], pg = x >> p.pshift;
    if (s >= t.n_seq || pg >= t.max_pages) return;
    const uint32_t id = t.table[(size_t)s * t.max_pages + pg];
    if (id >= p.n_pages) return;
    const uint32_t h = c / p.hd, d = c % p.hd;
    const uint64_t at = id * p.page_stride + h * p.head_stride + (uint64_t)(x & ((1u << p.pshift) - 1)) * p.hd + d;
    const float4* from = (const float4*)((blockIdx.y ? v : k) + (size_t)r * ld + c);
    const float4 a = from[0], b = from[1];
    void* pool = blockIdx.y ? p.v : p.k;
    if (p.f32) {
        float4* to = (float4*)((float*)pool + at);
        to[0] = a;
        to[1] = b;
    } else {
        const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
            o[e] = (uint32_t)__half_as_ushort(__float2half_rn(f[2 * e])) |
                   (uint32_t)__half_as_ushort(__float2half_rn(f[2 * e + 1])) << 16;
        *(uint4*)((uint16_t*)pool + at) = uint4{o[0], o[1], o[2], o[3]};
    }
}

// --------------------------------------------------------------- compact

// A block takes 256 columns of 16 bytes (of all layers, kv heads, K and V) of one entry, and its accepted rows 64 at a
// time: a lane each finds where the rows lie, then every thread moves its column of eight rows at a time, all loads
// before the stores.  As the places increase (path[j] > path[j - 1], so path[j] >= j), a row is never needed after its
// place was written: what is written last, place j, lies before every row that is read later.  (A thread that walks
// the path by itself: 8.9 us for 64 paths of up to 9 rows in 24 layers; so 4.8, half of it launch and the places.)
constexpr uint32_t kMove = 8;
__global__ __launch_bounds__(256) void pages_compact_kernel(LkPages p, LkTable t, const uint32_t* slots,
                                                            const uint32_t* from, const uint32_t* path,
                                                            uint32_t ld_path, const uint32_t* n_path, uint32_t n) {
    __shared__ uint64_t s_from[64], s_to[64];  // elements within a layer's kv head; ~0: not moved
    __shared__ uint32_t s_rows;
    const uint32_t i = blockIdx.y, s = slots[i];
    const uint64_t c0 = from[i];
    uint32_t count = n_path[i];
    count = count < ld_path ? count : ld_path;
    if (s >= t.n_seq || in_list(slots, i, s, n)) return;  // uniform
    const uint32_t es = p.f32 ? 4 : 2, cols = p.hd * es / 16;
    const uint32_t u = blockIdx.x * 256 + threadIdx.x;
    const uint32_t col = u % cols, hv = u / cols % (2 * p.n_kv), layer = u / cols / (2 * p.n_kv);
    char* const pool = (char*)(hv & 1 ? p.v : p.k) + (layer * p.layer_stride + (hv >> 1) * p.head_stride) * es + col * 16;
    const uint32_t* row = t.table + (size_t)s * t.max_pages;
    const uint32_t* mine = path + (size_t)i * ld_path;
    auto place = [&](uint64_t x) -> uint64_t {
        const uint64_t pg = x >> p.pshift;
        const uint32_t id = pg < t.max_pages ? row[pg] : LK_NO_PAGE;
        return id < p.n_pages ? id * p.page_stride + (x & ((1u << p.pshift) - 1)) * p.hd : ~0ull;
    };
    for (uint32_t j0 = 0; j0 < count; j0 += 64) {
        if (threadIdx.x < 64) {
            const uint32_t j = j0 + threadIdx.x;
            const bool in = j < count;
            const uint32_t at = in ? mine[j] : 0, before = in && j ? mine[j - 1] : 0;
            const uint64_t stop = __ballot(!in || (j && at <= before));  // not increasing: the path ends here
            const uint64_t a = place(c0 + at), b = place(c0 + j);
            s_from[threadIdx.x] = b == ~0ull || a == b ? ~0ull : a;
            s_to[threadIdx.x] = b;
            if (threadIdx.x == 0) s_rows = stop ? __builtin_ctzll(stop) : 64;
        }
        __syncthreads();
        const uint32_t rows = s_rows;
        if (layer < p.n_layers) {
            for (uint32_t j = 0; j < rows; j += kMove) {
                u4 r[kMove];  // a vector type, not the uint4 struct: held in registers
#pragma unroll
                for (uint32_t e = 0; e < kMove; e++)
                    if (j + e < rows && s_from[j + e] != ~0ull) r[e] = *(const u4*)(pool + s_from[j + e] * es);
#pragma unroll
                for (uint32_t e = 0; e < kMove; e++)
                    if (j + e < rows && s_from[j + e] != ~0ull) *(u4*)(pool + s_to[j + e] * es) = r[e];
            }
        }
        if (rows < 64) return;  // uniform: the last of the path
        __syncthreads();
    }
}

// ---------------------------------------------------------------- bounds

// min / max that keep a NaN: a page with one is always worth a look
__device__ __forceinline__ float lower(float a, float b) { return (b < a || b != b) ? b : a; }
__device__ __forceinline__ float upper(float a, float b) { return (b > a || b != b) ? b : a; }

// Block = (entry, kv head); its pages blockIdx.z, + gridDim.z, ...  A lane holds
// E values of a row (16 bytes), L lanes a row, the block 256 / L rows at once.  Bound by launch and its chain of reads
// where a step touches one page a sequence (5.4 us for 32 x 8 pages).
template <typename KV, int HD>
__global__ __launch_bounds__(256) void page_bounds_kernel(LkPages p, LkTable t, const uint32_t* slots,
                                                          const uint32_t* from, const uint32_t* to, KV* bounds) {
    constexpr int E = 16 / sizeof(KV), L = HD / E, R = 256 / L;
    __shared__ float s_lo[4][HD], s_hi[4][HD];
    const uint32_t i = blockIdx.x, h = blockIdx.y, s = slots ? slots[i] : i;
    if (s >= t.n_seq) return;  // uniform
    const uint32_t page = 1u << p.pshift;
    const uint64_t cap = (uint64_t)t.max_pages << p.pshift;
    const uint64_t a = from[i], b = to[i] < cap ? to[i] : cap;
    if (a >= b) return;
    const uint32_t r0 = threadIdx.x / L, c = threadIdx.x % L, w = threadIdx.x >> 6;
    for (uint64_t pg = (a >> p.pshift) + blockIdx.z; pg <= (b - 1) >> p.pshift; pg += gridDim.z) {
        const uint32_t id = t.table[(size_t)s * t.max_pages + pg];
        if (id >= p.n_pages) continue;  // uniform
        const uint64_t left = b - (pg << p.pshift);
        const uint32_t rows = left < page ? (uint32_t)left : page;
        const KV* k = (const KV*)p.k + id * p.page_stride + h * p.head_stride + c * E;
        float lo[E], hi[E];
#pragma unroll
        for (int e = 0; e < E; e++) lo[e] = INFINITY, hi[e] = -INFINITY;
        for (uint32_t r = r0; r < rows; r += R) {
            const uint4 x = *(const uint4*)(k + (size_t)r * HD);
            const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < E; e++) {
                float f;
                if constexpr (sizeof(KV) == 4) f = __uint_as_float(xw[e]);
                else f = lk_h2f((uint16_t)(xw[e / 2] >> (16 * (e & 1))));
                lo[e] = lower(lo[e], f);
                hi[e] = upper(hi[e], f);
            }
        }
        // rows of a wave, then of the four waves
#pragma unroll
        for (int d = L; d < 64; d *= 2)
#pragma unroll
            for (int e = 0; e < E; e++) {
                lo[e] = lower(lo[e], __shfl_xor(lo[e], d, 64));
                hi[e] = upper(hi[e], __shfl_xor(hi[e], d, 64));
            }
        __syncthreads();  // the last page's values are read
        if ((threadIdx.x & 63) < L)
#pragma unroll
            for (int e = 0; e < E; e++) s_lo[w][c * E + e] = lo[e], s_hi[w][c * E + e] = hi[e];
        __syncthreads();
        if (threadIdx.x < 2 * HD) {
            const uint32_t d = threadIdx.x % HD, top = threadIdx.x / HD;
            float f = top ? s_hi[0][d] : s_lo[0][d];
#pragma unroll
            for (int k2 = 1; k2 < 4; k2++) f = top ? upper(f, s_hi[k2][d]) : lower(f, s_lo[k2][d]);
            const size_t at = (((size_t)id * p.n_kv + h) * 2 + top) * HD + d;
            if constexpr (sizeof(KV) == 4) bounds[at] = f;
            else bounds[at] = __half_as_ushort(__float2half_rn(f));  // exact: it was an f16
        }
    }
}

}  // namespace

hipError_t lk_pages_fork_launch(const LkPages& p, const LkTable& t, const uint32_t* src, const uint32_t* dst,
                                uint32_t n, uint32_t* ok, hipStream_t st) {
    hipLaunchKernelGGL(pages_fork_kernel, dim3(n), dim3(256), 0, st, p, t, src, dst, n, ok);
    return hipGetLastError();
}
hipError_t lk_pages_grow_launch(const LkPages& p, const LkTable& t, const uint32_t* slots, const uint32_t* add,
                                uint32_t n, uint32_t* ok, uint32_t* copied, hipStream_t st) {
    // a short list over few pages: fewer waves to wait for
    if (n <= 256 && p.n_pages <= 8192)
        hipLaunchKernelGGL((pages_grow_kernel<256>), dim3(1), dim3(256), 0, st, p, t, slots, add, n, ok, copied);
    else
        hipLaunchKernelGGL((pages_grow_kernel<1024>), dim3(1), dim3(1024), 0, st, p, t, slots, add, n, ok, copied);
    hipLaunchKernelGGL(pages_copy_kernel, dim3(n, p.n_layers, 2 * p.n_kv), dim3(256), 0, st, p, t, slots, add, copied);
    return hipGetLastError();
}
hipError_t lk_pages_trim_launch(const LkPages& p, const LkTable& t, const uint32_t* slots, const uint32_t* keep,
                                uint32_t n, hipStream_t st) {
    hipLaunchKernelGGL(pages_trim_kernel, dim3(n), dim3(256), 0, st, p, t, slots, keep, n);
    return hipGetLastError();
}
hipError_t lk_pages_write_launch(const LkPages& p, const LkTable& t, const float* k, const float* v, uint32_t ld,
                                 const uint32_t* slots, const uint32_t* pos, uint32_t n_rows, hipStream_t st) {
    const uint64_t units = (uint64_t)n_rows * (p.n_kv * p.hd / 8);
    hipLaunchKernelGGL(pages_write_kernel, dim3((uint32_t)((units + 255) / 256), 2), dim3(256), 0, st, p, t, k, v, ld,
                       slots, pos, n_rows);
    return hipGetLastError();
}
hipError_t lk_pages_compact_launch(const LkPages& p, const LkTable& t, const uint32_t* slots, const uint32_t* from,
                                   const uint32_t* path, uint32_t ld_path, const uint32_t* n_path, uint32_t n,
                                   hipStream_t st) {
    const uint32_t units = p.n_layers * 2 * p.n_kv * (p.hd * (p.f32 ? 4 : 2) / 16);
    hipLaunchKernelGGL(pages_compact_kernel, dim3((units + 255) / 256, n), dim3(256), 0, st, p, t, slots, from, path,
                       ld_path, n_path, n);
    return hipGetLastError();
}
hipError_t lk_page_bounds_launch(const LkPages& p, const LkTable& t, const uint32_t* slots, const uint32_t* from,
                                 const uint32_t* to, uint32_t n, void* bounds, hipStream_t st) {
    // enough blocks for long prompts, few idle ones where each entry has one page
    uint32_t z = 1024 / (n * p.n_kv) + 1;
    if (z > t.max_pages) z = t.max_pages;
    const dim3 grid(n, p.n_kv, z);
#define LK_BOUNDS(T, HD) \
    hipLaunchKernelGGL((page_bounds_kernel<T, HD>), grid, dim3(256), 0, st, p, t, slots, from, to, (T*)bounds)
    if (p.f32 && p.hd == 64) LK_BOUNDS(float, 64);
    else if (p.f32) LK_BOUNDS(float, 128);
    else if (p.hd == 64) LK_BOUNDS(uint16_t, 64);
    else LK_BOUNDS(uint16_t, 128);
#undef LK_BOUNDS
    return hipGetLastError();
}
