// page_choose.hip -- the pages that a sparse attention reads (pages.h LkSparse):
// scores of a sequence's pages from the bounds of their keys, and the choice.
#include "lkhip_common.h"
#include "pages.h"

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// A number as an unsigned key of the same order, above all where it is not finite.
__device__ __forceinline__ uint64_t order_key(double x) {
    if (!(fabs(x) < (double)INFINITY)) return ~0ull;
    const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);  // -0 as 0
    return b >> 63 ? ~b : b | 1ull << 63;
}

// score(page) = max over the kv head's query heads of sum_d max(q_d lo_d, q_d hi_d),
// which no q.k of the page exceeds; products of f32 and f16 are exact in 64 bits and
// their sums wrong by 2^-52, so that which page is taken does not hang on the order of
// a sum (f64 products run at the f32 rate here).  HD / 8 lanes take a page, E = 8
// dims each; the bounds are widened once for all heads, and the sign of q_d says which
// one a dim needs.  A page with a bound that is not finite has the highest key.
template <int N>
__device__ __forceinline__ double dpp_add(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, N, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), N, 0xF, 0xF, false);
    return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// over N = 8 or 16 neighbouring lanes: quad pairs, quad halves, the half row mirrored, the row mirrored
template <int N>
__device__ __forceinline__ double lanes_sum(double x) {
    x = dpp_add<0x141>(dpp_add<0x4E>(dpp_add<0xB1>(x)));
    return N == 16 ? dpp_add<0x140>(x) : x;
}

template <typename KV, int HD>
struct PageBounds {
    static constexpr int E = 8, W = E * sizeof(KV) / 4;  // words of a lane's lower, and of its upper bounds
    uint32_t lo[W], hi[W];
    __device__ __forceinline__ void load(const void* bounds, const LkPages& p, uint32_t id, uint32_t kvh, uint32_t c) {
        const u4* b = (const u4*)((const KV*)bounds + ((size_t)id * p.n_kv + kvh) * 2 * HD + c * E);
        const u4* t = (const u4*)((const KV*)b + HD);
#pragma unroll
        for (int w = 0; w < W / 4; w++) {
            const u4 x = b[w], y = t[w];
#pragma unroll
            for (int e = 0; e < 4; e++) lo[4 * w + e] = x[e], hi[4 * w + e] = y[e];
        }
    }
    // The bounds of dim e of the lane.
    __device__ __forceinline__ float low(int e) const {
        if constexpr (sizeof(KV) == 4) return __uint_as_float(lo[e]);
        else return lk_h2f((uint16_t)(lo[e / 2] >> (16 * (e & 1))));
    }
    __device__ __forceinline__ float high(int e) const {
        if constexpr (sizeof(KV) == 4) return __uint_as_float(hi[e]);
        else return lk_h2f((uint16_t)(hi[e / 2] >> (16 * (e & 1))));
    }
};

// AND and OR over the wave, on lane 63: as a sum by lk_wave_sum's steps (a lane without a source meets itself).
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ uint64_t dpp_bits(uint64_t x) {
    const uint32_t lo = (uint32_t)x, hi = (uint32_t)(x >> 32);
    return (uint64_t)lk_dpp_u32<CTRL, ROW_MASK>(hi, hi) << 32 | lk_dpp_u32<CTRL, ROW_MASK>(lo, lo);
}
__device__ __forceinline__ void wave_bits(uint64_t& all, uint64_t& any) {
    all &= dpp_bits<0xB1, 0xF>(all), any |= dpp_bits<0xB1, 0xF>(any);
    all &= dpp_bits<0x4E, 0xF>(all), any |= dpp_bits<0x4E, 0xF>(any);
    all &= dpp_bits<0x124, 0xF>(all), any |= dpp_bits<0x124, 0xF>(any);
    all &= dpp_bits<0x128, 0xF>(all), any |= dpp_bits<0x128, 0xF>(any);
    all &= dpp_bits<0x142, 0xA>(all), any |= dpp_bits<0x142, 0xA>(any);
    all &= dpp_bits<0x143, 0xC>(all), any |= dpp_bits<0x143, 0xC>(any);
}

// What a sequence holds, for both kernels below.
__device__ __forceinline__ uint32_t sparse_held(const LkSparse& a, uint32_t slot, uint32_t s) {
    if (slot >= a.t.n_seq) return 0;
    const uint32_t cap = a.t.max_pages << a.p.pshift, ctx = a.ctx[s] < cap ? a.ctx[s] : cap;  // < 2^31
    return (ctx + (1u << a.p.pshift) - 1) >> a.p.pshift;
}
__device__ __forceinline__ bool sparse_forced(const LkSparse& a, uint32_t x, uint32_t held) {
    return x < a.first || x + a.last >= held;
}

// Keys of pages x0, x0 + step, .. below x1 for one (sequence, kv head), by groups of HD / 8
// lanes; put(page, key) runs on one lane of the group.  s_q: kHeads x HD doubles.
constexpr uint32_t kHeads = 8;
template <typename KV, int HD, class Put>
__device__ __forceinline__ void score_pages(const LkSparse& a, uint32_t s, uint32_t slot, uint32_t kvh, uint32_t held,
                                            uint32_t x0, uint32_t x1, uint32_t step, double* s_q, Put put) {
    constexpr int E = 8, L = HD / 8;
    const uint32_t c = threadIdx.x % L;
    const uint32_t* row = a.t.table + (size_t)slot * a.t.max_pages;
    // a page's id is read two pages ahead, its bounds one
    auto id_of = [&](uint32_t x) __attribute__((always_inline)) -> uint32_t {
        return x < x1 && !sparse_forced(a, x, held) ? row[x] : LK_NO_PAGE;
    };
    for (uint32_t g0 = 0; g0 < a.G; g0 += kHeads) {
        uint32_t id = id_of(x0), id1 = id_of(x0 + step);
        PageBounds<KV, HD> b;
        b.load(a.bounds, a.p, id < a.p.n_pages ? id : 0, kvh, c);
        const uint32_t gn = a.G - g0 < kHeads ? a.G - g0 : kHeads;
        __syncthreads();  // the last heads' q is read
        const float* q = a.q + ((size_t)s * a.n_heads + kvh * a.G + g0) * HD;
        // [head][pair of a lane's dims][lane][2]: neighbouring lanes read neighbouring 16 bytes
        for (uint32_t i = threadIdx.x; i < gn * HD; i += blockDim.x)
            s_q[i / HD * HD + (i % E / 2 * L + i % HD / E) * 2 + i % 2] = q[i];
        __syncthreads();
        for (uint32_t x = x0; x < x1; x += step) {
            const PageBounds<KV, HD> now = b;
            const bool there = id < a.p.n_pages;
            id = id1;
            b.load(a.bounds, a.p, id < a.p.n_pages ? id : 0, kvh, c);
            id1 = id_of(x + 2 * step);
            if (sparse_forced(a, x, held)) continue;
            uint64_t key = 0;  // a hole: below all
            if (there) {
                double bl[E], bh[E];
                float odd = 0.f;  // NaN where a bound is not finite
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const float u = now.low(e), v = now.high(e);
                    odd = fmaf(v, 0.f, fmaf(u, 0.f, odd));
                    bl[e] = u, bh[e] = v;
                }
                double top = -(double)INFINITY, off = odd;
                for (uint32_t g = 0; g < gn; g++) {
                    double sum = off;
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const double y = s_q[g * HD + (e / 2 * L + c) * 2 + e % 2];
                        sum = fma(y, __double2hiint(y) < 0 ? bl[e] : bh[e], sum);
                    }
                    sum = lanes_sum<L>(sum);
                    top = sum > top || !(fabs(sum) < (double)INFINITY) ? sum : top;
                    off = fabs(sum) < (double)INFINITY ? off : (double)NAN;  // and stays so
                }
                key = order_key(top);
            }
            if (c == 0) put(x, key, g0 == 0);
        }
    }
}

// Scores alone, of long tables: many blocks a (sequence, kv head).
template <typename KV, int HD>
__global__ __launch_bounds__(256) void sparse_score_kernel(const LkSparse a) {
    __shared__ __align__(16) double s_q[kHeads * HD];
    const uint32_t kvh = blockIdx.y, s = blockIdx.z, slot = a.slots ? a.slots[s] : s;
    const uint32_t held = sparse_held(a, slot, s);
    if (held <= a.take) return;  // uniform: all are taken
    uint64_t* keys = a.keys + ((size_t)s * a.p.n_kv + kvh) * a.t.max_pages;
    score_pages<KV, HD>(a, s, slot, kvh, held, blockIdx.x * (2048 / HD) + threadIdx.x / (HD / 8), held, gridDim.x * (2048 / HD), s_q,
                        [&](uint32_t x, uint64_t k, bool first) { keys[x] = first || k > keys[x] ? k : keys[x]; });
}

// The choice: the want-th largest key by bins of 11 bits, from the highest bit in which
// the pages still in question differ, so that two or three rounds settle it; then the
// pages above it and the first of those at it, in order: equal keys go to the lowest
// page.  One workgroup a (sequence, kv head); FUSED: it takes the scores itself and
// keeps the keys in LDS.  (A thread that walks 256 bins eight times: 62-78 us.)
constexpr uint32_t kBins = 2048, kFusedPages = 256;
template <typename KV, int HD, bool FUSED, uint32_t kChoose>
__global__ __launch_bounds__(kChoose) void sparse_choose_kernel(const LkSparse a) {
    __shared__ uint32_t s_bin[kBins], s_part[kChoose / 64], s_find[3];
    __shared__ uint64_t s_and[kChoose / 64], s_or[kChoose / 64];
    __shared__ uint64_t s_keys[FUSED ? kFusedPages : 1];
    __shared__ __align__(16) double s_q[FUSED ? kHeads * HD : 1];
    const uint32_t kvh = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint32_t slot = a.slots ? a.slots[s] : s;
    uint32_t* sel = a.sel + ((size_t)s * a.p.n_kv + kvh) * a.take;
    const uint32_t held = sparse_held(a, slot, s);
    if (held <= a.take) {  // uniform
        for (uint32_t x = tid; x < a.take; x += kChoose) sel[x] = x < held ? x : LK_NO_PAGE;
        return;
    }
    const uint64_t* keys;
    if constexpr (FUSED) {
        score_pages<KV, HD>(a, s, slot, kvh, held, tid / (HD / 8), held, kChoose / (HD / 8), s_q,
                            [&](uint32_t x, uint64_t k, bool first) { s_keys[x] = first || k > s_keys[x] ? k : s_keys[x]; });
        keys = s_keys;
        __syncthreads();
    } else {
        keys = a.keys + ((size_t)s * a.p.n_kv + kvh) * a.t.max_pages;
    }
    // sum of v over the threads before this one, and over all
    auto scan = [&](uint32_t v, uint32_t& all) {
        const uint32_t x = lk_wave_scan(v);
        __syncthreads();
        if (lane == 63) s_part[w] = x;
        __syncthreads();
        uint32_t before = 0;
        all = 0;
#pragma unroll
        for (uint32_t k = 0; k < kChoose / 64; k++) {
            const uint32_t y = s_part[k];
            before += k < w ? y : 0;
            all += y;
        }
        return before + x - v;
    };
    const uint32_t others = a.take - a.first - a.last;  // first + last <= take < held
    uint32_t want = others, shift = 63;
    uint64_t prefix = 0;  // pages in question: key >> shift >> 1 == prefix (shift 63: all)
    bool any = others > 0;
    auto asked = [&](uint32_t x, uint64_t k) { return !sparse_forced(a, x, held) && (k >> shift >> 1) == prefix; };
    while (any) {  // at most 6 rounds of 11 bits
        uint64_t all1 = ~0ull, any1 = 0;
        for (uint32_t x = tid; x < held; x += kChoose) {
            const uint64_t k = keys[x];
            if (asked(x, k)) all1 &= k, any1 |= k;
        }
        wave_bits(all1, any1);
        __syncthreads();
        if (lane == 63) s_and[w] = all1, s_or[w] = any1;
        for (uint32_t b = tid; b < kBins; b += kChoose) s_bin[b] = 0;
        __syncthreads();
        all1 = s_and[0], any1 = s_or[0];
#pragma unroll
        for (uint32_t k = 1; k < kChoose / 64; k++) all1 &= s_and[k], any1 |= s_or[k];
        const uint64_t differ = all1 ^ any1;
        if (!differ) {  // all in question are equal
            shift = 0;
            prefix = any1;
            break;
        }
        const uint32_t top = 63 - __clzll((long long)differ), sh = top > 10 ? top - 10 : 0;
        for (uint32_t x = tid; x < held; x += kChoose) {
            const uint64_t k = keys[x];
            if (asked(x, k)) atomicAdd(&s_bin[(uint32_t)(k >> sh) & (kBins - 1)], 1u);
        }
        __syncthreads();
        // thread t holds OF neighbouring bins, counted from the top
        constexpr uint32_t OF = kBins / kChoose;
        uint32_t c[OF], sum = 0, total;
#pragma unroll
        for (uint32_t k = 0; k < OF; k++) c[k] = s_bin[kBins - 1 - OF * tid - k], sum += c[k];
        uint32_t above = scan(sum, total);
        if (above < want && above + sum >= want) {  // one thread
#pragma unroll
            for (uint32_t k = 0; k < OF; k++) {
                if (above < want && above + c[k] >= want) {
                    s_find[0] = kBins - 1 - OF * tid - k;
                    s_find[1] = above;
                    s_find[2] = c[k];
                }
                above += c[k];
            }
        }
        __syncthreads();
        const uint32_t bin = s_find[0], count = s_find[2];
        want -= s_find[1];
        prefix = (any1 >> sh & ~(uint64_t)(kBins - 1)) | bin;  // bits above the bins are common
        // from here on in question: key >> sh == prefix
        any = count != want && sh > 0;
        shift = sh ? sh - 1 : 0;
        if (!any) {
            shift = sh;
            break;
        }
        __syncthreads();
    }
    // taken: key >> shift above prefix, and the first `want` of those at it
    uint32_t out = 0, equal = 0;
    for (uint32_t x0 = 0; x0 < held; x0 += kChoose) {
        const uint32_t x = x0 + tid;
        const bool in = x < held, f = in && sparse_forced(a, x, held);
        const uint64_t k = in && !f && others ? keys[x] >> shift : 0;
        const bool mine = in && !f && others, same = mine && k == prefix;
        uint32_t n_same, n_take;
        const uint32_t e = equal + scan(same, n_same);
        const bool takes = f || (mine && k > prefix) || (same && e < want);
        const uint32_t at = out + scan(takes, n_take);
        if (takes && at < a.take) sel[at] = x;
        equal += n_same;
        out += n_take;
    }
}

}  // namespace

template <typename KV, int HD>
static void select_launch(const LkSparse& a, hipStream_t st) {
    const dim3 pairs(a.p.n_kv, a.n);
    if (a.t.max_pages <= kFusedPages) {
        hipLaunchKernelGGL((sparse_choose_kernel<KV, HD, true, 256>), pairs, dim3(256), 0, st, a);
        return;
    }
    uint32_t blocks = 4096 / (a.n * a.p.n_kv) + 1;
    const uint32_t most = (a.t.max_pages + 2048 / HD - 1) / (2048 / HD);
    if (blocks > most) blocks = most;
    hipLaunchKernelGGL((sparse_score_kernel<KV, HD>), dim3(blocks, a.p.n_kv, a.n), dim3(256), 0, st, a);
    if (a.t.max_pages <= 2048) hipLaunchKernelGGL((sparse_choose_kernel<KV, HD, false, 256>), pairs, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((sparse_choose_kernel<KV, HD, false, 1024>), pairs, dim3(1024), 0, st, a);
}
hipError_t lk_sparse_select_launch(const LkSparse& a, hipStream_t st) {
    if (a.p.f32) a.p.hd == 64 ? select_launch<float, 64>(a, st) : select_launch<float, 128>(a, st);
    else a.p.hd == 64 ? select_launch<uint16_t, 64>(a, st) : select_launch<uint16_t, 128>(a, st);
    return hipGetLastError();
}
