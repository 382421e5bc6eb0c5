// paged_attn.hip -- attention over a paged KV cache (pages.h): several drafted
// tokens of a sequence at once, each seeing the cached context and what a bit
// mask lets it see of the draft; and one token over chosen pages.
//
//   o = sum_x 2^(s_x - m) v_x / sum_x 2^(s_x - m),  s_x = log2(e) q.k_x / sqrt(hd)
//
// over the positions x that the row sees, in one pass with running m and sum.
// All T * G rows of a kv head (T tokens, G query heads) share its K and V.
//
// A wave takes RT tiles of 16 rows over tiles of 64 (f32 cache: 32) positions;
// WR waves of a workgroup lie side by side in rows, the others take positions
// in turn, and the workgroup one chunk of positions.  Both products run on the
// matrix cores:
//   scores S[position][row] = K Q^T: K rows straight from memory as the first
//     operand (lane: position lane & 15, 8 dims), Q as the second;
//   O[row][dim] += P V: S's lanes hold row lane & 15, positions 4 (lane >> 4) + i
//     of each 16, which is the first operand of the second product once its k
//     index is taken as those positions; V is read with the same positions and
//     HD / 16 neighbouring dims per lane, column n of product d being dim
//     (HD / 16) n + d, so O's lanes hold neighbouring dims.
// No operand goes through LDS.  q carries log2(e) / sqrt(hd).  f16 cache: K and V
// are exact operands; q (scaled per row by a power of two, so that its largest value is in 2^13..2^14) and P
// are each split into two f16 parts (22 bits), as one part alone is off by
// 1.4e-4.  f32 cache: 16x16x4 f32 products.
// The running maximum lags: it moves when some score passes it by 8 (in log2),
// so most tiles neither reduce over lanes nor rescale O; P stays below 2^8.
//
// Positions that no row sees (behind the draft, in holes of the table) are
// clamped to readable rows; their scores become -inf and their V zero, so what
// lies there -- NaN too -- does not matter.  A draft position whose V is not
// finite would reach the rows that do not see it as 0 * NaN: such a tile takes
// its V with those values zeroed and then marks (row, dim) pairs that do see one.
//
// A chunk's rows go out as (m, sum, O) and paged_fold_kernel joins them; where a
// sequence has one chunk its workgroup writes the output itself.
#include "lkhip_common.h"
#include "pages.h"

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

constexpr float kLag = 8.f;  // log2: how far a score may pass the running maximum

__device__ __forceinline__ h8 bits_h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(h8, u4{a, b, c, d});
}
__device__ __forceinline__ bool half_not_finite(uint32_t w) {  // either half of w
    return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u;
}
// w with its non-finite halves as 1.0 and the others 0 (mark), or as 0 and the others kept (clean)
__device__ __forceinline__ uint32_t half_mark(uint32_t w) {
    return ((w & 0x7C00u) == 0x7C00u ? 0x3C00u : 0u) | ((w & 0x7C000000u) == 0x7C000000u ? 0x3C000000u : 0u);
}
__device__ __forceinline__ uint32_t half_clean(uint32_t w) {
    return ((w & 0x7C00u) == 0x7C00u ? 0u : w & 0xFFFFu) | ((w & 0x7C000000u) == 0x7C000000u ? 0u : w & 0xFFFF0000u);
}
__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7F800000u) == 0x7F800000u; }

// What a sequence shows: table row, context and drafted tokens, positions in all.
struct Seq {
    uint32_t slot, ctx, rows, total;
    bool live;
};
template <bool SPARSE>
__device__ __forceinline__ Seq seq_of(const LkPagedAttn& a, uint32_t s) {
    Seq q;
    q.slot = a.slots ? a.slots[s] : s;
    q.live = q.slot < a.t.n_seq;
    const uint32_t cap = a.t.max_pages << a.p.pshift;  // < 2^31
    const uint32_t ctx = a.ctx[s];
    q.ctx = ctx < cap ? ctx : cap;
    if constexpr (SPARSE) {
        q.rows = 1;
        // positions of the chosen pages, counted page by page
        const uint32_t held = (q.ctx + (1u << a.p.pshift) - 1) >> a.p.pshift;
        q.total = (held < a.take ? held : a.take) << a.p.pshift;
    } else {
        const uint32_t d = a.draft ? a.draft[s] : a.tokens;
        q.rows = d < a.tokens ? d : a.tokens;
        const uint32_t all = q.ctx + q.rows;
        q.total = all < cap ? all : cap;
    }
    return q;
}
__device__ __forceinline__ uint32_t chunks_of(uint32_t total, uint32_t chunk) {
    const uint32_t c = (total + chunk - 1) / chunk;
    return c ? c : 1;
}

template <int HD, bool F32, int RT, int WR, bool SPARSE>
__global__ __launch_bounds__(256) void paged_attn_kernel(const LkPagedAttn a) {
    constexpr int WP = 4 / WR;           // waves that share a row group's positions
    constexpr int NT = F32 ? 2 : 4;      // 16-position tiles of a step
    constexpr int ND = HD / 16;          // column tiles of O, neighbouring dims of a lane
    constexpr int KS = HD / 32;          // f16 score products of a tile
    constexpr int ROWS = WR * RT * 16;   // rows of the workgroup
    __shared__ float s_m[WP][ROWS], s_l[WP][ROWS];
    __shared__ __align__(16) float s_o[WP > 1 ? ROWS : 1][WP > 1 ? HD + 4 : 1];

    // Row groups of one (sequence, kv head, chunk) read the same K and V: they run
    // on one XCD (workgroups go round the 8), one after the other.
    const uint32_t xcd = blockIdx.x & 7, turn = blockIdx.x >> 3;
    const uint32_t rg = turn % a.n_rg, item = turn / a.n_rg * 8 + xcd;
    if (item >= a.n * a.p.n_kv * a.n_chunks) return;
    const uint32_t chunk = item % a.n_chunks, pair = item / a.n_chunks, kvh = pair % a.p.n_kv, s = pair / a.p.n_kv;
    const Seq sq = seq_of<SPARSE>(a, s);
    const uint32_t R = sq.rows * a.G, row0 = rg * ROWS;
    const uint32_t x0 = chunk * a.chunk;
    if (!sq.live || row0 >= R || (x0 >= sq.total && chunk)) return;  // uniform
    const uint32_t nch = chunks_of(sq.total, a.chunk);
    const uint32_t x1 = x0 + a.chunk < sq.total ? x0 + a.chunk : sq.total;

    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wr = (uint32_t)w % WR, wp = (uint32_t)w / WR;
    const uint32_t j = (uint32_t)lane >> 4, c16 = (uint32_t)lane & 15;
    const uint32_t rbase = row0 + wr * (RT * 16);
    const uint32_t pmask = (1u << a.p.pshift) - 1;
    const uint32_t* trow = a.t.table + (size_t)sq.slot * a.t.max_pages;
    const uint32_t* sel = SPARSE ? a.sel + ((size_t)s * a.p.n_kv + kvh) * a.take : nullptr;
    const uint64_t hoff = kvh * a.p.head_stride;

    // ---- this lane's row of each tile: q and its score factor
    h8 qh[F32 ? 1 : RT][F32 ? 1 : KS], ql[F32 ? 1 : RT][F32 ? 1 : KS];
    f4 qf[F32 ? RT : 1][F32 ? ND : 1];
    float fac[RT];
    uint32_t tok[RT];
    float m[RT], l[RT];
    f4 o[RT][ND];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const uint32_t row = rbase + rt * 16 + c16;
        const bool live = row < R;
        tok[rt] = live ? row / a.G : 0;
        const uint32_t g = live ? row % a.G : 0;
        const float* q = a.q + (((size_t)s * a.tokens + tok[rt]) * a.n_heads + kvh * a.G + g) * HD;
        m[rt] = -INFINITY;
        l[rt] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; d++) o[rt][d] = f4{0.f, 0.f, 0.f, 0.f};
        if constexpr (F32) {
            fac[rt] = 1.f;
#pragma unroll
            for (int b = 0; b < ND; b++) {  // dims 16 b + 4 j + e
                const float4 x = *(const float4*)(q + 16 * b + 4 * j);
                qf[rt][b] = live ? f4{x.x, x.y, x.z, x.w} * a.scale : f4{0.f, 0.f, 0.f, 0.f};
            }
        } else {
            float x[KS][8], top = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {  // dims 32 ks + 8 j + e
                const float4 u = *(const float4*)(q + 32 * ks + 8 * j), v = *(const float4*)(q + 32 * ks + 8 * j + 4);
                const float y[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    x[ks][e] = live ? y[e] * a.scale : 0.f;
                    top = fmaxf(top, fabsf(x[ks][e]));
                }
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            int up = 0;
            if (top > 0.f && top < INFINITY) {
                up = 13 - (int)((__float_as_uint(top) >> 23) & 255) + 127;
                up = up > 100 ? 100 : up;  // subnormal rows
            }
            fac[rt] = ldexpf(1.f, -up);
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float y = ldexpf(x[ks][e], up);
                    const _Float16 hi = (_Float16)y;
                    qh[rt][ks][e] = hi;
                    ql[rt][ks][e] = (_Float16)(y - (float)hi);
                }
        }
    }

    if (rbase < R) {  // wave-uniform
        for (uint32_t x = x0 + wp * (NT * 16); x < x1; x += WP * (NT * 16)) {
            // ---- where the step's 16-position tiles lie
            uint64_t base[NT];   // element of the tile's first row
            uint32_t pos[NT];    // its position in the sequence
            bool hole[NT];
            bool masked = false;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const uint32_t y = x + 16 * t;
                uint32_t pg = y >> a.p.pshift;
                hole[t] = y >= sq.total;
                if constexpr (SPARSE) {
                    pg = hole[t] ? LK_NO_PAGE : sel[pg];
                    hole[t] = pg >= a.t.max_pages;
                }
                const uint32_t id = hole[t] ? LK_NO_PAGE : trow[pg];
                hole[t] = id >= a.p.n_pages;
                pos[t] = hole[t] ? 0 : (pg << a.p.pshift) + (y & pmask);
                base[t] = (hole[t] ? 0 : id * a.p.page_stride + (uint64_t)(y & pmask) * HD) + hoff;
                masked |= hole[t] || pos[t] + 16 > sq.ctx;
            }
            masked = __builtin_amdgcn_readfirstlane(masked);
            // in a masked step: which of the lane's positions (4 j + i of tile t) no row sees
            uint32_t unseen = 0;
            if (masked) {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t y = pos[t] + 4 * j + i;
                        if (hole[t] || y >= (SPARSE ? sq.ctx : sq.total)) unseen |= 1u << (4 * t + i);
                    }
            }
            auto hide = [&](int rt, int t, int i, float v) -> float {
                bool see = !(unseen >> (4 * t + i) & 1);
                if constexpr (!SPARSE) {
                    const uint32_t y = pos[t] + 4 * j + i;
                    if (see && y >= sq.ctx) {
                        const uint32_t d = y - sq.ctx;
                        if (a.mask) {
                            const uint32_t words = (a.tokens + 31) / 32;
                            see = a.mask[((size_t)s * a.tokens + tok[rt]) * words + (d >> 5)] >> (d & 31) & 1;
                        } else {
                            see = d <= tok[rt];
                        }
                    }
                }
                return see ? v : -INFINITY;
            };
            // the running maximum and sum of tile rt's rows; sc becomes the weights
            auto weigh = [&](int rt, f4(&sc)[NT]) {
                if (masked) {
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) sc[t][i] = hide(rt, t, i, sc[t][i]);
                }
                float top = -INFINITY;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) top = fmaxf(top, sc[t][i]);
                top *= fac[rt];  // fac > 0
                if (__any(top > m[rt] + kLag)) {
                    top = fmaxf(top, __shfl_xor(top, 16, 64));
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const float mn = fmaxf(m[rt], top);
                    const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[rt] - mn);
                    m[rt] = mn;
                    l[rt] *= f;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float fi = __shfl(f, (int)(4 * j + i), 64);  // O's rows are 4 j + i
#pragma unroll
                        for (int d = 0; d < ND; d++) o[rt][d][i] *= fi;
                    }
                }
                const float ms = m[rt] == -INFINITY ? 0.f : m[rt];  // no score yet: weights of 0
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(sc[t][i], fac[rt], -ms));
                        sc[t][i] = p;
                        l[rt] += p;
                    }
            };
            if constexpr (F32) {
                const float *K = (const float*)a.p.k, *V = (const float*)a.p.v;
                f4 sc[RT][NT];
#pragma unroll
                for (int t = 0; t < NT; t++) {
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) sc[rt][t] = f4{0.f, 0.f, 0.f, 0.f};
                    const float* k = K + base[t] + (size_t)c16 * HD + 4 * j;
#pragma unroll
                    for (int b = 0; b < ND; b++) {
                        const f4 kk = *(const f4*)(k + 16 * b);
#pragma unroll
                        for (int e = 0; e < 4; e++)
#pragma unroll
                            for (int rt = 0; rt < RT; rt++)
                                sc[rt][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[e], qf[rt][b][e], sc[rt][t], 0, 0, 0);
                    }
                }
#pragma unroll
                for (int rt = 0; rt < RT; rt++) weigh(rt, sc[rt]);
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const f4* v = (const f4*)(V + base[t] + (size_t)(4 * j + i) * HD + ND * c16);
                        f4 vv[ND / 4];
#pragma unroll
                        for (int d = 0; d < ND / 4; d++) vv[d] = v[d];
                        bool odd = false;
                        if (masked) {
                            if (unseen >> (4 * t + i) & 1)
#pragma unroll
                                for (int d = 0; d < ND / 4; d++) vv[d] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int d = 0; d < ND; d++) odd |= not_finite(vv[d / 4][d % 4]);
                            odd = !SPARSE && __any(odd);
                        }
                        if (odd) {
#pragma unroll
                            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                                for (int d = 0; d < ND; d++) {
                                    const float y = vv[d / 4][d % 4];
                                    const float sees = hide(rt, t, i, 0.f) == 0.f ? 1.f : 0.f;
                                    f4 c = __builtin_amdgcn_mfma_f32_16x16x4f32(sees, not_finite(y) ? 1.f : 0.f,
                                                                                f4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                                    for (int e = 0; e < 4; e++)
                                        if (c[e] > 0.f) o[rt][d][e] = NAN;
                                }
#pragma unroll
                            for (int d = 0; d < ND; d++)
                                if (not_finite(vv[d / 4][d % 4])) vv[d / 4][d % 4] = 0.f;
                        }
#pragma unroll
                        for (int rt = 0; rt < RT; rt++)
#pragma unroll
                            for (int d = 0; d < ND; d++)
                                o[rt][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(sc[rt][t][i], vv[d / 4][d % 4], o[rt][d],
                                                                                0, 0, 0);
                    }
            } else {
                const uint16_t *K = (const uint16_t*)a.p.k, *V = (const uint16_t*)a.p.v;
                u4 kr[NT][KS];
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int ks = 0; ks < KS; ks++)
                        kr[t][ks] = *(const u4*)(K + base[t] + (size_t)c16 * HD + 32 * ks + 8 * j);
                uint32_t vr[NT][4][ND / 2];  // dims ND c16 .. of position 4 j + i
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint16_t* v = V + base[t] + (size_t)(4 * j + i) * HD + ND * c16;
                        if constexpr (ND == 4) {
                            const u2 y = *(const u2*)v;
                            vr[t][i][0] = y[0], vr[t][i][1] = y[1];
                        } else {
                            const u4 y = *(const u4*)v;
                            vr[t][i][0] = y[0], vr[t][i][1] = y[1], vr[t][i][2] = y[2], vr[t][i][3] = y[3];
                        }
                    }
                bool odd = false;
                if (masked) {
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int d = 0; d < ND / 2; d++) {
                                if (unseen >> (4 * t + i) & 1) vr[t][i][d] = 0;
                                odd |= half_not_finite(vr[t][i][d]);
                            }
                    odd = !SPARSE && __any(odd);
                }
                // operand of column tile d over tiles 2 g, 2 g + 1: halves d of eight positions
                auto column = [&](const uint32_t(&y)[NT][4][ND / 2], int g, int d) -> h8 {
                    const uint32_t sel2 = (d & 1) ? 0x07060302u : 0x05040100u;
                    uint32_t r[4];
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int i = 0; i < 2; i++)
                            r[2 * t + i] = __builtin_amdgcn_perm(y[2 * g + t][2 * i + 1][d / 2], y[2 * g + t][2 * i][d / 2],
                                                                 sel2);
                    return bits_h8(r[0], r[1], r[2], r[3]);
                };
                if (odd) {
                    uint32_t bad[NT][4][ND / 2];
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int d = 0; d < ND / 2; d++) bad[t][i][d] = half_mark(vr[t][i][d]);
                    // which rows see a marked position (a weight that underflowed to 0 counts: 0 * NaN)
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
#pragma unroll
                        for (int g = 0; g < NT / 2; g++) {
                            h8 sees;
#pragma unroll
                            for (int t = 0; t < 2; t++)
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    sees[4 * t + i] = hide(rt, 2 * g + t, i, 0.f) == 0.f ? (_Float16)1.f : (_Float16)0.f;
#pragma unroll
                            for (int d = 0; d < ND; d++) {
                                const f4 c = __builtin_amdgcn_mfma_f32_16x16x32_f16(sees, column(bad, g, d),
                                                                                    f4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    if (c[e] > 0.f) o[rt][d][e] = NAN;
                            }
                        }
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int d = 0; d < ND / 2; d++) vr[t][i][d] = half_clean(vr[t][i][d]);
                }
                h8 vb[NT / 2][ND];
#pragma unroll
                for (int g = 0; g < NT / 2; g++)
#pragma unroll
                    for (int d = 0; d < ND; d++) vb[g][d] = column(vr, g, d);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    f4 sc[NT];
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        f4 c = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int ks = 0; ks < KS; ks++) {
                            const h8 kk = __builtin_bit_cast(h8, kr[t][ks]);
                            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, qh[rt][ks], c, 0, 0, 0);
                            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, ql[rt][ks], c, 0, 0, 0);
                        }
                        sc[t] = c;
                    }
                    weigh(rt, sc);
#pragma unroll
                    for (int g = 0; g < NT / 2; g++) {
                        h8 ph, pl;
#pragma unroll
                        for (int t = 0; t < 2; t++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const float p = sc[2 * g + t][i];
                                const _Float16 hi = (_Float16)p;
                                ph[4 * t + i] = hi;
                                pl[4 * t + i] = (_Float16)(p - (float)hi);
                            }
#pragma unroll
                        for (int d = 0; d < ND; d++) {
                            o[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, vb[g][d], o[rt][d], 0, 0, 0);
                            o[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, vb[g][d], o[rt][d], 0, 0, 0);
                        }
                    }
                }
            }
        }
    }

    // ---- the waves of a row group join: m and sum per row, then O one wave after the other
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        l[rt] += __shfl_xor(l[rt], 16, 64);
        l[rt] += __shfl_xor(l[rt], 32, 64);
        if (j == 0) {
            s_m[wp][wr * (RT * 16) + rt * 16 + c16] = m[rt];
            s_l[wp][wr * (RT * 16) + rt * 16 + c16] = l[rt];
        }
    }
    __syncthreads();
    const size_t pbase = ((size_t)pair * a.n_chunks + chunk) * a.rows_pad + row0;
    for (int turn2 = 0; turn2 < WP; turn2++) {
        if ((int)wp == turn2) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t lr = wr * (RT * 16) + rt * 16 + 4 * j + i, row = row0 + lr;
                    float top = -INFINITY, sum = 0.f;
#pragma unroll
                    for (int k = 0; k < WP; k++) top = fmaxf(top, s_m[k][lr]);
                    const float ms = top == -INFINITY ? 0.f : top;
#pragma unroll
                    for (int k = 0; k < WP; k++) sum += s_l[k][lr] * __builtin_amdgcn_exp2f(s_m[k][lr] - ms);
                    const float f = __builtin_amdgcn_exp2f(s_m[wp][lr] - ms);  // 0 for a wave that saw nothing
                    float y[ND];
#pragma unroll
                    for (int d = 0; d < ND; d++) y[d] = o[rt][d][i] * f;
                    if constexpr (WP > 1) {
                        float* acc = &s_o[lr][ND * c16];
                        if (turn2 > 0)
#pragma unroll
                            for (int d = 0; d < ND; d++) y[d] += acc[d];
                        if (turn2 < WP - 1) {
#pragma unroll
                            for (int d = 0; d < ND; d++) acc[d] = y[d];
                            continue;
                        }
                    }
                    if (row >= R) continue;
                    float* to;
                    if (nch == 1) {
                        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing: zeros
#pragma unroll
                        for (int d = 0; d < ND; d++) y[d] *= inv;
                        to = a.out + (((size_t)s * a.tokens + row / a.G) * a.n_heads + kvh * a.G + row % a.G) * HD;
                    } else {
                        if (c16 == 0) *(float2*)(a.part_ml + 2 * (pbase + lr)) = float2{top, sum};
                        to = a.part_o + (pbase + lr) * HD;
                    }
#pragma unroll
                    for (int d = 0; d < ND; d += 4) *(f4*)(to + ND * c16 + d) = f4{y[d], y[d + 1], y[d + 2], y[d + 3]};
                }
        }
        if (turn2 < WP - 1) __syncthreads();
    }
}

// Chunks of a row, joined: HD / 4 lanes a row.
template <int HD, bool SPARSE>
__global__ __launch_bounds__(256) void paged_fold_kernel(const LkPagedAttn a) {
    constexpr uint32_t L = HD / 4;
    const uint32_t pair = blockIdx.x, kvh = pair % a.p.n_kv, s = pair / a.p.n_kv;
    const Seq sq = seq_of<SPARSE>(a, s);
    const uint32_t nch = chunks_of(sq.total, a.chunk);
    const uint32_t row = blockIdx.y * (256 / L) + threadIdx.x / L, c = threadIdx.x % L;
    if (!sq.live || nch == 1 || row >= sq.rows * a.G) return;
    const size_t base = (size_t)pair * a.n_chunks * a.rows_pad + row;
    float top = -INFINITY;
    for (uint32_t k = 0; k < nch; k++) top = fmaxf(top, a.part_ml[2 * (base + (size_t)k * a.rows_pad)]);
    const float ms = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f4 y = f4{0.f, 0.f, 0.f, 0.f};
    for (uint32_t k = 0; k < nch; k++) {
        const size_t at = base + (size_t)k * a.rows_pad;
        const float2 ml = *(const float2*)(a.part_ml + 2 * at);
        const float f = __builtin_amdgcn_exp2f(ml.x - ms);
        sum = fmaf(ml.y, f, sum);
        y += *(const f4*)(a.part_o + at * HD + 4 * c) * f;
    }
    y *= sum == 0.f ? 0.f : 1.f / sum;
    *(f4*)(a.out + (((size_t)s * a.tokens + row / a.G) * a.n_heads + kvh * a.G + row % a.G) * HD + 4 * c) = y;
}

// ------------------------------------------------------------ choosing pages

// A number as an unsigned key of the same order, NaN above all.
__device__ __forceinline__ uint64_t order_key(double x) {
    if (x != x) return ~0ull;
    const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);  // -0 as 0
    return b >> 63 ? ~b : b | 1ull << 63;
}

// score(page) = max over the kv head's query heads of sum_d max(q_d lo_d, q_d hi_d),
// which no q.k of the page exceeds; products of f32 and f16 are exact in 64 bits and
// their sums wrong by 2^-52, so that which page is taken does not hang on the order of
// a sum.  A group of 8 lanes takes a page, HD / 8 dims each.
template <typename KV, int HD>
__global__ __launch_bounds__(256) void sparse_score_kernel(const LkSparse a) {
    constexpr int E = HD / 8;
    const uint32_t kvh = blockIdx.y, s = blockIdx.z;
    const uint32_t slot = a.slots ? a.slots[s] : s;
    if (slot >= a.t.n_seq) return;
    const uint64_t cap = (uint64_t)a.t.max_pages << a.p.pshift;
    const uint64_t ctx = a.ctx[s] < cap ? a.ctx[s] : cap;
    const uint32_t held = (uint32_t)((ctx + (1u << a.p.pshift) - 1) >> a.p.pshift);
    if (held <= a.take) return;  // all are taken
    const uint32_t pg = blockIdx.x * 32 + threadIdx.x / 8, c = threadIdx.x % 8;
    if (pg >= held) return;  // whole groups of 8
    uint64_t key = ~0ull;
    if (pg >= a.first && pg + a.last < held) {
        const uint32_t id = a.t.table[(size_t)slot * a.t.max_pages + pg];
        key = 0;
        if (id < a.p.n_pages) {
            const KV* lo = (const KV*)a.bounds + (((size_t)id * a.p.n_kv + kvh) * 2) * HD + c * E;
            const KV* hi = lo + HD;
            double bl[E], bh[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                if constexpr (sizeof(KV) == 4) bl[e] = lo[e], bh[e] = hi[e];
                else bl[e] = lk_h2f(lo[e]), bh[e] = lk_h2f(hi[e]);
            }
            const float* q = a.q + ((size_t)s * a.n_heads + kvh * a.G) * HD + c * E;
            for (uint32_t g = 0; g < a.G; g++) {
                double sum = 0;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const double y = q[(size_t)g * HD + e];
                    sum = fma(y, y > 0 ? bh[e] : bl[e], sum);
                }
#pragma unroll
                for (int d = 1; d < 8; d *= 2) sum += __shfl_xor(sum, d, 64);
                const uint64_t k = order_key(sum);
                key = k > key ? k : key;
            }
        }
    }
    if (c == 0) a.keys[((size_t)s * a.p.n_kv + kvh) * a.t.max_pages + pg] = key;
}

// The `take` largest keys, equal ones by lowest page: the take-th largest key by its
// digits of 8 bits from the top (a histogram of the pages that agree so far), then the
// pages above it and the first of those at it, in order.  First and last pages have
// the highest key and a NaN score has it too, so it is looked at beside them.
constexpr uint32_t kSelect = 256;
__global__ __launch_bounds__(kSelect) void sparse_select_kernel(const LkSparse a) {
    __shared__ uint32_t hist[256], s_part[kSelect / 64], s_digit, s_above;
    const uint32_t kvh = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const uint32_t slot = a.slots ? a.slots[s] : s;
    uint32_t* sel = a.sel + ((size_t)s * a.p.n_kv + kvh) * a.take;
    const uint64_t cap = (uint64_t)a.t.max_pages << a.p.pshift;
    const uint64_t ctx = slot < a.t.n_seq ? (a.ctx[s] < cap ? a.ctx[s] : cap) : 0;
    const uint32_t held = (uint32_t)((ctx + (1u << a.p.pshift) - 1) >> a.p.pshift);
    if (held <= a.take) {  // uniform
        for (uint32_t x = tid; x < a.take; x += kSelect) sel[x] = x < held ? x : LK_NO_PAGE;
        return;
    }
    const uint64_t* keys = a.keys + ((size_t)s * a.p.n_kv + kvh) * a.t.max_pages;
    auto forced = [&](uint32_t x) { return x < a.first || x + a.last >= held; };
    // first + last <= take (host): what is left for the others
    const uint32_t want0 = a.take - a.first - a.last;
    uint32_t want = want0;  // of the pages that agree with `prefix` so far
    uint64_t prefix = 0, known = 0;
    for (int shift = 56; shift >= 0 && want; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        for (uint32_t x = tid; x < held; x += kSelect)
            if (!forced(x) && (keys[x] & known) == prefix) atomicAdd(&hist[keys[x] >> shift & 255], 1u);
        __syncthreads();
        if (tid == 0) {
            uint32_t above = 0;
            int d = 255;
            while (d > 0 && above + hist[d] < want) above += hist[d--];
            s_digit = d;
            s_above = above;
        }
        __syncthreads();
        prefix |= (uint64_t)s_digit << shift;
        known |= 255ull << shift;
        want -= s_above;
        __syncthreads();
    }
    // pages above `prefix`, and the first `want` of those equal to it
    uint32_t out = 0, equal = 0;
    for (uint32_t x0 = 0; x0 < held; x0 += kSelect) {
        const uint32_t x = x0 + tid;
        const bool in = x < held, f = in && forced(x);
        const uint64_t k = in ? keys[x] : 0;
        const bool same = in && !f && want0 && k == prefix;
        auto place = [&](bool v, uint32_t& all) {
            const uint64_t b = __ballot(v);
            __syncthreads();
            if ((tid & 63) == 0) s_part[tid >> 6] = __popcll(b);
            __syncthreads();
            uint32_t before = __popcll(b & ((1ull << (tid & 63)) - 1));
            all = 0;
            for (uint32_t i = 0; i < kSelect / 64; i++) {
                if (i < tid >> 6) before += s_part[i];
                all += s_part[i];
            }
            return before;
        };
        uint32_t n_same, n_take;
        const uint32_t e = equal + place(same, n_same);
        const bool takes = f || (in && want0 && k > prefix) || (same && e < want);
        const uint32_t at = out + place(takes, n_take);
        if (takes && at < a.take) sel[at] = x;
        equal += n_same;
        out += n_take;
    }
}

}  // namespace

LkPagedPlan lk_paged_plan(uint32_t hd, bool f32, bool sparse, uint32_t n, uint32_t n_kv, uint32_t rows,
                          uint64_t positions) {
    LkPagedPlan p{};
    p.rt = sparse || rows <= 16 ? 1 : rows <= 32 || hd == 128 || f32 ? 2 : 4;
    const uint32_t per = p.rt * 16;
    p.wr = sparse ? 1 : rows > 2 * per ? 4 : rows > per ? 2 : 1;
    p.n_rg = (rows + p.wr * per - 1) / (p.wr * per);
    p.rows_pad = p.n_rg * p.wr * per;
    const uint64_t base = (uint64_t)n * n_kv * p.n_rg;
    const uint32_t step = 64 * (4 / p.wr);  // every wave has a step
    const uint64_t steps = (positions + step - 1) / step;
    uint64_t c = (1024 + base - 1) / base;
    c = c > 64 ? 64 : c;
    c = c > steps ? steps : c;
    if (c < 1) c = 1;
    p.chunk = (uint32_t)((steps + c - 1) / c * step);
    if (!p.chunk) p.chunk = step;
    p.n_chunks = (uint32_t)((positions + p.chunk - 1) / p.chunk);
    if (!p.n_chunks) p.n_chunks = 1;
    const uint64_t items = (uint64_t)n * n_kv * p.n_chunks;
    p.blocks = (items + 7) / 8 * 8 * p.n_rg;
    p.part_bytes = p.n_chunks > 1 ? items * p.rows_pad * (hd + 2) * 4 : 0;
    return p;
}

template <int HD, bool F32, bool SPARSE>
static hipError_t launch(const LkPagedAttn& a, const LkPagedPlan& p, hipStream_t st) {
    const dim3 grid((uint32_t)p.blocks);
#define LK_PAGED(RT, WR) \
    hipLaunchKernelGGL((paged_attn_kernel<HD, F32, RT, WR, SPARSE>), grid, dim3(256), 0, st, a)
    constexpr int TOP = HD == 64 && !F32 ? 4 : 2;
    if constexpr (SPARSE) {
        if (p.rt != 1 || p.wr != 1) return hipErrorInvalidValue;
        LK_PAGED(1, 1);
    } else if (p.rt == 1 && p.wr == 1) LK_PAGED(1, 1);
    else if (p.rt == 2 && p.wr == 1) LK_PAGED(2, 1);
    else if (p.rt == TOP && p.wr == 1) LK_PAGED(TOP, 1);
    else if (p.rt == TOP && p.wr == 2) LK_PAGED(TOP, 2);
    else if (p.rt == TOP && p.wr == 4) LK_PAGED(TOP, 4);
    else return hipErrorInvalidValue;
#undef LK_PAGED
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.n_chunks == 1) return e;
    const uint32_t rows = a.tokens * a.G, per = 256 / (HD / 4);
    hipLaunchKernelGGL((paged_fold_kernel<HD, SPARSE>), dim3(a.n * a.p.n_kv, (rows + per - 1) / per), dim3(256), 0, st,
                       a);
    return hipGetLastError();
}

hipError_t lk_paged_attn_launch(LkPagedAttn a, const LkPagedPlan& p, void* ws, hipStream_t st) {
    a.chunk = p.chunk;
    a.n_chunks = p.n_chunks;
    a.n_rg = p.n_rg;
    a.rows_pad = p.rows_pad;
    a.scale = 1.44269504088896340736f * (a.p.hd == 64 ? 0.125f : 0.08838834764831845f);
    if (p.n_chunks > 1) {
        a.part_o = (float*)ws;
        a.part_ml = a.part_o + (size_t)a.n * a.p.n_kv * p.n_chunks * p.rows_pad * a.p.hd;
    }
#define LK_PAGED(HD, F32) (a.sel ? launch<HD, F32, true>(a, p, st) : launch<HD, F32, false>(a, p, st))
    if (a.p.hd == 64) return a.p.f32 ? LK_PAGED(64, true) : LK_PAGED(64, false);
    return a.p.f32 ? LK_PAGED(128, true) : LK_PAGED(128, false);
#undef LK_PAGED
}

hipError_t lk_sparse_select_launch(const LkSparse& a, hipStream_t st) {
    const dim3 grid((a.t.max_pages + 31) / 32, a.p.n_kv, a.n);
    if (a.t.max_pages > a.take) {
        if (a.p.f32 && a.p.hd == 64) hipLaunchKernelGGL((sparse_score_kernel<float, 64>), grid, dim3(256), 0, st, a);
        else if (a.p.f32) hipLaunchKernelGGL((sparse_score_kernel<float, 128>), grid, dim3(256), 0, st, a);
        else if (a.p.hd == 64) hipLaunchKernelGGL((sparse_score_kernel<uint16_t, 64>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((sparse_score_kernel<uint16_t, 128>), grid, dim3(256), 0, st, a);
    }
    hipLaunchKernelGGL(sparse_select_kernel, dim3(a.p.n_kv, a.n), dim3(kSelect), 0, st, a);
    return hipGetLastError();
}
