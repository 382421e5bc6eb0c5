// paged_attn.hip -- attention over a paged KV cache (pages.h): several drafted
// tokens of a sequence at once, each seeing the cached context and what a bit
// mask lets it see of the draft; and one token over chosen pages.
//
//   o = sum_x 2^(s_x - m) v_x / sum_x 2^(s_x - m),  s_x = log2(e) q.k_x / sqrt(hd)
//
// over the positions x that the row sees, in one pass with running m and sum.
// All T * G rows of a kv head (T tokens, G query heads) share its K and V.
//
// A wave takes RT tiles of 16 rows over steps of NT tiles of 16 positions.  Both
// products run on the matrix cores:
//   scores S[position][row] = K Q^T: K rows are the first operand (lane: position
//     lane & 15, 8 dims), Q the second;
//   O[row][dim] += P V: S's lanes hold row lane & 15, positions 4 (lane >> 4) + i
//     of each 16, which is the first operand of the second product once its k
//     index is taken as those positions; V is read with the same positions and
//     neighbouring dims per lane, so O's lanes hold neighbouring dims.
// q carries log2(e) / sqrt(hd).  f16 cache: K and V are exact operands; q (scaled
// per row by a power of two where its values need it) and P are each split into two
// f16 parts (22 bits), as one part alone is off by 1.4e-4.  f32 cache: 16x16x4 f32
// products up to 32 rows; more rows split K and V into two f16 parts too and take
// three of the four products (76 -> 64 us for 3 x 23 tokens when it came).
// The running maximum lags: it moves when some score passes it by 6 (in log2),
// so most steps neither reduce over lanes nor rescale O; f16 parts of P are
// held 2^9 times and stay below 2^15, sums and O alike.
//
// Two kernels.  Up to 32 rows (narrow): the four waves of a workgroup take steps in
// turn, K and V go straight from memory to registers, and the waves join at the end.
// More rows (wide): the waves lie side by side in rows and share each step's K and V
// through LDS, a ring of stages that loads write without registers.
//
// Positions that no row sees (behind the draft, in holes of the table) are clamped
// to readable rows; their scores become -inf and their V zero, so what lies there
// -- NaN too -- does not matter.  A draft position whose V is not finite would
// reach the rows that do not see it as 0 * NaN: such a step takes its V with those
// values zeroed and then marks the (row, dim) pairs that do see one.
//
// A chunk's rows go out as (m, sum, O) and paged_fold_kernel joins them; where a
// sequence has one chunk its workgroup writes the output itself.
#include "lkhip_common.h"
#include "pages.h"

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 hf2 __attribute__((ext_vector_type(2)));
typedef float fl2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

#define LK_INLINE __attribute__((always_inline))  // lambdas too: what they capture stays in registers
constexpr float kLag = 6.f;  // log2: how far a score may pass the running maximum
// Weights are held 2^kUp times: with kLag below 2^15, and small ones keep bits in f16, whose steps end at 2^-24.  (At
// once their size, 4096 weights of 2^-17 beside one of 1 were off by 2^-25 each, all to one side: 1.2e-4 of the sum.)
constexpr float kUp = 9.f;
constexpr uint32_t kMaxChunks = 64;

__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7F800000u) == 0x7F800000u; }
// bits 15 and 31: whether that half of w is not finite
__device__ __forceinline__ uint32_t halves_not_finite(uint32_t w) {
    return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
}
__device__ __forceinline__ uint64_t low_bits(int64_t n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }

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
// A sequence's chunks: as many as the table's capacity has (a short one is spread as wide), each of a.chunk
// positions at least, in whole steps of the workgroup.  (Chunks of the capacity's size: 17.0 us for one token over 4000
// positions where the table has room for 65536, here 10.3.)
struct Chunks {
    uint32_t size, count;
};
__device__ __forceinline__ Chunks chunks_of(const LkPagedAttn& a, uint32_t total) {
    const uint32_t units = (total + (1u << a.unit) - 1) >> a.unit, even = (units + a.n_chunks - 1) / a.n_chunks << a.unit;
    const uint32_t size = even > a.chunk ? even : a.chunk, count = (total + size - 1) / size;
    return Chunks{size, count ? count : 1};
}

// A workgroup's share: some of the positions of a (sequence, kv head), and one group of its rows.
struct Share {
    uint32_t s, kvh, row0, R, x0, x1;
    Seq sq;
    bool live;
    bool whole;   // all of the rows' positions: the output can be written
    size_t part;  // else: where the first row's part goes
};
// The narrow kernel's: one chunk.  Row groups of one chunk read the same K and V: they run on one XCD (workgroups go
// round the 8), one after the other.
template <bool SPARSE>
__device__ __forceinline__ Share share_of(const LkPagedAttn& a, uint32_t rows) {
    Share h{};
    const uint32_t xcd = blockIdx.x & 7, turn = blockIdx.x >> 3;
    const uint32_t rg = turn % a.n_rg, item = turn / a.n_rg * 8 + xcd;
    if (item >= a.n * a.p.n_kv * a.n_chunks) return h;
    const uint32_t pair = item / a.n_chunks;
    const uint32_t chunk = (item % a.n_chunks + pair) % a.n_chunks;  // short sequences lack the same chunks: not the same XCDs'
    h.kvh = pair % a.p.n_kv;
    h.s = pair / a.p.n_kv;
    h.sq = seq_of<SPARSE>(a, h.s);
    h.R = h.sq.rows * a.G;
    h.row0 = rg * rows;
    const Chunks of = chunks_of(a, h.sq.total);
    h.x0 = chunk * of.size;
    h.live = h.sq.live && h.row0 < h.R && chunk < of.count;
    h.whole = of.count == 1;
    h.part = ((size_t)pair * a.n_chunks + chunk) * a.rows_pad + h.row0;
    h.x1 = h.x0 + of.size < h.sq.total ? h.x0 + of.size : h.sq.total;
    return h;
}

// A tile's page id (LK_NO_PAGE or above: a hole) and the sequence position of its first row; y: its place among the
// positions shown, a multiple of 16.
template <bool SPARSE>
__device__ __forceinline__ uint32_t tile_page(const LkPagedAttn& a, const Share& h, uint32_t y, uint32_t& pos) {
    uint32_t pg = y >> a.p.pshift;
    bool hole = y >= h.sq.total;
    if constexpr (SPARSE) {
        pg = hole ? LK_NO_PAGE : a.sel[((size_t)h.s * a.p.n_kv + h.kvh) * a.take + pg];
        hole = pg >= a.t.max_pages;
    }
    pos = hole ? 0x7FFFFFF0u : (pg << a.p.pshift) + (y & ((1u << a.p.pshift) - 1));
    return hole ? LK_NO_PAGE : a.t.table[(size_t)h.sq.slot * a.t.max_pages + pg];
}
// element of the tile's first row, in the clamped place of a hole
__device__ __forceinline__ uint64_t tile_base(const LkPagedAttn& a, const Share& h, uint32_t id, uint32_t y, int hd) {
    return (id < a.p.n_pages ? id * a.p.page_stride + (uint64_t)(y & ((1u << a.p.pshift) - 1)) * hd : 0) +
           h.kvh * a.p.head_stride;
}

// Dim d (0..HD / 16 - 1) of lane column c16 in the second product.  TR: V comes through LDS's transposing reads.
template <int HD, bool F32, bool TR>
__device__ __forceinline__ constexpr uint32_t dim_of(uint32_t c16, int d) {
    return TR ? 16 * d + c16 : F32 ? (d / 4) * 64 + 4 * c16 + d % 4 : HD / 16 * c16 + d;
}

// A wave's RT tiles of 16 rows: their queries, running maxima and sums, and O.
template <int HD, bool F32, int RT, int NT, bool SPARSE, bool TR>
struct Rows {
    static constexpr int ND = HD / 16, KS = F32 ? ND : HD / 32, ES = F32 ? 4 : 2;
    static constexpr int VW = ND * ES / 4;  // words of a lane's dims of one V row
    static constexpr float UP = F32 ? 0.f : kUp;  // weights in f32 need none
    h8 qh[F32 ? 1 : RT][F32 ? 1 : KS], ql[F32 ? 1 : RT][F32 ? 1 : KS];
    f4 qf[F32 ? RT : 1][F32 ? ND : 1];
    float m[RT];     // log2: what row c16's weights are relative to; -inf before its first score
    float l[RT];     // lane's part of row c16's sum: on the adders, which round; the matrix cores' long sums drift
    uint32_t tok[RT];
    f4 o[RT][ND];
    int up[RT];      // q was taken times 2^up: 0 for rows whose largest value needs no scaling
    uint32_t j, c16;
    using Scores = f4[RT][NT];

    __device__ __forceinline__ void init(const LkPagedAttn& a, const Share& h, uint32_t rbase) {
        j = (threadIdx.x & 63) >> 4, c16 = threadIdx.x & 15;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const uint32_t row = rbase + rt * 16 + c16;
            const bool live = row < h.R;
            tok[rt] = live ? row / a.G : 0;
            const uint32_t g = live ? row - tok[rt] * a.G : 0;
            const float* q = a.q + (((size_t)h.s * a.tokens + tok[rt]) * a.n_heads + h.kvh * a.G + g) * HD;
            m[rt] = -INFINITY;
            l[rt] = 0.f;
            up[rt] = 0;
#pragma unroll
            for (int d = 0; d < ND; d++) o[rt][d] = f4{0.f, 0.f, 0.f, 0.f};
            if constexpr (F32) {
#pragma unroll
                for (int b = 0; b < ND; b++) {  // dims 16 b + 4 j + e
                    const f4 x = *(const f4*)(q + 16 * b + 4 * j);
                    qf[rt][b] = live ? x * a.scale : f4{0.f, 0.f, 0.f, 0.f};
                }
            } else {
                float x[KS][8], top = 0.f;
                int by = 0;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {  // dims 32 ks + 8 j + e
                    const f4 u = *(const f4*)(q + 32 * ks + 8 * j), v = *(const f4*)(q + 32 * ks + 8 * j + 4);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[ks][e] = live ? (e < 4 ? u[e & 3] : v[e & 3]) * a.scale : 0.f;
                        top = fmaxf(top, fabsf(x[ks][e]));
                    }
                }
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                // Rows whose largest value is in [1/4, 2^14) are split as they are: the second part, down to f16's
                // 2^-24, is off by 2^-23 of it at most.  Others are brought to 2^13..2^14 first.
                if (top > 0.f && top < INFINITY && (top < 0.25f || top >= 16384.f)) {
                    by = 13 + 127 - (int)((__float_as_uint(top) >> 23) & 255);
                    by = by > 126 ? 126 : by;  // subnormal rows
#pragma unroll
                    for (int ks = 0; ks < KS; ks++)
#pragma unroll
                        for (int e = 0; e < 8; e++) x[ks][e] = ldexpf(x[ks][e], by);
                }
                up[rt] = by;
#pragma unroll
                for (int ks = 0; ks < KS; ks++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const _Float16 hi = (_Float16)x[ks][e];
                        qh[rt][ks][e] = hi;
                        ql[rt][ks][e] = (_Float16)(x[ks][e] - (float)hi);
                    }
            }
        }
    }

    static __device__ __forceinline__ void start(Scores& sc) {
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int t = 0; t < NT; t++) sc[rt][t] = f4{0.f, 0.f, 0.f, 0.f};
    }
    // k: f16 the lane's 8 dims 32 ks + 8 j of position c16, f32 its 4 dims 16 ks + 4 j.  Products that follow each other
    // belong to different sums.
    // PARTS of q: 1 where k is the second part of K itself.
    template <int PARTS = 2>
    __device__ __forceinline__ void scores(const u4 (&k)[NT], int ks, Scores& sc) const {
        if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
                        sc[rt][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f4, k[t])[e], qf[rt][ks][e], sc[rt][t], 0, 0, 0);
        } else {
#pragma unroll
            for (int part = 0; part < PARTS; part++)
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
                        sc[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, k[t]), part ? ql[rt][ks] : qh[rt][ks],
                                                                           sc[rt][t], 0, 0, 0);
        }
    }

    // What row c16 of tile rt sees of the step at x: a bit a position.  live: positions that any row may see.
    __device__ __forceinline__ uint64_t sees(const LkPagedAttn& a, const Share& h, uint32_t x, uint64_t live, int rt) const {
        if constexpr (SPARSE) return live;
        const int64_t off = (int64_t)x - h.sq.ctx;  // of the step in the draft
        uint64_t draft;
        if (a.mask) {
            const int32_t words = (int32_t)((a.tokens + 31) / 32), w0 = off >= 0 ? (int32_t)(off >> 5) : 0;
            const uint32_t* row = a.mask + ((size_t)h.s * a.tokens + tok[rt]) * words;
            const uint64_t b0 = w0 < words ? row[w0] : 0, b1 = w0 + 1 < words ? row[w0 + 1] : 0,
                           b2 = w0 + 2 < words ? row[w0 + 2] : 0;
            if (off >= 0) {
                const uint32_t sh = off & 31;
                draft = (b0 | b1 << 32) >> sh;
                if (sh) draft |= b2 << (64 - sh);
            } else {
                draft = off > -64 ? (b0 | b1 << 32) << -off : 0;
            }
        } else {
            draft = low_bits((int64_t)tok[rt] + 1 - off);
        }
        return live & (low_bits(-off) | draft);
    }
    __device__ __forceinline__ void hide(int rt, uint64_t see, Scores& sc) const {
        const uint32_t b[2] = {(uint32_t)see >> (4 * j), (uint32_t)(see >> 32) >> (4 * j)};
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) sc[rt][t][i] = b[t / 2] >> (16 * (t & 1) + i) & 1 ? sc[rt][t][i] : -INFINITY;
    }

    // Products of K times 2^k_up become scores relative to m, and UP.
    __device__ __forceinline__ void relate(Scores& sc, int k_up) const {
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const int by = -(up[rt] + k_up);  // scores of 2^126 and more are all alike
            const float f = ldexpf(1.f, by < 126 ? by : 126), z = m[rt] == -INFINITY ? 0.f : UP - m[rt];
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) sc[rt][t][i] = fmaf(sc[rt][t][i], f, z);
        }
    }
    // Before scores become weights: m moves up where one passes it by kLag.
    __device__ __forceinline__ void move(Scores& sc) {
        float top[RT];
        bool far = false;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            top[rt] = -INFINITY;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) top[rt] = fmaxf(top[rt], sc[rt][t][i]);
            far |= top[rt] > (m[rt] == -INFINITY ? -INFINITY : kLag + UP);
        }
        if (!__any(far)) return;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const bool first = m[rt] == -INFINITY;
            float x = top[rt];
            x = fmaxf(x, __shfl_xor(x, 16, 64));
            x = fmaxf(x, __shfl_xor(x, 32, 64));
            const float by = first ? (x == -INFINITY ? 0.f : x - UP) : fmaxf(x - UP, 0.f);  // how far m goes up; first: scores down
            const float f = first ? 1.f : __builtin_amdgcn_exp2f(-by);
            m[rt] = first ? x : m[rt] + by;
#pragma unroll
            for (int t = 0; t < NT; t++) sc[rt][t] -= by;
            l[rt] *= f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float fi = __shfl(f, (int)(4 * j + i), 64);  // O's rows are 4 j + i
#pragma unroll
                for (int d = 0; d < ND; d++) o[rt][d][i] *= fi;
            }
        }
    }

    // f16: the weights of tiles 2 g and 2 g + 1 in two parts, and their sums.
    __device__ __forceinline__ void weights(const Scores& sc, int g, h8 (&ph)[RT], h8 (&pl)[RT]) {
        float minus = -1.f;  // a register: p - hi is then one mixed product, hi not widened first
        asm("" : "+s"(minus));
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const fl2 p = fl2{__builtin_amdgcn_exp2f(sc[rt][2 * g + e / 2][2 * (e & 1)]),
                                  __builtin_amdgcn_exp2f(sc[rt][2 * g + e / 2][2 * (e & 1) + 1])};
                l[rt] += p[0] + p[1];
                const hf2 u = __builtin_convertvector(p, hf2);
                hi[e] = __builtin_bit_cast(uint32_t, u);
                const fl2 rest = fl2{__builtin_fmaf((float)u[0], minus, p[0]), __builtin_fmaf((float)u[1], minus, p[1])};
                lo[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, hf2));
            }
            ph[rt] = __builtin_bit_cast(h8, u4{hi[0], hi[1], hi[2], hi[3]});
            pl[rt] = __builtin_bit_cast(h8, u4{lo[0], lo[1], lo[2], lo[3]});
        }
    }
    // vb: column tiles d0.. of their V, positions 4 j + i of the one tile, then of the other.  PARTS of the weights: 1
    // where vb is V's second part.
    template <int PARTS = 2, int N>
    __device__ __forceinline__ void add16(const h8 (&ph)[RT], const h8 (&pl)[RT], const h8 (&vb)[N], int d0) {
#pragma unroll
        for (int part = 0; part < PARTS; part++)
#pragma unroll
            for (int d = 0; d < N; d++)
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
                    o[rt][d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(part ? pl[rt] : ph[rt], vb[d], o[rt][d0 + d], 0, 0, 0);
    }
    __device__ __forceinline__ void add32(const Scores& sc, int t, int i, const uint32_t (&v)[VW]) {
        float p[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            p[rt] = __builtin_amdgcn_exp2f(sc[rt][t][i]);
            l[rt] += p[rt];
        }
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
                o[rt][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[rt], __uint_as_float(v[d % VW]), o[rt][d], 0, 0, 0);
    }

    // A word of V in a masked step: what is not finite becomes zero, and odd says so.
    static __device__ __forceinline__ uint32_t clean_word(uint32_t y, uint32_t& odd) {
        if constexpr (F32) {
            const bool bad = not_finite(__uint_as_float(y));
            odd |= bad;
            return bad ? 0 : y;
        } else {
            const uint32_t bad = halves_not_finite(y);
            odd |= bad;
            return y & ~((bad >> 15) * 0xFFFFu);
        }
    }
    // V of position 4 j + i of tile t: zero where no row sees it.
    __device__ __forceinline__ uint32_t clean(int t, int i, uint64_t live, uint32_t (&v)[VW]) const {
        const bool see = live >> (16 * t + 4 * j + i) & 1;
        uint32_t odd = 0;
#pragma unroll
        for (int d = 0; d < VW; d++) {
            v[d] = see ? v[d] : 0;
            if constexpr (!SPARSE) v[d] = clean_word(v[d], odd);
        }
        return odd;
    }
    // Rows that see a value that is not finite, in a step that had something to hide: NaN in its dim.  Rare, so short: a
    // position at a time, after all steps.
    template <bool OF32>  // the cache's type
    __device__ __forceinline__ void poison(const LkPagedAttn& a, const Share& h, uint32_t x) {
        uint64_t live = 0;
        bool masked = false;
        for (uint32_t t = 0; t < NT; t++) {
            uint32_t pos;
            const uint32_t id = tile_page<SPARSE>(a, h, x + 16 * t, pos);
            const uint32_t end = SPARSE ? h.sq.ctx : h.sq.total;
            if (id < a.p.n_pages) live |= (low_bits((int64_t)end - pos) & 0xFFFF) << (16 * t);
            masked |= id >= a.p.n_pages || pos + 16 > h.sq.ctx;
        }
        if (!masked) return;
        for (uint32_t p = 0; p < NT * 16; p++) {
            if (!(live >> p & 1)) continue;  // uniform
            uint32_t pos;
            const uint32_t y = x + (p & ~15u), id = tile_page<SPARSE>(a, h, y, pos);
            const uint64_t at = tile_base(a, h, id, y, HD) + (uint64_t)(p & 15) * HD;
            uint32_t bad = 0;
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const uint64_t e = at + dim_of<HD, F32, TR>(c16, d);
                bool b;
                if constexpr (OF32) b = not_finite(((const float*)a.p.v)[e]);
                else b = (((const uint16_t*)a.p.v)[e] & 0x7C00) == 0x7C00;
                bad |= (uint32_t)b << d;
            }
            if (!__any(bad)) continue;
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                const uint32_t see = sees(a, h, x, live, rt) >> p & 1;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t hit = __shfl(see, (int)(4 * j + i), 64) ? bad : 0;
#pragma unroll
                    for (int d = 0; d < ND; d++) o[rt][d][i] = hit >> d & 1 ? NAN : o[rt][d][i];
                }
            }
        }
    }

    // Sum of row 4 j + i of tile rt, on its lanes.
    __device__ __forceinline__ float sum_of(int rt, int i) const {
        float x = l[rt];
        x += __shfl_xor(x, 16, 64);
        x += __shfl_xor(x, 32, 64);
        return __shfl(x, (int)(4 * j + i), 64);
    }
    __device__ __forceinline__ float max_of(int rt, int i) const { return __shfl(m[rt], (int)(4 * j + i), 64); }
    // Row lr of the workgroup: the output where the sequence has one chunk, else the chunk's (m, sum, O).
    __device__ __forceinline__ void put(const LkPagedAttn& a, const Share& h, uint32_t lr, float top, float sum, float (&y)[ND]) const {
        const uint32_t row = h.row0 + lr;
        if (row >= h.R) return;
        float* to;
        if (h.whole) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing: zeros
#pragma unroll
            for (int d = 0; d < ND; d++) y[d] *= inv;
            const uint32_t t = row / a.G;
            to = a.out + (((size_t)h.s * a.tokens + t) * a.n_heads + h.kvh * a.G + row - t * a.G) * HD;
        } else {
            const size_t at = h.part + lr;
            if (c16 == 0) *(float2*)(a.part_ml + 2 * at) = float2{top, sum};
            to = a.part_o + at * HD;
        }
        if constexpr (TR) {
#pragma unroll
            for (int d = 0; d < ND; d++) to[dim_of<HD, F32, TR>(c16, d)] = y[d];
        } else {
#pragma unroll
            for (int d = 0; d < ND; d += 4) *(f4*)(to + dim_of<HD, F32, TR>(c16, d)) = f4{y[d], y[d + 1], y[d + 2], y[d + 3]};
        }
    }
};

// ---------------------------------------------------------------- narrow

// Bound by memory where there is work for the card: 32 sequences x 8 kv heads x 1536 positions of 128 (201 MB) 46.9 us,
// 4.3 TB/s; below that by a chain of dependent reads (length, page id, K) and the join: 1 x 1 token over 304 positions
// 8.7 us, 4 x 2 kv heads x 4096 positions 8.1 us.  All loads of a step go out before the first product; three waves a
// SIMD (head 64) hide them better than two with a step ahead.
template <int HD, bool F32, int RT, bool SPARSE>
__global__ __launch_bounds__(256, RT == 1 && HD == 64 ? 3 : 2) void paged_narrow_kernel(const LkPagedAttn a) {
    constexpr int NT = F32 || HD == 128 ? 2 : 4, W = 4, ROWS = RT * 16, STEP = NT * 16;
    using Wave = Rows<HD, F32, RT, NT, SPARSE, false>;
    constexpr int ND = Wave::ND, KS = Wave::KS, VW = Wave::VW, ES = Wave::ES;
    __shared__ float s_m[W][ROWS], s_l[W][ROWS];
    __shared__ __align__(16) float s_o[ROWS][HD + 4];
    const Share h = share_of<SPARSE>(a, ROWS);
    if (!h.live) return;  // uniform
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Wave r;
    // a step's tiles: loads go out for all of its K and V
    auto fetch = [&](uint32_t x, u4 (&k)[NT][KS], uint32_t (&v)[NT][4][VW], uint64_t& live, bool& masked) LK_INLINE {
        const uint32_t j = (threadIdx.x & 63) >> 4, c16 = threadIdx.x & 15;
        live = 0;
        masked = false;
        const char* kb[NT];
        const char* vb[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            uint32_t pos;
            const uint32_t y = x + 16 * t, id = tile_page<SPARSE>(a, h, y, pos);
            const uint64_t base = tile_base(a, h, id, y, HD) * ES;
            kb[t] = (const char*)a.p.k + base, vb[t] = (const char*)a.p.v + base;
            const uint32_t end = SPARSE ? h.sq.ctx : h.sq.total;
            if (id < a.p.n_pages) live |= (low_bits((int64_t)end - pos) & 0xFFFF) << (16 * t);
            masked |= id >= a.p.n_pages || pos + 16 > h.sq.ctx;
        }
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                k[t][ks] = *(const u4*)(kb[t] + (c16 * HD * ES + (4 * ks + j) * 16));
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const char* row = vb[t] + (4 * j + i) * HD * ES;
#pragma unroll
                for (int d = 0; d < ND; d += 16 / ES < ND ? 16 / ES : ND) {
                    const char* at = row + dim_of<HD, F32, false>(c16, d) * ES;
                    if constexpr (VW == 2) {
                        const u2 y = *(const u2*)at;
                        v[t][i][0] = y[0], v[t][i][1] = y[1];
                    } else {
                        const u4 y = *(const u4*)at;
#pragma unroll
                        for (int e = 0; e < 4; e++) v[t][i][d * ES / 4 + e] = y[e];
                    }
                }
            }
    };
    uint32_t odd = 0;
    auto use = [&](uint32_t x, u4 (&k)[NT][KS], uint32_t (&v)[NT][4][VW], uint64_t live, bool masked) LK_INLINE {
        f4 sc[RT][NT];
        r.start(sc);
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            u4 kk[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) kk[t] = k[t][ks];
            r.scores(kk, ks, sc);
        }
        r.relate(sc, 0);
        if (__builtin_amdgcn_readfirstlane(masked)) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++) r.hide(rt, r.sees(a, h, x, live, rt), sc);
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) odd |= r.clean(t, i, live, v[t][i]);
        }
        r.move(sc);
        if constexpr (F32) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) r.add32(sc, t, i, v[t][i]);
        } else {
#pragma unroll
            for (int g = 0; g < NT / 2; g++) {
                h8 vb[ND];
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    const uint32_t pick = (d & 1) ? 0x07060302u : 0x05040100u;  // halves d of two positions
                    u4 y;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        y[e] = __builtin_amdgcn_perm(v[2 * g + e / 2][2 * (e & 1) + 1][d / 2], v[2 * g + e / 2][2 * (e & 1)][d / 2], pick);
                    vb[d] = __builtin_bit_cast(h8, y);
                }
                h8 ph[RT], pl[RT];
                r.weights(sc, g, ph, pl);
                r.add16(ph, pl, vb, 0);
            }
        }
    };
    r.init(a, h, h.row0);
    uint32_t x = h.x0 + w * STEP;
    for (; x < h.x1; x += W * STEP) {
        u4 k[NT][KS];
        uint32_t v[NT][4][VW];
        uint64_t live;
        bool masked;
        fetch(x, k, v, live, masked);
        use(x, k, v, live, masked);
    }
    if (!SPARSE && __any(odd))
        for (x = h.x0 + w * STEP; x < h.x1; x += W * STEP) r.template poison<F32>(a, h, x);
    // ---- the waves join: m and sum per row, then O one wave after the other
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float mi = r.max_of(rt, i), li = r.sum_of(rt, i);
            if (r.c16 == 0) s_m[w][rt * 16 + 4 * r.j + i] = mi, s_l[w][rt * 16 + 4 * r.j + i] = li;
        }
    __syncthreads();
    for (uint32_t turn = 0; turn < W; turn++) {
        if (w == turn) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t lr = rt * 16 + 4 * r.j + i;
                    float top = -INFINITY, sum = 0.f;
#pragma unroll
                    for (int k = 0; k < W; k++) top = fmaxf(top, s_m[k][lr]);
                    const float ms = top == -INFINITY ? 0.f : top;
#pragma unroll
                    for (int k = 0; k < W; k++) sum += s_l[k][lr] * __builtin_amdgcn_exp2f(s_m[k][lr] - ms);
                    const float f = __builtin_amdgcn_exp2f(s_m[w][lr] - ms);  // 0 for a wave that saw nothing
                    float y[ND];
#pragma unroll
                    for (int d = 0; d < ND; d++) y[d] = r.o[rt][d][i] * f;
#pragma unroll
                    for (int d = 0; d < ND; d += 4) {
                        f4* acc = (f4*)&s_o[lr][dim_of<HD, F32, false>(r.c16, d)];
                        f4 z = f4{y[d], y[d + 1], y[d + 2], y[d + 3]};
                        if (turn > 0) z += *acc;
                        if (turn < W - 1) *acc = z;
#pragma unroll
                        for (int e = 0; e < 4; e++) y[d + e] = z[e];
                    }
                    if (turn == W - 1) r.put(a, h, lr, top, sum, y);
                }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ wide

// Work of the wide kernel is counted in steps of an item: a (sequence, kv head, group of ROWS rows), all items one
// after the other, row groups of a kv head together.  How many there are is known on the device only (contexts and
// drafts differ), so a fixed number of workgroups, as many as the card holds at once, takes equal runs of steps; a run
// may end one item and begin others.  Chunks, as long as the longest sequence's, leave the card idle
// behind the shorter ones: 8 x 64 tokens over up to 32768 positions 251 us against 171.
struct Plan {
    uint32_t total, run;  // steps in all (the host keeps them below 2^32) and of a workgroup
};
// Steps of one item of a sequence, and its items.
__device__ __forceinline__ uint32_t item_steps(const Seq& q, uint32_t step) { return (q.total + step - 1) / step; }
__device__ __forceinline__ uint32_t row_groups(const LkPagedAttn& a, const Seq& q, uint32_t rows) {
    return q.live ? (q.rows * a.G + rows - 1) / rows : 0;
}
constexpr uint32_t kLeast = 2;  // steps of a run at least

// All workgroups count all sequences; `start`: where this one's run begins.  Sequences are read twice (total, then
// the place) unless one round of the threads holds them.  Workgroup 0 leaves the sequences' places for the fold.
template <int NW>
__device__ __forceinline__ Plan plan_runs(const LkPagedAttn& a, uint32_t wg, uint32_t step, uint32_t rows, uint32_t& seq,
                                          uint32_t& in_seq) {
    constexpr uint32_t T = NW * 64;
    __shared__ uint32_t s_sum[NW], s_long[NW], s_at, s_seq;
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    Plan p{};
    uint32_t longest = 0;
    auto count = [&](uint32_t s, uint32_t& steps) LK_INLINE -> uint32_t {
        steps = 0;
        if (s >= a.n) return 0;
        const Seq q = seq_of<false>(a, s);
        const uint32_t g = row_groups(a, q, rows);
        steps = g ? item_steps(q, step) : 0;
        return g * a.p.n_kv * steps;
    };
    // exclusive sum over the block, and the sum
    auto scan = [&](uint32_t v, uint32_t& all) LK_INLINE -> uint32_t {
        uint32_t x = v;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t y = __shfl_up(x, d, 64);
            if ((int)lane >= d) x += y;
        }
        __syncthreads();
        if (lane == 63) s_sum[w] = x;
        __syncthreads();
        uint32_t before = 0;
        all = 0;
#pragma unroll
        for (uint32_t k = 0; k < NW; k++) {
            if (k < w) before += s_sum[k];
            all += s_sum[k];
        }
        return before + x - v;
    };
    uint32_t mine = 0, at = 0;
    for (uint32_t s0 = 0; s0 < a.n; s0 += T) {
        uint32_t steps, all;
        mine = count(s0 + threadIdx.x, steps);
        at = p.total + scan(mine, all);
        p.total += all;
        longest = steps > longest ? steps : longest;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t y = __shfl_xor(longest, d, 64);
        longest = y > longest ? y : longest;
    }
    if (lane == 0) s_long[w] = longest;
    if (threadIdx.x == 0) s_seq = a.n;
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < NW; k++) longest = s_long[k] > longest ? s_long[k] : longest;
    // at most kMaxChunks workgroups share an item
    const uint32_t even = p.total / gridDim.x + 1, few = (longest + kMaxChunks - 3) / (kMaxChunks - 2);
    p.run = even > few ? even : few;
    p.run = p.run > kLeast ? p.run : kLeast;
    const uint64_t start = (uint64_t)wg * p.run;
    uint32_t sum = 0;
    for (uint32_t s0 = 0; s0 < a.n; s0 += T) {
        const uint32_t s = s0 + threadIdx.x;
        if (a.n > T) {
            uint32_t steps, all;
            mine = count(s, steps);
            at = sum + scan(mine, all);
            sum += all;
        }
        if (s < a.n) {
            if (wg == 0) a.place[1 + s] = at;
            if (start >= at && start - at < mine) s_seq = s, s_at = (uint32_t)(start - at);
        }
    }
    if (wg == 0 && threadIdx.x == 0) a.place[0] = p.run;
    __syncthreads();
    seq = s_seq;
    in_seq = s_at;
    return p;
}

// NW waves side by side in rows, 32 rows each, over steps of NT tiles.  K and V of a step go to LDS, RING - 1 steps
// ahead; one barrier a step.  A place there holds rows of RB bytes, whose 16-byte pieces lie at their number ^ (row &
// 7), so that eight lanes that read one piece of eight rows meet eight different bank groups.  Loads write LDS in lane
// order, so the lane that lands in a place fetches the piece that belongs there.
// f32 cache: a step lands once, each thread takes its values to registers, the next step's loads go out, and the two f16
// parts are written to a place of their own: three barriers a step.
// What bounds it.  Many rows: the matrix cores and the adders in turn (31% and 41% of their cycles): 8 x 64 tokens, 32 / 4
// heads of 64, all over 32768 positions 374 us, 736 TFLOP/s with both parts counted, 67% of a large library product's.
// Few rows: the chain of a step's landing, products and weights in a workgroup: 24 x 12 tokens, 32 / 8 heads of 128, up
// to 2048 positions 43.6 us for 132 MB; f32, 3 x 23 tokens, up to 5000 positions 44.5 us for 77 MB.
template <int HD, bool F32, int NW>
struct Wide {
    static constexpr int NT = F32 || HD == 128 ? 2 : 4, STEP = NT * 16, ROWS = NW * 32;
    static constexpr int SIDE = STEP * HD * (F32 ? 4 : 2);  // bytes of a step's K or V
    static constexpr int RING = F32 ? 1 : SIDE <= 8192 && NW == 4 ? 3 : 2;
    // Waves on a SIMD: two of 256 registers, but where two waves share 64 KB of LDS two such workgroups fill a CU.
    static constexpr int OCC = F32 && HD == 128 && NW == 2 ? 1 : 2;
};
template <int HD, bool F32, int NW>
__global__ __launch_bounds__(NW * 64, (Wide<HD, F32, NW>::OCC)) void paged_wide_kernel(const LkPagedAttn a) {
    constexpr int RT = 2, NT = Wide<HD, F32, NW>::NT, STEP = Wide<HD, F32, NW>::STEP, ROWS = Wide<HD, F32, NW>::ROWS;
    using Wave = Rows<HD, false, RT, NT, false, true>;
    constexpr int ND = Wave::ND, KS = Wave::KS, ES = F32 ? 4 : 2;
    constexpr int RB = HD * ES, PIECES = RB / 16, PER = 64 / PIECES;  // rows that one load instruction covers
    constexpr int SIDE = STEP * RB, OPS = SIDE / 1024 / NW;           // a step's K or V; a wave's loads of it
    constexpr int RING = Wide<HD, F32, NW>::RING;
    static_assert(OPS >= 1 && SIDE % (1024 * NW) == 0 && 16 % PER == 0, "whole load instructions, each within a tile");
    // f16: K, then V.  f32: one stage as it comes, and K and V in two f16 parts each.
    constexpr int ROW = HD * 2, PART = STEP * ROW, V0 = F32 ? 2 * PART : SIDE;
    __shared__ __align__(1024) char ring[RING][2 * SIDE];
    __shared__ __align__(1024) char s_parts[F32 ? 4 * PART : 16];
    __shared__ float s_top[2][NW];
    __shared__ uint32_t s_odd;  // a V that is not finite was met
    typedef __attribute__((address_space(3))) uint32_t* lptr;
    typedef __attribute__((address_space(1))) uint32_t* gptr;
    typedef __attribute__((address_space(3))) s4* sptr;
    const uint32_t lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // neighbours in the order of work are on one XCD (workgroups go round the 8): row groups of a kv head meet in its L2
    const uint32_t wg = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const bool chunks = a.n_chunks != 0;
    uint32_t seq = 0, in_seq = 0, left = 0;
    Share h{};
    if (chunks) {
        h = share_of<false>(a, ROWS);
        if (!h.live) return;  // uniform
    } else {
        const Plan plan = plan_runs<NW>(a, wg, STEP, ROWS, seq, in_seq);
        const uint64_t start = (uint64_t)wg * plan.run;
        if (start >= plan.total) return;  // uniform
        left = plan.total - start < plan.run ? (uint32_t)(plan.total - start) : plan.run;
    }
    do {
        uint32_t steps;
        if (chunks) {
            steps = (h.x1 - h.x0 + STEP - 1) / STEP;
        } else {
            if (seq >= a.n) return;  // uniform; not reached unless the lengths change under the call
            h.s = seq;
            h.sq = seq_of<false>(a, seq);
            const uint32_t groups = row_groups(a, h.sq, ROWS), of_item = groups ? item_steps(h.sq, STEP) : 0;
            if (in_seq >= groups * a.p.n_kv * of_item) {  // the sequence is done, or has nothing: on to the next
                seq++;
                in_seq = 0;
                continue;
            }
            const uint32_t item = in_seq / of_item, step0 = in_seq - item * of_item;
            steps = of_item - step0 < left ? of_item - step0 : left;
            h.kvh = item / groups;
            h.row0 = (item - h.kvh * groups) * ROWS;
            h.R = h.sq.rows * a.G;
            h.x0 = step0 * STEP;
            h.x1 = (step0 + steps) * STEP < h.sq.total ? (step0 + steps) * STEP : h.sq.total;
            h.whole = steps == of_item;
            // a run has at most one part that began before it and one that goes on behind it
            h.part = ((size_t)wg * 2 + (step0 == 0)) * ROWS;
            left -= steps;
            in_seq += steps;
        }
        const uint32_t rbase = h.row0 + w * 32;
        const bool busy = rbase < h.R;  // wave-uniform; an idle wave loads with the others

        // Where the part's tiles lie, 64 at a time, one a lane (byte of the first row), and which are no holes; `ahead`:
        // page ids of the next 64.
        auto ids_of = [&](uint32_t block) LK_INLINE -> uint32_t {
            uint32_t pos;
            const uint64_t y = (uint64_t)h.x0 + ((uint64_t)block * 64 + lane) * 16;
            return y < h.x1 ? tile_page<false>(a, h, (uint32_t)y, pos) : LK_NO_PAGE;
        };
        uint32_t at_lo, at_hi, block = 0;
        uint64_t there;
        auto place = [&](uint32_t id) LK_INLINE {
            const uint64_t at = tile_base(a, h, id, h.x0 + (block * 64 + lane) * 16, HD) * ES;
            at_lo = (uint32_t)at, at_hi = (uint32_t)(at >> 32);
            there = __ballot(id < a.p.n_pages);
        };
        place(ids_of(0));
        uint32_t ahead = ids_of(1);
        // this lane's piece of an instruction's rows: the instruction's first row is a multiple of PER
        const uint32_t in_op = lane / PIECES, my_piece = lane % PIECES;
        auto issue = [&](uint32_t n, char* to) LK_INLINE {
#pragma unroll
            for (int k = 0; k < 2 * OPS; k++) {
                const uint32_t q = w * OPS + k % OPS, row0 = q * PER, tile = (n * NT + row0 / 16) & 63;
                const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(at_hi, tile) << 32 | (uint32_t)__builtin_amdgcn_readlane(at_lo, tile);
                const uint32_t mine = ((row0 & 15) + in_op) * RB + ((F32 ? my_piece : my_piece ^ ((row0 + in_op) & 7)) * 16);
                const char* from = (const char*)(k < OPS ? a.p.k : a.p.v) + at;
                __builtin_amdgcn_global_load_lds((gptr)(from + mine), (lptr)(to + (k < OPS ? 0 : SIDE) + q * 1024), 16, 0, 0);
            }
        };
        // before a step's issue: the next 64 tiles begin every 64 / NT steps
        auto turn_page = [&](uint32_t n) LK_INLINE {
            if (n * NT / 64 != block) {
                block++;
                place(ahead);
                ahead = ids_of(block + 1);
            }
        };
        auto look = [&](uint32_t n) LK_INLINE -> uint32_t { return (uint32_t)(there >> (n * NT & 63)) & ((1u << NT) - 1); };
        // the positions of a step that a row may see; tiles: which are no holes
        auto live_of = [&](uint32_t x, uint32_t tiles) LK_INLINE -> uint64_t {
            uint64_t b = 0;
#pragma unroll
            for (int t = 0; t < NT; t++) b |= tiles >> t & 1 ? 0xFFFFull << (16 * t) : 0;
            return b & low_bits((int64_t)h.sq.total - x);
        };
        __syncthreads();  // the last part's s_odd is read
        if (threadIdx.x == 0) s_odd = 0;  // set behind a barrier at the earliest
        constexpr int AHEAD = F32 ? 1 : RING - 1;
        uint32_t tiles[AHEAD];  // of the steps under way: which tiles are no holes
#pragma unroll
        for (int n = 0; n < AHEAD; n++) {
            tiles[n] = 0;
            if ((uint32_t)n < steps) {
                tiles[n] = look(n);
                issue(n, ring[n]);
            }
        }
        Wave r;
        r.init(a, h, rbase);
        // Where the lane reads: K piece 4 ks + j of row c16; of V the part of column tile d that it hands the transposing
        // read (of 16 lanes, four hold a row's 16 dims, and each gets one dim of the four rows).  A tile further is 16
        // rows on.
        uint32_t k_at[KS], v_at[ND];
#pragma unroll
        for (int ks = 0; ks < KS; ks++) k_at[ks] = r.c16 * ROW + ((4 * ks + r.j) ^ (r.c16 & 7)) * 16;
        {
            const uint32_t row = 4 * r.j + r.c16 / 4;
#pragma unroll
            for (int d = 0; d < ND; d++) v_at[d] = V0 + row * ROW + ((2 * d + r.c16 % 4 / 2) ^ (row & 7)) * 16 + (r.c16 & 1) * 8;
        }
        int v_up = 126;  // f32: O is in units of 2^-v_up
        uint32_t slot = 0;  // n % RING
        for (uint32_t n = 0; n < steps; n++) {
            // step n has landed for every wave, and every wave is done with the stage that is filled next
            if (!F32 && RING > 2 && n + RING - 2 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((RING - 2) * 2 * OPS) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            const uint32_t tl = tiles[0];
#pragma unroll
            for (int k = 0; k + 1 < AHEAD; k++) tiles[k] = tiles[k + 1];
            const uint32_t x = h.x0 + n * STEP;
            const bool masked = tl != (1u << NT) - 1 || x + STEP > h.sq.ctx;  // uniform: something to hide
            const uint64_t live = masked ? live_of(x, tl) : 0;
            char* stage;
            int k_up = 0;  // f32: K was taken times 2^k_up
            if constexpr (F32) {
                // K and V into f16 parts, each step's largest value brought to 2^13..2^14: 22 bits of those near it, and
                // 2^-39 of it for the others.  V's power only falls, O following it.
                stage = s_parts;
                constexpr uint32_t UNITS = STEP * HD / 8, EACH = (UNITS + NW * 64 - 1) / (NW * 64);
                f4 u[2][EACH][2];
                float top[2] = {0.f, 0.f};
                uint32_t any = 0;
#pragma unroll
                for (int side = 0; side < 2; side++)
#pragma unroll
                    for (uint32_t e = 0; e < EACH; e++) {
                        const f4* from = (const f4*)(ring[0] + side * SIDE + (threadIdx.x + e * NW * 64) * 32);
                        u[side][e][0] = from[0], u[side][e][1] = from[1];
                    }
                if (masked) {
#pragma unroll
                    for (uint32_t e = 0; e < EACH; e++) {
                        const bool see = live >> ((threadIdx.x + e * NW * 64) / (HD / 8)) & 1;
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float y = u[1][e][i / 4][i % 4];
                            const bool bad = not_finite(y);
                            any |= see && bad;
                            u[1][e][i / 4][i % 4] = see && !bad ? y : 0.f;
                        }
                    }
                }
#pragma unroll
                for (int side = 0; side < 2; side++) {
#pragma unroll
                    for (uint32_t e = 0; e < EACH; e++)
#pragma unroll
                        for (int i = 0; i < 8; i++) top[side] = fmaxf(top[side], fabsf(u[side][e][i / 4][i % 4]));
                    if (__any(top[side] == INFINITY)) {  // the largest finite one
                        top[side] = 0.f;
#pragma unroll
                        for (uint32_t e = 0; e < EACH; e++)
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                const float y = u[side][e][i / 4][i % 4];
                                top[side] = fmaxf(top[side], not_finite(y) ? 0.f : fabsf(y));
                            }
                    }
                }
#pragma unroll
                for (int side = 0; side < 2; side++) {
                    const float t = lk_wave_max(top[side]);
                    if (lane == 0) s_top[side][w] = t;
                }
                if (any) s_odd = 1;
                __syncthreads();  // the stage is read: the next one may come
                if (n + 1 < steps) {
                    turn_page(n + 1);
                    tiles[0] = look(n + 1);
                    issue(n + 1, ring[0]);
                }
                int up[2];
#pragma unroll
                for (int side = 0; side < 2; side++) {
                    float t = s_top[side][0];
#pragma unroll
                    for (int k = 1; k < NW; k++) t = fmaxf(t, s_top[side][k]);
                    const int e = 13 + 127 - (int)(__float_as_uint(t) >> 23);
                    up[side] = __builtin_amdgcn_readfirstlane(t > 0.f ? (e < 126 ? e : 126) : 126);
                }
                k_up = up[0];
                if (up[1] < v_up) {
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
#pragma unroll
                        for (int d = 0; d < ND; d++)
#pragma unroll
                            for (int i = 0; i < 4; i++) r.o[rt][d][i] = ldexpf(r.o[rt][d][i], up[1] - v_up);
                    v_up = up[1];
                }
                up[1] = v_up;
                float minus = -1.f;  // as in weights()
                asm("" : "+s"(minus));
                const float by[2] = {ldexpf(1.f, up[0]), ldexpf(1.f, up[1])};  // -115..126: a normal number
#pragma unroll
                for (int side = 0; side < 2; side++)
#pragma unroll
                    for (uint32_t e = 0; e < EACH; e++) {
                        const uint32_t at = threadIdx.x + e * NW * 64, row = at / (HD / 8), piece = (at % (HD / 8)) ^ (row & 7);
                        h8 hi, lo;
#pragma unroll
                        for (int i = 0; i < 8; i += 2) {
                            const fl2 y = fl2{u[side][e][i / 4][i % 4] * by[side], u[side][e][i / 4][i % 4 + 1] * by[side]};
                            const hf2 x = __builtin_convertvector(y, hf2);
                            const hf2 z = __builtin_convertvector(
                                (fl2{__builtin_fmaf((float)x[0], minus, y[0]), __builtin_fmaf((float)x[1], minus, y[1])}), hf2);
                            hi[i] = x[0], hi[i + 1] = x[1];
                            lo[i] = z[0], lo[i + 1] = z[1];
                        }
                        char* to = s_parts + side * 2 * PART + row * ROW + piece * 16;
                        *(h8*)to = hi;
                        *(h8*)(to + PART) = lo;
                    }
                __syncthreads();
            } else {
                if (n + RING - 1 < steps) {
                    turn_page(n + RING - 1);
                    tiles[AHEAD - 1] = look(n + RING - 1);
                    issue(n + RING - 1, ring[slot ? slot - 1 : RING - 1]);
                }
                stage = ring[slot];
                slot = slot + 1 < RING ? slot + 1 : 0;
                if (masked) {
                    // V of positions that no row sees becomes zero, and what is not finite too
                    uint32_t any = 0;
                    for (uint32_t p = threadIdx.x; p < SIDE / 16; p += NW * 64) {
                        u4* at = (u4*)(stage + SIDE + p * 16);
                        u4 y = *at;
                        const bool see = live >> (p / PIECES) & 1;
#pragma unroll
                        for (int e = 0; e < 4; e++) y[e] = Wave::clean_word(see ? y[e] : 0, any);
                        *at = y;
                    }
                    if (any) s_odd = 1;
                    __syncthreads();
                }
            }
            if (!busy) continue;
            f4 sc[RT][NT];
            r.start(sc);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                u4 kr[NT];
#pragma unroll
                for (int t = 0; t < NT; t++) kr[t] = *(const u4*)(stage + k_at[ks] + t * 16 * ROW);
                r.scores(kr, ks, sc);
                if constexpr (F32) {
#pragma unroll
                    for (int t = 0; t < NT; t++) kr[t] = *(const u4*)(stage + PART + k_at[ks] + t * 16 * ROW);
                    r.template scores<1>(kr, ks, sc);
                }
                if (HD == 128 && ks % 2) __builtin_amdgcn_sched_barrier(0);  // K operands of two at a time: registers
            }
            r.relate(sc, k_up);
            if (masked) {
#pragma unroll
                for (int rt = 0; rt < RT; rt++) r.hide(rt, r.sees(a, h, x, live, rt), sc);
            }
            r.move(sc);
#pragma unroll
            for (int g = 0; g < NT / 2; g++) {
                h8 ph[RT], pl[RT];
                r.weights(sc, g, ph, pl);
#pragma unroll
                for (int part = 0; part < (F32 ? 2 : 1); part++)
#pragma unroll
                    for (int d0 = 0; d0 < ND; d0 += 4) {
                        h8 vb[4];
#pragma unroll
                        for (int d = 0; d < 4; d++) {
                            u2 y[2];
#pragma unroll
                            for (int t = 0; t < 2; t++)
                                y[t] = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((sptr)(stage + part * PART + v_at[d0 + d] + (2 * g + t) * 16 * ROW)));
                            vb[d] = __builtin_bit_cast(h8, u4{y[0][0], y[0][1], y[1][0], y[1][1]});
                        }
                        if (part == 0) r.add16(ph, pl, vb, d0);
                        else r.template add16<1>(ph, pl, vb, d0);
                        if (HD == 128) __builtin_amdgcn_sched_barrier(0);
                    }
            }
        }
        __syncthreads();  // s_odd, and the stages, are settled
        if (s_odd && busy)
            for (uint32_t n = 0; n < steps; n++) r.template poison<F32>(a, h, h.x0 + n * STEP);
        if (!busy) continue;
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float y[ND];
#pragma unroll
                for (int d = 0; d < ND; d++) y[d] = F32 ? ldexpf(r.o[rt][d][i], -v_up) : r.o[rt][d][i];
                const float top = r.max_of(rt, i), sum = r.sum_of(rt, i);
                r.put(a, h, w * 32 + rt * 16 + 4 * r.j + i, top, sum, y);
            }
    } while (left);
}

// Parts of a row, joined.  A block takes four rows: a wave weighs a row's parts (lane = part, at most 64), then HD / 4
// lanes by SPLIT groups a row add them up, each group every SPLIT-th part: two dependent reads of memory in all.  (One
// thread group walking the parts of a row: 19.6 us for 33 parts of 112 rows x 8; now 4.3 us.)  ROWS: of a workgroup of
// the wide kernel; 0: parts are the narrow kernel's chunks.
template <int HD, bool SPARSE, int ROWS, uint32_t STEP>
__global__ __launch_bounds__(256) void paged_fold_kernel(const LkPagedAttn a) {
    constexpr uint32_t L = HD / 4, SPLIT = 64 / L;
    __shared__ float s_f[4][kMaxChunks];
    __shared__ __align__(16) f4 s_y[4][SPLIT][L];
    const uint32_t pair = blockIdx.x, kvh = pair % a.p.n_kv, s = pair / a.p.n_kv;
    const Seq sq = seq_of<SPARSE>(a, s);
    const uint32_t R = sq.rows * a.G, w = threadIdx.x >> 6, lane = threadIdx.x & 63, row = blockIdx.y * 4 + w;
    if (!sq.live || blockIdx.y * 4 >= R) return;  // uniform
    constexpr uint32_t RG = ROWS ? ROWS : 1;
    uint32_t parts;
    size_t base, stride;  // of the row's parts, but for the first of runs
    const bool runs = ROWS && !a.n_chunks;
    if (runs) {
        const uint32_t groups = row_groups(a, sq, RG), of_item = item_steps(sq, STEP), run = (uint32_t)a.place[0];
        const uint64_t at = a.place[1 + s] + (uint64_t)(kvh * groups + blockIdx.y * 4 / RG) * of_item;
        const uint64_t wg = at / run;
        parts = (uint32_t)((at + of_item - 1) / run - wg) + 1;
        base = wg * 2 * RG + row % RG;
        stride = 2 * RG;
    } else {
        parts = chunks_of(a, sq.total).count;
        base = (size_t)pair * a.n_chunks * a.rows_pad + row;
        stride = a.rows_pad;
    }
    if (parts == 1) return;  // uniform: written as it is
    auto at = [&](uint32_t k) LK_INLINE { return base + k * stride + (runs && k == 0 ? RG : 0); };
    if (row < R) {  // wave-uniform
        float2 ml{-INFINITY, 0.f};
        if (lane < parts) ml = *(const float2*)(a.part_ml + 2 * at(lane));
        const float top = lk_wave_max(ml.x), f = __builtin_amdgcn_exp2f(ml.x - (top == -INFINITY ? 0.f : top));
        const float sum = lk_wave_sum(ml.y * f);
        s_f[w][lane] = f * (sum == 0.f ? 0.f : 1.f / sum);
    }
    __syncthreads();
    const uint32_t c = lane % L, sp = lane / L;
    f4 y = f4{0.f, 0.f, 0.f, 0.f};
    if (row < R) {
#pragma unroll 4
        for (uint32_t k = sp; k < parts; k += SPLIT) y += *(const f4*)(a.part_o + at(k) * HD + 4 * c) * s_f[w][k];
    }
    s_y[w][sp][c] = y;
    __syncthreads();
    if (row >= R || sp) return;
#pragma unroll
    for (uint32_t k = 1; k < SPLIT; k++) y += s_y[w][k][c];
    const uint32_t t = row / a.G;
    *(f4*)(a.out + (((size_t)s * a.tokens + t) * a.n_heads + kvh * a.G + row - t * a.G) * HD + 4 * c) = y;
}

}  // namespace

// Narrow: enough chunks of the table's capacity to fill the card.  Wide: as many workgroups as it holds, each with two
// places for parts.
constexpr uint32_t kCus = 256;
LkPagedPlan lk_paged_plan(uint32_t hd, bool f32, bool sparse, uint32_t n, uint32_t n_kv, uint32_t rows,
                          uint64_t positions) {
    LkPagedPlan p{};
    p.narrow = sparse || rows <= 32;
    p.tiles = p.narrow ? (rows <= 16 || sparse ? 1 : 2) : 2;
    p.waves = p.narrow ? 4 : rows <= 64 ? 2 : 4;
    const uint32_t per = p.narrow ? p.tiles * 16 : p.waves * 32;
    p.n_rg = (rows + per - 1) / per;
    p.rows_pad = p.n_rg * per;
    const uint64_t base = (uint64_t)n * n_kv * p.n_rg;
    const uint32_t step = f32 || hd == 128 ? 32 : 64;
    const uint64_t steps = (positions + step - 1) / step, fill = (uint64_t)kCus * (p.waves == 4 || (f32 && hd == 128) ? 2 : 4);
    p.steps = base * steps;
    // Runs begin 7 us later than chunks (they count the work first), but share out what lengths there are; chunks are as
    // long as the longest sequence's.  Runs from 480 positions a workgroup on.  us, chunks / runs: sequences of one
    // length, 8 x 16 tokens, 32 / 8 heads of 128, 8192 positions (512 a workgroup) 86 / 90; 4 x 32, 32 / 4 of 64, 8000 of
    // 8192 (512) 69 / 74, 1000 of 4096 (256) 33 / 34; f32, 3 x 23, 32 / 8 of 128, 5000 (236) 56 / 64; of many lengths,
    // 8 x 64, up to 32768 (4096) 251 / 171.
    if (!p.narrow && p.steps * step > 480 * fill) {
        p.blocks = fill;
        p.part_rows = fill * 2 * per;
        p.place_bytes = (((uint64_t)n + 1) * 8 + 255) / 256 * 256;
    } else {
        const uint32_t all = p.narrow ? step * 4 : step;  // narrow: every wave has a step
        const uint64_t pieces = (positions + all - 1) / all;
        uint64_t c;
        if (p.narrow) {
            // two steps a wave cost less than a fold: 1 x 1 token, up to 304 positions, 9.4 -> 8.6 us
            c = pieces <= 2 ? 1 : (1024 + base - 1) / base;
        } else {  // as few rounds of the card as can be, each of a chunk's positions and some 128 to begin
            uint64_t least = ~0ull;
            c = 1;
            for (uint64_t k = 1; k <= kMaxChunks && k <= pieces; k++) {
                const uint64_t cost = (base * k + fill - 1) / fill * ((pieces + k - 1) / k * all + 128);
                if (cost < least) least = cost, c = k;
            }
        }
        c = c > kMaxChunks ? kMaxChunks : c;
        c = c > pieces ? pieces : c;
        if (c < 1) c = 1;
        p.chunk = (uint32_t)((pieces + c - 1) / c * all);
        if (!p.chunk) p.chunk = all;
        p.n_chunks = (uint32_t)((positions + p.chunk - 1) / p.chunk);
        if (!p.n_chunks) p.n_chunks = 1;
        while (1u << p.unit < all) p.unit++;  // a power of two
        // short sequences: chunks down to this.  f32, 3 x 23 tokens over 1000 positions, 5000 in the table: 37 -> 29 us
        const uint32_t spread = p.narrow ? all : f32 ? 128 : 256;
        if (p.n_chunks > 1 && p.chunk > spread) p.chunk = spread;
        const uint64_t items = (uint64_t)n * n_kv * p.n_chunks;
        p.blocks = (items + 7) / 8 * 8 * p.n_rg;
        p.part_rows = p.n_chunks > 1 ? items * p.rows_pad : 0;
    }
    p.part_bytes = p.place_bytes + p.part_rows * (hd + 2) * 4;
    return p;
}

template <int HD, bool F32, bool SPARSE>
static hipError_t launch(const LkPagedAttn& a, const LkPagedPlan& p, hipStream_t st) {
    const dim3 grid((uint32_t)p.blocks), fold(a.n * a.p.n_kv, (a.tokens * a.G + 3) / 4);
    if (p.narrow) {
        if (p.tiles == 1) hipLaunchKernelGGL((paged_narrow_kernel<HD, F32, 1, SPARSE>), grid, dim3(256), 0, st, a);
        else if (!SPARSE) hipLaunchKernelGGL((paged_narrow_kernel<HD, F32, 2, false>), grid, dim3(256), 0, st, a);
        else return hipErrorInvalidValue;
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || p.n_chunks == 1) return e;
        hipLaunchKernelGGL((paged_fold_kernel<HD, SPARSE, 0, 0>), fold, dim3(256), 0, st, a);
    } else if constexpr (!SPARSE) {
#define LK_WIDE(NW)                                                                                                   \
    hipLaunchKernelGGL((paged_wide_kernel<HD, F32, NW>), grid, dim3(NW * 64), 0, st, a);                              \
    const hipError_t e = hipGetLastError();                                                                           \
    if (e != hipSuccess || p.n_chunks == 1) return e;                                                                 \
    hipLaunchKernelGGL((paged_fold_kernel<HD, false, Wide<HD, F32, NW>::ROWS, Wide<HD, F32, NW>::STEP>), fold,        \
                       dim3(256), 0, st, a)
        if (p.waves == 2) {
            LK_WIDE(2);
        } else {
            LK_WIDE(4);
        }
#undef LK_WIDE
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t lk_paged_attn_launch(LkPagedAttn a, const LkPagedPlan& p, void* ws, hipStream_t st) {
    a.chunk = p.chunk;
    a.unit = p.unit;
    a.n_chunks = p.n_chunks;
    a.n_rg = p.n_rg;
    a.rows_pad = p.rows_pad;
    a.scale = 1.44269504088896340736f * (a.p.hd == 64 ? 0.125f : 0.08838834764831845f);
    a.place = (uint64_t*)ws;
    a.part_o = (float*)((char*)ws + p.place_bytes);
    a.part_ml = a.part_o + p.part_rows * a.p.hd;
#define LK_PAGED(HD, F32) (a.sel ? launch<HD, F32, true>(a, p, st) : launch<HD, F32, false>(a, p, st))
    if (a.p.hd == 64) return a.p.f32 ? LK_PAGED(64, true) : LK_PAGED(64, false);
    return a.p.f32 ? LK_PAGED(128, true) : LK_PAGED(128, false);
#undef LK_PAGED
}
