// Attention of a batch of sequences over one paged KV pool, gfx950.  The rows [0, prefix) are one
// copy that every sequence shares; the rows from `prefix` on are each sequence's own, found through
// its block table.
//
// Mathematics.  For query row r (token, head) with scaled query q (log2 units) and allowed rows j,
// o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m), s_j = q.k_j, over any m.  A work item is (KV head,
// 16*MT query rows, a range of rows of the pool): the prefix ranges take the rows of ALL tokens at
// once, so the prefix is read from memory once for the batch; the own ranges take one sequence's
// tokens.  Every item leaves (m, l = sum 2^(s - m), unnormalised o) per query row, and
// paged_combine_kernel joins the items of a row.
//
// 32 rows of the pool are taken at a time, S^T = K Q^T and O^T += V^T P^T with
// v_mfma_f32_16x16x32_f16.  Lane (n = lane % 16, g = lane / 16) holds A[n][8g + j], B[8g + j][n] and
// D[4g + i][n]:
//  - K: lane (n, g) loads dims 32s + 8g .. +7 of rows n and 16 + n: the A operands as they are.
//  - S^T's result lies as (query n, rows 4g + i), which is the B operand of the second product when
//    its 32 rows are taken in the order {4g .. 4g+3, 16 + 4g .. 16 + 4g + 3}.
//  - V: lane (n, g) loads dims 64c + 4n .. +3 of those 8 rows, 256 contiguous bytes a row.  Column t
//    of the four is one A operand whose 16 output rows stand for dims 64c + 4n + t: the transposition
//    costs nothing.
// Few query rows (attn_narrow, 16): each wave takes tiles of its own, straight from memory to registers
// to the matrix units, and the waves join at the end.  Many (attn_wide, 64 or 128): the four waves share
// each tile, every wave loads and splits a quarter of it into LDS, laid out as the operands are read, and
// multiplies all of it with query rows of its own.
// Precision: each fp32 operand is split in two fp16 parts and a product takes three MFMAs
// (hi*hi + hi*lo + lo*hi, ~2^-21 per term).  fp16 reaches from 2^-24 to 65504, so K is scaled by a
// power of two per 32 rows, V by one per wave that only grows, each query by its own: the parts
// keep their bits whatever the magnitudes in the pool.  Scores, sums and outputs are fp32.
#pragma once

#include "paged_args.h"
#include "prefill_kernels.h"

namespace llmp {
namespace pg {

typedef pk::f16x8 f16x8;
typedef pk::floatx4 floatx4;

constexpr int kSchedAlu = 0x6;   // of the scheduler's barriers: VALU and scalar instructions may cross
constexpr int kAttnThreads = 256, kAttnWaves = kAttnThreads / 64;
constexpr int kTile = 32;            // pool rows a wave takes at a time
constexpr float kPShift = 4.0f;      // 2^(s - m + 4): small probabilities keep their fp16 bits
constexpr float kNegBig = dk::kNegBig;

// max(m, |x|, |y|) in one instruction.  (The compiler quiets every loaded value first, one more each.)
__device__ __forceinline__ float max_abs(float m, float x, float y) {
    asm("v_max3_f32 %0, |%1|, |%2|, %0" : "+v"(m) : "v"(x), "v"(y));
    return m;
}

// Split of x*f: hi = fp16(x*f), lo = fp16(x*f - hi), one mixed-precision multiply-add each, the first
// rounded from the exact product and the second from the exact difference.
// In plain operations, not in assembly: the compiler has to see who writes an operand of a matrix
// instruction, which must not read it within two wait states.  The opaque step keeps lo to the `hi` that
// was rounded above.
__device__ __forceinline__ void split2(float x, float y, float fx, float fy, pk::f16x2& hi, pk::f16x2& lo) {
    const pk::f16x2 r = {(_Float16)(x * fx), (_Float16)(y * fy)};
    unsigned u = __builtin_bit_cast(unsigned, r);
    asm("" : "+v"(u));
    hi = __builtin_bit_cast(pk::f16x2, u);
    lo = pk::f16x2{(_Float16)__builtin_fmaf(x, fx, -(float)hi[0]), (_Float16)__builtin_fmaf(y, fy, -(float)hi[1])};
}
__device__ __forceinline__ void split8(const float (&x)[8], const float (&f)[8], f16x8& hi, f16x8& lo) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        pk::f16x2 h, l;
        split2(x[2 * j], x[2 * j + 1], f[2 * j], f[2 * j + 1], h, l);
        hi[2 * j] = h[0];
        hi[2 * j + 1] = h[1];
        lo[2 * j] = l[0];
        lo[2 * j + 1] = l[1];
    }
}
__device__ __forceinline__ void split8(const float (&x)[8], float f, f16x8& hi, f16x8& lo) {
    const float ff[8] = {f, f, f, f, f, f, f, f};
    split8(x, ff, hi, lo);
}
// Probabilities: no factor.
__device__ __forceinline__ void split8(const float (&x)[8], f16x8& hi, f16x8& lo) {
    float minus = -1.0f;
    asm("" : "+s"(minus));   // (x - hi stays one multiply-add)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        unsigned u = pk::pack_f16(x[2 * j], x[2 * j + 1]);
        asm("" : "+v"(u));
        const pk::f16x2 h = __builtin_bit_cast(pk::f16x2, u);
        hi[2 * j] = h[0];
        hi[2 * j + 1] = h[1];
        lo[2 * j] = (_Float16)__builtin_fmaf((float)h[0], minus, x[2 * j]);
        lo[2 * j + 1] = (_Float16)__builtin_fmaf((float)h[1], minus, x[2 * j + 1]);
    }
}

// ---- one tile of 32 rows in registers --------------------------------------------------------
template <int D, bool Q8>
struct Tile;

// Address of row `row` (alike in all lanes) of KV head h of a page, rows of `unit` bytes; a lane adds
// its own part as a 32-bit offset, so that one scalar base serves all of its loads.
__device__ __forceinline__ const char* page_rows(const void* p, const PoolPlanes& pool, int page, int h, int row, int unit) {
    return static_cast<const char*>(p) + ((((long long)page * pool.n_kv_heads + h) << pool.shift) + row) * unit;
}
template <class T>
__device__ __forceinline__ T at(const char* base, unsigned offset) {
    return *reinterpret_cast<const T*>(base + offset);
}

__device__ __forceinline__ bool finite_bits(unsigned b) { return (b & 0x7F800000u) != 0x7F800000u; }

template <int D>
struct Tile<D, false> {
    static constexpr int KS = D / 32, NC = D / 64, REM = D % 64 / 32;
    floatx4 k[2][KS][2];
    floatx4 v[8][NC];
    float vr[8][REM ? 2 : 1];

    __device__ __forceinline__ void load_k(const PoolPlanes& p, int page0, int page1, int h, int r0, int r1, int n, int g) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const char* b = page_rows(p.k, p, u ? page1 : page0, h, u ? r1 : r0, 4 * D);
            const unsigned lane = (unsigned)(4 * D * n + 32 * g);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                k[u][s][0] = at<floatx4>(b, lane + 128 * s);
                k[u][s][1] = at<floatx4>(b, lane + 128 * s + 16);
            }
        }
    }
    __device__ __forceinline__ void load_v(const PoolPlanes& p, int page0, int page1, int h, int r0, int r1, int n, int g) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const char* b = page_rows(p.v, p, j < 4 ? page0 : page1, h, j < 4 ? r0 : r1, 4 * D);
            const unsigned row = (unsigned)(4 * D * 4 * g) + 4 * D * (j & 3);
#pragma unroll
            for (int c = 0; c < NC; ++c) v[j][c] = at<floatx4>(b, row + 16 * n + 256 * c);
            if constexpr (REM) {
                const float2 w = at<float2>(b, row + 8 * n + 256 * NC);
                vr[j][0] = w.x;
                vr[j][1] = w.y;
            }
        }
    }
    __device__ __forceinline__ float max_k() const {
        float x = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int e = 0; e < 4; e += 2) x = max_abs(x, k[u][s][q][e], k[u][s][q][e + 1]);
        return x;
    }
    __device__ __forceinline__ float max_v() const {
        float x = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 4; e += 2) x = max_abs(x, v[j][c][e], v[j][c][e + 1]);
            if constexpr (REM) x = max_abs(x, vr[j][0], vr[j][1]);
        }
        return x;
    }
    // Value with what no row holds (keep 0, else ~0) and what is not finite taken out; worst: the
    // largest magnitude's bits before that.
    static __device__ __forceinline__ float clean(float x, unsigned keep, unsigned& worst) {
        const unsigned b = __float_as_uint(x) & keep, m = b & 0x7FFFFFFFu;
        worst = max(worst, m);
        int fin = (int)(m - 0x7F800000u) >> 31;   // all ones where it is finite
        asm("" : "+v"(fin));                      // (not a lane mask per value: they would not fit)
        return __uint_as_float(b & (unsigned)fin);
    }
    // ok: bit u of the lane's K rows; returns bit u for a K row with a value that is not finite.
    __device__ __forceinline__ unsigned clean_k(unsigned ok) {
        unsigned r = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            unsigned worst = 0;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) k[u][s][q][e] = clean(k[u][s][q][e], 0u - (ok >> u & 1u), worst);
            r |= (unsigned)(worst >= 0x7F800000u) << u;
        }
        return r;
    }
    // The same for the lane's 8 V rows.
    __device__ __forceinline__ unsigned clean_v(unsigned ok) {
        unsigned r = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            unsigned worst = 0;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[j][c][e] = clean(v[j][c][e], 0u - (ok >> j & 1u), worst);
            if constexpr (REM) {
                vr[j][0] = clean(vr[j][0], 0u - (ok >> j & 1u), worst);
                vr[j][1] = clean(vr[j][1], 0u - (ok >> j & 1u), worst);
            }
            r |= (unsigned)(worst >= 0x7F800000u) << j;
        }
        return r;
    }
    __device__ __forceinline__ void k_split(int u, int s, float f, f16x8& hi, f16x8& lo) const {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = k[u][s][e >> 2][e & 3];
        split8(x, f, hi, lo);
    }
    // Output tile tt's column of the 8 rows.
    __device__ __forceinline__ void v_split(int tt, float f, f16x8& hi, f16x8& lo) const {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = tt < 4 * NC ? v[j][tt >> 2][tt & 3] : vr[j][(tt - 4 * NC) & 1];
        split8(x, f, hi, lo);
    }
};

template <int D>
struct Tile<D, true> {
    static constexpr int KS = D / 32, NC = D / 64, REM = D % 64 / 32;
    uint2 k[2][KS];
    float ks[2][KS];
    unsigned v[8][NC + REM];    // REM: the low half only
    float vs[8][NC + REM];

    __device__ __forceinline__ void load_k(const PoolPlanes& p, int page0, int page1, int h, int r0, int r1, int n, int g) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const char* b = page_rows(p.k, p, u ? page1 : page0, h, u ? r1 : r0, D);
            const char* sc = page_rows(p.ks, p, u ? page1 : page0, h, u ? r1 : r0, 4 * KS);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                k[u][s] = at<uint2>(b, (unsigned)(D * n + 8 * g) + 32 * s);
                ks[u][s] = at<float>(sc, (unsigned)(4 * KS * n) + 4 * s);
            }
        }
    }
    __device__ __forceinline__ void load_v(const PoolPlanes& p, int page0, int page1, int h, int r0, int r1, int n, int g) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int page = j < 4 ? page0 : page1, r = j < 4 ? r0 : r1;
            const char* b = page_rows(p.v, p, page, h, r, D);
            const char* sc = page_rows(p.vs, p, page, h, r, 4 * KS);
            const unsigned row = (unsigned)(4 * g) + (j & 3);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                v[j][c] = at<unsigned>(b, row * D + 4 * n + 64 * c);
                vs[j][c] = at<float>(sc, row * (4 * KS) + 4 * (n >> 3) + 8 * c);
            }
            if constexpr (REM) {
                v[j][NC] = at<unsigned short>(b, row * D + 2 * n + 64 * NC);
                vs[j][NC] = at<float>(sc, row * (4 * KS) + 8 * NC);
            }
        }
    }
    __device__ __forceinline__ float max_k() const {
        float x = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int s = 0; s < KS; ++s) x = fmaxf(x, fabsf(ks[u][s]));
        return x * 128.0f;
    }
    __device__ __forceinline__ float max_v() const {
        float x = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int c = 0; c < NC + REM; ++c) x = fmaxf(x, fabsf(vs[j][c]));
        return x * 128.0f;
    }
    __device__ __forceinline__ unsigned clean_k(unsigned ok) {
        unsigned r = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            unsigned worst = 0;
#pragma unroll
            for (int s = 0; s < KS; ++s) ks[u][s] = Tile<D, false>::clean(ks[u][s], 0u - (ok >> u & 1u), worst);
            r |= (unsigned)(worst >= 0x7F800000u) << u;
        }
        return r;
    }
    __device__ __forceinline__ unsigned clean_v(unsigned ok) {
        unsigned r = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            unsigned worst = 0;
#pragma unroll
            for (int c = 0; c < NC + REM; ++c) vs[j][c] = Tile<D, false>::clean(vs[j][c], 0u - (ok >> j & 1u), worst);
            r |= (unsigned)(worst >= 0x7F800000u) << j;
        }
        return r;
    }
    __device__ __forceinline__ void k_split(int u, int s, float f, f16x8& hi, f16x8& lo) const {
        const unsigned w[2] = {k[u][s].x, k[u][s].y};
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)(signed char)(w[e >> 2] >> (8 * (e & 3)) & 0xFF);
        split8(x, ks[u][s] * f, hi, lo);
    }
    __device__ __forceinline__ void v_split(int tt, float f, f16x8& hi, f16x8& lo) const {
        const int c = tt < 4 * NC ? tt >> 2 : NC, t = tt < 4 * NC ? tt & 3 : tt - 4 * NC;
        float x[8], y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = (float)(signed char)(v[j][c] >> (8 * t) & 0xFF);
            y[j] = vs[j][c] * f;
        }
        split8(x, y, hi, lo);
    }
};

// Largest of non-negative floats (their bits) over the wave, and of two packed 16-bit halves each.
template <class Max>
__device__ __forceinline__ unsigned wave_reduce(unsigned x, const Max& max_of) {
    auto step = [&](auto ctrl) {
        x = max_of(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xF, 0xF, false));
    };
    step(std::integral_constant<int, dk::kDppQuadXor1>{});
    step(std::integral_constant<int, dk::kDppQuadXor2>{});
    step(std::integral_constant<int, dk::kDppRowHalfMirror>{});
    step(std::integral_constant<int, dk::kDppRowMirror>{});
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max_of((unsigned)a[0], (unsigned)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = max_of((unsigned)b[0], (unsigned)b[1]);
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ float wave_max(float x) {
    return __uint_as_float(wave_reduce(__float_as_uint(x), [](unsigned a, unsigned b) { return max(a, b); }));
}
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned max_halves(unsigned a, unsigned b) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// Exponent e with max * 2^-e in [2^13, 2^14) (0 for 0; clamped so that 2^e and 2^-e are normal).
__device__ __forceinline__ int fit_exp(float mx) {
    const int b = (int)(__float_as_uint(mx) >> 23) - 127 - 13;
    return mx == 0.0f ? 0 : max(min(b, 120), -120);
}

__device__ __forceinline__ unsigned wave_or(unsigned x) {
    return wave_reduce(x, [](unsigned a, unsigned b) { return a | b; });
}
__device__ __forceinline__ int wave_max_i(int x) {
    return (int)wave_reduce((unsigned)x, [](unsigned a, unsigned b) { return (unsigned)max((int)a, (int)b); });
}

// The rows of a tile (bit = row) that the lanes' bits name: bk the K rows n and 16 + n, bv the V
// rows 4g + i and 16 + 4g + i.
__device__ __forceinline__ unsigned tile_rows(unsigned bk, unsigned bv, int n, int g) {
    return wave_or((bk & 1u) << n | (bk >> 1) << (16 + n) | (bv & 15u) << (4 * g) | (bv >> 4) << (16 + 4 * g));
}

// The sequence of work item `item` of an own-rows launch (paged_item_base), its start and its end: a search
// by 64 lanes at once.
__device__ __forceinline__ int item_sequence(const AttnArgs& a, int item, int BM, int lane, int& start, int& end) {
    int lo = 0, len = a.n_seqs;
    for (;;) {
        const int step = (len + 63) / 64, b = min(lo + lane * step, a.n_seqs - 1);
        const int from = a.seq_start[b], to = a.seq_start[b + 1];
        const bool in = lane * step < len && paged_item_base(from, a.group, BM, b) <= item;
        const int c = max((int)__popcll(__ballot(in)), 1) - 1;
        lo += c * step;
        if (step == 1) {
            start = __builtin_amdgcn_readlane(from, c);
            end = __builtin_amdgcn_readlane(to, c);
            return __builtin_amdgcn_readfirstlane(lo);
        }
        len = min(step, len - c * step);
    }
}

// The query rows of a work item: `rows` per item of one KV head, of all tokens (prefix) or of one
// sequence (OWN).
struct ItemRows {
    int tok0, r0, r1;     // token tok0 + r / G, head h*G + r % G for r in [r0, r1)
    const int* blk;       // the block table
};
template <bool OWN>
__device__ __forceinline__ ItemRows item_rows(const AttnArgs& a, int item, int rows, int lane) {
    ItemRows x{0, item * rows, 0, a.blocks};
    if constexpr (OWN) {
        int st, en;
        const int b = item_sequence(a, item, rows, lane, st, en);
        st = min(max(st, 0), a.n_tokens);
        en = min(max(en, st), a.n_tokens);
        x.tok0 = st;
        x.r0 = (item - paged_item_base(st, a.group, rows, b)) * rows;
        x.r1 = x.r0 < 0 ? x.r0 : min((en - st) * a.group, x.r0 + rows);
        x.blk += (long long)b * a.width;
    } else {
        x.r1 = min(min(max(a.seq_start[a.n_seqs], 0), a.n_tokens) * a.group, x.r0 + rows);
    }
    return x;
}

// One tile of 16 query rows: scaled, divided by a power of two of their own (returned as fq), split, as
// the B operands take them; pos and first: the rows of the sequence that the lane's query attends.
template <int D>
__device__ __forceinline__ void load_queries(const AttnArgs& a, const ItemRows& x, int r, int h, int g, f16x8 (&qh)[D / 32],
                                             f16x8 (&ql)[D / 32], float& fq, int& pos, int& first) {
    constexpr int KS = D / 32;
    const bool have = r < x.r1;
    const int rr = have ? r : x.r0, tok = x.tok0 + rr / a.group, head = h * a.group + rr % a.group;
    const float* q = a.q + (long long)tok * a.q_stride + (long long)head * D + 8 * g;
    const int p = a.positions[tok];
    float v[KS][8], mx = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) pk::load8(q + 32 * s, v[s]);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[s][e] *= a.qk_scale;
            mx = fmaxf(mx, fabsf(v[s][e]));
        }
    mx = dk::lane_step<16, true>(mx);
    mx = dk::lane_step<32, true>(mx);
    const int e = finite_bits(__float_as_uint(mx)) ? fit_exp(mx) : 0;
    const float f = pk::pow2i(-e);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[s][i] *= f;
        split8(v[s], qh[s], ql[s]);
    }
    const bool live = have && (unsigned)p < (unsigned)a.max_seq;
    pos = live ? p : -1;
    first = !live ? 0x7fffffff : a.window > 0 ? max(p + 1 - a.window, 0) : 0;
    fq = pk::pow2i(e);
}

// The tiles [lo, hi) of one split of an item's rows [row_lo, row_hi).
template <bool OWN>
__device__ __forceinline__ void split_tiles(const AttnArgs& a, int row_lo, int row_hi, int split, int& lo, int& hi) {
    const int first = min(row_lo, row_hi) / kTile, end = row_lo < row_hi ? (row_hi + kTile - 1) / kTile : first;
    if constexpr (OWN) {
        const int per = (end - first + a.own_splits - 1) / a.own_splits;
        lo = min(first + split * per, end);
        hi = min(lo + per, end);
    } else {
        lo = max(split * a.prefix_tiles, first);
        hi = max(min(split * a.prefix_tiles + a.prefix_tiles, end), lo);
    }
}

// Scores to probabilities of one tile.  st: S^T in units of 1 / (fkr * fq); on return ph, pl hold the
// split of p = 2^(s - m).  The maxima are only raised where a score passes the present one by 2^12 or more
// (p stays below 2^12, which fp16 holds), so that most tiles leave o as it is: true where o has to be
// multiplied by alpha.  poison: rows of the tile that make a NaN of what attends them.
template <int MT, int NU, class Attended>
__device__ __forceinline__ bool tile_softmax(const AttnArgs& a, floatx4 (&st)[MT][NU], float fkr, const float (&fq)[MT],
                                             float (&m)[MT], float (&l)[MT], float (&alpha)[MT], f16x8 (&ph)[MT][NU / 2],
                                             f16x8 (&pl)[MT][NU / 2], bool masked, unsigned long long poison, int g,
                                             const Attended& attended) {
    float fs[MT], mx[MT];
    bool up = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        fs[mt] = fminf(fmaxf(fkr * fq[mt], 1.2e-38f), 1.7e38f);   // (0 * -inf would be a NaN)
        if (a.softcap > 0.0f) {
            const float isc = a.inv_softcap * fs[mt];
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) st[mt][u][i] = a.softcap_log2e * tanhf(st[mt][u][i] * isc);
            fs[mt] = 1.0f;
        }
        if (masked) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = 16 * u + 4 * g + i;
                    const float x = poison >> row & 1 ? __builtin_nanf("") : st[mt][u][i];
                    st[mt][u][i] = attended(mt, row) ? x : -__builtin_inff();
                }
        }
        float x = kNegBig;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) x = fmaxf(x, st[mt][u][i]);
        x = dk::lane_step<16, true>(x);
        x = dk::lane_step<32, true>(x);
        mx[mt] = x * fs[mt];
        up |= mx[mt] > m[mt] + 12.0f;
    }
    const bool rescale = __ballot(up) != 0;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const float mn = rescale ? fmaxf(m[mt], mx[mt] - kPShift) : m[mt];
        alpha[mt] = dk::fast_exp2(m[mt] - mn);
        m[mt] = mn;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NU / 2; ++w) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = dk::fast_exp2(__builtin_fmaf(st[mt][2 * w + (i >> 2)][i & 3], fs[mt], -mn));
                sum += p[i];
            }
            split8(p, ph[mt][w], pl[mt][w]);
        }
        l[mt] = __builtin_fmaf(l[mt], alpha[mt], sum);
    }
    return rescale;
}

// The factor that follows V's exponent: ev grows with the largest value seen.
__device__ __forceinline__ float raise_exp(int& ev, int evt) {
    const float f = evt <= ev ? 1.0f : ev < -500 ? 0.0f : pk::pow2i(max(ev - evt, -126));
    ev = max(ev, evt);
    return f;
}

// One tile of 16 query rows' state (o: lane's dims as D[4g + i][n] of each output tile) to its part.
template <int D>
__device__ __forceinline__ void store_part(const AttnArgs& a, const ItemRows& x, int r, int h, long long part, float m, float l,
                                           const floatx4 (&o)[D / 16], int g) {
    constexpr int NC = D / 64, REM = D % 64 / 32;
    if (r >= x.r1) return;
    const long long rows = (long long)a.n_tokens * a.n_heads;
    const long long row = (long long)(x.tok0 + r / a.group) * a.n_heads + h * a.group + r % a.group;
    if (g == 0) *reinterpret_cast<float2*>(a.part_ml + (part * rows + row) * 2) = make_float2(m, l);
    if (l == 0.0f) return;   // (the combine takes no outputs of such a part)
    float* po = a.part_o + (part * rows + row) * D;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<floatx4*>(po + 64 * c + 16 * g + 4 * i) =
                floatx4{o[4 * c][i], o[4 * c + 1][i], o[4 * c + 2][i], o[4 * c + 3][i]};
    if constexpr (REM) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float2*>(po + 64 * NC + 2 * (4 * g + i)) = make_float2(o[4 * NC][i], o[4 * NC + 1][i]);
    }
}

// 16 query rows against a split of the prefix, or (OWN) of one sequence's own rows; the waves take the
// split's tiles in turn.  Bound by memory latency: two waves per SIMD are all that K and V of a tile in
// registers leave, each with one tile on its way (one token of 32 sequences, 32 + 8 heads of 128, up to 1500 own fp32
// rows each: 50 us, 3.8 TB/s; 64 sequences, 32 + 8 heads of 64, up to 2000 Q8_0 rows: 40 us, where the split
// of the quants takes 17 us of every SIMD).  The four query heads of such a KV head fill a quarter of the 16 rows: the
// matrix units run 5 to 10 % of the time, so no smaller tile is made for them.
template <int D, bool Q8, bool OWN>
__device__ __forceinline__ void attn_narrow(const AttnArgs& a, uint4* lds, int item, int h, int split) {
    using T = Tile<D, Q8>;
    constexpr int KS = D / 32, DT = D / 16;
    // K and V of a tile in registers at once, where they leave room for two waves per SIMD.
    constexpr bool BOTH = D < 128 || Q8;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const ItemRows x = item_rows<OWN>(a, item, 16, lane);
    if (x.r0 >= x.r1) return;
    f16x8 qh[KS], ql[KS];
    float fq[1], m[1] = {kNegBig}, l[1] = {0.0f}, alpha[1];
    int pos, first;
    load_queries<D>(a, x, x.r0 + n, h, g, qh, ql, fq[0], pos, first);
    // Rows that some query attends, and those that all do.
    const bool real = x.r0 + n < x.r1;
    const int hi_any = wave_max_i(pos) + 1, lo_any = -wave_max_i(-first);
    const int hi_all = -wave_max_i(real ? -pos : -0x7ffffffe) + 1, lo_all = wave_max_i(real ? first : 0);
    const int lo = OWN ? max(a.prefix, lo_any) : lo_any, hi = OWN ? hi_any : min(a.prefix, hi_any);
    int t_lo, t_hi;
    split_tiles<OWN>(a, lo, hi, split, t_lo, t_hi);

    floatx4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = floatx4{0, 0, 0, 0};
    int ev = -1000;
    const int rmask = (1 << a.pool.shift) - 1;
    // Entries of the block table for the two half tiles of 16 rows, each of which lies in one page; one
    // outside the pool holds no rows (page 0 is read instead and masked).
    auto entry = [&](int tile, int u) { return x.blk[min((tile * kTile + 16 * u) >> a.pool.shift, a.width - 1)]; };
    auto in_pool = [&](int e) { return paged_page_ok(e, a.pool.n_pages); };
    // Software pipeline: a tile's K is loaded behind the scores of the tile before and lands during
    // its softmax and second product; its V is loaded behind that product and lands during the scores.
    // The table entries are one tile further ahead.
    T t;
    int tile = t_lo + wave;
    int n0 = 0, n1 = 0, c0 = 0, c1 = 0;
    auto load_k = [&](int at) {
        t.load_k(a.pool, in_pool(c0) ? c0 : 0, in_pool(c1) ? c1 : 0, h, at * kTile & rmask, (at * kTile + 16) & rmask, n, g);
    };
    auto load_v = [&](int at, int d0, int d1) {
        t.load_v(a.pool, in_pool(d0) ? d0 : 0, in_pool(d1) ? d1 : 0, h, at * kTile & rmask, (at * kTile + 16) & rmask, n, g);
    };
    if (tile < t_hi) {
        const int e0 = entry(tile, 0), e1 = entry(tile, 1);
        n0 = entry(tile + kAttnWaves, 0);
        n1 = entry(tile + kAttnWaves, 1);
        c0 = __builtin_amdgcn_readfirstlane(e0);
        c1 = __builtin_amdgcn_readfirstlane(e1);
        load_k(tile);
        if constexpr (BOTH) load_v(tile, c0, c1);
    }
    for (; tile < t_hi; tile += kAttnWaves) {
        const int k0 = tile * kTile, v0 = c0, v1 = c1;
        const bool there0 = in_pool(c0), there1 = in_pool(c1);
        const bool plain = k0 >= max(lo, lo_all) && k0 + kTile <= min(hi, hi_all) && there0 && there1;
        auto held = [&](int row) {   // row of the tile: whether the item has it
            return (row < 16 ? there0 : there1) && k0 + row >= lo && k0 + row < hi;
        };
        auto attended = [&](int, int row) { return held(row) && k0 + row >= first && k0 + row <= pos; };
        unsigned poison = 0;   // rows (bit = row of the tile) that hold a value that is not finite
        if (!plain) {
            const unsigned bk = t.clean_k((unsigned)held(n) | (unsigned)held(16 + n) << 1);
            if (__ballot(bk) != 0) poison = tile_rows(bk, 0, n, g);
        }
        float mk = wave_max(t.max_k());
        if (!finite_bits(__float_as_uint(mk))) {   // an infinity must not take the other rows' bits
            poison |= tile_rows(t.clean_k(3u), 0, n, g);
            mk = wave_max(t.max_k());
        }
        const int ek = fit_exp(mk);
        const float fk = pk::pow2i(-ek), fkr = pk::pow2i(ek);
        floatx4 st[1][2] = {{{0, 0, 0, 0}, {0, 0, 0, 0}}};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                f16x8 kh, kl;
                t.k_split(u, s, fk, kh, kl);
                st[0][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[s], st[0][u], 0, 0, 0);
                st[0][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[s], st[0][u], 0, 0, 0);
                st[0][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh[s], st[0][u], 0, 0, 0);
            }
        const int next = tile + kAttnWaves;
        if constexpr (!BOTH) load_v(tile, v0, v1);
        c0 = __builtin_amdgcn_readfirstlane(n0);
        c1 = __builtin_amdgcn_readfirstlane(n1);
        if (next < t_hi) {
            n0 = entry(next + kAttnWaves, 0);
            n1 = entry(next + kAttnWaves, 1);
            if constexpr (BOTH) load_k(next);
        }
        f16x8 ph[1][1], pl[1][1];
        const bool rescale = tile_softmax<1, 2>(a, st, fkr, fq, m, l, alpha, ph, pl, !plain || poison, poison, g, attended);
        unsigned bv = 0;
        if (!plain) {
            unsigned ok = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) ok |= (unsigned)held(16 * (j >> 2) + 4 * g + (j & 3)) << j;
            bv = t.clean_v(ok);
        }
        float mv = wave_max(t.max_v());
        if (!finite_bits(__float_as_uint(mv))) {
            bv |= t.clean_v(255u);
            mv = wave_max(t.max_v());
        }
        if (__ballot(bv) != 0) {
            // a lane's rows of P are its rows of V: their probabilities become NaN where attended
            poison = tile_rows(0, bv, n, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = 16 * (j >> 2) + 4 * g + (j & 3);
                if ((poison >> row & 1) && attended(0, row)) {
                    ph[0][0][j] = (_Float16)__builtin_nanf("");
                    l[0] = __builtin_nanf("");
                }
            }
        }
        const float fe = raise_exp(ev, fit_exp(mv));
        if (rescale || fe != 1.0f) {
            const float f = alpha[0] * fe;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] = o[d] * f;
        }
        const float fv = pk::pow2i(-ev);
#pragma unroll
        for (int tt = 0; tt < DT; ++tt) {
            f16x8 vh, vl;
            t.v_split(tt, fv, vh, vl);
            o[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph[0][0], o[tt], 0, 0, 0);
            o[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl[0][0], o[tt], 0, 0, 0);
            o[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph[0][0], o[tt], 0, 0, 0);
        }
        if (next < t_hi) {
            if constexpr (BOTH) load_v(next, c0, c1);
            else load_k(next);
        }
    }
    // l is a sum over the lane's own rows so far: the four groups of a query together.
    l[0] = dk::lane_step<16, false>(l[0]);
    l[0] = dk::lane_step<32, false>(l[0]);
    const float f = ev < -500 ? 0.0f : pk::pow2i(ev);
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = o[d] * f;
    // The waves' states, in a fixed order: 2 into 0 and 3 into 1, then 1 into 0.
    constexpr int XS = D / 4 + 2;
    float* xch = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int round = 0; round < 2; ++round) {
        const int from = round == 0 ? 2 : 1, count = round == 0 ? 2 : 1;
        if (wave >= from && wave < from + count) {
            float* y = xch + (size_t)(wave - from) * XS * 64 + lane;
            y[0] = m[0];
            y[64] = l[0];
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) y[(2 + 4 * d + i) * 64] = o[d][i];
        }
        __syncthreads();
        if (wave < count) {
            const float* y = xch + (size_t)wave * XS * 64 + lane;
            const float m2 = y[0], l2 = y[64];
            const float mn = fmaxf(m[0], m2), f1 = dk::fast_exp2(m[0] - mn), f2 = dk::fast_exp2(m2 - mn);
            m[0] = mn;
            l[0] = l[0] * f1 + l2 * f2;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][i] = o[d][i] * f1 + y[(2 + 4 * d + i) * 64] * f2;
        }
        __syncthreads();
    }
    if (wave == 0)
        store_part<D>(a, x, x.r0 + n, h, OWN ? a.prefix_splits + split : split, m[0], l[0], o, g);
}

// ---- a tile shared by four waves ---------------------------------------------------------------
// Rows of it: 64 at head_dim 64, 32 above (the same bytes).  In LDS: K as [16-row parts x D/32 steps][hi,
// lo][lane] and V as [32-row groups x D/16 output tiles][hi, lo][lane], 16 bytes a lane, exactly the
// operands: every read is one conflict-free b128.  A wave loads, cleans and splits operands of K and units
// of V (64 dims) of one 16-row part, so that one entry of the block table serves all of its loads; a unit's lane
// holds 4 rows of 4 dims, 8 bytes of four operands.
constexpr int wide_rows(int D) { return D == 64 ? 64 : 32; }
constexpr int wide_tiles(int D) { return D <= 128 ? 2 : 1; }

template <int D, bool Q8>
struct TilePart {
    static constexpr int KS = D / 32, NC = D / 64, REM = D % 64 / 32, DT = D / 16, NU = wide_rows(D) / 16;
    static constexpr int NK = NU * KS, NV = NC + REM, WPP = 4 / NU;   // WPP: waves of a part
    static constexpr int KP = (KS + WPP - 1) / WPP, VP = (NV + WPP - 1) / WPP;
    static constexpr int kBytes = (NK + NU / 2 * DT) * 2 * 64 * 16;
    floatx4 k[KP][2];      // Q8: 8 quants in the first two words, the scale in the third
    floatx4 v[VP][4];      // Q8: 4 quants and their scale

    // The wave's 16-row part; step s of its K operand i, and 64 dims c of its V unit i.
    static __device__ __forceinline__ int part(int wave) { return wave / WPP; }
    static __device__ __forceinline__ int k_step(int wave, int i) { return KP * (wave % WPP) + i; }
    static __device__ __forceinline__ int v_dims(int wave, int i) { return VP * (wave % WPP) + i; }
    static __device__ __forceinline__ bool no_k(int wave, int i) { return KS % WPP != 0 && k_step(wave, i) >= KS; }
    static __device__ __forceinline__ bool no_v(int wave, int i) { return NV % WPP != 0 && v_dims(wave, i) >= NV; }

    // From row `row` of `page` on.
    __device__ __forceinline__ void load(const PoolPlanes& p, int page, int row, int h, int wave, int n, int g) {
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            if (no_k(wave, i)) break;
            const int s = k_step(wave, i);
            if constexpr (Q8) {
                const uint2 w = at<uint2>(page_rows(p.k, p, page, h, row, D) + 32 * s, D * n + 8 * g);
                k[i][0] = floatx4{__uint_as_float(w.x), __uint_as_float(w.y),
                                  at<float>(page_rows(p.ks, p, page, h, row, 4 * KS) + 4 * s, 4 * KS * n), 0};
            } else {
                const char* b = page_rows(p.k, p, page, h, row, 4 * D) + 128 * s;
                k[i][0] = at<floatx4>(b, 4 * D * n + 32 * g);
                k[i][1] = at<floatx4>(b, 4 * D * n + 32 * g + 16);
            }
        }
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            if (no_v(wave, i)) break;
            const int c = v_dims(wave, i);
            if constexpr (Q8) {
                const char* b = page_rows(p.v, p, page, h, row, D) + 64 * c;
                const char* sc = page_rows(p.vs, p, page, h, row, 4 * KS) + 8 * c;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned r = 4 * g + j;
                    const bool full = REM == 0 || c < NC;
                    const unsigned w = full ? at<unsigned>(b, D * r + 4 * n) : at<unsigned short>(b, D * r + 2 * n);
                    v[i][j] = floatx4{__uint_as_float(w), at<float>(sc, 4 * KS * r + (full ? 4 * (n >> 3) : 0)), 0, 0};
                }
            } else {
                const char* b = page_rows(p.v, p, page, h, row, 4 * D) + 256 * c;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned r = 4 * D * (4 * g + j);
                    if (REM == 0 || c < NC) {
                        v[i][j] = at<floatx4>(b, r + 16 * n);
                    } else {
                        const float2 w = at<float2>(b, r + 8 * n);
                        v[i][j] = floatx4{w.x, w.y, 0, 0};
                    }
                }
            }
        }
    }
    // Takes out what no row holds (held(row) false) and what is not finite; returns the rows (bit = row
    // of the tile) of the lane's share that held such a value.
    template <class Held>
    __device__ __forceinline__ unsigned long long clean(const Held& held, int wave, int n, int g) {
        using C = Tile<D, false>;
        unsigned long long bad = 0;
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            if (no_k(wave, i)) break;
            const int row = 16 * part(wave) + n;
            const unsigned keep = 0u - (unsigned)held(row);
            unsigned worst = 0;
            if constexpr (Q8) {
                k[i][0][2] = C::clean(k[i][0][2], keep, worst);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) k[i][e >> 2][e & 3] = C::clean(k[i][e >> 2][e & 3], keep, worst);
            }
            bad |= (unsigned long long)(worst >= 0x7F800000u) << row;
        }
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            if (no_v(wave, i)) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = 16 * part(wave) + 4 * g + j;
                const unsigned keep = 0u - (unsigned)held(row);
                unsigned worst = 0;
                if constexpr (Q8) {
                    v[i][j][1] = C::clean(v[i][j][1], keep, worst);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[i][j][e] = C::clean(v[i][j][e], keep, worst);
                }
                bad |= (unsigned long long)(worst >= 0x7F800000u) << row;
            }
        }
        return bad;
    }
    // The wave's largest magnitudes: bits 16-31 of K's in the low half, of V's in the high half.
    __device__ __forceinline__ unsigned largest(int wave) const {
        float x = 0.0f, y = 0.0f;
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            if (no_k(wave, i)) break;
            if constexpr (Q8) {
                x = max_abs(x, k[i][0][2], k[i][0][2]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e += 2) x = max_abs(x, k[i][e >> 2][e & 3], k[i][e >> 2][(e & 3) + 1]);
            }
        }
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            if (no_v(wave, i)) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (Q8) {
                    y = max_abs(y, v[i][j][1], v[i][j][1]);
                } else {
                    y = max_abs(y, v[i][j][0], v[i][j][1]);
                    y = max_abs(y, v[i][j][2], v[i][j][3]);
                }
            }
        }
        return wave_reduce(__builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u), max_halves);
    }
    static __device__ __forceinline__ float quant(float word, int byte) {
        return (float)(signed char)(__float_as_uint(word) >> (8 * byte) & 0xFF);
    }
    __device__ __forceinline__ void store(uint4* lds, float fk, float fv, int wave, int lane) const {
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            if (no_k(wave, i)) break;
            const int q = part(wave) * KS + k_step(wave, i);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = Q8 ? quant(k[i][0][e >> 2], e & 3) : k[i][e >> 2][e & 3];
            f16x8 hi, lo;
            split8(x, Q8 ? k[i][0][2] * fk : fk, hi, lo);
            lds[(2 * q + 0) * 64 + lane] = __builtin_bit_cast(uint4, hi);
            lds[(2 * q + 1) * 64 + lane] = __builtin_bit_cast(uint4, lo);
        }
        uint2* lv = reinterpret_cast<uint2*>(lds + NK * 2 * 64);
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            if (no_v(wave, i)) break;
            const int u = part(wave), c = v_dims(wave, i);
#pragma unroll
            for (int t = 0; t < 4; t += 2) {   // columns t and t + 1
                if (REM && c >= NC && t > 0) break;
                float x[8], y[8];
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        x[4 * w + j] = Q8 ? quant(v[i][j][0], t + w) : v[i][j][t + w];
                        y[4 * w + j] = Q8 ? v[i][j][1] * fv : fv;
                    }
                f16x8 hi, lo;
                split8(x, y, hi, lo);
                const uint4 uh = __builtin_bit_cast(uint4, hi), ul = __builtin_bit_cast(uint4, lo);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const int tt = (u >> 1) * DT + 4 * c + t + w;
                    lv[((2 * tt + 0) * 64 + lane) * 2 + (u & 1)] = w ? make_uint2(uh.z, uh.w) : make_uint2(uh.x, uh.y);
                    lv[((2 * tt + 1) * 64 + lane) * 2 + (u & 1)] = w ? make_uint2(ul.z, ul.w) : make_uint2(ul.x, ul.y);
                }
            }
        }
    }
};

// 64*MT query rows, 16*MT a wave, against a split of the prefix, or (OWN) of one sequence's own rows.
// Two tiles in LDS (one at head_dim 256, whose two would leave room for one workgroup a CU): while the
// waves multiply tile i, they hold tile i + 2 in flight and have stored i + 1: one barrier a tile (an item of 128
// rows against 32001 shared rows of 128 dims: 109 us with one tile and two barriers, 84 us, 3.1 TB/s).
// Many rows are bound by the issue of two waves a SIMD: of its 340 us in 12 prompts of up to 700 tokens, 32 + 8
// heads of 64, behind 2000 shared rows (300 us a call unprofiled, 240 TFLOP/s, three times that in fp16
// products), vector instructions take 155, the matrix units 91: exponentials, the split of P, and the split of K and
// V, which 128 rows share (with 64 rows an item 430 us).  Few rows against a long prefix are bound by the latency of
// one tile in flight per workgroup; 64 rows an item read each tile twice and take 107 us where 128 take 90.
template <int D, int MT, bool Q8, bool OWN>
__device__ __forceinline__ void attn_wide(const AttnArgs& a, uint4* lds, int item, int h, int split) {
    using T = TilePart<D, Q8>;
    constexpr int KS = D / 32, DT = D / 16, NK = T::NK, NU = T::NU, TR = 16 * NU, kTileU4 = T::kBytes / 16;
    constexpr bool TWO = wide_tiles(D) == 2;
    __shared__ int s_range[4][kAttnWaves];
    __shared__ unsigned s_max[2][kAttnWaves], s_gone[2][kAttnWaves];
    __shared__ unsigned long long s_bad[2][kAttnWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
    const ItemRows x = item_rows<OWN>(a, item, 64 * MT, lane);
    if (x.r0 >= x.r1) return;
    const int rw = x.r0 + 16 * MT * wave;
    f16x8 qh[MT][KS], ql[MT][KS];
    float fq[MT], m[MT], l[MT], alpha[MT];
    int pos[MT], first[MT], hi_any = -1, lo_any = 0x7fffffff, hi_all = 0x7ffffffe, lo_all = 0;
    floatx4 o[MT][DT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int r = rw + 16 * mt + n;
        load_queries<D>(a, x, r, h, g, qh[mt], ql[mt], fq[mt], pos[mt], first[mt]);
        hi_any = max(hi_any, pos[mt]);
        lo_any = min(lo_any, first[mt]);
        if (r < x.r1) {
            hi_all = min(hi_all, pos[mt]);
            lo_all = max(lo_all, first[mt]);
        }
        m[mt] = kNegBig;
        l[mt] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[mt][d] = floatx4{0, 0, 0, 0};
    }
    hi_any = wave_max_i(hi_any) + 1;
    lo_any = -wave_max_i(-lo_any);
    hi_all = -wave_max_i(-hi_all) + 1;
    lo_all = wave_max_i(lo_all);
    if (lane == 0) {
        s_range[0][wave] = lo_any;
        s_range[1][wave] = hi_any;
        s_range[2][wave] = lo_all;
        s_range[3][wave] = hi_all;
    }
    __syncthreads();
    // Of all waves: the rows that some query attends, and those that every query does.
    auto all_waves = [&](int which, bool most) {
        int y = s_range[which][0];
#pragma unroll
        for (int w = 1; w < kAttnWaves; ++w) y = most ? max(y, s_range[which][w]) : min(y, s_range[which][w]);
        return __builtin_amdgcn_readfirstlane(y);
    };
    int lo = all_waves(0, false), hi = all_waves(1, true);
    const int lo_every = all_waves(2, true), hi_every = all_waves(3, false);
    if constexpr (OWN) lo = max(a.prefix, lo);
    else hi = min(a.prefix, hi);
    int t_lo, t_hi;
    split_tiles<OWN>(a, lo, hi, split, t_lo, t_hi);
    // The split's rows [lo, hi), taken TR at a time from row0 on.
    const int row0 = t_lo * kTile, tiles = (t_hi - t_lo + TR / kTile - 1) / (TR / kTile);
    lo = max(lo, row0);
    hi = min(hi, t_hi * kTile);

    int ev = -1000;
    const int rmask = (1 << a.pool.shift) - 1;
    // Entries of the block table for the 16-row parts, each of which lies in one page; one outside the
    // pool holds no rows (page 0 is read instead and masked).
    auto entry = [&](int tile, int u) { return x.blk[min((row0 + tile * TR + 16 * u) >> a.pool.shift, a.width - 1)]; };
    auto in_pool = [&](int e) { return paged_page_ok(e, a.pool.n_pages); };
    // The loaded tile t, the entry c of the wave's part of it, and the next tile's e.
    T t;
    int e = 0, c = 0;
    const int part = T::part(wave);
    auto load = [&](int tile) {
        c = __builtin_amdgcn_readfirstlane(e);
        e = entry(tile + 1, part);
        t.load(a.pool, in_pool(c) ? c : 0, (row0 + tile * TR + 16 * part) & rmask, h, wave, n, g);
    };
    auto held = [&](int k0, unsigned gone, int row) { return !(gone >> (row >> 4) & 1) && k0 + row >= lo && k0 + row < hi; };
    // The loaded tile's largest values, for the exponents; and where some query does not attend all of
    // it, or a value is infinite, what is not to be multiplied is taken out.
    auto inspect = [&](int tile) {
        const int k0 = row0 + tile * TR;
        const unsigned gone = (unsigned)!in_pool(c) << part;   // parts of it that no page of the pool holds: the wave's
        unsigned long long bad = 0;
        unsigned mx = t.largest(wave);
        const bool every = k0 >= max(lo, lo_every) && k0 + TR <= min(hi, hi_every) && gone == 0;
        if (!every || (mx & 0x7F80u) == 0x7F80u || mx >= 0x7F800000u) {
            bad = t.clean([&](int row) { return held(k0, gone, row); }, wave, n, g);
            bad = __ballot(bad != 0) != 0
                      ? (unsigned long long)wave_or((unsigned)(bad >> 32)) << 32 | wave_or((unsigned)bad) : 0ull;
            mx = t.largest(wave);
        }
        if (lane == 0) {
            s_max[tile & 1][wave] = mx;
            s_bad[tile & 1][wave] = bad;
            s_gone[tile & 1][wave] = gone;
        }
    };
    // The inspected tile to LDS, and what its multiplication has to know.
    struct Stored {
        int ek;
        float fe;                    // factor of the outputs that V's exponent brings
        unsigned long long poison;   // rows (bit = row of the tile) that hold a value that is not finite
        unsigned gone;               // 16-row parts that no page of the pool holds
    };
    auto store = [&](int tile) {
        const unsigned(&y)[kAttnWaves] = s_max[tile & 1];
        const unsigned mx = __builtin_amdgcn_readfirstlane(max_halves(max_halves(y[0], y[1]), max_halves(y[2], y[3])));
        const unsigned long long(&z)[kAttnWaves] = s_bad[tile & 1];
        const unsigned long long bad = z[0] | z[1] | z[2] | z[3];
        Stored r;
        r.poison = (unsigned long long)__builtin_amdgcn_readfirstlane((unsigned)(bad >> 32)) << 32 |
                   (unsigned)__builtin_amdgcn_readfirstlane((unsigned)bad);
        // (Q8: the largest scales, whose quants reach 128)
        r.ek = fit_exp(__uint_as_float(mx << 16)) + (Q8 ? 7 : 0);
        r.fe = raise_exp(ev, fit_exp(__uint_as_float(mx & 0xFFFF0000u)) + (Q8 ? 7 : 0));
        const unsigned(&w)[kAttnWaves] = s_gone[tile & 1];
        r.gone = __builtin_amdgcn_readfirstlane(w[0] | w[1] | w[2] | w[3]);
        t.store(lds + (TWO ? (tile & 1) * kTileU4 : 0), pk::pow2i(-r.ek), pk::pow2i(-ev), wave, lane);
        return r;
    };
    auto multiply = [&](int tile, const Stored& now) {
        if (rw >= x.r1) return;   // no rows of its own: only the loads are its work
        const int k0 = row0 + tile * TR;
        const f16x8* op = reinterpret_cast<const f16x8*>(lds + (TWO ? (tile & 1) * kTileU4 : 0));
        floatx4 st[MT][NU];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int u = 0; u < NU; ++u) st[mt][u] = floatx4{0, 0, 0, 0};
        // (Operand q + 1 is on its way out of LDS while q is multiplied.)
        f16x8 xh = op[lane], xl = op[64 + lane];
#pragma unroll
        for (int q = 0; q < NK; ++q) {
            const f16x8 kh = xh, kl = xl;
            if (q + 1 < NK) {
                xh = op[(2 * q + 2) * 64 + lane];
                xl = op[(2 * q + 3) * 64 + lane];
            }
            __builtin_amdgcn_sched_barrier(kSchedAlu);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                floatx4& y = st[mt][q / KS];
                y = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[mt][q % KS], y, 0, 0, 0);
                y = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[mt][q % KS], y, 0, 0, 0);
                y = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh[mt][q % KS], y, 0, 0, 0);
            }
        }
        auto attended = [&](int mt, int row) {
            return held(k0, now.gone, row) && k0 + row >= first[mt] && k0 + row <= pos[mt];
        };
        const bool plain = k0 >= max(lo, lo_all) && k0 + TR <= min(hi, hi_all) && now.gone == 0 && now.poison == 0;
        f16x8 ph[MT][NU / 2], pl[MT][NU / 2];
        const bool rescale =
            tile_softmax<MT, NU>(a, st, pk::pow2i(now.ek), fq, m, l, alpha, ph, pl, !plain, now.poison, g, attended);
        if (rescale || now.fe != 1.0f) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const float f = alpha[mt] * now.fe;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[mt][d] = o[mt][d] * f;
            }
        }
        xh = op[NK * 2 * 64 + lane];
        xl = op[(NK * 2 + 1) * 64 + lane];
#pragma unroll
        for (int q = 0; q < NU / 2 * DT; ++q) {
            const int w = q / DT, tt = q % DT;
            const f16x8 vh = xh, vl = xl;
            if (q + 1 < NU / 2 * DT) {
                xh = op[(NK + q + 1) * 2 * 64 + lane];
                xl = op[((NK + q + 1) * 2 + 1) * 64 + lane];
            }
            __builtin_amdgcn_sched_barrier(kSchedAlu);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                o[mt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph[mt][w], o[mt][tt], 0, 0, 0);
                o[mt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl[mt][w], o[mt][tt], 0, 0, 0);
                o[mt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph[mt][w], o[mt][tt], 0, 0, 0);
            }
        }
    };
    if (tiles > 0) {
        e = entry(0, part);
        load(0);
        inspect(0);
    }
    __syncthreads();
    if constexpr (TWO) {
        Stored now{};
        if (tiles > 0) {
            now = store(0);
            if (tiles > 1) {
                load(1);
                inspect(1);
            }
        }
        __syncthreads();
        for (int tile = 0; tile < tiles; ++tile) {
            Stored next = now;
            if (tile + 1 < tiles) next = store(tile + 1);   // over the tile that was multiplied before the barrier
            if (tile + 2 < tiles) load(tile + 2);
            multiply(tile, now);
            if (tile + 2 < tiles) inspect(tile + 2);
            now = next;
            __syncthreads();
        }
    } else {
        for (int tile = 0; tile < tiles; ++tile) {
            const Stored now = store(tile);
            if (tile + 1 < tiles) load(tile + 1);
            __syncthreads();
            multiply(tile, now);
            if (tile + 1 < tiles) inspect(tile + 1);
            __syncthreads();
        }
    }
    const float f = ev < -500 ? 0.0f : pk::pow2i(ev);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        l[mt] = dk::lane_step<16, false>(l[mt]);
        l[mt] = dk::lane_step<32, false>(l[mt]);
#pragma unroll
        for (int d = 0; d < DT; ++d) o[mt][d] = o[mt][d] * f;
        store_part<D>(a, x, rw + 16 * mt + n, h, OWN ? a.prefix_splits + split : split, m[mt], l[mt], o[mt], g);
    }
}

// Index of workgroup `id` of `count` (a multiple of 8) in an order that gives each of the chip's 8
// parts, which take the workgroups in turn, a consecutive range: items that read the same rows follow
// one another and share that part's L2.
__device__ __forceinline__ int by_part(int id, int count) { return (id & 7) * (count >> 3) + (id >> 3); }

// Dynamic LDS: the tiles of attn_wide, or the waves' states that attn_narrow joins.
template <int D>
constexpr size_t attn_lds(int wide) {
    return wide ? (size_t)wide_tiles(D) * TilePart<D, false>::kBytes : 2 * (size_t)(D / 4 + 2) * 64 * 4;
}

// WIDE 0: items of 16 query rows; else of 64*WIDE.
template <int D, int WIDE, bool Q8, bool OWN>
__device__ __forceinline__ void attn_item(const AttnArgs& a, uint4* lds, int item, int h, int split) {
    if constexpr (WIDE == 0) attn_narrow<D, Q8, OWN>(a, lds, item, h, split);
    else attn_wide<D, WIDE, Q8, OWN>(a, lds, item, h, split);
}

// Workgroups [0, prefix_wgs) take the prefix items (block of query rows fastest, then split, then KV
// head), the others the own rows' (item of item_sequence, split, KV head): one launch, so the one fills
// what the other leaves of the chip.
template <int D, int WP, int WO, bool Q8>
__global__ __launch_bounds__(kAttnThreads, D > 128 ? 1 : 2) void paged_attn_kernel(AttnArgs a) {
    extern __shared__ uint4 s_dyn4[];
    int id = blockIdx.x;
    if (id < a.prefix_wgs) {
        id = by_part(id, a.prefix_wgs);
        const int item = id % a.prefix_items, hs = id / a.prefix_items;
        if (hs >= a.pool.n_kv_heads * a.prefix_splits) return;
        attn_item<D, WP, Q8, false>(a, s_dyn4, item, hs / a.prefix_splits, hs % a.prefix_splits);
    } else {
        id = by_part(id - a.prefix_wgs, (int)gridDim.x - a.prefix_wgs);
        const int item = id % a.own_items, hs = id / a.own_items;
        if (hs >= a.pool.n_kv_heads * a.own_splits) return;
        attn_item<D, WO, Q8, true>(a, s_dyn4, item, hs / a.own_splits, hs % a.own_splits);
    }
}

// Joins the partials of each query row (prefix splits, then own splits) and applies sink and gate.  Bound by
// memory where there are many rows (4700 tokens of 32 heads of 64, two partials: 17 us, 6.5 TB/s), by its
// start where there are few (3 to 5 us).  A
// group of D/4 threads (four dims each) takes one row's partials; a row with several of them is taken by
// GR groups, every GR-th partial each, all loads in flight together, which meet in LDS in a fixed
// order.  A row with nothing to attend is zero; rows of tokens behind the last sequence are left as they
// are.
constexpr int kJoinThreads = 256;
template <int D>
constexpr int join_groups() { return kJoinThreads / (D / 4); }
// Groups per row for S partials: a power of two that leaves each at most about two.
template <int D>
__host__ __device__ constexpr int join_groups_per_row(int S) {
    int gr = 1;
    while (2 * gr <= join_groups<D>() && 2 * gr < S) gr *= 2;
    return gr;
}
template <int D>
__global__ __launch_bounds__(kJoinThreads) void paged_combine_kernel(AttnArgs a) {
    constexpr int TPR = D / 4, NG = join_groups<D>(), U = 4;
    __shared__ float2 s_ml[NG];
    __shared__ floatx4 s_o[NG][TPR];
    const int S = a.prefix_splits + a.own_splits, SG = join_groups_per_row<D>(S), RPB = NG / SG;
    const int grp = threadIdx.x / TPR, col = threadIdx.x % TPR, sg = grp % SG;
    const long long rows = (long long)a.n_tokens * a.n_heads, row = (long long)blockIdx.x * RPB + grp / SG;
    const int tok = (int)(row / a.n_heads), head = (int)(row % a.n_heads);
    const bool mine = grp < RPB * SG && row < rows && tok >= a.seq_start[0] && tok < a.seq_start[a.n_seqs];
    float M = kNegBig, L = 0.0f;
    floatx4 O = {0, 0, 0, 0};
    if (mine)
        for (int s0 = sg; s0 < S; s0 += SG * U) {
            float2 ml[U];
            floatx4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = s0 + u * SG;
                ml[u] = s < S ? *reinterpret_cast<const float2*>(a.part_ml + (s * rows + row) * 2) : make_float2(kNegBig, 0.0f);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = min(s0 + u * SG, S - 1);
                x[u] = *reinterpret_cast<const floatx4*>(a.part_o + (s * rows + row) * D + 4 * col);
            }
            float mn = M;
#pragma unroll
            for (int u = 0; u < U; ++u) mn = fmaxf(mn, ml[u].x);
            const float f0 = dk::fast_exp2(M - mn);
            M = mn;
            L *= f0;
            O = O * f0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (ml[u].y == 0.0f) continue;   // such a part wrote no outputs
                const float f = dk::fast_exp2(ml[u].x - M);
                L = __builtin_fmaf(ml[u].y, f, L);
#pragma unroll
                for (int i = 0; i < 4; ++i) O[i] = __builtin_fmaf(x[u][i], f, O[i]);
            }
        }
    if (SG > 1) {
        if (grp < NG) {
            if (col == 0) s_ml[grp] = make_float2(M, L);
            s_o[grp][col] = O;
        }
        __syncthreads();
        if (!mine || sg > 0) return;
        const int used = min(S, SG);
        float mn = M;
        for (int k = 1; k < used; ++k) mn = fmaxf(mn, s_ml[grp + k].x);
        const float f0 = dk::fast_exp2(M - mn);
        M = mn;
        L *= f0;
        O = O * f0;
        for (int k = 1; k < used; ++k) {
            const float f = dk::fast_exp2(s_ml[grp + k].x - M);
            L = __builtin_fmaf(s_ml[grp + k].y, f, L);
            const floatx4 x = s_o[grp + k][col];
#pragma unroll
            for (int i = 0; i < 4; ++i) O[i] = __builtin_fmaf(x[i], f, O[i]);
        }
    } else if (!mine) {
        return;
    }
    floatx4 r = {0, 0, 0, 0};
    if (L != 0.0f) {   // (true for NaN as well)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[i] = dk::finish_output(M, L, O[i], a.sinks, a.gate, head,
                                     (long long)tok * a.n_heads * D + (long long)head * D + 4 * col + i);
    }
    *reinterpret_cast<floatx4*>(a.out + (long long)tok * a.out_stride + (long long)head * D + 4 * col) = r;
}

}  // namespace pg
}  // namespace llmp
