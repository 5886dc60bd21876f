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
// One wave takes 32 rows of the pool at a time against all MT tiles of 16 query rows, straight from
// memory to registers: S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_16x16x32_f16.  Lane
// (n = lane % 16, g = lane / 16) holds A[n][8g + j], B[8g + j][n] and D[4g + i][n]:
//  - K: lane (n, g) loads dims 32s + 8g .. +7 of rows n and 16 + n: the A operands as they are.
//  - S^T's result lies as (query n, rows 4g + i), which is the B operand of the second product when
//    its 32 rows are taken in the order {4g .. 4g+3, 16 + 4g .. 16 + 4g + 3}.
//  - V: lane (n, g) loads dims 64c + 4n .. +3 of those 8 rows, 256 contiguous bytes a row.  Column t
//    of the four is one A operand whose 16 output rows stand for dims 64c + 4n + t: the transposition
//    costs nothing.
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

constexpr int kAttnThreads = 256, kAttnWaves = kAttnThreads / 64;
constexpr int kTile = 32;            // pool rows a wave takes at a time
constexpr float kPShift = 4.0f;      // 2^(s - m + 4): small probabilities keep their fp16 bits
constexpr float kNegBig = dk::kNegBig;

// ---- one tile of 32 rows in registers --------------------------------------------------------
template <int D, bool Q8>
struct Tile;

// Address of row r of a page of plane p (elements of `unit` values per row).
template <class T>
__device__ __forceinline__ const T* page_row(const void* p, const PoolPlanes& pool, int page, int h, int row, int unit) {
    return static_cast<const T*>(p) + ((((long long)page * pool.n_kv_heads + h) << pool.shift) + row) * unit;
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
            const float* x = page_row<float>(p.k, p, u ? page1 : page0, h, (u ? r1 : r0) + n, D) + 8 * g;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                k[u][s][0] = *reinterpret_cast<const floatx4*>(x + 32 * s);
                k[u][s][1] = *reinterpret_cast<const floatx4*>(x + 32 * s + 4);
            }
        }
    }
    __device__ __forceinline__ void load_v(const PoolPlanes& p, int page0, int page1, int h, int r0, int r1, int n, int g) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float* x = page_row<float>(p.v, p, j < 4 ? page0 : page1, h, (j < 4 ? r0 : r1) + 4 * g + (j & 3), D);
#pragma unroll
            for (int c = 0; c < NC; ++c) v[j][c] = *reinterpret_cast<const floatx4*>(x + 64 * c + 4 * n);
            if constexpr (REM) {
                const float2 w = *reinterpret_cast<const float2*>(x + 64 * NC + 2 * n);
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
                    for (int e = 0; e < 4; ++e) x = fmaxf(x, fabsf(k[u][s][q][e]));
        return x;
    }
    __device__ __forceinline__ float max_v() const {
        float x = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) x = fmaxf(x, fabsf(v[j][c][e]));
            if constexpr (REM) x = fmaxf(x, fmaxf(fabsf(vr[j][0]), fabsf(vr[j][1])));
        }
        return x;
    }
    // Value with what no row holds (keep 0, else ~0) and what is not finite taken out; worst: the
    // largest magnitude's bits before that.
    static __device__ __forceinline__ float clean(float x, unsigned keep, unsigned& worst) {
        const unsigned b = __float_as_uint(x) & keep, m = b & 0x7FFFFFFFu;
        worst = max(worst, m);
        return __uint_as_float(b & (unsigned)((int)(m - 0x7F800000u) >> 31));   // no lane mask per value
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
    __device__ __forceinline__ void k_values(int u, int s, float f, float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = k[u][s][e >> 2][e & 3] * f;
    }
    // Output tile tt's column of the 8 rows.
    __device__ __forceinline__ void v_values(int tt, float f, float (&x)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (tt < 4 * NC ? v[j][tt >> 2][tt & 3] : vr[j][(tt - 4 * NC) & 1]) * f;
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
            const signed char* x = page_row<signed char>(p.k, p, u ? page1 : page0, h, (u ? r1 : r0) + n, D) + 8 * g;
            const float* sc = page_row<float>(p.ks, p, u ? page1 : page0, h, (u ? r1 : r0) + n, KS);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                k[u][s] = *reinterpret_cast<const uint2*>(x + 32 * s);
                ks[u][s] = sc[s];
            }
        }
    }
    __device__ __forceinline__ void load_v(const PoolPlanes& p, int page0, int page1, int h, int r0, int r1, int n, int g) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int page = j < 4 ? page0 : page1, row = (j < 4 ? r0 : r1) + 4 * g + (j & 3);
            const signed char* x = page_row<signed char>(p.v, p, page, h, row, D);
            const float* sc = page_row<float>(p.vs, p, page, h, row, KS);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                v[j][c] = *reinterpret_cast<const unsigned*>(x + 64 * c + 4 * n);
                vs[j][c] = sc[2 * c + (n >> 3)];
            }
            if constexpr (REM) {
                v[j][NC] = *reinterpret_cast<const unsigned short*>(x + 64 * NC + 2 * n);
                vs[j][NC] = sc[2 * NC];
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
    __device__ __forceinline__ void k_values(int u, int s, float f, float (&x)[8]) const {
        const float sc = ks[u][s] * f;
        const unsigned w[2] = {k[u][s].x, k[u][s].y};
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)(signed char)(w[e >> 2] >> (8 * (e & 3)) & 0xFF) * sc;
    }
    __device__ __forceinline__ void v_values(int tt, float f, float (&x)[8]) const {
        const int c = tt < 4 * NC ? tt >> 2 : NC, t = tt < 4 * NC ? tt & 3 : tt - 4 * NC;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)(signed char)(v[j][c] >> (8 * t) & 0xFF) * (vs[j][c] * f);
    }
};

// hi = fp16(x), lo = fp16(x - hi): one conversion a pair and one mixed-precision multiply-add a value.
// In plain operations, not in assembly: the compiler has to see who writes an operand of a matrix
// instruction, which must not read it within two wait states.  Two opaque steps keep its hands off the
// arithmetic: `hi` as it was rounded is what lo starts from (a product may be rounded to fp16 in one
// step for the one and in two for the other), and x - hi stays a multiply-add by a -1 it cannot see.
__device__ __forceinline__ void split8(const float (&x)[8], f16x8& hi, f16x8& lo) {
    float minus = -1.0f;
    asm("" : "+s"(minus));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        unsigned u = pk::pack_f16(x[2 * j], x[2 * j + 1]);
        asm("" : "+v"(u));
        const pk::f16x2 h = __builtin_bit_cast(pk::f16x2, u);
        const pk::f16x2 l = {(_Float16)__builtin_fmaf((float)h[0], minus, x[2 * j]),
                             (_Float16)__builtin_fmaf((float)h[1], minus, x[2 * j + 1])};
        hi[2 * j] = h[0];
        hi[2 * j + 1] = h[1];
        lo[2 * j] = l[0];
        lo[2 * j + 1] = l[1];
    }
}

// Largest value over the wave.
__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, dk::dpp<dk::kDppQuadXor1>(x));
    x = fmaxf(x, dk::dpp<dk::kDppQuadXor2>(x));
    x = dk::lane_step<4, true>(x);
    x = dk::lane_step<8, true>(x);
    x = dk::lane_step<16, true>(x);
    x = dk::lane_step<32, true>(x);
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
// Exponent e with max * 2^-e in [2^13, 2^14) (0 for 0; clamped so that 2^e and 2^-e are normal).
__device__ __forceinline__ int fit_exp(float mx) {
    const int b = (int)(__float_as_uint(mx) >> 23) - 127 - 13;
    return mx == 0.0f ? 0 : max(min(b, 120), -120);
}

// The rows of a tile (bit = row) that the lanes' bits name: bk the K rows n and 16 + n, bv the V
// rows 4g + i and 16 + 4g + i.
__device__ __forceinline__ unsigned tile_rows(unsigned bk, unsigned bv, int n, int g) {
    unsigned x = (bk & 1u) << n | (bk >> 1) << (16 + n) | (bv & 15u) << (4 * g) | (bv >> 4) << (16 + 4 * g);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) x |= __shfl_xor(x, off);
    return __builtin_amdgcn_readfirstlane(x);
}

template <int D, int MT>
constexpr size_t attn_lds() {
    const size_t q = (size_t)MT * (D / 32) * 2 * 64 * 16, x = 2 * (size_t)MT * (D / 4 + 2) * 64 * 4;
    return q > x ? q : x;
}

// The sequence of work item `item` of an own-rows launch (paged_item_base).
__device__ __forceinline__ int item_sequence(const AttnArgs& a, int item, int BM, int lane) {
    int lo = 0, len = a.n_seqs;
    while (len > 1) {
        const int step = (len + 63) / 64, b = lo + lane * step;
        const bool in = lane * step < len && paged_item_base(a.seq_start[b], a.group, BM, b) <= item;
        const int c = max((int)__popcll(__ballot(in)), 1) - 1;
        lo += c * step;
        len = min(step, len - c * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// OWN: blockIdx = (item of item_sequence, KV head, split of the own rows).
// Else: blockIdx = (block of 16*MT query rows of all tokens, KV head, split of the prefix).
template <int D, int MT, bool Q8, bool OWN>
__global__ __launch_bounds__(kAttnThreads) void paged_attn_kernel(AttnArgs a) {
    using T = Tile<D, Q8>;
    constexpr int KS = D / 32, DT = D / 16, BM = 16 * MT, NC = D / 64, REM = D % 64 / 32;
    extern __shared__ uint4 s_dyn4[];
    __shared__ int s_pos[BM], s_first[BM];
    __shared__ float s_fq[BM];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const int h = blockIdx.y, split = blockIdx.z;
    const int G = a.group;
    // Query rows of the item: token tok0 + r / G, head h*G + r % G for r in [r0, r1).
    int tok0 = 0, r0, r1;
    const int* blk = a.blocks;
    if constexpr (OWN) {
        const int b = item_sequence(a, blockIdx.x, BM, lane);
        const int st = min(max(a.seq_start[b], 0), a.n_tokens), en = min(max(a.seq_start[b + 1], st), a.n_tokens);
        tok0 = st;
        r0 = ((int)blockIdx.x - paged_item_base(st, G, BM, b)) * BM;
        r1 = min((en - st) * G, r0 + BM);
        if (r0 < 0) return;
        blk += (long long)b * a.width;
    } else {
        r0 = blockIdx.x * BM;
        r1 = min(min(max(a.seq_start[a.n_seqs], 0), a.n_tokens) * G, r0 + BM);
    }
    if (r0 >= r1) return;

    // Queries: wave w prepares the tiles w, w + 4, ...: scaled, divided by a power of two of their
    // own, split and laid out as the B operands take them.
    uint4* s_q = s_dyn4;
    for (int mt = wave; mt < MT; mt += kAttnWaves) {
        const int r = r0 + 16 * mt + n;
        const bool have = r < r1;
        const int rr = have ? r : r0, tok = tok0 + rr / G, head = h * G + rr % G;
        const float* q = a.q + (long long)tok * a.q_stride + (long long)head * D + 8 * g;
        int pos = a.positions[tok];
        float x[KS][8], mx = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) pk::load8(q + 32 * s, x[s]);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[s][e] *= a.qk_scale;
                mx = fmaxf(mx, fabsf(x[s][e]));
            }
        mx = dk::lane_step<16, true>(mx);
        mx = dk::lane_step<32, true>(mx);
        const int e = finite_bits(__float_as_uint(mx)) ? fit_exp(mx) : 0;
        const float f = pk::pow2i(-e);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[s][i] *= f;
            f16x8 hi, lo;
            split8(x[s], hi, lo);
            s_q[((mt * KS + s) * 2 + 0) * 64 + lane] = __builtin_bit_cast(uint4, hi);
            s_q[((mt * KS + s) * 2 + 1) * 64 + lane] = __builtin_bit_cast(uint4, lo);
        }
        if (g == 0) {
            const bool live = have && (unsigned)pos < (unsigned)a.max_seq;
            s_pos[16 * mt + n] = live ? pos : -1;
            s_first[16 * mt + n] = !live ? 0x7fffffff : a.window > 0 ? max(pos + 1 - a.window, 0) : 0;
            s_fq[16 * mt + n] = pk::pow2i(e);
        }
    }
    __syncthreads();
    // Rows that some query attends, and those that all do.
    int hi_any = -1, lo_any = 0x7fffffff, hi_all = 0x7fffffff, lo_all = 0;
    {
        const int r = lane < BM ? lane : 0;
        const int p = s_pos[r], f = s_first[r];
        hi_any = p;
        lo_any = f;
        const bool real = r0 + r < r1;
        hi_all = real ? p : 0x7fffffff;
        lo_all = real ? f : 0;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            hi_any = max(hi_any, __shfl_xor(hi_any, off));
            lo_any = min(lo_any, __shfl_xor(lo_any, off));
            hi_all = min(hi_all, __shfl_xor(hi_all, off));
            lo_all = max(lo_all, __shfl_xor(lo_all, off));
        }
        hi_any = __builtin_amdgcn_readfirstlane(hi_any) + 1;
        lo_any = __builtin_amdgcn_readfirstlane(lo_any);
        hi_all = __builtin_amdgcn_readfirstlane(hi_all) + 1;
        lo_all = __builtin_amdgcn_readfirstlane(lo_all);
    }
    // The item's rows [lo, hi) and this split's tiles of them.
    const int lo = OWN ? max(a.prefix, lo_any) : lo_any;
    const int hi = OWN ? hi_any : min(a.prefix, hi_any);
    int t_lo, t_hi;
    if constexpr (OWN) {
        const int first = min(lo, hi) / kTile, all = lo < hi ? (hi + kTile - 1) / kTile - first : 0;
        const int per = (all + a.own_splits - 1) / a.own_splits;
        t_lo = first + min(split * per, all);
        t_hi = first + min(split * per + per, all);
    } else {
        t_lo = max(split * a.prefix_tiles, min(lo, hi) / kTile);
        t_hi = lo < hi ? min(split * a.prefix_tiles + a.prefix_tiles, (hi + kTile - 1) / kTile) : t_lo;
    }

    float m[MT], l[MT], fq[MT];
    floatx4 o[MT][DT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m[mt] = kNegBig;
        l[mt] = 0.0f;
        fq[mt] = s_fq[16 * mt + n];
#pragma unroll
        for (int d = 0; d < DT; ++d) o[mt][d] = floatx4{0, 0, 0, 0};
    }
    int ev = -1000;   // exponent that V is divided by: grows with the largest value seen
    const int rmask = (1 << a.pool.shift) - 1;
    const f16x8* qf = reinterpret_cast<const f16x8*>(s_q);
    T t;
    for (int tile = t_lo + wave; tile < t_hi; tile += kAttnWaves) {
        const int k0 = tile * kTile;
        // Each half tile of 16 rows lies in one page.  A block entry outside the pool holds no rows.
        int page[2];
        bool there[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int j = (k0 + 16 * u) >> a.pool.shift;
            page[u] = j < a.width ? __builtin_amdgcn_readfirstlane(blk[j]) : -1;
            there[u] = paged_page_ok(page[u], a.pool.n_pages);
            if (!there[u]) page[u] = 0;
        }
        const int r0k = k0 & rmask, r1k = (k0 + 16) & rmask;
        t.load_k(a.pool, page[0], page[1], h, r0k, r1k, n, g);
        t.load_v(a.pool, page[0], page[1], h, r0k, r1k, n, g);
        const bool inner = k0 >= lo && k0 + kTile <= hi && there[0] && there[1];
        const bool plain = inner && k0 >= lo_all && k0 + kTile <= hi_all;
        unsigned poison = 0;   // rows (bit = row of the tile) that hold a value that is not finite
        if (!plain) {
            unsigned ok = 0;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int key = k0 + 16 * u + n;
                ok |= (unsigned)(there[u] && key >= lo && key < hi) << u;
            }
            const unsigned bk = t.clean_k(ok);
            ok = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = k0 + 16 * (j >> 2) + 4 * g + (j & 3);
                ok |= (unsigned)(there[j >> 2] && key >= lo && key < hi) << j;
            }
            const unsigned bv = t.clean_v(ok);
            if (__ballot(bk | bv) != 0) poison = tile_rows(bk, bv, n, g);
        }
        float mk = wave_max(t.max_k());
        if (!finite_bits(__float_as_uint(mk))) {   // an infinity must not take the other rows' bits
            poison |= tile_rows(t.clean_k(3u), 0, n, g);
            mk = wave_max(t.max_k());
        }
        const int ek = fit_exp(mk);
        const float fk = pk::pow2i(-ek), fkr = pk::pow2i(ek);
        // S^T of both half tiles, in units of 2^(ek + eq).
        floatx4 st[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) st[mt][0] = st[mt][1] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                float x[8];
                t.k_values(u, s, fk, x);
                f16x8 kh, kl;
                split8(x, kh, kl);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const f16x8 qh = qf[((mt * KS + s) * 2 + 0) * 64 + lane], ql = qf[((mt * KS + s) * 2 + 1) * 64 + lane];
                    st[mt][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh, st[mt][u], 0, 0, 0);
                    st[mt][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql, st[mt][u], 0, 0, 0);
                    st[mt][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh, st[mt][u], 0, 0, 0);
                }
            }
        // V's exponent: the largest of the wave's tiles so far; what is summed follows it.
        float mv = wave_max(t.max_v());
        if (!finite_bits(__float_as_uint(mv))) {
            poison |= tile_rows(0, t.clean_v(255u), n, g);
            mv = wave_max(t.max_v());
        }
        const int evt = fit_exp(mv);
        float fo = 1.0f;
        if (evt > ev) {
            fo = ev < -500 ? 0.0f : pk::pow2i(max(ev - evt, -126));
            ev = evt;
        }
        const float fv = pk::pow2i(-ev);
        f16x8 ph[MT], pl[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float f = fkr * fq[mt];
            float mx = kNegBig;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = st[mt][u][i] * f;
                    if (a.softcap > 0.0f) x = a.softcap_log2e * tanhf(x * a.inv_softcap);
                    if (!plain || poison) {
                        const int key = k0 + 16 * u + 4 * g + i;
                        const bool ok = there[u] && key >= lo && key < hi && key >= s_first[16 * mt + n] && key <= s_pos[16 * mt + n];
                        if (poison >> (16 * u + 4 * g + i) & 1) x = __builtin_nanf("");
                        x = ok ? x : -__builtin_inff();
                    }
                    st[mt][u][i] = x;
                    mx = fmaxf(mx, x);
                }
            mx = dk::lane_step<16, true>(mx);
            mx = dk::lane_step<32, true>(mx);
            const float mn = fmaxf(m[mt], mx - kPShift);
            const float alpha = dk::fast_exp2(m[mt] - mn);
            m[mt] = mn;
            float sum = 0.0f;
            float p[8];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[4 * u + i] = dk::fast_exp2(st[mt][u][i] - mn);
                    sum += p[4 * u + i];
                }
            l[mt] = __builtin_fmaf(l[mt], alpha, sum);
            split8(p, ph[mt], pl[mt]);
            const float ao = alpha * fo;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[mt][d] = o[mt][d] * ao;
        }
#pragma unroll
        for (int tt = 0; tt < DT; ++tt) {
            float x[8];
            t.v_values(tt, fv, x);
            f16x8 vh, vl;
            split8(x, vh, vl);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                o[mt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph[mt], o[mt][tt], 0, 0, 0);
                o[mt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl[mt], o[mt][tt], 0, 0, 0);
                o[mt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph[mt], o[mt][tt], 0, 0, 0);
            }
        }
    }
    // l is a sum over the lane's own rows so far: the four groups of a query together.
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        l[mt] = dk::lane_step<16, false>(l[mt]);
        l[mt] = dk::lane_step<32, false>(l[mt]);
        const float f = ev < -500 ? 0.0f : pk::pow2i(ev);
#pragma unroll
        for (int d = 0; d < DT; ++d) o[mt][d] = o[mt][d] * f;
    }
    // The waves' states, in a fixed order: 2 into 0 and 3 into 1, then 1 into 0.
    __syncthreads();   // the last reads of the queries
    constexpr int XS = MT * (D / 4 + 2);
    float* xch = reinterpret_cast<float*>(s_dyn4);
#pragma unroll
    for (int round = 0; round < 2; ++round) {
        const int from = round == 0 ? 2 : 1, count = round == 0 ? 2 : 1;
        if (wave >= from && wave < from + count) {
            float* x = xch + (size_t)(wave - from) * XS * 64 + lane;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                x[(mt * (D / 4 + 2) + 0) * 64] = m[mt];
                x[(mt * (D / 4 + 2) + 1) * 64] = l[mt];
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[(mt * (D / 4 + 2) + 2 + 4 * d + i) * 64] = o[mt][d][i];
            }
        }
        __syncthreads();
        if (wave < count) {
            const float* x = xch + (size_t)wave * XS * 64 + lane;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const float m2 = x[(mt * (D / 4 + 2) + 0) * 64], l2 = x[(mt * (D / 4 + 2) + 1) * 64];
                const float mn = fmaxf(m[mt], m2), f1 = dk::fast_exp2(m[mt] - mn), f2 = dk::fast_exp2(m2 - mn);
                m[mt] = mn;
                l[mt] = l[mt] * f1 + l2 * f2;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[mt][d][i] = o[mt][d][i] * f1 + x[(mt * (D / 4 + 2) + 2 + 4 * d + i) * 64] * f2;
            }
        }
        __syncthreads();
    }
    if (wave != 0) return;
    const long long rows = (long long)a.n_tokens * a.n_heads;
    const long long part = OWN ? a.prefix_splits + split : split;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int r = r0 + 16 * mt + n;
        if (r >= r1) continue;
        const long long row = (long long)(tok0 + r / G) * a.n_heads + h * G + r % G;
        if (g == 0) *reinterpret_cast<float2*>(a.part_ml + (part * rows + row) * 2) = make_float2(m[mt], l[mt]);
        float* po = a.part_o + (part * rows + row) * D;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<floatx4*>(po + 64 * c + 16 * g + 4 * i) =
                    floatx4{o[mt][4 * c][i], o[mt][4 * c + 1][i], o[mt][4 * c + 2][i], o[mt][4 * c + 3][i]};
        if constexpr (REM) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float2*>(po + 64 * NC + 2 * (4 * g + i)) = make_float2(o[mt][4 * NC][i], o[mt][4 * NC + 1][i]);
        }
    }
}

// Joins the partials of each query row (prefix splits, then own splits, in that order) and applies
// sink and gate.  A thread takes four dims of one row.  A row with nothing to attend is zero; rows
// of tokens behind the last sequence are left as they are.
constexpr int kJoinThreads = 256;
template <int D>
__global__ __launch_bounds__(kJoinThreads) void paged_combine_kernel(AttnArgs a) {
    constexpr int TPR = D / 4, RPB = kJoinThreads / TPR;
    const int local = threadIdx.x / TPR, col = threadIdx.x % TPR;
    const long long rows = (long long)a.n_tokens * a.n_heads;
    const long long row = (long long)blockIdx.x * RPB + local;
    if (local >= RPB || row >= rows) return;
    const int tok = (int)(row / a.n_heads), head = (int)(row % a.n_heads);
    if (tok < a.seq_start[0] || tok >= a.seq_start[a.n_seqs]) return;
    const int S = a.prefix_splits + a.own_splits;
    float M = kNegBig;
    for (int s = 0; s < S; ++s) M = fmaxf(M, a.part_ml[(s * rows + row) * 2]);
    float L = 0.0f;
    floatx4 O = {0, 0, 0, 0};
    for (int s = 0; s < S; ++s) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (s * rows + row) * 2);
        if (ml.y == 0.0f) continue;
        const float f = dk::fast_exp2(ml.x - M);
        L = __builtin_fmaf(ml.y, f, L);
        const floatx4 x = *reinterpret_cast<const floatx4*>(a.part_o + (s * rows + row) * D + 4 * col);
#pragma unroll
        for (int i = 0; i < 4; ++i) O[i] = __builtin_fmaf(x[i], f, O[i]);
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
