// A batch of sequences over one paged KV pool, gfx950: the tables of a step and the append of its
// tokens.  (The attention over the pool: paged_attn_kernels.h.)
#pragma once

#include "paged_args.h"
#include "prefill_kernels.h"

#include <type_traits>

namespace llmp {
namespace pg {

typedef pk::floatx4 floatx4;

// ---- the tables of a step --------------------------------------------------------------------
// Per sequence b with len_b rows and grow_b new tokens (grow_b < 0: it has ended), P rows a page:
//   have = ceil(len/P), need = ceil((len + grow)/P) - have, back = have - shared (ended only);
//   the returned blocks [shared, have) of the ended sequences are pushed on the free stack in
//   order of (b, block), then the blocks [have, have + need) of the others are popped from its top
//   in the same order; seq_start is the exclusive sum of the new tokens, and token i of sequence b
//   has position len_b + i and slot blocks[b][pos / P] * P + pos % P.
constexpr int kTablesThreads = 1024;
constexpr int kTablesPer = kTablesMaxSeqs / kTablesThreads;   // sequences of a thread, at most
inline size_t tables_lds(int n) { return ((size_t)n * 4 + 3) * sizeof(int); }

__device__ __forceinline__ unsigned add_capped(unsigned a, unsigned b) { return min(a + b, 0x7fffffffu); }   // both below 2^31
// Inclusive sum over the wave's lanes, or over its rows of 16 each.
template <bool ROW>
__device__ __forceinline__ unsigned wave_scan(unsigned x) {
    auto step = [&](auto ctrl, auto rows) {   // (0 comes in from outside the row and to masked rows)
        x = add_capped(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
    };
    using All = std::integral_constant<int, 0xF>;
    step(std::integral_constant<int, 0x111>{}, All{});   // row_shr:1, 2, 4, 8
    step(std::integral_constant<int, 0x112>{}, All{});
    step(std::integral_constant<int, 0x114>{}, All{});
    step(std::integral_constant<int, 0x118>{}, All{});
    if constexpr (!ROW) {
        step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});   // row_bcast:15 to rows 1 and 3
        step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});   // row_bcast:31 to rows 2 and 3
    }
    return x;
}

// Every workgroup reads all lengths and forms the three exclusive sums itself (a few KB out of
// L2), then takes its share of the tokens, blocks and returned pages: one launch, no exchange.
// len_out and n_free_out may lie over the inputs, so the workgroup that is last to have read them
// writes both.  Bound by latency: the start, three dependent memory trips, the sums' barriers and, with
// thousands of sequences, the search of a token's one (48 sequences of one token: 4.6 us; 300 with
// prompts of up to 900: 7.1 us, with 64 workgroups in place of 256 8.8 us; 4096 of 4 tokens: 10.5 us).
__global__ __launch_bounds__(kTablesThreads) void paged_tables_kernel(TablesArgs a) {
    extern __shared__ int s_dyn[];
    const int n = a.n, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int* s_len = s_dyn;              // n: the length, or ~length for a sequence that has ended
    int* s_start = s_len + n;        // n + 1
    int* s_need = s_start + n + 1;   // n + 1
    int* s_back = s_need + n + 1;    // n + 1
    __shared__ uint4 s_sum[kTablesThreads / 64];
    __shared__ int s_last;
    const int n_free = *a.n_free;
    const int P1 = (1 << a.shift) - 1;
    // The thread's `per` consecutive sequences, all loads at once.
    const int per = (n + kTablesThreads - 1) / kTablesThreads, i0 = tid * per;
    int l[kTablesPer], grow[kTablesPer];
#pragma unroll
    for (int k = 0; k < kTablesPer; ++k) {
        const int i = min(i0 + k, n - 1);
        if (k < per) {
            l[k] = a.len[i];
            grow[k] = a.grow[i];
        }
    }
    // New tokens, blocks to take and blocks given back: sums that stop at 2^31 - 1, above all that a step
    // may hold.
    unsigned bad = n_free < 0 || n_free > a.n_pages, own[3] = {0, 0, 0};
    int need[kTablesPer], back[kTablesPer];
#pragma unroll
    for (int k = 0; k < kTablesPer; ++k) {
        if (k >= per || i0 + k >= n) break;
        const bool ended = grow[k] < 0;
        const int add = ended ? 0 : grow[k];
        const bool wrong = l[k] < 0 || (long long)l[k] + add > a.max_seq;
        bad |= wrong;
        const int len = wrong ? 0 : l[k];
        grow[k] = wrong ? 0 : add;
        const int have = (int)(((unsigned)len + P1) >> a.shift);
        const int after = (int)(((unsigned)len + (unsigned)grow[k] + P1) >> a.shift);
        need[k] = ended ? 0 : after - have;
        back[k] = ended && !wrong ? max(have - a.shared, 0) : 0;
        l[k] = ended ? ~len : len;
        own[0] = add_capped(own[0], grow[k]);
        own[1] = add_capped(own[1], need[k]);
        own[2] = add_capped(own[2], back[k]);
    }
    unsigned at[3], total[3];
#pragma unroll
    for (int q = 0; q < 3; ++q) at[q] = wave_scan<false>(own[q]);
    bad = __ballot(bad != 0) != 0;
    if (lane == 63) s_sum[wave] = make_uint4(at[0], at[1], at[2], bad);
    __syncthreads();
    const uint4 w = s_sum[lane & (kTablesThreads / 64 - 1)];
    const unsigned part[3] = {w.x, w.y, w.z};
    bad = __ballot(w.w != 0) != 0;
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        const unsigned sums = wave_scan<true>(part[q]);
        total[q] = __builtin_amdgcn_readlane(sums, kTablesThreads / 64 - 1);
        const unsigned before = __builtin_amdgcn_readlane(sums, max(__builtin_amdgcn_readfirstlane(wave) - 1, 0));
        // (an inclusive sum less the thread's own; where sums were capped the step is refused)
        at[q] = at[q] - own[q] + (wave > 0 ? before : 0);
    }
    int status = 0;
    if (bad || (long long)n_free + total[2] > a.n_pages) status = -1;
    else if (total[0] > (unsigned)a.max_tokens) status = -2;
    else if (total[1] > n_free + total[2]) status = (int)(total[1] - n_free - total[2]);
    const bool good = status == 0;
#pragma unroll
    for (int k = 0; k < kTablesPer; ++k) {
        const int i = i0 + k;
        if (k >= per || i >= n) break;
        s_len[i] = l[k];
        s_start[i] = good ? (int)at[0] : 0;
        s_need[i] = good ? (int)at[1] : 0;
        s_back[i] = good ? (int)at[2] : 0;
        at[0] += grow[k];
        at[1] += need[k];
        at[2] += back[k];
    }
    const int tokens = good ? (int)total[0] : 0, taken = good ? (int)total[1] : 0, given = good ? (int)total[2] : 0;
    if (tid == 0) {
        s_start[n] = tokens;
        s_need[n] = taken;
        s_back[n] = given;
    }
    __syncthreads();
    // All inputs of this workgroup are in LDS and registers: the last workgroup to come here may write over
    // them.  (It writes over what the others have read and reads nothing of theirs: no fence; and the
    // answer is not waited for before the end.)
    int ticket = 0;
    if (tid == 0 && gridDim.x > 1) ticket = atomicAdd(a.ticket, 1);
    // Entry e of the stack after the pushes, as the popping tokens see it.
    const int top = n_free + given;
    auto returned = [&](int r) {
        const int b = paged_owner(s_back, n, r);
        return a.blocks[(long long)b * a.width + a.shared + (r - s_back[b])];
    };
    auto popped = [&](int rank) {
        const int e = top - 1 - rank;
        return e < n_free ? a.free_pages[e] : returned(e - n_free);
    };
    const int g0 = blockIdx.x * kTablesThreads + tid, gn = gridDim.x * kTablesThreads;
    for (int i = g0; i <= n; i += gn) a.seq_start[i] = s_start[i];
    for (int i = g0; i < a.max_tokens; i += gn) {
        int pos = -1, slot = -1;
        if (i < tokens) {
            const int b = paged_owner(s_start, n, i);
            const int len = s_len[b];   // not an ended one: those hold no tokens
            pos = len + (i - s_start[b]);
            const int j = pos >> a.shift, have = (int)(((unsigned)len + P1) >> a.shift);
            const int page = j < have ? a.blocks[(long long)b * a.width + j] : popped(s_need[b] + j - have);
            if (paged_page_ok(page, a.n_pages)) slot = (page << a.shift) + (pos & P1);
        }
        a.positions[i] = pos;
        a.slots[i] = slot;
    }
    for (int r = g0; r < taken; r += gn) {
        const int b = paged_owner(s_need, n, r);
        const int have = (int)(((unsigned)s_len[b] + P1) >> a.shift);
        a.blocks[(long long)b * a.width + have + (r - s_need[b])] = popped(r);
    }
    for (int r = g0; r < given; r += gn) a.free_pages[n_free + r] = returned(r);
    if (blockIdx.x == 0 && tid == 0) *a.status = status;
    if (tid == 0) {
        s_last = gridDim.x == 1 || ticket == (int)gridDim.x - 1;
        if (s_last && gridDim.x > 1) *a.ticket = 0;
    }
    __syncthreads();
    if (s_last) {
        for (int i = tid; i < n; i += kTablesThreads) {
            const int l = s_len[i];
            const bool ended = l < 0;
            // (a refused step leaves every length as it was, a wrong one included)
            if (good) a.len_out[i] = ended ? 0 : l + (s_start[i + 1] - s_start[i]);
            else if (a.len_out != a.len) a.len_out[i] = a.len[i];
        }
        if (tid == 0) *a.n_free_out = good ? top - taken : n_free;
    }
}

// ---- rotation and append ---------------------------------------------------------------------
constexpr int kAppendThreads = 256;

__device__ __forceinline__ floatx4 load4_in(const void* p, long long i, int f32) {
    if (f32) return *reinterpret_cast<const floatx4*>(static_cast<const float*>(p) + i);
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const unsigned short*>(p) + i);
    return floatx4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u),
                   __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u)};
}

// Scale of 32 values.  Rounded quants take the largest magnitude times 1/127, one product (within one
// unit in the last place of the division, which moves a quant only at a border between two).  Truncated
// ones take a contiguous cache's division: there the last place decides the quant of the largest value.
constexpr float kInv127 = 1.0f / 127.0f;
__device__ __forceinline__ float q8_scale(float mx, bool trunc) { return trunc ? mx / 127.0f : mx * kInv127; }
__device__ __forceinline__ float block_scale(const float* x, bool trunc) {
    float mx = 0.0f;
    for (int i = 0; i < 32; ++i) mx = fmaxf(mx, fabsf(x[i]));
    return q8_scale(mx, trunc);
}

// Whether a call takes the register kernel: no sum over a head that runs from its first value to its last
// (LLMP_NORM_SEQUENTIAL's and the value norm's), rows that load in fours, and pairs and quantised blocks
// that lie in the lanes as that kernel has them.
inline bool append_in_registers(const AppendArgs& a, int D) {
    const uintptr_t row = a.in_f32 ? 15 : 7;
    const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
    if ((a.qnw != nullptr && a.norm_seq) || a.v_norm) return false;
    if ((at(a.q) | at(a.k) | at(a.v)) & row || at(a.out) & 15) return false;
    if ((a.q_stride | a.k_stride | a.v_stride | a.out_stride | (a.cos_t ? a.half_rope : 0)) & 3) return false;
    const bool halves = a.cos_t != nullptr && a.rope_type != 0;
    return !a.q8 || !halves || a.half_rope <= 16 || (a.half_rope % 32 == 0 && D % 64 == 0);
}

// A thread holds 8 values of a head, two fours that rotate within themselves (adjacent
// pairs) or with each other (halves: [i, i + 4) and [half + i, half + i + 4)), from their load to their store.
// A quantised block of 32 lies in 4 lanes (both fours), or in 8 lanes (the fours of two blocks): its maximum
// takes two or three lane exchanges.  Bound by HBM: every value is read once and written once (4099 tokens
// of 32 + 8 + 8 heads of 128, bf16 to fp32: 26 us, 5.8 TB/s; through LDS 55 us.  1500 tokens of
// 32 + 8 + 8 heads of 64, fp32 to Q8_0: 8 us, through LDS 17 us).
// NORM: a copy of the head in LDS gives the sum of its squares in the decode path's order, 8 chains of
// every eighth value, added up one after the other (4099 tokens of 16 + 8 + 8 heads of 128, fp32: 53 us to
// 28 us a call).
template <int D, bool F32, bool Q8, bool NORM>
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(AppendArgs a) {
    constexpr int TPH = D / 8, HPW = kAppendThreads / TPH;   // threads of a head, heads of a workgroup
    const int t = blockIdx.x, j = threadIdx.x % TPH;
    const int hh = blockIdx.y * HPW + threadIdx.x / TPH;
    const int Hq = a.n_heads, Hkv = a.pool.n_kv_heads;
    const bool live = threadIdx.x < TPH * HPW && hh < (a.k != nullptr ? Hq + 2 * Hkv : Hq);
    if (!NORM && !live) return;
    const bool is_q = hh < Hq, is_k = !is_q && hh < Hq + Hkv;
    const int h = is_q ? hh : is_k ? hh - Hq : hh - Hq - Hkv;
    const bool rope = a.cos_t != nullptr && (is_q || is_k), halves = rope && a.rope_type != 0;
    const int half = rope ? a.half_rope : 0;
    const bool rot = 4 * j < half, apart = halves && rot;
    const int ea = apart ? 4 * j : 8 * j, eb = apart ? half + 4 * j : ea + 4;
    const int pos = a.positions[t];
    floatx4 xa{}, xb{};
    if (live) {
        const void* in = is_q ? a.q : is_k ? a.k : a.v;
        const long long row = (is_q ? a.q_stride : is_k ? a.k_stride : a.v_stride) * t + h * D;
        xa = load4_in(in, row + ea, F32);
        xb = load4_in(in, row + eb, F32);
    }
    if ((unsigned)pos >= (unsigned)a.max_seq) return;   // (the workgroup's: it has one token)
    if constexpr (NORM) {
        constexpr int LD = D + 8;   // the rows of a wave's 8 heads start in banks 8 apart
        __shared__ __align__(16) float s_x[HPW * LD];
        __shared__ float s_r[HPW];
        const int lh = threadIdx.x / TPH;
        floatx4 wa{}, wb{};
        if (live) {
            const float* w = is_q ? a.qnw : a.knw;
            wa = *reinterpret_cast<const floatx4*>(w + ea);
            wb = *reinterpret_cast<const floatx4*>(w + eb);
        }
        if (lh < HPW) {
            *reinterpret_cast<floatx4*>(s_x + lh * LD + ea) = xa;
            *reinterpret_cast<floatx4*>(s_x + lh * LD + eb) = xb;
        }
        __syncthreads();
        for (int c = threadIdx.x; c < HPW * 8; c += kAppendThreads) {   // whole groups of 8 lanes
            const float* x = s_x + (c >> 3) * LD + (c & 7);
            float acc = 0.0f;
#pragma unroll
            for (int k = 0; k < D / 8; ++k) acc = __builtin_fmaf(x[8 * k], x[8 * k], acc);
            float sum = __shfl(acc, 0, 8);
#pragma unroll
            for (int ln = 1; ln < 8; ++ln) sum = sum + __shfl(acc, ln, 8);
            float v = sum / (float)D;
            v = v + a.eps;
            if ((c & 7) == 0) s_r[c >> 3] = 1.0f / (float)__builtin_sqrt((double)v);
        }
        __syncthreads();
        if (!live) return;
        if (is_q || is_k) {
            const float r = s_r[lh];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                xa[i] = (xa[i] * r) * wa[i];
                xb[i] = (xb[i] * r) * wb[i];
            }
        }
    }
    if (rot) {
        const floatx4 c = *reinterpret_cast<const floatx4*>(a.cos_t + (long long)pos * half + 4 * j);
        const floatx4 s = *reinterpret_cast<const floatx4*>(a.sin_t + (long long)pos * half + 4 * j);
        float x0[4], x1[4], y0[4], y1[4];   // the pairs
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const floatx4& x = i < 2 ? xa : xb;
            x0[i] = halves ? xa[i] : x[2 * (i & 1)];
            x1[i] = halves ? xb[i] : x[2 * (i & 1) + 1];
            const float t0 = x0[i] * c[i], t1 = x1[i] * s[i], t2 = x0[i] * s[i], t3 = x1[i] * c[i];
            y0[i] = t0 - t1;
            y1[i] = t2 + t3;
        }
        xa = halves ? floatx4{y0[0], y0[1], y0[2], y0[3]} : floatx4{y0[0], y1[0], y0[1], y1[1]};
        xb = halves ? floatx4{y1[0], y1[1], y1[2], y1[3]} : floatx4{y0[2], y1[2], y0[3], y1[3]};
    }
    if (is_q) {
        float* o = a.out + a.out_stride * t + h * D;
        *reinterpret_cast<floatx4*>(o + ea) = xa;
        *reinterpret_cast<floatx4*>(o + eb) = xb;
        return;
    }
    const int slot = a.slots[t];
    if (!paged_slot_ok(slot, a.pool.shift, a.pool.n_pages)) return;
    const long long to = ((((long long)(slot >> a.pool.shift) * Hkv + h) << a.pool.shift) + (slot & ((1 << a.pool.shift) - 1)));
    void* plane = is_k ? a.pool.k : a.pool.v;
    if constexpr (!Q8) {
        float* o = static_cast<float*>(plane) + to * D;
        *reinterpret_cast<floatx4*>(o + ea) = xa;
        *reinterpret_cast<floatx4*>(o + eb) = xb;
    } else {
        auto largest = [](const floatx4& x) {
            return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
        };
        auto over_four = [](float x) {
            x = fmaxf(x, dk::dpp<dk::kDppQuadXor1>(x));
            return fmaxf(x, dk::dpp<dk::kDppQuadXor2>(x));
        };
        const bool eight = apart && half % 32 == 0;
        float ma = largest(xa), mb = largest(xb);
        if (!eight) ma = mb = fmaxf(ma, mb);
        ma = over_four(ma);
        mb = over_four(mb);
        if (eight) {
            ma = fmaxf(ma, dk::dpp<dk::kDppRowHalfMirror>(ma));
            mb = fmaxf(mb, dk::dpp<dk::kDppRowHalfMirror>(mb));
        }
        const float sa = q8_scale(ma, a.q8_trunc != 0), sb = q8_scale(mb, a.q8_trunc != 0);
        float* so = (is_k ? a.pool.ks : a.pool.vs) + to * (D / 32);
        if ((ea & 31) == 0) so[ea / 32] = sa;
        if (eight && (eb & 31) == 0) so[eb / 32] = sb;
        const float ia = dk::q8_inv_scale(sa), ib = dk::q8_inv_scale(sb);
        unsigned wa = 0, wb = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            wa |= (unsigned)(dk::q8_code(xa[i], ia, a.q8_trunc != 0) & 0xFF) << (8 * i);
            wb |= (unsigned)(dk::q8_code(xb[i], ib, a.q8_trunc != 0) & 0xFF) << (8 * i);
        }
        signed char* o = static_cast<signed char*>(plane) + to * D;
        *reinterpret_cast<unsigned*>(o + ea) = wa;
        *reinterpret_cast<unsigned*>(o + eb) = wb;
    }
}

// The others (sequential norms, odd strides, blocks that do not lie in whole lanes).  One workgroup = (token,
// group of kAppendHeads heads): the heads [h0, h0 + kAppendHeads) of the token's query, key and value
// heads in that order, staged in LDS and prepared with the decode path's functions, so the rows are
// bit-identical to a decode append's (before they are quantised).
constexpr int kAppendHeads = 8;
template <int D>
__global__ __launch_bounds__(kAppendThreads) void paged_append_lds_kernel(AppendArgs a) {
    __shared__ float s_x[kAppendHeads * D], s_acc[kAppendHeads * 8], s_r[kAppendHeads], s_inv[kAppendHeads * (D / 32)];
    const int tid = threadIdx.x, t = blockIdx.x;
    const int Hq = a.n_heads, Hkv = a.pool.n_kv_heads;
    const int pos = a.positions[t], slot = a.k != nullptr ? a.slots[t] : -1;   // (slots may be null without k)
    if ((unsigned)pos >= (unsigned)a.max_seq) return;
    const bool store = a.k != nullptr && paged_slot_ok(slot, a.pool.shift, a.pool.n_pages);
    const int all = a.k != nullptr ? Hq + 2 * Hkv : Hq;
    const int h0 = blockIdx.y * kAppendHeads, h1 = min(h0 + kAppendHeads, all), nh = h1 - h0;
    if (!store && h0 >= Hq) return;
    for (int e = tid; e < nh * D; e += kAppendThreads) {
        const int hh = h0 + e / D, d = e % D;
        const bool is_q = hh < Hq, is_k = hh < Hq + Hkv;
        const void* p = is_q ? a.q : is_k ? a.k : a.v;
        const long long row = is_q ? a.q_stride * t + (long long)hh * D
                              : is_k ? a.k_stride * t + (long long)(hh - Hq) * D
                                     : a.v_stride * t + (long long)(hh - Hq - Hkv) * D;
        s_x[e] = pk::in_val(p, row + d, a.in_f32);
    }
    __syncthreads();
    const long long row = (long long)pos * a.half_rope;
    const dk::HeadPrep hp{a.qnw, a.knw, a.eps, a.cos_t ? a.cos_t + row : nullptr, a.sin_t ? a.sin_t + row : nullptr,
                          a.half_rope, a.rope_type};
    const int nq = max(min(h1, Hq) - h0, 0), nk = max(min(h1, Hq + Hkv) - h0 - nq, 0);
    if (a.norm_seq) {   // the sequential order is the key norm's only
        if (nq) dk::prep_heads_lds<D, kAppendThreads>(s_x, nq, nq, s_acc, s_r, hp, tid);
        if (nk) dk::prep_heads_lds<D, kAppendThreads>(s_x + nq * D, nk, 0, s_acc, s_r, hp, tid, true);
    } else if (nq + nk) {
        dk::prep_heads_lds<D, kAppendThreads>(s_x, nq + nk, nq, s_acc, s_r, hp, tid);
    }
    const int nv = nh - nq - nk;
    if (a.v_norm && nv) {
        float* sv = s_x + (nq + nk) * D;
        if (tid < nv) s_r[tid] = dk::seq_rms_inv<D>(sv + tid * D, a.eps);
        __syncthreads();
        for (int e = tid; e < nv * D; e += kAppendThreads) sv[e] = sv[e] * s_r[e / D];
    }
    __syncthreads();
    for (int e = tid; e < nq * D; e += kAppendThreads) a.out[a.out_stride * t + (long long)h0 * D + e] = s_x[e];
    if (!store || nk + nv == 0) return;
    const int page = slot >> a.pool.shift, r = slot & ((1 << a.pool.shift) - 1);
    auto row_of = [&](int hh) {   // row index of head hh (>= Hq) in its plane
        const int h = (hh - Hq) % Hkv;
        return (((long long)page * Hkv + h) << a.pool.shift) + r;
    };
    if (!a.q8) {
        for (int e = tid + nq * D; e < nh * D; e += kAppendThreads) {
            const int hh = h0 + e / D;
            static_cast<float*>(hh < Hq + Hkv ? a.pool.k : a.pool.v)[row_of(hh) * D + e % D] = s_x[e];
        }
        return;
    }
    constexpr int NB = D / 32;
    for (int b = tid + nq * NB; b < nh * NB; b += kAppendThreads) {
        const int hh = h0 + b / NB;
        const float scale = block_scale(s_x + 32 * b, a.q8_trunc != 0);
        s_inv[b] = dk::q8_inv_scale(scale);
        (hh < Hq + Hkv ? a.pool.ks : a.pool.vs)[row_of(hh) * NB + b % NB] = scale;
    }
    __syncthreads();
    for (int w = tid + nq * D / 4; w < nh * D / 4; w += kAppendThreads) {
        const int e = 4 * w, hh = h0 + e / D;
        unsigned word = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            word |= (unsigned)(dk::q8_code(s_x[e + j], s_inv[e / 32], a.q8_trunc != 0) & 0xFF) << (8 * j);
        *reinterpret_cast<unsigned*>(static_cast<signed char*>(hh < Hq + Hkv ? a.pool.k : a.pool.v) + row_of(hh) * D +
                                     e % D) = word;
    }
}

}  // namespace pg
}  // namespace llmp
