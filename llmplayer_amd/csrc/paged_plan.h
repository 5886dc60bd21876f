// Host side of the paged batch in plain C++ (no HIP dependency): the checks of its arguments, the
// launch plan of llmp_paged_attn, and the index rules that host and kernels share.
#pragma once

#include <algorithm>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "host_layout.h"

namespace llmp {

// Sequences of one llmp_paged_tables call: their four tables of offsets are held in LDS (128 KB of
// 160).
constexpr int kTablesMaxSeqs = 8192;

// What a paged handle is, as the checks need it.
struct PagedShape {
    int n_layers, n_pages, page_size, max_seq, n_kv_heads, head_dim, dtype;
    long long width() const { return ((long long)max_seq + page_size - 1) / page_size; }
};

struct PagedMessage {
    char text[256];
    int refuse(int code, const char* fmt, ...) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(text, sizeof text, fmt, ap);
        va_end(ap);
        return code;
    }
};

inline int paged_create_check(const PagedShape& s, PagedMessage& m) {
    if (s.n_layers <= 0 || s.n_pages <= 0 || s.max_seq <= 0 || s.n_kv_heads <= 0 || s.n_kv_heads > 65535)
        return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_create: n_layers=%d n_pages=%d max_seq=%d n_kv_heads=%d",
                        s.n_layers, s.n_pages, s.max_seq, s.n_kv_heads);
    if (s.page_size < 16 || s.page_size > 256 || (s.page_size & (s.page_size - 1)))
        return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_create: page_size %d (16, 32, 64, 128 or 256)", s.page_size);
    if (s.head_dim != 64 && s.head_dim != 96 && s.head_dim != 128 && s.head_dim != 256)
        return m.refuse(LLMP_ERR_UNSUPPORTED, "llmp_paged_create: head_dim %d (supported: 64, 96, 128, 256)", s.head_dim);
    if (s.dtype != LLMP_KV_F32 && s.dtype != LLMP_KV_Q8_0 && s.dtype != LLMP_KV_Q8_0_TRUNC)
        return m.refuse(LLMP_ERR_UNSUPPORTED,
                        "llmp_paged_create: dtype %d (LLMP_KV_F32, LLMP_KV_Q8_0 or LLMP_KV_Q8_0_TRUNC)", s.dtype);
    // Slots are int32, and so is every position that a tile of rows may pass.
    if ((long long)s.n_pages * s.page_size >= (1LL << 31) || s.max_seq > (1 << 30))
        return m.refuse(LLMP_ERR_INVALID_ARG,
                        "llmp_paged_create: n_pages*page_size=%lld (below 2^31), max_seq=%d (up to 2^30)",
                        (long long)s.n_pages * s.page_size, s.max_seq);
    return LLMP_OK;
}

inline int paged_tables_check(const PagedShape& s, int n_seqs, int shared_blocks, int max_tokens, const uint64_t* arrays,
                              int n_arrays, PagedMessage& m) {
    if (n_seqs <= 0 || n_seqs > kTablesMaxSeqs)
        return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_tables: n_seqs=%d (1 to %d)", n_seqs, kTablesMaxSeqs);
    if (max_tokens <= 0 || shared_blocks < 0 || shared_blocks > s.width())
        return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_tables: max_tokens=%d shared_blocks=%d (a table has %lld)",
                        max_tokens, shared_blocks, s.width());
    for (int i = 0; i < n_arrays; ++i)
        if (!arrays[i] || (arrays[i] & 3))
            return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_tables: array %d is null or not 4-byte aligned", i);
    return LLMP_OK;
}

inline int paged_append_check(const PagedShape& s, int n_heads, int n_tokens, uint64_t positions, uint64_t slots,
                              int in_type, uint64_t q, int64_t q_stride, uint64_t k, int64_t k_stride, uint64_t v,
                              int64_t v_stride, uint64_t q_out, int64_t out_stride, PagedMessage& m) {
    const int64_t qd = (int64_t)n_heads * s.head_dim, kvd = (int64_t)s.n_kv_heads * s.head_dim;
    if (n_tokens <= 0) return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_append: n_tokens=%d", n_tokens);
    if (in_type != LLMP_IN_F32 && in_type != LLMP_IN_BF16)
        return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_append: in_type=%d", in_type);
    if (!positions || !q || !q_out || (k == 0) != (v == 0) || (k && !slots))
        return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_append: null buffer (k, v and slots: all or none)");
    if ((positions | slots) & 3 || (q | k | v) & (in_type == LLMP_IN_F32 ? 3 : 1) || q_out & 3)
        return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_append: an array is not aligned to its elements");
    if (q_stride < qd || out_stride < qd || (k && (k_stride < kvd || v_stride < kvd)))
        return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_append: strides %lld/%lld/%lld/%lld below the rows' %lld and %lld",
                        (long long)q_stride, (long long)k_stride, (long long)v_stride, (long long)out_stride,
                        (long long)qd, (long long)kvd);
    if (q_out == q && (in_type != LLMP_IN_F32 || q_stride != out_stride))
        return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_append: in place only for fp32 at equal strides");
    return LLMP_OK;
}

inline int paged_attn_check(const PagedShape& s, int n_heads, int n_seqs, int n_tokens, int prefix_len, int max_len,
                            uint64_t seq_start, uint64_t positions, uint64_t blocks, uint64_t q, int64_t q_stride,
                            uint64_t gate, uint64_t out, int64_t out_stride, PagedMessage& m) {
    const int64_t qd = (int64_t)n_heads * s.head_dim;
    if (n_seqs <= 0 || n_tokens <= 0 || (int64_t)n_tokens * n_heads + n_seqs >= (1LL << 31))
        return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_attn: n_seqs=%d n_tokens=%d", n_seqs, n_tokens);
    if (prefix_len < 0 || prefix_len > s.max_seq || max_len > s.max_seq)
        return m.refuse(LLMP_ERR_OUT_OF_RANGE, "llmp_paged_attn: prefix_len=%d max_len=%d, at most max_seq=%d", prefix_len,
                        max_len, s.max_seq);
    if (!seq_start || !positions || !blocks || !q || !out)
        return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_attn: null buffer");
    if ((seq_start | positions | blocks | gate) & 3 || (q | out) & 15 || (q_stride | out_stride) & 3)
        return m.refuse(LLMP_ERR_INVALID_ARG,
                        "llmp_paged_attn: misaligned tables or gate (4 B), q or out (16 B), or strides (multiples of 4)");
    if (q_stride < qd || out_stride < qd)
        return m.refuse(LLMP_ERR_INVALID_ARG, "llmp_paged_attn: strides %lld/%lld below the rows' %lld", (long long)q_stride,
                        (long long)out_stride, (long long)qd);
    return LLMP_OK;
}

// ---- index rules, shared with the kernels ------------------------------------------------------
// Whether a page, or a slot's page, lies in the pool.
LLMP_HD inline bool paged_page_ok(int page, int n_pages) { return (unsigned)page < (unsigned)n_pages; }
LLMP_HD inline bool paged_slot_ok(int slot, int shift, int n_pages) { return slot >= 0 && (slot >> shift) < n_pages; }

// Largest b < n with s[b] <= x (s ascending, s[0] <= x): among equal starts the last one, which is
// the one that holds something.
LLMP_HD inline int paged_owner(const int* s, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Work items of the own rows: `rows` query rows each, sequence b's from this index on.  It leaves
// room for the ceil(tokens*group / rows) items of every sequence before b without a sum over them:
// floor(x + y) >= floor(x) + ceil(y) - 1.
LLMP_HD inline int paged_item_base(int start, int group, int rows, int b) {
    return (int)((long long)(start > 0 ? start : 0) * group / rows) + b;
}

// ---- launch plan -------------------------------------------------------------------------------
// Query rows of a work item: 16 (wide 0), or 64 or 128 (wide 1, 2).  At head_dim 256 neither the rows
// that a wave of the 16 takes by itself nor the outputs of 128 fit the registers.
LLMP_HD constexpr int paged_item_rows(int wide) { return wide ? 64 * wide : 16; }
constexpr int paged_wide_max(int head_dim) { return head_dim > 128 ? 1 : 2; }
constexpr bool paged_narrow(int head_dim) { return head_dim <= 128; }

struct PagedPlan {
    int prefix_wide, prefix_splits, prefix_tiles;   // item size, splits, 32-row tiles of a split
    int own_wide, own_splits;
};

// n_seqs and max_len (the longest sequence, a bound that the caller gives) set the size of the own
// rows' work: nothing but the speed depends on them.
inline PagedPlan paged_plan(int n_seqs, int n_tokens, int n_heads, int n_kv_heads, int head_dim, int prefix, int max_len,
                            int n_cu) {
    const long long cu = n_cu > 0 ? n_cu : 256, group = n_heads / n_kv_heads, rows = (long long)n_tokens * group;
    auto wide_of = [&](long long r) { return r <= 16 && paged_narrow(head_dim) ? 0 : r <= 64 ? 1 : paged_wide_max(head_dim); };
    auto items_of = [&](long long r, int wide) { return (r + paged_item_rows(wide) - 1) / paged_item_rows(wide); };
    // About two workgroups a CU for the prefix and three for the own rows, whose lengths differ, with at
    // least 4 tiles of 32 rows a split: a workgroup's start and its partial cost about as much (32 query
    // rows of 128 dims against 4001 rows take 26 us so, 31 us from 2 tiles on).  At head_dim 256 a CU holds one
    // workgroup, whose tiles take several times as long: one a CU, from 1 and 2 tiles on (48 sequences
    // of 4 heads against 5000 + 2000 rows: 45 us, 56 us with two and three a CU; 12 of 9 tokens against
    // 300 + 900: 20 us, 31 us from 4 tiles on).
    const bool one = head_dim > 128;
    auto splits_of = [&](long long tiles, long long items, int per_cu, int least) {
        return (int)std::max<long long>(1, std::min((per_cu * cu + items - 1) / items, (tiles + least - 1) / least));
    };
    PagedPlan p{};
    const long long each = (rows + n_seqs - 1) / n_seqs;
    p.prefix_wide = wide_of(rows);
    p.own_wide = wide_of(each);
    if (prefix > 0) {
        const long long tiles = (prefix + 31) / 32;
        const int s = splits_of(tiles, items_of(rows, p.prefix_wide) * n_kv_heads, one ? 1 : 2, one ? 1 : 4);
        p.prefix_tiles = (int)((tiles + s - 1) / s);
        p.prefix_splits = (int)((tiles + p.prefix_tiles - 1) / p.prefix_tiles);
    }
    p.own_splits = splits_of((std::max(max_len - prefix, 1) + 31) / 32, n_seqs * items_of(each, p.own_wide) * n_kv_heads,
                             one ? 1 : 3, one ? 2 : 4);
    return p;
}

}  // namespace llmp
