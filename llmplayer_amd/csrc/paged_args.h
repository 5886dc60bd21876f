// Arguments of the paged batch's launches (paged_kernels.h, paged_attn_kernels.h).
#pragma once

#include "paged_plan.h"

namespace llmp {
namespace pg {

// The pool of one layer.  K and V are pages [page][kv_head][row][D] of page_size = 1 << shift
// rows, fp32, or int8 quants with scales [page][kv_head][row][D/32] (Q8_0).
struct PoolPlanes {
    void* k;
    float* ks;
    void* v;
    float* vs;
    int n_pages, shift, n_kv_heads;
};

struct TablesArgs {
    int n, max_tokens, shared, shift, max_seq, width, n_pages;
    const int* len;
    const int* grow;
    int* free_pages;          // [n_pages], the stack; entries below *n_free are read, above written
    const int* n_free;
    int* blocks;              // [n][width]
    int* len_out;             // may be len
    int* n_free_out;          // may be n_free
    int* seq_start;           // [n + 1]
    int* positions;           // [max_tokens]
    int* slots;               // [max_tokens]
    int* status;
    int* ticket;              // workgroups that have read their inputs (zero between calls)
};

struct AppendArgs {
    PoolPlanes pool;
    const int* positions;
    const int* slots;
    const void* q;            // token t's row at q + t*q_stride elements; fp32 or bf16
    const void* k;
    const void* v;
    long long q_stride, k_stride, v_stride, out_stride;
    float* out;               // rotated queries, fp32
    const float* cos_t;       // [max_seq][half_rope] or nullptr
    const float* sin_t;
    const float* qnw;         // QK-norm weights or nullptr
    const float* knw;
    int n_tokens, n_heads, max_seq, half_rope, rope_type;
    int in_f32, q8, q8_trunc, norm_seq, v_norm;
    float eps;
};

struct AttnArgs {
    PoolPlanes pool;
    const int* seq_start;     // [n_seqs + 1]
    const int* positions;     // [n_tokens]
    const int* blocks;        // [n_seqs][width]
    const float* q;           // [n_tokens] rows of Hq*D, q_stride apart
    const float* gate;        // [n_tokens][Hq*D] or nullptr
    const float* sinks;       // [Hq] log2-domain logits or nullptr
    float* out;
    long long q_stride, out_stride;
    float* part_o;            // [splits][n_tokens*Hq][D]
    float* part_ml;           // [splits][n_tokens*Hq][2]
    int width, n_seqs, n_tokens, n_heads, group, max_seq;
    int prefix, window;
    int prefix_splits, own_splits;   // partials of a row: the prefix's, then its own rows'
    int prefix_tiles;                // 32-row tiles of one prefix split
    int prefix_items, own_items;     // blocks of query rows per (KV head, split)
    int prefix_wgs;                  // workgroups of the prefix items, padded to a multiple of 8
    float qk_scale, softcap, softcap_log2e, inv_softcap;
};

}  // namespace pg
}  // namespace llmp
