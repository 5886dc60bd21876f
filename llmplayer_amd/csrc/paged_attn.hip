// Instantiation and dispatch of the paged attention (paged_attn_kernels.h).
#include "paged_attn_kernels.h"

#include <algorithm>

namespace llmp {
namespace {

template <int D, int WP, int WO, bool Q8>
hipError_t launch(pg::AttnArgs a, hipStream_t st) {
    constexpr size_t lds = std::max(pg::attn_lds<D>(WP), pg::attn_lds<D>(WO));
    // LDS above 64 KB has to be asked for, once per kernel.
    static const hipError_t allowed = hipFuncSetAttribute(reinterpret_cast<const void*>(&pg::paged_attn_kernel<D, WP, WO, Q8>),
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (allowed != hipSuccess) return allowed;
    const long long rows = (long long)a.n_tokens * a.group, h = a.pool.n_kv_heads;
    const long long rp = paged_item_rows(WP), ro = paged_item_rows(WO);
    const long long p = (rows + rp - 1) / rp, o = rows / ro + a.n_seqs;
    const long long pw = (p * h * a.prefix_splits + 7) / 8 * 8, ow = (o * h * a.own_splits + 7) / 8 * 8;
    if (pw + ow >= (1LL << 31)) return hipErrorInvalidValue;
    a.prefix_items = (int)p;
    a.own_items = (int)o;
    a.prefix_wgs = (int)pw;
    hipLaunchKernelGGL((pg::paged_attn_kernel<D, WP, WO, Q8>), dim3((unsigned)(pw + ow)), dim3(pg::kAttnThreads), lds, st, a);
    return hipGetLastError();
}

// The pairs that paged_plan gives: an item of all tokens has at least the rows of one sequence's.
template <int D, bool Q8>
hipError_t launch_rows(const pg::AttnArgs& a, int wp, int wo, hipStream_t st) {
    if constexpr (paged_narrow(D)) {
        if (wp == 0 && wo == 0) return launch<D, 0, 0, Q8>(a, st);
        if (wp == 1 && wo == 0) return launch<D, 1, 0, Q8>(a, st);
    }
    if (wp == 1 && wo == 1) return launch<D, 1, 1, Q8>(a, st);
    if constexpr (paged_wide_max(D) == 2) {
        if (wp == 2 && wo == 0) return launch<D, 2, 0, Q8>(a, st);
        if (wp == 2 && wo == 1) return launch<D, 2, 1, Q8>(a, st);
        if (wp == 2 && wo == 2) return launch<D, 2, 2, Q8>(a, st);
    }
    return hipErrorInvalidValue;
}

template <int D>
hipError_t launch_d(const pg::AttnArgs& a, bool q8, int wp, int wo, hipStream_t st) {
    return q8 ? launch_rows<D, true>(a, wp, wo, st) : launch_rows<D, false>(a, wp, wo, st);
}

}  // namespace

hipError_t launch_paged_attn(const pg::AttnArgs& a, int head_dim, bool q8, int prefix_wide, int own_wide, hipStream_t st) {
    switch (head_dim) {
    case 64: return launch_d<64>(a, q8, prefix_wide, own_wide, st);
    case 96: return launch_d<96>(a, q8, prefix_wide, own_wide, st);
    case 128: return launch_d<128>(a, q8, prefix_wide, own_wide, st);
    case 256: return launch_d<256>(a, q8, prefix_wide, own_wide, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace llmp
