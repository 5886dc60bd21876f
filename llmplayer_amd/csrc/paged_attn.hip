// Instantiation and dispatch of the paged attention (paged_attn_kernels.h).
#include "paged_attn_kernels.h"

namespace llmp {
namespace {

template <int D, int MT, bool Q8, bool OWN>
hipError_t launch(const pg::AttnArgs& a, dim3 grid, hipStream_t st) {
    static const hipError_t allowed =
        hipFuncSetAttribute(reinterpret_cast<const void*>(&pg::paged_attn_kernel<D, MT, Q8, OWN>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, (int)pg::attn_lds<D, MT>());
    if (allowed != hipSuccess) return allowed;
    hipLaunchKernelGGL((pg::paged_attn_kernel<D, MT, Q8, OWN>), grid, dim3(pg::kAttnThreads), (pg::attn_lds<D, MT>()), st, a);
    return hipGetLastError();
}

template <int D, bool Q8, bool OWN>
hipError_t launch_rows(const pg::AttnArgs& a, int mt, hipStream_t st) {
    const int BM = 16 * mt, h = a.pool.n_kv_heads;
    const long long rows = (long long)a.n_tokens * a.group;
    const dim3 grid((unsigned)(OWN ? rows / BM + a.n_seqs : (rows + BM - 1) / BM), h, OWN ? a.own_splits : a.prefix_splits);
    if (mt == 1) return launch<D, 1, Q8, OWN>(a, grid, st);
    if (mt == 2) return launch<D, 2, Q8, OWN>(a, grid, st);
    if constexpr (D <= 128) {
        if (mt == 4) return launch<D, 4, Q8, OWN>(a, grid, st);
    }
    return hipErrorInvalidValue;
}

template <int D>
hipError_t launch_d(const pg::AttnArgs& a, bool q8, bool own, int mt, hipStream_t st) {
    if (q8) return own ? launch_rows<D, true, true>(a, mt, st) : launch_rows<D, true, false>(a, mt, st);
    return own ? launch_rows<D, false, true>(a, mt, st) : launch_rows<D, false, false>(a, mt, st);
}

}  // namespace

hipError_t launch_paged_attn(const pg::AttnArgs& a, int head_dim, bool q8, bool own, int mt, hipStream_t st) {
    switch (head_dim) {
    case 64: return launch_d<64>(a, q8, own, mt, st);
    case 96: return launch_d<96>(a, q8, own, mt, st);
    case 128: return launch_d<128>(a, q8, own, mt, st);
    case 256: return launch_d<256>(a, q8, own, mt, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace llmp
