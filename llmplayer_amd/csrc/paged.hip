// Launches of the paged batch's tables and append (paged_kernels.h) and of the attention's combine
// (paged_attn_kernels.h).
#include "paged_attn_kernels.h"
#include "paged_kernels.h"

#include <algorithm>

namespace llmp {
namespace {

// LDS above 64 KB has to be asked for, once per kernel.
template <class K>
hipError_t allow_lds(K kernel, size_t bytes) {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <int D, bool F32, bool Q8>
hipError_t launch_append_registers(const pg::AppendArgs& a, int all, hipStream_t st) {
    constexpr int per = pg::kAppendThreads / (D / 8);
    const dim3 grid(a.n_tokens, (all + per - 1) / per), block(pg::kAppendThreads);
    if (a.qnw != nullptr) hipLaunchKernelGGL((pg::paged_append_kernel<D, F32, Q8, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((pg::paged_append_kernel<D, F32, Q8, false>), grid, block, 0, st, a);
    return hipGetLastError();
}

template <int D>
hipError_t launch_append_d(const pg::AppendArgs& a, hipStream_t st) {
    const int all = a.k != nullptr ? a.n_heads + 2 * a.pool.n_kv_heads : a.n_heads;
    if (pg::append_in_registers(a, D)) {
        if (a.in_f32) return a.q8 ? launch_append_registers<D, true, true>(a, all, st) : launch_append_registers<D, true, false>(a, all, st);
        return a.q8 ? launch_append_registers<D, false, true>(a, all, st) : launch_append_registers<D, false, false>(a, all, st);
    }
    hipLaunchKernelGGL((pg::paged_append_lds_kernel<D>), dim3(a.n_tokens, (all + pg::kAppendHeads - 1) / pg::kAppendHeads),
                       dim3(pg::kAppendThreads), 0, st, a);
    return hipGetLastError();
}

template <int D>
hipError_t launch_combine_d(const pg::AttnArgs& a, hipStream_t st) {
    const int per = pg::join_groups<D>() / pg::join_groups_per_row<D>(a.prefix_splits + a.own_splits);
    const long long rows = (long long)a.n_tokens * a.n_heads;
    hipLaunchKernelGGL((pg::paged_combine_kernel<D>), dim3((unsigned)((rows + per - 1) / per)), dim3(pg::kJoinThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_tables(const pg::TablesArgs& a, hipStream_t st) {
    static const hipError_t allowed = allow_lds(pg::paged_tables_kernel, pg::tables_lds(kTablesMaxSeqs));
    if (allowed != hipSuccess) return allowed;
    const long long work = std::max<long long>(a.max_tokens, 8LL * a.n);
    const int wgs = (int)std::min<long long>(256, (work + pg::kTablesThreads - 1) / pg::kTablesThreads);
    hipLaunchKernelGGL(pg::paged_tables_kernel, dim3(std::max(wgs, 1)), dim3(pg::kTablesThreads), pg::tables_lds(a.n), st, a);
    return hipGetLastError();
}

hipError_t launch_paged_append(const pg::AppendArgs& a, int head_dim, hipStream_t st) {
    switch (head_dim) {
    case 64: return launch_append_d<64>(a, st);
    case 96: return launch_append_d<96>(a, st);
    case 128: return launch_append_d<128>(a, st);
    case 256: return launch_append_d<256>(a, st);
    default: return hipErrorInvalidValue;
    }
}

hipError_t launch_paged_combine(const pg::AttnArgs& a, int head_dim, hipStream_t st) {
    switch (head_dim) {
    case 64: return launch_combine_d<64>(a, st);
    case 96: return launch_combine_d<96>(a, st);
    case 128: return launch_combine_d<128>(a, st);
    case 256: return launch_combine_d<256>(a, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace llmp
