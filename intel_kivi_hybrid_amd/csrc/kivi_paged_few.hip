// Attention over a paged cache in steps whose sequences bring up to 16 query rows to a
// kv head each, 16-bit types: the launch of kivi_paged_few.hpp.
#include <hip/hip_runtime.h>

#include "kivi_paged_few.hpp"

namespace kivi {
namespace {

constexpr int kBlock = kFewWaves * kWave;

template <int DT, int DP>
__global__ void __launch_bounds__(kBlock) paged_few_kernel(PagedLaunch a) {
    __shared__ __align__(16) unsigned char lds[kFewWaves * Few<DP>::WAVE_BYTES];
    __shared__ FewJoin join;
    few_rows<DT, DP>(a, work_of(a), [&](int i) { return lds + i * Few<DP>::WAVE_BYTES; }, join);
}

template <int DT>
void launch_dim(const PagedLaunch& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_items * a.Hkv));
    if (a.D <= 64) paged_few_kernel<DT, 64><<<grid, kBlock, 0, s>>>(a);
    else if (a.D <= 96) paged_few_kernel<DT, 96><<<grid, kBlock, 0, s>>>(a);
    else if (a.D <= 128) paged_few_kernel<DT, 128><<<grid, kBlock, 0, s>>>(a);
    else paged_few_kernel<DT, 256><<<grid, kBlock, 0, s>>>(a);
}

}  // namespace

void launch_paged_few(const PagedLaunch& a, int dtype, hipStream_t s) {
    if (dtype == kSrcBF16) launch_dim<kSrcBF16>(a, s);
    else launch_dim<kSrcF16>(a, s);
}

}  // namespace kivi
