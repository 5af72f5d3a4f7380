// Attention over pages of 8 bits in steps whose sequences bring up to 16 query rows to a
// kv head each: single tokens (few8_rows() of kivi_paged8_attention.hpp).
//
// Memory-bound: each of a workgroup's four waves walks units of 64 positions of its own
// (32 above 128 channels), the next unit's codes in flight, and meets the others once, at
// the end.  64 single tokens of 4K to 8K positions, 32/8 heads of 128, bf16: 151 us for
// 811 MB, 5.4 TB/s (a stream that only reads 6.4); 287 in pages of 16 bits.  With both
// products on bf16 operands, whose widening takes a fifth more operations, the vector units
// bound it at 293 us.
#include <hip/hip_runtime.h>

#include "kivi_paged8_attention.hpp"

namespace kivi {
namespace {

constexpr int kBlock = kFew8Waves * kWave;

template <int DT, int DP>
__global__ void __launch_bounds__(kBlock, 2) paged8_few_kernel(Paged8Launch a) {
    __shared__ __align__(16) unsigned char lds[kFew8Waves * Few8<DP>::WAVE_BYTES];
    __shared__ Few8Join join;
    few8_rows<DT, DP>(a, work_of(a), [&](int i) { return lds + i * Few8<DP>::WAVE_BYTES; }, join);
}

template <int DT>
void launch_dim(const Paged8Launch& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_items * a.Hkv));
    if (a.D <= 64) paged8_few_kernel<DT, 64><<<grid, kBlock, 0, s>>>(a);
    else if (a.D <= 96) paged8_few_kernel<DT, 96><<<grid, kBlock, 0, s>>>(a);
    else if (a.D <= 128) paged8_few_kernel<DT, 128><<<grid, kBlock, 0, s>>>(a);
    else paged8_few_kernel<DT, 256><<<grid, kBlock, 0, s>>>(a);
}

}  // namespace

void launch_paged8_few(const Paged8Launch& a, int dtype, hipStream_t s) {
    if (dtype == kSrcF32) launch_dim<kSrcF32>(a, s);
    else if (dtype == kSrcBF16) launch_dim<kSrcBF16>(a, s);
    else launch_dim<kSrcF16>(a, s);
}

}  // namespace kivi
