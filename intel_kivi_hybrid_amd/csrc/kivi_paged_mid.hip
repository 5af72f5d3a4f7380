// Attention over a paged cache for 17 to 64 query rows per kv head, 16-bit types
// (gfx950 matrix cores): verification passes, short chunks.
//
// Bound by memory like fewer rows, but with as many products as a tile of 32 or
// two of them take.  Each of a workgroup's four waves walks tiles of 32 positions
// of its own, loaded straight into its two LDS buffers, with no barrier between
// the waves; their results are joined in LDS at the end.
#include <hip/hip_runtime.h>

#include "kivi_paged_tile.hpp"

namespace kivi {
namespace {

constexpr int kWaves = 4;
constexpr int kBlock = kWaves * kWave;
constexpr int kTile = 32;

template <int DT, int DP, int GROUPS>
__global__ void __launch_bounds__(kBlock) paged_mid_kernel(PagedLaunch a) {
    using M = TileShape<DP, kTile>;
    constexpr int OS = DP + 4;             // joining rows, padded by one vector
    static_assert(kWaves * 32 * OS * 4 <= kWaves * 4 * M::BYTES, "the join fits the buffers");
    // (two arrays: see the kernel of many rows)
    __shared__ __align__(16) unsigned char buf0[kWaves * 2 * M::BYTES];
    __shared__ __align__(16) unsigned char buf1[kWaves * 2 * M::BYTES];
    __shared__ float join_m[kWaves][32], join_l[kWaves][32];
    __shared__ int join_odd[kWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, col = lane % 32, half = lane / 32;
    const Work w = work_of(a);
    const int end = w.it.kv_end;

    // (two groups' queries and outputs do not fit the registers: every wave has
    // the same queries, and writes them)
    constexpr bool kQLds = GROUPS > 1;
    __shared__ u32x4_t q_lds[kQLds ? GROUPS * M::KS * kWave : 1];
    using Rows = TileRows<DT, DP, kTile, kQLds>;
    Rows rows[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
        rows[g].init(a, w, w.it.row0 + 32 * g, q_lds + g * M::KS * kWave);
    const int all_see = rows[0].all;
    TileLoads<DP, kTile, 1> loads;
    loads.wave = 0;

    bool odd = false;                      // some of the lane's values were not finite
    int t0 = w.it.kv_begin + wave * kTile;
    constexpr int kStep = kWaves * kTile;
    auto step = [&](unsigned char* now, unsigned char* next) {
        now += wave * 2 * M::BYTES;
        next += wave * 2 * M::BYTES;
        wait_loads();
        if (t0 + kTile > min(all_see, end)) odd |= loads.template mend<DT>(now, t0, end);
        wave_sync();
        if (t0 + kStep < end) loads.issue(a, w, next, t0 + kStep, t0 + 2 * kStep);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) rows[g].tile(now, now + M::BYTES, t0, end, a.qscale);
        wave_sync();
        t0 += kStep;
    };

    if (kQLds) wave_sync();
    if (a.D != M::SL * 8) {
        // (vectors behind the head's channels, which no load writes)
        for (int i = threadIdx.x; i < kWaves * 2 * M::BYTES / 16; i += kBlock) {
            reinterpret_cast<u32x4_t*>(buf0)[i] = u32x4_t{0, 0, 0, 0};
            reinterpret_cast<u32x4_t*>(buf1)[i] = u32x4_t{0, 0, 0, 0};
        }
        lds_barrier();
    }
    if (t0 < end) {
        loads.pages_of(a, w, t0);
        loads.issue(a, w, buf0 + wave * 2 * M::BYTES, t0, t0 + kStep);
        while (true) {
            step(buf0, buf1);
            if (t0 >= end) break;
            step(buf1, buf0);
            if (t0 >= end) break;
        }
    }

    // Join the waves: a row's largest maximum, then the rescaled sums, two waves'
    // in each buffer.
    __syncthreads();
    const bool any_odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    if (lane == 0) join_odd[wave] = any_odd;
    float* jo = reinterpret_cast<float*>(wave < 2 ? buf0 : buf1) + wave % 2 * 32 * OS;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        Rows& x = rows[g];
        x.l += __shfl_xor(x.l, 32);
        if (half == 0) {
            join_m[wave][col] = x.m;
            join_l[wave][col] = x.l;
        }
        __syncthreads();
        const float top = fmaxf(fmaxf(join_m[0][col], join_m[1][col]),
                                fmaxf(join_m[2][col], join_m[3][col]));
        const float f = exp2_fast(x.m - top);
#pragma unroll
        for (int cb = 0; cb < M::CB; ++cb) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4_t*>(jo + col * OS + 32 * cb + 8 * i + 4 * half) =
                    f32x4_t{x.O[cb][4 * i], x.O[cb][4 * i + 1], x.O[cb][4 * i + 2],
                            x.O[cb][4 * i + 3]} * f;
        }
        __syncthreads();
        join_waves<DT, DP, 32>(a, w, w.it.row0 + 32 * g, [&](int i) {
            return reinterpret_cast<const float*>(i < 2 ? buf0 : buf1) + i % 2 * 32 * OS;
        }, OS, join_m, join_l, join_odd, kTile);
        if (g + 1 < GROUPS) __syncthreads();
    }
}

template <int DT, int DP>
void launch_rows(const PagedLaunch& a, int kind, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_items * a.Hkv));
    if (kind == kFew32) paged_mid_kernel<DT, DP, 1><<<grid, kBlock, 0, s>>>(a);
    else paged_mid_kernel<DT, DP, 2><<<grid, kBlock, 0, s>>>(a);
}

template <int DT>
void launch_dim(const PagedLaunch& a, int kind, hipStream_t s) {
    if (a.D <= 64) launch_rows<DT, 64>(a, kind, s);
    else if (a.D <= 96) launch_rows<DT, 96>(a, kind, s);
    else launch_rows<DT, 128>(a, kind, s);
}

}  // namespace

void launch_paged_mid(const PagedLaunch& a, int dtype, int kind, hipStream_t s) {
    if (dtype == kSrcBF16) launch_dim<kSrcBF16>(a, kind, s);
    else launch_dim<kSrcF16>(a, kind, s);
}

}  // namespace kivi
