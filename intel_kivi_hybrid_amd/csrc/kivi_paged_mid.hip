// Attention over a paged cache for 17 to 64 query rows per kv head, 16-bit types
// (gfx950 matrix cores): verification passes, short chunks.
//
// Bound by memory like fewer rows, but with as many products as two tiles of 32
// rows take.  A workgroup walks tiles of 64 positions, loaded straight into one of
// four LDS buffers: three tiles are in flight (96 KB of a CU at head_dim 128; a
// tile ahead, as the kernel of many rows has it, left the loads' latency in
// sight: 27 us for 5 tokens of 16 sequences, 28/4 heads, 3K positions).  Wave w
// takes the 32 rows of group w % 2 and the 32 positions of half w / 2 of a tile;
// the halves are joined in LDS at the end.
#include <hip/hip_runtime.h>

#include "kivi_paged_tile.hpp"

namespace kivi {
namespace {

constexpr int kWaves = 4;
constexpr int kBlock = kWaves * kWave;
constexpr int kTile = 64;

template <int DT, int DP>
__global__ void __launch_bounds__(kBlock) paged_mid_kernel(PagedLaunch a) {
    using M = TileShape<DP, kTile>;
    constexpr int OS = DP + 4;             // joining rows, padded by one vector
    // (four arrays: see the kernel of many rows)
    __shared__ __align__(16) unsigned char buf0[2 * M::BYTES];
    __shared__ __align__(16) unsigned char buf1[2 * M::BYTES];
    __shared__ __align__(16) unsigned char buf2[2 * M::BYTES];
    __shared__ __align__(16) unsigned char buf3[2 * M::BYTES];
    __shared__ float join_m[2][2][32], join_l[2][2][32];
    __shared__ int odd;                    // some values were not finite
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, col = lane % 32, half = lane / 32;
    const int group = wave % 2, part = wave / 2;
    const Work w = work_of(a);
    const int end = w.it.kv_end;

    TileRows<DT, DP, 32> rows;
    rows.init(a, w, w.it.row0 + 32 * group);
    const int all_see = w.it.ctx - w.it.n + 1 + w.it.row0 / w.hg;
    TileLoads<DP, kTile, kWaves> loads;
    loads.init(a, wave);
    constexpr int kLoads = 2 * TileLoads<DP, kTile, kWaves>::LD;      // of a tile

    int t0 = w.it.kv_begin;
    auto step = [&](unsigned char* now, unsigned char* last) {
        // (tiles behind this one that were asked for: up to two)
        if (t0 + 2 * kTile < end) wait_loads<2 * kLoads>();
        else if (t0 + kTile < end) wait_loads<kLoads>();
        else wait_loads<0>();
        if (t0 + kTile > min(all_see, end) && loads.template mend<DT>(now, t0, end)) odd = 1;
        tile_barrier();
        if (t0 + 3 * kTile < end) loads.issue(a, w, last, t0 + 3 * kTile, t0 + 4 * kTile);
        const int at = t0 + 32 * part;
        if (at < rows.last)
            rows.tile(now, 32 * part * M::ROW, M::BYTES + 32 * part * M::ROW, at, end, a.qscale);
        t0 += kTile;
    };

    loads.pages_of(a, w, t0);
    if (threadIdx.x == 0) odd = 0;
    // (the queries' loads first: the waits count the tiles' alone)
    wait_loads<0>();
    tile_barrier();
    loads.issue(a, w, buf0, t0, t0 + kTile);
    if (t0 + kTile < end) loads.issue(a, w, buf1, t0 + kTile, t0 + 2 * kTile);
    if (t0 + 2 * kTile < end) loads.issue(a, w, buf2, t0 + 2 * kTile, t0 + 3 * kTile);
    while (true) {
        step(buf0, buf3);
        if (t0 >= end) break;
        step(buf1, buf0);
        if (t0 >= end) break;
        step(buf2, buf1);
        if (t0 >= end) break;
        step(buf3, buf2);
        if (t0 >= end) break;
    }

    // Join the halves: a row's larger maximum, then the rescaled sums, a group in
    // two buffers.
    rows.l += __shfl_xor(rows.l, 32);
    if (half == 0) {
        join_m[group][part][col] = rows.m;
        join_l[group][part][col] = rows.l;
    }
    __syncthreads();
    const float f = exp2_fast(rows.m - fmaxf(join_m[group][0][col], join_m[group][1][col]));
    auto at = [&](int g, int p) {
        unsigned char* b = g == 0 ? (p == 0 ? buf0 : buf1) : (p == 0 ? buf2 : buf3);
        return reinterpret_cast<float*>(b);
    };
    static_assert(32 * OS * 4 <= 2 * M::BYTES, "a wave's join fits a buffer");
    float* jo = at(group, part);
#pragma unroll
    for (int cb = 0; cb < M::CB; ++cb) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4_t*>(jo + col * OS + 32 * cb + 8 * i + 4 * half) =
                f32x4_t{rows.O[cb][4 * i], rows.O[cb][4 * i + 1], rows.O[cb][4 * i + 2],
                        rows.O[cb][4 * i + 3]} * f;
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < 2; ++g)
        join_waves<DT, DP, 32, 2>(a, w, w.it.row0 + 32 * g, [&](int p) { return at(g, p); }, OS,
                                  join_m[g], join_l[g], odd != 0, kTile);
}

template <int DT>
void launch_dim(const PagedLaunch& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_items * a.Hkv));
    if (a.D <= 64) paged_mid_kernel<DT, 64><<<grid, kBlock, 0, s>>>(a);
    else if (a.D <= 96) paged_mid_kernel<DT, 96><<<grid, kBlock, 0, s>>>(a);
    else paged_mid_kernel<DT, 128><<<grid, kBlock, 0, s>>>(a);
}

}  // namespace

void launch_paged_mid(const PagedLaunch& a, int dtype, hipStream_t s) {
    if (dtype == kSrcBF16) launch_dim<kSrcBF16>(a, s);
    else launch_dim<kSrcF16>(a, s);
}

}  // namespace kivi
