// Attention over a paged cache for more than 16 query rows per kv head, 16-bit
// types (gfx950 matrix cores): chunks of prompts, verification passes.
//
// A workgroup takes 128 rows of a kv head, 32 for each of its four waves
// (v_mfma_f32_32x32x16: a wave's operand tile is read from LDS once for all of
// them), and walks the positions in tiles of 64 (32 above 128 channels).  The
// next tile's keys and values go from memory straight to the other of two LDS
// buffers while this one is computed: one barrier per tile, no registers held
// for them, two workgroups per CU.
//
// Many rows are bound by the products: 2048 tokens after 8200, 32/8 heads of 128,
// bf16: 305 to 335 us, 920 to 1015 TFLOP/s, of the 1093 that a large product
// reaches (the matrix cores busy for 47 % of the cycles, at a clock that they bring
// down to 1.8 GHz).  Few rows are bound by memory, whatever the idle waves: 5 tokens
// of 16 sequences, 28/4 heads, 3K positions: 23 us with the join, of 64 at 8K 157 to
// 167, 5.0 TB/s (a kernel of 64 rows of its own, with its waves on both rows and
// positions and three tiles in flight, took 27 and 186).
//
// A workgroup whose sequence has up to 16 rows walks it as kivi_paged_few.hpp does, in
// the same LDS: two chunks of 777 tokens and 30 single ones, 64/8 heads, fp16: 281 us,
// as it took with those in tiles of 128 rows (whose weights had one piece); 63 single
// tokens of 8K beside 5 tokens, 32/8 heads, bf16: 327 and 331.
#include <hip/hip_runtime.h>

#include "kivi_paged_few.hpp"
#include "kivi_paged_tile.hpp"

namespace kivi {
namespace {

constexpr int kWaves = 4;
constexpr int kBlock = kWaves * kWave;

template <int DT, int DP>
__global__ void __launch_bounds__(kBlock, DP <= 128 ? 2 : 1) paged_many_kernel(PagedLaunch a) {
    constexpr int kTile = DP <= 128 ? 64 : 32;         // (what the registers hold)
    using M = TileShape<DP, kTile>;
    // (two arrays, not one: reads of this tile then need not wait for the next
    // one's loads, which the compiler knows to write the other array)
    constexpr int kFewBytes = 2 * Few<DP>::WAVE_BYTES;
    constexpr int kBytes = 2 * M::BYTES > kFewBytes ? 2 * M::BYTES : kFewBytes;
    __shared__ __align__(16) unsigned char buf0[kBytes];
    __shared__ __align__(16) unsigned char buf1[kBytes];
    __shared__ FewJoin join;
    __shared__ int odd;                    // some values were not finite
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, col = lane % 32, half = lane / 32;
    const Work w = work_of(a);
    if (w.rows <= paged_tile_rows(kFew16)) {
        few_rows<DT, DP>(a, w, [&](int i) {
            return (i < 2 ? buf0 : buf1) + i % 2 * Few<DP>::WAVE_BYTES;
        }, join);
        return;
    }
    const int end = w.it.kv_end;

    TileRows<DT, DP, kTile> rows;
    rows.init(a, w, w.it.row0 + 32 * wave);
    const int wg_all = w.it.ctx - w.it.n + 1 + w.it.row0 / w.hg;
    TileLoads<DP, kTile, kWaves> loads;
    loads.init(a, wave);

    int t0 = w.it.kv_begin;
    auto step = [&](unsigned char* now, unsigned char* next) {
        wait_loads();
        if (t0 + kTile > min(wg_all, end) && loads.template mend<DT>(now, t0, end)) odd = 1;
        tile_barrier();
        if (t0 + kTile < end) loads.issue(a, w, next, t0 + kTile, t0 + 2 * kTile);
        if (t0 < rows.last) rows.tile(now, 0, M::BYTES, t0, end, a.qscale);
        t0 += kTile;
    };

    loads.pages_of(a, w, t0);
    if (threadIdx.x == 0) odd = 0;
    tile_barrier();
    loads.issue(a, w, buf0, t0, t0 + kTile);
    while (true) {
        step(buf0, buf1);
        if (t0 >= end) break;
        step(buf1, buf0);
        if (t0 >= end) break;
    }

    float l = rows.l;
    l += __shfl_xor(l, 32);
    const int r = w.it.row0 + 32 * wave + col;
    if (r >= w.rows) return;
    const bool whole = w.it.part < 0;
    const float inv = whole ? inverse_sum(l) : 1.0f;
    const int64_t at = whole ? out_offset(a, w, r) : part_row(a, w, r);
    bool lost = false;
#pragma unroll
    for (int cb = 0; cb < M::CB; ++cb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = 32 * cb + 8 * i + 4 * half;
            if (c >= a.D) continue;
            const f32x16_t& O = rows.O[cb];
            f32x4_t o = {O[4 * i], O[4 * i + 1], O[4 * i + 2], O[4 * i + 3]};
            o *= inv;
            lost |= has_nan(o);
            if (whole) store4<DT>(a.out, at + c, o);
            else *reinterpret_cast<f32x4_t*>(a.part_o + at * a.D + c) = o;
        }
    }
    if (!whole && half == 0)
        *reinterpret_cast<float2*>(a.part_ml + 2 * at) = make_float2(rows.m, l);
    if (odd == 0 && !lost) return;
#pragma unroll 1
    for (int c = 4 * half; c < a.D; c += 8)
        mend_row<DT>(a, w, r, c, rows.m, l, odd != 0, M::TILE);
}

template <int DT>
void launch_dim(const PagedLaunch& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_items * a.Hkv));
    if (a.D <= 64) paged_many_kernel<DT, 64><<<grid, kBlock, 0, s>>>(a);
    else if (a.D <= 96) paged_many_kernel<DT, 96><<<grid, kBlock, 0, s>>>(a);
    else if (a.D <= 128) paged_many_kernel<DT, 128><<<grid, kBlock, 0, s>>>(a);
    else paged_many_kernel<DT, 256><<<grid, kBlock, 0, s>>>(a);
}

}  // namespace

void launch_paged_many(const PagedLaunch& a, int dtype, hipStream_t s) {
    if (dtype == kSrcBF16) launch_dim<kSrcBF16>(a, s);
    else launch_dim<kSrcF16>(a, s);
}

}  // namespace kivi
