// Attention over pages of 8 bits for more than 16 query rows per kv head: chunks of
// prompts, verification passes.
//
// As kivi_paged_many.hip: a workgroup takes 128 rows of a kv head (256 where the plan says
// so), 32 for each of its four (eight) waves (v_mfma_f32_32x32x16), and walks the positions
// in tiles of 64 (32 above 128 channels) in two LDS buffers.  A tile's codes are loaded
// into registers while the one before is computed, widened there once for all waves and
// written to the other buffer: one barrier per tile.
//
// What bounds it is the sum of two units: a SIMD's two waves do not hide a product behind
// the other's vector instructions (32 products of 16.4 ns and about 390 instructions of 1.4
// for a wave's tile of 64 positions at 128 channels; the products alone are two thirds of
// the time).  Hence little else is done per score: one multiply-add, one exponential, one
// sum, half a packing; scales enter once per block of 16 positions.  A chunk of 2048
// tokens after 8200, 32/8 heads of 128, bf16: 338 to 375 us from card to card (825 to 915
// TFLOP/s) in tiles of 256 rows, 373 in tiles of 128 where those took 345; sixteen times five
// tokens after 3000, 28/4 heads, fp16: 24 us.  At 64 channels a score has half the products
// and as many vector operations, which take 69 % of the cycles beside the products' 25 (four
// chunks of 1024 after 3000, 12/12 heads: 80 to 85 us, 400 to 425 TFLOP/s); at 256 a SIMD has
// one wave, whose operations (44 %) and products (25 %) nothing runs beside (2048 after 8200,
// 28/4 heads: 1005 us, 540 TFLOP/s).
//
// 16-bit types' weights are rounded once here.  A second piece would take the chunk from 338
// to 450 us and the verification from 24.2 to 27.5; with one the verification is off from
// float64 by 0.00024 of the outputs (fp16; their own rounding alone by 0.00021), the chunk
// by 0.0017 (bf16, as its rounding alone).
#include <hip/hip_runtime.h>

#include "kivi_paged8_attention.hpp"
#include "kivi_paged_tile.hpp"

namespace kivi {
namespace {

// How a workgroup's lanes load a tile: a lane takes 16 channels of a token.
template <int DP, int TOKENS, int WAVES>
struct Tile8Loads {
    using M = TileShape<DP, TOKENS>;
    static constexpr int kBlock = WAVES * kWave;
    static constexpr int CH = M::SL / 2;                    // lanes of a token
    static constexpr int LD = TOKENS * CH / kBlock;         // loads of a lane for a tile's keys
    static constexpr int NB = TOKENS / 16;
    int wave;
    int page[LD];                                           // of the loads
    u32x4_t k[LD], v[LD];
    BlockScales<NB> scales;

    // the first position of the block that load i lies in, and its token of the tile
    __device__ __forceinline__ int block_of(int i) const {
        return (i * kBlock + wave * kWave) / CH / 16 * 16;
    }
    __device__ __forceinline__ int token(int i) const {
        return (i * kBlock + (int)threadIdx.x) / CH;
    }
    __device__ __forceinline__ int channel() const { return threadIdx.x % CH * 16; }

    __device__ __forceinline__ void pages_of(const Paged8Launch& a, const Work& w, int t0) {
#pragma unroll
        for (int i = 0; i < LD; ++i) page[i] = block_page_ahead(a, w, t0 + block_of(i));
        scales.pages_of(a, w, t0);
    }
    // Loads the tile at t0 (whose pages are known), then its successor's pages.  (Lanes
    // behind the head's channels bring its first ones: queries are 0 there, and outputs are
    // not stored.)
    __device__ __forceinline__ void issue(const Paged8Launch& a, const Work& w, int t0) {
        const int c = channel() < a.D ? channel() : 0;
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const uint32_t off = token(i) % 16 * a.D + c;
            const int t = t0 + block_of(i), pg = __builtin_amdgcn_readfirstlane(page[i]);
            k[i] = *reinterpret_cast<const u32x4_t*>(
                block_at<uint8_t>(a, w, a.k_pages, pg, t) + off);
            v[i] = *reinterpret_cast<const u32x4_t*>(
                block_at<uint8_t>(a, w, a.v_pages, pg, t) + off);
        }
        scales.load(a, w, t0);
        pages_of(a, w, t0 + TOKENS);
    }
    // Writes the loaded tile, widened, to LDS.
    __device__ __forceinline__ void store(unsigned char* buf) const {
        const int c = channel();
        if (c >= DP) return;                                // (96 channels: six lanes of eight)
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int t = token(i);
            unsigned char* kr = buf + t * M::ROW;
            unsigned char* vr = kr + M::BYTES;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int x = c / 8 + h;
                *reinterpret_cast<u32x4_t*>(kr + ((x ^ M::key_swizzle(t)) << 4)) =
                    operand_of_codes(k[i][2 * h], k[i][2 * h + 1]);
                *reinterpret_cast<u32x4_t*>(vr + ((x ^ M::value_swizzle(t)) << 4)) =
                    operand_of_codes(v[i][2 * h], v[i][2 * h + 1]);
            }
        }
    }
};

// A wave's 32 query rows (lane: row lane % 32) and their softmax state.
template <int DT, int DP, int TOKENS>
struct Tile8Rows {
    using M = TileShape<DP, TOKENS>;
    static constexpr int NQ = query_pieces<DT>();
    static constexpr int NB = TOKENS / 16;
    u32x4_t qf[M::KS][NQ];
    f32x16_t O[M::CB];
    RowState row;
    float qscale;
    uint32_t far_from;
    int lim;                 // positions that the lane's row sees
    int all, last;           // that all, and any, of the 32 rows see

    __device__ __forceinline__ void init(const Paged8Launch& a, const Work& w, int row0) {
        const int lane = threadIdx.x % kWave, half = lane / 32, r = row0 + lane % 32;
        const bool live = r < w.rows;
        lim = live ? row_limit(w, r) : 0;
        row = RowState{-FLT_MAX, 0.f, 0.f};
        qscale = a.qscale * load_query<DT, M::KS>(
            a, live ? q_offset(a, w, r) : 0, live, [&](int ks) { return 16 * ks + 8 * half; },
            [](uint32_t x) { return max(x, (uint32_t)__shfl_xor((int)x, 32)); }, qf);
        far_from = far_keys(qscale);
#pragma unroll
        for (int cb = 0; cb < M::CB; ++cb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) O[cb][i] = 0.f;
        }
        const int base = w.it.ctx - w.it.n + 1;
        all = base + row0 / w.hg;
        last = row0 < w.rows ? min(base + min(row0 + 31, w.rows - 1) / w.hg, w.it.kv_end) : 0;
    }

    // A tile of keys and values in LDS, positions t0 ..
    __device__ __forceinline__ void tile(const unsigned char* buf, const BlockScales<NB>& sc,
                                         int t0, int end) {
        const int lane = threadIdx.x % kWave, col = lane % 32, half = lane / 32;
        f32x16_t s[M::TB];
#pragma unroll
        for (int tb = 0; tb < M::TB; ++tb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[tb][i] = 0.f;
        }
        const uint32_t krow = col * M::ROW + ((half ^ M::key_swizzle(col)) << 4);
#pragma unroll
        for (int ks = 0; ks < M::KS; ++ks) {
#pragma unroll
            for (int tb = 0; tb < M::TB; ++tb) {
                const u32x4_t kf = *reinterpret_cast<const u32x4_t*>(
                    buf + ((krow ^ (32 * ks)) + 32 * tb * M::ROW));
#pragma unroll
                for (int n = NQ - 1; n >= 0; --n) s[tb] = mfma32<kSrcF16>(kf, qf[ks][n], s[tb]);
            }
        }
        if constexpr (NQ == 1) {
            // (key vectors three k-steps ahead of their products)
            constexpr int kReads = M::KS * M::TB, kAhead = 3 * M::TB;
            __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, kAhead, 0);
#pragma unroll
            for (int i = 0; i < kReads - kAhead; ++i) {
                __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, kAhead, 0);
        }
        // score i of 32 tokens tb: token 32 tb + 8 (i / 4) + 4 half + i % 4, of block
        // 2 tb + i / 8
        float units[NB], vs[NB], most[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            units[b] = sc.k(b) * qscale;
            vs[b] = sc.v(b);
        }
        auto each_most = [&] {       // the lane's largest of each block's
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                most[b] = s[b / 2][b % 2 * 8];
#pragma unroll
                for (int i = 1; i < 8; ++i) most[b] = fmaxf(most[b], s[b / 2][b % 2 * 8 + i]);
            }
        };
        auto row_most = [](float x) { return fmaxf(x, __shfl_xor(x, 32)); };
        const bool loud = sc.loud(), far = sc.far(far_from);
        if (t0 + M::TILE > min(all, end) || loud || far) {
            asm volatile("");        // (or every tile does all of this and selects)
#pragma unroll
            for (int tb = 0; tb < M::TB; ++tb) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (t0 + 32 * tb + 8 * (i / 4) + 4 * half + i % 4 >= lim)
                        s[tb][i] = -INFINITY;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                units[b] = above_zero(units[b]);
                if (t0 + 16 * b >= lim) {
                    vs[b] = 0.f;
                    units[b] = FLT_MIN;
                }
            }
            if (__builtin_expect(far, 0)) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[b / 2][b % 2 * 8 + i] *= units[b];
                    units[b] = 1.0f;
                }
            }
            if (__builtin_expect(loud, 0)) {
                each_most();
                drop_far<NB>(vs, most, units, row.m, row_most);
            }
        }
        each_most();
        float f;
        if (move_row<NB>(row, sc, most, units, row_most, f)) {
#pragma unroll
            for (int cb = 0; cb < M::CB; ++cb) O[cb] *= f;
        }
        const float down = exp2_fast(-row.lead);
#pragma unroll
        for (int b = 0; b < NB; ++b) vs[b] *= down;
        // transposed: lanes of 16 take tokens 4 half .. + 3 of 16 channels
        const int t = 4 * half + lane % 16 / 4;
        const int c = lane / 16 % 2 * 2 + lane % 4 / 2;
        const uint32_t vrow = M::BYTES + t * M::ROW + ((c ^ M::value_swizzle(t)) << 4) + lane % 2 * 8;
        constexpr int NP = DT == kSrcF32 ? 2 : 1;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            u32x4_t pf[NP];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = s[b / 2][b % 2 * 8 + 2 * i], y = s[b / 2][b % 2 * 8 + 2 * i + 1];
                const float p0 = exp2_fast(fmaf(x, units[b], -row.m));
                const float p1 = exp2_fast(fmaf(y, units[b], -row.m));
                row.l += p0 + p1;
                if constexpr (NP == 2) {
                    const Pieces w = split_f16(p0 * vs[b], p1 * vs[b]);
                    pf[0][i] = w.hi;
                    pf[1][i] = w.lo;
                } else {
                    pf[0][i] = pack2<kSrcF16>(p0 * vs[b], p1 * vs[b]);
                }
            }
#pragma unroll
            for (int cb = 0; cb < M::CB; ++cb) {
                const uint32_t at = (vrow ^ (64 * cb)) + 16 * b * M::ROW;
                const uint2 lo = read_transposed(buf + at);
                const uint2 hi = read_transposed(buf + (at + 8 * M::ROW));
                const u32x4_t vt = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
                for (int n = NP - 1; n >= 0; --n) O[cb] = mfma32<kSrcF16>(vt, pf[n], O[cb]);
            }
        }
        if constexpr (NP == 1) {
            // A step's products run beside the next one's weights; its values are read a
            // step ahead.
            __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 2 * M::CB, 0);
            __builtin_amdgcn_sched_group_barrier(kSchedValu, 36, 0);
#pragma unroll
            for (int j = 0; j + 1 < NB; ++j) {
#pragma unroll
                for (int cb = 0; cb < M::CB; ++cb) {
                    __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 2, 0);
                    __builtin_amdgcn_sched_group_barrier(kSchedValu, 36 / M::CB, 0);
                }
            }
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, M::CB, 0);
        }
    }
};

template <int DT, int DP, int WAVES>
__global__ void __launch_bounds__(WAVES * kWave, DP <= 128 && DT != kSrcF32 && WAVES == 4 ? 2 : 1)
    paged8_many_kernel(Paged8Launch a) {
    constexpr int kTile = DP <= 128 ? 64 : 32;
    using M = TileShape<DP, kTile>;
    constexpr int kFewBytes = 2 * Few8<DP>::WAVE_BYTES;
    constexpr int kBytes = 2 * M::BYTES > kFewBytes ? 2 * M::BYTES : kFewBytes;
    __shared__ __align__(16) unsigned char buf0[kBytes];
    __shared__ __align__(16) unsigned char buf1[kBytes];
    __shared__ Few8Join join;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, col = lane % 32, half = lane / 32;
    const Work w = work_of(a);
    if constexpr (WAVES == kFew8Waves) {
        if (w.rows <= paged_tile_rows(kFew16)) {
            few8_rows<DT, DP>(a, w, [&](int i) {
                return (i < 2 ? buf0 : buf1) + i % 2 * Few8<DP>::WAVE_BYTES;
            }, join);
            return;
        }
    }
    const int end = w.it.kv_end;
    using R = Tile8Rows<DT, DP, kTile>;
    R rows;
    rows.init(a, w, w.it.row0 + 32 * wave);
    Tile8Loads<DP, kTile, WAVES> loads;
    loads.wave = wave;

    int t0 = w.it.kv_begin;
    loads.pages_of(a, w, t0);
    loads.issue(a, w, t0);
    loads.store(buf0);
    auto step = [&](unsigned char* now, unsigned char* next) {
        const BlockScales<R::NB> scales = loads.scales;
        // (behind it this tile is whole, and the other buffer read by all)
        __syncthreads();
        const bool more = t0 + kTile < end;
        if (more) loads.issue(a, w, t0 + kTile);
        if (t0 < rows.last) rows.tile(now, scales, t0, end);
        if (more) loads.store(next);
        t0 += kTile;
    };
    while (true) {
        step(buf0, buf1);
        if (t0 >= end) break;
        step(buf1, buf0);
        if (t0 >= end) break;
    }

    float l = rows.row.l;
    l += __shfl_xor(l, 32);
    const int r = w.it.row0 + 32 * wave + col;
    if (r >= w.rows) return;
    const bool whole = w.it.part < 0;
    const float f = (whole ? inverse_sum(l) : 1.0f) * exp2_fast(rows.row.lead);
    const int64_t at = whole ? out_offset(a, w, r) : part_row(a, w, r);
#pragma unroll
    for (int cb = 0; cb < M::CB; ++cb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = 32 * cb + 8 * i + 4 * half;
            if (c >= a.D) continue;
            const f32x16_t& O = rows.O[cb];
            f32x4_t o = {O[4 * i], O[4 * i + 1], O[4 * i + 2], O[4 * i + 3]};
            o *= f;
            if (whole) store4<DT>(a.out, at + c, o);
            else *reinterpret_cast<f32x4_t*>(a.part_o + at * a.D + c) = o;
        }
    }
    if (!whole && half == 0)
        *reinterpret_cast<float2*>(a.part_ml + 2 * at) = make_float2(rows.row.m, l);
}

template <int DT, int DP>
void launch_waves(const Paged8Launch& a, bool wide, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_items * a.Hkv));
    if constexpr (DP == 128 && DT != kSrcF32) {
        if (wide) {
            paged8_many_kernel<DT, DP, 8><<<grid, 8 * kWave, 0, s>>>(a);
            return;
        }
    }
    paged8_many_kernel<DT, DP, 4><<<grid, 4 * kWave, 0, s>>>(a);
}

template <int DT>
void launch_dim(const Paged8Launch& a, bool wide, hipStream_t s) {
    if (a.D <= 64) launch_waves<DT, 64>(a, wide, s);
    else if (a.D <= 96) launch_waves<DT, 96>(a, wide, s);
    else if (a.D <= 128) launch_waves<DT, 128>(a, wide, s);
    else launch_waves<DT, 256>(a, wide, s);
}

}  // namespace

void launch_paged8_many(const Paged8Launch& a, int dtype, bool wide, hipStream_t s) {
    if (dtype == kSrcF32) launch_dim<kSrcF32>(a, wide, s);
    else if (dtype == kSrcBF16) launch_dim<kSrcBF16>(a, wide, s);
    else launch_dim<kSrcF16>(a, wide, s);
}

}  // namespace kivi
