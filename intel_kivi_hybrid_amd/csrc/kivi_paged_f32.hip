// Attention over a paged fp32 cache (gfx950 matrix cores).
//
// v_mfma_f32_16x16x4_f32 takes one element per lane and operand; with the
// inner index and the output channels in an order of their own, every operand
// comes in vectors of four as it lies, keys and values alike:
//   scores  inner index c of step 4 kk + c at lane group gq: channel 16 kk + 4 gq + c
//   output  row i of tile (cg, c): channel 64 cg + 4 i + c; inner index: token
//           4 gq + i of step i, which is where the scores leave the weights
// so scores and weights never leave their lanes.  A wave takes 16 rows and units
// of 16 positions.
//
// Up to 16 rows are bound by memory: a workgroup's four waves walk units of their
// own, straight from memory to registers, and join at the end.  64 sequences of 4096
// positions, 32/8 heads of 128: 361 us, 5.9 TB/s.
//
// More are bound by the fp32 products (a sixteenth of the 16-bit rate): each wave
// takes 16 of 64 rows, and all read the same tiles from LDS, the next one on its way
// in registers.  1024 tokens over 8K positions of two sequences, 32/8 heads of 128:
// 113 TFLOP/s of the 154 that a large product reaches; 319 to 638 tokens of each of 5
// sequences, 28/4 heads: 95 to 104 us (with two tiles of 16 rows for each wave and the
// keys split over the waves, each reading all of them from L2: 157).  Small steps stay at a
// third of the rate: 256 workgroups of 36 units take 1.6 us a unit, of 132 1.2 (0.85
// are the products), wherever their operands come from.
#include <hip/hip_runtime.h>

#include "kivi_paged_tile.hpp"

namespace kivi {
namespace {

constexpr int kWaves = 4;
constexpr int kBlock = kWaves * kWave;
constexpr int kUnit = 16;

__device__ __forceinline__ f32x4_t mfma4(float a, float b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// A wave's 16 rows (lane: row lane % 16) and their softmax state.
template <int DP>
struct Rows32 {
    static constexpr int KK = DP / 16, CG = DP / 64;
    f32x4_t qf[KK], O[CG][4];
    float m, l;
    int lim;                  // positions that the lane's row sees

    __device__ __forceinline__ void init(const PagedLaunch& a, const Work& w, int row0) {
        const int lane = threadIdx.x % kWave, gq = lane / 16, r = row0 + lane % 16;
        const bool live = r < w.rows;
        lim = live ? row_limit(w, r) : 0;
        m = -FLT_MAX;
        l = 0.f;
        const float* q = static_cast<const float*>(a.q) + (live ? q_offset(a, w, r) : 0);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int c = 16 * kk + 4 * gq;
            qf[kk] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if (live && c < a.D) qf[kk] = *reinterpret_cast<const f32x4_t*>(q + c);
        }
#pragma unroll
        for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
            for (int c = 0; c < 4; ++c) O[cg][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
    }
    // Scores of the unit at t0 to weights; masked: some row does not see all of it.
    __device__ __forceinline__ void weights(f32x4_t& s, int t0, bool masked, float qscale) {
        const int gq = threadIdx.x % kWave / 16;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (masked && t0 + 4 * gq + i >= lim) s[i] = -INFINITY;
        float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])) * qscale;
        if (__builtin_amdgcn_ballot_w64(mx > m + kMoveMax) != 0) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float to = fmaxf(m, mx), f = exp2_fast(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
                for (int c = 0; c < 4; ++c) O[cg][c] *= f;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] = exp2_fast(fmaf(s[i], qscale, -m));
            l += s[i];
        }
    }
    // The sum of all lanes of a row, in each of them.
    __device__ __forceinline__ void sum() {
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
    }
    // Channels 64 cg + 16 gq + 4 r .. + 3 of the lane's row.
    __device__ __forceinline__ f32x4_t out(int cg, int r) const {
        return f32x4_t{O[cg][0][r], O[cg][1][r], O[cg][2][r], O[cg][3][r]};
    }
};

template <int DP>
__global__ void __launch_bounds__(kBlock) paged_f32_few_kernel(PagedLaunch a) {
    using R = Rows32<DP>;
    constexpr int KK = R::KK, CG = R::CG;
    constexpr int OS = DP + 4;             // joining rows, padded by one vector
    __shared__ __align__(16) float jo[kWaves * 16 * OS];
    __shared__ float join_m[kWaves][16], join_l[kWaves][16];
    __shared__ int join_odd[kWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, col = lane % 16, gq = lane / 16;
    const Work w = work_of(a);
    R rows;
    rows.init(a, w, w.it.row0);
    const int all_see = w.it.ctx - w.it.n + w.it.row0 / w.hg + 1;
    const int end = w.it.kv_end;

    f32x4_t kf[KK], vf[CG][4];
    const bool full = a.D == DP;
    auto load_k = [&](int t0, int page) {
        const float* p = block_at<float>(a, w, a.k_pages, page, t0);
        const uint32_t off = col * a.D + 4 * gq;
        if (full) {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
                kf[kk] = *reinterpret_cast<const f32x4_t*>(p + off + 16 * kk);
        } else {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                kf[kk] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                if (16 * kk + 4 * gq < a.D)
                    kf[kk] = *reinterpret_cast<const f32x4_t*>(p + off + 16 * kk);
            }
        }
    };
    auto load_v = [&](int t0, int page) {
        const float* p = block_at<float>(a, w, a.v_pages, page, t0);
        const uint32_t off = 4 * gq * a.D + 4 * col;
        if (full && t0 + kUnit <= end) {
#pragma unroll
            for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    vf[cg][i] = *reinterpret_cast<const f32x4_t*>(p + off + i * a.D + 64 * cg);
            }
        } else {
#pragma unroll
            for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // (zeros past the end: whatever lies there has weight 0)
                    vf[cg][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                    if (t0 + 4 * gq + i < end && 64 * cg + 4 * col < a.D)
                        vf[cg][i] = *reinterpret_cast<const f32x4_t*>(p + off + i * a.D + 64 * cg);
                }
            }
        }
    };

    bool odd = false;                     // some of the lane's values were not finite
    int t0 = w.it.kv_begin + wave * kUnit, page = 0, ahead = 0;
    if (t0 < end) {
        page = block_page(a, w, t0);
        load_k(t0, page);
        load_v(t0, page);
        ahead = block_page(a, w, t0 + kWaves * kUnit);
    }
    for (; t0 < end; t0 += kWaves * kUnit) {
        const int next = t0 + kWaves * kUnit;
        f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
            for (int c = 0; c < 4; ++c) s = mfma4(kf[kk][c], rows.qf[kk][c], s);
        }
        page = ahead;
        if (next < end) {
            load_k(next, page);
            ahead = block_page(a, w, next + kWaves * kUnit);
        }
        if (t0 + kUnit > all_see) {
#pragma unroll
            for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (!non_finite(vf[cg][i][c])) continue;
                        vf[cg][i][c] = 0.f;
                        odd = true;
                    }
                }
            }
        }
        rows.weights(s, t0, t0 + kUnit > min(all_see, end), a.qscale);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    rows.O[cg][c] = mfma4(vf[cg][i][c], s[i], rows.O[cg][c]);
            }
        }
        if (next < end) load_v(next, page);
    }

    // Join the waves: a row's largest maximum, then the rescaled sums.
    const bool any_odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    if (lane == 0) join_odd[wave] = any_odd;
    rows.sum();
    if (gq == 0) {
        join_m[wave][col] = rows.m;
        join_l[wave][col] = rows.l;
    }
    __syncthreads();
    const float f = exp2_fast(rows.m - fmaxf(fmaxf(join_m[0][col], join_m[1][col]),
                                             fmaxf(join_m[2][col], join_m[3][col])));
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            *reinterpret_cast<f32x4_t*>(jo + (wave * 16 + col) * OS + 64 * cg + 16 * gq + 4 * r) =
                rows.out(cg, r) * f;
    }
    __syncthreads();
    join_waves<kSrcF32, DP, 16, kWaves>(
        a, w, w.it.row0, [&](int i) { return jo + i * 16 * OS; }, OS, join_m, join_l,
        (join_odd[0] | join_odd[1] | join_odd[2] | join_odd[3]) != 0, kUnit);
}

// Tiles of 16 KB of keys and values (32 KB above 128 channels), and how a
// workgroup's lanes bring them from memory to LDS: load i of wave w covers ROWS
// tokens of one block of 16 positions.  Slot c ^ (t % 16) holds vector c of token t:
// the 16 tokens of a key read, and the 16 vectors of a value read, lie on all the
// banks.
template <int DP>
struct Tile32 {
    static constexpr int TILE = DP <= 64 ? 32 : 16, SL = DP / 4, ROW = SL * 16;
    static constexpr int BYTES = TILE * ROW, ROWS = kWave / SL, LD = TILE / ROWS / kWaves;
    static_assert(SL >= 16 && LD * ROWS * kWaves == TILE && 16 % ROWS == 0, "whole loads");
    int wave;
    int page[LD];
    f32x4_t k[LD], v[LD];

    __device__ __forceinline__ int row(int i) const {
        return (i * kWaves + wave) * ROWS + threadIdx.x % kWave / SL;
    }
    __device__ __forceinline__ int block_of(int i) const {
        return (i * kWaves + wave) * ROWS / 16 * 16;
    }
    __device__ __forceinline__ void pages_of(const PagedLaunch& a, const Work& w, int t0) {
#pragma unroll
        for (int i = 0; i < LD; ++i) page[i] = block_page(a, w, t0 + block_of(i));
    }
    // Loads the tile at t0, whose pages are known, and the next one's pages.
    __device__ __forceinline__ void load(const PagedLaunch& a, const Work& w, int t0) {
        const int c = threadIdx.x % SL * 4;
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int t = t0 + block_of(i);
            const uint32_t off = row(i) % 16 * a.D + c;
            k[i] = v[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if (c < a.D) {
                k[i] = *reinterpret_cast<const f32x4_t*>(
                    block_at<float>(a, w, a.k_pages, page[i], t) + off);
                v[i] = *reinterpret_cast<const f32x4_t*>(
                    block_at<float>(a, w, a.v_pages, page[i], t) + off);
            }
        }
        pages_of(a, w, t0 + TILE);
    }
    // Of a tile at t0 that some row does not see to its end: zeros for values behind
    // the end (weight 0 of whatever lies there) and for non-finite ones.  Whether
    // there was one of the latter.
    __device__ __forceinline__ bool mend(int t0, int end) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const bool behind = t0 + row(i) >= end;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!behind && !non_finite(v[i][j])) continue;
                any |= !behind;
                v[i][j] = 0.f;
            }
        }
        return any;
    }
    __device__ __forceinline__ void store(unsigned char* buf) const {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int t = row(i), at = t * ROW + ((threadIdx.x % SL ^ t % 16) << 4);
            *reinterpret_cast<f32x4_t*>(buf + at) = k[i];
            *reinterpret_cast<f32x4_t*>(buf + BYTES + at) = v[i];
        }
    }
};

template <int DP>
__global__ void __launch_bounds__(kBlock, DP <= 128 ? 3 : 2) paged_f32_many_kernel(PagedLaunch a) {
    using R = Rows32<DP>;
    using T = Tile32<DP>;
    constexpr int kTile = T::TILE;
    __shared__ __align__(16) unsigned char buf[2][2 * T::BYTES];
    __shared__ int odd;                    // some values were not finite
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, col = lane % 16, gq = lane / 16;
    const Work w = work_of(a);
    const int end = w.it.kv_end, row0 = w.it.row0 + 16 * wave;
    T tiles;
    tiles.wave = wave;
    int t0 = w.it.kv_begin;
    tiles.pages_of(a, w, t0);
    R rows;
    rows.init(a, w, row0);
    tiles.load(a, w, t0);
    const int see = w.it.ctx - w.it.n + 1;
    const int all_see = see + w.it.row0 / w.hg;               // all rows of the workgroup
    const int all = see + row0 / w.hg;                        // the wave's
    const int last = row0 < w.rows ? min(see + min(row0 + 15, w.rows - 1) / w.hg, end) : 0;
    if (threadIdx.x == 0) odd = 0;
    lds_barrier();
#pragma unroll 1
    for (int b = 0; t0 < end; b ^= 1, t0 += kTile) {
        // (the other buffer is read until the barrier, this one no longer)
        if (t0 + kTile > min(all_see, end) && tiles.mend(t0, end)) odd = 1;
        tiles.store(buf[b]);
        lds_barrier();
        if (t0 + kTile < end) tiles.load(a, w, t0 + kTile);
        const unsigned char* kb = buf[b];
        const unsigned char* vb = kb + T::BYTES;
#pragma unroll 1
        for (int at = t0; at < min(t0 + kTile, last); at += kUnit) {
            // (two sums: a product need not wait for the one before; operands are read
            // three steps of four products ahead: left to itself the compiler waits
            // for each of them)
            constexpr int kAheadReads = 3, kValues = 4 * R::CG;
            f32x4_t s = {0.f, 0.f, 0.f, 0.f}, s1 = s, vf[kValues];
#pragma unroll
            for (int kk = 0; kk < R::KK; ++kk) {
                const f32x4_t kf = *reinterpret_cast<const f32x4_t*>(
                    kb + col * T::ROW + (((4 * kk + gq) ^ col) << 4));
#pragma unroll
                for (int c = 0; c < 4; c += 2) {
                    s = mfma4(kf[c], rows.qf[kk][c], s);
                    s1 = mfma4(kf[c + 1], rows.qf[kk][c + 1], s1);
                }
            }
            auto value = [&](int j) {
                const int t = 4 * gq + j / R::CG, c = 16 * (j % R::CG) + col;
                vf[j] = *reinterpret_cast<const f32x4_t*>(vb + t * T::ROW + ((c ^ t) << 4));
            };
#pragma unroll
            for (int j = 0; j < kAheadReads; ++j) value(j);
            __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, kAheadReads, 0);
#pragma unroll
            for (int i = 0; i < R::KK; ++i) {
                __builtin_amdgcn_sched_group_barrier(kSchedMfma, 4, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 1, 0);
            }
            s += s1;
            rows.weights(s, at, at + kUnit > min(all, end), a.qscale);
#pragma unroll
            for (int j = 0; j < kValues; ++j) {
                if (j + kAheadReads < kValues) value(j + kAheadReads);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    rows.O[j % R::CG][c] =
                        mfma4(vf[j][c], s[j / R::CG], rows.O[j % R::CG][c]);
            }
#pragma unroll
            for (int j = kAheadReads; j < kValues; ++j) {
                __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedMfma, 4, 0);
            }
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, 4 * kAheadReads, 0);
            kb += kUnit * T::ROW;
            vb += kUnit * T::ROW;
        }
    }

    rows.sum();
    const int r = row0 + col;
    if (r >= w.rows) return;
    const float inv = w.it.part < 0 ? inverse_sum(rows.l) : 1.0f;
    bool lost = false;
#pragma unroll
    for (int cg = 0; cg < R::CG; ++cg) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = 64 * cg + 16 * gq + 4 * i;
            if (c >= a.D) continue;
            const f32x4_t o = rows.out(cg, i) * inv;
            lost |= has_nan(o);
            store_row<kSrcF32>(a, w, r, c, o, rows.m, rows.l);
        }
    }
    if (odd == 0 && !lost) return;
#pragma unroll 1
    for (int c = 16 * gq; c < a.D; c += c % 16 < 12 ? 4 : 52)
        mend_row<kSrcF32>(a, w, r, c, rows.m, rows.l, odd != 0, kTile);
}

template <int DP>
void launch_rows(const PagedLaunch& a, int kind, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_items * a.Hkv));
    if (kind == kFew16) paged_f32_few_kernel<DP><<<grid, kBlock, 0, s>>>(a);
    else paged_f32_many_kernel<DP><<<grid, kBlock, 0, s>>>(a);
}

}  // namespace

void launch_paged_f32(const PagedLaunch& a, int kind, hipStream_t s) {
    if (a.D <= 64) launch_rows<64>(a, kind, s);
    else if (a.D <= 128) launch_rows<128>(a, kind, s);
    else launch_rows<256>(a, kind, s);
}

}  // namespace kivi
