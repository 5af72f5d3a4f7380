// Attention over a paged fp32 cache (gfx950 matrix cores).
//
// v_mfma_f32_16x16x4_f32 takes one element per lane and operand; with the
// inner index and the output channels in an order of their own, every operand
// comes from memory in vectors of four as it lies, keys and values alike:
//   scores  inner index c of step 4 kk + c at lane group gq: channel 16 kk + 4 gq + c
//   output  row i of tile (cg, c): channel 64 cg + 4 i + c; inner index: token
//           4 gq + i of step i, which is where the scores leave the weights
// so nothing passes through LDS before the waves' results are joined.  A
// workgroup's four waves walk units of 16 positions in turn.  Few rows are bound
// by memory, many by the fp32 products (a sixteenth of the 16-bit rate).
#include <hip/hip_runtime.h>

#include "kivi_paged_attention.hpp"

namespace kivi {
namespace {

constexpr int kWaves = 4;
constexpr int kBlock = kWaves * kWave;
constexpr int kUnit = 16;

__device__ __forceinline__ f32x4_t mfma4(float a, float b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

template <int DP, int RT>
__global__ void __launch_bounds__(kBlock) paged_f32_kernel(PagedLaunch a) {
    constexpr int KK = DP / 16, CG = DP / 64;
    constexpr int OS = DP + 4;             // joining rows, padded by one vector
    __shared__ __align__(16) float jo[kWaves * 16 * OS];
    __shared__ float join_m[kWaves][16], join_l[kWaves][16];
    __shared__ int join_odd[kWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, col = lane % 16, gq = lane / 16;
    const Work w = work_of(a);

    f32x4_t qf[RT][KK], O[RT][CG][4];
    int lim[RT];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = w.it.row0 + 16 * rt + col;
        const bool live = r < w.rows;
        lim[rt] = live ? row_limit(w, r) : 0;
        m[rt] = -FLT_MAX;
        l[rt] = 0.f;
        const float* q = static_cast<const float*>(a.q) + (live ? q_offset(a, w, r) : 0);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int c = 16 * kk + 4 * gq;
            qf[rt][kk] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if (live && c < a.D) qf[rt][kk] = *reinterpret_cast<const f32x4_t*>(q + c);
        }
#pragma unroll
        for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
            for (int c = 0; c < 4; ++c) O[rt][cg][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
    }
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
        f32x4_t s[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) s[rt] = mfma4(kf[kk][c], qf[rt][kk][c], s[rt]);
            }
        }
        page = ahead;
        if (next < end) {
            load_k(next, page);
            ahead = block_page(a, w, next + kWaves * kUnit);
        }
        const bool masked = t0 + kUnit > min(all_see, end);
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
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (masked && t0 + 4 * gq + i >= lim[rt]) s[rt][i] = -INFINITY;
            float mx = fmaxf(fmaxf(s[rt][0], s[rt][1]), fmaxf(s[rt][2], s[rt][3])) * a.qscale;
            if (__builtin_amdgcn_ballot_w64(mx > m[rt] + kMoveMax) != 0) {
                mx = fmaxf(mx, __shfl_xor(mx, 16));
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float to = fmaxf(m[rt], mx), f = exp2_fast(m[rt] - to);
                m[rt] = to;
                l[rt] *= f;
#pragma unroll
                for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) O[rt][cg][c] *= f;
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[rt][i] = exp2_fast(fmaf(s[rt][i], a.qscale, -m[rt]));
                l[rt] += s[rt][i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        O[rt][cg][c] = mfma4(vf[cg][i][c], s[rt][i], O[rt][cg][c]);
                }
            }
        }
        if (next < end) load_v(next, page);
    }

    // Join the waves: a row's largest maximum, then the rescaled sums.
    const bool any_odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    if (lane == 0) join_odd[wave] = any_odd;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] += __shfl_xor(l[rt], 16);
        l[rt] += __shfl_xor(l[rt], 32);
        if (gq == 0) {
            join_m[wave][col] = m[rt];
            join_l[wave][col] = l[rt];
        }
        __syncthreads();
        const float f = exp2_fast(m[rt] - fmaxf(fmaxf(join_m[0][col], join_m[1][col]),
                                                fmaxf(join_m[2][col], join_m[3][col])));
#pragma unroll
        for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<f32x4_t*>(jo + (wave * 16 + col) * OS + 64 * cg + 16 * gq +
                                            4 * r) =
                    f32x4_t{O[rt][cg][0][r], O[rt][cg][1][r], O[rt][cg][2][r], O[rt][cg][3][r]} * f;
        }
        __syncthreads();
        join_waves<kSrcF32, DP, 16, kWaves>(
            a, w, w.it.row0 + 16 * rt, [&](int i) { return jo + i * 16 * OS; }, OS, join_m,
            join_l, (join_odd[0] | join_odd[1] | join_odd[2] | join_odd[3]) != 0, kUnit);
        __syncthreads();
    }
}

template <int DP>
void launch_rows(const PagedLaunch& a, int kind, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_items * a.Hkv));
    // (paged_kind(): the kinds that a head_dim comes with)
    if (kind == kFew16) {
        paged_f32_kernel<DP, 1><<<grid, kBlock, 0, s>>>(a);
    } else {
        if constexpr (DP <= 128) paged_f32_kernel<DP, 2><<<grid, kBlock, 0, s>>>(a);
    }
}

}  // namespace

void launch_paged_f32(const PagedLaunch& a, int kind, hipStream_t s) {
    if (a.D <= 64) launch_rows<64>(a, kind, s);
    else if (a.D <= 128) launch_rows<128>(a, kind, s);
    else launch_rows<256>(a, kind, s);
}

}  // namespace kivi
