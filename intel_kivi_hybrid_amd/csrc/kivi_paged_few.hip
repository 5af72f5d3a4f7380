// Attention over a paged cache for up to 64 query rows per kv head, 16-bit
// types (gfx950 matrix cores): single tokens, verification passes.
//
// Such calls read every key and value once for a few products: memory-bound.
// A workgroup's four waves walk the item's positions in units of 32, each wave
// units of its own with no barrier between them, its next unit's keys and values
// in flight while it computes.  Keys go from memory into the A operand of
// v_mfma_f32_16x16x32 as they lie (a lane takes 8 channels of one token); values
// need the token as the inner index and pass through the wave's own LDS, from
// which they are read transposed.  The waves' results are joined in LDS at the
// end; splits of a context are joined by a second launch.
#include <hip/hip_runtime.h>

#include "kivi_paged_attention.hpp"

namespace kivi {
namespace {

constexpr int kWaves = 4;
constexpr int kBlock = kWaves * kWave;
constexpr int kUnit = 32;

template <int DT, int DP, int RT>
struct Few {
    static constexpr int KS = DP / 32;            // k-steps of a score
    static constexpr int CB = DP / 16;            // blocks of 16 output channels
    static constexpr int CH = DP / 8;             // 16-byte vectors of a token
    static constexpr int VL = kUnit * CH / kWave; // value loads of a lane per unit
    // (32 bytes of padding per token: the 16 rows of a transposed read then
    // start on 8 different bank groups, as few as their 512 bytes need)
    static constexpr int VS = DP * 2 + 32;
    static constexpr int V_BYTES = kUnit * VS;
    // joining the waves: fp32 rows, padded by one vector
    static constexpr int OS = DP + 4;
    static constexpr int JOIN_BYTES = kWaves * 16 * OS * 4;
    static constexpr int LDS = kWaves * V_BYTES > JOIN_BYTES ? kWaves * V_BYTES : JOIN_BYTES;
};

template <int DT, int DP, int RT>
__global__ void __launch_bounds__(kBlock) paged_few_kernel(PagedLaunch a) {
    using F = Few<DT, DP, RT>;
    __shared__ __align__(16) unsigned char lds[F::LDS];
    __shared__ float join_m[kWaves][RT * 16], join_l[kWaves][RT * 16];
    __shared__ int join_odd[kWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const int col = lane % 16, gq = lane / 16;
    const Work w = work_of(a);
    unsigned char* vl = lds + wave * F::V_BYTES;

    u32x4_t qf[RT][F::KS];
    int lim[RT];
    float m[RT], l[RT];
    f32x4_t O[RT][F::CB];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = w.it.row0 + 16 * rt + col;
        const bool live = r < w.rows;
        lim[rt] = live ? row_limit(w, r) : 0;
        m[rt] = -FLT_MAX;
        l[rt] = 0.f;
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + (live ? q_offset(a, w, r) : 0);
#pragma unroll
        for (int ks = 0; ks < F::KS; ++ks) {
            const int c = 32 * ks + 8 * gq;
            qf[rt][ks] = u32x4_t{0, 0, 0, 0};
            if (live && c < a.D) qf[rt][ks] = *reinterpret_cast<const u32x4_t*>(q + c);
        }
#pragma unroll
        for (int cb = 0; cb < F::CB; ++cb) O[rt][cb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    // positions that every row sees, and whether some row is short of the end
    const int all_see = w.it.ctx - w.it.n + w.it.row0 / w.hg + 1;
    const int end = w.it.kv_end;

    u32x4_t kf[2][F::KS], vf[F::VL];
    // pages of the unit's two blocks
    struct Pages { int p[2]; };
    auto pages_of = [&](int t0) {
        return Pages{{block_page(a, w, t0), block_page(a, w, t0 + 16)}};
    };
    const bool full = a.D == DP;
    auto load_k = [&](int t0, Pages pg) {
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
            const uint16_t* p = block_at<uint16_t>(a, w, a.k_pages, pg.p[tb], t0 + 16 * tb);
            const uint32_t off = col * a.D + 8 * gq;
            if (full) {
#pragma unroll
                for (int ks = 0; ks < F::KS; ++ks)
                    kf[tb][ks] = *reinterpret_cast<const u32x4_t*>(p + off + 32 * ks);
            } else {
#pragma unroll
                for (int ks = 0; ks < F::KS; ++ks) {
                    kf[tb][ks] = u32x4_t{0, 0, 0, 0};
                    if (32 * ks + 8 * gq < a.D)
                        kf[tb][ks] = *reinterpret_cast<const u32x4_t*>(p + off + 32 * ks);
                }
            }
        }
    };
    auto load_v = [&](int t0, Pages pg) {
        const bool whole = full && t0 + kUnit <= end;
#pragma unroll
        for (int i = 0; i < F::VL; ++i) {
            constexpr int kPer = F::VL / 2;               // loads of a block
            const int at = i % kPer * kWave + lane, t = at / F::CH, c = at % F::CH * 8;
            const int tb = i / kPer;
            const uint16_t* p = block_at<uint16_t>(a, w, a.v_pages, pg.p[tb], t0 + 16 * tb);
            const uint32_t off = t * a.D + c;
            if (whole) {
                vf[i] = *reinterpret_cast<const u32x4_t*>(p + off);
            } else {
                // (zeros past the end: whatever lies there has weight 0)
                vf[i] = u32x4_t{0, 0, 0, 0};
                if (t0 + 16 * tb + t < end && c < a.D)
                    vf[i] = *reinterpret_cast<const u32x4_t*>(p + off);
            }
        }
    };

    bool odd = false;                     // some of the lane's values were not finite
    int t0 = w.it.kv_begin + wave * kUnit;
    Pages ahead = {{0, 0}};
    if (t0 < end) {
        const Pages pg = pages_of(t0);
        load_k(t0, pg);
        load_v(t0, pg);
        ahead = pages_of(t0 + kWaves * kUnit);
    }
    for (; t0 < end; t0 += kWaves * kUnit) {
        const int next = t0 + kWaves * kUnit;
        f32x4_t s[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
                s[rt][tb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < F::KS; ++ks)
                    s[rt][tb] = mfma16<DT>(kf[tb][ks], qf[rt][ks], s[rt][tb]);
            }
        }
        const Pages pg = ahead;
        if (next < end) {
            load_k(next, pg);
            ahead = pages_of(next + kWaves * kUnit);
        }
        const bool masked = t0 + kUnit > min(all_see, end);
        if (t0 + kUnit > all_see) {
#pragma unroll
            for (int i = 0; i < F::VL; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t x = finite_part<DT>(vf[i][j]);
                    odd |= x != vf[i][j];
                    vf[i][j] = x;
                }
            }
        }
        wave_sync();                      // the last unit's reads, before these writes
#pragma unroll
        for (int i = 0; i < F::VL; ++i) {
            const int at = i * kWave + lane;
            *reinterpret_cast<u32x4_t*>(vl + at / F::CH * F::VS + at % F::CH * 16) = vf[i];
        }
        if (next < end) load_v(next, pg);

        u32x4_t pf[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = s[rt][i / 4][i % 4];
                if (masked && t0 + 16 * (i / 4) + 4 * gq + i % 4 >= lim[rt]) x[i] = -INFINITY;
            }
            float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                             fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            mx *= a.qscale;
            if (__builtin_amdgcn_ballot_w64(mx > m[rt] + kMoveMax) != 0) {
                mx = fmaxf(mx, __shfl_xor(mx, 16));
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float to = fmaxf(m[rt], mx), f = exp2_fast(m[rt] - to);
                m[rt] = to;
                l[rt] *= f;
#pragma unroll
                for (int cb = 0; cb < F::CB; ++cb) O[rt][cb] *= f;
            }
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = exp2_fast(fmaf(x[i], a.qscale, -m[rt]));
                l[rt] += p[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) pf[rt][i] = pack2<DT>(p[2 * i], p[2 * i + 1]);
        }
        wave_sync();
        // rows of a transposed read: tokens 4 gq .. + 3, and 16 further on, in the
        // order in which a lane holds the weights
        const unsigned char* vr = vl + (4 * gq + col / 4) * F::VS + col % 4 * 8;
#pragma unroll
        for (int cb = 0; cb < F::CB; ++cb) {
            const uint2 lo = read_transposed(vr + cb * 32);
            const uint2 hi = read_transposed(vr + 16 * F::VS + cb * 32);
            const u32x4_t vt = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) O[rt][cb] = mfma16<DT>(vt, pf[rt], O[rt][cb]);
        }
    }

    // Join the waves: a row's largest maximum, then the rescaled sums.
    if (lane == 0) join_odd[wave] = 0;
    if (__builtin_amdgcn_ballot_w64(odd) != 0 && lane == 0) join_odd[wave] = 1;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] += __shfl_xor(l[rt], 16);
        l[rt] += __shfl_xor(l[rt], 32);
        if (gq == 0) {
            join_m[wave][16 * rt + col] = m[rt];
            join_l[wave][16 * rt + col] = l[rt];
        }
    }
    __syncthreads();
    float* jo = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int jr = 16 * rt + col;
        const float top = fmaxf(fmaxf(join_m[0][jr], join_m[1][jr]),
                                fmaxf(join_m[2][jr], join_m[3][jr]));
        const float f = exp2_fast(m[rt] - top);
        if (rt > 0) __syncthreads();
#pragma unroll
        for (int cb = 0; cb < F::CB; ++cb)
            *reinterpret_cast<f32x4_t*>(jo + (wave * 16 + col) * F::OS + 16 * cb + 4 * gq) =
                O[rt][cb] * f;
        __syncthreads();
        for (int at = threadIdx.x; at < 16 * (DP / 4); at += kBlock) {
            const int row = at / (DP / 4), c = at % (DP / 4) * 4;
            const int r = w.it.row0 + 16 * rt + row;
            if (r >= w.rows || c >= a.D) continue;
            f32x4_t o = {0.f, 0.f, 0.f, 0.f};
            float sum = 0.f, mt = -FLT_MAX;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) mt = fmaxf(mt, join_m[i][16 * rt + row]);
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                o += *reinterpret_cast<const f32x4_t*>(jo + (i * 16 + row) * F::OS + c);
                sum += join_l[i][16 * rt + row] * exp2_fast(join_m[i][16 * rt + row] - mt);
            }
            if (w.it.part < 0) o *= inverse_sum(sum);
            if (join_odd[0] | join_odd[1] | join_odd[2] | join_odd[3])
                o += odd_values<DT>(a, w, odd_from(w, all_see, kUnit), row_limit(w, r), c);
            if (w.it.part < 0) {
                store4<DT>(a.out, out_offset(a, w, r) + c, o);
            } else {
                const int64_t pr = part_row(a, w, r);
                *reinterpret_cast<f32x4_t*>(a.part_o + pr * a.D + c) = o;
                if (c == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * pr) = make_float2(mt, sum);
            }
        }
    }
}

template <int DT, int DP>
void launch_rows(const PagedLaunch& a, int kind, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_items * a.Hkv));
    // (paged_few_rows(): the kinds that a head_dim comes with)
    if (kind == kFew16) {
        paged_few_kernel<DT, DP, 1><<<grid, kBlock, 0, s>>>(a);
    } else if (kind == kFew32) {
        if constexpr (DP <= 128) paged_few_kernel<DT, DP, 2><<<grid, kBlock, 0, s>>>(a);
    } else {
        if constexpr (DP <= 128) paged_few_kernel<DT, DP, 4><<<grid, kBlock, 0, s>>>(a);
    }
}

template <int DT>
void launch_dim(const PagedLaunch& a, int kind, hipStream_t s) {
    if (a.D <= 64) launch_rows<DT, 64>(a, kind, s);
    else if (a.D <= 96) launch_rows<DT, 96>(a, kind, s);
    else if (a.D <= 128) launch_rows<DT, 128>(a, kind, s);
    else launch_rows<DT, 256>(a, kind, s);
}

}  // namespace

void launch_paged_few(const PagedLaunch& a, int dtype, int kind, hipStream_t s) {
    if (dtype == kSrcBF16) launch_dim<kSrcBF16>(a, kind, s);
    else launch_dim<kSrcF16>(a, kind, s);
}

}  // namespace kivi
