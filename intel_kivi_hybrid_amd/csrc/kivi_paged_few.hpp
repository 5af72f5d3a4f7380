// Attention over a paged cache for up to 16 query rows per kv head, 16-bit
// types (gfx950 matrix cores): single tokens.
//
// Such calls read every key and value once for a few products: memory-bound.
// A workgroup's four waves walk the item's positions in units of 32, each wave
// units of its own with no barrier between them, its next unit's keys and values
// in flight while it computes.  Keys go from memory into the A operand of
// v_mfma_f32_16x16x32 as they lie (a lane takes 8 channels of one token); values
// need the token as the inner index and pass through the wave's own LDS, from
// which they are read transposed.  The products cost nothing beside the loads, so
// the weights enter as two pieces (rounded, and what that left out): their
// rounding then does not show.  The waves' results are joined in LDS at the
// end; splits of a context are joined by a second launch.  Beside sequences of more
// rows the same is done in their launch (kivi_paged_many.hip).
//
// 64 sequences of up to 8K positions, 32/8 heads of 128, bf16: 287 us, 5.75 TB/s (a
// read-only stream reaches 6.4).  One sequence of 1K: 7 us, and the join 3 to 4.
#pragma once

#include "kivi_paged_attention.hpp"

namespace kivi {
namespace {

constexpr int kFewWaves = 4;
constexpr int kFewUnit = 32;

template <int DP>
struct Few {
    static constexpr int KS = DP / 32;            // k-steps of a score
    static constexpr int CB = DP / 16;            // blocks of 16 output channels
    static constexpr int CH = DP / 8;             // 16-byte vectors of a token
    static constexpr int VL = kFewUnit * CH / kWave; // value loads of a lane per unit
    // (32 bytes of padding per token: the 16 rows of a transposed read then
    // start on 8 different bank groups, as few as their 512 bytes need)
    static constexpr int VS = DP * 2 + 32;
    static constexpr int V_BYTES = kFewUnit * VS;
    // joining the waves: fp32 rows, padded by one vector
    static constexpr int OS = DP + 4;
    static constexpr int JOIN_BYTES = 16 * OS * 4;
    static constexpr int WAVE_BYTES = V_BYTES > JOIN_BYTES ? V_BYTES : JOIN_BYTES;
};

// What the waves leave for the join.
struct FewJoin {
    float m[kFewWaves][16], l[kFewWaves][16];
    int odd[kFewWaves];
};

// An item of up to 16 rows, by a workgroup of four waves; lds(i): wave i's WAVE_BYTES.
template <int DT, int DP, class L>
__device__ __forceinline__ void few_rows(const PagedLaunch& a, const Work& w, L lds, FewJoin& join) {
    using F = Few<DP>;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const int col = lane % 16, gq = lane / 16;
    unsigned char* vl = lds(wave);

    u32x4_t qf[F::KS];
    f32x4_t O[F::CB];
    float m = -FLT_MAX, l = 0.f;
    int lim = 0;
    {
        const int r = w.it.row0 + col;
        const bool live = r < w.rows;
        if (live) lim = row_limit(w, r);
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + (live ? q_offset(a, w, r) : 0);
#pragma unroll
        for (int ks = 0; ks < F::KS; ++ks) {
            const int c = 32 * ks + 8 * gq;
            qf[ks] = u32x4_t{0, 0, 0, 0};
            if (live && c < a.D) qf[ks] = *reinterpret_cast<const u32x4_t*>(q + c);
        }
    }
#pragma unroll
    for (int cb = 0; cb < F::CB; ++cb) O[cb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // positions that every row sees
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
        const bool whole = full && t0 + kFewUnit <= end;
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
    int t0 = w.it.kv_begin + wave * kFewUnit;
    Pages ahead = {{0, 0}};
    if (t0 < end) {
        const Pages pg = pages_of(t0);
        load_k(t0, pg);
        load_v(t0, pg);
        ahead = pages_of(t0 + kFewWaves * kFewUnit);
    }
    for (; t0 < end; t0 += kFewWaves * kFewUnit) {
        const int next = t0 + kFewWaves * kFewUnit;
        f32x4_t s[2];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
            s[tb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < F::KS; ++ks) s[tb] = mfma16<DT>(kf[tb][ks], qf[ks], s[tb]);
        }
        const Pages pg = ahead;
        if (next < end) {
            load_k(next, pg);
            ahead = pages_of(next + kFewWaves * kFewUnit);
        }
        const bool masked = t0 + kFewUnit > min(all_see, end);
        if (t0 + kFewUnit > all_see) {
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

        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = s[i / 4][i % 4];
            if (masked && t0 + 16 * (i / 4) + 4 * gq + i % 4 >= lim) x[i] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                         fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        mx = fmaf(mx, a.qscale, -weight_bits<DT>());
        if (__builtin_amdgcn_ballot_w64(mx > m + kMoveMax) != 0) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float to = fmaxf(m, mx), f = exp2_fast(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int cb = 0; cb < F::CB; ++cb) O[cb] *= f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = exp2_fast(fmaf(x[i], a.qscale, -m));
            l += x[i];
        }
        u32x4_t hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            hi[i] = pack2<DT>(x[2 * i], x[2 * i + 1]);
            lo[i] = pack2<DT>(x[2 * i] - half_of<DT>(hi[i], 0), x[2 * i + 1] - half_of<DT>(hi[i], 1));
        }
        wave_sync();
        // rows of a transposed read: tokens 4 gq .. + 3, and 16 further on, in the
        // order in which a lane holds the weights
        const unsigned char* vr = vl + (4 * gq + col / 4) * F::VS + col % 4 * 8;
#pragma unroll
        for (int cb = 0; cb < F::CB; ++cb) {
            const uint2 v0 = read_transposed(vr + cb * 32);
            const uint2 v1 = read_transposed(vr + 16 * F::VS + cb * 32);
            const u32x4_t vt = {v0.x, v0.y, v1.x, v1.y};
            O[cb] = mfma16<DT>(vt, lo, O[cb]);
            O[cb] = mfma16<DT>(vt, hi, O[cb]);
        }
    }

    // Join the waves: a row's largest maximum, then the rescaled sums.
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (gq == 0) {
        join.m[wave][col] = m;
        join.l[wave][col] = l;
    }
    const bool any_odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    if (lane == 0) join.odd[wave] = any_odd;
    __syncthreads();
    const float f = exp2_fast(m - fmaxf(fmaxf(join.m[0][col], join.m[1][col]),
                                        fmaxf(join.m[2][col], join.m[3][col])));
#pragma unroll
    for (int cb = 0; cb < F::CB; ++cb)
        *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(vl) + col * F::OS + 16 * cb + 4 * gq) =
            O[cb] * f;
    __syncthreads();
    join_waves<DT, DP, 16, kFewWaves>(
        a, w, w.it.row0, [&](int i) { return reinterpret_cast<const float*>(lds(i)); }, F::OS,
        join.m, join.l, (join.odd[0] | join.odd[1] | join.odd[2] | join.odd[3]) != 0, kFewUnit);
}

}  // namespace
}  // namespace kivi
