// Pieces shared by the attention kernels over pages of 8 bits (kivi_paged8.hip), and the
// walk of up to 16 query rows.
//
// Codes are whole numbers up to 127, which bf16 and fp16 hold exactly, so both products
// run on the 16-bit matrix instructions with codes as they are; the scales of a block of
// 16 positions, numbers that all its lanes share, come in outside: the keys' into what
// turns a score into log2 units, the values' into the weights.  The first product takes
// queries in their own type, fp32 ones as three bf16 pieces (their 24 bits); the second
// takes bf16 weights (fp16 has no room for scales): two pieces for up to 16 rows, three
// for fp32, which so keeps fp32's accuracy at three times the products, where the fp32
// instructions take sixteen times.
//
// Codes are finite, so what a row must not see is 0 times a number; but for a block's
// scales that are NaN, whose place numbers take for rows that see none of the block.
#pragma once

#include "kivi_paged_attention.hpp"

namespace kivi {

struct Paged8Launch : PagedLaunch {
    const float* k_scales;
    const float* v_scales;
};

namespace {

// The type of the key operand, and the pieces that queries and weights enter in.
template <int DT>
constexpr int key_type() { return DT == kSrcF16 ? kSrcF16 : kSrcBF16; }
template <int DT>
constexpr int query_pieces() { return DT == kSrcF32 ? 3 : 1; }

// Two codes of a word's bytes 2 i and 2 i + 1, as a pair of DT.
template <int DT>
__device__ __forceinline__ uint32_t pair_of_codes(uint32_t x, int i) {
    if constexpr (DT == kSrcBF16) {
        const float a = (float)(int8_t)(x >> (16 * i)), b = (float)(int8_t)(x >> (16 * i + 8));
        return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    } else {
        // 1024 + (code + 128), from which 1152 goes exactly
        const uint32_t u = __builtin_amdgcn_perm(0x64646464u, x ^ 0x80808080u,
                                                 i ? 0x04030402u : 0x04010400u);
        const f16x2_t v = __builtin_bit_cast(f16x2_t, u) - f16x2_t{(_Float16)1152, (_Float16)1152};
        return __builtin_bit_cast(uint32_t, v);
    }
}
// Eight codes as an operand.
template <int DT>
__device__ __forceinline__ u32x4_t operand_of_codes(uint32_t x, uint32_t y) {
    return u32x4_t{pair_of_codes<DT>(x, 0), pair_of_codes<DT>(x, 1), pair_of_codes<DT>(y, 0),
                   pair_of_codes<DT>(y, 1)};
}

// Eight consecutive channels of a query row as an operand of each piece.
template <int DT>
__device__ __forceinline__ void load_query(const void* q, int64_t i,
                                           u32x4_t (&f)[query_pieces<DT>()]) {
    if constexpr (DT == kSrcF32) {
        const SplitConsts k = split_consts();
        const f32x4_t* p = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(q) + i);
        const f32x4_t x = p[0], y = p[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t hi, mid, lo;
            split3_pair(j < 2 ? x[2 * j] : y[2 * j - 4], j < 2 ? x[2 * j + 1] : y[2 * j - 3], hi,
                        mid, lo, k);
            f[0][j] = hi;
            f[1][j] = mid;
            f[2][j] = lo;
        }
    } else {
        f[0] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(q) + i);
    }
}

// The scales of blocks of 16 positions (the last one's for blocks past the end), by
// scalar loads.
template <int N>
struct BlockScales {
    float k[N], v[N];

    __device__ __forceinline__ void load(const Paged8Launch& a, const Work& w, int t0,
                                         const int (&page)[N]) {
        typedef const __attribute__((address_space(4))) float* scalar_t;
        const int shift = a.page_shift - 4;
#pragma unroll
        for (int b = 0; b < N; ++b) {
            const int off = min(t0 + 16 * b, (w.it.kv_end - 1) & ~15) & ((1 << a.page_shift) - 1);
            const int64_t at = (((int64_t)page[b] * a.Hkv + w.kvh) << shift) + off / kScaleBlock;
            k[b] = ((scalar_t)a.k_scales)[at];
            v[b] = ((scalar_t)a.v_scales)[at];
        }
    }
};

// What turns a score of a block into log2 units.  Above 0, for what masks leave of a row
// is -infinity (a scale of 0 belongs to codes that do not matter); NaN stays.
__device__ __forceinline__ float score_units(float scale, float qscale) {
    const float x = scale * qscale;
    return x < FLT_MIN ? FLT_MIN : x;
}

constexpr int kFew8Waves = 4;

template <int DP>
struct Few8 {
    static constexpr int UNIT = DP <= 128 ? 64 : 32;   // positions of a wave at a time
    static constexpr int NB = UNIT / 16;
    static constexpr int KS = DP / 32;                 // k-steps of a score
    static constexpr int KP = (KS + 1) / 2;            // loads of a key, 16 bytes a lane
    static constexpr int CB = DP / 16;                 // blocks of 16 output channels
    // lanes of a value row in its load, 16 bytes each (96 channels: six of the eight)
    static constexpr int CH = DP <= 64 ? 4 : DP <= 128 ? 8 : 16;
    static constexpr int VT = kWave / CH;              // tokens of a load
    static constexpr int VB = 16 / VT;                 // loads of a block
    // (16 bytes of padding: the 16 rows that half a transposed read takes start on 16
    // different groups of four banks)
    static constexpr int VS = DP + 16;
    static constexpr int V_BYTES = UNIT * VS;
    static constexpr int OS = DP + 4;
    static constexpr int JOIN_BYTES = 16 * OS * 4;
    static constexpr int WAVE_BYTES = V_BYTES > JOIN_BYTES ? V_BYTES : JOIN_BYTES;
};

struct Few8Join {
    float m[kFew8Waves][16], l[kFew8Waves][16];
};

typedef int i32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2_t lds_i32x2_t;

// Eight rows' bytes, read transposed: lane 2 r + c of a group of 16 gives the address of
// row r's columns 8 c .. 8 c + 7; lane i receives column i of rows 0 .. 7.
__device__ __forceinline__ i32x2_t read_transposed8(const unsigned char* p) {
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2_t*)(p));
}

// An item of up to 16 rows, by a workgroup of four waves; lds(i): wave i's WAVE_BYTES.
template <int DT, int DP, class L>
__device__ __forceinline__ void few8_rows(const Paged8Launch& a, const Work& w, L lds,
                                          Few8Join& join) {
    using F = Few8<DP>;
    constexpr int NB = F::NB, KT = key_type<DT>(), NQ = query_pieces<DT>();
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const int col = lane % 16, gq = lane / 16;
    unsigned char* vl = lds(wave);
    const bool full = a.D == DP;

    // A lane takes 16 consecutive channels of a key with one load, which are its 8 of
    // two k-steps: k-step 2 p + h, group gq: channels 64 p + 16 gq + 8 h ..; an odd last
    // k-step its 8 as they lie.
    auto channel = [&](int ks) {
        return ks + 1 == F::KS && F::KS % 2 ? 32 * ks + 8 * gq : 32 * (ks & ~1) + 16 * gq + ks % 2 * 8;
    };
    u32x4_t qf[F::KS][NQ];
    f32x4_t O[F::CB];
    float m = -FLT_MAX, l = 0.f;
    int lim = 0;
    {
        const int r = w.it.row0 + col;
        const bool live = r < w.rows;
        if (live) lim = row_limit(w, r);
        const int64_t q = live ? q_offset(a, w, r) : 0;
#pragma unroll
        for (int ks = 0; ks < F::KS; ++ks) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) qf[ks][n] = u32x4_t{0, 0, 0, 0};
            if (live && channel(ks) < a.D) load_query<DT>(a.q, q + channel(ks), qf[ks]);
        }
    }
#pragma unroll
    for (int cb = 0; cb < F::CB; ++cb) O[cb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // positions that every row sees
    const int all_see = w.it.ctx - w.it.n + w.it.row0 / w.hg + 1;
    const int end = w.it.kv_end;

    u32x4_t kf[NB][F::KP], vf[NB][F::VB];
    struct Pages { int p[NB]; };
    auto pages_of = [&](int t0) {
        Pages pg;
#pragma unroll
        for (int b = 0; b < NB; ++b) pg.p[b] = block_page(a, w, t0 + 16 * b);
        return pg;
    };
    auto load_k = [&](int t0, const Pages& pg) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint8_t* p = block_at<uint8_t>(a, w, a.k_pages, pg.p[b], t0 + 16 * b);
#pragma unroll
            for (int kp = 0; kp < F::KP; ++kp) {
                const int c = channel(2 * kp);
                const uint8_t* at = p + (uint32_t)(col * a.D + c);
                kf[b][kp] = u32x4_t{0, 0, 0, 0};
                if (!full && c >= a.D) continue;
                if (2 * kp + 1 < F::KS) {
                    kf[b][kp] = *reinterpret_cast<const u32x4_t*>(at);
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(at);
                    kf[b][kp][0] = x.x;
                    kf[b][kp][1] = x.y;
                }
            }
        }
    };
    const int vt = lane / F::CH, vc = lane % F::CH * 16;
    auto load_v = [&](int t0, const Pages& pg) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint8_t* p = block_at<uint8_t>(a, w, a.v_pages, pg.p[b], t0 + 16 * b);
#pragma unroll
            for (int i = 0; i < F::VB; ++i) {
                vf[b][i] = u32x4_t{0, 0, 0, 0};
                if (full ? F::CH * 16 == DP || vc < DP : vc < a.D)
                    vf[b][i] = *reinterpret_cast<const u32x4_t*>(
                        p + (uint32_t)((vt + i * F::VT) * a.D + vc));
            }
        }
    };

    int t0 = w.it.kv_begin + wave * F::UNIT;
    constexpr int kStep = kFew8Waves * F::UNIT;
    Pages ahead{};
    BlockScales<NB> scales{}, coming{};
    if (t0 < end) {
        const Pages pg = pages_of(t0);
        load_k(t0, pg);
        load_v(t0, pg);
        coming.load(a, w, t0, pg.p);
        ahead = pages_of(t0 + kStep);
    }
    for (; t0 < end; t0 += kStep) {
        const int next = t0 + kStep;
        scales = coming;
        f32x4_t s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            s[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < F::KS; ++ks) {
                const u32x4_t x = operand_of_codes<KT>(kf[b][ks / 2][ks % 2 * 2],
                                                       kf[b][ks / 2][ks % 2 * 2 + 1]);
#pragma unroll
                for (int n = NQ - 1; n >= 0; --n) s[b] = mfma16<KT>(x, qf[ks][n], s[b]);
            }
        }
        const Pages pg = ahead;
        if (next < end) {
            load_k(next, pg);
            coming.load(a, w, next, pg.p);
            ahead = pages_of(next + kStep);
        }
        wave_sync();                      // the last unit's reads, before these writes
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int i = 0; i < F::VB; ++i)
                if (F::CH * 16 == DP || vc < DP)
                    *reinterpret_cast<u32x4_t*>(vl + (16 * b + vt + i * F::VT) * F::VS + vc) =
                        vf[b][i];
        }
        if (next < end) load_v(next, pg);

        float units[NB], vs[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            units[b] = score_units(scales.k[b], a.qscale);
            vs[b] = scales.v[b];
        }
        if (t0 + F::UNIT > min(all_see, end)) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (t0 + 16 * b >= lim) {
                    vs[b] = 0.f;
                    units[b] = FLT_MIN;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t0 + 16 * b + 4 * gq + i >= lim) s[b][i] = -INFINITY;
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < NB; ++b)
            mx = fmaxf(mx, fmaxf(fmaxf(s[b][0], s[b][1]), fmaxf(s[b][2], s[b][3])) * units[b]);
        if (__builtin_amdgcn_ballot_w64(mx > m + kMoveMax) != 0) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float to = fmaxf(m, mx), f = exp2_fast(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int cb = 0; cb < F::CB; ++cb) O[cb] *= f;
        }
        // rows of a transposed read: tokens 4 gq .. + 3 of a block and of the next, in
        // the order in which a lane holds the weights
        const unsigned char* vr = vl + (4 * gq + col / 2 % 4 + col / 8 * 16) * F::VS + col % 2 * 8;
        wave_sync();
#pragma unroll
        for (int j = 0; j < NB / 2; ++j) {
            constexpr int NP = DT == kSrcF32 ? 3 : 2;
            const SplitConsts k = split_consts();
            u32x4_t pf[NP];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int b = 2 * j + i / 2;
                const float p0 = exp2_fast(fmaf(s[b][i % 2 * 2], units[b], -m));
                const float p1 = exp2_fast(fmaf(s[b][i % 2 * 2 + 1], units[b], -m));
                l += p0 + p1;
                uint32_t x[3];
                if constexpr (NP == 3) split3_pair(p0 * vs[b], p1 * vs[b], x[0], x[1], x[2], k);
                else split_pair(p0 * vs[b], p1 * vs[b], x[0], x[1], k);
#pragma unroll
                for (int n = 0; n < NP; ++n) pf[n][i] = x[n];
            }
#pragma unroll
            for (int cb = 0; cb < F::CB; ++cb) {
                const i32x2_t v = read_transposed8(vr + 32 * j * F::VS + cb * 16);
                const u32x4_t vt8 = operand_of_codes<kSrcBF16>((uint32_t)v[0], (uint32_t)v[1]);
#pragma unroll
                for (int n = NP - 1; n >= 0; --n) O[cb] = mfma16<kSrcBF16>(vt8, pf[n], O[cb]);
            }
        }
    }

    // Join the waves: a row's largest maximum, then the rescaled sums.
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (gq == 0) {
        join.m[wave][col] = m;
        join.l[wave][col] = l;
    }
    __syncthreads();
    const float f = exp2_fast(m - fmaxf(fmaxf(join.m[0][col], join.m[1][col]),
                                        fmaxf(join.m[2][col], join.m[3][col])));
#pragma unroll
    for (int cb = 0; cb < F::CB; ++cb)
        *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(vl) + col * F::OS + 16 * cb + 4 * gq) =
            O[cb] * f;
    __syncthreads();
    join_waves<DT, DP, 16, kFew8Waves, false>(
        a, w, w.it.row0, [&](int i) { return reinterpret_cast<const float*>(lds(i)); }, F::OS,
        join.m, join.l, false, F::UNIT);
}

}  // namespace

void launch_paged8_few(const Paged8Launch& a, int dtype, hipStream_t s);
void launch_paged8_many(const Paged8Launch& a, int dtype, hipStream_t s);

}  // namespace kivi
