// Pieces shared by the attention kernels over pages of 8 bits (kivi_paged8_few.hip,
// kivi_paged8_many.hip), and the walk of up to 16 query rows.
//
// Codes are whole numbers up to 127, which fp16 holds exactly, so both products run on
// the fp16 matrix instructions with codes as they are; the scales of a block of 16
// positions, numbers that all its lanes share, come in outside: the keys' into what
// turns a score into log2 units, the values' into the weights.
//
// Queries enter as fp16 too: a row times the power of two that brings its largest
// element to 2^14, which keeps every bit of bf16's elements down to 2^-28 of that one,
// and fp32's as two pieces (22 bits).  Weights times value scales have no such bounds, so
// a row keeps a second maximum, that of these products, and its outputs in units of
// that one: the largest lies between 2^12 and 2^15, so that fp16's last step, 2^-24, is
// 2^-36 of it or less (RowState and drop_far() say how fp32 holds what lies between).  They are rounded to fp16 (as a bf16 cache's would be to bf16, or
// better), for up to 16 rows and for fp32 in two pieces.  (bf16 operands hold codes and any scale
// at once, but take a fifth more operations to widen codes, and fp32 three pieces.)
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

// The pieces that queries enter in.
template <int DT>
constexpr int query_pieces() { return DT == kSrcF32 ? 2 : 1; }

// Two codes of a word's bytes 2 i and 2 i + 1: 1024 + (code + 128), from which 1152 goes
// exactly.  x: the word with the codes' signs flipped.
__device__ __forceinline__ uint32_t pair_of_codes(uint32_t x, int i) {
    const uint32_t u = __builtin_amdgcn_perm(0x64646464u, x, i ? 0x04030402u : 0x04010400u);
    const f16x2_t v = __builtin_bit_cast(f16x2_t, u) - f16x2_t{(_Float16)1152, (_Float16)1152};
    return __builtin_bit_cast(uint32_t, v);
}
// Eight codes as an operand.
__device__ __forceinline__ u32x4_t operand_of_codes(uint32_t x, uint32_t y) {
    x ^= 0x80808080u;
    y ^= 0x80808080u;
    return u32x4_t{pair_of_codes(x, 0), pair_of_codes(x, 1), pair_of_codes(y, 0),
                   pair_of_codes(y, 1)};
}

// Two values as fp16 pieces: rounded, and what that left out.
struct Pieces { uint32_t hi, lo; };
__device__ __forceinline__ Pieces split_f16(float a, float b) {
    uint32_t hi = pack2<kSrcF16>(a, b);
    // (What is taken off must be the word that is multiplied: of a product the compiler
    // otherwise rounds it a second time, from the exact product, and one in 2^13 of
    // those lies on the other side of a border.)
    asm("" : "+v"(hi));
    const f16x2_t h = __builtin_bit_cast(f16x2_t, hi);
    return {hi, pack2<kSrcF16>(fmaf((float)h[0], -1.0f, a), fmaf((float)h[1], -1.0f, b))};
}

// A query row's operands, k-step i's 8 channels at channel(i), by the lanes that
// share(max) reduces over: f, and what a product with them is to be multiplied by.
template <int DT, int KS, class C, class S>
__device__ __forceinline__ float load_query(const PagedLaunch& a, int64_t at, bool live, C channel,
                                            S share, u32x4_t (&f)[KS][query_pieces<DT>()]) {
    if constexpr (DT == kSrcF16) {
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            f[i][0] = u32x4_t{0, 0, 0, 0};
            if (live && channel(i) < a.D)
                f[i][0] = *reinterpret_cast<const u32x4_t*>(
                    static_cast<const uint16_t*>(a.q) + at + channel(i));
        }
        return 1.0f;
    } else {
        f32x4_t x[KS][2];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                x[i][h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                if (live && channel(i) < a.D) x[i][h] = load4<DT>(a.q, at + channel(i) + 4 * h);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    top = max(top, __float_as_uint(x[i][h][j]) & 0x7fffffffu);
            }
        }
        const int e = (int)(share(top) >> 23);
        // 2^14 for the largest (a row of infinities or NaN, and one below 2^-112, may stay
        // where it is: its scores are no numbers, or 0)
        const int up = e == 255 ? 0 : min(141 - e, 126);
        const float factor = __int_as_float((127 + up) << 23);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float u = x[i][j / 2][j % 2 * 2] * factor;
                const float v = x[i][j / 2][j % 2 * 2 + 1] * factor;
                if constexpr (DT == kSrcF32) {
                    const Pieces p = split_f16(u, v);
                    f[i][0][j] = p.hi;
                    f[i][1][j] = p.lo;
                } else {
                    f[i][0][j] = pack2<kSrcF16>(u, v);
                }
            }
        }
        return __int_as_float((127 - up) << 23);
    }
}

// The largest weight times scale of a row is 2^kWeightBits, or half of it, when its units
// are set, and they are set anew where one comes out 2^kMoveTop times larger.
constexpr float kWeightBits = 13.0f, kMoveTop = 2.0f;

// Power of two above a scale, log2.
__device__ __forceinline__ float above(float scale) {
    return (float)((int)(__float_as_uint(scale) >> 23 & 0xff) - 126);
}

// A row's softmax state: weights are 2^(score - m), l their sum, outputs in units of
// 2^(m + lead).  (Units relative to m: beside a score of 2^28 fp32 holds no distance of 13.)
//
// fp32 has to hold 2^-lead too.  Where the values at a row's largest scores are quiet (zeros
// have the smallest scale, 2^-126) m lies below the largest score, by 75 at most, so that
// lead is -64 or more.  Rows with values of a scale of 2^-51 or more at their largest score
// have it at m.
constexpr float kLeastLead = -64.0f;
struct RowState {
    float m, lead, l;

    // Moves m to `to`, or below, where `next` is the least lead that the row's outputs and
    // the tile at hand ask for.  What the outputs are to be multiplied by.
    __device__ __forceinline__ float move(float to, float next) {
        float low = to + fminf(next - kLeastLead, 0.f);
        // (from 2^31 on the nearest number below is 128 away: weights of 2^128)
        if (to - low > 96.0f) low = to;
        next = fmaxf(next + (to - low), kLeastLead);
        const float gone = low - m, f = exp2_fast(lead - gone - next);
        l *= exp2_fast(-gone);
        m = low;
        lead = next;
        return f;
    }
};

// Value scales from 2^60 on may leave fp32 on the way into such units, where the scores
// of their block are 2^112 or more below the row's largest, and an infinity is NaN beside
// a weight of 0: such a block's weights count as 0.  most: the lane's largest of the blocks'
// scores, whose units these are, of(x): the row's of the lanes' x.
constexpr float kLoud = 0x1p60f;
template <int N, class F>
__device__ __forceinline__ void drop_far(float (&vs)[N], const float (&most)[N],
                                         const float (&units)[N], float m, F of) {
    float top = m;
#pragma unroll
    for (int b = 0; b < N; ++b) top = fmaxf(top, most[b] * units[b]);
    top = of(top);
#pragma unroll
    for (int b = 0; b < N; ++b)
        if (vs[b] >= kLoud && fmaf(most[b], units[b], -top) < -112.0f) vs[b] = 0.f;  // (NaN stays)
}

// The scales of N blocks of 16 positions (the last one's for blocks past the end).  Lane l
// loads one of them, its block l % N's for keys or values, and before that, while the
// tile before is loaded, its page.  (Scalar loads would do with no lanes, but LDS reads
// wait for whatever scalar loads are on their way: a chunk of 2048 tokens after 8200 took
// 397 us with them.)
template <int N>
struct BlockScales {
    int page;
    float own;

    __device__ __forceinline__ void pages_of(const Paged8Launch& a, const Work& w, int t0) {
        const int t = min(t0 + 16 * ((int)threadIdx.x % N), w.it.kv_end - 1);
        page = (a.pages + w.it.page0)[t >> a.page_shift];
    }
    __device__ __forceinline__ void load(const Paged8Launch& a, const Work& w, int t0) {
        const int lane = threadIdx.x % kWave;
        const int t = min(t0 + 16 * (lane % N), (w.it.kv_end - 1) & ~15);
        const int off = t & ((1 << a.page_shift) - 1);
        const int64_t at = (((int64_t)page * a.Hkv + w.kvh) << (a.page_shift - 4)) + off / kScaleBlock;
        own = (lane / N % 2 ? a.v_scales : a.k_scales)[at];
    }
    __device__ __forceinline__ int page_of(int b) const {
        return __builtin_amdgcn_readlane(page, b);
    }
    __device__ __forceinline__ float k(int b) const { return lane_f(own, b); }
    __device__ __forceinline__ float v(int b) const { return lane_f(own, N + b); }
    // Whether a value's reaches kLoud, and a key's far_keys().
    __device__ __forceinline__ bool loud() const {
        uint32_t most = 0;
#pragma unroll
        for (int b = 0; b < N; ++b) most = max(most, __float_as_uint(v(b)));
        return most >= __float_as_uint(kLoud);
    }
    __device__ __forceinline__ bool far(uint32_t from) const {
        uint32_t most = 0;
#pragma unroll
        for (int b = 0; b < N; ++b) most = max(most, __float_as_uint(k(b)));
        return most >= from;
    }
};

// Key scales (as bits) from which on scores of a wave's rows may pass 2^29, products with
// codes being 2^31 at most.  The largest score's distance from m is then no longer small, since
// m is its product with the units rounded: such scores are rounded themselves first.
__device__ __forceinline__ uint32_t far_keys(float qscale) {
    const int e = __float_as_int(wave_max(qscale)) >> 23;
    return (uint32_t)min(max(252 - e, 1), 255) << 23;
}

// Moves a row where a tile's blocks (most, units: as in drop_far()) ask for it: whether any
// row of the wave moved, and what outputs are then to be multiplied by.  of(x): the row's
// largest of its lanes' x.
template <int N, class F>
__device__ __forceinline__ bool move_row(RowState& row, const BlockScales<N>& scales,
                                         const float (&most)[N], const float (&units)[N], F of,
                                         float& f) {
    // the largest score less m, and of these plus above() of their value scales
    float x = -INFINITY, xv = -INFINITY;
#pragma unroll
    for (int b = 0; b < N; ++b) {
        const float y = fmaf(most[b], units[b], -row.m);
        x = fmaxf(x, y);
        xv = fmaxf(xv, y + above(scales.v(b)));
    }
    if (__builtin_amdgcn_ballot_w64((x > kMoveMax) |
                                    (xv > row.lead + (kWeightBits + kMoveTop))) == 0)
        return false;
    x = of(x);
    xv = of(xv);
    float to, next;
    if (__builtin_amdgcn_ballot_w64(x > 0x1p16f) == 0) {
        to = row.m + fmaxf(x, 0.f);
        next = fmaxf(row.lead, xv - kWeightBits) - (to - row.m);
    } else {
        // (a first tile's, or so far from m that the difference says little)
        to = row.m;
#pragma unroll
        for (int b = 0; b < N; ++b) to = fmaxf(to, most[b] * units[b]);
        to = of(to);
        xv = -INFINITY;
#pragma unroll
        for (int b = 0; b < N; ++b)
            xv = fmaxf(xv, fmaf(most[b], units[b], -to) + above(scales.v(b)));
        next = fmaxf(row.lead - (to - row.m), of(xv) - kWeightBits);
    }
    f = row.move(to, next);
    return true;
}

// A page id (one for the wave), by a vector load for the same reason.
__device__ __forceinline__ int block_page_ahead(const Paged8Launch& a, const Work& w, int t) {
    int at = min(t, w.it.kv_end - 1) >> a.page_shift;
    asm("" : "+v"(at));
    return (a.pages + w.it.page0)[at];
}

// What turns a score of a block into log2 units, where masks leave -infinity of some:
// above 0 (a scale of 0 belongs to codes that do not matter); NaN stays.
__device__ __forceinline__ float above_zero(float units) {
    return units < FLT_MIN ? FLT_MIN : units;
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
    constexpr int NB = F::NB, NQ = query_pieces<DT>();
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
    RowState row{-FLT_MAX, 0.f, 0.f};
    float qscale;
    uint32_t far_from;
    int lim = 0;
    {
        const int r = w.it.row0 + col;
        const bool live = r < w.rows;
        if (live) lim = row_limit(w, r);
        qscale = a.qscale * load_query<DT, F::KS>(a, live ? q_offset(a, w, r) : 0, live, channel,
                                                  [](uint32_t x) {
            x = max(x, (uint32_t)__shfl_xor((int)x, 16));
            return max(x, (uint32_t)__shfl_xor((int)x, 32));
        }, qf);
        far_from = far_keys(qscale);
    }
#pragma unroll
    for (int cb = 0; cb < F::CB; ++cb) O[cb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // positions that every row sees
    const int all_see = w.it.ctx - w.it.n + w.it.row0 / w.hg + 1;
    const int end = w.it.kv_end;

    u32x4_t kf[NB][F::KP], vf[NB][F::VB];
    auto load_k = [&](int t0, const BlockScales<NB>& of) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint8_t* p = block_at<uint8_t>(a, w, a.k_pages, of.page_of(b), t0 + 16 * b);
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
    auto load_v = [&](int t0, const BlockScales<NB>& of) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint8_t* p = block_at<uint8_t>(a, w, a.v_pages, of.page_of(b), t0 + 16 * b);
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
    // (a unit's scales and the next one's pages; the scales of the unit at hand)
    BlockScales<NB> coming{}, scales{};
    if (t0 < end) {
        coming.pages_of(a, w, t0);
        load_k(t0, coming);
        load_v(t0, coming);
        coming.load(a, w, t0);
        coming.pages_of(a, w, t0 + kStep);
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
                const u32x4_t x = operand_of_codes(kf[b][ks / 2][ks % 2 * 2],
                                                   kf[b][ks / 2][ks % 2 * 2 + 1]);
#pragma unroll
                for (int n = NQ - 1; n >= 0; --n) s[b] = mfma16<kSrcF16>(x, qf[ks][n], s[b]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (next < end) {
            load_k(next, coming);
            coming.load(a, w, next);
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
        if (next < end) {
            load_v(next, coming);
            coming.pages_of(a, w, next + kStep);
        }

        float units[NB], vs[NB], most[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            units[b] = scales.k(b) * qscale;
            vs[b] = scales.v(b);
        }
        auto each_most = [&] {                // the lane's largest of each block's
#pragma unroll
            for (int b = 0; b < NB; ++b)
                most[b] = fmaxf(fmaxf(s[b][0], s[b][1]), fmaxf(s[b][2], s[b][3]));
        };
        auto row_most = [](float x) {
            x = fmaxf(x, __shfl_xor(x, 16));
            return fmaxf(x, __shfl_xor(x, 32));
        };
        const bool loud = scales.loud(), far = scales.far(far_from);
        if (t0 + F::UNIT > min(all_see, end) || loud || far) {
            asm volatile("");            // (or every unit does all of this and selects)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                units[b] = above_zero(units[b]);
                if (t0 + 16 * b >= lim) {
                    vs[b] = 0.f;
                    units[b] = FLT_MIN;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t0 + 16 * b + 4 * gq + i >= lim) s[b][i] = -INFINITY;
            }
            if (__builtin_expect(far, 0)) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    s[b] *= units[b];
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
        if (move_row<NB>(row, scales, most, units, row_most, f)) {
#pragma unroll
            for (int cb = 0; cb < F::CB; ++cb) O[cb] *= f;
        }
        const float down = exp2_fast(-row.lead);
#pragma unroll
        for (int b = 0; b < NB; ++b) vs[b] *= down;
        // rows of a transposed read: tokens 4 gq .. + 3 of a block and of the next, in
        // the order in which a lane holds the weights
        const unsigned char* vr = vl + (4 * gq + col / 2 % 4 + col / 8 * 16) * F::VS + col % 2 * 8;
        wave_sync();
#pragma unroll
        for (int j = 0; j < NB / 2; ++j) {
            u32x4_t hi, lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int b = 2 * j + i / 2;
                const float p0 = exp2_fast(fmaf(s[b][i % 2 * 2], units[b], -row.m));
                const float p1 = exp2_fast(fmaf(s[b][i % 2 * 2 + 1], units[b], -row.m));
                row.l += p0 + p1;
                const Pieces w = split_f16(p0 * vs[b], p1 * vs[b]);
                hi[i] = w.hi;
                lo[i] = w.lo;
            }
            // (four reads, then their products: left to itself the compiler widens all of
            // a unit's codes first, in 100 registers more)
            constexpr int kAtOnce = F::CB % 4 == 0 ? 4 : 3;
#pragma unroll
            for (int c0 = 0; c0 < F::CB; c0 += kAtOnce) {
                i32x2_t v[kAtOnce];
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i)
                    v[i] = read_transposed8(vr + 32 * j * F::VS + (c0 + i) * 16);
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    const u32x4_t x = operand_of_codes((uint32_t)v[i][0], (uint32_t)v[i][1]);
                    O[c0 + i] = mfma16<kSrcF16>(x, lo, O[c0 + i]);
                    O[c0 + i] = mfma16<kSrcF16>(x, hi, O[c0 + i]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // Join the waves: a row's largest maximum, then the rescaled sums.
    row.l += __shfl_xor(row.l, 16);
    row.l += __shfl_xor(row.l, 32);
    if (gq == 0) {
        join.m[wave][col] = row.m;
        join.l[wave][col] = row.l;
    }
    __syncthreads();
    const float apart = row.lead + (row.m - fmaxf(fmaxf(join.m[0][col], join.m[1][col]),
                                                  fmaxf(join.m[2][col], join.m[3][col])));
    // (below 2^-126 in two steps: the outputs may be large)
    const float f = exp2_fast(fmaxf(apart, -100.0f)), rest = exp2_fast(fminf(apart + 100.0f, 0.f));
#pragma unroll
    for (int cb = 0; cb < F::CB; ++cb)
        *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(vl) + col * F::OS + 16 * cb + 4 * gq) =
            O[cb] * f * rest;
    __syncthreads();
    join_waves<DT, DP, 16, kFew8Waves, false>(
        a, w, w.it.row0, [&](int i) { return reinterpret_cast<const float*>(lds(i)); }, F::OS,
        join.m, join.l, false, F::UNIT);
}

}  // namespace

void launch_paged8_few(const Paged8Launch& a, int dtype, hipStream_t s);
void launch_paged8_many(const Paged8Launch& a, int dtype, bool wide, hipStream_t s);

}  // namespace kivi
