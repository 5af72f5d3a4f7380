// Rows of a step's queries, keys and values on their way into a paged cache: how lanes
// share a head's channels, its norm and its rotation (kivi_paged.hip, kivi_paged8.hip).
//
// A lane takes two 8-element vectors of a head, D/2 apart (r/2 in a rotated part of
// r channels), that hold whole pairs of either kind of rotation: neighbours, or
// i and i + r/2.  So a rotation never crosses lanes, and only the norm's sum does,
// over the D / 16 lanes of the head (a power of two of them, DPP steps).
#pragma once

#include "kivi_common.hpp"
#include "kivi_paged.hpp"

namespace kivi {

int paged_page_shift(int32_t page_size);
int paged_check_pool(int32_t dtype, int64_t num_pages, int32_t page_size, int32_t q_heads,
                     int32_t kv_heads, int32_t head_dim);
struct AppendArgs;
int paged_append_args(AppendArgs& a, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                      const void* k, int64_t k_token_stride, int64_t k_head_stride,
                      const void* v, int64_t v_token_stride, int64_t v_head_stride,
                      int32_t dtype, void* q_out, void* k_pages, void* v_pages,
                      int64_t num_pages, int32_t page_size, int32_t q_heads, int32_t kv_heads,
                      int32_t head_dim, const int32_t* plan, int32_t tokens, const float* cos,
                      const float* sin, int32_t rotary_dim, int32_t interleaved,
                      const void* q_norm, const void* k_norm, int32_t norm_dtype, float eps);


constexpr int kAppendBlock = 256;

struct AppendArgs {
    const void* q;
    const void* k;
    const void* v;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
    void* q_out;
    void* k_pages;
    void* v_pages;
    const int2* tokens;          // slot, position
    const float* cos;
    const float* sin;
    const void* q_norm;
    const void* k_norm;
    float eps, inv_d;
    int n_tokens, Hq, Hkv, D, page_shift, rot, lanes_log2;
    int norm_dt, norm_vec, interleaved, vec;
};

namespace {

typedef unsigned int kivi_u4v __attribute__((ext_vector_type(4)));

// Eight elements as they lie: one or two 16-byte loads (vec: aligned to 16), read once
// by this kernel.
template <int DT>
struct Eight {
    static constexpr int kWords = DT == kSrcF32 ? 8 : 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void load(const void* p, int64_t i, bool vec) {
        const char* from = static_cast<const char*>(p) + i * src_size(DT);
        if (vec) {
#pragma unroll
            for (int j = 0; j < kWords; j += 4) {
                const kivi_u4v x =
                    __builtin_nontemporal_load(reinterpret_cast<const kivi_u4v*>(from + 4 * j));
#pragma unroll
                for (int k = 0; k < 4; ++k) w[j + k] = x[k];
            }
        } else if constexpr (DT == kSrcF32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = reinterpret_cast<const uint32_t*>(from)[j];
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(from);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
        }
    }
    __device__ __forceinline__ void widen(float (&x)[8]) const {
        if constexpr (DT == kSrcF32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(w[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (DT == kSrcBF16) {
                    x[2 * j] = __uint_as_float(w[j] << 16);
                    x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                } else {
                    x[2 * j] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[j] & 0xffffu));
                    x[2 * j + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[j] >> 16));
                }
            }
        }
    }
    __device__ __forceinline__ void round(const float (&x)[8]) {
        if constexpr (DT == kSrcF32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(x[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint16_t lo, hi;
                if constexpr (DT == kSrcBF16) {
                    lo = __builtin_bit_cast(uint16_t, (__bf16)x[2 * j]);
                    hi = __builtin_bit_cast(uint16_t, (__bf16)x[2 * j + 1]);
                } else {
                    lo = __builtin_bit_cast(uint16_t, (_Float16)x[2 * j]);
                    hi = __builtin_bit_cast(uint16_t, (_Float16)x[2 * j + 1]);
                }
                w[j] = lo | (uint32_t)hi << 16;
            }
        }
    }
    __device__ __forceinline__ void store(void* p, int64_t i) const {
        uint4* to = reinterpret_cast<uint4*>(static_cast<char*>(p) + i * src_size(DT));
#pragma unroll
        for (int j = 0; j < kWords; j += 4)
            to[j / 4] = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
    }
};
// Eight of a type known at run time, widened.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int i, bool vec, float (&x)[8]) {
    Eight<DT> e;
    e.load(p, i, vec);
    e.widen(x);
}
__device__ __forceinline__ void load8_dt(const void* p, int i, int dt, bool vec, float (&x)[8]) {
    if (dt == kSrcF32) load8<kSrcF32>(p, i, vec, x);
    else if (dt == kSrcBF16) load8<kSrcBF16>(p, i, vec, x);
    else load8<kSrcF16>(p, i, vec, x);
}

// Sum over aligned segments of 1 << log2 lanes.
template <class T>
__device__ __forceinline__ T seg_sum(T v, int log2) {
    if (log2 > 0) v += seg_partner<1>(v);
    if (log2 > 1) v += seg_partner<2>(v);
    if (log2 > 2) v += seg_partner<4>(v);
    if (log2 > 3) v += seg_partner<8>(v);
    return v;
}

// The lane's two vectors of 8 channels: of the rotated part's halves, or of the rest's.
struct HeadLane {
    bool live, inside;
    int c0, c1;
};
__device__ __forceinline__ HeadLane head_lane(const AppendArgs& a, int unit) {
    HeadLane l;
    l.live = unit < a.D / 16;
    l.inside = 16 * unit < a.rot;
    const int start = l.inside ? 0 : a.rot, at = 8 * unit - start / 2;
    l.c0 = start + at;
    l.c1 = l.c0 + (l.inside ? a.rot : a.D - a.rot) / 2;
    return l;
}

// cos and sin of a position for pairs (c0 + j, c1 + j), or for the pairs in x and those
// in y.
struct Angles {
    float4 c[2], s[2];

    __device__ __forceinline__ void load(const AppendArgs& a, const HeadLane& l, int position) {
        const int half = a.rot / 2;
        const int64_t r = (int64_t)position * half;
        const int i0 = a.interleaved ? l.c0 / 2 : l.c0, i1 = a.interleaved ? l.c1 / 2 : l.c0 + 4;
        c[0] = *reinterpret_cast<const float4*>(a.cos + r + i0);
        c[1] = *reinterpret_cast<const float4*>(a.cos + r + i1);
        s[0] = *reinterpret_cast<const float4*>(a.sin + r + i0);
        s[1] = *reinterpret_cast<const float4*>(a.sin + r + i1);
    }
};

__device__ __forceinline__ float fma_of(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma_of(double a, double b, double c) { return fma(a, b, c); }
__device__ __forceinline__ float inverse_root(float x) { return rsqrtf(x); }
__device__ __forceinline__ double inverse_root(double x) { return 1.0 / sqrt(x); }

// The norm of a head's row over its segment of lanes (all of which call it), in T.
template <class T>
__device__ __forceinline__ void norm_row(const AppendArgs& a, const HeadLane& l, const void* norm,
                                         T (&x)[8], T (&y)[8]) {
    float u[8], w[8];
    if (l.live) {
        load8_dt(norm, l.c0, a.norm_dt, a.norm_vec, u);
        load8_dt(norm, l.c1, a.norm_dt, a.norm_vec, w);
    }
    T s = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fma_of(x[j], x[j], fma_of(y[j], y[j], s));
    s = seg_sum(s, a.lanes_log2);
    const T inv_d = sizeof(T) == 8 ? (T)1 / (T)a.D : (T)a.inv_d;
    const T r = inverse_root(fma_of(s, inv_d, (T)a.eps));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = x[j] * r * (T)u[j];
        y[j] = y[j] * r * (T)w[j];
    }
}

// The rotation of the lane's pairs, in T.
template <class T>
__device__ __forceinline__ void turn_row(const AppendArgs& a, const Angles& at, T (&x)[8],
                                         T (&y)[8]) {
    const T c[8] = {at.c[0].x, at.c[0].y, at.c[0].z, at.c[0].w,
                    at.c[1].x, at.c[1].y, at.c[1].z, at.c[1].w};
    const T s[8] = {at.s[0].x, at.s[0].y, at.s[0].z, at.s[0].w,
                    at.s[1].x, at.s[1].y, at.s[1].z, at.s[1].w};
    if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            T* v = j < 4 ? x + 2 * j : y + 2 * (j - 4);
            const T p = v[0], q = v[1];
            v[0] = fma_of(p, c[j], -(q * s[j]));
            v[1] = fma_of(q, c[j], p * s[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const T p = x[j], q = y[j];
            x[j] = fma_of(p, c[j], -(q * s[j]));
            y[j] = fma_of(q, c[j], p * s[j]);
        }
    }
}

// A head's row by its segment of lanes, normed and rotated where asked, in fp32 rounded
// once.  (What is only moved keeps its bits: to fp32 and back a signalling NaN loses one.)
template <int DT>
__device__ __forceinline__ void move_row(const AppendArgs& a, const HeadLane& l, const void* src,
                                         int64_t from, const void* norm, bool turn, int position,
                                         void* dst, int64_t to) {
    Eight<DT> ex{}, ey{};
    if (l.live) {
        ex.load(src, from + l.c0, a.vec);
        ey.load(src, from + l.c1, a.vec);
    }
    const bool turned = l.live && l.inside && turn;
    Angles at;
    if (turned) at.load(a, l, position);
    float x[8], y[8];
    ex.widen(x);
    ey.widen(y);
    if (norm != nullptr) norm_row(a, l, norm, x, y);
    if (!l.live) return;
    if (turned) turn_row(a, at, x, y);
    if (norm != nullptr || turned) {
        ex.round(x);
        ey.round(y);
    }
    ex.store(dst, to + l.c0);
    ey.store(dst, to + l.c1);
}

}  // namespace
}  // namespace kivi
