// Pieces shared by the paged-attention kernels: operand types, the products
// of each type, a step's rows and pages, and what is written at the end.
//
// All kernels form scores transposed, S^T = K Q^T, and outputs transposed,
// O^T = V^T P^T: a lane then holds scores, sums and outputs of one query row,
// so a row's softmax state is a per-lane scalar, and the weights go from the
// score registers into the second product's operand without moving between
// lanes (the order of a product's inner index is free as long as both operands
// agree).  Scores, softmax and outputs are fp32; the weights are rounded to
// the cache's type for the second product (fp32 caches keep them), which is
// off by at most half a step of that type, as the values themselves are.  Up to 16
// rows, where the products cost nothing, they enter in two pieces (kivi_paged_few.hpp);
// for more the second piece costs matrix instructions that bound the tile (5 tokens of
// 16 sequences of 3K, 28/4 heads, bf16: 23 us, with it 27; off from float64 by 0.0023 of
// the outputs, their own rounding alone by 0.0017).
//
// The softmax is online in the log2 domain.  A row's maximum moves only when
// exceeded by more than 8, so most steps rescale nothing.  Weights are formed against
// the maximum lowered by weight_bits(): in fp16 from 2^7 to 2^15 for a row's largest,
// so that the type's subnormal steps of 2^-24 are 2^-31 of it or less.  (Against the
// maximum itself weights below 2^-25 of the largest became 0: of 16K positions whose
// values count, 25.2 log2 units below every 32nd, nothing was left.)
#pragma once

#include <float.h>

#include "kivi_common.hpp"
#include "kivi_mfma.hpp"
#include "kivi_paged.hpp"

namespace kivi {
namespace {

constexpr float kMoveMax = 8.0f;       // log2 units
template <int DT>
constexpr float weight_bits() { return DT == kSrcF16 ? 7.0f : 0.0f; }

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

template <int DT>
__device__ __forceinline__ f32x4_t mfma16(u32x4_t a, u32x4_t b, f32x4_t c) {
    if constexpr (DT == kSrcBF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                      __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    if constexpr (DT == kSrcBF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                      __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// Two values rounded to nearest even.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == kSrcBF16) {
        return pack_bf16x2(a, b);
    } else {
        const f16x2_t v = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
}
// The low or high half of a word, widened.
template <int DT>
__device__ __forceinline__ float half_of(uint32_t w, int hi) {
    const uint32_t h = hi ? w >> 16 : w & 0xffffu;
    if constexpr (DT == kSrcBF16) return __uint_as_float(h << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}

// A value that a row must not see still meets it as 0 * value, which is NaN for
// an infinity or a NaN.  In steps where some row stops short, such elements
// enter the products as 0, and the rows that do see them get them back at the
// end (add_odd()): a weight is positive, so what they make of the sum does not
// depend on it.  In the other steps they enter as they are.  What the products hold of
// a weight may be 0 (one that rounds to it) or less (its second piece), which makes a
// NaN of an infinity; so where channels end as NaN in a row whose weights are numbers,
// the sum of what it sees there is formed anew, without weights.

// Zeroes the non-finite ones (an exponent of ones) of two 16-bit values.
template <int DT>
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
    constexpr uint32_t e = DT == kSrcBF16 ? 0x7f80u : 0x7c00u;
    if ((w & e) == e) w &= 0xffff0000u;
    if ((w >> 16 & e) == e) w &= 0xffffu;
    return w;
}
__device__ __forceinline__ bool non_finite(float x) {
    return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
}

// Four rows' 16-bit elements, read transposed: the 16 lanes of a group give the
// addresses of 4 consecutive elements each, lane 4r + c of row r's columns 4c ..
// 4c + 3; lane i receives column i of rows 0 .. 3.
__device__ __forceinline__ uint2 read_transposed(const unsigned char* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4_t*)(p)));
}

// A workgroup's item and where its sequence's pages lie.
struct Work {
    PagedItem it;
    int kvh, rows, hg;
    // (the constant address space: scalar loads, whatever else is written)
    const __attribute__((address_space(4))) int32_t* pages;
    uint32_t head_off;           // of the kv head within a page, in elements
    uint32_t page_elems;
};

__device__ __forceinline__ Work work_of(const PagedLaunch& a) {
    Work w;
    const int item = blockIdx.x / a.Hkv;
    w.kvh = blockIdx.x - item * a.Hkv;
    w.it = a.items[item];
    w.hg = a.hg;
    w.rows = w.it.n * a.hg;
    w.pages = (const __attribute__((address_space(4))) int32_t*)(a.pages + w.it.page0);
    w.head_off = ((uint32_t)w.kvh << a.page_shift) * a.D;
    w.page_elems = ((uint32_t)a.Hkv << a.page_shift) * a.D;
    return w;
}

// Positions are loaded in blocks of 16, which never cross a page.  A block's
// page id (the block of the last position for blocks past the end), and the
// address of its first row.
__device__ __forceinline__ int block_page(const PagedLaunch& a, const Work& w, int t) {
    return w.pages[min(t, w.it.kv_end - 1) >> a.page_shift];
}
template <class T>
__device__ __forceinline__ const T* block_at(const PagedLaunch& a, const Work& w,
                                             const void* pool, int page, int t) {
    const int off = min(t, (w.it.kv_end - 1) & ~15) & ((1 << a.page_shift) - 1);
    return static_cast<const T*>(pool) + (uint64_t)(uint32_t)page * w.page_elems + w.head_off +
           (uint32_t)(off * a.D);
}

// Positions that row r sees, within the split.
__device__ __forceinline__ int row_limit(const Work& w, int r) {
    return min(w.it.ctx - w.it.n + r / w.hg + 1, w.it.kv_end);
}
__device__ __forceinline__ int64_t out_offset(const PagedLaunch& a, const Work& w, int r) {
    const int i = r / w.hg;
    return ((int64_t)(w.it.tok0 + i) * a.Hq + w.kvh * w.hg + (r - i * w.hg)) * a.D;
}
__device__ __forceinline__ int64_t q_offset(const PagedLaunch& a, const Work& w, int r) {
    const int i = r / w.hg;
    return (w.it.tok0 + i) * a.q_st + (int64_t)(w.kvh * w.hg + (r - i * w.hg)) * a.q_sh;
}
// The first row of a partial of a sequence with `rows` rows.
__device__ __forceinline__ int64_t part_at(const PagedLaunch& a, int kvh, int part, int rows) {
    return kvh * a.part_total + (paged_few(rows) ? (int64_t)part * a.few_rows
                                                 : a.many_at + (int64_t)part * a.part_rows);
}
__device__ __forceinline__ int64_t part_row(const PagedLaunch& a, const Work& w, int r) {
    return part_at(a, w.kvh, w.it.part, w.rows) + (r - w.it.row0);
}

// Four consecutive elements, widened.
template <int DT>
__device__ __forceinline__ f32x4_t load4(const void* p, int64_t i) {
    if constexpr (DT == kSrcF32) {
        return *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p) + i);
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
        return f32x4_t{half_of<DT>(x.x, 0), half_of<DT>(x.x, 1), half_of<DT>(x.y, 0),
                       half_of<DT>(x.y, 1)};
    }
}

// Four consecutive channels of an output row, rounded once.
template <int DT>
__device__ __forceinline__ void store4(void* out, int64_t i, f32x4_t x) {
    if constexpr (DT == kSrcF32)
        *reinterpret_cast<f32x4_t*>(static_cast<float*>(out) + i) = x;
    else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i) =
            make_uint2(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]));
}

// The sum of the non-finite values of positions t .. lim - 1 (t a multiple of 8) in four
// channels, the ones asked for (done once all of these are NaN).  Eight loads at a time
// (one infinity early in one of 64 sequences of 8K: 0.78 ms a call, one load at a time
// 2.5, without it 0.29).
template <int DT>
__device__ __forceinline__ f32x4_t odd_values(const PagedLaunch& a, const Work& w, int t, int lim,
                                           int c, const bool (&asked)[4]) {
    constexpr int kAtOnce = 8;
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (; t < lim; t += kAtOnce) {
        const int64_t at = (int64_t)w.pages[t >> a.page_shift] * w.page_elems + w.head_off +
                           (t & ((1 << a.page_shift) - 1)) * a.D + c;
        f32x4_t x[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)                // (the last one again changes nothing)
            x[j] = load4<DT>(a.v_pages, at + min(j, lim - 1 - t) * a.D);
        bool done = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) sum[i] += non_finite(x[j][i]) ? x[j][i] : 0.f;
            done &= !asked[i] || sum[i] != sum[i];
        }
        if (done) break;
    }
    return sum;
}
__device__ __forceinline__ bool has_nan(f32x4_t o) {
    return o[0] != o[0] || o[1] != o[1] || o[2] != o[2] || o[3] != o[3];
}
// Four channels of a row that sees the positions up to lim, of weights' sum `sum`:
// the non-finite values added.  odd: some in the steps of `unit` positions that not all
// rows (which all see `all`) see to their ends, where they entered as 0.
template <int DT>
__device__ __forceinline__ void add_odd(const PagedLaunch& a, const Work& w, int all, int unit,
                                        int lim, int c, float sum, bool odd, f32x4_t& o) {
    const bool lost = sum == sum && has_nan(o);
    if (!odd && !lost) return;
    bool asked[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) asked[i] = odd || o[i] != o[i];
    const int from = lost ? 0 : max(0, all - w.it.kv_begin) / unit * unit;
    const f32x4_t x = odd_values<DT>(a, w, w.it.kv_begin + from, lim, c, asked);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (lost && asked[i]) o[i] = non_finite(x[i]) ? x[i] : o[i];
        else o[i] += asked[i] ? x[i] : 0.f;
    }
}

// 1 / sum; a row that saw nothing has sum 0 and comes out as zeros.
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.f ? 0.f : 1.0f / l; }

// Four channels of row r of an item that is done: `o` of sum `sum` at maximum
// `top`.
template <int DT>
__device__ __forceinline__ void store_row(const PagedLaunch& a, const Work& w, int r, int c,
                                          f32x4_t o, float top, float sum) {
    if (w.it.part < 0) {
        store4<DT>(a.out, out_offset(a, w, r) + c, o);
    } else {
        const int64_t at = part_row(a, w, r);
        *reinterpret_cast<f32x4_t*>(a.part_o + at * a.D + c) = o;
        if (c == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * at) = make_float2(top, sum);
    }
}
// add_odd() for channels that the lane has stored (a loop over them, once in the code,
// where the kernel has them in registers by constant numbers).
template <int DT>
__device__ __forceinline__ void mend_row(const PagedLaunch& a, const Work& w, int r, int c,
                                         float top, float sum, bool odd, int unit) {
    f32x4_t o;
    if (w.it.part < 0) o = load4<DT>(a.out, out_offset(a, w, r) + c);
    else o = *reinterpret_cast<const f32x4_t*>(a.part_o + part_row(a, w, r) * a.D + c);
    add_odd<DT>(a, w, w.it.ctx - w.it.n + w.it.row0 / w.hg + 1, unit, row_limit(w, r), c, sum, odd, o);
    store_row<DT>(a, w, r, c, o, top, sum);
}

// Joins WAVES waves' results of ROWS rows (row i of wave j at jo(j) + i * stride,
// each scaled to the largest of the waves' maxima) and finishes the rows from
// row0.  By all 256 threads of a workgroup.  ODD: values may not be finite (codes always
// are).
template <int DT, int DP, int ROWS, int WAVES, bool ODD = true, class F>
__device__ __forceinline__ void join_waves(const PagedLaunch& a, const Work& w, int row0, F jo,
                                           int stride, const float (*m)[ROWS],
                                           const float (*l)[ROWS], bool odd, int unit) {
    for (int at = threadIdx.x; at < ROWS * (DP / 4); at += 4 * kWave) {
        const int row = at / (DP / 4), c = at % (DP / 4) * 4, r = row0 + row;
        if (r >= w.rows || c >= a.D) continue;
        float top = m[0][row];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) top = fmaxf(top, m[i][row]);
        f32x4_t o = {0.f, 0.f, 0.f, 0.f};
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            o += *reinterpret_cast<const f32x4_t*>(jo(i) + row * stride + c);
            sum += l[i][row] * exp2_fast(m[i][row] - top);
        }
        if (w.it.part < 0) o *= inverse_sum(sum);
        if constexpr (ODD)
            add_odd<DT>(a, w, w.it.ctx - w.it.n + w.it.row0 / w.hg + 1, unit, row_limit(w, r), c,
                        sum, odd, o);
        store_row<DT>(a, w, r, c, o, top, sum);
    }
}

}  // namespace

void launch_paged_few(const PagedLaunch& a, int dtype, hipStream_t s);
void launch_paged_f32(const PagedLaunch& a, int kind, hipStream_t s);
void launch_paged_many(const PagedLaunch& a, int dtype, hipStream_t s);

}  // namespace kivi
