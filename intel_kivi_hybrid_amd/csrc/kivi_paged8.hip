// Paged cache of 8 bits: the append of a step's new tokens.
//
// Pages hold codes, [num_pages][kv_heads][page_size][head_dim] int8, and beside them a
// scale for each block of 16 positions of a page and kv head, [num_pages][kv_heads]
// [page_size / 16] fp32: a key or value is code * scale.  Scales are powers of two:
//   s = the least 2^k, k >= -126, with |x| <= 127 s for every x of the block,
//   code = x / s, rounded to nearest even.
// Quotients by a power of two are exact, so a code is off by half a scale at most, and
// code * scale is a number of the 16-bit types as it is.  A block fills over several
// steps: where new tokens need a larger scale, the codes that it holds are rounded
// again, to whole bits less, so that all roundings of a code together stay below one
// final scale.  (Scales of 24 bits would be 1.4 times finer on average, and a block
// that grows by a little 15 times would be rounded 15 times, half a scale each.)
//
// A code goes by which side of a border its value lies on, so keys that are normed or
// rotated are formed in fp64: from fp32 one in 3e4 of them came out next to its
// definition's code.  It costs nothing that shows beside the memory traffic.  Queries
// are as in paged_append_kernel.
//
// A wave takes the tokens of a block of a kv head, keys or values, that fit its lanes
// (8 of 128 channels; as many waves of a workgroup as that takes share a block and meet
// once, over the scale): their rows, read once and held in registers until the block's
// largest is known; the scale; and the older codes, read only where the scale grows.
// Memory-bound for prompts, with the latency of a wave's steps beside it (9.3K tokens of
// 32/8 heads of 128 with norms, bf16: 60 us, 3.6 TB/s; blocks alone 27, queries alone 38,
// as two launches 65; a whole block to a wave, 162 registers in place of 108: 72),
// launch-bound for single tokens (64 of 64/8 heads, fp16: 5.3 us on the GPU).
#include <hip/hip_runtime.h>

#include <float.h>

#include "kivi_paged_rows.hpp"
#include "../../include/kivi_hip.h"

namespace kivi {
namespace {

struct Append8Args {
    AppendArgs a;
    float* k_scales;
    float* v_scales;
    const PagedBlock* blocks;
    uint32_t n_parts;            // blocks x kv heads
    uint32_t block_wgs;          // workgroups that their keys and values take, the first ones
};

constexpr int kLeast = -126;     // exponent of the smallest scale
constexpr int kNotFinite = 1 << 20;

// The exponent of the least scale for values up to `top`: 2^k >= top / 127.
__device__ __forceinline__ int scale_exponent(float top) {
    const uint32_t b = __float_as_uint(top);
    return (int)(b >> 23) - 133 + ((b & 0x7fffffu) > 0x7e0000u ? 1 : 0);
}
__device__ __forceinline__ int scale_exponent(double top) {
    const uint64_t b = __builtin_bit_cast(uint64_t, top);
    return (int)(b >> 52) - 1029 + ((b & 0xfffffffffffffull) > 0xfc00000000000ull ? 1 : 0);
}

template <int M>
__device__ __forceinline__ int max_with(int v) {
    return max(v, __float_as_int(seg_partner<M>(__int_as_float(v))));
}
__device__ __forceinline__ int wave_max_int(int v) {
    return max_with<32>(max_with<16>(max_with<8>(max_with<4>(max_with<2>(max_with<1>(v))))));
}

// Eight codes as they lie.
template <class T>
__device__ __forceinline__ uint2 codes_of(const T (&x)[8], T inverse) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        T r = x[j] * inverse;
        r = sizeof(T) == 8 ? (T)rint((double)r) : (T)rintf((float)r);
        r = r > (T)127 ? (T)127 : r < (T)-127 ? (T)-127 : r;   // (scales of another's making)
        w[j / 4] |= ((uint32_t)(int)r & 0xffu) << (8 * (j % 4));
    }
    return make_uint2(w[0], w[1]);
}
// Eight codes times `ratio`, rounded again.
__device__ __forceinline__ uint2 codes_again(uint2 c, float ratio) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)(int8_t)((j < 4 ? c.x : c.y) >> (8 * (j % 4)));
    return codes_of(x, ratio);
}

// A block's new rows into it, by WAVES waves (this one's tokens: `part`).  T: what norm
// and rotation are formed in.  meet(k): the largest of the waves' k.
template <int DT, int WAVES, class T, class M>
__device__ __forceinline__ void fill_block(const Append8Args& g, const PagedBlock& b, int kvh,
                                           bool key, int part, M meet) {
    const AppendArgs& a = g.a;
    const int lane = threadIdx.x % kWave;
    const HeadLane l = head_lane(a, lane & ((1 << a.lanes_log2) - 1));
    const int slot = part * (kScaleBlock / WAVES) + (lane >> a.lanes_log2), i = slot - b.held;
    const void* src = key ? a.k : a.v;
    const int64_t st = key ? a.k_st : a.v_st;
    const int64_t from = (b.tok + i) * st + kvh * (key ? a.k_sh : a.v_sh);
    const void* norm = key ? a.k_norm : nullptr;
    const bool fresh = l.live && i >= 0 && i < b.n, turned = fresh && key && l.inside;

    const int64_t page = b.slot >> a.page_shift;
    const int off = b.slot & ((1 << a.page_shift) - 1);
    const int64_t row = ((page * a.Hkv + kvh) << a.page_shift) + off;
    int8_t* codes = static_cast<int8_t*>(key ? a.k_pages : a.v_pages) + row * a.D + slot * a.D;
    float* scale = (key ? g.k_scales : g.v_scales) + row / kScaleBlock;

    Eight<DT> ex{}, ey{};
    Angles at;
    if (fresh) {
        ex.load(src, from + l.c0, a.vec);
        ey.load(src, from + l.c1, a.vec);
    }
    if (turned) at.load(a, l, b.position + i);
    const float old = b.held > 0 ? *scale : 0.f;
    T x[8], y[8];
    {
        float u[8], w[8];
        ex.widen(u);
        ey.widen(w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = u[j];
            y[j] = w[j];
        }
    }
    if (norm != nullptr) norm_row<T>(a, l, norm, x, y);
    if (turned) turn_row<T>(a, at, x, y);
    T top = 0;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const T m = x[j] < 0 ? -x[j] : x[j], n = y[j] < 0 ? -y[j] : y[j];
        finite &= m <= (T)FLT_MAX && n <= (T)FLT_MAX;
        top = m > top ? m : top;
        top = n > top ? n : top;
    }
    const int k = meet(wave_max_int(
        !fresh ? kLeast : finite ? max(scale_exponent(top), kLeast) : kNotFinite));
    // (what a block holds that is not a number keeps it so, until it starts anew)
    float s = k == kNotFinite ? __int_as_float(0x7fc00000) : __int_as_float((k + 127) << 23);
    if (old != old || (s == s && old > s)) s = old;
    const bool number = s == s;
    const T inverse = number ? (T)1 / (T)s : (T)0;
    if (part == 0 && lane == 0 && b.n > 0 && __float_as_uint(s) != __float_as_uint(old)) *scale = s;
    if (fresh) {
        const uint2 zero = make_uint2(0, 0);
        *reinterpret_cast<uint2*>(codes + l.c0) = number ? codes_of(x, inverse) : zero;
        *reinterpret_cast<uint2*>(codes + l.c1) = number ? codes_of(y, inverse) : zero;
    }
    if (b.held == 0 || !number || s == old || !l.live || slot >= b.held) return;
    const float ratio = old / s;
    uint2* to = reinterpret_cast<uint2*>(codes + l.c0);
    uint2* too = reinterpret_cast<uint2*>(codes + l.c1);
    const uint2 c = *to, d = *too;
    *to = codes_again(c, ratio);
    *too = codes_again(d, ratio);
}

// Query rows of workgroup `wg`, a segment of lanes each.
template <int DT>
__device__ __forceinline__ void move_query(const AppendArgs& a, uint32_t wg) {
    const uint32_t t = wg * kAppendBlock + threadIdx.x;
    const uint32_t row = t >> a.lanes_log2;
    const int tok = (int)(row / (uint32_t)a.Hq), h = (int)(row - (uint32_t)tok * (uint32_t)a.Hq);
    if (tok >= a.n_tokens) return;                       // (whole segments leave)
    move_row<DT>(a, head_lane(a, (int)(t & ((1u << a.lanes_log2) - 1))), a.q,
                 tok * a.q_st + (int64_t)h * a.q_sh, a.q_norm, true, a.tokens[tok].y, a.q_out,
                 ((int64_t)tok * a.Hq + h) * a.D);
}

template <int DT, int WAVES>
__global__ void __launch_bounds__(kAppendBlock) paged8_append_kernel(Append8Args g) {
    constexpr int kParts = kAppendBlock / kWave / WAVES;      // blocks of a workgroup
    const AppendArgs& a = g.a;
    if (blockIdx.x < g.block_wgs) {
        __shared__ int largest[kAppendBlock / kWave];
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
        // (keys by the first half of the workgroups, values by the others)
        const bool key = blockIdx.x < g.block_wgs / 2;
        const uint32_t p = (blockIdx.x - (key ? 0 : g.block_wgs / 2)) * kParts + wave / WAVES;
        const uint32_t at = min(p, g.n_parts - 1), block = at / (uint32_t)a.Hkv;
        const int kvh = (int)(at - block * (uint32_t)a.Hkv);
        PagedBlock b = g.blocks[block];
        if (p >= g.n_parts) b.n = b.held = 0;
        auto meet = [&](int k) {
            if constexpr (WAVES > 1) {
                largest[wave] = k;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < WAVES; ++i) k = max(k, largest[wave / WAVES * WAVES + i]);
            }
            return k;
        };
        if (key && (a.k_norm != nullptr || a.rot > 0))
            fill_block<DT, WAVES, double>(g, b, kvh, true, wave % WAVES, meet);
        else
            fill_block<DT, WAVES, float>(g, b, kvh, key, wave % WAVES, meet);
        return;
    }
    move_query<DT>(a, blockIdx.x - g.block_wgs);
}

template <int DT>
void launch_append(const Append8Args& g, unsigned grid, hipStream_t s) {
    if (g.a.lanes_log2 <= 2) paged8_append_kernel<DT, 1><<<grid, kAppendBlock, 0, s>>>(g);
    else if (g.a.lanes_log2 == 3) paged8_append_kernel<DT, 2><<<grid, kAppendBlock, 0, s>>>(g);
    else paged8_append_kernel<DT, 4><<<grid, kAppendBlock, 0, s>>>(g);
}

}  // namespace
}  // namespace kivi

using namespace kivi;

extern "C" {

int kivi_paged8_append(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                       const void* k, int64_t k_token_stride, int64_t k_head_stride,
                       const void* v, int64_t v_token_stride, int64_t v_head_stride,
                       int32_t dtype, void* q_out, int8_t* k_pages, int8_t* v_pages,
                       float* k_scales, float* v_scales, int64_t num_pages, int32_t page_size,
                       int32_t q_heads, int32_t kv_heads, int32_t head_dim, const int32_t* plan,
                       const int64_t* info, const float* cos, const float* sin,
                       int32_t rotary_dim, int32_t interleaved, const void* q_norm,
                       const void* k_norm, int32_t norm_dtype, float eps, void* stream) {
    if (info == nullptr) return set_error(kErrInvalidArgument, "null plan info");
    Append8Args g{};
    AppendArgs& a = g.a;
    const int rc = paged_append_args(a, q, q_token_stride, q_head_stride, k, k_token_stride,
                                     k_head_stride, v, v_token_stride, v_head_stride, dtype, q_out,
                                     k_pages, v_pages, num_pages, page_size, q_heads, kv_heads,
                                     head_dim, plan, (int32_t)info[kInfoTokens], cos, sin,
                                     rotary_dim, interleaved, q_norm, k_norm, norm_dtype, eps);
    if (rc || a.n_tokens == 0) return rc;
    if (k_scales == nullptr || v_scales == nullptr)
        return set_error(kErrInvalidArgument, "null scales");
    if (paged_plain_info(info))
        return set_error(kErrInvalidArgument, "the plan is not one of kivi_paged8_plan");
    g.k_scales = k_scales;
    g.v_scales = v_scales;
    g.blocks = reinterpret_cast<const PagedBlock*>(plan + info[kInfoBlocksAt]);
    const int64_t parts = info[kInfoBlocks] * kv_heads;
    const int64_t lanes = (int64_t)a.n_tokens * a.Hq << a.lanes_log2;
    // waves of a block: 16 tokens in 64 lanes
    const int waves = a.lanes_log2 <= 2 ? 1 : 1 << (a.lanes_log2 - 2);
    const int64_t wgs = (parts * waves + kAppendBlock / kWave - 1) / (kAppendBlock / kWave) * 2;
    if (parts * waves * kWave > INT32_MAX / 2 || lanes > INT32_MAX)
        return set_error(kErrInvalidArgument, "%d tokens are too many for one launch", a.n_tokens);
    g.n_parts = (uint32_t)parts;
    g.block_wgs = (uint32_t)wgs;
    const unsigned grid = (unsigned)(wgs + (lanes + kAppendBlock - 1) / kAppendBlock);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == kSrcF32) launch_append<kSrcF32>(g, grid, s);
    else if (dtype == kSrcBF16) launch_append<kSrcBF16>(g, grid, s);
    else launch_append<kSrcF16>(g, grid, s);
    return check_launch("paged8_append");
}

}  // extern "C"
