// Logits changed before sampling: penalties for repeated tokens, biases, masks.
//
// For token v of a row with logit x, n times among the row's generated tokens:
//   x > 0 ? x / r : x * r      where v is among its tokens, prompt or generated
//   x - (f n + p)              where n > 0
//   x + b                      b: the biases that the row lists for v, added up in order
//   -infinity                  where the row's mask does not allow v
// in fp32, rounded once; a logit that none of this concerns keeps its bits.
//
// One launch: a workgroup takes a slice of a row's vocabulary.  It counts the row's tokens
// that lie in the slice in LDS (whole numbers: in any order the same), adds up the
// slice's biases there, and goes through its logits once.  Every slice reads all of its
// row's tokens, from L2.  The steps wait for each other, and for memory, rather than for
// operations, so whatever does not depend on a step before it is loaded at the start:
// logits, mask, biases and the first 16 tokens of each lane.
//
// A batch is bound by the instructions of counting and of what the counts change, half of
// the vector units' time (64 rows of 128256, bf16, lists of 4000, 40 biases and a mask:
// 16.0 us, 2.2 TB/s; in a captured graph 17.3, without tokens 9.7, with nothing 6.5), one row and long lists by the
// chain of their steps (50257 fp32 with a list of 300: 10 us a call, 3.9 on the GPU; 16 rows
// of 32000 with lists of 30000: 11).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "kivi_common.hpp"
#include "../../include/kivi_hip.h"

namespace kivi {
namespace {

// Tokens of a workgroup, as measured (64 rows of 128256 with lists of 4000: 256 lanes and
// 2048 tokens 17.3 us, 512 and 4096 17.7, 1024 and 8192 18.8; 16 rows of 32000 with lists of
// 30000: 1024 lanes and 4096 11 us).
constexpr int slice_of(int block) { return block == 256 ? 2048 : 4096; }
constexpr uint32_t kInPrompt = 1u << 31;     // of a count
constexpr uint32_t kNoBias = 0xffffffffu;    // (of no sum: NaN is stored as 0x7fc00000)
constexpr int kMostEntries = 1 << 30;        // (32-bit indexes look a turn past the last one)
// Longer lists are read by workgroups of 1024 lanes, shorter ones of 256.
constexpr int kManyTokens = 8192;

struct AdjustArgs {
    const void* logits;
    void* out;
    int64_t stride, out_stride;
    const void* tokens;                      // NULL: no penalties
    int64_t token_stride;
    const int32_t* lengths;
    const int32_t* prompts;
    const float* repetitions;
    const float* presences;
    const float* frequencies;
    const void* bias_ids;
    const float* bias;
    int64_t id_stride, bias_stride;
    const uint8_t* allowed;                  // bytes of the words
    int64_t allowed_stride;                  // in bytes
    float repetition, presence, frequency;
    int length, prompt, n_tokens, biases;
    int vocab, slices, token64, id64;
};

// Eight elements wherever they lie.
typedef uint32_t loose_u4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

template <int DT>
struct Eight {
    static constexpr int kWords = DT == kSrcF32 ? 8 : 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void load(const void* p, int64_t i) {
        const char* from = static_cast<const char*>(p) + i * src_size(DT);
#pragma unroll
        for (int j = 0; j < kWords; j += 4) {
            const u4 x = *reinterpret_cast<const loose_u4*>(from + 4 * j);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[j + k] = x[k];
        }
    }
    __device__ __forceinline__ void store(void* p, int64_t i) const {
        char* to = static_cast<char*>(p) + i * src_size(DT);
#pragma unroll
        for (int j = 0; j < kWords; j += 4)
            *reinterpret_cast<loose_u4*>(to + 4 * j) = u4{w[j], w[j + 1], w[j + 2], w[j + 3]};
    }
    __device__ __forceinline__ void load_some(const void* p, int64_t i, int n) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (DT == kSrcF32) {
                w[j] = j < n ? static_cast<const uint32_t*>(p)[i + j] : 0u;
            } else {
                const uint32_t h = j < n ? static_cast<const uint16_t*>(p)[i + j] : 0u;
                if (j % 2 == 0) w[j / 2] = h;
                else w[j / 2] |= h << 16;
            }
        }
    }
    __device__ __forceinline__ void store_some(void* p, int64_t i, int n) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (j >= n) continue;
            if (DT == kSrcF32) static_cast<uint32_t*>(p)[i + j] = w[j];
            else static_cast<uint16_t*>(p)[i + j] = (uint16_t)(w[j / 2] >> (16 * (j % 2)));
        }
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (DT == kSrcF32) return __uint_as_float(w[j]);
        const uint32_t h = w[j / 2] >> (16 * (j % 2)) & 0xffffu;
        if constexpr (DT == kSrcBF16) return __uint_as_float(h << 16);
        else return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
    }
    __device__ __forceinline__ void set(int j, float x) {
        if constexpr (DT == kSrcF32) {
            w[j] = __float_as_uint(x);
        } else {
            uint32_t h;
            if constexpr (DT == kSrcBF16) h = __builtin_bit_cast(uint16_t, (__bf16)x);
            else h = __builtin_bit_cast(uint16_t, (_Float16)x);
            w[j / 2] = j % 2 ? (w[j / 2] & 0xffffu) | h << 16 : (w[j / 2] & 0xffff0000u) | h;
        }
    }
};

__device__ __forceinline__ float setting(const float* rows, float all, int row) {
    return rows == nullptr ? all : rows[row];
}
__device__ __forceinline__ int64_t id_at(const void* ids, int64_t i, int wide) {
    return wide ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}

// A lane's next ids of a row's list: kLoads loads of 16 bytes, a turn of the workgroup's
// lanes apart.
template <int BLOCK, class I>
struct Ids {
    static constexpr int kLoads = 16 / sizeof(I) == 2 ? 8 : 4, kEach = 16 / sizeof(I);
    static constexpr int kTurn = BLOCK * kEach;
    I id[kLoads][kEach];

    // From `from` on, of `n` in the list; those behind its end are -1.
    __device__ __forceinline__ void load(const I* ids, int from, int n) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int left = n - from - j * kTurn, i = threadIdx.x * kEach;
            if (left <= 0) continue;
            const I* at = ids + from + j * kTurn + i;
            if (i + kEach <= left) {
                const u4 x = *reinterpret_cast<const loose_u4*>(at);
                __builtin_memcpy(id[j], &x, 16);
            } else {
#pragma unroll
                for (int k = 0; k < kEach; ++k) id[j][k] = i + k < left ? at[k] : (I)-1;
            }
        }
    }
    // Counts those that lie in the slice; the list's first `prompt` are the prompt.
    __device__ __forceinline__ void count(int from, int length, int prompt, uint32_t first,
                                          uint32_t n, uint32_t* counts) const {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            if (length - from - j * kTurn <= 0) continue;
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                const uint32_t at = (uint32_t)id[j][k] - first;
                if (at >= n || (sizeof(I) == 8 && (int64_t)id[j][k] >> 32 != 0)) continue;
                if (from + j * kTurn + (int)threadIdx.x * kEach + k < prompt)
                    atomicOr(counts + at, kInPrompt);
                else
                    atomicAdd(counts + at, 1u);
            }
        }
    }
};

// The slice's biases, each token's added up in the list's order: of the entries of a turn
// that name one token the first goes, then the next.  owner: 0 throughout, before and
// after.
template <int BLOCK>
struct Biases {
    int64_t id;
    float b;

    __device__ __forceinline__ void load(const AdjustArgs& a, int64_t row, int base) {
        const int i = base + threadIdx.x;
        id = -1;
        b = 0.f;
        if (i >= a.biases) return;
        id = id_at(a.bias_ids, row * a.id_stride + i, a.id64);
        b = a.bias[row * a.bias_stride + i];
    }
    __device__ __forceinline__ bool inside(uint32_t first, uint32_t n) const {
        return (uint64_t)(id - (int64_t)first) < n;
    }
    __device__ __forceinline__ void add(uint32_t first, uint32_t n, uint32_t* owner,
                                        uint32_t* sums) const {
        const uint64_t at = (uint64_t)(id - (int64_t)first);
        bool waits = inside(first, n);
        while (__syncthreads_or(waits)) {
            if (waits) atomicMax(owner + at, BLOCK - threadIdx.x);
            __syncthreads();
            const bool goes = waits && owner[at] == BLOCK - threadIdx.x;
            __syncthreads();
            if (goes) {
                const float s = sums[at] == kNoBias ? b : __uint_as_float(sums[at]) + b;
                sums[at] = s == s ? __float_as_uint(s) : 0x7fc00000u;
                owner[at] = 0;
                waits = false;
            }
        }
    }
};

template <int BLOCK, class I>
__device__ __forceinline__ void count_all(const AdjustArgs& a, int64_t row, int start, int length,
                                          int prompt, uint32_t first, uint32_t n,
                                          Ids<BLOCK, I>& ids, uint32_t* counts) {
    for (int from = start; from < length;) {
        ids.count(from, length, prompt, first, n, counts);
        if (length - from <= Ids<BLOCK, I>::kLoads * Ids<BLOCK, I>::kTurn) break;
        from += Ids<BLOCK, I>::kLoads * Ids<BLOCK, I>::kTurn;
        ids.load(static_cast<const I*>(a.tokens) + row * a.token_stride, from, length);
    }
}

// BIASED: sums of biases in LDS, behind the counts.
template <int DT, int OUT, int BLOCK, class I, bool BIASED>
__global__ void __launch_bounds__(BLOCK) adjust_logits_kernel(AdjustArgs a) {
    constexpr int kSlice = slice_of(BLOCK);
    static_assert(kSlice <= 8 * BLOCK, "eight logits of a lane");
    __shared__ __align__(16) uint32_t counts[kSlice];
    __shared__ __align__(16) uint32_t sums[BIASED ? kSlice : 4];
    const int row = blockIdx.x / a.slices;
    const uint32_t first = (blockIdx.x - row * a.slices) * (uint32_t)kSlice;
    const uint32_t n = min((uint32_t)kSlice, (uint32_t)a.vocab - first);

    const int64_t in = row * a.stride + first, to = row * a.out_stride + first;
    const uint8_t* allowed =
        a.allowed == nullptr ? nullptr : a.allowed + row * a.allowed_stride + first / 8;
    const uint32_t i = 8 * threadIdx.x;
    const int some = (int)min(8u, n - min(i, n));
    Eight<DT> x{};
    uint32_t bits = 0xff;
    if (some == 8) x.load(a.logits, in + i);
    else if (some > 0) x.load_some(a.logits, in + i, some);
    if (some > 0 && allowed != nullptr) bits = allowed[i / 8];
    Biases<BLOCK> biases;
    if constexpr (BIASED) biases.load(a, row, 0);

    float r = 1.f, p = 0.f, f = 0.f;
    int length = 0, prompt = 0;
    if (a.tokens != nullptr) {
        r = setting(a.repetitions, a.repetition, row);
        p = setting(a.presences, a.presence, row);
        f = setting(a.frequencies, a.frequency, row);
        if (!(r > 0.f)) r = 1.f;
        length = a.lengths == nullptr ? a.length : a.lengths[row];
        prompt = a.prompts == nullptr ? a.prompt : a.prompts[row];
        length = min(max(length, 0), a.n_tokens);
        prompt = min(max(prompt, 0), length);
    }
    const int start = r != 1.f ? 0 : prompt;
    const bool counted = start < length && (r != 1.f || p != 0.f || f != 0.f);
    Ids<BLOCK, I> ids;
    if (counted) ids.load(static_cast<const I*>(a.tokens) + row * a.token_stride, start, length);

    // (most slices have none of a short list's biases)
    bool biased = false;
    if (counted || BIASED) {
#pragma unroll
        for (int i = 0; i < kSlice; i += 4 * BLOCK)
            *reinterpret_cast<u4*>(counts + i + 4 * threadIdx.x) = u4{0, 0, 0, 0};
        if constexpr (BIASED)
            biased = __syncthreads_or(biases.inside(first, n)) || a.biases > BLOCK;
        else
            __syncthreads();
    }
    if (biased) {
#pragma unroll
        for (int i = 0; i < kSlice; i += 4 * BLOCK)
            *reinterpret_cast<u4*>(sums + i + 4 * threadIdx.x) =
                u4{kNoBias, kNoBias, kNoBias, kNoBias};
        biases.add(first, n, counts, sums);
        for (int base = BLOCK; base < a.biases; base += BLOCK) {
            biases.load(a, row, base);
            biases.add(first, n, counts, sums);
        }
    }
    if (counted) {
        count_all<BLOCK, I>(a, row, start, length, prompt, first, n, ids, counts);
        __syncthreads();
    }

    if (some == 0) return;
    Eight<OUT> y;
    if constexpr (DT == OUT) {
        y = x;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) y.set(j, x.get(j));
    }
    // (few lanes have a token that something concerns)
    uint32_t c[8], b[8], seen = 0, free = kNoBias;
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
        const u4 k = counted ? *reinterpret_cast<const u4*>(counts + i + h) : u4{0, 0, 0, 0};
        const u4 sum = biased ? *reinterpret_cast<const u4*>(sums + i + h)
                              : u4{kNoBias, kNoBias, kNoBias, kNoBias};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            c[h + j] = k[j];
            b[h + j] = sum[j];
            seen |= k[j];
            free &= sum[j];
        }
    }
    if (seen != 0 || free != kNoBias) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float v = x.get(j);
            if (c[j] != 0 && r != 1.f) v = v > 0.f ? v / r : v * r;
            const uint32_t k = c[j] & ~kInPrompt;
            if (k != 0) v = v - (f * (float)k + p);
            if (b[j] != kNoBias) v = v + __uint_as_float(b[j]);
            if (c[j] != 0 || b[j] != kNoBias) y.set(j, v);
        }
    }
    if (bits != 0xff) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if ((bits >> j & 1) == 0) y.set(j, -__builtin_inff());
    }
    if (some == 8) y.store(a.out, to + i);
    else y.store_some(a.out, to + i, some);
}

template <int DT, int OUT>
void launch(const AdjustArgs& a, unsigned grid, hipStream_t s) {
    auto with = [&](auto block, auto id) {
        constexpr int kBlock = decltype(block)::value;
        using I = decltype(id);
        if (a.biases > 0) adjust_logits_kernel<DT, OUT, kBlock, I, true><<<grid, kBlock, 0, s>>>(a);
        else adjust_logits_kernel<DT, OUT, kBlock, I, false><<<grid, kBlock, 0, s>>>(a);
    };
    const bool many = a.n_tokens > kManyTokens;
    if (many && a.token64) with(std::integral_constant<int, 1024>{}, int64_t{});
    else if (many) with(std::integral_constant<int, 1024>{}, int32_t{});
    else if (a.token64) with(std::integral_constant<int, 256>{}, int64_t{});
    else with(std::integral_constant<int, 256>{}, int32_t{});
}

}  // namespace
}  // namespace kivi

using namespace kivi;

extern "C" {

int kivi_adjust_logits(const void* logits, int32_t dtype, int64_t row_stride, int32_t rows,
                       int32_t vocab, const void* tokens, int32_t tokens_i64,
                       int64_t token_stride, int32_t n_tokens, const int32_t* lengths,
                       int32_t length, const int32_t* prompt_lengths, int32_t prompt_length,
                       const float* repetitions, float repetition, const float* presences,
                       float presence, const float* frequencies, float frequency,
                       const void* bias_ids, int32_t ids_i64, int64_t id_stride,
                       const float* bias, int64_t bias_stride, int32_t biases,
                       const uint32_t* allowed, int64_t allowed_stride, void* out,
                       int32_t out_dtype, int64_t out_stride, void* stream) {
    if (dtype < 0 || dtype > 2)
        return set_error(kErrInvalidArgument, "dtype %d is not 0 (f32), 1 (bf16) or 2 (f16)", dtype);
    if (out_dtype != dtype && out_dtype != kSrcF32)
        return set_error(kErrInvalidArgument, "out_dtype %d is neither 0 (f32) nor dtype", out_dtype);
    if (rows < 0 || vocab < 1)
        return set_error(kErrInvalidArgument, "%d rows of %d tokens", rows, vocab);
    if (n_tokens < 0 || n_tokens > kMostEntries || biases < 0 || biases > kMostEntries)
        return set_error(kErrInvalidArgument, "%d tokens, %d biases: at most %d of each are taken",
                         n_tokens, biases, kMostEntries);
    if (rows == 0) return kOk;
    if (logits == nullptr || out == nullptr || (n_tokens > 0 && tokens == nullptr) ||
        (biases > 0 && (bias_ids == nullptr || bias == nullptr)))
        return set_error(kErrInvalidArgument, "null pointer");
    if (((uintptr_t)logits & (src_size(dtype) - 1)) || ((uintptr_t)out & (src_size(out_dtype) - 1)))
        return set_error(kErrInvalidArgument, "logits and out must be aligned to their elements");
    // In place is one element at a time; any other overlap would read what was written.
    const char* from = static_cast<const char*>(logits);
    const char* to = static_cast<const char*>(out);
    const int64_t in_bytes = ((rows - 1) * row_stride + vocab) * src_size(dtype);
    const int64_t out_bytes = ((rows - 1) * out_stride + vocab) * src_size(out_dtype);
    const bool same = from == to && dtype == out_dtype && (rows == 1 || row_stride == out_stride);
    if (out_stride < vocab && rows > 1)
        return set_error(kErrInvalidArgument, "rows of out overlap");
    // (rows may lie between the other's, the same distance apart)
    const int64_t apart = row_stride * src_size(dtype), row = (int64_t)vocab * src_size(dtype);
    bool between = false;
    if (rows > 1 && apart > row && apart == out_stride * src_size(out_dtype)) {
        const int64_t off = ((to - from) % apart + apart) % apart;
        between = off >= row && off + (int64_t)vocab * src_size(out_dtype) <= apart;
    }
    if (!same && !between && from < to + out_bytes && to < from + in_bytes)
        return set_error(kErrInvalidArgument, "out must be logits or apart from them");
    AdjustArgs a{};
    a.logits = logits; a.out = out;
    a.stride = row_stride; a.out_stride = out_stride;
    a.tokens = n_tokens > 0 ? tokens : nullptr;
    a.token64 = tokens_i64; a.token_stride = token_stride; a.n_tokens = n_tokens;
    a.lengths = lengths; a.length = length;
    a.prompts = prompt_lengths; a.prompt = prompt_length;
    a.repetitions = repetitions; a.repetition = repetition;
    a.presences = presences; a.presence = presence;
    a.frequencies = frequencies; a.frequency = frequency;
    a.bias_ids = bias_ids; a.id64 = ids_i64; a.id_stride = id_stride;
    a.bias = bias; a.bias_stride = bias_stride; a.biases = biases;
    a.allowed = reinterpret_cast<const uint8_t*>(allowed);
    a.allowed_stride = 4 * allowed_stride;
    a.vocab = vocab;
    const bool many = n_tokens > kManyTokens;
    const int slice = slice_of(many ? 1024 : 256);
    a.slices = (int)(((int64_t)vocab + slice - 1) / slice);
    const int64_t blocks = (int64_t)rows * a.slices;
    if (blocks > (int64_t)UINT32_MAX / 1024)
        return set_error(kErrInvalidArgument, "%d rows of %d tokens are too many for one launch",
                         rows, vocab);
    const unsigned grid = (unsigned)blocks;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == kSrcF32) launch<kSrcF32, kSrcF32>(a, grid, s);
    else if (dtype == kSrcBF16 && out_dtype == dtype) launch<kSrcBF16, kSrcBF16>(a, grid, s);
    else if (dtype == kSrcBF16) launch<kSrcBF16, kSrcF32>(a, grid, s);
    else if (out_dtype == dtype) launch<kSrcF16, kSrcF16>(a, grid, s);
    else launch<kSrcF16, kSrcF32>(a, grid, s);
    return check_launch("adjust_logits");
}

}  // extern "C"
