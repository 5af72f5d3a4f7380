// Sampling next tokens from logits with given random numbers.
//
// A row's tokens are ordered by (logit descending, index ascending), with
// weights w = exp((x - max) / temperature).  Kept are the first top_k; of these
// the shortest prefix that holds top_p of their mass; of those the tokens with
// w >= min_p (the first one always).  All three cut the order to a prefix, so
// the kept mass is one of the order's running sums S, and the token is the first
// whose S exceeds u times it.  Nothing is sorted: what is needed of the order is
// where its running count or mass crosses a border, three times at most for the
// kept prefix and once for the token.
//
// A border is found by bucket, then within one: the row's 4096 buckets are
// 1/128 wide in (max - x) / temperature, whose counts and masses one pass sums;
// a second pass collects the border's bucket (a few tokens; where it holds more
// than a workgroup's threads, sub-buckets of its keys narrow it first), and its
// tokens are ranked against each other.
//
// Precision: neighbouring tokens' borders lie as close as a token's share of the
// mass, 1e-6 and less, and sums of fp32 weights over 10^5 tokens are off by more
// than that.  Weights are computed in fp64 (2^-47 relative) and summed as
// integers in units of 2^-43 of the largest weight, exactly and in any order.
// Tokens below half a unit (w < 2^-44) have no mass: all of a million of them
// together are below 2^-24 of it.
#include <hip/hip_runtime.h>

#include <math.h>

#include "kivi_common.hpp"
#include "kivi_mfma.hpp"
#include "../../include/kivi_hip.h"

namespace kivi {
namespace {

constexpr int kBlock = 1024;
constexpr int kBuckets = 4096;
constexpr float kPerUnit = 128.f;         // buckets per unit of (max - x) / t
constexpr int kUnitBits = 43;
constexpr int kMaxVocab = 1 << 20;        // (sums stay below 2^63)
constexpr int kSub = 2048;                // sub-buckets of a crowded bucket

struct SampleArgs {
    const void* logits;
    int64_t stride;
    int V;
    const void* u;
    int u_f64;
    const float* t_row;      // per row, or NULL: the scalar
    const int* k_row;
    const float* p_row;
    const float* m_row;
    double t, p, m;
    int k;
    int64_t* out;
};

// Order-preserving bits of a logit, largest first: keys ascend as logits
// descend.  -0 counts as 0, NaN as -infinity.
__device__ __forceinline__ uint32_t order_bits(float x) {
    x = x == 0.f ? 0.f : x;
    x = x != x ? -INFINITY : x;
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ float logit_of(uint32_t bits) {
    return __uint_as_float(bits & 0x80000000u ? bits : ~bits & 0x7fffffffu);
}

// The tokens' weights in units of 2^-43 of the largest.
struct Weights {
    double top, per;         // the largest logit, log2(e) / temperature
    float top32, bucket;     // buckets per unit of logit

    __device__ __forceinline__ void set(float mx, double t) {
        top = mx;
        top32 = mx;
        per = 1.4426950408889634074 / t;
        bucket = (float)(kPerUnit / t);
    }
    // 2^y by its series in y ln 2 around the nearest integer: the eleventh
    // power's remainder is 0.35^12 / 12! < 2^-46.
    __device__ __forceinline__ uint64_t mass(float x) const {
        const double y = ((double)x - top) * per;
        if (x == top32) return 1ull << kUnitBits;          // (infinities too)
        if (!(y > -46.0)) return 0;
        const double n = __builtin_rint(y), z = (y - n) * 0.69314718055994530942;
        double e = 1.0 / 39916800.0;
        e = __builtin_fma(e, z, 1.0 / 3628800.0);
        e = __builtin_fma(e, z, 1.0 / 362880.0);
        e = __builtin_fma(e, z, 1.0 / 40320.0);
        e = __builtin_fma(e, z, 1.0 / 5040.0);
        e = __builtin_fma(e, z, 1.0 / 720.0);
        e = __builtin_fma(e, z, 1.0 / 120.0);
        e = __builtin_fma(e, z, 1.0 / 24.0);
        e = __builtin_fma(e, z, 1.0 / 6.0);
        e = __builtin_fma(e, z, 0.5);
        e = __builtin_fma(e, z, 1.0);
        e = __builtin_fma(e, z, 1.0);
        return (uint64_t)__builtin_rint(ldexp(e, (int)n + kUnitBits));
    }
    // (monotone: each step rounds monotonely; at 4096 w is below 2^-46)
    __device__ __forceinline__ int bucket_of(float x) const {
        if (x == top32) return 0;
        const float b = (top32 - x) * bucket;
        return b < (float)kBuckets ? (int)b : kBuckets;
    }
};

// f(x, index) for the row's tokens: 16-byte loads between the first and the last
// 16-byte border, single ones outside.
template <int DT, class F>
__device__ __forceinline__ void each_token(const SampleArgs& a, int row, F f) {
    constexpr int kSize = src_size(DT), kVec = 16 / kSize;
    const char* base = static_cast<const char*>(a.logits) + row * a.stride * kSize;
    const int head = min(a.V, (int)((16 - ((uintptr_t)base & 15)) & 15) / kSize);
    const int vecs = (a.V - head) / kVec, tail = head + vecs * kVec;
    if ((int)threadIdx.x < head) f(widen<DT>(base, threadIdx.x), (int)threadIdx.x);
    if ((int)threadIdx.x < a.V - tail)
        f(widen<DT>(base, tail + threadIdx.x), tail + (int)threadIdx.x);
    const uint4* v = reinterpret_cast<const uint4*>(base + head * kSize);
#pragma unroll 2
    for (int i = threadIdx.x; i < vecs; i += kBlock) {
        const uint4 w = v[i];
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
        const int at = head + i * kVec;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == kSrcF32) {
                f(__uint_as_float(words[j]), at + j);
            } else if constexpr (DT == kSrcBF16) {
                f(__uint_as_float(words[j] << 16), at + 2 * j);
                f(__uint_as_float(words[j] & 0xffff0000u), at + 2 * j + 1);
            } else {
                f((float)__builtin_bit_cast(_Float16, (uint16_t)(words[j] & 0xffffu)), at + 2 * j);
                f((float)__builtin_bit_cast(_Float16, (uint16_t)(words[j] >> 16)), at + 2 * j + 1);
            }
        }
    }
}

struct Shared {
    uint64_t mass[kBuckets];         // then the running sum before each bucket
    uint32_t count[kBuckets];
    union {
        struct {
            uint64_t key[kBlock];
            uint64_t mass[kBlock];
        } list;
        struct {
            uint64_t mass[kSub];
            uint32_t count[kSub];
        } sub;
    };
    uint64_t wave_mass[kBlock / kWave];
    uint32_t wave_count[kBlock / kWave];
    uint64_t key_min, key_max, hit_mass;
    uint32_t listed, hit;
};

// A place in the order: the running count or mass to be reached.
enum Border : int {
    kByCount,       // the token that is number `at`
    kByMass,        // the first whose running sum reaches `at`
    kPast,          // the first whose running sum exceeds `at`
};

template <int DT>
struct Sampler {
    const SampleArgs& a;
    Shared& s;
    int row;
    Weights w;
    uint64_t all_mass;
    uint32_t all_count;

    // Exclusive running sums of n counts and masses, in place; the totals.
    __device__ void scan(uint64_t* mass, uint32_t* count, int n, uint64_t& tm, uint32_t& tc) {
        const int tid = threadIdx.x, lane = tid % kWave, per = n / kBlock;
        uint64_t m = 0;
        uint32_t c = 0;
        for (int i = 0; i < per; ++i) {
            m += mass[tid * per + i];
            c += count[tid * per + i];
        }
        uint64_t im = m;
        uint32_t ic = c;
        for (int d = 1; d < kWave; d *= 2) {
            const uint64_t om = __shfl_up(im, d);
            const uint32_t oc = __shfl_up(ic, d);
            if (lane >= d) {
                im += om;
                ic += oc;
            }
        }
        if (lane == kWave - 1) {
            s.wave_mass[tid / kWave] = im;
            s.wave_count[tid / kWave] = ic;
        }
        __syncthreads();
        uint64_t bm = im - m;
        uint32_t bc = ic - c;
        tm = tc = 0;
        for (int i = 0; i < kBlock / kWave; ++i) {
            if (i < tid / kWave) {
                bm += s.wave_mass[i];
                bc += s.wave_count[i];
            }
            tm += s.wave_mass[i];
            tc += s.wave_count[i];
        }
        for (int i = 0; i < per; ++i) {
            const uint64_t xm = mass[tid * per + i];
            const uint32_t xc = count[tid * per + i];
            mass[tid * per + i] = bm;
            count[tid * per + i] = bc;
            bm += xm;
            bc += xc;
        }
        __syncthreads();
    }

    // The last of n entries whose running sum before it has not reached the
    // border: the one that crosses it.
    __device__ static int crossing(const uint64_t* mass, const uint32_t* count, int n, Border kind,
                                   uint64_t at) {
        int lo = 0, hi = n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            const uint64_t v = kind == kByCount ? count[mid] : mass[mid];
            if (kind == kPast ? v <= at : v < at) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    }

    // The running sum up to and with the token at the border, and its index.
    // `at` lies in the total of all buckets.
    __device__ uint64_t find(Border kind, uint64_t at, int& index) {
        const int tid = threadIdx.x;
        const int b = crossing(s.mass, s.count, kBuckets, kind, at);
        uint64_t base_mass = s.mass[b], lo = 0, hi = ~0ull;
        uint32_t base_count = s.count[b];
        while (true) {
            // collect the bucket's tokens between two keys
            __syncthreads();
            if (tid == 0) {
                s.listed = 0;
                s.key_min = ~0ull;
                s.key_max = 0;
            }
            __syncthreads();
            uint64_t mn = ~0ull, mx = 0;
            each_token<DT>(a, row, [&](float x, int i) {
                if (w.bucket_of(x) != b) return;
                const uint64_t key = (uint64_t)order_bits(x) << 32 | (uint32_t)i;
                if (key < lo || key > hi) return;
                mn = min(mn, key);
                mx = max(mx, key);
                const uint32_t n = atomicAdd(&s.listed, 1u);
                if (n < kBlock) s.list.key[n] = key;
            });
            if (mx >= mn) {
                atomicMin((unsigned long long*)&s.key_min, (unsigned long long)mn);
                atomicMax((unsigned long long*)&s.key_max, (unsigned long long)mx);
            }
            __syncthreads();
            const uint32_t n = s.listed;
            if (n <= kBlock) {
                uint64_t key = 0, mass = 0;
                if (tid < (int)n) {
                    key = s.list.key[tid];
                    mass = w.mass(logit_of((uint32_t)(key >> 32)));
                    s.list.mass[tid] = mass;
                }
                __syncthreads();
                if (tid < (int)n) {
                    uint64_t before = base_mass;
                    uint32_t rank = base_count;
                    for (uint32_t j = 0; j < n; ++j) {
                        if (s.list.key[j] < key) {
                            before += s.list.mass[j];
                            ++rank;
                        }
                    }
                    const bool hit = kind == kByCount  ? rank + 1 == at
                                     : kind == kByMass ? before < at && at <= before + mass
                                                       : before <= at && at < before + mass;
                    if (hit) {
                        s.hit = (uint32_t)key;
                        s.hit_mass = before + mass;
                    }
                }
                __syncthreads();
                index = (int)s.hit;
                return s.hit_mass;
            }
            // too many: counts and masses of 2048 stretches of their keys
            const uint64_t first = s.key_min, span = s.key_max - first;
            int shift = 0;
            while (span >> shift >= kSub) ++shift;
            __syncthreads();
            for (int i = tid; i < kSub; i += kBlock) {
                s.sub.mass[i] = 0;
                s.sub.count[i] = 0;
            }
            __syncthreads();
            each_token<DT>(a, row, [&](float x, int i) {
                if (w.bucket_of(x) != b) return;
                const uint64_t key = (uint64_t)order_bits(x) << 32 | (uint32_t)i;
                if (key < lo || key > hi) return;
                const int at_sub = (int)((key - first) >> shift);
                atomicAdd((unsigned long long*)&s.sub.mass[at_sub], (unsigned long long)w.mass(x));
                atomicAdd(&s.sub.count[at_sub], 1u);
            });
            __syncthreads();
            uint64_t tm;
            uint32_t tc;
            scan(s.sub.mass, s.sub.count, kSub, tm, tc);
            const uint64_t rest = kind == kByCount ? at - base_count : at - base_mass;
            const int at_sub = crossing(s.sub.mass, s.sub.count, kSub, kind, rest);
            base_mass += s.sub.mass[at_sub];
            base_count += s.sub.count[at_sub];
            lo = first + ((uint64_t)at_sub << shift);
            hi = lo + ((1ull << shift) - 1);
        }
    }
};

template <int DT>
__global__ void __launch_bounds__(kBlock) sample_kernel(SampleArgs a) {
    __shared__ Shared s;
    const int row = blockIdx.x, tid = threadIdx.x;
    Sampler<DT> r{a, s, row, {}, 0, 0};

    // the first token of the order
    uint64_t best = ~0ull;
    each_token<DT>(a, row, [&](float x, int i) {
        best = min(best, (uint64_t)order_bits(x) << 32 | (uint32_t)i);
    });
    for (int d = 1; d < kWave; d *= 2) best = min(best, (uint64_t)__shfl_xor(best, d));
    if (tid % kWave == 0) s.wave_mass[tid / kWave] = best;
    for (int i = tid; i < kBuckets; i += kBlock) {
        s.mass[i] = 0;
        s.count[i] = 0;
    }
    __syncthreads();
    for (int i = 0; i < kBlock / kWave; ++i) best = min(best, s.wave_mass[i]);
    const float top = logit_of((uint32_t)(best >> 32));

    const double t = a.t_row ? (double)a.t_row[row] : a.t;
    const double p = a.p_row ? (double)a.p_row[row] : a.p;
    const double m = a.m_row ? (double)a.m_row[row] : a.m;
    const int k = a.k_row ? a.k_row[row] : a.k;
    double u = a.u_f64 ? static_cast<const double*>(a.u)[row]
                       : (double)static_cast<const float*>(a.u)[row];
    u = u > 0.0 ? fmin(u, 1.0) : 0.0;          // (NaN: 0)

    const bool none = top == -INFINITY;
    if (none || !(t > 0.0) || k == 1 || p <= 0.0) {
        if (tid == 0) a.out[row] = none ? -1 : (int64_t)(uint32_t)best;
        return;
    }
    r.w.set(top, t);
    __syncthreads();                           // (wave_mass was read)
    each_token<DT>(a, row, [&](float x, int) {
        const int b = r.w.bucket_of(x);
        if (b >= kBuckets) return;
        atomicAdd((unsigned long long*)&s.mass[b], (unsigned long long)r.w.mass(x));
        atomicAdd(&s.count[b], 1u);
    });
    __syncthreads();
    uint64_t kept;
    uint32_t count;
    r.scan(s.mass, s.count, kBuckets, kept, count);
    int index = 0;
    if (k > 0 && (uint32_t)k < count) kept = r.find(kByCount, (uint64_t)k, index);
    if (p < 1.0) {
        uint64_t want = (uint64_t)ceil(p * (double)kept);
        want = want < 1 ? 1 : want > kept ? kept : want;
        kept = r.find(kByMass, want, index);
    }
    if (m > 0.0) {
        // the running sum of tokens with w >= min_p (the first one at least)
        const double unit = (double)(1ull << kUnitBits);
        uint64_t sum = 0;
        __syncthreads();
        if (tid == 0) s.hit_mass = 0;
        __syncthreads();
        each_token<DT>(a, row, [&](float x, int) {
            const uint64_t mass = r.w.mass(x);
            if ((double)mass >= m * unit) sum += mass;
        });
        for (int d = 1; d < kWave; d *= 2) sum += __shfl_xor(sum, d);
        if (tid % kWave == 0) atomicAdd((unsigned long long*)&s.hit_mass, (unsigned long long)sum);
        __syncthreads();
        sum = s.hit_mass;
        kept = min(kept, max(sum, (uint64_t)1 << kUnitBits));
    }
    uint64_t past = (uint64_t)(u * (double)kept);
    past = past >= kept ? kept - 1 : past;
    r.find(kPast, past, index);
    if (tid == 0) a.out[row] = index;
}

}  // namespace
}  // namespace kivi

using namespace kivi;

extern "C" {

int kivi_sample(const void* logits, int32_t dtype, int64_t row_stride, int32_t rows,
                int32_t vocab, const void* uniforms, int32_t uniforms_f64,
                const float* temperatures, double temperature, const int32_t* top_ks,
                int32_t top_k, const float* top_ps, double top_p, const float* min_ps,
                double min_p, int64_t* out, void* stream) {
    if (dtype < 0 || dtype > 2)
        return set_error(kErrInvalidArgument, "dtype %d is not 0 (f32), 1 (bf16) or 2 (f16)", dtype);
    if (rows < 0 || vocab < 1 || vocab > kMaxVocab)
        return set_error(kErrInvalidArgument, "logits of %d rows and %d tokens (1 to %d)", rows,
                         vocab, kMaxVocab);
    if (rows == 0) return kOk;
    if (row_stride < 0)
        return set_error(kErrInvalidArgument, "row_stride %lld must not be negative",
                         (long long)row_stride);
    if (logits == nullptr || uniforms == nullptr || out == nullptr)
        return set_error(kErrInvalidArgument, "null pointer");
    SampleArgs a{};
    a.logits = logits;
    a.stride = row_stride;
    a.V = vocab;
    a.u = uniforms;
    a.u_f64 = uniforms_f64 != 0;
    a.t_row = temperatures;
    a.k_row = top_ks;
    a.p_row = top_ps;
    a.m_row = min_ps;
    a.t = temperature;
    a.k = top_k;
    a.p = top_p;
    a.m = min_p;
    a.out = out;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == kSrcF32) sample_kernel<kSrcF32><<<rows, kBlock, 0, s>>>(a);
    else if (dtype == kSrcBF16) sample_kernel<kSrcBF16><<<rows, kBlock, 0, s>>>(a);
    else sample_kernel<kSrcF16><<<rows, kBlock, 0, s>>>(a);
    return check_launch("sample");
}

}  // extern "C"
