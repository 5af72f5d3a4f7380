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
// Two launches.  The first, a workgroup for each slice of 8192 tokens, sums counts
// and masses of the slice's buckets, 1/16 wide in x / temperature, and leaves its
// tokens in the buckets' order (a token's place is its bucket's count when it was
// added).  The borders lie in a few buckets that these sums name (the second to
// last border moves the last by less than a bucket's mass); the second launch, a
// workgroup for each row, takes their tokens from the slices and ranks those
// against each other, by sub-buckets where they are many.  Where they are more than
// fit its list (a flat distribution, or thousands of equal logits) it goes through the
// row instead: 64 rows of 128256 normal logits of deviation 1, temperature 1.3, top_p
// 0.9: fp32 268 us, bf16 410.
//
// Precision: neighbouring borders lie as close as a token's share of the mass,
// 1e-6 and less, and sums of fp32 weights over 10^5 tokens are off by more than
// that.  A token's weight is formed in fp64 as (edge of its bucket) x rel, with
// rel in [1, e^(1/16)) rounded to 2^-36 and summed as an integer, exactly and in
// any order; a bucket's sum is rounded to 2^-43 of the row's largest edge.  Tokens
// below e^-32 of a slice's largest have no mass (2^-46 of it, each).
//
// 64 rows of 128256 bf16 logits with settings of their own: 46 to 49 us a call (in a
// serialised trace the first launch 19, bound by its 55 vector operations for each
// token, the second 34, bound by the passes that one CU makes over a warm row's list of
// 4500 tokens); one row of 50257 fp32: 20 us (8 and 12, both the latency of their
// steps).  The logits' bytes alone would take 3 us.
#include <hip/hip_runtime.h>

#include <math.h>

#include "kivi_common.hpp"
#include "kivi_mfma.hpp"
#include "../../include/kivi_hip.h"

namespace kivi {
namespace {

constexpr int kSlice = 8192;              // tokens of a workgroup
constexpr int kBlock = 512;               // its threads
constexpr int kPickBlock = 1024;
// tokens that are ranked against each other (64 rows of 128256 bf16: 64 52 us, 128
// 49, 256 51, 512 59)
constexpr int kFew = 128;
constexpr int kBuckets = 512;
constexpr double kPerUnit = 16.0;         // buckets per unit of x / t
constexpr int kRelBits = 36, kMassBits = 43;
constexpr int kCountShift = 50;           // a slice's rels stay below 2^50
constexpr uint64_t kRelMask = (1ull << kCountShift) - 1;
constexpr int kMaxVocab = 1 << 20;        // (a row's rels stay below 2^57)
constexpr int kList = 6144;               // tokens that a row's list holds
constexpr int kOrder = kSlice + 16;       // a slice's tokens, and the ones outside of vectors
constexpr int kStarts = kBuckets + 8;     // (whole 16 bytes)
// sub-buckets of a crowded bucket, in copies of which a lane takes one (16-bit logits
// have few values: their tokens meet in few sub-buckets)
constexpr int kSub = 512, kCopies = 4;

struct SampleArgs {
    const void* logits;
    int64_t stride;
    int V, slices;
    const void* u;
    int u_f64;
    const float* t_row;      // per row, or NULL: the scalar
    const int* k_row;
    const float* p_row;
    const float* m_row;
    double t, p, m;
    int k;
    int64_t* out;
    // workspace
    uint64_t* hist;          // [row][slice][bucket]: count << 50 | sum of rels
    uint64_t* best;          // [row][slice]: the first token's key
    uint16_t* order;         // [row][slice][kOrder]: its tokens by bucket
    uint16_t* starts;        // [row][slice][kStarts]: where each bucket's begin
};

struct Settings {
    double t, p, m, u;
    int k;
    bool first;              // the first token of the order, whatever u
};

__device__ __forceinline__ Settings settings_of(const SampleArgs& a, int row) {
    Settings s;
    s.t = a.t_row ? (double)a.t_row[row] : a.t;
    s.p = a.p_row ? (double)a.p_row[row] : a.p;
    s.m = a.m_row ? (double)a.m_row[row] : a.m;
    s.k = a.k_row ? a.k_row[row] : a.k;
    const double u = a.u_f64 ? static_cast<const double*>(a.u)[row]
                             : (double)static_cast<const float*>(a.u)[row];
    s.u = u > 0.0 ? fmin(u, 1.0) : 0.0;                  // (NaN: 0)
    s.first = !(s.t > 0.0) || s.k == 1 || s.p <= 0.0 || s.m > 1.0;
    // (of any fp32 logits, x / t and its multiples stay finite; beyond these bounds
    // all others weigh nothing, or all the same)
    s.t = fmin(fmax(s.t, 0x1p-300), 0x1p300);
    return s;
}

// Order-preserving bits of a logit: they ascend as logits descend.  -0 counts
// as 0, NaN as -infinity.
__device__ __forceinline__ uint32_t order_bits(float x) {
    x = x == 0.f ? 0.f : x;
    x = x != x ? -INFINITY : x;
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t bits = (uint32_t)(key >> 32);
    return __uint_as_float(bits & 0x80000000u ? bits : ~bits & 0x7fffffffu);
}

// Buckets and weights of a row or slice whose largest logit is `top`.
struct Scale {
    float top;
    double inv_t, edge;      // 1 / temperature; the largest logit's bucket

    __device__ __forceinline__ void set(float largest, double t) {
        top = largest;
        inv_t = 1.0 / t;
        edge = floor((double)top * inv_t * kPerUnit);
    }
    // Buckets below the largest's (kBuckets: no mass), and rel.
    __device__ __forceinline__ int bucket(float x, uint64_t& rel) const {
        rel = 1ull << kRelBits;
        if (x == top && isinf(x)) return 0;
        const double z = (double)x * inv_t, e = floor(z * kPerUnit), below = edge - e;
        if (!(below < (double)kBuckets)) return kBuckets;      // (NaN too)
        // e^r, r in [0, 1/16]: the series' remainder is r^7 / 7! < 2^-40
        const double r = __builtin_fma(e, -1.0 / kPerUnit, z);
        double w = 1.0 / 720.0;
        w = __builtin_fma(w, r, 1.0 / 120.0);
        w = __builtin_fma(w, r, 1.0 / 24.0);
        w = __builtin_fma(w, r, 1.0 / 6.0);
        w = __builtin_fma(w, r, 0.5);
        w = __builtin_fma(w, r, 1.0);
        w = __builtin_fma(w, r, 1.0);
        // (rounded to an integer in the low bits by the 2^52 added)
        w = __builtin_fma(w, (double)(1ull << kRelBits), 0x1p52);
        rel = __double_as_longlong(w) & ((1ull << 52) - 1);
        return (int)below;
    }
};

__device__ __forceinline__ int bucket_gap(double row_edge, double slice_edge) {
    if (row_edge == slice_edge) return 0;                // (infinities too)
    const double d = row_edge - slice_edge;
    return d < (double)kBuckets ? (int)d : kBuckets;
}

// A row as 16-byte vectors between its first and last 16-byte borders, and the
// tokens before and behind them.
template <int DT>
struct RowView {
    static constexpr int kVec = 16 / src_size(DT);
    const char* base;
    const uint4* vecs;
    int head, n_vecs, tail;              // tail: the first token behind
    __device__ __forceinline__ RowView(const SampleArgs& a, int row) {
        base = static_cast<const char*>(a.logits) + row * a.stride * src_size(DT);
        head = min(a.V, (int)((16 - ((uintptr_t)base & 15)) & 15) / src_size(DT));
        n_vecs = (a.V - head) / kVec;
        tail = head + n_vecs * kVec;
        vecs = reinterpret_cast<const uint4*>(base + head * src_size(DT));
    }
    // f(logit, index) for the tokens of vector i, loaded as w
    template <class F>
    __device__ __forceinline__ void tokens(uint4 w, int i, F f) const {
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
    // The same without unrolling, for bodies of some size: code that runs once is
    // bound by its own fetch.
    template <class F>
    __device__ __forceinline__ void tokens_rolled(uint4 w, int i, F f) const {
        int at = head + i * kVec;
#pragma unroll 1
        for (int j = 0; j < kVec; ++j, ++at) {
            float x;
            if constexpr (DT == kSrcF32) {
                x = __uint_as_float(w.x);
            } else {
                x = DT == kSrcBF16 ? __uint_as_float(w.x << 16)
                                   : (float)__builtin_bit_cast(_Float16, (uint16_t)(w.x & 0xffffu));
                w.x >>= 16;
            }
            if (DT == kSrcF32 || j % 2 == 1) {
                w.x = w.y;
                w.y = w.z;
                w.z = w.w;
            }
            f(x, at);
        }
    }
    // the token before or behind the vectors that a thread takes (-1: none):
    // the first slice takes those before, the last slice those behind
    __device__ __forceinline__ int single(int tid, int slice, int slices, int V) const {
        if (slice == 0 && tid < head) return tid;
        if (slice == slices - 1 && tid >= 8 && tid - 8 < V - tail) return tail + tid - 8;
        return -1;
    }
};

// A slice's tokens in registers.
template <int DT>
struct Slice {
    using R = RowView<DT>;
    static constexpr int kLoads = kSlice / R::kVec / kBlock;
    R row;
    uint4 w[kLoads];
    int first, single;
    float lone;
    // a thread's first vector, the others kBlock further each
    static __device__ __forceinline__ int vec_of(int slice, int thread) {
        return slice * (kSlice / R::kVec) + thread;
    }
    __device__ __forceinline__ Slice(const SampleArgs& a, int r, int slice) : row(a, r) {
        first = vec_of(slice, threadIdx.x);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int v = first + i * kBlock;
            if (v < row.n_vecs) w[i] = row.vecs[v];
        }
        single = row.single(threadIdx.x, slice, a.slices, a.V);
        lone = single >= 0 ? widen<DT>(row.base, single) : 0.f;
    }
    // f(logit, index, slot) for the thread's tokens: slots 0 .. kLone
    static constexpr int kLone = kLoads * R::kVec;
    template <class F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int v = first + i * kBlock;
            if (v >= row.n_vecs) continue;
            int slot = i * R::kVec;
            row.tokens(w[i], v, [&](float x, int at) { f(x, at, slot++); });
        }
        if (single >= 0) f(lone, single, kLone);
    }
    // A token's number within the slice, and the token of a number.
    static __device__ __forceinline__ int number(int slot) {
        return slot == kLone ? kSlice + (int)threadIdx.x
                             : (slot / R::kVec * kBlock + (int)threadIdx.x) * R::kVec +
                                   slot % R::kVec;
    }
    static __device__ __forceinline__ int token(const R& row, int slice, int number) {
        if (number < kSlice) return row.head + slice * kSlice + number;
        number -= kSlice;
        return number < 8 ? number : row.tail + number - 8;
    }
};

template <int DT>
__global__ void __launch_bounds__(kBlock) sample_sums_kernel(SampleArgs a) {
    __shared__ uint64_t hist[kBuckets];
    __shared__ uint32_t starts[kBuckets];
    __shared__ __align__(16) uint16_t order[kOrder];
    __shared__ float wave_top[kBlock / kWave];
    __shared__ uint32_t wave_count[kBlock / kWave], first;
    const int row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
    const int tid = threadIdx.x;
    using S = Slice<DT>;
    const S tokens(a, row, slice);
    const Settings s = settings_of(a, row);
    hist[tid] = 0;
    static_assert(kBuckets == kBlock, "a thread for each bucket");
    if (tid == 0) first = ~0u;
    float top = -INFINITY;
    tokens.each([&](float x, int, int) { top = fmaxf(top, x); });       // (NaN never)
    top = wave_max(top);
    if (tid % kWave == 0) wave_top[tid / kWave] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBlock / kWave; ++i) top = fmaxf(top, wave_top[i]);
    const int64_t at = (int64_t)row * a.slices + slice;
    uint32_t index = ~0u;
    if (s.first) {
        tokens.each([&](float x, int i, int) {
            index = x == top ? min(index, (uint32_t)i) : index;
        });
        if (index != ~0u) atomicMin(&first, index);
        __syncthreads();
        if (tid == 0) a.best[at] = (uint64_t)order_bits(top) << 32 | first;
        return;
    }
    Scale scale;
    scale.set(top, s.t);
    uint32_t place[S::kLone + 1];          // bucket << 16 | number in the bucket
#pragma unroll
    for (int i = 0; i <= S::kLone; ++i) place[i] = ~0u;
    if (top > -INFINITY) {
        tokens.each([&](float x, int i, int slot) {
            index = x == top ? min(index, (uint32_t)i) : index;
            uint64_t rel;
            const int b = scale.bucket(x, rel);
            if (b >= kBuckets) return;
            const uint64_t old = atomicAdd((unsigned long long*)&hist[b],
                                           (unsigned long long)(rel | 1ull << kCountShift));
            place[slot] = (uint32_t)b << 16 | (uint32_t)(old >> kCountShift);
        });
    }
    if (index != ~0u) atomicMin(&first, index);
    __syncthreads();
    if (tid == 0) a.best[at] = (uint64_t)order_bits(top) << 32 | first;
    const uint64_t sum = hist[tid];
    a.hist[at * kBuckets + tid] = sum;
    // where each bucket's tokens start
    const int lane = tid % kWave;
    const uint32_t count = (uint32_t)(sum >> kCountShift);
    uint32_t end = count;
    for (int d = 1; d < kWave; d *= 2) {
        const uint32_t o = __shfl_up(end, d);
        if (lane >= d) end += o;
    }
    if (lane == kWave - 1) wave_count[tid / kWave] = end;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < kBlock / kWave; ++i) {
        if (i < tid / kWave) end += wave_count[i];
        all += wave_count[i];
    }
    starts[tid] = end - count;
    a.starts[at * kStarts + tid] = (uint16_t)(end - count);
    if (tid == 0) a.starts[at * kStarts + kBuckets] = (uint16_t)all;
    __syncthreads();
#pragma unroll
    for (int i = 0; i <= S::kLone; ++i)
        if (place[i] != ~0u)
            order[starts[place[i] >> 16] + (place[i] & 0xffffu)] = (uint16_t)S::number(i);
    __syncthreads();
    uint4* to = reinterpret_cast<uint4*>(a.order + at * kOrder);
    for (uint32_t i = tid; i < (all + 7) / 8; i += kBlock)
        to[i] = reinterpret_cast<const uint4*>(order)[i];
}

// The first token of a row from its slices' (every lane).
__device__ __forceinline__ uint64_t first_of(const SampleArgs& a, int row) {
    uint64_t best = ~0ull;
    for (int i = threadIdx.x % kWave; i < a.slices; i += kWave)
        best = min(best, a.best[(int64_t)row * a.slices + i]);
    for (int d = 1; d < kWave; d *= 2)
        best = min(best, (uint64_t)__shfl_xor((unsigned long long)best, d));
    return best;
}

// A row's running sums before each bucket (entry kBuckets: the totals).
struct Sums {
    uint64_t mass[kBuckets + 1];
    uint32_t count[kBuckets + 1];
    uint64_t rel[kBuckets];              // the buckets' sums of rels
};

// Inclusive running sums over the wave's lanes.
__device__ __forceinline__ void wave_scan(uint64_t& m, uint32_t& c) {
    const int lane = threadIdx.x % kWave;
    for (int d = 1; d < kWave; d *= 2) {
        const uint64_t om = __shfl_up((unsigned long long)m, d);
        const uint32_t oc = __shfl_up(c, d);
        if (lane >= d) {
            m += om;
            c += oc;
        }
    }
}

// The border kinds, and whether entry i of running sums crosses one (exactly one
// does, for a border within the total).
enum Border : int {
    kByCount,       // the token that is number `at`
    kByMass,        // the first whose running sum reaches `at`
    kPast,          // the first whose running sum exceeds `at`
};
template <class T>
__device__ __forceinline__ bool crosses(const T* sums, int i, Border kind, uint64_t at) {
    const uint64_t from = sums[i], to = sums[i + 1];
    return kind == kPast ? from <= at && at < to : from < at && at <= to;
}

__device__ __forceinline__ uint64_t mass_wanted(double p, uint64_t kept) {
    const uint64_t want = (uint64_t)ceil(p * (double)kept);
    return want < 1 ? 1 : want > kept ? kept : want;
}
__device__ __forceinline__ uint64_t mass_passed(double u, uint64_t kept) {
    const uint64_t past = (uint64_t)(u * (double)kept);
    return past >= kept ? kept - 1 : past;
}

// min_p: w >= m where x / t reaches this.
__device__ __forceinline__ double min_p_border(const Scale& s, double m) {
    return (double)s.top * s.inv_t + log(m);
}
// its bucket (kBuckets: it cuts nothing that has mass)
__device__ __forceinline__ int min_p_bucket(const Scale& s, double border) {
    if (isinf(s.top)) return 0;
    const double below = s.edge - floor(border * kPerUnit);
    return below < (double)kBuckets ? (int)below : kBuckets;
}

// Ranges of buckets that may hold a border (lo > hi: none).
struct Wanted {
    int lo[4], hi[4];
};

// Where the borders can lie: each is known up to its bucket, so the kept mass
// lies between two of the running sums.  By all threads of a workgroup.
__device__ void wanted_buckets(const Settings& s, const Scale& scale, const Sums& sums,
                               Wanted& w) {
    const int b = threadIdx.x;
    if (b < 4) {
        w.lo[b] = 1;
        w.hi[b] = 0;
    }
    __syncthreads();
    uint64_t low = sums.mass[kBuckets], high = low;
    if (s.k > 0 && (uint32_t)s.k < sums.count[kBuckets]) {
        if (b < kBuckets && crosses(sums.count, b, kByCount, (uint64_t)s.k))
            w.lo[0] = w.hi[0] = b;
        __syncthreads();
        low = max(sums.mass[w.lo[0]], (uint64_t)1);
        high = max(sums.mass[w.hi[0] + 1], (uint64_t)1);
    }
    if (s.p < 1.0) {
        if (b < kBuckets) {
            if (crosses(sums.mass, b, kByMass, mass_wanted(s.p, low))) w.lo[1] = b;
            if (crosses(sums.mass, b, kByMass, mass_wanted(s.p, high))) w.hi[1] = b;
        }
        __syncthreads();
        low = max(sums.mass[w.lo[1]], (uint64_t)1);
        high = min(high, sums.mass[w.hi[1] + 1]);
    }
    if (s.m > 0.0) {
        const int at = min_p_bucket(scale, min_p_border(scale, s.m));
        if (at < kBuckets) {
            if (b == 0) w.lo[2] = w.hi[2] = at;
            low = min(low, max(sums.mass[at], (uint64_t)1));
            high = min(high, max(sums.mass[at + 1], (uint64_t)1));
        }
    }
    if (b < kBuckets) {
        if (crosses(sums.mass, b, kPast, mass_passed(s.u, low))) w.lo[3] = b;
        if (crosses(sums.mass, b, kPast, mass_passed(s.u, high))) w.hi[3] = b;
    }
    __syncthreads();
}

template <int DT>
struct Picker {
    struct Shared {
        Sums sums;
        uint64_t key[kList];             // the wanted buckets' tokens
        uint64_t rel[kList];             // bucket << 40 | rel
        union {
            struct {
                uint64_t key[kFew], rel[kFew], before[kPickBlock / kFew][kFew];
                uint32_t count[kPickBlock / kFew][kFew];
            } few;
            struct {
                uint64_t rel[kSub + 1], part_rel[kCopies][kSub];
                uint32_t count[kSub + 1], part_count[kCopies][kSub];
            } sub;
        };
        Wanted wanted;
        uint64_t wave_rel[kPickBlock / kWave];
        uint32_t wave_count[kPickBlock / kWave];
        int gap[kMaxVocab / kSlice];
        uint64_t hit_rel;
        // a range of wanted buckets in a slice: its first token there, and in the list
        uint32_t from[4 * kMaxVocab / kSlice], to[4 * kMaxVocab / kSlice + 1];
        uint32_t bits_min, bits_max, n, hit;
        int entry;
    };
    const SampleArgs& a;
    Shared& s;
    int row;
    Scale scale;
    int listed;                          // tokens of the list, -1: too many

    // f(key, rel) for the tokens of bucket b
    template <class F>
    __device__ __forceinline__ void each(int b, F f) {
        if (listed >= 0) {
            for (int i = threadIdx.x; i < listed; i += kPickBlock) {
                const uint64_t rel = s.rel[i];
                if ((int)(rel >> 40) == b) f(s.key[i], rel & ((1ull << 40) - 1));
            }
            return;
        }
        const RowView<DT> r(a, row);
        auto token = [&](float x, int i) {
            uint64_t rel;
            if (scale.bucket(x, rel) == b) f((uint64_t)order_bits(x) << 32 | (uint32_t)i, rel);
        };
        const int single = r.single(threadIdx.x, 0, 1, a.V);
        if (single >= 0) token(widen<DT>(r.base, single), single);
#pragma unroll 1
        for (int i = threadIdx.x; i < r.n_vecs; i += kPickBlock) r.tokens_rolled(r.vecs[i], i, token);
    }

    // The row's sums from its slices', and the buckets that may hold a border;
    // their tokens to the list.
    __device__ void collect(const Settings& set) {
        const int tid = threadIdx.x, bucket = tid % kBuckets, lane = tid % kWave;
        static_assert(kPickBlock == 2 * kBuckets, "two threads for each bucket");
        // (buckets that each slice's lie below the row's)
        for (int i = tid; i < a.slices; i += kPickBlock) {
            Scale other;
            other.set(logit_of(a.best[(int64_t)row * a.slices + i]), set.t);
            s.gap[i] = other.top == -INFINITY ? kBuckets : bucket_gap(scale.edge, other.edge);
        }
        __syncthreads();
        uint64_t rel = 0;
        uint32_t count = 0;
        const uint64_t* hist = a.hist + (int64_t)row * a.slices * kBuckets;
#pragma unroll 4
        for (int i = tid / kBuckets; i < a.slices; i += 2) {
            const int b = bucket - s.gap[i];
            const uint64_t h = b >= 0 ? hist[i * kBuckets + b] : 0;
            rel += h & kRelMask;
            count += (uint32_t)(h >> kCountShift);
        }
        if (tid >= kBuckets) {
            s.sums.rel[bucket] = rel;
            s.sums.count[bucket] = count;
        }
        __syncthreads();
        uint64_t mass = 0;
        if (tid < kBuckets) {
            rel += s.sums.rel[tid];
            count += s.sums.count[tid];
            s.sums.rel[tid] = rel;
            const double unit = exp(-tid / kPerUnit) * (double)(1ull << (kMassBits - kRelBits));
            mass = (uint64_t)__builtin_rint((double)rel * unit);
            wave_scan(mass, count);
            if (lane == kWave - 1) {
                s.wave_rel[tid / kWave] = mass;
                s.wave_count[tid / kWave] = count;
            }
        }
        __syncthreads();
        if (tid < kBuckets) {
            for (int i = 0; i < tid / kWave; ++i) {
                mass += s.wave_rel[i];
                count += s.wave_count[i];
            }
            s.sums.mass[tid + 1] = mass;
            s.sums.count[tid + 1] = count;
            if (tid == 0) {
                s.sums.mass[0] = 0;
                s.sums.count[0] = 0;
            }
        }
        __syncthreads();
        wanted_buckets(set, scale, s.sums, s.wanted);
        // The ranges without what an earlier one has: each token once.
        int lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo[i] = s.wanted.lo[i];
            hi[i] = s.wanted.hi[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < i; ++j) {
                if (lo[i] > hi[i] || lo[j] > hi[j] || lo[i] > hi[j] + 1 || hi[i] < lo[j] - 1)
                    continue;
                // (they meet: one range, in the later's place)
                lo[i] = min(lo[i], lo[j]);
                hi[i] = max(hi[i], hi[j]);
                lo[j] = 1;
                hi[j] = 0;
            }
        }
        // Their stretches of each slice's order, one after the other in the list.
        const int stretches = 4 * a.slices;
        uint64_t unused = 0;
        uint32_t length = 0;
        static_assert(4 * kMaxVocab / kSlice <= kBuckets, "a thread for each stretch");
        if (tid < stretches) {
            const int i = tid / a.slices, slice = tid - i * a.slices;
            const int l = i == 0 ? lo[0] : i == 1 ? lo[1] : i == 2 ? lo[2] : lo[3];
            const int h = i == 0 ? hi[0] : i == 1 ? hi[1] : i == 2 ? hi[2] : hi[3];
            const int b0 = max(l - s.gap[slice], 0), b1 = min(h - s.gap[slice], kBuckets - 1);
            if (l <= h && b0 <= b1) {
                const uint16_t* starts = a.starts + ((int64_t)row * a.slices + slice) * kStarts;
                s.from[tid] = starts[b0];
                length = starts[b1 + 1] - starts[b0];
            }
        }
        uint32_t to = length;
        if (tid < kBuckets) {
            wave_scan(unused, to);
            if (lane == kWave - 1) s.wave_count[tid / kWave] = to;
        }
        __syncthreads();
        uint32_t all = 0;
        for (int i = 0; i < kBuckets / kWave; ++i) {
            if (i < tid / kWave) to += s.wave_count[i];
            all += s.wave_count[i];
        }
        if (tid < stretches) s.to[tid] = to - length;
        if (tid == 0) s.to[stretches] = all;
        __syncthreads();
        listed = all <= (uint32_t)kList ? (int)all : -1;
        const RowView<DT> r(a, row);
#pragma unroll 1
        for (int j = tid; j < listed; j += kPickBlock) {
            int at = 0;                              // the last stretch that starts by j
            for (int d = kBuckets; d > 0; d /= 2)
                if (at + d < stretches && s.to[at + d] <= (uint32_t)j) at += d;
            const int slice = at % a.slices;
            const uint16_t* order = a.order + ((int64_t)row * a.slices + slice) * kOrder;
            const int i = Slice<DT>::token(r, slice, order[s.from[at] + (j - s.to[at])]);
            const float x = widen<DT>(r.base, i);
            uint64_t rel;
            const int b = scale.bucket(x, rel);
            s.key[j] = (uint64_t)order_bits(x) << 32 | (uint32_t)i;
            s.rel[j] = (uint64_t)b << 40 | rel;
        }
        __syncthreads();
    }

    // The sub-buckets' running sums from their copies.
    __device__ void scan_sub() {
        static_assert(kSub <= kPickBlock, "a thread for each sub-bucket");
        const int tid = threadIdx.x, lane = tid % kWave;
        uint64_t rel = 0;
        uint32_t count = 0;
        if (tid < kSub) {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                rel += s.sub.part_rel[i][tid];
                count += s.sub.part_count[i][tid];
            }
            wave_scan(rel, count);
            if (lane == kWave - 1) {
                s.wave_rel[tid / kWave] = rel;
                s.wave_count[tid / kWave] = count;
            }
        }
        __syncthreads();
        if (tid < kSub) {
            for (int i = 0; i < tid / kWave; ++i) {
                rel += s.wave_rel[i];
                count += s.wave_count[i];
            }
            s.sub.rel[tid + 1] = rel;
            s.sub.count[tid + 1] = count;
            if (tid == 0) {
                s.sub.rel[0] = 0;
                s.sub.count[0] = 0;
            }
        }
        __syncthreads();
    }

    // A border within bucket b: a number of tokens, or a sum of rels.
    struct Need {
        uint64_t base, mass, rels, at;
        double per;
    };
    __device__ __forceinline__ Need need_of(Border kind, uint64_t at, int b) const {
        Need x;
        x.base = s.sums.mass[b];
        x.mass = s.sums.mass[b + 1] - x.base;
        x.rels = s.sums.rel[b];
        x.per = (double)x.rels / (double)x.mass;
        if (kind == kByCount) {
            x.at = at - s.sums.count[b];
        } else if (kind == kByMass) {
            const uint64_t need = (uint64_t)ceil((double)(at - x.base) * x.per);
            x.at = need < 1 ? 1 : need > x.rels ? x.rels : need;
        } else {
            const uint64_t need = (uint64_t)((double)(at - x.base) * x.per);
            x.at = need >= x.rels ? x.rels - 1 : need;
        }
        return x;
    }
    // Whether a token with `r` rels and `c` tokens before it is the border's.
    static __device__ __forceinline__ bool hits(Border kind, uint64_t at, uint64_t r, uint32_t c,
                                                uint64_t rel) {
        return kind == kByCount  ? c + 1 == at
               : kind == kByMass ? r < at && at <= r + rel
                                 : r <= at && at < r + rel;
    }
    // The running mass at `rel` rels of the bucket (one whose mass is rounded to 0 adds
    // none: the row's total is never passed).
    static __device__ __forceinline__ uint64_t mass_at(const Need& x, uint64_t rel) {
        const uint64_t part = (uint64_t)__builtin_rint((double)rel / x.per);
        return x.base + min(max(part, (uint64_t)1), x.mass);
    }

    // One wave, a token of the list for each lane: its rank in its bucket.
    uint64_t my_key, my_rel, my_before;
    uint32_t my_count;
    int my_bucket;
    __device__ void gather_wave() {
        const int lane = threadIdx.x;
        my_key = my_rel = my_before = 0;
        my_count = 0;
        my_bucket = -1;
        if (lane < listed) {
            my_key = s.key[lane];
            my_rel = s.rel[lane] & ((1ull << 40) - 1);
            my_bucket = (int)(s.rel[lane] >> 40);
        }
#pragma unroll 1
        for (int j = 0; j < listed; ++j) {
            const uint64_t rel = s.rel[j];
            const bool ahead = (int)(rel >> 40) == my_bucket && s.key[j] < my_key;
            my_before += ahead ? rel & ((1ull << 40) - 1) : 0;
            my_count += ahead;
        }
    }
    __device__ uint64_t find_wave(Border kind, uint64_t at, uint32_t& index) {
        int b = 0;
#pragma unroll 1
        for (int i = threadIdx.x; i < kBuckets; i += kWave) {
            const uint64_t lanes = __builtin_amdgcn_ballot_w64(
                kind == kByCount ? crosses(s.sums.count, i, kind, at)
                                 : crosses(s.sums.mass, i, kind, at));
            if (lanes == 0) continue;
            b = __builtin_amdgcn_readfirstlane(i) + __ffsll((unsigned long long)lanes) - 1;
            break;
        }
        const Need x = need_of(kind, at, b);
        const uint64_t lanes = __builtin_amdgcn_ballot_w64(
            my_bucket == b && hits(kind, x.at, my_before, my_count, my_rel));
        const int lane = __ffsll((unsigned long long)lanes) - 1;
        index = __shfl((uint32_t)my_key, lane);
        return mass_at(x, __shfl((unsigned long long)(my_before + my_rel), lane));
    }
    __device__ uint64_t min_p_mass_wave(double m) {
        const double border = min_p_border(scale, m);
        const int b = min_p_bucket(scale, border);
        if (b >= kBuckets) return s.sums.mass[kBuckets];
        const float t = logit_of(my_key);
        const bool in = my_bucket == b && (t == scale.top || (double)t * scale.inv_t >= border);
        uint64_t sum = in ? my_rel : 0;
        for (int d = 1; d < kWave; d *= 2) sum += __shfl_xor((unsigned long long)sum, d);
        return sum == 0 ? s.sums.mass[b] : mass_at(need_of(kByCount, 0, b), sum);
    }

    // The running mass up to and with the token at the border, and its index.
    // `at` lies in the row's total.
    __device__ uint64_t find(Border kind, uint64_t at, uint32_t& index) {
        const int tid = threadIdx.x;
        if (tid < kBuckets && (kind == kByCount ? crosses(s.sums.count, tid, kind, at)
                                                : crosses(s.sums.mass, tid, kind, at)))
            s.entry = tid;
        __syncthreads();
        const int b = s.entry;
        const Need x = need_of(kind, at, b);
        uint64_t lo = 0, hi = ~0ull, before_rel = 0;
        uint32_t before_count = 0, n = s.sums.count[b + 1] - s.sums.count[b];
        // (a round leaves a 512th of a range of 2^64 at most: 7 rounds and a bit)
        for (int round = 0; n > kFew && round < 8; ++round) {
            // counts and sums of 512 stretches of the keys between lo and hi, from
            // the least to the most logit (or index, where all are equal)
            __syncthreads();
            if (tid == 0) {
                s.bits_min = ~0u;
                s.bits_max = 0;
            }
            for (int i = tid; i < kCopies * kSub; i += kPickBlock) {
                (&s.sub.part_rel[0][0])[i] = 0;
                (&s.sub.part_count[0][0])[i] = 0;
            }
            __syncthreads();
            uint32_t mn = ~0u, mx = 0;
            each(b, [&](uint64_t key, uint64_t) {
                if (key < lo || key > hi) return;
                mn = min(mn, (uint32_t)(key >> 32));
                mx = max(mx, (uint32_t)(key >> 32));
            });
            for (int d = 1; d < kWave; d *= 2) {
                mn = min(mn, (uint32_t)__shfl_xor(mn, d));
                mx = max(mx, (uint32_t)__shfl_xor(mx, d));
            }
            if (tid % kWave == 0) {
                atomicMin(&s.bits_min, mn);
                atomicMax(&s.bits_max, mx);
            }
            __syncthreads();
            const uint64_t first = max((uint64_t)s.bits_min << 32, lo);
            const uint64_t span = min(((uint64_t)s.bits_max << 32) + a.V - 1, hi) - first;
            int shift = 0;
            while (span >> shift >= kSub) ++shift;
            each(b, [&](uint64_t key, uint64_t rel) {
                if (key < lo || key > hi) return;
                const int i = (int)((key - first) >> shift);
                const int copy = tid % kCopies;
                atomicAdd((unsigned long long*)&s.sub.part_rel[copy][i], (unsigned long long)rel);
                atomicAdd(&s.sub.part_count[copy][i], 1u);
            });
            __syncthreads();
            scan_sub();
            const uint64_t rest = x.at - (kind == kByCount ? before_count : before_rel);
            for (int j = tid; j < kSub; j += kPickBlock)
                if (kind == kByCount ? crosses(s.sub.count, j, kind, rest)
                                     : crosses(s.sub.rel, j, kind, rest))
                    s.entry = j;
            __syncthreads();
            const int i = s.entry;
            before_rel += s.sub.rel[i];
            before_count += s.sub.count[i];
            n = s.sub.count[i + 1] - s.sub.count[i];
            lo = first + ((uint64_t)i << shift);
            hi = lo + ((1ull << shift) - 1);
        }
        __syncthreads();
        if (tid == 0) s.n = 0;
        __syncthreads();
        each(b, [&](uint64_t key, uint64_t rel) {
            if (key < lo || key > hi) return;
            const uint32_t i = atomicAdd(&s.n, 1u);
            if (i >= (uint32_t)kFew) return;
            s.few.key[i] = key;
            s.few.rel[i] = rel;
        });
        __syncthreads();
        // each against the others, an eighth of them a thread
        constexpr int kParts = kPickBlock / kFew;
        const int mine = tid % kFew, part = tid / kFew;
        const uint64_t key = mine < (int)n ? s.few.key[mine] : 0;
        uint64_t r = 0;
        uint32_t c = 0;
        for (int j = part; j < (int)n; j += kParts) {
            const bool ahead = s.few.key[j] < key;
            r += ahead ? s.few.rel[j] : 0;
            c += ahead;
        }
        s.few.before[part][mine] = r;
        s.few.count[part][mine] = c;
        __syncthreads();
        if (tid < (int)n) {
            const uint64_t rel = s.few.rel[tid];
            r = before_rel;
            c = before_count;
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                r += s.few.before[i][tid];
                c += s.few.count[i][tid];
            }
            if (hits(kind, x.at, r, c, rel)) {
                s.hit = (uint32_t)key;
                s.hit_rel = r + rel;
            }
        }
        __syncthreads();
        index = s.hit;
        return mass_at(x, s.hit_rel);
    }

    // The running mass of the tokens with w >= m.
    __device__ uint64_t min_p_mass(double m) {
        const double border = min_p_border(scale, m);
        const int b = min_p_bucket(scale, border);
        if (b >= kBuckets) return s.sums.mass[kBuckets];
        __syncthreads();
        if (threadIdx.x == 0) s.hit_rel = 0;
        __syncthreads();
        uint64_t sum = 0;
        each(b, [&](uint64_t key, uint64_t rel) {
            const float x = logit_of(key);
            if (x == scale.top || (double)x * scale.inv_t >= border) sum += rel;
        });
        if (sum) atomicAdd((unsigned long long*)&s.hit_rel, (unsigned long long)sum);
        __syncthreads();
        return s.hit_rel == 0 ? s.sums.mass[b] : mass_at(need_of(kByCount, 0, b), s.hit_rel);
    }
};

template <int DT>
__global__ void __launch_bounds__(kPickBlock) sample_pick_kernel(SampleArgs a) {
    using P = Picker<DT>;
    __shared__ typename P::Shared s;
    const int row = blockIdx.x, tid = threadIdx.x;
    const Settings set = settings_of(a, row);
    const uint64_t best = first_of(a, row);
    P p{a, s, row, {}, 0, 0, 0, 0, 0, 0};
    p.scale.set(logit_of(best), set.t);
    const bool none = p.scale.top == -INFINITY;
    if (none || set.first) {
        if (tid == 0) a.out[row] = none ? -1 : (int64_t)(uint32_t)best;
        return;
    }
    p.collect(set);
    uint64_t kept = s.sums.mass[kBuckets];
    uint32_t index = 0;
    // (few tokens: one wave, without barriers)
    const bool alone = p.listed >= 0 && p.listed <= kWave;
    if (alone) {
        if (tid >= kWave) return;
        p.gather_wave();
    }
    // (one loop for the three borders: one copy of the search's code)
#pragma unroll 1
    for (int step = 0; step < 3; ++step) {
        Border kind;
        uint64_t at;
        if (step == 0) {
            if (set.k <= 0 || (uint32_t)set.k >= s.sums.count[kBuckets]) continue;
            kind = kByCount;
            at = (uint64_t)set.k;
        } else if (step == 1) {
            if (!(set.p < 1.0)) continue;
            kind = kByMass;
            at = mass_wanted(set.p, kept);
        } else {
            if (set.m > 0.0)
                kept = max(min(kept, alone ? p.min_p_mass_wave(set.m) : p.min_p_mass(set.m)),
                           (uint64_t)1);
            kind = kPast;
            at = mass_passed(set.u, kept);
        }
        kept = alone ? p.find_wave(kind, at, index) : p.find(kind, at, index);
    }
    if (tid == 0) a.out[row] = (int64_t)index;
}

int64_t slices_of(int32_t vocab) { return ((int64_t)vocab + kSlice - 1) / kSlice; }

template <int DT>
void launch(const SampleArgs& a, int rows, hipStream_t s) {
    sample_sums_kernel<DT><<<(unsigned)(rows * a.slices), kBlock, 0, s>>>(a);
    sample_pick_kernel<DT><<<rows, kPickBlock, 0, s>>>(a);
}

}  // namespace
}  // namespace kivi

using namespace kivi;

extern "C" {

size_t kivi_sample_workspace_size(int32_t rows, int32_t vocab) {
    if (rows < 1 || vocab < 1 || vocab > kMaxVocab) return 0;
    return (size_t)(rows * slices_of(vocab)) *
           (8 * kBuckets + 2 * kOrder + 2 * kStarts + 8);
}

int kivi_sample(const void* logits, int32_t dtype, int64_t row_stride, int32_t rows,
                int32_t vocab, const void* uniforms, int32_t uniforms_f64,
                const float* temperatures, double temperature, const int32_t* top_ks,
                int32_t top_k, const float* top_ps, double top_p, const float* min_ps,
                double min_p, int64_t* out, void* workspace, size_t workspace_bytes,
                void* stream) {
    if (dtype < 0 || dtype > 2)
        return set_error(kErrInvalidArgument, "dtype %d is not 0 (f32), 1 (bf16) or 2 (f16)", dtype);
    if (rows < 0 || vocab < 1 || vocab > kMaxVocab)
        return set_error(kErrInvalidArgument, "logits of %d rows and %d tokens (1 to %d)", rows,
                         vocab, kMaxVocab);
    if (row_stride < 0)
        return set_error(kErrInvalidArgument, "row_stride %lld must not be negative",
                         (long long)row_stride);
    if (rows == 0) return kOk;
    if (logits == nullptr || uniforms == nullptr || out == nullptr)
        return set_error(kErrInvalidArgument, "null pointer");
    const int64_t slices = slices_of(vocab);
    // (a launch has fewer than 2^32 lanes)
    if (rows * slices > (int64_t)UINT32_MAX / kBlock || rows > (int64_t)UINT32_MAX / kPickBlock)
        return set_error(kErrInvalidArgument, "%d rows of %d tokens are too many for one launch",
                         rows, vocab);
    const size_t need = kivi_sample_workspace_size(rows, vocab);
    if (workspace == nullptr || ((uintptr_t)workspace & 15) || workspace_bytes < need)
        return set_error(kErrInvalidArgument, "workspace must be 16-byte aligned and hold %zu "
                         "bytes, got %zu", need, workspace_bytes);
    SampleArgs a{};
    a.logits = logits;
    a.stride = row_stride;
    a.V = vocab;
    a.slices = (int)slices;
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
    uint64_t* w = static_cast<uint64_t*>(workspace);
    const int64_t n = rows * slices;
    a.hist = w;
    a.order = reinterpret_cast<uint16_t*>(a.hist + n * kBuckets);
    a.starts = a.order + n * kOrder;
    a.best = reinterpret_cast<uint64_t*>(a.starts + n * kStarts);
    static_assert(kOrder % 8 == 0 && kStarts % 8 == 0, "whole 16 bytes");
    hipStream_t s = (hipStream_t)stream;
    if (dtype == kSrcF32) launch<kSrcF32>(a, rows, s);
    else if (dtype == kSrcBF16) launch<kSrcBF16>(a, rows, s);
    else launch<kSrcF16>(a, rows, s);
    return check_launch("sample");
}

}  // extern "C"
