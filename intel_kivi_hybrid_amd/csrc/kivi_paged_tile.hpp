// Tiles of keys and values in LDS and the products of 32 query rows with them
// (16-bit types), where tiles go from memory straight into LDS.
//
// Such a load (64 lanes of 16 bytes) fills 1024 consecutive bytes, so token rows
// lie unpadded there, and the vectors of a token are permuted instead, by the
// address that each lane loads from.
#pragma once

#include "kivi_paged_attention.hpp"

namespace kivi {
namespace {

template <int DP, int TOKENS>
struct TileShape {
    static constexpr int TILE = TOKENS, TB = TILE / 32;
    static constexpr int KS = DP / 16;                 // k-steps of a score
    static constexpr int CB = DP / 32;                 // blocks of 32 output channels
    // slots of 16 bytes of a token's row in LDS (DP 96: the last four unused)
    static constexpr int SL = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;
    static constexpr int ROW = SL * 16;
    static constexpr int BYTES = TILE * ROW;           // of a tile's keys
    static constexpr int ROWS = kWave / SL;            // tokens of a load

    // Slot c ^ swizzle(t) holds vector c of token t.  The 16 tokens of a
    // half-wave's key reads then start on 16 different bank groups, and the 8
    // tokens of a transposed read (64 bytes each) meet each bank twice.
    static __device__ __forceinline__ int key_swizzle(int t) {
        return SL == 8 ? t / 2 % 8 : t % 16;
    }
    static __device__ __forceinline__ int value_swizzle(int t) {
        return SL == 8 ? t / 2 % 2 * 4 : t % 4 * 4;
    }
};

// 64 lanes' 16 bytes from memory to 1024 consecutive bytes of LDS; lanes behind the
// head's channels bring zeros, so no load stands behind a branch that depends on the
// lane and no LDS has to be cleared.
__device__ __forceinline__ void load_lds(const PagedLaunch& a, const void* from, bool inside,
                                         unsigned char* lds) {
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)(inside ? from : a.zeros),
        (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
// The wave's loads have arrived.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// Workgroup barrier behind which the tiles waited for are whole, and the buffers
// read before it free.  A fence would wait for the loads in flight too: they write
// LDS, which it orders.
__device__ __forceinline__ void tile_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Instruction kinds of __builtin_amdgcn_sched_group_barrier.
constexpr int kSchedValu = 0x2, kSchedMfma = 0x8, kSchedLdsRead = 0x100;

// A wave's 32 query rows (lane: row lane % 32) and their softmax state.
template <int DT, int DP, int TOKENS>
struct TileRows {
    using M = TileShape<DP, TOKENS>;
    u32x4_t qf[M::KS];
    f32x16_t O[M::CB];
    float m, l;
    int lim;                 // positions that the lane's row sees
    int all, last;           // that all, and any, of the 32 rows see

    // rows row0 .. row0 + 31 of the item's sequence
    __device__ __forceinline__ void init(const PagedLaunch& a, const Work& w, int row0) {
        const int lane = threadIdx.x % kWave, half = lane / 32, r = row0 + lane % 32;
        const bool live = r < w.rows;
        lim = live ? row_limit(w, r) : 0;
        m = -FLT_MAX;
        l = 0.f;
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + (live ? q_offset(a, w, r) : 0);
#pragma unroll
        for (int ks = 0; ks < M::KS; ++ks) {
            const int c = 16 * ks + 8 * half;
            qf[ks] = u32x4_t{0, 0, 0, 0};
            if (live && c < a.D) qf[ks] = *reinterpret_cast<const u32x4_t*>(q + c);
        }
#pragma unroll
        for (int cb = 0; cb < M::CB; ++cb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) O[cb][i] = 0.f;
        }
        const int base = w.it.ctx - w.it.n + 1;
        all = base + row0 / w.hg;
        last = row0 < w.rows ? min(base + min(row0 + 31, w.rows - 1) / w.hg, w.it.kv_end) : 0;
    }

    // A tile of keys (at kb of buf) and values (at vb) in LDS, positions t0 ..  (buf is
    // the array itself and each address one sum: through a longer chain the compiler
    // loses which array a read is of, and it then waits for the loads into the others)
    __device__ __forceinline__ void tile(const unsigned char* buf, uint32_t kb, uint32_t vb,
                                         int t0, int end, float qscale) {
        const int lane = threadIdx.x % kWave, col = lane % 32, half = lane / 32;
        f32x16_t s[M::TB];
#pragma unroll
        for (int tb = 0; tb < M::TB; ++tb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[tb][i] = 0.f;
        }
        const uint32_t krow = col * M::ROW + ((half ^ M::key_swizzle(col)) << 4);
#pragma unroll
        for (int ks = 0; ks < M::KS; ++ks) {
#pragma unroll
            for (int tb = 0; tb < M::TB; ++tb) {
                const u32x4_t kf = *reinterpret_cast<const u32x4_t*>(
                    buf + (kb + (krow ^ (32 * ks)) + 32 * tb * M::ROW));
                s[tb] = mfma32<DT>(kf, qf[ks], s[tb]);
            }
        }
        // (key vectors three k-steps ahead of their products: left to itself the
        // compiler waits for each pair)
        constexpr int kReads = M::KS * M::TB, kAhead = 3 * M::TB;
        __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, kAhead, 0);
#pragma unroll
        for (int i = 0; i < kReads - kAhead; ++i) {
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, kAhead, 0);
        // score i of block tb: token 32 tb + 8 (i / 4) + 4 half + i % 4
        if (t0 + M::TILE > min(all, end)) {
#pragma unroll
            for (int tb = 0; tb < M::TB; ++tb) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (t0 + 32 * tb + 8 * (i / 4) + 4 * half + i % 4 >= lim)
                        s[tb][i] = -INFINITY;
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int tb = 0; tb < M::TB; ++tb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[tb][i]);
        }
        mx = fmaf(mx, qscale, -weight_bits<DT>());
        if (__builtin_amdgcn_ballot_w64(mx > m + kMoveMax) != 0) {
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float to = fmaxf(m, mx), f = exp2_fast(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int cb = 0; cb < M::CB; ++cb) O[cb] *= f;
        }
        // transposed: lanes of 16 take tokens 4 half .. + 3 of 16 channels
        const int t = 4 * half + lane % 16 / 4;
        const int c = lane / 16 % 2 * 2 + lane % 4 / 2;
        const uint32_t vrow = t * M::ROW + ((c ^ M::value_swizzle(t)) << 4) + lane % 2 * 8;
        constexpr int kSteps = 2 * M::TB;          // of 16 tokens
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            u32x4_t pf;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = s[j / 2][j % 2 * 8 + 2 * i];
                const float y = s[j / 2][j % 2 * 8 + 2 * i + 1];
                const float p0 = exp2_fast(fmaf(x, qscale, -m)), p1 = exp2_fast(fmaf(y, qscale, -m));
                l += p0 + p1;
                pf[i] = pack2<DT>(p0, p1);
            }
#pragma unroll
            for (int cb = 0; cb < M::CB; ++cb) {
                const uint32_t at = vb + (vrow ^ (64 * cb)) + 16 * j * M::ROW;
                const uint2 lo = read_transposed(buf + at);
                const uint2 hi = read_transposed(buf + (at + 8 * M::ROW));
                O[cb] = mfma32<DT>(u32x4_t{lo.x, lo.y, hi.x, hi.y}, pf, O[cb]);
            }
        }
        // A step's products run beside the next one's weights; its values are read
        // a step ahead.
        __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 2 * M::CB, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedValu, 28, 0);
#pragma unroll
        for (int j = 0; j + 1 < kSteps; ++j) {
#pragma unroll
            for (int cb = 0; cb < M::CB; ++cb) {
                __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 2, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedValu, 28 / M::CB, 0);
            }
        }
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, M::CB, 0);
    }
};

// How a workgroup's lanes load a tile: load i of one of its WAVES waves covers
// ROWS tokens of one block of 16 positions, whose page is the same for the whole
// wave; a lane's place in the block is the same for every tile.  Pages of at
// least a tile's size hold the whole tile: one page and one address for it (four
// of each, with their 64-bit products, were 160 scalar instructions a tile).
template <int DP, int TOKENS, int WAVES>
struct TileLoads {
    using M = TileShape<DP, TOKENS>;
    static constexpr int LD = TOKENS / M::ROWS / WAVES;     // loads of a wave for a tile's keys
    int wave;
    int page[LD];                                           // (whole: the first alone)
    uint32_t k_off[LD], v_off[LD];                          // the lane's, in the tile's rows
    bool whole;                                             // pages hold tiles

    __device__ __forceinline__ void init(const PagedLaunch& a, int w) {
        wave = w;
        whole = 1 << a.page_shift >= TOKENS;
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int row = (whole ? block_of(i) : 0) + token(i);
            k_off[i] = row * a.D + channel(i, true);
            v_off[i] = row * a.D + channel(i, false);
        }
    }
    __device__ __forceinline__ int block_of(int i) const {
        return (i * WAVES + wave) * M::ROWS / 16 * 16;
    }
    // the token (of its block) and channel that the lane loads
    __device__ __forceinline__ int token(int i) const {
        return ((i * WAVES + wave) * M::ROWS + threadIdx.x % kWave / M::SL) % 16;
    }
    __device__ __forceinline__ int channel(int i, bool key) const {
        const int t = token(i), slot = threadIdx.x % kWave % M::SL;
        return (slot ^ (key ? M::key_swizzle(t) : M::value_swizzle(t))) * 8;
    }
    __device__ __forceinline__ void pages_of(const PagedLaunch& a, const Work& w, int t0) {
        // (a store of page[0] on either side of a branch is merged with another's, and
        // the array then lies in scratch memory)
        page[0] = block_page(a, w, t0 + (whole ? 0 : block_of(0)));
        if (whole) return;
#pragma unroll
        for (int i = 1; i < LD; ++i) page[i] = block_page(a, w, t0 + block_of(i));
    }
    // Loads the tile at t0 (whose pages are known), then its successor's pages.
    __device__ __forceinline__ void issue(const PagedLaunch& a, const Work& w, unsigned char* buf,
                                          int t0, int next) {
        unsigned char* to = buf + wave * 1024;
        const uint16_t *k[LD], *v[LD];
        k[0] = block_at<uint16_t>(a, w, a.k_pages, page[0], t0 + (whole ? 0 : block_of(0)));
        v[0] = block_at<uint16_t>(a, w, a.v_pages, page[0], t0 + (whole ? 0 : block_of(0)));
#pragma unroll
        for (int i = 1; i < LD; ++i) {
            k[i] = k[0];
            v[i] = v[0];
        }
        if (!whole) {
#pragma unroll
            for (int i = 1; i < LD; ++i) {
                k[i] = block_at<uint16_t>(a, w, a.k_pages, page[i], t0 + block_of(i));
                v[i] = block_at<uint16_t>(a, w, a.v_pages, page[i], t0 + block_of(i));
            }
        }
        pages_of(a, w, next);
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            load_lds(a, k[i] + k_off[i], channel(i, true) < a.D, to + i * WAVES * 1024);
            load_lds(a, v[i] + v_off[i], channel(i, false) < a.D, to + i * WAVES * 1024 + M::BYTES);
        }
    }
    // The lane's own part of a tile that has arrived and that some row does not see
    // to its end: zeros behind the end (weight 0 of whatever lies there) and for
    // non-finite values.  Whether there was one of the latter.
    template <int DT>
    __device__ __forceinline__ bool mend(unsigned char* buf, int t0, int end) const {
        bool any = false;
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            u32x4_t* v = reinterpret_cast<u32x4_t*>(
                buf + (M::BYTES + (i * WAVES + wave) * 1024 + threadIdx.x % kWave * 16));
            u32x4_t x = *v;
            if (t0 + block_of(i) + token(i) >= end) {
                x = u32x4_t{0, 0, 0, 0};
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t y = finite_part<DT>(x[j]);
                    any |= y != x[j];
                    x[j] = y;
                }
            }
            *v = x;
        }
        return any;
    }
};

}  // namespace
}  // namespace kivi
