// Attention over a paged cache for many query rows per kv head, 16-bit types
// (gfx950 matrix cores): chunks of prompts.
//
// A workgroup takes 128 rows of a kv head, 32 for each of its four waves
// (v_mfma_f32_32x32x16: a wave's operand tile is read from LDS once for all of
// them), and walks the positions in tiles of 64 (32 above 128 channels).  The
// next tile's keys and values go from memory straight to the other of two LDS
// buffers while this one is computed: one barrier per tile, no registers held
// for them.  Such a load fills consecutive LDS, so rows lie unpadded there and
// the vectors of a token are permuted instead, by the address that each lane
// loads from (Many::key_swizzle, value_swizzle).
#include <hip/hip_runtime.h>

#include "kivi_paged_attention.hpp"

namespace kivi {
namespace {

constexpr int kWaves = 4;
constexpr int kBlock = kWaves * kWave;

template <int DP>
struct Many {
    static constexpr int TILE = DP <= 128 ? 64 : 32;   // (what the registers hold)
    static constexpr int TB = TILE / 32;
    static constexpr int KS = DP / 16;                 // k-steps of a score
    static constexpr int CB = DP / 32;                 // blocks of 32 output channels
    // slots of 16 bytes of a token's row in LDS (DP 96: the last four unused)
    static constexpr int SL = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;
    static constexpr int ROW = SL * 16;
    static constexpr int BYTES = TILE * ROW;           // of a tile's keys
    static constexpr int ROWS = kWave / SL;            // tokens of a load
    static constexpr int LD = TILE / ROWS / kWaves;    // a wave's loads of a tile's keys

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

// 64 lanes' 16 bytes from memory to 1024 consecutive bytes of LDS.
__device__ __forceinline__ void load_lds(const uint16_t* base, uint32_t off, unsigned char* lds) {
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)(base + off),
        (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
// All of the wave's loads have arrived.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// A wave's 32 query rows (lane: row lane % 32) and their softmax state.
template <int DT, int DP>
struct ManyRows {
    using M = Many<DP>;
    u32x4_t qf[M::KS];
    f32x16_t O[M::CB];
    float m, l;
    int lim;                 // positions that the lane's row sees
    int all, last;           // that all, and any, of the wave's rows see

    // A tile of keys (kb) and values (vb) in LDS, positions t0 ..
    __device__ __forceinline__ void tile(const unsigned char* kb, const unsigned char* vb,
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
                    kb + (krow ^ (32 * ks)) + 32 * tb * M::ROW);
                s[tb] = mfma32<DT>(kf, qf[ks], s[tb]);
            }
        }
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
        mx *= qscale;
        if (__builtin_amdgcn_ballot_w64(mx > m + kMoveMax) != 0) {
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float to = fmaxf(m, mx), f = exp2_fast(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int cb = 0; cb < M::CB; ++cb) O[cb] *= f;
        }
        u32x4_t pf[2 * M::TB];        // weights of tokens 16 j .. + 15
#pragma unroll
        for (int tb = 0; tb < M::TB; ++tb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[tb][i] = exp2_fast(fmaf(s[tb][i], qscale, -m));
                l += s[tb][i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                pf[2 * tb + i / 4][i % 4] = pack2<DT>(s[tb][2 * i], s[tb][2 * i + 1]);
        }
        // transposed: lanes of 16 take tokens 4 half .. + 3 of 16 channels
        const int t = 4 * half + lane % 16 / 4;
        const int c = lane / 16 % 2 * 2 + lane % 4 / 2;
        const uint32_t vrow = t * M::ROW + ((c ^ M::value_swizzle(t)) << 4) + lane % 2 * 8;
#pragma unroll
        for (int j = 0; j < 2 * M::TB; ++j) {
#pragma unroll
            for (int cb = 0; cb < M::CB; ++cb) {
                const unsigned char* p = vb + (vrow ^ (64 * cb)) + 16 * j * M::ROW;
                const uint2 lo = read_transposed(p);
                const uint2 hi = read_transposed(p + 8 * M::ROW);
                O[cb] = mfma32<DT>(u32x4_t{lo.x, lo.y, hi.x, hi.y}, pf[j], O[cb]);
            }
        }
    }
};

template <int DT, int DP>
__global__ void __launch_bounds__(kBlock, DP <= 128 ? 2 : 1) paged_many_kernel(PagedLaunch a) {
    using M = Many<DP>;
    // (two arrays, not one: reads of this tile then need not wait for the next
    // one's loads, which the compiler knows to write the other array)
    __shared__ __align__(16) unsigned char buf0[2 * M::BYTES];
    __shared__ __align__(16) unsigned char buf1[2 * M::BYTES];
    __shared__ int odd;                    // some values were not finite
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, col = lane % 32, half = lane / 32;
    const Work w = work_of(a);
    const int end = w.it.kv_end;

    const int r = w.it.row0 + 32 * wave + col;
    const bool live = r < w.rows;
    ManyRows<DT, DP> rows;
    rows.lim = live ? row_limit(w, r) : 0;
    rows.m = -FLT_MAX;
    rows.l = 0.f;
    {
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + (live ? q_offset(a, w, r) : 0);
#pragma unroll
        for (int ks = 0; ks < M::KS; ++ks) {
            const int c = 16 * ks + 8 * half;
            rows.qf[ks] = u32x4_t{0, 0, 0, 0};
            if (live && c < a.D) rows.qf[ks] = *reinterpret_cast<const u32x4_t*>(q + c);
        }
    }
#pragma unroll
    for (int cb = 0; cb < M::CB; ++cb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) rows.O[cb][i] = 0.f;
    }
    const int base = w.it.ctx - w.it.n + 1, first = w.it.row0 + 32 * wave;
    const int wg_all = base + w.it.row0 / w.hg;
    rows.all = base + first / w.hg;
    rows.last = first < w.rows ? min(base + min(first + 31, w.rows - 1) / w.hg, end) : 0;

    // A load covers ROWS tokens of one block of 16 positions, whose page is the
    // same for the whole wave; a lane's place in it is the same for every tile.
    const bool full = a.D == M::SL * 8;
    auto vec_off = [&](int i, bool key) {
        const int t = ((i * kWaves + wave) * M::ROWS + lane / M::SL) % 16;
        const int c = lane % M::SL ^ (key ? M::key_swizzle(t) : M::value_swizzle(t));
        return make_int2(t, c * 8);
    };
    auto block_of = [&](int i) { return (i * kWaves + wave) * M::ROWS / 16 * 16; };
    int page[M::LD];
    auto pages_of = [&](int t0) {
#pragma unroll
        for (int i = 0; i < M::LD; ++i) page[i] = block_page(a, w, t0 + block_of(i));
    };
    auto issue = [&](unsigned char* buf, int t0) {
#pragma unroll
        for (int i = 0; i < M::LD; ++i) {
            const int t = t0 + block_of(i);
            const uint16_t* k = block_at<uint16_t>(a, w, a.k_pages, page[i], t);
            const uint16_t* v = block_at<uint16_t>(a, w, a.v_pages, page[i], t);
            unsigned char* to = buf + (i * kWaves + wave) * 1024;
            const int2 kc = vec_off(i, true), vc = vec_off(i, false);
            if (full) {
                load_lds(k, kc.x * a.D + kc.y, to);
                load_lds(v, vc.x * a.D + vc.y, to + M::BYTES);
            } else {
                if (kc.y < a.D) load_lds(k, kc.x * a.D + kc.y, to);
                if (vc.y < a.D) load_lds(v, vc.x * a.D + vc.y, to + M::BYTES);
            }
        }
        pages_of(t0 + M::TILE);
    };
    // Waits for the wave's part of the tile.  What lies behind the end has
    // weight 0: zeros there, as it may be anything.
    auto arrive = [&](unsigned char* buf, int t0) {
        wait_loads();
        if (t0 + M::TILE > min(wg_all, end)) {
            bool any = false;
#pragma unroll
            for (int i = 0; i < M::LD; ++i) {
                u32x4_t* v = reinterpret_cast<u32x4_t*>(buf + M::BYTES +
                                                        (i * kWaves + wave) * 1024 + lane * 16);
                u32x4_t x = *v;
                if (t0 + block_of(i) + vec_off(i, false).x >= end) {
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
            if (any) odd = 1;
        }
        lds_barrier();
    };
    int t0 = w.it.kv_begin;
    auto step = [&](unsigned char* now, unsigned char* next) {
        arrive(now, t0);
        if (t0 + M::TILE < end) issue(next, t0 + M::TILE);
        if (t0 < rows.last) rows.tile(now, now + M::BYTES, t0, end, a.qscale);
        t0 += M::TILE;
    };

    pages_of(t0);
    if (!full) {
        // (vectors behind the head's channels, which no load writes)
        for (int i = threadIdx.x; i < 2 * M::BYTES / 16; i += kBlock) {
            reinterpret_cast<u32x4_t*>(buf0)[i] = u32x4_t{0, 0, 0, 0};
            reinterpret_cast<u32x4_t*>(buf1)[i] = u32x4_t{0, 0, 0, 0};
        }
    }
    if (threadIdx.x == 0) odd = 0;
    lds_barrier();
    issue(buf0, t0);
    while (true) {
        step(buf0, buf1);
        if (t0 >= end) break;
        step(buf1, buf0);
        if (t0 >= end) break;
    }

    float l = rows.l;
    l += __shfl_xor(l, 32);
    if (!live) return;
    const bool whole = w.it.part < 0;
    const float inv = whole ? inverse_sum(l) : 1.0f;
    const int64_t at = whole ? out_offset(a, w, r) : part_row(a, w, r);
#pragma unroll
    for (int cb = 0; cb < M::CB; ++cb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = 32 * cb + 8 * i + 4 * half;
            if (c >= a.D) continue;
            const f32x16_t& O = rows.O[cb];
            f32x4_t o = {O[4 * i], O[4 * i + 1], O[4 * i + 2], O[4 * i + 3]};
            o *= inv;
            if (odd != 0) o += odd_values<DT>(a, w, odd_from(w, wg_all, M::TILE), rows.lim, c);
            if (whole) store4<DT>(a.out, at + c, o);
            else *reinterpret_cast<f32x4_t*>(a.part_o + at * a.D + c) = o;
        }
    }
    if (!whole && half == 0)
        *reinterpret_cast<float2*>(a.part_ml + 2 * at) = make_float2(rows.m, l);
}

template <int DT>
void launch_dim(const PagedLaunch& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_items * a.Hkv));
    if (a.D <= 64) paged_many_kernel<DT, 64><<<grid, kBlock, 0, s>>>(a);
    else if (a.D <= 96) paged_many_kernel<DT, 96><<<grid, kBlock, 0, s>>>(a);
    else if (a.D <= 128) paged_many_kernel<DT, 128><<<grid, kBlock, 0, s>>>(a);
    else paged_many_kernel<DT, 256><<<grid, kBlock, 0, s>>>(a);
}

}  // namespace

void launch_paged_many(const PagedLaunch& a, int dtype, hipStream_t s) {
    if (dtype == kSrcBF16) launch_dim<kSrcBF16>(a, s);
    else launch_dim<kSrcF16>(a, s);
}

}  // namespace kivi
