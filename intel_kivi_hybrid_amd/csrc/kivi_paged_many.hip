// Attention over a paged cache for many query rows per kv head, 16-bit types
// (gfx950 matrix cores): chunks of prompts.
//
// A workgroup takes 128 rows of a kv head, 32 for each of its four waves
// (v_mfma_f32_32x32x16: a wave's operand tile is read from LDS once for all of
// them), and walks the positions in tiles of 64 (32 above 128 channels).  Keys and values of the next
// tile are in flight to registers while the current one is computed, and go to
// the other of two LDS buffers after it: one barrier per tile.  Token rows in
// LDS are padded so that keys (8 channels of 32 tokens) and the transposed reads
// of values (4 tokens of 16 channels) meet every bank equally often.
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
    static constexpr int CH = DP / 8;                  // 16-byte vectors of a token
    static constexpr int LD = TILE * CH / kBlock;     // loads of a lane per tile
    static constexpr int KST = DP * 2 + 16, VST = DP * 2 + 64;
    static constexpr int K_BYTES = TILE * KST, V_BYTES = TILE * VST;
    static constexpr int BUF = K_BYTES + V_BYTES;
};

template <int DT, int DP>
__global__ void __launch_bounds__(kBlock) paged_many_kernel(PagedLaunch a) {
    using M = Many<DP>;
    constexpr int kTile = M::TILE;
    __shared__ __align__(16) unsigned char lds[2 * M::BUF];
    // Whether tile k's values are not all finite, at k % 3: set while tile k - 1
    // is computed, read with tile k, cleared with tile k + 1 (three, so that a
    // barrier lies between each of these and the next).
    __shared__ int odd_tile[3];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, col = lane % 32, half = lane / 32;
    const Work w = work_of(a);
    const int end = w.it.kv_end;

    const int r = w.it.row0 + 32 * wave + col;
    const bool live = r < w.rows;
    const int lim = live ? row_limit(w, r) : 0;
    u32x4_t qf[M::KS];
    {
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + (live ? q_offset(a, w, r) : 0);
#pragma unroll
        for (int ks = 0; ks < M::KS; ++ks) {
            const int c = 16 * ks + 8 * half;
            qf[ks] = u32x4_t{0, 0, 0, 0};
            if (live && c < a.D) qf[ks] = *reinterpret_cast<const u32x4_t*>(q + c);
        }
    }
    // positions that all of the workgroup's, all and any of the wave's rows see
    const int base = w.it.ctx - w.it.n + 1;
    const int wg_all = base + w.it.row0 / w.hg;
    const int first = w.it.row0 + 32 * wave;
    const int wave_all = base + first / w.hg;
    const int wave_end =
        first < w.rows ? min(base + min(first + 31, w.rows - 1) / w.hg, end) : 0;

    float m = -FLT_MAX, l = 0.f;
    f32x16_t O[M::CB];
#pragma unroll
    for (int cb = 0; cb < M::CB; ++cb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) O[cb][i] = 0.f;
    }

    // A load covers part of one block of 16 positions (64 lanes divide its
    // 16 * CH vectors): its page is the same for the whole wave.
    u32x4_t kr[M::LD], vr[M::LD];
    auto block_of = [&](int i) { return (i * kWaves + wave) * 4 / M::CH; };
    auto load = [&](int t0, const int (&page)[M::LD]) {
#pragma unroll
        for (int i = 0; i < M::LD; ++i) {
            const int blk = block_of(i);
            const int at = i * kBlock + threadIdx.x - blk * 16 * M::CH;
            const int t = at / M::CH, c = at % M::CH * 8;
            kr[i] = vr[i] = u32x4_t{0, 0, 0, 0};
            if (c < a.D) {
                const uint32_t off = t * a.D + c;
                kr[i] = *reinterpret_cast<const u32x4_t*>(
                    block_at<uint16_t>(a, w, a.k_pages, page[i], t0 + 16 * blk) + off);
                // (zeros past the end: whatever lies there has weight 0)
                if (t0 + 16 * blk + t < end)
                    vr[i] = *reinterpret_cast<const u32x4_t*>(
                        block_at<uint16_t>(a, w, a.v_pages, page[i], t0 + 16 * blk) + off);
            }
        }
    };
    auto pages_of = [&](int t0, int (&page)[M::LD]) {
#pragma unroll
        for (int i = 0; i < M::LD; ++i) page[i] = block_page(a, w, t0 + 16 * block_of(i));
    };
    auto stage = [&](int buf, int slot, int t0) {
        unsigned char* kb = lds + buf * M::BUF;
        unsigned char* vb = kb + M::K_BYTES;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < M::LD; ++i) {
            const int at = i * kBlock + threadIdx.x, t = at / M::CH, c = at % M::CH * 16;
            *reinterpret_cast<u32x4_t*>(kb + t * M::KST + c) = kr[i];
            *reinterpret_cast<u32x4_t*>(vb + t * M::VST + c) = vr[i];
            if (t0 + kTile > wg_all)
                odd |= non_finite<DT>(vr[i][0]) || non_finite<DT>(vr[i][1]) ||
                       non_finite<DT>(vr[i][2]) || non_finite<DT>(vr[i][3]);
        }
        if (odd) odd_tile[slot] = 1;
    };

    int page[M::LD];
    if (threadIdx.x < 3) odd_tile[threadIdx.x] = 0;
    int t0 = w.it.kv_begin;
    pages_of(t0, page);
    load(t0, page);
    pages_of(t0 + kTile, page);
    __syncthreads();
    stage(0, 0, t0);
    __syncthreads();
    for (int buf = 0, slot = 0; t0 < end; t0 += kTile, buf ^= 1, slot = slot == 2 ? 0 : slot + 1) {
        if (threadIdx.x == 0) odd_tile[slot == 0 ? 2 : slot - 1] = 0;
        const bool more = t0 + kTile < end;
        if (more) {
            load(t0 + kTile, page);
            pages_of(t0 + 2 * kTile, page);
        }
        if (t0 < wave_end) {
            const unsigned char* kb = lds + buf * M::BUF;
            const unsigned char* vb = kb + M::K_BYTES;
            f32x16_t s[M::TB];
#pragma unroll
            for (int tb = 0; tb < M::TB; ++tb) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[tb][i] = 0.f;
            }
#pragma unroll
            for (int ks = 0; ks < M::KS; ++ks) {
#pragma unroll
                for (int tb = 0; tb < M::TB; ++tb) {
                    const u32x4_t kf = *reinterpret_cast<const u32x4_t*>(
                        kb + (32 * tb + col) * M::KST + 32 * ks + 16 * half);
                    s[tb] = mfma32<DT>(kf, qf[ks], s[tb]);
                }
            }
            // score i of block tb: token 32 tb + 8 (i / 4) + 4 half + i % 4
            if (t0 + kTile > min(wave_all, end)) {
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
            mx *= a.qscale;
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
                    s[tb][i] = exp2_fast(fmaf(s[tb][i], a.qscale, -m));
                    l += s[tb][i];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    pf[2 * tb + i / 4][i % 4] = pack2<DT>(s[tb][2 * i], s[tb][2 * i + 1]);
            }
            if (odd_tile[slot] == 0) {
                // transposed: lanes of 16 take tokens 4 half .. + 3 of 16 channels
                const unsigned char* vt = vb + (4 * half + lane % 16 / 4) * M::VST +
                                          lane / 16 % 2 * 32 + lane % 4 * 8;
#pragma unroll
                for (int j = 0; j < 2 * M::TB; ++j) {
#pragma unroll
                    for (int cb = 0; cb < M::CB; ++cb) {
                        const uint2 lo = read_transposed(vt + 16 * j * M::VST + 64 * cb);
                        const uint2 hi = read_transposed(vt + (16 * j + 8) * M::VST + 64 * cb);
                        O[cb] = mfma32<DT>(u32x4_t{lo.x, lo.y, hi.x, hi.y}, pf[j], O[cb]);
                    }
                }
            } else {
                // A value that some row must not see would reach it as 0 * value:
                // token by token, for the rows that see it.
                for (int j = 0; j < kTile && t0 + j < end; ++j) {
                    // token 16 j4 + 8 (e / 4) + 4 h + e % 4 is element e of pf[j4]
                    const int j4 = j / 16, e = j % 16 / 8 * 4 + j % 4, h = j / 4 % 2;
                    u32x4_t f = pf[0];
#pragma unroll
                    for (int i = 1; i < 2 * M::TB; ++i)
                        if (j4 == i) f = pf[i];
                    const uint32_t word = e < 4 ? (e < 2 ? f[0] : f[1]) : (e < 6 ? f[2] : f[3]);
                    // (a weight that rounds to 0 still carries an infinity)
                    const float p =
                        fmaxf(half_of<DT>(__shfl(word, col + 32 * h), e & 1), FLT_MIN);
                    if (t0 + j >= lim) continue;
#pragma unroll
                    for (int cb = 0; cb < M::CB; ++cb) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint2 x = *reinterpret_cast<const uint2*>(
                                vb + j * M::VST + 64 * cb + 16 * i + 8 * half);
                            O[cb][4 * i] = fmaf(p, half_of<DT>(x.x, 0), O[cb][4 * i]);
                            O[cb][4 * i + 1] = fmaf(p, half_of<DT>(x.x, 1), O[cb][4 * i + 1]);
                            O[cb][4 * i + 2] = fmaf(p, half_of<DT>(x.y, 0), O[cb][4 * i + 2]);
                            O[cb][4 * i + 3] = fmaf(p, half_of<DT>(x.y, 1), O[cb][4 * i + 3]);
                        }
                    }
                }
            }
        }
        if (more) stage(buf ^ 1, slot == 2 ? 0 : slot + 1, t0 + kTile);
        __syncthreads();
    }

    l += __shfl_xor(l, 32);
    if (!live) return;
    const float inv = inverse_sum(l);
    const bool whole = w.it.part < 0;
    const int64_t at = whole ? out_offset(a, w, r) : part_row(a, w, r);
#pragma unroll
    for (int cb = 0; cb < M::CB; ++cb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = 32 * cb + 8 * i + 4 * half;
            if (c >= a.D) continue;
            const f32x4_t o = {O[cb][4 * i], O[cb][4 * i + 1], O[cb][4 * i + 2], O[cb][4 * i + 3]};
            if (whole) store4<DT>(a.out, at + c, o * inv);
            else *reinterpret_cast<f32x4_t*>(a.part_o + at * a.D + c) = o;
        }
    }
    if (!whole && half == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * at) = make_float2(m, l);
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
