// Attention of a step's new tokens over a paged cache: the launches of a plan
// and the merge of split contexts.
//
// For sequence b with n new tokens in a context of c (these included), query
// head h of kv head h / (q_heads / kv_heads), new token i:
//   o = sum_p softmax_p(q . k_p * scale) v_p   over positions p <= c - n + i.
// A plan's items are workgroups' shares of this (kivi_paged.hpp); each kind of
// row tile is one launch.  Block b takes kv head b % kv_heads: blocks go to the
// eight XCDs in turn, so with 8 kv heads (or a multiple) the tiles that read
// one head's pages meet in one XCD's L2.
#include <hip/hip_runtime.h>

#include <math.h>

#include <type_traits>

#include "kivi_paged8_attention.hpp"
#include "../../include/kivi_hip.h"

namespace kivi {
namespace {

constexpr int kMergeBlock = 256;
// (a launch has fewer than 2^32 lanes; all of these have 256 to a workgroup, but for
// tiles of 256 rows, which have 512)
constexpr int64_t kMostBlocks = (int64_t)UINT32_MAX / kMergeBlock;

// Joins partials: a thread takes four channels of a row.  Bound by its reads of the
// partials, and for few of them by one trip to memory: 4 us for a single token's 8
// splits, 17 us for 45 MB (80 pieces of 128 rows, 8 kv heads).
template <int DT>
__global__ void __launch_bounds__(kMergeBlock) paged_merge_kernel(PagedLaunch a) {
    const int per_row = a.D / 4;
    const int blocks = (a.part_rows * per_row + kMergeBlock - 1) / kMergeBlock;   // of a tile
    const int tile = blockIdx.x / blocks;
    const int kvh = tile % a.Hkv;
    const PagedMerge g = a.merges[tile / a.Hkv];
    const int at = (blockIdx.x - tile * blocks) * kMergeBlock + threadIdx.x;
    const int row = at / per_row, c = (at - row * per_row) * 4, r = g.row0 + row;
    if (row >= g.rows) return;
    const int64_t p0 = part_at(a, kvh, g.part, g.n * a.hg) + row;
    const float* ml = a.part_ml + 2 * p0;
    const float* po = a.part_o + p0 * a.D + c;
    const int64_t rows = paged_few(g.n * a.hg) ? a.few_rows : a.part_rows;
    const int64_t next_ml = 2 * rows, next_o = rows * a.D;
    float top = -FLT_MAX;
#pragma unroll 4
    for (int s = 0; s < g.splits; ++s) top = fmaxf(top, ml[s * next_ml]);
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll 4
    for (int s = 0; s < g.splits; ++s) {
        const float2 x = *reinterpret_cast<const float2*>(ml + s * next_ml);
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(po + s * next_o);
        const float f = exp2_fast(x.x - top);
        sum = fmaf(x.y, f, sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = fmaf(y[i], f, o[i]);
    }
    if (sum == sum && has_nan(o)) {
        // (an infinity of a partial whose weight is 0 here: it is one all the same)
        o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int s = 0; s < g.splits; ++s) {
            const f32x4_t y = *reinterpret_cast<const f32x4_t*>(po + s * next_o);
            const float f = exp2_fast(ml[s * next_ml] - top);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = non_finite(y[i]) ? o[i] + y[i] : fmaf(y[i], f, o[i]);
        }
    }
    const int i = r / a.hg;
    store4<DT>(a.out, ((int64_t)(g.tok0 + i) * a.Hq + kvh * a.hg + (r - i * a.hg)) * a.D + c,
               o * inverse_sum(sum));
}

int64_t part_rows_of(const int64_t* info) {
    return info[kInfoFewParts] * info[kInfoFewRows] +
           (info[kInfoParts] - info[kInfoFewParts]) * info[kInfoPartRows];
}
int64_t part_floats(const int64_t* info, int32_t kv_heads, int32_t head_dim) {
    return part_rows_of(info) * kv_heads * (head_dim + 2);
}

// Checks a call's arguments and fills what its launches share; Hq 0: there is nothing to
// do.
int launch_args(PagedLaunch& a, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                int32_t dtype, const void* k_pages, const void* v_pages, int64_t num_pages,
                int32_t page_size, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                const int32_t* plan, const int64_t* info, float softmax_scale, void* out,
                void* workspace, size_t workspace_bytes) {
    if (info == nullptr) return set_error(kErrInvalidArgument, "null plan info");
    if (dtype < 0 || dtype > 2)
        return set_error(kErrInvalidArgument, "dtype %d is not 0 (f32), 1 (bf16) or 2 (f16)", dtype);
    int shift = -1;
    for (int s = 4; s <= 8; ++s)
        if (page_size == 1 << s) shift = s;
    if (shift < 0 || num_pages < 1 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads != 0 ||
        head_dim < 16 || head_dim > 256 || head_dim % 16 != 0 ||
        (int64_t)kv_heads * page_size * head_dim > INT32_MAX)
        return set_error(kErrInvalidArgument,
                         "unsupported geometry: page_size %d, %d query heads over %d kv heads, "
                         "head_dim %d", page_size, q_heads, kv_heads, head_dim);
    const float qscale = softmax_scale * (float)M_LOG2E;
    if (!(softmax_scale > 0.f) || !isfinite(qscale))
        return set_error(kErrInvalidArgument,
                         "softmax_scale must be positive and below 2^127, got %g",
                         (double)softmax_scale);
    a.Hq = 0;
    if (info[kInfoTokens] == 0) return kOk;
    if (q == nullptr || k_pages == nullptr || v_pages == nullptr || plan == nullptr ||
        out == nullptr)
        return set_error(kErrInvalidArgument, "null pointer");
    const int per = 16 / src_size(dtype);
    if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out |
         (uintptr_t)plan | (uintptr_t)workspace) & 15 ||
        q_token_stride % per != 0 || q_head_stride % per != 0)
        return set_error(kErrInvalidArgument,
                         "q's rows, pages, plan, out and workspace must be 16-byte aligned");
    const int64_t floats = part_floats(info, kv_heads, head_dim);
    if (floats > 0 && (workspace == nullptr || workspace_bytes < (size_t)floats * 4))
        return set_error(kErrInvalidArgument, "workspace must hold %lld bytes, got %zu",
                         (long long)floats * 4, workspace_bytes);
    a.q = q;
    a.q_st = q_token_stride;
    a.q_sh = q_head_stride;
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.out = out;
    a.pages = plan + info[kInfoPagesAt];
    a.merges = reinterpret_cast<const PagedMerge*>(plan + info[kInfoMergesAt]);
    a.zeros = plan + info[kInfoZerosAt];
    a.n_merges = (int)info[kInfoMerges];
    a.part_rows = (int)info[kInfoPartRows];
    a.few_rows = (int)info[kInfoFewRows];
    a.part_total = part_rows_of(info);
    a.many_at = info[kInfoFewParts] * (info[kInfoFewRows] - info[kInfoPartRows]);
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + a.part_total * kv_heads * head_dim;
    a.Hq = q_heads;
    a.Hkv = kv_heads;
    a.hg = q_heads / kv_heads;
    a.D = head_dim;
    a.page_shift = shift;
    a.qscale = qscale;
    return kOk;
}

// The launches of a plan: launch(kind) makes that of a kind's items.
template <class L, class F>
int run_items(L& a, int dtype, const int32_t* plan, const int64_t* info, hipStream_t s, F launch) {
    const PagedItem* items = reinterpret_cast<const PagedItem*>(plan + info[kInfoItemsAt]);
    // (the largest tiles first: the small ones fill in behind them)
    for (int kind = kPagedKinds - 1; kind >= 0; --kind) {
        int64_t before = 0;
        for (int j = 0; j < kind; ++j) before += info[kInfoItems + j];
        a.items = items + before;
        a.n_items = (int)info[kInfoItems + kind];
        if (a.n_items == 0) continue;
        const bool wide = std::is_same_v<L, Paged8Launch> && kind == kWide8;
        if ((int64_t)a.n_items * a.Hkv > kMostBlocks / (wide ? 2 : 1))
            return set_error(kErrInvalidArgument, "%d items are too many for one launch",
                             a.n_items);
        launch(kind);
        const int rc = check_launch("paged_attention");
        if (rc) return rc;
    }
    if (a.n_merges == 0) return kOk;
    const int64_t blocks = (int64_t)a.n_merges * a.Hkv *
                           ((a.part_rows * (a.D / 4) + kMergeBlock - 1) / kMergeBlock);
    if (blocks > kMostBlocks)
        return set_error(kErrInvalidArgument, "%d tiles to merge are too many for one launch",
                         a.n_merges);
    const dim3 grid((unsigned)blocks);
    if (dtype == kSrcF32) paged_merge_kernel<kSrcF32><<<grid, kMergeBlock, 0, s>>>(a);
    else if (dtype == kSrcBF16) paged_merge_kernel<kSrcBF16><<<grid, kMergeBlock, 0, s>>>(a);
    else paged_merge_kernel<kSrcF16><<<grid, kMergeBlock, 0, s>>>(a);
    return check_launch("paged_merge");
}

}  // namespace
}  // namespace kivi

using namespace kivi;

extern "C" {

size_t kivi_paged_attention_workspace_size(const int64_t* info, int32_t kv_heads,
                                           int32_t head_dim) {
    if (info == nullptr || kv_heads < 1 || head_dim < 1) return 0;
    return (size_t)part_floats(info, kv_heads, head_dim) * 4;
}

int kivi_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                         int32_t dtype, const void* k_pages, const void* v_pages,
                         int64_t num_pages, int32_t page_size, int32_t q_heads,
                         int32_t kv_heads, int32_t head_dim, const int32_t* plan,
                         const int64_t* info, float softmax_scale, void* out, void* workspace,
                         size_t workspace_bytes, void* stream) {
    PagedLaunch a{};
    const int rc = launch_args(a, q, q_token_stride, q_head_stride, dtype, k_pages, v_pages,
                               num_pages, page_size, q_heads, kv_heads, head_dim, plan, info,
                               softmax_scale, out, workspace, workspace_bytes);
    if (rc || a.Hq == 0) return rc;
    // (a kind that the type's plans do not have: those of pages of 8 bits do)
    if (info[kInfoItems + (dtype == kSrcF32 ? kMany : kFew64)] != 0)
        return set_error(kErrInvalidArgument, "the plan is not one of kivi_paged_plan");
    hipStream_t s = (hipStream_t)stream;
    return run_items(a, dtype, plan, info, s, [&](int kind) {
        if (kind == kMany) launch_paged_many(a, dtype, s);
        else if (dtype == kSrcF32) launch_paged_f32(a, kind, s);
        else launch_paged_few(a, dtype, s);
    });
}

int kivi_paged8_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                          int32_t dtype, const int8_t* k_pages, const int8_t* v_pages,
                          const float* k_scales, const float* v_scales, int64_t num_pages,
                          int32_t page_size, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                          const int32_t* plan, const int64_t* info, float softmax_scale, void* out,
                          void* workspace, size_t workspace_bytes, void* stream) {
    Paged8Launch a{};
    const int rc = launch_args(a, q, q_token_stride, q_head_stride, dtype, k_pages, v_pages,
                               num_pages, page_size, q_heads, kv_heads, head_dim, plan, info,
                               softmax_scale, out, workspace, workspace_bytes);
    if (rc || a.Hq == 0) return rc;
    if (k_scales == nullptr || v_scales == nullptr)
        return set_error(kErrInvalidArgument, "null scales");
    if (paged_plain_info(info) ||
        (info[kInfoItems + kWide8] != 0 && !paged_wide(dtype == kSrcF32, head_dim)))
        return set_error(kErrInvalidArgument, "the plan is not one of kivi_paged8_plan");
    a.k_scales = k_scales;
    a.v_scales = v_scales;
    hipStream_t s = (hipStream_t)stream;
    return run_items(a, dtype, plan, info, s, [&](int kind) {
        if (kind == kMany || kind == kWide8) launch_paged8_many(a, dtype, kind == kWide8, s);
        else launch_paged8_few(a, dtype, s);
    });
}

}  // extern "C"
