// Paged K/V cache: a step's plan (host) and the append of its new tokens.
//
// The append takes a projection's queries, keys and values of the step's
// tokens, token-major as a model's projections leave them.  For a head row x
// of the queries or keys:
//   y = x * rsqrt(mean(x^2) + eps) * weight          (where a weight is given)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)   for each rotated pair
// with the token's position's row of the tables, all in fp32 and rounded once
// to the tensors' type; values are copied.  Keys and values go to their pages,
// queries to an output of their own: one launch, each element read and
// written once.  Memory-bound for prompts (12.3K tokens of 32/8 heads of 128 with
// norms, bf16: 59 us, 4.7 TB/s, where a copy reaches 5.0), launch-bound for single
// tokens (64 of 64/8 heads, fp16: 3.7 us on the GPU, 12 us a call).
// How lanes share a head: kivi_paged_rows.hpp.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <functional>
#include <new>
#include <vector>

#include "kivi_paged_rows.hpp"
#include "../../include/kivi_hip.h"

namespace kivi {
namespace {

// A segment of lanes takes a head of a token.  (Several heads to a segment, to
// share the angles and have more loads in flight, cost more in waves on a SIMD
// than it gave: 12.3K tokens of 32/8 heads with norms, 1 head 60 us, 2 heads 67, 4
// heads 83.)
template <int DT>
__global__ void __launch_bounds__(kAppendBlock) paged_append_kernel(AppendArgs a) {
    const int heads = a.Hq + 2 * a.Hkv;
    const uint32_t t = blockIdx.x * kAppendBlock + threadIdx.x;
    const uint32_t row = t >> a.lanes_log2;
    const int tok = (int)(row / (uint32_t)heads), h = (int)(row - (uint32_t)tok * heads);
    if (tok >= a.n_tokens) return;                       // (whole segments leave)
    const HeadLane lane = head_lane(a, (int)(t & ((1u << a.lanes_log2) - 1)));
    const int2 place = a.tokens[tok];

    const void* src = a.v;
    const void* norm = nullptr;
    int64_t from = tok * a.v_st + (int64_t)(h - a.Hq - a.Hkv) * a.v_sh;
    if (h < a.Hq) {
        src = a.q;
        norm = a.q_norm;
        from = tok * a.q_st + (int64_t)h * a.q_sh;
    } else if (h < a.Hq + a.Hkv) {
        src = a.k;
        norm = a.k_norm;
        from = tok * a.k_st + (int64_t)(h - a.Hq) * a.k_sh;
    }
    void* dst = a.q_out;
    int64_t to = ((int64_t)tok * a.Hq + h) * a.D;
    if (h >= a.Hq) {
        const int kvh = h < a.Hq + a.Hkv ? h - a.Hq : h - a.Hq - a.Hkv;
        const int64_t page = place.x >> a.page_shift;
        const int off = place.x & ((1 << a.page_shift) - 1);
        dst = h < a.Hq + a.Hkv ? a.k_pages : a.v_pages;
        to = (((page * a.Hkv + kvh) << a.page_shift) + off) * a.D;
    }
    move_row<DT>(a, lane, src, from, norm, h < a.Hq + a.Hkv, place.y, dst, to);
}

}  // namespace

int paged_page_shift(int32_t page_size) {
    for (int s = 4; s <= 8; ++s)
        if (page_size == 1 << s) return s;
    return -1;
}

int paged_check_pool(int32_t dtype, int64_t num_pages, int32_t page_size, int32_t q_heads,
                     int32_t kv_heads, int32_t head_dim) {
    if (dtype < 0 || dtype > 2)
        return set_error(kErrInvalidArgument, "dtype %d is not 0 (f32), 1 (bf16) or 2 (f16)", dtype);
    if (paged_page_shift(page_size) < 0)
        return set_error(kErrInvalidArgument,
                         "page_size must be 16, 32, 64, 128 or 256, got %d", page_size);
    if (num_pages < 1 || num_pages > INT32_MAX / page_size)
        return set_error(kErrInvalidArgument,
                         "num_pages must be positive and hold fewer than 2^31 tokens, got %lld",
                         (long long)num_pages);
    if (kv_heads < 1 || q_heads < 1 || q_heads % kv_heads != 0)
        return set_error(kErrInvalidArgument,
                         "q_heads (%d) must be a positive multiple of kv_heads (%d)", q_heads,
                         kv_heads);
    if (head_dim < 16 || head_dim > 256 || head_dim % 16 != 0)
        return set_error(kErrUnsupported,
                         "head_dim must be a multiple of 16 up to 256, got %d", head_dim);
    if ((int64_t)kv_heads * page_size * head_dim > INT32_MAX)
        return set_error(kErrUnsupported, "a page of %d kv heads is too large", kv_heads);
    return kOk;
}

namespace {

struct Tile {
    int seq, row0;
    int64_t end;                 // positions that its rows see
};

// How one kind's tiles (the longest first) are cut: the first `whole` stay
// whole, the others into pieces of at most `length` positions (a multiple of 64).
struct Cut {
    size_t whole;
    int64_t length;
    int64_t end;                 // when the last piece ends, in positions
    int64_t pieces(size_t tile, int64_t len) const {
        return tile < whole ? 1 : std::max<int64_t>(1, (len + length - 1) / length);
    }
};

// Costs in positions, as measured: an item's start; what a row of a partial
// adds to it (written, then read by the merge); the merge's launch.
struct Costs {
    int64_t start, partial_row, merge;
};
constexpr Costs paged_costs(int kind, bool eight, int head_dim) {
    // A position of 8 bits takes few rows half the time up to 128 channels, so what is
    // not positions weighs more (64 single tokens of 4K to 8K positions, 32/8 heads of 128,
    // 152 us and 163 with {64, 4, 96}; 16 of 3000, 24 and 31; 64 of 8K, 12/12 of 64, 115 and
    // 126; 116 steps of four geometries 0.97 of the time, none above 1.04; with 256
    // channels 29 steps 1.01).
    if (eight && kind == kFew16 && head_dim <= 128) return Costs{256, 8, 256};
    // (fp32's products of 64 rows take four times as long for a position; the eight waves
    // of kWide8 write twice the rows in the time of one)
    return kind != kFew64 ? Costs{64, 4, 96} : eight ? Costs{64, 2, 96} : Costs{16, 1, 24};
}

// Pages of 8 bits: a position's time in tiles of 256 rows (one workgroup on a CU), in
// hundredths of its time in tiles of 128 (two), and the positions on the longest way from
// which on they are taken.
constexpr int64_t kWideCost = 93, kWideFrom = 2048;

// The cut whose items, dealt in order to `machines` workgroups as these come
// free, end first.
Cut best_cut(const std::vector<Tile>& tiles, const std::vector<int>& rows, int64_t machines,
             Costs cost) {
    Cut best{tiles.size(), 64, INT64_MAX};
    const int64_t longest = tiles.empty() ? 0 : tiles.front().end;
    std::vector<int64_t> busy;                    // a heap: when each comes free
    const size_t rounds = tiles.size() / (size_t)machines * (size_t)machines;
    for (int64_t n : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
        const int64_t T = ((longest + n - 1) / n + 63) / 64 * 64;
        if (n > 1 && T < 128) break;
        // (with whole rounds of tiles first, only the rest is cut)
        for (int keep = 0; keep < (n > 1 && rounds > 0 ? 2 : 1); ++keep) {
            Cut cut{keep ? rounds : 0, T, 0};
            int64_t items = 0;
            for (size_t i = 0; i < tiles.size(); ++i) items += cut.pieces(i, tiles[i].end);
            if (n > 1 && items > 4 * machines) continue;
            busy.assign((size_t)machines, 0);
            int64_t& end = cut.end;
            bool merge = false;
            for (size_t i = 0; i < tiles.size() && end < best.end; ++i) {
                const int64_t k = cut.pieces(i, tiles[i].end);
                merge |= k > 1;
                const int64_t each =
                    tiles[i].end / k + cost.start + (k > 1 ? cost.partial_row * rows[i] : 0);
                for (int64_t j = 0; j < k; ++j) {
                    std::pop_heap(busy.begin(), busy.end(), std::greater<int64_t>());
                    busy.back() += each;
                    end = std::max(end, busy.back());
                    std::push_heap(busy.begin(), busy.end(), std::greater<int64_t>());
                }
            }
            if (merge) end += cost.merge;
            if (end < best.end) best = cut;
        }
    }
    return best;
}

// The plan of kivi_paged_plan, and with `eight` of kivi_paged8_plan.
int make_plan(bool eight, int32_t n_seqs, const int32_t* new_lens, const int32_t* context_lens,
              const int32_t* page_table, int64_t table_stride, int32_t table_pages,
              int32_t page_size, int64_t num_pages, int32_t dtype, int32_t q_heads,
              int32_t kv_heads, int32_t head_dim, int32_t* plan, int64_t plan_ints,
              int64_t* info) {
    int rc = paged_check_pool(dtype, num_pages, page_size, q_heads, kv_heads, head_dim);
    if (rc) return rc;
    if (n_seqs < 0 || info == nullptr || table_pages < 0 || table_stride < table_pages ||
        (n_seqs > 0 && (new_lens == nullptr || context_lens == nullptr ||
                        (page_table == nullptr && table_pages > 0))))
        return set_error(kErrInvalidArgument, "null or negative plan argument");
    const int shift = paged_page_shift(page_size);
    const int hg = q_heads / kv_heads;
    const bool f32 = dtype == 0 && !eight;   // (8 bits: their products run on the 16-bit units)
    try {
        int64_t tokens = 0, pages = 0, longest = 0;
        for (int s = 0; s < n_seqs; ++s) {
            const int64_t n = new_lens[s], c = context_lens[s];
            if (n < 0 || c < n)
                return set_error(kErrInvalidArgument,
                                 "sequence %d: %lld new tokens in a context of %lld", s,
                                 (long long)n, (long long)c);
            if (c > kPagedMost)
                return set_error(kErrInvalidArgument,
                                 "sequence %d: a context of %lld, at most %lld positions are taken",
                                 s, (long long)c, (long long)kPagedMost);
            const int64_t p = (c + page_size - 1) >> shift;
            if (p > table_pages)
                return set_error(kErrInvalidArgument,
                                 "sequence %d: a context of %lld needs %lld pages, the table has "
                                 "%d", s, (long long)c, (long long)p, table_pages);
            if (n == 0) continue;
            for (int64_t j = 0; j < p; ++j) {
                const int32_t page = page_table[s * table_stride + j];
                if (page < 0 || page >= num_pages)
                    return set_error(kErrInvalidArgument,
                                     "sequence %d: page %d outside the pool of %lld", s, page,
                                     (long long)num_pages);
            }
            tokens += n;
            pages += p;
            longest = std::max(longest, c);
        }
        if (tokens > INT32_MAX / 4 || tokens * (int64_t)hg > kPagedMost || pages > INT32_MAX / 4)
            return set_error(kErrInvalidArgument, "a step of %lld tokens over %lld pages is too "
                             "large", (long long)tokens, (long long)pages);

        // No slot is written twice: the new tokens' stretches of pages, sorted.
        struct Run { int32_t page, from, to; };
        std::vector<Run> runs;
        for (int s = 0; s < n_seqs; ++s) {
            if (new_lens[s] == 0) continue;
            const int64_t first = context_lens[s] - new_lens[s], last = context_lens[s] - 1;
            for (int64_t j = first >> shift; j <= last >> shift; ++j)
                runs.push_back({page_table[s * table_stride + j],
                                (int32_t)(std::max(first, j << shift) - (j << shift)),
                                (int32_t)(std::min<int64_t>(last, (j << shift) + page_size - 1) -
                                          (j << shift))});
        }
        std::sort(runs.begin(), runs.end(), [](const Run& a, const Run& b) {
            return a.page != b.page ? a.page < b.page : a.from < b.from;
        });
        for (size_t i = 1; i < runs.size(); ++i) {
            if (runs[i].page != runs[i - 1].page) continue;
            if (runs[i].from <= runs[i - 1].to)
                return set_error(kErrInvalidArgument, "page %d: a slot is given to two new tokens",
                                 runs[i].page);
            // (each would rescale the other's)
            if (eight && runs[i].from / kScaleBlock <= runs[i - 1].to / kScaleBlock)
                return set_error(kErrInvalidArgument,
                                 "page %d: a block of %d positions is given to two sequences' new "
                                 "tokens", runs[i].page, kScaleBlock);
        }

        // Row tiles, and the positions that the last row of each sees.  Beside 16-bit
        // sequences of more than 16 rows those of fewer go into the same launch, where
        // their loads run beside the others' products (64/8 heads, fp16, two chunks of 777
        // tokens and 30 single ones: 281 us, as two launches 354; 32/8 heads, bf16, 63
        // single tokens of 8K beside five tokens: 327 and 354, 128 of 2K beside eight
        // times five: 177 and 188, eight of 500 beside 200: 29 and 38; 28/4 heads of 256,
        // where a CU holds one workgroup, 18 of 2K beside 200: 58 and 78, but 30 of 8K
        // beside 200: 244 and 228).  In fp32, where a tile of many rows takes few at the
        // time of products that only one of its waves has, up to 2^23 elements of their
        // keys (32/8 heads of 128, 28 single tokens beside two of 200: 2^23 75 and 88 us,
        // 2^24 102 and 97; eight beside 94: 2^22 31 and 35, 2^23 46 and 41, 2^24 60 and
        // 51; 16/2 heads of 256, eight beside 94: 2^23 52 and 54, 2^24 71 and 64).
        int64_t small = 0;
        bool large = false;
        for (int s = 0; s < n_seqs; ++s) {
            const int64_t rows = (int64_t)new_lens[s] * hg;
            if (rows > 0 && rows <= 16) small += context_lens[s];
            large |= rows > 16;
        }
        int few = kFew16;
        if (large && !f32) few = kMany;
        if (large && f32 && small <= (1 << 23) / head_dim / kv_heads) few = kFew64;
        std::vector<Tile> tiles[kPagedKinds];
        auto add_tiles = [&](int s, int kind) {
            const int64_t n = new_lens[s], rows = n * hg;
            const int step = paged_tile_rows(kind, eight);
            for (int64_t r = 0; r < rows; r += step) {
                const int64_t last = std::min(rows, r + step) - 1;
                tiles[kind].push_back({s, (int)r, context_lens[s] - n + last / hg + 1});
            }
        };
        for (int s = 0; s < n_seqs; ++s) {
            const int64_t rows = (int64_t)new_lens[s] * hg;
            if (rows > 0) add_tiles(s, std::max(few, paged_kind(rows, f32)));
        }
        auto tile_rows = [&](const Tile& t, int kind) {
            return (int)std::min<int64_t>(paged_tile_rows(kind, eight),
                                          (int64_t)new_lens[t.seq] * hg - t.row0);
        };
        auto cut_tiles = [&](int kind) {
            // longest first: the last workgroups to start are short ones
            std::vector<Tile>& of = tiles[kind];
            std::stable_sort(of.begin(), of.end(),
                             [](const Tile& a, const Tile& b) { return a.end > b.end; });
            std::vector<int> rows;
            for (const Tile& t : of) rows.push_back(tile_rows(t, kind));
            const int64_t slots = paged_slots(kind, head_dim, eight, dtype == 0);
            return best_cut(of, rows, std::max<int64_t>(1, slots / kv_heads),
                            paged_costs(kind, eight, head_dim));
        };
        Cut cuts[kPagedKinds];
        for (int kind = 0; kind < kPagedKinds; ++kind) cuts[kind] = cut_tiles(kind);
        // Tiles of 256 rows, whose eight waves share the widening of a tile of codes, where by
        // these costs they end first (bf16, heads of 128, in tiles of 256 and of 128 rows: a
        // chunk of 2048 tokens after 8200, 32/8 heads, 348 and 373 us; 400 after 30000, 32/32,
        // 255 and 289; four of 256 after 3000, 32/8, 72 and 75; 520 after 8000, 32/32, whose
        // third tile is nearly empty, 135 and 117; shorter ways, as eight of 256 after
        // 1000, 32/32: 50 and 44).  Sequences of few rows would need a launch of their own.
        if (eight && large && small == 0 && paged_wide(dtype == 0, head_dim) &&
            cuts[kMany].end >= kWideFrom) {
            for (int s = 0; s < n_seqs; ++s)
                if (new_lens[s] > 0) add_tiles(s, kWide8);
            cuts[kWide8] = cut_tiles(kWide8);
            tiles[cuts[kWide8].end * kWideCost < cuts[kMany].end * 100 ? kMany : kWide8].clear();
        }
        auto is_few = [&](const Tile& t) { return paged_few((int64_t)new_lens[t.seq] * hg); };
        int64_t items = 0, merges = 0, parts = 0, part_rows = 0, kinds[kPagedKinds] = {0, 0, 0, 0};
        int64_t few_parts = 0, few_rows = 0;
        for (int kind = 0; kind < kPagedKinds; ++kind) {
            const std::vector<Tile>& of = tiles[kind];
            for (size_t i = 0; i < of.size(); ++i) {
                const int64_t splits = cuts[kind].pieces(i, of[i].end);
                items += splits;
                kinds[kind] += splits;
                if (splits == 1) continue;
                merges += 1;
                parts += splits;
                part_rows = std::max<int64_t>(part_rows, tile_rows(of[i], kind));
                if (!is_few(of[i])) continue;
                few_parts += splits;
                few_rows = std::max<int64_t>(few_rows, tile_rows(of[i], kind));
            }
        }
        const int64_t pages_at = 2 * tokens, items_at = (pages_at + pages + 7) / 8 * 8;
        const int64_t merges_at = items_at + 8 * items, zeros_at = merges_at + 8 * merges;
        int64_t blocks = 0;
        for (int s = 0; s < n_seqs && eight; ++s)
            if (new_lens[s] > 0)
                blocks += (int64_t)(context_lens[s] - 1) / kScaleBlock -
                          (context_lens[s] - new_lens[s]) / kScaleBlock + 1;
        const int64_t blocks_at = zeros_at + 8;
        const int64_t ints = tokens > 0 ? blocks_at + 4 * blocks : 0;
        if (ints > INT32_MAX || parts > INT32_MAX / 64)
            return set_error(kErrInvalidArgument, "a plan of %lld words is too large",
                             (long long)ints);
        for (int i = 0; i < (eight ? kInfoCount8 : kInfoCount); ++i) info[i] = 0;
        info[kInfoInts] = ints;
        info[kInfoTokens] = tokens;
        info[kInfoPagesAt] = pages_at;
        info[kInfoItemsAt] = items_at;
        info[kInfoMergesAt] = merges_at;
        info[kInfoMerges] = merges;
        for (int i = 0; i < kPagedKinds; ++i) info[kInfoItems + i] = kinds[i];
        info[kInfoParts] = parts;
        info[kInfoPartRows] = part_rows;
        info[kInfoContext] = longest;
        info[kInfoZerosAt] = zeros_at;
        info[kInfoFewParts] = few_parts;
        info[kInfoFewRows] = few_rows;
        if (eight) {
            info[kInfoBlocksAt] = blocks_at;
            info[kInfoBlocks] = blocks;
        }
        if (plan == nullptr || tokens == 0) return kOk;
        if (plan_ints < ints)
            return set_error(kErrInvalidArgument, "the plan needs %lld words, got %lld",
                             (long long)ints, (long long)plan_ints);

        std::vector<int32_t> tok0(n_seqs), page0(n_seqs);
        int32_t t = 0, pg = 0;
        for (int s = 0; s < n_seqs; ++s) {
            tok0[s] = t;
            page0[s] = pg;
            if (new_lens[s] == 0) continue;
            const int32_t* row = page_table + s * table_stride;
            const int64_t np = ((int64_t)context_lens[s] + page_size - 1) >> shift;
            for (int64_t j = 0; j < np; ++j) plan[pages_at + pg + j] = row[j];
            pg += (int32_t)np;
            for (int32_t i = 0; i < new_lens[s]; ++i, ++t) {
                const int32_t pos = context_lens[s] - new_lens[s] + i;
                plan[2 * t] = row[pos >> shift] * page_size + (pos & (page_size - 1));
                plan[2 * t + 1] = pos;
            }
        }
        for (int64_t i = pages_at + pages; i < items_at; ++i) plan[i] = 0;
        for (int64_t i = zeros_at; i < blocks_at; ++i) plan[i] = 0;
        PagedBlock* block = reinterpret_cast<PagedBlock*>(plan + blocks_at);
        for (int s = 0; s < n_seqs && eight; ++s) {
            const int32_t from = context_lens[s] - new_lens[s], c = context_lens[s];
            for (int32_t p = from; p < c; p = p / kScaleBlock * kScaleBlock + kScaleBlock) {
                const int32_t first = p / kScaleBlock * kScaleBlock;
                *block++ = PagedBlock{
                    page_table[s * table_stride + (first >> shift)] * page_size +
                        (first & (page_size - 1)),
                    tok0[s] + (p - from), p, (int16_t)(p - first),
                    (int16_t)(std::min(kScaleBlock, c - first) - (p - first))};
            }
        }
        PagedItem* item = reinterpret_cast<PagedItem*>(plan + items_at);
        PagedMerge* merge = reinterpret_cast<PagedMerge*>(plan + merges_at);
        int32_t next_few = 0, next_many = (int32_t)few_parts;
        for (int kind = 0; kind < kPagedKinds; ++kind) {
            for (size_t j = 0; j < tiles[kind].size(); ++j) {
                const Tile& x = tiles[kind][j];
                const int64_t splits = cuts[kind].pieces(j, x.end);
                // (whole units of 64 positions, shared out evenly)
                const int64_t units = (x.end + 63) / 64;
                const int s = x.seq;
                int32_t& part = is_few(x) ? next_few : next_many;
                if (splits > 1)
                    *merge++ = PagedMerge{tok0[s], new_lens[s], x.row0, (int32_t)splits, part,
                                          tile_rows(x, kind), {0, 0}};
                for (int64_t i = 0; i < splits; ++i) {
                    const int64_t b = units * i / splits * 64;
                    const int64_t e = std::min(x.end, units * (i + 1) / splits * 64);
                    *item++ = PagedItem{tok0[s], new_lens[s], context_lens[s], page0[s], x.row0,
                                        (int32_t)b, (int32_t)e, splits > 1 ? part++ : -1};
                }
            }
        }
        return kOk;
    } catch (...) {                                      // (bad_alloc, length_error)
        return set_error(kErrRuntime, "out of host memory for a plan");
    }
}

}  // namespace

// Checks an append's arguments and fills the kernels'; n_tokens 0: there is nothing to do.
int paged_append_args(AppendArgs& a, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                      const void* k, int64_t k_token_stride, int64_t k_head_stride,
                      const void* v, int64_t v_token_stride, int64_t v_head_stride,
                      int32_t dtype, void* q_out, void* k_pages, void* v_pages,
                      int64_t num_pages, int32_t page_size, int32_t q_heads, int32_t kv_heads,
                      int32_t head_dim, const int32_t* plan, int32_t tokens, const float* cos,
                      const float* sin, int32_t rotary_dim, int32_t interleaved,
                      const void* q_norm, const void* k_norm, int32_t norm_dtype, float eps) {
    const int32_t hq = q == nullptr ? 0 : q_heads;
    const int rc = paged_check_pool(dtype, num_pages, page_size,
                                    q == nullptr ? kv_heads : q_heads, kv_heads, head_dim);
    if (rc) return rc;
    if (tokens < 0) return set_error(kErrInvalidArgument, "tokens %d must not be negative", tokens);
    if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16 != 0)
        return set_error(kErrInvalidArgument,
                         "rotary_dim must be a multiple of 16 up to head_dim, got %d", rotary_dim);
    if (rotary_dim > 0 && (cos == nullptr || sin == nullptr))
        return set_error(kErrInvalidArgument, "rotation needs cos and sin");
    if (rotary_dim > 0 && (((uintptr_t)cos | (uintptr_t)sin) & 15))
        return set_error(kErrInvalidArgument, "cos and sin must be 16-byte aligned");
    if (norm_dtype < 0 || norm_dtype > 2)
        return set_error(kErrInvalidArgument, "norm_dtype %d is not 0, 1 or 2", norm_dtype);
    a = AppendArgs{};
    if (tokens == 0) return kOk;
    if (k == nullptr || v == nullptr || k_pages == nullptr || v_pages == nullptr ||
        plan == nullptr || (q != nullptr && q_out == nullptr))
        return set_error(kErrInvalidArgument, "null pointer");
    const uintptr_t align = 15;
    if (((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)(q != nullptr ? q_out : nullptr)) &
        align)
        return set_error(kErrInvalidArgument, "pages and q_out must be 16-byte aligned");
    a.q = q; a.k = k; a.v = v;
    a.q_st = q_token_stride; a.q_sh = q_head_stride;
    a.k_st = k_token_stride; a.k_sh = k_head_stride;
    a.v_st = v_token_stride; a.v_sh = v_head_stride;
    a.q_out = q_out; a.k_pages = k_pages; a.v_pages = v_pages;
    a.tokens = reinterpret_cast<const int2*>(plan);
    a.cos = cos; a.sin = sin;
    a.q_norm = q_norm; a.k_norm = k_norm; a.norm_dt = norm_dtype;
    a.eps = eps;
    a.inv_d = 1.0f / (float)head_dim;
    a.n_tokens = tokens; a.Hq = hq; a.Hkv = kv_heads; a.D = head_dim;
    a.page_shift = paged_page_shift(page_size);
    a.rot = rotary_dim; a.interleaved = interleaved != 0;
    a.lanes_log2 = 0;
    while ((1 << a.lanes_log2) < head_dim / 16) ++a.lanes_log2;
    // vectors of eight elements where every row starts on 16 bytes
    int64_t strides = k_token_stride | k_head_stride | v_token_stride | v_head_stride;
    uintptr_t bases = (uintptr_t)k | (uintptr_t)v;
    if (q != nullptr) {
        strides |= q_token_stride | q_head_stride;
        bases |= (uintptr_t)q;
    }
    a.vec = (strides * src_size(dtype) & 15) == 0 && (bases & 15) == 0;
    a.norm_vec = (((uintptr_t)q_norm | (uintptr_t)k_norm) & 15) == 0;
    return kOk;
}

}  // namespace kivi

using namespace kivi;

extern "C" {

int kivi_paged_plan(int32_t n_seqs, const int32_t* new_lens, const int32_t* context_lens,
                    const int32_t* page_table, int64_t table_stride, int32_t table_pages,
                    int32_t page_size, int64_t num_pages, int32_t dtype, int32_t q_heads,
                    int32_t kv_heads, int32_t head_dim, int32_t* plan, int64_t plan_ints,
                    int64_t* info) {
    return make_plan(false, n_seqs, new_lens, context_lens, page_table, table_stride, table_pages,
                     page_size, num_pages, dtype, q_heads, kv_heads, head_dim, plan, plan_ints,
                     info);
}

int kivi_paged8_plan(int32_t n_seqs, const int32_t* new_lens, const int32_t* context_lens,
                     const int32_t* page_table, int64_t table_stride, int32_t table_pages,
                     int32_t page_size, int64_t num_pages, int32_t dtype, int32_t q_heads,
                     int32_t kv_heads, int32_t head_dim, int32_t* plan, int64_t plan_ints,
                     int64_t* info) {
    return make_plan(true, n_seqs, new_lens, context_lens, page_table, table_stride, table_pages,
                     page_size, num_pages, dtype, q_heads, kv_heads, head_dim, plan, plan_ints,
                     info);
}

int kivi_paged_append(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                      const void* k, int64_t k_token_stride, int64_t k_head_stride,
                      const void* v, int64_t v_token_stride, int64_t v_head_stride,
                      int32_t dtype, void* q_out, void* k_pages, void* v_pages,
                      int64_t num_pages, int32_t page_size, int32_t q_heads, int32_t kv_heads,
                      int32_t head_dim, const int32_t* plan, int32_t tokens, const float* cos,
                      const float* sin, int32_t rotary_dim, int32_t interleaved,
                      const void* q_norm, const void* k_norm, int32_t norm_dtype, float eps,
                      void* stream) {
    AppendArgs a;
    const int rc = paged_append_args(a, q, q_token_stride, q_head_stride, k, k_token_stride,
                                     k_head_stride, v, v_token_stride, v_head_stride, dtype, q_out,
                                     k_pages, v_pages, num_pages, page_size, q_heads, kv_heads,
                                     head_dim, plan, tokens, cos, sin, rotary_dim, interleaved,
                                     q_norm, k_norm, norm_dtype, eps);
    if (rc || a.n_tokens == 0) return rc;
    const int64_t lanes = (int64_t)tokens * (a.Hq + 2 * kv_heads) << a.lanes_log2;
    if (lanes > INT32_MAX)
        return set_error(kErrInvalidArgument, "%d tokens are too many for one launch", tokens);
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)((lanes + kAppendBlock - 1) / kAppendBlock));
    if (dtype == kSrcF32) paged_append_kernel<kSrcF32><<<grid, kAppendBlock, 0, s>>>(a);
    else if (dtype == kSrcBF16) paged_append_kernel<kSrcBF16><<<grid, kAppendBlock, 0, s>>>(a);
    else paged_append_kernel<kSrcF16><<<grid, kAppendBlock, 0, s>>>(a);
    return check_launch("paged_append");
}

}  // extern "C"
