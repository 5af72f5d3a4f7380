// The plan of one step over a paged cache, shared by the host that writes it
// (kivi_paged.hip) and the kernels that read it.
//
// A paged cache holds keys and values as [num_pages][kv_heads][page_size]
// [head_dim] of the model's type; a sequence's position p lies on its page
// p / page_size.  A step brings n new tokens to each of some sequences.  The
// plan is one int32 array, written and checked on the host once per step and
// read by every layer's launches:
//   tokens  [tokens][2]   slot (page * page_size + offset) and position of
//                         each new token, the sequences one after the other
//   pages   [pages]       the sequences' page lists, one after the other
//   items   [items][8]    PagedItem: one workgroup's work for one kv head
//   merges  [merges][8]   PagedMerge: row tiles whose context is split
//   zeros   [8]           what lanes behind the head's channels load
#pragma once

#include "kivi_common.hpp"

namespace kivi {

// Query rows of a sequence and kv head: row r is new token r / hg, head
// r % hg of the kv head's hg = q_heads / kv_heads.  Token i sees positions
// 0 .. ctx - n + i.
struct PagedItem {
    int32_t tok0;        // the sequence's first new token among the step's
    int32_t n;           // its new tokens
    int32_t ctx;         // its length, the new tokens included
    int32_t page0;       // where its page list starts
    int32_t row0;        // first row of the tile
    int32_t kv_begin;    // positions of the split
    int32_t kv_end;
    int32_t part;        // the split's partial (-1: the only one, written out)
};

struct PagedMerge {
    int32_t tok0;
    int32_t n;
    int32_t row0;
    int32_t splits;
    int32_t part;        // first partial
    int32_t rows;        // of the tile
    int32_t pad[2];
};

static_assert(sizeof(PagedItem) == 32 && sizeof(PagedMerge) == 32, "plan records");

// Kinds of attention items: kind k takes 16 << k rows (none 32), and is one launch
// (kFew64: fp32, kMany: the 16-bit types).
enum PagedKind : int { kFew16 = 0, kFew64 = 2, kMany = 3, kPagedKinds = 4 };

constexpr int paged_tile_rows(int kind) { return 16 << kind; }

// The kind that takes `rows` rows of a kv head: fp32 has kernels of 16 and 64 rows,
// the 16-bit types of 16 and 128.  Up to 16 rows a kernel that streams them is
// faster (64 single tokens, 32/8 heads of 128: bf16, up to 8K positions, 287 us, in tiles
// of more rows 317; fp32, 4096 positions, 361 and 390, 512 positions 43 and 52), from
// there on the larger tiles.
constexpr int paged_kind(int64_t rows, bool f32) {
    return rows <= 16 ? kFew16 : f32 ? kFew64 : kMany;
}
// Sequences whose partials have rows of their own number (beside tiles of many rows
// those of single tokens would otherwise be mostly empty: eight tokens of 32K beside
// five of another sequence, 32/4 heads of 128, took 55 MB).
constexpr bool paged_few(int64_t rows) { return rows <= paged_tile_rows(kFew16); }

// Workgroups that the card works on at once: 256 CUs, and as many on each as the
// kernels' registers or LDS leave room for (fp32's 64 rows: as bring more; more
// than that share the matrix cores that bound it).
constexpr int paged_slots(int kind, int head_dim) {
    const int per_cu = kind == kMany    ? (head_dim <= 64 ? 4 : head_dim <= 128 ? 2 : 1)
                       : kind == kFew16 ? (head_dim <= 64 ? 3 : head_dim <= 128 ? 2 : 1)
                                        : 2;
    return 256 * per_cu;
}

// Positions of a sequence, and rows of a step (tokens x heads of a kv head), at most:
// kernels look a few tiles past the last one in 32 bits.
constexpr int64_t kPagedMost = ((int64_t)1 << 31) - 4096;

// info[] of kivi_paged_plan
enum PagedInfo : int {
    kInfoInts = 0,        // int32s of the plan
    kInfoTokens = 1,
    kInfoPagesAt = 2,     // offset of the page lists
    kInfoItemsAt = 3,
    kInfoMergesAt = 4,
    kInfoMerges = 5,
    kInfoItems = 6,       // items of each kind, in order
    kInfoParts = 10,      // partials of a kv head
    kInfoPartRows = 11,   // rows of a partial (of the split tile that has most)
    kInfoContext = 12,    // the longest sequence
    kInfoZerosAt = 13,
    kInfoFewParts = 14,   // partials of sequences with few rows (the first ones),
    kInfoFewRows = 15,    // and rows of these
    kInfoCount = 16,
};

struct PagedLaunch {
    const void* q;
    int64_t q_st, q_sh;           // strides of tokens and heads, in elements
    const void* k_pages;
    const void* v_pages;
    void* out;                    // [tokens][q_heads][head_dim]
    float* part_o;                // [kv head][partial][its rows][head_dim]
    float* part_ml;               // [kv head][partial][its rows][2]: maximum and sum
    const int32_t* pages;
    const PagedItem* items;
    const PagedMerge* merges;
    const int32_t* zeros;
    int n_items, n_merges, part_rows, few_rows;
    int64_t part_total;           // rows of a kv head's partials
    int64_t many_at;              // row of partial p with many rows: this + p * part_rows
    int Hq, Hkv, hg, D, page_shift;
    float qscale;                 // softmax scale * log2 e
};

}  // namespace kivi
