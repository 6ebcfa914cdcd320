// pd_prefix_args.cuh — what the shared-prefix kernels are given.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace pd {

// FP16 work items: two streams over their own pages of one row tile, or two row tiles over the same pages.
enum : int { kItemSplit = 0, kItemPaired = 1 };

// A partial's l (else 0 or more, or NaN) where the row's live table has other pages than the plan's.
constexpr float kPieceMoved = -1.f;

struct PrefixArgs {
    const void *q;              // [B, Hq, D]
    const void *k, *v;          // [P, T, Hkv, D]
    // Work items.  FP32: 2 words of 4: {first member, members, KV head, row tile}, {first of the
    // group's pages in `pages`, first and end page of the piece, partial slot}.  FP16: 4 of them:
    // {first member, members, KV head, kind}, {first of the group's pages in `pages`, 0, 0, 0},
    // and per stream {row tile, first page, end page, slot}; kind kItem*.
    const int4 *items;
    // Per sequence: {member index in its group or -1, first row tile of KV head 0, row tiles per KV
    // head, first of the group's pages in `pages`}, {shared pages, planned tokens, 0, 0}.
    const int4 *seqs;
    const int2 *tiles;          // per row tile: {first partial slot, pieces}
    const int32_t *members;     // sequences of the groups, one after another
    const int32_t *pages;       // shared pages of the groups, one after another
    const int32_t *lengths;     // [B]
    const int32_t *table;       // a dynamic launch's page table [B, width]; NULL: the plan's, which is `pages`
    int64_t width;
    const float *rows;          // the suffix decode: FP32 [B, Hq, D] and (m, l) [B, Hq, 2]; NULL: no suffix
    const float *stats;
    float *part_o;              // [slots][D / 8][tile rows][8]
    float2 *part_ml;            // [slots][tile rows]
    void *out;                  // [B, Hq, D]
    uint32_t *error;
    int32_t B, Hq, Hkv, group, page_size, tile_rows, step_pages;
    int64_t P;                  // physical pages
    float scale_log2;           // log2(e) / sqrt(D)
};

}  // namespace pd
