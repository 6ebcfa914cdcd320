// pd_prefix.hpp — plans of shared-prefix decode attention (host side).
#pragma once

#include <cstddef>
#include <cstdint>
#include <vector>

#include "paged_decode.h"
#include "pd_plan.hpp"

namespace pd {

// Sections of the plan's device buffer (256-byte aligned).
struct PrefixImage {
    size_t off_error = 0, off_items = 0, off_seqs = 0, off_tiles = 0, off_members = 0, off_pages = 0, off_lengths = 0;
    size_t off_suffix = 0;                        // the suffix plan's own buffer
    size_t off_rows = 0, off_stats = 0;           // the suffix decode's FP32 rows and (m, l)
    size_t off_part_o = 0, off_part_ml = 0;       // the prefix pieces' partials
    size_t metadata = 0, bytes = 0;
};

struct PrefixGroup {
    std::vector<int32_t> members;   // sequences, ascending
    int32_t pages = 0;              // shared leading pages
};

}  // namespace pd

struct pd_prefix_plan {
    pd_layout layout{};
    pd_dtype dtype = PD_FLOAT16;
    int32_t device = -1;
    int64_t width = 0;
    int32_t group = 0;              // G = Hq / Hkv
    int32_t tile_rows = 0;          // query rows of one prefix tile
    int32_t slots = 0;              // partial slots (tile pieces)
    int32_t step_pages = 0;         // pages of one step of the prefix kernel
    int64_t item_steps = 1;         // steps of the longest work item (choose_pieces)
    int32_t suffix_ctas = 0;        // SMs left to the suffix's decode beside the prefix kernel, 0: it runs behind it
    int32_t merge_ways = 1;         // thread sets that share a row's pieces in the merge
    bool dynamic = false;
    bool suffix_empty = false;      // no sequence has pages past its prefix: nothing for the decode kernel
    std::vector<pd::PrefixGroup> groups;
    int32_t item_words = 0;
    std::vector<int32_t> items;     // item_words per work item, see PrefixArgs::items
    std::vector<int32_t> seqs;      // 8 per sequence, see PrefixArgs::seqs
    std::vector<int32_t> tiles;     // 2 per row tile: first slot, pieces
    pd_plan *suffix = nullptr;
    pd::PrefixImage image;
    std::vector<uint8_t> host_image;
    uint8_t *dev = nullptr;

    ~pd_prefix_plan() { delete suffix; }
};

namespace pd {

// Groups of sequences whose leading pages are the same.  A candidate is all
// sequences that start with some pages; disjoint candidates are chosen so that
// the page reads saved are the most.
void find_prefix_groups(const pd_layout &layout, const int32_t *table, int64_t width, const int32_t *lengths,
                        std::vector<PrefixGroup> &groups);

// Check the groups against the table and lengths.
pd_status check_prefix_groups(const pd_layout &layout, const int32_t *table, int64_t width, const int32_t *lengths,
                              const std::vector<PrefixGroup> &groups);

// What follows from the layout and the type alone (group, item_words, step_pages).
void set_shape(pd_prefix_plan &p);

// Of the found groups, those that an estimate of the call's time says are worth it:
// the ones that save the most page reads, as long as more of them make the call
// shorter (all, some or none).  suffix_pages: the pages outside of all groups.
void keep_paying_groups(pd_prefix_plan &p, int64_t suffix_pages, int32_t sm_count);

// How the groups' work is cut (tile_rows, item_steps) and which SMs the suffix gets
// (suffix_ctas), from the groups and the pages outside of them.
void choose_pieces(pd_prefix_plan &p, int64_t suffix_pages, int32_t sm_count);

// Lay the groups' work out and build the device image; the suffix plan is set.
// span: the tokens that each sequence is planned for (max_lengths, or lengths).
pd_status build_prefix_plan(pd_prefix_plan &p, const int32_t *table, const int32_t *lengths, const int32_t *span,
                            int32_t sm_count);

}  // namespace pd
