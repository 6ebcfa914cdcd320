// pd_prefix.cpp — plan builder of shared-prefix decode attention.
//
// Sequences that share leading pages form a group.  For each KV head the
// group's queries are one matrix of n * G rows (n members, G query heads per
// KV head) against the prefix, read once; each sequence's remaining pages are
// left to a decode plan that starts behind the prefix.
#include "pd_prefix.hpp"

#include <algorithm>
#include <cstring>
#include <numeric>

namespace pd {

namespace {
size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
}  // namespace

void find_prefix_groups(const pd_layout &layout, const int32_t *table, int64_t width, const int32_t *lengths,
                        std::vector<PrefixGroup> &groups) {
    groups.clear();
    const int B = layout.batch;
    const auto full = [&](int b) { return int64_t(lengths[b]) / layout.page_size; };   // whole live pages
    const auto common = [&](int a, int b) {
        const int32_t *x = table + a * width, *y = table + b * width;
        const int64_t n = std::min(full(a), full(b));
        return int64_t(std::mismatch(x, x + n, y).first - x);
    };
    std::vector<int32_t> order(B);
    std::iota(order.begin(), order.end(), 0);
    std::sort(order.begin(), order.end(), [&](int a, int b) {
        const int32_t *x = table + a * width, *y = table + b * width;
        const int64_t na = full(a), nb = full(b);
        const auto d = std::mismatch(x, x + std::min(na, nb), y);
        if (d.first != x + std::min(na, nb)) return *d.first < *d.second;
        return na != nb ? na < nb : a < b;
    });
    // Runs of neighbours with common leading pages form a tree (a run is inside
    // another or apart from it).  Bottom up, a run is taken as one group where
    // that saves more than the best choice inside it.
    struct Run {
        int64_t pages, saved;         // common pages; the most that can be saved inside
        int left, right;
        bool whole;                   // taken as one group
        std::vector<int> inside;
    };
    std::vector<Run> runs;
    std::vector<int> open;            // runs still growing, each inside the one before
    std::vector<int> top;             // closed runs inside no other
    for (int k = 1; k <= B; ++k) {
        const int64_t pages = k < B ? common(order[k - 1], order[k]) : 0;
        int left = k - 1, closed = -1;
        while (!open.empty() && runs[open.back()].pages > pages) {
            const int id = open.back();
            open.pop_back();
            Run &r = runs[id];
            r.right = k - 1;
            if (closed >= 0) {
                r.inside.push_back(closed);
                r.saved += runs[closed].saved;
            }
            const int64_t own = int64_t(r.right - r.left) * r.pages;
            r.whole = own >= r.saved && own > 0;
            if (r.whole) r.saved = own;
            left = r.left;
            closed = id;
        }
        if (pages > 0 && (open.empty() || runs[open.back()].pages < pages)) {
            runs.push_back(Run{pages, 0, left, k, false, {}});
            open.push_back(int(runs.size()) - 1);
        }
        if (closed >= 0) {
            if (open.empty()) {
                top.push_back(closed);
            } else {
                runs[open.back()].inside.push_back(closed);
                runs[open.back()].saved += runs[closed].saved;
            }
        }
    }
    while (!top.empty()) {
        const int id = top.back();
        top.pop_back();
        const Run &r = runs[id];
        if (!r.whole) {
            top.insert(top.end(), r.inside.begin(), r.inside.end());
            continue;
        }
        PrefixGroup g;
        g.pages = int32_t(r.pages);
        g.members.assign(order.begin() + r.left, order.begin() + r.right + 1);
        std::sort(g.members.begin(), g.members.end());
        groups.push_back(std::move(g));
    }
    std::sort(groups.begin(), groups.end(),
              [](const PrefixGroup &a, const PrefixGroup &b) { return a.members[0] < b.members[0]; });
}

pd_status check_prefix_groups(const pd_layout &layout, const int32_t *table, int64_t width, const int32_t *lengths,
                              const std::vector<PrefixGroup> &groups) {
    std::vector<char> seen(layout.batch, 0);
    for (const PrefixGroup &g : groups) {
        if (g.members.empty()) return fail(PD_ERR_VALUE, "a prefix group needs at least one sequence");
        if (g.pages < 1 || g.pages > width) return fail(PD_ERR_VALUE, "a prefix must have 1 .. table width pages");
        for (const int32_t b : g.members) {
            if (b < 0 || b >= layout.batch) return fail(PD_ERR_VALUE, "prefix group names a sequence outside the batch");
            if (seen[b]) return fail(PD_ERR_VALUE, "a sequence can be in one prefix group only");
            seen[b] = 1;
            if (int64_t(lengths[b]) < int64_t(g.pages) * layout.page_size)
                return fail(PD_ERR_VALUE, "a prefix is longer than one of its sequences");
            if (!std::equal(table + b * width, table + b * width + g.pages, table + g.members[0] * width))
                return fail(PD_ERR_VALUE, "the sequences of a prefix group must share its pages");
        }
    }
    return PD_OK;
}

namespace {

// FP32 (CUDA cores): tiles of 16 rows, or of 64 where a group has more than 16
// (32 rows: half a tile of 64 runs at 13 TFLOP/s, two of 16 at 10),
// 32-token steps, about as many CTAs as are resident at once.
struct SimtPlan {
    static constexpr int64_t step_tokens = 32;
};

// FP16 (tcgen05): tiles of 128 rows, 64-token steps, one CTA per SM with two
// streams (see pd_prefix_mma.cuh).
struct MmaShape {
    static constexpr int64_t rows = 128, step_tokens = 64;
    // In steps (0.9 us): start and end of a CTA (launch, first loads, rows out); the merge kernel; and
    // the partials' way through memory, FP32 values a step.
    static constexpr int64_t overhead_steps = 7, merge_steps = 3, values_per_step = 20 * 128 * 128;
};

}  // namespace

pd_status build_prefix_plan(pd_prefix_plan &p, const int32_t *table, const int32_t *lengths, int32_t sm_count) {
    const pd_layout &L = p.layout;
    const int D = L.head_dim;
    const bool mma = p.dtype == PD_FLOAT16;
    p.group = L.query_heads / L.kv_heads;
    int64_t most_rows = 0;
    for (const PrefixGroup &g : p.groups) most_rows = std::max(most_rows, int64_t(g.members.size()) * p.group);
    p.tile_rows = int32_t(mma ? MmaShape::rows : most_rows > 16 ? 64 : 16);
    const int64_t simt_ctas_per_sm = p.tile_rows == 16 ? 4 : 2;
    p.item_words = mma ? 16 : 8;
    const int64_t step_pages = (mma ? MmaShape::step_tokens : SimtPlan::step_tokens) / L.page_size;
    const auto tiles_of = [&](const PrefixGroup &g) {
        return (int64_t(g.members.size()) * p.group + p.tile_rows - 1) / p.tile_rows;
    };
    const auto steps_of = [&](const PrefixGroup &g) { return (g.pages + step_pages - 1) / step_pages; };
    // FP16: what finishes first when the CTAs run in waves of one per SM and each
    // costs its steps and the fixed overhead: a CTA per pair of row tiles or per tile
    // that sees the whole prefix and writes the output (direct), or any number of
    // pieces that leave partials for the merge kernel.
    int64_t item_steps = 1;
    bool pair_tiles = true;
    p.direct = false;
    if (mma) {
        int64_t most = 1, pairs = 0, tiles = 0, best = INT64_MAX;
        for (const PrefixGroup &g : p.groups) {
            most = std::max<int64_t>(most, steps_of(g));
            pairs += L.kv_heads * ((tiles_of(g) + 1) / 2);
            tiles += L.kv_heads * tiles_of(g);
        }
        int64_t values = 0;     // of the partials
        const auto items = [&](int64_t steps) {     // CTAs of so many steps
            int64_t n = 0;
            values = 0;
            for (const PrefixGroup &g : p.groups) {
                const int64_t t = tiles_of(g), s = steps_of(g), pieces = (s + steps - 1) / steps;
                n += L.kv_heads * (t / 2 * pieces + t % 2 * ((pieces + 1) / 2));
                values += L.query_heads * int64_t(g.members.size()) * D * pieces;
            }
            return n;
        };
        const auto waves = [&](int64_t ctas) { return (ctas + sm_count - 1) / sm_count; };
        for (int64_t steps = 1; steps <= most; ++steps) {
            const int64_t n = items(steps);
            const int64_t cost = waves(n) * (MmaShape::overhead_steps + steps) + MmaShape::merge_steps +
                                 values / MmaShape::values_per_step;
            if (cost < best) best = cost, item_steps = steps;
        }
        const int64_t by_pair = waves(pairs) * (MmaShape::overhead_steps + most);
        const int64_t by_tile = waves(tiles) * (MmaShape::overhead_steps + (most + 1) / 2);
        if (by_pair <= best || by_tile <= best) {
            p.direct = !p.groups.empty();
            pair_tiles = by_pair <= by_tile;
            item_steps = most;
        }
    } else {
        int64_t work = 0;
        for (const PrefixGroup &g : p.groups) work += L.kv_heads * tiles_of(g) * steps_of(g);
        item_steps = std::max<int64_t>(1, work / std::max<int64_t>(1, simt_ctas_per_sm * sm_count));
    }
    p.seqs.assign(size_t(L.batch) * 8, 0);
    for (int b = 0; b < L.batch; ++b) p.seqs[size_t(b) * 8] = -1;
    p.items.clear();
    p.tiles.clear();
    std::vector<int32_t> members, pages;
    int64_t slots = 0, count = 0;
    for (const PrefixGroup &g : p.groups) {
        const int64_t ntiles = tiles_of(g), steps = steps_of(g);
        count += L.kv_heads * ntiles * steps;
        if (count > INT32_MAX / 1024) return fail(PD_ERR_VALUE, "too many prefix tiles");
        for (size_t j = 0; j < g.members.size(); ++j) {
            int32_t *s = &p.seqs[size_t(g.members[j]) * 8];
            s[0] = int32_t(j);
            s[1] = int32_t(p.tiles.size() / 2);
            s[2] = int32_t(ntiles);
            s[3] = int32_t(pages.size());
            s[4] = g.pages;
        }
        const int32_t m0 = int32_t(members.size()), n = int32_t(g.members.size()), pg = int32_t(pages.size());
        // piece c of `pieces`: whole steps, as even as they come
        const auto bound = [&](int64_t c, int64_t pieces) {
            return int32_t(std::min<int64_t>(g.pages, c * steps / pieces * step_pages));
        };
        for (int h = 0; h < L.kv_heads; ++h) {
            for (int64_t t = 0; t < ntiles; ++t) {
                const bool paired = mma && pair_tiles && (t ^ 1) < ntiles;
                const bool split = mma && !paired && steps > 1;
                int64_t pieces = (steps + item_steps - 1) / item_steps;
                if (split) pieces = (steps + 2 * item_steps - 1) / (2 * item_steps) * 2;
                pieces = std::min(pieces, steps);
                p.tiles.insert(p.tiles.end(), {int32_t(slots), int32_t(pieces)});
                const int32_t slot = int32_t(slots), tile = int32_t(t);
                slots += pieces;
                if (!mma) {
                    for (int64_t c = 0; c < pieces; ++c)
                        p.items.insert(p.items.end(), {m0, n, h, tile, pg, bound(c, pieces), bound(c + 1, pieces),
                                                       int32_t(slot + c)});
                } else if (!paired) {
                    // two neighbouring pieces of one tile, the longer one first
                    for (int64_t c = 0; c < pieces; c += 2) {
                        int32_t x[4] = {bound(c, pieces), bound(c + 1, pieces), 0, 0};
                        int32_t sx = int32_t(slot + c), sy = sx;
                        if (c + 1 < pieces) {
                            x[2] = x[1], x[3] = bound(c + 2, pieces), sy = sx + 1;
                            if (x[3] - x[2] > x[1] - x[0]) {
                                std::swap(x[0], x[2]);
                                std::swap(x[1], x[3]);
                                std::swap(sx, sy);
                            }
                        }
                        p.items.insert(p.items.end(), {m0, n, h, 0, pg, g.pages, 0, 0, tile, x[0], x[1], sx, tile, x[2],
                                                       x[3], sy});
                    }
                } else if (t % 2) {
                    // both tiles of a pair have the same pieces; this one's slots follow the other's
                    for (int64_t c = 0; c < pieces; ++c)
                        p.items.insert(p.items.end(),
                                       {m0, n, h, 1, pg, g.pages, 0, 0, tile - 1, bound(c, pieces), bound(c + 1, pieces),
                                        int32_t(slot - pieces + c), tile, bound(c, pieces), bound(c + 1, pieces),
                                        int32_t(slot + c)});
                }
            }
        }
        members.insert(members.end(), g.members.begin(), g.members.end());
        const int32_t *row = table + int64_t(g.members[0]) * p.width;
        pages.insert(pages.end(), row, row + g.pages);
    }
    if (p.direct) {
        // every row is written by the prefix kernel: sequences of no group, four to a CTA
        slots = 0;
        const size_t first = members.size();
        for (int b = 0; b < L.batch; ++b)
            if (p.seqs[size_t(b) * 8] < 0) members.push_back(b);
        for (size_t at = first; at < members.size(); at += 4) {
            p.items.insert(p.items.end(), {int32_t(at), int32_t(std::min<size_t>(4, members.size() - at)), 0, 2});
            p.items.insert(p.items.end(), 12, 0);
        }
    }
    p.slots = int32_t(slots);
    // Merge: at most four pieces (one batch of loads) per thread set, while the
    // sets' threads still fit the device at once (2048 per SM).
    int32_t most_pieces = 1;
    for (size_t t = 1; t < p.tiles.size(); t += 2) most_pieces = std::max(most_pieces, p.tiles[t]);
    p.merge_ways = 1;
    while (p.merge_ways < 8 && p.merge_ways * 4 < most_pieces &&
           int64_t(L.batch) * L.query_heads * (D / 8) * p.merge_ways * 2 <= int64_t(sm_count) * 2048)
        p.merge_ways *= 2;

    PrefixImage &im = p.image;
    size_t off = 0;
    im.off_error = off;    off = align256(off + 4);
    im.off_items = off;    off = align256(off + p.items.size() * 4);
    im.off_seqs = off;     off = align256(off + p.seqs.size() * 4);
    im.off_tiles = off;    off = align256(off + p.tiles.size() * 4);
    im.off_members = off;  off = align256(off + members.size() * 4);
    im.off_pages = off;    off = align256(off + pages.size() * 4);
    im.off_lengths = off;  off = align256(off + size_t(L.batch) * 4);
    im.metadata = off;
    im.off_suffix = off;   off = align256(off + p.suffix->image.bytes);
    im.off_rows = off;     off = align256(off + size_t(L.batch) * L.query_heads * D * 4);
    im.off_stats = off;    off = align256(off + size_t(L.batch) * L.query_heads * 8);
    im.off_part_o = off;   off = align256(off + size_t(slots) * p.tile_rows * D * 4);
    im.off_part_ml = off;  off = align256(off + size_t(slots) * p.tile_rows * 8);
    im.bytes = off;
    p.host_image.assign(im.metadata, 0);
    const auto put = [&](size_t at, const void *data, size_t bytes) {
        if (bytes) std::memcpy(p.host_image.data() + at, data, bytes);
    };
    put(im.off_items, p.items.data(), p.items.size() * 4);
    put(im.off_seqs, p.seqs.data(), p.seqs.size() * 4);
    put(im.off_tiles, p.tiles.data(), p.tiles.size() * 4);
    put(im.off_members, members.data(), members.size() * 4);
    put(im.off_pages, pages.data(), pages.size() * 4);
    put(im.off_lengths, lengths, size_t(L.batch) * 4);
    return PD_OK;
}

}  // namespace pd
