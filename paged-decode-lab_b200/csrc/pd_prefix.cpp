// pd_prefix.cpp — plan builder of shared-prefix decode attention.
//
// Sequences that share leading pages form a group.  For each KV head the
// group's queries are one matrix of n * G rows (n members, G query heads per
// KV head) against the prefix, read once; each sequence's remaining pages are
// left to a decode plan that starts behind the prefix.
#include "pd_prefix.hpp"

#include <algorithm>
#include <cstring>
#include <map>
#include <numeric>
#include <set>
#include <utility>

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
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Groups of one shape: `count` of them, each with so many members and shared pages.
struct GroupShape {
    int64_t members, pages, count;
    int64_t saved() const { return (members - 1) * pages; }
};

// The shapes of some groups, those of which one saves the most first.
std::vector<GroupShape> shapes_of(const std::vector<PrefixGroup> &groups) {
    std::map<std::pair<int64_t, int64_t>, int64_t> counts;
    for (const PrefixGroup &g : groups) ++counts[{int64_t(g.members.size()), int64_t(g.pages)}];
    std::vector<GroupShape> shapes;
    for (const auto &c : counts) shapes.push_back({c.first.first, c.first.second, c.second});
    std::stable_sort(shapes.begin(), shapes.end(),
                     [](const GroupShape &a, const GroupShape &b) { return a.saved() > b.saved(); });
    return shapes;
}

struct PrefixCut {
    double us = 0;                  // estimated time of a call
    int64_t item_steps = 1;
    int32_t suffix_ctas = 0;
};

int32_t tile_rows_for(bool mma, int64_t most_rows) { return int32_t(mma ? MmaShape::rows : most_rows > 16 ? 64 : 16); }

// The decode kernel reads copies of pages that others read too from L2 (B/us, measured on a B200).
double copy_rate(const pd_prefix_plan &p) { return p.dtype != PD_FLOAT16 ? 9e6 : p.group > 16 ? 7.5e6 : 14e6; }

double page_bytes_of(const pd_prefix_plan &p) {
    return (p.dtype == PD_FLOAT16 ? 4.0 : 8.0) * p.layout.page_size * p.layout.kv_heads * p.layout.head_dim;
}

// How these groups' work is best cut, and what a call then takes; the decode kernel has
// suffix_pages beside them, and `copies` reads of pages that it could have shared.
PrefixCut cut_of(const pd_prefix_plan &p, const std::vector<GroupShape> &shapes, int64_t suffix_pages, int64_t copies,
                 int32_t sm_count) {
    const pd_layout &L = p.layout;
    const bool mma = p.dtype == PD_FLOAT16;
    const double page_bytes = page_bytes_of(p);
    int64_t most_rows = 0, shared_pages = 0;
    for (const GroupShape &g : shapes) {
        most_rows = std::max(most_rows, g.members * p.group);
        shared_pages += g.count * g.pages;
    }
    const int64_t rows = tile_rows_for(mma, most_rows);
    const auto tiles_of = [&](const GroupShape &g) { return ceil_div(g.members * p.group, rows); };
    const auto steps_of = [&](const GroupShape &g) { return ceil_div(g.pages, p.step_pages); };
    PrefixCut cut;
    if (!mma) {
        int64_t work = 0;
        double flops = 0;
        for (const GroupShape &g : shapes) {
            work += g.count * L.kv_heads * tiles_of(g) * steps_of(g);
            flops += 4.0 * L.kv_heads * double(g.count * tiles_of(g) * rows) * g.pages * L.page_size * L.head_dim;
        }
        cut.item_steps = std::max<int64_t>(1, work / std::max<int64_t>(1, (rows == 16 ? 4 : 2) * sm_count));
        cut.us = 22 + suffix_pages * page_bytes / 5.5e6 + copies * page_bytes / copy_rate(p) +
                 std::max(shared_pages * page_bytes / 5e6, flops / (rows == 16 ? 15e6 : 23e6));
        return cut;
    }
    // Estimated times in us, fitted to whole calls on a B200.  A CTA of the prefix kernel takes 7 steps
    // for its start and end and 0.94 a step; the prefix's bytes come at 6.2e6 B/us at best.  The decode kernel
    // takes 9 and its bytes at 5.5e6 B/us, or 48e3 per SM, and 3 for each sequence on an SM.  The merge takes
    // 3 and 350e3 FP32 values of partials a us.  The two kernels run beside each other where both fit and that is
    // sooner done.  (256 sequences of 64:8 heads, 4096 shared and 512 own tokens each: 64 CTAs beside 84 took
    // 136 us, 128 and then 148 174, 128 beside 20 364.)
    const double segments = double(L.batch) * ceil_div(L.kv_heads, 8) * ceil_div(p.group, 32);
    const auto suffix_us = [&](int64_t sms) {
        if (suffix_pages + copies == 0) return 0.0;
        return 9 + suffix_pages * page_bytes / std::min(5.5e6, 48e3 * double(sms)) +
               copies * page_bytes / (copy_rate(p) * double(sms) / sm_count) + 3 * segments / double(sms);
    };
    // the shortest item for every number of pieces of the first (largest) few shapes
    std::set<int64_t> lengths;
    for (size_t i = 0; i < std::min<size_t>(shapes.size(), 8); ++i)
        for (int64_t steps = 1, all = steps_of(shapes[i]); steps <= all;) {
            lengths.insert(steps);
            const int64_t pieces = ceil_div(all, steps);
            if (pieces == 1) break;
            steps = ceil_div(all, pieces - 1);
        }
    cut.us = 1e300;
    for (const int64_t steps : lengths) {
        int64_t ctas = 0, total = 0, longest = 0, values = 0;      // total, longest: in steps
        for (const GroupShape &g : shapes) {
            const int64_t tiles = tiles_of(g), pieces = ceil_div(steps_of(g), steps);
            const int64_t own = L.kv_heads * g.count * (tiles / 2 * pieces + tiles % 2 * ceil_div(pieces, 2));
            const int64_t length = 7 + ceil_div(steps_of(g), pieces);
            ctas += own;
            total += own * length;
            longest = std::max(longest, length);
            values += L.query_heads * g.count * g.members * L.head_dim * pieces;
        }
        // waves of CTAs of the mean length, but no less than the longest
        const double prefix = std::max(0.94 * std::max(double(longest), double(ceil_div(ctas, sm_count)) * total / ctas),
                                       7 + shared_pages * page_bytes / 6.2e6);
        const double behind = prefix + suffix_us(sm_count);
        const double beside = suffix_pages + copies > 0 && ctas < sm_count ? std::max(prefix, suffix_us(sm_count - ctas))
                                                                           : behind;
        const double us = 4 + std::min(beside, behind) + 3 + double(values) / 350e3;
        if (us < cut.us) cut = PrefixCut{us, steps, beside < behind ? int32_t(sm_count - ctas) : 0};
    }
    return cut;
}

}  // namespace

void keep_paying_groups(pd_prefix_plan &p, int64_t suffix_pages, int32_t sm_count) {
    const std::vector<GroupShape> shapes = shapes_of(p.groups);
    int64_t copies = 0;             // of the shapes that are not used
    for (const GroupShape &g : shapes) copies += g.count * g.members * g.pages;
    // without any: the decode kernel alone, 12 us and its bytes
    const double page_bytes = page_bytes_of(p);
    double best = 12 + suffix_pages * page_bytes / 5.5e6 + copies * page_bytes / copy_rate(p);
    size_t kept = 0;
    // the first k shapes, for at most some 64 values of k
    std::vector<GroupShape> used;
    const size_t stride = std::max<size_t>(1, shapes.size() / 64);
    for (size_t k = 1; k <= shapes.size(); ++k) {
        const GroupShape &g = shapes[k - 1];
        used.push_back(g);
        copies -= g.count * g.members * g.pages;
        if (k > 16 && k % stride && k < shapes.size()) continue;
        const double us = cut_of(p, used, suffix_pages, copies, sm_count).us;
        if (us < best) best = us, kept = k;
    }
    std::set<std::pair<int64_t, int64_t>> keep;
    for (size_t k = 0; k < kept; ++k) keep.insert({shapes[k].members, shapes[k].pages});
    p.groups.erase(std::remove_if(p.groups.begin(), p.groups.end(),
                                  [&](const PrefixGroup &g) {
                                      return !keep.count({int64_t(g.members.size()), int64_t(g.pages)});
                                  }),
                   p.groups.end());
}

void choose_pieces(pd_prefix_plan &p, int64_t suffix_pages, int32_t sm_count) {
    int64_t most_rows = 0;
    for (const PrefixGroup &g : p.groups) most_rows = std::max(most_rows, int64_t(g.members.size()) * p.group);
    p.tile_rows = tile_rows_for(p.dtype == PD_FLOAT16, most_rows);
    p.item_steps = 1;
    p.suffix_ctas = 0;
    if (p.groups.empty()) return;
    const PrefixCut cut = cut_of(p, shapes_of(p.groups), suffix_pages, 0, sm_count);
    p.item_steps = cut.item_steps;
    p.suffix_ctas = cut.suffix_ctas;
}

void set_shape(pd_prefix_plan &p) {
    const bool mma = p.dtype == PD_FLOAT16;
    p.group = p.layout.query_heads / p.layout.kv_heads;
    p.item_words = mma ? 16 : 8;
    p.step_pages = int32_t((mma ? MmaShape::step_tokens : SimtPlan::step_tokens) / p.layout.page_size);
}

pd_status build_prefix_plan(pd_prefix_plan &p, const int32_t *table, const int32_t *lengths, const int32_t *span,
                            int32_t sm_count) {
    const pd_layout &L = p.layout;
    const int D = L.head_dim;
    const bool mma = p.dtype == PD_FLOAT16;
    const int64_t item_steps = p.item_steps;
    const int64_t step_pages = p.step_pages;
    const auto tiles_of = [&](const PrefixGroup &g) { return ceil_div(int64_t(g.members.size()) * p.group, p.tile_rows); };
    const auto steps_of = [&](const PrefixGroup &g) { return ceil_div(g.pages, step_pages); };
    p.seqs.assign(size_t(L.batch) * 8, 0);
    for (int b = 0; b < L.batch; ++b) {
        p.seqs[size_t(b) * 8] = -1;
        p.seqs[size_t(b) * 8 + 5] = span[b];
    }
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
        // piece c of `pieces`: whole steps, as even as they come (prefix_merge_kernel has the same cut)
        const auto bound = [&](int64_t c, int64_t pieces) {
            return int32_t(std::min<int64_t>(g.pages, c * steps / pieces * step_pages));
        };
        for (int h = 0; h < L.kv_heads; ++h) {
            for (int64_t t = 0; t < ntiles; ++t) {
                const bool paired = mma && (t ^ 1) < ntiles;
                const bool split = mma && !paired && steps > 1;
                int64_t pieces = ceil_div(steps, item_steps);
                if (split) pieces = std::min(steps, ceil_div(pieces, 2) * 2);
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
                        p.items.insert(p.items.end(), {m0, n, h, 0, pg, 0, 0, 0, tile, x[0], x[1], sx, tile, x[2],
                                                       x[3], sy});
                    }
                } else if (t % 2) {
                    // both tiles of a pair have the same pieces; this one's slots follow the other's
                    for (int64_t c = 0; c < pieces; ++c)
                        p.items.insert(p.items.end(),
                                       {m0, n, h, 1, pg, 0, 0, 0, tile - 1, bound(c, pieces), bound(c + 1, pieces),
                                        int32_t(slot - pieces + c), tile, bound(c, pieces), bound(c + 1, pieces),
                                        int32_t(slot + c)});
                }
            }
        }
        members.insert(members.end(), g.members.begin(), g.members.end());
        const int32_t *row = table + int64_t(g.members[0]) * p.width;
        pages.insert(pages.end(), row, row + g.pages);
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
