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
                        int64_t overhead_pages, std::vector<PrefixGroup> &groups) {
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
            const int64_t own = int64_t(r.right - r.left) * r.pages - overhead_pages;
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

pd_status build_prefix_plan(pd_prefix_plan &p, const int32_t *table, const int32_t *lengths, int32_t sm_count) {
    const pd_layout &L = p.layout;
    const int D = L.head_dim;
    p.group = L.query_heads / L.kv_heads;
    p.tile_rows = 16;
    const int64_t step_pages = std::max(1, 32 / L.page_size);
    int64_t tiles = 0;
    for (const PrefixGroup &g : p.groups)
        tiles += int64_t(L.kv_heads) * ((int64_t(g.members.size()) * p.group + p.tile_rows - 1) / p.tile_rows);
    p.seqs.assign(size_t(L.batch) * 4, 0);
    for (int b = 0; b < L.batch; ++b) p.seqs[size_t(b) * 4] = -1;
    p.items.clear();
    std::vector<int32_t> members, pages;
    int64_t slots = 0;
    for (const PrefixGroup &g : p.groups) {
        const int64_t rows = int64_t(g.members.size()) * p.group;
        const int64_t ntiles = (rows + p.tile_rows - 1) / p.tile_rows;
        const int64_t steps = (g.pages + step_pages - 1) / step_pages;
        const int64_t pieces = std::min(steps, std::max<int64_t>(1, (4 * int64_t(sm_count) + tiles - 1) / tiles));
        for (size_t j = 0; j < g.members.size(); ++j) {
            int32_t *s = &p.seqs[size_t(g.members[j]) * 4];
            s[0] = int32_t(j);
            s[1] = int32_t(slots);
            s[2] = int32_t(ntiles);
            s[3] = int32_t(pieces);
        }
        if (slots + int64_t(L.kv_heads) * ntiles * pieces > INT32_MAX / 256)
            return fail(PD_ERR_VALUE, "too many prefix tiles");
        for (int h = 0; h < L.kv_heads; ++h)
            for (int64_t t = 0; t < ntiles; ++t)
                for (int64_t c = 0; c < pieces; ++c, ++slots) {
                    const int64_t first = c * steps / pieces * step_pages;
                    const int64_t end = std::min<int64_t>(g.pages, (c + 1) * steps / pieces * step_pages);
                    p.items.insert(p.items.end(),
                                   {int32_t(members.size()), int32_t(g.members.size()), h, int32_t(t),
                                    int32_t(pages.size()), int32_t(first), int32_t(end), int32_t(slots)});
                }
        members.insert(members.end(), g.members.begin(), g.members.end());
        const int32_t *row = table + int64_t(g.members[0]) * p.width;
        pages.insert(pages.end(), row, row + g.pages);
    }
    p.slots = int32_t(slots);

    PrefixImage &im = p.image;
    size_t off = 0;
    im.off_error = off;    off = align256(off + 4);
    im.off_items = off;    off = align256(off + p.items.size() * 4);
    im.off_seqs = off;     off = align256(off + p.seqs.size() * 4);
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
    put(im.off_members, members.data(), members.size() * 4);
    put(im.off_pages, pages.data(), pages.size() * 4);
    put(im.off_lengths, lengths, size_t(L.batch) * 4);
    return PD_OK;
}

}  // namespace pd
