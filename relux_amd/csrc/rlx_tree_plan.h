// Cuts along the keys of a tree attention call.  Host code.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <vector>

namespace rlx {

// One sequence: live tokens, tiles of query rows a kv head, query rows a kv head.
struct TreeLoad {
    int len, tiles, rows;
};

// A work-group (one per CU, two of 64 rows) walks its keys 128 at a time, a step.
// For one round of them, two, three ... the shortest cut is taken whose work-groups fit them, so
// that the rounds end together whatever the mix of lengths; of these, and of whole
// sequences, the one whose estimate is least: between the CUs' share of the work
// and the rounds' longest work-groups, with a start for each and the merge's launch
// and traffic.
inline std::vector<int> tree_cuts(const std::vector<TreeLoad> &load, int kvh, int cus, int tile_rows, int hd,
                                  bool fine) {
    const auto steps = [](int len) { return (len + 127) / 128; };
    const int per_cu = tile_rows == 64 && hd <= 128 ? 2 : 1, slots = per_cu * cus;
    int64_t all = 0, keys = 0;
    int most = 1;
    for (const TreeLoad &l : load) {
        all += (int64_t)l.tiles * kvh * steps(l.len);
        keys += (int64_t)kvh * steps(l.len);
        most = std::max(most, steps(l.len));
    }
    const auto count = [&](int at, int64_t *parts) {
        int64_t wgs = 0;
        *parts = 0;
        for (const TreeLoad &l : load) {
            const int n = (steps(l.len) + at - 1) / at;
            wgs += (int64_t)l.tiles * kvh * n;
            if (n > 1) *parts += (int64_t)l.rows * kvh * n;
        }
        return wgs;
    };
    // us: a step (its share of HBM where tiles do not share the keys, or the
    // arithmetic), a work-group's start, the merge's launch, a partial row
    const double wide = hd / 128.0;
    const double mem = 2.5 * wide * keys / all;
    const double math = wide * (tile_rows <= 64 ? 0.8 : tile_rows <= 128 ? 1.6 : 2.8) * (fine ? 2.0 : 1.0);
    const double step = per_cu * std::max(mem, math), start = 3.0, launch = 5.0, row = hd * 8 / 4.0e6;
    double best = 0.0;
    int best_at = most, last = 0;
    for (int k = 0; k <= 8; k++) {
        int at = most;
        int64_t parts, wgs = count(most, &parts);
        if (k > 0) {  // the least cut of at most k rounds
            if (wgs > (int64_t)k * slots) continue;
            int lo = 1, hi = most;
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (count(mid, &parts) <= (int64_t)k * slots)
                    hi = mid;
                else
                    lo = mid + 1;
            }
            at = lo;
            if (at == last) continue;
            wgs = count(at, &parts);
        }
        last = at;
        const double rounds = (double)((wgs + slots - 1) / slots) * (at * step + start);
        const double share = std::max(at * step + start, (all * step + wgs * start) / slots);
        const double us = 0.5 * (rounds + share) + (parts ? launch + parts * row : 0.0);
        if (best == 0.0 || us < best) {
            best = us;
            best_at = at;
        }
    }
    std::vector<int> n(load.size());
    for (size_t i = 0; i < load.size(); i++) n[i] = (steps(load[i].len) + best_at - 1) / best_at;
    return n;
}

}  // namespace rlx
