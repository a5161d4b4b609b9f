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

// A work-group (one per CU) walks its keys 128 at a time, a step.  Of a few cut
// lengths the one whose estimate is least is taken: the longest work-group or the
// CUs' share of the steps, a start for each work-group, half a work-group's time
// for the last round, and the merge's launch and traffic.
inline std::vector<int> tree_cuts(const std::vector<TreeLoad> &load, int kvh, int cus, int tile_rows, int hd,
                                  bool fine) {
    const auto steps = [](int len) { return (len + 127) / 128; };
    int64_t all = 0;
    int most = 1;
    for (const TreeLoad &l : load) {
        all += (int64_t)l.tiles * kvh * steps(l.len);
        most = std::max(most, steps(l.len));
    }
    // us: a step, a work-group's start, the merge's launch, a partial row
    const double step = 0.6 + hd / 128.0 * 1.0, start = 3.0, launch = 5.0, row = hd * 8 / 4.0e6;
    (void)tile_rows;
    (void)fine;
    double best = 0.0;
    int best_len = most;
    for (int k = 0; k <= 8; k++) {
        static const double share[] = {0, 0.25, 0.34, 0.5, 0.67, 1.0, 1.34, 2.0, 4.0};
        const int at = k == 0 ? most
                              : (int)std::min<double>(most, std::max(1.0, std::ceil(all * share[k] / cus)));
        int64_t wgs = 0, parts = 0;
        for (const TreeLoad &l : load) {
            const int n = (steps(l.len) + at - 1) / at;
            wgs += (int64_t)l.tiles * kvh * n;
            if (n > 1) parts += (int64_t)l.rows * kvh * n;
        }
        const double share_us = (all * step + wgs * start) / cus;
        const double last = wgs > cus ? 0.5 * (all * step / wgs + start) : 0.0;
        const double us = std::max(at * step + start, share_us + last) + (parts ? launch + parts * row : 0.0);
        if (k == 0 || us < best) {
            best = us;
            best_len = at;
        }
    }
    std::vector<int> n(load.size());
    for (size_t i = 0; i < load.size(); i++) n[i] = (steps(load[i].len) + best_len - 1) / best_len;
    return n;
}

}  // namespace rlx
