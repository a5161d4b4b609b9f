// Tiles and cuts of a tree attention call.  Host code.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <vector>

namespace rlx {

// One sequence: live tokens, query rows a kv head.
struct TreeLoad {
    int len, rows;
};
struct TreePlan {
    int tile = 16;          // query rows of a work-group
    std::vector<int> cuts;  // of each sequence's keys
};

// Whether a tile has a kernel: 16 and 32 rows at every stored head dim (256: 16),
// more from 64 dims on (256: 64; f32: 128), as a wave's registers allow.
inline bool tree_has_tile(int tile, int hd, bool fine) {
    if (tile == 16) return true;
    if (tile == 32) return hd < 256;
    if (hd < 64) return false;
    return tile == 64 || (hd < 256 && (tile == 128 || !fine));
}

// A work-group walks its keys 128 at a time, a step; a tile of more rows reads the
// keys less often, and takes longer to start and to end.  Estimates in us, for a
// head dim of 128 (steps scale with it; f32 rows take 1.6 times as long), measured
// on single work-groups and full chips (tiles of 16 and 64 rows: two a CU, but 16
// of f32 or past 128 dims): a step up to a work-group a CU, past it, and a
// work-group's own time
//
//   rows        16    32    64   128   256
//   alone     0.67   0.8  2.35   2.4   3.6
//   full       1.2   0.8   3.2   2.5   4.2
//   own          8  10.5     9    10    14
//
// The chip reads 128 keys of a kv head in 2.5 us / CUs; every further tile of 16 or
// 32 rows, reading them from L2, adds a quarter where it is not there at the same
// time (more than one round).
//
// For one round of the CUs, two, three ... the shortest cut is taken whose
// work-groups fit them, so that the rounds end together whatever the mix of
// lengths; of these, of whole sequences and of the tiles, the plan whose estimate
// is least: the memory's time, or half way between the CUs' share of the work and
// the rounds' longest work-groups, and the merge's.  Over 20 calls of 1 to 32
// sequences, 10 to 8000 tokens, 12 to 256 rows the plan taken is 2 % slower on
// average than the fastest one; 32/8 heads, us by tile (best cuts): 1 x 10 tokens, 28
// rows 7.7 / 9.9 / 7.3 / 7.6 / 9.4; 1 x 1000, 256 rows 14.3 / 15.9 / 18 / 18 / 22; 8 x
// 4000, 256 rows 103 / 70 / 70 / 61 / 59; 32 x 2000, 28 rows 46 / 48 / 50 / 50 / 72.
inline TreePlan tree_plan(const std::vector<TreeLoad> &load, int kvh, int cus, int hd, bool fine) {
    static const struct {
        int tile;
        double alone, full, own;
    } kinds[] = {{16, 0.67, 1.2, 8.0}, {32, 0.8, 0.8, 10.5}, {64, 2.35, 3.2, 9.0}, {128, 2.4, 2.5, 10.0}, {256, 3.6, 4.2, 14.0}};
    const auto steps = [](int len) { return (len + 127) / 128; };
    int64_t keys = 0;
    int most = 1;
    for (const TreeLoad &l : load) {
        keys += (int64_t)kvh * steps(l.len);
        most = std::max(most, steps(l.len));
    }
    const double wide = std::max(hd, 64) / 128.0;
    const double mem = 2.5 * wide * keys / cus;
    TreePlan plan;
    double best = 0.0;
    int best_at = most;
    for (const auto &kind : kinds) {
        if (!tree_has_tile(kind.tile, hd, fine)) continue;
        const int per_cu = hd <= 128 && (kind.tile == 64 || (kind.tile == 16 && !fine)) ? 2 : 1, slots = per_cu * cus;
        const auto tiles = [&](const TreeLoad &l) { return (l.rows + kind.tile - 1) / kind.tile; };
        int64_t all = 0;
        for (const TreeLoad &l : load) all += (int64_t)tiles(l) * kvh * steps(l.len);
        const auto count = [&](int at, int64_t *parts) {
            int64_t wgs = 0;
            *parts = 0;
            for (const TreeLoad &l : load) {
                const int n = (steps(l.len) + at - 1) / at;
                wgs += (int64_t)tiles(l) * kvh * n;
                if (n > 1) *parts += (int64_t)l.rows * kvh * n;
            }
            return wgs;
        };
        // (a tile's share of reading the keys again; wide tiles stream a little worse)
        const double again = std::min((double)all / keys - 1.0, 4.0);
        const double own = kind.own * (fine ? 1.5 : 1.0);
        int last = 0;
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
                wgs = count(at, &parts);
            }
            if (at == last) continue;
            last = at;
            const double step = (wgs <= cus ? kind.alone : kind.full) * wide * (fine ? 1.6 : 1.0);
            const double one = at * step + own;
            const double rounds = (double)((wgs + slots - 1) / slots) * one;
            const double share = std::max(one, (all * step + wgs * own) / slots);
            const double read = kind.tile <= 32 ? 1.0 + (wgs > slots ? 0.25 : 0.05) * again : kind.tile == 64 ? 1.0 : 1.15;
            double us = std::max(mem * read + own, 0.5 * (rounds + share));
            if (parts) us += 2.0 + 1.6 * ((most + at - 1) / at + 7) / 8 + parts * hd * 2e-6;
            if (best == 0.0 || us < best) {
                best = us;
                best_at = at;
                plan.tile = kind.tile;
            }
        }
    }
    for (const TreeLoad &l : load) plan.cuts.push_back((steps(l.len) + best_at - 1) / best_at);
    return plan;
}

}  // namespace rlx
