// Trees of drafted tokens over the paged GQA cache: plan records and launchers
// (rlx_tree.hip, rlx_tree_accept.hip, rlx_rope.hip).
#pragma once
#include "rlx_common.h"

namespace rlx {

constexpr int kTreeMaxNodes = 256;  // nodes of one sequence's tree
constexpr int kTreeKeys = 32;       // keys a wave takes at a time

// One sequence of a tree attention call.
struct TreeRow {
    int32_t tab;     // flat index of the sequence's first live table entry
    int32_t len;     // live tokens, the tree's nodes the last of them
    int32_t nodes;   // nodes | query rows << 16 (the last nodes)
    int32_t qrow;    // first call-row of this sequence's queries / outputs
    int32_t node0;   // first entry of this sequence in `parents`
    int32_t nsplit;  // cuts along the keys
    int32_t wg0;     // first work-group
    int32_t part;    // first partial slot (nsplit > 1)
};
static_assert(sizeof(TreeRow) == 32, "TreeRow is 8 int32");

struct TreeArgs {
    const uint16_t *kpool, *vpool;
    const int32_t *table;
    const TreeRow *rows;     // device rows, or nullptr: in the plan argument
    const int32_t *work;     // device rows only: the row of each work-group
    const int32_t *parents;
    const void *q;
    void *out;
    float *part_o, *part_ml;  // [slot][rows of a tile][D], [slot][rows of a tile][max, sum]
    int n_rows, H, KVH, DQ, P, pshift;  // pshift: log2(P), or -1
    int q_bf16, out_bf16, layout;
    float qscale;  // scale * log2(e)
};

// fine: queries and weights in parts of bf16, for f32 queries or outputs.
hipError_t launch_tree_attend(hipStream_t s, const PlanArg &plan, const TreeArgs &a, int hd, int tile_rows,
                              bool fine, int n_wgs, bool merge, int max_qr, hipEvent_t e0, hipEvent_t e1);

// One (layer, sequence) whose accepted nodes move: node path[path0 + j] to slot
// base + j, j in [0, n) (path[j] > j: an unmoved beginning is left out).
struct KeepRow {
    uint16_t *kpool, *vpool;
    int32_t tab, base, n, path0;
};
static_assert(sizeof(KeepRow) == 32, "KeepRow is 32 bytes");
hipError_t launch_tree_keep(hipStream_t s, const PlanArg *plan, const KeepRow *rows, const int32_t *path, int path_off,
                            int n_rows, const int32_t *table, int kvh, int hd, int P);

// Rotary positions of `heads` heads a row (rlx_rope).
struct RopeArgs {
    const void *x;
    void *out;
    int64_t x_row, x_head, out_row, out_head;  // strides, elements
    const int32_t *pos;
    const float *inv_freq;
    float scale;
    int64_t rows;
    int heads, D, rd;
    int x_bf16, out_bf16, halves;
};
hipError_t launch_rope(hipStream_t s, const RopeArgs &a, int cus);

// Acceptance of trees of drafts (rlx_tree_accept_async).
struct TreeAcceptArgs {
    const float *t_logits, *d_logits;  // [nodes][V] (d_logits: nullptr: drafts without probabilities)
    int64_t t_stride, d_stride;
    const int32_t *tok, *parents;
    const float *u;
    int V;
    float temperature;
    const int2 *trees;  // (first node, nodes) of each sequence, or nullptr: in the plan argument
    int32_t *path, *n_acc, *next;
    int path_stride;
};
hipError_t launch_tree_accept(hipStream_t s, const PlanArg *plan, const TreeAcceptArgs &a, int n_seqs,
                              hipEvent_t e0, hipEvent_t e1);

}  // namespace rlx
