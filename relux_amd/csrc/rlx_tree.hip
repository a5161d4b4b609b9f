// Attention of a tree of drafted tokens over the paged bf16 GQA cache, and the
// move that keeps a tree's accepted path.
//
// The last N live tokens of a sequence are the nodes of a tree in the order they
// were appended; parents[j] < j names node j's parent.  Query j is node j and
// attends every token before the tree, itself and its ancestors:
//
//   out_j = sum_t w_jt v_t / sum_t w_jt,  w_jt = exp(scale q_j.k_t),
//   t < len - N, or t - (len - N) in {j, parents[j], parents[parents[j]], ...}
#include <type_traits>

#include "rlx_tree.h"

namespace rlx {

typedef __attribute__((address_space(4))) const int32_t kconst_i32;

// A record of n int32 from the plan argument (rows == nullptr) or device memory,
// by scalar loads either way: the kernel-argument segment is ordinary memory.
__device__ __forceinline__ kconst_i32 *plan_ints(const void *rows, int i, int n) {
    return rows ? (kconst_i32 *)(uintptr_t)rows + (int64_t)i * n : (kconst_i32 *)kernarg_plan() + i * n;
}
__device__ __forceinline__ TreeRow tree_row(const TreeRow *rows, int i) {
    kconst_i32 *p = plan_ints(rows, i, 8);
    return TreeRow{p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]};
}

__device__ __forceinline__ void tree_store4(void *out, int64_t o, const float (&v)[4], int out_bf16) {
    if (out_bf16) {
        uint16_t *dst = (uint16_t *)out + o;
        if (((uintptr_t)out & 7) == 0) {
            *(uint2 *)dst = make_uint2(bf16_rne(v[0]) | ((uint32_t)bf16_rne(v[1]) << 16),
                                       bf16_rne(v[2]) | ((uint32_t)bf16_rne(v[3]) << 16));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) dst[i] = bf16_rne(v[i]);
        }
    } else {
        float *dst = (float *)out + o;
        if (((uintptr_t)out & 15) == 0) {
            *(float4 *)dst = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) dst[i] = v[i];
        }
    }
}

// Element of the outputs (and queries) where query row qr of kv head kvh starts.
__device__ __forceinline__ int64_t tree_qbase(const TreeArgs &a, const TreeRow &R, int kvh, int G, int qr) {
    const int qi = qr / G, h = kvh * G + (qr - qi * G), nq = R.nodes >> 16;
    return (a.layout == kLayoutSHD ? (int64_t)(R.qrow + qi) * a.H + h
                                   : (int64_t)R.qrow * a.H + (int64_t)h * nq + qi) * a.DQ;
}

// Ancestor sets of a tree's nodes, bit k of word w of node j: node 32 w + k is j
// or an ancestor.  Each round joins a node's set with that of the node it
// points to and doubles how far it points (8 rounds for a chain of 256).  A
// parent outside [0, j) ends the chain.  Words past the tree's are zero up to one
// more than its last.
__device__ __forceinline__ void tree_ancestors(int parent, int n, uint32_t (*anc)[kTreeMaxNodes], int16_t *up) {
    const int j = threadIdx.x, words = (n + 31) >> 5;
    int u = -1;
    if (j < n) {
        u = parent >= 0 && parent < j ? parent : -1;
        for (int w = 0; w <= words; w++) anc[w][j] = w == (j >> 5) ? 1u << (j & 31) : 0u;
        up[j] = (int16_t)u;
    }
    while (__syncthreads_or(u >= 0)) {
        uint32_t s[kTreeMaxNodes / 32];
        int far = -1;
        if (u >= 0) {
#pragma unroll
            for (int w = 0; w < kTreeMaxNodes / 32; w++) s[w] = w < words ? anc[w][u] : 0u;
            far = up[u];
        }
        __syncthreads();
        if (u >= 0) {
#pragma unroll
            for (int w = 0; w < kTreeMaxNodes / 32; w++)
                if (w < words) anc[w][j] |= s[w];
            up[j] = (int16_t)far;
        }
        u = far;
    }
}

// What a work-group computes: a cut of one kv head's keys for a tile of query rows.
struct TreeItem {
    TreeRow R;
    int nodes, nq, G, QR, tiles, split, kvh, tile, ctx, u0, u1;  // ctx: first key of the tree; u: units of 32 keys
};
// The item of work-group blockIdx.x.
//
// Work-group b runs on XCD b mod 8, each with its own L2: the tiles of a (cut, kv
// head) pair read the same keys and are put 8 apart, the pairs dealt out.
template <int QT>
__device__ __forceinline__ void tree_item(const TreeArgs &a, TreeItem &w) {
    const int b = blockIdx.x;
    int r;
    if (a.rows) {
        r = ((kconst_i32 *)(uintptr_t)a.work)[b];
    } else {
        int lo = 0, hi = a.n_rows - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (plan_ints(nullptr, mid, 8)[6] <= b)
                lo = mid;
            else
                hi = mid - 1;
        }
        r = lo;
    }
    w.R = tree_row(a.rows, r);
    w.nodes = w.R.nodes & 0xFFFF;
    w.nq = w.R.nodes >> 16;
    w.G = a.H / a.KVH;
    w.QR = w.nq * w.G;
    w.tiles = (w.QR + QT - 1) / QT;
    const int pairs = w.R.nsplit * a.KVH, i = b - w.R.wg0;
    const int s0 = i / (8 * w.tiles) * 8, m = min(8, pairs - s0), rem = i - s0 * w.tiles;
    w.tile = rem / m;
    const int pair = s0 + rem - w.tile * m;
    w.split = pair / a.KVH;
    w.kvh = pair - w.split * a.KVH;
    w.ctx = w.R.len - w.nodes;
    const int units = (w.R.len + kTreeKeys - 1) / kTreeKeys;
    w.u0 = (int)((int64_t)w.split * units / w.R.nsplit);
    w.u1 = (int)((int64_t)(w.split + 1) * units / w.R.nsplit);
}
// Partial slot of (cut, kv head, tile) of a row.
__device__ __forceinline__ int64_t tree_slot(const TreeRow &R, int KVH, int tiles, int split, int kvh, int tile) {
    return (int64_t)R.part + ((int64_t)split * KVH + kvh) * tiles + tile;
}

// The bf16 parts (the high one, or three whose sum is the f32 value) of 8 values.
template <int PARTS>
__device__ __forceinline__ void tree_parts(float (&v)[8], u32x4 (&o)[PARTS]) {
#pragma unroll
    for (int p = 0; p < PARTS; p++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            o[p][i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
            v[2 * i] -= bf16_lo(o[p][i]);
            v[2 * i + 1] -= bf16_hi(o[p][i]);
        }
}

// A wave's 16 NQT query rows and their running softmax over units of 32 keys:
//
//   S^T[32 keys][16 rows] = K[32 x D] . Q^T         2 D/32 MFMA 16x16x32 a tile
//   P = exp2(S c - m), lane-local
//   O^T[D][16 rows]      += V^T[D x 32 keys] . P^T  D/16 MFMA 16x16x32 a tile
//
// Rows of the two 16-key score tiles are given the keys 8 (row / 4) + row % 4 and
// 4 more, so that a lane's scores are those of 8 consecutive keys: the operand of
// the second product as they are, against V read 8 keys (16 bytes) at a time.
//
// The maximum of a row moves only when a score exceeds it by 2^8 (weights stay
// below 256 in f32 and bf16 alike), so that rescaling and the reduction over
// lanes are rare.
//
// Weights are rounded to bf16 for the second product, and the sum is of the
// rounded ones.  FINE (f32 queries or outputs): queries and weights in three
// bf16 parts, as exact as f32.
//
// A masked weight is a selected zero; a value that is not finite in a masked
// place must not reach other rows through 0 x inf, so such values of the tree's
// keys stay out of the product and replace the sums of the rows that attend them.
template <int D, int NQT, bool FINE, bool ACC>
struct TreeWave {
    static constexpr int KS = D < 32 ? 1 : D / 32, MT = D / 16, PARTS = FINE ? 3 : 1;
    u32x4 qb[NQT][KS][PARTS];
    int node[NQT];
    float m_run[NQT], l_part[NQT];
    fl4 acc[NQT][MT];
    bool odd = false;  // a value of the tree's keys that is not finite
    int col, grp, len, ctx;
    const uint32_t (*anc)[kTreeMaxNodes];

    // Query rows row0 + 16 nt + col; rows past the last one hold zeros.
    __device__ __forceinline__ void init(const TreeArgs &a, const TreeItem &w, int row0, const uint32_t (*an)[kTreeMaxNodes]) {
        const int lane = threadIdx.x & 63;
        col = lane & 15;
        grp = lane >> 4;
        len = w.R.len;
        ctx = w.ctx;
        anc = an;
#pragma unroll
        for (int nt = 0; nt < NQT; nt++) {
            const int qr = row0 + nt * 16 + col;
            const bool ok = qr < w.QR;
            const int qc = ok ? qr : 0;
            node[nt] = w.nodes - w.nq + qc / w.G;
            const int64_t base = tree_qbase(a, w.R, w.kvh, w.G, qc);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const int d0 = ks * 32 + grp * 8;
                const bool in = ok && d0 < a.DQ;
                if (a.q_bf16) {
                    qb[nt][ks][0] = in ? *(const u32x4 *)((const uint16_t *)a.q + base + d0) : u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int p = 1; p < PARTS; p++) qb[nt][ks][p] = u32x4{0, 0, 0, 0};
                } else {
                    const float4 z = float4{0.f, 0.f, 0.f, 0.f};
                    const float4 x = in ? *(const float4 *)((const float *)a.q + base + d0) : z;
                    const float4 y = in ? *(const float4 *)((const float *)a.q + base + d0 + 4) : z;
                    float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                    tree_parts<PARTS>(v, qb[nt][ks]);
                }
            }
            m_run[nt] = -INFINITY;
            l_part[nt] = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; mt++) acc[nt][mt] = fl4{0.f, 0.f, 0.f, 0.f};
        }
    }

    // The queries are here: no wait for them sits in the loop, where it would
    // wait for the keys requested ahead as well.
    __device__ __forceinline__ void ready() const {
#pragma unroll
        for (int nt = 0; nt < NQT; nt++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int p = 0; p < PARTS; p++) asm volatile("" ::"v"(qb[nt][ks][p]));
    }

    typedef fl4 Scores[NQT][2];
    typedef u32x4 Weights[NQT][PARTS];

    // Scores of a unit; kf(k, ks): the keys' fragments.
    template <class KF>
    __device__ __forceinline__ void scores(Scores &s, KF kf) {
#pragma unroll
        for (int nt = 0; nt < NQT; nt++) s[nt][0] = s[nt][1] = fl4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const bf16x8 kr = __builtin_bit_cast(bf16x8, kf(k, ks));
#pragma unroll
                for (int p = PARTS - 1; p >= 0; p--)
#pragma unroll
                    for (int nt = 0; nt < NQT; nt++)
                        s[nt][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kr, __builtin_bit_cast(bf16x8, qb[nt][ks][p]),
                                                                          s[nt][k], 0, 0, 0);
            }
    }
    // FINE: an infinite key against a query's parts of both signs is a NaN; its
    // score is the first part's.
    template <class KF>
    __device__ __forceinline__ void mend(Scores &s, KF kf) {
        if constexpr (FINE) {
            float sum = 0.f;
#pragma unroll
            for (int nt = 0; nt < NQT; nt++)
#pragma unroll
                for (int i = 0; i < 8; i++) sum += s[nt][i >> 2][i & 3];
            if (__builtin_amdgcn_ballot_w64(sum != sum)) {
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    fl4 h[NQT];
#pragma unroll
                    for (int nt = 0; nt < NQT; nt++) h[nt] = fl4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ks = 0; ks < KS; ks++)
#pragma unroll
                        for (int nt = 0; nt < NQT; nt++)
                            h[nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kf(k, ks)),
                                                                            __builtin_bit_cast(bf16x8, qb[nt][ks][0]),
                                                                            h[nt], 0, 0, 0);
#pragma unroll
                    for (int nt = 0; nt < NQT; nt++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (s[nt][k][i] != s[nt][k][i]) s[nt][k][i] = h[nt][i];
                }
            }
        }
    }
    // The keys tl .. tl + 7 that row tile nt's row attends, as bits (none past the
    // last token: it has no node there).
    __device__ __forceinline__ uint32_t seen8(int tl, int nt) const {
        const int k = tl - ctx;
        if (k <= -8) return 0xFFu;
        if (k < 0) return (anc[0][node[nt]] << -k) | ((1u << -k) - 1u);
        const int w = min(k >> 5, kTreeMaxNodes / 32 - 1);
        const uint64_t bits = (uint64_t)anc[w + 1][node[nt]] << 32 | anc[w][node[nt]];
        return tl < len ? (uint32_t)(bits >> (k & 31)) : 0u;
    }
    // Masks a unit from key t0 that holds keys of the tree, or past the last token.
    __device__ __forceinline__ void mask(Scores &s, int t0) const {
#pragma unroll
        for (int nt = 0; nt < NQT; nt++) {
            const uint32_t m = seen8(t0 + grp * 8, nt);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (!(m & (1u << i))) s[nt][i >> 2][i & 3] = -INFINITY;
        }
    }
    // A lane's largest scores.
    __device__ __forceinline__ void largest(const Scores &s, float (&mx)[NQT]) const {
#pragma unroll
        for (int nt = 0; nt < NQT; nt++)
            mx[nt] = max3(max3(max3(s[nt][0][0], s[nt][0][1], s[nt][0][2]), s[nt][0][3], s[nt][1][0]), s[nt][1][1],
                          max3(s[nt][1][2], s[nt][1][3], s[nt][1][3]));
    }
    // (as one instruction: fmaxf makes its operands canonical first)
    static __device__ __forceinline__ float max3(float x, float y, float z) {
        float r;
        asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
        return r;
    }
    // Moves the maximum (and what was summed under it) where a score exceeds it far.
    __device__ __forceinline__ void grow(const float (&mx)[NQT], float qscale) {
        bool far = false;
#pragma unroll
        for (int nt = 0; nt < NQT; nt++) far |= mx[nt] * qscale > m_run[nt] + 8.f;
        if (!__builtin_amdgcn_ballot_w64(far)) return;
#pragma unroll
        for (int nt = 0; nt < NQT; nt++) {
            const float m_new = fmaxf(m_run[nt], rows4_max(mx[nt]) * qscale);
            const float c = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run[nt] - m_new);
            m_run[nt] = m_new;
            l_part[nt] *= c;
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                // (pinned on both sides, so that the loop does not carry copies
                // for this branch)
                pin(acc[nt][mt]);
                acc[nt][mt] *= c;
                pin(acc[nt][mt]);
            }
        }
    }
    // Accumulators live in accumulation registers where a wave has more than 256.
    static __device__ __forceinline__ void pin(fl4 &x) {
        if constexpr (ACC)
            asm volatile("" : "+a"(x));
        else
            asm volatile("" : "+v"(x));
    }
    __device__ __forceinline__ void weights(const Scores &s, Weights &pw, float qscale) {
#pragma unroll
        for (int nt = 0; nt < NQT; nt++) {
            const float m = m_run[nt] == -INFINITY ? 0.f : m_run[nt];
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = __builtin_amdgcn_exp2f(fmaf(s[nt][i >> 2][i & 3], qscale, -m));
            if constexpr (FINE) l_part[nt] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            tree_parts<PARTS>(p, pw[nt]);
            if constexpr (!FINE)
#pragma unroll
                for (int i = 0; i < 4; i++) l_part[nt] = add_bf16x2(pw[nt][0][i], l_part[nt]);
        }
    }
    // The values' product; vf(mt): their fragments.  TREE: as mask(); values past the
    // last token are zeroed, and those of the tree that are not finite taken out.
    template <bool TREE, class VF>
    __device__ __forceinline__ void values(const Weights &pw, int t0, VF vf) {
        u32x4 v[MT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) v[mt] = vf(mt);
        if constexpr (TREE) {
            const int tl = t0 + grp * 8;
            u32x4 live, tree;  // halves before the last token; of the tree
#pragma unroll
            for (int i = 0; i < 4; i++) {
                live[i] = (tl + 2 * i < len ? 0xFFFFu : 0u) | (tl + 2 * i + 1 < len ? 0xFFFF0000u : 0u);
                tree[i] = (tl + 2 * i >= ctx ? 0x8000u : 0u) | (tl + 2 * i + 1 >= ctx ? 0x80000000u : 0u);
            }
            uint32_t bad = 0;
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    v[mt][i] &= live[i];
                    bad |= ((v[mt][i] & 0x7F807F80u) + 0x00800080u) & tree[i];  // an exponent of ones carries
                }
            if (__builtin_amdgcn_ballot_w64(bad != 0)) {
                odd = true;
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t x = ((v[mt][i] & 0x7F807F80u) + 0x00800080u) & tree[i];
                        v[mt][i] &= ~((x >> 15) * 0xFFFFu);
                    }
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int p = PARTS - 1; p >= 0; p--)
#pragma unroll
                for (int nt = 0; nt < NQT; nt++)
                    acc[nt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, v[mt]), __builtin_bit_cast(bf16x8, pw[nt][p]), acc[nt][mt], 0, 0, 0);
    }
};

// The tree's values that are not finite, taken out of the product: where the row qt
// of the tile attends one in dims d0 .. d0 + 3 it is the sum, whatever the weights.
// Run by the lane that stored these dims, after it.
__device__ __forceinline__ void tree_odd(const TreeArgs &a, const TreeItem &w, const uint32_t (*anc)[kTreeMaxNodes],
                                         int64_t slot, int D, int QT, int qt, int d0) {
    const int qr = w.tile * QT + qt;
    if (qr >= w.QR || (w.R.nsplit == 1 && d0 >= a.DQ)) return;
    const int node = w.nodes - w.nq + qr / w.G;
#pragma unroll 1
    for (int i = 0; i < 4; i++) {
        float x = 0.f;
#pragma unroll 1
        for (int t = max(w.u0 * kTreeKeys, w.ctx); t < min(w.u1 * kTreeKeys, w.R.len); t++) {
            const int k = t - w.ctx, e = t / a.P;
            if (!((anc[k >> 5][node] >> (k & 31)) & 1u)) continue;
            const uint16_t v = a.vpool[(((int64_t)a.table[w.R.tab + e] * a.KVH + w.kvh) * D + d0 + i) * a.P + (t - e * a.P)];
            if ((v & 0x7F80) == 0x7F80) x += bf16_f32(v);
        }
        if (x == 0.f) continue;
        if (w.R.nsplit > 1) {
            a.part_o[(slot * QT + qt) * D + d0 + i] = x;
        } else {
            const int64_t o = tree_qbase(a, w.R, w.kvh, w.G, qr) + d0 + i;
            if (a.out_bf16)
                ((uint16_t *)a.out)[o] = bf16_rne(x);
            else
                ((float *)a.out)[o] = x;
        }
    }
}

// Byte offsets into the K and V pools of a lane's block (lane & 1) of unit j +
// lane / 2, of `nu` units `step` apart from unit `first`.  A block past the last
// token is the last token's (its keys are masked).
template <int D>
struct TreePages {
    int64_t k, v;
    int page, slot;
    __device__ __forceinline__ void request(const TreeArgs &a, const TreeItem &w, int first, int step, int nu, int j) {
        const int lane = threadIdx.x & 63;
        int t = (first + step * min(j + (lane >> 1), nu - 1)) * kTreeKeys + 16 * (lane & 1);
        t = min(t, (w.R.len - 1) & ~15);
        const int e = a.pshift >= 0 ? t >> a.pshift : t / a.P;
        slot = t - e * a.P;
        page = a.table[w.R.tab + e];
    }
    __device__ __forceinline__ void take(const TreeArgs &a, const TreeItem &w) {
        const int64_t base = ((int64_t)page * a.KVH + w.kvh) * a.P * D;
        k = (base + (int64_t)slot * D) * 2;
        v = (base + slot) * 2;
        // wait here, so that no wait for these sits on the common path
        asm volatile("" ::"v"(k), "v"(v));
    }
    __device__ __forceinline__ void fetch(const TreeArgs &a, const TreeItem &w, int first, int step, int nu, int j) {
        request(a, w, first, step, nu, j);
        take(a, w);
    }
    // A lane's offset in unit j of the fetched ones: that of its block.
    static __device__ __forceinline__ int64_t pick(int64_t off, int j, bool second) {
        const int src = (2 * j) & 63;
        const auto at = [&](int l) {
            const uint32_t lo = __builtin_amdgcn_readlane((int)off, l), hi = __builtin_amdgcn_readlane((int)(off >> 32), l);
            return (int64_t)((uint64_t)hi << 32 | lo);
        };
        const int64_t x = at(src), y = at(src + 1);
        return second ? y : x;
    }
};
// A lane's places in a unit: K of key 8 (col / 4) + col % 4 (kKeys4 bytes on: the
// second score tile's, 4 keys further; kStep: the next 32 dims), dims 8 grp ..;
// V of dim col, keys 8 grp ...
template <int D>
struct TreeLane {
    static constexpr int kKeys4 = D <= 32 ? 4 * D * 2 : 256, kStep = 1024;
    const char *k, *v;
    bool k2, v2;  // in the unit's second block
    __device__ __forceinline__ explicit TreeLane(const TreeArgs &a) {
        const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4, row = ((col >> 2) & 1) * 8 + (col & 3);
        k = (const char *)a.kpool + (D == 16 ? row * 32 + (grp & 1) * 16 : row * 64 + grp * 16);
        v = (const char *)a.vpool + (col * a.P + (grp & 1) * 8) * 2;
        k2 = col >= 8;
        v2 = grp >= 2;
    }
};

// Few query rows: 4 waves, each holding all 16 NQT rows of the tile and taking
// every fourth unit, straight from HBM into registers in the operands' order -- no
// LDS and no barrier in the loop.  HBM-bound: 16 sequences of 8192 tokens, 16 nodes,
// 32 / 8 heads of 128, bf16, 99 us, 5.4 TB/s (a large copy moves 5.2).  One of 200
// tokens, 7 nodes, f32: 12 us, a launch and the chain of reads (plan, table, keys),
// products and joins of its one round.
// SHARED: other tiles read the same keys, which stay in L2 (else non-temporal loads).
template <int D, int NQT, bool FINE, bool SHARED>
__global__ __launch_bounds__(256, 1) void tree_narrow_kernel(PlanArg plan, TreeArgs a) {
    using W = TreeWave<D, NQT, FINE, true>;
    constexpr int KS = W::KS, MT = W::MT, QT = 16 * NQT;
    constexpr int MC = MT < 8 ? MT : 8;  // m-tiles merged at a time
    __shared__ uint32_t anc[kTreeMaxNodes / 32 + 1][kTreeMaxNodes];
    __shared__ int16_t up[kTreeMaxNodes];
    __shared__ float sm[4][QT], sl[4][QT];
    __shared__ fl4 so[4][MC][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    TreeItem w;
    tree_item<QT>(a, w);
    const int parent = threadIdx.x < w.nodes ? a.parents[w.R.node0 + threadIdx.x] : -1;

    const int first = w.u0 + wave, nu = first < w.u1 ? (w.u1 - first + 3) / 4 : 0;
    const int nc = max(0, min(nu, (w.ctx / kTreeKeys - first + 3) / 4));  // units before the tree's
    TreePages<D> pages;
    if (nu > 0) pages.request(a, w, first, 4, nu, 0);
    const TreeLane<D> at(a);
    W q;
    q.init(a, w, w.tile * QT, anc);
    if (nu > 0) pages.take(a, w);

    const auto get = [](const char *p) {
        if constexpr (SHARED)
            return *(const u32x4 *)p;
        else
            return __builtin_nontemporal_load((const u32x4 *)p);
    };
    auto load = [&](int j, u32x4(&kr)[2][KS], u32x4(&vr)[MT]) {
        j = min(j, nu - 1);
        if ((j & 31) == 0 && j) pages.fetch(a, w, first, 4, nu, j);
        const char *kp = at.k + pages.pick(pages.k, j, at.k2), *vp = at.v + pages.pick(pages.v, j, at.v2);
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int k = 0; k < 2; k++)
                kr[k][ks] = get(kp + ks * at.kStep + k * at.kKeys4);
#pragma unroll
        for (int mt = 0; mt < MT; mt++) vr[mt] = get(vp + mt * a.P * 32);
    };
    auto consume = [&](auto tree, int j, u32x4(&kr)[2][KS], u32x4(&vr)[MT]) {
        constexpr bool TREE = decltype(tree)::value;
        const int t0 = (first + 4 * j) * kTreeKeys;
        const auto kf = [&](int k, int ks) { return D == 16 && q.grp >= 2 ? u32x4{0, 0, 0, 0} : kr[k][ks]; };
        typename W::Scores sc;
        typename W::Weights pw;
        float mx[NQT];
        q.scores(sc, kf);
        q.mend(sc, kf);
        if constexpr (TREE) q.mask(sc, t0);
        q.largest(sc, mx);
        q.grow(mx, a.qscale);
        q.weights(sc, pw, a.qscale);
        q.template values<TREE>(pw, t0, [&](int mt) { return vr[mt]; });
    };
    using Ctx = std::integral_constant<bool, false>;
    using Tree = std::integral_constant<bool, true>;
    // Two register sets alternate, so that the next unit's loads are in flight
    // while one is consumed (past the last unit they read it again).  Stored head
    // dim 256 has registers for one.
    u32x4 ka[2][KS], kb[2][KS], va[MT], vb[MT];
    int j = 0;
    if constexpr (D <= 128)
        if (nu > 0) load(0, ka, va);
    if (w.u1 * kTreeKeys > w.ctx) tree_ancestors(parent, w.nodes, anc, up);
    if constexpr (D <= 128) {
        q.ready();
        for (; j + 1 < nc; j += 2) {
            load(j + 1, kb, vb);
            consume(Ctx{}, j, ka, va);
            load(j + 2, ka, va);
            consume(Ctx{}, j + 1, kb, vb);
        }
        for (; j < nu; j++) {
            load(j + 1, kb, vb);
            consume(Tree{}, j, ka, va);
#pragma unroll
            for (int i = 0; i < KS; i++) ka[0][i] = kb[0][i], ka[1][i] = kb[1][i];
#pragma unroll
            for (int i = 0; i < MT; i++) va[i] = vb[i];
        }
    } else {
        for (; j < nc; j++) {
            load(j, ka, va);
            consume(Ctx{}, j, ka, va);
        }
        for (; j < nu; j++) {
            load(j, ka, va);
            consume(Tree{}, j, ka, va);
        }
    }

    // ---- merge of the 4 waves ----
#pragma unroll
    for (int nt = 0; nt < NQT; nt++) {
        const float l = rows4_sum(q.l_part[nt]);
        if (q.grp == 0) {
            sm[wave][nt * 16 + q.col] = q.m_run[nt];
            sl[wave][nt * 16 + q.col] = l;
        }
    }
    const bool any_odd = __syncthreads_or(q.odd);
    const int64_t slot = tree_slot(w.R, a.KVH, w.tiles, w.split, w.kvh, w.tile);
#pragma unroll
    for (int nt = 0; nt < NQT; nt++) {
        const int qt = nt * 16 + q.col, qr = w.tile * QT + qt;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) M = fmaxf(M, sm[i][qt]);
#pragma unroll
        for (int i = 0; i < 4; i++) L += sm[i][qt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[i][qt] - M) * sl[i][qt];
        const float f = q.m_run[nt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(q.m_run[nt] - M);
        const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
        for (int m0 = 0; m0 < MT; m0 += MC) {
            if (nt || m0) __syncthreads();
#pragma unroll
            for (int mt = 0; mt < MC; mt++) so[wave][mt][lane] = q.acc[nt][m0 + mt] * f;
            __syncthreads();
#pragma unroll 1
            for (int mt = wave; mt < MC; mt += 4) {
                const fl4 o = (so[0][mt][lane] + so[1][mt][lane]) + (so[2][mt][lane] + so[3][mt][lane]);
                const int d0 = (m0 + mt) * 16 + q.grp * 4;
                if (w.R.nsplit > 1) {
                    *(fl4 *)(a.part_o + (slot * QT + qt) * D + d0) = o;
                } else if (qr < w.QR && d0 < a.DQ) {
                    const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
                    tree_store4(a.out, tree_qbase(a, w.R, w.kvh, w.G, qr) + d0, v, a.out_bf16);
                }
            }
        }
        if (w.R.nsplit > 1 && wave == 0 && q.grp == 0) {
            float *pm = a.part_ml + (slot * QT + qt) * 2;
            pm[0] = M;
            pm[1] = L;
        }
    }
    if (any_odd) {
#pragma unroll 1
        for (int nt = 0; nt < NQT; nt++)
#pragma unroll 1
            for (int mt = wave; mt < MT; mt += 4)
                tree_odd(a, w, anc, slot, D, QT, nt * 16 + q.col, mt * 16 + q.grp * 4);
    }
}

// Many query rows: WAVES waves of 16 NQT rows each share the keys, which stream
// through a ring of units in LDS in the operands' order (a lane's 16 bytes of a
// fragment at 16 lane: reads without bank conflicts).  A wave takes the scores of unit
// u + 1 while it turns those of unit u into weights, so that the matrix unit works
// through the softmax; two waves a SIMD hide the rest.  HBM-bound at few rows, by
// the matrix and softmax units at many: 24 sequences of 1000 to 12000 tokens, 40 to
// 64 nodes, 64 / 8 heads of 128, bf16: 255 to 265 us with the merge's 20, 670 to 695 TFLOP/s (a large
// library product reaches 1200), matrix units 36 % busy.
template <int D, int NQT, int WAVES, bool FINE>
__global__ __launch_bounds__(64 * WAVES, (D > 128 && WAVES == 4 ? 1 : 2)) void tree_wide_kernel(PlanArg plan, TreeArgs a) {
    using W = TreeWave<D, NQT, FINE, (D > 128 && WAVES == 4)>;
    constexpr int KS = W::KS, MT = W::MT, QT = 16 * NQT * WAVES;
    static_assert(D >= 64 && 2 * KS == MT, "K and V of a unit take as many loads");
    constexpr int UNIT = 2 * MT * 64;                       // u32x4 of a unit: K, then V
    constexpr int UPS = WAVES == 8 && D <= 128 ? 2 : 1;     // units a stage
    constexpr int STAGES = 4;                               // of 16 KB a unit (D 128) or 32
    constexpr int SLABS = UPS * 2 * MT, LOADS = (SLABS + WAVES - 1) / WAVES;  // fragments of a stage; a wave's of them
    static_assert(SLABS % WAVES == 0 && MT % LOADS == 0, "a wave loads K or V");
    __shared__ uint32_t anc[kTreeMaxNodes / 32 + 1][kTreeMaxNodes];
    __shared__ int16_t up[kTreeMaxNodes];
    __shared__ u32x4 ring[STAGES * UPS][UNIT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    TreeItem w;
    tree_item<QT>(a, w);
    const int parent = threadIdx.x < w.nodes ? a.parents[w.R.node0 + threadIdx.x] : -1;

    const int nu = w.u1 - w.u0;
    const int nc = max(0, min(nu, w.ctx / kTreeKeys - w.u0));  // units before the tree's
    const bool shared = w.QR > QT;  // other tiles read the same keys
    const uint32_t ring_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) u32x4 *)&ring[0][0];
    TreePages<D> pages;
    pages.request(a, w, w.u0, 1, nu, 0);
    const TreeLane<D> at(a);
    W q;
    q.init(a, w, w.tile * QT + wave * 16 * NQT, anc);
    q.ready();
    pages.take(a, w);
    const int ns = (nu + UPS - 1) / UPS;
    // a wave's fragments are of one unit, and of K or V alone
    const int i0 = wave * LOADS % (2 * MT), uu = wave * LOADS / (2 * MT);
    const bool is_v = i0 >= MT;
    auto issue = [&](int s) {
        if ((s * UPS & 31) == 0 && s) pages.fetch(a, w, w.u0, 1, nu, s * UPS);
        const uint32_t dst = ring_lds + (uint32_t)(s % STAGES * UPS * UNIT + wave * LOADS * 64) * 16;
        const char *src = is_v ? at.v + pages.pick(pages.v, s * UPS + uu, at.v2) + (i0 - MT) * a.P * 32
                               : at.k + pages.pick(pages.k, s * UPS + uu, at.k2);
#pragma unroll
        for (int l = 0; l < LOADS; l++) {
            const int i = i0 + l;
            const char *p = is_v ? src + l * a.P * 32 : src + (i >> 1) * at.kStep + (i & 1) * at.kKeys4;
            if (shared)
                lds_dma16_keep(p, dst + l * 1024);
            else
                lds_dma16(p, dst + l * 1024);
        }
    };
    // Stage s is here: this wave's loads of it are done, then everybody's.  Stages
    // up to s + STAGES - 3 were requested.
    auto arrive = [&](int s) {
        if (s + STAGES - 3 < ns)
            RLX_WAIT_VM(LOADS * (STAGES - 3));
        else
            RLX_WAIT_VM(0);
        ring_barrier();
    };
    const auto kfrag = [&](int u) {
        const u32x4 *st = &ring[u % (STAGES * UPS)][lane];
        return [st](int k, int ks) { return st[(2 * ks + k) * 64]; };
    };
    const auto vfrag = [&](int u) {
        const u32x4 *st = &ring[u % (STAGES * UPS)][MT * 64 + lane];
        return [st](int mt) { return st[mt * 64]; };
    };
    for (int s = 0; s < STAGES - 2 && s < ns; s++) issue(s);
    if (w.u1 * kTreeKeys > w.ctx) tree_ancestors(parent, w.nodes, anc, up);
    typename W::Scores sc;
    float mx[NQT];
    arrive(0);
    if (STAGES - 2 < ns) issue(STAGES - 2);
    q.scores(sc, kfrag(0));
    q.mend(sc, kfrag(0));
    if (nc == 0) q.mask(sc, w.u0 * kTreeKeys);
    q.largest(sc, mx);
    // Before the scores of unit u + 1: its stage; then every wave is past the scores
    // and values of the stage two before, whose place the next request takes.
    auto ahead = [&](int u) {
        if ((u + 1) % UPS) return;
        const int s = (u + 1) / UPS;
        arrive(s);
        if (s + STAGES - 2 < ns) issue(s + STAGES - 2);
    };
    int u = 0;
    for (; u + UPS < nc; u += UPS) {
#pragma unroll
        for (int i = 0; i < UPS; i++) {
            q.grow(mx, a.qscale);
            ahead(u + i);
            typename W::Scores next;
            typename W::Weights pw;
            q.scores(next, kfrag(u + i + 1));
            q.weights(sc, pw, a.qscale);
            q.mend(next, kfrag(u + i + 1));
            q.template values<false>(pw, 0, vfrag(u + i));
            q.largest(next, mx);
#pragma unroll
            for (int nt = 0; nt < NQT; nt++) sc[nt][0] = next[nt][0], sc[nt][1] = next[nt][1];
        }
    }
    for (; u < nu; u++) {
        q.grow(mx, a.qscale);
        typename W::Weights pw;
        q.weights(sc, pw, a.qscale);
        q.template values<true>(pw, (w.u0 + u) * kTreeKeys, vfrag(u));
        if (u + 1 < nu) {
            ahead(u);
            q.scores(sc, kfrag(u + 1));
            q.mend(sc, kfrag(u + 1));
            q.mask(sc, (w.u0 + u + 1) * kTreeKeys);
            q.largest(sc, mx);
        }
    }

    const bool any_odd = __builtin_amdgcn_ballot_w64(q.odd) != 0;
    const int64_t slot = tree_slot(w.R, a.KVH, w.tiles, w.split, w.kvh, w.tile);
#pragma unroll
    for (int nt = 0; nt < NQT; nt++) {
        const int qt = (wave * NQT + nt) * 16 + q.col, qr = w.tile * QT + qt;
        const float L = rows4_sum(q.l_part[nt]), inv = L > 0.f ? 1.f / L : 0.f;
        if (qr >= w.QR) continue;
        const int64_t base = tree_qbase(a, w.R, w.kvh, w.G, qr);
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const fl4 o = q.acc[nt][mt];
            const int d0 = mt * 16 + q.grp * 4;
            if (w.R.nsplit > 1) {
                *(fl4 *)(a.part_o + (slot * QT + qt) * D + d0) = o;
            } else if (d0 < a.DQ) {
                const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
                tree_store4(a.out, base + d0, v, a.out_bf16);
            }
        }
        if (w.R.nsplit > 1 && q.grp == 0) {
            float *pm = a.part_ml + (slot * QT + qt) * 2;
            pm[0] = q.m_run[nt];
            pm[1] = L;
        }
    }
    if (any_odd) {
#pragma unroll 1
        for (int i = 0; i < NQT * MT; i++)
            tree_odd(a, w, anc, slot, D, QT, (wave * NQT + i / MT) * 16 + q.col, i % MT * 16 + q.grp * 4);
    }
}

// Joins the partials of the sequences whose keys were cut: a thread holds 4 dims
// of a query row.  out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.  HBM-bound.
__global__ __launch_bounds__(256) void tree_merge_kernel(PlanArg plan, TreeArgs a, int D, int QT) {
    const TreeRow R = tree_row(a.rows, blockIdx.x);
    if (R.nsplit <= 1) return;
    const int G = a.H / a.KVH, nq = R.nodes >> 16, QR = nq * G, kvh = blockIdx.y;
    const int Q4 = D >> 2, TQ = 256 / Q4, t = threadIdx.x;
    const int qr = blockIdx.z * TQ + t / Q4, d0 = (t - t / Q4 * Q4) * 4;
    if (t >= TQ * Q4 || qr >= QR) return;
    const int tiles = (QR + QT - 1) / QT, tile = qr / QT, qt = qr - tile * QT;
    const auto at = [&](int s) { return tree_slot(R, a.KVH, tiles, s, kvh, tile) * QT + qt; };
    constexpr int kFew = 8;  // partials read in one round trip
    float M = -INFINITY, L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < R.nsplit; s0 += kFew) {
        float2 ml[kFew];
        float4 o[kFew];
#pragma unroll
        for (int i = 0; i < kFew; i++) {
            const int64_t p = at(min(s0 + i, R.nsplit - 1));
            ml[i] = *(const float2 *)(a.part_ml + p * 2);
            o[i] = *(const float4 *)(a.part_o + p * D + d0);
        }
        float m = M;
#pragma unroll
        for (int i = 0; i < kFew; i++)
            if (s0 + i < R.nsplit) m = fmaxf(m, ml[i].x);
        if (m == -INFINITY) continue;
        const float c = __builtin_amdgcn_exp2f(M - m);
        L *= c;
        O.x *= c, O.y *= c, O.z *= c, O.w *= c;
#pragma unroll
        for (int i = 0; i < kFew; i++) {
            if (s0 + i >= R.nsplit || ml[i].x == -INFINITY) continue;
            const float f = __builtin_amdgcn_exp2f(ml[i].x - m);
            L += f * ml[i].y;
            O.x += f * o[i].x, O.y += f * o[i].y, O.z += f * o[i].z, O.w += f * o[i].w;
        }
        M = m;
    }
    if (d0 >= a.DQ) return;
    const float inv = L > 0.f ? 1.f / L : 0.f;
    const float v[4] = {O.x * inv, O.y * inv, O.z * inv, O.w * inv};
    tree_store4(a.out, tree_qbase(a, R, kvh, G, qr) + d0, v, a.out_bf16);
}

hipError_t launch_tree_attend(hipStream_t s, const PlanArg &plan, const TreeArgs &a, int hd, int tile_rows,
                              bool fine, int n_wgs, bool merge, int max_qr, hipEvent_t e0, hipEvent_t e1) {
    if (n_wgs <= 0) return hipSuccess;
    void (*k)(PlanArg, TreeArgs) = nullptr;
    const bool shared = max_qr > tile_rows;
#define RLX_TREE_NARROW(DD, NN)                                                                                   \
    if (hd == DD && tile_rows == 16 * NN)                                                                         \
        k = fine ? (shared ? tree_narrow_kernel<DD, NN, true, true> : tree_narrow_kernel<DD, NN, true, false>)    \
                 : (shared ? tree_narrow_kernel<DD, NN, false, true> : tree_narrow_kernel<DD, NN, false, false>);
#define RLX_TREE_WIDE(DD, NN, WW, FF) \
    if (hd == DD && tile_rows == 16 * NN * WW && fine == FF) k = tree_wide_kernel<DD, NN, WW, FF>;
    RLX_TREE_NARROW(16, 1)
    RLX_TREE_NARROW(16, 2)
    RLX_TREE_NARROW(32, 1)
    RLX_TREE_NARROW(32, 2)
    RLX_TREE_NARROW(64, 1)
    RLX_TREE_NARROW(64, 2)
    RLX_TREE_NARROW(96, 1)
    RLX_TREE_NARROW(96, 2)
    RLX_TREE_NARROW(128, 1)
    RLX_TREE_NARROW(128, 2)
    RLX_TREE_NARROW(256, 1)
    RLX_TREE_WIDE(64, 1, 4, false)
    RLX_TREE_WIDE(64, 1, 4, true)
    RLX_TREE_WIDE(64, 1, 8, false)
    RLX_TREE_WIDE(64, 1, 8, true)
    RLX_TREE_WIDE(64, 2, 8, false)
    RLX_TREE_WIDE(96, 1, 4, false)
    RLX_TREE_WIDE(96, 1, 4, true)
    RLX_TREE_WIDE(96, 1, 8, false)
    RLX_TREE_WIDE(96, 1, 8, true)
    RLX_TREE_WIDE(96, 2, 8, false)
    RLX_TREE_WIDE(128, 1, 4, false)
    RLX_TREE_WIDE(128, 1, 4, true)
    RLX_TREE_WIDE(128, 1, 8, false)
    RLX_TREE_WIDE(128, 1, 8, true)
    RLX_TREE_WIDE(128, 2, 8, false)
    RLX_TREE_WIDE(256, 1, 4, false)
    RLX_TREE_WIDE(256, 1, 4, true)
#undef RLX_TREE_NARROW
#undef RLX_TREE_WIDE
    if (!k) return hipErrorInvalidValue;
    hipError_t e = launch_timed(k, dim3(n_wgs), dim3(tile_rows <= 64 ? 256 : 512), s, e0, e1, plan, a);
    if (e != hipSuccess || !merge) return e;
    const int TQ = 256 / (hd / 4);
    tree_merge_kernel<<<dim3(a.n_rows, a.KVH, (max_qr + TQ - 1) / TQ), 256, 0, s>>>(plan, a, hd, tile_rows);
    return hipGetLastError();
}

// Moves the accepted nodes' K and V rows of (layer, sequence) blockIdx.x, kv head
// blockIdx.y, dims [32 blockIdx.z, + 32): node path[j] to the tree's slot j, every
// row read before the first is written (a slot may be both).  Latency-bound: 64 bytes of K
// and 32 2-byte elements of V a node.  16 layers of 16 sequences of 24 to 48 nodes, 8 kv
// heads of 128: 19 us.
__global__ __launch_bounds__(256) void tree_keep_kernel(PlanArg plan, const KeepRow *rows, const int32_t *path,
                                                        int path_off, const int32_t *__restrict__ table, int kvh,
                                                        int hd, int P) {
    kconst_i32 *p = plan_ints(rows, blockIdx.x, 8);
    uint16_t *kpool = (uint16_t *)((uint64_t)(uint32_t)p[0] | (uint64_t)(uint32_t)p[1] << 32);
    uint16_t *vpool = (uint16_t *)((uint64_t)(uint32_t)p[2] | (uint64_t)(uint32_t)p[3] << 32);
    const int tab = p[4], base = p[5], n = p[6];
    kconst_i32 *way = (path ? (kconst_i32 *)(uintptr_t)path : (kconst_i32 *)(kernarg_plan() + path_off)) + p[7];
    __shared__ u32x4 sk[kTreeMaxNodes * 4];
    __shared__ uint16_t sv[kTreeMaxNodes * 32];
    __shared__ int64_t from[kTreeMaxNodes], to[kTreeMaxNodes];  // the head's page
    __shared__ int from_slot[kTreeMaxNodes], to_slot[kTreeMaxNodes];
    const int h = blockIdx.y, d0 = blockIdx.z * 32, w = min(32, hd - d0), t = threadIdx.x;
    if (t < n) {
        const auto page = [&](int node, int *slot) {
            const int at = base + node, e = at / P;
            *slot = at - e * P;
            return ((int64_t)table[tab + e] * kvh + h) * P * hd;
        };
        from[t] = page(way[t], &from_slot[t]);
        to[t] = page(t, &to_slot[t]);
    }
    __syncthreads();
    // K: a thread a node and 8 dims; V: a thread a node and dim
    const int kj = t >> 2, kc = (t & 3) * 8, vj = t >> 5, vd = t & 31;
    if (kc < w)
        for (int j = kj; j < n; j += 64)
            sk[j * 4 + (t & 3)] = *(const u32x4 *)(kpool + from[j] + k_page_off(from_slot[j], d0 + kc, hd));
    if (vd < w)
        for (int j = vj; j < n; j += 8) sv[j * 32 + vd] = vpool[from[j] + (int64_t)(d0 + vd) * P + from_slot[j]];
    __syncthreads();
    if (kc < w)
        for (int j = kj; j < n; j += 64)
            *(u32x4 *)(kpool + to[j] + k_page_off(to_slot[j], d0 + kc, hd)) = sk[j * 4 + (t & 3)];
    if (vd < w)
        for (int j = vj; j < n; j += 8) vpool[to[j] + (int64_t)(d0 + vd) * P + to_slot[j]] = sv[j * 32 + vd];
}

hipError_t launch_tree_keep(hipStream_t s, const PlanArg *plan, const KeepRow *rows, const int32_t *path, int path_off,
                            int n_rows, const int32_t *table, int kvh, int hd, int P) {
    if (n_rows <= 0) return hipSuccess;
    static const PlanArg none{};
    tree_keep_kernel<<<dim3(n_rows, kvh, (hd + 31) / 32), 256, 0, s>>>(plan ? *plan : none, rows, path, path_off, table,
                                                                      kvh, hd, P);
    return hipGetLastError();
}

}  // namespace rlx
