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

// Place of (stream, tile) among a row's work-groups.  A stream is one kv head's
// keys of one cut; its tiles read the same keys, so they stand 8 apart: the
// same XCD (work-group b runs on XCD b mod 8), at about the same time.
__device__ __forceinline__ int tree_place(int stream, int tile, int streams, int tiles) {
    const int s0 = stream & ~7, m = min(8, streams - s0);
    return s0 * tiles + tile * m + (stream - s0);
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
// parent outside [0, j) ends the chain.
__device__ __forceinline__ void tree_ancestors(const int32_t *parents, int n, uint32_t (*anc)[kTreeMaxNodes],
                                               int16_t *up) {
    const int j = threadIdx.x, words = (n + 31) >> 5;
    int u = -1;
    if (j < n) {
        const int p = parents[j];
        u = p >= 0 && p < j ? p : -1;
        for (int w = 0; w < words; w++) anc[w][j] = w == (j >> 5) ? 1u << (j & 31) : 0u;
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

// Work-group = (cut of the keys, kv head, tile of query rows): 4 waves, each
// holding all of the tile's 16 NQT query rows and taking every fourth unit of 32
// keys, straight from HBM (or L2) into registers in the operand order of the
// matrix instructions -- no LDS and no barrier in the loop:
//
//   S^T[32 keys][16 rows] = K[32 x D] . Q^T         2 D/32 MFMA 16x16x32 a tile
//   P = exp2(S c - m), lane-local
//   O^T[D][16 rows]      += V^T[D x 32 keys] . P^T  D/16 MFMA 16x16x32 a tile
//
// The 32 keys are two 16-token blocks of the pages; the order in which the
// second product sums them is free, so a lane's 4 + 4 scores of the blocks are
// its 8 operands as they are.
//
// The maximum of a row moves only when a score exceeds it by 2^8 (weights stay
// below 256 in f32 and bf16 alike), so that rescaling and the reduction over
// lanes are rare.
//
// Weights are rounded to bf16 for the second product, and the sum is of the
// rounded ones.  FINE (f32 queries or outputs): queries in three bf16 parts
// (exact), weights in two (2^-17).
//
// A masked weight is a selected zero; a value that is not finite in a masked
// place must not reach other rows through 0 x inf, so such values of the tree's
// keys stay out of the product and are added at the end to the rows that attend
// them (an infinity or NaN whatever its weight).
template <int D, int NQT, bool FINE>
__global__ __launch_bounds__(256, 1) void tree_attend_kernel(PlanArg plan, TreeArgs a) {
    constexpr int KS = D < 32 ? 1 : D / 32;
    constexpr int MT = D / 16;
    constexpr int QP = FINE ? 3 : 1;  // bf16 parts of a query
    constexpr int QT = 16 * NQT;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    __shared__ uint32_t anc[kTreeMaxNodes / 32][kTreeMaxNodes];
    __shared__ int16_t up[kTreeMaxNodes];
    __shared__ float sm[4][QT], sl[4][QT];
    constexpr int MC = MT < 8 ? MT : 8;  // m-tiles merged at a time
    __shared__ fl4 so[4][MC][64];

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
    const TreeRow R = tree_row(a.rows, r);
    const int nodes = R.nodes & 0xFFFF, nq = R.nodes >> 16;
    const int KVH = a.KVH, G = a.H / KVH, QR = nq * G;
    const int tiles = (QR + QT - 1) / QT, streams = R.nsplit * KVH;
    int tile, stream;
    {
        const int i = b - R.wg0, s0 = i / (8 * tiles) * 8, m = min(8, streams - s0), rem = i - s0 * tiles;
        tile = rem / m;
        stream = s0 + rem - tile * m;
    }
    const int split = stream / KVH, kvh = stream - split * KVH;
    const int len = R.len, ctx = len - nodes;  // first key of the tree
    const int units = (len + kTreeKeys - 1) / kTreeKeys;
    const int u0 = (int)((int64_t)split * units / R.nsplit), u1 = (int)((int64_t)(split + 1) * units / R.nsplit);
    const bool has_tree = u1 * kTreeKeys > ctx;
    if (has_tree) tree_ancestors(a.parents + R.node0, nodes, anc, up);

    // ---- this wave's units: u0 + wave, + 4, ... --------------------------------
    const int first = u0 + wave, nu = first < u1 ? (u1 - first + 3) / 4 : 0;
    // Pages and slots of 32 units' blocks, one block a lane.  A block past the
    // last token reads the last token's (its keys are masked).
    int pg = 0, sl0 = 0;
    auto fetch_pages = [&](int j0) {
        const int j = j0 + (lane >> 1);
        int t = (first + 4 * min(j, nu - 1)) * kTreeKeys + 16 * (lane & 1);
        t = min(t, (len - 1) & ~15);
        const int e = a.pshift >= 0 ? t >> a.pshift : t / a.P;
        pg = a.table[R.tab + e];
        sl0 = t - e * a.P;
    };
    if (nu > 0) fetch_pages(0);
    asm volatile("" ::"v"(pg), "v"(sl0));

    // ---- queries: B operand, lane (row col, dims grp * 8 ..) -------------------
    u32x4 qb[NQT][KS][QP];
    int node[NQT];  // the row's node; rows past the tile's hold zeros
#pragma unroll
    for (int nt = 0; nt < NQT; nt++) {
        const int qr = tile * QT + nt * 16 + col;
        const bool ok = qr < QR;
        const int qc = ok ? qr : 0;
        node[nt] = nodes - nq + qc / G;
        const int64_t base = tree_qbase(a, R, kvh, G, qc);
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const int d0 = ks * 32 + grp * 8;
            const bool in = ok && d0 < a.DQ;
            float v[8];
            if (a.q_bf16) {
                const u32x4 w = in ? *(const u32x4 *)((const uint16_t *)a.q + base + d0) : u32x4{0, 0, 0, 0};
                qb[nt][ks][0] = w;
                if constexpr (FINE) qb[nt][ks][1] = qb[nt][ks][2] = u32x4{0, 0, 0, 0};
                continue;
            }
            const float4 x = in ? *(const float4 *)((const float *)a.q + base + d0) : float4{0.f, 0.f, 0.f, 0.f};
            const float4 y = in ? *(const float4 *)((const float *)a.q + base + d0 + 4) : float4{0.f, 0.f, 0.f, 0.f};
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
#pragma unroll
            for (int p = 0; p < QP; p++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint16_t h0 = bf16_rne(v[2 * i]), h1 = bf16_rne(v[2 * i + 1]);
                    qb[nt][ks][p][i] = (uint32_t)h0 | ((uint32_t)h1 << 16);
                    v[2 * i] -= bf16_f32(h0);
                    v[2 * i + 1] -= bf16_f32(h1);
                }
        }
    }

    float m_run[NQT], l_part[NQT];
    fl4 acc[NQT][MT];
#pragma unroll
    for (int nt = 0; nt < NQT; nt++) {
        m_run[nt] = -INFINITY;
        l_part[nt] = 0.f;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) acc[nt][mt] = fl4{0.f, 0.f, 0.f, 0.f};
    }

    const int64_t head = (int64_t)a.P * D;  // one kv head of one page
    const uint32_t k_lane = (D == 16 ? col * 16 + (grp & 1) * 8 : col * 32 + grp * 8) * 2u;  // bytes
    uint32_t v_lane[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) v_lane[mt] = (uint32_t)((mt * 16 + col) * a.P + grp * 4) * 2u;
    auto load_unit = [&](int j, u32x4(&kr)[2][KS], u32x4(&vr)[MT]) {
        j = min(j, nu - 1);
        if ((j & 31) == 0 && j) {
            fetch_pages(j);
            asm volatile("" ::"v"(pg), "v"(sl0));
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int src = (2 * j + k) & 63;
            const int page = __builtin_amdgcn_readlane(pg, src), slot = __builtin_amdgcn_readlane(sl0, src);
            const int64_t base = ((int64_t)page * KVH + kvh) * head;
            const char *kp = (const char *)(a.kpool + base + (int64_t)slot * D);
            const char *vp = (const char *)(a.vpool + base + slot);
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                kr[k][ks] = __builtin_nontemporal_load((const u32x4 *)(kp + (k_lane + ks * 1024)));
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                const u32x2 w = __builtin_nontemporal_load((const u32x2 *)(vp + v_lane[mt]));
                vr[mt][2 * k] = w[0];
                vr[mt][2 * k + 1] = w[1];
            }
        }
    };

    // Key i of block k in a lane: t0 + 16 k + 4 grp + i.
    auto allowed = [&](int t, int nt) {
        if (t < ctx) return true;
        const int k = t - ctx;
        return t < len && ((anc[k >> 5][node[nt]] >> (k & 31)) & 1u);
    };

    bool odd = false;  // a value of the tree's keys that is not finite
    // tree: a unit that holds keys of the tree (or past the last token)
    auto consume = [&](auto tree, int j, u32x4(&kr)[2][KS], u32x4(&vr)[MT]) {
        constexpr bool TREE = decltype(tree)::value;
        const int t0 = (first + 4 * j) * kTreeKeys;
        if constexpr (TREE) {
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = t0 + 16 * k + 4 * grp + i;
                    const uint32_t keep = (i & 1) ? 0x0000FFFFu : 0xFFFF0000u;
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        const uint32_t w = vr[mt][2 * k + (i >> 1)] & ~keep, ex = 0x7F807F80u & ~keep;
                        const bool inf = t >= ctx && (w & ex) == ex;
                        odd |= inf && t < len;
                        if (t >= len || inf) vr[mt][2 * k + (i >> 1)] &= keep;
                    }
                }
        }
        if (D == 16) {
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (grp >= 2) kr[k][0] = u32x4{0, 0, 0, 0};
        }
        fl4 s[NQT][2];
#pragma unroll
        for (int nt = 0; nt < NQT; nt++) s[nt][0] = s[nt][1] = fl4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int p = QP - 1; p >= 0; p--)
#pragma unroll
                for (int nt = 0; nt < NQT; nt++)
#pragma unroll
                    for (int k = 0; k < 2; k++)
                        s[nt][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[k][ks]),
                                                                          __builtin_bit_cast(bf16x8, qb[nt][ks][p]),
                                                                          s[nt][k], 0, 0, 0);
        if constexpr (FINE) {
            // An infinite key against a query's parts of both signs is a NaN; its
            // score is the first part's.
            float sum = 0.f;
#pragma unroll
            for (int nt = 0; nt < NQT; nt++)
#pragma unroll
                for (int i = 0; i < 8; i++) sum += s[nt][i >> 2][i & 3];
            if (__builtin_amdgcn_ballot_w64(sum != sum)) {
#pragma unroll
                for (int nt = 0; nt < NQT; nt++)
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        fl4 h = fl4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int ks = 0; ks < KS; ks++)
                            h = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[k][ks]),
                                                                        __builtin_bit_cast(bf16x8, qb[nt][ks][0]), h,
                                                                        0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (s[nt][k][i] != s[nt][k][i]) s[nt][k][i] = h[i];
                    }
            }
        }
        if constexpr (TREE) {
#pragma unroll
            for (int nt = 0; nt < NQT; nt++)
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (!allowed(t0 + 16 * k + 4 * grp + i, nt)) s[nt][k][i] = -INFINITY;
        }
        float mx[NQT];
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NQT; nt++) {
            mx[nt] = fmaxf(fmaxf(fmaxf(s[nt][0][0], s[nt][0][1]), fmaxf(s[nt][0][2], s[nt][0][3])),
                           fmaxf(fmaxf(s[nt][1][0], s[nt][1][1]), fmaxf(s[nt][1][2], s[nt][1][3])));
            grow |= mx[nt] * a.qscale > m_run[nt] + 8.f;
        }
        if (__builtin_amdgcn_ballot_w64(grow)) {
#pragma unroll
            for (int nt = 0; nt < NQT; nt++) {
                const float m_new = fmaxf(m_run[nt], rows4_max(mx[nt]) * a.qscale);
                const float c = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run[nt] - m_new);
                m_run[nt] = m_new;
                l_part[nt] *= c;
#pragma unroll
                for (int mt = 0; mt < MT; mt++) acc[nt][mt] *= c;
            }
        }
#pragma unroll
        for (int nt = 0; nt < NQT; nt++) {
            const float m = m_run[nt] == -INFINITY ? 0.f : m_run[nt];
            u32x4 pw, pl;
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = __builtin_amdgcn_exp2f(fmaf(s[nt][i >> 2][i & 3], a.qscale, -m));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                pw[i] = pack_bf16x2(p[2 * i], p[2 * i + 1]);
                if constexpr (FINE) {
                    pl[i] = pack_bf16x2(p[2 * i] - bf16_lo(pw[i]), p[2 * i + 1] - bf16_hi(pw[i]));
                    l_part[nt] += p[2 * i] + p[2 * i + 1];
                } else {
                    l_part[nt] = add_bf16x2(pw[i], l_part[nt]);
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                if constexpr (FINE)
                    acc[nt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, vr[mt]), __builtin_bit_cast(bf16x8, pl), acc[nt][mt], 0, 0, 0);
                acc[nt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8, vr[mt]), __builtin_bit_cast(bf16x8, pw), acc[nt][mt], 0, 0, 0);
            }
        }
    };
    using Ctx = std::integral_constant<bool, false>;
    using Tree = std::integral_constant<bool, true>;

    // Two register sets alternate, so that the next unit's loads are in flight
    // while one is consumed (past the last unit they read it again).  Stored head
    // dim 256 has registers for one.
    const int nc = max(0, min(nu, (ctx / kTreeKeys - first + 3) / 4));  // units before the tree's
    u32x4 ka[2][KS], kb[2][KS];
    u32x4 va[MT], vb[MT];
    int j = 0;
    if constexpr (D <= 128) {
        if (nu > 0) load_unit(0, ka, va);
        for (; j + 1 < nc; j += 2) {
            load_unit(j + 1, kb, vb);
            consume(Ctx{}, j, ka, va);
            load_unit(j + 2, ka, va);
            consume(Ctx{}, j + 1, kb, vb);
        }
        for (; j < nu; j++) {
            load_unit(j + 1, kb, vb);
            if (j < nc)
                consume(Ctx{}, j, ka, va);
            else
                consume(Tree{}, j, ka, va);
#pragma unroll
            for (int i = 0; i < KS; i++) ka[0][i] = kb[0][i], ka[1][i] = kb[1][i];
#pragma unroll
            for (int i = 0; i < MT; i++) va[i] = vb[i];
        }
    } else {
        for (; j < nc; j++) {
            load_unit(j, ka, va);
            consume(Ctx{}, j, ka, va);
        }
        for (; j < nu; j++) {
            load_unit(j, ka, va);
            consume(Tree{}, j, ka, va);
        }
    }

    // ---- merge of the 4 waves --------------------------------------------------
#pragma unroll
    for (int nt = 0; nt < NQT; nt++) {
        const float l = rows4_sum(l_part[nt]);
        if (grp == 0) {
            sm[wave][nt * 16 + col] = m_run[nt];
            sl[wave][nt * 16 + col] = l;
        }
    }
    const bool any_odd = __syncthreads_or(odd);
    const int slot = R.part + b - R.wg0;
#pragma unroll
    for (int nt = 0; nt < NQT; nt++) {
        const int qt = nt * 16 + col, qr = tile * QT + qt;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) M = fmaxf(M, sm[w][qt]);
#pragma unroll
        for (int w = 0; w < 4; w++) L += sm[w][qt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[w][qt] - M) * sl[w][qt];
        const float f = m_run[nt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[nt] - M);
        const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
        for (int m0 = 0; m0 < MT; m0 += MC) {
            if (nt || m0) __syncthreads();
#pragma unroll
            for (int mt = 0; mt < MC; mt++) so[wave][mt][lane] = acc[nt][m0 + mt] * f;
            __syncthreads();
            for (int mt = wave; mt < MC; mt += 4) {
                fl4 o = (so[0][mt][lane] + so[1][mt][lane]) + (so[2][mt][lane] + so[3][mt][lane]);
                const int d0 = (m0 + mt) * 16 + grp * 4;
                if (any_odd) {
#pragma unroll 1
                    for (int t = max(u0 * kTreeKeys, ctx); t < min(u1 * kTreeKeys, len); t++) {
                        if (!allowed(t, nt)) continue;
                        const int e = t / a.P;
                        const uint16_t *vp = a.vpool + ((int64_t)a.table[R.tab + e] * KVH + kvh) * head + (t - e * a.P);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint16_t w = vp[(d0 + i) * a.P];
                            if ((w & 0x7F80) == 0x7F80) o[i] += bf16_f32(w);
                        }
                    }
                }
                if (R.nsplit > 1) {
                    *(fl4 *)(a.part_o + ((int64_t)slot * QT + qt) * D + d0) = o;
                } else if (qr < QR && d0 < a.DQ) {
                    const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
                    tree_store4(a.out, tree_qbase(a, R, kvh, G, qr) + d0, v, a.out_bf16);
                }
            }
        }
        if (R.nsplit > 1 && wave == 0 && grp == 0) {
            float *pm = a.part_ml + ((int64_t)slot * QT + qt) * 2;
            pm[0] = M;
            pm[1] = L;
        }
    }
}

// Joins the partials of the sequences whose keys were cut: a thread holds 4 dims
// of a query row.  out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.
__global__ __launch_bounds__(256) void tree_merge_kernel(PlanArg plan, TreeArgs a, int D, int QT) {
    const TreeRow R = tree_row(a.rows, blockIdx.x);
    if (R.nsplit <= 1) return;
    const int G = a.H / a.KVH, nq = R.nodes >> 16, QR = nq * G, kvh = blockIdx.y;
    const int Q4 = D >> 2, TQ = 256 / Q4, t = threadIdx.x;
    const int qr = blockIdx.z * TQ + t / Q4, d0 = (t - t / Q4 * Q4) * 4;
    if (t >= TQ * Q4 || qr >= QR) return;
    const int tiles = (QR + QT - 1) / QT, streams = R.nsplit * a.KVH, tile = qr / QT, qt = qr - tile * QT;
    const auto at = [&](int s) {
        return ((int64_t)R.part + tree_place(s * a.KVH + kvh, tile, streams, tiles)) * QT + qt;
    };
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

int tree_tile_rows(int hd, int max_qr, bool fine) {
    if (hd > 128 || max_qr <= 16) return 16;
    return max_qr <= 32 || fine || hd > 64 ? 32 : 64;
}

hipError_t launch_tree_attend(hipStream_t s, const PlanArg &plan, const TreeArgs &a, int hd, int tile_rows,
                              bool fine, int n_wgs, bool merge, int max_qr, hipEvent_t e0, hipEvent_t e1) {
    if (n_wgs <= 0) return hipSuccess;
    void (*k)(PlanArg, TreeArgs) = nullptr;
#define RLX_TREE_CASE(DD, NN)                                                              \
    if (hd == DD && tile_rows == 16 * NN)                                                  \
        k = fine ? tree_attend_kernel<DD, (NN < 4 ? NN : 2), true> : tree_attend_kernel<DD, NN, false>;
    RLX_TREE_CASE(16, 1)
    RLX_TREE_CASE(16, 2)
    RLX_TREE_CASE(16, 4)
    RLX_TREE_CASE(32, 1)
    RLX_TREE_CASE(32, 2)
    RLX_TREE_CASE(32, 4)
    RLX_TREE_CASE(64, 1)
    RLX_TREE_CASE(64, 2)
    RLX_TREE_CASE(64, 4)
    RLX_TREE_CASE(96, 1)
    RLX_TREE_CASE(96, 2)
    RLX_TREE_CASE(96, 4)
    RLX_TREE_CASE(128, 1)
    RLX_TREE_CASE(128, 2)
    RLX_TREE_CASE(128, 4)
    RLX_TREE_CASE(256, 1)
#undef RLX_TREE_CASE
    if (!k) return hipErrorInvalidValue;
    hipError_t e = launch_timed(k, dim3(n_wgs), dim3(256), s, e0, e1, plan, a);
    if (e != hipSuccess || !merge) return e;
    const int TQ = 256 / (hd / 4);
    tree_merge_kernel<<<dim3(a.n_rows, a.KVH, (max_qr + TQ - 1) / TQ), 256, 0, s>>>(plan, a, hd, tile_rows);
    return hipGetLastError();
}

// Moves the accepted nodes' K and V rows of (layer, sequence) blockIdx.x, kv head
// blockIdx.y, dims [32 blockIdx.z, + 32): node path[j] to the tree's slot j, every
// row read before the first is written (a slot may be both).  Latency-bound: 64 bytes of K
// and 32 2-byte elements of V a node.
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
    const int h = blockIdx.y, d0 = blockIdx.z * 32, w = min(32, hd - d0), kc = w / 8;
    const auto page = [&](int node, int *slot) {
        const int t = base + node, e = t / P;
        *slot = t - e * P;
        return ((int64_t)table[tab + e] * kvh + h) * P * hd;
    };
    for (int i = threadIdx.x; i < n * kc; i += 256) {
        const int j = i / kc, c = i - j * kc;
        int s;
        const int64_t pb = page(way[j], &s);
        sk[j * 4 + c] = *(const u32x4 *)(kpool + pb + k_page_off(s, d0 + c * 8, hd));
    }
    for (int i = threadIdx.x; i < n * w; i += 256) {
        const int d = i / n, j = i - d * n;
        int s;
        const int64_t pb = page(way[j], &s);
        sv[d * n + j] = vpool[pb + (int64_t)(d0 + d) * P + s];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * kc; i += 256) {
        const int j = i / kc, c = i - j * kc;
        int s;
        const int64_t pb = page(j, &s);
        *(u32x4 *)(kpool + pb + k_page_off(s, d0 + c * 8, hd)) = sk[j * 4 + c];
    }
    for (int i = threadIdx.x; i < n * w; i += 256) {
        const int d = i / n, j = i - d * n;
        int s;
        const int64_t pb = page(j, &s);
        vpool[pb + (int64_t)(d0 + d) * P + s] = sv[d * n + j];
    }
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
