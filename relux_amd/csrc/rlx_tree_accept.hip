// Acceptance of a tree of drafts: the walk from the root along accepted nodes, and
// the draw of the token after the last one.
//
// At node v with target p = softmax(t_v / T) and draft q = softmax(d_v / T), v's
// children are tried in order; they were drawn from q without replacement.  With
// p_1 = p and q_1 = q, child i (token x, uniform u) is accepted when
//
//   u q_i(x) < p_i(x),
//
// else p_{i+1} = max(0, p_i - q_i) / sum, and q_{i+1} is q_i without x, rescaled.
// After the last rejection the next token is drawn from what p has become.  The
// result is distributed as the target alone would draw it.
//
// q_i is q / S_i off the rejected tokens, S_i = 1 - sum of their q, and repeated
// subtraction with a floor of zero is one: p_i ~ max(0, p - C_i q) with C_1 = 0,
// C_{i+1} = C_i + A_i / S_i, A_i = sum max(0, p - C_i q) (a rejected token's value
// is zero from its rejection on).  So a rejection costs one pass over the two
// rows and no distribution is stored.
//
// Without draft logits a draft is a choice without a distribution (q_i = the
// child's token): accepted when u A_i < p(x), else its probability is removed.
//
// Weights are exp2((l - m) log2(e) / T) in f32, m near the row's maximum, sums over
// the vocabulary in f64: a draw's place among V tokens moves by V times a sum's
// rounding.
#include "rlx_tree.h"

namespace rlx {

typedef __attribute__((address_space(4))) const int32_t kconst_i32;
constexpr int kAccWaves = 16, kAccThreads = 64 * kAccWaves;

namespace {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

// Entries i .. i + 3 of a row's [0, end): `full`, all inside; else -inf past the end.
__device__ __forceinline__ float4 acc_load4(const float *row, int i, int end, bool full) {
    if (full) {
        const f4u v = *(const f4u *)(row + i);
        return make_float4(v[0], v[1], v[2], v[3]);
    }
    float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (i < end) v.x = row[i];
    if (i + 1 < end) v.y = row[i + 1];
    if (i + 2 < end) v.z = row[i + 2];
    if (i + 3 < end) v.w = row[i + 3];
    return v;
}

// Weight of a logit: exp2(l k - m k), mk = m k rounded once for the whole row.
__device__ __forceinline__ float acc_e(float l, float k, float mk) { return __builtin_amdgcn_exp2f(fmaf(l, k, -mk)); }

// v of the lane that a row move (16 lanes) takes; 0 where it takes none or the row is masked.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ float row_move(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ double row_move(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, false),
                   hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_of(double v, int lane) {  // lane: the same in every lane
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
constexpr int kRor = 0x120, kShr = 0x110, kBcast15 = 0x142, kBcast31 = 0x143;  // rotate and shift within a row; a row's last lane to later ones

// Over the 16 lanes of a row, the same in each.
__device__ __forceinline__ double row_sum(double v) {
    v += row_move<kRor + 8>(v);
    v += row_move<kRor + 4>(v);
    v += row_move<kRor + 2>(v);
    return v + row_move<kRor + 1>(v);
}
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, row_move<kRor + 8>(v));
    v = fmaxf(v, row_move<kRor + 4>(v));
    v = fmaxf(v, row_move<kRor + 2>(v));
    return fmaxf(v, row_move<kRor + 1>(v));
}
// Over the wave.
__device__ __forceinline__ double wave_sum(double v) {
    v = row_sum(v);
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
__device__ __forceinline__ float wave_max(float v) { return rows4_max(row_max(v)); }
// Sums of lanes 0 .. lane.
__device__ __forceinline__ double wave_scan(double v) {
    v += row_move<kShr + 1>(v);
    v += row_move<kShr + 2>(v);
    v += row_move<kShr + 4>(v);
    v += row_move<kShr + 8>(v);
    v += row_move<kBcast15, 0xA>(v);
    return v + row_move<kBcast31, 0xC>(v);
}

// A condition that is the same in every lane, as a scalar one.
__device__ __forceinline__ bool same(bool c) { return __builtin_amdgcn_ballot_w64(c) != 0; }

constexpr int kAccBatch = 4;  // float4 of a row a lane has in flight

// A wave's sum of exp2(l k - mk), mk of the wave's first batch's maximum unless a
// later entry exceeds it by 2^60.  kNone: only -inf so far, below any other maximum
// and finite, so that -inf - mk is -inf.
constexpr float kNone = -3e38f;
struct Online {
    float mk = kNone;
    double s = 0.0;  // this lane's
    __device__ __forceinline__ void add(const float4 (&v)[kAccBatch], float k, bool first) {
        float x = -INFINITY;
#pragma unroll
        for (int i = 0; i < kAccBatch; i++) x = fmaxf(x, fmaxf(fmaxf(v[i].x, v[i].y), fmaxf(v[i].z, v[i].w)));
        if (first || __builtin_amdgcn_ballot_w64(x * k > mk + 60.f)) {
            const float to = fmaxf(wave_max(x) * k, kNone);
            if (!first) s *= (double)__builtin_amdgcn_exp2f(mk - to);
            mk = to;
        }
        float sum[kAccBatch];
#pragma unroll
        for (int i = 0; i < kAccBatch; i++)
            sum[i] = (acc_e(v[i].x, k, mk) + acc_e(v[i].y, k, mk)) + (acc_e(v[i].z, k, mk) + acc_e(v[i].w, k, mk));
        s += (double)((sum[0] + sum[1]) + (sum[2] + sum[3]));
    }
};

struct RowStat {
    float mk;
    double z;
};

}  // namespace

// One work-group a sequence: the walk reads the rows of the accepted path alone, each
// once the node before it is decided.  Bound by that chain of passes, at most one a
// node of the path and one a rejection: V / 4 entries a SIMD, half of the time their
// exponentials and sums, half a row's latency and the joins.  64 trees of 32 nodes, 32000
// tokens: 45 to 52 us, up to 7 passes; 12 of 9 to 61, 50257 tokens: 63 to 70 us; one of 8
// without draft logits, 32000 tokens: 13 us.  16 waves: 8 take 46 and 64 us, 4 take 69 and 91;
// batches of 8 loads instead of 4, 62 and 76.  Weights of 16 float4 a lane kept in
// registers between passes: 43 and 67, for a second form of every pass.
template <bool Q>
__global__ __launch_bounds__(kAccThreads) void tree_accept_kernel(PlanArg plan, TreeAcceptArgs a) {
    __shared__ int par[kTreeMaxNodes], tok[kTreeMaxNodes], gone[kTreeMaxNodes], way[kTreeMaxNodes];
    __shared__ float uni[kTreeMaxNodes], lt[kTreeMaxNodes], lq[kTreeMaxNodes];
    __shared__ float red_m[2][2][kAccWaves];  // the waves' sums, two passes in turn: one barrier a pass
    __shared__ double red_s[2][2][kAccWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int first, n;
    {
        kconst_i32 *p = (a.trees ? (kconst_i32 *)(uintptr_t)a.trees : (kconst_i32 *)kernarg_plan()) + 2 * blockIdx.x;
        first = p[0];
        n = p[1];
    }
    const int V = a.V;
    const float k = 1.4426950408889634f / a.temperature;
    // (used when the root's rows have been read)
    int my_par = 0, my_tok = 0;
    float my_u = 0.f;
    if (tid < n) {
        my_par = a.parents[first + tid];
        my_tok = a.tok[first + tid];
        my_u = a.u[first + tid];
    }

    // Wave w covers entries [w * span, (w + 1) * span) of a row, 256 at a time.
    const int span = (V + kAccWaves * 256 - 1) / (kAccWaves * 256) * 256;
    const int v0 = min(V, wave * span), v1 = min(V, v0 + span);
    int cur = 0, steps = 0, n_gone = 0;
    if (tid == 0) way[0] = 0;
    const float *t, *d;
    RowStat T{0.f, 0.0}, D{0.f, 1.0};
    double C, S, A;  // A in units of the target's weights (p's mass = T.z)
    bool subtract = false;  // ratio > 0
    float ratio;     // C in those units: max(0, e_t - ratio e_q)
    auto rest = [&](float et, float eq) __attribute__((always_inline)) {
        return Q ? fmaxf(0.f, fmaf(-ratio, eq, et)) : et;
    };
    auto load = [&](const float *row, float4 (&v)[kAccBatch], int base, int end) __attribute__((always_inline)) {
        const bool full = base + kAccBatch * 256 <= end;
#pragma unroll
        for (int i = 0; i < kAccBatch; i++) v[i] = acc_load4(row, base + i * 256 + lane * 4, end, full);
    };
    // Sum of what remains of entries [lo, hi) by this wave's lanes, the rejected
    // tokens left out where they have no distribution.
    auto mass = [&](int lo, int hi) {
        double s = 0.0;
        for (int base = lo; base < hi; base += kAccBatch * 256) {
            float4 x[kAccBatch], y[kAccBatch];
            load(t, x, base, hi);
            if (Q && subtract) load(d, y, base, hi);
            float sum[kAccBatch];
#pragma unroll
            for (int i = 0; i < kAccBatch; i++) {
                float e[4] = {acc_e(x[i].x, k, T.mk), acc_e(x[i].y, k, T.mk), acc_e(x[i].z, k, T.mk), acc_e(x[i].w, k, T.mk)};
                if (Q && subtract) {
                    e[0] = rest(e[0], acc_e(y[i].x, k, D.mk));
                    e[1] = rest(e[1], acc_e(y[i].y, k, D.mk));
                    e[2] = rest(e[2], acc_e(y[i].z, k, D.mk));
                    e[3] = rest(e[3], acc_e(y[i].w, k, D.mk));
                }
                if (!Q) {
                    for (int g = 0; g < n_gone; g++) {
                        const int at = gone[g] - (base + i * 256 + lane * 4);
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            if (at == c) e[c] = 0.f;
                    }
                }
                sum[i] = (e[0] + e[1]) + (e[2] + e[3]);
            }
            s += (double)((sum[0] + sum[1]) + (sum[2] + sum[3]));
        }
        return s;
    };
    int turn = 0;
    double waves;  // lane w of a row: what remains in wave w's span
    // Sum of what remains over the row.
    auto total = [&]() {
        const double s = wave_sum(mass(v0, v1));
        turn ^= 1;
        if (lane == 0) red_s[turn][0][wave] = s;
        __syncthreads();
        waves = red_s[turn][0][lane & 15];
        return row_sum(waves);
    };

    for (;;) {
        t = a.t_logits + (int64_t)(first + cur) * a.t_stride;
        d = Q ? a.d_logits + (int64_t)(first + cur) * a.d_stride : nullptr;
        // this node's children, and their logits
        uint64_t kids[kTreeMaxNodes / 64];
        float my_t = 0.f, my_d = 0.f;
        bool mine = false;
        auto children = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int w = 0; w < kTreeMaxNodes / 64; w++) {
                const int j = w * 64 + lane;
                kids[w] = __builtin_amdgcn_ballot_w64(j > cur && j < n && par[j] == cur);
            }
            mine = tid > cur && tid < n && par[tid] == cur && tok[tid] >= 0 && tok[tid] < V;
            if (mine) {
                my_t = t[tok[tid]];
                if (Q) my_d = d[tok[tid]];
            }
        };
        // the rows' masses (the draft's only where there are children)
        bool parent = Q && n > 1;
        if (steps > 0) {
            children();
            parent = Q && (kids[0] | kids[1] | kids[2] | kids[3]);
        }
        Online ot, oq;
        for (int base = v0; base < v1; base += kAccBatch * 256) {
            float4 x[kAccBatch], y[kAccBatch];
            load(t, x, base, v1);
            if (parent) load(d, y, base, v1);
            ot.add(x, k, base == v0);
            if (parent) oq.add(y, k, base == v0);
        }
        turn ^= 1;
        auto fold = [&](Online &o, int side) {
            const double z = wave_sum(o.s);
            if (lane == 0) {
                red_m[turn][side][wave] = o.mk;
                red_s[turn][side][wave] = z;
            }
        };
        fold(ot, 0);
        if (parent) fold(oq, 1);
        if (steps == 0) {
            if (tid < n) {
                par[tid] = my_par;
                tok[tid] = my_tok;
                uni[tid] = my_u;
            }
            __syncthreads();
            children();
        }
        if (mine) {
            lt[tid] = my_t;
            if (Q) lq[tid] = my_d;
        }
        __syncthreads();
        auto join = [&](int side, double &each) {
            const float m = red_m[turn][side][lane & 15], mk = row_max(m);
            each = red_s[turn][side][lane & 15] * (double)__builtin_amdgcn_exp2f(m - mk);
            return RowStat{mk, row_sum(each)};
        };
        T = join(0, waves);
        if (parent) {
            double each;
            D = join(1, each);
        }
        C = 0.0;
        S = 1.0;
        A = T.z;
        ratio = 0.f;
        subtract = false;
        n_gone = 0;
        int went = -1;
#pragma unroll 1
        for (int w = 0; w < kTreeMaxNodes / 64 && went < 0; w++) {
            uint64_t left = w == 0 ? kids[0] : w == 1 ? kids[1] : w == 2 ? kids[2] : kids[3];
            while (left) {
                const int c = w * 64 + __builtin_ctzll(left);
                left &= left - 1;
                const int x = __builtin_amdgcn_readfirstlane(tok[c]);
                bool skip = x < 0 || x >= V;  // no token: rejected without effect, as a rejected token again is
                for (int g = lane; g < n_gone; g += 64) skip |= gone[g] == x;
                if (same(skip)) continue;
                const float et = acc_e(lt[c], k, T.mk);
                if constexpr (Q) {
                    const float eq = acc_e(lq[c], k, D.mk);
                    const double qx = (double)eq / D.z, px = (double)rest(et, eq);
                    if (same(S > 0.0 ? (double)uni[c] * qx * A < px * S : px > 0.0)) {
                        went = c;
                        break;
                    }
                    if (tid == 0) gone[n_gone] = x;
                    n_gone++;
                    if (same(S > 0.0)) {
                        C += A / T.z / S;
                        S -= qx;
                        ratio = (float)fmin(C * T.z / D.z, 3e38);  // (finite: 0 where a draft weight is 0)
                        subtract = true;
                        A = total();
                        if (same(!(A > 0.0))) {  // nothing is left by rounding alone
                            C = 0.0;
                            ratio = 0.f;
                            subtract = false;
                            A = total();
                        }
                    } else {
                        __syncthreads();
                    }
                } else {
                    if (same((double)uni[c] * A < (double)et)) {
                        went = c;
                        break;
                    }
                    A -= (double)et;
                    if (tid == 0) gone[n_gone] = x;
                    n_gone++;
                    __syncthreads();
                }
            }
        }
        if (went < 0) break;
        cur = went;
        steps++;
        if (tid == 0) way[steps] = cur;
    }

    // ---- the next token: the first whose cumulated mass exceeds u A --------------
    if (!Q && n_gone) A = total();
    double want = (double)uni[0] * A;
    // Which of `waves` `want` falls in (else the last that holds any); want becomes
    // what is left of it there.
    auto pick = [&]() {
        const double s = lane < kAccWaves ? fmax(waves, 0.0) : 0.0, c = wave_scan(s);
        const uint64_t any = __builtin_amdgcn_ballot_w64(s > 0.0), over = __builtin_amdgcn_ballot_w64(s > 0.0 && c > want);
        const int w = over ? __builtin_ctzll(over) : any ? 63 - __builtin_clzll(any) : 0;
        want -= lane_of(c - s, w);
        return w;
    };
    // the wave's span again by all the waves, then a part of it by one
    int lo = pick() * span;
    const int sub = span / kAccWaves, hi = min(V, lo + span);
    const int s0 = min(hi, lo + wave * sub), s1 = min(hi, s0 + sub);
    {
        const double s = wave_sum(mass(s0, s1));
        turn ^= 1;
        if (lane == 0) red_s[turn][0][wave] = s;
    }
    __syncthreads();
    waves = red_s[turn][0][lane & 15];
    const int owner = pick();
    if (wave == owner) {
        int found = -1, some = -1;
        for (int base = s0; base < s1 && found < 0; base += 256) {
            const int at = base + lane * 4;
            const bool full = base + 256 <= s1;
            const float4 x = acc_load4(t, at, s1, full);
            float e[4] = {acc_e(x.x, k, T.mk), acc_e(x.y, k, T.mk), acc_e(x.z, k, T.mk), acc_e(x.w, k, T.mk)};
            if (Q && subtract) {
                const float4 y = acc_load4(d, at, s1, full);
                e[0] = rest(e[0], acc_e(y.x, k, D.mk));
                e[1] = rest(e[1], acc_e(y.y, k, D.mk));
                e[2] = rest(e[2], acc_e(y.z, k, D.mk));
                e[3] = rest(e[3], acc_e(y.w, k, D.mk));
            }
            for (int g = 0; !Q && g < n_gone; g++)
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (gone[g] == at + c) e[c] = 0.f;
            const double s = (double)((e[0] + e[1]) + (e[2] + e[3])), c = wave_scan(s);
            // this lane's first entry past `want`, and its last that holds any
            double run = c - s;
            int hit = -1, any = -1;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                run += (double)e[i];
                if (!(e[i] > 0.f)) continue;
                any = at + i;
                if (hit < 0 && run > want) hit = at + i;
            }
            const uint64_t hits = __builtin_amdgcn_ballot_w64(hit >= 0), anys = __builtin_amdgcn_ballot_w64(any >= 0);
            if (hits) found = __builtin_amdgcn_readlane(hit, __builtin_ctzll(hits));
            if (anys) some = __builtin_amdgcn_readlane(any, 63 - __builtin_clzll(anys));
            want -= lane_of(c, 63);
        }
        if (lane == 0) {
            a.n_acc[blockIdx.x] = steps;
            // (rows that hold no probability: some token of the vocabulary)
            a.next[blockIdx.x] = found >= 0 ? found : some >= 0 ? some : min(s0, V - 1);
        }
    }
    for (int i = tid; i < a.path_stride; i += kAccThreads)
        a.path[(int64_t)blockIdx.x * a.path_stride + i] = i <= steps ? way[i] : -1;
}

hipError_t launch_tree_accept(hipStream_t s, const PlanArg *plan, const TreeAcceptArgs &a, int n_seqs,
                              hipEvent_t e0, hipEvent_t e1) {
    if (n_seqs <= 0) return hipSuccess;
    static const PlanArg none{};
    auto k = a.d_logits ? tree_accept_kernel<true> : tree_accept_kernel<false>;
    return launch_timed(k, dim3(n_seqs), dim3(kAccThreads), s, e0, e1, plan ? *plan : none, a);
}

}  // namespace rlx
