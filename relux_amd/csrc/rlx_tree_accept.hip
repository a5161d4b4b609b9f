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
// Weights are e = exp2((l - max) log2(e) / T) in f32, sums over the vocabulary in
// f64: a draw's place among V tokens moves by V times a sum's rounding.
#include "rlx_tree.h"

namespace rlx {

typedef __attribute__((address_space(4))) const int32_t kconst_i32;
constexpr int kAccWaves = 16, kAccThreads = 64 * kAccWaves;

namespace {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

// Entries i .. i + 3 of a row, -inf past the end.
__device__ __forceinline__ float4 acc_load4(const float *row, int i, int end) {
    if (i + 4 <= end) {
        const f4u v = *(const f4u *)(row + i);
        return make_float4(v[0], v[1], v[2], v[3]);
    }
    float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (i < end) v.x = row[i];
    if (i + 1 < end) v.y = row[i + 1];
    if (i + 2 < end) v.z = row[i + 2];
    return v;
}

__device__ __forceinline__ float acc_e(float l, float m, float k) { return __builtin_amdgcn_exp2f((l - m) * k); }

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// A thread's running maximum and sum of exp2((l - max) k).
struct Online {
    float m = -INFINITY;
    double s = 0.0;
    __device__ __forceinline__ void add(const float4 &v, float k) {
        const float x = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
        if (x > m) {
            s *= (double)acc_e(m, x, k);
            m = x;
        }
        if (m > -INFINITY) s += (double)((acc_e(v.x, m, k) + acc_e(v.y, m, k)) + (acc_e(v.z, m, k) + acc_e(v.w, m, k)));
    }
};

struct RowStat {
    float m;
    double z;
};

}  // namespace

template <bool Q>
__global__ __launch_bounds__(kAccThreads) void tree_accept_kernel(PlanArg plan, TreeAcceptArgs a) {
    __shared__ int par[kTreeMaxNodes], tok[kTreeMaxNodes], gone[kTreeMaxNodes], way[kTreeMaxNodes];
    __shared__ float uni[kTreeMaxNodes], lt[kTreeMaxNodes], lq[kTreeMaxNodes];
    __shared__ float red_m[2][kAccWaves];
    __shared__ double red_s[2][kAccWaves], part[2][kAccWaves];  // part: the waves' sums, two passes in turn
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int first, n;
    {
        kconst_i32 *p = (a.trees ? (kconst_i32 *)(uintptr_t)a.trees : (kconst_i32 *)kernarg_plan()) + 2 * blockIdx.x;
        first = p[0];
        n = p[1];
    }
    const int V = a.V;
    const float k = 1.4426950408889634f / a.temperature;
    if (tid < n) {
        par[tid] = a.parents[first + tid];
        tok[tid] = a.tok[first + tid];
        uni[tid] = a.u[first + tid];
    }
    __syncthreads();

    // Wave w covers entries [w * span, (w + 1) * span) of a row, 256 at a time.
    const int span = (V + kAccWaves * 256 - 1) / (kAccWaves * 256) * 256;
    const int v0 = min(V, wave * span), v1 = min(V, v0 + span);
    int cur = 0, steps = 0, n_gone = 0;
    if (tid == 0) way[0] = 0;
    const float *t, *d;
    RowStat T, D{0.f, 1.0};
    double C, S, A;  // A in units of the target's weights (p's mass = T.z)
    float ratio;     // C in those units: max(0, e_t - ratio e_q)
    auto rest = [&](float et, float eq) { return Q && eq > 0.f ? fmaxf(0.f, fmaf(-ratio, eq, et)) : et; };
    // Sum of what remains of entries [lo, hi) by this wave's lanes, the rejected
    // tokens left out where they have no distribution.
    auto mass = [&](int lo, int hi) {
        double s = 0.0;
        for (int base = lo; base < hi; base += 256) {
            const int i = base + lane * 4;
            const float4 x = acc_load4(t, i, hi);
            float e[4] = {acc_e(x.x, T.m, k), acc_e(x.y, T.m, k), acc_e(x.z, T.m, k), acc_e(x.w, T.m, k)};
            if constexpr (Q) {
                const float4 y = acc_load4(d, i, hi);
                e[0] = rest(e[0], acc_e(y.x, D.m, k));
                e[1] = rest(e[1], acc_e(y.y, D.m, k));
                e[2] = rest(e[2], acc_e(y.z, D.m, k));
                e[3] = rest(e[3], acc_e(y.w, D.m, k));
            } else {
                for (int g = 0; g < n_gone; g++) {
                    const int at = gone[g] - i;
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (at == c) e[c] = 0.f;
                }
            }
            s += (double)((e[0] + e[1]) + (e[2] + e[3]));
        }
        return s;
    };
    int turn = 0;
    // Sum over the row; the waves' sums stay in part[turn].
    auto total = [&]() {
        const double s = wave_sum(mass(v0, v1));
        turn ^= 1;
        if (lane == 0) part[turn][wave] = s;
        __syncthreads();
        double z = 0.0;
#pragma unroll
        for (int w = 0; w < kAccWaves; w++) z += part[turn][w];
        return z;
    };

    for (;;) {
        t = a.t_logits + (int64_t)(first + cur) * a.t_stride;
        d = Q ? a.d_logits + (int64_t)(first + cur) * a.d_stride : nullptr;
        // this node's children, and their logits
        uint64_t kids[kTreeMaxNodes / 64];
#pragma unroll
        for (int w = 0; w < kTreeMaxNodes / 64; w++) {
            const int j = w * 64 + lane;
            kids[w] = __builtin_amdgcn_ballot_w64(j > cur && j < n && par[j] == cur);
        }
        if (tid > cur && tid < n && par[tid] == cur && tok[tid] >= 0 && tok[tid] < V) {
            lt[tid] = t[tok[tid]];
            if (Q) lq[tid] = d[tok[tid]];
        }
        // maximum and mass of both rows in one pass
        {
            Online ot, oq;
            for (int base = v0; base < v1; base += 256) {
                ot.add(acc_load4(t, base + lane * 4, v1), k);
                if (Q) oq.add(acc_load4(d, base + lane * 4, v1), k);
            }
            auto fold = [&](Online &o, int side) {
                float m = o.m;
#pragma unroll
                for (int s = 32; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
                const double z = wave_sum(o.m == -INFINITY ? 0.0 : o.s * (double)acc_e(o.m, m, k));
                if (lane == 0) {
                    red_m[side][wave] = m;
                    red_s[side][wave] = z;
                }
            };
            fold(ot, 0);
            if (Q) fold(oq, 1);
            __syncthreads();
            auto join = [&](int side) {
                RowStat r{-INFINITY, 0.0};
#pragma unroll
                for (int w = 0; w < kAccWaves; w++) r.m = fmaxf(r.m, red_m[side][w]);
                if (r.m == -INFINITY) r.m = 0.f;
#pragma unroll
                for (int w = 0; w < kAccWaves; w++) r.z += red_s[side][w] * (double)acc_e(red_m[side][w], r.m, k);
                return r;
            };
            T = join(0);
            if (Q) D = join(1);
            turn ^= 1;
            if (tid < kAccWaves) part[turn][tid] = red_s[0][tid] * (double)acc_e(red_m[0][tid], T.m, k);
            __syncthreads();
        }
        C = 0.0;
        S = 1.0;
        A = T.z;
        ratio = 0.f;
        n_gone = 0;
        int went = -1;
#pragma unroll 1
        for (int w = 0; w < kTreeMaxNodes / 64 && went < 0; w++) {
            uint64_t left = w == 0 ? kids[0] : w == 1 ? kids[1] : w == 2 ? kids[2] : kids[3];
            while (left) {
                const int c = w * 64 + __builtin_ctzll(left);
                left &= left - 1;
                const int x = tok[c];
                bool skip = x < 0 || x >= V;  // no token: rejected without effect, as a rejected token again is
                for (int g = 0; g < n_gone; g++) skip |= gone[g] == x;
                if (skip) continue;
                const float et = acc_e(lt[c], T.m, k);
                if constexpr (Q) {
                    const float eq = acc_e(lq[c], D.m, k);
                    const double qx = (double)eq / D.z, px = (double)rest(et, eq);
                    if (S > 0.0 ? (double)uni[c] * qx * A < px * S : px > 0.0) {
                        went = c;
                        break;
                    }
                    if (S > 0.0) {
                        C += A / T.z / S;
                        S -= qx;
                        ratio = (float)(C * T.z / D.z);
                        A = total();
                        if (!(A > 0.0)) {  // nothing is left by rounding alone
                            C = 0.0;
                            ratio = 0.f;
                            A = total();
                        }
                    }
                } else {
                    if ((double)uni[c] * A < (double)et) {
                        went = c;
                        break;
                    }
                    A -= (double)et;
                }
                __syncthreads();
                if (tid == 0) gone[n_gone] = x;
                n_gone++;
                __syncthreads();
            }
        }
        if (went < 0) break;
        cur = went;
        steps++;
        if (tid == 0) way[steps] = cur;
        __syncthreads();
    }

    // ---- the next token: the first whose cumulated mass exceeds u A --------------
    if (!Q && n_gone) A = total();
    double want = (double)uni[0] * A;
    // The part of `n` sums where `want` falls (else the last one that holds any),
    // want becoming what is left of it there.
    auto pick = [&](const double *s) {
        double c = 0.0;
        int last = 0;
        double before = 0.0;
#pragma unroll 1
        for (int w = 0; w < kAccWaves; w++) {
            const double x = s[w];
            if (!(x > 0.0)) continue;
            last = w;
            before = c;
            c += x;
            if (c > want) break;
        }
        want -= before;
        return last;
    };
    int lo = pick(part[turn]) * span;
    const int sub = span / kAccWaves, hi = min(V, lo + span);
    {
        const int s0 = min(hi, lo + wave * sub), s1 = min(hi, s0 + sub);
        const double s = wave_sum(mass(s0, s1));
        turn ^= 1;
        if (lane == 0) part[turn][wave] = s;
        __syncthreads();
        lo += pick(part[turn]) * sub;
    }
    if (wave == 0) {
        const int end = min(hi, lo + sub);
        int found = -1, some = -1;
        for (int base = lo; base < end && found < 0; base += 64) {
            const int i = base + lane;
            float e = 0.f;
            if (i < end) {
                e = acc_e(t[i], T.m, k);
                if (Q) e = rest(e, acc_e(d[i], D.m, k));
                for (int g = 0; !Q && g < n_gone; g++)
                    if (gone[g] == i) e = 0.f;
            }
            double c = (double)e;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double up = __shfl_up(c, o);
                if (lane >= o) c += up;
            }
            const uint64_t over = __builtin_amdgcn_ballot_w64(e > 0.f && c > want);
            const uint64_t any = __builtin_amdgcn_ballot_w64(e > 0.f);
            if (over) found = base + __builtin_ctzll(over);
            if (any) some = base + 63 - __builtin_clzll(any);
            want -= __shfl(c, 63);
        }
        if (lane == 0) {
            a.n_acc[blockIdx.x] = steps;
            // (rows that hold no probability: some token of the vocabulary)
            a.next[blockIdx.x] = found >= 0 ? found : some >= 0 ? some : min(lo, V - 1);
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
