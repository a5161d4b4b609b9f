// Rotary positions: heads rotated by angles pos * inv_freq, any position, in the
// interleaved (2i, 2i + 1) or half (i, i + rd/2) pairing, over the first rd of D
// dims:
//
//   a = pos * inv_freq[i]
//   (x0, x1) -> scale (x0 cos a - x1 sin a, x0 sin a + x1 cos a)
//
// dims from rd on are copied.  The gradient of the rotation is the rotation by
// the negated positions.
//
// The product pos * inv_freq and its remainder by a turn are taken in 64 bits (an
// f32 angle at position 10^6 is off by 0.03), the sine and cosine of what is left
// in f32.
//
// Bound: HBM, one read and one write of the rows.  A thread computes the angles
// of its dims once and rotates them for several heads of the row, neighbouring
// threads on neighbouring heads, so that the trigonometry hides behind the stream.
// 8192 rows of 40 heads of 128, bf16: 28 to 36 us a call (warm and cold; 6.0 and
// 4.7 TB/s, where a large copy moves 5.2); a head a thread 45 us.  3001 rows of 32
// heads of 80, f32, 32 dims rotated: 13 us.  16 rows of 40 heads: 3 us, a launch.
#include <algorithm>

#include "rlx_tree.h"

namespace rlx {

__device__ __forceinline__ void rope_load8(const void *p, int64_t o, int bf16, float (&v)[8]) {
    if (bf16) {
        const u32x4 w = *(const u32x4 *)((const uint16_t *)p + o);
#pragma unroll
        for (int i = 0; i < 4; i++) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
    } else {
        const float4 x = *(const float4 *)((const float *)p + o), y = *(const float4 *)((const float *)p + o + 4);
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    }
}
__device__ __forceinline__ void rope_store8(void *p, int64_t o, int bf16, const float (&v)[8]) {
    if (bf16) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = (uint32_t)bf16_rne(v[2 * i]) | ((uint32_t)bf16_rne(v[2 * i + 1]) << 16);
        *(u32x4 *)((uint16_t *)p + o) = w;
    } else {
        *(float4 *)((float *)p + o) = make_float4(v[0], v[1], v[2], v[3]);
        *(float4 *)((float *)p + o + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
}
__device__ __forceinline__ float rope_load1(const void *p, int64_t o, int bf16) {
    return bf16 ? bf16_f32(((const uint16_t *)p)[o]) : ((const float *)p)[o];
}
__device__ __forceinline__ void rope_store1(void *p, int64_t o, int bf16, float v) {
    if (bf16)
        ((uint16_t *)p)[o] = bf16_rne(v);
    else
        ((float *)p)[o] = v;
}

// (cos, sin) of pos * inv_freq, times scale.
__device__ __forceinline__ float2 rope_angle(int32_t pos, float inv_freq, float scale) {
    const double turns = (double)pos * (double)inv_freq * 0.15915494309189535;
    const float left = (float)(turns - rint(turns));  // of a turn, in [-1/2, 1/2]
    float s, c;
    sincospif(2.f * left, &s, &c);
    return make_float2(c * scale, s * scale);
}

// The rotated pair, by the same operations whichever way a call is laid out.
__device__ __forceinline__ float2 rope_turn(float x0, float x1, float2 cs) {
    return make_float2(fmaf(x0, cs.x, -(x1 * cs.y)), fmaf(x0, cs.y, x1 * cs.x));
}

// Thread = (row, head h of `step`, unit): heads h, h + step, ...  VEC: units of 8
// dims -- pairs: D/8 of a head; halves: rd/16 of a pair of pieces, then (D - rd)/8
// copied ones.  Otherwise (odd widths, strides or addresses, and small calls):
// units of a pair, then of one copied dim.
template <bool VEC>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, int units, int step) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t hu = id / units;
    const int u = (int)(id - hu * units);
    const int64_t row = hu / step;
    if (row >= a.rows) return;
    const int h0 = (int)(hu - row * step), half = a.rd >> 1;
    const int64_t xr = row * a.x_row, orow = row * a.out_row;
    if constexpr (VEC) {
        const int rot = a.halves ? a.rd / 16 : a.rd / 8;  // rotated units
        const int d0 = a.halves && u >= rot ? a.rd + (u - rot) * 8 : u * 8;
        float2 cs[8];
        if (u < rot) {
            const int32_t pos = a.pos[row];
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (a.halves || i < 4) cs[i] = rope_angle(pos, a.inv_freq[a.halves ? d0 + i : d0 / 2 + i], a.scale);
        }
        for (int h = h0; h < a.heads; h += step) {
            const int64_t xo = xr + h * a.x_head + d0, oo = orow + h * a.out_head + d0;
            float v[8], w[8];
            rope_load8(a.x, xo, a.x_bf16, v);
            if (u < rot && a.halves) {
                float y[8];
                rope_load8(a.x, xo + half, a.x_bf16, w);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float2 r = rope_turn(v[i], w[i], cs[i]);
                    y[i] = r.x;
                    w[i] = r.y;
                }
                rope_store8(a.out, oo, a.out_bf16, y);
                rope_store8(a.out, oo + half, a.out_bf16, w);
                continue;
            }
            if (u < rot) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 r = rope_turn(v[2 * i], v[2 * i + 1], cs[i]);
                    v[2 * i] = r.x;
                    v[2 * i + 1] = r.y;
                }
            }
            rope_store8(a.out, oo, a.out_bf16, v);
        }
    } else {
        const bool rot = u < half;
        const int d0 = !rot ? a.rd + (u - half) : a.halves ? u : 2 * u, d1 = a.halves ? d0 + half : d0 + 1;
        const float2 cs = rot ? rope_angle(a.pos[row], a.inv_freq[u], a.scale) : make_float2(1.f, 0.f);
        for (int h = h0; h < a.heads; h += step) {
            const int64_t xo = xr + h * a.x_head, oo = orow + h * a.out_head;
            const float x0 = rope_load1(a.x, xo + d0, a.x_bf16);
            if (!rot) {
                rope_store1(a.out, oo + d0, a.out_bf16, x0);
                continue;
            }
            const float x1 = rope_load1(a.x, xo + d1, a.x_bf16);
            const float2 r = rope_turn(x0, x1, cs);
            rope_store1(a.out, oo + d0, a.out_bf16, r.x);
            rope_store1(a.out, oo + d1, a.out_bf16, r.y);
        }
    }
}

hipError_t launch_rope(hipStream_t s, const RopeArgs &a, int cus) {
    if (a.rows <= 0 || a.heads <= 0) return hipSuccess;
    const auto whole = [](int64_t n) { return n % 8 == 0; };
    // Small calls take the pairs too, a thread's eight angles one after another being
    // longer than the rows' stream.  40 heads of 128, us by pairs and by units of 8: 16
    // rows 3.0 / 4.2 (halves), 3.0 / 3.4 (pairs); 128 rows 3.9 / 4.6, 3.9 / 4.0; 512
    // rows 5.9 / 6.2, 6.1 / 5.7; 8192 rows 48 / 28 (pairs).
    const int64_t pairs = a.rows * a.heads * (a.rd / 2 + (a.D - a.rd));
    const bool vec = pairs > (int64_t)cus * 2048 && whole(a.D) && whole(a.halves ? a.rd / 2 : a.rd) && whole(a.x_row) && whole(a.x_head) &&
                     whole(a.out_row) && whole(a.out_head) && ((uintptr_t)a.x & 15) == 0 && ((uintptr_t)a.out & 15) == 0;
    const int units = !vec ? a.rd / 2 + (a.D - a.rd) : a.halves ? a.rd / 16 + (a.D - a.rd) / 8 : a.D / 8;
    // Heads a thread takes: as many as 8, while 16 waves a CU remain.  8192 rows of 40
    // heads of 128: 45 us with 1, 27 with 4, 28 with 8 and 16.
    const int64_t all = a.rows * a.heads * units;
    const int per = (int)std::max<int64_t>(1, std::min<int64_t>(8, all / ((int64_t)cus * 1024)));
    const int step = (a.heads + per - 1) / per;
    const int64_t blocks = (a.rows * step * units + 255) / 256;
    if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
    if (vec)
        rope_kernel<true><<<(unsigned)blocks, 256, 0, s>>>(a, units, step);
    else
        rope_kernel<false><<<(unsigned)blocks, 256, 0, s>>>(a, units, step);
    return hipGetLastError();
}

}  // namespace rlx
