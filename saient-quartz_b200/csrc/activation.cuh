// The 16-bit block-fixed-point form in which the streaming GEMVs read their activation vector, and the conversion
// into it that producers of such vectors (norms, SwiGLU, attention) carry in their epilogue.
#pragma once

#include "common.cuh"

namespace qz {

// Block-fixed-point activations.  xl/xh: low/high int8 limbs [K]; xs: f32 scale per
// 32-run [K/32]; xsum: exact f32 sum of x per 16-run [K/16].
struct XQ {
    const int8_t *xl;
    const int8_t *xh;
    const float *xs;
    const float *xsum;
};

constexpr float XQ_RANGE = 32512.0f;   // 127 * 256: h, l both fit int8
// Runs whose largest magnitude is below this (2^-110) are taken as zero: XQ_RANGE / amax would overflow and the
// scale amax / XQ_RANGE would be subnormal; products of such activations underflow in f32 anyway.
constexpr float XQ_TINY = 7.703719777548943e-34f;

// Scale handling shared by every conversion site.  amax: largest magnitude of the 32-run; sum32: the run's f32
// sum, used only to notice a NaN or an infinity anywhere in the run (fmaxf drops NaNs): such a run gets a NaN
// scale, so every output that touches it becomes NaN, as it would in f32 arithmetic.
__device__ __forceinline__ void xq_run_scale(float amax, float sum32, float &inv, float &scale)
{
    if (!(fabsf(sum32) <= 3.0e38f) || !(amax <= 3.0e38f)) {   // NaN or infinite
        inv = 0.f;
        scale = __int_as_float(0x7FC00000);
    } else if (amax > XQ_TINY) {
        inv = XQ_RANGE / amax;
        scale = amax / XQ_RANGE;
    } else {
        inv = 0.f;
        scale = 0.f;
    }
}

struct XQOut {
    int8_t *xl, *xh;
    float *xs, *xsum;
};

// Convert four consecutive values (elements 4t .. 4t+3, t = global thread-of-4 index) exactly
// as quantize_x_kernel does.  All 32 lanes of the warp must call it (shuffles inside); lanes
// past the end pass valid = false.
__device__ __forceinline__ void quantize4_store(const float v[4], int t, bool valid, const XQOut &o)
{
    float amax = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
    float sum = (v[0] + v[1]) + (v[2] + v[3]);
    amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
    amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 4));
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
    const float sum32 = sum + __shfl_xor_sync(0xFFFFFFFFu, sum, 4);
    if (!valid) return;
    float inv, scale;
    xq_run_scale(amax, sum32, inv, scale);
    uint32_t wl = 0, wh = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        int X = __float2int_rn(v[i] * inv);
        int l = ((X + 128) & 0xFF) - 128;
        int h = (X - l) >> 8;
        wl |= (uint32_t)(l & 0xFF) << (8 * i);
        wh |= (uint32_t)(h & 0xFF) << (8 * i);
    }
    ((uint32_t *)o.xl)[t] = wl;
    ((uint32_t *)o.xh)[t] = wh;
    if ((t & 7) == 0) o.xs[t >> 3] = scale;
    if ((t & 3) == 0) o.xsum[t >> 2] = sum;
}

}  // namespace qz
