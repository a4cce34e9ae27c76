// Rotation angles of RoPE / YaRN, shared by every kernel that rotates queries and keys.
#pragma once

#include "common.cuh"

namespace qz {

constexpr int ATT_MAX_HD = 128;   // largest head_dim of the attention kernels

// rotation (cos, sin) of pair i at one position, exactly as rope_kv_kernel / src/cuda_kernels.cu:588-620 compute it
struct RopeArgsLite {
    int pos;
    float theta, yarn_scale;
    int yarn_orig_ctx;
};
__device__ __forceinline__ void rope_cs_lite(const RopeArgsLite &r, int i, int head_dim, float &c, float &s)
{
    const float PI = 3.14159265358979f;
    float inv = 1.f / powf(r.theta, 2.f * (float)i / (float)head_dim);
    float eff = inv;
    if (r.yarn_scale > 1.f && r.yarn_orig_ctx > 0) {
        float hi_w = (float)r.yarn_orig_ctx / 32.f, lo_w = (float)r.yarn_orig_ctx / 1.f;
        float wavelen = 2.f * PI / inv;
        float ramp = fmaxf(0.f, fminf(1.f, (lo_w - wavelen) / (lo_w - hi_w)));
        eff = ramp * inv + (1.f - ramp) * (inv / r.yarn_scale);
    }
    sincosf((float)r.pos * eff, &s, &c);
}

struct RopeArgs {
    int pos;
    float theta, yarn_scale;
    int yarn_orig_ctx, neox;
};

// rotation (cos, sin) of pair i, exactly as rope_kv_kernel / src/cuda_kernels.cu:588-620 compute it
__device__ __forceinline__ void rope_cs(const RopeArgs &r, int i, int head_dim, float &c, float &s)
{
    const float PI = 3.14159265358979f;
    float inv = 1.f / powf(r.theta, 2.f * (float)i / (float)head_dim);
    float eff = inv;
    if (r.yarn_scale > 1.f && r.yarn_orig_ctx > 0) {
        float hi_w = (float)r.yarn_orig_ctx / 32.f, lo_w = (float)r.yarn_orig_ctx / 1.f;
        float wavelen = 2.f * PI / inv;
        float ramp = fmaxf(0.f, fminf(1.f, (lo_w - wavelen) / (lo_w - hi_w)));
        eff = ramp * inv + (1.f - ramp) * (inv / r.yarn_scale);
    }
    sincosf((float)r.pos * eff, &s, &c);
}

}  // namespace qz
