// Attention over the 4-bit cache (kv4.cuh): one token of a decode step, or the tokens of a prompt.
#pragma once

#include "kv4.cuh"

namespace qz {

constexpr int AK_THREADS = 256, AK_WARPS = AK_THREADS / 32;
constexpr int AK_MAX_G = 16;

struct AttnKv4Args {
    float *out;
    const float *q, *k_new, *v_new;      // step: before rotation; prompt: already rotated, k_new / v_new NULL
    uint8_t *cache;
    const int *step;                     // device words {token, pos}, or NULL: pos
    int pos;
    int n_heads, n_kv, max_seq, n_blocks;
    int window;
    float scale;
    const float *sinks;
    float theta, yarn_scale;             // theta <= 0: nothing is rotated
    int yarn_orig_ctx, neox;
    XQOut o;
    int emit_q;
    const float2 *rope_tab;
};

// One CTA per (kv head, token); a warp takes every eighth position for one query head after the other.
template <int NG>
__global__ void __launch_bounds__(AK_THREADS) attn_kv4_kernel(const AttnKv4Args a)
{
    constexpr int HD = 32 * NG, half = HD / 2;
    __shared__ __align__(16) float qs[AK_MAX_G * HD];
    __shared__ __align__(16) float kn[HD];
    __shared__ float part[AK_WARPS][HD + 2];
    const int head = blockIdx.x, tok = blockIdx.y, G = a.n_heads / a.n_kv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    int pos = (a.step ? __ldcg(a.step + 1) : a.pos) + tok;
    pos = max(0, min(pos, a.max_seq - 1));
    const int first = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    const RopeArgs rope{pos, a.theta, a.yarn_scale, a.yarn_orig_ctx, a.neox};
    for (int e = threadIdx.x; e < (G + 1) * half; e += AK_THREADS) {
        const int g = e / half, i = e - g * half;
        const int i0 = a.neox ? i : 2 * i, i1 = a.neox ? i + half : 2 * i + 1;
        if (g == G && !a.k_new) break;
        const float *src = g == G ? a.k_new + (size_t)head * HD : a.q + ((size_t)tok * a.n_heads + (size_t)head * G + g) * HD;
        float x0 = __ldcg(src + i0), x1 = __ldcg(src + i1);
        if (a.theta > 0.f) {
            float c, s;
            rope_cs(rope, i, HD, c, s);
            const float r0 = x0 * c - x1 * s, r1 = x0 * s + x1 * c;
            x0 = r0;
            x1 = r1;
        }
        float *dst = g == G ? kn : qs + g * HD;
        dst[i0] = x0;
        dst[i1] = x1;
    }
    __syncthreads();
    if (a.k_new && warp < 2 && lane < 4 * NG) {
        const float *src = warp ? a.v_new + (size_t)head * HD : kn;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = src[8 * lane + e];
        kv4_store8<NG>(x, kv4_block(a.cache, a.n_blocks, head, pos / KV4_BLOCK, HD), pos % KV4_BLOCK, lane >> 2, lane & 3, warp == 1,
                       4 * NG == 32 ? 0xFFFFFFFFu : (1u << (4 * NG)) - 1u);
    }
    __syncthreads();
    for (int g = 0; g < G; g++) {
        float m_run = -INFINITY, l_run = 0.f, acc[NG];
#pragma unroll
        for (int j = 0; j < NG; j++) acc[j] = 0.f;
        for (int p = first + warp; p <= pos; p += AK_WARPS) {
            const uint8_t *blk = kv4_block(a.cache, a.n_blocks, head, p / KV4_BLOCK, HD);
            const int row = p % KV4_BLOCK;
            const uint32_t *kc = (const uint32_t *)(blk + row * half);
            const uint16_t *vc = (const uint16_t *)(blk + 20 * HD + row * half);
            const __half *kp = (const __half *)(blk + 16 * HD) + row * 2 * NG, *vp = (const __half *)(blk + 36 * HD) + row * 2 * NG;
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < NG; j++) {
                const float c = (float)((kc[(lane >> 3) * NG + j] >> (4 * (lane & 7))) & 15u);
                s = fmaf(fmaf(__half2float(kp[NG + j]), c, __half2float(kp[j])), qs[g * HD + 32 * j + lane], s);
            }
            s = warp_sum(s) * a.scale;
            const float m_new = fmaxf(m_run, s), corr = m_run == m_new ? 1.f : expf(m_run - m_new), w = expf(s - m_new);
            l_run = l_run * corr + w;
#pragma unroll
            for (int j = 0; j < NG; j++) {
                const float c = (float)((vc[(lane >> 2) * NG + j] >> (4 * (lane & 3))) & 15u);
                acc[j] = fmaf(w, fmaf(__half2float(vp[NG + j]), c, __half2float(vp[j])), acc[j] * corr);
            }
            m_run = m_new;
        }
        if (lane == 0) {
            part[warp][HD] = m_run;
            part[warp][HD + 1] = l_run;
        }
#pragma unroll
        for (int j = 0; j < NG; j++) part[warp][32 * j + lane] = acc[j];
        __syncthreads();
        const int h = head * G + g;
        float top = a.sinks ? a.sinks[h] : -INFINITY;
        for (int w = 0; w < AK_WARPS; w++) top = fmaxf(top, part[w][HD]);
        float total = a.sinks ? expf(a.sinks[h] - top) : 0.f;
        for (int w = 0; w < AK_WARPS; w++) total += part[w][HD + 1] * expf(part[w][HD] - top);
        for (int d = threadIdx.x; d < HD; d += AK_THREADS) {
            float o = 0.f;
            for (int w = 0; w < AK_WARPS; w++) o = fmaf(part[w][d], expf(part[w][HD] - top), o);
            o /= total;
            a.out[((size_t)tok * a.n_heads + h) * HD + d] = o;
            qs[g * HD + d] = o;   // (this head's query is no longer read)
        }
        __syncthreads();
    }
    if (a.emit_q) {
        for (int e = warp * 128; e < G * HD; e += AK_WARPS * 128) {
            const int i = e + 4 * lane;
            const bool valid = i < G * HD;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            for (int j = 0; j < 4 && valid; j++) v[j] = qs[i + j];
            quantize4_store(v, (head * G * HD + i) >> 2, valid, a.o);
        }
    }
}

}  // namespace qz
