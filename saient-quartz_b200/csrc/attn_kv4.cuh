// Attention over the 4-bit cache (kv4.cuh) for one token of a decode step, or a few tokens of a prompt one by one.
#pragma once

#include <cooperative_groups.h>

#include "async_copy.cuh"
#include "kv4.cuh"

namespace qz {

// six warps: two CTAs of them per SM leave 168 registers a thread (12 bytes of a thread are spilled; eight warps leave 128, which
// spill far more: 131072 positions take 58 us, not 51)
constexpr int AK_THREADS = 192, AK_WARPS = AK_THREADS / 32;
constexpr int AK_MAX_G = 16;
constexpr float AK_RAISE = 2.f;                       // weights are at most 2^AK_RAISE,
constexpr float AK_STEP_TOP = 8192.f;                 // scaled steps at most this, set to [1/4, 1/2) of it: products below 2^15
constexpr int AK_MAX_CLUSTERS = 128;                  // of all units together when a unit has several
constexpr int AK_COUNTERS = AK_MAX_CLUSTERS * 32;     // one per run of 32 outputs of a unit
constexpr size_t AK_WORKSPACE = sizeof(float) * (AK_COUNTERS + (size_t)AK_MAX_CLUSTERS * 32 * 34);

struct AttnKv4Args {
    float *out;
    const float *q, *k_new, *v_new;      // before rotation; token blockIdx.y (at pos + blockIdx.y) has row blockIdx.y of q and out
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
    int splits;                          // units that share a kv head's query heads
    int clusters;                        // clusters per unit
    float *workspace;                    // clusters > 1: AK_COUNTERS zeroed counters, then [units * 32 runs][clusters][34]
    int prefetch;                        // the launch may overlap the one before it: fetch into L2 ahead of the wait
    int *status;
};

// ---- one token ---------------------------------------------------------------------------------------------------
// One launch whose shape does not depend on the position.  A unit is a kv head (two units when more than eight query heads
// share it); it has NC clusters of CL CTAs, of which as many work as the context has a block for every warp of.  Warp w of
// CTA r (of all R working ones) takes the blocks of 32 positions r + R (w + 6 i), so that a short context is spread over the
// CTAs first.  A warp works alone: it streams its blocks through a ring of its own (one bulk copy per block: the block is
// contiguous) and keeps scores, weights and outputs of all heads in registers.  A cluster's CTAs push their results into
// the CTA that finishes a run of 32 outputs; with several clusters at work, that CTA leaves the run in a workspace and the
// last one to arrive merges them in the clusters' order (clusters of 16 need no workspace, but only 7 of them fit on the
// chip at once, 8 kv heads took two turns).
//
// Both products run on the tensor cores with the CODES as one operand, exactly, and 22 bits of the other:
//   scores   s[pos, head] = sum_g d_g ((codes_g - 8) . q_g) + (m_g + 8 d_g) sum(q_g)
//   outputs  o[dim, head] = sum_pos (codes[dim, pos] - 8) (p d_g)[pos, head]  +  sum_pos (p (m_g + 8 d_g))[pos, head]
// The codes are taken around 8 because the two terms of either line otherwise cancel (m is a group's minimum).  A nibble
// becomes the f16 number code - 8, two at a time, by one logical operation (1024 + code or 1024 + 16 code: the nibble in
// the mantissa) and one exact HADD2 / HFMA2.  (The nibbles alone, as f16 subnormals, would need no second step, but the
// tensor core aligns products by their nominal exponents: 6 to 10 bits of the sum were lost, 5e-6 of the output.)
// q and p * d are split into two f16 parts, hi + lo, in neighbouring columns of the 8-column operand, so four heads fill
// one mma.m16n8k16; both parts are scaled by powers of two (per head for q, per group of 32 dims for d: a group's outputs
// owe nothing to the other groups) that keep them clear of f16's ends.  Sums are f32.
// The softmax reference of a head is raised only when a score exceeds it by 2^AK_RAISE; until then weights up to that do no
// harm, and f16 has as many binades more for small ones.  With the largest step that the warp has met in a group at 2^11 or
// above, 22 bits of p d are whole down to 2^-14 of that step (p d = 2^-3), and below that the error is 2^-35 of it at most.
//
// Measured (32 / 8 heads of 128, replayed over caches that together exceed L2): context 1024 6.0 us (8 / 2 heads of 64, context 18:
// 4.0), 4096 10.7, 16384 14.9 (13.4 from L2), 131072 51 us = 3.3 TB/s of the cache.  Short contexts are bound by the launch, two cluster
// barriers and one block's latency; long ones by the warps' dependent instructions: a warp spends some 400 on a tile of 16
// positions (unpacking, the hi / lo parts, 24 MMAs), three warps a scheduler issue 0.52 a cycle; the same launch that only loads
// takes 32 us.
// Clusters join a unit only when every warp still has a block: at twice that 16384 positions take 14.2 us, 8192 13.4 (12.3).
__host__ __device__ constexpr int attn_kv4_stages(int NG) { return NG == 1 ? 8 : NG == 2 ? 4 : 2; }   // ~10 KB in flight per warp

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t *)&h;
}
// (v & mask) | magic as ONE instruction: both constants live in registers (two immediates would make it two)
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t magic)
{
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(v), "r"(mask), "r"(magic));
    return y;
}
struct Nibbles {
    uint32_t even, odd, magic;
    __device__ __forceinline__ Nibbles()
    {
        asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(even));   // (volatile: kept in registers, not rebuilt at each use)
        asm volatile("mov.b32 %0, 0x00F000F0;" : "=r"(odd));
        asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
    }
    // The four pairs (i, i + 4) of a word's eight nibbles as pairs of f16 numbers code - 8.
    __device__ __forceinline__ void pairs(uint32_t w, uint32_t (&x)[4]) const
    {
        const __half2 m1032 = __half2half2(__ushort_as_half((unsigned short)0xE408)), m72 = __half2half2(__ushort_as_half((unsigned short)0xD480)),
                      sixteenth = __half2half2(__ushort_as_half((unsigned short)0x2C00));
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const uint32_t v = i ? w >> 8 : w;
            const uint32_t e = and_or(v, even, magic), o = and_or(v, odd, magic);   // 1024 + c, 1024 + 16 c
            const __half2 he = __hadd2(*(const __half2 *)&e, m1032), ho = __hfma2(*(const __half2 *)&o, sixteenth, m72);
            x[i] = *(const uint32_t *)&he;
            x[i + 1] = *(const uint32_t *)&ho;
        }
    }
};
// N halves (N = 1..4) at a 2N-aligned address, as floats
template <int N>
__device__ __forceinline__ void lds_halves(const void *p, float (&x)[N])
{
    if constexpr (N == 4) {
        const uint2 w = *(const uint2 *)p;
        const float2 a = __half22float2(*(const __half2 *)&w.x), b = __half22float2(*(const __half2 *)&w.y);
        x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    } else if constexpr (N == 2) {
        const float2 a = __half22float2(*(const __half2 *)p);
        x[0] = a.x; x[1] = a.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = __half2float(((const __half *)p)[i]);
    }
}
template <int N>
__device__ __forceinline__ void lds_words(const void *p, uint32_t (&x)[N])
{
    if constexpr (N == 4) {
        const uint4 w = *(const uint4 *)p;
        x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
    } else if constexpr (N == 2) {
        const uint2 w = *(const uint2 *)p;
        x[0] = w.x; x[1] = w.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = ((const uint32_t *)p)[i];
    }
}
// the 16-bit words j of two positions side by side: out[j] = a[j] | b[j] << 16
template <int N>
__device__ __forceinline__ void lds_pairs(const void *a, const void *b, uint32_t (&out)[N])
{
    if constexpr (N == 4) {
        const uint2 x = *(const uint2 *)a, y = *(const uint2 *)b;
        out[0] = __byte_perm(x.x, y.x, 0x5410); out[1] = __byte_perm(x.x, y.x, 0x7632);
        out[2] = __byte_perm(x.y, y.y, 0x5410); out[3] = __byte_perm(x.y, y.y, 0x7632);
    } else if constexpr (N == 2) {
        const uint32_t x = *(const uint32_t *)a, y = *(const uint32_t *)b;
        out[0] = __byte_perm(x, y, 0x5410); out[1] = __byte_perm(x, y, 0x7632);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) out[i] = (uint32_t)((const uint16_t *)a)[i] | (uint32_t)((const uint16_t *)b)[i] << 16;
    }
}

// N floats at a 4N-aligned address (16 N = 64: one vector)
template <int N>
__device__ __forceinline__ void lds_floats(const float *p, float (&x)[N])
{
    if constexpr (N == 4) {
        const float4 v = *(const float4 *)p;
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else if constexpr (N == 2) {
        const float2 v = *(const float2 *)p;
        x[0] = v.x; x[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = p[i];
    }
}

// The running state of a warp over the blocks of one kv head, for 4 NT heads, and one block's turn.
// lane = 4 gr + t.  Scores: rows gr, gr + 8 of a tile of 16 positions, columns (hi, lo) of head t.  Outputs: dims
// 32 j + 4 gr + i of head t.  Weights as operand: head gr / 2 (part gr % 2), positions t, t + 4, t + 8, t + 12 of a tile.
template <int NG, int NT>
struct Kv4Warp {
    // floats of shared memory a warp needs: d, m + 8 d of K and of V per position, powers of two that p * d of group j carries
    static constexpr int VE = 4 * 32 * NG, SCRATCH = VE + 4;
    uint32_t qf[NT][NG][4];   // q as the column operand: dims (0,4) (1,5) (2,6) (3,7) of 32 j + 8 t, column gr
    float qs[NT][NG];         // sum of q over group j, head t
    float back[NT];           // scores in log2 units = back * what the products give, head t
    float ref[NT], l[NT];     // reference and partial sum of weights, head t
    float o[NT][2 * NG][4];   // sums of the tensor core since the last flush
    float acc[NT][2 * NG][2]; // flushed sums (hi + lo)
    float mo[NT][NG];         // partial sums of p * (m + 8 d), head gr / 2
    Nibbles nib;

    __device__ __forceinline__ void clear(float *scratch, int lane)
    {
        if (lane < NG) scratch[VE + lane] = 1.2676506e30f;   // 2^100: the first block with a step above zero sets it
        __syncwarp();
#pragma unroll
        for (int n = 0; n < NT; n++) {
            ref[n] = -3.0e38f;
            l[n] = 0.f;
#pragma unroll
            for (int j = 0; j < NG; j++) mo[n][j] = 0.f;
#pragma unroll
            for (int j = 0; j < 2 * NG; j++) {
                o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
                acc[n][j][0] = acc[n][j][1] = 0.f;
            }
        }
    }

    // The tensor core rounds its running f32 sums towards zero, half an ulp too low at each step on average: 64 steps cost
    // 2e-6.  Sums of at most 8 steps are therefore moved to ordinary ones (1e-7), which round to nearest.
    __device__ __forceinline__ void flush()
    {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 2 * NG; j++) {
                acc[n][j][0] += o[n][j][0] + o[n][j][1];
                acc[n][j][1] += o[n][j][2] + o[n][j][3];
                o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
            }
    }

    // rows lo .. hi of the block are visible; the others may hold anything
    __device__ __forceinline__ void block(const uint8_t *blk, float *scratch, int lo, int hi, int lane)
    {
        constexpr int HD = 32 * NG, ROW = HD / 2, PAR = 4 * NG;
        const int gr = lane >> 2, t = lane & 3;
        float *kd = scratch, *km = kd + 32 * NG, *vd = km + 32 * NG, *vm = vd + 32 * NG;
        // ---- parameters: lane = position, converted once for the warp ----
        const bool whole = lo == 0 && hi == KV4_BLOCK - 1;
        {
            float m[NG], d[NG], ve[NG];
            bool above = false;
            lds_floats<NG>(scratch + VE, ve);
            const bool seen = lane >= lo && lane <= hi;
#pragma unroll
            for (int side = 0; side < 2; side++) {
                const uint8_t *p = blk + (side ? 36 : 16) * HD + lane * PAR;
                lds_halves<NG>(p, m);
                lds_halves<NG>(p + 2 * NG, d);
                if (!whole && !seen) {
#pragma unroll
                    for (int j = 0; j < NG; j++) m[j] = d[j] = 0.f;
                }
                float *dd = (side ? vd : kd) + lane * NG, *mm = (side ? vm : km) + lane * NG;
#pragma unroll
                for (int j = 0; j < NG; j++) m[j] = fmaf(8.f, d[j], m[j]);
                if (side) {   // values: d as p will meet it, scaled
#pragma unroll
                    for (int j = 0; j < NG; j++) {
                        d[j] *= ve[j];
                        above |= d[j] > AK_STEP_TOP;
                    }
                }
                if constexpr (NG == 4) {
                    *(float4 *)dd = make_float4(d[0], d[1], d[2], d[3]);
                    *(float4 *)mm = make_float4(m[0], m[1], m[2], m[3]);
                } else {
#pragma unroll
                    for (int j = 0; j < NG; j++) {
                        dd[j] = d[j];
                        mm[j] = m[j];
                    }
                }
            }
            if (__any_sync(0xFFFFFFFFu, above)) set_scale(d, ve, vd + lane * NG, scratch + VE);   // (rare)
        }
        __syncwarp();
        // ---- scores ----
        float s[2][NT][2];
#pragma unroll
        for (int tile = 0; tile < 2; tile++) {
            const int r0 = 16 * tile + gr, r1 = r0 + 8;
            uint32_t k0[NG], k1[NG];
            float m0[NG], m1[NG], d0[NG], d1[NG];
            lds_words<NG>(blk + r0 * ROW + 4 * NG * t, k0);
            lds_words<NG>(blk + r1 * ROW + 4 * NG * t, k1);
            lds_floats<NG>(kd + r0 * NG, d0);
            lds_floats<NG>(km + r0 * NG, m0);
            lds_floats<NG>(kd + r1 * NG, d1);
            lds_floats<NG>(km + r1 * NG, m1);
#pragma unroll
            for (int n = 0; n < NT; n++) s[tile][n][0] = s[tile][n][1] = 0.f;
#pragma unroll
            for (int j = 0; j < NG; j++) {
                uint32_t x[4], y[4];
                nib.pairs(k0[j], x);
                nib.pairs(k1[j], y);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float c[4];
                    mma16816_first(c, x[0], y[0], x[1], y[1], qf[n][j][0], qf[n][j][1]);
                    mma16816(c, x[2], y[2], x[3], y[3], qf[n][j][2], qf[n][j][3]);
                    s[tile][n][0] = fmaf(d0[j], c[0] + c[1], fmaf(m0[j], qs[n][j], s[tile][n][0]));
                    s[tile][n][1] = fmaf(d1[j], c[2] + c[3], fmaf(m1[j], qs[n][j], s[tile][n][1]));
                }
            }
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = gr + 8 * i;
                if (r < lo || r > hi) {
#pragma unroll
                    for (int n = 0; n < NT; n++) s[i >> 1][n][i & 1] = -INFINITY;   // (back is positive)
                }
            }
        }
        // ---- weights ----
        bool raise = false;
#pragma unroll
        for (int n = 0; n < NT; n++) raise |= fmaxf(fmaxf(s[0][n][0], s[0][n][1]), fmaxf(s[1][n][0], s[1][n][1])) * back[n] > ref[n] + AK_RAISE;
        if (__any_sync(0xFFFFFFFFu, raise)) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float top = fmaxf(fmaxf(s[0][n][0], s[0][n][1]), fmaxf(s[1][n][0], s[1][n][1])) * back[n];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
                top = fmaxf(top, ref[n]);
                const float corr = ex2(ref[n] - top);
                ref[n] = top;
                l[n] *= corr;
                const float corr_m = __shfl_sync(0xFFFFFFFFu, corr, gr >> 1);   // of the head whose weights this lane carries
#pragma unroll
                for (int j = 0; j < NG; j++) mo[n][j] *= corr_m;
                scale_outputs(n, corr);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float &x = s[i >> 1][n][i & 1];
                x = ex2(fmaf(x, back[n], -ref[n]));
                l[n] += x;
            }
        // ---- outputs ----
        const uint8_t *vb = blk + 20 * HD;
        const int part = gr & 1;
        const float is_lo = (float)part;
        const uint32_t flip = (uint32_t)part << 31;
#pragma unroll
        for (int tile = 0; tile < 2; tile++) {
            const int r = 16 * tile + t;
            float d[4][NG], m[2][NG];
#pragma unroll
            for (int i = 0; i < 4; i++) lds_floats<NG>(vd + (r + 4 * i) * NG, d[i]);
#pragma unroll
            for (int i = 0; i < 2; i++) lds_floats<NG>(vm + (r + 8 * part + 4 * i) * NG, m[i]);
            uint32_t v01[NG], v23[NG];
            lds_pairs<NG>(vb + r * ROW + 2 * NG * gr, vb + (r + 4) * ROW + 2 * NG * gr, v01);
            lds_pairs<NG>(vb + (r + 8) * ROW + 2 * NG * gr, vb + (r + 12) * ROW + 2 * NG * gr, v23);
            float p[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int src = 4 * t + (gr >> 1);
                p[n][0] = __shfl_sync(0xFFFFFFFFu, s[tile][n][0], src);
                p[n][1] = __shfl_sync(0xFFFFFFFFu, s[tile][n][0], src + 16);
                p[n][2] = __shfl_sync(0xFFFFFFFFu, s[tile][n][1], src);
                p[n][3] = __shfl_sync(0xFFFFFFFFu, s[tile][n][1], src + 16);
                const float a = part ? p[n][2] : p[n][0], b = part ? p[n][3] : p[n][1];
#pragma unroll
                for (int j = 0; j < NG; j++) mo[n][j] = fmaf(a, m[0][j], fmaf(b, m[1][j], mo[n][j]));
            }
#pragma unroll
            for (int j = 0; j < NG; j++) {
                uint32_t x[4], y[4];   // dims 4 gr + 0 .. 3 of positions (t, t + 4) and (t + 8, t + 12)
                nib.pairs(v01[j], x);
                nib.pairs(v23[j], y);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // hi: the leading 11 bits; lo: the rest
                        const float v = p[n][i] * d[i][j];
                        w[i] = fmaf(is_lo, v, __uint_as_float((__float_as_uint(v) & 0xFFFFE000u) ^ flip));
                    }
                    const uint32_t b0 = pack_half2(w[0], w[1]), b1 = pack_half2(w[2], w[3]);
                    mma16816(o[n][2 * j], x[0], x[1], y[0], y[1], b0, b1);
                    mma16816(o[n][2 * j + 1], x[2], x[3], y[2], y[3], b0, b1);
                }
            }
        }
    }

    __device__ __forceinline__ void scale_outputs(int n, float f)
    {
#pragma unroll
        for (int j = 0; j < 2 * NG; j++) {
            o[n][j][0] *= f; o[n][j][1] *= f; o[n][j][2] *= f; o[n][j][3] *= f;
            acc[n][j][0] *= f; acc[n][j][1] *= f;
        }
    }
    // `scaled`: the block's steps times ve, this lane's position.  Groups that need it get the power of two that brings the largest
    // into [1/4, 1/2) of AK_STEP_TOP; the scaled steps once more, to dst.  (ve lives in shared memory: in registers 64 / 8 heads at
    // 131072 positions take 97 us, not 95.)
    __device__ __forceinline__ void set_scale(const float (&scaled)[NG], const float (&ve)[NG], float *dst, float *ve_dst)
    {
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(scaled[j]));   // (steps are not negative)
            const float f = __uint_as_float(top) > AK_STEP_TOP ? __uint_as_float((127 + 11 + 127 - (top >> 23)) << 23) : 1.f;
            ve_dst[j] = ve[j] * f;   // (all lanes the same)
            dst[j] = scaled[j] * f;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 2 * j; k < 2 * j + 2; k++) {
                    o[n][k][0] *= f; o[n][k][1] *= f; o[n][k][2] *= f; o[n][k][3] *= f;
                    acc[n][k][0] *= f; acc[n][k][1] *= f;
                }
        }
    }

    // after the last flush: the sum of weights of head t, and outputs (times it) of dims 32 j + 4 gr .. + 3 of head t
    __device__ __forceinline__ float sum(int n) const
    {
        float x = l[n];
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, k);
        return x;
    }
    __device__ __forceinline__ float4 out(int n, int j, int lane, const float *scratch) const
    {
        float m = mo[n][j];
#pragma unroll
        for (int k = 1; k < 8; k <<= 1) m += __shfl_xor_sync(0xFFFFFFFFu, m, k);
        m = __shfl_sync(0xFFFFFFFFu, m, 8 * (lane & 3));
        const float e = __uint_as_float((254u << 23) - __float_as_uint(scratch[VE + j]));   // 1 / ve (a division a group costs 0.3 us)
        return make_float4(fmaf(acc[n][2 * j][0], e, m), fmaf(acc[n][2 * j][1], e, m), fmaf(acc[n][2 * j + 1][0], e, m),
                           fmaf(acc[n][2 * j + 1][1], e, m));
    }
};

struct AttnKv4Smem {
    int ring, params, qf, qs, rot, cs, recv, bar, total;   // byte offsets
};
__host__ __device__ constexpr AttnKv4Smem attn_kv4_smem(int NG, int NT, int GV, int CL)
{
    AttnKv4Smem s = {};
    const int HD = 32 * NG;
    s.ring = 0;                                               // [warps][stages] blocks; a warp's results replace its own
    int at = AK_WARPS * attn_kv4_stages(NG) * 40 * HD;
    s.params = at;                                            // [warps]{[4][32][NG], 4} floats
    at += AK_WARPS * (4 * 32 * NG + 4) * 4;
    s.qf = at;                                                // [8 NT columns][HD] halves
    at += 8 * NT * HD * 2;
    s.qs = at;                                                // [4 NT heads][NG + 1] floats
    at += 4 * NT * (NG + 1) * 4;
    s.rot = at;                                               // [warps][HD] floats: rotated rows
    at += AK_WARPS * HD * 4;
    s.cs = at;                                                // [HD / 2] (cos, sin)
    at += HD * 4;
    s.recv = at;                                              // [slots][CL][34] floats
    at += ((GV * NG + CL - 1) / CL) * CL * 34 * 4;
    s.bar = (at + 7) & ~7;
    s.total = s.bar + AK_WARPS * attn_kv4_stages(NG) * 8;
    return s;
}

template <int NG, int NT>
__global__ void __launch_bounds__(AK_THREADS, NT == 1 ? 2 : 1) attn_step_kv4_kernel(const AttnKv4Args a)
{
    namespace cg = cooperative_groups;
    constexpr int HD = 32 * NG, half = HD / 2, BB = 40 * HD, RS = HD + 2, STAGES = attn_kv4_stages(NG);
    cg::cluster_group cluster = cg::this_cluster();
    const int CL = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    extern __shared__ __align__(128) uint8_t smem[];
    const int G = a.n_heads / a.n_kv, GV = (G + a.splits - 1) / a.splits;   // query heads per kv head, and of a cluster
    const AttnKv4Smem at = attn_kv4_smem(NG, NT, GV, CL);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int unit = blockIdx.x / CL / a.clusters, nth = blockIdx.x / CL - unit * a.clusters;   // which cluster of its unit
    const int kvh = unit / a.splits, split = unit - kvh * a.splits;
    const int tok = blockIdx.y;
    const int h_lo = kvh * G + split * GV, n_h = min(GV, G - split * GV);   // this cluster's query heads
    uint8_t *ring = smem + at.ring + warp * (STAGES * BB);
    uint64_t *bar = (uint64_t *)(smem + at.bar) + warp * STAGES;
    __half *qf = (__half *)(smem + at.qf);
    float *qs = (float *)(smem + at.qs);
    float *rot = (float *)(smem + at.rot) + warp * HD;
    float2 *cs = (float2 *)(smem + at.cs);
    float *recv = (float *)(smem + at.recv);

    cluster_arrive();   // another CTA's shared memory may be written once it runs: waited for before the pushes
    if (lane == 0) {
        for (int s = 0; s < STAGES; s++) mbar_init(&bar[s], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    auto place = [&](int pos, int &first, int &b0, int &n_blk) {   // the blocks of the visible positions
        pos = max(0, min(pos, a.max_seq - 1));
        first = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
        b0 = first / KV4_BLOCK;
        n_blk = pos / KV4_BLOCK - b0 + 1;
        return pos;
    };
    auto at_work = [&](int n_blk) { return max(1, min(a.clusters, n_blk / (CL * AK_WARPS))); };
    const uint8_t *head_blocks = kv4_block(a.cache, a.n_blocks, kvh, 0, HD);
    int first, b0, n_blk;
    if (a.prefetch) {
        // Ahead of the kernel that may still be writing q, k_new or the cache: into L2 only, whatever is there
        const int p = __ldcg(a.step + 1);
        place(p, first, b0, n_blk);
        const int R = CL * at_work(n_blk), b = nth * CL + rank + R * warp;
        if (nth < at_work(n_blk) && lane < STAGES && b + R * AK_WARPS * lane < n_blk)
            l2_prefetch_bulk(head_blocks + (size_t)(b0 + b + R * AK_WARPS * lane) * BB, BB);
    }
    pdl_trigger();
    pdl_wait();
    const int pos = place(a.step ? __ldcg(a.step + 1) : a.pos + tok, first, b0, n_blk);
    const int NC = at_work(n_blk), R = CL * NC, cta = nth * CL + rank;
    if (nth >= NC) {
        cluster_wait();
        return;
    }
    const int stride = R * AK_WARPS, mine = cta + R * warp;
    const int n_mine = mine < n_blk ? (n_blk - mine + stride - 1) / stride : 0;
    auto load = [&](int i) {   // (lane 0) this warp's i-th block into its stage
        uint64_t *b = &bar[i % STAGES];
        mbar_arrive_expect_tx(b, BB);
        tma_load_1d(ring + (i % STAGES) * BB, head_blocks + (size_t)(b0 + mine + i * stride) * BB, BB, b);
    };
    if (lane == 0)
        for (int i = 0; i < min(n_mine, STAGES); i++) load(i);
    const bool rotate = a.theta > 0.f;
    if (rotate) {
        if (threadIdx.x < half) {
            float c, s;
            if (a.rope_tab && __float_as_int(__ldcg(&a.rope_tab[ATT_MAX_HD / 2].x)) == pos) {
                const float2 v = __ldcg(&a.rope_tab[threadIdx.x]);
                c = v.x;
                s = v.y;
            } else {
                rope_cs(RopeArgs{pos, a.theta, a.yarn_scale, a.yarn_orig_ctx, a.neox}, threadIdx.x, HD, c, s);
            }
            cs[threadIdx.x] = make_float2(c, s);
        }
        __syncthreads();
    }
    // a row of q or k, rotated, into this warp's `rot`
    auto rotated = [&](const float *src) {
        for (int i = lane; i < half; i += 32) {
            const int i0 = a.neox ? i : 2 * i, i1 = a.neox ? i + half : 2 * i + 1;
            float x0 = __ldcg(src + i0), x1 = __ldcg(src + i1);
            if (rotate) {
                const float2 v = cs[i];
                const float r0 = x0 * v.x - x1 * v.y, r1 = x0 * v.y + x1 * v.x;
                x0 = r0;
                x1 = r1;
            }
            rot[i0] = x0;
            rot[i1] = x1;
        }
        __syncwarp();
    };
    // ---- q as the column operand: head h is columns 2 h and 2 h + 1 ----
    for (int h = warp; h < 4 * NT; h += AK_WARPS) {
        float x[NG], top = 0.f;
        if (h < n_h) {
            rotated(a.q + ((size_t)tok * a.n_heads + h_lo + h) * HD);
#pragma unroll
            for (int j = 0; j < NG; j++) {
                x[j] = rot[32 * j + lane] * (a.scale * 1.44269504f);
                top = fmaxf(top, fabsf(x[j]));
            }
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
        } else {
#pragma unroll
            for (int j = 0; j < NG; j++) x[j] = 0.f;
        }
        // 2^e brings the largest element into [2^13, 2^14)
        const int e = top > 0.f ? max(-120, min(100, 127 + 13 - (int)(__float_as_uint(top) >> 23))) : 0;
        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
        float *head_qs = qs + h * (NG + 1);
        if (lane == 0) head_qs[NG] = 1.f / up;
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const float total = warp_sum(x[j]);
            if (lane == 0) head_qs[j] = total * up;
            // dim 32 j + lane = 8 tt + i: halves of word (j, tt): pairs (0,4) (1,5) (2,6) (3,7)
            const int tt = lane >> 3, i = lane & 7;
            const float y = x[j] * up;
            const __half hi = __float2half_rn(y), lo = __float2half_rn(y - __half2float(hi));
            const int slot = (j * 4 + tt) * 8 + (i & 3) * 2 + (i >> 2);
            qf[(2 * h) * HD + slot] = hi;
            qf[(2 * h + 1) * HD + slot] = lo;
        }
    }
    __syncthreads();
    Kv4Warp<NG, NT> w;
    float *scratch = (float *)(smem + at.params) + warp * w.SCRATCH;
    w.clear(scratch, lane);
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const float *head_qs = qs + (4 * n + (lane & 3)) * (NG + 1);
        w.back[n] = head_qs[NG];
#pragma unroll
        for (int j = 0; j < NG; j++) {
            w.qs[n][j] = head_qs[j];
            const uint4 v = *(const uint4 *)(qf + (8 * n + (lane >> 2)) * HD + (j * 4 + (lane & 3)) * 8);
            w.qf[n][j][0] = v.x; w.qf[n][j][1] = v.y; w.qf[n][j][2] = v.z; w.qf[n][j][3] = v.w;
        }
    }
    // ---- this warp's blocks ----
    for (int i = 0; i < n_mine; i++) {
        const int stage = i % STAGES;
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(&bar[stage], (i / STAGES) & 1))) {
            if (lane == 0) {
                if (a.status) *a.status = QZ_ERR_TIMEOUT;
                for (int k = i; k < min(n_mine, i + STAGES); k++) mbar_wait(&bar[k % STAGES], (k / STAGES) & 1);   // copies in flight
            }
            break;
        }
        uint8_t *blk = ring + stage * BB;
        const int base = (b0 + mine + i * stride) * KV4_BLOCK;
        const int lo = max(0, first - base), hi = min(KV4_BLOCK - 1, pos - base);
        if (a.k_new && base + hi == pos) {
            {
                // the new position: lanes 0.. quantise its key, lanes 16.. its value, into the staged block; split 0
                // copies the row to the cache
                rotated(a.k_new + (size_t)kvh * HD);
                const int e = lane & 15;
                const bool is_v = lane >= 16;
                if (e < 4 * NG) {
                    float x[8];
                    const float *v = a.v_new + (size_t)kvh * HD + 8 * e;
#pragma unroll
                    for (int c = 0; c < 8; c++) x[c] = is_v ? __ldcg(v + c) : rot[8 * e + c];
                    kv4_store8<NG>(x, blk, hi, e >> 2, e & 3, is_v, ((1u << (4 * NG)) - 1u) * 0x00010001u);
                }
                __syncwarp();
                if (split == 0) {
                    uint32_t *dst = (uint32_t *)(kv4_block(a.cache, a.n_blocks, kvh, pos / KV4_BLOCK, HD));
                    const uint32_t *src = (const uint32_t *)blk;
                    for (int c = lane; c < 10 * NG; c += 32) {   // K codes, K parameters, V codes, V parameters of the row
                        const int side = c / (5 * NG), k = c - side * 5 * NG;
                        const int word = side * 5 * HD + (k < 4 * NG ? hi * 4 * NG + k : 4 * HD + hi * NG + (k - 4 * NG));
                        dst[word] = src[word];
                    }
                }
            }
            __syncwarp();
        }
        w.block(blk, scratch, lo, hi, lane);
        if ((i & 3) == 3) w.flush();
        __syncwarp();   // every lane is done with the stage
        if (lane == 0 && i + STAGES < n_mine) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // (a patched block is overwritten by the copy)
            load(i + STAGES);
        }
    }
    w.flush();
    // ---- results of this warp over its own ring, then of the CTA ----
    float *part = (float *)(smem + at.ring);
    constexpr int WS = STAGES * BB / 4;   // floats from one warp's results to the next
    __syncwarp();
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const float total = w.sum(n);
        const int h = 4 * n + (lane & 3);
        float *dst = part + warp * WS + h * RS;
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const float4 v = w.out(n, j, lane, scratch);
            if (h < n_h) {
                *(float2 *)(dst + 2 + 32 * j + 4 * (lane >> 2)) = make_float2(v.x, v.y);
                *(float2 *)(dst + 4 + 32 * j + 4 * (lane >> 2)) = make_float2(v.z, v.w);
            }
        }
        if (lane < 4 && h < n_h) {
            dst[0] = w.ref[n];
            dst[1] = total;
        }
    }
    __syncthreads();
    // runs of 32 outputs: run e belongs to CTA e % CL, in its slot e / CL
    const int n_runs = n_h * NG, active = min(AK_WARPS, max(1, (n_blk - cta + R - 1) / R));
    cluster_wait();   // (arrived at the top) every CTA of the cluster has started
    for (int e = warp; e < n_runs; e += AK_WARPS) {
        const int h = e / NG, j = e - h * NG;
        float top = -3.0e38f;
        for (int k = 0; k < active; k++) top = fmaxf(top, part[k * WS + h * RS]);
        float l = 0.f, o = 0.f;
        for (int k = 0; k < active; k++) {
            const float *src = part + k * WS + h * RS;
            const float f = ex2(src[0] - top);
            l = fmaf(src[1], f, l);
            o = fmaf(src[2 + 32 * j + lane], f, o);
        }
        float *dst = cluster.map_shared_rank(recv, e % CL) + ((e / CL) * CL + rank) * 34;
        dst[2 + lane] = o;
        if (lane == 0) {
            dst[0] = top;
            dst[1] = l;
        }
    }
    cluster_arrive();
    cluster_wait();   // every push has landed
    for (int e = rank + CL * warp; e < n_runs; e += CL * AK_WARPS) {
        const float *src = recv + (e / CL) * CL * 34;
        const int head = h_lo + e / NG;
        float top = -3.0e38f, l = 0.f, o = 0.f;
        for (int c = 0; c < CL; c++) top = fmaxf(top, src[34 * c]);
        for (int c = 0; c < CL; c++) {
            const float f = ex2(src[34 * c] - top);
            l = fmaf(src[34 * c + 1], f, l);
            o = fmaf(src[34 * c + 2 + lane], f, o);
        }
        if (NC > 1) {
            const int run = (tok * a.n_kv * a.splits + unit) * 32 + e;
            float *ws = a.workspace + AK_COUNTERS + (size_t)run * a.clusters * 34;
            __stcg(ws + nth * 34 + 2 + lane, o);
            if (lane < 2) __stcg(ws + nth * 34 + lane, lane ? l : top);
            __syncwarp();
            int *count = (int *)a.workspace + run;
            int before = 0;
            // releases the warp's stores (ordered before it by the warp barrier), acquires the other clusters'
            if (lane == 0) asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
            before = __shfl_sync(0xFFFFFFFFu, before, 0);
            __syncwarp();   // (the shuffle orders no memory: lane 0's acquire is the warp's from here on)
            if (before != NC - 1) continue;
            if (lane == 0) *count = 0;   // for the next call
            float all_top = -3.0e38f;
            for (int c = 0; c < NC; c++) all_top = fmaxf(all_top, __ldcg(ws + 34 * c));
            l = o = 0.f;
            top = all_top;
            for (int c = 0; c < NC; c++) {
                const float f = ex2(__ldcg(ws + 34 * c) - top);
                l = fmaf(__ldcg(ws + 34 * c + 1), f, l);
                o = fmaf(__ldcg(ws + 34 * c + 2 + lane), f, o);
            }
        }
        if (a.sinks) {
            const float sink = a.sinks[head] * 1.44269504f, all = fmaxf(sink, top), f = ex2(top - all);
            l = fmaf(l, f, ex2(sink - all));
            o *= f;
        }
        const float r = o / l;
        const int first_out = head * HD + 32 * (e % NG);
        a.out[(size_t)tok * a.n_heads * HD + first_out + lane] = r;
        if (a.emit_q) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = __shfl_sync(0xFFFFFFFFu, r, (4 * lane + k) & 31);
            quantize4_store(v, (first_out >> 2) + (lane & 7), lane < 8, a.o);
        }
    }
}

}  // namespace qz
