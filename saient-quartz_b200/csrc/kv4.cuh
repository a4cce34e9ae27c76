// The 4-bit KV cache: rows of keys and values are quantised as they are written and read back as the values they
// stand for.  The reference keeps f32 caches (src/cuda.rs:361-492, cuda_kv_append src/cuda_kernels.cu:622-638).
//
// A group is 32 consecutive dims of one (position, kv head).  With lo and hi its smallest and largest element
//   m = the largest f16 <= lo,   d = the smallest f16 with m + 15 d >= hi,
//   code = (x - m) / d rounded to nearest, ties to even, 0 .. 15,   value = m + d * code (one rounding to f32).
// m is rounded down and d up so that every element lies inside [m, m + 15 d]: |value - x| <= d / 2.  The two
// parameters cost 32 bits per 32 values (5 bits per value in all); f16 because a group's offset may be many steps
// large (keys have channels with a large mean), where bf16's 8 bits would shift the whole group by half a step.
// Beyond f16's range m and d saturate and the codes clamp.  A group with an element that is not finite stores m = NaN
// and reads back as NaN throughout.
//
// Layout: [kv head][block of 32 positions], a block being K codes | K parameters | V codes | V parameters, 40 head_dim
// bytes in all and contiguous, so that an attention warp fetches 32 positions of a head with one bulk copy.  Every
// position owns whole bytes (an append never reads its neighbours).  Inside a row the codes are permuted so that a
// lane's fragment of mma.m16n8k16 is one aligned vector (NG = head_dim / 32 groups per row):
//   K  32-bit word t * NG + g, t < 4: dims 32 g + 8 t + i in nibbles i < 8   (K is the row operand: k runs over dims)
//   V  16-bit word r * NG + g, r < 8: dims 32 g + 4 r + i in nibbles i < 4   (V^T is: k runs over positions)
//   parameters: NG halves m, then NG halves d.
//
// Writing and reading are bound by HBM: 4 bytes on one side, 0.625 on the other.  Eight dims per thread make every access
// of a warp whole sectors.  8192 rows of 8 heads of 128, appended and read back: 36 us, 4.3 TB/s; 8189 of 4 heads of 96:
// 17.0 us, 3.4 TB/s; a few rows are bound by the two launches (2.8 us in a replayed graph).
#pragma once

#include "activation.cuh"
#include "rope.cuh"

namespace qz {

constexpr int KV4_BLOCK = 32;   // positions per block

__host__ __device__ inline size_t kv4_block_bytes(int head_dim) { return (size_t)40 * head_dim; }
__host__ __device__ inline int kv4_blocks(int max_seq) { return (int)(((long long)max_seq + KV4_BLOCK - 1) / KV4_BLOCK); }

__device__ __forceinline__ uint8_t *kv4_block(uint8_t *cache, int n_blocks, int head, int block, int head_dim)
{
    return cache + ((size_t)head * n_blocks + block) * kv4_block_bytes(head_dim);
}

// Parameters of a group from its extremes.  The two borders (is m + 15 d >= hi, would one f16 less do) are decided in
// 64 bits, where every quantity is exact for operands within 2^29 of one another.
__device__ __forceinline__ void kv4_params(float lo, float hi, __half &m, __half &d)
{
    m = __float2half_rd(fmaxf(lo, -65504.f) + 0.f);   // (+ 0: a minimum of -0 is stored as 0)
    const double span = fmax((double)hi - (double)__half2float(m), 0.0);
    float df = __half2float(__float2half_ru(fminf((float)(span * (1.0 / 15.0)), 65504.f)));
    // the product above may be one ulp (of f32) to either side of span / 15: at most one f16 away from the answer
    if (15.0 * (double)df < span && df < 65504.f) df = __half2float(__ushort_as_half((unsigned short)(__half_as_ushort(__float2half_rn(df)) + 1)));
    if (df > 0.f) {
        const float less = __half2float(__ushort_as_half((unsigned short)(__half_as_ushort(__float2half_rn(df)) - 1)));
        if (15.0 * (double)less >= span) df = less;
    }
    d = __float2half_rn(df);
}

// (x - m) / d to nearest, ties to even.  The f32 quotient is off by less than 2^-18 (15 * 2^-22), so only a quotient
// that close to a border needs the exact comparison, in 64 bits; it is rare.
__device__ __forceinline__ uint32_t kv4_code(float x, float m, float d, float inv)
{
    const float y = fminf(fmaxf((x - m) * inv, 0.f), 15.f);
    float c = rintf(y);
    if (fabsf(fabsf(y - c) - 0.5f) < 1e-5f) {
        const float below = floorf(y), half = below + 0.5f;
        const double r = ((double)x - (double)m) - (double)half * (double)d;
        c = r > 0.0 ? below + 1.f : (r < 0.0 ? below : ((((int)below) & 1) ? below + 1.f : below));
        c = fminf(c, 15.f);
    }
    return (uint32_t)c;
}

// Quantise eight consecutive dims (32 g + 8 t ..) of a row; the four lanes of a group (t = 0..3, consecutive lanes of
// a warp, all present) call it together.  `blk` is the block, `row` the position inside it.
template <int NG>
__device__ __forceinline__ void kv4_store8(const float (&x)[8], uint8_t *blk, int row, int g, int t, bool is_v, unsigned mask)
{
    constexpr int HD = 32 * NG;
    float lo = x[0], hi = x[0];
    bool ok = isfinite(x[0]);
#pragma unroll
    for (int i = 1; i < 8; i++) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        ok = ok && isfinite(x[i]);
    }
    int all_ok = ok ? 1 : 0;
#pragma unroll
    for (int s = 1; s < 4; s <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(mask, lo, s));
        hi = fmaxf(hi, __shfl_xor_sync(mask, hi, s));
        all_ok &= __shfl_xor_sync(mask, all_ok, s);
    }
    __half m, d;
    uint32_t w = 0;
    if (all_ok) {
        kv4_params(lo, hi, m, d);
        const float mf = __half2float(m), df = __half2float(d), inv = df > 0.f ? 1.f / df : 0.f;
        if (df > 0.f) {
#pragma unroll
            for (int i = 0; i < 8; i++) w |= kv4_code(x[i], mf, df, inv) << (4 * i);
        }
    } else {
        m = __ushort_as_half((unsigned short)0x7FFF);
        d = __ushort_as_half((unsigned short)0);
    }
    uint8_t *side = blk + (is_v ? 20 * HD : 0);
    if (is_v) {
        uint16_t *c = (uint16_t *)(side + row * (HD / 2));
        c[(2 * t) * NG + g] = (uint16_t)w;
        c[(2 * t + 1) * NG + g] = (uint16_t)(w >> 16);
    } else {
        ((uint32_t *)(side + row * (HD / 2)))[t * NG + g] = w;
    }
    if (t == 0) {
        __half *p = (__half *)(side + 16 * HD) + row * (2 * NG);
        p[g] = m;
        p[NG + g] = d;
    }
}

// Rows k, v [n_tok][n_kv_heads * head_dim] into positions pos0 .. : one thread per eight dims; grid.y 0 keys, 1 values.
template <int NG>
__global__ void __launch_bounds__(256) kv4_append_kernel(uint8_t *__restrict__ cache, const float *__restrict__ k,
                                                         const float *__restrict__ v, long long n_rows, int n_kv, int n_blocks, int pos0)
{
    constexpr int PER = 4 * NG;   // threads per row
    pdl_wait();
    pdl_trigger();
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long row = e / PER;
    const int j = (int)(e - row * PER), g = j >> 2, t = j & 3;
    const unsigned mask = __ballot_sync(0xFFFFFFFFu, row < n_rows);
    if (row >= n_rows) return;
    const float *src = (blockIdx.y ? v : k) + row * (32 * NG) + 32 * g + 8 * t;
    const float4 a = __ldg((const float4 *)src), b = __ldg((const float4 *)src + 1);
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const long long tok = row / n_kv;
    const int head = (int)(row - tok * n_kv);
    const int pos = pos0 + (int)tok;
    kv4_store8<NG>(x, kv4_block(cache, n_blocks, head, pos / KV4_BLOCK, 32 * NG), pos % KV4_BLOCK, g, t, blockIdx.y != 0, mask);
}

// The reverse: the values of positions pos0 .. as f32 rows.
template <int NG>
__global__ void __launch_bounds__(256) kv4_read_kernel(float *__restrict__ k, float *__restrict__ v, const uint8_t *__restrict__ cache,
                                                       long long n_rows, int n_kv, int n_blocks, int pos0)
{
    constexpr int PER = 4 * NG, HD = 32 * NG;
    pdl_wait();
    pdl_trigger();
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long row = e / PER;
    if (row >= n_rows) return;
    const int j = (int)(e - row * PER), g = j >> 2, t = j & 3;
    const long long tok = row / n_kv;
    const int head = (int)(row - tok * n_kv);
    const int pos = pos0 + (int)tok, r = pos % KV4_BLOCK;
    const uint8_t *side = kv4_block(const_cast<uint8_t *>(cache), n_blocks, head, pos / KV4_BLOCK, HD) + (blockIdx.y ? 20 * HD : 0);
    uint32_t w;
    if (blockIdx.y) {
        const uint16_t *c = (const uint16_t *)(side + r * (HD / 2));
        w = (uint32_t)c[(2 * t) * NG + g] | (uint32_t)c[(2 * t + 1) * NG + g] << 16;
    } else {
        w = ((const uint32_t *)(side + r * (HD / 2)))[t * NG + g];
    }
    const __half *p = (const __half *)(side + 16 * HD) + r * (2 * NG);
    const float m = __half2float(p[g]), d = __half2float(p[NG + g]);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = fmaf(d, (float)((w >> (4 * i)) & 15u), m);
    float4 *dst = (float4 *)((blockIdx.y ? v : k) + row * HD + 32 * g + 8 * t);
    dst[0] = make_float4(x[0], x[1], x[2], x[3]);
    dst[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// rope_kv_rows_kernel with a 4-bit cache: token t = blockIdx.y at position pos0 + t; q and k rotated in place (theta <= 0:
// left as they are), then warp 0 of a key head quantises its k and warp 1 its v.  grid.x = query heads, then kv heads.
template <int NG>
__global__ void __launch_bounds__(64) rope_kv4_rows_kernel(float *q, float *k, const float *__restrict__ v, uint8_t *__restrict__ cache,
                                                           int n_heads, int n_kv, int n_blocks, int pos0, float theta,
                                                           float yarn_scale, int yarn_orig_ctx, int neox)
{
    constexpr int HD = 32 * NG, half = HD / 2;
    __shared__ __align__(16) float ks[HD];
    pdl_wait();
    pdl_trigger();
    const int i = threadIdx.x, tok = blockIdx.y, pos = pos0 + tok;
    const bool is_k = (int)blockIdx.x >= n_heads;
    const int head = is_k ? blockIdx.x - n_heads : blockIdx.x;
    float *xh = is_k ? k + ((size_t)tok * n_kv + head) * HD : q + ((size_t)tok * n_heads + head) * HD;
    if (i < half) {
        const int i0 = neox ? i : 2 * i, i1 = neox ? i + half : 2 * i + 1;
        float a = xh[i0], b = xh[i1];
        if (theta > 0.f) {
            const RopeArgsLite r{pos, theta, yarn_scale, yarn_orig_ctx};
            float s, c;
            rope_cs_lite(r, i, HD, c, s);
            const float r0 = a * c - b * s, r1 = a * s + b * c;
            a = r0;
            b = r1;
            xh[i0] = a;
            xh[i1] = b;
        }
        if (is_k) {
            ks[i0] = a;
            ks[i1] = b;
        }
    }
    if (!is_k) return;
    __syncthreads();
    const int lane = i & 31;
    if (lane >= 4 * NG) return;
    const bool is_v = i >= 32;
    const float *src = (is_v ? v + ((size_t)tok * n_kv + head) * HD : ks) + 8 * lane;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = src[e];
    kv4_store8<NG>(x, kv4_block(cache, n_blocks, head, pos / KV4_BLOCK, HD), pos % KV4_BLOCK, lane >> 2, lane & 3, is_v,
                   4 * NG == 32 ? 0xFFFFFFFFu : (1u << (4 * NG)) - 1u);
}

}  // namespace qz
