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
// of a warp whole sectors.  Over rows that together exceed L2, 8192 of 8 heads of 128: written 20.3 us, 3.8 TB/s (bound by the
// quantiser's issue slots as much as by HBM; 64-bit borders for every code and clamps took 21.3), read back 15.8 us, 4.9 TB/s; 8189 of 4
// heads of 96: 8.8 and 7.9 us; a few rows are bound by the launches (1.3 and 1.0 us in a replayed graph).
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

// Does m + 15 d reach hi?  Decided exactly: 15 d is exact, its sum with m is taken with the error that it leaves.
__device__ __forceinline__ bool kv4_reaches(float m, __half d, float hi)
{
    const float t = 15.f * __half2float(d), s = __fadd_rn(t, m), b = __fadd_rn(s, -t), err = __fadd_rn(__fadd_rn(t, -__fadd_rn(s, -b)), __fadd_rn(m, -b));
    return __fadd_rn(__fadd_rn(s, -hi), err) >= 0.f;   // (where s and hi differ by more than err, their difference has its sign)
}
// Parameters of a group from its extremes.  The f32 quotient (rounded up: a range of a few subnormals is not none) is right to
// 2^-22 of itself: only if it lies that close to an f16 number can that number, or the one above it, be the answer instead, and is
// asked exactly.
__device__ __forceinline__ void kv4_params(float lo, float hi, __half &m, __half &d)
{
    m = __float2half_rd(fmaxf(lo, -65504.f) + 0.f);   // (+ 0: a minimum of -0 is stored as 0)
    const float mf = __half2float(m), q = __fmul_ru(fmaxf(hi - mf, 0.f), 1.f / 15.f), near = q * (1.f / (1 << 20));
    d = __float2half_ru(fminf(q, 65504.f));
    const unsigned short bits = __half_as_ushort(d);
    const __half less = __ushort_as_half((unsigned short)(bits - 1));   // (of 0: NaN, which nothing is near to)
    if (__half2float(d) - q < near || q - __half2float(less) < near) {
        if (!kv4_reaches(mf, d, hi)) {
            if (bits < 0x7BFF) d = __ushort_as_half((unsigned short)(bits + 1));
        } else if (bits && kv4_reaches(mf, less, hi)) {
            d = less;
        }
    }
}

// (x - m) / d to nearest, ties to even, where its f32 value y, off by less than 2^-18 (15 * 2^-22), is too close to a border
// to tell: in 64 bits.
__device__ __forceinline__ float kv4_code_exact(float x, float m, float d, float y)
{
    const float below = floorf(y), half = below + 0.5f;
    const double r = ((double)x - (double)m) - (double)half * (double)d;
    return r > 0.0 || (r == 0.0 && ((int)below & 1)) ? fminf(below + 1.f, 15.f) : below;
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
    if (!ok) lo = -INFINITY;
#pragma unroll
    for (int s = 1; s < 4; s <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(mask, lo, s));
        hi = fmaxf(hi, __shfl_xor_sync(mask, hi, s));
    }
    __half m, d;
    uint32_t w = 0;
    if (lo > -INFINITY) {
        kv4_params(lo, hi, m, d);
        const float mf = __half2float(m), df = __half2float(d), inv = df > 0.f ? 1.f / df : 0.f;
        constexpr float WHOLE = 12582912.f;   // 1.5 * 2^23: a sum's low bits are the nearest integer
        bool odd = lo < -65504.f || df >= 65504.f;   // rare: saturated (codes may lie outside 0 .. 15), or close to a border
        float c[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float y = (x[i] - mf) * inv;
            c[i] = (y + WHOLE) - WHOLE;
            odd |= fabsf(fabsf(y - c[i]) - 0.5f) < 1e-5f;
        }
        if (odd) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = fminf(fmaxf((x[i] - mf) * inv, 0.f), 15.f);
                c[i] = (y + WHOLE) - WHOLE;
                if (fabsf(fabsf(y - c[i]) - 0.5f) < 1e-5f) c[i] = kv4_code_exact(x[i], mf, df, y);
            }
        }
        // four codes as one number of 16 bits
        const float a = fmaf(fmaf(fmaf(c[3], 16.f, c[2]), 16.f, c[1]), 16.f, c[0]) + WHOLE, b = fmaf(fmaf(fmaf(c[7], 16.f, c[6]), 16.f, c[5]), 16.f, c[4]) + WHOLE;
        w = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x5410);
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
                                                         const float *__restrict__ v, unsigned n_rows, int n_kv, int n_blocks, int pos0)
{
    constexpr int PER = 4 * NG;   // threads per row
    pdl_wait();
    pdl_trigger();
    const unsigned row = (blockIdx.x * 256ull + threadIdx.x) / PER;   // (memory holds less than 2^31 rows)
    const int j = (int)((blockIdx.x * 256ull + threadIdx.x) % PER), g = j >> 2, t = j & 3;
    const unsigned mask = __ballot_sync(0xFFFFFFFFu, row < n_rows);
    if (row >= n_rows) return;
    const float *src = (blockIdx.y ? v : k) + (size_t)row * (32 * NG) + 32 * g + 8 * t;
    const float4 a = __ldg((const float4 *)src), b = __ldg((const float4 *)src + 1);
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const unsigned tok = row / (unsigned)n_kv;
    const int head = (int)(row - tok * n_kv);
    const int pos = pos0 + (int)tok;
    kv4_store8<NG>(x, kv4_block(cache, n_blocks, head, pos / KV4_BLOCK, 32 * NG), pos % KV4_BLOCK, g, t, blockIdx.y != 0, mask);
}

// The reverse: the values of positions pos0 .. as f32 rows.
template <int NG>
__global__ void __launch_bounds__(256) kv4_read_kernel(float *__restrict__ k, float *__restrict__ v, const uint8_t *__restrict__ cache,
                                                       unsigned n_rows, int n_kv, int n_blocks, int pos0)
{
    constexpr int PER = 4 * NG, HD = 32 * NG;
    pdl_wait();
    pdl_trigger();
    const unsigned row = (blockIdx.x * 256ull + threadIdx.x) / PER;
    if (row >= n_rows) return;
    const int j = (int)((blockIdx.x * 256ull + threadIdx.x) % PER), g = j >> 2, t = j & 3;
    const unsigned tok = row / (unsigned)n_kv;
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
    float4 *dst = (float4 *)((blockIdx.y ? v : k) + (size_t)row * HD + 32 * g + 8 * t);
    dst[0] = make_float4(x[0], x[1], x[2], x[3]);
    dst[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// cuda_rope_kv_rows with a 4-bit cache: token blockIdx.x at position pos0 + blockIdx.x; q and k rotated in place (theta <= 0: left
// as they are), k and v quantised.  The angles of a token are computed once for all of its rows: 512 tokens of 32 / 8
// heads of 128 take 6.1 us (3.9 TB/s; 5.4 from L2), 8192 take 61 (6.2 TB/s; at 57 registers instead of 40 69 us); one block per row, as the f32 form has it, took 21.7 and 338, most
// of it for angles and for starting blocks.
// Rows are q's, k's, then v's; 4 NG threads share one, each with four pairs, two vectors of four dims.  grid.y blocks share
// a token's rows where there are few tokens.
constexpr int RK4_THREADS = 256;

template <int NG>
__global__ void __launch_bounds__(RK4_THREADS, 6) rope_kv4_rows_kernel(float *q, float *k, const float *__restrict__ v, uint8_t *__restrict__ cache,
                                                                    int n_heads, int n_kv, int n_blocks, int pos0, float theta,
                                                                    float yarn_scale, int yarn_orig_ctx, int neox)
{
    constexpr int HD = 32 * NG, half = HD / 2, PER = 4 * NG, ROWS = 32 / PER;   // threads per row, rows per warp
    __shared__ float2 cs[half];   // (cos, sin)
    pdl_wait();
    pdl_trigger();
    const int tok = blockIdx.x, pos = pos0 + tok, lane = threadIdx.x & 31;
    const bool rotate = theta > 0.f;
    if (rotate) {
        if (threadIdx.x < half) {
            const RopeArgsLite r{pos, theta, yarn_scale, yarn_orig_ctx};
            float s, c;
            rope_cs_lite(r, threadIdx.x, HD, c, s);
            cs[threadIdx.x] = make_float2(c, s);
        }
        __syncthreads();
    }
    const int in_warp = lane / PER, j = lane % PER, n_q = rotate ? n_heads : 0, n_rows = n_q + 2 * n_kv;
    const int at0 = neox ? 4 * j : 8 * j, at1 = neox ? half + 4 * j : 8 * j + 4;
    for (int r0 = ((int)blockIdx.y * (RK4_THREADS / 32) + (threadIdx.x >> 5)) * ROWS; r0 < n_rows; r0 += gridDim.y * (RK4_THREADS / 32) * ROWS) {
        const int row = r0 + in_warp;
        const bool there = in_warp < ROWS && row < n_rows;
        const unsigned mask = __ballot_sync(0xFFFFFFFFu, there);
        if (!there) continue;
        const bool is_q = row < n_q, is_v = row >= n_q + n_kv;
        const int head = is_q ? row : is_v ? row - n_q - n_kv : row - n_q;
        float x[8];
        if (is_v) {
            const float4 *src = (const float4 *)(v + ((size_t)tok * n_kv + head) * HD + 8 * j);
            const float4 a = __ldg(src), b = __ldg(src + 1);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else {
            float *at = is_q ? q + ((size_t)tok * n_heads + head) * HD : k + ((size_t)tok * n_kv + head) * HD;
            const float4 a = *(const float4 *)(at + at0), b = *(const float4 *)(at + at1);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
            if (rotate) {
                auto turn = [&](float &x0, float &x1, int pair) {
                    const float2 w = cs[pair];
                    const float y0 = x0 * w.x - x1 * w.y, y1 = x0 * w.y + x1 * w.x;
                    x0 = y0;
                    x1 = y1;
                };
                if (neox) {
#pragma unroll
                    for (int c = 0; c < 4; c++) turn(x[c], x[4 + c], 4 * j + c);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; c++) turn(x[2 * c], x[2 * c + 1], 4 * j + c);
                }
                *(float4 *)(at + at0) = make_float4(x[0], x[1], x[2], x[3]);
                *(float4 *)(at + at1) = make_float4(x[4], x[5], x[6], x[7]);
            }
        }
        // all threads of the warp's rows take part in the exchange; a query's have nothing to store
        if (neox) {   // dims 8 j ..: vectors 2 j and 2 j + 1 of the row, which threads 2 j .. of its first or second half hold
            const int from = in_warp * PER + (2 * j) % PER;
            float y[8];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float a0 = __shfl_sync(mask, x[c], from), a1 = __shfl_sync(mask, x[c], from + 1);
                const float b0 = __shfl_sync(mask, x[4 + c], from), b1 = __shfl_sync(mask, x[4 + c], from + 1);
                y[c] = 2 * j < PER ? a0 : b0;
                y[4 + c] = 2 * j < PER ? a1 : b1;
            }
            if (!is_v) {
#pragma unroll
                for (int c = 0; c < 8; c++) x[c] = y[c];
            }
        }
        const unsigned stored = __ballot_sync(mask, !is_q);
        if (!is_q)
            kv4_store8<NG>(x, kv4_block(cache, n_blocks, head, pos / KV4_BLOCK, HD), pos % KV4_BLOCK, j >> 2, j & 3, is_v, stored);
    }
}

}  // namespace qz
