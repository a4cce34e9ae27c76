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
// heads of 128 take 5.7 us (4.2 TB/s), 8192 take 66 (5.8 TB/s); one block per row, as the f32 form has it, took 21.7 and 338, most
// of it for angles and for starting blocks.
// Rows are q's, k's, then v's; 4 NG threads share one, each with four pairs, two vectors of four dims.  grid.y blocks share
// a token's rows where there are few tokens.
constexpr int RK4_THREADS = 256;

template <int NG>
__global__ void __launch_bounds__(RK4_THREADS) rope_kv4_rows_kernel(float *q, float *k, const float *__restrict__ v, uint8_t *__restrict__ cache,
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
