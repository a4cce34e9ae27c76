// Causal attention of a prompt's tokens over the 4-bit cache (kv4.cuh), on the 5th-generation tensor cores.
//
// One CTA per (kv head, 128 query rows: 128 / G tokens by the G query heads of the kv head), one KV tile of 64 positions
// after the other, longest CTAs first.  f32 in and out means 22 bits in both products, so every operand is split into two
// f16 parts and a product takes three MMAs, the two small ones first (lo hi + hi lo + hi hi):
//   S[row, pos]  = Q K^T   A = Q in tensor memory (rows scaled by a power of two), B = K tile in shared memory, K-major
//   O[row, dim]  = P V     A = P in tensor memory, over S's own columns, B = V tile in shared memory, dims contiguous
// A value is d (code - 8) + (m + 8 d).  The first term's two parts are exact and cost two packed instructions for two
// values (hi = d c rounded, lo = d c - hi by one HFMA2: d has 11 bits, c four); the second is the same for the 32 dims of a
// group, so it is a product of its own, with m and 8 d as they are: 8 more k of S against the sums of q over the groups, 8
// more columns of O.  (Values split in f32 take ten instructions for two: 2048 tokens of 32 / 8 heads of
// 128 took 182 us so, 171 with this.)
// A operands live in tensor memory because a 64-wide MMA that fetched them from shared memory would be bound by that.
// The tensor core rounds its sums towards zero, so O is never carried across tiles there: each tile's O starts from zero
// and is added to f32 registers, where a raised softmax reference is also paid for (one factor per row and tile).
//
//   warps 0-3   one row per thread: S from tensor memory, mask, weights 2^11 exp2(s - ref), their sum, P back.  The
//               reference is raised only when a score exceeds it by 2^4: weights stay below 2^15, and their lo parts keep
//               clear of f16's subnormals down to weights of 2^-14 (many small ones beside a large one, as a sink has, add up).
//   warps 4-11  fill a ring of three (K, V) stages from the cache, 8 dims of a position at a time.  The keys, or the values, of
//               a tile with a step above 8188 (8 d would overflow) are taken by an eighth: exact but for steps and minima
//               below 2^-11, which are then off by 2^-22 at most.  Between two stages they add a finished O tile to their
//               half of a row.
//   warp 12     issues S(j), then P V of tile j - 1: the tensor core works while the weights are computed.
// Columns of tensor memory: Q 144 (hi, lo, sums over groups), S / P 2 x 64, O 144 (two halves of 64 dims, 16 for m and 8 d).
// Within every 8 dims the tiles' order is (0,4,1,5,2,6,3,7), which unpacking produces for free; Q is put in that order,
// and O's columns are written out by it.
// Positions outside [first visible, last visible] of the CTA count as zero whatever the cache holds there; a visible V
// group that is NaN is taken as zero by the MMA (0 * NaN would reach rows that do not see it) and noted in a bit mask,
// from which the rows that see it are set to NaN.
//
// Measured (32 / 8 heads of 128, replayed): 512 tokens 21.8 us, 2048 122 us = 281 TF of attention, 843 TF with the three
// products; 512 tokens at 16000 404 us, 338 TF.  Bound by the unpacking and softmax warps' issue and by shared memory: a tile takes
// some 3600 cycles, of which the MMAs need 1660 (13.6 MFLOP at 8192 a cycle), its operands' way through shared memory some
// 1350; the tensor pipe is active 44 % of the time.  Tried: weights before the maximum is known, repeated when it rises (2048
// tokens: 137 us); parameters checked by a warp of their own (124 us).
#pragma once

#include "attn_kv4.cuh"
#include "tcgen05.cuh"

namespace qz {

constexpr int APK_BN = 64, APK_STAGES = 3, APK_THREADS = 512;
constexpr float APK_RAISE = 4.f, APK_CARRY = 11.f;   // log2: how far a score may exceed the reference, what weights carry

struct AttnPromptKv4Args {
    float *out;
    const float *q;
    const uint8_t *cache;
    int n_tok, n_heads, n_kv, n_blocks, pos0, window, tq;   // tq: tokens per CTA
    float scale;
    const float *sinks;
    int *status;
};

struct AttnPromptKv4Shared {
    uint64_t full[APK_STAGES], free_[APK_STAGES], s_full[2], p_full[2], o_free, q_done;
    float corr[4][UMMA_M];           // factor of a row's earlier outputs at tile j (slot j % 4)
    float scale_k[4], scale_v[4];    // 1 / what the tile's K and V were multiplied with
    uint32_t nan_v[4][4][2];         // positions of the tile whose V group is NaN, by group
    float inv[UMMA_M];               // 1 / sum of weights
    uint32_t nan_row[UMMA_M];        // groups of the row's output that are NaN
    uint32_t tmem;
};

__host__ __device__ constexpr size_t attn_prompt_kv4_smem(int NG)
{
    return (size_t)APK_STAGES * (4 * ((NG + 1) / 2) + 1) * APK_BN * 128 + 1024 + sizeof(AttnPromptKv4Shared);
}

// eight products d (code - 8) of a word as two 16-byte rows of f16, hi and lo, in the order (0,4,1,5,2,6,3,7)
__device__ __forceinline__ void kv4_split8(const Nibbles &nib, uint32_t w, __half2 d, uint4 &hi, uint4 &lo)
{
    uint32_t x[4], h[4], l[4];
    nib.pairs(w, x);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 c = *(const __half2 *)&x[i], p = __hmul2_rn(d, c), r = __hfma2(d, c, __hneg2(p));
        h[i] = *(const uint32_t *)&p;
        l[i] = *(const uint32_t *)&r;
    }
    hi = make_uint4(h[0], h[1], h[2], h[3]);
    lo = make_uint4(l[0], l[1], l[2], l[3]);
}

template <int N>
__device__ __forceinline__ void ldg_words(const void *p, uint32_t (&x)[N])
{
    if constexpr (N == 4) {
        const uint4 w = __ldcg((const uint4 *)p);
        x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
    } else if constexpr (N == 2) {
        const uint2 w = __ldcg((const uint2 *)p);
        x[0] = w.x; x[1] = w.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = __ldcg((const uint32_t *)p + i);
    }
}
// half k of an array of words
template <int N>
__device__ __forceinline__ uint32_t bits_of(const uint32_t (&x)[N], int k) { return (x[k >> 1] >> (16 * (k & 1))) & 0xFFFFu; }
template <int N>
__device__ __forceinline__ float half_of(const uint32_t (&x)[N], int k) { return __half2float(__ushort_as_half((unsigned short)bits_of(x, k))); }

template <int NG>
__global__ void __launch_bounds__(APK_THREADS, 1) attn_prompt_kv4_kernel(const AttnPromptKv4Args a)
{
    constexpr int HD = 32 * NG, NH = (NG + 1) / 2, HALF = APK_BN * 128, SIDE = NH * HALF, STAGE = 4 * SIDE + HALF;   // bytes: 64 dims, a part, K and V and their m and 8 d
    constexpr int AT_K = 0, AT_V_LO = 2 * SIDE, AT_V = 3 * SIDE, AT_X = 4 * SIDE;   // (the m and 8 d follow V's hi part as its next columns)
    constexpr uint32_t T_Q = 0, T_S = 160, T_O = 288, T_X = T_O + 64 * NH;          // tensor-memory columns
    extern __shared__ unsigned char smem_raw[];
    unsigned char *ring = (unsigned char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    AttnPromptKv4Shared &s = *(AttnPromptKv4Shared *)(ring + APK_STAGES * STAGE);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = blockIdx.x, G = a.n_heads / a.n_kv;
    const int t0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * a.tq, nt = min(a.tq, a.n_tok - t0);
    const int p_first = a.pos0 + t0, p_last = p_first + nt - 1;
    const int k_lo = a.window > 0 ? max(0, p_first + 1 - a.window) : 0, b0 = k_lo / KV4_BLOCK;
    const int base0 = b0 * KV4_BLOCK, n_tiles = (p_last - base0) / APK_BN + 1;
    if (threadIdx.x == 0) {
        for (int i = 0; i < APK_STAGES; i++) {
            mbar_init(&s.full[i], 8);
            mbar_init(&s.free_[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s.s_full[i], 1);
            mbar_init(&s.p_full[i], 4);
        }
        mbar_init(&s.o_free, 8);
        mbar_init(&s.q_done, 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x < 32) ((uint32_t *)s.nan_v)[threadIdx.x] = 0;
    for (int i = threadIdx.x; i < APK_STAGES * HALF / 16; i += APK_THREADS)   // what the m and 8 d do not fill stays zero
        *(uint4 *)(ring + (i / (HALF / 16)) * STAGE + AT_X + 16 * (i % (HALF / 16))) = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (warp == 12) tmem_alloc(&s.tmem, 512);
    pdl_trigger();
    pdl_wait();   // q and the cache's rows come from the launches before
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    bool ok = true;
    const int row = 32 * (warp & 3) + lane;   // (warps 0 to 11) this thread's row, and its token and head
    const int tok = row / G, head = kvh * G + row % G;
    const bool is_row = row < nt * G;

    // registers: 128 a thread at launch; the issuing warpgroup gives 64 of each of its threads away, the others take 16, 24 and
    // 24 a thread: as many together
    if (warp < 4) asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    else if (warp < 12) asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp < 4) {
        // ---- Q into tensor memory ----
        const uint32_t lanes = (uint32_t)(32 * warp) << 16;
        const float to_log2 = a.scale * 1.44269504f;
        // rows come in one after the other, copied to the last stage, which the filling warps
        // leave alone until then (a thread that reads its own row touches 32 rows at once: 2048 tokens took 151 us so, 129 with
        // this); 16-byte columns are rotated by the row against bank conflicts
        constexpr int COLS = HD / 4;
        float4 *stage_q = (float4 *)(ring + (APK_STAGES - 1) * STAGE) + warp * 32 * COLS;
        const float4 *q0 = (const float4 *)(a.q + ((size_t)t0 * a.n_heads + (size_t)kvh * G) * HD);
        const int my_row = is_row ? (tok * a.n_heads + row % G) * COLS : -1;
#pragma unroll 8
        for (int i = lane; i < 32 * COLS; i += 32) {
            const int r = i / COLS, from = __shfl_sync(0xFFFFFFFFu, my_row, r);
            cp_async16(stage_q + r * COLS + (i % COLS + r) % COLS, q0 + max(from, 0) + i % COLS, from >= 0);
        }
        cp_async_wait_all();
        __syncwarp();
        auto q_at = [&](int c) { return stage_q[lane * COLS + (c + lane) % COLS]; };
        float top = 0.f;
#pragma unroll 8
        for (int c = 0; c < COLS; c++) {
            const float4 v = q_at(c);
            top = fmaxf(top, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        }
        top *= fabsf(to_log2);
        const int e = top > 0.f ? max(-120, min(100, 127 + 8 - (int)(__float_as_uint(top) >> 23))) : 0;   // the largest element into [2^8, 2^9): 32 of them fit f16
        const float up = __uint_as_float((uint32_t)(127 + e) << 23), back = __uint_as_float((uint32_t)(127 - e) << 23);
        float sum[4] = {0.f, 0.f, 0.f, 0.f};   // of q over the groups
#pragma unroll
        for (int g = 0; g < NG; g++) {
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float4 u = q_at(8 * g + 2 * c), v = q_at(8 * g + 2 * c + 1);
                const float x[4] = {u.x, u.y, u.z, u.w}, y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = x[i] * to_log2 * up, r = y[i] * to_log2 * up;
                    const uint32_t h = pack_half2(p, r);
                    const float2 f = __half22float2(*(const __half2 *)&h);
                    sum[g] += p + r;
                    hi[4 * c + i] = h;
                    lo[4 * c + i] = pack_half2(p - f.x, r - f.y);
                }
            }
            tc_st16(tmem + lanes + T_Q + 16 * g, hi);
            tc_st16(tmem + lanes + T_Q + 64 + 16 * g, lo);
        }
        {
            uint32_t x[16] = {};   // hi: (0,1) (2,3) for m, the same for 8 d, zeros; then lo
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t h = pack_half2(sum[2 * i], sum[2 * i + 1]);
                const float2 f = __half22float2(*(const __half2 *)&h);
                x[i] = x[2 + i] = h;
                x[8 + i] = x[10 + i] = pack_half2(sum[2 * i] - f.x, sum[2 * i + 1] - f.y);
            }
            tc_st16(tmem + lanes + T_Q + 128, x);
        }
        tc_wait_st();
        tc_fence_before();
        asm volatile("bar.sync 1, 160;" ::: "memory");   // with the issuing warp: Q is in place
        if (lane == 0) mbar_arrive(&s.q_done);           // the last stage may be filled
        // ---- tiles ----
        const int p_row = p_first + tok, lo_row = a.window > 0 ? max(0, p_row + 1 - a.window) : 0;
        float ref = -3.0e38f, l = 0.f;
        uint32_t nan_groups = 0;
        for (int j = 0; j < n_tiles; j++) {
            const uint32_t t_s = tmem + lanes + T_S + 64 * (j & 1);
            ok = ok && mbar_wait(&s.s_full[j & 1], (j >> 1) & 1) && mbar_wait(&s.full[j % APK_STAGES], (j / APK_STAGES) & 1);
            if (!__all_sync(0xFFFFFFFFu, ok)) break;
            tc_fence_after();
            const float f = back * s.scale_k[j & 3];
            const int lo = lo_row - (base0 + APK_BN * j), hi = p_row - (base0 + APK_BN * j);   // visible columns
            const bool partial = __any_sync(0xFFFFFFFFu, lo > 0 || hi < APK_BN - 1);
            auto load = [&](int c, uint32_t (&v)[32]) {   // (twice: 64 values do not fit the registers beside the rest)
                tc_ld32(t_s + 32 * c, v);
                if (partial) {
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (32 * c + i < lo || 32 * c + i > hi) v[i] = 0xFF800000u;
                }
            };
            float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t v[32];
                load(c, v);
#pragma unroll
                for (int i = 0; i < 32; i++) top4[i & 3] = fmaxf(top4[i & 3], __uint_as_float(v[i]));
            }
            const float y = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * f;
            float corr = 1.f;
            if (y > ref + APK_RAISE) {
                corr = ex2(ref - y);
                l *= corr;
                ref = y;
            }
            s.corr[j & 3][row] = corr;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const uint32_t n0 = s.nan_v[j & 3][g][0], n1 = s.nan_v[j & 3][g][1];
                if (n0 | n1) {   // rare: does this row see one of them?
                    const uint64_t seen = hi < 0 || lo > 63 ? 0 : (~0ull >> (63 - min(63, hi))) & (~0ull << max(0, lo));
                    if (seen & ((uint64_t)n1 << 32 | n0)) nan_groups |= 1u << g;
                }
            }
            float l4[4] = {0.f, 0.f, 0.f, 0.f};
            const float minus = APK_CARRY - ref;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t v[32], ph[16], pl[16];
                load(c, v);
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float p0 = ex2(fmaf(__uint_as_float(v[2 * i]), f, minus)), p1 = ex2(fmaf(__uint_as_float(v[2 * i + 1]), f, minus));
                    l4[(2 * i) & 3] += p0;
                    l4[(2 * i + 1) & 3] += p1;
                    const float h0 = __uint_as_float(__float_as_uint(p0) & 0xFFFFE000u), h1 = __uint_as_float(__float_as_uint(p1) & 0xFFFFE000u);
                    ph[i] = pack_half2(h0, h1);
                    pl[i] = pack_half2(p0 - h0, p1 - h1);
                }
                tc_st16(t_s + 32 * c, ph);
                tc_st16(t_s + 32 * c + 16, pl);
            }
            l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.p_full[j & 1]);
        }
        if (a.sinks && is_row) {
            const float sink = a.sinks[head] * 1.44269504f, all = fmaxf(ref, sink), down = ex2(ref - all);
            s.inv[row] = down / fmaf(l, down, ex2(sink - all + APK_CARRY));
        } else {
            s.inv[row] = 1.f / l;
        }
        s.nan_row[row] = nan_groups;
        asm volatile("bar.sync 2, 384;" ::: "memory");
    } else if (warp < 12) {
        const int tid = threadIdx.x - 128, w8 = warp - 4, p_tile = tid >> 2, t = tid & 3;
        const uint8_t *head_blocks = kv4_block(const_cast<uint8_t *>(a.cache), a.n_blocks, kvh, 0, HD);
        const Nibbles nib;
        float acc[16 * NG];   // columns [part * HD / 2, ...) of row
#pragma unroll
        for (int i = 0; i < 16 * NG; i++) acc[i] = 0.f;
        const int part = w8 >> 2;
        float acc_x[2] = {0.f, 0.f};                    // sum of p (m + 8 d) of the one or two groups they lie in
        constexpr int GROUPS = NG == 1 ? 1 : 2;
        const int g0 = part * (HD / 2) / 32;
        // O of tile j is finished: add it
        auto collect = [&](int j) {
            ok = ok && mbar_wait(&s.free_[j % APK_STAGES], (j / APK_STAGES) & 1);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                ok = false;
                return;
            }
            tc_fence_after();
            const float corr = s.corr[j & 3][row], f = s.scale_v[j & 3];
            const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
            if (!__all_sync(0xFFFFFFFFu, corr == 1.f)) {   // (a reference is raised a few times in all)
#pragma unroll
                for (int i = 0; i < 16 * NG; i++) acc[i] *= corr;
                acc_x[0] *= corr;
                acc_x[1] *= corr;
            }
            uint32_t x[8];
            tc_ld8(tmem + lanes + T_X, x);
#pragma unroll
            for (int g = 0; g < GROUPS; g++) {
                constexpr int G1 = HD / 64;   // (indexes known to the compiler: the values stay in registers)
                const float m0 = __uint_as_float(x[g]) + __uint_as_float(x[4 + g]), m1 = __uint_as_float(x[G1 + g]) + __uint_as_float(x[4 + G1 + g]);
                const float m = part ? m1 : m0;
                acc_x[g] = fmaf(m, f, acc_x[g]);
            }
#pragma unroll
            for (int c = 0; c < NG / 2; c++) {
                uint32_t o[32];
                tc_ld32(tmem + lanes + T_O + part * (HD / 2) + 32 * c, o);
#pragma unroll
                for (int i = 0; i < 32; i++) acc[32 * c + i] = fmaf(__uint_as_float(o[i]), f, acc[32 * c + i]);
            }
            if constexpr (NG % 2 == 1) {
                uint32_t o[16];
                tc_ld16(tmem + lanes + T_O + part * (HD / 2) + 16 * (NG - 1), o);
#pragma unroll
                for (int i = 0; i < 16; i++) acc[16 * (NG - 1) + i] = fmaf(__uint_as_float(o[i]), f, acc[16 * (NG - 1) + i]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.o_free);
        };
        // 8 dims of NG groups, and the position's parameters (m .., d ..): of this tile, and of the next, on its way
        uint32_t kw[NG], vw[NG], kp[NG], vp[NG], kw1[NG], vw1[NG], kp1[NG], vp1[NG];
        const uint8_t *at0 = head_blocks + (size_t)(b0 + p_tile / KV4_BLOCK) * (40 * HD) + 4 * NG * (p_tile % KV4_BLOCK);   // (a tile is two blocks on)
        auto fetch = [&](int j) {
            const unsigned pos = (unsigned)base0 + APK_BN * j + p_tile;   // (may pass 2^31 where a cache ends there)
            if (pos - k_lo <= (unsigned)(p_last - k_lo)) {
                const uint8_t *at = at0 + (size_t)j * (2 * 40 * HD);
                ldg_words<NG>(at + 16 * HD, kp1);
                ldg_words<NG>(at + 36 * HD, vp1);
                at += 4 * NG * (3 * (p_tile % KV4_BLOCK) + t);   // (a row of codes is four rows of parameters long)
                ldg_words<NG>(at, kw1);
                ldg_words<NG>(at + 20 * HD, vw1);
            } else {
#pragma unroll
                for (int i = 0; i < NG; i++) kp1[i] = vp1[i] = kw1[i] = vw1[i] = 0;   // m = d = 0
            }
        };
        // is it so for any of these warps' threads?
        auto any_thread = [](bool x) {
            uint32_t any;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 3, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
                         : "=r"(any) : "r"((uint32_t)x) : "memory");
            return any != 0;
        };
        // (rare) note V groups that are NaN and take them as zero; bring steps whose eightfold overflows into range
        auto mend = [&](int j, float &uk, float &uv) {
            bool big_k = false, big_v = false;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                if ((bits_of(vp, g) & 0x7FFFu) > 0x7C00u) {
                    if (t == 0) atomicOr(&s.nan_v[j & 3][g][p_tile >> 5], 1u << (p_tile & 31));
                    vp[g >> 1] &= g & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                }
                big_k |= bits_of(kp, NG + g) > 0x6FFFu;
                big_v |= bits_of(vp, NG + g) > 0x6FFFu;
            }
            if (any_thread(big_k)) uk = 0.125f;
            if (any_thread(big_v)) uv = 0.125f;
            auto times = [](uint32_t w, float u) {
                const float2 x = __half22float2(*(const __half2 *)&w);
                return pack_half2(x.x * u, x.y * u);
            };
#pragma unroll
            for (int i = 0; i < NG; i++) {
                kp[i] = times(kp[i], uk);
                vp[i] = times(vp[i], uv);
            }
        };
        fetch(0);
        for (int j = 0; j < n_tiles; j++) {
            if (j >= APK_STAGES) collect(j - APK_STAGES);   // (a wait that gave up does not leave the loop: the barrier below is for all)
#pragma unroll
            for (int i = 0; i < NG; i++) {
                kw[i] = kw1[i];
                vw[i] = vw1[i];
                kp[i] = kp1[i];
                vp[i] = vp1[i];
            }
            if (j + 1 < n_tiles) fetch(j + 1);
            if (tid < 8) s.nan_v[(j + 1) & 3][tid >> 1][tid & 1] = 0;   // (its last readers have finished: tile j - 3 is)
            // a step whose eightfold overflows f16, or a NaN among V's minima (a sum of them that is NaN)?  Subnormal steps do no
            // harm: their multiples are exact.
            bool odd;
            if constexpr (NG % 2 == 0) {
                uint32_t top = 0;
                __half2 sum = __half2half2(__ushort_as_half((unsigned short)0));
#pragma unroll
                for (int i = 0; i < NG / 2; i++) {
                    top = __vmaxu2(top, __vmaxu2(kp[NG / 2 + i], vp[NG / 2 + i]));
                    sum = __hadd2(sum, *(const __half2 *)&vp[i]);
                }
                const uint32_t w = *(const uint32_t *)&sum & 0x7FFF7FFFu;
                odd = (__vmaxu2(top, 0x6FFF6FFFu) != 0x6FFF6FFFu) | (__vmaxu2(w, 0x7C007C00u) != 0x7C007C00u);
            } else {
                odd = false;
#pragma unroll
                for (int g = 0; g < NG; g++)
                    odd |= bits_of(kp, NG + g) > 0x6FFFu || bits_of(vp, NG + g) > 0x6FFFu || (bits_of(vp, g) & 0x7FFFu) > 0x7C00u;
            }
            float uk = 1.f, uv = 1.f;
            if (any_thread(odd)) mend(j, uk, uv);
            if (tid == 0) {
                s.scale_k[j & 3] = 1.f / uk;
                s.scale_v[j & 3] = 1.f / uv;
            }
            unsigned char *stage = ring + (j % APK_STAGES) * STAGE;
            if (j == APK_STAGES - 1) ok = ok && mbar_wait(&s.q_done, 0);
#pragma unroll
            for (int g = 0; g < NG; g++) {
                // odd positions take a pair of groups the other way round: eight lanes then fill eight different 16-byte columns
                const int other = (g ^ 1) < NG ? g ^ 1 : g;
                const bool swap = (p_tile & 1) && other != g;
                const uint32_t at = (g >> 1) * HALF + sw128(p_tile, ((swap ? other : g) & 1) * 4 + t);
                uint4 hi, lo;
                kv4_split8(nib, swap ? kw[other] : kw[g], __half2half2(__ushort_as_half((unsigned short)(swap ? bits_of(kp, NG + other) : bits_of(kp, NG + g)))), hi, lo);
                *(uint4 *)(stage + AT_K + at) = hi;
                *(uint4 *)(stage + AT_K + SIDE + at) = lo;
                // dims 8 t .., and 8 t + 4 ..
                const uint32_t w = swap ? bits_of(vw, other) | bits_of(vw, NG + other) << 16 : bits_of(vw, g) | bits_of(vw, NG + g) << 16;
                kv4_split8(nib, w, __half2half2(__ushort_as_half((unsigned short)(swap ? bits_of(vp, NG + other) : bits_of(vp, NG + g)))), hi, lo);
                *(uint4 *)(stage + AT_V + at) = hi;
                *(uint4 *)(stage + AT_V_LO + at) = lo;
            }
            if (t < 2) {   // m and 8 d of the position: K's as k 32 .. of the extra tile, V's as its first columns
                uint32_t x[4] = {0, 0, 0, 0};
                const __half2 eight = __half2half2(__ushort_as_half((unsigned short)0x4800));
#pragma unroll
                for (int i = 0; i < (NG + 1) / 2; i++) {
                    uint32_t m, d;
                    if constexpr (NG % 2 == 0) {
                        m = t ? vp[i] : kp[i];
                        d = t ? vp[NG / 2 + i] : kp[NG / 2 + i];
                    } else {
                        const bool two = 2 * i + 1 < NG;
                        constexpr int L = NG - 1;
                        m = t ? bits_of(vp, 2 * i) | (two ? bits_of(vp, min(2 * i + 1, L)) << 16 : 0) : bits_of(kp, 2 * i) | (two ? bits_of(kp, min(2 * i + 1, L)) << 16 : 0);
                        d = t ? bits_of(vp, NG + 2 * i) | (two ? bits_of(vp, NG + min(2 * i + 1, L)) << 16 : 0)
                              : bits_of(kp, NG + 2 * i) | (two ? bits_of(kp, NG + min(2 * i + 1, L)) << 16 : 0);
                    }
                    const __half2 d8 = __hmul2(*(const __half2 *)&d, eight);
                    x[i] = m;
                    x[2 + i] = *(const uint32_t *)&d8;
                }
                *(uint4 *)(stage + AT_X + sw128(p_tile, t ? 0 : 4)) = make_uint4(x[0], x[1], x[2], x[3]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.full[j % APK_STAGES]);
        }
        for (int j = max(0, n_tiles - APK_STAGES); j < n_tiles; j++) collect(j);
        asm volatile("bar.sync 2, 384;" ::: "memory");
        if (is_row && ok) {
            const float inv = s.inv[row];
            const uint32_t bad = s.nan_row[row];
            float *dst = a.out + ((size_t)(t0 + tok) * a.n_heads + head) * HD + part * (HD / 2);
#pragma unroll
            for (int c = 0; c < 2 * NG; c++) {   // eight columns: dims (0,4,1,5,2,6,3,7)
                const int g = (part * (HD / 2) + 8 * c) >> 5;
                const float f = bad >> g & 1 ? __int_as_float(0x7FC00000) : inv, x = g == g0 ? acc_x[0] : acc_x[1];
                const float *o = acc + 8 * c;
                *(float4 *)(dst + 8 * c) = make_float4((o[0] + x) * f, (o[2] + x) * f, (o[4] + x) * f, (o[6] + x) * f);
                *(float4 *)(dst + 8 * c + 4) = make_float4((o[1] + x) * f, (o[3] + x) * f, (o[5] + x) * f, (o[7] + x) * f);
            }
        }
    } else if (warp == 12) {   // (warps 13 to 15 only lend their registers)
        asm volatile("bar.sync 1, 160;" ::: "memory");
        tc_fence_after();
        const bool leader = elect_one();
        constexpr uint32_t i_s = umma_idesc_f16(APK_BN, false), i_o = umma_idesc_f16(64 * NH + 16, true), i_lo = umma_idesc_f16(64 * NH, true);
        const uint32_t ring_addr = smem_u32(ring), t_base = __shfl_sync(0xFFFFFFFFu, tmem, 0);
        int scored = -1, done = -1;   // last tiles whose S and whose P V were issued
        for (int j = 0; j <= n_tiles; j++) {
            if (j < n_tiles) {
                // S(j) may overwrite P(j - 2): the MMAs that read it were issued before and execute in order
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s.full[j % APK_STAGES], (j / APK_STAGES) & 1));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = t_base + T_S + 64 * (j & 1);
                const uint64_t stage = umma_desc_sw128(ring_addr + (j % APK_STAGES) * STAGE);   // (its low word counts 16 bytes)
#pragma unroll
                for (int m = 0; m < 3; m++) {   // lo hi, hi lo, hi hi
#pragma unroll
                    for (int k = 0; k < HD / 16; k++)
                        tc_mma_f16_ta(leader, d, t_base + T_Q + (m == 0 ? 64 : 0) + 8 * k,
                                      stage + ((AT_K + (m == 1 ? SIDE : 0) + (k >> 2) * HALF + 32 * (k & 3)) >> 4), i_s, (m | k) ? 1u : 0u);
                    if (m != 1) tc_mma_f16_ta(leader, d, t_base + T_Q + (m == 0 ? 136 : 128), stage + ((AT_X + 64) >> 4), i_s, 1u);
                }
                if (leader) tc_commit(&s.s_full[j & 1]);
                scored = j;
            }
            if (j > 0) {
                const int i = j - 1;
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s.p_full[i & 1], (i >> 1) & 1) && (i < 1 || mbar_wait(&s.o_free, (i - 1) & 1)));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = t_base + T_O, p = t_base + T_S + 64 * (i & 1);
                const uint64_t stage = umma_desc_sw128_mn(ring_addr + (i % APK_STAGES) * STAGE, HALF);
#pragma unroll
                for (int m = 0; m < 3; m++)
#pragma unroll
                    for (int k = 0; k < APK_BN / 16; k++)
                        tc_mma_f16_ta(leader, d, p + 32 * (k >> 1) + 8 * (k & 1) + (m == 0 ? 16 : 0), stage + (((m == 1 ? AT_V_LO : AT_V) + 2048 * k) >> 4),
                                      m == 1 ? i_lo : i_o, (m | k) ? 1u : 0u);
                if (leader) tc_commit(&s.free_[i % APK_STAGES]);
                done = i;
            }
        }
        // nothing in flight at the exit, also where a wait gave up between the two
        if (scored >= 0) mbar_wait(&s.s_full[scored & 1], (scored >> 1) & 1);
        if (done >= 0) mbar_wait(&s.free_[done % APK_STAGES], (done / APK_STAGES) & 1);
        __syncwarp();
    }
    if (!ok && a.status) *a.status = QZ_ERR_TIMEOUT;
    tc_fence_before();
    __syncthreads();
    if (warp == 12) tmem_dealloc(tmem, 512);
}

}  // namespace qz
