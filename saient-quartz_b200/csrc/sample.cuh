// Choosing the next token from a row of logits, given a uniform random number (the reference samples on the host from
// logits that it copies back, src/main.rs).
//
// With M the largest logit and T the temperature, token i weighs w_i = exp((z_i - M) / T).  Tokens are ordered by logit,
// ties by the lower index.  Kept are the first top_k of that order; of those the shortest prefix whose weights reach
// top_p of their sum; of those the tokens with w_i >= min_p.  The answer is the first token, in the order of the
// vocabulary, at which the running sum of the kept weights exceeds u times their total.
//
// Weights are held as 64-bit integers in units of 2^-44, so that every sum is exact and does not depend on its order:
// 2^19 tokens of weight 1 still fit.  A logit of -inf or NaN has no weight and is never chosen.
#pragma once

#include "common.cuh"

namespace qz {

typedef unsigned long long u64;
constexpr int SMP_THREADS = 1024;
constexpr int SMP_MAX_VOCAB = 1 << 19;
constexpr double SMP_ONE = 17592186044416.0;   // 2^44

struct SampleArgs {
    const float *logits;
    size_t ld;
    int vocab;
    float temperature;
    int top_k;
    float top_p, min_p;
    const float *u;
    int *tokens;
    float *probs;
};

// order of f32 values as unsigned integers; -0 counts as +0, NaN comes last
__device__ __forceinline__ uint32_t smp_key(float z)
{
    if (!(z == z)) return 0;
    const uint32_t b = __float_as_uint(z + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t SMP_KEY_MIN = 0x00800000u;   // keys from here on are logits above -inf

// weight of logit z in units of 2^-44.  Weights above 2^-13 carry the sums and are taken in 64 bits; below, the f32
// error (1e-6 of a weight under 1e-4) is lost in the total.
__device__ __forceinline__ u64 smp_weight(float z, float M, float inv_t, double inv_t64)
{
    if (z == M) return (u64)SMP_ONE;
    const float x = (z - M) * inv_t;
    if (x < -31.5f) return 0;
    if (x < -9.f) return (u64)__float2uint_rn(expf(x) * (float)SMP_ONE);
    return (u64)__double2ull_rn(exp(((double)z - (double)M) * inv_t64) * SMP_ONE);
}

template <class T, class Op>
__device__ __forceinline__ T smp_block_reduce(T v, T *sm, Op op)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sm[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}
__device__ __forceinline__ u64 smp_block_sum(u64 v, u64 *sm)
{
    return smp_block_reduce(v, sm, [](u64 a, u64 b) { return a + b; });
}
// sum over the threads before this one; *total over all
__device__ __forceinline__ u64 smp_block_before(u64 v, u64 *sm, u64 *total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();
    if (lane == 31) sm[warp] = inc;
    __syncthreads();
    u64 w = sm[lane], winc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xFFFFFFFFu, winc, o);
        if (lane >= o) winc += y;
    }
    *total = __shfl_sync(0xFFFFFFFFu, winc, 31);
    return __shfl_sync(0xFFFFFFFFu, winc - w, warp) + inc - v;
}

// One CTA per row; thresholds found by bisecting the 32 bits of the key.
__global__ void __launch_bounds__(SMP_THREADS) sample_kernel(const SampleArgs a)
{
    __shared__ u64 sm[32];
    pdl_wait();
    pdl_trigger();
    const float *z = a.logits + (size_t)blockIdx.x * a.ld;
    const int n = a.vocab, tid = threadIdx.x;
    // strided passes for sums, a contiguous chunk per thread where the order of the indices matters
    auto sum = [&](auto f) {
        u64 s = 0;
        for (int i = tid; i < n; i += SMP_THREADS) s += f(z[i]);
        return smp_block_sum(s, sm);
    };
    u64 best = 0;
    for (int i = tid; i < n; i += SMP_THREADS) {
        const uint32_t k = smp_key(z[i]);
        if (k >= SMP_KEY_MIN) best = max(best, (u64)k << 32 | (uint32_t)~i);
    }
    best = smp_block_reduce(best, sm, [](u64 x, u64 y) { return x > y ? x : y; });
    if (best == 0 || a.temperature == 0.f) {
        if (tid == 0) {
            a.tokens[blockIdx.x] = best ? (int)~(uint32_t)best : -1;
            if (a.probs) a.probs[blockIdx.x] = best ? 1.f : 0.f;
        }
        return;
    }
    const float M = z[~(uint32_t)best];
    const uint32_t key_max = (uint32_t)(best >> 32);
    const double inv64 = 1.0 / (double)a.temperature;
    const float inv = (float)inv64;
    // ---- top_k: the smallest key of the set, and how many tokens of that key belong to it ----
    uint32_t t_k = SMP_KEY_MIN;
    u64 r_k = (u64)n;
    if (a.top_k > 0 && a.top_k < n && sum([&](float x) { return (u64)(smp_key(x) >= SMP_KEY_MIN); }) > (u64)a.top_k) {
        t_k = 0;
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t c = t_k | 1u << bit;
            if (sum([&](float x) { return (u64)(smp_key(x) >= c); }) >= (u64)a.top_k) t_k = c;
        }
        r_k = (u64)a.top_k - sum([&](float x) { return (u64)(smp_key(x) > t_k); });
    }
    // ---- top_p ----
    uint32_t t_f = t_k;
    u64 r_f = r_k;
    if (a.top_p <= 0.f) {
        t_f = key_max;
        r_f = 1;
    } else if (a.top_p < 1.f) {
        const u64 ties = sum([&](float x) { return (u64)(smp_key(x) == t_k); });
        const u64 above_k = sum([&](float x) { return smp_key(x) > t_k ? smp_weight(x, M, inv, inv64) : 0; });
        const u64 tie_w = sum([&](float x) { return smp_key(x) == t_k ? smp_weight(x, M, inv, inv64) : 0; });
        const double goal = (double)a.top_p * (double)(above_k + (ties ? tie_w / ties * min(ties, r_k) : 0));
        // the largest key whose tokens above it do not reach the goal yet is one more than the largest that do
        uint32_t t = 0;
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t c = t | 1u << bit;
            if (c <= t_k || (double)sum([&](float x) { return smp_key(x) > c - 1 ? smp_weight(x, M, inv, inv64) : 0; }) >= goal) t = c;
        }
        // (weight of the tokens with key >= t reaches the goal, that of key >= t + 1 does not)
        if (t > t_k) {
            t_f = t;
            r_f = (u64)n;
        }
        const u64 eq = sum([&](float x) { return (u64)(smp_key(x) == t_f); });
        const double above = (double)sum([&](float x) { return smp_key(x) > t_f ? smp_weight(x, M, inv, inv64) : 0; });
        const u64 w = eq ? sum([&](float x) { return smp_key(x) == t_f ? smp_weight(x, M, inv, inv64) : 0; }) / eq : 0;
        if (w > 0 && above < goal) r_f = min(r_f, max((u64)1, (u64)ceil((goal - above) / (double)w)));
    }
    // ---- min_p is a lower bound of the weight ----
    const double lowest = fmin((double)a.min_p, 1.0);
    const int per = (n + SMP_THREADS - 1) / SMP_THREADS, lo = min(n, tid * per), hi = min(n, lo + per);
    u64 eq = 0, total;
    for (int i = lo; i < hi; i++) eq += smp_key(z[i]) == t_f;
    const u64 eq_before = smp_block_before(eq, sm, &total);
    auto kept = [&](float x, u64 &rank) -> u64 {
        const uint32_t k = smp_key(x);
        if (k < t_f || k < SMP_KEY_MIN || (k == t_f && rank++ >= r_f)) return 0;
        if (lowest > 0.0 && k != key_max && exp(((double)x - (double)M) * inv64) < lowest) return 0;
        return smp_weight(x, M, inv, inv64);
    };
    u64 s = 0, rank = eq_before;
    for (int i = lo; i < hi; i++) s += kept(z[i], rank);
    const u64 before = smp_block_before(s, sm, &total);
    const float u = fminf(fmaxf(a.u[blockIdx.x], 0.f), 1.f);
    const u64 goal = min((u64)floor((double)u * (double)total), total - 1);
    if (before <= goal && goal < before + s) {
        u64 run = before;
        rank = eq_before;
        for (int i = lo; i < hi; i++) {
            const u64 w = kept(z[i], rank);
            run += w;
            if (run > goal) {
                a.tokens[blockIdx.x] = i;
                if (a.probs) a.probs[blockIdx.x] = (float)((double)w / (double)total);
                break;
            }
        }
    }
}

}  // namespace qz
