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

#include <cooperative_groups.h>

#include "common.cuh"

namespace qz {

typedef unsigned long long u64;
constexpr int SMP_THREADS = 512;
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
    int chunk;   // tokens per CTA, a multiple of 4
};

// Order of f32 values as unsigned integers; -0 counts as +0, NaN comes last.  A token's place in its row is the number
// key << 32 | ~index: larger = earlier.
__device__ __forceinline__ uint32_t smp_key(float z)
{
    if (!(z == z)) return 0;
    const uint32_t b = __float_as_uint(z + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float smp_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// exp of a weight's argument in units of 2^-44.  In 64 bits: with thousands of tokens kept, an error of 1e-7 in their sums
// moves the border of top_p, or the token that u falls on, once in some thousand rows. 2^(n / 16) from a table, the rest (below ln 2 / 32) by its
// Taylor series up to the fifth power (1.4e-13).  (CUDA's exp: 730 us, not 610, for 256 rows of 128256.)
struct SampleExp {
    double M, scale;        // scale = 16 log2(e) / temperature
    const double *table;    // 2^(k / 16), k < 16
    __device__ __forceinline__ u64 operator()(float z) const
    {
        const double t = ((double)z - M) * scale, whole = t + 6755399441055744.0;   // 1.5 * 2^52: the sum's low word is t's nearest integer
        const int n = __double2loint(whole);
        constexpr double A = 0.04332169878499658;   // ln(2) / 16
        const double f = (t - (whole - 6755399441055744.0)) * A;
        const double p = fma(f, fma(f, fma(f, fma(f, fma(f, 1.0 / 120, 1.0 / 24), 1.0 / 6), 0.5), 1.0), 1.0) * table[n & 15];
        const double w = __hiloint2double(__double2hiint(p) + (((n >> 4) + 44) << 20), __double2loint(p));
        return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;   // + 2^52: rounded to a whole number
    }
};
// Weights below exp(-9) are taken in 32 bits: their errors (2e-6 of a weight, either way) average out of sums to which
// such tokens contribute by the thousand.
__device__ __forceinline__ u64 smp_light(float x) { return x < -31.5f ? 0 : __float2uint_rn(exp2f(x * 1.44269504f) * (float)SMP_ONE); }

// ---- the kernel -------------------------------------------------------------------------------------------------
// A cluster of CL CTAs per row; each keeps a contiguous part of the row in shared memory, read once from HBM.  Nothing is
// sorted: a threshold is the number of the last token kept, and is found by counting.
//   1. the largest number of the row (M; at temperature 0 the answer)
//   2. a histogram of the logits over 1024 bins of 1/32 of the temperature below M
//   3. top_k: the bin of the k-th token follows from the counts; its tokens are gathered and ranked against one another.
//      When all tokens down to that bin fit the list (k up to some hundreds), everything else is done on the list.
//   4. top_p: the counts bracket the bin in which the weights reach their goal (a bin's tokens weigh the same within 1/32);
//      one pass sums the weights above the bracket and below it, and those inside in 1024 finer bins; the tokens of the
//      right bin are gathered and ranked.
//   5. the kept weights are summed warp by warp in the order of the vocabulary (above the bracket step 4 did that, only
//      tokens inside it are looked at again); the warp in whose range u falls walks its part.
// Tokens that need more than a few instructions (64-bit weights, histogram entries) are first collected, so that a warp
// takes 32 of them at a time.
// A bin with more tokens than the list takes (ties, high temperatures) is divided further, by the number itself.
// A histogram is reduced in slices, one per CTA, that are pushed to every CTA: all find the same bin without asking.
constexpr int SMP_BINS = 2 * SMP_THREADS, SMP_LIST = 512,   // (a thread looks after two bins, and one token of the list)
              SMP_WARPS = SMP_THREADS / 32, SMP_MAX_CLUSTER = 16;

struct SampleShared {
    uint32_t cnt[SMP_BINS], part[3][SMP_BINS];    // this CTA's histogram: tokens, and their weights in parts of 15 bits
    uint32_t all_cnt[SMP_BINS];                   // the row's
    u64 all_w[SMP_BINS];
    union {
        u64 slice[SMP_BINS];                      // while a histogram is collected: this CTA's slice of everybody's
        struct { u64 mine[SMP_LIST], list[SMP_LIST]; };   // gathered tokens: this CTA's; (CTA 0) the row's
    };
    u64 list_w[SMP_LIST];
    u64 from[2][SMP_MAX_CLUSTER][3];              // what the cluster's CTAs pushed last, and before
    u64 red[SMP_WARPS];
    double exp2_16[16];
    u64 own[2], got[SMP_MAX_CLUSTER][2];          // sums beside a histogram: this CTA's, everybody's
    u64 result;
    u64 before;
    int n_mine, n_list, at, bin;
    uint16_t later[SMP_WARPS][64];                // tokens that a warp has put off
};

// sum, or largest, over the block; every thread gets it
template <bool MAX>
__device__ __forceinline__ u64 smp_reduce(u64 v, u64 *sm)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 y = __shfl_xor_sync(0xFFFFFFFFu, v, o);
        v = MAX ? (v > y ? v : y) : v + y;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < SMP_WARPS ? sm[threadIdx.x & 31] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 y = __shfl_xor_sync(0xFFFFFFFFu, v, o);
        v = MAX ? (v > y ? v : y) : v + y;
    }
    return v;
}
template <class T>
__device__ __forceinline__ T smp_warp_inclusive(T v)
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}
// sum over the threads before this one; *total over all
template <class T>
__device__ __forceinline__ T smp_before(T v, u64 *scratch, T *total)
{
    static_assert(sizeof(T) <= 8, "");
    T *sm = (T *)scratch;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T inc = smp_warp_inclusive(v);
    __syncthreads();
    if (lane == 31) sm[warp] = inc;
    __syncthreads();
    const T w = lane < SMP_WARPS ? sm[lane] : T(0), winc = smp_warp_inclusive(w);
    *total = __shfl_sync(0xFFFFFFFFu, winc, 31);
    return __shfl_sync(0xFFFFFFFFu, winc - w, warp) + inc - v;
}

struct Sampler {
    SampleShared &s;
    const float *z;       // this CTA's part of the row
    int n, base;          // tokens in it, index of the first
    int CL, rank, turn;
    float M, inv, per_bin;
    float fine0, fine;    // inside the bracket: bin (t - fine0) * fine of t = (M - z) * per_bin
    SampleExp e;
    float keep_z;         // the set: logits above keep_z, and those equal to it with an index up to keep_i
    int keep_i;

    __device__ __forceinline__ SampleShared *peer(int r) const { return cooperative_groups::this_cluster().map_shared_rank(&s, r); }
    __device__ __forceinline__ void sync() const { cooperative_groups::this_cluster().sync(); }
    __device__ __forceinline__ bool in_set(int i) const { return z[i] > keep_z || (z[i] == keep_z && base + i <= keep_i); }
    __device__ __forceinline__ void keep_to(u64 last)
    {
        keep_z = smp_unkey((uint32_t)(last >> 32));
        keep_i = (int)~(uint32_t)last;
    }
    __device__ __forceinline__ u64 number(int i) const { return (u64)smp_key(z[i]) << 32 | (uint32_t)~(base + i); }
    __device__ __forceinline__ int bin(float x) const
    {
        const float t = (M - x) * per_bin;
        return x == M ? 0 : t < (float)(SMP_BINS - 1) ? (int)t : SMP_BINS - 1;
    }
    __device__ __forceinline__ int fine_bin(float x) const   // of a token inside the bracket
    {
        const float t = x == M ? 0.f : fminf((M - x) * per_bin, (float)SMP_BINS);
        return max(0, min(SMP_BINS - 1, (int)((t - fine0) * fine)));
    }
    __device__ __forceinline__ float log_weight(float x) const { return x == M ? 0.f : (x - M) * inv; }
    __device__ __forceinline__ u64 weight(float x) const
    {
        const float y = log_weight(x);
        return x == M ? (u64)SMP_ONE : y < -9.f ? smp_light(y) : e(x);
    }
    // Calls now(i) for tokens lo + lane, lo + 32 + lane, .. below hi; what it returns true for is done by put_off(i), 32 at a time.
    template <class Now, class PutOff>
    __device__ __forceinline__ void sweep(int lo, int hi, Now now, PutOff put_off) const
    {
        const int lane = threadIdx.x & 31;
        uint16_t *later = s.later[threadIdx.x >> 5];
        int held = 0;
        for (int i0 = lo; i0 < hi; i0 += 32) {
            const int i = i0 + lane;
            const bool more = i < hi && now(i);
            const unsigned mask = __ballot_sync(0xFFFFFFFFu, more);
            if (more) later[held + __popc(mask & ((1u << lane) - 1))] = (uint16_t)i;
            held += __popc(mask);
            if (held >= 32) {
                __syncwarp();
                put_off((int)later[lane]);
                held -= 32;
                const uint16_t rest = later[32 + lane];
                __syncwarp();
                later[lane] = rest;
            }
        }
        __syncwarp();
        if (lane < held) put_off((int)later[lane]);
        __syncwarp();
    }
    __device__ __forceinline__ u64 weight_of(u64 number) const { return weight(smp_unkey((uint32_t)(number >> 32))); }

    // three values of this CTA to every CTA: afterwards s.from[turn][r] holds those of CTA r (two turns' worth are kept:
    // a CTA may still read the last ones while another pushes the next)
    __device__ __forceinline__ void exchange(u64 a, u64 b, u64 c)
    {
        turn ^= 1;
        if ((int)threadIdx.x < CL) {
            u64 *to = peer(threadIdx.x)->from[turn][rank];
            to[0] = a;
            to[1] = b;
            to[2] = c;
        }
        sync();
    }
    __device__ __forceinline__ void clear(bool weights)
    {
        for (int b = threadIdx.x; b < SMP_BINS; b += SMP_THREADS) {
            s.cnt[b] = 0;
            if (weights) s.part[0][b] = s.part[1][b] = s.part[2][b] = 0;
        }
        if (threadIdx.x == 0) s.bin = -1;
        __syncthreads();
    }
    __device__ __forceinline__ void no_list()
    {
        if (threadIdx.x == 0) s.n_mine = s.n_list = 0;   // (the cluster meets before the next tokens arrive)
    }
    __device__ __forceinline__ void add(int b, bool weights, u64 w)
    {
        atomicAdd(&s.cnt[b], 1u);
        if (weights) {
            atomicAdd(&s.part[0][b], (uint32_t)(w & 0x7FFF));
            atomicAdd(&s.part[1][b], (uint32_t)(w >> 15 & 0x7FFF));
            atomicAdd(&s.part[2][b], (uint32_t)(w >> 30));
        }
    }
    // the row's histogram into every CTA: this one sums a slice of all CTAs' bins and pushes it (lanes run over bins)
    __device__ __forceinline__ void collect(bool weights)
    {
        sync();
        const int per = SMP_BINS / CL;
        for (int what = weights ? 1 : 0; what >= 0; what--) {   // weights, then tokens
            for (int t = threadIdx.x; t < SMP_BINS; t += SMP_THREADS) {
                const SampleShared *from = peer(t / per);
                const int b = rank * per + t % per;
                if (what && t < 2 * CL) s.got[t >> 1][t & 1] = peer(t >> 1)->own[t & 1];
                s.slice[t] = what ? (u64)from->part[0][b] + ((u64)from->part[1][b] << 15) + ((u64)from->part[2][b] << 30) : from->cnt[b];
            }
            __syncthreads();
            for (int t = threadIdx.x; t < SMP_BINS; t += SMP_THREADS) {
                const int k = t % per, b = rank * per + k;
                u64 sum = 0;
                for (int r = 0; r < CL; r++) sum += s.slice[r * per + k];
                if (what) peer(t / per)->all_w[b] = sum;
                else peer(t / per)->all_cnt[b] = (uint32_t)sum;
            }
            if (what) __syncthreads();
        }
        sync();
    }
    // The first bin at which `above` plus the sum up to and with it reaches the goal; *before: the sum above it.
    // (The last bin that holds anything where the goal is not reached: fewer tokens than top_k.)
    __device__ __forceinline__ int boundary(bool weights, u64 above, double goal, u64 *before)
    {
        u64 v[2], total;
        for (int k = 0; k < 2; k++) v[k] = weights ? s.all_w[2 * threadIdx.x + k] : s.all_cnt[2 * threadIdx.x + k];
        u64 sum = above + smp_before(v[0] + v[1], s.red, &total);
        for (int k = 0; k < 2; k++) {
            if (v[k] && (double)sum < goal && (goal <= (double)(sum + v[k]) || sum + v[k] == above + total)) {
                s.bin = 2 * threadIdx.x + k;
                s.before = sum;
            }
            sum += v[k];
        }
        __syncthreads();
        const int b = s.bin;
        *before = s.before;
        __syncthreads();   // (read before the next clear)
        return b;
    }
    // The tokens for which pred holds, as numbers, in CTA 0's list (it takes them all: the caller has counted)
    template <class Pred>
    __device__ __forceinline__ void gather(Pred pred)
    {
        for (int i = threadIdx.x; i < n; i += SMP_THREADS)
            if (pred(i)) s.mine[atomicAdd(&s.n_mine, 1)] = number(i);
        __syncthreads();
        if (threadIdx.x == 0) s.at = atomicAdd(&peer(0)->n_list, s.n_mine);
        __syncthreads();
        for (int i = threadIdx.x; i < s.n_mine; i += SMP_THREADS) peer(0)->list[s.at + i] = s.mine[i];
        sync();
    }
    // Number of the last token with `above` + (weights, or count, of the set's tokens before it) < goal, given that it is
    // among the `count` tokens for which in_bin holds (a run of the order).
    template <class Bin>
    __device__ __forceinline__ u64 last_in_bin(Bin in_bin, uint32_t count, u64 above, double goal, bool weights)
    {
        bool ranged = false;
        u64 lo = 0, hi = ~(u64)0;
        if (count > SMP_LIST) {
            u64 small = 0, large = 0;   // largest of ~number and of number
            for (int i = threadIdx.x; i < n; i += SMP_THREADS) {
                const u64 x = number(i);
                if (in_set(i) && in_bin(z[i])) {
                    small = max(small, ~x);
                    large = max(large, x);
                }
            }
            small = smp_reduce<true>(small, s.red);
            large = smp_reduce<true>(large, s.red);
            exchange(small, large, 0);
            for (int r = 0; r < CL; r++) {
                small = max(small, s.from[turn][r][0]);
                large = max(large, s.from[turn][r][1]);
            }
            lo = ~small;
            hi = large;
            while (count > SMP_LIST && lo < hi) {
                const int shift = max(0, 54 - __clzll((long long)(hi - lo)));   // (hi - lo) >> shift < 1024
                clear(weights);
                for (int i = threadIdx.x; i < n; i += SMP_THREADS) {
                    const u64 x = number(i);
                    if (x >= lo && x <= hi) add((int)((hi - x) >> shift), weights, weights ? weight(z[i]) : 0);
                }
                collect(weights);
                const int sub = boundary(weights, above, goal, &above);
                count = s.all_cnt[sub];
                hi -= (u64)sub << shift;
                lo = max(lo, hi - (((u64)1 << shift) - 1));
            }
            if (lo == hi) return hi;
            ranged = true;
        }
        gather([&](int i) {
            if (!ranged) return in_set(i) && in_bin(z[i]);
            const u64 x = number(i);
            return x >= lo && x <= hi;
        });
        if (rank == 0) {
            const int c = s.n_list;
            const u64 x = (int)threadIdx.x < c ? s.list[threadIdx.x] : 0;
            if ((int)threadIdx.x < c) s.list_w[threadIdx.x] = weights ? weight_of(x) : 1;
            __syncthreads();
            u64 before = above;
            if ((int)threadIdx.x < c)
                for (int j = 0; j < c; j++) before += s.list[j] > x ? s.list_w[j] : 0;
            const u64 last = ~smp_reduce<true>((int)threadIdx.x < c && (double)before < goal ? ~x : 0, s.red);
            if ((int)threadIdx.x < CL) peer(threadIdx.x)->result = last;
        }
        sync();
        no_list();
        return s.result;
    }
};

__global__ void __launch_bounds__(SMP_THREADS) sample_kernel(const SampleArgs a)
{
    extern __shared__ __align__(16) unsigned char smem[];
    SampleShared &s = *(SampleShared *)smem;
    float *z = (float *)(smem + ((sizeof(SampleShared) + 15) & ~(size_t)15));
    const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Sampler c = {s, z};
    c.CL = (int)cluster.num_blocks();
    c.rank = (int)cluster.block_rank();
    c.turn = 0;
    c.base = c.rank * a.chunk;
    c.n = max(0, min(a.chunk, a.vocab - c.base));
    const int row = blockIdx.x / c.CL, n = c.n;
    pdl_wait();
    pdl_trigger();
    // ---- 1. the row into shared memory; its first token ----
    const float *src = a.logits + (size_t)row * a.ld + c.base;
    float top = -INFINITY;
    int at = -1;
    auto take = [&](float x, int i) {   // (in rising order of i: the first of equals stays)
        z[i] = x;
        if (x > top) {
            top = x;
            at = i;
        }
    };
    if (((uintptr_t)src & 15) == 0) {
#pragma unroll 4
        for (int i = tid; i < n / 4; i += SMP_THREADS) {
            const float4 v = __ldcs((const float4 *)src + i);
            take(v.x, 4 * i);
            take(v.y, 4 * i + 1);
            take(v.z, 4 * i + 2);
            take(v.w, 4 * i + 3);
        }
        if (tid < (n & 3)) take(src[(n & ~3) + tid], (n & ~3) + tid);
    } else {
#pragma unroll 4
        for (int i = tid; i < n; i += SMP_THREADS) take(__ldcs(src + i), i);
    }
    if (tid < 16) s.exp2_16[tid] = exp2((double)tid / 16.0);
    c.no_list();
    c.clear(false);   // (synchronises)
    u64 best = at >= 0 ? c.number(at) : 0;
    best = smp_reduce<true>(best, s.red);
    c.exchange(best, 0, 0);
    for (int r = 0; r < c.CL; r++) best = max(best, s.from[c.turn][r][0]);
    const bool none = best == 0;
    if (none || a.temperature == 0.f) {
        if (c.rank == 0 && tid == 0) {
            a.tokens[row] = none ? -1 : (int)~(uint32_t)best;
            if (a.probs) a.probs[row] = none ? 0.f : 1.f;
        }
        return;
    }
    c.M = smp_unkey((uint32_t)(best >> 32));
    const double inv64 = 1.0 / (double)a.temperature;
    c.inv = (float)inv64;
    c.per_bin = (float)(32.0 * inv64);
    c.e = {(double)c.M, 16.0 * 1.4426950408889634 * inv64, s.exp2_16};
    c.keep_z = -INFINITY;
    c.keep_i = -1;
    const double u = (double)fminf(fmaxf(a.u[row], 0.f), 1.f), lowest = fmin((double)a.min_p, 1.0);
    const float log_lowest = lowest > 0.0 ? (float)log(lowest) : -INFINITY;
    auto heavy = [&](float x) {   // weight >= min_p: decided in 64 bits where 32 could be wrong
        const float y = (x - c.M) * c.inv;
        if (x == c.M || y > log_lowest + 1e-3f) return true;
        if (y < log_lowest - 1e-3f) return false;
        return exp(((double)x - (double)c.M) * inv64) >= lowest;
    };
    const bool by_k = a.top_k > 0 && a.top_k < a.vocab, by_p = a.top_p > 0.f && a.top_p < 1.f;
    if (by_k || by_p) {
        // ---- 2. counts ----
        for (int i = tid; i < n; i += SMP_THREADS)
            if (c.in_set(i)) c.add(c.bin(z[i]), false, 0);
        c.collect(false);
    }
    if (a.top_p <= 0.f) {
        c.keep_to(best);
    } else if (by_k) {
        // ---- 3. top_k ----
        u64 before;
        const int b = c.boundary(false, 0, (double)a.top_k, &before);
        const uint32_t in_bin = s.all_cnt[b];
        if (before + in_bin <= SMP_LIST) {
            c.gather([&](int i) { return c.in_set(i) && c.bin(z[i]) <= b; });
            if (c.rank != 0) return;   // (nobody pushes to this CTA or reads from it any more)
            const int m = s.n_list;
            const u64 x = tid < m ? s.list[tid] : 0;
            int place = 0;
            if (tid < m)
                for (int j = 0; j < m; j++) place += s.list[j] > x;
            const u64 w = tid < m && place < a.top_k ? c.weight_of(x) : 0;
            if (tid < m) s.list_w[tid] = w;
            u64 total = smp_reduce<false>(w, s.red), earlier = 0;
            if (w && a.top_p < 1.f)
                for (int j = 0; j < m; j++) earlier += s.list[j] > x ? s.list_w[j] : 0;
            const bool in = w && (a.top_p >= 1.f || (double)earlier < (double)a.top_p * (double)total) && heavy(smp_unkey((uint32_t)(x >> 32)));
            __syncthreads();
            if (tid < m) s.list_w[tid] = in ? w : 0;
            total = smp_reduce<false>(in ? w : 0, s.red);
            const u64 goal = min((u64)floor(u * (double)total), total - 1);
            if (in) {
                u64 run = 0;   // weights of lower indices (larger low words)
                for (int j = 0; j < m; j++) run += (uint32_t)s.list[j] > (uint32_t)x ? s.list_w[j] : 0;
                if (run <= goal && goal < run + w) {
                    a.tokens[row] = (int)~(uint32_t)x;
                    if (a.probs) a.probs[row] = (float)((double)w / (double)total);
                }
            }
            return;
        }
        c.keep_to(c.last_in_bin([&](float x) { return c.bin(x) == b; }, in_bin, before, (double)a.top_k, false));
    }
    const int seg = ((n + SMP_WARPS - 1) / SMP_WARPS + 31) & ~31, lo = min(n, warp * seg), hi = min(n, lo + seg);   // this warp's part
    int first = 0, last = -1;
    u64 above_here = 0;   // weights above the bracket that this lane has summed
    if (by_p) {
        // ---- 4. top_p ----
        if (by_k) {   // the counts of the set (last_in_bin may have used the histogram)
            c.clear(false);
            for (int i = tid; i < n; i += SMP_THREADS)
                if (c.in_set(i)) c.add(c.bin(z[i]), false, 0);
            c.collect(false);
        }
        // a token of bin b weighs between exp(-(b + 1) / 32) and exp(-b / 32); 1e-3 covers the rounding of its bin and of these sums
        float most[2], least[2], most_all, least_all;
        for (int k = 0; k < 2; k++) {
            const int b = 2 * tid + k;
            const float count = (float)s.all_cnt[b];
            most[k] = count * expf(-(float)b / 32.f) * 1.001f;
            least[k] = b < SMP_BINS - 1 ? count * expf(-(float)(b + 1) / 32.f) * 0.999f : 0.f;
        }
        float most_before = smp_before(most[0] + most[1], s.red, &most_all), least_before = smp_before(least[0] + least[1], s.red, &least_all);
        // the first bin that may hold the border is the last with most_before < goal, the last one the first with least up to it >= goal
        int from_end = 0;
        first = 0;
        for (int k = 0; k < 2; k++) {
            if (most_before < a.top_p * least_all) first = 2 * tid + k;
            least_before += least[k];
            if (least_before >= a.top_p * most_all) from_end = max(from_end, SMP_BINS - 1 - (2 * tid + k));
            most_before += most[k];
        }
        first = (int)smp_reduce<true>((u64)first, s.red);
        last = SMP_BINS - 1 - (int)smp_reduce<true>((u64)from_end, s.red);
        c.fine0 = (float)first;
        c.fine = (float)SMP_BINS / (float)(last + 1 - first);
        c.clear(true);
        u64 above = 0, below = 0;
        c.sweep(lo, hi, [&](int i) {
            const float x = z[i], y = c.log_weight(x);
            const int b = c.bin(x);
            const bool light = y < -9.f, inside = b >= first && b <= last, in = c.in_set(i);
            if (in && light && !inside) {
                if (b < first) above += smp_light(y);
                else below += smp_light(y);
            }
            return in && (!light || inside);
        }, [&](int i) {
            const int b = c.bin(z[i]);
            const u64 w = c.weight(z[i]);
            if (b < first) above += w;
            else if (b > last) below += w;
            else c.add(c.fine_bin(z[i]), true, w);
        });
        above_here = above;
        above = smp_reduce<false>(above, s.red);
        below = smp_reduce<false>(below, s.red);
        if (tid == 0) {
            s.own[0] = above;
            s.own[1] = below;
        }
        c.collect(true);
        above = below = 0;
        for (int r = 0; r < c.CL; r++) {
            above += s.got[r][0];
            below += s.got[r][1];
        }
        u64 inside;
        smp_before(s.all_w[2 * tid] + s.all_w[2 * tid + 1], s.red, &inside);
        const double goal = (double)a.top_p * (double)(above + inside + below);
        u64 before;
        const int b = c.boundary(true, above, goal, &before);
        if (b >= 0)
            c.keep_to(c.last_in_bin([&](float x) { const int k = c.bin(x); return k >= first && k <= last && c.fine_bin(x) == b; }, s.all_cnt[b], before, goal, true));
    }
    // ---- 5. the token ----
    u64 mine = 0, cta;
    if (by_p && lowest <= 0.0) {
        mine = above_here;
        c.sweep(lo, hi, [&](int i) {
            const int b = c.bin(z[i]);
            return b >= first && b <= last && c.in_set(i);
        }, [&](int i) { mine += c.weight(z[i]); });
    } else {
        c.sweep(lo, hi, [&](int i) {
            const float y = c.log_weight(z[i]);
            const bool in = c.in_set(i) && heavy(z[i]);
            if (in && y < -9.f) mine += smp_light(y);
            return in && y >= -9.f;
        }, [&](int i) { mine += c.weight(z[i]); });
    }
    u64 warp_sum = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) warp_sum += __shfl_xor_sync(0xFFFFFFFFu, warp_sum, o);
    u64 run = smp_before(lane == 0 ? warp_sum : 0, s.red, &cta);
    run = __shfl_sync(0xFFFFFFFFu, run, 0);
    c.exchange(cta, 0, 0);
    u64 total = 0;
    for (int r = 0; r < c.CL; r++) {
        if (r < c.rank) run += s.from[c.turn][r][0];
        total += s.from[c.turn][r][0];
    }
    const u64 goal = min((u64)floor(u * (double)total), total - 1);
    if (goal < run || goal >= run + warp_sum) return;
    for (int i0 = lo; i0 < hi; i0 += 128) {   // four runs of 32 at once: their weights do not wait for one another
        u64 w[4], sum[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = i0 + 32 * k + lane;
            w[k] = i < hi && c.in_set(i) && heavy(z[i]) ? c.weight(z[i]) : 0;
            sum[k] = smp_warp_inclusive(w[k]);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const unsigned hit = __ballot_sync(0xFFFFFFFFu, run + sum[k] > goal);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    a.tokens[row] = c.base + i0 + 32 * k + lane;
                    if (a.probs) a.probs[row] = (float)((double)w[k] / (double)total);
                }
                return;
            }
            run += __shfl_sync(0xFFFFFFFFu, sum[k], 31);
        }
    }
}

}  // namespace qz
