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
//
// With c = 32 log2(e) / T as a sum of two f32 numbers, z c is a whole number k and a rest f, |f| < 0.8: one FMA rounds z c to
// k, two more give f with an error of 2^-26.  The weight is then 2^((k - k_M) / 32), from a table of 32 and a shift, times
// 2^((f - f_M) / 32): the table carries f_M, four terms of the exponential's series give the rest (|y| < 0.017: 1e-11), and
// only table times series is taken in 32 bits, two roundings of half a unit in 2^26 to 2^27: a weight is right to 2^-26, to 2^-28 as a
// rule.  (CUDA's exp in 64 bits took twice the time
// of the rest.)  Where z c passes 2^22, at temperatures near 0 or logits of any size, M - z takes the place of z, exact as two
// f32 numbers, times a power of two that brings c to [1, 2) (c itself leaves f32 at temperatures below 2^-122).  Why so exact: with thousands of tokens kept, an error of 1e-7 in their sums would move the border of top_p, or
// the token that u falls on, once in some thousand rows.  b = k_M - k is also the bin in which tokens are counted: it follows
// the order of the logits.
#pragma once

#include <cooperative_groups.h>

#include "async_copy.cuh"

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
    double inv_t, c, one_over_c;   // 1 / temperature; 32 log2(e) / temperature
    int top_k;
    float top_p;
    double min_p;        // (at most 1)
    float log_min_p;
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

// ---- the kernel -------------------------------------------------------------------------------------------------
// A cluster of CL CTAs per row; each keeps a contiguous part of the row in shared memory, read once from HBM.  Nothing is
// sorted: a threshold is the number of the last token kept, and is found by counting.
//   1. the largest number of the row (M; at temperature 0 the answer)
//   2. top_k: a histogram of the tokens over the bins b; the bin of the k-th token is known then, its tokens are gathered
//      and ranked against one another.  When all tokens down to that bin fit the list (k up to some hundreds), everything
//      else is done on the list.
//   3. top_p: the same with a histogram of the weights, bin by bin in units of the bin's own size.
//   4. the kept weights are summed warp by warp in the order of the vocabulary; the part of the warp in whose
//      range u falls is weighed again, token by token.  (Few are kept as a rule: a warp collects them and weighs 32 at a time.)
// A bin with more tokens than the list takes (ties, high temperatures) is divided further, by the number itself.
// A histogram is reduced in slices, one per CTA, that are pushed to every CTA: all find the same bin without asking.
//
// Measured (128256 tokens, replayed): one row, top_k 40 12.3 us, top_p alone 21.4, no filter 8.2; 256 rows, top_k 142 us,
// top_p 266, no filter 117, temperature 0 47 us = 2.8 TB/s.  One row is bound by cluster barriers (five or six, 1 to 2 us each),
// many rows by instruction issue (150 a warp and 32 tokens with top_p) and the histogram's shared-memory atomics (two per token)
// between the same barriers: two CTAs of an SM, of different rows, are all there is to overlap them (a part of a row and the
// histograms take 107 KB).  Sizes cut to whole units cost 2 per cent of top_p, the barrier that every CTA runs 1.
constexpr int SMP_PER = 3, SMP_BINS = SMP_PER * SMP_THREADS, SMP_LIST = 512;   // (a thread looks after three bins, and one token of the list)
constexpr int SMP_WARPS = SMP_THREADS / 32, SMP_MAX_CLUSTER = 16;
static_assert(SMP_BINS >= 32 * 46 && SMP_BINS % SMP_MAX_CLUSTER == 0, "bins cover weights down to 2^-45");

struct SampleShared {
    uint32_t part[2][SMP_BINS];                   // this CTA's histogram: tokens in [0], or the two halves of their sizes
    u64 all[SMP_BINS];                            // the row's: tokens, or weights
    union {
        u64 slice[SMP_BINS];                      // while a histogram is collected: this CTA's slice of everybody's
        struct { u64 mine[SMP_LIST], list[SMP_LIST], list_w[SMP_LIST]; };   // gathered tokens: this CTA's; the row's, their weights
    };
    u64 from[2][SMP_MAX_CLUSTER][2];              // what the cluster's CTAs pushed last, and before
    u64 red[SMP_WARPS];
    uint2 table[32];                              // 2^27 * 2^(-(k + f_M) / 32): rounded to a whole number, and that as f32
    u64 before;
    int n_mine, n_list, at, bin;
    uint16_t later[SMP_WARPS][160];               // tokens that a warp has put off
};

// largest over the warp, and over the block; every thread gets it
__device__ __forceinline__ u64 smp_warp_largest(u64 v)
{
    const uint32_t hi = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(v >> 32));
    return (u64)hi << 32 | __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0);
}
__device__ __forceinline__ u64 smp_largest(u64 v, u64 *sm)
{
    v = smp_warp_largest(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    return smp_warp_largest((threadIdx.x & 31) < SMP_WARPS ? sm[threadIdx.x & 31] : 0);
}
__device__ __forceinline__ u64 smp_warp_inclusive(u64 v)
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}
// sum over the threads before this one; *total over all
__device__ __forceinline__ u64 smp_before(u64 v, u64 *sm, u64 *total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const u64 inc = smp_warp_inclusive(v);
    __syncthreads();
    if (lane == 31) sm[warp] = inc;
    __syncthreads();
    const u64 w = lane < SMP_WARPS ? sm[lane] : 0, winc = smp_warp_inclusive(w);
    *total = __shfl_sync(0xFFFFFFFFu, winc, 31);
    return __shfl_sync(0xFFFFFFFFu, winc - w, warp) + inc - v;
}

struct Sampler {
    SampleShared &s;
    const float *z;       // this CTA's part of the row
    int n, base;          // tokens in it, index of the first
    int CL, rank, turn;
    float M, c_hi, c_lo;  // c = up (c_hi + c_lo)
    float up;             // plain: 1
    bool plain;           // z c stays below 2^22
    float low;            // plain: all logits up to here share the last bin
    int top;              // plain: the bits of 1.5 * 2^23 + k_M
    float keep_z;         // the set: logits above keep_z, and those equal to it with an index up to keep_i
    int keep_i;

    __device__ __forceinline__ SampleShared *peer(int r) const { return cooperative_groups::this_cluster().map_shared_rank(&s, r); }
    __device__ __forceinline__ void sync() const { cooperative_groups::this_cluster().sync(); }
    __device__ __forceinline__ bool in_set(float x, int i) const { return x > keep_z || (x == keep_z && base + i <= keep_i); }
    // f(logit, i) for this CTA's tokens i, in any order (-inf behind the last)
    template <class F>
    __device__ __forceinline__ void each(F f) const
    {
#pragma unroll 2
        for (int i = threadIdx.x; 4 * i < n; i += SMP_THREADS) {
            const float4 v = ((const float4 *)z)[i];
            f(v.x, 4 * i);
            f(v.y, 4 * i + 1);
            f(v.z, 4 * i + 2);
            f(v.w, 4 * i + 3);
        }
    }
    __device__ __forceinline__ void keep_to(u64 last)
    {
        keep_z = smp_unkey((uint32_t)(last >> 32));
        keep_i = (int)~(uint32_t)last;
    }
    __device__ __forceinline__ u64 number(int i) const { return (u64)smp_key(z[i]) << 32 | (uint32_t)~(base + i); }
    // (ends with the threads synchronised)
    __device__ __forceinline__ void scale(double c, double one_over_c)
    {
        constexpr double LAST = SMP_BINS - 1;
        const double Mc = (double)M * c;
        c_hi = (float)c;
        c_lo = (float)(c - (double)c_hi);
        plain = fabs(Mc) < 4190000.0 && c_hi < 1e30f && c_hi > 1e-30f;
        up = 1.f;
        if (!plain) {
            const int e = max(-126, min(127, ilogb(c)));
            const double rest = ldexp(c, -e);
            up = (float)ldexp(1.0, e);
            c_hi = (float)rest;
            c_lo = (float)(rest - (double)c_hi);
        }
        low = -INFINITY;
        top = __float_as_int(fmaf(M, c_hi, 12582912.f));   // 1.5 * 2^23: the sum's low bits are the nearest integer
        if (plain) {
            const float last = (float)((Mc - LAST) * one_over_c);   // (its product is off by 1/4 at most: bin LAST - 1, LAST or LAST + 1)
            low = bin(last) == SMP_BINS - 1 ? last : (float)((Mc - LAST + 0.75) * one_over_c);
        }
        if (threadIdx.x < 32) {
            const double f = plain ? Mc - (double)(top - 0x4B400000) : 0.0;
            const uint32_t e = (uint32_t)rint(exp2(27.0 - ((double)threadIdx.x + f) / 32.0));
            s.table[threadIdx.x] = make_uint2(e, __float_as_uint((float)e));
        }
        __syncthreads();
    }
    // b, at most SMP_BINS - 1
    __device__ __forceinline__ int bin(float x) const
    {
        if (plain) return top - __float_as_int(fmaf(fmaxf(x, low), c_hi, 12582912.f));   // (NaN goes with the lowest)
        const float t = x == M ? 0.f : __fmul_rn((M - x) * up, c_hi);   // (M = inf: t may not be a number)
        return t < (float)(SMP_BINS - 1) ? __float2int_rn(t) : SMP_BINS - 1;
    }
    // the weight of logit x is size << 17 >> b / 32, b its bin
    __device__ __forceinline__ uint32_t size(float x, int &b) const
    {
        float f;
        bool far = false;
        if (plain) {
            const float y = fmaxf(x, low), whole = fmaf(y, c_hi, 12582912.f);
            b = top - __float_as_int(whole);
            f = fmaf(y, c_lo, fmaf(y, c_hi, 12582912.f - whole));
        } else {
            const float diff = M - x, back = diff - M, d = diff * up, rest = ((M - (diff - back)) - (x + back)) * up;   // d + rest = up (M - x)
            const float t = __fmul_rn(d, c_hi), t_lo = fmaf(d, c_hi, -t) + fmaf(d, c_lo, rest * c_hi);
            const bool first = x == M;
            far = !first && !(t < (float)(SMP_BINS - 1));
            b = first ? 0 : far ? SMP_BINS - 1 : __float2int_rn(t);
            f = first || far ? 0.f : ((float)b - t) - t_lo;
        }
        constexpr float L = 0.0216608494f;   // ln 2 / 32
        const float r = f * fmaf(f, fmaf(f, fmaf(f, L * L * L * L / 24, L * L * L / 6), L * L / 2), L);
        const uint2 e = s.table[b & 31];
        const uint32_t v = e.x + (__float_as_uint(fmaf(__uint_as_float(e.y), r, 12582912.f)) - 0x4B400000);
        return far ? 0 : v;
    }
    // a size of bin b without what its weight is rounded down by: the sum over a bin is then the sum of its weights
    __device__ __forceinline__ static uint32_t whole(uint32_t size, int b) { return size & 0xFFFFFFFFu << max((b >> 5) - 17, 0); }
    __device__ __forceinline__ u64 weight(float x) const
    {
        int b;
        const uint32_t v = size(x, b);
        return (u64)v << 17 >> (b >> 5);
    }
    __device__ __forceinline__ u64 weight_of(u64 number) const { return weight(smp_unkey((uint32_t)(number >> 32))); }
    // Tokens lo .. below hi for which now(logit, i) holds are passed to put_off(i), 32 at a time.
    template <class Now, class PutOff>
    __device__ __forceinline__ void sweep(int lo, int hi, Now now, PutOff put_off) const
    {
        const int lane = threadIdx.x & 31;
        uint16_t *later = s.later[threadIdx.x >> 5];
        int held = 0;
        for (int i0 = lo; i0 < hi; i0 += 128) {
            const int i = i0 + 4 * lane;
            const float4 v = i < hi ? *(const float4 *)(z + i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const bool more = now(x[k], i + k);
                const unsigned mask = __ballot_sync(0xFFFFFFFFu, more);
                if (more) later[held + __popc(mask & ((1u << lane) - 1))] = (uint16_t)(i + k);
                held += __popc(mask);
            }
            __syncwarp();
            while (held >= 32) {
                held -= 32;
                put_off((int)later[held + lane]);
            }
            __syncwarp();
        }
        if (lane < held) put_off((int)later[lane]);
        __syncwarp();
    }

    // two values of this CTA to every CTA: afterwards s.from[turn][r] holds those of CTA r (two turns' worth are kept:
    // a CTA may still read the last ones while another pushes the next)
    __device__ __forceinline__ void exchange(u64 a, u64 b)
    {
        turn ^= 1;
        if ((int)threadIdx.x < CL) {
            u64 *to = peer(threadIdx.x)->from[turn][rank];
            to[0] = a;
            to[1] = b;
        }
        sync();
    }
    // the largest of what the CTAs pushed last
    __device__ __forceinline__ u64 largest(int which = 0) const
    {
        return smp_warp_largest((int)(threadIdx.x & 31) < CL ? s.from[turn][threadIdx.x & 31][which] : 0);
    }
    __device__ __forceinline__ void clear()
    {
        for (int b = threadIdx.x; b < SMP_BINS; b += SMP_THREADS) s.part[0][b] = s.part[1][b] = 0;
        if (threadIdx.x == 0) s.bin = -1;
        __syncthreads();
    }
    __device__ __forceinline__ void no_list()
    {
        if (threadIdx.x == 0) s.n_mine = s.n_list = 0;   // (the cluster meets before the next tokens arrive)
    }
    __device__ __forceinline__ void add(int b, bool weights, uint32_t size)   // (sizes are below 2^28: 2^17 halves fit a sum)
    {
        atomicAdd(&s.part[0][b], weights ? size & 0x3FFF : 1u);
        if (weights) atomicAdd(&s.part[1][b], size >> 14);
    }
    // The row's histogram into every CTA: each gets a slice of all CTAs' bins, sums it and pushes it (lanes run over bins).  Weights:
    // the bins' sizes are in units of 2^(17 - shift), shift = b / 32 or (of a bin divided further) as given.
    __device__ __forceinline__ void collect(bool weights, int shift = -1)
    {
        const int log_third = 10 - __ffs(CL), per = 3 << log_third;   // (SMP_BINS = 3 * 512)
        __syncthreads();
        for (int t = threadIdx.x; t < SMP_BINS; t += SMP_THREADS) {
            const int to = (t >> log_third) / 3;
            peer(to)->slice[(rank - to) * per + t] = weights ? (u64)s.part[0][t] + ((u64)s.part[1][t] << 14) : s.part[0][t];
        }
        sync();
        for (int k = threadIdx.x; k < per; k += SMP_THREADS) {
            const int b = rank * per + k;
            u64 sum = 0;
#pragma unroll 4
            for (int r = 0; r < CL; r++) sum += s.slice[r * per + k];
            if (weights) sum = sum << 17 >> (shift < 0 ? b >> 5 : shift);
            for (int r = 0; r < CL; r++) peer(r)->all[b] = sum;
        }
        sync();
    }
    // The first bin at which `above` plus the sum up to and with it reaches the goal; *before: the sum above it.
    // (The last bin that holds anything where the goal is not reached: fewer tokens than top_k.)  part < 0: `goal` is the goal,
    // else that part of the sum over all bins, and becomes it.
    __device__ __forceinline__ int boundary(u64 above, double &goal, u64 *before, double part = -1.0)
    {
        u64 v[SMP_PER], total, mine = 0;
        for (int k = 0; k < SMP_PER; k++) mine += v[k] = s.all[SMP_PER * threadIdx.x + k];
        u64 sum = above + smp_before(mine, s.red, &total);
        if (part >= 0.0) goal = part * (double)total;
        for (int k = 0; k < SMP_PER; k++) {
            if (v[k] && (double)sum < goal && (goal <= (double)(sum + v[k]) || sum + v[k] == above + total)) {
                s.bin = SMP_PER * threadIdx.x + k;
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
    // The tokens for which pred holds, as numbers, in the first `lists` CTAs' lists (a list takes them all: the caller has counted)
    template <class Pred>
    __device__ __forceinline__ void gather(int lists, Pred pred)
    {
        each([&](float x, int i) {
            if (pred(x, i)) s.mine[atomicAdd(&s.n_mine, 1)] = number(i);
        });
        __syncthreads();
        if (threadIdx.x == 0) s.at = atomicAdd(&peer(0)->n_list, s.n_mine);
        __syncthreads();
        for (int i = threadIdx.x; i < s.n_mine; i += SMP_THREADS)
            for (int r = 0; r < lists; r++) peer(r)->list[s.at + i] = s.mine[i];
        sync();
    }
    // Number of the last token with `above` + (weights, or count, of the set's tokens before it) < goal, given that it is
    // among the set's tokens of bin b, at most `count` of them.
    __device__ __forceinline__ u64 last_in_bin(int b, u64 count, u64 above, double goal, bool weights)
    {
        u64 lo = 0, hi = ~(u64)0;
        bool ranged = false;
        if (count > SMP_LIST) {
            u64 small = 0, large = 0;   // largest of ~number and of number
            for (int i = threadIdx.x; i < n; i += SMP_THREADS) {
                const u64 x = number(i);
                if (in_set(z[i], i) && bin(z[i]) == b) {
                    small = max(small, ~x);
                    large = max(large, x);
                }
            }
            small = smp_largest(small, s.red);
            large = smp_largest(large, s.red);
            exchange(small, large);
            small = largest();
            large = largest(1);
            lo = ~small;
            hi = large;
            while (count > SMP_LIST && lo < hi) {
                const int shift = max(0, 54 - __clzll((long long)(hi - lo)));   // (hi - lo) >> shift < 1024
                clear();
                for (int i = threadIdx.x; i < n; i += SMP_THREADS) {
                    const u64 x = number(i);
                    int same;   // (all lie in bin b)
                    if (x >= lo && x <= hi) add((int)((hi - x) >> shift), weights, weights ? whole(size(z[i], same), b) : 0);
                }
                collect(weights, b >> 5);
                const int sub = boundary(above, goal, &above);
                count = held_by(s.all[sub], weights, b);
                hi -= (u64)sub << shift;
                lo = max(lo, hi - (((u64)1 << shift) - 1));
                __syncthreads();
            }
            if (lo == hi) return hi;
            ranged = true;
        }
        if (ranged)
            gather(CL, [&](float, int i) { return i < n && number(i) >= lo && number(i) <= hi; });
        else
            gather(CL, [&](float x, int i) { return in_set(x, i) && bin(x) == b; });
        // each CTA ranks every CL-th token of the list, CL threads to a token
        const int c = peer(0)->n_list, e = rank + CL * ((int)threadIdx.x / CL), first = (int)threadIdx.x % CL;
        if ((int)threadIdx.x < c) s.list_w[threadIdx.x] = weights ? weight_of(s.list[threadIdx.x]) : 1;
        __syncthreads();
        const u64 x = e < c ? s.list[e] : 0;
        u64 before = 0;
        if (e < c)
            for (int j = first; j < c; j += CL) before += s.list[j] > x ? s.list_w[j] : 0;
        for (int o = CL >> 1; o > 0; o >>= 1) before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
        exchange(smp_largest(e < c && (double)(above + before) < goal ? ~x : 0, s.red), 0);
        no_list();
        return ~largest();
    }
    // At most so many tokens make up v, tokens or weights of bin b (a token's weight is 2^(-b / 32) within 1.7 per cent, rounded down
    // to a unit; where that can be none, v tells nothing)
    __device__ __forceinline__ u64 held_by(u64 v, bool weights, int b) const
    {
        if (!weights) return v;
        const float least = floorf(__uint_as_float(s.table[b & 31].y) * (float)(1ull << 17) / (float)(1ull << (b >> 5)) * (1 / 1.02f));
        return least < 1.f ? SMP_MAX_VOCAB : (u64)((float)v / least * 1.0001f) + 1;
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
    cluster_arrive();   // another CTA's shared memory may be written once it runs: waited for before the first exchange
    pdl_wait();
    pdl_trigger();
    // ---- 1. the row into shared memory; its first token ----
    const float *src = a.logits + (size_t)row * a.ld + c.base;
    const float4 *z4 = (const float4 *)z;
    float top = -INFINITY;
    int at = 0;
    auto look = [&](const float4 &v, int i) {   // (in rising order of i: the first of equals stays)
        const float m = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
        if (m > top) {
            top = m;
            at = i;
        }
    };
    const bool vectors = ((uintptr_t)src & 15) == 0;
    if (vectors) {
#pragma unroll 4
        for (int i = tid; i < n / 4; i += SMP_THREADS) {
            const float4 v = __ldcs((const float4 *)src + i);
            *((float4 *)z + i) = v;
            look(v, i);
        }
        if (tid < (n & 3)) z[(n & ~3) + tid] = __ldcs(src + (n & ~3) + tid);
    } else {
#pragma unroll 4
        for (int i = tid; i < n; i += SMP_THREADS) z[i] = __ldcs(src + i);
    }
    if (tid < ((n + 3) & ~3) - n) z[n + tid] = -INFINITY;   // up to a vector
    c.no_list();
    c.clear();   // (synchronises)
    for (int i = vectors ? n / 4 + (tid - n / 4 & SMP_THREADS - 1) : tid; 4 * i < n; i += SMP_THREADS) look(z4[i], i);   // what was not looked at
    u64 best = 0;
    if (top > -INFINITY) {
        const float4 v = z4[at];
        best = c.number(4 * at + (v.x == top ? 0 : v.y == top ? 1 : v.z == top ? 2 : 3));
    }
    best = smp_largest(best, s.red);
    cluster_wait();   // (arrived at the top; the row was loaded meanwhile)
    c.exchange(best, 0);
    best = c.largest();
    const bool none = best == 0;
    if (none || a.temperature == 0.f) {
        if (c.rank == 0 && tid == 0) {
            a.tokens[row] = none ? -1 : (int)~(uint32_t)best;
            if (a.probs) a.probs[row] = none ? 0.f : 1.f;
        }
        return;
    }
    c.M = smp_unkey((uint32_t)(best >> 32));
    c.keep_z = -INFINITY;
    c.keep_i = -1;
    c.scale(a.c, a.one_over_c);
    const float inv = (float)(a.inv_t / c.up);
    const double u = (double)fminf(fmaxf(a.u[row], 0.f), 1.f);
    auto heavy = [&](float x) {   // weight >= min_p: decided in 64 bits where 32 could be wrong
        if (a.min_p <= 0.0 || x == c.M) return true;
        const float y = (x - c.M) * c.up * inv;
        if (y > a.log_min_p + 1e-3f) return true;
        if (y < a.log_min_p - 1e-3f) return false;
        return exp(((double)x - (double)c.M) * a.inv_t) >= a.min_p;
    };
    const bool by_k = a.top_k > 0 && a.top_k < a.vocab, by_p = a.top_p > 0.f && a.top_p < 1.f;
    if (a.top_p <= 0.f) {
        c.keep_to(best);
    } else if (by_k) {
        // ---- 2. top_k ----
        c.each([&](float x, int i) {
            if (c.in_set(x, i)) c.add(c.bin(x), false, 0);
        });
        c.collect(false);
        u64 before;
        double goal = a.top_k;
        const int b = c.boundary(0, goal, &before);
        const u64 in_bin = s.all[b];
        if (before + in_bin <= SMP_LIST) {
            c.gather(1, [&](float x, int i) { return c.in_set(x, i) && c.bin(x) <= b; });
            if (c.rank != 0) return;   // (nobody pushes to this CTA or reads from it any more)
            const int m = s.n_list;
            const u64 x = tid < m ? s.list[tid] : 0;
            int place = 0;
            if (tid < m)
                for (int j = 0; j < m; j++) place += s.list[j] > x;
            const u64 w = tid < m && place < a.top_k ? c.weight_of(x) : 0;
            if (tid < m) s.list_w[tid] = w;
            u64 total, earlier = 0;
            smp_before(w, s.red, &total);
            if (w && a.top_p < 1.f)
                for (int j = 0; j < m; j++) earlier += s.list[j] > x ? s.list_w[j] : 0;
            const bool in = w && (a.top_p >= 1.f || (double)earlier < (double)a.top_p * (double)total) && heavy(smp_unkey((uint32_t)(x >> 32)));
            __syncthreads();
            if (tid < m) s.list_w[tid] = in ? w : 0;
            smp_before(in ? w : 0, s.red, &total);
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
        c.keep_to(c.last_in_bin(b, in_bin, before, goal, false));
        if (by_p) c.clear();
    }
    if (by_p) {
        // ---- 3. top_p ----
        c.each([&](float x, int i) {
            int b;
            const uint32_t v = c.size(x, b);
            if (c.in_set(x, i)) c.add(b, true, c.whole(v, b));
        });
        c.collect(true);
        u64 before;
        double goal;
        const int b = c.boundary(0, goal, &before, (double)a.top_p);
        c.keep_to(c.last_in_bin(b, c.held_by(s.all[b], true, b), before, goal, true));
    }
    // ---- 4. the token ----
    const int seg = ((n + SMP_WARPS - 1) / SMP_WARPS + 127) & ~127, lo = min(n, warp * seg), hi = min(n, lo + seg);   // this warp's part
    u64 mine = 0, cta;
    if (!by_k && !by_p && a.top_p > 0.f && a.min_p <= 0.0) {   // all of them
#pragma unroll 4
        for (int i = lo + lane; i < hi; i += 32) mine += z[i] > -INFINITY ? c.weight(z[i]) : 0;
    } else {
        c.sweep(lo, hi, [&](float x, int i) { return c.in_set(x, i) && heavy(x); }, [&](int i) { mine += c.weight(z[i]); });
    }
    u64 warp_sum = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) warp_sum += __shfl_xor_sync(0xFFFFFFFFu, warp_sum, o);
    u64 run = smp_before(lane == 0 ? warp_sum : 0, s.red, &cta);
    run = __shfl_sync(0xFFFFFFFFu, run, 0);   // of the warps before this one
    c.exchange(cta, 0);
    u64 total = 0, before = 0;
    for (int r = 0; r < c.CL; r++) {
        if (r < c.rank) before += s.from[c.turn][r][0];
        total += s.from[c.turn][r][0];
    }
    const u64 goal = min((u64)floor(u * (double)total), total - 1);
    if (goal < before || goal >= before + cta) return;   // another CTA's
    run += before;
    if (lane == 0 && goal >= run && goal < run + warp_sum) {
        s.at = warp;
        s.before = run;
    }
    __syncthreads();
    // the part of the warp in whose range the goal lies, by all threads: up to four tokens each
    constexpr int MOST = SMP_MAX_VOCAB / SMP_MAX_CLUSTER / SMP_WARPS / SMP_THREADS;
    const int from = s.at * seg, each = (seg + SMP_THREADS - 1) / SMP_THREADS, end = min(n, from + seg);
    run = s.before;
    u64 w[MOST], sum = 0, all;
#pragma unroll
    for (int k = 0; k < MOST; k++) {
        const int i = from + each * tid + k;
        w[k] = k < each && i < end && c.in_set(z[i], i) && heavy(z[i]) ? c.weight(z[i]) : 0;
        sum += w[k];
    }
    run += smp_before(sum, s.red, &all);
#pragma unroll
    for (int k = 0; k < MOST; k++) {
        if (goal >= run && goal < run + w[k]) {
            a.tokens[row] = c.base + from + each * tid + k;
            if (a.probs) a.probs[row] = (float)((double)w[k] / (double)total);
        }
        run += w[k];
    }
}

}  // namespace qz
