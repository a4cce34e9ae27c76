// C entry points of the 4-bit KV cache and of the attention over it.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <memory>
#include <vector>

#include "attn_prompt_kv4.cuh"
#include "host.cuh"

using namespace qz;

namespace {

constexpr const char *GEOMETRY = "head_dim must be 32, 64, 96 or 128";

bool head_dim_ok(int head_dim) { return head_dim > 0 && head_dim % 32 == 0 && head_dim <= ATT_MAX_HD; }
bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// Arguments that every call on a cache shares; records what is wrong.
bool cache_ok(const char *who, const void *cache, int n_kv_heads, int head_dim, int max_seq)
{
    static char msg[160];
    const char *why = !head_dim_ok(head_dim) ? GEOMETRY
                      : n_kv_heads <= 0 || max_seq <= 0 ? "n_kv_heads and max_seq must be positive"
                      : !cache || !aligned16(cache) ? "the cache must be a 16-byte aligned device pointer" : nullptr;
    if (!why) return true;
    snprintf(msg, sizeof msg, "%s: %s", who, why);
    set_error(QZ_ERR_BAD_SHAPE, msg);
    return false;
}

bool refuse(const char *why)
{
    set_error(QZ_ERR_BAD_SHAPE, why);
    return false;
}

// Shape of the step kernel: clusters of CL <= 8 CTAs, `clusters` of them per unit.  8 is the widest size that leaves (almost)
// no SM without a cluster at two CTAs per SM; narrower when the units alone would not fit on the chip at once or the cache
// has fewer blocks.
struct StepShape {
    int cl, clusters;
};
template <int NG, int NT>
StepShape step_shape(int units, int n_blocks, int GV)
{
    static int fit[4 * NT + 1][4] = {};   // clusters of 1, 2, 4, 8 CTAs that the device holds at once (every B200 alike)
    static PerDevice ready;
    int (&f)[4] = fit[GV];
    const auto kernel = attn_step_kv4_kernel<NG, NT>;
    ready.once([&] {
        QZ_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, attn_kv4_smem(NG, NT, 4 * NT, 8).total));
    });
    if (!f[0]) {
        for (int i = 0; i < 4; i++) {
            cudaLaunchConfig_t cfg = {};
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = 1u << i;
            at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
            cfg.gridDim = dim3(1u << i);
            cfg.blockDim = dim3(AK_THREADS);
            cfg.dynamicSmemBytes = attn_kv4_smem(NG, NT, GV, 1 << i).total;
            cfg.attrs = at;
            cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&f[i], kernel, &cfg) != cudaSuccess || f[i] < 1) {
                cudaGetLastError();
                f[i] = i ? 0 : 1;
            }
        }
    }
    int i = 3;
    while (i > 0 && (f[i] < units || (1 << (i - 1)) >= n_blocks)) i--;
    // Of more than four query heads per kv head one CTA fits an SM, and clusters of 8 may leave half of them out (8 units: 64
    // CTAs against 128).  Narrower ones pay once a context is long, which the shape knows by the cache only: 64 / 8 heads
    // of 128 at 131072 positions 95 us against 172, at 8192 16.9 against 18.4; 28 / 4 (96 CTAs against 128) 54 against 64, at 16384
    // 16.4 against 16.3.  The price is paid where the context is short and the cache is not: at 2048 of 131072 positions 15.4 us
    // against 10.7, 28 / 4 14.4 against 10.2.
    if (i == 3) {
        const int wide = (f[3] / units) << 3, narrow = (f[2] / units) << 2;
        if (2 * narrow >= 3 * wide ? n_blocks >= 256 : 4 * narrow >= 5 * wide && n_blocks >= 1024) i = 2;
    }
    const int useful = std::max(1, n_blocks / (AK_WARPS << i));
    return {1 << i, std::max(1, std::min({f[i] / units, useful, AK_MAX_CLUSTERS / units}))};
}

// The workspace in which the clusters of a unit meet.  Calls on one stream follow one another and share one; every graph
// that is being captured gets one of its own (graphs may be replayed side by side), which returns to the pool when the
// last executable form of the graph is gone.  Streams are told apart by their ids: a handle may come back for a new stream while
// work of the old one is still running.  Nothing tells when a stream is gone, so only the first AK_OWN_STREAMS of a device have
// their own; all later ones share one more, which an event passes from call to call.
// ptr NULL: it cannot be had (then one cluster per unit works).
constexpr int AK_OWN_STREAMS = 16;   // (0.57 MB each; the event costs a call a microsecond or two on the host)
struct Workspace {
    int device;
    unsigned long long stream;    // its id (its handle in a capture); 0: shared
    unsigned long long capture;   // 0: calls that run at once
    float *ptr;
    cudaEvent_t passed;           // shared: recorded behind the last call
    std::atomic<bool> in_use;
};
struct MergeWorkspace {
    float *ptr;
    cudaEvent_t record;           // to be recorded behind the launch, or NULL
};
MergeWorkspace merge_workspace()
{
    static std::vector<std::unique_ptr<Workspace>> all;
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long capture = 0, id = 0;
    cudaGraph_t graph = nullptr;
    if (cudaStreamGetCaptureInfo_v2(stream(), &status, &capture, &graph, nullptr, nullptr) != cudaSuccess) cudaGetLastError();
    if (status == cudaStreamCaptureStatusInvalidated) return {};
    const bool capturing = status == cudaStreamCaptureStatusActive;
    if (!capturing) capture = 0;
    int device = 0;
    // (asked for its id, a stream loses its capture; while that lasts the handle will do)
    if (capturing) id = (uintptr_t)stream();
    if (cudaGetDevice(&device) != cudaSuccess || (!capturing && cudaStreamGetId(stream(), &id) != cudaSuccess)) {
        cudaGetLastError();
        return {};
    }
    Workspace *w = nullptr, *shared = nullptr;
    int owners = 0;
    for (auto &e : all) {
        if (e->device != device) continue;
        if (!e->in_use) w = e.get();
        else if (e->passed) shared = e.get();
        else if (e->stream == id && e->capture == capture) return {e->ptr, nullptr};
        else if (!e->capture) owners++;
    }
    const bool share = !capturing && owners >= AK_OWN_STREAMS;
    if (share && shared) {
        if (cudaStreamWaitEvent(stream(), shared->passed, 0) != cudaSuccess) {
            cudaGetLastError();
            return {};
        }
        return {shared->ptr, shared->passed};
    }
    if (!w) {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;   // allocating does not disturb a capture
        cudaThreadExchangeStreamCaptureMode(&mode);
        float *p = nullptr;
        cudaStream_t side = nullptr;
        bool ok = cudaMalloc(&p, AK_WORKSPACE) == cudaSuccess && cudaStreamCreateWithFlags(&side, cudaStreamNonBlocking) == cudaSuccess &&
                  cudaMemsetAsync(p, 0, AK_COUNTERS * sizeof(int), side) == cudaSuccess && cudaStreamSynchronize(side) == cudaSuccess;
        if (side) cudaStreamDestroy(side);
        if (!ok) {
            cudaGetLastError();
            if (p) cudaFree(p);
        }
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (!ok) return {};
        all.push_back(std::make_unique<Workspace>());
        w = all.back().get();
        w->device = device;
        w->ptr = p;
    }
    if (capturing) {
        cudaUserObject_t owner = nullptr;
        const auto release = [](void *e) { ((Workspace *)e)->in_use = false; };
        if (cudaUserObjectCreate(&owner, w, release, 1, cudaUserObjectNoDestructorSync) != cudaSuccess ||
            cudaGraphRetainUserObject(graph, owner, 1, cudaGraphUserObjectMove) != cudaSuccess) {
            cudaGetLastError();
            return {};
        }
    }
    if (share && cudaEventCreateWithFlags(&w->passed, cudaEventDisableTiming) != cudaSuccess) {
        cudaGetLastError();
        w->passed = nullptr;
        return {};
    }
    w->stream = share ? 0 : id;
    w->capture = capture;
    w->in_use = true;
    return {w->ptr, w->passed};
}

// NG = head_dim / 32 as a template argument
template <class F>
void by_groups(int head_dim, F f)
{
    switch (head_dim / 32) {
    case 1: f(std::integral_constant<int, 1>()); break;
    case 2: f(std::integral_constant<int, 2>()); break;
    case 3: f(std::integral_constant<int, 3>()); break;
    default: f(std::integral_constant<int, 4>()); break;
    }
}

// The step kernel for n_tok tokens at consecutive positions.
void launch_step(AttnKv4Args &a, int n_tok, int head_dim)
{
    const int G = a.n_heads / a.n_kv;
    a.splits = (G + 7) / 8;
    a.prefetch = pdl_enabled() && a.step;
    a.status = status_word_if_ready();
    const int GV = (G + a.splits - 1) / a.splits, units = a.n_kv * a.splits;
    by_groups(head_dim, [&](auto ng) {
        auto go = [&](auto nt) {
            StepShape s = step_shape<ng.value, nt.value>(units * n_tok, a.n_blocks, GV);
            MergeWorkspace w = {};
            if (s.clusters > 1 && !(w = merge_workspace()).ptr) s.clusters = 1;
            a.workspace = w.ptr;
            a.clusters = s.clusters;
            launch_cluster(attn_step_kv4_kernel<ng.value, nt.value>, dim3(units * s.clusters * s.cl, n_tok), dim3(AK_THREADS),
                           (size_t)attn_kv4_smem(ng.value, nt.value, GV, s.cl).total, s.cl, a);
            if (w.record) QZ_CUDA_CHECK(cudaEventRecord(w.record, stream()));
        };
        if (GV <= 4) go(std::integral_constant<int, 1>());
        else go(std::integral_constant<int, 2>());
    });
}

}  // namespace

extern "C" {

size_t cuda_kv4_bytes(int max_seq, int n_kv_heads, int head_dim)
{
    if (max_seq <= 0 || n_kv_heads <= 0 || !head_dim_ok(head_dim)) return 0;
    return (size_t)n_kv_heads * kv4_blocks(max_seq) * kv4_block_bytes(head_dim);
}

void cuda_kv4_append_rows(void *d_cache, const float *k, const float *v, int n_tok, int n_kv_heads, int head_dim, int max_seq, int pos0)
{
    if (n_tok == 0 || !cache_ok("cuda_kv4_append_rows", d_cache, n_kv_heads, head_dim, max_seq)) return;
    if (n_tok < 0 || pos0 < 0 || (long long)pos0 + n_tok > max_seq) {
        refuse("cuda_kv4_append_rows: 0 <= pos0 and pos0 + n_tok <= max_seq");
        return;
    }
    if (!k || !v || !aligned16(k) || !aligned16(v)) {
        refuse("cuda_kv4_append_rows: k and v must be 16-byte aligned");
        return;
    }
    const long long rows = (long long)n_tok * n_kv_heads, threads = rows * (head_dim / 8);
    if (rows >= 1ll << 31) {
        set_error(QZ_ERR_TOO_LARGE, "cuda_kv4_append_rows: n_tok * n_kv_heads must be below 2^31");
        return;
    }
    by_groups(head_dim, [&](auto ng) {
        launch(kv4_append_kernel<ng.value>, dim3((unsigned)((threads + 255) / 256), 2), dim3(256), 0, (uint8_t *)d_cache, k, v, (unsigned)rows, n_kv_heads,
               kv4_blocks(max_seq), pos0);
    });
}

void cuda_kv4_read_rows(float *k, float *v, const void *d_cache, int n_tok, int n_kv_heads, int head_dim, int max_seq, int pos0)
{
    if (n_tok == 0 || !cache_ok("cuda_kv4_read_rows", d_cache, n_kv_heads, head_dim, max_seq)) return;
    if (n_tok < 0 || pos0 < 0 || (long long)pos0 + n_tok > max_seq) {
        refuse("cuda_kv4_read_rows: 0 <= pos0 and pos0 + n_tok <= max_seq");
        return;
    }
    if (!k || !v || !aligned16(k) || !aligned16(v)) {
        refuse("cuda_kv4_read_rows: k and v must be 16-byte aligned");
        return;
    }
    const long long rows = (long long)n_tok * n_kv_heads, threads = rows * (head_dim / 8);
    if (rows >= 1ll << 31) {
        set_error(QZ_ERR_TOO_LARGE, "cuda_kv4_read_rows: n_tok * n_kv_heads must be below 2^31");
        return;
    }
    by_groups(head_dim, [&](auto ng) {
        launch(kv4_read_kernel<ng.value>, dim3((unsigned)((threads + 255) / 256), 2), dim3(256), 0, k, v, (const uint8_t *)d_cache, (unsigned)rows, n_kv_heads,
               kv4_blocks(max_seq), pos0);
    });
}

void cuda_rope_kv4_rows(float *q, float *k, const float *v, void *d_cache, int n_tok, int n_heads, int n_kv_heads, int head_dim, int max_seq,
                        int pos0, float theta, float yarn_scale, int yarn_orig_ctx, int neox)
{
    if (n_tok == 0 || !cache_ok("cuda_rope_kv4_rows", d_cache, n_kv_heads, head_dim, max_seq)) return;
    if (n_tok < 0 || n_tok > 65535 || n_heads <= 0 || pos0 < 0 || (long long)pos0 + n_tok > max_seq) {
        refuse("cuda_rope_kv4_rows: 0 <= pos0, pos0 + n_tok <= max_seq, n_tok <= 65535");
        return;
    }
    if (!q || !k || !v || !aligned16(q) || !aligned16(k) || !aligned16(v)) {
        refuse("cuda_rope_kv4_rows: q, k and v must be 16-byte aligned device pointers");
        return;
    }
    by_groups(head_dim, [&](auto ng) {
        // blocks of a token: all of its rows at once while they still find room on the chip, one from there on
        const int at_once = RK4_THREADS / 32 * (8 / ng.value), rows = (theta > 0.f ? n_heads : 0) + 2 * n_kv_heads;
        const int share = std::max(1, std::min((rows + at_once - 1) / at_once, 8 * sm_count() / n_tok));
        launch(rope_kv4_rows_kernel<ng.value>, dim3(n_tok, share), dim3(RK4_THREADS), 0, q, k, v, (uint8_t *)d_cache, n_heads, n_kv_heads,
               kv4_blocks(max_seq), pos0, theta, yarn_scale, yarn_orig_ctx, neox);
    });
}

int cuda_attn_kv4_supported(int n_heads, int n_kv_heads, int head_dim)
{
    return n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads / n_kv_heads <= AK_MAX_G && head_dim_ok(head_dim) ? 1 : 0;
}

void cuda_attn_step_kv4(float *out, const float *q, const float *k_new, const float *v_new, void *d_cache, int n_heads, int n_kv_heads,
                        int head_dim, int max_seq, const int *d_step, int pos, int window, float scale, const float *sinks, float theta,
                        float yarn_scale, int yarn_orig_ctx, int neox, int out_slot)
{
    if (!cache_ok("cuda_attn_step_kv4", d_cache, n_kv_heads, head_dim, max_seq)) return;
    if (!cuda_attn_kv4_supported(n_heads, n_kv_heads, head_dim) || (!d_step && (pos < 0 || pos >= max_seq))) {
        refuse("cuda_attn_step_kv4: n_heads a multiple of n_kv_heads, at most 16 query heads per kv head, 0 <= pos < max_seq");
        return;
    }
    if (!out || !q || !aligned16(out) || !aligned16(q) || (!k_new) != (!v_new) || !aligned16(k_new) || !aligned16(v_new)) {
        refuse("cuda_attn_step_kv4: out and q must be 16-byte aligned device pointers, k_new and v_new too or both NULL");
        return;
    }
    AttnKv4Args a = {out, q, k_new, v_new, (uint8_t *)d_cache, d_step, pos, n_heads, n_kv_heads, max_seq, kv4_blocks(max_seq), window, scale, sinks,
                     theta, yarn_scale, yarn_orig_ctx, neox, XQOut{nullptr, nullptr, nullptr, nullptr}, 0,
                     theta > 0.f ? step_rope_table(d_step, head_dim, theta, yarn_scale, yarn_orig_ctx) : nullptr};
    if (out_slot >= 0) {
        if (!activation_slot(out_slot, n_heads * head_dim, &a.o)) return;
        a.emit_q = 1;
    }
    launch_step(a, 1, head_dim);
}

void cuda_attn_prompt_kv4(float *out, const float *q, const void *d_cache, int n_tok, int n_heads, int n_kv_heads, int head_dim, int max_seq,
                          int pos0, int window, float scale, const float *sinks)
{
    if (n_tok == 0 || !cache_ok("cuda_attn_prompt_kv4", d_cache, n_kv_heads, head_dim, max_seq)) return;
    if (!cuda_attn_kv4_supported(n_heads, n_kv_heads, head_dim) || n_tok < 0 || n_tok > 65535 || pos0 < 0 || (long long)pos0 + n_tok > max_seq) {
        refuse("cuda_attn_prompt_kv4: n_heads a multiple of n_kv_heads, at most 16 query heads per kv head, pos0 + n_tok <= max_seq, n_tok <= 65535");
        return;
    }
    if (!out || !q || !aligned16(out) || !aligned16(q)) {
        refuse("cuda_attn_prompt_kv4: out and q must be 16-byte aligned device pointers");
        return;
    }
    // A few tokens on a long cache leave the prompt kernel, one CTA per kv head and 128 rows, with most SMs idle: there
    // the step kernel takes them one by one, all in one launch.  Time of either in us, fitted to measurements: waves of units
    // (more than four query heads: one to an SM, else two) and what a unit spends on a position, or what a CTA spends on a
    // tile of 64.  Step / prompt, 32 / 8 heads of 128: 32 tokens at 0 7.7 / 10.4, 64 at 0 14.7 / 10.8, 64 at 2000 56 / 58, 64
    // at 16000 338 / 384; 64 / 8: 16 at 200 13 / 15, 32 at 0 21 / 11, 16 at 2000 30 / 56, 64 at 2000 119 / 58; 12 / 6 of 64:
    // 32 at 0 4.7 / 6.3, 64 at 0 8.5 / 7.1, 64 at 16000 178 / 259.
    const int G = n_heads / n_kv_heads, ctas = n_kv_heads * ((n_tok + UMMA_M / G - 1) / (UMMA_M / G)), splits = (G + 7) / 8, units = n_kv_heads * splits * n_tok;
    const bool wide = (G + splits - 1) / splits > 4;
    const double h = head_dim / 128.0, sms = sm_count(), most = pos0 + (double)n_tok, mean = pos0 + 0.5 * n_tok;
    const double by_step = 2 + (wide ? 1.8 + 7.6 * h : 1 + 5 * h) * std::ceil(units / (wide ? sms : 2 * sms)) +
                           (wide ? 51 + 26 * h : 16 + 24 * h) * 1e-6 * units * (window > 0 ? std::min((double)window, mean) : mean);
    const double by_prompt = 3 + 6 * h + (0.5 + h) * std::ceil((window > 0 ? std::min((double)window + UMMA_M / G, most) : most) / APK_BN) * std::ceil(ctas / sms);
    if (by_step < by_prompt) {
        AttnKv4Args s = {out, q, nullptr, nullptr, (uint8_t *)d_cache, nullptr, pos0, n_heads, n_kv_heads, max_seq, kv4_blocks(max_seq), window, scale, sinks};
        launch_step(s, n_tok, head_dim);
        return;
    }
    AttnPromptKv4Args a = {out, q, (const uint8_t *)d_cache, n_tok, n_heads, n_kv_heads, kv4_blocks(max_seq), pos0, window, UMMA_M / G,
                           scale, sinks, status_word_if_ready()};
    by_groups(head_dim, [&](auto ng) {
        static PerDevice ready;
        ready.once([&] {
            QZ_CUDA_CHECK(cudaFuncSetAttribute(attn_prompt_kv4_kernel<ng.value>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)attn_prompt_kv4_smem(ng.value)));
        });
        launch(attn_prompt_kv4_kernel<ng.value>, dim3(n_kv_heads, (n_tok + a.tq - 1) / a.tq), dim3(APK_THREADS), attn_prompt_kv4_smem(ng.value), a);
    });
}

}  // extern "C"
