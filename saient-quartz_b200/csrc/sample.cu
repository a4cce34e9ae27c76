// C entry point of the token sampler.
#include <algorithm>
#include <cmath>

#include "host.cuh"
#include "sample.cuh"

using namespace qz;

namespace {

size_t sample_smem(int chunk) { return ((sizeof(SampleShared) + 15) & ~(size_t)15) + (size_t)chunk * 4; }

// CTAs per row: enough for two CTAs and their parts of rows to fit an SM (16 for the longest rows), then, while that leaves
// SMs idle, more of them as long as a thread keeps four tokens (the device holds 7 clusters of 16).
int sample_cluster(int n_rows, int vocab)
{
    static PerDevice ready;
    ready.once([] {
        QZ_CUDA_CHECK(cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        if (cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) cudaGetLastError();
    });
    int cl = 1;
    while (cl < SMP_MAX_CLUSTER && sample_smem((vocab + cl - 1) / cl + 3) > 112 * 1024) cl *= 2;
    while (cl < SMP_MAX_CLUSTER && (long long)n_rows * cl * 2 <= (cl == 8 ? 112 : sm_count()) && vocab / (cl * 2) >= 4 * SMP_THREADS) cl *= 2;
    return cl;
}

}  // namespace

extern "C" int cuda_sample_supported(int vocab, float temperature, float top_p, float min_p)
{
    return vocab >= 1 && vocab <= SMP_MAX_VOCAB && temperature >= 0.f && std::isfinite(temperature) && top_p == top_p && min_p == min_p ? 1 : 0;
}

extern "C" void cuda_sample(const float *d_logits, int n_rows, int vocab, size_t row_stride, float temperature, int top_k, float top_p,
                            float min_p, const float *d_u, int *d_tokens, float *d_probs)
{
    if (n_rows == 0) return;
    if (n_rows < 0 || vocab <= 0 || vocab > SMP_MAX_VOCAB || row_stride < (size_t)vocab) {
        set_error(vocab > SMP_MAX_VOCAB ? QZ_ERR_TOO_LARGE : QZ_ERR_BAD_SHAPE, "cuda_sample: 1 <= vocab <= 524288 and row_stride >= vocab");
        return;
    }
    if (!cuda_sample_supported(vocab, temperature, top_p, min_p)) {
        set_error(QZ_ERR_BAD_SHAPE, "cuda_sample: temperature must be finite and at least 0, top_p and min_p must be numbers");
        return;
    }
    if (!d_logits || !d_tokens || (!d_u && temperature > 0.f)) {
        set_error(QZ_ERR_BAD_SHAPE, "cuda_sample: d_logits, d_tokens and (temperature > 0) d_u must be device pointers");
        return;
    }
    const int cl = sample_cluster(n_rows, vocab), chunk = ((vocab + cl - 1) / cl + 3) & ~3;
    const double inv_t = 1.0 / (double)temperature, c = 32.0 * 1.4426950408889634 * inv_t, lowest = std::min((double)min_p, 1.0);
    const SampleArgs a = {d_logits, row_stride, vocab, temperature, inv_t, c, 1.0 / c, top_k, top_p, lowest,
                          lowest > 0.0 ? (float)std::log(lowest) : 0.f, d_u, d_tokens, d_probs, chunk};
    launch_cluster(sample_kernel, dim3((unsigned)n_rows * cl), dim3(SMP_THREADS), sample_smem(chunk), cl, a);
}
