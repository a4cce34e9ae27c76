// C entry point of the token sampler.
#include "host.cuh"
#include "sample.cuh"

using namespace qz;

extern "C" void cuda_sample(const float *d_logits, int n_rows, int vocab, size_t row_stride, float temperature, int top_k, float top_p,
                            float min_p, const float *d_u, int *d_tokens, float *d_probs)
{
    if (n_rows == 0) return;
    if (n_rows < 0 || vocab <= 0 || vocab > SMP_MAX_VOCAB || row_stride < (size_t)vocab) {
        set_error(vocab > SMP_MAX_VOCAB ? QZ_ERR_TOO_LARGE : QZ_ERR_BAD_SHAPE, "cuda_sample: 1 <= vocab <= 524288 and row_stride >= vocab");
        return;
    }
    if (!(temperature >= 0.f) || !isfinite(temperature) || !(top_p == top_p) || !(min_p == min_p)) {
        set_error(QZ_ERR_BAD_SHAPE, "cuda_sample: temperature must be finite and at least 0, top_p and min_p must be numbers");
        return;
    }
    if (!d_logits || !d_tokens || (!d_u && temperature > 0.f)) {
        set_error(QZ_ERR_BAD_SHAPE, "cuda_sample: d_logits, d_tokens and (temperature > 0) d_u must be device pointers");
        return;
    }
    const SampleArgs a = {d_logits, row_stride, vocab, temperature, top_k, top_p, min_p, d_u, d_tokens, d_probs};
    launch(sample_kernel, dim3((unsigned)n_rows), dim3(SMP_THREADS), 0, a);
}
