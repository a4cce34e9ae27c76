// Host-side state of the library that its translation units share.
#pragma once

#include "activation.cuh"

namespace qz {

bool pdl_enabled();            // kernels are being recorded into a graph as programmatic dependents
cudaStream_t replay_stream();  // stream on which the step words are written, in order with the replays of recorded graphs
int *status_word();            // device word that bounded waits set when they run out; NULL if it cannot be created
int *status_word_if_ready();   // the same for calls that may be captured before anything created it (then NULL)
// activation-form scratch slot 0..3 for a vector of n values; false (and the sticky error) if there is none
bool activation_slot(int slot, int n, XQOut *o);
// the (cos, sin) table registered for these step words and parameters, or NULL
const float2 *step_rope_table(const int *d_step, int head_dim, float theta, float yarn_scale, int yarn_orig_ctx);

// What is set once per device, as a kernel's attributes are.  (Devices beyond the table: every time.)
struct PerDevice {
    bool done[16] = {};
    template <class F>
    void once(F f)
    {
        int device = 0;
        if (cudaGetDevice(&device) != cudaSuccess) cudaGetLastError();
        if (device < 16 && done[device]) return;
        f();
        if (device < 16) done[device] = true;
    }
};

// Ordinary launch, or programmatic dependent launch when enabled; cluster > 1: clusters of that many CTAs along x.
template <class... KArgs, class... Args>
static void launch_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, int cluster, Args... args)
{
    g_launch_count++;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream();
    cudaLaunchAttribute at[2];
    int n = 0;
    if (pdl_enabled()) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = (unsigned)cluster;
        at[n].val.clusterDim.y = 1;
        at[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    QZ_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...));
}

template <class... KArgs, class... Args>
static void launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, Args... args)
{
    launch_cluster(kernel, grid, block, smem, 1, args...);
}

}  // namespace qz
