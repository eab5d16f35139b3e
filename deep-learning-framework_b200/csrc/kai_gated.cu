// Gated linear layer: the pass of its backward call that is not a product.
#include "kai_act.cuh"
#include "kai_common.cuh"

namespace kai {
namespace {

// gg = gh * u * act'(g), gu = gh * act(g); every value is read before its outputs are written, so the outputs may lie
// in the inputs' buffers.
__global__ void __launch_bounds__(256)
gate_backward_kernel(float* gg, float* gu, const float* gh, const float* g, const float* u, int64_t total, int act,
                     const float* __restrict__ leaky_alpha) {
    const float alpha = (leaky_alpha != nullptr) ? __ldg(leaky_alpha) : 0.0f;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total; i += stride) {
        const float d = gh[i], gv = g[i], uv = u[i];
        const float2 v = act_value_slope(act, gv, alpha);
        gg[i] = d * uv * v.y;
        gu[i] = d * v.x;
    }
}

inline unsigned gate_grid(int64_t total, int sm_count) {
    int64_t blocks = (total + 255) / 256;
    const int64_t cap = static_cast<int64_t>(sm_count) * 16;
    return static_cast<unsigned>(blocks < cap ? blocks : cap);
}

}  // namespace

int gated_apply_backward(DeviceState* st, float* gg, float* gu, const float* gh, const float* g, const float* u,
                         int64_t total, int act, const float* leaky_alpha, cudaStream_t s) {
    gate_backward_kernel<<<gate_grid(total, st->sm_count), 256, 0, s>>>(gg, gu, gh, g, u, total, act, leaky_alpha);
    count_launch();
    return check_launch("gate_backward_kernel");
}

}  // namespace kai
