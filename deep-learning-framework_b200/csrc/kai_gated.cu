// Gated linear layer: h = act(x Wg^T + bg) * (x Wu^T + bu), and the passes of its backward call that are not products.
#include "kai_act.cuh"
#include "kai_common.cuh"

namespace kai {
namespace {

// h = act(g) * u over `total` values, after the biases have been added (in place when `save` is set).
__global__ void __launch_bounds__(256)
gate_kernel(float* __restrict__ h, float* g, float* u, const float* __restrict__ bg, const float* __restrict__ bu,
            int64_t total, int64_t ncol, int act, const float* __restrict__ leaky_alpha, int save) {
    const float alpha = (leaky_alpha != nullptr) ? __ldg(leaky_alpha) : 0.0f;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total; i += stride) {
        float gv = g[i], uv = u[i];
        if (bg != nullptr) gv += bg[i % ncol];
        if (bu != nullptr) uv += bu[i % ncol];
        if (save) {
            if (bg != nullptr) g[i] = gv;
            if (bu != nullptr) u[i] = uv;
        }
        h[i] = act_forward(act, gv, alpha) * uv;
    }
}

// gg = gh * u * act'(g), gu = gh * act(g); every value is read before its outputs are written, so the outputs may lie
// in the inputs' buffers.
__global__ void __launch_bounds__(256)
gate_backward_kernel(float* gg, float* gu, const float* gh, const float* g, const float* u, int64_t total, int act,
                     const float* __restrict__ leaky_alpha) {
    const float alpha = (leaky_alpha != nullptr) ? __ldg(leaky_alpha) : 0.0f;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total; i += stride) {
        const float d = gh[i], gv = g[i], uv = u[i];
        gg[i] = d * uv * act_grad_from_x(act, gv, alpha);
        gu[i] = d * act_forward(act, gv, alpha);
    }
}

inline unsigned gate_grid(int64_t total, int sm_count) {
    int64_t blocks = (total + 255) / 256;
    const int64_t cap = static_cast<int64_t>(sm_count) * 16;
    return static_cast<unsigned>(blocks < cap ? blocks : cap);
}

}  // namespace

int gated_apply(DeviceState* st, float* h, float* g, float* u, const float* bg, const float* bu, int64_t ndat,
                int64_t yvec, int act, const float* leaky_alpha, int save, cudaStream_t s) {
    const int64_t total = ndat * yvec;
    gate_kernel<<<gate_grid(total, st->sm_count), 256, 0, s>>>(h, g, u, bg, bu, total, yvec, act, leaky_alpha, save);
    count_launch();
    return check_launch("gate_kernel");
}

int gated_apply_backward(DeviceState* st, float* gg, float* gu, const float* gh, const float* g, const float* u,
                         int64_t total, int act, const float* leaky_alpha, cudaStream_t s) {
    gate_backward_kernel<<<gate_grid(total, st->sm_count), 256, 0, s>>>(gg, gu, gh, g, u, total, act, leaky_alpha);
    count_launch();
    return check_launch("gate_backward_kernel");
}

}  // namespace kai
