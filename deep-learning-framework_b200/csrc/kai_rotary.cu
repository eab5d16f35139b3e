// Rotary positions: pairs of a head's values turned by an angle that grows with the token's position.
//
//   a' = s (a cos t - b sin t),  b' = s (b cos t + a sin t),  t = pos * freq[i]       (backward: t -> -t)
//
// One read and one write of the tensor; HBM-bound from a few hundred tokens on, launch-bound below.
//
// The angle of a far position does not survive fp32 (pos = 1e5, freq = 1: half a unit in the last place is 4e-3
// radians), so it is formed in 64 bits, in turns: u = pos * (freq / 2 pi), u - rint(u) in [-1/2, 1/2] is exact, and
// only that remainder is rounded to fp32 (1.5e-8 turns = 9.4e-8 radians at most) for sincospif.  64-bit arithmetic is
// slow, but an angle belongs to all heads of a token: a thread owns the pairs of one unit of the head and walks over
// heads with the sines in registers.
#include "kai_common.cuh"

namespace kai {
namespace {

constexpr double kInvTwoPi = 0.15915494309189533577;

template <int V> struct Vec;
template <> struct Vec<1> { using T = float; };
template <> struct Vec<2> { using T = float2; };
template <> struct Vec<4> { using T = float4; };

template <int V>
__device__ __forceinline__ void load_v(const float* p, float* r) {
    const typename Vec<V>::T t = *reinterpret_cast<const typename Vec<V>::T*>(p);
    const float* f = reinterpret_cast<const float*>(&t);
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = f[i];
}
template <int V>
__device__ __forceinline__ void store_v(float* p, const float* r) {
    typename Vec<V>::T t;
    float* f = reinterpret_cast<float*>(&t);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = r[i];
    *reinterpret_cast<typename Vec<V>::T*>(p) = t;
}

struct RotaryParams {
    float* y;
    const float* x;
    const double* freq;
    const int64_t* pos;
    const float* scale;
    int64_t pos0, ntimes, rows, ldy, ldx;
    int nhead, npiece, nrot;
    int rot_units;        // units of V pairs (2 V values)
    int units;            // rotated units + copied units of the rest of the head (0 copied in place)
    int head_groups;      // threads that share the heads of one (row, unit)
    int backward;
};

// A unit is 2 V values of every head: V pairs, or 2 V values behind nrot that are copied.  Thread index =
// (row, head group, unit), unit fastest, so that a warp touches whole heads.
template <int V, bool HALF>
__global__ void __launch_bounds__(256)
rotary_kernel(const RotaryParams p) {
    const int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
    const int64_t rg = i / p.units;
    const int unit = static_cast<int>(i - rg * p.units);
    const int64_t row = rg / p.head_groups;
    const int group = static_cast<int>(rg - row * p.head_groups);
    if (row >= p.rows) return;
    const float* x = p.x + row * p.ldx;
    float* y = p.y + row * p.ldy;
    int ca, cb;                         // where the unit's two vectors begin in a head
    bool two = true;
    float c[V], s[V];
    if (unit < p.rot_units) {
        const int pair = unit * V;
        ca = HALF ? pair : 2 * pair;
        cb = HALF ? pair + p.nrot / 2 : 2 * pair + V;
        const int64_t pos = (p.pos != nullptr) ? p.pos[row] : p.pos0 + row % p.ntimes;
        const float scale = (p.scale != nullptr) ? __ldg(p.scale) : 1.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const double turns = static_cast<double>(pos) * (p.freq[pair + j] * kInvTwoPi);
            const float rest = static_cast<float>(turns - rint(turns));
            float sn, cs;
            sincospif(2.0f * rest, &sn, &cs);
            c[j] = cs * scale;
            s[j] = (p.backward ? -sn : sn) * scale;
        }
    } else {
        ca = p.nrot + (unit - p.rot_units) * 2 * V;
        cb = ca + V;
        two = cb < p.npiece;
    }
    const bool turn = unit < p.rot_units;
#pragma unroll 4
    for (int h = group; h < p.nhead; h += p.head_groups) {
        const int64_t at = static_cast<int64_t>(h) * p.npiece;
        float a[V], b[V];
        load_v<V>(x + at + ca, a);
        if (two) load_v<V>(x + at + cb, b);
        if (turn) {
            if (HALF) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float u = a[j], w = b[j];
                    a[j] = fmaf(u, c[j], -(w * s[j]));
                    b[j] = fmaf(w, c[j], u * s[j]);
                }
            } else {
                float v[2 * V];
#pragma unroll
                for (int j = 0; j < V; ++j) { v[j] = a[j]; v[V + j] = b[j]; }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float u = v[2 * j], w = v[2 * j + 1];
                    v[2 * j] = fmaf(u, c[j], -(w * s[j]));
                    v[2 * j + 1] = fmaf(w, c[j], u * s[j]);
                }
#pragma unroll
                for (int j = 0; j < V; ++j) { a[j] = v[j]; b[j] = v[V + j]; }
            }
        }
        store_v<V>(y + at + ca, a);
        if (two) store_v<V>(y + at + cb, b);
    }
}

template <int V>
int launch(const RotaryParams& p0, bool half, bool in_place, int sm_count, cudaStream_t s) {
    RotaryParams p = p0;
    p.rot_units = p.nrot / (2 * V);
    const int rest = in_place ? 0 : p.npiece - p.nrot;
    p.units = p.rot_units + (rest + 2 * V - 1) / (2 * V);
    if (p.units == 0) return KAI_OK;
    // Four heads per thread and angle, fewer where that leaves the SMs' thread slots empty.  3 x 32771 tokens, 12 heads: 123 us with
    // 3 or 4 heads per thread, 132 with 12, 166 with one; 32 x 512 tokens, 8 heads: 16.6 us with 2 to 8, 20 with one.
    const int64_t slots = static_cast<int64_t>(sm_count) * 2048;
    int64_t groups = (slots + p.rows * p.units - 1) / (p.rows * p.units);
    if (groups < (p.nhead + 3) / 4) groups = (p.nhead + 3) / 4;
    if (groups > p.nhead) groups = p.nhead;
    p.head_groups = static_cast<int>(groups);
    const int64_t blocks = (p.rows * p.units * groups + 255) / 256;
    if (blocks >= (int64_t(1) << 31)) return fail(KAI_E_TOO_LARGE, "rotary: too many values for one launch");
    if (half) rotary_kernel<V, true><<<static_cast<unsigned>(blocks), 256, 0, s>>>(p);
    else rotary_kernel<V, false><<<static_cast<unsigned>(blocks), 256, 0, s>>>(p);
    count_launch();
    return check_launch("rotary_kernel");
}

__global__ void rotary_frequencies_kernel(double* freq, int npair, double base, int scaling, double factor, double slow,
                                          double fast, double times) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= npair) return;
    if (scaling == KAI_ROTARY_BASE) base *= pow(factor, static_cast<double>(npair) / (npair - 1));
    double f = pow(base, -static_cast<double>(i) / npair);
    if (scaling == KAI_ROTARY_LINEAR) f /= factor;
    if (scaling == KAI_ROTARY_BY_PARTS) {
        double keep = (times * f * kInvTwoPi - slow) / (fast - slow);
        keep = fmin(fmax(keep, 0.0), 1.0);
        f *= keep + (1.0 - keep) / factor;
    }
    freq[i] = f;
}

}  // namespace

int rotary(DeviceState* st, float* y, const float* x, const double* freq, const int64_t* pos, int64_t pos0, int64_t nbat,
           int64_t ntimes, int64_t nhead, int64_t npiece, int64_t nrot, int layout, const float* scale, int64_t ldy,
           int64_t ldx, int backward, cudaStream_t s) {
    RotaryParams p{};
    p.y = y; p.x = x; p.freq = freq; p.pos = pos; p.scale = scale; p.pos0 = pos0;
    p.ntimes = ntimes; p.rows = nbat * ntimes; p.ldy = ldy; p.ldx = ldx;
    p.nhead = static_cast<int>(nhead); p.npiece = static_cast<int>(npiece); p.nrot = static_cast<int>(nrot);
    p.backward = backward;
    const bool in_place = x == y;
    // Width of a thread's loads: whole units must fall on vector boundaries in both tensors.
    const int64_t both = npiece | ldy | ldx;
    const uintptr_t at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y);
    const bool half = layout == KAI_ROTARY_HALF;
    if ((both & 3) == 0 && (nrot & 7) == 0 && (at & 15) == 0) return launch<4>(p, half, in_place, st->sm_count, s);
    if ((both & 1) == 0 && (nrot & 3) == 0 && (at & 7) == 0) return launch<2>(p, half, in_place, st->sm_count, s);
    return launch<1>(p, half, in_place, st->sm_count, s);
}

int rotary_frequencies(double* freq, int64_t nrot, double base, int scaling, double factor, double slow, double fast,
                       int64_t times, cudaStream_t s) {
    const int npair = static_cast<int>(nrot / 2);
    rotary_frequencies_kernel<<<(npair + 127) / 128, 128, 0, s>>>(freq, npair, base, scaling, factor, slow, fast,
                                                                 static_cast<double>(times));
    count_launch();
    return check_launch("rotary_frequencies_kernel");
}

}  // namespace kai
