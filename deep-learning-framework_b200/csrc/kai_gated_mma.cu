// Gated linear layer for small and middle sizes: one launch forward, one for all products of the backward call.
//
//   forward    h = act(x Wg^T + bg) * (x Wu^T + bu)
//   backward   gx = gg Wg + gu Wu,   gWg = gg^T x,   gWu = gu^T x
//
// With a few hundred rows or less the tensor-core GEMM of kai_gemm_tc.cu spends its time on what it does around the
// product: planes of both weights written and read again (12 bytes per weight where 4 are needed), three launches.  Here
// operands come into shared memory as they are and are split into TF32 hi / lo parts in registers, on the warp-level
// instruction mma.sync.m16n8k8 (2.09 clocks each per SM, measured: 276 TFLOP/s, so 92 for three of them per product).
//
// A block of four warps owns a 64 x 64 tile of the product and walks the reduction 32 values at a time through a ring of three
// stages (cp.async).  A forward tile is 64 rows of x by 32 gate and the same 32 up columns, so that a thread's
// accumulators hold both factors of its outputs.  Fragments are 32-bit loads from rows padded to a stride of 4 (reduction
// contiguous) or 8 (reduction along the rows) modulo 32 banks, both without conflicts, so the three layouts of the call
// (NT, NN, TN) need no transpose.  Accumulation: the tensor core truncates; a fragment collects 32 values of the reduction
// and is then added to fp32 registers with rounding.
// Few tiles: the reduction is shared by the 1 to 8 CTAs of a cluster; each leaves its tile in its shared memory, and after a
// cluster barrier every CTA finishes its share of the rows by adding the tiles in rank order (the same bits on every run).
#include <initializer_list>

#include "kai_act.cuh"
#include "kai_common.cuh"

namespace kai {
namespace {

constexpr int kTile = 64, kStep = 32, kStages = 3, kThreads = 128;
constexpr int kRowStride = 36;                     // [64][32] tiles, reduction contiguous
constexpr int kColStride = 72;                     // [32][64] tiles, reduction along the rows
constexpr int kOperand = 64 * kRowStride;          // floats of an operand's tile, either way (2304)
static_assert(kOperand == 32 * kColStride, "both layouts take the same room");
constexpr int kStageFloats = 2 * kOperand;
constexpr int kOutStride = 68;
constexpr int kSmemBytes = kStages * kStageFloats * 4;
static_assert(kTile * kOutStride <= kStages * kStageFloats, "the finished tile reuses the ring");

__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// A [ROWS][COLS] box of a row-major matrix into shared memory; what lies outside the matrix becomes zero.
template <int ROWS, int COLS, int STRIDE>
__device__ __forceinline__ void load_box(float* dst, const float* __restrict__ src, int64_t ld, int64_t r0, int64_t c0, int64_t rows,
                                         int64_t cols, bool vec) {
    if (vec) {                                     // rows on 16-byte boundaries: a piece is inside or outside as a whole
        constexpr int PER_ROW = COLS / 4;
#pragma unroll
        for (int i = threadIdx.x; i < ROWS * PER_ROW; i += kThreads) {
            const int r = i / PER_ROW, c = i % PER_ROW * 4;
            const bool in = r0 + r < rows && c0 + c < cols;
            const float* at = in ? src + (r0 + r) * ld + c0 + c : src;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_at(dst + r * STRIDE + c)), "l"(at), "r"(in ? 16 : 0)
                         : "memory");
        }
    } else {
#pragma unroll 4
        for (int i = threadIdx.x; i < ROWS * COLS; i += kThreads) {
            const int r = i / COLS, c = i % COLS;
            const bool in = r0 + r < rows && c0 + c < cols;
            const float* at = in ? src + (r0 + r) * ld + c0 + c : src;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_at(dst + r * STRIDE + c)), "l"(at), "r"(in ? 4 : 0)
                         : "memory");
        }
    }
}

// hi = v rounded to TF32 by integer arithmetic (the conversion instruction issues at a fraction of the rate), lo = v - hi, exact.
__device__ __forceinline__ void split_frag(float v, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(v) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(v - __uint_as_float(hi));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// One stage: acc += A(64 x 32) . B(32 x 64).  A_ROWS: A's tile is [64][32] (else [32][64]); B_ROWS: B's is [64][32] (else [32][64]).
// PAIRED: columns 0 to 31 are gate, 32 to 63 up; a warp takes 16 of each.
template <bool A_ROWS, bool B_ROWS, bool PAIRED>
__device__ __forceinline__ void multiply(float (&acc)[2][4][4], const float* a, const float* b) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3, wm = warp >> 1, wn = warp & 1;
    float c[2][4][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[i][j][e] = 0.0f;
#pragma unroll
    for (int k0 = 0; k0 < kStep; k0 += 8) {
        uint32_t ah[2][4], al[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int m = wm * 32 + i * 16 + g;
#pragma unroll
            for (int e = 0; e < 4; ++e) {                // e: row + 8 (bit 0), column + 4 (bit 1)
                const int r = m + (e & 1) * 8, k = k0 + t + (e >> 1) * 4;
                split_frag(A_ROWS ? a[r * kRowStride + k] : a[k * kColStride + r], ah[i][e], al[i][e]);
            }
        }
        uint32_t bh[4][2], bl[4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = PAIRED ? (j >> 1) * 32 + wn * 16 + (j & 1) * 8 + g : wn * 32 + j * 8 + g;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = k0 + t + e * 4;
                split_frag(B_ROWS ? b[n * kRowStride + k] : b[k * kColStride + n], bh[j][e], bl[j][e]);
            }
        }
        // the small terms first; eight independent sums between two instructions on the same one
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) mma_tf32(c[i][j], al[i], bh[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) mma_tf32(c[i][j], ah[i], bl[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) mma_tf32(c[i][j], ah[i], bh[j]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] += c[i][j][e];
}

// The accumulators as a [64][kOutStride] tile in shared memory.
template <bool PAIRED>
__device__ __forceinline__ void leave_tile(const float (&acc)[2][4][4], float* out) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3, wm = warp >> 1, wn = warp & 1;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = PAIRED ? (j >> 1) * 32 + wn * 16 + (j & 1) * 8 + 2 * t : wn * 32 + j * 8 + 2 * t;
            float* at = out + (wm * 32 + i * 16 + g) * kOutStride + n;
            *reinterpret_cast<float2*>(at) = make_float2(acc[i][j][0], acc[i][j][1]);
            *reinterpret_cast<float2*>(at + 8 * kOutStride) = make_float2(acc[i][j][2], acc[i][j][3]);
        }
}

__device__ __forceinline__ void cluster_sync(int ranks) {
    if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
}
// Four values of the finished tile: the ranks' tiles added in rank order.
__device__ __forceinline__ float4 gather4(const float* tile, int at, int ranks) {
    const uint32_t local = smem_at(tile + at);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = 0; r < ranks; ++r) {
        uint32_t remote;
        float4 v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(r));
        asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    return s;
}

// The stages of a reduction of `steps` steps: load(step, stage) orders one, use(step, stage) works on it.
template <class Load, class Use>
__device__ __forceinline__ void run_ring(int begin, int end, Load load, Use use) {
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        if (begin + i < end) load(begin + i, i);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    int stage = 0;
    for (int k = begin; k < end; ++k) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncthreads();                                 // stage k is there for everybody, and stage k - 1 is free
        const int ahead = k + kStages - 1;
        if (ahead < end) load(ahead, stage == 0 ? kStages - 1 : stage - 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        use(k, stage);
        if (++stage == kStages) stage = 0;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
}

struct ForwardParams {
    float *h, *g, *u;
    const float *x, *wg, *wu, *bg, *bu, *leaky_alpha;
    int64_t M, F, K;
    int act, m_tiles, ranks, vec, vec_out;
};

__global__ void __launch_bounds__(kThreads, 4)
gated_mma_forward_kernel(const ForwardParams p) {
    extern __shared__ __align__(16) float ring[];
    const int rank = blockIdx.x % p.ranks, tile = blockIdx.x / p.ranks;
    const int64_t m0 = static_cast<int64_t>(tile % p.m_tiles) * kTile, f0 = static_cast<int64_t>(tile / p.m_tiles) * 32;
    const int steps = static_cast<int>((p.K + kStep - 1) / kStep), per = (steps + p.ranks - 1) / p.ranks;
    float acc[2][4][4] = {};
    run_ring(
        min(rank * per, steps), min((rank + 1) * per, steps),
        [&](int step, int stage) {
            float* a = ring + stage * kStageFloats;
            float* b = a + kOperand;
            const int64_t k0 = static_cast<int64_t>(step) * kStep;
            load_box<64, 32, kRowStride>(a, p.x, p.K, m0, k0, p.M, p.K, p.vec);
            load_box<32, 32, kRowStride>(b, p.wg, p.K, f0, k0, p.F, p.K, p.vec);
            load_box<32, 32, kRowStride>(b + 32 * kRowStride, p.wu, p.K, f0, k0, p.F, p.K, p.vec);
        },
        [&](int, int stage) {
            const float* a = ring + stage * kStageFloats;
            multiply<true, true, true>(acc, a, a + kOperand);
        });
    leave_tile<true>(acc, ring);
    cluster_sync(p.ranks);
    const float alpha = (p.leaky_alpha != nullptr) ? __ldg(p.leaky_alpha) : 0.0f;
    const int rows = kTile / p.ranks;                    // a power of two of ranks
#pragma unroll 1
    for (int i = threadIdx.x; i < rows * 8; i += kThreads) {
        const int r = rank * rows + i / 8, c = i % 8 * 4;
        const int64_t m = m0 + r, f = f0 + c;
        if (m >= p.M || f >= p.F) continue;
        float4 g4 = gather4(ring, r * kOutStride + c, p.ranks), u4 = gather4(ring, r * kOutStride + 32 + c, p.ranks), h4;
        float* g = reinterpret_cast<float*>(&g4);
        float* u = reinterpret_cast<float*>(&u4);
        float* h = reinterpret_cast<float*>(&h4);
        const int64_t at = m * p.F + f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (f + e < p.F) {
                if (p.bg) g[e] += __ldg(p.bg + f + e);
                if (p.bu) u[e] += __ldg(p.bu + f + e);
            }
            h[e] = act_forward(p.act, g[e], alpha) * u[e];
        }
        if (p.vec_out) {
            *reinterpret_cast<float4*>(p.h + at) = h4;
            if (p.g) { *reinterpret_cast<float4*>(p.g + at) = g4; *reinterpret_cast<float4*>(p.u + at) = u4; }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (f + e < p.F) {
                    p.h[at + e] = h[e];
                    if (p.g) { p.g[at + e] = g[e]; p.u[at + e] = u[e]; }
                }
        }
    }
    if (p.ranks > 1) cluster_sync(p.ranks);              // no CTA's tile goes away while another reads it
}

struct BackwardParams {
    float *gx, *gwg, *gwu;
    const float *gg, *gu, *wg, *wu, *x;
    int64_t M, F, K;
    int x_tiles, w_tiles;        // tiles of gx, tiles of one weight gradient
    int n_tiles;                 // tiles along K of either
    int ranks, acc_x, acc_w, vec_f, vec_k, vec_out;
};

__global__ void __launch_bounds__(kThreads, 4)
gated_mma_backward_kernel(const BackwardParams p) {
    extern __shared__ __align__(16) float ring[];
    const int rank = blockIdx.x % p.ranks;
    int tile = blockIdx.x / p.ranks;
    float acc[2][4][4] = {};
    const int which = tile < p.x_tiles ? 0 : 1 + (tile - p.x_tiles) / p.w_tiles;
    if (which > 0) tile = (tile - p.x_tiles) % p.w_tiles;
    const int64_t n0 = static_cast<int64_t>(tile % p.n_tiles) * kTile, r0 = static_cast<int64_t>(tile / p.n_tiles) * kTile;
    if (which == 0) {
        // gx: the reduction runs over the hidden units of the gate, then over those of the up projection
        const int half = static_cast<int>((p.F + kStep - 1) / kStep), steps = 2 * half, per = (steps + p.ranks - 1) / p.ranks;
        run_ring(
            min(rank * per, steps), min((rank + 1) * per, steps),
            [&](int step, int stage) {
                float* a = ring + stage * kStageFloats;
                const bool up = step >= half;
                const int64_t f0 = static_cast<int64_t>(up ? step - half : step) * kStep;
                load_box<64, 32, kRowStride>(a, up ? p.gu : p.gg, p.F, r0, f0, p.M, p.F, p.vec_f);
                load_box<32, 64, kColStride>(a + kOperand, up ? p.wu : p.wg, p.K, f0, n0, p.F, p.K, p.vec_k);
            },
            [&](int, int stage) {
                const float* a = ring + stage * kStageFloats;
                multiply<true, false, false>(acc, a, a + kOperand);
            });
    } else {
        const float* d = which == 1 ? p.gg : p.gu;
        const int steps = static_cast<int>((p.M + kStep - 1) / kStep), per = (steps + p.ranks - 1) / p.ranks;
        run_ring(
            min(rank * per, steps), min((rank + 1) * per, steps),
            [&](int step, int stage) {
                float* a = ring + stage * kStageFloats;
                const int64_t m0 = static_cast<int64_t>(step) * kStep;
                load_box<32, 64, kColStride>(a, d, p.F, m0, r0, p.M, p.F, p.vec_f);
                load_box<32, 64, kColStride>(a + kOperand, p.x, p.K, m0, n0, p.M, p.K, p.vec_k);
            },
            [&](int, int stage) {
                const float* a = ring + stage * kStageFloats;
                multiply<false, false, false>(acc, a, a + kOperand);
            });
    }
    leave_tile<false>(acc, ring);
    cluster_sync(p.ranks);
    float* out = which == 0 ? p.gx : which == 1 ? p.gwg : p.gwu;
    const bool add = which == 0 ? p.acc_x != 0 : p.acc_w != 0;
    const int64_t out_rows = which == 0 ? p.M : p.F;
    const int rows = kTile / p.ranks;
#pragma unroll 1
    for (int i = threadIdx.x; i < rows * 16; i += kThreads) {
        const int r = rank * rows + i / 16, c = i % 16 * 4;
        const int64_t row = r0 + r, col = n0 + c;
        if (row >= out_rows || col >= p.K) continue;
        float4 s4 = gather4(ring, r * kOutStride + c, p.ranks);
        float* s = reinterpret_cast<float*>(&s4);
        float* at = out + row * p.K + col;
        if (p.vec_out) {
            if (add) {
                const float4 o = *reinterpret_cast<const float4*>(at);
                s4 = make_float4(o.x + s4.x, o.y + s4.y, o.z + s4.z, o.w + s4.w);
            }
            *reinterpret_cast<float4*>(at) = s4;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col + e < p.K) at[e] = add ? at[e] + s[e] : s[e];
        }
    }
    if (p.ranks > 1) cluster_sync(p.ranks);
}

// CTAs that share a reduction: 1 to 8, whichever makes the busiest SM's steps fewest.  `work` is the number of steps of all tiles,
// `longest` that of one tile's reduction; a tile alone on an SM takes about 1000 clocks per step, the tensor instructions of
// two or three on one SM take turns, and meeting in the cluster costs about three steps.
int share(int64_t work, int longest, int sm_count) {
    int best = 1;
    double least = 0.0;
    for (int ranks = 1; ranks <= 8; ranks *= 2) {
        const double chain = (longest + ranks - 1) / ranks, each = static_cast<double>(work) / sm_count;
        const double cost = (chain > each ? chain : each) + 0.3 * (chain < each ? chain : each) + (ranks > 1 ? 2.0 + 0.5 * ranks : 0.0);
        if (ranks == 1 || cost < least) { best = ranks; least = cost; }
    }
    return best;
}

template <auto kernel, class P>
int launch(const char* name, const P& p, int64_t tiles, cudaStream_t s) {
    if (tiles * p.ranks >= (int64_t(1) << 31)) return fail(KAI_E_TOO_LARGE, "%s: too many tiles", name);
    static bool configured[kMaxDevices] = {};
    int dev = 0;
    KAI_CUDA(cudaGetDevice(&dev));
    if (dev < kMaxDevices && !configured[dev]) {
        KAI_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * p.ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = static_cast<unsigned>(p.ranks);
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.ranks > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess) { cudaGetLastError(); return cuda_fail(e, name); }
    count_launch();
    return KAI_OK;
}

bool on16(std::initializer_list<const float*> ps) {
    uintptr_t all = 0;
    for (const float* v : ps) all |= reinterpret_cast<uintptr_t>(v);
    return (all & 15) == 0;
}

}  // namespace

int gated_forward_mma(DeviceState* st, float* h, float* g, float* u, const float* wg, const float* wu, const float* x,
                      const float* bg, const float* bu, int64_t F, int64_t M, int64_t K, int act, const float* leaky_alpha,
                      cudaStream_t s) {
    ForwardParams p{};
    p.h = h; p.g = g; p.u = u; p.x = x; p.wg = wg; p.wu = wu; p.bg = bg; p.bu = bu; p.leaky_alpha = leaky_alpha;
    p.M = M; p.F = F; p.K = K; p.act = act;
    p.m_tiles = static_cast<int>((M + kTile - 1) / kTile);
    const int64_t tiles = p.m_tiles * ((F + 31) / 32);
    const int steps = static_cast<int>((K + kStep - 1) / kStep);
    p.ranks = share(tiles * steps, steps, st->sm_count);
    p.vec = (K & 3) == 0 && on16({x, wg, wu});
    p.vec_out = (F & 3) == 0 && on16({h, g, u});
    return launch<gated_mma_forward_kernel>("gated_mma_forward_kernel", p, tiles, s);
}

int gated_backward_mma(DeviceState* st, float* gx, float* gwg, float* gwu, const float* gg, const float* gu, const float* wg,
                       const float* wu, const float* x, int64_t F, int64_t M, int64_t K, int acc_x, int acc_w, cudaStream_t s) {
    BackwardParams p{};
    p.gx = gx; p.gwg = gwg; p.gwu = gwu; p.gg = gg; p.gu = gu; p.wg = wg; p.wu = wu; p.x = x;
    p.M = M; p.F = F; p.K = K; p.acc_x = acc_x; p.acc_w = acc_w;
    const int64_t n_tiles = (K + kTile - 1) / kTile;
    const int64_t x_tiles = gx ? (M + kTile - 1) / kTile * n_tiles : 0, w_tiles = gwg ? (F + kTile - 1) / kTile * n_tiles : 0;
    if (x_tiles + 2 * w_tiles >= (int64_t(1) << 31)) return fail(KAI_E_TOO_LARGE, "gated_linear_backward: too many tiles");
    p.n_tiles = static_cast<int>(n_tiles); p.x_tiles = static_cast<int>(x_tiles); p.w_tiles = static_cast<int>(w_tiles > 0 ? w_tiles : 1);
    // The split of the reductions is that of a call for all three gradients, so that each comes out the same whichever others are
    // wanted.
    const int sx = static_cast<int>(2 * ((F + kStep - 1) / kStep)), sw = static_cast<int>((M + kStep - 1) / kStep);
    p.ranks = share(((M + kTile - 1) / kTile * sx + 2 * ((F + kTile - 1) / kTile) * sw) * n_tiles, sx > sw ? sx : sw, st->sm_count);
    p.vec_f = (F & 3) == 0 && on16({gg, gu});
    p.vec_k = (K & 3) == 0 && on16({wg, wu, x});
    p.vec_out = (K & 3) == 0 && on16({gx, gwg, gwu});
    return launch<gated_mma_backward_kernel>("gated_mma_backward_kernel", p, x_tiles + 2 * w_tiles, s);
}

}  // namespace kai
