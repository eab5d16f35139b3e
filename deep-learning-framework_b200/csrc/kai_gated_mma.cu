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
// contiguous; read as 8 x 4 blocks) or 8 (reduction along the rows; read value by value) modulo 32 banks, both without
// conflicts, so the three layouts of the call (NT, NN, TN) need no transpose.  Accumulation: the tensor core truncates; a fragment collects 32 values of the reduction
// and is then added to fp32 registers with rounding.
// Few tiles: a reduction is shared by the 1 to 8 CTAs of a cluster (in the backward launch, where gx may have few tiles with a long
// reduction and the weight gradients many with a short one, the CTAs of some clusters share a tile and those of
// others take one each); each leaves its tile in its shared memory, and after a
// cluster barrier every CTA finishes its share of the rows by adding the tiles in rank order (the same bits on every run).
// Measured: 48 x 512 x 512 forward 10.5 us, 391 x 512 x 1365 forward 36, backward 68 us (the tensor-core GEMM: 42 and 83); 4096 x
// 512 x 512 forward 84 us, 51 TFLOP/s.  The tensor pipe is busy 54 % (backward), the issue slots 49 %: per 96 MMAs a warp spends 64 operations
// on loads, 192 on splits and 100 on copies and their bounds.  Part of that: operand blocks by ldmatrix and the bounds of a copy hoisted out of
// its loop gained 12 %, four blocks per SM instead of three 17 %.
#include <math.h>

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

// A [ROWS][COLS] box of a row-major matrix into shared memory, `rows` and `cols` of it inside the matrix (0 or less: nothing); what
// lies outside becomes zero (a copy of 0 bytes reads nothing).  src: the box's first value.
template <int ROWS, int COLS, int STRIDE>
__device__ __forceinline__ void load_box(float* dst, const float* __restrict__ src, int64_t ld, int64_t rows, int64_t cols, bool vec) {
    const int in_rows = rows < ROWS ? static_cast<int>(rows) : ROWS;
    const int in_cols = cols < COLS ? static_cast<int>(cols) : COLS;
    if (vec) {                                     // rows on 16-byte boundaries: a piece is inside or outside as a whole
        constexpr int PER_ROW = COLS / 4, ROW_STEP = kThreads / PER_ROW;
        const int r0 = threadIdx.x / PER_ROW, c = threadIdx.x % PER_ROW * 4;
        const float* at = src + r0 * ld + c;
        uint32_t to = smem_at(dst + r0 * STRIDE + c);
        const int limit = c < in_cols ? in_rows : 0;
#pragma unroll
        for (int i = 0; i < ROWS / ROW_STEP; ++i) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(at), "r"(r0 + i * ROW_STEP < limit ? 16 : 0)
                         : "memory");
            at += ROW_STEP * ld;
            to += ROW_STEP * STRIDE * 4;
        }
    } else {
        constexpr int ROW_STEP = kThreads / COLS;
        const int r0 = threadIdx.x / COLS, c = threadIdx.x % COLS;
        const float* at = src + r0 * ld + c;
        uint32_t to = smem_at(dst + r0 * STRIDE + c);
        const int limit = c < in_cols ? in_rows : 0;
#pragma unroll 4
        for (int i = 0; i < ROWS / ROW_STEP; ++i) {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(at), "r"(r0 + i * ROW_STEP < limit ? 4 : 0)
                         : "memory");
            at += ROW_STEP * ld;
            to += ROW_STEP * STRIDE * 4;
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

// D = A . B: the first product of a chain.
__device__ __forceinline__ void mma_tf32_first(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.0f));
}
// Four 8 x 4 blocks of 32-bit values, a lane naming one of their 32 rows: lane (g, t) receives row g, column t of each -- the
// fragment layout of the instruction above.
__device__ __forceinline__ void load_blocks(uint32_t (&v)[4], const float* row) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(smem_at(row))
                 : "memory");
}

// One stage: acc += A(64 x 32) . B(32 x 64).  A_ROWS: A's tile is [64][32] (else [32][64]); B_ROWS: B's is [64][32] (else [32][64]).
// PAIRED: columns 0 to 31 are gate, 32 to 63 up; a warp takes 16 of each.
template <bool A_ROWS, bool B_ROWS, bool PAIRED>
__device__ __forceinline__ void multiply(float (&acc)[2][4][4], const float* a, const float* b) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3, wm = warp >> 1, wn = warp & 1;
    float c[2][4][4];
    // the row and the 16-byte piece that this lane names for load_blocks: blocks are (row + 8: bit 0, column + 4: bit 1) for A,
    // (column + 4: bit 0, row + 8: bit 1) for two column tiles of B
    const int block = lane >> 3, in = lane & 7;
    const float* a_row = a + (wm * 32 + (block & 1) * 8 + in) * kRowStride + (block >> 1) * 4;
    const float* b_row = b + ((PAIRED ? wn * 16 : wn * 32) + (block >> 1) * 8 + in) * kRowStride + (block & 1) * 4;
#pragma unroll
    for (int k0 = 0; k0 < kStep; k0 += 8) {
        uint32_t ah[2][4], al[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t v[4];
            if (A_ROWS) {
                load_blocks(v, a_row + i * 16 * kRowStride + k0);
            } else {
                const int m = wm * 32 + i * 16 + g;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = __float_as_uint(a[(k0 + t + (e >> 1) * 4) * kColStride + m + (e & 1) * 8]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) split_frag(__uint_as_float(v[e]), ah[i][e], al[i][e]);
        }
        uint32_t bh[4][2], bl[4][2];
#pragma unroll
        for (int j = 0; j < 4; j += 2) {                 // column tiles j and j + 1
            uint32_t v[4];
            if (B_ROWS) {
                load_blocks(v, b_row + (PAIRED ? j * 16 : j * 8) * kRowStride + k0);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = __float_as_uint(b[(k0 + t + (e & 1) * 4) * kColStride + wn * 32 + (j + (e >> 1)) * 8 + g]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) split_frag(__uint_as_float(v[e]), bh[j + (e >> 1)][e & 1], bl[j + (e >> 1)][e & 1]);
        }
        // the small terms first; eight independent sums between two instructions on the same one
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (k0 == 0) mma_tf32_first(c[i][j], al[i], bh[j]);
                else mma_tf32(c[i][j], al[i], bh[j]);
            }
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
// Four values of the finished tile: the ranks' tiles added in rank order.  `own`: the CTA's own tile alone, whatever its rank.
__device__ __forceinline__ float4 gather4(const float* tile, int at, int ranks, bool own = false) {
    if (own) return *reinterpret_cast<const float4*>(tile + at);
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
            load_box<64, 32, kRowStride>(a, p.x + m0 * p.K + k0, p.K, p.M - m0, p.K - k0, p.vec);
            load_box<32, 32, kRowStride>(b, p.wg + f0 * p.K + k0, p.K, p.F - f0, p.K - k0, p.vec);
            load_box<32, 32, kRowStride>(b + 32 * kRowStride, p.wu + f0 * p.K + k0, p.K, p.F - f0, p.K - k0, p.vec);
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
    int ranks, split_x, split_w;     // CTAs of a cluster; whether they share a tile of gx / of a weight gradient or take one each
    int acc_x, acc_w, vec_f, vec_k, vec_out;
};

__global__ void __launch_bounds__(kThreads, 4)
gated_mma_backward_kernel(const BackwardParams p) {
    extern __shared__ __align__(16) float ring[];
    int rank = blockIdx.x % p.ranks, tile = blockIdx.x / p.ranks, ranks = 1;
    float acc[2][4][4] = {};
    // clusters of gx come first, then those of the weight gradients
    const int x_clusters = p.split_x ? p.x_tiles : (p.x_tiles + p.ranks - 1) / p.ranks;
    int which = 0;
    bool idle = false;
    if (tile < x_clusters) {
        if (p.split_x) ranks = p.ranks;
        else { tile = tile * p.ranks + rank; rank = 0; idle = tile >= p.x_tiles; }
    } else {
        tile -= x_clusters;
        if (p.split_w) ranks = p.ranks;
        else { tile = tile * p.ranks + rank; rank = 0; idle = tile >= 2 * p.w_tiles; }
        which = 1 + tile / p.w_tiles;
        tile %= p.w_tiles;
    }
    const int64_t n0 = static_cast<int64_t>(tile % p.n_tiles) * kTile, r0 = static_cast<int64_t>(tile / p.n_tiles) * kTile;
    if (which == 0) {
        // gx: the reduction runs over the hidden units of the gate, then over those of the up projection
        const int half = static_cast<int>((p.F + kStep - 1) / kStep), steps = 2 * half, per = (steps + ranks - 1) / ranks;
        run_ring(
            idle ? 0 : min(rank * per, steps), idle ? 0 : min((rank + 1) * per, steps),
            [&](int step, int stage) {
                float* a = ring + stage * kStageFloats;
                const bool up = step >= half;
                const int64_t f0 = static_cast<int64_t>(up ? step - half : step) * kStep;
                load_box<64, 32, kRowStride>(a, (up ? p.gu : p.gg) + r0 * p.F + f0, p.F, p.M - r0, p.F - f0, p.vec_f);
                load_box<32, 64, kColStride>(a + kOperand, (up ? p.wu : p.wg) + f0 * p.K + n0, p.K, p.F - f0, p.K - n0, p.vec_k);
            },
            [&](int, int stage) {
                const float* a = ring + stage * kStageFloats;
                multiply<true, false, false>(acc, a, a + kOperand);
            });
    } else {
        const float* d = which == 1 ? p.gg : p.gu;
        const int steps = static_cast<int>((p.M + kStep - 1) / kStep), per = (steps + ranks - 1) / ranks;
        run_ring(
            idle ? 0 : min(rank * per, steps), idle ? 0 : min((rank + 1) * per, steps),
            [&](int step, int stage) {
                float* a = ring + stage * kStageFloats;
                const int64_t m0 = static_cast<int64_t>(step) * kStep;
                load_box<32, 64, kColStride>(a, d + m0 * p.F + r0, p.F, p.M - m0, p.F - r0, p.vec_f);
                load_box<32, 64, kColStride>(a + kOperand, p.x + m0 * p.K + n0, p.K, p.M - m0, p.K - n0, p.vec_k);
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
    const int rows = idle ? 0 : kTile / ranks;
#pragma unroll 1
    for (int i = threadIdx.x; i < rows * 16; i += kThreads) {
        const int r = rank * rows + i / 16, c = i % 16 * 4;
        const int64_t row = r0 + r, col = n0 + c;
        if (row >= out_rows || col >= p.K) continue;
        float4 s4 = gather4(ring, r * kOutStride + c, ranks, p.ranks > ranks);
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

// Work of a launch in steps of a block, and how it is best dealt out.  A block that has started, filled its ring and left its tile
// has spent about one and a half steps; an SM with three or four blocks does a step in 1450 clocks, a block alone on its SM
// takes about 1.4 times that.
struct Job {
    int64_t tiles;
    int steps;
    int64_t blocks(bool split, int ranks) const { return split ? tiles * ranks : tiles; }
    int chain(bool split, int ranks) const { return tiles == 0 ? 0 : split ? (steps + ranks - 1) / ranks : steps; }
};
double cost(const Job& a, bool split_a, const Job& b, bool split_b, int ranks, int sm_count) {
    const double blocks = static_cast<double>(a.blocks(split_a, ranks) + b.blocks(split_b, ranks));
    const double work = static_cast<double>(a.blocks(split_a, ranks)) * a.chain(split_a, ranks) +
                        static_cast<double>(b.blocks(split_b, ranks)) * b.chain(split_b, ranks);
    const int ca = a.chain(split_a, ranks), cb = b.chain(split_b, ranks);
    const double chain = 1.4 * ((ca > cb ? ca : cb) + 1.5);
    const double share = ceil(blocks / sm_count) * (work / blocks + 1.5);
    return (chain > share ? chain : share) + (ranks > 1 ? 1.0 : 0.0);
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
    const Job job{tiles, static_cast<int>((K + kStep - 1) / kStep)}, none{0, 0};
    p.ranks = 1;
    for (int r = 2; r <= 8; r *= 2)
        if (cost(job, true, none, false, r, st->sm_count) < cost(job, true, none, false, p.ranks, st->sm_count)) p.ranks = r;
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
    const Job jx{(M + kTile - 1) / kTile * n_tiles, static_cast<int>(2 * ((F + kStep - 1) / kStep))};
    const Job jw{2 * ((F + kTile - 1) / kTile) * n_tiles, static_cast<int>((M + kStep - 1) / kStep)};
    p.ranks = 1;
    double least = cost(jx, false, jw, false, 1, st->sm_count);
    for (int r = 2; r <= 8; r *= 2)
        for (int split = 1; split < 4; ++split) {
            const double c = cost(jx, (split & 1) != 0, jw, (split & 2) != 0, r, st->sm_count);
            if (c < least) { least = c; p.ranks = r; p.split_x = split & 1; p.split_w = split >> 1; }
        }
    const int64_t groups = (p.split_x ? x_tiles : (x_tiles + p.ranks - 1) / p.ranks) +
                           (p.split_w ? 2 * w_tiles : (2 * w_tiles + p.ranks - 1) / p.ranks);
    p.vec_f = (F & 3) == 0 && on16({gg, gu});
    p.vec_k = (K & 3) == 0 && on16({wg, wu, x});
    p.vec_out = (K & 3) == 0 && on16({gx, gwg, gwu});
    return launch<gated_mma_backward_kernel>("gated_mma_backward_kernel", p, groups, s);
}

}  // namespace kai
