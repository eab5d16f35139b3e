// Losses on rows of logits: distillation from a teacher's top logits, and the clipped policy loss with a KL term.
//
// Both are functions of log q at a few columns, q = softmax(x / T), and both have gradients of one form,
//   gx_c = gy (k q_c - w_c),     w_c = 0 but for the columns named by the row's labels,
//   distillation   k = T,          w = T p_j at column pidx_j              (p = softmax of the teacher's entries / T)
//   policy         k = -dl / T,    w = -dl / T at column pz                (dl = d loss / d log q)
// so they share three kernels, which differ only in a small description of the row (Distill / Policy below):
//   row_loss_kernel   one read of the row with a running maximum and sum per thread; loss and the row's statistics
//   row_grad_kernel   one read, one write, from the saved statistics
//   row_step_kernel   loss and gradient with ONE read: the row stays in the registers of a cluster of CTAs
// All are HBM-bound: 4, 8 and 8 bytes per logit.
//
// Precision: exponentials and their sums are fp32 (sums over at most a few hundred values per thread, then joined in
// a fixed order); log q = (x - max) / T - log(sum) is formed in 64 bits per row, with the logarithm of the sum split into
// exponent and mantissa: log(sum) rounded to fp32 would alone be off by up to 5e-7, which the ratio of two
// probabilities and a clip bound next to it would see.
#include <math.h>

#include "kai_common.cuh"

namespace kai {
namespace {

constexpr int kRowThreads = 512;
constexpr int kRowWarps = kRowThreads / 32;

// ---- row geometry ----------------------------------------------------------------------------------
// A row of any length at any 4-byte alignment is `head` scalars up to a 16-byte boundary, `quads` 16-byte pieces, and the
// rest.  Part r of `parts` takes quads [r * per, (r + 1) * per); part 0 also takes the scalars, one for each of its first
// threads.
struct RowShape {
    int64_t ncol, quads, per;
    int head, loose;        // loose: scalars in front of and behind the quads, at most 6
    __device__ __forceinline__ RowShape(const float* x, int64_t ncol_, int parts) {
        ncol = ncol_;
        head = static_cast<int>((4 - ((reinterpret_cast<uintptr_t>(x) >> 2) & 3)) & 3);
        if (head > ncol) head = static_cast<int>(ncol);
        quads = (ncol - head) >> 2;
        loose = static_cast<int>(ncol - 4 * quads);
        per = (quads + parts - 1) / parts;
    }
    __device__ __forceinline__ int64_t loose_col(int i) const { return i < head ? i : 4 * quads + i; }
    __device__ __forceinline__ bool owned(int64_t c, int part) const {
        const int64_t q = (c - head) >> 2;
        if (c < head || q >= quads) return part == 0;
        return q >= part * per && q < (part + 1) * per;
    }
};

__device__ __forceinline__ void max4(const float4& v, float& m) { m = fmaxf(fmaxf(m, fmaxf(v.x, v.y)), fmaxf(v.z, v.w)); }

// log of a positive sum, to about 1e-8 absolute
__device__ __forceinline__ double log_sum(float s) {
    if (!(s > 0.0f) || isinf(s)) return static_cast<double>(logf(s));
    int e;
    float f = frexpf(s, &e);
    if (f < 0.70710678f) { f *= 2.0f; --e; }
    return e * 0.69314718055994530942 + static_cast<double>(logf(f));
}

// Block-wide maximum / sum, the same value in every thread; `red` holds one float per warp.
__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[threadIdx.x & (kRowWarps - 1)];
#pragma unroll
    for (int o = kRowWarps / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[threadIdx.x & (kRowWarps - 1)];
#pragma unroll
    for (int o = kRowWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// exp((x - m) / T); a part of a row that holds nothing but -inf has m = -inf and no weight
__device__ __forceinline__ float weight(float x, float m, float inv_t) {
    return (m == -INFINITY && x == -INFINITY) ? 0.0f : expf((x - m) * inv_t);
}

// What a row's labels make of it.
enum : int { kLive = 0, kPadding = 1, kBad = 2 };

struct RowResult {
    float loss;
    float slope;   // d loss / d log q, without gy (distillation: the p_j carry the labels, slope is 1)
    float logp;
};

// ---- distillation ------------------------------------------------------------------------------------
struct Distill {
    const int* idx;
    const float* t;
    const float* temp;
    int ntop;

    // Shared memory of a row: the ids, the teacher's weights, and the student's logits there.
    struct Smem {
        int* id;        // [ntop] column, -1 = unused; `first` marks the entry that speaks for repeated ids
        float* p;       // [ntop] probability of the entry
        float* sum;     // [ntop] probability of all entries with that id (first occurrence), negative elsewhere
        float* xz;      // [ntop] logit of the student
        float* scalar;  // [0] sum of teacher weights
        int* state;
    };
    static __host__ __device__ size_t smem_bytes(int ntop) { return 16 * static_cast<size_t>(ntop) + 16; }
    __device__ __forceinline__ Smem smem(uint8_t* base) const {
        Smem m;
        m.id = reinterpret_cast<int*>(base);
        m.p = reinterpret_cast<float*>(m.id + ntop);
        m.sum = m.p + ntop;
        m.xz = m.sum + ntop;
        m.scalar = m.xz + ntop;
        m.state = reinterpret_cast<int*>(m.scalar + 2);
        return m;
    }
    __device__ __forceinline__ float temperature() const { return temp != nullptr ? __ldg(temp) : 1.0f; }

    // Step 1 (before the first block-wide barrier): ids, and what the student says there.  Every thread, strided.
    __device__ __forceinline__ void gather(const Smem& m, const float* x, int64_t row, int64_t ncol) const {
        for (int j = threadIdx.x; j < ntop; j += kRowThreads) {
            const int id = idx[row * ntop + j];
            m.id[j] = id;
            m.p[j] = t[row * ntop + j];
            m.xz[j] = (x != nullptr && id >= 0 && id < ncol) ? x[id] : 0.0f;
        }
    }
    // Step 2 (after a barrier): warp 0 turns the teacher's entries into probabilities.  p = 0 for unused entries.
    __device__ __forceinline__ void teacher(const Smem& m, int64_t ncol) const {
        if (threadIdx.x >= 32) return;
        const int lane = threadIdx.x;
        const float inv_t = 1.0f / temperature();
        float top = -INFINITY;
        bool bad = false, some = false, nan = false;
        for (int j = lane; j < ntop; j += 32) {
            const int id = m.id[j];
            if (id < -1 || id >= ncol) bad = true;
            if (id >= 0) {
                some = some || m.p[j] > -INFINITY;
                nan = nan || isnan(m.p[j]);
                top = fmaxf(top, m.p[j]);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        bad = __any_sync(0xffffffffu, bad);
        some = __any_sync(0xffffffffu, some || nan);
        float sum = 0.0f;
        for (int j = lane; j < ntop; j += 32) {
            const float e = (m.id[j] >= 0 && some) ? expf((m.p[j] - top) * inv_t) : 0.0f;
            sum += e;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float inv = 1.0f / sum;
        // the logit makes room for the probability; its logarithm is formed again from that logit, so keep it in `sum`
        for (int j = lane; j < ntop; j += 32) {
            const float v = m.p[j];
            m.sum[j] = (v - top) * inv_t;
            m.p[j] = (m.id[j] >= 0 && some) ? expf((v - top) * inv_t) * inv : 0.0f;
        }
        if (lane == 0) {
            m.scalar[0] = sum;
            *m.state = bad ? kBad : (some ? kLive : kPadding);
        }
    }
    __device__ __forceinline__ int state(const Smem& m) const { return *m.state; }

    // Step 3 (after a barrier, statistics known; one warp): the loss.
    __device__ __forceinline__ RowResult finish(const Smem& m, float top, float total, int64_t) const {
        const float tv = temperature();
        const float inv_t = 1.0f / tv;
        double s = 0.0;
        for (int j = threadIdx.x & 31; j < ntop; j += 32) {
            const float p = m.p[j];
            if (p != 0.0f)   // NaN included
                s += static_cast<double>(p) * (static_cast<double>(m.sum[j]) -
                                               (static_cast<double>(m.xz[j]) - static_cast<double>(top)) * inv_t);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s += log_sum(total) - log_sum(m.scalar[0]);
        RowResult r;
        r.loss = static_cast<float>(static_cast<double>(tv) * tv * s);
        r.slope = 1.0f;
        r.logp = 0.0f;
        return r;
    }
    // Step 4 (after a barrier): one entry speaks for all that name the same column.  Overwrites `sum`.
    __device__ __forceinline__ void merge(const Smem& m) const {
        for (int j = threadIdx.x; j < ntop; j += kRowThreads) {
            const int id = m.id[j];
            float sum = 0.0f;
            bool first = id >= 0;
            for (int i = 0; i < ntop; ++i) {
                const bool same = m.id[i] == id;
                if (same && i < j) first = false;
                if (same) sum += m.p[i];
            }
            m.sum[j] = first ? sum : -1.0f;
        }
    }
    // gx = gy T (q - sum p)
    __device__ __forceinline__ float q_coef(float gy, float) const { return gy * temperature(); }
    __device__ __forceinline__ int labels() const { return ntop; }
    __device__ __forceinline__ bool label(const Smem& m, int j, int64_t& c, float& w) const {
        c = m.id[j];
        w = m.sum[j];
        return w >= 0.0f || isnan(w);
    }
    __device__ __forceinline__ void extra(int64_t, float) const {}
};

// ---- policy loss ---------------------------------------------------------------------------------------
struct Policy {
    const int* z;
    const float* old_logp;
    const float* ref_logp;
    const float* adv;
    const float* low;
    const float* high;
    const float* beta;
    const float* temp;
    float* logp;

    struct Smem {
        int* id;
        float* xz;
        int* state;
    };
    static __host__ __device__ size_t smem_bytes(int) { return 16; }
    __device__ __forceinline__ Smem smem(uint8_t* base) const {
        return Smem{reinterpret_cast<int*>(base), reinterpret_cast<float*>(base) + 1, reinterpret_cast<int*>(base) + 2};
    }
    __device__ __forceinline__ float temperature() const { return temp != nullptr ? __ldg(temp) : 1.0f; }
    __device__ __forceinline__ void gather(const Smem& m, const float* x, int64_t row, int64_t ncol) const {
        if (threadIdx.x == 0) {
            const int id = z[row];
            const bool in = id >= 0 && id < ncol;
            *m.id = id;
            *m.state = in ? kLive : (id == -1 ? kPadding : kBad);
            *m.xz = (x != nullptr && in) ? x[id] : 0.0f;
        }
    }
    __device__ __forceinline__ void teacher(const Smem&, int64_t) const {}
    __device__ __forceinline__ int state(const Smem& m) const { return *m.state; }
    __device__ __forceinline__ RowResult finish(const Smem& m, float top, float total, int64_t row) const {
        const double l = (static_cast<double>(*m.xz) - static_cast<double>(top)) / temperature() - log_sum(total);
        const float a = adv[row];
        const float rho = (old_logp != nullptr) ? expf(static_cast<float>(l - static_cast<double>(old_logp[row]))) : 1.0f;
        float bound = rho;
        if (low != nullptr) bound = fmaxf(bound, 1.0f - __ldg(low));
        if (high != nullptr) bound = fminf(bound, 1.0f + __ldg(high));
        if (isnan(rho)) bound = rho;
        // without an advantage there is no loss, even where rho has overflowed
        const float ra = (a == 0.0f && !isnan(rho)) ? 0.0f : rho * a;
        const float ba = (a == 0.0f) ? 0.0f : bound * a;
        const bool free = !(ra > ba);
        RowResult r;
        r.loss = free ? -ra : -ba;
        r.slope = free ? -ra : 0.0f;
        if (ref_logp != nullptr && beta != nullptr) {
            const float b = __ldg(beta);
            const float d = static_cast<float>(static_cast<double>(ref_logp[row]) - l);
            const float e1 = expm1f(d);          // e^d - 1: the term is d^2 / 2 next to 0, e^d - d - 1 would cancel
            r.loss = fmaf(b, e1 - d, r.loss);
            r.slope = fmaf(-b, e1, r.slope);
        }
        r.logp = static_cast<float>(l);
        return r;
    }
    __device__ __forceinline__ void merge(const Smem&) const {}
    __device__ __forceinline__ float q_coef(float gy, float slope) const { return -(gy * slope) / temperature(); }
    __device__ __forceinline__ int labels() const { return 1; }
    __device__ __forceinline__ bool label(const Smem& m, int, int64_t& c, float& w) const {
        c = *m.id;
        w = 1.0f;
        return true;
    }
    __device__ __forceinline__ void extra(int64_t row, float v) const {
        if (logp != nullptr) logp[row] = v;
    }
};

struct RowParams {
    const float* x;
    float* y;
    float* ps;
    float* gx;
    const float* gy;
    int64_t ncol;
    int parts;       // CTAs per row
    int* flag;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Writes two floats to the same shared-memory variable of CTA `rank` of the cluster.
__device__ __forceinline__ void push_stat(float2* local, uint32_t rank, float a, float b) {
    const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(local));
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(rank));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(a), "f"(b) : "memory");
}

// Joins the parts' (maximum, sum of exponentials against it).  Rank order, the same in every CTA.
__device__ __forceinline__ void join(const float2* stat, int parts, float inv_t, float& top, float& total) {
    top = stat[0].x;
    for (int i = 1; i < parts; ++i) top = fmaxf(top, stat[i].x);
    total = 0.0f;
    for (int i = 0; i < parts; ++i) total += stat[i].y * weight(stat[i].x, top, inv_t);
}

// ---- loss alone ------------------------------------------------------------------------------------------
// A thread keeps a running maximum m and sum s over its pieces of the row, four 16-byte loads at a time: the maximum of
// the sixteen values first, one rescaling of s if it rose, then sixteen exponentials.
template <class L>
__global__ void __launch_bounds__(kRowThreads)
row_loss_kernel(const RowParams p, const L loss) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ float red_m[kRowWarps], red_s[kRowWarps];
    __shared__ float2 stat[8];
    const int64_t row = blockIdx.x / p.parts;
    const int part = blockIdx.x % p.parts;
    if (p.parts > 1) cluster_arrive();
    const float* x = p.x + row * p.ncol;
    const RowShape shape(x, p.ncol, p.parts);
    const typename L::Smem sm = loss.smem(dyn);
    const float inv_t = 1.0f / loss.temperature();
    if (part == 0) loss.gather(sm, x, row, p.ncol);

    const float4* xq = reinterpret_cast<const float4*>(x + shape.head);
    const int64_t q_end = min(shape.quads, (part + 1) * shape.per);
    float m = -INFINITY, s = 0.0f;
    for (int64_t q0 = part * shape.per + threadIdx.x; q0 < q_end; q0 += 4 * kRowThreads) {
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t q = q0 + u * kRowThreads;
            v[u] = (q < q_end) ? __ldcs(xq + q) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        }
        float m1 = m;
#pragma unroll
        for (int u = 0; u < 4; ++u) max4(v[u], m1);
        if (m1 > m) { s *= weight(m, m1, inv_t); m = m1; }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            s += (weight(v[u].x, m, inv_t) + weight(v[u].y, m, inv_t)) + (weight(v[u].z, m, inv_t) + weight(v[u].w, m, inv_t));
    }
    if (part == 0 && static_cast<int>(threadIdx.x) < shape.loose) {
        const float v = x[shape.loose_col(threadIdx.x)];
        if (v > m) { s *= weight(m, v, inv_t); m = v; }
        s += weight(v, m, inv_t);
    }
    float top = block_max(m, red_m);
    if (part == 0) loss.teacher(sm, p.ncol);
    float total = block_sum(s * weight(m, top, inv_t), red_s);
    if (p.parts > 1) {
        cluster_wait();                         // every CTA of the cluster has begun
        if (threadIdx.x == 0) push_stat(&stat[part], 0, top, total);
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (part != 0) return;
        join(stat, p.parts, inv_t, top, total);
    }
    if (threadIdx.x < 32) {
        const int state = loss.state(sm);
        RowResult r = loss.finish(sm, top, total, row);
        if (state == kPadding) r.loss = r.slope = r.logp = 0.0f;
        if (state == kBad) r.loss = r.slope = r.logp = nanf("");
        if (threadIdx.x == 0) {
            p.y[row] = r.loss;
            loss.extra(row, r.logp);
            p.ps[3 * row + 0] = top;
            p.ps[3 * row + 1] = total;
            p.ps[3 * row + 2] = r.slope;
            if (state == kBad) *p.flag = 1;
        }
    }
}

// Stores the gradients of four neighbouring columns; `vec`: the output row has the input row's alignment.
__device__ __forceinline__ void store4(float* g, float4 v, bool vec) {
    if (vec) {
        __stcs(reinterpret_cast<float4*>(g), v);
    } else {
        g[0] = v.x; g[1] = v.y; g[2] = v.z; g[3] = v.w;
    }
}

// ---- gradient from saved statistics ----------------------------------------------------------------------
template <class L, int NV>
__global__ void __launch_bounds__(kRowThreads)
row_grad_kernel(const RowParams p, const L loss) {
    extern __shared__ __align__(16) uint8_t dyn[];
    const int64_t row = blockIdx.x / p.parts;
    const int part = blockIdx.x % p.parts;
    const float* x = p.x + row * p.ncol;
    float* gx = p.gx + row * p.ncol;
    const RowShape shape(x, p.ncol, p.parts);
    const typename L::Smem sm = loss.smem(dyn);
    const bool vec = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(gx)) & 15) == 0;
    const float4* xq = reinterpret_cast<const float4*>(x + shape.head);
    const int64_t q_end = min(shape.quads, (part + 1) * shape.per);
    const int64_t q_begin = part * shape.per + threadIdx.x;
    float4 v[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int64_t q = q_begin + u * kRowThreads;
        v[u] = (q < q_end) ? __ldcs(xq + q) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const bool has_loose = part == 0 && static_cast<int>(threadIdx.x) < shape.loose;
    const float lv = has_loose ? x[shape.loose_col(threadIdx.x)] : 0.0f;
    loss.gather(sm, nullptr, row, p.ncol);
    // the labels' logits are read before anything is written: gx may be x
    const float inv_t = 1.0f / loss.temperature();
    const float top = p.ps[3 * row], total = p.ps[3 * row + 1], slope = p.ps[3 * row + 2];
    const float gy = (p.gy != nullptr) ? p.gy[row] : 1.0f;
    __syncthreads();
    loss.teacher(sm, p.ncol);
    __syncthreads();
    loss.merge(sm);
    const int state = loss.state(sm);
    const float k = loss.q_coef(gy, slope);
    // one factor for all columns; a padding row's logits are not looked at, a bad label poisons the row
    const float f = k / total;
    auto grad = [&](float xv) {
        return state == kLive ? weight(xv, top, inv_t) * f : (state == kPadding ? 0.0f : nanf(""));
    };
    // labelled columns of this part: value in registers until the columns around them are written
    for (int base = 0; base < loss.labels(); base += kRowThreads) {
        // gathered in rounds of one label per thread; rounds beyond the first only for more than 512 labels
        const int j = base + threadIdx.x;
        int64_t c = 0;
        float w = 0.0f;
        bool mine = state == kLive && j < loss.labels() && loss.label(sm, j, c, w) && shape.owned(c, part);
        float g = 0.0f;
        if (mine) g = weight(x[c], top, inv_t) * f - k * w;
        __syncthreads();
        if (mine) sm.xz[j] = g;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int64_t q = q_begin + u * kRowThreads;
        if (q < q_end)
            store4(gx + shape.head + 4 * q, make_float4(grad(v[u].x), grad(v[u].y), grad(v[u].z), grad(v[u].w)), vec);
    }
    if (has_loose) gx[shape.loose_col(threadIdx.x)] = grad(lv);
    __syncthreads();
    for (int j = threadIdx.x; j < loss.labels(); j += kRowThreads) {
        int64_t c = 0;
        float w = 0.0f;
        if (state == kLive && loss.label(sm, j, c, w) && shape.owned(c, part)) gx[c] = sm.xz[j];
    }
}

// ---- loss and gradient with one read -----------------------------------------------------------------------
// The row is spread over the registers of `parts` CTAs (a cluster, 1 to 8), NV 16-byte pieces per thread.  Each CTA
// forms its maximum and sum of exponentials, the cluster exchanges the two numbers through distributed shared memory,
// and the gradient is one multiplication per value.
template <class L, int NV>
__global__ void __launch_bounds__(kRowThreads)
row_step_kernel(const RowParams p, const L loss) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ float red_m[kRowWarps], red_s[kRowWarps];
    __shared__ float2 stat[8];
    __shared__ float slope_sh;
    const int64_t row = blockIdx.x / p.parts;
    const int part = blockIdx.x % p.parts;
    if (p.parts > 1) cluster_arrive();
    const float* x = p.x + row * p.ncol;
    float* gx = p.gx + row * p.ncol;
    const RowShape shape(x, p.ncol, p.parts);
    const typename L::Smem sm = loss.smem(dyn);
    const bool vec = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(gx)) & 15) == 0;
    const float4* xq = reinterpret_cast<const float4*>(x + shape.head);
    const int64_t q_end = min(shape.quads, (part + 1) * shape.per);
    const int64_t q_begin = part * shape.per + threadIdx.x;
    float4 v[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int64_t q = q_begin + u * kRowThreads;
        v[u] = (q < q_end) ? __ldcs(xq + q) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
    const bool has_loose = part == 0 && static_cast<int>(threadIdx.x) < shape.loose;
    float lv = has_loose ? x[shape.loose_col(threadIdx.x)] : -INFINITY;
    loss.gather(sm, x, row, p.ncol);
    const float inv_t = 1.0f / loss.temperature();
    const float gy = (p.gy != nullptr) ? p.gy[row] : 1.0f;

    float m = lv;
#pragma unroll
    for (int u = 0; u < NV; ++u) max4(v[u], m);
    const float mine_top = block_max(m, red_m);
    loss.teacher(sm, p.ncol);
    float s = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        v[u] = make_float4(weight(v[u].x, mine_top, inv_t), weight(v[u].y, mine_top, inv_t),
                           weight(v[u].z, mine_top, inv_t), weight(v[u].w, mine_top, inv_t));
        s += (v[u].x + v[u].y) + (v[u].z + v[u].w);
    }
    if (has_loose) { lv = weight(lv, mine_top, inv_t); s += lv; }
    float top = mine_top, total = block_sum(s, red_s);
    if (p.parts > 1) {
        cluster_wait();                         // every CTA of the cluster has begun
        if (static_cast<int>(threadIdx.x) < p.parts) push_stat(&stat[part], threadIdx.x, top, total);
        __syncwarp();
        cluster_arrive();
        cluster_wait();                         // all labels are gathered and all statistics here: x may be written
        join(stat, p.parts, inv_t, top, total);
    }
    const int state = loss.state(sm);
    if (threadIdx.x < 32) {
        RowResult r = loss.finish(sm, top, total, row);
        if (state == kPadding) r.loss = r.slope = r.logp = 0.0f;
        if (state == kBad) r.loss = r.slope = r.logp = nanf("");
        if (threadIdx.x == 0) {
            slope_sh = r.slope;
            if (part == 0) {
                p.y[row] = r.loss;
                loss.extra(row, r.logp);
                if (state == kBad) *p.flag = 1;
            }
        }
    }
    __syncthreads();
    loss.merge(sm);
    const float k = loss.q_coef(gy, slope_sh);
    const float f = k / total;
    const float f_mine = f * weight(mine_top, top, inv_t);
    auto grad = [&](float e) { return state == kLive ? e * f_mine : (state == kPadding ? 0.0f : nanf("")); };
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int64_t q = q_begin + u * kRowThreads;
        if (q < q_end)
            store4(gx + shape.head + 4 * q, make_float4(grad(v[u].x), grad(v[u].y), grad(v[u].z), grad(v[u].w)), vec);
    }
    if (has_loose) gx[shape.loose_col(threadIdx.x)] = grad(lv);
    __syncthreads();
    for (int j = threadIdx.x; j < loss.labels(); j += kRowThreads) {
        int64_t c = 0;
        float w = 0.0f;
        if (state == kLive && loss.label(sm, j, c, w) && shape.owned(c, part))
            gx[c] = weight(sm.xz[j], top, inv_t) * f - k * w;
    }
}

// ---- host side -----------------------------------------------------------------------------------------------
template <class K, class L>
int launch_rows(K kernel, const char* name, const RowParams& p, const L& loss, int64_t nrow, bool cluster, size_t smem,
                cudaStream_t s) {
    if (nrow * p.parts >= (int64_t(1) << 31)) return fail(KAI_E_TOO_LARGE, "%s: too many rows for one launch", name);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(nrow * p.parts));
    cfg.blockDim = dim3(kRowThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = static_cast<unsigned>(p.parts);
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster && p.parts > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, loss);
    if (e != cudaSuccess) { cudaGetLastError(); return cuda_fail(e, name); }
    count_launch();
    return KAI_OK;
}

// CTAs per row of a call that may use up to `most`: as few as hold the row (`need`), and more while the rows alone do not
// fill the SMs twice and every thread still has a piece.
int parts_for(int64_t nrow, int64_t ncol, int need, int most, int sm_count) {
    int parts = need;
    while (parts * 2 <= most && nrow * parts < 2 * static_cast<int64_t>(sm_count) &&
           ncol >= static_cast<int64_t>(parts) * 2 * 4 * kRowThreads)
        parts *= 2;
    return parts;
}

template <class L>
int run_loss(DeviceState* st, RowParams p, const L& loss, int64_t nrow, size_t smem, cudaStream_t s) {
    p.flag = st->flag_dev + 2;
    p.parts = parts_for(nrow, p.ncol, 1, 8, st->sm_count);
    return launch_rows(row_loss_kernel<L>, "row_loss_kernel", p, loss, nrow, true, smem, s);
}

template <class L>
int run_grad(DeviceState* st, RowParams p, const L& loss, int64_t nrow, size_t smem, cudaStream_t s) {
    p.flag = st->flag_dev + 2;
    const int64_t per = 4 * kRowThreads;
    const int64_t pieces = (p.ncol + per - 1) / per;       // 16-byte pieces per thread over the whole row
    int64_t parts = (pieces + 7) / 8;
    if (parts < 1) parts = 1;
    const int64_t each = (pieces + parts - 1) / parts;
    p.parts = static_cast<int>(parts);
    if (each <= 1) return launch_rows(row_grad_kernel<L, 1>, "row_grad_kernel", p, loss, nrow, false, smem, s);
    if (each <= 2) return launch_rows(row_grad_kernel<L, 2>, "row_grad_kernel", p, loss, nrow, false, smem, s);
    if (each <= 4) return launch_rows(row_grad_kernel<L, 4>, "row_grad_kernel", p, loss, nrow, false, smem, s);
    return launch_rows(row_grad_kernel<L, 8>, "row_grad_kernel", p, loss, nrow, false, smem, s);
}

template <class L>
int run_step(DeviceState* st, RowParams p, const L& loss, int64_t nrow, size_t smem, cudaStream_t s) {
    const int64_t cap = 8 * 4 * kRowThreads;        // values a CTA holds at 8 pieces per thread
    int need = 1;
    while (need < 8 && need * cap < p.ncol) need *= 2;
    if (need * cap < p.ncol) {                      // a row that a cluster cannot hold: two kernels, two reads
        KAI_TRY(ensure_aux(st, nrow * 3 * 4));
        p.ps = static_cast<float*>(st->aux);
        KAI_TRY(run_loss(st, p, loss, nrow, smem, s));
        return run_grad(st, p, loss, nrow, smem, s);
    }
    p.flag = st->flag_dev + 2;
    p.parts = parts_for(nrow, p.ncol, need, 8, st->sm_count);
    const int64_t per = static_cast<int64_t>(p.parts) * 4 * kRowThreads;
    const int64_t each = (p.ncol + per - 1) / per;
    if (each <= 1) return launch_rows(row_step_kernel<L, 1>, "row_step_kernel", p, loss, nrow, true, smem, s);
    if (each <= 2) return launch_rows(row_step_kernel<L, 2>, "row_step_kernel", p, loss, nrow, true, smem, s);
    if (each <= 4) return launch_rows(row_step_kernel<L, 4>, "row_step_kernel", p, loss, nrow, true, smem, s);
    return launch_rows(row_step_kernel<L, 8>, "row_step_kernel", p, loss, nrow, true, smem, s);
}

RowParams row_params(const float* x, int64_t ncol) {
    RowParams p{};
    p.x = x;
    p.ncol = ncol;
    p.parts = 1;
    return p;
}

}  // namespace

int loss_distill(DeviceState* st, float* y, float* ps, const float* x, const int* idx, const float* t, int64_t nrow,
                 int64_t ncol, int64_t ntop, const float* temp, cudaStream_t s) {
    RowParams p = row_params(x, ncol);
    p.y = y; p.ps = ps;
    const Distill d{idx, t, temp, static_cast<int>(ntop)};
    return run_loss(st, p, d, nrow, Distill::smem_bytes(d.ntop), s);
}
int loss_distill_backward(DeviceState* st, float* gx, const float* gy, const float* x, const float* ps, const int* idx,
                          const float* t, int64_t nrow, int64_t ncol, int64_t ntop, const float* temp, cudaStream_t s) {
    RowParams p = row_params(x, ncol);
    p.gx = gx; p.gy = gy; p.ps = const_cast<float*>(ps);
    const Distill d{idx, t, temp, static_cast<int>(ntop)};
    return run_grad(st, p, d, nrow, Distill::smem_bytes(d.ntop), s);
}
int loss_distill_step(DeviceState* st, float* y, float* gx, const float* gy, const float* x, const int* idx,
                      const float* t, int64_t nrow, int64_t ncol, int64_t ntop, const float* temp, cudaStream_t s) {
    RowParams p = row_params(x, ncol);
    p.y = y; p.gx = gx; p.gy = gy;
    const Distill d{idx, t, temp, static_cast<int>(ntop)};
    return run_step(st, p, d, nrow, Distill::smem_bytes(d.ntop), s);
}

int loss_policy(DeviceState* st, float* y, float* logp, float* ps, const float* x, const int* z, const float* old_logp,
                const float* ref_logp, const float* adv, int64_t nrow, int64_t ncol, const float* low, const float* high,
                const float* beta, const float* temp, cudaStream_t s) {
    RowParams p = row_params(x, ncol);
    p.y = y; p.ps = ps;
    const Policy l{z, old_logp, ref_logp, adv, low, high, beta, temp, logp};
    return run_loss(st, p, l, nrow, Policy::smem_bytes(1), s);
}
int loss_policy_backward(DeviceState* st, float* gx, const float* gy, const float* x, const float* ps, const int* z,
                         int64_t nrow, int64_t ncol, const float* temp, cudaStream_t s) {
    RowParams p = row_params(x, ncol);
    p.gx = gx; p.gy = gy; p.ps = const_cast<float*>(ps);
    const Policy l{z, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, temp, nullptr};
    return run_grad(st, p, l, nrow, Policy::smem_bytes(1), s);
}
int loss_policy_step(DeviceState* st, float* y, float* logp, float* gx, const float* gy, const float* x, const int* z,
                     const float* old_logp, const float* ref_logp, const float* adv, int64_t nrow, int64_t ncol,
                     const float* low, const float* high, const float* beta, const float* temp, cudaStream_t s) {
    RowParams p = row_params(x, ncol);
    p.y = y; p.gx = gx; p.gy = gy;
    const Policy l{z, old_logp, ref_logp, adv, low, high, beta, temp, logp};
    return run_step(st, p, l, nrow, Policy::smem_bytes(1), s);
}

}  // namespace kai
