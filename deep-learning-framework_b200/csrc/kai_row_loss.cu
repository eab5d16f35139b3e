// Losses on rows of logits: distillation from a teacher's top logits, and the clipped policy loss with a KL term.
//
// Both are functions of log q at a few columns, q = softmax(x / T), and both have gradients of one form,
//   gx_c = k q_c - k w_c,     w_c = 0 but for the columns that the row's labels name,
//   distillation   k = gy T,          w_c = sum of p_j with pidx_j = c        (p = softmax of the teacher's entries / T)
//   policy         k = -gy dl / T,    w_c = 1 at c = pz                       (dl = d loss / d log q)
// so they share their kernels, which differ only in a small description of a row's labels (Distill / Policy below).
//
// row_stream_kernel<L, T, MODE> is one persistent kernel for the three calls: kLoss (read the row: loss and
// statistics), kGrad (read, write, from saved statistics) and kStep (loss and gradient with ONE read of the row).
// All are HBM-bound: 4, 8 and 8 bytes per logit.
//   * A row is spread over the shared memory of `parts` CTAs (kLoss, kStep: a cluster of 1 to 8): one bulk copy in, a pass for
//     the maximum, a pass for the exponentials' sum, and (kStep, kGrad) a pass that turns the logits into the gradient
//     in place, then one bulk copy out.  A CTA holds one part of one row; what hides its waits are the other
//     CTAs of the SM, four parts of up to 50 KB or six of 32 KB.
//   * Statistics: each warp takes its own reference and sum of exponentials and sends both to all CTAs of the row
//     (distributed shared memory); ONE cluster barrier per row later every warp joins the same list in the same order.
//   * Labels: a warp of its own prepares the next row's labels (teacher softmax, the student's logits at the ids) and parks
//     what the row's loss is made of; eight parked rows are settled together, one per lane.
// Measured on the way, 8192 x 32000, loss and gradient (2.1 GB, 320 us at the copy rate): row in registers, one CTA per
// part and launch, 725 us; the same persistent, next rows fetched by cp.async, 640 us -- 21 instructions per value, most of
// them addresses and bounds; by bulk copies, 657 us, the label warp's 13,000 clocks per row of 64-bit arithmetic now in
// everybody's way; with the losses parked, 537 us.  There the registers still held the row (96 KB per SM) while twice
// that lay prefetched in shared memory, and 8,000 clocks from load to store of each part bounded the rate; stores from
// registers stood in the way of the label warp's loads.  As it is: 431 to 445 us (4.8 TB/s), policy loss 4096 x 50257 324 us (5.1 TB/s),
// loss alone 195 us (5.4 TB/s), two calls 550 us.  A part takes 17,000 to 24,000 clocks from load to store (3700 waiting
// for its load, 3500 in the two passes, 3500 to 5000 at the cluster barrier, 2000 to 2700 for statistics and slope, 3000 for the
// gradient, 2500 until the store has read its source), with 26 to 39 % of the issue slots used: it is bound by the latency of that
// chain.  Measured without gain: parts of 4096 to 16384 columns, 64 to 256 threads, cluster sizes between the powers of two.
// row_short_kernel takes rows of up to 4096 columns (kGrad with many rows: 2048) with up to 256 labels, a warp each: there the barriers and the label warp of
// row_stream_kernel cost more than the row.  Loss and gradient of 8192 rows, the stream's time first: 97 columns, 64 labels 37 us and
// 14.5; 1000 columns, 256 labels 155 and 40 (64 labels: 44 and 23); 2000 columns, 200 labels 123 and 50; policy loss, 8191 x 1000 29
// and 17 (10 at the copy rate; bound by the chain of one row in the 24 warps per SM that its registers leave).
// row_loss_wide_kernel takes the rows that the shared memory of a cluster cannot hold (more than 445000 columns, 280000 with 2048 labels), for kLoss;
// kStep is then kLoss and kGrad.
//
// Precision.  exp((x - m) / T) is formed as 2^(x c - k) with c = log2(e) / T and k = m c, each rounded once: one fused multiply-add,
// rounded relative to the exponent itself; what k lost stands in every term and in the logarithm below alike, and rounding
// c is a temperature off by 2^-24 at most, the same for every term: log q is off by as much of the difference between the label's argument and
// the row's mean one (a label 20 below the maximum: 1.2e-6 at most; a label's logarithm with the exact factor over a sum with the rounded
// one is further off in most rows).  The largest term is 2^0 to within rounding: with k the integer above
// m c, which joins sums by exact powers of two, it is a power of a fraction, and the instruction's 2^-22 on a term that is nearly
// the whole sum cost log-probabilities next to 0 three binary digits (a policy row of 1e-6 relative error, 2e-7 so).
// Exponentials and their sums are fp32 (a few dozen values per thread, then joined in a fixed order); log q = ln 2 (x c - k) - log(sum) is formed in 64 bits per row, with
// the logarithm of the sum split into exponent and mantissa: log(sum) rounded to fp32 would alone be off by up to
// 5e-7, which the ratio of two probabilities and a clip bound next to it would see.  The instruction's results are 5e-8 low on average
// wherever its argument lies, and are taken twice where warps' sums are joined: sums measured 2e-8 to 8e-8 low, 7e-8 to 1.2e-7 off (root mean
// square, 1000 to 128256 columns); the ratio of a policy row 8e-8 to 2e-7.
#include <math.h>

#include <mutex>
#include <type_traits>

#include "kai_common.cuh"
#include "kai_tcgen05.cuh"

namespace kai {
namespace {

enum Mode : int { kLoss, kGrad, kStep };

// What a row's labels make of it.
enum : int { kLive = 0, kPadding = 1, kBad = 2 };

constexpr double kLn2 = 0.69314718055994530942;
constexpr int kMaxParts = 8;
constexpr int kShortWarps = 4, kShortLeast = 8;

// ---- row geometry ----------------------------------------------------------------------------------
// A row of any length at any 4-byte alignment is `head` scalars up to a 16-byte boundary, `quads` 16-byte pieces, and the
// rest.  Part r of `parts` takes quads [r * per, (r + 1) * per); part 0 also takes the scalars, one for each of its first
// threads.
struct RowShape {
    int quads, per;
    int head, loose;        // loose: scalars in front of and behind the quads, at most 6
    // per_: pieces of a part, the same for all rows (the alignment of a row costs at most one piece)
    __device__ __forceinline__ RowShape(const float* x, int ncol, int per_) : per(per_) {
        head = static_cast<int>((4 - ((reinterpret_cast<uintptr_t>(x) >> 2) & 3)) & 3);
        if (head > ncol) head = ncol;
        quads = (ncol - head) >> 2;
        loose = ncol - 4 * quads;
    }
    __device__ __forceinline__ int begin(int part) const { return min(part * per, quads); }
    __device__ __forceinline__ int count(int part) const { return min(per, quads - begin(part)); }
    __device__ __forceinline__ int loose_col(int i) const { return i < head ? i : 4 * quads + i; }
    __device__ __forceinline__ bool owned(int c, int part) const {
        const int q = (c - head) >> 2;
        if (c < head || q >= quads) return part == 0;
        return q >= begin(part) && q < begin(part) + per;
    }
};

__device__ __forceinline__ float max4(const float4& v, float m) {
    return fmaxf(fmaxf(m, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
}
__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
template <class V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// log of a positive sum, to about 1e-8 absolute; NaN for a sum of nothing
__device__ __forceinline__ double log_sum(float s) {
    if (!(s > 0.0f) || isinf(s)) return static_cast<double>(nanf(""));     // no distribution
    int e;
    float f = frexpf(s, &e);
    if (f < 0.70710678f) { f *= 2.0f; --e; }
    return e * kLn2 + static_cast<double>(logf(f));
}

// 2^(x c - k).  Against k = -inf (nothing but -inf was seen) the caller uses 0, so that -inf has no weight instead of
// being NaN.
__device__ __forceinline__ float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float weight(float x, float k, float c) { return exp2_approx(fmaf(x, c, -k)); }
__device__ __forceinline__ float reference(float m, float c) { return m * c; }
__device__ __forceinline__ float finite_ref(float k) { return k == -INFINITY ? 0.0f : k; }
__device__ __forceinline__ float weight4(float4 v, float k, float c) {
    v = make_float4(weight(v.x, k, c), weight(v.y, k, c), weight(v.z, k, c), weight(v.w, k, c));
    return (v.x + v.y) + (v.z + v.w);
}
struct RowParams {
    const float* x;
    float* y;
    float* ps;
    float* gx;
    const float* gy;
    const float* temp;
    int64_t nrow, ncol;
    int parts;       // CTAs per row
    int per;         // 16-byte pieces of a part, and of a stage
    int* flag;       // label outside its range
    int* status;     // a bounded wait ran out
};

// What both kinds of labels keep of a row in shared memory.
struct alignas(16) RowHead {
    float gy;
    float stat[3];           // the saved row of ps (kGrad): reference, sum, slope
    int state;
    float teacher, weights;  // distillation: reference and sum of the teacher's weights
    int lone;                // distillation: no id occurs twice
};
constexpr int kParked = 8;  // rows whose losses are settled together
static_assert(sizeof(RowHead) % 16 == 0, "what follows it in shared memory is read 16 bytes at a time");

struct Temp {
    float t, c;       // temperature, log2(e) / T
    __device__ __forceinline__ explicit Temp(const float* p) {
        t = (p != nullptr) ? __ldg(p) : 1.0f;
        c = static_cast<float>(1.44269504088896340736 / static_cast<double>(t));
    }
    // log2 of the weight of x against k
    __device__ __forceinline__ double exponent(float x, float k) const {
        return static_cast<double>(x) * static_cast<double>(c) - static_cast<double>(k);
    }
};

struct Result {
    float loss, slope, logp;     // slope: d loss / d log q, without gy (distillation: the p_j carry the labels, slope is 1)
};

// ---- distillation ------------------------------------------------------------------------------------
struct Distill {
    const int* idx;
    const float* t;
    int ntop, ntop4;       // ntop4: rounded up to a multiple of 4, unused entries behind ntop
    int bits;              // log2 of the 16-bit places that `merged` has room for

    struct Row : RowHead {};
    // row_short_kernel has room for a table of its own, four to eight places for a label (row_stream_kernel: 512 bytes more would
    // cost it a CTA per SM at 8000 columns, 98 us becoming 106).
    __host__ __device__ size_t table_bytes() const { return size_t(2) << (bits + 2); }
    __host__ __device__ size_t bytes() const { return sizeof(RowHead) + 20 * static_cast<size_t>(ntop4); }
    static __device__ __forceinline__ int* ids(Row* r) { return reinterpret_cast<int*>(r + 1); }
    __device__ __forceinline__ float* probs(Row* r) const { return reinterpret_cast<float*>(ids(r) + ntop4); }
    __device__ __forceinline__ float* logits(Row* r) const { return probs(r) + ntop4; }
    __device__ __forceinline__ float* teacher(Row* r) const { return logits(r) + ntop4; }
    __device__ __forceinline__ float* merged(Row* r) const { return teacher(r) + ntop4; }
    __host__ __device__ __forceinline__ int labels() const { return ntop; }

    // The label warp works ahead so that no load of its own is waited for: ids and teacher logits are fetched two rows ahead
    // (Ahead), the student's logits there one row ahead (Flight), up to kAhead labels per lane; what is beyond is loaded in
    // place.
    static constexpr int kAhead = 4;
    struct Ahead {
        int id[kAhead];
        float t[kAhead];
    };
    struct Flight {
        float x[kAhead];
    };
    __device__ __forceinline__ void ahead(Ahead& a, int64_t row) const {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int j = (threadIdx.x & 31) + 32 * i;
            a.id[i] = j < ntop ? idx[row * ntop + j] : -1;
            a.t[i] = j < ntop ? t[row * ntop + j] : 0.0f;
        }
    }
    // The student's logits at ids of this part, or at all of them.
    __device__ __forceinline__ void depart(Flight& f, const Ahead& a, const float* x, const RowShape& shape, int part, bool all,
                                           int64_t, int64_t ncol) const {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int z = a.id[i];
            f.x[i] = (z >= 0 && z < ncol && (all || shape.owned(z, part))) ? x[z] : 0.0f;
        }
    }
    // Whether no id of the row is repeated, by one warp.  Each label writes its place into a table of any content, where a hash of
    // its id says, and reads back who stands there: itself, and it is done; the same id, and there is a repetition;
    // another id, and it tries again without those that are done.  Labels of one id that both lost try again together.  Every try
    // settles one label for each place in use, so tries end.  Against a search for each label, loss and gradient: 2048 x 32000
    // with 256 labels 227 us and 146, with 1000 labels 2115 and 505; 8192 x 2500 with 64 labels 68 and 58.5.
    __device__ __forceinline__ bool distinct(const int* id, uint16_t* table, int log) const {
        const int lane = threadIdx.x & 31;
        uint64_t open = 0;                     // of the labels lane + 32 i (KAI_TOP_MAX: 64 of them)
        for (int i = 0, j = lane; j < ntop; ++i, j += 32)
            if (id[j] >= 0) open |= uint64_t(1) << i;
        bool twice = false;
        while (__any_sync(0xffffffffu, open != 0)) {
            for (int i = 0, j = lane; j < ntop; ++i, j += 32)
                if (open >> i & 1) table[place(id[j], log)] = static_cast<uint16_t>(j);
            __syncwarp();
            for (int i = 0, j = lane; j < ntop; ++i, j += 32)
                if (open >> i & 1) {
                    const int who = table[place(id[j], log)];
                    if (who == j) open &= ~(uint64_t(1) << i);
                    else if (id[who] == id[j]) twice = true;
                }
            if (__any_sync(0xffffffffu, twice)) return false;
            __syncwarp();                      // the next try writes where this one has read
        }
        return true;
    }
    __device__ __forceinline__ uint32_t place(int z, int log) const { return static_cast<uint32_t>(z) * 2654435761u >> (32 - log); }
    // One warp: labels and logits into shared memory, the teacher's entries as probabilities (0 for unused entries), and
    // the row's state.
    __device__ __forceinline__ void arrive(Row* r, const Flight& f, const Ahead& a, const float* x, const RowShape& shape,
                                           int part, bool all, int64_t row, int64_t ncol, const Temp& tv, bool gradient,
                                           uint16_t* table) const {
        const int lane = threadIdx.x & 31;
        int* id = ids(r);
        float* p = probs(r);
        float* xz = logits(r);
        float* te = teacher(r);
        float top = -INFINITY;
        bool bad = false, some = false;
        auto take = [&](int j, int z, float v, float xv) {
            id[j] = z;
            te[j] = v;
            xz[j] = xv;
            if (z < -1 || z >= ncol) bad = true;
            if (z >= 0) {
                some = some || !(v == -INFINITY);      // NaN counts: it poisons the row
                top = fmaxf(top, v);
            }
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (lane + 32 * i < ntop4) take(lane + 32 * i, a.id[i], a.t[i], f.x[i]);
#pragma unroll 4
        for (int j = lane + 32 * kAhead; j < ntop4; j += 32) {
            const int z = j < ntop ? idx[row * ntop + j] : -1;
            const bool read = z >= 0 && z < ncol && (all || shape.owned(z, part));
            take(j, z, j < ntop ? t[row * ntop + j] : 0.0f, read ? x[z] : 0.0f);
        }
        top = warp_max(top);
        bad = __any_sync(0xffffffffu, bad);
        some = __any_sync(0xffffffffu, some);
        const float k = finite_ref(reference(top, tv.c));
        float sum = 0.0f;
        for (int j = lane; j < ntop4; j += 32) {
            const float e = (id[j] >= 0) ? weight(te[j], k, tv.c) : 0.0f;
            sum += e;
            p[j] = e;
        }
        sum = warp_sum(sum);
        const float inv = some ? 1.0f / sum : 0.0f;
        for (int j = lane; j < ntop4; j += 32) p[j] *= inv;
        bool lone = gradient && !bad;
        if (gradient) {
            __syncwarp();
            if (lone)
                lone = (table != nullptr) ? distinct(id, table, bits + 2) : distinct(id, reinterpret_cast<uint16_t*>(merged(r)), bits);
            __syncwarp();
            if (lone || ntop <= kMergeAhead) {
                // repeated ids: the first place of an id takes the sum, the others are marked
                for (int j = lane; j < ntop; j += 32) {
                    int first = j;
                    float sum_j = p[j];
                    if (!lone && id[j] >= 0) { sum_j = 0.0f; search(r, id[j], 0, 1, first, sum_j); }
                    merged(r)[j] = (id[j] >= 0 && first == j) ? sum_j : -1.0f;
                }
            }
        }
        if (lane == 0) {
            r->teacher = k;
            r->weights = sum;
            r->lone = lone;
            r->state = bad ? kBad : (some ? kLive : kPadding);
        }
    }
    // What the loss of a row is made of: loss = T^2 (ln 2 sum_j p_j (log2-weight of the teacher - of the student) + log S - log W).
    // Each lane leaves its part of the sum.
    struct Parked {
        double part[kParked][33];
        float k[kParked], total[kParked], weights[kParked];
        int state[kParked];
    };
    __device__ __forceinline__ void park(Parked* q, int slot, Row* r, float k, float total, const Temp& tv) const {
        const int lane = threadIdx.x & 31;
        const double shift = static_cast<double>(r->teacher) - static_cast<double>(finite_ref(k));
        double s = 0.0;
        for (int j = lane; j < ntop; j += 32) {
            const float p = probs(r)[j];
            if (p != 0.0f)
                s += static_cast<double>(p) *
                     ((static_cast<double>(teacher(r)[j]) - static_cast<double>(logits(r)[j])) * static_cast<double>(tv.c) - shift);
        }
        q->part[slot][lane] = s;
        if (lane == 0) {
            q->k[slot] = k; q->total[slot] = total; q->weights[slot] = r->weights; q->state[slot] = r->state;
        }
    }
    __device__ __forceinline__ Result settle(const Parked* q, int slot, const Temp& tv) const {
        double s4[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int i = 0; i < 32; ++i) s4[i & 3] += q->part[slot][i];
        double s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
        s = kLn2 * s + log_sum(q->total[slot]) - log_sum(q->weights[slot]);
        return Result{static_cast<float>(static_cast<double>(tv.t) * tv.t * s), 1.0f, 0.0f};
    }
    __device__ __forceinline__ float finish_slope(Row*, float, float, const Temp&) const { return 1.0f; }
    __device__ __forceinline__ float coef(Row* r, float, const Temp& tv) const { return r->gy * tv.t; }
    // Where ids are repeated, up to this many labels the label warp joins them while it waits for the others anyway (as part of the
    // gradient's pass it cost 3500 clocks per row at 64 labels); beyond, its time would grow with the square, and all threads
    // share it.
    static constexpr int kMergeAhead = 128;
    // Places of id z: the first of them, and the sum of their probabilities.  Thread `sub` of `g` looks at every g-th group of four.
    __device__ __forceinline__ void search(Row* r, int z, int sub, int g, int& first, float& sum) const {
        const int4* id4 = reinterpret_cast<const int4*>(ids(r));
        const float4* p4 = reinterpret_cast<const float4*>(probs(r));
#pragma unroll 4
        for (int i = sub; i < ntop4 / 4; i += g) {
            const int4 v = id4[i];
            if (v.x == z || v.y == z || v.z == z || v.w == z) {
                const float4 q = p4[i];
                if (v.x == z) { sum += q.x; first = min(first, 4 * i); }
                if (v.y == z) { sum += q.y; first = min(first, 4 * i + 1); }
                if (v.z == z) { sum += q.z; first = min(first, 4 * i + 2); }
                if (v.w == z) { sum += q.w; first = min(first, 4 * i + 3); }
            }
        }
    }
    // Threads that share the search for one label's repetitions, as a power of two (32 at most), `threads` being a multiple of 32.
    __device__ __forceinline__ int sharers(const Row* r, int threads) const {
        int g = 0;
        while (!r->lone && ntop > kMergeAhead && g < 5 && (ntop << (g + 1)) <= threads) ++g;
        return g;
    }
    // Label j's column and weight; an id that occurs again belongs to its first place.  Called by whole warps.
    __device__ __forceinline__ bool label(Row* r, int j, int sub, int g, int& c, float& w, float& x) const {
        const int z = j < ntop ? ids(r)[j] : -1;
        c = z;
        if (r->lone || ntop <= kMergeAhead) {
            if (z < 0) return false;
            w = merged(r)[j];
            x = logits(r)[j];
            return w >= 0.0f || isnan(w);
        }
        int first = j;
        float sum = 0.0f;
        if (z >= 0) {
            search(r, z, sub, g, first, sum);
            x = logits(r)[j];
        }
        for (int o = 1; o < g; o *= 2) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
        }
        w = sum;
        return z >= 0 && first == j && sub == 0;
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
    float* logp;

    // The label warp's pipeline, as above: the token two rows ahead, what belongs to it one row ahead.
    struct Ahead {
        int id;
    };
    struct Flight {
        float x, old, ref, adv;
    };

    __host__ __device__ size_t table_bytes() const { return 0; }
    struct Row : RowHead {
        Flight token;
        int id;
    };
    __host__ __device__ size_t bytes() const { return sizeof(Row); }
    __host__ __device__ __forceinline__ int labels() const { return 1; }

    __device__ __forceinline__ void ahead(Ahead& a, int64_t row) const { a.id = z[row]; }
    __device__ __forceinline__ void depart(Flight& f, const Ahead& a, const float* x, const RowShape& shape, int part, bool all,
                                           int64_t row, int64_t ncol) const {
        f.x = (a.id >= 0 && a.id < ncol && (all || shape.owned(a.id, part))) ? x[a.id] : 0.0f;
        f.old = (old_logp != nullptr) ? old_logp[row] : 0.0f;
        f.ref = (ref_logp != nullptr) ? ref_logp[row] : 0.0f;
        f.adv = (adv != nullptr) ? adv[row] : 0.0f;
    }
    __device__ __forceinline__ void arrive(Row* r, const Flight& f, const Ahead& a, const float*, const RowShape&, int, bool,
                                           int64_t, int64_t ncol, const Temp&, bool, uint16_t*) const {
        if ((threadIdx.x & 31) == 0) {
            r->id = a.id;
            r->state = (a.id >= 0 && a.id < ncol) ? kLive : (a.id == -1 ? kPadding : kBad);
            r->token = f;
        }
    }
    // e^d - d - 1, from d in 64 bits, d rounded and e1 = expm1f of that.  Next to 0 it is d^2 / 2 and e1 - d the difference of two numbers
    // that agree to d / 2, which leaves 2^-24 / d of it (4e-4 at d = 1e-4): up to 1 it is d^2 (1/2 + d (1/6 + d/24 + ...)), nine
    // terms behind the first (what is left out: 4e-9), of which only the sum behind 1/2 is rounded to fp32.  (exp and expm1 in 64 bits
    // for ratio and term: 8192 x 97, loss alone, 8.4 us instead of 7.4.)
    static __device__ __forceinline__ double kl_value(double d, float d32, float e1) {
        if (!(fabsf(d32) <= 1.0f)) return static_cast<double>(e1) - d;
        float s = 1.0f / 39916800.0f;
        s = fmaf(s, d32, 1.0f / 3628800.0f);
        s = fmaf(s, d32, 1.0f / 362880.0f);
        s = fmaf(s, d32, 1.0f / 40320.0f);
        s = fmaf(s, d32, 1.0f / 5040.0f);
        s = fmaf(s, d32, 1.0f / 720.0f);
        s = fmaf(s, d32, 1.0f / 120.0f);
        s = fmaf(s, d32, 1.0f / 24.0f);
        s = fmaf(s, d32, 1.0f / 6.0f);
        return d * d * (0.5 + static_cast<double>(s * d32));
    }
    __device__ __forceinline__ Result finish(const Flight& v, float k, float total, const Temp& tv) const {
        const double l = kLn2 * tv.exponent(v.x, finite_ref(k)) - log_sum(total);
        const float a = v.adv;
        // expf is within a unit in the last place of e^near; what l - old lost in its rounding, up to 1.2e-7 of the ratio, is a factor
        const double gap = l - static_cast<double>(v.old);
        const float near = static_cast<float>(gap);
        const float rho = (old_logp == nullptr) ? 1.0f
                          : expf(near) * (isinf(near) ? 1.0f : 1.0f + static_cast<float>(gap - static_cast<double>(near)));
        float bound = rho;
        if (low != nullptr) bound = fmaxf(bound, 1.0f - __ldg(low));
        if (high != nullptr) bound = fminf(bound, 1.0f + __ldg(high));
        if (isnan(rho)) bound = rho;
        // without an advantage there is no loss, even where rho has overflowed
        const float ra = (a == 0.0f && !isnan(rho)) ? 0.0f : rho * a;
        const float ba = (a == 0.0f) ? 0.0f : bound * a;
        const bool free = !(ra > ba);
        Result out;
        out.loss = free ? -ra : -ba;
        out.slope = free ? -ra : 0.0f;
        const float b = (ref_logp != nullptr && beta != nullptr) ? __ldg(beta) : 0.0f;
        if (b != 0.0f) {          // a coefficient of 0 is no term, even where e^d has overflowed
            const double d = static_cast<double>(v.ref) - l;
            const float d32 = static_cast<float>(d), e1 = expm1f(d32);
            out.loss = static_cast<float>(static_cast<double>(out.loss) + static_cast<double>(b) * kl_value(d, d32, e1));
            out.slope = fmaf(-b, e1, out.slope);
        }
        out.logp = static_cast<float>(l);
        return out;
    }
    // kGrad brings the saved slope; kStep works it out in every warp, which spares a second barrier.
    __device__ __forceinline__ float finish_slope(Row* r, float k, float total, const Temp& tv) const {
        return finish(r->token, k, total, tv).slope;
    }
    __device__ __forceinline__ float coef(Row* r, float slope, const Temp& tv) const {
        return -(r->gy * slope) / tv.t;
    }
    __device__ __forceinline__ int sharers(const Row*, int) const { return 0; }
    __device__ __forceinline__ bool label(Row* r, int j, int, int, int& c, float& w, float& x) const {
        c = r->id;
        w = 1.0f;
        x = r->token.x;
        return j == 0;
    }
    struct Parked {
        Flight token[kParked];
        float k[kParked], total[kParked];
        int state[kParked];
    };
    __device__ __forceinline__ void park(Parked* q, int slot, Row* r, float k, float total, const Temp&) const {
        if ((threadIdx.x & 31) == 0) {
            q->token[slot] = r->token;
            q->k[slot] = k; q->total[slot] = total; q->state[slot] = r->state;
        }
    }
    __device__ __forceinline__ Result settle(const Parked* q, int slot, const Temp& tv) const {
        return finish(q->token[slot], q->k[slot], q->total[slot], tv);
    }
    __device__ __forceinline__ void extra(int64_t row, float v) const {
        if (logp != nullptr) logp[row] = v;
    }
};

// ---- clusters ------------------------------------------------------------------------------------------
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Writes two floats to the same shared-memory variable of CTA `rank` of the cluster.
__device__ __forceinline__ void push_stat(float2* local, uint32_t rank, float a, float b) {
    const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(local));
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(rank));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(a), "f"(b) : "memory");
}
// Raises the same shared-memory flag of CTA `rank`.
__device__ __forceinline__ void push_flag(int* local, uint32_t rank) {
    const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(local));
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(rank));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(1) : "memory");
}
// `bytes` (a multiple of 16, both addresses on 16-byte boundaries) into shared memory; the barrier is credited as they land.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// The way back; returns when the copy has read its source (the bytes land in order for whoever waits for the kernel).
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.commit_group;\n cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// Joins `n` pairs (reference, sum of exponentials against it); every warp does the same in the same order.
__device__ __forceinline__ void join(const float2* stat, int n, float& k, float& total) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY;
    for (int i = lane; i < n; i += 32) m = fmaxf(m, stat[i].x);
    k = warp_max(m);
    const float kf = finite_ref(k);
    float s = 0.0f;
    for (int i = lane; i < n; i += 32) s += stat[i].y * exp2_approx(stat[i].x - kf);
    total = warp_sum(s);
}

// Losses and statistics of `n` parked rows first, first + step, ...: a lane each.
template <class L>
__device__ __forceinline__ void settle_rows(const RowParams& p, const L& loss, const typename L::Parked* q, int n, int64_t first,
                                            int64_t step, const Temp& tv) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    if (lane < n) {
        const int64_t row = first + lane * step;
        Result res = loss.settle(q, lane, tv);
        const int state = q->state[lane];
        if (state == kPadding) res.loss = res.slope = res.logp = 0.0f;
        if (state == kBad) res.loss = res.slope = res.logp = nanf("");
        p.y[row] = res.loss;
        loss.extra(row, res.logp);
        if (p.ps != nullptr) {
            p.ps[3 * row + 0] = q->k[lane];
            p.ps[3 * row + 1] = q->total[lane];
            p.ps[3 * row + 2] = res.slope;
        }
        if (state == kBad) *p.flag = 1;
    }
    __syncwarp();
}

template <class L, int T, int MODE>
__global__ void __launch_bounds__(T + 32, T == 64 ? 10 : T == 128 ? 6 : 1)
row_stream_kernel(const RowParams p, const L loss) {
    constexpr int W = T / 32;
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ float2 stat[2][kMaxParts * W];
    __shared__ float loose_sh[8];
    __shared__ uint64_t full;
    __shared__ int abort_flag;
    using Row = typename L::Row;
    float4* stage = reinterpret_cast<float4*>(dyn);                      // this part of the row
    uint8_t* rows = dyn + p.per * sizeof(float4);                        // [2] label buffers
    const size_t row_bytes = loss.bytes();
    typename L::Parked* parked = reinterpret_cast<typename L::Parked*>(rows + 2 * row_bytes);
    const int ncol = static_cast<int>(p.ncol);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
    const bool labels = warp == W;                                       // the warp that prepares labels
    const int part = blockIdx.x % p.parts;
    const int64_t first = blockIdx.x / p.parts, step = gridDim.x / p.parts;
    const Temp tv(p.temp);
    const bool cluster = MODE != kGrad && p.parts > 1;
    if (tid == 0) {
        mbar_init(smem_u32(&full), 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (cluster) { cluster_arrive(); cluster_wait(); } else { __syncthreads(); }

    auto fetch = [&](int64_t row) {
        const float* x = p.x + row * p.ncol;
        const RowShape shape(x, ncol, p.per);
        const uint32_t bytes = static_cast<uint32_t>(shape.count(part)) * 16u;
        mbar_expect_tx(smem_u32(&full), bytes);
        if (bytes > 0)
            bulk_load(stage, reinterpret_cast<const float4*>(x + shape.head) + shape.begin(part), bytes, smem_u32(&full));
    };

    // A wait ran out in a CTA of this row: from here on its rows have no logits, whatever the barriers' phases say of them.  They become NaN
    // (padding rows stay 0), and the CTAs keep in step.  Whoever asks behind the row's barrier gets the same answer in all of them.
    auto lost = [&] { return *static_cast<volatile int*>(&abort_flag) != 0; };

    // The label warp's three stages; every part of a row needs all labels' logits (kStep: the policy's slope hangs on them)
    // or its own (kGrad).
    typename L::Ahead ids, ids_next;
    typename L::Flight flight;
    float gy_next = 1.0f, ps_next = 0.0f;
    auto depart = [&](int64_t row) {
        const float* x = p.x + row * p.ncol;
        const RowShape shape(x, ncol, p.per);
        loss.depart(flight, ids, x, shape, part, MODE != kGrad, row, p.ncol);
        if (MODE != kLoss && p.gy != nullptr) gy_next = p.gy[row];
        if (MODE == kGrad && lane < 3) ps_next = p.ps[3 * row + lane];
    };
    auto arrive = [&](int64_t row, int buf) {
        const float* x = p.x + row * p.ncol;
        const RowShape shape(x, ncol, p.per);
        Row* r = reinterpret_cast<Row*>(rows + buf * row_bytes);
        if (lane == 0) r->gy = gy_next;
        if (MODE == kGrad && lane < 3) r->stat[lane] = ps_next;
        loss.arrive(r, flight, ids, x, shape, part, MODE != kGrad, row, p.ncol, tv, MODE != kLoss, nullptr);
    };

    if (first < p.nrow) {
        if (labels) {
            loss.ahead(ids, first);
            depart(first);
            arrive(first, 0);
            if (first + step < p.nrow) loss.ahead(ids, first + step);
        } else if (tid == 0) {
            fetch(first);
        }
    }

    int buf = 0, waiting = 0;
    uint32_t phase = 0;
    for (int64_t row = first; row < p.nrow; row += step, buf ^= 1, phase ^= 1u) {
        const int64_t next = row + step;
        Row* r = reinterpret_cast<Row*>(rows + buf * row_bytes);
        const float* x = p.x + row * p.ncol;
        const RowShape shape(x, ncol, p.per);
        const int n = shape.count(part);           // 16-byte pieces of this part
        const bool loose = part == 0 && tid < shape.loose;
        float lv = -INFINITY;
        if (!labels) {
            if (loose) lv = x[shape.loose_col(tid)];
            if (!mbar_wait(smem_u32(&full), phase, &abort_flag, p.status, 40) && cluster)
                for (int i = 0; i < p.parts; ++i) push_flag(&abort_flag, i);
            if (MODE != kGrad) {
                float m = lv;
#pragma unroll 4
                for (int i = tid; i < n; i += T) m = max4(stage[i], m);
                const float k = reference(warp_max(m), tv.c);
                const float kf = finite_ref(k);
                float s = weight(lv, kf, tv.c);
#pragma unroll 4
                for (int i = tid; i < n; i += T) s += weight4(stage[i], kf, tv.c);
                s = warp_sum(s);
                if (cluster) {
                    if (lane < p.parts) push_stat(&stat[buf][part * W + warp], lane, k, s);
                } else if (lane == 0) {
                    stat[buf][warp] = make_float2(k, s);
                }
                __syncwarp();
            }
        }
        // The one barrier of all parts: the row's statistics and labels are there, and the labels' logits have been read
        // everywhere, so that the gradient may be written over them.  The list of statistics and the label buffer are used
        // in turn: a CTA that fills one again has passed the next row's barrier, where everybody is done with it.
        if (cluster) { cluster_arrive(); cluster_wait(); } else { __syncthreads(); }

        if (labels) {
            if (next < p.nrow) {
                depart(next);
                if (next + step < p.nrow) loss.ahead(ids_next, next + step);
            }
            if (MODE != kGrad && part == 0) {
                float k, total;
                join(stat[buf], p.parts * W, k, total);
                if (lost()) total = nanf("");
                loss.park(parked, waiting, r, k, total, tv);
                if (++waiting == kParked || next >= p.nrow) {
                    settle_rows(p, loss, parked, waiting, row - (waiting - 1) * step, step, tv);
                    waiting = 0;
                }
            } else if (MODE == kGrad && part == 0 && lane == 0 && r->state == kBad) {
                *p.flag = 1;
            }
            if (next < p.nrow) {
                arrive(next, buf ^ 1);
                ids = ids_next;
            }
        } else if (MODE == kLoss) {
            if (tid == 0 && next < p.nrow && !lost()) fetch(next);
        } else {
            float k, total, slope;
            if (MODE == kGrad) {
                k = r->stat[0]; total = r->stat[1]; slope = r->stat[2];
            } else {
                join(stat[buf], p.parts * W, k, total);
                slope = loss.finish_slope(r, k, total, tv);
            }
            const float kf = finite_ref(k);
            const float coef = loss.coef(r, slope, tv);
            const float f = coef / total;                                   // gradient = f * 2^(x c - k)
            const int state = r->state;
            float* gx = p.gx + row * p.ncol;
            if (state == kLive) {
#pragma unroll 4
                for (int i = tid; i < n; i += T) {
                    const float4 v = stage[i];
                    stage[i] = make_float4(weight(v.x, kf, tv.c) * f, weight(v.y, kf, tv.c) * f, weight(v.z, kf, tv.c) * f,
                                           weight(v.w, kf, tv.c) * f);
                }
                if (loose) loose_sh[tid] = weight(lv, kf, tv.c) * f;
                asm volatile("bar.sync 1, %0;" ::"n"(T) : "memory");
                // the labels' columns, over what has just been written there
                const int g = loss.sharers(r, T);
                for (int j0 = 0; j0 < loss.labels(); j0 += T >> g) {
                    const int j = j0 + (tid >> g);
                    int c;
                    float w, xv;
                    if (loss.label(r, j, tid & ((1 << g) - 1), 1 << g, c, w, xv) && shape.owned(c, part)) {
                        const float v = weight(xv, kf, tv.c) * f - coef * w;
                        const int q = (c - shape.head) >> 2;
                        if (c < shape.head) loose_sh[c] = v;
                        else if (q >= shape.quads) loose_sh[c - 4 * shape.quads] = v;
                        else reinterpret_cast<float*>(stage)[c - shape.head - 4 * shape.begin(part)] = v;
                    }
                }
            } else {
                // a padding row's logits are not looked at; a bad label poisons the row
                const float fixed = state == kPadding ? 0.0f : nanf("");
                for (int i = tid; i < n; i += T) stage[i] = make_float4(fixed, fixed, fixed, fixed);
                if (loose) loose_sh[tid] = fixed;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the bulk copy reads what this thread wrote
            asm volatile("bar.sync 1, %0;" ::"n"(T) : "memory");
            if (loose) gx[shape.loose_col(tid)] = loose_sh[tid];
            float* out = gx + shape.head + 4 * shape.begin(part);
            if (lost()) {
                // a copy may still land in the stage: what goes out does not come from there, and nothing more is fetched
                const float fixed = state == kPadding ? 0.0f : nanf("");
                for (int i = tid; i < 4 * n; i += T) out[i] = fixed;
            } else if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(gx)) & 15) == 0) {
                if (tid == 0) {
                    if (n > 0) bulk_store(out, stage, static_cast<uint32_t>(n) * 16u);
                    if (next < p.nrow) fetch(next);
                }
            } else {
                // the gradient's rows lie on another 4-byte phase than the logits'
                for (int i = tid; i < 4 * n; i += T) out[i] = reinterpret_cast<const float*>(stage)[i];
                asm volatile("bar.sync 1, %0;" ::"n"(T) : "memory");
                if (tid == 0 && next < p.nrow) fetch(next);
            }
        }
    }
    __syncthreads();
    if (abort_flag) {          // copies may still be on their way into this CTA's memory
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
}

// ---- short rows: a warp each -------------------------------------------------------------------------------
// A row of up to 32 E columns lies in the registers of one warp, column lane + 32 i in value i: loads and stores of 128 bytes
// whatever the row's alignment, no barrier beyond the warp, and the label's work between the row's loads and their use.  Beyond the
// smallest E a row has more than 16 E columns (run_short), so that half of the values need no bound.
template <class L, int E, int MODE>
__global__ void __launch_bounds__(kShortWarps * 32, E <= 16 ? 8 : E <= 32 ? 6 : E <= 64 ? 4 : 3)
row_short_kernel(const RowParams p, const L loss) {
    extern __shared__ __align__(16) uint8_t dyn[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const size_t row_bytes = loss.bytes();
    typename L::Row* r = reinterpret_cast<typename L::Row*>(dyn + warp * row_bytes);
    typename L::Parked* parked = reinterpret_cast<typename L::Parked*>(dyn + kShortWarps * row_bytes) + warp;
    const int ncol = static_cast<int>(p.ncol);
    uint16_t* table = reinterpret_cast<uint16_t*>(dyn + kShortWarps * (row_bytes + (MODE == kGrad ? 0 : sizeof(typename L::Parked))) +
                                                  warp * loss.table_bytes());
    const int rest = ncol - lane;
    auto inside = [&](int i) { return (E > kShortLeast && 2 * i < E) || 32 * i < rest; };
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kShortWarps + warp, step = static_cast<int64_t>(gridDim.x) * kShortWarps;
    const Temp tv(p.temp);
    typename L::Ahead ids;
    if (first < p.nrow) loss.ahead(ids, first);
    int waiting = 0;
    for (int64_t row = first; row < p.nrow; row += step) {
        const int64_t next = row + step;
        const float* x = p.x + row * p.ncol;
        float v[E];
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = inside(i) ? __ldcs(x + lane + 32 * i) : -INFINITY;
        const RowShape shape(x, ncol, ncol);                 // one part
        typename L::Flight flight;
        loss.depart(flight, ids, x, shape, 0, true, row, p.ncol);
        float k = 0.0f, total = 0.0f, slope = 0.0f;
        if (MODE == kGrad) { k = p.ps[3 * row]; total = p.ps[3 * row + 1]; slope = p.ps[3 * row + 2]; }
        if (lane == 0) r->gy = (MODE != kLoss && p.gy != nullptr) ? p.gy[row] : 1.0f;
        loss.arrive(r, flight, ids, x, shape, 0, true, row, p.ncol, tv, MODE != kLoss, table);
        if (next < p.nrow) loss.ahead(ids, next);
        __syncwarp();
        if (MODE != kGrad) {
            float m = v[0];
#pragma unroll
            for (int i = 1; i < E; ++i) m = fmaxf(m, v[i]);
            k = reference(warp_max(fmaxf(m, -INFINITY)), tv.c);
            const float kf = finite_ref(k);
            float part[4] = {};
#pragma unroll
            for (int i = 0; i < E; ++i) {
                v[i] = weight(v[i], kf, tv.c);               // all that kStep needs of it from here on
                part[i & 3] += v[i];
            }
            total = warp_sum((part[0] + part[1]) + (part[2] + part[3]));
            if (MODE == kStep) slope = loss.finish_slope(r, k, total, tv);
        }
        const int state = r->state;
        if (MODE != kLoss) {
            const float kf = finite_ref(k);
            const float coef = loss.coef(r, slope, tv);
            const float f = coef / total;                                   // gradient = f * 2^(x c - k)
            float* gx = p.gx + row * p.ncol;
            if (state == kLive) {
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (inside(i)) gx[lane + 32 * i] = (MODE == kStep ? v[i] : weight(v[i], kf, tv.c)) * f;
                __syncwarp();
                // the labels' columns, over what has just been written there
                for (int j0 = 0; j0 < loss.labels(); j0 += 32) {
                    int c;
                    float w, xv;
                    if (loss.label(r, j0 + lane, 0, 1, c, w, xv)) gx[c] = weight(xv, kf, tv.c) * f - coef * w;
                }
            } else {
                // a padding row's logits are not looked at; a bad label poisons the row
                const float fixed = state == kPadding ? 0.0f : nanf("");
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (inside(i)) gx[lane + 32 * i] = fixed;
            }
        }
        if (MODE != kGrad) {
            loss.park(parked, waiting, r, k, total, tv);
            if (++waiting == kParked || next >= p.nrow) {
                settle_rows(p, loss, parked, waiting, row - (waiting - 1) * step, step, tv);
                waiting = 0;
            }
        } else if (lane == 0 && state == kBad) {
            *p.flag = 1;
        }
        __syncwarp();                                        // the label buffer is filled again
    }
}

// ---- rows of any length, loss and statistics alone -------------------------------------------------------
// A thread keeps a running reference k and sum s over its pieces of the row, four 16-byte loads at a time: the maximum of
// the sixteen values first, one rescaling of s if it rose, then sixteen exponentials.
template <class L>
__global__ void __launch_bounds__(512 + 32)
row_loss_wide_kernel(const RowParams p, const L loss) {
    constexpr int T = 512, W = T / 32;
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ float2 stat[kMaxParts * W];
    const int64_t row = blockIdx.x / p.parts;
    const int part = blockIdx.x % p.parts;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Temp tv(p.temp);
    const int ncol = static_cast<int>(p.ncol);
    const float* x = p.x + row * p.ncol;
    const RowShape shape(x, ncol, p.per);
    typename L::Row* r = reinterpret_cast<typename L::Row*>(dyn);
    if (p.parts > 1) { cluster_arrive(); cluster_wait(); }
    if (warp == W) {
        if (part == 0) {
            typename L::Ahead ids;
            typename L::Flight flight;
            loss.ahead(ids, row);
            loss.depart(flight, ids, x, shape, part, true, row, p.ncol);
            loss.arrive(r, flight, ids, x, shape, part, true, row, p.ncol, tv, false, nullptr);
        }
    } else {
        const float4* xq = reinterpret_cast<const float4*>(x + shape.head);
        const int q_end = shape.begin(part) + shape.count(part);
        float k = -INFINITY, s = 0.0f;
        if (part == 0 && static_cast<int>(threadIdx.x) < shape.loose) {
            const float v = x[shape.loose_col(threadIdx.x)];
            k = reference(v, tv.c);
            s = weight(v, finite_ref(k), tv.c);
        }
        for (int q0 = shape.begin(part) + threadIdx.x; q0 < q_end; q0 += 4 * T) {
            float4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                v[u] = (q0 + u * T < q_end) ? __ldcs(xq + q0 + u * T)
                                            : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            float m = -INFINITY;
#pragma unroll
            for (int u = 0; u < 4; ++u) m = max4(v[u], m);
            const float k1 = reference(m, tv.c);
            if (k1 > k) { s *= exp2_approx(k - k1); k = k1; }
#pragma unroll
            for (int u = 0; u < 4; ++u) s += weight4(v[u], finite_ref(k), tv.c);
        }
        const float kw = warp_max(k);
        s = warp_sum(s * exp2_approx(k - finite_ref(kw)));
        if (p.parts > 1) {
            if (lane == 0) push_stat(&stat[part * W + warp], 0, kw, s);
        } else if (lane == 0) {
            stat[warp] = make_float2(kw, s);
        }
        __syncwarp();
    }
    if (p.parts > 1) { cluster_arrive(); cluster_wait(); } else { __syncthreads(); }
    if (warp == W && part == 0) {
        float k, total;
        join(stat, p.parts * W, k, total);
        __shared__ typename L::Parked parked;
        loss.park(&parked, 0, r, k, total, tv);
        settle_rows(p, loss, &parked, 1, row, 1, tv);
    }
}

// ---- host side -----------------------------------------------------------------------------------------------
constexpr int64_t kPart = 12800;      // columns of a part at most, where a row has several: 50 KB, four parts to an SM
constexpr int64_t kPartOne = 16384;   // columns from which on a part is a matter for 256 threads
// Columns that a warp takes by itself, with kShortLabels labels at most.  Beyond 2048 kGrad alone loses by it where warps have several
// rows (8192 x 4090, 64 labels: 56 us in the stream, 66; 1000 x 4000, both calls: 23 us and 19), while loss and gradient in one still gain (policy, 8192 x 2500: 47 us
// and 39, 8192 x 4090: 60 and 53; 64 labels 58 and 50, 69 and 68; 200 labels, 8192 x 2500: 105 and 67).
constexpr int64_t kShort = 4096, kShortGrad = 2048;
constexpr int kShortLabels = 256;
constexpr size_t kSmemMost = 220 * 1024;

// Clusters (or, for `parts` = 1, CTAs) of a kernel that are resident on the device at once: the size of a persistent grid.
// Asked once per kernel, cluster size and shared-memory size.
int resident_clusters(const void* kernel, int threads, int parts, size_t smem, int sm_count, int* out) {
    struct Known { const void* kernel; int device, parts; size_t smem; int clusters; };
    static std::mutex mu;
    static Known known[64];          // the first of them; what does not fit any more is asked again
    static int count = 0;
    int device = 0;
    KAI_CUDA(cudaGetDevice(&device));
    {
        std::lock_guard<std::mutex> lock(mu);
        for (int i = 0; i < count; ++i) {
            const Known& k = known[i];
            if (k.kernel == kernel && k.device == device && k.parts == parts && k.smem == smem) { *out = k.clusters; return KAI_OK; }
        }
    }
    KAI_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemMost)));
    int clusters = 0;
    if (parts == 1) {
        int per_sm = 0;
        KAI_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem));
        clusters = per_sm * sm_count;
    } else {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(parts));
        cfg.blockDim = dim3(static_cast<unsigned>(threads));
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = static_cast<unsigned>(parts);
        at[0].val.clusterDim.y = 1;
        at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        KAI_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg));
    }
    if (clusters < 1) return fail(KAI_E_TOO_LARGE, "row losses: %zu bytes of shared memory do not fit", smem);
    *out = clusters;
    std::lock_guard<std::mutex> lock(mu);
    if (count < 64) known[count++] = Known{kernel, device, parts, smem, clusters};
    return KAI_OK;
}

template <class L>
int launch_rows(void (*kernel)(const RowParams, const L), const char* name, const RowParams& p, const L& loss, int64_t groups,
                int threads, bool cluster, size_t smem, cudaStream_t s) {
    if (groups * p.parts >= (int64_t(1) << 31)) return fail(KAI_E_TOO_LARGE, "%s: too many rows for one launch", name);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(groups * p.parts));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
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

template <class L, int MODE>
size_t stream_smem(int64_t ncol, int parts, const L& loss) {
    return ((ncol >> 2) + parts - 1) / parts * sizeof(float4) + 2 * loss.bytes() + (MODE == kGrad ? 0 : sizeof(typename L::Parked));
}

template <class L, int T, int MODE>
int launch_stream(DeviceState* st, const RowParams& p0, const L& loss, cudaStream_t s) {
    RowParams p = p0;
    auto kernel = row_stream_kernel<L, T, MODE>;
    p.status = st->status_dev;
    p.per = static_cast<int>(((p.ncol >> 2) + p.parts - 1) / p.parts);
    const size_t smem = stream_smem<L, MODE>(p.ncol, p.parts, loss);
    int clusters = 0;
    const int group = MODE == kGrad ? 1 : p.parts;
    KAI_TRY(resident_clusters(reinterpret_cast<const void*>(kernel), T + 32, group, smem, st->sm_count, &clusters));
    if (MODE == kGrad) clusters = clusters / p.parts < 1 ? 1 : clusters / p.parts;
    const int64_t groups = p.nrow < clusters ? p.nrow : clusters;
    return launch_rows(kernel, "row_stream_kernel", p, loss, groups, T + 32, MODE != kGrad, smem, s);
}

template <class L>
int run_wide(DeviceState* st, RowParams p, const L& loss, cudaStream_t s) {
    p.parts = kMaxParts;
    p.per = static_cast<int>(((p.ncol >> 2) + kMaxParts - 1) / kMaxParts);
    (void)st;
    return launch_rows(row_loss_wide_kernel<L>, "row_loss_wide_kernel", p, loss, p.nrow, 512 + 32, true, loss.bytes(), s);
}

// Parts of a row: as many as hold it at kPart columns, and more while the rows alone do not fill the SMs and a part keeps 1024
// columns.
int row_parts(int64_t nrow, int64_t ncol, int64_t most, int sm_count) {
    int64_t parts = 1;
    while (parts < most && parts * kPart < ncol) parts *= 2;
    while (parts * 2 <= most && nrow * parts < 2 * static_cast<int64_t>(sm_count) && ncol >= parts * 2 * 1024) parts *= 2;
    return static_cast<int>(parts);
}

// Threads of a CTA: 64 for many short rows (a part of 2048 columns at most; only rows with more labels than row_short_kernel takes get
// here, so none of the policy loss: 8192 x 250, 200 labels, loss 29 us, with 128 threads 43), 256 for parts beyond kPartOne and where there are too
// few parts to give every SM four, 128 otherwise.
template <class L, int MODE>
int launch_threads(DeviceState* st, const RowParams& p, const L& loss, cudaStream_t s) {
    const int64_t each = (p.ncol + p.parts - 1) / p.parts, ctas = p.nrow * p.parts;
    if (each > kPartOne || ctas < 4 * static_cast<int64_t>(st->sm_count)) return launch_stream<L, 256, MODE>(st, p, loss, s);
    if constexpr (std::is_same_v<L, Distill>)
        if (each <= 2048) return launch_stream<L, 64, MODE>(st, p, loss, s);
    return launch_stream<L, 128, MODE>(st, p, loss, s);
}

// Rows that lie in a warp's registers.
template <class L, int E, int MODE>
int launch_short(DeviceState* st, const RowParams& p, const L& loss, cudaStream_t s) {
    auto kernel = row_short_kernel<L, E, MODE>;
    const size_t smem = kShortWarps * (loss.bytes() + (MODE == kGrad ? 0 : sizeof(typename L::Parked)) +
                                       (MODE == kLoss ? 0 : loss.table_bytes()));
    int blocks = 0;
    KAI_TRY(resident_clusters(reinterpret_cast<const void*>(kernel), kShortWarps * 32, 1, smem, st->sm_count, &blocks));
    const int64_t groups = (p.nrow + kShortWarps - 1) / kShortWarps;
    return launch_rows(kernel, "row_short_kernel", p, loss, groups < blocks ? groups : blocks, kShortWarps * 32, false, smem, s);
}
template <class L, int MODE>
bool takes_short(const RowParams& p, const L& loss, int sm_count) {
    const bool several = p.nrow > 3 * kShortWarps * static_cast<int64_t>(sm_count);       // at 168 registers
    return p.ncol <= (MODE == kGrad && several ? kShortGrad : kShort) && loss.labels() <= kShortLabels;
}
template <class L, int MODE>
int run_short(DeviceState* st, RowParams p, L loss, cudaStream_t s) {
    p.parts = 1;
    if (p.ncol <= 32 * kShortLeast) return launch_short<L, kShortLeast, MODE>(st, p, loss, s);
    if (p.ncol <= 512) return launch_short<L, 16, MODE>(st, p, loss, s);
    if (p.ncol <= 1024) return launch_short<L, 32, MODE>(st, p, loss, s);
    if (p.ncol <= 2048) return launch_short<L, 64, MODE>(st, p, loss, s);
    return launch_short<L, 128, MODE>(st, p, loss, s);
}

// What every call with bounded waits answers while an expired one has not been cleared.
int answer(const DeviceState* st) {
    if (st->status_host[0] != 0)
        return fail(KAI_E_DEVICE_WAIT, "a device-side wait ran out earlier (where=%d)", st->status_host[1]);
    return KAI_OK;
}

template <class L>
int launch_grad(DeviceState* st, RowParams p, const L& loss, cudaStream_t s) {
    p.flag = st->flag_dev + 2;
    if (takes_short<L, kGrad>(p, loss, st->sm_count)) return run_short<L, kGrad>(st, p, loss, s);
    p.parts = row_parts(p.nrow, p.ncol, int64_t(1) << 20, st->sm_count);
    return launch_threads<L, kGrad>(st, p, loss, s);
}

template <class L, int MODE>
int launch_any(DeviceState* st, RowParams p, const L& loss, cudaStream_t s) {
    p.flag = st->flag_dev + 2;
    if (takes_short<L, MODE>(p, loss, st->sm_count)) return run_short<L, MODE>(st, p, loss, s);
    if (stream_smem<L, MODE>(p.ncol, kMaxParts, loss) > kSmemMost) {
        if (MODE == kLoss) return run_wide(st, p, loss, s);
        KAI_TRY(ensure_aux(st, p.nrow * 3 * 4));
        p.ps = static_cast<float*>(st->aux);
        KAI_TRY(run_wide(st, p, loss, s));
        return launch_grad(st, p, loss, s);
    }
    p.parts = row_parts(p.nrow, p.ncol, kMaxParts, st->sm_count);
    return launch_threads<L, MODE>(st, p, loss, s);
}

template <class L>
int run_grad(DeviceState* st, const RowParams& p, const L& loss, cudaStream_t s) {
    KAI_TRY(launch_grad(st, p, loss, s));
    return answer(st);
}
template <class L, int MODE>
int run_rows(DeviceState* st, const RowParams& p, const L& loss, cudaStream_t s) {
    KAI_TRY((launch_any<L, MODE>(st, p, loss, s)));
    return answer(st);
}

RowParams row_params(const float* x, int64_t nrow, int64_t ncol, const float* temp) {
    RowParams p{};
    p.x = x;
    p.nrow = nrow;
    p.ncol = ncol;
    p.temp = temp;
    p.parts = 1;
    return p;
}
Distill distill(const int* idx, const float* t, int64_t ntop) {
    const int ntop4 = static_cast<int>((ntop + 3) / 4 * 4);
    int bits = 3;
    while ((2 << bits) <= 2 * ntop4) ++bits;
    return Distill{idx, t, static_cast<int>(ntop), ntop4, bits};
}

}  // namespace

int loss_distill(DeviceState* st, float* y, float* ps, const float* x, const int* idx, const float* t, int64_t nrow,
                 int64_t ncol, int64_t ntop, const float* temp, cudaStream_t s) {
    RowParams p = row_params(x, nrow, ncol, temp);
    p.y = y; p.ps = ps;
    return run_rows<Distill, kLoss>(st, p, distill(idx, t, ntop), s);
}
int loss_distill_backward(DeviceState* st, float* gx, const float* gy, const float* x, const float* ps, const int* idx,
                          const float* t, int64_t nrow, int64_t ncol, int64_t ntop, const float* temp, cudaStream_t s) {
    RowParams p = row_params(x, nrow, ncol, temp);
    p.gx = gx; p.gy = gy; p.ps = const_cast<float*>(ps);
    return run_grad(st, p, distill(idx, t, ntop), s);
}
int loss_distill_step(DeviceState* st, float* y, float* gx, const float* gy, const float* x, const int* idx,
                      const float* t, int64_t nrow, int64_t ncol, int64_t ntop, const float* temp, cudaStream_t s) {
    RowParams p = row_params(x, nrow, ncol, temp);
    p.y = y; p.gx = gx; p.gy = gy;
    return run_rows<Distill, kStep>(st, p, distill(idx, t, ntop), s);
}

int loss_policy(DeviceState* st, float* y, float* logp, float* ps, const float* x, const int* z, const float* old_logp,
                const float* ref_logp, const float* adv, int64_t nrow, int64_t ncol, const float* low, const float* high,
                const float* beta, const float* temp, cudaStream_t s) {
    RowParams p = row_params(x, nrow, ncol, temp);
    p.y = y; p.ps = ps;
    return run_rows<Policy, kLoss>(st, p, Policy{z, old_logp, ref_logp, adv, low, high, beta, logp}, s);
}
int loss_policy_backward(DeviceState* st, float* gx, const float* gy, const float* x, const float* ps, const int* z,
                         int64_t nrow, int64_t ncol, const float* temp, cudaStream_t s) {
    RowParams p = row_params(x, nrow, ncol, temp);
    p.gx = gx; p.gy = gy; p.ps = const_cast<float*>(ps);
    return run_grad(st, p, Policy{z, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr}, s);
}
int loss_policy_step(DeviceState* st, float* y, float* logp, float* gx, const float* gy, const float* x, const int* z,
                     const float* old_logp, const float* ref_logp, const float* adv, int64_t nrow, int64_t ncol,
                     const float* low, const float* high, const float* beta, const float* temp, cudaStream_t s) {
    RowParams p = row_params(x, nrow, ncol, temp);
    p.y = y; p.gx = gx; p.gy = gy;
    return run_rows<Policy, kStep>(st, p, Policy{z, old_logp, ref_logp, adv, low, high, beta, logp}, s);
}

}  // namespace kai
