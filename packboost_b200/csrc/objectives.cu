// Losses on the scores of rows with their gradients: preferences between two rows, choices among the
// rows of a group, and a clipped policy over groups (include/packboost_b200.h has the formulas).
//
// Sums over a row's pairs, over a group and over the whole table are taken in a fixed order, so a
// result does not change from run to run.  The log of a group's sum of exponentials comes from 64 bits:
// whether a policy's ratio is beyond its border must not hang on the rounding of a sum over a whole era, and
// with a reference near the policy the difference of the two log-probabilities is all there is.
//
// Groups of rows in order are bound neither by memory nor by the instructions that the SMs issue, but by waiting: 32 rows of a policy
// are 640 bytes and some 190 instructions of a warp, half of the time at four a cycle; 2.2 to 2.5 are issued.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace pb {

namespace {

// ---- scores of any type ---------------------------------------------------------------------------

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ double warp_sum(double v) {
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
    for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
    return v;
}

// The sum over the CTA, the same in every thread.  `scratch` holds a value per warp.
template <int THREADS>
__device__ __forceinline__ double cta_sum(double v, double* scratch) {
    v = warp_sum(v);
    __syncthreads();  // (the scratch may still be read from the call before)
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    const int k = threadIdx.x & 31;
    return warp_sum(k < THREADS / 32 ? scratch[k] : 0.0);
}

// ---- launches that overlap, and the totals of an evaluation ------------------------------------------
//
// The kernels of one evaluation write different rows, so the next may start while one runs (its CTAs fill SMs that the
// last of this one's leave idle); each waits for the one before it at its end, so that the last one's end is
// everyone's.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// What a CTA leaves of the totals.  The CTA that leaves the last of them adds them up, in the order of their slots, and
// resets the count: a launch only for that would take longer than the sums.
struct Part {
    double loss, kl, clipped;
};
struct Totals {
    unsigned* ticket;  // null: not wanted
    Part* parts;
    int n_parts;
    double scale;
    float *loss, *kl;
    int64_t* clipped;
};

// (acquire and release: what the count is for)
__device__ __forceinline__ void fence() { asm volatile("fence.acq_rel.gpu;" ::: "memory"); }

template <int THREADS>
__device__ __forceinline__ void put_totals(const Totals& out, int slot, double loss, double kl, int clipped, bool policy) {
    if (!out.ticket) return;
    constexpr int kWarps = THREADS / 32;
    __shared__ Part s_part[kWarps];
    __shared__ int s_last;
    const int lane = threadIdx.x & 31;
    auto sum_in_warp = [&](Part& v) {
        v.loss = warp_sum(v.loss);
        if (policy) {
            v.kl = warp_sum(v.kl);
            v.clipped = warp_sum(v.clipped);
        }
    };
    Part mine{loss, kl, 0.0};
    mine.clipped = (double)clipped;
    sum_in_warp(mine);
    if (lane == 0) s_part[threadIdx.x >> 5] = mine;
    __syncthreads();
    if (threadIdx.x < 32) {
        mine = lane < kWarps ? s_part[lane] : Part{0.0, 0.0, 0.0};
        sum_in_warp(mine);
    }
    if (out.n_parts > 1) {
        if (threadIdx.x == 0) {
            out.parts[slot] = mine;
            fence();  // the part is visible before the ticket is
            s_last = atomicAdd(out.ticket, 1u) == (unsigned)out.n_parts - 1u;
            fence();
        }
        __syncthreads();
        if (!s_last) return;
        mine = Part{0.0, 0.0, 0.0};
        for (int i = threadIdx.x; i < out.n_parts; i += THREADS) {
            mine.loss += __ldcg(&out.parts[i].loss);
            if (policy) {
                mine.kl += __ldcg(&out.parts[i].kl);
                mine.clipped += __ldcg(&out.parts[i].clipped);
            }
        }
        sum_in_warp(mine);
        if (lane == 0) s_part[threadIdx.x >> 5] = mine;
        __syncthreads();
        if (threadIdx.x < 32) {
            mine = lane < kWarps ? s_part[lane] : Part{0.0, 0.0, 0.0};
            sum_in_warp(mine);
        }
    }
    if (threadIdx.x == 0) {
        if (out.n_parts > 1) *out.ticket = 0u;
        if (out.loss) *out.loss = (float)(mine.loss * out.scale);
        if (out.kl) *out.kl = (float)(mine.kl * out.scale);
        if (out.clipped) *out.clipped = (int64_t)mine.clipped;
    }
}

// ---- pairs ---------------------------------------------------------------------------------------

struct PairArgs {
    pb_pairs p;
    float beta, beta_log2e, smoothing, half_tau;  // half_tau: 1 / (2 beta)
    double factor;                                // of the sum of a row's terms: scale and what the terms leave out (32 bits need not hold it)
    double* sums;                                 // [n_chunks]
    unsigned* counts;                             // [n_split], 0 before and after
};

__device__ __forceinline__ float exp2_of(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float reciprocal(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Derivative with respect to d, without the factor 2 (squared) or beta, of a pair whose (reference-corrected)
// score difference is d.  Of softplus(-z) + e z it is e - sigmoid(-z); the units' 2^x and 1 / x (2 and 1 ulp) are off
// by less than 4 roundings of the slope's range.
template <bool SQUARED>
__device__ __forceinline__ float pair_slope(const PairArgs& a, float d) {
    if (SQUARED) return d - a.half_tau;
    return a.smoothing - reciprocal(1.f + exp2_of(d * a.beta_log2e));
}

// The same pair's loss, from its slope.  With h the smaller of q = sigmoid(-z) and 1 - q, softplus(-z) is max(-z, 0) -
// log(1 - h), and -log(1 - h) = 2 atanh(h / (2 - h)), an argument of at most 1/3; the term after the last one kept is
// s^14 / 15 of the sum, below 2^-26.
template <bool SQUARED>
__device__ __forceinline__ float pair_loss(const PairArgs& a, float d, float slope) {
    if (SQUARED) return slope * slope;
    const float z = a.beta * d, q = reciprocal(1.f + exp2_of(d * a.beta_log2e)), h = fminf(q, 1.f - q);
    const float s = h * reciprocal(2.f - h), s2 = s * s;
    float p = fmaf(s2, 1.f / 13.f, 1.f / 11.f);
    p = fmaf(s2, p, 1.f / 9.f);
    p = fmaf(s2, p, 1.f / 7.f);
    p = fmaf(s2, p, 1.f / 5.f);
    p = fmaf(s2, p, 1.f / 3.f);
    p = fmaf(s2 * s, p, s);
    const float loss = fmaf(2.f, p, fmaxf(-z, 0.f));
    return a.smoothing != 0.f ? fmaf(a.smoothing, z, loss) : loss;
}

// Every pair is an item of both of its rows and is evaluated for each: a row then adds up its own items, with no
// atomics, and 4 to 12 bytes of an item are read in order; only the other row's score is looked up, mostly in L1, since rows
// that are compared lie together.  Two rows of few items are one lane of a slice of 64 rows whose items are stored by
// columns; rows of a slice have equal numbers of chosen and of rejected items, or nearly, because the layout
// sorts the rows of a window by them.  So few lanes idle, and which side a column is on is the same for the whole
// warp.  A row of many items has warps of its own, PB_CHUNK_ITEMS items each.
constexpr int kPairThreads = 512;
constexpr int kPairWarps = kPairThreads / 32;
constexpr int kAhead = 8;  // times 32 items of a chunk are asked for at once

// What a lane has of a slice: two rows, their scores, their numbers of items.
struct LaneRows {
    float own0, own1;
    int chosen0, end0, chosen1, end1;  // columns of the chosen side, of the rejected side from the slice's `chosen` on
    double sum0, sum1, loss;
};

// N columns from the c0-th on.
template <int N, typename T, bool SQUARED>
__device__ __forceinline__ void slice_columns(const PairArgs& a, const T* scores, int64_t item, int c0, int chosen, bool want,
                                              LaneRows& r) {
    int2 o[N];
    float2 off[N], w[N];
    T s0[N], s1[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        // (read once: L1 is for the scores)
        o[u] = __ldcs(reinterpret_cast<const int2*>(a.p.other + item + (c0 + u) * 64));
        off[u] = a.p.offset ? __ldcs(reinterpret_cast<const float2*>(a.p.offset + item + (c0 + u) * 64)) : make_float2(0.f, 0.f);
        w[u] = a.p.weight ? __ldcs(reinterpret_cast<const float2*>(a.p.weight + item + (c0 + u) * 64)) : make_float2(1.f, 1.f);
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
        s0[u] = scores[o[u].x];
        s1[u] = scores[o[u].y];
    }
    float p0 = 0.f, p1 = 0.f, cost = 0.f;  // (eight terms at most in 32 bits)
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int c = c0 + u;
        const float d0 = (r.own0 - to_f32(s0[u])) - off[u].x, d1 = (r.own1 - to_f32(s1[u])) - off[u].y;
        if (c < chosen) {
            const float t0 = pair_slope<SQUARED>(a, d0), t1 = pair_slope<SQUARED>(a, d1);
            if (c < r.chosen0) p0 = fmaf(w[u].x, t0, p0);
            if (c < r.chosen1) p1 = fmaf(w[u].y, t1, p1);
            if (want) {
                const float l0 = pair_loss<SQUARED>(a, d0, t0), l1 = pair_loss<SQUARED>(a, d1, t1);
                if (c < r.chosen0) cost = fmaf(w[u].x, l0, cost);
                if (c < r.chosen1) cost = fmaf(w[u].y, l1, cost);
            }
        } else {
            const float t0 = pair_slope<SQUARED>(a, -d0), t1 = pair_slope<SQUARED>(a, -d1);
            if (c < r.end0) p0 = fmaf(-w[u].x, t0, p0);
            if (c < r.end1) p1 = fmaf(-w[u].y, t1, p1);
        }
    }
    r.sum0 += (double)p0;
    r.sum1 += (double)p1;
    r.loss += (double)cost;
}

// (The scores may still be written by the kernel in front when this one begins: nothing tells the compiler that they stay as they
// are.)
template <typename T, bool SQUARED>
__global__ void __launch_bounds__(kPairThreads) pair_kernel(PairArgs a, const T* scores, T* __restrict__ grad, Totals totals) {
    let_next_start();
    wait_for_previous();  // (see launch_pairs)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool want = totals.ticket != nullptr;
    double loss = 0.0;
    // rows of many items first: their chunks are added up while others are still at their slices
    const int h0 = (int)(a.p.n_chunks * blockIdx.x / gridDim.x), h1 = (int)(a.p.n_chunks * (blockIdx.x + 1) / gridDim.x);
    for (int k = h0 + warp; k < h1; k += kPairWarps) {
        const int4 chunk = reinterpret_cast<const int4*>(a.p.chunks)[2 * k], of = reinterpret_cast<const int4*>(a.p.chunks)[2 * k + 1];
        const int row = chunk.x, count = chunk.z, chosen = chunk.w;
        const int64_t begin = chunk.y;
        const float own = to_f32(scores[row]);
        double sum = 0.0;
        for (int i0 = lane; i0 < count; i0 += 32 * kAhead) {
            int o[kAhead];
            float off[kAhead], w[kAhead];
            T s[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int64_t i = begin + min(i0 + u * 32, count - 1);
                o[u] = a.p.other[i];
                off[u] = a.p.offset ? a.p.offset[i] : 0.f;
                w[u] = a.p.weight ? a.p.weight[i] : 1.f;
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) s[u] = scores[o[u]];
            float four = 0.f, four_loss = 0.f;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int i = i0 + u * 32;
                const bool better = i < chosen;
                const float d = (own - to_f32(s[u])) - off[u], t = pair_slope<SQUARED>(a, better ? d : -d);
                if (i < count) four = fmaf(better ? w[u] : -w[u], t, four);
                if (want) {
                    const float l = pair_loss<SQUARED>(a, d, t);
                    if (better) four_loss = fmaf(w[u], l, four_loss);
                }
            }
            sum += (double)four;
            loss += (double)four_loss;
        }
        sum = warp_sum(sum);
        if (lane == 0) {
            if (of.z == 1)
                grad[row] = from_f32<T>((float)(sum * a.factor));
            else
                a.sums[k] = sum;
        }
    }
    if (a.p.n_split && h0 < h1) {
        // A row of several chunks: the CTA with its last ones adds all of them up, in their order.  (CTAs count for their chunks of a
        // row at once: 4 000 chunks of three rows that counted one by one took 3 us of 19.)
        __syncthreads();
        for (int k = h0 + warp; k < h1; k += kPairWarps) {
            const int4 of = reinterpret_cast<const int4*>(a.p.chunks)[2 * k + 1];
            if (of.z == 1 || (k != h0 && k != of.y)) continue;
            const unsigned mine = (unsigned)(min(h1, of.y + of.z) - k);
            int last = 0;
            if (lane == 0) {
                fence();  // the sums (of all warps, which the barrier has put before this) are visible before the count is
                last = atomicAdd(a.counts + of.x, mine) + mine == (unsigned)of.z;
            }
            if (!__shfl_sync(0xFFFFFFFFu, last, 0)) continue;
            __syncwarp();  // (orders the lanes' reads after the first lane's count)
            fence();
            double sum = 0.0;
#pragma unroll 8
            for (int i = lane; i < of.z; i += 32) sum += __ldcg(a.sums + of.y + i);
            sum = warp_sum(sum);
            if (lane == 0) {
                grad[a.p.chunks[8 * (int64_t)k]] = from_f32<T>((float)(sum * a.factor));
                a.counts[of.x] = 0u;
            }
        }
    }
    // neighbouring slices to one CTA: their rows are compared with the same ones
    const int s0 = (int)(a.p.n_slices * blockIdx.x / gridDim.x), s1 = (int)(a.p.n_slices * (blockIdx.x + 1) / gridDim.x);
    // (a slice's description is read one slice ahead)
    const int2* slices = reinterpret_cast<const int2*>(a.p.slices);
    const int4* slice_rows = reinterpret_cast<const int4*>(a.p.slice_rows);
    auto describe = [&](int k) { return k < s1 ? slices[k] : make_int2(0, 0); };
    auto rows_of = [&](int k) { return k < s1 ? slice_rows[(int64_t)k * 32 + lane] : make_int4(-1, 0, -1, 0); };
    int2 slice = describe(s0 + warp);
    int4 mine = rows_of(s0 + warp);
    for (int k = s0 + warp; k < s1; k += kPairWarps) {
        const int2 next_slice = describe(k + kPairWarps);
        const int4 next_mine = rows_of(k + kPairWarps);
        const int chosen = slice.y & 0xFFFF, columns = chosen + (slice.y >> 16);
        LaneRows r;
        r.own0 = mine.x >= 0 ? to_f32(scores[mine.x]) : 0.f;
        r.own1 = mine.z >= 0 ? to_f32(scores[mine.z]) : 0.f;
        r.chosen0 = mine.y & 0xFFFF;
        r.end0 = chosen + (mine.y >> 16);
        r.chosen1 = mine.w & 0xFFFF;
        r.end1 = chosen + (mine.w >> 16);
        r.sum0 = r.sum1 = 0.0;
        r.loss = loss;
        const int64_t item = (int64_t)slice.x * 64 + 2 * lane;
        int c = 0;
        for (; c + 4 <= columns; c += 4) slice_columns<4, T, SQUARED>(a, scores, item, c, chosen, want, r);
        if (columns - c == 3)
            slice_columns<3, T, SQUARED>(a, scores, item, c, chosen, want, r);
        else if (columns - c == 2)
            slice_columns<2, T, SQUARED>(a, scores, item, c, chosen, want, r);
        else if (columns - c == 1)
            slice_columns<1, T, SQUARED>(a, scores, item, c, chosen, want, r);
        loss = r.loss;
        if (mine.x >= 0) grad[mine.x] = from_f32<T>((float)(r.sum0 * a.factor));
        if (mine.z >= 0) grad[mine.z] = from_f32<T>((float)(r.sum1 * a.factor));
        slice = next_slice;
        mine = next_mine;
    }
    put_totals<kPairThreads>(totals, blockIdx.x, loss, 0.0, 0, false);
}

// ---- groups ---------------------------------------------------------------------------------------
//
// A group needs three sums in turn: the largest score and the sum of exponentials, then what its rows add to
// one another's gradients, then nothing: the gradients.  The sum of exponentials is taken in 64 bits; from its log
// on, numbers are pairs of floats (value and rounding error), which the 32-bit units add faster than the
// few 64-bit ones would convert them.

enum GroupOp { kChoice, kPolicy, kLogProbs };

struct Pair32 {  // hi + lo
    float hi, lo;
};

// a - b without rounding, plus a small `lo`.  Where hi is infinite, lo comes out as NaN; fminf(lo, 1) is then 1, with which sums
// and exp come out right, and changes nothing else: lo is above 1 only where hi is beyond 2^24 (see Normaliser).
__device__ __forceinline__ Pair32 difference(float a, float b, float lo) {
    const float t = a - b, v = t - a;
    return Pair32{t, (a - (t - v)) - (b + v) + lo};
}

__host__ __device__ __forceinline__ Pair32 split(double x) {
    const float hi = (float)x, lo = (float)(x - (double)hi);
    return Pair32{hi, lo - lo == 0.f ? lo : 0.f};
}

__device__ __forceinline__ float sum_of(Pair32 x) { return x.hi + fminf(x.lo, 1.f); }

// exp(hi + lo): 2^y with y = hi log2 e rounded, by the unit that has 2^x to 2 ulp, times 1 + what y left out.  BEYOND: it may be
// beyond 32 bits.  y is then held below 128, where 2^y is a number, and what that leaves out makes it infinite: infinity less a
// part of itself would be no number.  (574 groups of a policy: 27.5 us so, 28.1 with a choice after the product, 26.7 without.)  The
// correction is of first order: to float32 as long as |lo| is below 2e-4.
template <bool BEYOND>
__device__ __forceinline__ float exp_of(Pair32 x) {
    constexpr float log2e = 1.44269502f, rest = 1.33498e-8f;  // log2 e as a float, and (log2 e - that) ln 2
    constexpr double off = (1.4426950408889634 - (double)log2e) * 0.6931471805599453 - (double)rest;
    static_assert(off < 1e-13 && off > -1e-13, "what the float of log2 e leaves out");
    float y = x.hi * log2e;
    if (BEYOND) asm("min.NaN.f32 %0, %0, %1;" : "+f"(y) : "f"(127.999992f));  // (the largest float below 128)
    float more = fmaf(fmaf(x.hi, log2e, -y), 0.693147181f, x.lo);
    more = fminf(fmaf(x.hi, rest, more), 1.f);
    const float e = exp2_of(y);
    return fmaf(e, more, e);
}

// The log of a group's sum, for differences from it.  Of a large log its float leaves out what is no longer small against the
// difference: of three scores of 1e8 the probabilities were -0.1.  From 4 096 on scores and log are therefore both taken
// relative to its float: the scores near it, which are all that have a probability, stay exact.  Below, what the float leaves out is at
// most 1.3e-4, whose square is none of float32's.
struct Normaliser {
    float zero;
    Pair32 log;  // from zero on
    __device__ __forceinline__ explicit Normaliser(double lse64)
        : zero(fabs(lse64) < 4096.0 ? 0.f : (float)lse64), log(split(lse64 - (double)zero)) {}
    __device__ __forceinline__ Pair32 log_prob(float s) const { return difference(s - zero, log.hi, -log.lo); }
};

// exp(x) for x <= 0, exactly 1 at 0: with n = rint(x / ln 2), 2^n times the Taylor polynomial of degree 11 at
// |f| <= ln 2 / 2.  Off by up to 1.1e-14 of the value from -60 on (7e-15 the rest of the polynomial, and 2.3e-17 a unit of n the one
// constant for ln 2), by 3.1e-14 near -700; below that: 0.  (The log of the sum has to be exact to some 1e-13: a divergence of nearly
// equal policies is a mean of differences of that size.)
__device__ __forceinline__ double exp_negative(double x) {
    const double shift = 6755399441055744.0;  // 1.5 * 2^52: the low word of x + shift is x as an integer
    const double t = fma(x, 1.4426950408889634, shift);
    const double f = fma(t - shift, -0.6931471805599453, x);
    double p = fma(f, 1.0 / 39916800.0, 1.0 / 3628800.0);
    p = fma(f, p, 1.0 / 362880.0);
    p = fma(f, p, 1.0 / 40320.0);
    p = fma(f, p, 1.0 / 5040.0);
    p = fma(f, p, 1.0 / 720.0);
    p = fma(f, p, 1.0 / 120.0);
    p = fma(f, p, 1.0 / 24.0);
    p = fma(f, p, 1.0 / 6.0);
    p = fma(f, p, 0.5);
    p = fma(f, p, 1.0);
    p = fma(f, p, 1.0);
    p *= __hiloint2double((__double2loint(t) + 1023) << 20, 0);
    return x < -700.0 ? 0.0 : p;
}

// m + log(z), z a sum of exponentials whose largest is 1 (or 0: nothing left in the group, every p is 0; or NaN).  With y
// the units' log2(z) times ln 2, log z = y + log(1 + w), w = z exp(-y) - 1 of some 1e-6, where four terms are exact.
__device__ __forceinline__ double log_sum(float m, double z) {
    float y2;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y2) : "f"((float)z));
    const double y = (double)y2 * 0.6931471805599453;
    const double w = fma(z, exp_negative(-y), -1.0);
    const double l = y + w * fma(w, fma(w, fma(w, -0.25, 1.0 / 3.0), -0.5), 1.0);
    return z == 0.0 ? 0.0 : (double)m + l;
}

struct GroupArgs {
    pb_groups g;
    const float *target, *advantage, *old, *reference;
    Pair32 log_high, log_low;  // borders of the log of the ratio
    float bound_high, bound_low;
    float kl_coef;
    float scale;
};

// Up to N rows of one group that a thread has: places first, first + stride ... of those from `low` to below `end`.  VECTOR:
// four neighbouring ones, whose first is a multiple of 4, moved as one word where all are in the table and the arrays allow it (which
// changes nothing in the order of sums).  FULL (of the members): all are the group's.
template <typename T, int OP, int N, bool VECTOR = false>
struct Rows {
    const GroupArgs& a;
    int first, stride, low, end;  // places
    int used;                     // rows that any thread of the warp has
    bool words;                   // VECTOR: all arrays begin on the border of a word
    int row[N];                   // only with a list of rows
    // (s becomes p, main (target or advantage) the fixed part; of more than four rows, the three inputs of a policy come four rows
    // at a time: interleaved lists of 1M rows took 39 us with all at once, which spills, and 35 so)
    static constexpr bool LATE = OP == kPolicy && N > 4;
    static constexpr int HELD = LATE ? 4 : N;
    alignas(16) float s[N], main[N], old[HELD], reference[HELD];  // (four of them are moved as one word)
    double loss = 0.0, kl = 0.0, share = 0.0;
    int clipped = 0;
    static_assert(!VECTOR || N == 4, "rows of a word");

    __device__ __forceinline__ Rows(const GroupArgs& args) : a(args) {}

    __device__ __forceinline__ int place(int u) const { return VECTOR ? first + u : first + u * stride; }
    template <bool FULL>
    __device__ __forceinline__ bool has(int u) const { return FULL || (place(u) < end && (!VECTOR || place(u) >= low)); }
    __device__ __forceinline__ int row_of(int u) const { return !VECTOR && a.g.rows ? row[u] : place(u); }
    // (half of the rows are there more often than not: only the others are worth a branch)
    template <bool FULL>
    __device__ __forceinline__ bool on(int u) const { return VECTOR || FULL || u < N / 2 || u < used; }

    // COUNT values from the u0-th on
    template <bool FULL, int COUNT = N, typename V>
    __device__ __forceinline__ void take(const V* from, V* to, int u0 = 0) const {
        if (VECTOR && words && (FULL || (first < end && first + 3 < (int)a.g.n_rows))) {
            if (sizeof(V) == 4)
                *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from + first);
            else
                *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(from + first);
        } else {
#pragma unroll
            for (int u = 0; u < COUNT; ++u)
                if (on<FULL>(u0 + u) && has<FULL>(u0 + u)) to[u] = from[row_of(u0 + u)];
        }
    }

    // Everything is asked for before anything is used.
    template <bool FULL>
    __device__ __forceinline__ void load(const T* scores, bool inputs) {
        alignas(16) T raw[N];
        if (!VECTOR && a.g.rows) {
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (on<FULL>(u) && has<FULL>(u)) row[u] = a.g.rows[place(u)];
        }
        take<FULL>(scores, raw);
        if (OP != kLogProbs && inputs && !LATE) {
            take<FULL>(OP == kChoice ? a.target : a.advantage, main);
            if (OP == kPolicy) {
                take<FULL, HELD>(a.old, old);
                if (a.reference) take<FULL, HELD>(a.reference, reference);
            }
        }
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const bool mine = on<FULL>(u) && has<FULL>(u);
            s[u] = mine ? to_f32(raw[u]) : -INFINITY;
            if (OP == kChoice && inputs) main[u] = mine ? main[u] : 0.f;
        }
    }

    __device__ __forceinline__ float largest() const {
        float m = s[0];
#pragma unroll
        for (int u = 1; u < N; ++u) m = fmaxf(m, s[u]);
        return m;
    }

    // Sum of exp(s - m).  (m = -inf: no row is left, all of them add exp(-inf) to 0.)
    template <bool FULL>
    __device__ __forceinline__ double mass(float m) const {
        const double top = m == -INFINITY ? 0.0 : (double)m;
        double z = 0.0;
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (on<FULL>(u)) z += exp_negative((double)s[u] - top);
        return z;
    }

    // With the log of the group's sum: p, the part of the gradient that does not hang on the rest of the group, and what
    // goes into the sums.  A row's gradient is (fixed + p * share) * scale: of a choice -t + p * sum t, of a policy, with h
    // the slopes of the taken rows and D the divergence, h + p (k (l - reference - D) - sum h).  A masked row's other
    // inputs, and the old log-probability of a row that was not taken, may be anything.
    template <bool FULL>
    __device__ __forceinline__ void terms(double lse64) {
        const Normaliser lse(lse64);
        float part = 0.f, part_loss = 0.f, part_kl = 0.f;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            if (LATE && u % 4 == 0 && on<FULL>(u)) {
                take<FULL, 4>(a.advantage, main + u, u);
                take<FULL, 4>(a.old, old, u);
                if (a.reference) take<FULL, 4>(a.reference, reference, u);
            }
            if (on<FULL>(u)) {
                const bool live = s[u] != -INFINITY;
                const Pair32 l = lse.log_prob(s[u]);
                const float p = live ? exp_of<false>(l) : 0.f;
                float fixed, own;
                if (OP == kChoice) {
                    const float t = main[u];
                    if (t != 0.f) loss += (double)t * (lse64 - (double)s[u]);  // (in 64 bits: terms may be of very different size)
                    fixed = -t;
                    own = t;
                } else {
                    const float adv = live ? main[u] : 0.f;
                    const bool up = adv > 0.f, taken = adv != 0.f;
                    Pair32 x = difference(l.hi, old[u % HELD], l.lo);
                    // (two log-probabilities below some -4 000: of the difference of their floats less may be left than of what they leave out)
                    if (fabsf(x.lo) > 2e-4f) x = Pair32{x.hi + x.lo, x.lo - ((x.hi + x.lo) - x.hi)};
                    const float past = (x.hi - (up ? a.log_high.hi : a.log_low.hi)) + (fminf(x.lo, 1.f) - (up ? a.log_high.lo : a.log_low.lo));
                    const bool beyond = taken && (up ? past : -past) > 0.f;
                    const float q = beyond ? (up ? a.bound_high : a.bound_low) : exp_of<true>(x);
                    const float cost = -adv * (taken ? q : 0.f);
                    fixed = beyond ? 0.f : cost;
                    part_loss += cost;
                    clipped += beyond ? 1 : 0;
                    own = -fixed;
                    if (a.reference) {
                        const float k = live ? p * sum_of(difference(l.hi, reference[u % HELD], l.lo)) : 0.f;
                        fixed = fmaf(a.kl_coef, k, fixed);
                        own = fmaf(-a.kl_coef, k, own);
                        part_kl += k;
                    }
                }
                part += own;
                s[u] = p;
                main[u] = fixed;
            }
            if ((u & 3) == 3 && on<FULL>(u - 3)) {  // (four terms in 32 bits, the sums of fours in 64)
                share += (double)part;
                if (OP == kPolicy) {
                    loss += (double)fmaf(a.kl_coef, part_kl, part_loss);
                    kl += (double)part_kl;
                }
                part = part_loss = part_kl = 0.f;
            }
        }
    }

    // (v becomes what is written)
    template <bool FULL>
    __device__ __forceinline__ void put(const float v[N], T* out) const {
        if (VECTOR && words && (FULL || (first >= low && first + 3 < end))) {
            alignas(16) const T w[4] = {from_f32<T>(v[0]), from_f32<T>(v[1]), from_f32<T>(v[2]), from_f32<T>(v[3])};
            if (sizeof(T) == 4)
                *reinterpret_cast<uint4*>(out + first) = *reinterpret_cast<const uint4*>(w);
            else
                *reinterpret_cast<uint2*>(out + first) = *reinterpret_cast<const uint2*>(w);
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (on<FULL>(u) && has<FULL>(u)) out[row_of(u)] = from_f32<T>(v[u]);
        }
    }

    template <bool FULL>
    __device__ __forceinline__ void gradient(float total, T* out) const {
        float g[N];
#pragma unroll
        for (int u = 0; u < N; ++u) g[u] = fmaf(s[u], total, main[u]) * a.scale;
        // The total may be infinite, and with it the fixed part of a row whose ratio is: that row's gradient is its own part, and
        // rows without a share of the total have none.
        if (!(fabsf(total) < INFINITY)) {
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (s[u] == 0.f || fabsf(main[u]) == INFINITY) g[u] = main[u] * a.scale;
        }
        put<FULL>(g, out);
    }

    template <bool FULL>
    __device__ __forceinline__ void log_probs(double lse64, T* out) const {
        const Normaliser lse(lse64);
        float l[N];
#pragma unroll
        for (int u = 0; u < N; ++u) l[u] = sum_of(lse.log_prob(s[u]));
        put<FULL>(l, out);
    }
};

// The sums of several threads into one: z is relative to m.
__device__ __forceinline__ double rescaled(double z, float m, float top) {
    return z == 0.0 ? 0.0 : z * exp_negative((double)m - (double)top);
}

// ---- short groups: lanes of a warp ----
//
// 1, 2, 4 ... 32 neighbouring lanes have a group, up to eight rows each; the groups of a warp have equal lengths, or nearly,
// because the layout sorts them by length; sums over a group are shuffles within its lanes.
constexpr int kTeamThreads = 256;
__host__ __device__ constexpr int team_ctas(bool policy) { return policy ? 2 : 4; }  // on an SM
constexpr int kTeamRows = PB_TEAM_ROWS / 32;

// (Registers: of a choice, 4 CTAs per SM took 27 us over 2.7M rows, 2 took 33, 5 took 30.  Of a policy over 1M rows in interleaved
// lists, where what the SMs can look up bounds it, 2 took 35, 3 took 39 and 4 took 37.)
template <typename T, int OP>
__global__ void __launch_bounds__(kTeamThreads, team_ctas(OP == kPolicy))
    team_kernel(GroupArgs a, int slot0, const T* __restrict__ scores, T* __restrict__ out, Totals totals) {
    let_next_start();
    const int lane = threadIdx.x & 31;
    double loss = 0.0, kl = 0.0;
    int clipped = 0;
    for (int w = (blockIdx.x * kTeamThreads + threadIdx.x) >> 5; w < (int)a.g.n_team_warps; w += gridDim.x * (kTeamThreads / 32)) {
        const int2 what = reinterpret_cast<const int2*>(a.g.team_warps)[w];  // first team; class and rows of a lane
        const int shift = what.y & 0xFF, lanes = 1 << shift;
        const int2 group = reinterpret_cast<const int2*>(a.g.teams)[what.x + (lane >> shift)];
        Rows<T, OP, kTeamRows> rows(a);
        rows.first = group.x + (lane & (lanes - 1));
        rows.stride = lanes;
        rows.low = group.x;
        rows.end = group.x + group.y;
        rows.used = what.y >> 8;
        rows.template load<false>(scores, true);
        float m = rows.largest();
        for (int d = lanes >> 1; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
        double z = rows.template mass<false>(m);
        for (int d = lanes >> 1; d > 0; d >>= 1) z += __shfl_xor_sync(0xFFFFFFFFu, z, d);
        const double lse = log_sum(m, z);
        if (OP == kLogProbs) {
            rows.template log_probs<false>(lse, out);
            continue;
        }
        rows.template terms<false>(lse);
        double share = rows.share;
        for (int d = lanes >> 1; d > 0; d >>= 1) share += __shfl_xor_sync(0xFFFFFFFFu, share, d);
        rows.template gradient<false>((float)share, out);
        loss += rows.loss;
        kl += rows.kl;
        clipped += rows.clipped;
    }
    if (OP != kLogProbs) put_totals<kTeamThreads>(totals, slot0 + blockIdx.x, loss, kl, clipped, OP == kPolicy);
    wait_for_previous();
}

// ---- longer groups: a CTA ----
//
// The scores are gone through twice, the second time from L1; p and the fixed part of the gradient stay in shared memory for
// the third step, so that the other inputs are read once.  Few threads with many rows each: what a warp does per group (sums
// over its lanes, the log) is as much as five rows.
template <int THREADS>
__device__ __forceinline__ double cta_log_sum(float m, double z, float* s_m, double* s_z) {
    const int lane = threadIdx.x & 31;
    const float wm = warp_max(m);
    z = warp_sum(rescaled(z, m, wm));
    if (lane == 0) {
        s_m[threadIdx.x >> 5] = wm;
        s_z[threadIdx.x >> 5] = z;
    }
    __syncthreads();
    m = lane < THREADS / 32 ? s_m[lane] : -INFINITY;
    z = lane < THREADS / 32 ? s_z[lane] : 0.0;
    const float top = warp_max(m);
    return log_sum(top, warp_sum(rescaled(z, m, top)));
}

constexpr int kBlockRows = 4;  // of a thread at a time

// (MANY: a CTA takes one group after the other; as a loop that runs once it costs ragged eras 2 us of 18.)
template <typename T, int OP, int THREADS, bool VECTOR, bool MANY>
__global__ void __launch_bounds__(THREADS) block_kernel(GroupArgs a, const int2* __restrict__ list, int most, bool words, int slot0,
                                                        const T* __restrict__ scores, T* __restrict__ out, Totals totals) {
    extern __shared__ float4 kept4[];  // p, then the fixed parts, `most` each: a thread's four are one word
    __shared__ float s_m[THREADS / 32];
    __shared__ double s_z[THREADS / 32], scratch[THREADS / 32];
    let_next_start();
    constexpr int kStep = THREADS * kBlockRows;
    using Four = Rows<T, OP, kBlockRows, VECTOR>;
    static_assert(alignof(Four) % 16 == 0, "four rows are moved as one word");
    float4* const kept_p = kept4 + threadIdx.x;
    float4* const kept_fixed = kept4 + most / 4 + threadIdx.x;
    double loss = 0.0, kl = 0.0;
    int clipped = 0;
    for (int g = blockIdx.x; MANY ? g < (int)a.g.n_blocks : g == (int)blockIdx.x; g += gridDim.x) {
        const int2 group = list[g];
        const int begin = VECTOR ? group.x & ~3 : group.x, end = group.x + group.y;
        // all steps of the group in turn: f(rows, step, whether all rows are the group's)
        auto steps = [&](auto f) {
            for (int at = begin, k = 0; at < end; at += kStep, ++k) {
                Four rows(a);
                rows.first = at + (int)threadIdx.x * (VECTOR ? kBlockRows : 1);
                rows.stride = THREADS;
                rows.low = group.x;
                rows.end = end;
                rows.used = (end - at + THREADS - 1) / THREADS;
                rows.words = words;
                if (at >= group.x && at + kStep <= end)
                    f(rows, k, std::true_type());
                else
                    f(rows, k, std::false_type());
            }
        };
        float m = -INFINITY;
        double z = 0.0, share = 0.0;
        steps([&](Four& rows, int, auto full) {
            rows.template load<decltype(full)::value>(scores, false);
            const float top = fmaxf(m, rows.largest());
            z = rescaled(z, m, top) + rows.template mass<decltype(full)::value>(top);
            m = top;
        });
        const double lse = cta_log_sum<THREADS>(m, z, s_m, s_z);
        if (OP == kLogProbs) {
            steps([&](Four& rows, int, auto full) {
                rows.template load<decltype(full)::value>(scores, false);
                rows.template log_probs<decltype(full)::value>(lse, out);
            });
            if (MANY) __syncthreads();  // (the next group's sums go where this one's were)
            continue;
        }
        steps([&](Four& rows, int k, auto full) {
            rows.template load<decltype(full)::value>(scores, true);
            rows.template terms<decltype(full)::value>(lse);
            if (decltype(full)::value || (k * THREADS + (int)threadIdx.x) * 4 < most) {
                kept_p[k * THREADS] = make_float4(rows.s[0], rows.s[1], rows.s[2], rows.s[3]);
                kept_fixed[k * THREADS] = make_float4(rows.main[0], rows.main[1], rows.main[2], rows.main[3]);
            }
            loss += rows.loss;
            kl += rows.kl;
            share += rows.share;
            clipped += rows.clipped;
        });
        const float total = (float)cta_sum<THREADS>(share, scratch);
        steps([&](Four& rows, int k, auto full) {
            if (!decltype(full)::value && (k * THREADS + (int)threadIdx.x) * 4 >= most) return;
            *reinterpret_cast<float4*>(rows.s) = kept_p[k * THREADS];
            *reinterpret_cast<float4*>(rows.main) = kept_fixed[k * THREADS];
            if (!VECTOR && a.g.rows) {
#pragma unroll
                for (int u = 0; u < kBlockRows; ++u)
                    if (rows.template has<decltype(full)::value>(u)) rows.row[u] = a.g.rows[rows.place(u)];
            }
            rows.template gradient<decltype(full)::value>(total, out);
        });
    }
    if (OP != kLogProbs) put_totals<THREADS>(totals, slot0 + blockIdx.x, loss, kl, clipped, OP == kPolicy);
    wait_for_previous();
}

// ---- long groups: many CTAs each ----
//
// Pieces of up to 2048 rows; the sums of a group's pieces go through memory from one launch to the next: sums of
// exponentials, then (of a policy; a choice's are its targets, known at once) shares, then the gradient.  The rows are read
// again each time, from L2 mostly, while the launch before still runs.
struct alignas(16) PieceSums {
    double z;
    float m, unused;
    double share, unused2;
};
enum PieceStep { kPieceMass, kPieceTerms, kPieceOut };
constexpr int kPieceThreads = 256;
constexpr int kPieceRows = PB_PIECE_ROWS / kPieceThreads;

// (A launch begins before the one in front has left its sums: they are read from L2, after the wait, and nothing tells the compiler
// that they stay as they are.)
template <typename T, int OP, int STEP>
__global__ void __launch_bounds__(kPieceThreads) piece_kernel(GroupArgs a, PieceSums* pieces, int slot0,
                                                              const T* __restrict__ scores, T* __restrict__ out, Totals totals) {
    constexpr int kWarps = kPieceThreads / 32;
    __shared__ float s_m[kWarps];
    __shared__ double s_z[kWarps], scratch[kWarps];
    let_next_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int4 piece = reinterpret_cast<const int4*>(a.g.pieces)[blockIdx.x];
    const int first = piece.z, count = piece.w;  // the group's pieces
    Rows<T, OP, kPieceRows> rows(a);
    rows.first = piece.x + threadIdx.x;
    rows.stride = kPieceThreads;
    rows.low = piece.x;
    rows.end = piece.x + piece.y;
    rows.used = (piece.y + kPieceThreads - 1) / kPieceThreads;
    rows.template load<false>(scores, STEP != kPieceMass || OP == kChoice);
    constexpr bool kTotalsAtEnd = OP == kChoice;
    if (STEP == kPieceMass) {
        if (OP == kChoice) {
            double targets = 0.0;
#pragma unroll
            for (int u = 0; u < kPieceRows; ++u) targets += (double)rows.main[u];
            targets = cta_sum<kPieceThreads>(targets, scratch);
            if (threadIdx.x == 0) pieces[blockIdx.x].share = targets;
        }
        float m = rows.largest();
        const float wm = warp_max(m);
        double z = warp_sum(rows.template mass<false>(wm));
        if (lane == 0) {
            s_m[warp] = wm;
            s_z[warp] = z;
        }
        __syncthreads();
        if (warp == 0) {
            m = lane < kWarps ? s_m[lane] : -INFINITY;
            z = lane < kWarps ? s_z[lane] : 0.0;
            const float top = warp_max(m);
            z = warp_sum(rescaled(z, m, top));
            if (lane == 0) {
                pieces[blockIdx.x].m = top;
                pieces[blockIdx.x].z = z;
            }
        }
        wait_for_previous();
        return;
    }
    wait_for_previous();  // (the rows do not come from the launch before, the sums do)
    float m = -INFINITY;
    double z = 0.0;
    for (int k = threadIdx.x; k < count; k += kPieceThreads) {
        const float4 zm = __ldcg(reinterpret_cast<const float4*>(pieces + first + k));  // (z and m in one word)
        const float mk = zm.z, top = fmaxf(m, mk);
        z = rescaled(z, m, top) + rescaled(__hiloint2double(__float_as_int(zm.y), __float_as_int(zm.x)), mk, top);
        m = top;
    }
    const double lse = cta_log_sum<kPieceThreads>(m, z, s_m, s_z);
    if (OP == kLogProbs) {
        rows.template log_probs<false>(lse, out);
        return;
    }
    rows.template terms<false>(lse);
    if (STEP == kPieceTerms) {
        const double share = cta_sum<kPieceThreads>(rows.share, scratch);
        if (threadIdx.x == 0) pieces[blockIdx.x].share = share;
        put_totals<kPieceThreads>(totals, slot0 + blockIdx.x, rows.loss, rows.kl, rows.clipped, OP == kPolicy);
        return;
    }
    double share = 0.0;
    for (int k = threadIdx.x; k < count; k += kPieceThreads) share += __ldcg(&pieces[first + k].share);
    rows.template gradient<false>((float)cta_sum<kPieceThreads>(share, scratch), out);
    if (kTotalsAtEnd) put_totals<kPieceThreads>(totals, slot0 + blockIdx.x, rows.loss, 0.0, 0, false);
}

// ---- launches ---------------------------------------------------------------------------------------

constexpr double kMostFactor = 1e30, kLeastSquaredBeta = 1e-15;
constexpr int64_t kMost = (1ll << 31) - 1;
constexpr int64_t kMostRows = PB_OBJECTIVE_MOST_ROWS;  // (a CTA's places past the last row are still 32-bit numbers)

int check_groups(const pb_groups* g) {
    PB_REQUIRE(g != nullptr, "groups are null");
    PB_REQUIRE(g->n_rows >= 0 && g->n_rows <= kMostRows, "n_rows=%lld out of range", (long long)g->n_rows);
    PB_REQUIRE(g->n_groups >= 0 && g->n_groups <= g->n_rows, "n_groups=%lld out of range", (long long)g->n_groups);
    PB_REQUIRE((g->n_groups == 0) == (g->n_rows == 0), "rows without a group");
    PB_REQUIRE(g->n_team_warps >= 0 && g->n_team_warps < kMost / 32 && g->n_pieces >= 0 && g->n_pieces < kMost && g->n_blocks >= 0 &&
                   g->n_blocks <= g->n_groups,
               "counts of the groups' layout are out of range");
    PB_REQUIRE(g->n_blocks == 0 || (g->block_rows > 0 && g->block_rows <= PB_BLOCK_ROWS), "block_rows is out of range");
    PB_REQUIRE((g->n_team_warps == 0 || (g->team_warps && g->teams)) && (g->n_blocks == 0 || g->blocks) && (g->n_pieces == 0 || g->pieces),
               "a table of the groups' layout is null");
    PB_REQUIRE((uintptr_t)g->team_warps % 8 == 0 && (uintptr_t)g->teams % 8 == 0 && (uintptr_t)g->blocks % 8 == 0 && (uintptr_t)g->pieces % 16 == 0,
               "tables of the groups' layout must be aligned");
    PB_REQUIRE(g->n_groups == 0 || g->n_team_warps + g->n_blocks + g->n_pieces > 0, "the groups are not laid out");
    return PB_OK;
}

int check_pairs(const pb_pairs* p) {
    PB_REQUIRE(p != nullptr, "pairs are null");
    PB_REQUIRE(p->n_rows >= 0 && p->n_rows <= kMostRows, "n_rows=%lld out of range", (long long)p->n_rows);
    PB_REQUIRE(p->n_slices >= 0 && p->n_slices < kMost / 64 && p->n_chunks >= 0 && p->n_chunks < kMost && p->n_split >= 0 &&
                   2 * p->n_split <= p->n_chunks,
               "counts of the pairs' layout are out of range");
    PB_REQUIRE(p->n_rows == 0 || p->n_slices + p->n_chunks > 0, "the pairs are not laid out");
    PB_REQUIRE((p->n_slices == 0 || (p->slices && p->slice_rows)) && (p->n_chunks == 0 || p->chunks) && (p->n_rows == 0 || p->other),
               "a table of the pairs' layout is null");
    PB_REQUIRE((uintptr_t)p->slices % 8 == 0 && (uintptr_t)p->slice_rows % 16 == 0 && (uintptr_t)p->chunks % 16 == 0,
               "tables of the pairs' layout must be aligned");
    PB_REQUIRE((uintptr_t)p->other % 8 == 0 && (uintptr_t)p->offset % 8 == 0 && (uintptr_t)p->weight % 8 == 0,
               "items must be 8-byte aligned");
    return PB_OK;
}

int check_objective(const pb_objective* o) {
    PB_REQUIRE(o != nullptr, "objective is null");
    // (factors that stay numbers in 32 bits)
    PB_REQUIRE(fabs(o->scale) <= kMostFactor, "scale is out of range");
    if (o->kind == PB_OBJECTIVE_PREFERENCE) {
        PB_TRY(check_pairs(o->pairs));
        PB_REQUIRE(o->beta >= 1.0 / kMostFactor && o->beta <= kMostFactor, "beta outside [1e-30, 1e30]");
        // (1 / (2 beta) and its square)
        PB_REQUIRE(!o->squared || o->beta >= kLeastSquaredBeta, "beta of the squared form below 1e-15");
        PB_REQUIRE(o->smoothing >= 0.0 && o->smoothing < 0.5, "smoothing outside [0, 0.5)");
        return PB_OK;
    }
    PB_REQUIRE(o->kind == PB_OBJECTIVE_CHOICE || o->kind == PB_OBJECTIVE_POLICY, "unknown objective %lld", (long long)o->kind);
    PB_TRY(check_groups(o->groups));
    if (o->groups->n_rows == 0) return PB_OK;
    if (o->kind == PB_OBJECTIVE_CHOICE) {
        PB_REQUIRE(o->target != nullptr, "target is null");
        return PB_OK;
    }
    PB_REQUIRE(o->advantage && o->old, "advantage or old is null");
    PB_REQUIRE(o->clip_low >= 0.0 && o->clip_low <= 1.0, "clip_low outside [0, 1]");
    PB_REQUIRE(o->clip_high >= 0.0, "clip_high must not be negative");
    PB_REQUIRE(fabs(o->kl_coef) <= kMostFactor, "kl_coef is out of range");
    PB_REQUIRE(o->reference || o->kl_coef == 0.0, "kl_coef needs a reference");
    return PB_OK;
}

int64_t n_rows_of(const pb_objective* o) {
    return o->kind == PB_OBJECTIVE_PREFERENCE ? o->pairs->n_rows : o->groups->n_rows;
}

// CTAs of the launch whose warps take one team task after the other: as many as the SMs hold at once (with more of them, 1M rows in
// interleaved lists took 34 us for 31), or as there are tasks.
int64_t team_grid(const pb_groups* g, bool policy) {
    const int64_t most = 148 * team_ctas(policy);
    return g->n_team_warps < most * (kTeamThreads / 32) ? (g->n_team_warps + kTeamThreads / 32 - 1) / (kTeamThreads / 32) : most;
}

// (two CTAs per SM: with more, of which each looks up scores in another window of rows, L1 holds too little of each)
int64_t n_parts_of(const pb_pairs* p) {
    const int64_t tasks = p->n_slices > p->n_chunks ? p->n_slices : p->n_chunks;
    return tasks < 148 * 2 * kPairWarps ? (tasks + kPairWarps - 1) / kPairWarps : 148 * 2;
}
// CTAs of the launch for longer groups: one each, up to so many that the totals are few against the rows.  (8 000 groups of 300 rows, one
// CTA each and so many: policy 78.5 and 75.4 us, choice 58.5 and 56.3; 2 400 groups: 27.7 and 30.4, 21.5 and 23.1.)
int64_t block_grid(const pb_groups* g) { return g->n_blocks < 148 * 16 ? g->n_blocks : 148 * 16; }

int64_t n_parts_of(const pb_groups* g, bool policy) { return team_grid(g, policy) + block_grid(g) + g->n_pieces; }

// Scratch: the ticket; of pairs, counts and sums of the rows in several chunks; of groups, the sums of pieces; the totals.
constexpr int64_t kTicketBytes = 16;
int64_t sums_bytes(const pb_pairs* p) { return (int64_t)align_up((size_t)p->n_split * 4, 8) + (p->n_split ? p->n_chunks * 8 : 0); }
int64_t sums_bytes(const pb_groups* g) { return g->n_pieces * (int64_t)sizeof(PieceSums); }
// (a layout's scratch is the same whatever the objective)
int64_t scratch_bytes(const pb_pairs* p) { return kTicketBytes + sums_bytes(p) + n_parts_of(p) * (int64_t)sizeof(Part); }
int64_t scratch_bytes(const pb_groups* g) { return kTicketBytes + sums_bytes(g) + n_parts_of(g, false) * (int64_t)sizeof(Part); }
int64_t scratch_bytes(const pb_objective* o) {
    return o->kind == PB_OBJECTIVE_PREFERENCE ? scratch_bytes(o->pairs) : scratch_bytes(o->groups);
}
Totals totals_of(int64_t n_parts, int64_t sums, double scale, float* loss, float* kl, int64_t* clipped, char* scratch) {
    const bool want = loss || kl || clipped;
    return Totals{want ? reinterpret_cast<unsigned*>(scratch) : nullptr, reinterpret_cast<Part*>(scratch + kTicketBytes + sums),
                  (int)n_parts, scale, loss, kl, clipped};
}

// A launch; `early`: it may begin before the one in front of it on the stream has ended, and waits for that itself.
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), int64_t grid, int block, size_t smem, bool early, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = early ? 1 : 0;
    count_launch(1);
    return cudaLaunchKernelEx(&cfg, kernel, (P)args...);
}

// Whether a launch may begin before the kernel in front of it has ended.  (In a capture what is before it may be no kernel.)
bool early_allowed(cudaStream_t stream) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream, &status) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    return status == cudaStreamCaptureStatusNone;
}

// No rows: nothing to launch, all totals 0.
int no_totals(float* loss, float* kl, int64_t* clipped, cudaStream_t stream) {
    if (loss) PB_CUDA_TRY(cudaMemsetAsync(loss, 0, sizeof(*loss), stream));
    if (kl) PB_CUDA_TRY(cudaMemsetAsync(kl, 0, sizeof(*kl), stream));
    if (clipped) PB_CUDA_TRY(cudaMemsetAsync(clipped, 0, sizeof(*clipped), stream));
    return PB_OK;
}

template <typename T>
int launch_pairs(const pb_objective* o, const T* scores, T* grad, const Totals& totals, char* scratch, cudaStream_t stream) {
    const pb_pairs& p = *o->pairs;
    unsigned* counts = reinterpret_cast<unsigned*>(scratch + kTicketBytes);
    double* sums = reinterpret_cast<double*>(scratch + kTicketBytes + align_up((size_t)p.n_split * 4, 8));
    const PairArgs a{p, (float)o->beta, (float)(o->beta * 1.4426950408889634), (float)o->smoothing, (float)(0.5 / o->beta), o->scale * (o->squared ? 2.0 : o->beta), sums, counts};
    // It may be launched before the kernel in front of it has ended, and waits for that: 1.3 us less from one evaluation to the next
    // (of 18 for 2M pairs).  The SMs are full with its CTAs, so none of them waits where another should run; the kernels of groups
    // lose by it: CTAs that are early crowd on the SMs that are free first, 100 groups of 5 000 rows took 14 us for 10.
    const bool early = early_allowed(stream);
    if (o->squared)
        PB_CUDA_TRY(launch(pair_kernel<T, true>, n_parts_of(&p), kPairThreads, 0, early, stream, a, scores, grad, totals));
    else
        PB_CUDA_TRY(launch(pair_kernel<T, false>, n_parts_of(&p), kPairThreads, 0, early, stream, a, scores, grad, totals));
    return PB_OK;
}

template <typename T, int OP>
int launch_groups(const GroupArgs& a, const T* scores, T* out, const Totals& totals, char* scratch, cudaStream_t stream) {
    const pb_groups& g = a.g;
    int slot = 0;
    // (rows in order: four neighbouring ones to a thread, as one word where all arrays are on the border of one)
    const uintptr_t bits = (uintptr_t)a.target | (uintptr_t)a.advantage | (uintptr_t)a.old | (uintptr_t)a.reference;
    const bool words = bits % 16 == 0 && ((uintptr_t)scores | (uintptr_t)out) % (4 * sizeof(T)) == 0;
    bool early = false;  // the first launch begins when all before it on the stream is done, the others may overlap with it
    if (g.n_team_warps) {
        const int64_t grid = team_grid(&g, OP == kPolicy);
        PB_CUDA_TRY(launch(team_kernel<T, OP>, grid, kTeamThreads, 0, early, stream, a, slot, scores, out, totals));
        slot += (int)grid;
        early = true;
    }
    if (g.n_blocks) {
        // Threads of a group: as few as keep an SM busy, since each warp costs its group as much as five rows: 8 warps where an SM has
        // three groups, else 16.  Policies with 256 and 512 threads: 100 groups of 5 000 rows 13.5 and 12.0 us, 443 of them 20.4 and 24.2,
        // 600 of them 28.3 and 34.4, 1 000 of 2 000 rows 21.9 and 28.4.  On the wrong side of the rule: 443 groups of 500 rows (9.7 and
        // 14.9), 1 000 of 8 000 (73.6 and 66.4).  (`most`: the first place is rounded down; with a list of rows the last step's threads have
        // places that are not used.)
        const int threads = g.n_blocks >= 148 * 3 ? 256 : 512;
        const int most = (int)(g.block_rows + 7) / 4 * 4 + (g.rows ? threads * kBlockRows : 0);
        const size_t smem = OP == kLogProbs ? 0 : (size_t)most * 8;
        const int2* list = reinterpret_cast<const int2*>(g.blocks);
        auto block = [&](auto kernel) -> int {
            PB_TRY(allow_shared(kernel, smem));
            PB_CUDA_TRY(launch(kernel, block_grid(&g), threads, smem, early, stream, a, list, most, words, slot, scores, out, totals));
            return PB_OK;
        };
        if (block_grid(&g) < g.n_blocks)
            PB_TRY(g.rows ? block(block_kernel<T, OP, 256, false, true>) : block(block_kernel<T, OP, 256, true, true>));
        else if (threads == 256)
            PB_TRY(g.rows ? block(block_kernel<T, OP, 256, false, false>) : block(block_kernel<T, OP, 256, true, false>));
        else
            PB_TRY(g.rows ? block(block_kernel<T, OP, 512, false, false>) : block(block_kernel<T, OP, 512, true, false>));
        slot += (int)block_grid(&g);
        early = true;
    }
    if (g.n_pieces) {
        PieceSums* sums = reinterpret_cast<PieceSums*>(scratch + kTicketBytes);
        PB_CUDA_TRY(launch(piece_kernel<T, OP, kPieceMass>, g.n_pieces, kPieceThreads, 0, early, stream, a, sums, slot, scores, out, totals));
        if constexpr (OP == kPolicy)
            PB_CUDA_TRY(launch(piece_kernel<T, OP, kPieceTerms>, g.n_pieces, kPieceThreads, 0, true, stream, a, sums, slot, scores, out, totals));
        PB_CUDA_TRY(launch(piece_kernel<T, OP, kPieceOut>, g.n_pieces, kPieceThreads, 0, true, stream, a, sums, slot, scores, out, totals));
    }
    return PB_OK;
}

template <typename T>
int launch_objective(const pb_objective* o, const void* scores_, void* grad_, float* loss, float* kl, int64_t* clipped, void* scratch_,
                     cudaStream_t stream) {
    const T* scores = static_cast<const T*>(scores_);
    T* grad = static_cast<T*>(grad_);
    char* scratch = static_cast<char*>(scratch_);
    if (o->kind == PB_OBJECTIVE_PREFERENCE)
        return launch_pairs<T>(o, scores, grad, totals_of(n_parts_of(o->pairs), sums_bytes(o->pairs), o->scale, loss, kl, clipped, scratch), scratch,
                               stream);
    const double high = 1.0 + o->clip_high > kMostFactor ? INFINITY : o->clip_high;  // (beyond it nothing is cut off)
    const GroupArgs a{*o->groups, o->target, o->advantage, o->old, o->reference, split(log1p(high)), split(log1p(-o->clip_low)),
                      (float)(1.0 + high), (float)(1.0 - o->clip_low), (float)o->kl_coef, (float)o->scale};
    const Totals totals = totals_of(n_parts_of(o->groups, o->kind == PB_OBJECTIVE_POLICY), sums_bytes(o->groups), o->scale, loss, kl, clipped,
                                    scratch);
    if (o->kind == PB_OBJECTIVE_CHOICE) return launch_groups<T, kChoice>(a, scores, grad, totals, scratch, stream);
    return launch_groups<T, kPolicy>(a, scores, grad, totals, scratch, stream);
}

int check_scratch(const void* workspace, int64_t given, int64_t need) {
    PB_REQUIRE(workspace != nullptr && (uintptr_t)workspace % 16 == 0, "workspace is null or not aligned");
    if (given < need) {
        set_error("objective workspace: %lld bytes given, %lld needed", (long long)given, (long long)need);
        return PB_ERR_WORKSPACE;
    }
    return PB_OK;
}

// (a row's score is read for other rows too, after its own result is written)
int check_apart(const void* scores, const void* out, int64_t n_rows, int64_t score_type) {
    const uintptr_t a = (uintptr_t)scores, b = (uintptr_t)out, bytes = (uintptr_t)n_rows * (score_type == PB_SCORE_F32 ? 4 : 2);
    PB_REQUIRE(a + bytes <= b || b + bytes <= a, "what is written overlaps the scores");
    return PB_OK;
}

}  // namespace

int objective_gradient(const pb_objective* o, const void* scores, int64_t score_type, void* grad, float* loss, float* kl,
                       int64_t* clipped, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
    PB_REQUIRE(score_type >= PB_SCORE_F32 && score_type <= PB_SCORE_BF16, "unknown type of scores %lld", (long long)score_type);
    if (n_rows_of(o) == 0) return no_totals(loss, kl, clipped, stream);
    PB_REQUIRE(scores && grad, "scores or gradient is null");
    PB_TRY(objective_check_workspace(o, workspace, workspace_bytes));
    PB_TRY(check_apart(scores, grad, n_rows_of(o), score_type));
    if (score_type == PB_SCORE_F32) return launch_objective<float>(o, scores, grad, loss, kl, clipped, workspace, stream);
    if (score_type == PB_SCORE_F16) return launch_objective<__half>(o, scores, grad, loss, kl, clipped, workspace, stream);
    return launch_objective<__nv_bfloat16>(o, scores, grad, loss, kl, clipped, workspace, stream);
}

int objective_check_workspace(const pb_objective* o, const void* workspace, int64_t workspace_bytes) {
    return check_scratch(workspace, workspace_bytes, scratch_bytes(o));
}

int objective_check(const pb_objective* o, int64_t n_rows) {
    PB_TRY(check_objective(o));
    PB_REQUIRE(n_rows < 0 || n_rows_of(o) == n_rows, "the objective has %lld rows, the state %lld", (long long)n_rows_of(o),
               (long long)n_rows);
    return PB_OK;
}

}  // namespace pb

using namespace pb;

extern "C" int64_t pb_objective_struct_bytes(int64_t which) {
    return which == 0 ? (int64_t)sizeof(pb_pairs) : which == 1 ? (int64_t)sizeof(pb_groups) : (int64_t)sizeof(pb_objective);
}

extern "C" int64_t pb_objective_workspace_bytes(const pb_objective* o) {
    if (check_objective(o)) return PB_ERR_ARG;
    return scratch_bytes(o);
}

extern "C" int pb_objective_evaluate(const pb_objective* o, const void* scores, int64_t score_type, void* grad, float* loss,
                                     float* kl, int64_t* clipped, void* workspace, int64_t workspace_bytes, void* stream) {
    NvtxRange nvtx("pb.objective kind=%lld", o ? (long long)o->kind : -1);
    PB_TRY(objective_check(o, -1));
    return objective_gradient(o, scores, score_type, grad, loss, kl, clipped, workspace, workspace_bytes, (cudaStream_t)stream);
}

extern "C" int64_t pb_group_log_probs_bytes(const pb_groups* g) {
    if (check_groups(g)) return PB_ERR_ARG;
    return g->n_pieces ? kTicketBytes + sums_bytes(g) : 0;
}

extern "C" int pb_group_log_probs(const pb_groups* g, const void* scores, int64_t score_type, void* out, void* workspace,
                                  int64_t workspace_bytes, void* stream_) {
    NvtxRange nvtx("pb.group_log_probs n=%lld", g ? (long long)g->n_rows : -1);
    PB_TRY(check_groups(g));
    PB_REQUIRE(score_type >= PB_SCORE_F32 && score_type <= PB_SCORE_BF16, "unknown type of scores %lld", (long long)score_type);
    if (g->n_rows == 0) return PB_OK;
    PB_REQUIRE(scores && out, "scores or output is null");
    if (g->n_pieces) PB_TRY(check_scratch(workspace, workspace_bytes, kTicketBytes + sums_bytes(g)));
    PB_TRY(check_apart(scores, out, g->n_rows, score_type));
    cudaStream_t stream = (cudaStream_t)stream_;
    GroupArgs a{};
    a.g = *g;
    const Totals none{};
    char* scratch = static_cast<char*>(workspace);
    if (score_type == PB_SCORE_F32)
        return launch_groups<float, kLogProbs>(a, static_cast<const float*>(scores), static_cast<float*>(out), none, scratch, stream);
    if (score_type == PB_SCORE_F16)
        return launch_groups<__half, kLogProbs>(a, static_cast<const __half*>(scores), static_cast<__half*>(out), none, scratch, stream);
    return launch_groups<__nv_bfloat16, kLogProbs>(a, static_cast<const __nv_bfloat16*>(scores), static_cast<__nv_bfloat16*>(out), none, scratch, stream);
}
