// Losses on the scores of rows with their gradients: preferences between two rows, choices among the
// rows of a group, and a clipped policy over groups (include/packboost_b200.h has the formulas).
//
// Sums over a row's pairs, over a group and over the whole table are taken in a fixed order, so a
// result does not change from run to run.  Within a group, the log of the sum of exponentials and the
// differences of log-probabilities are held in 64 bits: whether a policy's ratio is beyond its border
// must not hang on the rounding of a sum over a whole era, and with a reference near the policy the
// difference of the two log-probabilities is all there is.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace pb {

namespace {

// ---- scores of either type ---------------------------------------------------------------------

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// What a CTA leaves of the three totals; finish_kernel adds them up.
struct Part {
    double loss, kl, clipped;
};

__device__ __forceinline__ double warp_sum(double v) {
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    return v;
}

__device__ __forceinline__ float warp_max(float v) {
    for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
    return v;
}

// The sum over the CTA, the same in every thread.  `scratch` holds a value per warp.
__device__ __forceinline__ double block_sum(double v, double* scratch) {
    v = warp_sum(v);
    __syncthreads();  // (the scratch may still be read from the call before)
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t += scratch[w];
    return t;
}

constexpr int kFinishThreads = 512;

__global__ void __launch_bounds__(kFinishThreads) finish_kernel(const Part* __restrict__ parts, int64_t n, double scale,
                                                                float* loss, float* kl, int64_t* clipped) {
    __shared__ double scratch[kFinishThreads / 32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Part t{0.0, 0.0, 0.0};
    for (int64_t i = threadIdx.x; i < n; i += kFinishThreads) {
        t.loss += parts[i].loss;
        t.kl += parts[i].kl;
        t.clipped += parts[i].clipped;
    }
    t.loss = block_sum(t.loss, scratch);
    t.kl = block_sum(t.kl, scratch);
    t.clipped = block_sum(t.clipped, scratch);
    if (threadIdx.x == 0) {
        if (loss) *loss = (float)(t.loss * scale);
        if (kl) *kl = (float)(t.kl * scale);
        if (clipped) *clipped = (int64_t)t.clipped;
    }
}

// ---- pairs ---------------------------------------------------------------------------------------

struct PairArgs {
    pb_pairs p;
    float beta, smoothing, half_tau;  // half_tau: 1 / (2 beta)
    float factor;                     // of the sum of a row's terms: scale and what the terms leave out
};

// log(1 + e) for e in [0, 1]: with s = e / (2 + e), 2 atanh(s), s <= 1/3; the term after the last one kept is
// s^14 / 15 of the sum, below 2^-26.
__device__ __forceinline__ float log1p_of(float e) {
    const float s = __fdividef(e, 2.f + e), q = s * s;
    float p = fmaf(q, 1.f / 13.f, 1.f / 11.f);
    p = fmaf(q, p, 1.f / 9.f);
    p = fmaf(q, p, 1.f / 7.f);
    p = fmaf(q, p, 1.f / 5.f);
    p = fmaf(q, p, 1.f / 3.f);
    return 2.f * fmaf(s * q, p, s);
}

// Derivative with respect to d, without the factor 2 (squared) or beta, of a pair whose (reference-corrected)
// score difference is d; its loss, if wanted.
template <bool SQUARED>
__device__ __forceinline__ float pair_slope(const PairArgs& a, float d, bool want, float* loss) {
    if (SQUARED) {
        const float off = d - a.half_tau;
        *loss = off * off;
        return off;
    }
    // softplus(-z) + e z has the derivative e - sigmoid(-z)
    const float z = a.beta * d;
    const float e = expf(-fabsf(z));
    if (want) *loss = fmaxf(-z, 0.f) + log1p_of(e) + (a.smoothing != 0.f ? a.smoothing * z : 0.f);
    return a.smoothing - __fdividef(z > 0.f ? e : 1.f, 1.f + e);
}

// A thread takes eight neighbouring items, a CTA a tile of them at a time and a run of tiles in all; a row's
// items are neighbours, so a segmented scan over the threads gives every row its sum however many items it
// has: rows of one pair and a row that all pairs share cost the same per item.  Rows cut by the border of
// two runs leave a piece on either side, which pair_finish_kernel adds up in order.
constexpr int kPairThreads = 128;
constexpr int kPairItems = 8;
constexpr int kPairTile = kPairThreads * kPairItems;
static_assert(kPairTile == PB_PAIR_TILE && kPairItems == PB_PAIR_ITEMS, "layout of the items");

struct PairPieces {
    double *lead, *tail, *loss;  // per run: sums before its first row starts and after its last one has
};

template <typename T, bool SQUARED>
__global__ void __launch_bounds__(kPairThreads) pair_kernel(PairArgs a, const T* __restrict__ scores, T* __restrict__ grad,
                                                            PairPieces pieces, double scale, float* loss_out) {
    __shared__ double s_tail[2][kPairThreads / 32];
    __shared__ int s_seen[2][kPairThreads / 32];
    __shared__ double scratch[kPairThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t tile0 = (int64_t)blockIdx.x * a.p.run_tiles;
    const int64_t tile1 = min(tile0 + a.p.run_tiles, a.p.n_items / kPairTile);
    const bool want = pieces.loss || loss_out;
    double carry = 0.0, loss = 0.0;  // carry: of the row that is open where the tile begins
    bool seen = false;               // a row has started in this run
    int last_row = 0;
    for (int64_t tile = tile0; tile < tile1; ++tile) {
        const int64_t chunk = tile * kPairThreads + threadIdx.x, i0 = chunk * kPairItems;
        uint32_t word[kPairItems];
        float off[kPairItems], w[kPairItems];
        *reinterpret_cast<uint4*>(word) = *reinterpret_cast<const uint4*>(a.p.other + i0);
        *reinterpret_cast<uint4*>(word + 4) = *reinterpret_cast<const uint4*>(a.p.other + i0 + 4);
        int row = a.p.chunk_rows[chunk];
        const uint32_t heads = a.p.chunk_heads[chunk];
        if (a.p.offset) {
            *reinterpret_cast<float4*>(off) = *reinterpret_cast<const float4*>(a.p.offset + i0);
            *reinterpret_cast<float4*>(off + 4) = *reinterpret_cast<const float4*>(a.p.offset + i0 + 4);
        } else {
#pragma unroll
            for (int u = 0; u < kPairItems; ++u) off[u] = 0.f;
        }
        if (a.p.weight) {
            *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(a.p.weight + i0);
            *reinterpret_cast<float4*>(w + 4) = *reinterpret_cast<const float4*>(a.p.weight + i0 + 4);
        } else {
#pragma unroll
            for (int u = 0; u < kPairItems; ++u) w[u] = 1.f;
        }
        float term[kPairItems];
        {
            T own[kPairItems], other[kPairItems];
            int r = row;
#pragma unroll
            for (int u = 0; u < kPairItems; ++u) {
                other[u] = scores[word[u] & 0x7FFFFFFFu];
                if (u > 0) r += (int)((heads >> u) & 1u);
                own[u] = scores[r];
            }
            r = row;
            float chunk_loss = 0.f;
#pragma unroll
            for (int u = 0; u < kPairItems; ++u) {
                if (u > 0) r += (int)((heads >> u) & 1u);
                const uint32_t sign = word[u] & 0x80000000u;
                const float d = (to_f32(own[u]) - to_f32(other[u])) - off[u];
                float l;
                float t = pair_slope<SQUARED>(a, __uint_as_float(__float_as_uint(d) ^ sign), want, &l);
                t = __uint_as_float(__float_as_uint(t) ^ sign) * w[u];
                // (an item of a row with itself fills a row without pairs, or the last tile)
                term[u] = (int)(word[u] ^ sign) != r ? t : 0.f;
                if (want && !sign && (int)word[u] != r) chunk_loss = fmaf(w[u], l, chunk_loss);
            }
            loss += (double)chunk_loss;
        }
        const int row_open = row - (int)(heads & 1u);  // the row that is open where the chunk begins
        float acc = 0.f, lead = 0.f;
        bool any = false;                              // a row has started in this chunk
#pragma unroll
        for (int u = 0; u < kPairItems; ++u) {
            if ((heads >> u) & 1u) {
                if (any)
                    grad[row] = from_f32<T>(acc * a.factor);
                else
                    lead = acc;
                if (u > 0) ++row;
                any = true;
                acc = 0.f;
            }
            acc += term[u];
        }
        if (!any) lead = acc;

        // inclusive scan of what is open at the end of each chunk
        const uint32_t mask = __ballot_sync(0xFFFFFFFFu, any);
        const uint32_t below = mask & (0xFFFFFFFFu >> (31 - lane));
        const int reach = below ? lane - (31 - __clz(below)) : lane;
        double v = (double)(any ? acc : lead);
        for (int d = 1; d < 32; d <<= 1) {
            const double o = __shfl_up_sync(0xFFFFFFFFu, v, d);
            if (d <= reach) v += o;
        }
        const int b = (int)(tile - tile0) & 1;
        if (lane == 31) {
            s_tail[b][warp] = v;
            s_seen[b][warp] = mask != 0u;
        }
        __syncthreads();  // (two buffers: the other one was last read before this barrier's predecessor)
        double before = carry;  // open where this warp begins
        bool started = seen;
        for (int k = 0; k < warp; ++k) {
            before = s_seen[b][k] ? s_tail[b][k] : before + s_tail[b][k];
            started |= s_seen[b][k] != 0;
        }
        double open = __shfl_up_sync(0xFFFFFFFFu, v, 1);
        if (lane == 0) open = 0.0;
        const uint32_t prior = mask & ((1u << lane) - 1u);
        if (!prior) open += before;
        if (any) {
            const double sum = open + (double)lead;
            if (started || prior)
                grad[row_open] = from_f32<T>((float)sum * a.factor);
            else if (pieces.lead)   // (there are several runs)
                pieces.lead[blockIdx.x] = sum;
        }
        for (int k = 0; k < kPairThreads / 32; ++k) {
            carry = s_seen[b][k] ? s_tail[b][k] : carry + s_tail[b][k];
            seen |= s_seen[b][k] != 0;
        }
        last_row = row;
    }
    if (threadIdx.x == kPairThreads - 1) {
        // the row that is open at the end: done, or continued in the next run
        const int64_t next = tile1 * kPairThreads;
        const bool ends = tile1 == a.p.n_items / kPairTile || (a.p.chunk_heads[next] & 1u);
        if (seen && ends) grad[last_row] = from_f32<T>((float)carry * a.factor);
        if (pieces.lead) {
            if (!seen) pieces.lead[blockIdx.x] = carry;
            pieces.tail[blockIdx.x] = carry;
        }
    }
    if (want) {
        loss = block_sum(loss, scratch);
        if (threadIdx.x == 0) {
            if (loss_out)  // one run: nothing else to add
                *loss_out = (float)(loss * scale);
            else
                pieces.loss[blockIdx.x] = loss;
        }
    }
}

// Rows cut by borders of runs: a warp each; the loss: the last CTA.
constexpr int kPairFinishThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kPairFinishThreads) pair_finish_kernel(PairArgs a, PairPieces pieces, int64_t n_runs,
                                                                         double scale, T* __restrict__ grad, float* loss_out) {
    __shared__ double scratch[kPairFinishThreads / 32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (blockIdx.x == gridDim.x - 1) {
        if (!loss_out) return;
        double t = 0.0;
        for (int64_t i = threadIdx.x; i < n_runs; i += kPairFinishThreads) t += pieces.loss[i];
        t = block_sum(t, scratch);
        if (threadIdx.x == 0) *loss_out = (float)(t * scale);
        return;
    }
    const int64_t k = (int64_t)blockIdx.x * (kPairFinishThreads / 32) + (threadIdx.x >> 5);
    if (k >= a.p.n_cuts) return;
    const int lane = threadIdx.x & 31;
    const int row = a.p.cuts[3 * k], first = a.p.cuts[3 * k + 1], last = a.p.cuts[3 * k + 2];
    double t = 0.0;
    for (int r = first + 1 + lane; r <= last; r += 32) t += pieces.lead[r];
    t = warp_sum(t) + pieces.tail[first];
    if (lane == 0) grad[row] = from_f32<T>((float)t * a.factor);
}

// A launch; `early`: it may begin before the one in front of it on the stream has ended, and waits for that itself.
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, bool early, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = early ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, (P)args...);
}

int64_t n_runs_of(const pb_pairs* p) {
    return p->n_items ? (p->n_items / kPairTile + p->run_tiles - 1) / p->run_tiles : 0;
}

template <typename T>
int launch_pairs(const PairArgs& a, bool squared, double scale, const T* scores, T* grad, float* loss, double* scratch, cudaStream_t stream) {
    const int64_t n_runs = n_runs_of(&a.p);
    if (n_runs == 0) {
        if (loss) PB_CUDA_TRY(cudaMemsetAsync(loss, 0, 4, stream));
        return PB_OK;
    }
    const bool one = n_runs == 1;
    PairPieces pieces{nullptr, nullptr, nullptr};
    if (!one) pieces = PairPieces{scratch, scratch + n_runs, loss ? scratch + 2 * n_runs : nullptr};
    if (squared)
        pair_kernel<T, true><<<(unsigned)n_runs, kPairThreads, 0, stream>>>(a, scores, grad, pieces, scale, one ? loss : nullptr);
    else
        pair_kernel<T, false><<<(unsigned)n_runs, kPairThreads, 0, stream>>>(a, scores, grad, pieces, scale, one ? loss : nullptr);
    count_launch(1);
    if (!one && (loss || a.p.n_cuts)) {
        const int64_t grid = (a.p.n_cuts + kPairFinishThreads / 32 - 1) / (kPairFinishThreads / 32) + 1;
        PB_CUDA_TRY(launch_after(pair_finish_kernel<T>, (unsigned)grid, kPairFinishThreads, 0, true, stream, a, pieces, n_runs, scale,
                                 grad, loss));
        count_launch(1);
    }
    return PB_OK;
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

// a - b without rounding, plus a small `lo`
__device__ __forceinline__ Pair32 difference(float a, float b, float lo) {
    const float t = a - b, v = t - a;
    const float err = (a - (t - v)) - (b + v);
    return Pair32{t, fabsf(t) <= 3.402823466e38f ? err + lo : 0.f};  // (nothing to correct at infinity)
}

__host__ __device__ __forceinline__ Pair32 split(double x) {
    const float hi = (float)x, lo = (float)(x - (double)hi);
    return Pair32{hi, lo - lo == 0.f ? lo : 0.f};
}

__device__ __forceinline__ float exp_of(Pair32 x) {
    const float e = expf(x.hi);
    return fmaf(e, x.lo, e);
}

struct GroupArgs {
    pb_groups g;
    const float *target, *advantage, *old, *reference;
    Pair32 log_high, log_low;  // borders of the log of the ratio
    float bound_high, bound_low;
    float kl_coef;
    float scale;
};

struct RowInputs {
    float main, old, reference;  // main: target, or advantage
};

// What a row has and gives: its gradient is (fixed + p * share) * scale, the share being the group's sum.
struct RowTerm {
    float fixed, p;
    float share;  // what the row adds to the group's
    float loss, kl;
    int clipped;
};

template <int OP>
__device__ __forceinline__ RowTerm row_term(const GroupArgs& a, float s, Pair32 lse, const RowInputs& in) {
    RowTerm t{0.f, 0.f, 0.f, 0.f, 0.f, 0};
    const bool live = s != -INFINITY;
    const Pair32 l = difference(s, lse.hi, -lse.lo);
    if (live) t.p = exp_of(l);
    if (OP == kChoice) {
        t.fixed = -in.main;
        t.share = in.main;
    } else if (live) {
        const float adv = in.main;
        if (adv != 0.f) {
            const Pair32 x = difference(l.hi, in.old, l.lo);
            const Pair32 edge = adv > 0.f ? a.log_high : a.log_low;
            const float past = (x.hi - edge.hi) + (x.lo - edge.lo);
            const bool beyond = adv > 0.f ? past > 0.f : past < 0.f;
            t.loss = -adv * (beyond ? (adv > 0.f ? a.bound_high : a.bound_low) : exp_of(x));
            t.fixed = beyond ? 0.f : t.loss;
            t.clipped = beyond ? 1 : 0;
        }
        t.share = -t.fixed;
        if (a.reference) {
            const Pair32 gap = difference(l.hi, in.reference, l.lo);
            t.kl = t.p * (gap.hi + gap.lo);
            t.fixed = fmaf(a.kl_coef, t.kl, t.fixed);
            t.share = fmaf(-a.kl_coef, t.kl, t.share);
        }
    }
    return t;
}

__device__ __forceinline__ float row_gradient(const GroupArgs& a, float fixed, float p, float share) {
    return (p == 0.f ? fixed : fmaf(p, share, fixed)) * a.scale;  // (the share may be infinite)
}

// What the loss of a choice gets from a row, in 64 bits: the terms of a group may be of very different size.
__device__ __forceinline__ double choice_loss(float s, double lse, float target) {
    return target != 0.f ? (double)target * (lse - (double)s) : 0.0;
}

__device__ __forceinline__ double log_sum(float m, double z) {
    return z == 0.0 ? 0.0 : (double)m + log(z);  // (nothing left in the group: every p is 0)
}

// exp(s - m), 0 for a masked row
__device__ __forceinline__ double mass_of(float s, float m) { return s == -INFINITY ? 0.0 : exp((double)s - (double)m); }

// Where a CTA puts its totals; the only CTA of an evaluation puts the outputs.
struct Totals {
    Part* parts;  // null: not wanted
    double scale;
    float *loss, *kl;
    int64_t* clipped;
    int only;
    float kl_coef;
};
__device__ __forceinline__ void put_totals(const Totals& out, int slot, double loss, double kl, double clipped) {
    loss += (double)out.kl_coef * kl;
    if (out.only) {
        if (out.loss) *out.loss = (float)(loss * out.scale);
        if (out.kl) *out.kl = (float)(kl * out.scale);
        if (out.clipped) *out.clipped = (int64_t)clipped;
    } else {
        out.parts[slot] = Part{loss, kl, clipped};
    }
}
// (all threads of the CTA)
template <int OP>
__device__ __forceinline__ void put_cta_totals(const Totals& out, int slot, double loss, double kl, int clipped, double* scratch) {
    if (!out.parts && !out.only) return;
    loss = block_sum(loss, scratch);
    if (OP == kPolicy) {
        kl = block_sum(kl, scratch);
        const double c = block_sum((double)clipped, scratch);
        if (threadIdx.x == 0) put_totals(out, slot, loss, kl, c);
    } else if (threadIdx.x == 0) {
        put_totals(out, slot, loss, 0.0, 0.0);
    }
}

template <int OP>
__device__ __forceinline__ RowInputs row_inputs(const GroupArgs& a, int r) {
    RowInputs v;
    v.main = OP == kChoice ? a.target[r] : a.advantage[r];
    v.old = OP == kPolicy ? a.old[r] : 0.f;
    v.reference = OP == kPolicy && a.reference ? a.reference[r] : 0.f;
    return v;
}

// The kernels of one evaluation write different rows, so the next may start while one runs (its CTAs fill SMs that the
// last of this one's leave idle); each waits for the one before it at its end, so that the last one's end is
// everyone's.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- short groups: lanes of a warp ----
//
// 1, 2, 4 ... 32 neighbouring lanes have a group, ROWS rows each; a warp's groups are of one class (so many lanes), and
// sums over a group are shuffles within its lanes.  Of up to 4 x lanes rows at least half are there; one launch
// takes all classes.
constexpr int kTeamThreads = 256;

template <typename T, int OP, int ROWS>
__global__ void __launch_bounds__(kTeamThreads) team_kernel(GroupArgs a, const int2* __restrict__ teams, const int first_class,
                                                            int64_t n_warps, int slot0, const T* __restrict__ scores,
                                                            T* __restrict__ out, Totals totals) {
    __shared__ double scratch[kTeamThreads / 32];
    let_next_start();
    const int lane = threadIdx.x & 31;
    double loss = 0.0, kl = 0.0;
    int clipped = 0;
    for (int64_t w = ((int64_t)blockIdx.x * kTeamThreads + threadIdx.x) >> 5; w < n_warps; w += (int64_t)gridDim.x * (kTeamThreads / 32)) {
        // the class of this warp, and its first team
        int c = first_class;
        int64_t left = w, team = 0;
        while (left >= a.g.team_warps[c]) {
            left -= a.g.team_warps[c];
            team += a.g.team_warps[c] * (32 >> min(c, 5));
            ++c;
        }
        c = min(c, 5);
        const int lanes = 1 << c, me = lane & (lanes - 1);
        const int2 group = teams[team + left * (32 >> c) + (lane >> c)];
        int r[ROWS];
        float s[ROWS];
        RowInputs in[ROWS];
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            const int i = u * lanes + me;
            r[u] = i < group.y ? group.x + i : -1;
            if (a.g.rows && r[u] >= 0) r[u] = a.g.rows[r[u]];
        }
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            s[u] = -INFINITY;
            in[u] = RowInputs{0.f, 0.f, 0.f};
            if (r[u] >= 0) {
                s[u] = to_f32(scores[r[u]]);
                if (OP != kLogProbs) in[u] = row_inputs<OP>(a, r[u]);
            }
        }
        float m = s[0];
#pragma unroll
        for (int u = 1; u < ROWS; ++u) m = fmaxf(m, s[u]);
        for (int d = lanes >> 1; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
        double z = 0.0;
#pragma unroll
        for (int u = 0; u < ROWS; ++u) z += mass_of(s[u], m);
        for (int d = lanes >> 1; d > 0; d >>= 1) z += __shfl_xor_sync(0xFFFFFFFFu, z, d);
        const double lse64 = log_sum(m, z);
        const Pair32 lse = split(lse64);
        if (OP == kLogProbs) {
#pragma unroll
            for (int u = 0; u < ROWS; ++u)
                if (r[u] >= 0) {
                    const Pair32 l = difference(s[u], lse.hi, -lse.lo);
                    out[r[u]] = from_f32<T>(l.hi + l.lo);
                }
            continue;
        }
        float fixed[ROWS], part = 0.f, part_loss = 0.f, part_kl = 0.f;
        double part64 = 0.0;
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            if (r[u] >= 0) {
                if (OP == kChoice) loss += choice_loss(s[u], lse64, in[u].main);
                const RowTerm t = row_term<OP>(a, s[u], lse, in[u]);
                s[u] = t.p;
                fixed[u] = t.fixed;
                part += t.share;
                part_loss += t.loss;
                part_kl += t.kl;
                clipped += t.clipped;
            }
            if ((u & 3) == 3) {  // (four terms in 32 bits, the sums of fours in 64)
                part64 += (double)part;
                if (OP == kPolicy) {
                    loss += (double)part_loss;
                    kl += (double)part_kl;
                }
                part = part_loss = part_kl = 0.f;
            }
        }
        for (int d = lanes >> 1; d > 0; d >>= 1) part64 += __shfl_xor_sync(0xFFFFFFFFu, part64, d);
        const float share = (float)part64;
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
            if (r[u] >= 0) out[r[u]] = from_f32<T>(row_gradient(a, fixed[u], s[u], share));
    }
    if (OP != kLogProbs) put_cta_totals<OP>(totals, slot0 + blockIdx.x, loss, kl, clipped, scratch);
    wait_for_previous();
}

// ---- groups that a CTA holds ----
//
// The rows of a group stay in the shared memory of one CTA, each thread using the words it filled itself: the
// inputs that the gradient needs are on their way there (cp.async) while the scores are summed.
__device__ __forceinline__ void copy_word(float* to, const float* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from));
}

// Largest score and log of the sum of exponentials over the CTA, from the threads' own ones.
template <int THREADS>
__device__ __forceinline__ double cta_log_sum(float m, double z, float* s_m, double* s_z) {
    float wm = warp_max(m);
    z = z == 0.0 ? 0.0 : z * exp((double)m - (double)wm);
    z = warp_sum(z);
    if ((threadIdx.x & 31) == 0) {
        s_m[threadIdx.x >> 5] = wm;
        s_z[threadIdx.x >> 5] = z;
    }
    __syncthreads();
    constexpr int kWarps = THREADS / 32;
    const int k = threadIdx.x & 31;
    wm = k < kWarps ? s_m[k] : -INFINITY;
    z = k < kWarps ? s_z[k] : 0.0;
    const float all = warp_max(wm);
    z = z == 0.0 ? 0.0 : z * exp((double)wm - (double)all);
    return log_sum(all, warp_sum(z));
}

template <int THREADS>
__device__ __forceinline__ double cta_sum(double v, double* scratch) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    const int k = threadIdx.x & 31;
    return warp_sum(k < THREADS / 32 ? scratch[k] : 0.0);
}

template <typename T, int OP, int THREADS>
__global__ void __launch_bounds__(THREADS) held_kernel(GroupArgs a, const int2* __restrict__ list, int most, int slot0,
                                                       const T* __restrict__ scores, T* __restrict__ out, Totals totals) {
    extern __shared__ float held[];  // scores (then p) | main (then fixed) | old | reference, `most` each
    __shared__ float s_m[THREADS / 32];
    __shared__ double s_z[THREADS / 32], scratch[THREADS / 32];
    let_next_start();
    const int2 group = list[blockIdx.x];
    const int begin = group.x, n = group.y;
    float* const h_main = held + most;
    float* const h_old = held + 2 * most;
    float* const h_ref = held + 3 * most;
    auto row_of = [&](int i) { return a.g.rows ? a.g.rows[begin + i] : begin + i; };
    if (OP != kLogProbs) {
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const int r = row_of(i);
            copy_word(h_main + i, (OP == kChoice ? a.target : a.advantage) + r);
            if (OP == kPolicy) {
                copy_word(h_old + i, a.old + r);
                if (a.reference) copy_word(h_ref + i, a.reference + r);
            }
        }
        asm volatile("cp.async.commit_group;");
    }
    float m = -INFINITY;
    {
        constexpr int kAhead = 8;
        for (int i0 = threadIdx.x; i0 < n; i0 += THREADS * kAhead) {
            float v[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int i = i0 + u * THREADS;
                v[u] = i < n ? to_f32(scores[row_of(i)]) : -INFINITY;
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int i = i0 + u * THREADS;
                m = fmaxf(m, v[u]);
                if (i < n) held[i] = v[u];
            }
        }
    }
    double z = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += THREADS) z += mass_of(held[i], m);
    const double lse64 = cta_log_sum<THREADS>(m, z, s_m, s_z);
    const Pair32 lse = split(lse64);
    if (OP == kLogProbs) {
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const Pair32 l = difference(held[i], lse.hi, -lse.lo);
            out[row_of(i)] = from_f32<T>(l.hi + l.lo);
        }
        wait_for_previous();
        return;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    double part = 0.0, loss = 0.0, kl = 0.0;
    int clipped = 0;
    for (int i0 = threadIdx.x; i0 < n; i0 += THREADS * 4) {
        float p4 = 0.f, l4 = 0.f, k4 = 0.f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * THREADS;
            if (i < n) {
                const float s = held[i];
                const RowInputs in{h_main[i], OP == kPolicy ? h_old[i] : 0.f, OP == kPolicy && a.reference ? h_ref[i] : 0.f};
                if (OP == kChoice) loss += choice_loss(s, lse64, in.main);
                const RowTerm t = row_term<OP>(a, s, lse, in);
                held[i] = t.p;
                h_main[i] = t.fixed;
                p4 += t.share;
                l4 += t.loss;
                k4 += t.kl;
                clipped += t.clipped;
            }
        }
        part += (double)p4;
        if (OP == kPolicy) {
            loss += (double)l4;
            kl += (double)k4;
        }
    }
    const float share = (float)cta_sum<THREADS>(part, scratch);
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += THREADS) out[row_of(i)] = from_f32<T>(row_gradient(a, h_main[i], held[i], share));
    put_cta_totals<OP>(totals, slot0 + blockIdx.x, loss, kl, clipped, scratch);
    wait_for_previous();
}

// ---- long groups: many CTAs each ----
//
// Pieces of PB_PIECE_ROWS rows; the sums of a group's pieces go through memory from one launch to the next: sums of
// exponentials, then shares, then the gradient.  The rows are read again each time, from L2 mostly.
struct PieceSums {
    double z, share;
    float m, unused;
};
constexpr int kPieceThreads = 512;
constexpr int kPieceRows = PB_PIECE_ROWS / kPieceThreads;
enum PieceStep { kPieceMass, kPieceTerms, kPieceOut };

template <typename T, int OP, int STEP>
__global__ void __launch_bounds__(kPieceThreads) piece_kernel(GroupArgs a, PieceSums* __restrict__ pieces, int slot0,
                                                              const T* __restrict__ scores, T* __restrict__ out, Totals totals) {
    constexpr int THREADS = kPieceThreads, ROWS = kPieceRows;
    __shared__ float s_m[THREADS / 32];
    __shared__ double s_z[THREADS / 32], scratch[THREADS / 32];
    let_next_start();
    if (STEP == kPieceMass) wait_for_previous();
    const int4 piece = reinterpret_cast<const int4*>(a.g.pieces)[blockIdx.x];
    const int begin = piece.x, n = piece.y, first = piece.z, count = piece.w;  // (first, count: the group's pieces)
    int r[ROWS];
    float s[ROWS];
    RowInputs in[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        const int i = u * THREADS + threadIdx.x;
        r[u] = i < n ? begin + i : -1;
        if (a.g.rows && r[u] >= 0) r[u] = a.g.rows[r[u]];
    }
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        s[u] = -INFINITY;
        if (r[u] >= 0) {
            s[u] = to_f32(scores[r[u]]);
            if (OP != kLogProbs && STEP != kPieceMass) in[u] = row_inputs<OP>(a, r[u]);
        }
    }
    float m = -INFINITY;
    double z = 0.0;
    if (STEP == kPieceMass) {
#pragma unroll
        for (int u = 0; u < ROWS; ++u) m = fmaxf(m, s[u]);
#pragma unroll
        for (int u = 0; u < ROWS; ++u) z += mass_of(s[u], m);
        const float wm = warp_max(m);
        z = warp_sum(z == 0.0 ? 0.0 : z * exp((double)m - (double)wm));
        if ((threadIdx.x & 31) == 0) {
            s_m[threadIdx.x >> 5] = wm;
            s_z[threadIdx.x >> 5] = z;
        }
        __syncthreads();
        if (threadIdx.x < 32) {
            const float k = threadIdx.x < THREADS / 32 ? s_m[threadIdx.x] : -INFINITY;
            z = threadIdx.x < THREADS / 32 ? s_z[threadIdx.x] : 0.0;
            m = warp_max(k);
            z = warp_sum(z == 0.0 ? 0.0 : z * exp((double)k - (double)m));
            if (threadIdx.x == 0) {
                pieces[blockIdx.x].m = m;
                pieces[blockIdx.x].z = z;
            }
        }
        return;
    }
    wait_for_previous();   // (the rows' inputs do not come from the launch before, the sums do)
    for (int k = threadIdx.x; k < count; k += THREADS) m = fmaxf(m, pieces[first + k].m);
    for (int k = threadIdx.x; k < count; k += THREADS) {
        const double zk = pieces[first + k].z;
        if (zk != 0.0) z += zk * exp((double)pieces[first + k].m - (double)m);
    }
    const double lse64 = cta_log_sum<THREADS>(m, z, s_m, s_z);
    const Pair32 lse = split(lse64);
    if (OP == kLogProbs) {
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
            if (r[u] >= 0) {
                const Pair32 l = difference(s[u], lse.hi, -lse.lo);
                out[r[u]] = from_f32<T>(l.hi + l.lo);
            }
        return;
    }
    float share = 0.f;
    if (STEP == kPieceOut) {
        double sum = 0.0;
        for (int k = threadIdx.x; k < count; k += THREADS) sum += pieces[first + k].share;
        share = (float)cta_sum<THREADS>(sum, scratch);
    }
    double part = 0.0, loss = 0.0, kl = 0.0;
    int clipped = 0;
    float p4 = 0.f, l4 = 0.f, k4 = 0.f;
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        if (r[u] >= 0) {
            const RowTerm t = row_term<OP>(a, s[u], lse, in[u]);
            if (STEP == kPieceOut) {
                out[r[u]] = from_f32<T>(row_gradient(a, t.fixed, t.p, share));
            } else {
                if (OP == kChoice) loss += choice_loss(s[u], lse64, in[u].main);
                p4 += t.share;
                l4 += t.loss;
                k4 += t.kl;
                clipped += t.clipped;
            }
        }
        if (STEP == kPieceTerms && (u & 3) == 3) {
            part += (double)p4;
            if (OP == kPolicy) {
                loss += (double)l4;
                kl += (double)k4;
            }
            p4 = l4 = k4 = 0.f;
        }
    }
    if (STEP == kPieceTerms) {
        part = cta_sum<THREADS>(part, scratch);
        if (threadIdx.x == 0) pieces[blockIdx.x].share = part;
        put_cta_totals<OP>(totals, slot0 + blockIdx.x, loss, kl, clipped, scratch);
    }
}

// ---- launches ---------------------------------------------------------------------------------------

int check_groups(const pb_groups* g) {
    PB_REQUIRE(g != nullptr, "groups are null");
    PB_REQUIRE(g->n_rows >= 0 && g->n_rows < (1ll << 31) - 1, "n_rows=%lld out of range", (long long)g->n_rows);
    PB_REQUIRE(g->n_groups >= 0 && g->n_groups <= g->n_rows, "n_groups=%lld out of range", (long long)g->n_groups);
    PB_REQUIRE((g->n_groups == 0) == (g->n_rows == 0), "rows without a group");
    const int64_t most = (1ll << 31) - 1;
    int64_t warps = 0;
    for (int c = 0; c < 7; ++c) {
        PB_REQUIRE(g->team_warps[c] >= 0 && g->team_warps[c] < most, "team_warps[%d] is out of range", c);
        warps += g->team_warps[c];
    }
    PB_REQUIRE(g->n_medium >= 0 && g->n_large >= 0 && g->n_medium + g->n_large <= g->n_groups && g->n_pieces >= 0 && g->n_pieces < most,
               "counts of the groups' layout are out of range");
    PB_REQUIRE(g->n_medium == 0 || (g->medium_rows > 0 && g->medium_rows <= PB_MEDIUM_ROWS), "medium_rows is out of range");
    PB_REQUIRE(g->n_large == 0 || (g->large_rows > 0 && g->large_rows <= PB_LARGE_ROWS), "large_rows is out of range");
    PB_REQUIRE((warps == 0 || g->teams) && (g->n_medium + g->n_large == 0 || g->held) && (g->n_pieces == 0 || g->pieces),
               "a table of the groups' layout is null");
    PB_REQUIRE((uintptr_t)g->teams % 8 == 0 && (uintptr_t)g->held % 8 == 0 && (uintptr_t)g->pieces % 16 == 0,
               "tables of the groups' layout must be aligned");
    PB_REQUIRE(g->n_groups == 0 || warps + g->n_medium + g->n_large + g->n_pieces > 0, "the groups are not laid out");
    return PB_OK;
}

int check_objective(const pb_objective* o) {
    PB_REQUIRE(o != nullptr, "objective is null");
    PB_REQUIRE(isfinite(o->scale), "scale is not finite");
    if (o->kind == PB_OBJECTIVE_PREFERENCE) {
        const pb_pairs* p = o->pairs;
        PB_REQUIRE(p != nullptr, "pairs are null");
        PB_REQUIRE(p->n_rows >= 0 && p->n_rows < (1ll << 31) - 1, "n_rows=%lld out of range", (long long)p->n_rows);
        PB_REQUIRE(p->n_items >= 0 && p->n_items < (1ll << 31) - 1, "n_items=%lld out of range", (long long)p->n_items);
        PB_REQUIRE(p->n_items % kPairTile == 0 && (p->n_items == 0) == (p->n_rows == 0), "items are not laid out in tiles");
        PB_REQUIRE(p->n_items == 0 || (p->other && p->chunk_rows && p->chunk_heads && p->run_tiles >= 1),
                   "a table of the pairs' layout is null");
        PB_REQUIRE(p->n_cuts >= 0 && p->n_cuts <= p->n_items / kPairTile && (p->n_cuts == 0 || p->cuts), "cuts of the pairs' layout");
        PB_REQUIRE((uintptr_t)p->other % 16 == 0 && (uintptr_t)p->offset % 16 == 0 && (uintptr_t)p->weight % 16 == 0,
                   "items must be 16-byte aligned");
        PB_REQUIRE(o->beta > 0.0 && isfinite(o->beta), "beta must be positive");
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
    PB_REQUIRE(isfinite(o->kl_coef) && (o->reference || o->kl_coef == 0.0), "kl_coef needs a reference");
    return PB_OK;
}

int64_t n_rows_of(const pb_objective* o) {
    return o->kind == PB_OBJECTIVE_PREFERENCE ? o->pairs->n_rows : o->groups->n_rows;
}

// CTAs of the launch that takes all warps of short groups: what the SMs hold at once, or as many as there are warps.
constexpr int64_t kTeamGrid = 148 * 6;
int64_t team_grid(int64_t warps) { return warps == 0 ? 0 : warps / 8 + 1 < kTeamGrid ? (warps + 7) / 8 : kTeamGrid; }
int64_t team_warps(const pb_groups* g, int from, int to) {
    int64_t n = 0;
    for (int c = from; c < to; ++c) n += g->team_warps[c];
    return n;
}

int64_t n_group_parts(const pb_groups* g) {
    return team_grid(team_warps(g, 0, 6)) + team_grid(g->team_warps[6]) + g->n_medium + g->n_large + g->n_pieces;
}

// Scratch: the sums of pieces, then what the CTAs leave of the totals, if there are several.
int64_t group_scratch_bytes(const pb_groups* g, bool totals) {
    const int64_t n = n_group_parts(g);
    return (totals && n > 1 ? n * (int64_t)sizeof(Part) : 0) + g->n_pieces * (int64_t)sizeof(PieceSums);
}
int64_t scratch_bytes(const pb_objective* o) {
    if (o->kind == PB_OBJECTIVE_PREFERENCE) return n_runs_of(o->pairs) > 1 ? 3 * n_runs_of(o->pairs) * (int64_t)sizeof(double) : 0;
    return group_scratch_bytes(o->groups, true);
}

template <typename T, int OP>
int launch_groups(const GroupArgs& a, double scale, const void* scores_, void* out_, float* loss, float* kl, int64_t* clipped,
                  void* scratch, cudaStream_t stream) {
    const T* scores = static_cast<const T*>(scores_);
    T* out = static_cast<T*>(out_);
    const pb_groups& g = a.g;
    const int64_t n_parts = n_group_parts(&g);
    const bool want = loss || kl || clipped;
    PieceSums* const sums = static_cast<PieceSums*>(scratch);
    const Totals totals{want && n_parts > 1 ? reinterpret_cast<Part*>(sums + g.n_pieces) : nullptr, scale, loss, kl, clipped, want && n_parts == 1, a.kl_coef};
    const int2* teams = reinterpret_cast<const int2*>(g.teams);
    int slot = 0, launches = 0;
    // the first launch waits for what is before it on the stream, the others may overlap with the ones before
    auto launch = [&](auto kernel, int64_t grid, int block, size_t smem, auto... args) -> int {
        PB_TRY(allow_shared(kernel, smem));
        PB_CUDA_TRY(launch_after(kernel, (unsigned)grid, (unsigned)block, smem, launches > 0, stream, args...));
        ++launches;
        return PB_OK;
    };
    const int64_t small = team_warps(&g, 0, 6);
    if (small) {
        PB_TRY(launch(team_kernel<T, OP, 4>, team_grid(small), kTeamThreads, 0, a, teams, 0, small, slot, scores, out, totals));
        slot += (int)team_grid(small);
    }
    if (g.team_warps[6]) {
        int64_t before = 0;
        for (int c = 0; c < 6; ++c) before += g.team_warps[c] * (32 >> c);
        PB_TRY(launch(team_kernel<T, OP, 8>, team_grid(g.team_warps[6]), kTeamThreads, 0, a, teams + before, 6, g.team_warps[6], slot,
                      scores, out, totals));
        slot += (int)team_grid(g.team_warps[6]);
    }
    const int arrays = OP == kLogProbs ? 1 : OP == kChoice ? 2 : a.reference ? 4 : 3;
    const int2* held = reinterpret_cast<const int2*>(g.held);
    if (g.n_medium) {
        PB_TRY(launch(held_kernel<T, OP, 128>, g.n_medium, 128, (size_t)(g.medium_rows * arrays * 4), a, held, (int)g.medium_rows, slot,
                      scores, out, totals));
        slot += (int)g.n_medium;
    }
    if (g.n_large) {
        PB_TRY(launch(held_kernel<T, OP, 512>, g.n_large, 512, (size_t)(g.large_rows * arrays * 4), a, held + g.n_medium,
                      (int)g.large_rows, slot, scores, out, totals));
        slot += (int)g.n_large;
    }
    if (g.n_pieces) {
        PB_TRY(launch(piece_kernel<T, OP, kPieceMass>, g.n_pieces, kPieceThreads, 0, a, sums, slot, scores, out, totals));
        if (OP != kLogProbs)
            PB_TRY(launch(piece_kernel<T, OP, kPieceTerms>, g.n_pieces, kPieceThreads, 0, a, sums, slot, scores, out, totals));
        PB_TRY(launch(piece_kernel<T, OP, kPieceOut>, g.n_pieces, kPieceThreads, 0, a, sums, slot, scores, out, totals));
    }
    if (want && n_parts != 1)
        PB_TRY(launch(finish_kernel, 1, kFinishThreads, 0, (const Part*)totals.parts, n_parts, scale, loss, kl, clipped));
    count_launch(launches);
    return PB_OK;
}

template <typename T>
int launch_objective(const pb_objective* o, const void* scores, void* grad, float* loss, float* kl, int64_t* clipped, void* scratch,
                     cudaStream_t stream) {
    if (o->kind == PB_OBJECTIVE_PREFERENCE) {
        const PairArgs a{*o->pairs, (float)o->beta, (float)o->smoothing, (float)(0.5 / o->beta),
                         (float)(o->scale * (o->squared ? 2.0 : o->beta))};
        if (kl) PB_CUDA_TRY(cudaMemsetAsync(kl, 0, sizeof(*kl), stream));
        if (clipped) PB_CUDA_TRY(cudaMemsetAsync(clipped, 0, sizeof(*clipped), stream));
        return launch_pairs<T>(a, o->squared != 0, o->scale, static_cast<const T*>(scores), static_cast<T*>(grad), loss, static_cast<double*>(scratch), stream);
    }
    const GroupArgs a{*o->groups, o->target, o->advantage, o->old, o->reference, split(log1p(o->clip_high)), split(log1p(-o->clip_low)),
                      (float)(1.0 + o->clip_high), (float)(1.0 - o->clip_low), (float)o->kl_coef, (float)o->scale};
    if (o->kind == PB_OBJECTIVE_CHOICE) return launch_groups<T, kChoice>(a, o->scale, scores, grad, loss, kl, clipped, scratch, stream);
    return launch_groups<T, kPolicy>(a, o->scale, scores, grad, loss, kl, clipped, scratch, stream);
}

}  // namespace

int objective_gradient(const pb_objective* o, const void* scores, int64_t score_type, void* grad, float* loss, float* kl,
                       int64_t* clipped, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
    PB_REQUIRE(n_rows_of(o) == 0 || (scores && grad), "scores or gradient is null");
    const int64_t need = scratch_bytes(o);
    if (need > 0) {
        PB_REQUIRE(workspace != nullptr && (uintptr_t)workspace % 8 == 0, "workspace is null or not aligned");
        if (workspace_bytes < need) {
            set_error("objective workspace: %lld bytes given, %lld needed", (long long)workspace_bytes, (long long)need);
            return PB_ERR_WORKSPACE;
        }
    }
    int rc;
    switch (score_type) {
        case PB_SCORE_F32: rc = launch_objective<float>(o, scores, grad, loss, kl, clipped, workspace, stream); break;
        case PB_SCORE_F16: rc = launch_objective<__half>(o, scores, grad, loss, kl, clipped, workspace, stream); break;
        case PB_SCORE_BF16: rc = launch_objective<__nv_bfloat16>(o, scores, grad, loss, kl, clipped, workspace, stream); break;
        default: return fail_arg("unknown type of scores %lld", (long long)score_type);
    }
    if (rc) return rc;
    PB_LAUNCH_CHECK("objective");
    return PB_OK;
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
    return group_scratch_bytes(g, false);
}

extern "C" int pb_group_log_probs(const pb_groups* g, const void* scores, int64_t score_type, void* out, void* workspace,
                                  int64_t workspace_bytes, void* stream_) {
    NvtxRange nvtx("pb.group_log_probs n=%lld", g ? (long long)g->n_rows : -1);
    PB_TRY(check_groups(g));
    PB_REQUIRE(g->n_rows == 0 || (scores && out), "scores or output is null");
    if (g->n_pieces) {
        PB_REQUIRE(workspace != nullptr && (uintptr_t)workspace % 8 == 0, "workspace is null or not aligned");
        if (workspace_bytes < group_scratch_bytes(g, false)) {
            set_error("workspace of the log-probabilities: %lld bytes given, %lld needed", (long long)workspace_bytes,
                      (long long)pb_group_log_probs_bytes(g));
            return PB_ERR_WORKSPACE;
        }
    }
    cudaStream_t stream = (cudaStream_t)stream_;
    GroupArgs a{};
    a.g = *g;
    int rc;
    switch (score_type) {
        case PB_SCORE_F32: rc = launch_groups<float, kLogProbs>(a, 1.0, scores, out, nullptr, nullptr, nullptr, workspace, stream); break;
        case PB_SCORE_F16: rc = launch_groups<__half, kLogProbs>(a, 1.0, scores, out, nullptr, nullptr, nullptr, workspace, stream); break;
        case PB_SCORE_BF16: rc = launch_groups<__nv_bfloat16, kLogProbs>(a, 1.0, scores, out, nullptr, nullptr, nullptr, workspace, stream); break;
        default: return fail_arg("unknown type of scores %lld", (long long)score_type);
    }
    if (rc) return rc;
    PB_LAUNCH_CHECK("group_log_probs");
    return PB_OK;
}
