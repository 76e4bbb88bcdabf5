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
    int squared;
    float scale;
};

// Loss and derivative with respect to d of a pair whose (reference-corrected) score difference is d.
__device__ __forceinline__ float pair_slope(const PairArgs& a, float d, float* loss) {
    if (a.squared) {
        const float off = d - a.half_tau;
        *loss = off * off;
        return 2.f * off;
    }
    // softplus(-z) + e z has the derivative e - sigmoid(-z)
    const float z = a.beta * d;
    const float e = expf(-fabsf(z));
    *loss = fmaxf(-z, 0.f) + log1pf(e) + (a.smoothing != 0.f ? a.smoothing * z : 0.f);
    const float q = __fdividef(z > 0.f ? e : 1.f, 1.f + e);
    return a.beta * (a.smoothing - q);
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

template <typename T>
__global__ void __launch_bounds__(kPairThreads) pair_kernel(PairArgs a, const T* __restrict__ scores, T* __restrict__ grad,
                                                            PairPieces pieces, double scale, float* loss_out) {
    __shared__ double s_tail[2][kPairThreads / 32];
    __shared__ int s_seen[2][kPairThreads / 32];
    __shared__ double scratch[kPairThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t tile0 = (int64_t)blockIdx.x * a.p.run_tiles;
    const int64_t tile1 = min(tile0 + a.p.run_tiles, a.p.n_items / kPairTile);
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
        }
        if (a.p.weight) {
            *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(a.p.weight + i0);
            *reinterpret_cast<float4*>(w + 4) = *reinterpret_cast<const float4*>(a.p.weight + i0 + 4);
        }
        float other[kPairItems];
#pragma unroll
        for (int u = 0; u < kPairItems; ++u) other[u] = to_f32(scores[word[u] & 0x7FFFFFFFu]);
        const int row_open = row - (int)(heads & 1u);  // the row that is open where the chunk begins
        float own = to_f32(scores[row]);
        float acc = 0.f, lead = 0.f, chunk_loss = 0.f;
        bool any = false;                              // a row has started in this chunk
#pragma unroll
        for (int u = 0; u < kPairItems; ++u) {
            if ((heads >> u) & 1u) {
                if (any)
                    grad[row] = from_f32<T>(acc * a.scale);
                else
                    lead = acc;
                if (u > 0) own = to_f32(scores[++row]);
                any = true;
                acc = 0.f;
            }
            const uint32_t o = word[u] & 0x7FFFFFFFu;
            const bool rejected = word[u] >> 31;
            float d = own - other[u];
            if (a.p.offset) d -= off[u];
            if (rejected) d = -d;
            float l;
            float sl = pair_slope(a, d, &l);
            if (a.p.weight) {
                sl *= w[u];
                l *= w[u];
            }
            if (o != (uint32_t)row) {                  // (else it fills a row without pairs, or the last tile)
                acc += rejected ? -sl : sl;
                if (!rejected) chunk_loss += l;
            }
        }
        if (!any) lead = acc;
        loss += (double)chunk_loss;

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
                grad[row_open] = from_f32<T>((float)sum * a.scale);
            else
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
        if (seen && ends) grad[last_row] = from_f32<T>((float)carry * a.scale);
        if (!seen) pieces.lead[blockIdx.x] = carry;
        pieces.tail[blockIdx.x] = carry;
    }
    if (pieces.loss || loss_out) {
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
    if (lane == 0) grad[row] = from_f32<T>((float)t * a.scale);
}

// A launch that may begin before the one in front of it on the stream has ended, and waits for it itself.
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), unsigned grid, unsigned block, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.stream = stream;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, (P)args...);
}

int64_t n_runs_of(const pb_pairs* p) {
    return p->n_items ? (p->n_items / kPairTile + p->run_tiles - 1) / p->run_tiles : 0;
}

template <typename T>
int launch_pairs(const PairArgs& a, double scale, const T* scores, T* grad, float* loss, double* scratch, cudaStream_t stream) {
    const int64_t n_runs = n_runs_of(&a.p);
    if (n_runs == 0) {
        if (loss) PB_CUDA_TRY(cudaMemsetAsync(loss, 0, 4, stream));
        return PB_OK;
    }
    const bool one = n_runs == 1;
    PairPieces pieces{scratch, scratch + n_runs, loss && !one ? scratch + 2 * n_runs : nullptr};
    pair_kernel<T><<<(unsigned)n_runs, kPairThreads, 0, stream>>>(a, scores, grad, pieces, scale, one ? loss : nullptr);
    count_launch(1);
    if (!one && (loss || a.p.n_cuts)) {
        const int64_t grid = (a.p.n_cuts + kPairFinishThreads / 32 - 1) / (kPairFinishThreads / 32) + 1;
        PB_CUDA_TRY(launch_after(pair_finish_kernel<T>, (unsigned)grid, kPairFinishThreads, stream, a, pieces, n_runs, scale,
                                 grad, loss));
        count_launch(1);
    }
    return PB_OK;
}

// ---- groups ---------------------------------------------------------------------------------------

enum GroupOp { kChoice, kPolicy, kLogProbs };

struct GroupArgs {
    pb_groups g;
    const float *target, *advantage, *old, *reference;
    double log_high, log_low;  // borders of the log of the ratio
    float bound_high, bound_low;
    double kl_coef;
    float scale;
};

// exp of a 64-bit value that 32 bits would round by more than exp forgives
__device__ __forceinline__ float exp_of(double x) {
    const float hi = (float)x;
    const float lo = (float)(x - (double)hi);
    const float e = expf(hi);
    return isfinite(lo) ? fmaf(e, lo, e) : e;
}

// A taken row: its term of the loss, and that term's derivative with respect to its log-probability.
struct Taken {
    float loss, slope;
    bool beyond;
};
__device__ __forceinline__ Taken taken_row(const GroupArgs& a, double adv_x, float adv) {
    Taken t;
    t.beyond = adv > 0.f ? adv_x > a.log_high : adv_x < a.log_low;
    const float q = t.beyond ? (adv > 0.f ? a.bound_high : a.bound_low) : exp_of(adv_x);
    t.loss = -adv * q;
    t.slope = t.beyond ? 0.f : t.loss;
    return t;
}

// Sums and divergence of one group, and what its rows get: a slope plus p times a number of the group.
struct RowTerm {
    float slope;  // of the row's own term (policy), or minus its target (choice)
    float p;
    float gap;    // p (l - reference), times kl_coef in the gradient
};

// What one row contributes.  `s` is its score, l its log-probability; the row's other inputs are read here.
template <int OP>
struct RowSums {
    double sum = 0.0;   // targets, or slopes of taken rows
    double kl = 0.0;
    double loss = 0.0;
    int clipped = 0;
};
struct RowInputs {
    float target_or_advantage, old, reference;
};

template <int OP>
__device__ __forceinline__ RowInputs row_inputs(const GroupArgs& a, int r, bool in) {
    RowInputs v{0.f, 0.f, 0.f};
    if (in) {
        v.target_or_advantage = OP == kChoice ? a.target[r] : a.advantage[r];
        if (OP == kPolicy) v.old = a.old[r];
        if (OP == kPolicy && a.reference) v.reference = a.reference[r];
    }
    return v;
}

template <int OP>
__device__ __forceinline__ RowTerm row_term(const GroupArgs& a, float s, double l, const RowInputs& in, RowSums<OP>& sums) {
    RowTerm t{0.f, 0.f, 0.f};
    const bool live = s != -INFINITY;
    if (live) t.p = exp_of(l);
    if (OP == kChoice) {
        t.slope = -in.target_or_advantage;
        sums.sum += (double)in.target_or_advantage;
        if (in.target_or_advantage != 0.f) sums.loss -= (double)in.target_or_advantage * l;
    } else if (live) {
        const float adv = in.target_or_advantage;
        if (adv != 0.f) {
            const Taken k = taken_row(a, l - (double)in.old, adv);
            t.slope = k.slope;
            sums.sum += (double)k.slope;
            sums.loss += (double)k.loss;
            sums.clipped += k.beyond ? 1 : 0;
        }
        if (a.reference) {
            t.gap = t.p * (float)(l - (double)in.reference);
            sums.kl += (double)t.gap;
        }
    }
    return t;
}

// The gradient of a row: with H the sum of the slopes (or T of the targets) and D the divergence,
// slope + p (k (l - reference - D) - H), or p T - target.
template <int OP>
__device__ __forceinline__ float row_gradient(const GroupArgs& a, const RowTerm& t, float share) {
    const float fixed = OP == kChoice ? t.slope : fmaf((float)a.kl_coef, t.gap, t.slope);
    return (t.p == 0.f ? fixed : fmaf(t.p, share, fixed)) * a.scale;  // (the share may be infinite)
}
template <int OP>
__device__ __forceinline__ float group_share(const GroupArgs& a, double sum, double kl) {
    return OP == kChoice ? (float)sum : (float)(-a.kl_coef * kl - sum);
}

__device__ __forceinline__ double log_sum(float m, double z) {
    return z == 0.0 ? 0.0 : (double)m + log(z);  // (nothing left in the group: every p is 0)
}

// exp(s - m), 0 for a masked row
__device__ __forceinline__ double mass_of(float s, float m) { return s == -INFINITY ? 0.0 : exp((double)s - (double)m); }

// Writes the totals of a CTA, or, where it is the only one, the outputs.
struct Totals {
    Part* parts;           // null: not wanted
    double scale;
    float *loss, *kl;
    int64_t* clipped;
    int only;              // this launch's one CTA is all there is
};
__device__ __forceinline__ void put_totals(const Totals& out, int slot, double loss, double kl, double clipped) {
    if (out.only) {
        if (out.loss) *out.loss = (float)(loss * out.scale);
        if (out.kl) *out.kl = (float)(kl * out.scale);
        if (out.clipped) *out.clipped = (int64_t)clipped;
    } else {
        out.parts[slot] = Part{loss, kl, clipped};
    }
}
__device__ __forceinline__ bool wants_totals(const Totals& out) { return out.only ? (out.loss || out.kl || out.clipped) : out.parts != nullptr; }

// ---- short groups: a window of rows per CTA ----
//
// A window is 1024 neighbouring places; every short group belongs to the window its first row is in, and
// windows start 896 apart so that it ends there too.  A thread has four places; sums over groups are
// segmented scans over the CTA's threads, so groups of one row and groups of 128 cost the same per row.
constexpr int kWindowThreads = 256;
static_assert(kWindowThreads * 4 == PB_WINDOW_ROWS, "layout of the windows");

// Bits of a thread's word: first rows of groups 0-3, rows of this window 4-7, last rows 8-11, groups begun before the thread 12-.
__device__ __forceinline__ bool word_head(uint32_t w, int u) { return (w >> u) & 1u; }
__device__ __forceinline__ bool word_in(uint32_t w, int u) { return (w >> (4 + u)) & 1u; }
__device__ __forceinline__ bool word_last(uint32_t w, int u) { return (w >> (8 + u)) & 1u; }
__device__ __forceinline__ int word_group(uint32_t w, int u) { return (int)(w >> 12) + __popc(w & ((2u << u) - 1u)) - 1; }

struct AddOp {
    template <typename V> __device__ static V apply(V x, V y) { return x + y; }
};
struct MaxOp {
    __device__ static float apply(float x, float y) { return fmaxf(x, y); }
};

// Totals of the groups of a window, by group, in `total`.  A group of at most 128 rows is open in one warp
// before the one that ends it at most, since a warp has 128 places.
template <typename V, typename Op>
__device__ __forceinline__ void window_totals(const V x[4], uint32_t word, uint32_t mask, V none, V* warp_open, V* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V v = none;
#pragma unroll
    for (int u = 0; u < 4; ++u) v = word_head(word, u) ? x[u] : Op::apply(v, x[u]);
    const uint32_t below = mask & (0xFFFFFFFFu >> (31 - lane));
    const int reach = below ? lane - (31 - __clz(below)) : lane;
    for (int d = 1; d < 32; d <<= 1) {
        const V o = __shfl_up_sync(0xFFFFFFFFu, v, d);
        if (d <= reach) v = Op::apply(o, v);
    }
    if (lane == 31) warp_open[warp] = v;
    V open = __shfl_up_sync(0xFFFFFFFFu, v, 1);
    if (lane == 0) open = none;
    __syncthreads();
    if (!(mask & ((1u << lane) - 1u)) && warp > 0) open = Op::apply(warp_open[warp - 1], open);
    v = open;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        v = word_head(word, u) ? x[u] : Op::apply(v, x[u]);
        if (word_last(word, u)) total[word_group(word, u)] = v;
    }
    __syncthreads();
}

// Four neighbouring places of an array, or of the rows that an index lists.
template <typename T>
__device__ __forceinline__ void load4(const T* p, const int r[4], bool straight, uint32_t word, T v[4]) {
    if (straight) {
        if (sizeof(T) == 4)
            *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p + r[0]);
        else
            *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(p + r[0]);
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (word_in(word, u)) v[u] = p[r[u]];
    }
}

template <typename T, int OP>
__global__ void __launch_bounds__(kWindowThreads) window_kernel(GroupArgs a, int vectors, const T* __restrict__ scores,
                                                                T* __restrict__ out, Totals totals) {
    __shared__ double s_z[PB_WINDOW_ROWS], s_open[3][kWindowThreads / 32];
    __shared__ float s_m[PB_WINDOW_ROWS], s_open_m[kWindowThreads / 32];
    __shared__ double s_kl[OP == kPolicy ? PB_WINDOW_ROWS : 1];
    __shared__ double scratch[kWindowThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;");
    const int64_t i0 = (int64_t)a.g.windows[blockIdx.x] * PB_WINDOW_STEP + threadIdx.x * 4;
    const uint32_t word = a.g.window_words[(int64_t)blockIdx.x * kWindowThreads + threadIdx.x];
    const uint32_t mask = __ballot_sync(0xFFFFFFFFu, (word & 15u) != 0u);
    int r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = (int)(i0 + u);
    if (a.g.rows) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (word_in(word, u)) r[u] = a.g.rows[i0 + u];
    }
    const bool straight = vectors && i0 + 3 < a.g.n_rows && (word & 0xF0u);
    T raw[4];
    RowInputs in[4];
    load4(scores, r, straight, word, raw);
    if (OP != kLogProbs) {
        float v[4];
        load4(OP == kChoice ? a.target : a.advantage, r, straight, word, v);
#pragma unroll
        for (int u = 0; u < 4; ++u) in[u].target_or_advantage = v[u];
        if (OP == kPolicy) {
            load4(a.old, r, straight, word, v);
#pragma unroll
            for (int u = 0; u < 4; ++u) in[u].old = v[u];
            if (a.reference) {
                load4(a.reference, r, straight, word, v);
#pragma unroll
                for (int u = 0; u < 4; ++u) in[u].reference = v[u];
            }
        }
    }
    float s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) s[u] = word_in(word, u) ? to_f32(raw[u]) : -INFINITY;
    window_totals<float, MaxOp>(s, word, mask, -INFINITY, s_open_m, s_m);
    double e[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) e[u] = word_in(word, u) ? mass_of(s[u], s_m[word_group(word, u)]) : 0.0;
    window_totals<double, AddOp>(e, word, mask, 0.0, s_open[0], s_z);
    // (the log of each group's sum once, by the thread of its last row)
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (word_last(word, u)) {
            const int k = word_group(word, u);
            s_z[k] = log_sum(s_m[k], s_z[k]);
        }
    __syncthreads();
    double l[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) l[u] = word_in(word, u) ? (double)s[u] - s_z[word_group(word, u)] : 0.0;
    float g[4];
    if (OP == kLogProbs) {
#pragma unroll
        for (int u = 0; u < 4; ++u) g[u] = (float)l[u];
    } else {
        RowSums<OP> all;
        RowTerm t[4];
        double sum[4], kl[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            RowSums<OP> one;
            t[u] = RowTerm{0.f, 0.f, 0.f};
            if (word_in(word, u)) t[u] = row_term<OP>(a, s[u], l[u], in[u], one);
            sum[u] = one.sum;
            kl[u] = one.kl;
            all.loss += one.loss;
            all.kl += one.kl;
            all.clipped += one.clipped;
        }
        window_totals<double, AddOp>(sum, word, mask, 0.0, s_open[1], s_z);
        if (OP == kPolicy && a.reference) window_totals<double, AddOp>(kl, word, mask, 0.0, s_open[2], s_kl);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            g[u] = 0.f;
            if (word_in(word, u)) {
                const int k = word_group(word, u);
                g[u] = row_gradient<OP>(a, t[u], group_share<OP>(a, s_z[k], OP == kPolicy && a.reference ? s_kl[k] : 0.0));
            }
        }
        if (wants_totals(totals)) {
            const double loss = block_sum(all.loss, scratch);
            double kl_all = 0.0, clipped = 0.0;
            if (OP == kPolicy) {
                kl_all = block_sum(all.kl, scratch);
                clipped = block_sum((double)all.clipped, scratch);
            }
            if (threadIdx.x == 0) put_totals(totals, blockIdx.x, loss + a.kl_coef * kl_all, kl_all, clipped);
        }
    }
    if (straight && (word & 0xF0u) == 0xF0u) {
        T v[4] = {from_f32<T>(g[0]), from_f32<T>(g[1]), from_f32<T>(g[2]), from_f32<T>(g[3])};
        if (sizeof(T) == 4)
            *reinterpret_cast<uint4*>(out + r[0]) = *reinterpret_cast<const uint4*>(v);
        else
            *reinterpret_cast<uint2*>(out + r[0]) = *reinterpret_cast<const uint2*>(v);
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (word_in(word, u)) out[r[u]] = from_f32<T>(g[u]);
    }
}

// ---- groups that a CTA holds ----
//
// A group of up to THREADS x ROWS rows stays in the registers of one CTA: its scores are read once, and of the
// rest of a row two numbers are kept between the sums and the gradient.
template <int THREADS>
__device__ __forceinline__ double cta_sum(double v, double* scratch) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) t += scratch[w];
    return t;
}

// Largest score and the log of the sum of exponentials over the CTA's threads, from the threads' own ones.
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

template <typename T, int OP, int THREADS, int ROWS>
__global__ void __launch_bounds__(THREADS) held_kernel(GroupArgs a, const int32_t* __restrict__ list, int slot0,
                                                       const T* __restrict__ scores, T* __restrict__ out, Totals totals) {
    __shared__ float s_m[THREADS / 32];
    __shared__ double s_z[THREADS / 32], scratch[THREADS / 32];
    asm volatile("griddepcontrol.launch_dependents;");
    const int group = list[blockIdx.x];
    const int begin = a.g.offsets[group], n = a.g.offsets[group + 1] - begin;
    auto row_of = [&](int i) { return a.g.rows ? a.g.rows[begin + i] : begin + i; };
    float s[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        const int i = u * THREADS + threadIdx.x;
        s[u] = i < n ? to_f32(scores[row_of(i)]) : -INFINITY;
    }
    float m = s[0];
#pragma unroll
    for (int u = 1; u < ROWS; ++u) m = fmaxf(m, s[u]);
    double z = 0.0;
#pragma unroll
    for (int u = 0; u < ROWS; ++u)
        if (u * THREADS < n) z += mass_of(s[u], m);
    const double lse = cta_log_sum<THREADS>(m, z, s_m, s_z);
    if (OP == kLogProbs) {
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            const int i = u * THREADS + threadIdx.x;
            if (i < n) out[row_of(i)] = from_f32<T>((float)((double)s[u] - lse));
        }
        return;
    }
    RowSums<OP> sums;
    float fixed[ROWS];  // what does not hang on the group; s becomes p
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        const int i = u * THREADS + threadIdx.x;
        if (i < n) {
            const RowInputs in = row_inputs<OP>(a, row_of(i), true);
            const RowTerm t = row_term<OP>(a, s[u], (double)s[u] - lse, in, sums);
            s[u] = t.p;
            fixed[u] = OP == kChoice ? t.slope : fmaf((float)a.kl_coef, t.gap, t.slope);
        }
    }
    const double sum = cta_sum<THREADS>(sums.sum, scratch);
    const double kl = OP == kPolicy && a.reference ? cta_sum<THREADS>(sums.kl, scratch) : 0.0;
    const float share = group_share<OP>(a, sum, kl);
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        const int i = u * THREADS + threadIdx.x;
        if (i < n) out[row_of(i)] = from_f32<T>((s[u] == 0.f ? fixed[u] : fmaf(s[u], share, fixed[u])) * a.scale);
    }
    if (wants_totals(totals)) {
        const double loss = cta_sum<THREADS>(sums.loss, scratch);
        const double clipped = OP == kPolicy ? cta_sum<THREADS>((double)sums.clipped, scratch) : 0.0;
        if (threadIdx.x == 0) put_totals(totals, slot0 + blockIdx.x, loss + a.kl_coef * kl, kl, clipped);
    }
}

// ---- long groups: many CTAs each ----
//
// Pieces of PB_PIECE_ROWS rows; the sums of a group's pieces go through memory from one launch to the next: sums of
// exponentials, then slopes and divergence, then the gradient.  The rows are read again each time, from L2 mostly.
struct PieceSums {
    double z, sum, kl;
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
    const int begin = a.g.pieces[4 * blockIdx.x], n = a.g.pieces[4 * blockIdx.x + 1];
    const int first = a.g.pieces[4 * blockIdx.x + 2], count = a.g.pieces[4 * blockIdx.x + 3];  // of the group's pieces
    auto row_of = [&](int i) { return a.g.rows ? a.g.rows[begin + i] : begin + i; };
    float s[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        const int i = u * THREADS + threadIdx.x;
        s[u] = i < n ? to_f32(scores[row_of(i)]) : -INFINITY;
    }
    float m = -INFINITY;
    double z = 0.0;
    if (STEP == kPieceMass) {
#pragma unroll
        for (int u = 0; u < ROWS; ++u) m = fmaxf(m, s[u]);
#pragma unroll
        for (int u = 0; u < ROWS; ++u) z += mass_of(s[u], m);
        float wm = warp_max(m);
        z = warp_sum(z == 0.0 ? 0.0 : z * exp((double)m - (double)wm));
        if ((threadIdx.x & 31) == 0) {
            s_m[threadIdx.x >> 5] = wm;
            s_z[threadIdx.x >> 5] = z;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 0; w < THREADS / 32; ++w) wm = fmaxf(wm, s_m[w]);
            z = 0.0;
            for (int w = 0; w < THREADS / 32; ++w)
                if (s_z[w] != 0.0) z += s_z[w] * exp((double)s_m[w] - (double)wm);
            pieces[blockIdx.x].m = wm;
            pieces[blockIdx.x].z = z;
        }
        return;
    }
    // the group's log of the sum, from all its pieces
    for (int k = threadIdx.x; k < count; k += THREADS) m = fmaxf(m, pieces[first + k].m);
    for (int k = threadIdx.x; k < count; k += THREADS) {
        const double zk = pieces[first + k].z;
        if (zk != 0.0) z += zk * exp((double)pieces[first + k].m - (double)m);
    }
    const double lse = cta_log_sum<THREADS>(m, z, s_m, s_z);
    if (OP == kLogProbs) {
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            const int i = u * THREADS + threadIdx.x;
            if (i < n) out[row_of(i)] = from_f32<T>((float)((double)s[u] - lse));
        }
        return;
    }
    double sum = 0.0, kl = 0.0;
    if (STEP == kPieceOut) {
        for (int k = threadIdx.x; k < count; k += THREADS) {
            sum += pieces[first + k].sum;
            kl += pieces[first + k].kl;
        }
        sum = cta_sum<THREADS>(sum, scratch);
        kl = OP == kPolicy && a.reference ? cta_sum<THREADS>(kl, scratch) : 0.0;
    }
    const float share = group_share<OP>(a, sum, kl);
    RowSums<OP> sums;
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        const int i = u * THREADS + threadIdx.x;
        if (i < n) {
            const int r = row_of(i);
            const RowInputs in = row_inputs<OP>(a, r, true);
            const RowTerm t = row_term<OP>(a, s[u], (double)s[u] - lse, in, sums);
            if (STEP == kPieceOut) out[r] = from_f32<T>(row_gradient<OP>(a, t, share));
        }
    }
    if (STEP == kPieceTerms) {
        sum = cta_sum<THREADS>(sums.sum, scratch);
        kl = OP == kPolicy ? cta_sum<THREADS>(sums.kl, scratch) : 0.0;
        if (threadIdx.x == 0) {
            pieces[blockIdx.x].sum = sum;
            pieces[blockIdx.x].kl = kl;
        }
        if (wants_totals(totals)) {
            const double loss = cta_sum<THREADS>(sums.loss, scratch);
            const double clipped = OP == kPolicy ? cta_sum<THREADS>((double)sums.clipped, scratch) : 0.0;
            if (threadIdx.x == 0) put_totals(totals, slot0 + blockIdx.x, loss + a.kl_coef * kl, kl, clipped);
        }
    }
}

// ---- launches ---------------------------------------------------------------------------------------

int check_groups(const pb_groups* g) {
    PB_REQUIRE(g != nullptr, "groups are null");
    PB_REQUIRE(g->n_rows >= 0 && g->n_rows < (1ll << 31) - 1, "n_rows=%lld out of range", (long long)g->n_rows);
    PB_REQUIRE(g->n_groups >= 0 && g->n_groups <= g->n_rows, "n_groups=%lld out of range", (long long)g->n_groups);
    PB_REQUIRE((g->n_groups == 0) == (g->n_rows == 0), "rows without a group");
    PB_REQUIRE(g->n_groups == 0 || g->offsets, "offsets of the groups are null");
    const int64_t most = (1ll << 31) - 1;
    PB_REQUIRE(g->n_windows >= 0 && g->n_medium >= 0 && g->n_large >= 0 && g->n_pieces >= 0 && g->n_windows < most &&
                   g->n_pieces < most && g->n_medium + g->n_large <= g->n_groups,
               "counts of the groups' layout are out of range");
    PB_REQUIRE((g->n_windows == 0 || (g->windows && g->window_words)) && (g->n_medium + g->n_large == 0 || g->listed) &&
                   (g->n_pieces == 0 || g->pieces),
               "a table of the groups' layout is null");
    PB_REQUIRE(g->n_groups == 0 || g->n_windows + g->n_medium + g->n_large + g->n_pieces > 0, "the groups are not laid out");
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

int64_t n_group_parts(const pb_groups* g) { return g->n_windows + g->n_medium + g->n_large + g->n_pieces; }

// Scratch: what the CTAs leave of the totals, then the sums of pieces.
int64_t scratch_bytes(const pb_objective* o) {
    if (o->kind == PB_OBJECTIVE_PREFERENCE) return 3 * n_runs_of(o->pairs) * (int64_t)sizeof(double);
    return n_group_parts(o->groups) * (int64_t)sizeof(Part) + o->groups->n_pieces * (int64_t)sizeof(PieceSums);
}

template <typename T, int OP>
int launch_groups(const GroupArgs& a, double scale, const void* scores_, void* out_, float* loss, float* kl, int64_t* clipped,
                  void* scratch, cudaStream_t stream) {
    const T* scores = static_cast<const T*>(scores_);
    T* out = static_cast<T*>(out_);
    const pb_groups& g = a.g;
    const int64_t n_parts = n_group_parts(&g);
    const bool want = loss || kl || clipped;
    Totals totals{want ? static_cast<Part*>(scratch) : nullptr, scale, loss, kl, clipped, n_parts == 1};
    if (g.n_windows) {
        const uintptr_t bits = (uintptr_t)scores | (uintptr_t)out | (uintptr_t)a.target | (uintptr_t)a.advantage | (uintptr_t)a.old | (uintptr_t)a.reference;
        const int vectors = !g.rows && bits % 16 == 0;
        window_kernel<T, OP><<<(unsigned)g.n_windows, kWindowThreads, 0, stream>>>(a, vectors, scores, out, totals);
        count_launch(1);
    }
    if (g.n_medium) {
        held_kernel<T, OP, 128, PB_MEDIUM_ROWS / 128><<<(unsigned)g.n_medium, 128, 0, stream>>>(
            a, g.listed, (int)g.n_windows, scores, out, totals);
        count_launch(1);
    }
    if (g.n_large) {
        held_kernel<T, OP, 512, PB_LARGE_ROWS / 512><<<(unsigned)g.n_large, 512, 0, stream>>>(
            a, g.listed + g.n_medium, (int)(g.n_windows + g.n_medium), scores, out, totals);
        count_launch(1);
    }
    if (g.n_pieces) {
        PieceSums* sums = reinterpret_cast<PieceSums*>(static_cast<Part*>(scratch) + n_parts);
        const int slot0 = (int)(n_parts - g.n_pieces);
        piece_kernel<T, OP, kPieceMass><<<(unsigned)g.n_pieces, kPieceThreads, 0, stream>>>(a, sums, slot0, scores, out, totals);
        if (OP != kLogProbs) {
            piece_kernel<T, OP, kPieceTerms><<<(unsigned)g.n_pieces, kPieceThreads, 0, stream>>>(a, sums, slot0, scores, out, totals);
            count_launch(1);
        }
        piece_kernel<T, OP, kPieceOut><<<(unsigned)g.n_pieces, kPieceThreads, 0, stream>>>(a, sums, slot0, scores, out, totals);
        count_launch(2);
    }
    if (want && n_parts != 1) {
        PB_CUDA_TRY(launch_after(finish_kernel, 1u, (unsigned)kFinishThreads, stream, (const Part*)totals.parts, n_parts, scale, loss, kl, clipped));
        count_launch(1);
    }
    return PB_OK;
}

template <typename T>
int launch_objective(const pb_objective* o, const void* scores, void* grad, float* loss, float* kl, int64_t* clipped, void* scratch,
                     cudaStream_t stream) {
    if (o->kind == PB_OBJECTIVE_PREFERENCE) {
        const PairArgs a{*o->pairs, (float)o->beta, (float)o->smoothing, (float)(0.5 / o->beta), o->squared != 0, (float)o->scale};
        if (kl) PB_CUDA_TRY(cudaMemsetAsync(kl, 0, sizeof(*kl), stream));
        if (clipped) PB_CUDA_TRY(cudaMemsetAsync(clipped, 0, sizeof(*clipped), stream));
        return launch_pairs<T>(a, o->scale, static_cast<const T*>(scores), static_cast<T*>(grad), loss, static_cast<double*>(scratch), stream);
    }
    const GroupArgs a{*o->groups, o->target, o->advantage, o->old, o->reference, log1p(o->clip_high), log1p(-o->clip_low),
                      (float)(1.0 + o->clip_high), (float)(1.0 - o->clip_low), o->kl_coef, (float)o->scale};
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
    return n_group_parts(g) * (int64_t)sizeof(Part) + g->n_pieces * (int64_t)sizeof(PieceSums);
}

extern "C" int pb_group_log_probs(const pb_groups* g, const void* scores, int64_t score_type, void* out, void* workspace,
                                  int64_t workspace_bytes, void* stream_) {
    NvtxRange nvtx("pb.group_log_probs n=%lld", g ? (long long)g->n_rows : -1);
    PB_TRY(check_groups(g));
    PB_REQUIRE(g->n_rows == 0 || (scores && out), "scores or output is null");
    if (g->n_pieces) {
        PB_REQUIRE(workspace != nullptr && (uintptr_t)workspace % 8 == 0, "workspace is null or not aligned");
        if (workspace_bytes < pb_group_log_probs_bytes(g)) {
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
