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
    *loss = fmaxf(-z, 0.f) + log1pf(expf(-fabsf(z))) + (a.smoothing != 0.f ? a.smoothing * z : 0.f);
    return a.beta * (a.smoothing - 1.f / (1.f + expf(z)));
}

constexpr int kPairThreads = 128;

// A thread per row adds up the row's items.
template <typename T>
__global__ void __launch_bounds__(kPairThreads) pair_rows_kernel(PairArgs a, const T* __restrict__ scores,
                                                                 T* __restrict__ grad, Part* __restrict__ parts) {
    __shared__ double scratch[kPairThreads / 32];
    const int64_t row = (int64_t)blockIdx.x * kPairThreads + threadIdx.x;
    double loss = 0.0;
    if (row < a.p.n_rows) {
        const float own = to_f32(scores[row]);
        double g = 0.0;
        const int end = a.p.item_offsets[row + 1];
        for (int i = a.p.item_offsets[row]; i < end; ++i) {
            const uint32_t o = a.p.other[i];
            const bool rejected = o >> 31;
            float d = own - to_f32(scores[o & 0x7FFFFFFFu]);
            if (a.p.offset) d -= a.p.offset[i];
            if (rejected) d = -d;
            float l;
            float s = pair_slope(a, d, &l);
            const float w = a.p.weight ? a.p.weight[i] : 1.f;
            s *= w;
            g += rejected ? -s : s;
            if (!rejected) loss += (double)(w * l);
        }
        grad[row] = from_f32<T>((float)g * a.scale);
    }
    if (parts) {
        loss = block_sum(loss, scratch);
        if (threadIdx.x == 0) parts[blockIdx.x] = Part{loss, 0.0, 0.0};
    }
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

constexpr int kGroupThreads = 256;

// A CTA per group, three passes over its rows.
template <typename T, int OP>
__global__ void __launch_bounds__(kGroupThreads) group_kernel(GroupArgs a, const T* __restrict__ scores,
                                                              T* __restrict__ out, Part* __restrict__ parts) {
    __shared__ double scratch[kGroupThreads / 32];
    __shared__ float s_max[kGroupThreads / 32];
    const int begin = a.g.offsets[blockIdx.x], end = a.g.offsets[blockIdx.x + 1];
    auto row_of = [&](int i) { return a.g.rows ? a.g.rows[i] : i; };

    float m = -INFINITY;
    for (int i = begin + threadIdx.x; i < end; i += kGroupThreads) m = fmaxf(m, to_f32(scores[row_of(i)]));
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int w = 0; w < kGroupThreads / 32; ++w) m = fmaxf(m, s_max[w]);
    double z = 0.0;
    for (int i = begin + threadIdx.x; i < end; i += kGroupThreads) {
        const float s = to_f32(scores[row_of(i)]);
        if (s != -INFINITY) z += exp((double)s - (double)m);
    }
    z = block_sum(z, scratch);
    const double lse = z == 0.0 ? 0.0 : (double)m + log(z);  // (nothing left in the group: every p is 0)

    if (OP == kLogProbs) {
        for (int i = begin + threadIdx.x; i < end; i += kGroupThreads) {
            const int r = row_of(i);
            out[r] = from_f32<T>((float)((double)to_f32(scores[r]) - lse));
        }
        return;
    }
    double loss = 0.0, sum = 0.0, kl = 0.0, clipped = 0.0;  // sum: of the targets, or of the slopes
    for (int i = begin + threadIdx.x; i < end; i += kGroupThreads) {
        const int r = row_of(i);
        const float s = to_f32(scores[r]);
        const double l = (double)s - lse;
        if (OP == kChoice) {
            const float t = a.target[r];
            sum += t;
            if (t != 0.f) loss -= (double)t * l;
        } else if (s != -INFINITY) {
            const float adv = a.advantage[r];
            if (adv != 0.f) {
                const Taken t = taken_row(a, l - (double)a.old[r], adv);
                loss += t.loss;
                sum += t.slope;
                clipped += t.beyond ? 1.0 : 0.0;
            }
            if (a.reference) kl += exp_of(l) * (l - (double)a.reference[r]);
        }
    }
    sum = block_sum(sum, scratch);
    if (OP == kPolicy && a.reference) kl = block_sum(kl, scratch);
    for (int i = begin + threadIdx.x; i < end; i += kGroupThreads) {
        const int r = row_of(i);
        const float s = to_f32(scores[r]);
        const double l = (double)s - lse;
        const float p = s == -INFINITY ? 0.f : exp_of(l);
        float g = 0.f;
        if (OP == kChoice) {
            g = p * (float)sum - a.target[r];
        } else if (s != -INFINITY) {
            const float adv = a.advantage[r];
            const float slope = adv != 0.f ? taken_row(a, l - (double)a.old[r], adv).slope : 0.f;
            const double gap = a.reference ? a.kl_coef * (l - (double)a.reference[r] - kl) : 0.0;
            g = slope + p * (float)(gap - sum);
        }
        out[r] = from_f32<T>(g * a.scale);
    }
    if (parts) {
        loss = block_sum(loss, scratch);
        if (OP == kPolicy) {
            clipped = block_sum(clipped, scratch);
            loss += a.kl_coef * kl;
        }
        if (threadIdx.x == 0) parts[blockIdx.x] = Part{loss, kl, clipped};
    }
}

// ---- launches ---------------------------------------------------------------------------------------

int check_groups(const pb_groups* g) {
    PB_REQUIRE(g != nullptr, "groups are null");
    PB_REQUIRE(g->n_rows >= 0 && g->n_rows < (1ll << 31) - 1, "n_rows=%lld out of range", (long long)g->n_rows);
    PB_REQUIRE(g->n_groups >= 0 && g->n_groups <= g->n_rows, "n_groups=%lld out of range", (long long)g->n_groups);
    PB_REQUIRE((g->n_groups == 0) == (g->n_rows == 0), "rows without a group");
    PB_REQUIRE(g->n_groups == 0 || g->offsets, "offsets of the groups are null");
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
        PB_REQUIRE(p->n_rows == 0 || p->item_offsets, "offsets of the items are null");
        PB_REQUIRE(p->n_items == 0 || (p->other && p->n_rows >= 2), "items without rows");
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

int64_t n_parts_of(const pb_objective* o) {
    return o->kind == PB_OBJECTIVE_PREFERENCE ? (o->pairs->n_rows + kPairThreads - 1) / kPairThreads : o->groups->n_groups;
}

template <typename T, int OP>
void launch_groups(const GroupArgs& a, const void* scores, void* out, Part* parts, cudaStream_t stream) {
    if (a.g.n_groups == 0) return;
    group_kernel<T, OP><<<(unsigned)a.g.n_groups, kGroupThreads, 0, stream>>>(a, static_cast<const T*>(scores),
                                                                            static_cast<T*>(out), parts);
    count_launch(1);
}

template <typename T>
void launch_objective(const pb_objective* o, const void* scores, void* grad, Part* parts, cudaStream_t stream) {
    if (o->kind == PB_OBJECTIVE_PREFERENCE) {
        PairArgs a{*o->pairs, (float)o->beta, (float)o->smoothing, (float)(0.5 / o->beta), o->squared != 0, (float)o->scale};
        if (a.p.n_rows == 0) return;
        pair_rows_kernel<T><<<(unsigned)n_parts_of(o), kPairThreads, 0, stream>>>(a, static_cast<const T*>(scores),
                                                                                static_cast<T*>(grad), parts);
        count_launch(1);
        return;
    }
    GroupArgs a{*o->groups, o->target, o->advantage, o->old, o->reference, log1p(o->clip_high), log1p(-o->clip_low),
                (float)(1.0 + o->clip_high), (float)(1.0 - o->clip_low), o->kl_coef, (float)o->scale};
    if (o->kind == PB_OBJECTIVE_CHOICE)
        launch_groups<T, kChoice>(a, scores, grad, parts, stream);
    else
        launch_groups<T, kPolicy>(a, scores, grad, parts, stream);
}

}  // namespace

int objective_gradient(const pb_objective* o, const void* scores, int64_t score_type, void* grad, float* loss, float* kl,
                       int64_t* clipped, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
    const bool totals = loss || kl || clipped;
    const int64_t n_parts = n_parts_of(o);
    PB_REQUIRE(n_rows_of(o) == 0 || (scores && grad), "scores or gradient is null");
    Part* parts = totals ? static_cast<Part*>(workspace) : nullptr;
    if (totals && n_parts > 0) {
        PB_REQUIRE(workspace != nullptr && (uintptr_t)workspace % 8 == 0, "workspace is null or not aligned");
        if (workspace_bytes < n_parts * (int64_t)sizeof(Part)) {
            set_error("objective workspace: %lld bytes given, %lld needed", (long long)workspace_bytes,
                      (long long)(n_parts * (int64_t)sizeof(Part)));
            return PB_ERR_WORKSPACE;
        }
    }
    switch (score_type) {
        case PB_SCORE_F32: launch_objective<float>(o, scores, grad, parts, stream); break;
        case PB_SCORE_F16: launch_objective<__half>(o, scores, grad, parts, stream); break;
        case PB_SCORE_BF16: launch_objective<__nv_bfloat16>(o, scores, grad, parts, stream); break;
        default: return fail_arg("unknown type of scores %lld", (long long)score_type);
    }
    if (totals) {
        finish_kernel<<<1, kFinishThreads, 0, stream>>>(parts, n_parts, o->scale, loss, kl, clipped);
        count_launch(1);
    }
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
    return n_parts_of(o) * (int64_t)sizeof(Part) + 16;
}

extern "C" int pb_objective_evaluate(const pb_objective* o, const void* scores, int64_t score_type, void* grad, float* loss,
                                     float* kl, int64_t* clipped, void* workspace, int64_t workspace_bytes, void* stream) {
    NvtxRange nvtx("pb.objective kind=%lld", o ? (long long)o->kind : -1);
    PB_TRY(objective_check(o, -1));
    return objective_gradient(o, scores, score_type, grad, loss, kl, clipped, workspace, workspace_bytes, (cudaStream_t)stream);
}

extern "C" int pb_group_log_probs(const pb_groups* g, const void* scores, int64_t score_type, void* out, void* stream_) {
    NvtxRange nvtx("pb.group_log_probs n=%lld", g ? (long long)g->n_rows : -1);
    PB_TRY(check_groups(g));
    PB_REQUIRE(g->n_rows == 0 || (scores && out), "scores or output is null");
    cudaStream_t stream = (cudaStream_t)stream_;
    GroupArgs a{};
    a.g = *g;
    switch (score_type) {
        case PB_SCORE_F32: launch_groups<float, kLogProbs>(a, scores, out, nullptr, stream); break;
        case PB_SCORE_F16: launch_groups<__half, kLogProbs>(a, scores, out, nullptr, stream); break;
        case PB_SCORE_BF16: launch_groups<__nv_bfloat16, kLogProbs>(a, scores, out, nullptr, stream); break;
        default: return fail_arg("unknown type of scores %lld", (long long)score_type);
    }
    PB_LAUNCH_CHECK("group_log_probs");
    return PB_OK;
}
