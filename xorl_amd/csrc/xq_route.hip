// The choice of experts: scores, groups, top-k, weights, and the gradient of the router's logits.
//
//   s = softmax(z) or sigmoid(z)     c = s + bias, without a bias the order of z      chosen: the top_k largest c in the top_groups best groups
//   w = scale s_chosen / (renormalize: sum of the chosen s, otherwise 1)
// An expert whose logit or bias is -inf is out: never chosen, and its group is as strong as it is without it.  Places that no expert is left for
// hold id -1 and weight 0.  A NaN in a row (an infinite logit under softmax too) makes its weights and its gradient NaN, its ids 0 .. top_k - 1.
#include "xq_common.h"

namespace xq {
namespace {

constexpr int kMaxExperts = 1024, kMaxTopK = 32, kMaxGroups = 64;

struct RouteArgs {
    xq_moe_route q;
    float* weights;
    int64_t* selected;
};
struct RouteGradArgs {
    xq_moe_route q;
    const float* weights;
    const int64_t* selected;
    const float* grad;
    void* dz;
    int64_t ld_dz;
};

__device__ __forceinline__ float load_logit(const xq_moe_route& q, int64_t row, int e) {
    const int64_t at = row * q.ld + e;
    return q.dtype == XQ_DT_F32 ? ((const float*)q.logits)[at] : bf16_to_f32(((const bf16_t*)q.logits)[at]);
}
__device__ __forceinline__ double wave_max(double v) {
    for (int o = 32; o; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ int wave_min(int v) {
    for (int o = 32; o; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
    return v;
}

// one wave a row, everything in 64 bits
__global__ void __launch_bounds__(64) moe_route_kernel(RouteArgs a) {
    __shared__ double score[kMaxExperts], order[kMaxExperts], strength[kMaxGroups];
    __shared__ double chosen[kMaxTopK];
    const xq_moe_route& q = a.q;
    const int lane = threadIdx.x, E = q.num_experts, K = q.top_k;
    const int64_t row = blockIdx.x;
    const double kOut = -INFINITY;
    double top = kOut;
    int bad = 0;
    for (int e = lane; e < E; e += 64) {
        const float z = load_logit(q, row, e), b = q.bias ? q.bias[e] : 0.0f;
        bad |= z != z || b != b || (q.scoring == XQ_ROUTE_SOFTMAX && z == INFINITY);
        score[e] = z;
        top = fmax(top, (double)z);
    }
    top = wave_max(top);
    if (__any(bad)) {
        for (int i = lane; i < K; i += 64) {
            a.weights[row * K + i] = NAN;
            a.selected[row * K + i] = i;
        }
        return;
    }
    double total = 0.0;
    for (int e = lane; e < E; e += 64) {
        const double z = score[e], b = q.bias ? (double)q.bias[e] : 0.0;
        const bool out = z == kOut || b == kOut;
        const double s = z == kOut ? 0.0 : q.scoring == XQ_ROUTE_SOFTMAX ? exp(z - top) : 1.0 / (1.0 + exp(-z));
        total += s;
        score[e] = s;
        order[e] = out ? kOut : q.bias ? 0.0 : z;
    }
    total = q.scoring == XQ_ROUTE_SOFTMAX ? wave_sum(total) : 1.0;
    __syncthreads();
    for (int e = lane; e < E; e += 64) {
        score[e] = total > 0.0 ? score[e] / total : 0.0;
        if (q.bias && order[e] != kOut) order[e] = score[e] + (double)q.bias[e];
    }
    __syncthreads();
    if (q.top_groups < q.num_groups) {
        const int size = E / q.num_groups;
        for (int g = lane; g < q.num_groups; g += 64) {
            double first = kOut, second = kOut;
            for (int e = g * size; e < (g + 1) * size; ++e) {
                const double c = order[e] == kOut ? kOut : q.bias ? order[e] : q.group_score == XQ_ROUTE_GROUP_MAX ? order[e] : score[e];
                second = fmax(second, fmin(first, c));
                first = fmax(first, c);
            }
            strength[g] = first + (q.group_score == XQ_ROUTE_GROUP_SUM2 && second != kOut ? second : 0.0);
        }
        __syncthreads();
        for (int e = lane; e < E; e += 64) {
            const int g = e / size;
            int better = 0;
            for (int h = 0; h < q.num_groups; ++h) better += strength[h] > strength[g] || (strength[h] == strength[g] && h < g);
            if (better >= q.top_groups) order[e] = kOut;
        }
        __syncthreads();
    }
    double sum = 0.0;
    int mine = -1;
    for (int i = 0; i < K; ++i) {
        double best = kOut;
        int at = E;
        for (int e = lane; e < E; e += 64)
            if (order[e] > best) { best = order[e]; at = e; }
        const double m = wave_max(best);
        at = wave_min(best == m && m != kOut ? at : E);
        if (lane == i) mine = at < E ? at : -1;
        const double s = at < E ? score[at] : 0.0;
        if (lane == 0) chosen[i] = s;
        sum += s;
        __syncthreads();
        if (at < E && lane == 0) order[at] = kOut;
        __syncthreads();
    }
    if (lane < K) {
        const double w = q.renormalize ? (sum > 0.0 ? chosen[lane] / sum : 0.0) : chosen[lane];
        a.weights[row * K + lane] = (float)((double)q.scale * w);
        a.selected[row * K + lane] = mine;
    }
}

// dz of a row: with g = scale * dw and u = w / scale
//   renormalized: d = u (g - sum g u), under sigmoid times 1 - s        softmax as it is: p_j (g_j - sum g p) for every j        sigmoid: g s (1 - s)
__global__ void __launch_bounds__(64) moe_route_grad_kernel(RouteGradArgs a) {
    __shared__ float d[kMaxExperts];
    const xq_moe_route& q = a.q;
    const int lane = threadIdx.x, E = q.num_experts, K = q.top_k;
    const int64_t row = blockIdx.x;
    const float w = lane < K ? a.weights[row * K + lane] : 0.0f;
    const int64_t id = lane < K ? a.selected[row * K + lane] : -1;
    const bool is = id >= 0 && id < E;
    const bool bad = __any(w != w);
    const double u = (double)w / q.scale, g = is ? (double)q.scale * a.grad[row * K + lane] : 0.0;
    const double dot = wave_sum(is ? g * u : 0.0);
    for (int e = lane; e < E; e += 64) d[e] = 0.0f;
    __syncthreads();
    if (is) {
        const bool soft = q.scoring == XQ_ROUTE_SOFTMAX;
        const double z = soft ? 0.0 : load_logit(q, row, (int)id);
        const double t = exp(-fabs(z)), rest = z > 0.0 ? t / (1.0 + t) : 1.0 / (1.0 + t), s = z > 0.0 ? 1.0 / (1.0 + t) : t / (1.0 + t);
        d[id] = (float)(q.renormalize ? u * (g - dot) * (soft ? 1.0 : rest) : soft ? g * u : g * s * rest);
    }
    __syncthreads();
    double top = -INFINITY, total = 0.0;
    const bool whole = q.scoring == XQ_ROUTE_SOFTMAX && !q.renormalize;
    if (whole && !bad) {
        for (int e = lane; e < E; e += 64) top = fmax(top, (double)load_logit(q, row, e));
        top = wave_max(top);
        for (int e = lane; e < E; e += 64) total += top == -INFINITY ? 0.0 : exp((double)load_logit(q, row, e) - top);
        total = wave_sum(total);
    }
    for (int e = lane; e < E; e += 64) {
        float v = d[e];
        if (whole && !bad && top != -INFINITY) v = (float)((double)v - exp((double)load_logit(q, row, e) - top) / total * dot);
        if (bad) v = NAN;
        const int64_t at = row * a.ld_dz + e;
        if (q.dtype == XQ_DT_F32) ((float*)a.dz)[at] = v;
        else ((bf16_t*)a.dz)[at] = to_bf16(v);
    }
}

int check_route(const char* who, const xq_moe_route* q, bool reads_logits) {
    XQ_REQUIRE(q, "%s: the problem is NULL", who);
    XQ_REQUIRE(q->n_tokens >= 0 && q->n_tokens < (1 << 26), "%s: %lld tokens", who, (long long)q->n_tokens);
    XQ_REQUIRE(q->num_experts >= 1 && q->num_experts <= kMaxExperts, "%s: 1 to %d experts, got %d", who, kMaxExperts, q->num_experts);
    XQ_REQUIRE(q->top_k >= 1 && q->top_k <= kMaxTopK && q->top_k <= q->num_experts, "%s: top_k must be 1 to %d and at most the number of experts, got %d of %d", who,
               kMaxTopK, q->top_k, q->num_experts);
    XQ_REQUIRE(q->scoring == XQ_ROUTE_SOFTMAX || q->scoring == XQ_ROUTE_SIGMOID, "%s: unknown scoring %d", who, q->scoring);
    XQ_REQUIRE(q->num_groups >= 1 && q->num_groups <= kMaxGroups && q->num_experts % q->num_groups == 0, "%s: 1 to %d groups that divide the experts, got %d of %d", who,
               kMaxGroups, q->num_groups, q->num_experts);
    XQ_REQUIRE(q->top_groups >= 1 && q->top_groups <= q->num_groups, "%s: top_groups must be 1 to %d, got %d", who, q->num_groups, q->top_groups);
    XQ_REQUIRE(q->top_k <= q->num_experts / q->num_groups * q->top_groups, "%s: top_k %d is more than the %d experts of %d groups", who, q->top_k,
               q->num_experts / q->num_groups * q->top_groups, q->top_groups);
    XQ_REQUIRE(q->group_score == XQ_ROUTE_GROUP_MAX || q->group_score == XQ_ROUTE_GROUP_SUM2, "%s: unknown group score %d", who, q->group_score);
    XQ_REQUIRE(q->scale >= 0x1p-60f && q->scale <= 0x1p60f, "%s: scale must be positive, from 2^-60 to 2^60, got %g", who, (double)q->scale);
    XQ_REQUIRE(q->dtype == XQ_DT_F32 || q->dtype == XQ_DT_BF16, "%s: logits are fp32 or bf16", who);
    const size_t size = q->dtype == XQ_DT_F32 ? 4 : 2;
    XQ_REQUIRE(q->n_tokens == 0 || !reads_logits || (q->logits && xq_aligned(q->logits, size) && (q->n_tokens == 1 || q->ld >= q->num_experts)), "%s: logits are NULL, misaligned, or rows overlap", who);
    XQ_REQUIRE(xq_aligned(q->bias, 4), "%s: the bias is misaligned", who);
    return XQ_OK;
}

}  // namespace
}  // namespace xq

using namespace xq;

extern "C" int xq_moe_route_fwd(const xq_moe_route* q, float* weights, int64_t* selected, void* stream) {
    const int rc = check_route("xq_moe_route_fwd", q, true);
    if (rc != XQ_OK) return rc;
    if (q->n_tokens == 0) return XQ_OK;
    XQ_REQUIRE(weights && selected && xq_aligned(weights, 4) && xq_aligned(selected, 8), "xq_moe_route_fwd: weights or selected is NULL or misaligned");
    moe_route_kernel<<<dim3((unsigned)q->n_tokens), 64, 0, (hipStream_t)stream>>>(RouteArgs{*q, weights, selected});
    XQ_CHECK_LAUNCH("xq_moe_route_fwd");
    return XQ_OK;
}

extern "C" int xq_moe_route_bwd(const xq_moe_route* q, const float* weights, const int64_t* selected, const float* grad, void* dlogits, int64_t ld_dlogits, void* stream) {
    const int rc = check_route("xq_moe_route_bwd", q, q && (q->scoring != XQ_ROUTE_SOFTMAX || !q->renormalize));
    if (rc != XQ_OK) return rc;
    if (q->n_tokens == 0) return XQ_OK;
    XQ_REQUIRE(weights && selected && grad && xq_aligned(weights, 4) && xq_aligned(selected, 8) && xq_aligned(grad, 4),
               "xq_moe_route_bwd: weights, selected or the gradient is NULL or misaligned");
    XQ_REQUIRE(dlogits && xq_aligned(dlogits, q->dtype == XQ_DT_F32 ? 4 : 2) && (q->n_tokens == 1 || ld_dlogits >= q->num_experts),
               "xq_moe_route_bwd: dlogits is NULL, misaligned, or its rows overlap");
    moe_route_grad_kernel<<<dim3((unsigned)q->n_tokens), 64, 0, (hipStream_t)stream>>>(RouteGradArgs{*q, weights, selected, grad, dlogits, ld_dlogits});
    XQ_CHECK_LAUNCH("xq_moe_route_bwd");
    return XQ_OK;
}
