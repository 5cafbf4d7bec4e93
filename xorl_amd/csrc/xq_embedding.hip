// Embedding:  out[t] = scale W[id_t],   dW[v] = scale sum over the tokens t of v of grad[t], in their order.
// An id outside [0, V) gives a row of NaN and no gradient; tokens of padding_idx give none either.  dW is written whole.
#include <algorithm>

#include "xq_common.h"

namespace xq {
namespace {

__device__ __forceinline__ int64_t token_id(const xq_embedding& q, int64_t t) {
    return q.id_bytes == 8 ? ((const int64_t*)q.ids)[t] : (int64_t)((const int32_t*)q.ids)[t];
}
__device__ __forceinline__ float load_value(const void* p, int dtype, int64_t at) {
    return dtype == XQ_DT_F32 ? ((const float*)p)[at] : bf16_to_f32(((const bf16_t*)p)[at]);
}
__device__ __forceinline__ void store_value(void* p, int dtype, int64_t at, float v) {
    if (dtype == XQ_DT_F32) ((float*)p)[at] = v;
    else ((bf16_t*)p)[at] = to_bf16(v);
}

__global__ void __launch_bounds__(256) embedding_kernel(xq_embedding q, void* out, int64_t ld_out) {
    for (int64_t t = blockIdx.x; t < q.n_tokens; t += gridDim.x) {
        const int64_t id = token_id(q, t);
        const bool is = id >= 0 && id < q.V;
        for (int64_t h = threadIdx.x; h < q.H; h += 256)
            store_value(out, q.dtype, t * ld_out + h, is ? q.scale * load_value(q.weight, q.dtype, id * q.ldw + h) : NAN);
    }
}

// a block a vocabulary row: it looks through all ids
__global__ void __launch_bounds__(256) embedding_grad_kernel(xq_embedding q, const void* grad, int64_t ld_grad, void* dw, int64_t ld_dw) {
    __shared__ int64_t list[256];
    __shared__ int wave_n[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int64_t v = blockIdx.x; v < q.V; v += gridDim.x)
        for (int64_t h0 = 0; h0 < q.H; h0 += 256) {
            const int64_t h = h0 + tid;
            float sum = 0.0f;
            for (int64_t t0 = 0; t0 < q.n_tokens; t0 += 256) {
                const bool is = v != q.padding_idx && t0 + tid < q.n_tokens && token_id(q, t0 + tid) == v;
                const uint64_t mask = __ballot(is);
                if (lane == 0) wave_n[wave] = __popcll(mask);
                __syncthreads();
                int at = __popcll(mask & ((1ull << lane) - 1)), n = 0;
                for (int w = 0; w < 4; ++w) {
                    at += w < wave ? wave_n[w] : 0;
                    n += wave_n[w];
                }
                if (is) list[at] = t0 + tid;
                __syncthreads();
                if (h < q.H)
                    for (int i = 0; i < n; ++i) sum += load_value(grad, q.dtype, list[i] * ld_grad + h);
                __syncthreads();
            }
            if (h < q.H) store_value(dw, q.dtype, v * ld_dw + h, q.scale * sum);
        }
}

int check_embedding(const char* who, const xq_embedding* q) {
    XQ_REQUIRE(q, "%s: the problem is NULL", who);
    XQ_REQUIRE(q->n_tokens >= 0 && q->n_tokens < (1ll << 31) && q->V >= 1 && q->V < (1ll << 31) && q->H >= 1 && q->H < (1ll << 31), "%s: %lld tokens, [%lld, %lld]", who,
               (long long)q->n_tokens, (long long)q->V, (long long)q->H);
    XQ_REQUIRE(q->dtype == XQ_DT_F32 || q->dtype == XQ_DT_BF16, "%s: the weight is fp32 or bf16", who);
    XQ_REQUIRE(q->id_bytes == 4 || q->id_bytes == 8, "%s: ids are int32 or int64, got %d bytes", who, q->id_bytes);
    XQ_REQUIRE(q->n_tokens == 0 || (q->ids && xq_aligned(q->ids, q->id_bytes)), "%s: ids are NULL or misaligned", who);
    XQ_REQUIRE(q->scale == q->scale && q->scale - q->scale == 0.0f, "%s: scale must be finite, got %g", who, (double)q->scale);
    XQ_REQUIRE(q->padding_idx >= -1 && q->padding_idx < q->V, "%s: padding_idx must be -1 (none) or a row of the weight, got %lld", who, (long long)q->padding_idx);
    return XQ_OK;
}
bool rows_ok(const void* p, int dtype, int64_t rows, int64_t ld, int64_t H) { return p && xq_aligned(p, dtype == XQ_DT_F32 ? 4 : 2) && (rows <= 1 || ld >= H); }

}  // namespace
}  // namespace xq

using namespace xq;

extern "C" int xq_embedding_fwd(const xq_embedding* q, void* out, int64_t ld_out, void* stream) {
    const int rc = check_embedding("xq_embedding_fwd", q);
    if (rc != XQ_OK) return rc;
    if (q->n_tokens == 0) return XQ_OK;
    XQ_REQUIRE(rows_ok(q->weight, q->dtype, q->V, q->ldw, q->H), "xq_embedding_fwd: the weight is NULL or misaligned, or its rows overlap");
    XQ_REQUIRE(rows_ok(out, q->dtype, q->n_tokens, ld_out, q->H), "xq_embedding_fwd: out is NULL or misaligned, or its rows overlap");
    embedding_kernel<<<dim3((unsigned)std::min<int64_t>(q->n_tokens, 1 << 20)), 256, 0, (hipStream_t)stream>>>(*q, out, ld_out);
    XQ_CHECK_LAUNCH("xq_embedding_fwd");
    return XQ_OK;
}

extern "C" int64_t xq_embedding_workspace_bytes(int64_t n_tokens, int64_t V, int64_t H) {
    if (n_tokens < 0 || n_tokens >= (1ll << 31) || V < 1 || V >= (1ll << 31) || H < 1 || H >= (1ll << 31)) return -1;
    return 256;
}

extern "C" int xq_embedding_bwd(const xq_embedding* q, const void* grad, int64_t ld_grad, void* dw, int64_t ld_dw, void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = check_embedding("xq_embedding_bwd", q);
    if (rc != XQ_OK) return rc;
    XQ_REQUIRE(q->n_tokens == 0 || rows_ok(grad, q->dtype, q->n_tokens, ld_grad, q->H), "xq_embedding_bwd: the gradient is NULL or misaligned, or its rows overlap");
    XQ_REQUIRE(rows_ok(dw, q->dtype, q->V, ld_dw, q->H), "xq_embedding_bwd: dw is NULL or misaligned, or its rows overlap");
    const int64_t need = xq_embedding_workspace_bytes(q->n_tokens, q->V, q->H);
    XQ_REQUIRE(workspace && xq_aligned(workspace, 256) && workspace_bytes >= need, "xq_embedding_bwd: a workspace of %lld bytes, 256-byte aligned, is needed", (long long)need);
    embedding_grad_kernel<<<dim3((unsigned)std::min<int64_t>(q->V, 1 << 20)), 256, 0, (hipStream_t)stream>>>(*q, grad, ld_grad, dw, ld_dw);
    XQ_CHECK_LAUNCH("xq_embedding_bwd");
    return XQ_OK;
}
