// Adapters of many requests beside one projection:  out = bf16(base + s_a (x A_a^T) B_a^T), a = the row's adapter.
// A row whose id is outside [0, n_adapters) has none: out = base.
#include <algorithm>

#include "xq_common.h"

namespace xq {
namespace {

struct AdapterArgs {
    xq_adapters q;
    float* t;             // [M, r]: x A_a^T
};

// the adapter of a row, or -1
__device__ __forceinline__ int adapter_of(const xq_adapters& q, int64_t row) {
    const int64_t id = q.id_bytes == 8 ? ((const int64_t*)q.ids)[row] : ((const int32_t*)q.ids)[row];
    return id >= 0 && id < q.n_adapters ? (int)id : -1;
}
__device__ __forceinline__ float load_factor(const void* p, int dtype, int64_t at) {
    return dtype == XQ_DT_F32 ? ((const float*)p)[at] : bf16_to_f32(((const bf16_t*)p)[at]);
}

// a wave a value of t
__global__ void __launch_bounds__(256) adapter_down_kernel(AdapterArgs a) {
    const xq_adapters& q = a.q;
    for (int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); at < q.M * q.r; at += (int64_t)gridDim.x * 4) {
        const int64_t row = at / q.r, j = at - row * q.r;
        const int id = adapter_of(q, row);
        float sum = 0.0f;
        if (id >= 0)
            for (int64_t k = threadIdx.x & 63; k < q.K; k += 64)
                sum = fmaf(bf16_to_f32(((const bf16_t*)q.x)[row * q.ldx + k]), load_factor(q.A, q.factor_dtype, ((int64_t)id * q.r + j) * q.K + k), sum);
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if ((threadIdx.x & 63) == 0) a.t[at] = sum;
    }
}

__global__ void __launch_bounds__(256) adapter_up_kernel(AdapterArgs a) {
    const xq_adapters& q = a.q;
    const int64_t chunks = (q.N + 255) / 256;
    for (int64_t at = blockIdx.x; at < q.M * chunks; at += gridDim.x) {
        const int64_t row = at / chunks, n = (at - row * chunks) * 256 + threadIdx.x;
        if (n >= q.N) continue;
        const int id = adapter_of(q, row);
        const bf16_t base = ((const bf16_t*)q.base)[row * q.ld_base + n];
        bf16_t out = base;
        if (id >= 0) {
            float sum = 0.0f;
            for (int j = 0; j < q.r; ++j) sum = fmaf(a.t[row * q.r + j], load_factor(q.B, q.factor_dtype, ((int64_t)id * q.N + n) * q.r + j), sum);
            out = to_bf16(fmaf(q.scaling[id], sum, bf16_to_f32(base)));
        }
        ((bf16_t*)q.out)[row * q.ld_out + n] = out;
    }
}

bool sizes_fit(int64_t M, int64_t N, int64_t K, int r) {
    return M >= 0 && M < (1 << 24) && N >= 16 && N < (1 << 24) && N % 16 == 0 && K >= 64 && K < (1 << 24) && K % 64 == 0 && r >= 1 && r <= 64;
}

}  // namespace
}  // namespace xq

using namespace xq;

extern "C" int64_t xq_adapters_workspace_bytes(int64_t M, int64_t N, int64_t K, int r) {
    if (!sizes_fit(M, N, K, r)) return -1;
    return M * r * 4 + 256;
}

extern "C" int xq_adapters_add(const xq_adapters* q, void* workspace, int64_t workspace_bytes, void* stream) {
    XQ_REQUIRE(q, "xq_adapters_add: the problem is NULL");
    XQ_REQUIRE(sizes_fit(q->M, q->N, q->K, q->r), "xq_adapters_add: %lld rows, [%lld, %lld], rank %d: in_features must be a multiple of 64, out_features of 16, the rank 1 to 64",
               (long long)q->M, (long long)q->N, (long long)q->K, q->r);
    XQ_REQUIRE(q->n_adapters >= 0, "xq_adapters_add: %d adapters", q->n_adapters);
    XQ_REQUIRE(q->factor_dtype == XQ_DT_F32 || q->factor_dtype == XQ_DT_BF16, "xq_adapters_add: factors are fp32 or bf16");
    XQ_REQUIRE(q->id_bytes == 4 || q->id_bytes == 8, "xq_adapters_add: ids are int32 or int64, got %d bytes", q->id_bytes);
    if (q->M == 0) return XQ_OK;
    XQ_REQUIRE(q->ids && xq_aligned(q->ids, q->id_bytes), "xq_adapters_add: ids are NULL or misaligned");
    XQ_REQUIRE(q->n_adapters == 0 || (q->A && q->B && q->scaling && xq_aligned(q->A, 16) && xq_aligned(q->B, 16) && xq_aligned(q->scaling, 4)),
               "xq_adapters_add: factors or scalings are NULL or misaligned");
    const struct { const void* p; int64_t ld, width; const char* name; } rows[] = {
        {q->x, q->ldx, q->K, "x"}, {q->base, q->ld_base, q->N, "base"}, {q->out, q->ld_out, q->N, "out"}};
    for (const auto& m : rows)
        XQ_REQUIRE(m.p && xq_aligned(m.p, 16) && m.ld >= m.width && m.ld % 8 == 0, "xq_adapters_add: %s must be 16-byte aligned with a row stride that is a multiple of 8 elements", m.name);
    XQ_REQUIRE(workspace && xq_aligned(workspace, 256) && workspace_bytes >= xq_adapters_workspace_bytes(q->M, q->N, q->K, q->r),
               "xq_adapters_add: a workspace of %lld bytes, 256-byte aligned, is needed", (long long)xq_adapters_workspace_bytes(q->M, q->N, q->K, q->r));
    hipStream_t st = (hipStream_t)stream;
    const AdapterArgs a = {*q, (float*)workspace};
    adapter_down_kernel<<<dim3((unsigned)std::min<int64_t>(xq_cdiv(q->M * q->r, 4), 1 << 22)), 256, 0, st>>>(a);
    adapter_up_kernel<<<dim3((unsigned)std::min<int64_t>(q->M * xq_cdiv(q->N, 256), 1 << 22)), 256, 0, st>>>(a);
    XQ_CHECK_LAUNCH("xq_adapters_add");
    return XQ_OK;
}
