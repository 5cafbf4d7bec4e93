// The choice of experts: scores, groups, top-k, weights, and the gradient of the router's logits.
//
//   s = softmax(z) or sigmoid(z)     c = s + bias, without a bias the order of z      chosen: the top_k largest c in the top_groups best groups
//   w = scale s_chosen / (renormalize: sum of the chosen s, otherwise 1)
// An expert whose logit or bias is -inf is out: never chosen, and its group is as strong as it is without it.  Places that no expert is left for
// hold id -1 and weight 0.  A NaN in a row (an infinite logit under softmax too) makes its weights and its gradient NaN, its ids 0 .. top_k - 1.
#include <algorithm>

#include "xq_common.h"

namespace xq {
namespace {

constexpr int kMaxExperts = 1024, kMaxTopK = 32, kMaxGroups = 64;

struct RouteArgs {
    xq_moe_route q;
    float* weights;
    int64_t* selected;
    bool wide, wide_bias;         // rows of logits, and the bias, are read in fours
    uint32_t per_group;           // ceil(2^32 / experts of a group): their quotient is the high word of a product (below 2^16)
};
struct RouteGradArgs {
    xq_moe_route q;
    const float* weights;
    const int64_t* selected;
    const float* grad;
    void* dz;
    int64_t ld_dz;
    bool wide, wide_dz;
};

// L lanes have a row (16: four rows a wave, sums and maxima within a quarter of it are register moves), V logits each, four neighbours at a time: lane l has
// experts (j L + l) 4 + i.  A block is one wave: what goes through LDS needs no barrier.
//
// Without a bias the order is that of the logits, exactly.  A score with a bias is compared as fp32 where that tells the chosen apart from each other and from the
// first that is left out: sums whose difference is within their error, of experts that differ in logit or bias, send the row to be done again in 64 bits, which is the definition.
// Groups by two scores likewise, at the border between those that stay and those that go.  Errors, in steps of 2^-24 of a score: sigmoid 4 for the exponential, 2 for
// sum and quotient; softmax 88 for the difference in the exponent (below that there is no score), 4, 22 for the sum (16 terms a lane, 6 steps), 1; one
// more, of itself, for the sum with the bias.
constexpr float kSigmoidError = 0x1p-20f, kSoftmaxError = 0x1p-17f;

template <int L>
struct Lanes {
    // the value of all L lanes, the same in each
    template <typename T, typename F>
    static __device__ __forceinline__ T all(T v, F f) {
        v = f(v, move<0x128>(v));                          // from 8, 4, 2, 1 lanes around in the row of 16
        v = f(v, move<0x124>(v));
        v = f(v, move<0x122>(v));
        v = f(v, move<0x121>(v));
        if (L == 64) {                                     // rows of 16, then halves, change places
            v = swapped<16>(v, f);
            v = swapped<32>(v, f);
        }
        return v;
    }
    template <int BY>
    static __device__ __forceinline__ u32x2 swap(uint32_t v) {
        const auto r = BY == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return u32x2{r[0], r[1]};
    }
    template <int BY, typename F>
    static __device__ __forceinline__ float swapped(float v, F f) {
        const u32x2 r = swap<BY>(__float_as_uint(v));
        return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    template <int BY, typename F>
    static __device__ __forceinline__ int swapped(int v, F f) {
        const u32x2 r = swap<BY>((uint32_t)v);
        return f((int)r[0], (int)r[1]);
    }
    template <int BY, typename F>
    static __device__ __forceinline__ double swapped(double v, F f) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const u32x2 lo = swap<BY>((uint32_t)u), hi = swap<BY>((uint32_t)(u >> 32));
        return f(__builtin_bit_cast(double, lo[0] | (uint64_t)hi[0] << 32), __builtin_bit_cast(double, lo[1] | (uint64_t)hi[1] << 32));
    }
    template <int HOW>
    static __device__ __forceinline__ float move(float v) { return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), HOW, 0xf, 0xf, true)); }
    template <int HOW>
    static __device__ __forceinline__ int move(int v) { return __builtin_amdgcn_update_dpp(0, v, HOW, 0xf, 0xf, true); }
    template <int HOW>
    static __device__ __forceinline__ double move(double v) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint64_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, HOW, 0xf, 0xf, true), hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), HOW, 0xf, 0xf, true);
        return __builtin_bit_cast(double, lo | hi << 32);
    }
    template <typename T>
    static __device__ __forceinline__ T largest(T v) { return all(v, [](T a, T b) { return a > b ? a : b; }); }
    template <typename T>
    static __device__ __forceinline__ T sum(T v) { return all(v, [](T a, T b) { return a + b; }); }
    static __device__ __forceinline__ int least(int v) { return all(v, [](int a, int b) { return min(a, b); }); }
    static __device__ __forceinline__ bool any(bool v) { return all((int)v, [](int a, int b) { return a | b; }) != 0; }
};

__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ float logit(const float* row, int e) { return row[e]; }
__device__ __forceinline__ float logit(const bf16_t* row, int e) { return bf16_to_f32(row[e]); }

// a lane's part of a row, `none` behind its end
template <typename T, int L, int V>
__device__ __forceinline__ void load_row(const T* row, int E, bool wide, int l, float none, float (&z)[V]) {
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
        const int e = (j * L + l) * 4;
        if (wide) {                                        // (whole fours at aligned addresses)
            if (e < E) {
                if constexpr (sizeof(T) == 4) {
                    const f32x4 v = *(const f32x4*)(row + e);
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[j * 4 + i] = v[i];
                } else {
                    const u32x2 v = *(const u32x2*)(row + e);
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[j * 4 + i] = bf16_to_f32((bf16_t)(v[i >> 1] >> (i & 1) * 16));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) z[j * 4 + i] = none;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                z[j * 4 + i] = none;
                if (e + i < E) {
                    if constexpr (sizeof(T) == 4) z[j * 4 + i] = row[e + i];
                    else z[j * 4 + i] = bf16_to_f32(row[e + i]);
                }
            }
        }
    }
}

// e^v for comparisons: 2^t of the hardware and what t leaves of v log2(e), 4 steps of 2^-24 in all; nothing below 2^-126
__device__ __forceinline__ float exp_of(float v) {
    const float t = v * 0x1.715476p+0f, rest = fmaf(v, 0x1.715476p+0f, -t) + v * 0x1.4ae0cp-26f, p = __builtin_amdgcn_exp2f(t);
    return v < -88.0f ? 0.0f : fmaf(p, rest * 0x1.62e43p-1f, p);
}
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float reciprocal(float v) { return __builtin_amdgcn_rcpf(v); }
__device__ __forceinline__ double reciprocal(double v) { return 1.0 / v; }

// what the steps of a row share in LDS
template <int L, int V>
struct RowPlace {
    double value[L * V];                                   // as R: scores by expert; or the two largest of every four
    double strength[kMaxGroups];
    float at[kMaxTopK + 1];                                // what the chosen, and the first left out, were chosen by
    int e[kMaxTopK + 1];
};

template <typename R>
__device__ __forceinline__ void take_in(R c, R& first, R& second) {
    const R low = c < first ? c : first;
    second = second > low ? second : low;
    first = first > c ? first : c;
}

// One choice with R = float or double: false where float cannot tell.  top, total: the row's largest logit and sum of exponentials (softmax)
template <typename R, typename T, int L, int V>
__device__ __forceinline__ bool choose(const RouteArgs& a, const T* row, const float (&z)[V], const float (&b)[V], float bias_most, R top, R total, int l, RowPlace<L, V>* place) {
    using A = Lanes<L>;
    const xq_moe_route& q = a.q;
    const R kOut = -INFINITY;
    const int E = q.num_experts, K = q.top_k;
    const bool has_bias = q.bias != nullptr, grouped = q.top_groups < q.num_groups, soft = q.scoring == XQ_ROUTE_SOFTMAX;
    const bool two = grouped && q.group_score == XQ_ROUTE_GROUP_SUM2, scored = has_bias || two;
    const float error = soft ? kSoftmaxError : kSigmoidError;
    bool sure = true;
    R v[V];                                                // what is compared
    R* value = (R*)place->value;
    R* strength = (R*)place->strength;
    const int size = E / q.num_groups;
    const bool fours = size % 4 == 0;
    const R over = scored && soft ? reciprocal(total) : (R)1;
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
        R c[4];                                            // what counts for a group
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = j * 4 + k;
            R s = 0;
            if (scored) s = soft ? exp_of((R)z[i] - top) * over : reciprocal((R)1 + exp_of(-(R)z[i]));
            const bool out = z[i] == -INFINITY || b[i] == -INFINITY;
            v[i] = out ? kOut : has_bias ? s + (R)b[i] : (R)z[i];
            c[k] = out || !two || has_bias ? v[i] : s;
        }
        if (grouped && fours) {
            R first = c[0] > c[1] ? c[0] : c[1], second = c[0] > c[1] ? c[1] : c[0];
            take_in(c[2], first, second);
            take_in(c[3], first, second);
            value[(j * L + l) * 2] = first;
            value[(j * L + l) * 2 + 1] = second;
        } else if (grouped) {
#pragma unroll
            for (int k = 0; k < 4; ++k) value[(j * L + l) * 4 + k] = c[k];
        }
    }
    if (grouped) {
        wave_fence();
        const int G = q.num_groups, n = fours ? size / 2 : size;
        for (int g = l; g < G; g += L) {
            R first = kOut, second = kOut;
#pragma unroll 8
            for (int k = 0; k < n; ++k) take_in(value[g * n + k], first, second);
            strength[g] = first + (two && second != kOut ? second : (R)0);
        }
        wave_fence();
        // a group stays if fewer than top_groups are better; float: the weakest that stays and the strongest that goes have to lie apart
        R least = INFINITY, most = kOut;
        uint64_t kept = 0;
        for (int mine = l; mine < G; mine += L) {
            const R own = strength[mine];
            int better = 0;
#pragma unroll 8
            for (int h = 0; h < G; ++h) {
                const R other = strength[h];
                better += other > own || (other == own && h < mine);
            }
            if (better < q.top_groups) {
                least = least < own ? least : own;
                kept |= 1ull << mine;
            } else {
                most = most > own ? most : own;
            }
        }
        const int lo = A::all((int)(uint32_t)kept, [](int x, int y) { return x | y; }), hi = G > 32 ? A::all((int)(kept >> 32), [](int x, int y) { return x | y; }) : 0;
        kept = (uint32_t)lo | (uint64_t)(uint32_t)hi << 32;
        if (sizeof(R) == 4 && scored) {
            least = -A::largest(-least);
            most = A::largest(most);
            // (two scores and the sums with the bias on either side)
            if (most != kOut && !(least - most > (R)(2 * error) * (fabsf((float)least) + fabsf((float)most) + 4 * bias_most))) sure = false;
        }
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            const int e = (j * L + l) * 4;
            if (fours) {
                const bool stays = kept >> (__umulhi((uint32_t)e, a.per_group) & 63) & 1;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[j * 4 + i] = stays ? v[j * 4 + i] : kOut;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[j * 4 + i] = kept >> ((size == 1 ? e + i : (int)__umulhi((uint32_t)(e + i), a.per_group)) & 63) & 1 ? v[j * 4 + i] : kOut;
            }
        }
    }
    const int picks = K + (sizeof(R) == 4 && has_bias ? 1 : 0);
    int k = 0;
    for (; k < picks; ++k) {
        R best = v[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = best > v[i] ? best : v[i];
        const R m = A::largest(best);
        if (m == kOut) break;                              // none left
        int at = -1;
#pragma unroll
        for (int i = V - 1; i >= 0; --i) at = v[i] == m ? i : at;
        const int mine = at >= 0 ? ((at >> 2) * L + l) * 4 + (at & 3) : kMaxExperts, e = A::least(mine);
        if (mine != e) at = -1;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i == at ? kOut : v[i];
        if (l == 0) {
            place->at[k] = (float)m;
            place->e[k] = e;
        }
    }
    if (l == 0)
        for (; k < picks; ++k) place->e[k] = -1;
    wave_fence();
    if (sizeof(R) == 4 && has_bias)
        for (int i = l; i + 1 < picks; i += L) {
            const int e = place->e[i], f = place->e[i + 1];
            if (e < 0 || f < 0) continue;
            const float x = place->at[i], y = place->at[i + 1];
            if (x - y > error * (fabsf(x) + fabsf(y) + 2 * bias_most)) continue;
            if (logit(row, e) != logit(row, f) || q.bias[e] != q.bias[f]) sure = false;
        }
    return !A::any(!sure);
}

template <typename T, int L, int V>
__global__ void __launch_bounds__(64) moe_route_kernel(RouteArgs a) {
    using A = Lanes<L>;
    __shared__ RowPlace<L, V> places[64 / L];
    const xq_moe_route& q = a.q;
    const int l = threadIdx.x & (L - 1), E = q.num_experts, K = q.top_k;
    RowPlace<L, V>* place = places + threadIdx.x / L;
    const bool soft = q.scoring == XQ_ROUTE_SOFTMAX;
    for (int64_t row = (int64_t)blockIdx.x * (64 / L) + threadIdx.x / L; row < q.n_tokens; row += (int64_t)gridDim.x * (64 / L)) {
        float z[V], b[V];
        const T* from = (const T*)q.logits + row * q.ld;
        load_row<T, L, V>(from, E, a.wide, l, -INFINITY, z);
        if (q.bias) {
            load_row<float, L, V>(q.bias, E, a.wide_bias, l, 0.0f, b);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) b[i] = 0.0f;
        }
        float top = -INFINITY, most = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            bad |= z[i] != z[i] || b[i] != b[i];
            top = fmaxf(top, z[i]);
            if (b[i] != -INFINITY) most = fmaxf(most, fabsf(b[i]));
        }
        top = A::largest(top);
        bad = A::any(bad || (soft && top == INFINITY));
        most = q.bias ? A::largest(most) : 0.0f;
        if (bad) {
            for (int k = l; k < K; k += L) {
                a.weights[row * K + k] = NAN;
                a.selected[row * K + k] = k;
            }
            continue;
        }
        // the scores' denominator where anything needs it: chosen by scores, or weights that are not renormalized
        float total = 0.0f;
        const bool sums = soft && top != -INFINITY;
        if (sums && (q.bias || !q.renormalize || (q.group_score == XQ_ROUTE_GROUP_SUM2 && q.top_groups < q.num_groups))) {
#pragma unroll
            for (int i = 0; i < V; ++i) total += q.renormalize ? exp_of(z[i] - top) : expf(z[i] - top);
            total = A::sum(total);
        }
        if (!choose<float, T, L, V>(a, from, z, b, most, top, total, l, place)) {
            double total64 = 0.0;
            if (sums) {
#pragma unroll
                for (int i = 0; i < V; ++i) total64 += exp((double)z[i] - (double)top);
                total64 = A::sum(total64);
            }
            choose<double, T, L, V>(a, from, z, b, most, (double)top, total64, l, place);
        }
        // the weights.  Renormalized: exp(z - largest chosen) under softmax; under sigmoid e^(z - m) / (1 + e^z) with m the largest chosen if that is negative, so
        // that scores which are no fp32 numbers keep their ratios
        constexpr int N = (kMaxTopK + L - 1) / L;
        float x[N], w[N], chosen = -INFINITY, sum = 0.0f;
        int e[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = i * L + l;
            e[i] = k < K ? place->e[k] : -1;
            x[i] = e[i] < 0 ? -INFINITY : q.bias ? logit(from, e[i]) : place->at[k];
            chosen = fmaxf(chosen, x[i]);
        }
        chosen = A::largest(chosen);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w[i] = 0.0f;
            if (e[i] >= 0) {
                if (soft) w[i] = q.renormalize ? expf(x[i] - chosen) : expf(x[i] - top) / total;
                else if (x[i] >= 0.0f) w[i] = 1.0f / (1.0f + expf(-x[i]));
                else w[i] = expf(q.renormalize ? x[i] - fminf(chosen, 0.0f) : x[i]) / (1.0f + expf(x[i]));
            }
            sum += w[i];
        }
        sum = q.renormalize ? A::sum(sum) : 1.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = i * L + l;
            if (k < K) {
                a.weights[row * K + k] = sum > 0.0f ? q.scale * (w[i] / sum) : 0.0f;
                a.selected[row * K + k] = e[i];
            }
        }
        wave_fence();                                      // (the place is the next row's)
    }
}

// dz of a row: with g = scale * dw and u = w / scale
//   renormalized: d = u (g - sum g u), under sigmoid times 1 - s        softmax as it is: p_j (g_j - sum g p) for every j        sigmoid: g s (1 - s)
template <typename T, int L, int V>
__global__ void __launch_bounds__(64) moe_route_grad_kernel(RouteGradArgs a) {
    using A = Lanes<L>;
    __shared__ float places[64 / L][L * V];
    const xq_moe_route& q = a.q;
    const int l = threadIdx.x & (L - 1), E = q.num_experts, K = q.top_k;
    const bool soft = q.scoring == XQ_ROUTE_SOFTMAX;
    float* place = places[threadIdx.x / L];
    for (int64_t row = (int64_t)blockIdx.x * (64 / L) + threadIdx.x / L; row < q.n_tokens; row += (int64_t)gridDim.x * (64 / L)) {
        constexpr int N = (kMaxTopK + L - 1) / L;
        float u[N], g[N], dot = 0.0f;
        int id[N];
        bool bad = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = i * L + l;
            const int64_t at = row * K + min(k, K - 1), e = a.selected[at];
            const float w = a.weights[at];
            id[i] = k < K && e >= 0 && e < E ? (int)e : -1;
            bad |= w != w;
            u[i] = w / q.scale;
            g[i] = id[i] >= 0 ? q.scale * a.grad[at] : 0.0f;
            if (id[i] >= 0) dot += g[i] * u[i];
        }
        bad = A::any(bad);
        dot = A::sum(dot);
        float z[V], top = 0.0f, total = 1.0f;
        const bool whole = soft && !q.renormalize;
        if (whole) {
            load_row<T, L, V>((const T*)q.logits + row * q.ld, E, a.wide, l, -INFINITY, z);
            top = -INFINITY;
#pragma unroll
            for (int i = 0; i < V; ++i) top = fmaxf(top, z[i]);
            top = A::largest(top);
            total = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                z[i] = top == -INFINITY ? 0.0f : expf(z[i] - top);
                total += z[i];
            }
            total = A::sum(total);
        }
#pragma unroll
        for (int j = 0; j < V / 4; ++j) *(f32x4*)(place + (j * L + l) * 4) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        wave_fence();
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (id[i] >= 0) {
                float d = q.renormalize ? u[i] * (g[i] - dot) : g[i] * u[i];
                if (!soft) {
                    const T raw = ((const T*)q.logits)[row * q.ld + id[i]];
                    float x;
                    if constexpr (sizeof(T) == 4) x = raw;
                    else x = bf16_to_f32(raw);
                    const float t = expf(-fabsf(x)), rest = x > 0.0f ? t / (1.0f + t) : 1.0f / (1.0f + t);       // 1 - s
                    d *= rest;
                }
                place[id[i]] = d;
            }
        wave_fence();
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            const int e = (j * L + l) * 4;
            f32x4 d = *(const f32x4*)(place + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (whole && total > 0.0f) d[i] -= z[j * 4 + i] / total * dot;
                if (bad) d[i] = NAN;
            }
            T* to = (T*)a.dz + row * a.ld_dz + e;
            if (a.wide_dz) {
                if (e < E) {
                    if constexpr (sizeof(T) == 4) *(f32x4*)to = d;
                    else *(u32x2*)to = u32x2{pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3])};
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (e + i < E) {
                        if constexpr (sizeof(T) == 4) to[i] = d[i];
                        else to[i] = to_bf16(d[i]);
                    }
            }
        }
        wave_fence();                                      // (the place is the next row's)
    }
}

// four elements at a time: whole fours, at addresses that are multiples of them
bool in_fours(const void* p, int dtype, int64_t rows, int64_t ld, int E) { return p && E % 4 == 0 && (rows <= 1 || ld % 4 == 0) && xq_aligned(p, dtype == XQ_DT_F32 ? 16 : 8); }

constexpr int64_t kFewRows = 2048;

template <typename T, int L, int V>
void launch(const RouteArgs* f, const RouteGradArgs* g, hipStream_t st) {
    const xq_moe_route& q = f ? f->q : g->q;
    const dim3 blocks((unsigned)std::min<int64_t>(xq_cdiv(q.n_tokens, 64 / L), 1 << 24));
    if (f) moe_route_kernel<T, L, V><<<blocks, 64, 0, st>>>(*f);
    else moe_route_grad_kernel<T, L, V><<<blocks, 64, 0, st>>>(*g);
}
template <typename T>
void launch(const RouteArgs* f, const RouteGradArgs* g, hipStream_t st) {
    const xq_moe_route& q = f ? f->q : g->q;
    const int E = q.num_experts;
    if (E > 512) launch<T, 64, 16>(f, g, st);
    else if (E > 256) launch<T, 64, 8>(f, g, st);
    else if (q.n_tokens <= kFewRows) launch<T, 64, 4>(f, g, st);
    else if (E > 128) launch<T, 16, 16>(f, g, st);
    else if (E > 64) launch<T, 16, 8>(f, g, st);
    else launch<T, 16, 4>(f, g, st);
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
    const RouteArgs a = {*q, weights, selected, in_fours(q->logits, q->dtype, q->n_tokens, q->ld, q->num_experts), in_fours(q->bias, XQ_DT_F32, 1, 0, q->num_experts),
                         (uint32_t)(((1ull << 32) + q->num_experts / q->num_groups - 1) / (q->num_experts / q->num_groups))};
    q->dtype == XQ_DT_F32 ? launch<float>(&a, nullptr, (hipStream_t)stream) : launch<bf16_t>(&a, nullptr, (hipStream_t)stream);
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
    const RouteGradArgs a = {*q, weights, selected, grad, dlogits, ld_dlogits, in_fours(q->logits, q->dtype, q->n_tokens, q->ld, q->num_experts),
                             in_fours(dlogits, q->dtype, q->n_tokens, ld_dlogits, q->num_experts)};
    q->dtype == XQ_DT_F32 ? launch<float>(nullptr, &a, (hipStream_t)stream) : launch<bf16_t>(nullptr, &a, (hipStream_t)stream);
    XQ_CHECK_LAUNCH("xq_moe_route_bwd");
    return XQ_OK;
}
