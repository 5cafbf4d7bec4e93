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

// What bounds it: a row is read once and a few numbers of it written, but a choice is a chain of maxima over lanes, about 1500 instructions for four rows of 256 with
// groups and a bias.  Their issue is 41 of the 62 us that 65536 such rows take (the reads alone would be 14); 16384 rows of 128 take 7.4 us.  Small calls are one launch:
// one row 4.2 us, 333 rows of 256 in groups 7.4 of a pass.
//
// L lanes have a row (16: four rows a wave, sums and maxima within a quarter of it are register moves), V logits each, four neighbours at a time; of 16 lanes each
// next such round begins four lanes on, so that the experts of a few groups are not all in a few lanes.  A block is one wave: what goes through LDS needs no
// barrier.  With one row a wave and the same steps 65536 rows in groups took 154 us.
//
// Without a bias the order is that of the logits, exactly.  A score with a bias is compared as fp32 where that tells the chosen apart from each other and from
// those that are left out: sums whose difference is within their error, of experts that differ in logit or bias, send the row to be done again in 64 bits, which is
// the definition (every score in 64 bits: 524 us).  Groups by two scores likewise, at the border between those that stay and those that go, equal groups too.  What that makes of
// 65536 rows of 256 (us, a pass): in groups 57, where all logits and biases are equal 309, with biases of the type's lowest value, in whose error all scores lie, 236; without
// groups 44, 134 and 166.  Errors, in steps of
// 2^-24 of a score: sigmoid 4 for the exponential, 2 for sum and quotient; softmax 88 for the difference in the exponent (below that there is no score), 4, 22 for
// the sum (16 terms a lane, 6 steps), 1; one more, of itself, for the sum with the bias.
// Scores below 2^-125 may be 0 here: what lies nearer than kNoScore is told apart in 64 bits too.
constexpr float kSigmoidError = 0x1p-20f, kSoftmaxError = 0x1p-17f, kNoScore = 0x1p-120f;

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
    // (L 16) the n-th largest of the lanes' values
    template <typename T>
    static __device__ __forceinline__ T nth(T v, int n) {
        int larger = 0;
        T r = v;
#pragma unroll
        for (int i = 1; i < 16; ++i) {
            r = move<0x121>(r);
            larger += r > v;
        }
        return all(larger < n ? v : (T)INFINITY, [](T a, T b) { return a < b ? a : b; });
    }
    // the next lane's value
    static __device__ __forceinline__ int next(int v) {
        return L == 16 ? __builtin_amdgcn_update_dpp(0, v, 0x101, 0xf, 0xf, true) : __shfl_down(v, 1, 64);
    }
    static __device__ __forceinline__ float next(float v) { return __uint_as_float((uint32_t)next((int)__float_as_uint(v))); }
    // (L 16) the sum of the lanes before
    static __device__ __forceinline__ int before(int v) {
        int u = v;
        u += __builtin_amdgcn_update_dpp(0, u, 0x111, 0xf, 0xf, true);      // from 1, 2, 4, 8 lanes below in the row, 0 where there is none
        u += __builtin_amdgcn_update_dpp(0, u, 0x112, 0xf, 0xf, true);
        u += __builtin_amdgcn_update_dpp(0, u, 0x114, 0xf, 0xf, true);
        u += __builtin_amdgcn_update_dpp(0, u, 0x118, 0xf, 0xf, true);
        return u - v;
    }
    static __device__ __forceinline__ uint64_t bits(uint64_t v) {
        auto either = [](int a, int b) { return a | b; };
        return (uint32_t)all((int)(uint32_t)v, either) | (uint64_t)(uint32_t)all((int)(v >> 32), either) << 32;
    }
    static __device__ __forceinline__ bool any(bool v) { return all((int)v, [](int a, int b) { return a | b; }) != 0; }
};

// the first expert of lane l's j-th four
template <int L>
__device__ __forceinline__ int first_of(int j, int l) { return (j * L + (L == 16 ? (l - 4 * j) & 15 : l)) * 4; }

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
        const int e = first_of<L>(j, l);
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
__device__ __forceinline__ float near_exp(float v) {
    const float t = v * 0x1.715476p+0f, rest = fmaf(v, 0x1.715476p+0f, -t) + v * 0x1.4ae0cp-26f, p = __builtin_amdgcn_exp2f(t);
    return v < -87.0f ? 0.0f : v > 88.0f ? INFINITY : fmaf(p, rest * 0x1.62e43p-1f, p);
}

// what the steps of a row share in LDS
template <int L, int V>
struct RowPlace {
    float value[L * V];       // what is compared by expert, the two largest of every four, those that are picked from
    float strength[kMaxGroups];
    int who[L == 16 ? 4 * L : 1];
};
// a wave's rows, or one row that the whole wave chooses for in 64 bits
template <int L, int V>
union WavePlace {
    RowPlace<L, V> rows[64 / L];
    struct {
        double value[L * V], strength[kMaxGroups];
    } wide;
};
// the k-th choice, in lane k
struct Chosen {
    int e;                    // or -1
    float at;                 // what it was chosen by
};

template <typename R>
__device__ __forceinline__ void take_in(R c, R& first, R& second) {
    const R low = c < first ? c : first;
    second = second > low ? second : low;
    first = first > c ? first : c;
}

// the largest values and whose they are, equal ones by their index
template <int L, int V>
__device__ __forceinline__ Chosen pick(float (&v)[V], const int (&who)[V], int picks, int l) {
    using A = Lanes<L>;
    Chosen c = {-1, 0.0f};
    for (int k = 0; k < picks; ++k) {
        float best = v[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = fmaxf(best, v[i]);
        const float m = A::largest(best);
        if (m == -INFINITY) break;
        int mine = kMaxExperts;
#pragma unroll
        for (int i = 0; i < V; ++i) mine = v[i] == m ? min(mine, who[i]) : mine;
        const int e = A::least(mine);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = who[i] == e ? -INFINITY : v[i];
        if (l == k) c = {e, m};
    }
    return c;
}
// among the first n of a list in LDS
template <int L, int V>
__device__ __forceinline__ Chosen pick_listed(const float* value, const int* who, int n, int picks, int l) {
    float v[V];
    int e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const bool is = i * L + l < n;
        v[i] = is ? value[i * L + l] : -INFINITY;
        e[i] = is ? who[i * L + l] : kMaxExperts;
    }
    return pick<L, V>(v, e, picks, l);
}

// among V of every lane in LDS, the i-th of lane l at i L + l: for the rows that have no short list, in few registers
template <int L, int V>
__device__ __forceinline__ Chosen pick_stored(float* value, int picks, int l) {
    using A = Lanes<L>;
    Chosen c = {-1, 0.0f};
#pragma unroll 1
    for (int k = 0; k < picks; ++k) {
        float best = -INFINITY;
        int at = -1;
#pragma unroll 4
        for (int i = 0; i < V; ++i) {                      // (not in order of the experts only where j turns around: the least of equal ones is looked for)
            const float v = value[i * L + l];
            const bool more = v > best || (v == best && at >= 0 && first_of<L>(i >> 2, l) + (i & 3) < first_of<L>(at >> 2, l) + (at & 3));
            best = more ? v : best;
            at = more ? i : at;
        }
        const float m = A::largest(best);
        if (m == -INFINITY) break;
        const int mine = first_of<L>(at >> 2, l) + (at & 3), e = A::least(best == m ? mine : kMaxExperts);
        if (best == m && mine == e) value[at * L + l] = -INFINITY;
        if (l == k) c = {e, m};
    }
    return c;
}

// The choice in 32 bits: false where they cannot tell.  top, total: the row's largest logit and sum of exponentials (softmax)
template <bool SOFT, bool SCORED, typename T, int L, int V>
__device__ __forceinline__ bool choose(const RouteArgs& a, const T* row, const float (&z)[V], const float (&b)[V], float bias_most, float top, float total, int l, RowPlace<L, V>* place, Chosen* chosen) {
    using A = Lanes<L>;
    const xq_moe_route& q = a.q;
    const float kOut = -INFINITY;
    const int E = q.num_experts, K = q.top_k;
    const bool has_bias = SCORED && q.bias != nullptr, grouped = q.top_groups < q.num_groups, two = SCORED && grouped && q.group_score == XQ_ROUTE_GROUP_SUM2;
    constexpr float error = SOFT ? kSoftmaxError : kSigmoidError;
    bool sure = true;
    float v[V];                                            // what is compared
    float* value = place->value;
    float* strength = place->strength;
    const int size = E / q.num_groups;
    const bool fours = size % 4 == 0;
    const float over = SCORED && SOFT ? __builtin_amdgcn_rcpf(total) : 1.0f;
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
        float c[4];                                        // what counts for a group
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = j * 4 + k;
            float s = 0.0f;
            if (SCORED) s = SOFT ? near_exp(z[i] - top) * over : __builtin_amdgcn_rcpf(1.0f + near_exp(-z[i]));
            const bool out = z[i] == -INFINITY;
            // (-inf with such a bias too; without one the bias is 0 here)
            v[i] = out ? kOut : has_bias ? s + b[i] : z[i];
            c[k] = !SCORED ? z[i] : out ? kOut : has_bias || two ? s + b[i] : z[i];
        }
        if (grouped && fours) {
            float first = fmaxf(c[0], c[1]), second = fminf(c[0], c[1]);
            take_in(c[2], first, second);
            take_in(c[3], first, second);
            value[first_of<L>(j, l) / 2] = first;
            value[first_of<L>(j, l) / 2 + 1] = second;
        } else if (grouped) {
#pragma unroll
            for (int k = 0; k < 4; ++k) value[first_of<L>(j, l) + k] = c[k];
        }
    }
    if (grouped) {
        wave_fence();
        const int G = q.num_groups, n = fours ? size / 2 : size;
        for (int g = l; g < G; g += L) {
            float first = kOut, second = kOut;
#pragma unroll 8
            for (int k = 0; k < n; ++k) take_in(value[g * n + k], first, second);
            const float both = first + (two && second != kOut ? second : 0.0f);
            if (SCORED && both == kOut && first != kOut) sure = false;        // (below every fp32 number, and yet above a group that has no experts)
            strength[g] = both;
        }
        wave_fence();
        // a group stays if fewer than top_groups are better; the weakest that stays and the strongest that goes have to lie apart
        float least = INFINITY, most = kOut;
        uint64_t kept = 0;
        for (int mine = l; mine < G; mine += L) {
            const float own = strength[mine];
            int better = 0;
#pragma unroll 8
            for (int h = 0; h < G; ++h) {
                const float other = strength[h];
                better += other > own || (other == own && h < mine);
            }
            if (better < q.top_groups) {
                least = fminf(least, own);
                kept |= 1ull << mine;
            } else {
                most = fmaxf(most, own);
            }
        }
        kept = A::bits(kept);
        if (SCORED) {
            least = -A::largest(-least);
            most = A::largest(most);
            // (two scores and the sums with the bias on either side)
            if (most != kOut && !(least - most > 2 * error * (fabsf(least) + fabsf(most) + 4 * bias_most) + kNoScore)) sure = false;
        }
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            const int e = first_of<L>(j, l);
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
    const int picks = K + (has_bias ? 1 : 0);              // (at most L)
    Chosen c;
    bool listed = false;
    if constexpr (L == 16 && V > 4) {
        // Many values a lane: the picks are among those that are at least as large as the picks-th of the lanes' largest, which are not many more
        // (256 values, 9 picks: 13 on average, 22 where half of the groups are out)
        float best = v[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = fmaxf(best, v[i]);
        const float border = A::nth(best, picks);
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) mine |= (v[i] >= border && v[i] != kOut ? 1u : 0u) << i;
        const int n = __popc(mine), before = A::before(n), all = A::sum(n);
        listed = all <= 4 * L;                             // (values in fewer lanes than there are picks, or many equal ones: not)
        if (listed) {
            int to = before;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (mine >> i & 1) {
                    value[to] = v[i];
                    place->who[to++] = first_of<L>(i >> 2, l) + (i & 3);
                }
            wave_fence();
            c = all <= 2 * L ? pick_listed<L, 2>(value, place->who, all, picks, l) : pick_listed<L, 4>(value, place->who, all, picks, l);
        }
    }
    if (!listed) {
        if constexpr (L == 16 && V > 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) value[i * L + l] = v[i];
            c = pick_stored<L, V>(value, picks, l);
        } else {
            int who[V];
#pragma unroll
            for (int i = 0; i < V; ++i) who[i] = first_of<L>(i >> 2, l) + (i & 3);
            c = pick<L, V>(v, who, picks, l);
        }
    }
    if (has_bias) {                                        // each against the next
        const float y = A::next(c.at);
        const int f = A::next(c.e);
        bool tied = false;
        if (l + 1 < picks && c.e >= 0 && f >= 0 && !(c.at - y > error * (fabsf(c.at) + fabsf(y) + 2 * bias_most) + kNoScore)) {
            const bool same = logit(row, c.e) == logit(row, f) && q.bias[c.e] == q.bias[f];
            sure &= same;
            tied = same && l == K - 1;
        }
        // The last chosen and the first left out are equal: by their index, if what lies as near as 32 bits tell is equal to them too (all of it is where a router
        // starts at zero: the row stays here).
        if (A::any(tied)) {
            const int last = A::largest(l == K - 1 ? c.e : -1);
            const float zl = logit(row, last), bl = q.bias[last], at = A::largest(l == K - 1 ? c.at : kOut);
#pragma unroll 1
            for (int e = l; e < E; e += L) {
                const float ze = logit(row, e), be = q.bias[e];
                if (ze == kOut || be == kOut || (ze == zl && be == bl)) continue;
                const float x = (SOFT ? near_exp(ze - top) * over : __builtin_amdgcn_rcpf(1.0f + near_exp(-ze))) + be;
                if (!(fabsf(x - at) > error * (fabsf(x) + fabsf(at) + 2 * bias_most) + kNoScore)) sure = false;
            }
        }
    }
    *chosen = c;
    return !A::any(!sure);
}

// The choice in 64 bits, of one row by the whole wave: rows that are chosen by scores, few of them
template <typename T, int L, int V>
__device__ __forceinline__ Chosen choose64(const RouteArgs& a, const T* row, float top, int l, WavePlace<L, V>* wave) {
    using A = Lanes<64>;
    auto* place = &wave->wide;
    const xq_moe_route& q = a.q;
    constexpr int N = L * V / 64, kTogether = N < 4 ? N : 4;          // experts a lane, l, l + 64, ..
    const double kOut = -INFINITY;
    const int E = q.num_experts, size = E / q.num_groups;
    const bool soft = q.scoring == XQ_ROUTE_SOFTMAX, grouped = q.top_groups < q.num_groups, two = q.group_score == XQ_ROUTE_GROUP_SUM2;
    double total = 0.0;
#pragma unroll kTogether
    for (int i = 0; i < N; ++i) {
        const double z = i * 64 + l < E ? (double)logit(row, i * 64 + l) : kOut;
        const double x = exp(soft ? z - (double)top : -z);
        place->value[i * 64 + l] = soft ? x : 1.0 / (1.0 + x);
        total += x;
    }
    total = soft ? A::sum(total) : 1.0;
#pragma unroll 1
    for (int e = l; e < 64 * N; e += 64) {
        const int at = min(e, E - 1);
        const double z = logit(row, at), bias = q.bias ? (double)q.bias[at] : 0.0;
        place->value[e] = e >= E || z == kOut || bias == kOut ? kOut : place->value[e] / total + bias;
    }
    if (grouped) {
        wave_fence();
        if (l < q.num_groups) {
            double first = kOut, second = kOut;
#pragma unroll 4
            for (int e = l * size; e < (l + 1) * size; ++e) take_in(place->value[e], first, second);
            place->strength[l] = first + (two && second != kOut ? second : 0.0);
        }
        wave_fence();
        const double own = l < q.num_groups ? place->strength[l] : kOut;
        int better = 0;
#pragma unroll 4
        for (int h = 0; h < q.num_groups; ++h) {
            const double other = place->strength[h];
            better += other > own || (other == own && h < l);
        }
        const uint64_t kept = __ballot(l < q.num_groups && better < q.top_groups);
#pragma unroll 1
        for (int e = l; e < E; e += 64) {
            if (!(kept >> (e / size) & 1)) place->value[e] = kOut;
            else if (!q.bias && place->value[e] != kOut) place->value[e] = logit(row, e);
        }
    }
    double v[N];                                           // (what this lane wrote)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = place->value[i * 64 + l];
    Chosen c = {-1, 0.0f};
#pragma unroll 1
    for (int k = 0; k < q.top_k; ++k) {
        double best = v[0];
#pragma unroll
        for (int i = 1; i < N; ++i) best = v[i] > best ? v[i] : best;
        const double m = A::largest(best);
        if (m == kOut) break;
        int mine = kMaxExperts;
#pragma unroll
        for (int i = N - 1; i >= 0; --i) mine = v[i] == m ? i * 64 + l : mine;
        const int e = A::least(mine);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i * 64 + l == e ? kOut : v[i];
        if (l == k) c = {e, (float)m};
    }
    return c;
}

// (16 lanes: four waves a SIMD, 128 registers)
template <typename T, int L, int V, bool SOFT, bool SCORED>
__global__ void __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(L == 16 ? 4 : 3))) moe_route_kernel(RouteArgs a) {
    using A = Lanes<L>;
    __shared__ WavePlace<L, V> places;
    const xq_moe_route& q = a.q;
    const int lane = threadIdx.x & (L - 1), E = q.num_experts, K = q.top_k;
    RowPlace<L, V>* place = places.rows + threadIdx.x / L;
    constexpr bool soft = SOFT;
    float b[V], most = 0.0f;
    bool bad_bias = false;
    if (SCORED && q.bias) {
        load_row<float, L, V>(q.bias, E, a.wide_bias, lane, 0.0f, b);
#pragma unroll
        for (int i = 0; i < V; ++i) bad_bias |= b[i] != b[i];
        bad_bias = A::any(bad_bias);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            b[i] = bad_bias ? 0.0f : b[i];                 // (then no row's choice matters)
            most = b[i] != -INFINITY ? fmaxf(most, fabsf(b[i])) : most;
        }
        most = A::largest(most);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) b[i] = 0.0f;
    }
    for (int64_t first = (int64_t)blockIdx.x * (64 / L); first < q.n_tokens; first += (int64_t)gridDim.x * (64 / L)) {
        int l = lane;
        asm volatile("" : "+v"(l));                        // (what follows from it is worked out again for every row: kept, it is 90 registers)
        const int64_t row = first + threadIdx.x / L;
        const bool real = row < q.n_tokens;                // (lanes behind the last row go along with it)
        const T* from = (const T*)q.logits + (real ? row : q.n_tokens - 1) * q.ld;
        float z[V], top = -INFINITY;
        bool bad = bad_bias;
        load_row<T, L, V>(from, E, a.wide, l, -INFINITY, z);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            bad |= z[i] != z[i];
            top = fmaxf(top, z[i]);
        }
        top = A::largest(top);
        bad = A::any(bad || (soft && top == INFINITY));
        if (bad) {
            top = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) z[i] = z[i] == -INFINITY ? -INFINITY : 0.0f;       // (a choice among equals, which is not used)
        }
        // the scores' denominator where anything needs it: chosen by scores, or weights that are not renormalized
        float total = 0.0f;
        const bool sums = soft && top != -INFINITY;
        if (sums && (SCORED || !q.renormalize)) {
#pragma unroll
            for (int i = 0; i < V; ++i) total += q.renormalize ? near_exp(z[i] - top) : expf(z[i] - top);
            total = A::sum(total);
        }
        Chosen c;
        [[maybe_unused]] const bool sure = choose<SOFT, SCORED, T, L, V>(a, from, z, b, most, top, total, l, place, &c);
        if constexpr (SCORED)
            for (uint64_t left = __ballot(!sure && !bad && real); left;) {
                const int of = __builtin_ctzll(left) / L;
                left &= L == 64 ? 0 : ~(0xffffull << of * L);
                wave_fence();
                const Chosen d = choose64<T, L, V>(a, (const T*)q.logits + (first + of) * q.ld, __shfl(top, of * L, 64), threadIdx.x, &places);
                const int e = __shfl(d.e, l, 64);
                const float at = __shfl(d.at, l, 64);
                if ((int)threadIdx.x / L == of) c = {e, at};
            }
        // the weights.  Renormalized: exp(z - largest chosen) under softmax; under sigmoid e^(z - m) / (1 + e^z) with m the largest chosen if that is negative, so
        // that scores which are no fp32 numbers keep their ratios
        const bool is = l < K && c.e >= 0;
        const float x = !is ? -INFINITY : SCORED && q.bias ? logit(from, c.e) : c.at, largest = A::largest(x);
        float w = 0.0f;
        if (is) {
            if (soft) w = q.renormalize ? expf(x - largest) : expf(x - top) / total;
            else if (x >= 0.0f) w = 1.0f / (1.0f + expf(-x));
            else w = expf(q.renormalize ? x - fminf(largest, 0.0f) : x) / (1.0f + expf(x));
        }
        const float sum = q.renormalize ? A::sum(w) : 1.0f;
        if (real && l < K) {
            a.weights[row * K + l] = bad ? NAN : sum > 0.0f ? q.scale * (w / sum) : 0.0f;
            a.selected[row * K + l] = bad ? l : is ? c.e : -1;
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
        for (int j = 0; j < V / 4; ++j) *(f32x4*)(place + first_of<L>(j, l)) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
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
            const int e = first_of<L>(j, l);
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

// From 129 to 256 experts few rows are done by 64 lanes each, whose chain is shorter, many by 16.  Sigmoid with a bias in groups, 64 against 16 lanes: one row 6.6 and
// 8.9 us, 512 rows 7.2 and 9.4, 4096 17.4 and 16.0, 8192 25 and 17.  Up to 128 experts 16 lanes are never behind (128: one row 4.5 and 4.6, 2048 rows 5.7 and 5.0, 8192 13.1
// and 5.7).  Rows of more choices than 16 lanes can hold, with the one behind them, take 64.
constexpr int64_t kFewRows = 2048;

template <typename T, int L, int V>
void launch(const RouteArgs* f, const RouteGradArgs* g, hipStream_t st) {
    const xq_moe_route& q = f ? f->q : g->q;
    const dim3 blocks((unsigned)std::min<int64_t>(xq_cdiv(q.n_tokens, 64 / L), 4096));        // (the 16 waves that a compute unit holds at 128 registers; then several rows each, the bias read once)
    if (f) {
        const bool scored = q.bias || (q.group_score == XQ_ROUTE_GROUP_SUM2 && q.top_groups < q.num_groups);
        if (q.scoring == XQ_ROUTE_SOFTMAX) scored ? moe_route_kernel<T, L, V, true, true><<<blocks, 64, 0, st>>>(*f) : moe_route_kernel<T, L, V, true, false><<<blocks, 64, 0, st>>>(*f);
        else scored ? moe_route_kernel<T, L, V, false, true><<<blocks, 64, 0, st>>>(*f) : moe_route_kernel<T, L, V, false, false><<<blocks, 64, 0, st>>>(*f);
    }
    else {
        moe_route_grad_kernel<T, L, V><<<blocks, 64, 0, st>>>(*g);
    }
}
template <typename T>
void launch(const RouteArgs* f, const RouteGradArgs* g, hipStream_t st) {
    const xq_moe_route& q = f ? f->q : g->q;
    const int E = q.num_experts;
    if (E > 512) launch<T, 64, 16>(f, g, st);
    else if (E > 256) launch<T, 64, 8>(f, g, st);
    else if (q.top_k > 15 || (E > 128 && q.n_tokens <= kFewRows)) launch<T, 64, 4>(f, g, st);
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
