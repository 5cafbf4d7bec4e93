// AdamW over many tensors at once, with 32- or 8-bit states, and the global norm of their gradients.
//
//   m' = b1 m + (1 - b1) g        v' = b2 v + (1 - b2) g^2        t = step + 1
//   p' = p - lr wd p - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)            g scaled by min(1, max_norm / (|g| + 1e-6))
//
// 8-bit states: blocks of 256 consecutive elements of a tensor share a scale each for m and for s = sqrt(v):
//   m = sign(c) (c / 127)^2 A_m   c in -127 .. 127          s = (d / 255)^2 A_s   d in 0 .. 255          A = the block's largest magnitude
// The squared codes spend their levels near zero, where most of a block lies: a code's neighbours are 2 / c of its value away, 0.8 % (d) and
// 1.6 % (c) at the top, and the smallest level is 1.5e-5 (s) of the largest.  s is kept, not v: v would need twice the range, and the
// update divides by s.  A positive s never takes code 0: the next step would divide its m by eps alone.  The update itself uses m' and s' as
// computed, before they are rounded to codes.  A NaN or an infinity in a block makes its scale NaN or infinite, so that it shows.
//
// Bound by memory: 28 bytes an element (fp32 parameters and gradients, 32-bit states) or 16.06 (8-bit ones).  The factors of a model are
// hundreds of tensors of 10^4 to 10^6 elements.  Their addresses change from step to step (autograd allocates gradients), so a call takes
// them by value: adamw_table_kernel's arguments carry 84 to 256 tensors a launch, and it writes them into a table in the workspace, with the
// step counts advanced and the bias corrections in 64 bits.  One launch then walks all tensors: chunks of 4096 elements, numbered through,
// are dealt out to the blocks in ranges; a block looks a chunk up in the table (two steps of 64 lanes) and goes on from there.
//
// 504 factors, 87 M elements: 465 us (fp32 states, 5.25 TB/s) and 268 us (8 bits, 5.2 TB/s), the norm 55 to 100 us before it; a [65536, 4096] bf16
// parameter with bf16 gradients: 614 us (10 bytes an element, 4.4 TB/s, near the vector units' limit); a large copy: 4.8 TB/s.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "xq_common.h"

namespace xq {
namespace {

constexpr int kBlock = 256;                 // elements that share a scale: a wave's four a lane
constexpr int kChunk = 4096;                // of a thread block at a time: four 256-element pieces of each of its waves
constexpr int kThreads = 256;
constexpr int kTableWords = 1008;           // of tensors by value in one launch: 4032 bytes, of the 4096 that arguments may take
constexpr int kNormBlocks = 2048;
constexpr int kStepBlocks = 2048;           // eight of a compute unit

struct Row {                                // what the walking kernels read of a tensor
    void* param;
    const void* grad;
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    int64_t numel;
    int64_t chunk0;                         // its first chunk, counted over all tensors
    float first, root;                      // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    int32_t param16, grad16;                // bf16 (otherwise fp32)
};

// A tensor in 3 words of 32 bits (its gradient alone), 9 (with 32-bit states) or 12: 504 factors are 5 or 6 launches of 2 to 5 us.
//   0  elements, low      1  elements, high (11 bits), bf16 parameter (bit 14), bf16 gradient (bit 15), gradient's top 16 bits      2  gradient
//   3 .. 6  parameter, states, step count; 7, 8  their top 16 bits, two a word      9 .. 11  scales, and theirs
struct TableArgs {
    uint32_t word[kTableWords];
    Row* rows;
    int32_t chunk0, n;
};
struct TableScalars {
    double lr, log_beta1, log_beta2;
    const float* lr_device;
};
static_assert(sizeof(TableArgs) + sizeof(TableScalars) <= 4096, "kernel arguments");
constexpr int table_tensors(int words) { return kTableWords / words < 256 ? kTableWords / words : 256; }
constexpr int kAddressBits = 48;
template <typename P>
__device__ __forceinline__ P* address(uint32_t low, uint32_t high16) { return (P*)((uint64_t)(high16 & 0xffffu) << 32 | low); }

template <int WORDS>
__global__ void __launch_bounds__(256) adamw_table_kernel(TableArgs a, TableScalars s) {
    __shared__ int wave_end[4];
    const int i = threadIdx.x, lane = i & 63, wave = i >> 6;
    const uint32_t* w = a.word + min(i, a.n - 1) * WORDS;
    const int64_t numel = (int64_t)(w[1] & 0x7ffu) << 32 | w[0];
    const int own = i < a.n ? (int)((numel + kChunk - 1) / kChunk) : 0;
    int end = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int before = __shfl_up(end, d);
        if (lane >= d) end += before;
    }
    if (lane == 63) wave_end[wave] = end;
    __syncthreads();
    if (i >= a.n) return;
    for (int k = 0; k < wave; ++k) end += wave_end[k];
    Row r = {};
    r.grad = address<const void>(w[2], w[1] >> 16);
    r.numel = numel;
    r.chunk0 = a.chunk0 + end - own;
    r.grad16 = (int)(w[1] >> 15 & 1);
    if constexpr (WORDS >= 9) {
        r.param16 = (int)(w[1] >> 14 & 1);
        r.param = address<void>(w[3], w[7]); r.m = address<void>(w[4], w[7] >> 16); r.v = address<void>(w[5], w[8]);
        float* const count = address<float>(w[6], w[8] >> 16);
        const float step = *count + 1.0f;
        *count = step;
        const double lr = s.lr_device ? (double)*s.lr_device : s.lr;
        r.first = (float)(lr / (1.0 - exp(step * s.log_beta1)));           // b^t; a beta of 0 has the logarithm -inf
        r.root = (float)(1.0 / sqrt(1.0 - exp(step * s.log_beta2)));
    }
    if constexpr (WORDS == 12) { r.m_scale = address<float>(w[9], w[11]); r.v_scale = address<float>(w[10], w[11] >> 16); }
    a.rows[i] = r;
}

// the last row whose first chunk is not behind `chunk` (rows in order of their first chunks, no row without chunks)
__device__ __forceinline__ int row_of(const Row* rows, int n, int64_t chunk, int lane) {
    const int step = (n + 63) >> 6;
    const int a = min(lane * step, n - 1);
    const int seg = __builtin_popcountll(__ballot(lane * step < n && rows[a].chunk0 <= chunk)) - 1;
    int at = seg * step;
    for (int base = at; base < min(n, at + step); base += 64) {
        const int k = base + lane;
        const uint64_t below = __ballot(k < min(n, (seg + 1) * step) && rows[min(k, n - 1)].chunk0 <= chunk);
        if (!below) break;
        at = base + __builtin_popcountll(below) - 1;
    }
    return __builtin_amdgcn_readfirstlane(at);
}

template <bool BF16>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
    return BF16 ? bf16_to_f32(((const bf16_t*)p)[i]) : ((const float*)p)[i];
}
// What a step reads and writes goes past the caches, but for the gradients: nothing else of it is read again before the next step, and the
// gradients that the norm read last are still there (504 factors, 87 M elements: 595 us otherwise, 545 so).
template <bool PAST, typename V>
__device__ __forceinline__ V load_as(const void* p) {
    if constexpr (PAST) return __builtin_nontemporal_load((const V*)p);
    else return *(const V*)p;
}
// four elements from i on.  WHOLE: all there, at an address for one access; otherwise one by one, zeros behind the tensor's end
template <bool WHOLE, bool PAST>
__device__ __forceinline__ f32x4 load4(bool bf16, const void* p, int64_t i, int64_t n) {
    if constexpr (WHOLE) {
        if (!bf16) return load_as<PAST, f32x4>((const float*)p + i);
        const u32x2 w = load_as<PAST, u32x2>((const bf16_t*)p + i);
        return f32x4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xffff0000u)};
    } else {
        f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) r[k] = bf16 ? load1<true>(p, i + k) : load1<false>(p, i + k);
        return r;
    }
}
template <bool WHOLE>
__device__ __forceinline__ void store4(bool bf16, void* p, int64_t i, int64_t n, f32x4 v) {
    if constexpr (WHOLE) {
        if (bf16) __builtin_nontemporal_store(u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])}, (u32x2*)((bf16_t*)p + i));
        else __builtin_nontemporal_store(v, (f32x4*)((float*)p + i));
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) {
                if (bf16) ((bf16_t*)p)[i + k] = to_bf16(v[k]);
                else ((float*)p)[i + k] = v[k];
            }
    }
}
template <bool WHOLE>
__device__ __forceinline__ uint32_t load4_codes(const void* p, int64_t i, int64_t n) {
    if constexpr (WHOLE) return load_as<true, uint32_t>((const uint8_t*)p + i);
    uint32_t r = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (i + k < n) r |= (uint32_t)((const uint8_t*)p)[i + k] << (8 * k);
    return r;
}
template <bool WHOLE>
__device__ __forceinline__ void store4_codes(void* p, int64_t i, int64_t n, uint32_t c) {
    if constexpr (WHOLE) {
        __builtin_nontemporal_store(c, (uint32_t*)((uint8_t*)p + i));
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) ((uint8_t*)p)[i + k] = (uint8_t)(c >> (8 * k));
    }
}
// whether four elements from a multiple of four on can be accessed as one
__device__ __forceinline__ bool whole4(const void* p, bool bf16) { return ((uintptr_t)p & (bf16 ? 7 : 15)) == 0; }

// the largest over a wave of the bits of non-negative floats: NaN lies above infinity, so that neither is lost
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
    // (0 for the lanes that get nothing: the identity, with which each step is one instruction)
    auto from = [](uint32_t x, auto ctrl, auto rows) {
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    };
    using All = std::integral_constant<int, 0xf>;
    v = max(v, from(v, std::integral_constant<int, 0xb1>{}, All{}));       // lanes 1, 0, 3, 2 of four
    v = max(v, from(v, std::integral_constant<int, 0x4e>{}, All{}));       // 2, 3, 0, 1
    v = max(v, from(v, std::integral_constant<int, 0x141>{}, All{}));      // mirrored within eight
    v = max(v, from(v, std::integral_constant<int, 0x140>{}, All{}));      // within sixteen
    v = max(v, from(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{}));     // lane 15 of a row of sixteen to the next
    v = max(v, from(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{}));     // lane 31 to the upper half
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t bits_abs(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// Codes of four elements: the nearest to 127 sqrt(|m| / A) and 255 sqrt(s / A), exactly.  A product, the hardware's root and the instruction
// that packs a byte (to nearest even, saturating; m goes in as 128 + c, whose top bit is flipped afterwards) decide all but the elements
// that come near the middle between two codes: the errors of reciprocal, product and root together are below 2e-7 (m) and 3e-7 (s, a root
// itself) of the code.  A wave with such an element, 7 % of them, compares |m| 127^2 with (c + 1/2)^2 A in 64 bits, where both sides
// are exact.  That a code does not hang on an ulp matters a step later: the neighbour of a small s is several per cent away.
__device__ __forceinline__ bool near_middle(float f, float by) { return fabsf(__builtin_amdgcn_fractf(f) - 0.5f) < by; }
__device__ __forceinline__ int exact_code(float x, float f, double top2, float amax) {
    const int c = (int)f;
    const double half = (double)c + 0.5, at = (double)x * top2, middle = half * half * (double)amax;
    return at > middle || (at == middle && (c & 1)) ? c + 1 : c;               // (in the middle: the even one)
}
__device__ __forceinline__ uint32_t m_codes(f32x4 m, float amax, float inv) {
    f32x4 f;
    bool near = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        f[k] = __builtin_amdgcn_sqrtf(fabsf(m[k]) * inv);
        near |= near_middle(f[k], 4e-5f);
    }
    if (__any(near)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = f[k] <= 127.0f ? (float)exact_code(fabsf(m[k]), f[k], 127.0 * 127.0, amax) : f[k];
    }
    uint32_t c = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_cvt_pk_u8_f32(128.0f + __builtin_copysignf(f[k], m[k]), k, c);
    return c ^ 0x80808080u;
}
__device__ __forceinline__ uint32_t s_codes(f32x4 s, f32x4 v, float amax, float inv) {
    f32x4 f;
    bool near = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        f[k] = __builtin_amdgcn_sqrtf(s[k] * inv);
        near |= near_middle(f[k], 1e-4f);
    }
    if (__any(near)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = f[k] <= 255.0f ? (float)exact_code(sqrtf(v[k]), f[k], 255.0 * 255.0, amax) : f[k];
    }
    uint32_t c = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float least = __builtin_amdgcn_fmed3f(s[k] * 0x1p120f, 0.0f, 1.0f);      // 1, or 0 for 0
        c = __builtin_amdgcn_cvt_pk_u8_f32(fmaxf(f[k], least), k, c);
    }
    return c;
}
// what they stand for: scale is the block's largest magnitude over the top code squared
__device__ __forceinline__ float m_value(uint32_t codes, int k, float scale) {
    const float c = (float)(int8_t)(codes >> (8 * k));
    return c * fabsf(c) * scale;
}
__device__ __forceinline__ float s_value(uint32_t codes, int k, float scale) {
    const float d = (float)((codes >> (8 * k)) & 0xffu);
    return d * d * scale;
}
constexpr float kM2 = 127.0f * 127.0f, kS2 = 255.0f * 255.0f;
constexpr float kSmallest = 1e-30f;         // blocks below it take the lowest codes: the quotient stays finite

struct StepArgs {
    const Row* rows;
    int64_t chunks;
    const float* norm;                      // of the gradients, or NULL
    int32_t n;
    float max_norm, beta1, beta2, one_minus_beta1, one_minus_beta2, eps, lr, weight_decay;
    const float* lr_device;
};

// constants of a call
struct Call {
    float clip, keep;                       // of the gradients; minus the decay
};

// a wave's four pieces of a chunk, from element base on (lane 0's) 1024 apart; everything is read before anything is computed
// (types known to the compiler where the pieces are whole: a branch on them between the loads would wait for each)
template <bool EIGHT, bool WHOLE, bool P16, bool G16>
__device__ __forceinline__ void step_chunk(const StepArgs& a, const Row& r, int64_t base, int lane, const Call& c) {
    constexpr int N = WHOLE ? 4 : 1;
    const bool p16 = WHOLE ? P16 : r.param16, g16 = WHOLE ? G16 : r.grad16;
    const int64_t n = r.numel;
#pragma unroll 1
    for (int u0 = 0; u0 < 4; u0 += N) {
        if (!WHOLE && base + u0 * (kThreads * 4) >= n) break;                // (the whole wave's piece lies behind the end)
        f32x4 p[N], g[N], m[N], v[N];
        uint32_t mc[N], vc[N];
        float ms[N], vs[N];
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int64_t i = base + (u0 + u) * (kThreads * 4) + lane * 4;
            g[u] = load4<WHOLE, false>(g16, r.grad, i, n);
            if constexpr (EIGHT) {
                mc[u] = load4_codes<WHOLE>(r.m, i, n);
                vc[u] = load4_codes<WHOLE>(r.v, i, n);
                ms[u] = r.m_scale[i >> 8];
                vs[u] = r.v_scale[i >> 8];
            } else {
                m[u] = load4<WHOLE, true>(false, r.m, i, n);
                v[u] = load4<WHOLE, true>(false, r.v, i, n);
            }
            p[u] = load4<WHOLE, true>(p16, r.param, i, n);
        }
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int64_t i = base + (u0 + u) * (kThreads * 4) + lane * 4;
            f32x4 s;
            uint32_t mb = 0, sb = 0;
            if constexpr (EIGHT) {
                // m' and v' by the formula's products and sums, each rounded as it stands: the codes are of these numbers.  For the update root and
                // reciprocal are the hardware's (an ulp each)
                const float mk = ms[u] * (1.0f / kM2), sk = vs[u] * (1.0f / kS2);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float gk = g[u][k] * c.clip, old = s_value(vc[u], k, sk);
                    m[u][k] = m_value(mc[u], k, mk) * a.beta1 + gk * a.one_minus_beta1;
                    v[u][k] = old * old * a.beta2 + gk * gk * a.one_minus_beta2;
                    s[k] = __builtin_amdgcn_sqrtf(v[u][k]);
                    p[u][k] = fmaf(p[u][k], c.keep, p[u][k]) - m[u][k] * r.first * __builtin_amdgcn_rcpf(fmaf(s[k], r.root, a.eps));
                    mb = max(mb, bits_abs(m[u][k]));
                    sb = max(sb, __float_as_uint(v[u][k]));
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float gk = g[u][k] * c.clip;
                    m[u][k] = fmaf(a.beta1, m[u][k], a.one_minus_beta1 * gk);
                    v[u][k] = fmaf(a.beta2, v[u][k], a.one_minus_beta2 * (gk * gk));
                    p[u][k] = fmaf(p[u][k], c.keep, p[u][k]) - m[u][k] * r.first / fmaf(sqrtf(v[u][k]), r.root, a.eps);
                }
            }
            store4<WHOLE>(p16, r.param, i, n, p[u]);
            if constexpr (EIGHT) {
                const float mt = __uint_as_float(wave_max_bits(mb)), st = sqrtf(__uint_as_float(wave_max_bits(sb) & 0x7fffffffu));
                store4_codes<WHOLE>(r.m, i, n, m_codes(m[u], mt, mt > kSmallest ? kM2 * __builtin_amdgcn_rcpf(mt) : 0.0f));
                store4_codes<WHOLE>(r.v, i, n, s_codes(s, v[u], st, st > kSmallest ? kS2 * __builtin_amdgcn_rcpf(st) : 0.0f));
                if (lane == 0) {
                    r.m_scale[i >> 8] = mt;
                    r.v_scale[i >> 8] = st;
                }
            } else {
                store4<WHOLE>(false, r.m, i, n, m[u]);
                store4<WHOLE>(false, r.v, i, n, v[u]);
            }
        }
    }
}

template <bool EIGHT>
__global__ void __launch_bounds__(kThreads) adamw_kernel(StepArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (from the last chunk to the first: what grad_norm_kernel, with the same ranges, read last is what caches still have)
    const int64_t c0 = a.chunks * blockIdx.x / gridDim.x;
    int64_t c = a.chunks * (blockIdx.x + 1) / gridDim.x - 1;
    if (c < c0) return;
    Call k;
    k.keep = -(a.lr_device ? *a.lr_device : a.lr) * a.weight_decay;
    // (written so that a NaN norm makes the gradients NaN)
    float clip = 1.0f;
    if (a.norm) {
        clip = 1.0f / (*a.norm + 1e-6f) * a.max_norm;
        clip = clip > 1.0f ? 1.0f : clip;
    }
    k.clip = clip;
    int t = row_of(a.rows, a.n, c, lane);
    Row r = a.rows[t];
    for (; c >= c0; --c) {
        while (r.chunk0 > c) r = a.rows[--t];
        const int64_t at = (c - r.chunk0) * kChunk;
        const bool whole = at + kChunk <= r.numel && whole4(r.param, r.param16) && whole4(r.grad, r.grad16) &&
                           (((uintptr_t)r.m | (uintptr_t)r.v) & (EIGHT ? 3 : 15)) == 0;
        const int64_t base = at + wave * kBlock;
        if (!whole) step_chunk<EIGHT, false, false, false>(a, r, base, lane, k);
        else if (r.param16) r.grad16 ? step_chunk<EIGHT, true, true, true>(a, r, base, lane, k) : step_chunk<EIGHT, true, true, false>(a, r, base, lane, k);
        else r.grad16 ? step_chunk<EIGHT, true, false, true>(a, r, base, lane, k) : step_chunk<EIGHT, true, false, false>(a, r, base, lane, k);
    }
}

// ---------------------------------------------------------------- the norm of all gradients
// Squares and sums in 64 bits, in an order fixed by the sizes alone: partial sums of the blocks, then one block over them.
__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) v += lds[w];
    return v;
}

__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const Row* rows, int n_rows, int64_t chunks, double* partial) {
    __shared__ double lds[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t c = chunks * blockIdx.x / gridDim.x;
    const int64_t c1 = chunks * (blockIdx.x + 1) / gridDim.x;
    double sum = 0.0;
    if (c < c1) {
        int t = row_of(rows, n_rows, c, lane);
        Row r = rows[t];
        for (; c < c1; ++c) {
            while (t + 1 < n_rows && rows[t + 1].chunk0 <= c) r = rows[++t];
            const int64_t base = (c - r.chunk0) * kChunk + wave * kBlock + lane * 4;
            f32x4 g[4];
            const bool whole = (c - r.chunk0 + 1) * kChunk <= r.numel && whole4(r.grad, r.grad16);
            if (whole && r.grad16) {
#pragma unroll
                for (int u = 0; u < 4; ++u) g[u] = load4<true, false>(true, r.grad, base + u * (kThreads * 4), r.numel);
            } else if (whole) {
#pragma unroll
                for (int u = 0; u < 4; ++u) g[u] = load4<true, false>(false, r.grad, base + u * (kThreads * 4), r.numel);
            } else {
#pragma unroll
                for (int u = 0; u < 4; ++u) g[u] = load4<false, false>(r.grad16, r.grad, base + u * (kThreads * 4), r.numel);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) sum += (double)g[u][k] * (double)g[u][k];
        }
    }
    sum = block_sum(sum, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kThreads) grad_norm_finish_kernel(const double* partial, int n, float* out) {
    __shared__ double lds[kThreads / 64];
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) sum += partial[i];
    sum = block_sum(sum, lds);
    if (threadIdx.x == 0) *out = (float)sqrt(sum);
}

// ---------------------------------------------------------------- what 8-bit states stand for
template <bool WHOLE>
__device__ __forceinline__ void values4(const uint8_t* mc, const uint8_t* vc, const float* ms, const float* vs, int64_t i, int64_t n, void* m_out, void* v_out,
                                        bool out16) {
    const uint32_t a = load4_codes<WHOLE>(mc, i, n), b = load4_codes<WHOLE>(vc, i, n);
    const float sm = ms[i >> 8] * (1.0f / kM2), sv = vs[i >> 8] * (1.0f / kS2);
    f32x4 m, v;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        m[k] = m_value(a, k, sm);
        const float s = s_value(b, k, sv);
        v[k] = s * s;
    }
    store4<WHOLE>(out16, m_out, i, n, m);
    store4<WHOLE>(out16, v_out, i, n, v);
}
template <bool OUT16>
__global__ void __launch_bounds__(kThreads) adamw_values_kernel(const uint8_t* mc, const uint8_t* vc, const float* ms, const float* vs, int64_t n, void* m_out,
                                                                void* v_out, bool vec) {
    const int64_t stride = (int64_t)gridDim.x * kThreads * 4;
    for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4; i < n; i += stride) {
        if (vec && i + 4 <= n) values4<true>(mc, vc, ms, vs, i, n, m_out, v_out, OUT16);
        else values4<false>(mc, vc, ms, vs, i, n, m_out, v_out, OUT16);
    }
}

int check_tensors(const char* who, const xq_adamw_tensor* t, int64_t n, int state_bits, bool grads_only, int64_t* chunks) {
    XQ_REQUIRE(n >= 0 && n < (1 << 24), "%s: bad number of tensors %lld", who, (long long)n);
    XQ_REQUIRE(n == 0 || t, "%s: tensors are NULL", who);
    *chunks = 0;
    for (int64_t i = 0; i < n; ++i) {
        const xq_adamw_tensor& a = t[i];
        uintptr_t bits = (uintptr_t)a.grad;
        if (!grads_only) {
            bits |= (uintptr_t)a.param | (uintptr_t)a.exp_avg | (uintptr_t)a.exp_avg_sq | (uintptr_t)a.step;
            if (state_bits == 8) bits |= (uintptr_t)a.exp_avg_scale | (uintptr_t)a.exp_avg_sq_scale;
        }
        XQ_REQUIRE(bits >> kAddressBits == 0, "%s: an address of tensor %lld has more than %d bits", who, (long long)i, kAddressBits);
        XQ_REQUIRE(a.numel > 0, "%s: tensor %lld has %lld elements", who, (long long)i, (long long)a.numel);
        XQ_REQUIRE(a.grad_dtype == XQ_DT_BF16 || a.grad_dtype == XQ_DT_F32, "%s: gradient %lld is neither fp32 nor bf16", who, (long long)i);
        XQ_REQUIRE(a.grad && xq_aligned(a.grad, a.grad_dtype == XQ_DT_BF16 ? 2 : 4), "%s: gradient %lld is NULL or misaligned", who, (long long)i);
        *chunks += xq_cdiv(a.numel, kChunk);
        XQ_REQUIRE(*chunks < (1ll << 31), "%s: more than %lld elements", who, (long long)kChunk << 31);
        if (grads_only) continue;
        XQ_REQUIRE(a.param_dtype == XQ_DT_BF16 || a.param_dtype == XQ_DT_F32, "%s: parameter %lld is neither fp32 nor bf16", who, (long long)i);
        XQ_REQUIRE(a.param && xq_aligned(a.param, a.param_dtype == XQ_DT_BF16 ? 2 : 4), "%s: parameter %lld is NULL or misaligned", who, (long long)i);
        XQ_REQUIRE(a.exp_avg && a.exp_avg_sq && a.step && xq_aligned(a.step, 4), "%s: a state of tensor %lld is NULL or misaligned", who, (long long)i);
        if (state_bits == 8)
            XQ_REQUIRE(a.exp_avg_scale && a.exp_avg_sq_scale && xq_aligned(a.exp_avg_scale, 4) && xq_aligned(a.exp_avg_sq_scale, 4),
                       "%s: 8-bit states of tensor %lld have no scales, or misaligned ones", who, (long long)i);
        else
            XQ_REQUIRE(xq_aligned(a.exp_avg, 4) && xq_aligned(a.exp_avg_sq, 4), "%s: a state of tensor %lld is misaligned", who, (long long)i);
    }
    return XQ_OK;
}

int64_t table_bytes(int64_t n) { return xq_cdiv(n * (int64_t)sizeof(Row), 256) * 256; }

int check_workspace(const char* who, int64_t n, const void* workspace, int64_t bytes) {
    XQ_REQUIRE(workspace && xq_aligned(workspace, 256) && bytes >= xq_adamw_workspace_bytes(n), "%s: a workspace of %lld bytes, 256-byte aligned, is needed", who,
               (long long)xq_adamw_workspace_bytes(n));
    return XQ_OK;
}

// words 3: for the norm alone
template <int WORDS>
void write_table(const xq_adamw_tensor* t, int64_t n, void* workspace, const xq_adamw_options* o, hipStream_t s) {
    TableScalars c = {};
    if (o) c = TableScalars{o->lr, std::log(o->beta1), std::log(o->beta2), o->lr_device};
    int64_t chunk0 = 0;
    for (int64_t at = 0; at < n; at += table_tensors(WORDS)) {
        TableArgs a;
        a.rows = (Row*)workspace + at;
        a.chunk0 = (int32_t)chunk0;
        a.n = (int32_t)std::min<int64_t>(table_tensors(WORDS), n - at);
        for (int i = 0; i < a.n; ++i) {
            const xq_adamw_tensor& q = t[at + i];
            uint32_t* w = a.word + i * WORDS;
            auto low = [](const void* p) { return (uint32_t)(uintptr_t)p; };
            auto high = [](const void* p) { return (uint32_t)((uintptr_t)p >> 32); };
            w[0] = (uint32_t)q.numel;
            w[1] = (uint32_t)(q.numel >> 32) | (uint32_t)(q.grad_dtype == XQ_DT_BF16) << 15 | high(q.grad) << 16;
            w[2] = low(q.grad);
            if (WORDS >= 9) {
                w[1] |= (uint32_t)(q.param_dtype == XQ_DT_BF16) << 14;
                w[3] = low(q.param); w[4] = low(q.exp_avg); w[5] = low(q.exp_avg_sq); w[6] = low(q.step);
                w[7] = high(q.param) | high(q.exp_avg) << 16; w[8] = high(q.exp_avg_sq) | high(q.step) << 16;
            }
            if (WORDS == 12) { w[9] = low(q.exp_avg_scale); w[10] = low(q.exp_avg_sq_scale); w[11] = high(q.exp_avg_scale) | high(q.exp_avg_sq_scale) << 16; }
            chunk0 += xq_cdiv(q.numel, kChunk);
        }
        adamw_table_kernel<WORDS><<<dim3(1), 256, 0, s>>>(a, c);
    }
}

void norm_of(int64_t n, int64_t chunks, void* workspace, float* norm, hipStream_t s) {
    double* partial = (double*)((uint8_t*)workspace + table_bytes(n));
    const int blocks = (int)std::min<int64_t>(chunks, kNormBlocks);
    if (blocks) grad_norm_kernel<<<dim3(blocks), kThreads, 0, s>>>((const Row*)workspace, (int)n, chunks, partial);
    grad_norm_finish_kernel<<<dim3(1), kThreads, 0, s>>>(partial, blocks, norm);
}

}  // namespace
}  // namespace xq

using namespace xq;

extern "C" int64_t xq_adamw_workspace_bytes(int64_t n_tensors) { return n_tensors < 0 ? -1 : table_bytes(n_tensors) + kNormBlocks * 8; }

extern "C" int xq_grad_norm(const xq_adamw_tensor* tensors, int64_t n, float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
    int64_t chunks;
    int rc = check_tensors("xq_grad_norm", tensors, n, 32, true, &chunks);
    if (rc == XQ_OK) rc = check_workspace("xq_grad_norm", n, workspace, workspace_bytes);
    if (rc != XQ_OK) return rc;
    XQ_REQUIRE(norm && xq_aligned(norm, 4), "xq_grad_norm: norm is NULL or misaligned");
    write_table<3>(tensors, n, workspace, nullptr, (hipStream_t)stream);
    norm_of(n, chunks, workspace, norm, (hipStream_t)stream);
    XQ_CHECK_LAUNCH("xq_grad_norm");
    return XQ_OK;
}

extern "C" int xq_adamw_step(const xq_adamw_tensor* tensors, int64_t n, const xq_adamw_options* o, void* workspace, int64_t workspace_bytes, void* stream) {
    XQ_REQUIRE(o, "xq_adamw_step: options are NULL");
    XQ_REQUIRE(o->state_bits == 8 || o->state_bits == 32, "xq_adamw_step: states of 8 or 32 bits, got %d", o->state_bits);
    XQ_REQUIRE(o->lr >= 0.0 && o->beta1 >= 0.0 && o->beta1 < 1.0 && o->beta2 >= 0.0 && o->beta2 < 1.0 && o->eps >= 0.0 && o->weight_decay >= 0.0,
               "xq_adamw_step: lr %g, betas %g and %g, eps %g, weight_decay %g", o->lr, o->beta1, o->beta2, o->eps, o->weight_decay);
    XQ_REQUIRE(!o->norm || (o->max_norm > 0.0 && xq_aligned(o->norm, 4)), "xq_adamw_step: a norm needs max_norm > 0 (got %g) and 4-byte alignment", o->max_norm);
    XQ_REQUIRE(!o->norm_given || o->norm, "xq_adamw_step: norm_given without a norm");
    XQ_REQUIRE(!o->lr_device || xq_aligned(o->lr_device, 4), "xq_adamw_step: lr_device is misaligned");
    int64_t chunks;
    int rc = check_tensors("xq_adamw_step", tensors, n, o->state_bits, false, &chunks);
    if (rc == XQ_OK) rc = check_workspace("xq_adamw_step", n, workspace, workspace_bytes);
    if (rc != XQ_OK) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (o->state_bits == 8) write_table<12>(tensors, n, workspace, o, s);
    else write_table<9>(tensors, n, workspace, o, s);
    if (o->norm && !o->norm_given) norm_of(n, chunks, workspace, o->norm, s);
    if (n) {
        const StepArgs a = {(const Row*)workspace, chunks, o->norm, (int32_t)n, (float)o->max_norm, (float)o->beta1, (float)o->beta2,
                            (float)(1.0 - o->beta1), (float)(1.0 - o->beta2), (float)o->eps, (float)o->lr, (float)o->weight_decay, o->lr_device};
        const dim3 grid((unsigned)std::min<int64_t>(chunks, kStepBlocks));
        if (o->state_bits == 8) adamw_kernel<true><<<grid, kThreads, 0, s>>>(a);
        else adamw_kernel<false><<<grid, kThreads, 0, s>>>(a);
    }
    XQ_CHECK_LAUNCH("xq_adamw_step");
    return XQ_OK;
}

extern "C" int xq_adamw_values(const void* exp_avg, const void* exp_avg_sq, const float* exp_avg_scale, const float* exp_avg_sq_scale, int64_t numel,
                               void* exp_avg_out, void* exp_avg_sq_out, int out_dtype, void* stream) {
    XQ_REQUIRE(numel >= 0, "xq_adamw_values: %lld elements", (long long)numel);
    XQ_REQUIRE(out_dtype == XQ_DT_BF16 || out_dtype == XQ_DT_F32, "xq_adamw_values: the outputs are fp32 or bf16");
    if (numel == 0) return XQ_OK;
    XQ_REQUIRE(exp_avg && exp_avg_sq && exp_avg_scale && exp_avg_sq_scale && exp_avg_out && exp_avg_sq_out, "xq_adamw_values: NULL buffer");
    const size_t e = out_dtype == XQ_DT_BF16 ? 2 : 4;
    XQ_REQUIRE(xq_aligned(exp_avg_scale, 4) && xq_aligned(exp_avg_sq_scale, 4) && xq_aligned(exp_avg_out, e) && xq_aligned(exp_avg_sq_out, e),
               "xq_adamw_values: misaligned buffer");
    const bool vec = xq_aligned(exp_avg, 4) && xq_aligned(exp_avg_sq, 4) && xq_aligned(exp_avg_out, 4 * e) && xq_aligned(exp_avg_sq_out, 4 * e);
    const dim3 grid((unsigned)std::min<int64_t>(xq_cdiv(numel, 4 * kThreads), kStepBlocks));
    const auto *m = (const uint8_t*)exp_avg, *v = (const uint8_t*)exp_avg_sq;
    if (e == 2) adamw_values_kernel<true><<<grid, kThreads, 0, (hipStream_t)stream>>>(m, v, exp_avg_scale, exp_avg_sq_scale, numel, exp_avg_out, exp_avg_sq_out, vec);
    else adamw_values_kernel<false><<<grid, kThreads, 0, (hipStream_t)stream>>>(m, v, exp_avg_scale, exp_avg_sq_scale, numel, exp_avg_out, exp_avg_sq_out, vec);
    XQ_CHECK_LAUNCH("xq_adamw_values");
    return XQ_OK;
}
