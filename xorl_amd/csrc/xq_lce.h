// Tile kernels of the cross entropy over an output head: products of bf16 matrices whose logits never reach memory.
//
// lce_logits_kernel   S = A . B^T, both with the contraction along their rows (hidden states and head), and one of three ends:
//   STATS   a row's largest logit and its sum of exponentials, by column tile (nothing else is written)
//   EXP     the same sums relative to a reference logit of the row, and E = exp(l - reference) as a bf16 image
//   GRAD    A the head, B the tokens: G = g_i (p_iv - [v = t_i]) as a bf16 image with the tokens along the contraction
// lce_product_kernel  C = image . B, B with the contraction across its rows: E . W (input gradients), G . X (the head's)
//
//  * Tiles of 32 TM x 256, K-steps of 32, four LDS stages filled by direct-to-LDS loads, eight waves of 16 TM x 64 on
//    v_mfma_f32_16x16x32_bf16.  In iteration kt every wave reads stages kt and kt + 1 and fills stage kt + 3; the loads of kt + 2 are waited
//    for at its end.  A K-step is TM chunks of four MFMAs; a chunk's fragment of A is read three chunks ahead, the fragments of B a
//    K-step ahead (two register sets).  Loads behind the last K-step repeat it, so that every iteration is the same.
//  * Stage.  A: [row][32 k], the 16-byte chunk c of a row at c ^ ((row >> 2) & 2): 16 rows x 4 chunks meet no bank twice.  B of
//    the logits the same.  B of the product: [32 k][256 columns], the 32-byte unit u of row k at u ^ (k & 7); fragments come out by
//    the transposing read, which takes 4 rows x 16 columns for 16 lanes: eight rows of a half wave lie in eight bank groups.
//  * Image.  [tile of 32 TM rows][K-step][row][32 k], as the stage of A wants it: loads are copies.  Slot 8 g + e of a K-step is its column
//    4 g + e (e < 4) or 16 + 4 g + e - 4: what lane group g of the logits kernel holds of two neighbouring fragments, stored as 16 bytes;
//    the product's transposing reads pick the rows of B to match.
#pragma once

#include "xq_common.h"

namespace xq {

enum { kLceStats = 0, kLceExp = 1, kLceGrad = 2 };

template <int TM>
struct LceTile {
    static constexpr int ROWS = 32 * TM, COLS = 256, BK = 32, STAGES = 4;
    static constexpr int A_BYTES = ROWS * 64, B_BYTES = COLS * 64, STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int AP = (ROWS / 8 + 15) / 16, BP = 2, NP = AP + BP;        // direct loads of a wave and K-step: 16 rows of 64 bytes each
    static constexpr int LDS_BYTES = STAGES * STAGE_BYTES;
};

struct LceRows {                        // what is kept of the labels: the rows that count, in order
    const int32_t* count;
    const int32_t* row;                 // of x
    const int32_t* label;               // -1: out of range
};

struct LceLogitsArgs {
    const bf16_t* A;
    const bf16_t* B;
    int64_t lda, ldb;
    int32_t H, first_v, n_v;            // the piece of the vocabulary: its first row of the head and how many
    LceRows rows;
    float scale2;                       // of the logits, times log2(e)
    const float* ref;                   // EXP: reference of a row, in log2 units;  GRAD: log2 of the row's sum of exponentials
    const float* grad;                  // GRAD: upstream gradient of a row times the logit scale
    const float* rest;                  // GRAD: 1 - p of the label
    f32x2* part;                        // STATS, EXP: [column tile][rows_pad] (largest, sum)
    float* at_label;                    // STATS: the label's logit
    int64_t rows_pad;
    bf16_t* image;
    int32_t image_steps;                // K-steps of the image's rows
    const int32_t* redo;                // EXP: row tiles to do again, or NULL
};

// C[r, n] over the tile's K-steps; issue(kt, part, dst): one of NP direct loads of K-step kt
template <int TM, bool BT, typename Issue>
__device__ __forceinline__ void lce_core(f32x4 (&acc)[TM][4], unsigned char* dsm, int nk, int wave, int lane, Issue issue) {
    using T = LceTile<TM>;
    constexpr int NC = TM, LA = NC < 3 ? NC : 3, FB = NC < 4 ? 4 / NC : 1;
    const int wm = wave >> 2, wn = wave & 3, l16 = lane & 15, lg = lane >> 4;
    const int sw = (l16 >> 2) & 2;
    const int a_at = (wm * 16 * TM + l16) * 64 + ((lg ^ sw) << 4);
    int b_at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (BT) {
            const int k = 4 * lg + (l16 >> 2);
            b_at[j] = T::A_BYTES + k * 512 + (((wn * 4 + j) ^ (k & 7)) << 5) + (l16 & 3) * 8;
        } else {
            b_at[j] = T::A_BYTES + (wn * 64 + j * 16 + l16) * 64 + ((lg ^ sw) << 4);
        }
    }
    auto read_a = [&](const unsigned char* stage, int c) -> bf16x8 { return *(const bf16x8*)(stage + a_at + c * 1024); };
    auto read_b = [&](const unsigned char* stage, int j) -> bf16x8 {
        if constexpr (BT) {
            typedef __attribute__((ext_vector_type(4))) short s16x4;
            typedef __attribute__((ext_vector_type(8))) short s16x8;
            const unsigned char* at = stage + b_at[j];
            s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(at));
            s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(at + 8192));
            return __builtin_bit_cast(bf16x8, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
        } else {
            return *(const bf16x8*)(stage + b_at[j]);
        }
    };
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (nk <= 0) return;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)dsm;
#pragma unroll
    for (int kt = 0; kt < 3; ++kt)
#pragma unroll
        for (int part = 0; part < T::NP; ++part) issue(min(kt, nk - 1), part, lds0 + kt * T::STAGE_BYTES);
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(T::NP) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    bf16x8 fa[4], fb[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) fb[0][j] = read_b(dsm, j);
#pragma unroll
    for (int c = 0; c < LA; ++c) fa[c] = read_a(dsm, c);
    auto iteration = [&](int kt, auto P_) {
        constexpr int P = decltype(P_)::value;
        const unsigned char* here = dsm + (kt & 3) * T::STAGE_BYTES;
        const unsigned char* next = dsm + ((kt + 1) & 3) * T::STAGE_BYTES;
        const uint32_t fill = lds0 + ((kt + 3) & 3) * T::STAGE_BYTES;
        const int kf = min(kt + 3, nk - 1);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int at = (P * NC + c) & 3;
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[P][j], fa[at], acc[c][j], 0, 0, 0);
            fa[(at + LA) & 3] = c + LA < NC ? read_a(here, c + LA) : read_a(next, c + LA - NC);
#pragma unroll
            for (int q = 0; q < FB; ++q)
                if (c * FB + q < 4) fb[P ^ 1][c * FB + q] = read_b(next, c * FB + q);
#pragma unroll
            for (int part = c * T::NP / NC; part < (c + 1) * T::NP / NC; ++part) issue(kf, part, fill);
            __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("s_waitcnt vmcnt(%0)" :: "n"(T::NP) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    int kt = 0;
    for (; kt + 1 < nk; kt += 2) {
        iteration(kt, std::integral_constant<int, 0>{});
        iteration(kt + 1, std::integral_constant<int, 1>{});
    }
    if (kt < nk) iteration(kt, std::integral_constant<int, 0>{});
    // nothing is on its way into LDS, and nobody reads it, from here on
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ void lce_load_lds(uint32_t dst, const void* src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(dst), "v"(src) : "memory");
}

// blocks to tiles: neighbours in time on one XCD share rows of A and B; blocks behind the last tile have none
__device__ __forceinline__ bool lce_tile(int tiles_a, int tiles_b, int* ta, int* tb) {
    const int nb = tiles_a * tiles_b, b = blockIdx.x, per = nb >> 3;
    if (b >= nb) return false;
    const int logical = b < per * 8 ? (b & 7) * per + (b >> 3) : b;
    constexpr int GM = 4;
    const int width = GM * tiles_b, grp = logical / width, first = grp * GM, gsz = min(tiles_a - first, GM), in = logical - grp * width;
    *ta = first + in % gsz;
    *tb = in / gsz;
    return true;
}

template <int TM, int MODE>
__global__ void __launch_bounds__(512, TM <= 2 ? 4 : 2) lce_logits_kernel(LceLogitsArgs g) {
    using T = LceTile<TM>;
    extern __shared__ __attribute__((aligned(16))) unsigned char dsm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3, l16 = lane & 15, lg = lane >> 4;
    const int count = *g.rows.count;
    const int n_a = MODE == kLceGrad ? g.n_v : count, n_b = MODE == kLceGrad ? count : g.n_v;
    int ta, tb;
    if (!lce_tile((n_a + T::ROWS - 1) / T::ROWS, (n_b + 255) >> 8, &ta, &tb)) return;
    if (MODE == kLceExp && g.redo && !g.redo[ta]) return;
    const int r0 = ta * T::ROWS, c0 = tb * 256;

    // ---- sources of the direct loads: a wave brings in an eighth of either side's rows, 64 bytes of each, 16 rows to a load
    const bf16_t* src[T::NP];
#pragma unroll
    for (int p = 0; p < T::NP; ++p) {
        const bool of_a = p < T::AP;
        const int rt = of_a ? wave * (T::ROWS / 8) + p * 16 + (lane >> 2) : wave * 32 + (p - T::AP) * 16 + (lane >> 2);
        const int n = min(of_a ? r0 + rt : c0 + rt, (of_a ? n_a : n_b) - 1);
        const bool tokens = of_a != (MODE == kLceGrad);
        const int64_t row = tokens ? g.rows.row[n] : g.first_v + n;
        src[p] = (of_a ? g.A + row * g.lda : g.B + row * g.ldb) + (((lane & 3) ^ ((rt >> 2) & 2)) << 3);
    }
    f32x4 acc[TM][4];
    lce_core<TM, false>(acc, dsm, g.H / T::BK, wave, lane, [&](int kt, int part, uint32_t stage) {
        const bool of_a = part < T::AP;
        const int p = of_a ? part : part - T::AP, rows = of_a ? T::ROWS / 8 : 32;
        const uint32_t dst = stage + (of_a ? 0 : T::A_BYTES) + wave * rows * 64 + p * 1024;
        if (p * 16 + 16 <= rows || lane < (rows - p * 16) * 4) lce_load_lds(dst, src[part] + kt * T::BK);
    });

    // ---- lane (l16, lg) holds rows r0 + wm 16 TM + 16 i + l16, columns c0 + 64 wn + 16 j + 4 lg + 0..3
    const int row_w = wm * 16 * TM + l16, col_w = wn * 64 + 4 * lg;
    if constexpr (MODE == kLceGrad) {
        f32x4 lse[4], up[4], rest[4];
        int label[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {               // (the arrays are as long as whole tiles: behind the last row up = 0, lse = inf)
            const int c = c0 + col_w + 16 * j;
            lse[j] = *(const f32x4*)(g.ref + c);
            up[j] = *(const f32x4*)(g.grad + c);
            rest[j] = *(const f32x4*)(g.rest + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) label[j][e] = g.rows.label[c + e];
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int v = g.first_v + r0 + row_w + 16 * i;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], g.scale2, -lse[j][e]));
                    acc[i][j][e] = up[j][e] * (label[j][e] == v ? -rest[j][e] : p);
                }
        }
    } else {
        // columns that the piece does not have, and the label's, count as -inf
        const bool tail = c0 + 256 > g.n_v;
        float ref[TM];
        int at[TM];                                     // the label's column in the tile, by the lane's own numbering of its 16
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int r = min(r0 + row_w + 16 * i, count - 1);
            at[i] = g.rows.label[r] - g.first_v - c0 - col_w;
            if (MODE == kLceExp) ref[i] = g.ref[r];
        }
        f32x2* lds = (f32x2*)dsm;                       // [row][wave column]
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] *= g.scale2;
            if (__any(at[i] >= 0 && at[i] < 52)) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at[i] == 16 * j + e) {
                            if (MODE == kLceStats && r0 + row_w + 16 * i < count) g.at_label[r0 + row_w + 16 * i] = acc[i][j][e];
                            acc[i][j][e] = -INFINITY;
                        }
            }
            if (tail) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c0 + col_w + 16 * j + e >= g.n_v) acc[i][j][e] = -INFINITY;
            }
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, acc[i][j][e]);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float base = MODE == kLceExp ? ref[i] : (top == -INFINITY ? 0.0f : top);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = __builtin_amdgcn_exp2f(acc[i][j][e] - base);
                    if (MODE == kLceExp) acc[i][j][e] = x;
                    sum += x;
                }
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (lg == 0) lds[(row_w + 16 * i) * 4 + wn] = f32x2{top, sum};
        }
        __syncthreads();
        if (tid < T::ROWS && r0 + tid < count) {
            f32x2 a = lds[tid * 4], b;
#pragma unroll
            for (int w = 1; w < 4; ++w) {
                b = lds[tid * 4 + w];
                const float top = fmaxf(a[0], b[0]);
                if (MODE == kLceExp) a[1] += b[1];
                else if (top != -INFINITY) a[1] = a[1] * __builtin_amdgcn_exp2f(a[0] - top) + b[1] * __builtin_amdgcn_exp2f(b[0] - top);
                a[0] = top;
            }
            g.part[(int64_t)tb * g.rows_pad + r0 + tid] = a;
        }
    }
    if constexpr (MODE != kLceStats) {
        bf16_t* out = g.image + ((int64_t)ta * g.image_steps + (c0 >> 5) + wn * 2) * (T::ROWS * 32);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int row = row_w + 16 * i;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const f32x4 a = acc[i][2 * q], b = acc[i][2 * q + 1];
                *(u32x4*)(out + (q * T::ROWS + row) * 32 + ((lg ^ ((row >> 2) & 2)) << 3)) =
                    u32x4{pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3])};
            }
        }
    }
}

struct LceProductArgs {
    const bf16_t* image;
    int32_t image_steps;                // K-steps of the image's rows
    int32_t rows, k;                    // rows of the result and contraction; < 0: as many as count
    const int32_t* count;
    const bf16_t* B;                    // [k, H]
    int64_t ldb;
    int32_t H, splits;
    float* out;                         // [split][rows_pad][H]: sums, added to what is there where `add`, that times alpha[row]
    int64_t split_stride;
    const float* alpha;
    int32_t add;
    bf16_t* out16;                      // or [rows, ld16] bf16
    int64_t ld16;
};

template <int TM>
__global__ void __launch_bounds__(512, TM <= 2 ? 4 : 2) lce_product_kernel(LceProductArgs g) {
    using T = LceTile<TM>;
    extern __shared__ __attribute__((aligned(16))) unsigned char dsm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3, l16 = lane & 15, lg = lane >> 4;
    const int rows = g.rows < 0 ? *g.count : g.rows, k = g.k < 0 ? *g.count : g.k;
    int ta, tb;
    if (!lce_tile((rows + T::ROWS - 1) / T::ROWS, (g.H + 255) >> 8, &ta, &tb)) return;
    const int r0 = ta * T::ROWS, c0 = tb * 256, s = blockIdx.y;
    const int steps = (k + 31) >> 5, kt0 = (int)((int64_t)steps * s / g.splits), nk = (int)((int64_t)steps * (s + 1) / g.splits) - kt0;

    const bf16_t* const a_src = g.image + ((int64_t)ta * g.image_steps + kt0) * (T::ROWS * 32) + wave * (T::ROWS / 8) * 32 + lane * 8;
    const int kr = wave * 4 + (lane >> 5);             // of a K-step's rows, two more with the second load
    const bf16_t* b_col[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int unit = ((lane & 31) >> 1) ^ ((kr + 2 * p) & 7);
        b_col[p] = g.B + min(c0 + unit * 16 + (lane & 1) * 8, g.H - 8);
    }
    f32x4 acc[TM][4];
    lce_core<TM, true>(acc, dsm, nk, wave, lane, [&](int kt, int part, uint32_t stage) {
        if (part < T::AP) {
            constexpr int rows8 = T::ROWS / 8;
            if (part * 16 + 16 <= rows8 || lane < (rows8 - part * 16) * 4)
                lce_load_lds(stage + wave * rows8 * 64 + part * 1024, a_src + (int64_t)kt * (T::ROWS * 32) + part * 512);
        } else {
            const int p = part - T::AP;
            const int row = min((kt0 + kt) * 32 + kr + 2 * p, k - 1);
            lce_load_lds(stage + T::A_BYTES + wave * 2048 + p * 1024, b_col[p] + row * g.ldb);
        }
    });

    const int row_w = wm * 16 * TM + l16, col_w = c0 + wn * 64 + 4 * lg;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int row = r0 + row_w + 16 * i;
        if (row >= rows) continue;
        const float alpha = g.add ? g.alpha[row] : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = col_w + 16 * j;
            if (col >= g.H) continue;
            if (g.out16) {
                *(u32x2*)(g.out16 + row * g.ld16 + col) = u32x2{pack_bf16x2(acc[i][j][0], acc[i][j][1]), pack_bf16x2(acc[i][j][2], acc[i][j][3])};
            } else {
                f32x4* o = (f32x4*)(g.out + s * g.split_stride + (int64_t)row * g.H + col);
                *o = g.add ? *o * alpha + acc[i][j] : acc[i][j];
            }
        }
    }
}

}  // namespace xq
