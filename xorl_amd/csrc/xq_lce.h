// Tile kernels of the cross entropy over an output head: products of bf16 matrices whose logits never reach memory.
//
// lce_logits_kernel   S = A . B^T, both with the contraction along their rows (hidden states and head), and one of three ends:
//   STATS   a row's largest logit and its sum of exponentials, by column tile (nothing else is written)
//   EXP     the same sums relative to a reference logit of the row, E = exp(l - reference) as a bf16 image, and the sum of what the image holds
//   GRAD    A the head, B the tokens: G = g_i (p_iv - [v = t_i]) as a bf16 image with the tokens along the contraction
// lce_product_kernel  C = image . B, B with the contraction across its rows: E . W (input gradients), G . X (the head's)
//
//  * Tiles of 32 TM x 64 TN, K-steps of 32, LDS stages (four or eight) filled by direct-to-LDS loads, eight waves of 16 TM x 16 TN on
//    v_mfma_f32_16x16x32_bf16.  In iteration kt every wave reads stages kt and kt + 1 and fills stage kt + 3 (or kt + 7); the loads of
//    kt + 2 are waited for at its end.  A K-step is TM chunks of TN MFMAs; a chunk's fragment of A is read three chunks ahead, the fragments of B a
//    K-step ahead (two register sets).  Every iteration is the same: behind a tile's last K-step the logits kernel loads the next tile's, the product
//    the last one again (a branch around the loads cost both 5 %).
//  * What bounds it.  Many rows: the matrix units, two thirds (logits) to three quarters (product) busy, and the power they draw: 1.36 PFLOP/s of
//    STATS at 8192 rows under [131072, 4096], 1.25 of EXP (its 1 GiB pieces of E are 5 % of it, the sum of what they hold 1.5 %, the other ends 3 %, reading 64-byte pieces of
//    rows and not whole lines 5 %), 1.36 of E . W; a library product of the same operands 1.41.  Up to 128 rows: reading the head, 1 GiB of it in 180 us
//    (6.0 TB/s) under one row, 174 us for E . W.
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

template <int TM, int TN = 4, int ST = 4>
struct LceTile {
    static constexpr int ROWS = 32 * TM, COLS = 64 * TN, BK = 32, STAGES = ST;
    static constexpr int A_BYTES = ROWS * 64, B_BYTES = COLS * 64, STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int AP = (ROWS / 8 + 15) / 16, BP = COLS / 128, NP = AP + BP;       // direct loads of a wave and K-step: 16 rows of 64 bytes each
    // a block goes on to its next tile, whose first K-steps are on their way while the ends of this one are computed; 64 rows: two blocks
    // of one tile each share a compute unit instead
    static constexpr bool AHEAD = TM >= 4;
    static constexpr int END_BYTES = ROWS * 64 + 1024 * 4;      // of the ends: up to four numbers by row and wave; four by row or column
    static constexpr int LDS_BYTES = STAGES * STAGE_BYTES + (AHEAD ? END_BYTES : 0);
    static_assert(AHEAD || END_BYTES <= STAGES * STAGE_BYTES, "the ends reuse the stages");
    static_assert((STAGES & (STAGES - 1)) == 0 && LDS_BYTES <= 160 * 1024, "stages are counted by a mask, and fit");
};

struct LceRows {                        // what is kept of the labels: the rows that count, in order
    const int32_t* count;
    const int32_t* row;                 // of x
    const int32_t* label;               // -1: out of range
};

// Up to kLceOwnRows labels: every wave of a STATS launch finds the rows that count by itself, a lane each
constexpr int kLceOwnRows = 64;
struct LceLabels {
    const void* label;                  // NULL: LceRows has them
    int32_t bytes, M;
    int64_t ignore, V;
};
__device__ __forceinline__ int64_t lce_label(const void* labels, int bytes, int64_t i) {
    return bytes == 8 ? ((const int64_t*)labels)[i] : (int64_t)((const int32_t*)labels)[i];
}

struct LceLogitsArgs {
    const bf16_t* A;
    const bf16_t* B;
    int64_t lda, ldb;
    int32_t H, first_v, n_v;            // the piece of the vocabulary: its first row of the head and how many
    int32_t cols;                       // of a tile, up to 256 (GRAD, and above 128 rows: 256)
    LceRows rows;
    LceLabels labels;                   // STATS
    float scale2;                       // of the logits, times log2(e)
    const float* ref;                   // EXP: reference of a row, in log2 units;  GRAD: log2 of the row's sum of exponentials
    const float* grad;                  // GRAD: upstream gradient of a row, but for what all rows share
    const float* rest;                  // GRAD: 1 - p of the label
    f32x2* part;                        // [column tile][rows_pad], STATS: a row's (largest, sum);  EXP: (sum of E as the image holds it, sum)
    float* top;                         // EXP: [column tile][rows_pad] the largest
    float* at_label;                    // STATS: the label's logit
    int64_t rows_pad;
    bf16_t* image;
    int32_t image_steps;                // K-steps of the image's rows
    int32_t* redo;                      // EXP: row tiles that found a logit too far above its reference
    int32_t again;                      // do those again, and those only, with the row's largest logit as its reference
    float* new_ref;                     // of the rows done again, and what their sums so far count by
    float* alpha;
};
constexpr float kLceFar = 64.0f;        // log2

// G of few tokens is kept as two bf16 numbers, the value and what its rounding left, in two runs of columns (K-steps of the product) of this length
// each: a row of the head's gradient is often one token's, whose rounded G would be a second error of half a step beside the result's own.  With
// many tokens the errors of G are as many and no larger, and the product would be twice the work; for 128 it is still level with writing the
// gradient (512 FLOP an element against 2 bytes).
constexpr int kLceSplit = 128;
__device__ __forceinline__ int lce_half(int count) { return count <= kLceSplit ? (count + 31) & ~31 : 1 << 30; }

// The first of a stream of K-steps, all stages but one: K-step k of it goes to stage k % STAGES.  issue(at, part, stage): one of NP direct loads of a K-step.
template <typename T, typename Advance, typename Issue>
__device__ __forceinline__ void lce_begin(unsigned char* dsm, Advance advance, Issue issue) {
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)dsm;
#pragma unroll
    for (int kt = 0; kt < T::STAGES - 1; ++kt) {
        const int at = advance(kt);
#pragma unroll
        for (int part = 0; part < T::NP; ++part) issue(at, part, lds0 + kt * T::STAGE_BYTES);
    }
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(T::NP * (T::STAGES - 3)) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// C[r, n] over the stream's K-steps first .. first + nk - 1 (an even number, not 0), the first two of which have landed; the same holds of the
// two behind them in the end.  advance(k): what issue is to be told for the tile's K-step k, which goes on behind the last.
template <int TM, int TN, int ST, bool BT, typename Advance, typename Issue>
__device__ __forceinline__ void lce_run(f32x4 (&acc)[TM][TN], unsigned char* dsm, int first, int nk, int wave, int lane, Advance advance, Issue issue) {
    using T = LceTile<TM, TN, ST>;
    constexpr int NC = TM, LA = NC < 3 ? NC : 3, FB = (TN + NC - 1) / NC, D = ST - 1;
    static_assert(!BT || TN == 4, "the transposed stage is 256 columns wide");
    const int wm = wave >> 2, wn = wave & 3, l16 = lane & 15, lg = lane >> 4;
    const int sw = (l16 >> 2) & 2;
    const int a_at = (wm * 16 * TM + l16) * 64 + ((lg ^ sw) << 4);
    int b_at[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        if constexpr (BT) {
            const int k = 4 * lg + (l16 >> 2);
            b_at[j] = T::A_BYTES + k * 512 + (((wn * 4 + j) ^ (k & 7)) << 5) + (l16 & 3) * 8;
        } else {
            b_at[j] = T::A_BYTES + (wn * 16 * TN + j * 16 + l16) * 64 + ((lg ^ sw) << 4);
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
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)dsm;
    bf16x8 fa[4], fb[2][TN];
    {
        const unsigned char* stage = dsm + (first & D) * T::STAGE_BYTES;
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[0][j] = read_b(stage, j);
#pragma unroll
        for (int c = 0; c < LA; ++c) fa[c] = read_a(stage, c);
    }
    auto iteration = [&](int kt, auto P_) {
        constexpr int P = decltype(P_)::value;
        const unsigned char* here = dsm + ((first + kt) & D) * T::STAGE_BYTES;
        const unsigned char* next = dsm + ((first + kt + 1) & D) * T::STAGE_BYTES;
        const uint32_t fill = lds0 + ((first + kt + D) & D) * T::STAGE_BYTES;
        const int ahead = advance(kt + D);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int at = (P * NC + c) & 3;
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[P][j], fa[at], acc[c][j], 0, 0, 0);
            fa[(at + LA) & 3] = c + LA < NC ? read_a(here, c + LA) : read_a(next, c + LA - NC);
#pragma unroll
            for (int q = 0; q < FB; ++q)
                if (c * FB + q < TN) fb[P ^ 1][c * FB + q] = read_b(next, c * FB + q);
#pragma unroll
            for (int part = c * T::NP / NC; part < (c + 1) * T::NP / NC; ++part) issue(ahead, part, fill);
            __builtin_amdgcn_sched_barrier(0);
        }
        // K-step kt + 2 has landed
        asm volatile("s_waitcnt vmcnt(%0)" :: "n"(T::NP * (ST - 3)) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    // (one loop and one exit: with several the sums met with no register to spare)
    for (int kt = 0; kt < nk; kt += 2) {
        iteration(kt, std::integral_constant<int, 0>{});
        iteration(kt + 1, std::integral_constant<int, 1>{});
    }
}
// before LDS is used for something else, or given back
__device__ __forceinline__ void lce_loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ void lce_load_lds(uint32_t dst, const void* src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(__builtin_amdgcn_readfirstlane(dst)), "v"(src) : "memory");
}

// What a block works on.  XCD x (blocks are dealt to the eight of them in turn) has an eighth of the tiles, in order; its blocks take them one
// after the other, so that what it works on at a time shares rows of A (4 tiles) and of B (8).
struct LceWalk {
    int at, end, step;
    __device__ LceWalk(int tiles) {
        const int x = blockIdx.x & 7, slots = gridDim.x >> 3;
        if (gridDim.x & 7) {                    // (fewer than eight, or an odd number: in turn)
            at = blockIdx.x; end = tiles; step = gridDim.x;
        } else {
            const int first = (int)((int64_t)tiles * x >> 3);
            at = first + (int)(blockIdx.x >> 3); end = (int)((int64_t)tiles * (x + 1) >> 3); step = slots;
        }
    }
    __device__ bool more() const { return at < end; }
};
__device__ __forceinline__ void lce_tile(int logical, int tiles_a, int tiles_b, int* ta, int* tb) {
    constexpr int GM = 4;
    const int width = GM * tiles_b, grp = logical / width, first = grp * GM, gsz = min(tiles_a - first, GM), in = logical - grp * width;
    *ta = first + in % gsz;
    *tb = in / gsz;
}

// (as fmaxf twice it is four instructions: the compiler makes its arguments quiet first)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float over_groups_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float over_groups_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

template <int TM, int TN, int ST, int MODE>
__global__ void __launch_bounds__(512, TM <= 2 ? 4 : 2) lce_logits_kernel(LceLogitsArgs g) {
    using T = LceTile<TM, TN, ST>;
    static_assert(MODE != kLceGrad || TN == 4, "what the ends keep of 256 columns");
    extern __shared__ __attribute__((aligned(16))) unsigned char dsm[];
    unsigned char* const ends = T::AHEAD ? dsm + T::STAGES * T::STAGE_BYTES : dsm;
    f32x4* const sums = (f32x4*)ends;                       // [row][wave column], STATS: largest, sum;  EXP: sum of the image's E, sum, largest
    float* const info = (float*)(ends + T::ROWS * 64);      // EXP, STATS: label and reference by row;  GRAD: label, lse, up, rest by column
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3, l16 = lane & 15, lg = lane >> 4;
    constexpr bool OWN = MODE == kLceStats && 32 * TM <= kLceOwnRows;
    int count, own_row = 0, own_label = -1;                 // (a lane's of the rows that count)
    if (OWN && g.labels.label) {
        const int64_t label = lane < g.labels.M ? lce_label(g.labels.label, g.labels.bytes, lane) : g.labels.ignore;
        const uint64_t in = __ballot(label != g.labels.ignore), below = (1ull << lane) - 1;
        count = __builtin_popcountll(in);
        const int to = 4 * (in >> lane & 1 ? __builtin_popcountll(in & below) : count + __builtin_popcountll(~in & below));
        own_row = __builtin_amdgcn_ds_permute(to, lane);
        own_label = __builtin_amdgcn_ds_permute(to, label >= 0 && label < g.labels.V ? (int)label : -1);
    } else {
        count = __builtin_amdgcn_readfirstlane(*g.rows.count);
    }
    const int n_a = MODE == kLceGrad ? g.n_v : count, n_b = MODE == kLceGrad ? count : g.n_v;
    const int tiles_a = (n_a + T::ROWS - 1) / T::ROWS, cols = MODE == kLceGrad || TM > 4 ? 256 : min(g.cols, T::COLS), tiles_b = (n_b + cols - 1) / cols, nk = g.H / T::BK;

    const int half = MODE == kLceGrad ? lce_half(count) : 0;
    // a column of the tile to a token of it
    auto token = [&](int c) -> int { return c >= half ? c - half : c; };

    LceWalk walk(tiles_a * tiles_b);
    int ta, tb;
    auto find = [&]() -> bool {                             // the block's next tile
        for (; walk.more(); walk.at += walk.step) {
            lce_tile(walk.at, tiles_a, tiles_b, &ta, &tb);
            if (MODE != kLceExp || !g.again || __builtin_amdgcn_readfirstlane(g.redo[ta])) return true;
        }
        return false;
    };
    // ---- sources of the direct loads: a wave brings in an eighth of either side's rows, 64 bytes of each, 16 rows to a load; and what
    // the ends want to know of the rows (EXP, STATS) or columns (GRAD) that are tokens
    constexpr int N_INFO = MODE == kLceGrad ? 256 : T::ROWS;
    auto own_label_of = [&](int r) -> int { return __shfl(own_label, r); };         // (N_INFO threads: whole waves)
    auto sources = [&](const bf16_t* (&src)[T::NP], float (&about)[4]) {
#pragma unroll
        for (int p = 0; p < T::NP; ++p) {
            const bool of_a = p < T::AP;
            const int rt = of_a ? wave * (T::ROWS / 8) + p * 16 + (lane >> 2) : wave * (T::COLS / 8) + (p - T::AP) * 16 + (lane >> 2);
            // (rows behind the last, of either side or of the tile's columns: that one again, for nothing)
            const int n = of_a ? min(ta * T::ROWS + rt, n_a - 1) : min(tb * cols + (MODE == kLceGrad ? token(rt) : min(rt, cols - 1)), n_b - 1);
            const bool tokens = of_a != (MODE == kLceGrad);
            const int64_t row = !tokens ? g.first_v + n : OWN && g.labels.label ? __shfl(own_row, n) : g.rows.row[n];
            src[p] = (of_a ? g.A + row * g.lda : g.B + row * g.ldb) + (((lane & 3) ^ ((rt >> 2) & 2)) << 3);
        }
        if (tid < N_INFO) {
            // (GRAD: the arrays are as long as whole tiles; behind the last row up = 0, lse = inf)
            const int r = MODE == kLceGrad ? tb * 256 + token(tid) : min(ta * T::ROWS + tid, count - 1);
            about[0] = __int_as_float((OWN && g.labels.label ? own_label_of(r) : g.rows.label[r]) - g.first_v);
            if (MODE != kLceStats) about[1] = g.ref[r];
            if (MODE == kLceGrad) { about[2] = g.grad[r]; about[3] = g.rest[r]; }
            if (MODE == kLceExp && g.again) {
                // done again: the largest logit of the row's tiles is its reference, where that is far from the one it had
                float top = -INFINITY;
                for (int t = 0; t < tiles_b; ++t) top = fmaxf(top, g.top[(int64_t)t * g.rows_pad + r]);
                const float old = about[1];
                const bool far = top - old > kLceFar;
                if (far) about[1] = top;
                if (tb == 0 && ta * T::ROWS + tid < count) {
                    g.new_ref[r] = about[1];
                    g.alpha[r] = far ? __builtin_amdgcn_exp2f(old - top) : 1.0f;
                }
            }
        }
    };
    auto note = [&](const float (&about)[4]) {
        if (tid < N_INFO) {
            info[tid] = about[0];
            if (MODE != kLceStats) info[N_INFO + tid] = about[1];
            if (MODE == kLceGrad) { info[512 + tid] = about[2]; info[768 + tid] = about[3]; }
        }
    };
    const bf16_t* src[T::NP];
    const bf16_t* src_next[T::NP];
    auto issue = [&](int at, int part, uint32_t stage) {
        const bool of_a = part < T::AP;
        const int p = of_a ? part : part - T::AP, rows = (of_a ? T::ROWS : T::COLS) / 8;
        const uint32_t dst = stage + (of_a ? 0 : T::A_BYTES) + wave * rows * 64 + p * 1024;
        if (p * 16 + 16 <= rows || lane < (rows - p * 16) * 4) lce_load_lds(dst, src[part] + at * T::BK);
    };
    float about[4];
    bool more = false;
    // Few rows: the head is all that is read, by all blocks at the same pace.  Starting each column tile at another K-step (and going round)
    // spreads what they read at a time over the memory channels: rows of the head are often a power of two apart (65536 x 4096 under one row:
    // 138 us in step, 110 so).
    auto turn = [&](int tile) -> int { return TM <= 4 ? (int)((uint32_t)tile * 37u % (uint32_t)nk) : 0; };
    int turned = 0, turned_next = 0;
    // (behind the tile's last K-step: the next tile's; without one, this one's again, for nothing)
    auto advance = [&](int kt) -> int {
        if (kt == nk && more) {
#pragma unroll
            for (int p = 0; p < T::NP; ++p) src[p] = src_next[p];
            turned = turned_next;
        }
        const int k = (kt < nk ? kt : kt - nk < nk ? kt - nk : 0) + turned;
        return k < nk ? k : k - nk;
    };
    if (!find()) return;
    const bool stream = T::AHEAD && nk >= ST;               // (fewer: a tile's end is nearer than the loads are ahead)
    sources(src, about);
    turned = turn(tb);
    lce_begin<T>(dsm, advance, issue);
    if (T::AHEAD) note(about);
    int first = 0;
    do {
        const int r0 = ta * T::ROWS, c0 = tb * cols, this_a = ta, this_b = tb;
        if (stream) {
            walk.at += walk.step;
            more = find();
            if (more) {
                sources(src_next, about);
                turned_next = turn(tb);
            }
        }
        f32x4 acc[TM][TN];
        lce_run<TM, TN, ST, false>(acc, dsm, first, nk, wave, lane, advance, issue);
        first += nk;
        if (!stream) {
            lce_loads_done();
            __syncthreads();
            if (!T::AHEAD) note(about);
            __syncthreads();
        }

        // ---- lane (l16, lg) holds rows r0 + wm 16 TM + 16 i + l16, columns c0 + 16 TN wn + 16 j + 4 lg + 0..3
        const int row_w = wm * 16 * TM + l16, col_w = wn * 16 * TN + 4 * lg;
        if constexpr (MODE == kLceGrad) {
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int c = col_w + 16 * j;
                const f32x4 label = *(const f32x4*)(info + c), lse = *(const f32x4*)(info + 256 + c), up = *(const f32x4*)(info + 512 + c), rest = *(const f32x4*)(info + 768 + c);
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const int v = r0 + row_w + 16 * i;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], g.scale2, -lse[e]));
                        acc[i][j][e] = up[e] * (__float_as_int(label[e]) == v ? -rest[e] : p);
                    }
                }
                if (wn * 64 + 16 * j >= half) {             // what the rounding of the same token's value left (nothing of an infinity)
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float hi = bf16_to_f32(to_bf16(acc[i][j][e]));
                            acc[i][j][e] = fabsf(hi) == INFINITY ? 0.0f : acc[i][j][e] - hi;
                        }
                }
            }
        } else {
            // columns that the piece does not have, and the label's, count as -inf
            const int end = min(cols, g.n_v - c0);
            if (end < T::COLS) {
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (col_w + 16 * j + e >= end) acc[i][j][e] = -INFINITY;
            }
            float ref[TM], top[TM], sum[TM], kept[TM];
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                int at = __float_as_int(info[row_w + 16 * i]) - c0 - col_w;           // the label's column by the lane's own numbering of its 4 TN
                if (col_w + at >= end) at = -1;
                if (MODE == kLceExp) ref[i] = info[N_INFO + row_w + 16 * i];
                if (__any(at >= 0 && at < 16 * TN - 12)) {
#pragma unroll
                    for (int j = 0; j < TN; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (at == 16 * j + e) {
                                if (MODE == kLceStats && r0 + row_w + 16 * i < count) g.at_label[r0 + row_w + 16 * i] = acc[i][j][e] * g.scale2;
                                acc[i][j][e] = -INFINITY;
                            }
                }
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                top[i] = acc[i][0][0];
#pragma unroll
                for (int j = 0; j < TN; ++j) top[i] = max3(max3(top[i], acc[i][j][0], acc[i][j][1]), acc[i][j][2], acc[i][j][3]);
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) top[i] = over_groups_max(top[i]) * g.scale2;
            bool far = false;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const float base = MODE == kLceExp ? ref[i] : (top[i] == -INFINITY ? 0.0f : top[i]);
                if (MODE == kLceExp) far |= top[i] - base > kLceFar;
                f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
                f32x2 k = {0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < TN; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], g.scale2, -base));
                    s += acc[i][j];
                    if (MODE == kLceExp) {                  // as the image is to have it, and what that stands for
                        const uint32_t lo = pack_bf16x2(acc[i][j][0], acc[i][j][1]), hi = pack_bf16x2(acc[i][j][2], acc[i][j][3]);
                        k += f32x2{__uint_as_float(lo << 16), __uint_as_float(lo & 0xffff0000u)};
                        k += f32x2{__uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u)};
                        acc[i][j][0] = __uint_as_float(lo);
                        acc[i][j][1] = __uint_as_float(hi);
                    }
                }
                sum[i] = (s[0] + s[1]) + (s[2] + s[3]);
                kept[i] = k[0] + k[1];
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                sum[i] = over_groups_sum(sum[i]);
                if (MODE == kLceExp) kept[i] = over_groups_sum(kept[i]);
                if (lg == 0) sums[(row_w + 16 * i) * 4 + wn] = MODE == kLceExp ? f32x4{kept[i], sum[i], top[i], 0.0f} : f32x4{top[i], sum[i], 0.0f, 0.0f};
            }
            if (MODE == kLceExp && !g.again && __any(far)) {
                if (lane == 0) g.redo[this_a] = 1;          // (several may say so, all the same)
            }
            __syncthreads();
            if (tid < T::ROWS && r0 + tid < count) {
                f32x4 a = sums[tid * 4], b;
#pragma unroll
                for (int w = 1; w < 4; ++w) {
                    b = sums[tid * 4 + w];
                    if (MODE == kLceExp) {
                        a = f32x4{a[0] + b[0], a[1] + b[1], fmaxf(a[2], b[2]), 0.0f};
                        continue;
                    }
                    const float most = fmaxf(a[0], b[0]);
                    if (most != -INFINITY) a[1] = a[1] * __builtin_amdgcn_exp2f(a[0] - most) + b[1] * __builtin_amdgcn_exp2f(b[0] - most);
                    a[0] = most;
                }
                const int64_t at = (int64_t)this_b * g.rows_pad + r0 + tid;
                g.part[at] = f32x2{a[0], a[1]};
                // (done again: the largest stays what it was, the other tiles' blocks read it)
                if (MODE == kLceExp && !g.again) g.top[at] = a[2];
            }
        }
        if constexpr (MODE != kLceStats) {
            bf16_t* out = g.image + ((int64_t)this_a * g.image_steps + (c0 >> 5) + wn * (TN / 2)) * (T::ROWS * 32);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int row = row_w + 16 * i;
#pragma unroll
                for (int q = 0; q < TN / 2; ++q) {
                    if (TM <= 4) {
                        // the next tile's;  (the last tile goes on to the end of the image: the product takes K-steps in pairs)
                        const int step = wn * (TN / 2) + q;
                        if ((step * 32 >= cols && this_b + 1 < tiles_b) || (c0 >> 5) + step >= g.image_steps) continue;
                    }
                    const f32x4 a = acc[i][2 * q], b = acc[i][2 * q + 1];
                    u32x4* const to = (u32x4*)(out + (q * T::ROWS + row) * 32 + ((lg ^ ((row >> 2) & 2)) << 3));
                    if (MODE == kLceExp) *to = u32x4{__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(b[0]), __float_as_uint(b[1])};
                    else *to = u32x4{pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3])};
                }
            }
            if (MODE == kLceGrad) __syncthreads();          // (what the ends read of the columns is written anew)
        }
        if (stream) {
            if (more) note(about);
        } else if (T::AHEAD) {
            walk.at += walk.step;
            if (find()) {
                sources(src, about);
                turned = turn(tb);
                __syncthreads();
                lce_begin<T>(dsm, advance, issue);
                note(about);
                __syncthreads();
                first = 0;
                continue;
            }
        }
        if (!more) break;
    } while (true);
    lce_loads_done();
}

struct LceProductArgs {
    const bf16_t* image;
    int32_t image_steps;                // K-steps of the image's rows
    int32_t rows, k;                    // rows of the result and contraction; < 0: as many as count
    const int32_t* count;
    const bf16_t* B;                    // [k, H]
    int64_t ldb;
    int32_t H;
    const int32_t* parts;               // of the contraction, or NULL: it is not divided
    float* out;                         // [part of the contraction][row][H]: sums, added to what is there where `add`, that times alpha[row]
    const float* alpha;                 // (of row tiles that were done again; 1 otherwise)
    const int32_t* redo;
    int32_t add;
    bf16_t* out16;                      // or [rows, ld16] bf16: times *scale (NULL: 1)
    int64_t ld16;
    const float* scale;
};

// Parts of a contraction of E . W: as many as leave the least of the chip idle, where tiles alone would (a part costs its sums once more in
// memory: 2 % a part).  The rows that count are known on the device only, so that the kernel that counts them works it out, a wave with
// a number of parts in each lane.  Divided, tiles and parts are three rounds of the chip at most, one where the tiles are few (more would
// gain nothing), which bounds the sums.
constexpr int kLceMostParts = 64;
__host__ __device__ inline int lce_rounds(int tiles, int slots) { return 4 * tiles <= slots ? 1 : 3; }
__device__ __forceinline__ int lce_parts(int tiles, int steps, int slots, int lane) {
    const int s = lane + 1, all = tiles * s;
    const bool may = s == 1 || (all <= lce_rounds(tiles, slots) * slots && steps >= 16 * s);
    const float cost = may ? (float)((all + slots - 1) / slots) / (float)s * (1.0f + 0.02f * (float)(s - 1)) : INFINITY;
    float least = cost;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) least = fminf(least, __shfl_xor(least, d));
    return __builtin_ctzll(__ballot(cost <= least * 1.001f)) + 1;
}

template <int TM>
__global__ void __launch_bounds__(512, TM <= 2 ? 4 : 2) lce_product_kernel(LceProductArgs g) {
    using T = LceTile<TM>;
    extern __shared__ __attribute__((aligned(16))) unsigned char dsm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3, l16 = lane & 15, lg = lane >> 4;
    const int count = __builtin_amdgcn_readfirstlane(*g.count), rows = g.rows < 0 ? count : g.rows;
    const int half = g.k < 0 ? lce_half(count) : 1 << 30, k = g.k >= 0 ? g.k : half <= kLceSplit ? 2 * half : count, last = (g.k < 0 ? count : k) - 1;
    const int tiles_a = (rows + T::ROWS - 1) / T::ROWS, tiles_b = (g.H + 255) >> 8, tiles = tiles_a * tiles_b, pairs = (k + 63) >> 6;        // of K-steps
    const int parts = g.parts ? __builtin_amdgcn_readfirstlane(*g.parts) : 1;
    // an XCD has an eighth of all tiles and parts, in order of the parts: what it reads of E and W at a time are few rows and the same K-steps
    const int all = tiles * parts, b = blockIdx.x, per = all >> 3;
    if (b >= all) return;
    const int logical = b < per * 8 ? (b & 7) * per + (b >> 3) : b, s = logical / tiles;
    int ta, tb;
    lce_tile(logical - s * tiles, tiles_a, tiles_b, &ta, &tb);
    const int r0 = ta * T::ROWS, c0 = tb * 256;
    const int kt0 = 2 * (int)((int64_t)pairs * s / parts), nk = 2 * (int)((int64_t)pairs * (s + 1) / parts) - kt0;

    const bf16_t* const a_src = g.image + ((int64_t)ta * g.image_steps + kt0) * (T::ROWS * 32) + wave * (T::ROWS / 8) * 32 + lane * 8;
    const int kr = wave * 4 + (lane >> 5);             // of a K-step's rows, two more with the second load
    const bf16_t* b_col[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int unit = ((lane & 31) >> 1) ^ ((kr + 2 * p) & 7);
        b_col[p] = g.B + min(c0 + unit * 16 + (lane & 1) * 8, g.H - 8);
    }
    auto issue = [&](int kt, int part, uint32_t stage) {
        if (part < T::AP) {
            constexpr int rows8 = T::ROWS / 8;
            if (part * 16 + 16 <= rows8 || lane < (rows8 - part * 16) * 4)
                lce_load_lds(stage + wave * rows8 * 64 + part * 1024, a_src + (int64_t)kt * (T::ROWS * 32) + part * 512);
        } else {
            const int p = part - T::AP;
            const int at = (kt0 + kt) * 32, row = min((at >= half ? at - half : at) + kr + 2 * p, last);
            lce_load_lds(stage + T::A_BYTES + wave * 2048 + p * 1024, b_col[p] + row * g.ldb);
        }
    };
    f32x4 acc[TM][4];
    if (nk > 0) {
        auto advance = [&](int kt) { return min(kt, nk - 1); };         // (behind the last K-step: that one again, for nothing)
        lce_begin<T>(dsm, advance, issue);
        lce_run<TM, 4, 4, true>(acc, dsm, 0, nk, wave, lane, advance, issue);
        lce_loads_done();
    } else {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const int row_w = r0 + wm * 16 * TM + l16, col_w = c0 + wn * 64;
    if (g.out16) {
        const float scale = g.scale ? *g.scale : 1.0f;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int row = row_w + 16 * i;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                // eight columns in a row for each lane: fragments 2 q and 2 q + 1 exchange halves, then rows of sixteen lanes
                const f32x4 u = acc[i][2 * q] * scale, v = acc[i][2 * q + 1] * scale;
                uint32_t x[2] = {pack_bf16x2(u[0], u[1]), pack_bf16x2(u[2], u[3])}, y[2] = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    const auto h = __builtin_amdgcn_permlane32_swap(x[d], y[d], false, false);
                    const auto r = __builtin_amdgcn_permlane16_swap(h[0], h[1], false, false);
                    x[d] = r[0];
                    y[d] = r[1];
                }
                const int col = col_w + q * 32 + lg * 8;
                if (row < rows && col < g.H) *(u32x4*)(g.out16 + row * g.ld16 + col) = u32x4{x[0], x[1], y[0], y[1]};
            }
        }
        return;
    }
    float* const out = g.out + (int64_t)s * rows * g.H;
    const bool again = g.add && g.redo[ta];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int row = row_w + 16 * i;
        if (row >= rows) continue;
        const float alpha = again ? g.alpha[row] : 1.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = col_w + 16 * j + 4 * lg;
            if (col >= g.H) continue;
            f32x4* o = (f32x4*)(out + (int64_t)row * g.H + col);
            *o = g.add ? *o * alpha + acc[i][j] : acc[i][j];
        }
    }
}

}  // namespace xq
