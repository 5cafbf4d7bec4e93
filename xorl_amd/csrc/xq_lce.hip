// Cross entropy over an output head, in pieces of the vocabulary, with its gradients; no logits are kept.
//
//   l_iv = c x_i . w_v        loss_i = log sum_v exp(l_iv) - l_it        t = label of row i
//   dx_i = g_i c (sum_v p_iv w_v - w_t)        dw_v = c sum_i g_i (p_iv - [v = t_i]) x_i
//
// Rows whose label is ignore_index are taken out first (prepare_kernel lists the others in order), so that they cost nothing: every launch
// covers the most rows there can be and blocks behind the last one end at once.  The label's column is left out of all sums and joined
// at the end: with Z' = sum_{v != t} exp(l_v - ref), e_t = exp(l_t - ref),
//   loss = log(Z' + e_t) + ref - l_t        (log1p(Z') where ref is the label's own logit)
//   dx_i = g_i c (O_i - Y w_t) / (Z' + e_t),        O_i = sum_{v != t} E_v w_v,        Y = sum_{v != t} E_v,        E_v = exp(l_v - ref) as bf16
// which keeps what a confident row has left of its loss and gradient, where p_t - 1 would cancel.  Y, and not Z', is taken off: the roundings of
// E then count on differences w_v - w_t, and what the rows of the head have in common cancels (300 tokens under rows whose common part is 16 times
// their spread, [4096, 256]: the gradient is off by 0.0017 of it, 0.0022 at worst, which is the result's own rounding; 0.0029 and 0.0152 with Z').
//
//  * Scores (no gradient wanted): one product whose ends are the largest logit and the sum of exponentials of 256 columns; one joining pass.
//  * Training: E = exp(l - ref) of a piece goes to the workspace as bf16, and E . W is added to O in fp32: the forward leaves
//    the whole input gradient but its factor, in two products, where forming the logits again in the backward would take three.  E needs
//    a reference before the row's largest logit is known: the label's own logit (lce_target_kernel).  E is right as long as no logit is more
//    than 2^64 times e above it; a piece that finds one takes the largest as the new reference (O and Z' are scaled to it) and is done
//    again for the row tiles concerned.  bf16 keeps E to half a step (up to 2^-8 of each term, of either sign).
//  * A trained head: the backward forms the logits again with the roles exchanged, G = g (p - [v = t]) as bf16 with the tokens along the
//    contraction, and multiplies it with the rows that count.  What all rows share of g (the mean's 1 / count, the logit scale) is left to the
//    result in 32 bits: in G it would be one and the same rounding error, up to half a step, of the whole gradient.
//
// 8192 rows, 5735 of which count, under [131072, 4096], forward and backward: 10.3 ms, in two pieces of 2.6 (logits) and 2.45 ms (product) each, 0.1 ms of
// everything else.  One row, scored: 188 us (192 with a launch of its own that lists the rows, as above 64 rows).  96 rows under [32003, 2048], forward and
// backward: 82 us, of which 32 and 27 are the products and the rest four small launches.
#include <algorithm>
#include <atomic>

#include "xq_lce.h"

namespace xq {
namespace {

constexpr int64_t kPieceBytes = 1ll << 30;          // of E or G at a time
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kBeginRows = 1024;                    // rows whose labels every block of a launch looks through by itself

inline int64_t up256(int64_t n) { return (n + 255) & ~255ll; }

// the rows that count, in order; arrays as long as whole tiles (behind the last row: no label)
struct Prep {
    const void* labels;
    int32_t label_bytes;
    int64_t M, M_pad, V, ignore;
    int32_t *count, *row, *label, *place;           // place: of a row of x among those that count, or -1
    int32_t* redo;                                  // flags to clear
    int32_t n_redo;
    float* loss_out;                                // losses by row, 0 for those that do not count; or NULL
    int32_t tile_rows, tiles_h, steps, slots;       // of E . W, for the parts of its contraction (count[1])
};
__device__ __forceinline__ int64_t label_of(const Prep& a, int64_t i) { return i < a.M ? lce_label(a.labels, a.label_bytes, i) : a.ignore; }
// a thread's label among 1024: whether it counts, and how many before it do; all: how many of the 1024
__device__ __forceinline__ bool place_of(bool in, int* before, int* all, int* wave_n) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t mask = __ballot(in);
    __syncthreads();
    if (lane == 0) wave_n[wave] = __builtin_popcountll(mask);
    __syncthreads();
    int n = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        if (w == wave) n = sum;
        sum += wave_n[w];
    }
    *before = n + __builtin_popcountll(mask & ((1ull << lane) - 1));
    *all = sum;
    return in;
}
__device__ __forceinline__ void write_row(const Prep& a, int64_t i, int64_t label, bool in, int c) {
    if (in) {
        a.row[c] = (int)i;
        a.label[c] = label >= 0 && label < a.V ? (int)label : -1;
    }
    if (i < a.M) {
        a.place[i] = in ? c : -1;
        if (!in && a.loss_out) a.loss_out[i] = 0.0f;
    }
}
__device__ __forceinline__ void write_rest(const Prep& a, int n) {
    if (threadIdx.x < 64) {
        const int parts = lce_parts((n + a.tile_rows - 1) / a.tile_rows * a.tiles_h, a.steps, a.slots, threadIdx.x);
        if (threadIdx.x == 0) {
            a.count[0] = n;
            a.count[1] = parts;
        }
    }
    for (int64_t c = n + threadIdx.x; c < a.M_pad; c += 1024) {
        a.row[c] = 0;
        a.label[c] = -1;
    }
    for (int i = threadIdx.x; i < a.n_redo; i += 1024) a.redo[i] = 0;
}

// A block of 1024 threads finds the rows that count, of up to kBeginRows labels, and notes the sixteen from first on; the first block does what
// lce_prepare_kernel does
__device__ __forceinline__ void own_rows_of(const Prep& a, int64_t first, int* count, int* wave_n, int* rows, int* labels) {
    const int64_t i = threadIdx.x, label = label_of(a, i);
    int at;
    const bool in = place_of(label != a.ignore, &at, count, wave_n);
    if (in && at >= first && at < first + 16) {
        rows[at - first] = (int)i;
        labels[at - first] = label >= 0 && label < a.V ? (int)label : -1;
    }
    if (blockIdx.x == 0) {
        write_row(a, i, label, in, at);
        write_rest(a, *count);
    }
    __syncthreads();
}

__global__ void __launch_bounds__(1024) lce_prepare_kernel(Prep a) {
    __shared__ int wave_n[16];
    int base = 0;
    for (int64_t at = 0; at < a.M; at += 1024) {
        const int64_t i = at + threadIdx.x, label = label_of(a, i);
        int c, all;
        const bool in = place_of(label != a.ignore, &c, &all, wave_n);
        write_row(a, i, label, in, base + c);
        base += all;
    }
    write_rest(a, base);
}

__device__ __forceinline__ f32x4 bf16x4_f32(u32x2 w) {
    return f32x4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xffff0000u)};
}

// The label's logit of every row (log2 units): the first reference.  A wave has a row.  own_rows (up to kBeginRows labels): every block finds
// its rows by itself, and the first does what lce_prepare_kernel does.
__global__ void __launch_bounds__(1024) lce_target_kernel(Prep a, int own_rows, const bf16_t* x, int64_t ldx, const bf16_t* w, int64_t ldw, int H, float scale2,
                                                          float* at_label, float* ref, f32x2* z) {
    __shared__ int wave_n[16], rows[16], labels[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t first = (int64_t)blockIdx.x * 16, c = first + wave;
    int count;
    if (own_rows) {
        own_rows_of(a, first, &count, wave_n, rows, labels);
    } else {
        count = *a.count;
    }
    if (c >= count) return;
    const int label = own_rows ? labels[wave] : a.label[c];
    const int64_t row = own_rows ? rows[wave] : a.row[c];
    float sum = 0.0f;
    if (label >= 0) {
        const bf16_t *xr = x + row * ldx, *wr = w + label * ldw;
#pragma unroll 4
        for (int k = lane * 8; k < H; k += 512) {
            const u32x4 p = *(const u32x4*)(xr + k), q = *(const u32x4*)(wr + k);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                sum += __uint_as_float(p[j] << 16) * __uint_as_float(q[j] << 16) + __uint_as_float(p[j] & 0xffff0000u) * __uint_as_float(q[j] & 0xffff0000u);
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) {
        at_label[c] = ref[c] = label >= 0 ? sum * scale2 : __builtin_nanf("");
        z[c] = f32x2{0.0f, 0.0f};
    }
}

// ---- joins over the column tiles: 16 rows a block, 64 groups of lanes over the tiles
struct Join {
    const int32_t* count;
    const f32x2* part;
    int64_t rows_pad;
    int32_t tiles, tile_rows;
    float* ref;
    f32x2* z;                           // (Y, Z') so far
    const float *new_ref, *alpha;       // of row tiles that were done again
    const int32_t* redo;
};

// in the first 16 threads of a block, for rows that count: the row's join
template <typename F>
__device__ __forceinline__ bool join_rows(const Join& a, int count, f32x2 start, F fold, f32x2* out, int64_t* row) {
    __shared__ f32x2 lds[16][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r = (int64_t)blockIdx.x * 16 + (lane & 15);
    if ((int64_t)blockIdx.x * 16 >= count) return false;
    f32x2 v = start;
    const f32x2* p = a.part + r;                            // (behind the last row: whatever is there, for nothing)
#pragma unroll 8
    for (int t = threadIdx.x >> 4; t < a.tiles; t += 64) v = fold(v, p[t * a.rows_pad]);
#pragma unroll
    for (int d = 16; d < 64; d <<= 1) v = fold(v, f32x2{__shfl_xor(v[0], d), __shfl_xor(v[1], d)});
    if (lane < 16) lds[wave][lane] = v;
    __syncthreads();
    if (threadIdx.x >= 16 || r >= count) return false;
    v = lds[0][lane];
#pragma unroll
    for (int w = 1; w < 16; ++w) v = fold(v, lds[w][lane]);
    *out = v;
    *row = r;
    return true;
}
__device__ __forceinline__ f32x2 fold_sum(f32x2 p, f32x2 q) { return p + q; }

// a row's sums and reference with those of a piece
__device__ __forceinline__ void add_piece(const Join& a, int64_t r, f32x2 sum, f32x2* z, float* ref) {
    *z = a.z[r];
    *ref = a.ref[r];
    if (a.redo[r / a.tile_rows]) {
        *z *= a.alpha[r];
        *ref = a.new_ref[r];
    }
    *z += sum;
}
__global__ void __launch_bounds__(1024) lce_sum_kernel(Join a) {
    f32x2 v;
    int64_t r;
    if (!join_rows(a, *a.count, f32x2{0.0f, 0.0f}, fold_sum, &v, &r)) return;
    f32x2 z;
    float ref;
    add_piece(a, r, v, &z, &ref);
    a.z[r] = z;
    a.ref[r] = ref;
}

// what is kept of a row: 1 / Z, Z' / Z, Y / Z (EXP), log2 of the sum of exponentials
struct RowEnd {
    float *inv, *rest, *off, *lse2, *loss;
    const int32_t* row;
    float* out;                         // losses by row of x, or NULL
};
__device__ __forceinline__ float end_row(const RowEnd& e, int64_t c, int row, float z, float ref, float t) {
    // (ref - t is 0 where the label's own logit is the reference, and NaN where that is infinite)
    const float apart = ref - t, et = __builtin_amdgcn_exp2f(-apart), sum = z + et;
    const float loss = apart == 0.0f ? log1pf(z) : logf(sum) + apart * kLn2;
    e.loss[c] = loss;
    if (e.out) e.out[row] = loss;
    const float inv = 1.0f / sum;
    e.inv[c] = inv;
    e.rest[c] = z / sum;
    e.lse2[c] = apart == 0.0f ? log1pf(z) * kLog2e + t : log2f(sum) + ref;
    return inv;
}

// STATS: joins and ends.  own_rows: as the logits kernel, every block finds the rows that count by itself, and the first notes them
__global__ void __launch_bounds__(1024) lce_score_kernel(Join a, Prep p, int own_rows, const float* at_label, RowEnd e) {
    __shared__ int wave_n[16], rows[16], labels[16];
    const int64_t first = (int64_t)blockIdx.x * 16, c = first + (threadIdx.x & 15);
    int count, row = 0, label = -1;
    // (read before the count is known: arrays as long as whole tiles)
    const float found = at_label[c];
    if (own_rows) {
        own_rows_of(p, first, &count, wave_n, rows, labels);
        row = rows[threadIdx.x & 15];
        label = labels[threadIdx.x & 15];
    } else {
        row = p.row[c];
        label = p.label[c];
        count = *a.count;
    }
    f32x2 v;
    int64_t r;
    auto fold = [](f32x2 p, f32x2 q) {
        const float top = fmaxf(p[0], q[0]), by = top == -INFINITY ? 0.0f : top;
        return f32x2{top, p[1] * __builtin_amdgcn_exp2f(p[0] - by) + q[1] * __builtin_amdgcn_exp2f(q[0] - by)};
    };
    if (!join_rows(a, count, f32x2{-INFINITY, 0.0f}, fold, &v, &r)) return;
    const float t = label >= 0 ? found : __builtin_nanf("");
    const float ref = v[0] > t ? v[0] : t;
    end_row(e, r, row, v[1] * __builtin_amdgcn_exp2f(v[0] - ref), ref, t);
}
// EXP: the last piece's sums, and ends; the label's logit is the first reference
__global__ void __launch_bounds__(1024) lce_end_kernel(Join a, const float* at_label, RowEnd e) {
    f32x2 v;
    int64_t r;
    if (!join_rows(a, *a.count, f32x2{0.0f, 0.0f}, fold_sum, &v, &r)) return;
    f32x2 z;
    float ref;
    add_piece(a, r, v, &z, &ref);
    e.off[r] = z[0] * end_row(e, r, e.row[r], z[1], ref, at_label[r]);
}

// sum or mean of the losses: one block, in an order that the sizes fix
__global__ void __launch_bounds__(1024) lce_reduce_kernel(const int32_t* count, const float* loss, int mean, float* out) {
    __shared__ double lds[16];
    const int n = *count;
    double s = 0.0;
    for (int c = threadIdx.x; c < n; c += 1024) s += (double)loss[c];
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < 16; ++w) s += lds[w];
    *out = (float)(mean ? s / n : s);
}

// ---- backward
struct Upstream {
    const float* grad;
    int32_t reduction;
    const int32_t* count;
    float scale;
};
// (upstream is the product of the two behind it)
__device__ __forceinline__ float upstream_of_row(const Upstream& u, int64_t row) { return u.reduction == XQ_LCE_NONE ? u.grad[row] : 1.0f; }
__device__ __forceinline__ float upstream_of_all(const Upstream& u) {
    const int count = *u.count;
    if (u.reduction == XQ_LCE_NONE || count == 0) return u.scale;
    return u.reduction == XQ_LCE_MEAN ? *u.grad * u.scale / (float)count : *u.grad * u.scale;
}
__device__ __forceinline__ float upstream(const Upstream& u, int64_t row) {
    const float g = u.grad[u.reduction == XQ_LCE_NONE ? row : 0] * u.scale;
    return u.reduction == XQ_LCE_MEAN ? g / (float)*u.count : g;
}

// dx: a block has 512 columns of a row of x, a thread 8 of them
__global__ void __launch_bounds__(64) lce_dx_kernel(const int32_t* place, const int32_t* label, int H, const float* o,
                                                    const float* inv, const float* off, const bf16_t* w, int64_t ldw, Upstream u, bf16_t* dx, int64_t lddx) {
    const int64_t i = blockIdx.x;
    const int k = blockIdx.y * 512 + threadIdx.x * 8;
    if (k >= H) return;
    const int c = place[i];
    u32x4* out = (u32x4*)(dx + i * lddx + k);
    if (c < 0) {
        *out = u32x4{0, 0, 0, 0};
        return;
    }
    const int t = label[c], count = u.count[0], parts = u.count[1];
    const u32x4 wt = *(const u32x4*)(w + max(t, 0) * ldw + k);
    const float g = upstream(u, i);
    const float a = g * inv[c], b = t < 0 ? __builtin_nanf("") : g * off[c];
    const float* oc = o + (int64_t)c * H + k;
    f32x4 lo = {0.0f, 0.0f, 0.0f, 0.0f}, hi = lo;
#pragma unroll 4
    for (int s = 0; s < parts; ++s) {
        lo += *(const f32x4*)(oc + s * (int64_t)count * H);
        hi += *(const f32x4*)(oc + s * (int64_t)count * H + 4);
    }
    lo = lo * a - bf16x4_f32(u32x2{wt[0], wt[1]}) * b;
    hi = hi * a - bf16x4_f32(u32x2{wt[2], wt[3]}) * b;
    *out = u32x4{pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]), pack_bf16x2(hi[0], hi[1]), pack_bf16x2(hi[2], hi[3])};
}

// the factors of the head's gradient by row, and the rows of x that count in order
__global__ void __launch_bounds__(256) lce_factors_kernel(LceRows rows, int64_t M_pad, const float* lse2, const float* rest, Upstream u, float* lse_out, float* up_out,
                                                          float* rest_out, float* all_out) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= M_pad) return;
    const bool in = c < *rows.count;
    lse_out[c] = in ? lse2[c] : INFINITY;
    up_out[c] = in ? upstream_of_row(u, rows.row[c]) : 0.0f;
    if (c == 0) *all_out = upstream_of_all(u);
    rest_out[c] = in ? rest[c] : 0.0f;
}
__global__ void __launch_bounds__(256) lce_gather_kernel(LceRows rows, const bf16_t* x, int64_t ldx, int H, bf16_t* out) {
    const int64_t c = blockIdx.x;
    if (c >= *rows.count) return;
    const bf16_t* xr = x + rows.row[c] * ldx;
    for (int k = threadIdx.x * 8; k < H; k += 2048) *(u32x4*)(out + c * H + k) = *(const u32x4*)(xr + k);
}

// ---------------------------------------------------------------- host side
int compute_units() {
    static std::atomic<int> cached{0};
    int n = cached.load(std::memory_order_relaxed), dev = 0;
    if (n > 0) return n;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cached.store(n, std::memory_order_relaxed);
    return n;
}

// blocks of a product that run at a time, for lce_parts
int slots(int tm) { return (tm == 2 ? 2 : 1) * compute_units(); }

// a kernel may have as much LDS as it asks for on the current device; raised: by device (a race only repeats the call)
int raise_lds(const void* kernel, int bytes, std::atomic<uint64_t>& raised) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (e == hipSuccess && dev < 64 && (raised.load(std::memory_order_relaxed) & bit)) return XQ_OK;
    if (e == hipSuccess) e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) { xq_set_error("xq_lce: cannot raise the dynamic LDS limit: %s", hipGetErrorString(e)); return XQ_ERR_LAUNCH; }
    raised.fetch_or(bit, std::memory_order_relaxed);
    return XQ_OK;
}

struct Plan {
    int tm, cols;                       // rows of a logits tile: 32 tm, and its columns
    int64_t rows_pad, piece, pieces;    // columns of the vocabulary at a time (a multiple of 256), and how many times
};

int tile_for(int64_t rows) { return rows <= 64 ? 2 : rows <= 128 ? 4 : 8; }

// Columns of a tile.  Up to 128 rows reading the head is what counts, and a compute unit reads at a rate of its own: as many columns as leave
// the busiest the least to read (100003 columns: 481 tiles of 208 and not 391 of 256, of which some units have two and some one).
// A tile costs what 16 columns do beside.  E: whole K-steps of 32.
int columns_for(int tm, int64_t V, bool steps) {
    if (tm > 4) return 256;
    int best = 256;
    int64_t least = INT64_MAX;
    for (int c = 256; c >= 64; c -= steps ? 32 : 16) {
        const int64_t cost = xq_cdiv(xq_cdiv(V, c), compute_units()) * (c + 16);
        if (cost < least) { least = cost; best = c; }
    }
    return best;
}

// tm 0: by the rows;  steps: E is wanted
Plan plan_for(int64_t M, int64_t V, int tm, bool steps) {
    Plan p;
    p.tm = tm ? tm : tile_for(M);
    p.rows_pad = up256(std::max<int64_t>(M, 1));
    const int64_t most = std::max<int64_t>(256, kPieceBytes / (p.rows_pad * 2) / 256 * 256);
    p.pieces = xq_cdiv(up256(V), most);
    p.piece = up256(xq_cdiv(up256(V), p.pieces));
    p.pieces = xq_cdiv(V, p.piece);
    p.cols = columns_for(p.tm, steps ? std::min(V, p.piece) : V, steps);
    return p;
}
Plan plan_tokens(int64_t M, int64_t V, int keep) { return plan_for(M, V, 0, keep == XQ_LCE_KEEP_DX); }
Plan plan_head(int64_t M, int64_t V) { return plan_for(M, V, 8, true); }          // G: rows of the vocabulary, tokens along the contraction

// rows of E, whole tiles of them
int64_t image_rows(const Plan& p, int64_t M) { return xq_cdiv(std::max<int64_t>(M, 1), 32 * p.tm) * 32 * p.tm; }

// fp32 sums of E . W over the parts of the contraction, however many of the rows count (lce_parts)
int64_t sums_bytes(const Plan& p, int64_t M, int64_t H) {
    const int64_t tiles_h = xq_cdiv(H, 256), rows = 32 * p.tm, free = slots(p.tm);
    int64_t most = M * H;
    for (int64_t t = 1; t <= xq_cdiv(M, rows); ++t) {
        const int64_t tiles = t * tiles_h, parts = std::min<int64_t>({kLceMostParts, lce_rounds((int)tiles, (int)free) * free / tiles, p.piece / 512});
        if (parts > 1) most = std::max(most, parts * std::min(t * rows, M) * H);
        else if (tiles > free) break;
    }
    return 4 * most;
}

// what a forward leaves for the backward
struct Saved {
    int32_t *count, *row, *label, *place;       // count[1]: parts of the contraction of E . W
    float *at_label, *inv, *rest, *off, *lse2, *loss, *o;
    int64_t bytes;
};
Saved saved_of(void* base, int64_t M, int64_t V, int64_t H, int keep) {
    const Plan p = plan_tokens(M, V, keep);
    uint8_t* at = (uint8_t*)base;
    auto take = [&](int64_t n) { uint8_t* r = at; at += up256(n); return r; };
    Saved s;
    s.count = (int32_t*)take(8);
    s.row = (int32_t*)take(4 * p.rows_pad);
    s.label = (int32_t*)take(4 * p.rows_pad);
    s.place = (int32_t*)take(4 * p.rows_pad);
    s.at_label = (float*)take(4 * p.rows_pad);
    s.inv = (float*)take(4 * p.rows_pad);
    s.rest = (float*)take(4 * p.rows_pad);
    s.off = keep == XQ_LCE_KEEP_DX ? (float*)take(4 * p.rows_pad) : nullptr;
    s.lse2 = (float*)take(4 * p.rows_pad);
    s.loss = (float*)take(4 * p.rows_pad);
    s.o = keep == XQ_LCE_KEEP_DX ? (float*)take(sums_bytes(p, M, H)) : nullptr;
    s.bytes = at - (uint8_t*)base;
    return s;
}

struct Scratch {
    float *ref, *rest, *alpha, *up, *new_ref, *top;
    int32_t* redo;
    f32x2 *part, *z;
    bf16_t *image, *x;
    int64_t bytes;
};
Scratch scratch_of(void* base, int64_t M, int64_t V, int64_t H, int pass) {
    const Plan p = pass == XQ_LCE_KEEP_HEAD_BWD ? plan_head(M, V) : plan_tokens(M, V, pass);
    uint8_t* at = (uint8_t*)base;
    auto take = [&](int64_t n) { uint8_t* r = at; at += up256(n); return r; };
    Scratch s = {};
    s.ref = (float*)take(4 * p.rows_pad);
    s.alpha = (float*)take(4 * p.rows_pad);
    s.up = (float*)take(4 * p.rows_pad);
    s.new_ref = (float*)take(4 * p.rows_pad);
    s.redo = (int32_t*)take(4 * p.pieces * (p.rows_pad / 64));
    if (pass == XQ_LCE_KEEP_HEAD_BWD) {
        s.rest = (float*)take(4 * p.rows_pad);
        s.x = (bf16_t*)take(2 * M * H);
        s.image = (bf16_t*)take(2 * p.rows_pad * p.piece);
    } else {
        const int64_t tiles = xq_cdiv(pass == XQ_LCE_KEEP_DX ? p.piece : V, p.cols);
        s.part = (f32x2*)take(8 * p.rows_pad * tiles);
        if (pass == XQ_LCE_KEEP_DX) {
            s.z = (f32x2*)take(8 * p.rows_pad);
            s.top = (float*)take(4 * p.rows_pad * tiles);
            s.image = (bf16_t*)take(2 * image_rows(p, M) * p.piece);
        }
    }
    s.bytes = at - (uint8_t*)base;
    return s;
}

template <int TM, int TN, int ST, int MODE>
int launch_logits(const LceLogitsArgs& a, int64_t rows, int64_t cols, hipStream_t s) {
    using T = LceTile<TM, TN, ST>;
    auto k = lce_logits_kernel<TM, TN, ST, MODE>;
    static std::atomic<uint64_t> raised{0};
    const int rc = raise_lds((const void*)k, T::LDS_BYTES, raised);
    if (rc != XQ_OK) return rc;
    int64_t blocks = xq_cdiv(rows, T::ROWS) * xq_cdiv(cols, a.cols);
    if (T::AHEAD) blocks = std::min<int64_t>(blocks, compute_units());
    k<<<dim3((unsigned)blocks), 512, T::LDS_BYTES, s>>>(a);
    return XQ_OK;
}
// tokens as rows.  Up to 128 columns a tile: eight stages, as a unit with one block reads no faster than its loads in flight allow
template <int MODE>
int launch_logits(int tm, const LceLogitsArgs& a, int64_t rows, int64_t cols, hipStream_t s) {
    if (tm == 2) return a.cols <= 128 ? launch_logits<2, 2, 8, MODE>(a, rows, cols, s) : launch_logits<2, 4, 4, MODE>(a, rows, cols, s);
    if (tm == 4) return a.cols <= 128 ? launch_logits<4, 2, 8, MODE>(a, rows, cols, s) : launch_logits<4, 4, 4, MODE>(a, rows, cols, s);
    return launch_logits<8, 4, 4, MODE>(a, rows, cols, s);
}
template <int TM>
int launch_product(const LceProductArgs& a, int64_t rows, hipStream_t s) {
    using T = LceTile<TM>;
    auto k = lce_product_kernel<TM>;
    static std::atomic<uint64_t> raised{0};
    const int rc = raise_lds((const void*)k, T::LDS_BYTES, raised);
    if (rc != XQ_OK) return rc;
    int64_t blocks = xq_cdiv(rows, T::ROWS) * xq_cdiv(a.H, 256);
    if (a.parts) blocks = std::max<int64_t>(blocks, std::min<int64_t>(kLceMostParts * blocks, 3ll * slots(TM)));
    k<<<dim3((unsigned)blocks), 512, T::LDS_BYTES, s>>>(a);
    return XQ_OK;
}
int launch_product(int tm, const LceProductArgs& a, int64_t rows, hipStream_t s) {
    return tm == 2 ? launch_product<2>(a, rows, s) : tm == 4 ? launch_product<4>(a, rows, s) : launch_product<8>(a, rows, s);
}

// (a launch has fewer than 2^32 threads: 256 a row in the gather, 512 for 64 columns of few rows)
bool sizes_fit(int64_t M, int64_t V, int64_t H) { return M >= 0 && M < (1 << 24) && V >= 1 && V < (1 << 28) && H >= 1 && H < (1 << 24); }

int check_problem(const char* who, const xq_lce_problem* q, const void* ws, int64_t ws_bytes, int64_t need, const void* saved, int64_t saved_need) {
    XQ_REQUIRE(q, "%s: the problem is NULL", who);
    XQ_REQUIRE(sizes_fit(q->M, q->V, q->H), "%s: %lld rows, %lld columns of logits, hidden size %lld", who, (long long)q->M, (long long)q->V, (long long)q->H);
    XQ_REQUIRE(q->H >= 64 && q->H % 64 == 0, "%s: the hidden size must be a multiple of 64, got %lld", who, (long long)q->H);
    XQ_REQUIRE(q->reduction >= XQ_LCE_NONE && q->reduction <= XQ_LCE_SUM, "%s: unknown reduction %d", who, q->reduction);
    XQ_REQUIRE(q->label_bytes == 4 || q->label_bytes == 8, "%s: labels are int32 or int64, got %d bytes", who, q->label_bytes);
    XQ_REQUIRE(q->logit_scale > 0.0f && q->logit_scale < INFINITY, "%s: logit_scale must be positive and finite, got %g", who, (double)q->logit_scale);
    XQ_REQUIRE(q->w && xq_aligned(q->w, 16) && q->ldw >= q->H && q->ldw % 8 == 0, "%s: the head must be 16-byte aligned with a row stride that is a multiple of 8 elements", who);
    XQ_REQUIRE(q->M == 0 || (q->x && xq_aligned(q->x, 16) && q->ldx >= q->H && q->ldx % 8 == 0),
               "%s: x must be 16-byte aligned with a row stride that is a multiple of 8 elements", who);
    XQ_REQUIRE(q->M == 0 || (q->labels && xq_aligned(q->labels, q->label_bytes)), "%s: labels are NULL or misaligned", who);
    XQ_REQUIRE(ws && xq_aligned(ws, 256) && ws_bytes >= need, "%s: a workspace of %lld bytes, 256-byte aligned, is needed", who, (long long)need);
    XQ_REQUIRE(saved_need == 0 || (saved && xq_aligned(saved, 256)), "%s: the saved buffer is NULL or not 256-byte aligned", who);
    return XQ_OK;
}

}  // namespace
}  // namespace xq

using namespace xq;

extern "C" int64_t xq_lce_saved_bytes(int64_t M, int64_t V, int64_t H, int keep) {
    if (!sizes_fit(M, V, H)) return -1;
    return saved_of(nullptr, M, V, H, keep).bytes;
}

extern "C" int64_t xq_lce_workspace_bytes(int64_t M, int64_t V, int64_t H, int pass) {
    if (!sizes_fit(M, V, H)) return -1;
    return scratch_of(nullptr, M, V, H, pass).bytes;
}

extern "C" int xq_lce_fwd(const xq_lce_problem* q, float* loss, void* saved, int keep, void* workspace, int64_t workspace_bytes, void* stream) {
    XQ_REQUIRE(q && keep >= XQ_LCE_KEEP_NONE && keep <= XQ_LCE_KEEP_DX, "xq_lce_fwd: the problem is NULL or keep is unknown");
    int rc = check_problem("xq_lce_fwd", q, workspace, workspace_bytes, xq_lce_workspace_bytes(q->M, q->V, q->H, keep), saved, 1);
    if (rc != XQ_OK) return rc;
    XQ_REQUIRE((loss && xq_aligned(loss, 4)) || (q->M == 0 && q->reduction == XQ_LCE_NONE), "xq_lce_fwd: loss is NULL or misaligned");
    hipStream_t st = (hipStream_t)stream;
    const int64_t M = q->M, V = q->V, H = q->H;
    const Plan p = plan_tokens(M, V, keep);
    const Saved s = saved_of(saved, M, V, H, keep);
    const Scratch c = scratch_of(workspace, M, V, H, keep);
    const float scale2 = q->logit_scale * kLog2e;
    const bool none = q->reduction == XQ_LCE_NONE;
    const int row_tiles = (int)xq_cdiv(M, 32 * p.tm);
    const RowEnd end = {s.inv, s.rest, s.off, s.lse2, s.loss, s.row, none ? loss : nullptr};
    const Prep prep = {q->labels, q->label_bytes, M, p.rows_pad, V, q->ignore_index, s.count, s.row, s.label, s.place, c.redo,
                       keep == XQ_LCE_KEEP_DX ? (int32_t)(p.pieces * row_tiles) : 0, none ? loss : nullptr,
                       32 * p.tm, (int32_t)xq_cdiv(H, 256), (int32_t)(p.piece / 32), slots(p.tm)};
    const dim3 by16((unsigned)xq_cdiv(M, 16));
    Join join = {s.count, c.part, p.rows_pad, 0, 32 * p.tm, c.ref, c.z, c.new_ref, c.alpha, nullptr};
    LceLogitsArgs a = {};
    a.A = (const bf16_t*)q->x; a.lda = q->ldx; a.B = (const bf16_t*)q->w; a.ldb = q->ldw;
    a.H = (int32_t)H; a.cols = p.cols; a.rows = {s.count, s.row, s.label}; a.scale2 = scale2; a.part = c.part; a.rows_pad = p.rows_pad;
    // few rows: no launch before the others that finds those that count
    const bool own_rows = M > 0 && M <= (keep == XQ_LCE_KEEP_DX ? kBeginRows : kLceOwnRows);
    if (!own_rows) lce_prepare_kernel<<<dim3(1), 1024, 0, st>>>(prep);
    if (M > 0 && keep != XQ_LCE_KEEP_DX) {
        a.n_v = (int32_t)V; a.at_label = s.at_label;
        if (own_rows) a.labels = {q->labels, q->label_bytes, (int32_t)M, q->ignore_index, V};
        if ((rc = launch_logits<kLceStats>(p.tm, a, M, V, st)) != XQ_OK) return rc;
        join.tiles = (int32_t)xq_cdiv(V, p.cols);
        lce_score_kernel<<<by16, 1024, 0, st>>>(join, prep, own_rows, s.at_label, end);
    } else if (M > 0) {
        lce_target_kernel<<<by16, 1024, 0, st>>>(prep, own_rows, a.A, a.lda, a.B, a.ldb, (int)H, scale2, s.at_label, c.ref, c.z);
        a.ref = c.ref; a.new_ref = c.new_ref; a.alpha = c.alpha; a.top = c.top; a.image = c.image; a.image_steps = (int32_t)(p.piece / 32); a.redo = c.redo;
        for (int64_t v0 = 0; v0 < V; v0 += p.piece, a.redo += row_tiles) {
            const int64_t n = std::min(p.piece, V - v0);
            a.first_v = (int32_t)v0; a.n_v = (int32_t)n;
            for (a.again = 0; a.again < 2; ++a.again)
                if ((rc = launch_logits<kLceExp>(p.tm, a, M, n, st)) != XQ_OK) return rc;
            join.tiles = (int32_t)xq_cdiv(n, p.cols); join.redo = a.redo;
            if (v0 + n < V) lce_sum_kernel<<<by16, 1024, 0, st>>>(join);
            else lce_end_kernel<<<by16, 1024, 0, st>>>(join, s.at_label, end);
            LceProductArgs o = {};
            o.image = c.image; o.image_steps = a.image_steps; o.rows = -1; o.k = (int32_t)n; o.count = s.count;
            o.B = a.B + v0 * a.ldb; o.ldb = a.ldb; o.H = (int32_t)H; o.parts = s.count + 1;
            o.out = s.o; o.alpha = c.alpha; o.redo = a.redo; o.add = v0 > 0;
            if ((rc = launch_product(p.tm, o, M, st)) != XQ_OK) return rc;
        }
    }
    if (!none) lce_reduce_kernel<<<dim3(1), 1024, 0, st>>>(s.count, s.loss, q->reduction == XQ_LCE_MEAN, loss);
    XQ_CHECK_LAUNCH("xq_lce_fwd");
    return XQ_OK;
}

extern "C" int xq_lce_bwd(const xq_lce_problem* q, const float* grad, const void* saved, int keep, void* dx, int64_t lddx, void* dw, int64_t lddw,
                          void* workspace, int64_t workspace_bytes, void* stream) {
    XQ_REQUIRE(q && (keep == XQ_LCE_KEEP_HEAD || keep == XQ_LCE_KEEP_DX), "xq_lce_bwd: the problem is NULL, or its forward kept nothing");
    int rc = check_problem("xq_lce_bwd", q, dw ? workspace : (const void*)256, dw ? workspace_bytes : 0, dw ? xq_lce_workspace_bytes(q->M, q->V, q->H, XQ_LCE_KEEP_HEAD_BWD) : 0,
                           saved, 1);
    if (rc != XQ_OK) return rc;
    XQ_REQUIRE((grad && xq_aligned(grad, 4)) || q->M == 0, "xq_lce_bwd: the upstream gradient is NULL or misaligned");
    XQ_REQUIRE(!dx || keep == XQ_LCE_KEEP_DX, "xq_lce_bwd: the forward was not asked to keep what dx needs");
    XQ_REQUIRE(!dx || (xq_aligned(dx, 16) && lddx >= q->H && lddx % 8 == 0), "xq_lce_bwd: dx must be 16-byte aligned with a row stride that is a multiple of 8 elements");
    XQ_REQUIRE(!dw || (xq_aligned(dw, 16) && lddw >= q->H && lddw % 8 == 0), "xq_lce_bwd: dw must be 16-byte aligned with a row stride that is a multiple of 8 elements");
    hipStream_t st = (hipStream_t)stream;
    const int64_t M = q->M, V = q->V, H = q->H;
    const Saved s = saved_of((void*)saved, M, V, H, keep);
    const LceRows rows = {s.count, s.row, s.label};
    const Upstream u = {grad, q->reduction, s.count, q->logit_scale};
    if (dx && M > 0)
        lce_dx_kernel<<<dim3((unsigned)M, (unsigned)xq_cdiv(H, 512)), 64, 0, st>>>(s.place, s.label, (int)H, s.o, s.inv, s.off, (const bf16_t*)q->w, q->ldw, u, (bf16_t*)dx, lddx);
    if (dw) {
        const Plan h = plan_head(M, V);
        const Scratch c = scratch_of(workspace, M, V, H, XQ_LCE_KEEP_HEAD_BWD);
        if (M > 0) {
            lce_factors_kernel<<<dim3((unsigned)(h.rows_pad / 256)), 256, 0, st>>>(rows, h.rows_pad, s.lse2, s.rest, u, c.ref, c.up, c.rest, c.alpha);
            lce_gather_kernel<<<dim3((unsigned)M), 256, 0, st>>>(rows, (const bf16_t*)q->x, q->ldx, (int)H, c.x);
        }
        LceLogitsArgs a = {};
        a.A = (const bf16_t*)q->w; a.lda = q->ldw; a.B = (const bf16_t*)q->x; a.ldb = q->ldx;
        a.H = (int32_t)H; a.cols = 256; a.rows = rows; a.scale2 = q->logit_scale * kLog2e; a.ref = c.ref; a.grad = c.up; a.rest = c.rest; a.rows_pad = h.rows_pad;
        a.image = c.image; a.image_steps = (int32_t)(h.rows_pad / 32);
        for (int64_t v0 = 0; v0 < V; v0 += h.piece) {
            const int64_t n = std::min(h.piece, V - v0);
            a.first_v = (int32_t)v0; a.n_v = (int32_t)n;
            if (M > 0 && (rc = launch_logits<8, 4, 4, kLceGrad>(a, n, M, st)) != XQ_OK) return rc;
            LceProductArgs o = {};
            o.image = c.image; o.image_steps = a.image_steps; o.rows = (int32_t)n; o.k = -1; o.count = s.count;
            o.B = c.x; o.ldb = H; o.H = (int32_t)H;
            o.out16 = (bf16_t*)dw + v0 * lddw; o.ld16 = lddw; o.scale = M > 0 ? c.alpha : nullptr;
            if ((rc = launch_product(h.tm, o, n, st)) != XQ_OK) return rc;
        }
    }
    XQ_CHECK_LAUNCH("xq_lce_bwd");
    return XQ_OK;
}
