// Embedding:  out[t] = scale W[id_t],   dW[v] = scale sum over the tokens t of v of grad[t], in their order.
// An id outside [0, V) gives a row of NaN and no gradient; tokens of padding_idx give none either.  dW is written whole.
//
// What bounds it: memory.  The forward reads and writes a row a token (16385 rows of 2048 bf16, 134 MB: 21.0 us, 6.4 TB/s, many of the rows from the caches; 64 rows 5 us, a
// launch).  The gradient reads one row a token and writes the whole of dW, nearly all of it zeros: 8192 tokens, [131072, 4096] bf16: 1.27 GB of the pass's traffic, 231 us
// with the forward, 198 at the rates of a copy and a fill.  Sorted tokens and not atomics: the same bits on every call, fp32 sums, and no pass that rounds them afterwards.
#include <algorithm>

#include "xq_common.h"

namespace xq {
namespace {

__device__ __forceinline__ int64_t token_id(const xq_embedding& q, int64_t t) {
    return q.id_bytes == 8 ? ((const int64_t*)q.ids)[t] : (int64_t)((const int32_t*)q.ids)[t];
}

// W elements of a row as one access: 16 bytes, or one element where addresses or pitches allow no more
template <typename T, int W>
struct Piece {
    T v[W];
};
template <typename T, int W>
__device__ __forceinline__ Piece<T, W> load_piece(const T* p) {
    Piece<T, W> r;
    if constexpr (W > 1) {
        static_assert(sizeof(r) == 16, "");
        r = __builtin_bit_cast(Piece<T, W>, *(const u32x4*)p);
    } else {
        r.v[0] = *p;
    }
    return r;
}
template <typename T, int W>
__device__ __forceinline__ void store_piece(T* p, const Piece<T, W>& r) {
    if constexpr (W > 1) *(u32x4*)p = __builtin_bit_cast(u32x4, r);
    else *p = r.v[0];
}
__device__ __forceinline__ float value(float v) { return v; }
__device__ __forceinline__ float value(bf16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ void put(float& to, float v) { to = v; }
__device__ __forceinline__ void put(bf16_t& to, float v) { to = to_bf16(v); }

// out[t] = scale W[id]: `lanes` threads U tokens after each other, whose rows are on their way together (16385 rows of 2048 bf16: 25.4 us one by one, 21.0 by four)
template <typename T, int W, int U>
__global__ void __launch_bounds__(256) embedding_kernel(xq_embedding q, T* out, int64_t ld_out, int32_t lanes) {
    const int per = 256 / lanes, lane = threadIdx.x & (lanes - 1);
    for (int64_t t0 = ((int64_t)blockIdx.x * per + threadIdx.x / lanes) * U; t0 < q.n_tokens; t0 += (int64_t)gridDim.x * per * U) {
        int64_t id[U];
        bool is[U];
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = token_id(q, min(t0 + u, q.n_tokens - 1));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            is[u] = id[u] >= 0 && id[u] < q.V;
            if (!is[u]) id[u] = 0;
        }
        for (int64_t h = lane * W; h < q.H; h += lanes * W) {
            Piece<T, W> r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) r[u] = load_piece<T, W>((const T*)q.weight + id[u] * q.ldw + h);
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < W; ++i) put(r[u].v[i], is[u] ? q.scale * value(r[u].v[i]) : NAN);
                if (t0 + u < q.n_tokens) store_piece<T, W>(out + (t0 + u) * ld_out + h, r[u]);
            }
        }
    }
}

// ---- the gradient: tokens sorted by id (stable), then a pass over the vocabulary that adds each row's tokens or writes its zeros
// Row v belongs to block v % blocks, as its row v / blocks: ids that come often lie next to each other in a vocabulary, and so go to different blocks.
typedef __attribute__((ext_vector_type(2))) int32_t i32x2;

struct Sorted {
    int32_t* start;           // [blocks * rows + 1]: where the tokens of a row begin in token[], by (v % blocks) * rows + v / blocks
    i32x2* token;             // [n_tokens]: the tokens and their ids, row by row, each row's in their order
    float* part;              // [n_tokens / kChunk, H]: sums over kChunk tokens in that order, where they are all of one row
    int32_t log_blocks, rows;
};
constexpr int kChunk = 16, kSlots = 8, kSortRows = 4096, kSortList = 3000, kSortEach = 8, kSortAtOnce = 256 * kSortEach;      // (list and counters: 35 KB, four blocks a unit)

// The tokens of a list go to their places, `next` of their row: 256 at a time, each wave's 64 ranked among themselves (those of one row agree in every bit
// of it), then the waves take their places in turn.
__device__ __forceinline__ void place_tokens(const uint16_t* row, const int32_t* token, int n, int bits, int32_t* next, const Sorted& s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i0 = 0; i0 < n; i0 += 256) {
        const int i = i0 + threadIdx.x;
        const bool is = i < n;
        const int r = is ? row[i] : 0;
        uint64_t same = __ballot(is);
        for (int b = 0; b < bits; ++b) {
            const bool bit = (r >> b) & 1;
            const uint64_t m = __ballot(bit);
            same &= bit ? m : ~m;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        int at = 0;
        for (int w = 0; w < 4 && i0 + w * 64 < n; ++w) {
            if (wave == w && is) {
                at = next[r] + rank;
                if (rank == __popcll(same) - 1) next[r] = at + 1;
            }
            __syncthreads();
        }
        if (is) s.token[at] = i32x2{token[i], (r << s.log_blocks) + (int)blockIdx.x};
    }
}

// Every sorting block looks through all ids: it counts its own rows' tokens, and those of the blocks before it, so that no launch is needed that adds counts
// up, and lists its own.  More of them than the list holds (a token that fills a batch) are found again in a second look.
// Blocks behind the sorting ones write zeros, 16 bytes a thread in the order of addresses: 1 GiB takes 150 us with four blocks on a unit, 175 to 240 in any
// other order that was tried (several pieces a thread, a share of the rows a block); the sort (8192 ids 9 us by itself) goes on beside them.
__global__ void __launch_bounds__(256) embedding_sort_kernel(xq_embedding q, Sorted s, u32x4* zeros, int64_t n_zeros) {
    __shared__ int32_t count[kSortRows], of_wave[2][4], token[kSortList];
    __shared__ uint16_t row[kSortList];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, block = blockIdx.x;
    const int64_t mask = (1 << s.log_blocks) - 1;
    if (block > (int)mask) {
        const int64_t stride = ((int64_t)gridDim.x - mask - 1) * 256;
        for (int64_t i = ((int64_t)block - mask - 1) * 256 + tid; i < n_zeros; i += stride) zeros[i] = u32x4{0, 0, 0, 0};
        return;
    }
    auto sum_up = [&](int v, int* all, int turn) {          // the values of the threads before this one, and all threads'; one barrier, two turns
        int upto = v;
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(upto, o, 64);
            if (lane >= o) upto += u;
        }
        if (lane == 63) of_wave[turn][wave] = upto;
        __syncthreads();
        int to = upto - v, sum = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int n = of_wave[turn][w];
            to += w < wave ? n : 0;
            sum += n;
        }
        *all = sum;
        return to;
    };
    for (int r = tid; r < s.rows; r += 256) count[r] = 0;
    __syncthreads();
    int before = 0, listed = 0, turn = 0;
    for (int64_t t0 = 0; t0 < q.n_tokens; t0 += kSortAtOnce, turn ^= 1) {
        // consecutive tokens a thread, so that the block's come in order
        int own[kSortEach], n = 0, found;
#pragma unroll
        for (int i = 0; i < kSortEach; ++i) {
            const int64_t t = t0 + tid * kSortEach + i, id = t < q.n_tokens ? token_id(q, t) : -1;
            const bool real = id >= 0 && id < q.V && id != q.padding_idx;
            const int at = (int)(id & mask);
            before += real && at < block;
            own[i] = real && at == block ? (int)(id >> s.log_blocks) : -1;
            n += own[i] >= 0;
        }
        int to = listed + sum_up(n, &found, turn);
        if (n)
#pragma unroll
            for (int i = 0; i < kSortEach; ++i)
                if (own[i] >= 0) {
                    atomicAdd(&count[own[i]], 1);
                    if (to < kSortList) {
                        row[to] = (uint16_t)own[i];
                        token[to] = (int)(t0 + tid * kSortEach + i);
                    }
                    ++to;
                }
        listed += found;
    }
    sum_up(before, &before, turn);
    turn ^= 1;
    // counts to places: each thread the rows it owns
    const int each = (s.rows + 255) / 256, first = tid * each, last = min(first + each, s.rows);
    int mine = 0, all;
    for (int r = first; r < last; ++r) mine += count[r];
    int at = before + sum_up(mine, &all, turn);
    turn ^= 1;
    for (int r = first; r < last; ++r) {
        const int n = count[r];
        count[r] = at;
        s.start[(int64_t)block * s.rows + r] = at;
        at += n;
    }
    if (block == (int)mask && tid == 0) s.start[(int64_t)(block + 1) * s.rows] = before + all;
    if (listed == 0) return;
    int bits = 0;
    while ((1 << bits) < s.rows) ++bits;
    __syncthreads();
    if (listed <= kSortList) {
        place_tokens(row, token, listed, bits, count, s);
        return;
    }
    for (int64_t t0 = 0; t0 < q.n_tokens; t0 += kSortAtOnce, turn ^= 1) {
        int own[kSortEach], n = 0, found;
#pragma unroll
        for (int i = 0; i < kSortEach; ++i) {
            const int64_t t = t0 + tid * kSortEach + i, id = t < q.n_tokens ? token_id(q, t) : -1;
            own[i] = id >= 0 && id < q.V && id != q.padding_idx && (int)(id & mask) == block ? (int)(id >> s.log_blocks) : -1;
            n += own[i] >= 0;
        }
        int to = sum_up(n, &found, turn);                  // (behind its barrier the list of the round before has been read)
#pragma unroll
        for (int i = 0; i < kSortEach; ++i)
            if (own[i] >= 0) {
                row[to] = (uint16_t)own[i];
                token[to++] = (int)(t0 + tid * kSortEach + i);
            }
        __syncthreads();
        place_tokens(row, token, found, bits, count, s);
    }
}

// `AHEAD` rows on their way at a time
template <typename T, int W, int AHEAD>
__device__ __forceinline__ void add_tokens(const i32x2* token, int from, int to, const T* grad, int64_t ld, int64_t h, float* sum) {
    int i = from;
    for (; i + AHEAD <= to; i += AHEAD) {
        Piece<T, W> r[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) r[u] = load_piece<T, W>(grad + token[i + u][0] * ld + h);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int j = 0; j < W; ++j) sum[j] += value(r[u].v[j]);
    }
    for (; i < to; ++i) {
        const Piece<T, W> r = load_piece<T, W>(grad + token[i][0] * ld + h);
#pragma unroll
        for (int j = 0; j < W; ++j) sum[j] += value(r.v[j]);
    }
}

// chunks of kChunk sorted tokens that are all of one row
template <typename T, int W>
__global__ void __launch_bounds__(256) embedding_part_kernel(xq_embedding q, Sorted s, const T* grad, int64_t ld) {
    const int64_t all = s.start[(int64_t)s.rows << s.log_blocks];
    for (int64_t c = blockIdx.x; (c + 1) * kChunk <= all; c += gridDim.x) {
        const i32x2* token = s.token + c * kChunk;
        if (token[0][1] != token[kChunk - 1][1]) continue;
        for (int64_t h = ((int64_t)blockIdx.y * 256 + threadIdx.x) * W; h < q.H; h += (int64_t)gridDim.y * 256 * W) {
            float sum[W] = {};
            add_tokens<T, W, kChunk>(token, 0, kChunk, grad, ld, h, sum);
#pragma unroll
            for (int j = 0; j < W; ++j) s.part[c * q.H + h + j] = sum[j];
        }
    }
}

// the tokens [from, to) of a row: those before its first whole chunk and behind its last one by one
template <typename T, int W>
__device__ __forceinline__ void add_row(const Sorted& s, int from, int to, const T* grad, int64_t ld, int64_t H, int64_t h, float* sum) {
    const int c0 = (from + kChunk - 1) / kChunk, c1 = max(c0, to / kChunk);
    add_tokens<T, W, 4>(s.token, from, c0 < c1 ? c0 * kChunk : to, grad, ld, h, sum);
    if (c0 == c1) return;
    for (int c = c0; c < c1; c += 8) {
        Piece<float, (W > 1 ? 4 : 1)> r[8][W > 1 ? W / 4 : 1];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int j = 0; j < (W > 1 ? W / 4 : 1); ++j) r[u][j] = load_piece<float, (W > 1 ? 4 : 1)>(s.part + min(c + u, c1 - 1) * H + h + 4 * j);
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int j = 0; j < W; ++j) sum[j] += c + u < c1 ? r[u][j / 4].v[j % 4] : 0.0f;
    }
    add_tokens<T, W, 4>(s.token, c1 * kChunk, to, grad, ld, h, sum);
}

template <typename T, int W, bool PAST = false>
__device__ __forceinline__ void store_sum(T* to, float scale, const float* sum) {
    Piece<T, W> r;
#pragma unroll
    for (int j = 0; j < W; ++j) put(r.v[j], scale * sum[j]);
    if constexpr (PAST && W > 1) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, r), (u32x4*)to);
    else store_piece<T, W>(to, r);
}

// Rows that have tokens, where the others hold their zeros already: `lanes` threads U sorted tokens after each other, whose gradients are on their way
// together.  A row is finished where its first token is.
template <typename T, int W, int U>
__global__ void __launch_bounds__(256) embedding_grad_kernel(xq_embedding q, Sorted s, const T* grad, int64_t ld, T* dw, int64_t ld_dw, int32_t lanes) {
    const int per = 256 / lanes, lane = threadIdx.x & (lanes - 1);
    const int64_t n = s.start[(int64_t)s.rows << s.log_blocks];
    for (int64_t i0 = ((int64_t)blockIdx.x * per + threadIdx.x / lanes) * U; i0 < n; i0 += (int64_t)gridDim.x * per * U) {
        i32x2 token[U + 2];                                // one before and one behind (ids are not negative: -1 is no row)
        token[0] = i0 > 0 ? s.token[i0 - 1] : i32x2{0, -1};
#pragma unroll
        for (int u = 1; u < U + 2; ++u) token[u] = i0 + u - 1 < n ? s.token[i0 + u - 1] : i32x2{0, -1};
        for (int64_t h = lane * W; h < q.H; h += lanes * W) {
            Piece<T, W> r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) r[u] = load_piece<T, W>(grad + token[u + 1][0] * ld + h);
            float sum[W];
            bool own = false;                              // whether the row's first token is among these
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int id = token[u + 1][1];
                if (id < 0) break;
                if (token[u][1] != id) {
                    own = true;
#pragma unroll
                    for (int j = 0; j < W; ++j) sum[j] = 0.0f;
                }
                if (!own) continue;
#pragma unroll
                for (int j = 0; j < W; ++j) sum[j] += value(r[u].v[j]);
                if (token[u + 2][1] == id && u < U - 1) continue;
                if (token[u + 2][1] == id) {
                    const int end = s.start[(int64_t)(id & ((1 << s.log_blocks) - 1)) * s.rows + (id >> s.log_blocks) + 1];
                    add_row<T, W>(s, (int)i0 + U, end, grad, ld, q.H, h, sum);
                }
                store_sum<T, W>(dw + id * ld_dw + h, q.scale, sum);
            }
        }
    }
}

// All rows: `lanes` threads kSlots of one sorting block after each other, whose tokens' places they look up together.
template <typename T, int W>
__global__ void __launch_bounds__(256) embedding_grad_rows_kernel(xq_embedding q, Sorted s, const T* grad, int64_t ld, T* dw, int64_t ld_dw, int32_t lanes) {
    const int per = 256 / lanes, lane = threadIdx.x & (lanes - 1);
    const int64_t slots = (int64_t)s.rows << s.log_blocks;
    for (int64_t p = ((int64_t)blockIdx.x * per + threadIdx.x / lanes) * kSlots; p < slots; p += (int64_t)gridDim.x * per * kSlots) {
        int32_t at[kSlots + 1];
#pragma unroll
        for (int i = 0; i < kSlots; i += 4) {
            const u32x4 four = *(const u32x4*)(s.start + p + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) at[i + j] = (int32_t)four[j];
        }
        at[kSlots] = s.start[p + kSlots];
        int64_t block = p / s.rows, row = p - block * s.rows;
#pragma unroll
        for (int i = 0; i < kSlots; ++i, ++row) {
            if (row == s.rows) { row = 0; ++block; }
            const int64_t v = (row << s.log_blocks) + block;
            if (v >= q.V) continue;
            for (int64_t h = lane * W; h < q.H; h += lanes * W) {
                float sum[W] = {};
                if (at[i] < at[i + 1]) add_row<T, W>(s, at[i], at[i + 1], grad, ld, q.H, h, sum);
                store_sum<T, W, true>(dw + v * ld_dw + h, q.scale, sum);
            }
        }
    }
}

// Gradients from 256 MiB on (what the memory-side cache holds) whose rows mostly have no token get their zeros first, in the order of addresses beside the sort, at
// 7 TB/s; others are gone through row by row, at 5.  us with forward, zeros first / row by row: 8192 tokens, [131072, 4096] bf16 231 / 287, [65536, 4096] 159 / 172,
// [65536, 2048] 83 / 94, 1000 tokens, [131072, 2048] 100 / 119; below: 4000, [60000, 2048] 71 / 71, 4001, [32003, 2048] fp32 90 / 83.
constexpr int64_t kFillBytes = 256ll << 20;

// the sorting blocks: 256 of them, more where one would own more rows than fit its counters
Sorted plan_of(void* base, int64_t n_tokens, int64_t V, int64_t H, int64_t* bytes) {
    Sorted s = {};
    s.log_blocks = 8;
    while (xq_cdiv(V, 1ll << s.log_blocks) > kSortRows) ++s.log_blocks;
    s.rows = (int32_t)xq_cdiv(V, 1ll << s.log_blocks);
    uint8_t* at = (uint8_t*)base;
    auto take = [&](int64_t n) {
        uint8_t* p = at;
        at += (n + 255) & ~255ll;
        return p;
    };
    s.start = (int32_t*)take((((int64_t)s.rows << s.log_blocks) + 1) * 4);
    s.token = (i32x2*)take(n_tokens * 8);
    s.part = (float*)take(n_tokens / kChunk * H * 4);
    *bytes = at - (uint8_t*)base;
    return s;
}

int32_t lanes_for(int64_t pieces) {
    int32_t n = 8;
    while (n < 256 && n < pieces) n <<= 1;
    return n;
}
bool by_16(const void* p, int64_t ld, int64_t rows, int64_t H, int64_t size) { return xq_aligned(p, 16) && H * size % 16 == 0 && (rows <= 1 || ld * size % 16 == 0); }

// (items of `lanes` threads four at a time where that leaves four blocks and more for every compute unit)
template <typename T, int W>
void launch_fwd(const xq_embedding& q, void* out, int64_t ld_out, hipStream_t st) {
    const int32_t lanes = lanes_for(xq_cdiv(q.H, W));
    const int64_t blocks = xq_cdiv(q.n_tokens, 256 / lanes);
    if (blocks >= 4096) embedding_kernel<T, W, 4><<<dim3((unsigned)std::min<int64_t>(xq_cdiv(blocks, 4), 1 << 20)), 256, 0, st>>>(q, (T*)out, ld_out, lanes);
    else embedding_kernel<T, W, 1><<<dim3((unsigned)blocks), 256, 0, st>>>(q, (T*)out, ld_out, lanes);
}
template <typename T, int W>
void launch_bwd(const xq_embedding& q, const Sorted& s, const void* grad, int64_t ld_grad, void* dw, int64_t ld_dw, hipStream_t st) {
    const int64_t bytes = q.V * q.H * (int64_t)sizeof(T);
    const bool filled = W > 1 && q.n_tokens < q.V / 2 && bytes >= kFillBytes && ld_dw == q.H;
    const unsigned sorts = 1u << s.log_blocks;
    embedding_sort_kernel<<<dim3(sorts + (filled ? (unsigned)std::min<int64_t>(xq_cdiv(bytes, 4096), (1 << 23)) : 0u)), 256, 0, st>>>(q, s, (u32x4*)dw, filled ? bytes / 16 : 0);
    if (q.n_tokens >= kChunk)
        embedding_part_kernel<T, W><<<dim3((unsigned)std::min<int64_t>(q.n_tokens / kChunk, 1 << 16), (unsigned)std::min<int64_t>(xq_cdiv(q.H, 256 * W), 16)), 256, 0, st>>>(
            q, s, (const T*)grad, ld_grad);
    const int32_t lanes = lanes_for(xq_cdiv(q.H, W));
    const int64_t rows = filled ? q.n_tokens : ((int64_t)s.rows << s.log_blocks) / kSlots, blocks = xq_cdiv(rows, 256 / lanes);
    const T* g = (const T*)grad;
    if (!filled) embedding_grad_rows_kernel<T, W><<<dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), 256, 0, st>>>(q, s, g, ld_grad, (T*)dw, ld_dw, lanes);
    else if (blocks >= 4096) embedding_grad_kernel<T, W, 4><<<dim3((unsigned)std::min<int64_t>(xq_cdiv(blocks, 4), 1 << 20)), 256, 0, st>>>(q, s, g, ld_grad, (T*)dw, ld_dw, lanes);
    else if (blocks > 0) embedding_grad_kernel<T, W, 1><<<dim3((unsigned)blocks), 256, 0, st>>>(q, s, g, ld_grad, (T*)dw, ld_dw, lanes);
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
    hipStream_t st = (hipStream_t)stream;
    const int64_t size = q->dtype == XQ_DT_F32 ? 4 : 2;
    const bool wide = by_16(q->weight, q->ldw, q->V, q->H, size) && by_16(out, ld_out, q->n_tokens, q->H, size);
    if (size == 4) wide ? launch_fwd<float, 4>(*q, out, ld_out, st) : launch_fwd<float, 1>(*q, out, ld_out, st);
    else wide ? launch_fwd<bf16_t, 8>(*q, out, ld_out, st) : launch_fwd<bf16_t, 1>(*q, out, ld_out, st);
    XQ_CHECK_LAUNCH("xq_embedding_fwd");
    return XQ_OK;
}

extern "C" int64_t xq_embedding_workspace_bytes(int64_t n_tokens, int64_t V, int64_t H) {
    if (n_tokens < 0 || n_tokens >= (1ll << 31) || V < 1 || V >= (1ll << 31) || H < 1 || H >= (1ll << 31)) return -1;
    int64_t bytes;
    plan_of(nullptr, n_tokens, V, H, &bytes);
    return bytes;
}

extern "C" int xq_embedding_bwd(const xq_embedding* q, const void* grad, int64_t ld_grad, void* dw, int64_t ld_dw, void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = check_embedding("xq_embedding_bwd", q);
    if (rc != XQ_OK) return rc;
    XQ_REQUIRE(q->n_tokens == 0 || rows_ok(grad, q->dtype, q->n_tokens, ld_grad, q->H), "xq_embedding_bwd: the gradient is NULL or misaligned, or its rows overlap");
    XQ_REQUIRE(rows_ok(dw, q->dtype, q->V, ld_dw, q->H), "xq_embedding_bwd: dw is NULL or misaligned, or its rows overlap");
    const int64_t need = xq_embedding_workspace_bytes(q->n_tokens, q->V, q->H);
    XQ_REQUIRE(workspace && xq_aligned(workspace, 256) && workspace_bytes >= need, "xq_embedding_bwd: a workspace of %lld bytes, 256-byte aligned, is needed", (long long)need);
    hipStream_t st = (hipStream_t)stream;
    int64_t bytes;
    const Sorted s = plan_of(workspace, q->n_tokens, q->V, q->H, &bytes);
    const int64_t size = q->dtype == XQ_DT_F32 ? 4 : 2;
    const bool wide = by_16(grad, ld_grad, q->n_tokens, q->H, size) && by_16(dw, ld_dw, q->V, q->H, size);
    if (size == 4) wide ? launch_bwd<float, 4>(*q, s, grad, ld_grad, dw, ld_dw, st) : launch_bwd<float, 1>(*q, s, grad, ld_grad, dw, ld_dw, st);
    else wide ? launch_bwd<bf16_t, 8>(*q, s, grad, ld_grad, dw, ld_dw, st) : launch_bwd<bf16_t, 1>(*q, s, grad, ld_grad, dw, ld_dw, st);
    XQ_CHECK_LAUNCH("xq_embedding_bwd");
    return XQ_OK;
}
