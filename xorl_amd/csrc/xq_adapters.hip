// Adapters of many requests beside one projection:  out = bf16(base + s_a (x A_a^T) B_a^T), a = the row's adapter.
// A row whose id is outside [0, n_adapters) has none: out = base.
#include <algorithm>

#include "xq_common.h"

namespace xq {
namespace {

// Two launches: t = x A_a^T in parts of K, fp32, to the workspace; then out = base + (s t) B_a^T.  Both multiply on 16x16x32 MFMA tiles straight from memory:
// all four operands have the contraction along their rows, so that a lane's eight elements are one 16-byte load.  t goes into the second product as two bf16
// numbers (16 bits: one would lose as much of a large update as the result's own rounding), laid out along the contraction: lanes 0-31 hold the high
// halves of 16 ranks, lanes 32-63 the low ones, and B's 16 ranks stand in both, so that 16 ranks are one MFMA.  fp32 factors are two bf16 numbers in the same way.
// Low halves count where the high halves' sum is finite: an infinity times a low half has any sign or is none (the first product keeps them in sums of their own, the
// second one takes sums that are no numbers again; 0 to 2 % of a call).
//
// What bounds it: few rows, the latency of two launches that each wait for memory two or three times (one row 8.7 us, 48 of 128 adapters 10.2); many, memory: 16384 rows of
// prompts, 12288 by 4096, rank 64, read and write 0.68 GB, 139 us at a copy's rate, and take 176 (down 104 us, up 73).  Between them (2049 rows, 4096 by 12288, fp32 rank 16: 46 us
// against 27) the down launch has too few blocks to keep memory busy (12 us against 4 of bytes), the up launch is within a third of its bytes (30 against 23).
//
// A tile is rows of one adapter.  Up to kLeaderRows rows in any order: a tile belongs to the row that is the first, 17th, 33rd .. of its adapter, and blocks find the
// tiles themselves among the ids (no launch that sorts them).  Up to 64 rows each launch does, and a block has one row to look at; from 65 on the first one leaves its tiles to the
// second, and a block looks at four rows: half of all blocks would do no more than find that their row leads none (1024 rows 81 against 41 us, 64 rows 9.7 against 10.2).  More rows are taken in
// windows of 16 or 64 that follow each other, and a window once for every adapter in it: of prompts' rows, each window has one or two.  By tiles against by windows, 4096 by
// 4096, 8 adapters: rank 16, 256 rows in any order 16 and 49 us, 512 27 and 49, 1024 36 and 54; sorted by adapter 17 and 18, 27 and 18, 39 and 17.  The order is not known when the
// launches are made: at 512 rows tiles take 27 us whatever it is, windows 18 or 49; from 1024 on windows cost rows in any order 1.5 times as much and sorted ones less than half.
constexpr int kLeaderRows = 512;
constexpr int kMostParts = 16, kLeadsNone = -2;

struct AdapterPlan {
    int32_t leaders;      // tiles are found by their first row: how many rows a block looks at, 1 or 4; or 0
    int32_t down_subs, up_subs;      // 16-row pieces of a window: 1 or 4
    int32_t down_tiles, up_tiles;
    int32_t parts;        // of K
    int32_t cols;         // of N a block
};
struct AdapterArgs {
    xq_adapters q;
    AdapterPlan p;
    float* t;             // [parts][M][r_pad]
    int32_t* led;         // (more than 64 rows, tiles by leaders) [M][16]: the rows of a leader's tile, or -1; kLeadsNone in the first place of a row that leads none
    int32_t r_pad;
};

// MFMA instructions are done whatever lanes are active, so that what decides about them has to be one value a wave, and known as that
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// the adapter of a row, or -1
__device__ __forceinline__ int adapter_of(const xq_adapters& q, int64_t row) {
    const int64_t id = q.id_bytes == 8 ? ((const int64_t*)q.ids)[row] : (int64_t)((const int32_t*)q.ids)[row];
    return id >= 0 && id < q.n_adapters ? (int)id : -1;
}

// the rows of a leader's tile, in each wave by itself: lane l gets the row of column l % 16, or -1; false: the row leads no tile
template <int U>
__device__ __forceinline__ bool leader_rows(const xq_adapters& q, int lead, int* id, int* row) {
    const int lane = threadIdx.x & 63, M = (int)q.M;
    const int mine = uniform(adapter_of(q, lead));
    *id = mine;
    int before = 0, seen = 0, want = lane & 15, found = -1;
    for (int c0 = 0; c0 < M; c0 += 64 * U) {
        int ids[U];                                        // (so many loads on their way)
#pragma unroll
        for (int u = 0; u < U; ++u) ids[u] = adapter_of(q, min(c0 + u * 64 + lane, M - 1));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = c0 + u * 64;
            uint64_t same = __ballot(c + lane < M && ids[u] == mine);
            if (lead >= c + 64) { before += __popcll(same); continue; }
            if (lead > c) {
                const uint64_t below = (1ull << (lead - c)) - 1;
                before += __popcll(same & below);
                same &= ~below;
            }
            if (before & 15) return false;
            const int n = __popcll(same);
            if (want >= seen && want < seen + n) {
                uint64_t m = same;
                for (int k = want - seen; k > 0; --k) m &= m - 1;
                found = c + __ffsll((unsigned long long)m) - 1;
            }
            seen += n;
        }
        if (seen >= 16) break;
    }
    *row = found;
    return true;
}

struct Split { bf16x8 hi, lo; };
__device__ __forceinline__ Split split8(const f32x4& a, const f32x4& b) {
    Split s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = i < 4 ? a[i] : b[i - 4];
        s.hi[i] = (__bf16)v;
        s.lo[i] = (__bf16)(v - (float)s.hi[i]);
    }
    return s;
}
__device__ __forceinline__ f32x4 mfma(const bf16x8& a, const bf16x8& b, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// what a factor's eight elements are before they are split
template <bool F32>
struct Raw { f32x4 a, b; };
template <>
struct Raw<false> { bf16x8 a; };
template <bool F32>
__device__ __forceinline__ Raw<F32> load_raw8(const void* p, int64_t at) {
    if constexpr (F32) return {*(const f32x4*)((const float*)p + at), *(const f32x4*)((const float*)p + at + 4)};
    else return {*(const bf16x8*)((const bf16_t*)p + at)};
}
template <bool F32>
__device__ __forceinline__ Split split_raw(const Raw<F32>& r) {
    if constexpr (F32) return split8(r.a, r.b);
    else return {r.a, r.a};
}

// the first n of them, the rest zero, one by one
template <bool F32>
__device__ __forceinline__ Raw<F32> load_raw_n(const void* p, int64_t at, int n) {
    Raw<F32> r = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) {
            if constexpr (F32) {
                if (i < 4) r.a[i & 3] = ((const float*)p)[at + i];
                else r.b[i & 3] = ((const float*)p)[at + i];
            } else {
                r.a[i] = ((const __bf16*)p)[at + i];
            }
        }
    return r;
}

// An MFMA operand has 16 rows in neighbouring lanes; a load that asks for it so touches a cache line a lane.  So rows are loaded whole cache lines at a time, eight
// lanes on each, and the lanes exchange them through LDS, a wave in a place of its own, pieces of 16 bytes exclusive-ored so that neither side
// meets a bank twice.  (16384 rows, K 12288, rank 64, us: operands loaded as they lie 133 down and 106 up, exchanged in pieces of 64 bytes 122, in cache lines 104 and 76)
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
template <int PIECES>
__device__ __forceinline__ int slot(int row, int piece) { return row * PIECES + (piece ^ (row & 7)); }
constexpr int kPlaceKb = 8;           // of a wave

// acc[sub][block of 16 ranks] += x A^T over n units of 64 elements (a cache line of x), four apart, the first `turn` of them last: AHEAD units are on their way
// while the AHEAD before them are multiplied.  (Rows lie a power of two apart, or nearly: tiles that all began with their first unit would ask the same few memory
// channels at the same time.)  x[t][h], a_at[b][h]: the rows that this lane loads; ex: this wave's place
template <int SUBS, int RB, bool F32, int AHEAD>
__device__ __forceinline__ void down_units(const bf16_t* const (&x)[SUBS][2], const void* A, const uint32_t (&a_at)[RB][F32 ? 4 : 2], int first, int n, int turn, u32x4* ex,
                                           f32x4 (&acc)[SUBS][RB]) {
    f32x4 low[F32 ? SUBS : 1][F32 ? RB : 1] = {};          // of A's low halves
    constexpr int FL = F32 ? 4 : 2, AP = F32 ? 16 : 8;    // loads, and pieces a row, of 16 rows of a factor
    constexpr int GROUP = kPlaceKb / FL;                   // blocks of ranks that the place holds
    const int lane = threadIdx.x & 63, col = lane & 15, group = lane >> 4;
    u32x4 xv[AHEAD][SUBS][2], av[AHEAD][RB][FL];
    auto unit = [&](int i) {
        const int at = i + turn;
        return (first + 4 * (at < n ? at : at - n)) * 64;
    };
    auto load_x = [&](int from) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (from + u >= n) break;
            const int64_t k = unit(from + u);
#pragma unroll
            for (int t = 0; t < SUBS; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) xv[u][t][h] = *(const u32x4*)(x[t][h] + k);
        }
    };
    auto load_a = [&](int from) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (from + u >= n) break;
            const char* base = (const char*)A + (int64_t)unit(from + u) * (F32 ? 4 : 2);
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int h = 0; h < FL; ++h) av[u][b][h] = *(const u32x4*)(base + a_at[b][h]);
        }
    };
    load_x(0);
    load_a(0);
    for (int i = 0; i < n; i += AHEAD) {
        bf16x8 xo[AHEAD][SUBS][2];
        wave_fence();                                      // (what was exchanged before has been read)
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int t = 0; t < SUBS; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) ex[(u * SUBS + t) * 128 + slot<8>(h * 8 + (lane >> 3), lane & 7)] = xv[u][t][h];
        wave_fence();
        load_x(i + AHEAD);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int t = 0; t < SUBS; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) xo[u][t][h] = __builtin_bit_cast(bf16x8, ex[(u * SUBS + t) * 128 + slot<8>(col, h * 4 + group)]);
#pragma unroll
        for (int b0 = 0; b0 < AHEAD * RB; b0 += GROUP) {
            wave_fence();
#pragma unroll
            for (int g = 0; g < GROUP; ++g)
                if (b0 + g < AHEAD * RB)
#pragma unroll
                    for (int h = 0; h < FL; ++h)
                        ex[g * AP * 16 + slot<AP>(F32 ? h * 4 + (lane >> 4) : h * 8 + (lane >> 3), lane & (AP - 1))] = av[(b0 + g) / RB][(b0 + g) % RB][h];
            wave_fence();
            if (b0 + GROUP >= AHEAD * RB) load_a(i + AHEAD);
#pragma unroll
            for (int g = 0; g < GROUP; ++g) {
                const int u = (b0 + g) / RB, b = (b0 + g) % RB;
                if (b0 + g >= AHEAD * RB || i + u >= n) break;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    Split s;
                    const u32x4* from = ex + g * AP * 16;
                    if constexpr (F32) s = split8(__builtin_bit_cast(f32x4, from[slot<AP>(col, h * 8 + group * 2)]), __builtin_bit_cast(f32x4, from[slot<AP>(col, h * 8 + group * 2 + 1)]));
                    else s.hi = __builtin_bit_cast(bf16x8, from[slot<AP>(col, h * 4 + group)]);
#pragma unroll
                    for (int t = 0; t < SUBS; ++t) {
                        acc[t][b] = mfma(s.hi, xo[u][t][h], acc[t][b]);
                        if constexpr (F32) low[t][b] = mfma(s.lo, xo[u][t][h], low[t][b]);
                    }
                }
            }
        }
    }
    // (where the high halves' sum is infinite or none, it is the sum: an infinity times a low half has any sign, or is no number)
    if constexpr (F32)
#pragma unroll
        for (int t = 0; t < SUBS; ++t)
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][b][i] += fabsf(acc[t][b][i]) < INFINITY ? low[t][b][i] : 0.0f;
}
// units on their way: up to four of x in a wave's place, and 16 loads of factors
constexpr int ahead_for(int subs, int rb, bool f32) { return subs == 4 ? 1 : std::min(4, std::max(1, 16 / (rb * (f32 ? 8 : 4)))); }

// one adapter's part of t for SUBS pieces of 16 rows: row[t] is the row of this lane's column in piece t, or -1
template <int SUBS, int RB, bool F32>
__device__ __forceinline__ void down_tile(const AdapterArgs& a, int id, const int (&row)[SUBS], int part, int turn, float* red) {
    constexpr int FL = F32 ? 4 : 2;
    const xq_adapters& q = a.q;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), group = lane >> 4;
    // this part's units, the four waves side by side: this wave's are first, first + 4 ..
    const int units = (int)(q.K / 64), begin = (int)((int64_t)units * part / a.p.parts), end = (int)((int64_t)units * (part + 1) / a.p.parts);
    const int first = begin + wave, n = (end - first + 3) >> 2;
    const bf16_t* x[SUBS][2];
    uint32_t a_at[RB][FL];                                 // (an adapter's A is below 4 GiB)
#pragma unroll
    for (int t = 0; t < SUBS; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) x[t][h] = (const bf16_t*)q.x + (int64_t)max(__shfl(row[t], h * 8 + (lane >> 3), 64), 0) * q.ldx + (lane & 7) * 8;
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int h = 0; h < FL; ++h)
            a_at[b][h] = (uint32_t)min(b * 16 + (F32 ? h * 4 + (lane >> 4) : h * 8 + (lane >> 3)), q.r - 1) * (uint32_t)q.K * (F32 ? 4 : 2) + (lane & (F32 ? 15 : 7)) * 16;
    f32x4 acc[SUBS][RB] = {};
    __syncthreads();                                       // (what the tile before left in red has been read)
    const char* A = (const char*)q.A + (int64_t)id * q.r * q.K * (F32 ? 4 : 2);
    down_units<SUBS, RB, F32, ahead_for(SUBS, RB, F32)>(x, A, a_at, first, n, n > 0 ? (int)((uint32_t)turn * 5 % n) : 0, (u32x4*)red + wave * kPlaceKb * 64, acc);
    // the four waves' sums: lane's four ranks of its column
    __syncthreads();
#pragma unroll
    for (int half = 2; half; half >>= 1) {
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int t = 0; t < SUBS; ++t)
#pragma unroll
                for (int b = 0; b < RB; ++b) *(f32x4*)(red + (((wave - half) * SUBS + t) * RB + b) * 256 + lane * 4) = acc[t][b];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int t = 0; t < SUBS; ++t)
#pragma unroll
                for (int b = 0; b < RB; ++b) acc[t][b] += *(const f32x4*)(red + ((wave * SUBS + t) * RB + b) * 256 + lane * 4);
        __syncthreads();
    }
    if (wave == 0)
#pragma unroll
        for (int t = 0; t < SUBS; ++t)
            if (row[t] >= 0)
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    f32x4 v = acc[t][b];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = b * 16 + group * 4 + i < q.r ? v[i] : 0.0f;
                    *(f32x4*)(a.t + ((int64_t)part * q.M + row[t]) * a.r_pad + b * 16 + group * 4) = v;
                }
}

// Blocks go to the eight XCDs in turn: neighbouring items, which are of one adapter as a rule, go to one of them, so that each reads few adapters through its L2
// (4096 by 4096, us so and in the order of launch: 1024 rows of 128 an adapter, rank 16 12.9 and 13.7, 4096 of 512, rank 32 30.7 and 32.0, 16384 of 2048, rank 64 in fp32 179 and
// 181, rank 16 in fp32 103 and 101; 12288 by 4096, 16384 rows, rank 64 the same; 4096 by 12288, 2049 rows in fp32, rank 16 40.5 and 39.2, rank 64 132 and 119)
__device__ __forceinline__ int64_t item_of(int64_t at, int64_t n) {
    const int64_t each = n / 8, rest = n - each * 8, xcd = at & 7, i = at >> 3;
    return xcd * each + min(xcd, rest) + i;
}

template <int SUBS, int RB, bool F32>
__global__ void __launch_bounds__(256) adapter_down_kernel(AdapterArgs a) {
    __shared__ __attribute__((aligned(16))) float red[4 * kPlaceKb * 256];       // (and the waves' sums: at most 2 * SUBS * RB KB)
    static_assert(2 * SUBS * RB <= 4 * kPlaceKb, "");
    __shared__ int found[4][16];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int64_t items = (int64_t)a.p.down_tiles * a.p.parts;
    for (int64_t b = blockIdx.x; b < items; b += gridDim.x) {
        const int64_t at = a.p.leaders ? b : item_of(b, items);
        const int tile = (int)(at / a.p.parts), part = (int)(at - (int64_t)tile * a.p.parts);
        if (a.p.leaders) {
            int id, row = -1;
            if (a.p.leaders == 1) {                        // (at most 64 rows: one look at them, by each wave for itself)
                const bool leads = leader_rows<1>(a.q, tile, &id, &row);
                const int one[1] = {row};
                if (leads && id >= 0) down_tile<1, RB, F32>(a, id, one, part, tile, red);
                continue;
            }
            // each wave looks at a row, and the block does the tiles of those that lead one after the other
            const int lead = tile + wave * a.p.down_tiles;
            const bool leads = lead < a.q.M && leader_rows<4>(a.q, lead, &id, &row);
            __syncthreads();                               // (the rows before have been read)
            if (lane < 16) {
                found[wave][lane] = leads ? row : kLeadsNone;
                if (part == 0 && lead < a.q.M) a.led[lead * 16 + lane] = leads ? row : kLeadsNone;
            }
            __syncthreads();
            for (int j = 0; j < 4; ++j) {
                const int one[1] = {found[j][lane & 15]}, of = uniform(one[0]);
                if (of == kLeadsNone) continue;
                id = uniform(adapter_of(a.q, of));
                if (id >= 0) down_tile<1, RB, F32>(a, id, one, part, tile + j * a.p.down_tiles, red);
            }
            continue;
        }
        // a window of SUBS * 16 rows: once for every adapter in it
        const int64_t row0 = (int64_t)tile * (SUBS * 16);
        const int own = lane < SUBS * 16 && row0 + lane < a.q.M ? adapter_of(a.q, row0 + lane) : -1;
        uint64_t left = __ballot(own >= 0);
        while (left) {
            const int id = __builtin_amdgcn_readlane(own, __ffsll((unsigned long long)left) - 1);
            const uint64_t same = __ballot(own == id) & left;
            left &= ~same;
            int row[SUBS], pieces = 0;
#pragma unroll
            for (int t = 0; t < SUBS; ++t) {
                pieces += (same >> (t * 16) & 0xffff) != 0;
                row[t] = same >> (t * 16 + (lane & 15)) & 1 ? (int)row0 + t * 16 + (lane & 15) : -1;
            }
            if (SUBS == 1 || pieces > 2) {
                down_tile<SUBS, RB, F32>(a, id, row, part, tile, red);
            } else {
#pragma unroll
                for (int t = 0; t < SUBS; ++t) {
                    const int one[1] = {row[t]};
                    if (same >> (t * 16) & 0xffff) down_tile<1, RB, F32>(a, id, one, part, tile, red);
                }
            }
        }
    }
}

// s t of SUBS pieces of 16 rows as MFMA operands, to LDS: [piece][block of 16 ranks][lane]
template <int SUBS, int RB>
__device__ __forceinline__ void up_operands(const AdapterArgs& a, float scale, const int (&row)[SUBS], bf16x8* ts) {
    constexpr int AT_ONCE = SUBS > 1 ? 4 : 8;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4;
#pragma unroll
    for (int t = 0; t < SUBS; ++t)
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            if (((t * RB + b) & 3) != wave) continue;
            f32x4 v0 = {}, v1 = {};
            if (row[t] >= 0) {
                const float* from = a.t + (int64_t)row[t] * a.r_pad + b * 16 + (group & 1) * 8;
                for (int p0 = 0; p0 < a.p.parts; p0 += AT_ONCE) {
                    f32x4 r[AT_ONCE][2];
#pragma unroll
                    for (int p = 0; p < AT_ONCE; ++p)
                        if (p0 + p < a.p.parts) {
                            r[p][0] = *(const f32x4*)(from + (int64_t)(p0 + p) * a.q.M * a.r_pad);
                            r[p][1] = *(const f32x4*)(from + (int64_t)(p0 + p) * a.q.M * a.r_pad + 4);
                        }
#pragma unroll
                    for (int p = 0; p < AT_ONCE; ++p)
                        if (p0 + p < a.p.parts) {
                            v0 += r[p][0];
                            v1 += r[p][1];
                        }
                }
            }
            const Split s = split8(v0 * scale, v1 * scale);
            ts[(t * RB + b) * 64 + lane] = group < 2 ? s.hi : s.lo;
        }
}

__device__ __forceinline__ bool has_nan(const f32x4 (&v)[2]) {
    bool is = false;
#pragma unroll
    for (int j = 0; j < 2; ++j) is |= __builtin_isunordered(v[j][0], v[j][1]) || __builtin_isunordered(v[j][2], v[j][3]);
    return is;
}
// Sums that are no numbers again, of the high halves alone: an infinity in t or B times a low half has any sign, or is none where the sum of the whole
// numbers is infinite.  factor(j, b): B's operand, as high halves
template <int RB, typename F>
__device__ __forceinline__ void sums_again(const bf16x8* ts, F factor, f32x4 (&acc)[2]) {
    const int lane = threadIdx.x & 63;
    f32x4 lead[2] = {};
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const bf16x8 tv = lane < 32 ? ts[b * 64 + lane] : bf16x8{};
#pragma unroll
        for (int j = 0; j < 2; ++j) lead[j] = mfma(lane < 32 ? factor(j, b) : bf16x8{}, tv, lead[j]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = acc[j][i] != acc[j][i] ? lead[j][i] : acc[j][i];
}

// eight columns of a row: base and the sums, rounded
__device__ __forceinline__ u32x4 add8(u32x4 base, const f32x4& lo, const f32x4& hi) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x4& d = i < 2 ? lo : hi;
        base[i] = pack_bf16x2(bf16_to_f32((bf16_t)base[i]) + d[(i & 1) * 2], bf16_to_f32((bf16_t)(base[i] >> 16)) + d[(i & 1) * 2 + 1]);
    }
    return base;
}
// B's row among 32 that this lane has as the operand of the j-th of two tiles: so that a lane's eight sums are of neighbouring columns
__device__ __forceinline__ int b_row(int col, int j) { return (col >> 2) * 8 + j * 4 + (col & 3); }

// out of 16 rows of one adapter, columns [n0, n1), a wave 32 at a time, loaded and stored as the operands lie: such blocks have no more than a few loads, and wait for
// them and not for the cache.  WHOLE: ranks in pieces of eight, at multiples of 16 bytes
template <int RB, bool F32, bool WHOLE>
__device__ __forceinline__ void up_piece(const AdapterArgs& a, int id, int row, int64_t n0, int64_t n1, bf16x8* ts) {
    const xq_adapters& q = a.q;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, group = lane >> 4;
    if (id < 0 && q.out == q.base && q.ld_out == q.ld_base) return;
    Raw<F32> bv[2][RB];
    u32x4 base;
    auto load = [&](int64_t n) {
        if (id >= 0)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t at = ((int64_t)id * q.N + min(n + b_row(col, j), q.N - 1)) * q.r;
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    const int k = b * 16 + (group & 1) * 8;
                    if (!WHOLE) bv[j][b] = load_raw_n<F32>(q.B, at + k, min(q.r - k, 8));
                    else if (b + 1 < RB || k < q.r) bv[j][b] = load_raw8<F32>(q.B, at + k);
                    else bv[j][b] = {};
                }
            }
        base = *(const u32x4*)((const bf16_t*)q.base + (int64_t)max(row, 0) * q.ld_base + min(n + group * 8, q.N - 8));
    };
    const int64_t from = n0 + wave * 32;                   // (the four waves side by side: 256 bytes of a row)
    load(from);
    if (id >= 0) {
        const int rows[1] = {row};
        __syncthreads();                                   // (what the tile before left in ts has been read)
        up_operands<1, RB>(a, q.scaling[id], rows, ts);
        __syncthreads();
    }
    for (int64_t n = from; n < n1; n += 128) {
        u32x4 out = base;
        if (id >= 0) {
            f32x4 acc[2] = {};
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const bf16x8 tv = ts[b * 64 + lane];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const Split s = split_raw<F32>(bv[j][b]);
                    acc[j] = mfma(s.hi, tv, acc[j]);
                    if (F32) acc[j] = mfma(s.lo, tv, acc[j]);
                }
            }
            if (__ballot(has_nan(acc))) sums_again<RB>(ts, [&](int j, int b) { return split_raw<F32>(bv[j][b]).hi; }, acc);
            out = add8(base, acc[0], acc[1]);
        }
        const int64_t mine = n + group * 8;
        if (n + 128 < n1) load(n + 128);
        if (row >= 0 && mine < n1) *(u32x4*)((bf16_t*)q.out + (int64_t)row * q.ld_out + mine) = out;
    }
}

// Where the eight ranks kc of B's row nl (of 32) lie after their exchange, m such pieces a row: exclusive-ored where m is a power of two
__device__ __forceinline__ int b_slot(int nl, int kc, int m) {
    const int f = m == 8 ? (nl & 3) | (nl >> 3 & 1) << 2 : m == 4 ? (nl >> 1 & 1) | (nl >> 3 & 1) << 1 : m == 2 ? nl >> 3 & 1 : 0;
    return nl * m + (kc ^ f);
}

// the same for four pieces, those in `pieces`, ranks in pieces of eight: B's rows, and the sums of each piece, exchange their lanes in ex, this wave's place
template <int RB, bool F32>
__device__ __forceinline__ void up_window(const AdapterArgs& a, int id, const int (&row)[4], int pieces, int64_t n0, int64_t n1, bf16x8* ts, u32x4* ex) {
    constexpr int FR = F32 ? 2 : 1, BP = RB * FR;         // KB of B's 32 rows
    const xq_adapters& q = a.q;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, group = lane >> 4;
    if (id < 0 && q.out == q.base && q.ld_out == q.ld_base) return;
    const int m = q.r / 8;
    // loads and stores: four lanes a row, eight columns each
    int own[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) own[t] = __shfl(row[t], lane >> 2, 64);
    u32x4 base[2][4], braw[BP];
    int put[BP];                                           // where this lane's pieces of B go
#pragma unroll
    for (int i = 0; i < BP; ++i) {
        const int piece = (i * 64 + lane) / FR, nl = piece / m;
        put[i] = nl < 32 ? b_slot(nl, piece - nl * m, m) * FR + (F32 ? lane & 1 : 0) : -1;
    }
    auto load = [&](int buf, int64_t n) {
        n = min(n, q.N - 16);
        if (id >= 0) {
            const int64_t size = F32 ? 4 : 2, last = min(q.N - n, (int64_t)32) * q.r * size - 16;
            const char* from = (const char*)q.B + ((int64_t)id * q.N + n) * q.r * size;
#pragma unroll
            for (int i = 0; i < BP; ++i) braw[i] = *(const u32x4*)(from + min((int64_t)(i * 64 + lane) * 16, last));
        }
        const int64_t mine = min(n + (lane & 3) * 8, q.N - 8);
#pragma unroll
        for (int t = 0; t < 4; ++t) base[buf][t] = *(const u32x4*)((const bf16_t*)q.base + (int64_t)max(own[t], 0) * q.ld_base + mine);
    };
    auto finish = [&](int buf, int64_t n) {
        Split sv[2][RB];
        if (id >= 0) {
            wave_fence();                                  // (what was exchanged before has been read)
#pragma unroll
            for (int i = 0; i < BP; ++i)
                if (put[i] >= 0) ex[put[i]] = braw[i];
            wave_fence();
        }
        load(buf ^ 1, n + 128);
        if (id >= 0)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    const int kc = b * 2 + (group & 1);
                    Raw<F32> r = {};
                    if (kc < m) {
                        const u32x4* from = ex + b_slot(b_row(col, j), kc, m) * FR;
                        r.a = __builtin_bit_cast(decltype(r.a), from[0]);
                        if constexpr (F32) r.b = __builtin_bit_cast(f32x4, from[1]);
                    }
                    sv[j][b] = split_raw<F32>(r);
                }
        const int64_t mine = n + (lane & 3) * 8;
        u32x4* sums = ex + BP * 64;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (!(pieces >> t & 1)) continue;
            u32x4 out = base[buf][t];
            if (id >= 0) {
                f32x4 acc[2] = {};
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    const bf16x8 tv = ts[(t * RB + b) * 64 + lane];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        acc[j] = mfma(sv[j][b].hi, tv, acc[j]);
                        if (F32) acc[j] = mfma(sv[j][b].lo, tv, acc[j]);
                    }
                }
                if (__ballot(has_nan(acc))) sums_again<RB>(ts + t * RB * 64, [&](int j, int b) { return sv[j][b].hi; }, acc);
                wave_fence();
#pragma unroll
                for (int j = 0; j < 2; ++j) sums[slot<8>(col, group * 2 + j)] = __builtin_bit_cast(u32x4, acc[j]);
                wave_fence();
                const u32x4 lo = sums[slot<8>(lane >> 2, (lane & 3) * 2)], hi = sums[slot<8>(lane >> 2, (lane & 3) * 2 + 1)];
                out = add8(out, __builtin_bit_cast(f32x4, lo), __builtin_bit_cast(f32x4, hi));
            }
            if (own[t] >= 0 && mine < n1) *(u32x4*)((bf16_t*)q.out + (int64_t)own[t] * q.ld_out + mine) = out;
        }
    };
    const int64_t from = n0 + wave * 32;                   // (the four waves side by side: 256 bytes of a row)
    load(0, from);
    if (id >= 0) {
        __syncthreads();                                   // (what the tile before left in ts has been read)
        up_operands<4, RB>(a, q.scaling[id], row, ts);
        __syncthreads();
    }
    for (int64_t n = from; n < n1; n += 256) {
        finish(0, n);
        if (n + 128 < n1) finish(1, n + 128);
    }
}

// LEADERS: tiles of rows in any order; otherwise windows of 16 rows, or with SUBS 4 of 64
template <int SUBS, int RB, bool F32, bool WHOLE>
__global__ void __launch_bounds__(256) adapter_up_kernel(AdapterArgs a) {
    constexpr int kb = SUBS > 1 ? RB * (F32 ? 2 : 1) + 2 : 0;
    __shared__ bf16x8 ts[SUBS * RB * 64];
    __shared__ u32x4 exchange[4 * kb * 64 + 1];           // (SUBS 1 has no use for it, and an array no zero elements)
    const int lane = threadIdx.x & 63;
    const int64_t chunks = (a.q.N + a.p.cols - 1) / a.p.cols, items = a.p.up_tiles * chunks;
    for (int64_t b = blockIdx.x; b < items; b += gridDim.x) {
        const int64_t at = a.p.leaders ? b : item_of(b, items);
        const int tile = (int)(at / chunks);
        const int64_t n0 = (at - tile * chunks) * a.p.cols, n1 = min(n0 + a.p.cols, a.q.N);
        if (SUBS == 1 && a.p.leaders) {
            for (int lead = tile; lead < a.q.M; lead += a.p.up_tiles) {
                int id, row;
                if (a.p.leaders == 1) {                    // (one look at the ids, which are in the cache, is shorter than reading what was just written: 48 rows 10.2 against 10.5 us)
                    if (!leader_rows<1>(a.q, lead, &id, &row)) continue;
                } else {
                    row = a.led[lead * 16 + (lane & 15)];
                    id = uniform(adapter_of(a.q, lead));
                    if (uniform(row) == kLeadsNone) continue;
                }
                up_piece<RB, F32, WHOLE>(a, id, row, n0, n1, ts);
            }
            continue;
        }
        const int64_t row0 = (int64_t)tile * (SUBS * 16);
        const bool real = lane < SUBS * 16 && row0 + lane < a.q.M;
        const int own = real ? adapter_of(a.q, row0 + lane) : -1;
        uint64_t left = __ballot(real);
        while (left) {
            const int id = __builtin_amdgcn_readlane(own, __ffsll((unsigned long long)left) - 1);
            const uint64_t same = __ballot(own == id) & left;
            left &= ~same;
            int row[SUBS], pieces = 0;
#pragma unroll
            for (int t = 0; t < SUBS; ++t) {
                pieces |= ((same >> (t * 16) & 0xffff) != 0) << t;
                row[t] = same >> (t * 16 + (lane & 15)) & 1 ? (int)row0 + t * 16 + (lane & 15) : -1;
            }
            if constexpr (SUBS == 4) up_window<RB, F32>(a, id, row, pieces, n0, n1, ts, exchange + (threadIdx.x >> 6) * kb * 64);
            else up_piece<RB, F32, WHOLE>(a, id, row[0], n0, n1, ts);
        }
    }
}

AdapterPlan plan_adapters(int64_t M, int64_t N, int64_t K, int r) {
    AdapterPlan p;
    p.leaders = M > kLeaderRows ? 0 : M > 64 ? 4 : 1;
    // (rank 16 and 64, rows sorted by adapter, 16 against 64 rows: 4096 rows 28 and 48 against 34 and 67 us, 16384 109 and 140 against 110 and 132; in any order 330 and 603 against 288 and 460)
    p.down_subs = p.leaders || M < 8192 ? 1 : 4;
    // (2049 rows, 12288 columns, rank 16 in fp32: windows of 64 rows 29 us, of 16 41; ranks that are no multiple of 8 are read one by one, 16 rows at a time)
    p.up_subs = p.leaders || r % 8 != 0 ? 1 : 4;
    // (a block's rows lie apart by an odd number: those that lead are often the first ones, or every 16th)
    const int64_t led = p.leaders > 1 ? xq_cdiv(M, p.leaders) | 1 : M;
    p.down_tiles = (int32_t)(p.leaders ? led : xq_cdiv(M, p.down_subs * 16));
    p.up_tiles = (int32_t)(p.leaders ? led : xq_cdiv(M, p.up_subs * 16));
    // parts that bring two blocks to every compute unit where the tiles do not, of at least two cache lines of x a wave
    const int64_t full = xq_cdiv(M, p.down_subs * 16), units = K / 64;
    p.parts = (int32_t)std::max<int64_t>(1, std::min<int64_t>({512 / std::max<int64_t>(full, 1), units / 8, kMostParts}));
    // columns of a block: fewer blocks repeat the reading of t and its roundings less, as long as there are four of them a compute unit (the same, of 128, 256 and 512 columns: 34.5, 29.1
    // and 31.2 us; 1024 rows in any order, tiles of 16, rank 16 and 64: of 128 45 and 70, of 256 36 and 59)
    p.cols = p.leaders ? (xq_cdiv(M, 16) * xq_cdiv(N, 256) >= 1024 ? 256 : 128) : p.up_tiles * xq_cdiv(N, 1024) >= 1024 ? 1024 : p.up_tiles * xq_cdiv(N, 512) >= 1024 ? 512 : 256;
    return p;
}
int r_pad(int r) { return (r + 15) / 16 * 16; }

template <int RB, bool F32>
void launch_adapters(const AdapterArgs& a, hipStream_t st) {
    const int64_t most = (1 << 24) - 1;
    const dim3 down((unsigned)std::min((int64_t)a.p.down_tiles * a.p.parts, most)), up((unsigned)std::min(a.p.up_tiles * xq_cdiv(a.q.N, a.p.cols), most));
    if (a.p.down_subs == 1) adapter_down_kernel<1, RB, F32><<<down, 256, 0, st>>>(a);
    else adapter_down_kernel<4, RB, F32><<<down, 256, 0, st>>>(a);
    if (a.p.up_subs == 4) adapter_up_kernel<4, RB, F32, true><<<up, 256, 0, st>>>(a);
    else if (a.q.r % 8 == 0) adapter_up_kernel<1, RB, F32, true><<<up, 256, 0, st>>>(a);
    else adapter_up_kernel<1, RB, F32, false><<<up, 256, 0, st>>>(a);
}
template <bool F32>
void launch_adapters(const AdapterArgs& a, hipStream_t st) {
    switch (a.r_pad / 16) {
        case 1: return launch_adapters<1, F32>(a, st);
        case 2: return launch_adapters<2, F32>(a, st);
        case 3: return launch_adapters<3, F32>(a, st);
        default: return launch_adapters<4, F32>(a, st);
    }
}

bool sizes_fit(int64_t M, int64_t N, int64_t K, int r) {
    return M >= 0 && M < (1 << 24) && N >= 16 && N < (1 << 24) && N % 16 == 0 && K >= 64 && K < (1 << 23) && K % 64 == 0 && r >= 1 && r <= 64;
}

}  // namespace
}  // namespace xq

using namespace xq;

extern "C" int64_t xq_adapters_workspace_bytes(int64_t M, int64_t N, int64_t K, int r) {
    if (!sizes_fit(M, N, K, r)) return -1;
    const AdapterPlan p = plan_adapters(M, N, K, r);
    return std::max<int64_t>((int64_t)p.parts * M * r_pad(r) * 4 + (p.leaders > 1 ? M * 64 : 0), 256);
}

extern "C" int xq_adapters_add(const xq_adapters* q, void* workspace, int64_t workspace_bytes, void* stream) {
    XQ_REQUIRE(q, "xq_adapters_add: the problem is NULL");
    XQ_REQUIRE(sizes_fit(q->M, q->N, q->K, q->r), "xq_adapters_add: %lld rows, [%lld, %lld], rank %d: in_features must be a multiple of 64 below 2^23, out_features of 16 below 2^24, the rows below 2^24, the rank 1 to 64",
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
    AdapterArgs a = {*q, plan_adapters(q->M, q->N, q->K, q->r), (float*)workspace, nullptr, r_pad(q->r)};
    a.led = (int32_t*)(a.t + (int64_t)a.p.parts * q->M * a.r_pad);
    q->factor_dtype == XQ_DT_F32 ? launch_adapters<true>(a, st) : launch_adapters<false>(a, st);
    XQ_CHECK_LAUNCH("xq_adapters_add");
    return XQ_OK;
}
