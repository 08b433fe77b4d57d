// Embedding lookup with scaling and its gradient, for gfx950.
//   out[n] = scale * table[ids[n]]              dtable[v] = scale * sum_{n: ids[n] = v} dout[n]  (+ dtable[v])
// A negative id is a place without a token: its row is zero and it has no gradient.  An id >= V is treated so too and
// reported through the status word.
//
// Lookup: bound by memory.  A thread moves 8 neighbouring columns of four rows, the four ids fetched together, then the four
// pieces of the table, then the stores.  65 536 tokens of 512 columns in bf16: 17.0 us (at best 14.5), 67 MB of rows written at 4.0
// TB/s (the table, 19 MB, comes from the caches); 128 tokens of 128: 3.0 us.
//
// Gradient: the tokens are put in the order of their ids (a stable radix sort of 8 bits a pass), and the sorted list is cut
// into chunks of equal length, whatever the ids: a row that half of the tokens read costs the sums no more than as many different
// rows (its parts, one a chunk, are joined by one workgroup for 256 columns: 65 536 tokens of 512 columns that all, or every
// second one of them, read one row, join in 16 to 26 us instead of 8.2).
// A team of lanes walks a chunk, holding one row's sum in registers; a row that lies inside the chunk is written at once, one
// that crosses its ends leaves partial sums, which a last launch joins in order.  Rows that no token reads are zeroed beside
// the chunks: the sort marks those that have one (looking them up in the sorted list, fifteen dependent loads, held the
// launch up: 22 983 tokens over 38 569 rows of 43 columns 16.2 us, 7.2 with marks and a team a row; up to 4096 tokens over more
// than 2^18 rows they are looked up all the same).  The order of every sum is fixed by the ids alone: no atomics, the same bits on every call.
// Few tokens (128) and few table rows (8: conditions) need no order and take one and two launches (below).
// Up to 4096 tokens are sorted by one workgroup in LDS, in one launch (over 19 000 rows of 512: 4096 tokens 30.0 us, 4097 in
// four launches 32.6; 8192 in one 38.5, in four 33.5).  Beyond, a pass is one launch in which every workgroup forms its own
// offsets from the digit counts of all tiles (no scan launch), which a launch before it has made.  (Counts of the
// next digit added up by the pass before, with atomics where the tokens land: 17 us a pass instead of 2.5 + 6, frequent ids
// meet in one counter.)
// 65 536 tokens over 19 000 rows of 512 columns in bf16, 48.5-49 us: two passes of count 3.0 and sort 6.4, sums 21.0 (106 MB, 5.0
// TB/s: a large copy's rate), joins 8.2, and what the starts of six launches leave between them.
#include <algorithm>

#include "vec8.h"

namespace c2 {
namespace embed {

constexpr int kSortOne = 4096;  // tokens that one workgroup sorts
constexpr int kBins = 256;

// ------------------------------------------------------------------------------------------------ lookup
template <typename T, typename TO, typename TI, bool EL>  // EL: rows shorter than eight columns
__global__ __launch_bounds__(256) void lookup_kernel(const T* __restrict__ table, int64_t ldt, int64_t V,
                                                     const TI* __restrict__ ids, unsigned count, unsigned dg, int64_t D,
                                                     float scale, TO* __restrict__ out, int64_t ldo, int32_t* status) {
    const unsigned stride = gridDim.x * 256;
    const unsigned i0 = blockIdx.x * 256 + threadIdx.x;
    unsigned n[4], g[4];
    int64_t id[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const unsigned i = i0 + u * stride;
        n[u] = i / dg;
        g[u] = i - n[u] * dg;
        id[u] = i < count ? (int64_t)ids[n[u]] : -1;
    }
    Raw8<T> x[4];
    float v[4][8];
    int64_t c[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        if (id[u] >= V) {
            if (status) *status = 1;
            id[u] = -1;
        }
        c[u] = min((int64_t)g[u] * 8, D - 8);  // a row's last, partial piece: its last eight columns
        if (id[u] >= 0) {
            if (EL) load_short(table + id[u] * ldt, D, v[u]);
            else x[u] = raw8(table + id[u] * ldt + c[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        if (i0 + u * stride >= count) continue;
        if (id[u] >= 0) {
            if (!EL) unraw8(x[u], v[u]);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[u][j] *= scale;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[u][j] = 0.f;
        }
        if (EL) store_row8(out + (int64_t)n[u] * ldo, 0, D, v[u]);
        else store8(out + (int64_t)n[u] * ldo + c[u], v[u]);
    }
}

// ------------------------------------------------------------------------------------------------ sort
// A token's key: its id, or V where it has none (sorted behind all rows).
__device__ __forceinline__ int key_of(int64_t i, int64_t V, int32_t* status) {
    if (i >= V && status) *status = 1;
    return (int)(i >= 0 && i < V ? i : V);
}

// Lanes of this wave whose digit equals this lane's, among the active ones.
__device__ __forceinline__ uint64_t same_digit(int digit, int bits, uint64_t active) {
    uint64_t peers = active;
    for (int b = 0; b < bits; ++b) {
        const uint64_t m = __ballot((digit >> b) & 1);
        peers &= ((digit >> b) & 1) ? m : ~m;
    }
    return peers;
}

// Stable ranks of a workgroup's items, 16 waves of ITEMS * 64 consecutive items each (item u of lane l: 64 u + l): on return
// rank[u] is the item's place among the wave's items of its digit, and hist[w][d] the wave's count.  hist zeroed by the caller.
template <int ITEMS>
__device__ __forceinline__ void wave_ranks(const int (&digit)[ITEMS], const bool (&on)[ITEMS], int bits, volatile int* hist,
                                           int (&rank)[ITEMS]) {
    const int lane = threadIdx.x & 63;
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
        const uint64_t act = __ballot(on[u]);
        if (act == 0) break;
        const uint64_t peers = same_digit(digit[u], bits, act);
        int base = 0;
        if (on[u]) base = hist[digit[u]];
        __builtin_amdgcn_wave_barrier();
        rank[u] = base + __popcll(peers & below);
        if (on[u] && (peers & below) == 0) hist[digit[u]] = base + __popcll(peers);  // the first of its digit
        __builtin_amdgcn_wave_barrier();
    }
}

// Exclusive prefix of 256 values held by the first four waves (thread t: value t); part: 4 ints in LDS.  All threads call it.
__device__ __forceinline__ int prefix_256(int v, int* part) {
    const int t = threadIdx.x, lane = t & 63;
    int s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(s, o, 64);
        if (lane >= o) s += x;
    }
    if (t < 256 && lane == 63) part[t >> 6] = s;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int w = 0; w < 3; ++w) before += (w < (t >> 6)) ? part[w] : 0;
    return before + s - v;
}

// hist[w][d], the digit counts of 16 waves -> the place of wave w's first item of digit d: base[d] (the workgroup's own prefix
// over the digits when LOCAL) plus the waves before.
template <bool LOCAL>
__device__ __forceinline__ void wave_offsets(int* hist, int* part, int base) {
    const int t = threadIdx.x;
    int c[16], tot = 0;
    if (t < kBins) {
#pragma unroll
        for (int w = 0; w < 16; ++w) c[w] = hist[w * kBins + t];
#pragma unroll
        for (int w = 0; w < 16; ++w) tot += c[w];
    }
    if (LOCAL) base = prefix_256(tot, part);
    if (t < kBins) {
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            hist[w * kBins + t] = base;
            base += c[w];
        }
    }
    __syncthreads();
}

// All of up to kSortOne tokens in one workgroup of 1024 threads.
template <typename TI, int ITEMS>
__global__ __launch_bounds__(1024) void sort_one_kernel(const TI* __restrict__ ids, int N, int64_t V, int bits, int width,
                                                        int* __restrict__ sid, int* __restrict__ pos,
                                                        uint8_t* __restrict__ seen, int32_t* status) {
    extern __shared__ __attribute__((aligned(16))) int sm[];
    int* keys = sm;                          // [1024 * ITEMS]
    int* from = sm + 1024 * ITEMS;           // [1024 * ITEMS]
    int* hist = sm + 2 * 1024 * ITEMS;       // [16][kBins]
    int* part = hist + 16 * kBins;           // [4]
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    int key[ITEMS], src[ITEMS], digit[ITEMS], rank[ITEMS];
    TI tok[ITEMS];
    bool on[ITEMS];
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
        const int i = w * 64 * ITEMS + u * 64 + lane;
        on[u] = i < N;
        tok[u] = ids[min(i, N - 1)];
        src[u] = i;
        rank[u] = 0;
    }
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) key[u] = on[u] ? key_of((int64_t)tok[u], V, status) : 0;  // (all asked for by then)
    if (seen)
        for (int64_t i = t * 16; i < V; i += 16384) *reinterpret_cast<u32x4*>(seen + i) = u32x4{0, 0, 0, 0};
    for (int lo = 0; lo < bits; lo += width) {
        const int nb = min(width, bits - lo);
        for (int i = t; i < 16 * kBins; i += 1024) hist[i] = 0;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < ITEMS; ++u) digit[u] = (key[u] >> lo) & ((1 << nb) - 1);
        wave_ranks<ITEMS>(digit, on, nb, hist + w * kBins, rank);
        __syncthreads();
        wave_offsets<true>(hist, part, 0);
#pragma unroll
        for (int u = 0; u < ITEMS; ++u)
            if (on[u]) {
                const int d = hist[w * kBins + digit[u]] + rank[u];
                keys[d] = key[u];
                from[d] = src[u];
            }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < ITEMS; ++u) {
            const int i = w * 64 * ITEMS + u * 64 + lane;
            if (on[u]) {
                key[u] = keys[i];
                src[u] = from[i];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < ITEMS; ++u)
        if (on[u]) {
            sid[w * 64 * ITEMS + u * 64 + lane] = key[u];
            pos[w * 64 * ITEMS + u * 64 + lane] = src[u];
            if (seen && key[u] < V) seen[key[u]] = 1;  // (behind the passes' barriers)
        }
}

// More tokens: the counts of a digit, hist [tiles][kBins], tiles of 1024 * ITEMS tokens.  FIRST: ids are the tokens themselves,
// else the keys of the pass before.
template <typename TI, bool FIRST, int ITEMS>
__global__ __launch_bounds__(1024) void sort_count_kernel(const TI* __restrict__ ids, int N, int64_t V, int lo, int nb,
                                                          int* __restrict__ hist, uint8_t* __restrict__ seen, int32_t* status) {
    __shared__ int cnt[kBins];
    const int t = threadIdx.x;
    TI tok[ITEMS];
    if (FIRST && seen)  // (16 bytes a thread; the workspace has room behind the last row)
        for (int64_t i = ((int64_t)blockIdx.x * 1024 + t) * 16; i < V; i += (int64_t)gridDim.x * 16384)
            *reinterpret_cast<u32x4*>(seen + i) = u32x4{0, 0, 0, 0};
    if (t < kBins) cnt[t] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
        const int64_t i = ((int64_t)blockIdx.x * ITEMS + u) * 1024 + t;
        tok[u] = ids[min(i, (int64_t)N - 1)];
    }
#pragma unroll
    for (int u = 0; u < ITEMS; ++u)
        if (((int64_t)blockIdx.x * ITEMS + u) * 1024 + t < N) {
            const int k = FIRST ? key_of((int64_t)tok[u], V, status) : (int)tok[u];
            atomicAdd(&cnt[(k >> lo) & ((1 << nb) - 1)], 1);
        }
    __syncthreads();
    if (t < kBins) hist[(int64_t)blockIdx.x * kBins + t] = cnt[t];
}

// One pass: every tile's items to their places by digit (bits lo .. lo + nb).
template <typename TI, bool FIRST, int ITEMS>
__global__ __launch_bounds__(1024) void sort_pass_kernel(const TI* __restrict__ ids, const int* __restrict__ src, int N,
                                                         int64_t V, int lo, int nb, int tiles, const int* __restrict__ hist,
                                                         int* __restrict__ sid, int* __restrict__ pos,
                                                         uint8_t* __restrict__ seen) {
    __shared__ int wh[16 * kBins], part[4];
    __shared__ int tot[4][kBins], bef[4][kBins];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    int key[ITEMS], from[ITEMS], digit[ITEMS], rank[ITEMS];
    bool on[ITEMS];
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
        const int64_t i = (int64_t)blockIdx.x * 1024 * ITEMS + w * 64 * ITEMS + u * 64 + lane;
        on[u] = i < N;
        const int64_t at = min(i, (int64_t)N - 1);
        const TI id = ids[at];
        key[u] = FIRST ? key_of((int64_t)id, V, nullptr) : (int)id;
        from[u] = FIRST ? (int)i : src[at];
        digit[u] = (key[u] >> lo) & ((1 << nb) - 1);
        rank[u] = 0;
    }
    // where digit d of this tile starts: all of the smaller digits, and digit d of the tiles before
    {
        const int d = t & (kBins - 1), q = t >> 8;
        int all = 0, before = 0;
        for (int b0 = q; b0 < tiles; b0 += 32) {
            int c[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) c[u] = hist[(int64_t)min(b0 + 4 * u, tiles - 1) * kBins + d];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (b0 + 4 * u >= tiles) c[u] = 0;
                all += c[u];
                if (b0 + 4 * u < (int)blockIdx.x) before += c[u];
            }
        }
        tot[q][d] = all;
        bef[q][d] = before;
    }
    for (int i = t; i < 16 * kBins; i += 1024) wh[i] = 0;
    __syncthreads();
    wave_ranks<ITEMS>(digit, on, nb, wh + w * kBins, rank);
    int base = 0, mine = 0;
    if (t < kBins) {
        mine = tot[0][t] + tot[1][t] + tot[2][t] + tot[3][t];
        base = bef[0][t] + bef[1][t] + bef[2][t] + bef[3][t];
    }
    base += prefix_256(mine, part);  // (its barrier also ends the ranks)
    wave_offsets<false>(wh, part, base);
#pragma unroll
    for (int u = 0; u < ITEMS; ++u)
        if (on[u]) {
            const int d = wh[w * kBins + digit[u]] + rank[u];
            sid[d] = key[u];
            pos[d] = from[u];
            if (FIRST && seen && key[u] < V) seen[key[u]] = 1;  // (whoever writes it writes the same)
        }
}

// ------------------------------------------------------------------------------------------------ sums
struct Sum {
    const void* dout;
    const int* sid;
    const int* pos;
    float* dtable;
    float* part;   // [chunks][2][dpad]: a chunk's open row at its head / at its tail
    const uint8_t* seen;  // [V] 1: the row has a token (null: looked up in the sorted list)
    int64_t ldd, ldt, V, D;
    float scale;
    int N, chunk, nchunk, accumulate;
    int lpr;       // lanes of a team: a power of two, 8 columns each
    int cblk;      // blocks of 8 * lpr columns
    int sum_blocks;
    __device__ __forceinline__ int64_t dpad() const { return (D + 7) & ~(int64_t)7; }
};

__device__ __forceinline__ int lower_bound(const int* sid, int N, int v) {  // first place whose id is >= v
    int lo = 0, hi = N;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sid[mid] < v) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// Columns c .. c + 7 of table row v (those < D, and from c + own on where the old value is added to: one writer a column)
__device__ __forceinline__ void write_row(const Sum& a, int v, int64_t c, int own, float (&s)[8]) {
    float* row = a.dtable + (int64_t)v * a.ldt;
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] *= a.scale;
    if (!a.accumulate) {
        store_row8(row, c, a.D, s);
    } else if (own == 0 && c + 8 <= a.D) {
        float o[8];
        load8(row + c, o);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] += o[j];
        store8(row + c, s);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j >= own && c + j < a.D) row[c + j] += s[j];
    }
}

constexpr int kZeroRows = 16;  // table rows that a wave looks through for rows without a token

// A column group is eight columns from c; a row's last, partial group is its last eight columns, which its neighbour forms too,
// with the same bits (own: the first column that only this group has).  EL: rows shorter than eight columns.
template <typename T, bool EL>
__global__ __launch_bounds__(256) void sum_kernel(Sum a) {
    const int lane = threadIdx.x & 63;
    if ((int)blockIdx.x >= a.sum_blocks) {  // rows without a token
        const int64_t v0 = (((int64_t)blockIdx.x - a.sum_blocks) * 4 + (threadIdx.x >> 6)) * kZeroRows;
        bool absent = false;
        if (lane < kZeroRows && v0 + lane < a.V) {
            const int v = (int)(v0 + lane);
            if (a.seen) {
                absent = a.seen[v] == 0;
            } else {
                const int p = lower_bound(a.sid, a.N, v);
                absent = p == a.N || a.sid[p] != v;
            }
        }
        const uint64_t m = __ballot(absent);
        const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int r = lane / a.lpr; r < kZeroRows; r += 64 / a.lpr) {  // (a team a row)
            if (!(m >> r & 1)) continue;
            for (int64_t c = (lane & (a.lpr - 1)) * 8; c < a.D; c += a.lpr * 8) store_row8(a.dtable + (v0 + r) * a.ldt, c, a.D, zero);
        }
        return;
    }
    const int tpb = 256 / a.lpr;
    const int64_t team = (int64_t)blockIdx.x * tpb + threadIdx.x / a.lpr;
    const int64_t ch = team / a.cblk;
    const int64_t c0 = ((team - ch * a.cblk) * a.lpr + (threadIdx.x & (a.lpr - 1))) * 8;
    if (ch >= a.nchunk || c0 >= a.D) return;
    const int64_t c = EL ? 0 : min(c0, a.D - 8);
    const int own = (int)(c0 - c);
    const T* dout = reinterpret_cast<const T*>(a.dout);
    const int beg = (int)ch * a.chunk, end = min(a.N, beg + a.chunk);
    int cur = a.sid[beg];
    bool head = beg > 0 && a.sid[beg - 1] == cur;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    // eight tokens at a time: their places, then their rows, then the sums (behind the end: the last token again, not added)
    for (int i0 = beg; i0 < end; i0 += 8) {
        int id[8], p[8];
        Raw8<T> raw[8];
        float x[8][8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = min(i0 + u, end - 1);
            id[u] = a.sid[i];
            p[u] = a.pos[i];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (EL) load_short(dout + (int64_t)p[u] * a.ldd, a.D, x[u]);
            else raw[u] = raw8(dout + (int64_t)p[u] * a.ldd + c);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (i0 + u >= end) continue;
            if (!EL) unraw8(raw[u], x[u]);
            if (id[u] != cur) {  // the row before is complete (cur < V: the places without a token come last)
                if (head) store8(a.part + ch * 2 * a.dpad() + c, s);
                else write_row(a, cur, c, own, s);
                head = false;
                cur = id[u];
#pragma unroll
                for (int j = 0; j < 8; ++j) s[j] = 0.f;
            }
            if (id[u] < a.V) {
#pragma unroll
                for (int j = 0; j < 8; ++j) s[j] += x[u][j];
            }
        }
    }
    if (cur >= a.V) return;
    const bool open = end < a.N && a.sid[end] == cur;
    if (head) store8(a.part + ch * 2 * a.dpad() + c, s);
    else if (open) store8(a.part + (ch * 2 + 1) * a.dpad() + c, s);
    else write_row(a, cur, c, own, s);
}

// Rows that cross chunk ends, joined by the wave of the chunk in which such a row begins: a row goes on into the next chunk
// where that chunk's first token has its id (64 chunks looked at together).  A long chain of parts (a row of very many
// tokens) is shared by the workgroup's sixteen waves.
constexpr int kShort = 16;

// s += parts k0 .. k1 - 1 of the chain that starts at chunk `first`, sixteen on their way at once; four columns a lane
__device__ __forceinline__ void add_parts(const Sum& a, int64_t c, int first, int k0, int k1, f32x4& s) {
    for (int k = k0; k < k1; k += 16) {
        f32x4 x[16];
#pragma unroll
        for (int u = 0; u < 16; ++u)
            x[u] = *reinterpret_cast<const f32x4*>(a.part + (int64_t)(first + min(k + u, k1 - 1)) * 2 * a.dpad() + c);
#pragma unroll
        for (int u = 0; u < 16; ++u)
            if (k + u < k1) s += x[u];
    }
}

// (added to what is there: a sum of zero leaves it as it is, bit for bit -- that of a row without a token in few_rows_join_kernel)
__device__ __forceinline__ void write_row4(const Sum& a, int v, int64_t c, f32x4 s) {
    float* row = a.dtable + (int64_t)v * a.ldt;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (c + j >= a.D) continue;
        if (!a.accumulate) row[c + j] = s[j] * a.scale;
        else if (s[j] != 0.f) row[c + j] += s[j] * a.scale;
    }
}

__global__ __launch_bounds__(1024) void join_kernel(Sum a) {
    __shared__ f32x4 red[16][64];
    __shared__ int chain[16], row[16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int ch = (int)blockIdx.x * 16 + w;
    const int64_t c = ((int64_t)blockIdx.y * 64 + lane) * 4;  // (parts lie in rows of dpad, D rounded up to 8)
    int n = 0, v = 0;                                         // parts behind the chunk's own
    if (ch + 1 < a.nchunk) {
        const int beg = ch * a.chunk, end = beg + a.chunk;
        // the first token of chunk ch + k has id v: for k = 1 + lane and, for very long rows, k = base + 64 (1 + lane)
        auto first_of = [&](int64_t k) { return ch + k < a.nchunk ? a.sid[(ch + k) * a.chunk] : -1; };
        auto run = [&](int id) {
            const uint64_t other = __ballot(id != v);
            return other == 0 ? 64 : __ffsll((unsigned long long)other) - 1;
        };
        const int near = first_of(1 + lane), vb = a.sid[beg], vp = beg > 0 ? a.sid[beg - 1] : -1;
        int far = first_of(64 + 64 * (1 + lane));  // (asked for with the rest: one trip to memory)
        v = a.sid[end - 1];
        if (v < a.V && !(vb == v && vp == v)) {  // (a token's row, and it did not begin in an earlier chunk)
            n = run(near);
            if (n == 64) {
                for (;;) {
                    const int r = run(far);
                    n += 64 * r;
                    if (r < 64) break;
                    far = first_of(n + 64 * (1 + lane));
                }
                n += run(first_of(n + 1 + lane));
            }
        }
    }
    if (lane == 0) {
        chain[w] = n;
        row[w] = v;
    }
    if (n > 0 && n <= kShort && c < a.dpad()) {
        f32x4 s = *reinterpret_cast<const f32x4*>(a.part + ((int64_t)ch * 2 + 1) * a.dpad() + c);
        add_parts(a, c, ch + 1, 0, n, s);
        write_row4(a, v, c, s);
    }
    __syncthreads();
    for (int o = 0; o < 16; ++o) {
        const int m = chain[o];
        if (m <= kShort) continue;  // (uniform)
        const int first = (int)blockIdx.x * 16 + o + 1, q = (m + 15) / 16;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        if (c < a.dpad()) {
            if (w == 0) s = *reinterpret_cast<const f32x4*>(a.part + ((int64_t)(first - 1) * 2 + 1) * a.dpad() + c);
            add_parts(a, c, first, min(m, w * q), min(m, w * q + q), s);
        }
        red[w][lane] = s;
        __syncthreads();
        if (w == 0 && c < a.dpad()) {
            s = red[0][lane];
#pragma unroll
            for (int i = 1; i < 16; ++i) s += red[i][lane];
            write_row4(a, row[o], c, s);
        }
        __syncthreads();
    }
}

// ---- up to kFewTokens tokens: one launch.  Every workgroup looks through all ids for its table rows' tokens (in their order);
// a wave takes four rows and 512 columns and sums each row's tokens, eight on their way at once.  Bound by the launch and by a row's
// chain of loads: 64 tokens over three rows of 256 columns 5.0 us (sorted 11).
constexpr int kFewTokens = 128;
constexpr int kRowsPerGroup = 16;

template <typename T, typename TI, bool EL>
__global__ __launch_bounds__(256) void few_tokens_kernel(Sum a, const TI* __restrict__ ids, int32_t* status) {
    __shared__ int key[kFewTokens];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    if (t < kFewTokens) key[t] = t < a.N ? key_of((int64_t)ids[t], a.V, status) : (int)a.V;
    __syncthreads();
    const int64_t c0 = ((int64_t)blockIdx.y * 64 + lane) * 8;
    const bool live = c0 < a.D;
    const int64_t c = EL ? 0 : min(c0, a.D - 8);
    const T* dout = reinterpret_cast<const T*>(a.dout);
    const int k[2] = {key[lane], key[64 + lane]};
    for (int r = w; r < kRowsPerGroup; r += 4) {
        const int64_t v = (int64_t)blockIdx.x * kRowsPerGroup + r;
        if (v >= a.V) break;
        float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        bool any = false;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            uint64_t m = __ballot(k[b] == (int)v);
            any |= m != 0;
            while (m) {
                int p[8], n = 0;
#pragma unroll
                for (int u = 0; u < 8; ++u) {  // the next eight of them; behind the last: the last again, not added
                    if (m) {
                        p[u] = b * 64 + __ffsll((unsigned long long)m) - 1;
                        m &= m - 1;
                        n = u + 1;
                    } else {
                        p[u] = p[u > 0 ? u - 1 : 0];
                    }
                }
                if (!live) continue;
                Raw8<T> raw[8];
                float x[8][8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (EL) load_short(dout + (int64_t)p[u] * a.ldd, a.D, x[u]);
                    else raw[u] = raw8(dout + (int64_t)p[u] * a.ldd + c);
                }
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (u < n) {
                        if (!EL) unraw8(raw[u], x[u]);
#pragma unroll
                        for (int j = 0; j < 8; ++j) s[j] += x[u][j];
                    }
            }
        }
        if (live && (any || !a.accumulate)) write_row(a, (int)v, c, (int)(c0 - c), s);
    }
}

// ---- up to kFewRows table rows (conditions): no sort.  A team keeps one sum for each row over a chunk of tokens, and a second
// launch adds the chunks up.  4096 tokens over three rows of 1024 columns in fp32 12.6 us (sorted 16.9): 8.0 for the sums, 5.2 for
// the join; half of either is a launch's start.
constexpr int kFewRows = 8;

template <typename T, typename TI, bool EL, int NV>  // NV >= V sums
__global__ __launch_bounds__(256) void few_rows_kernel(Sum a, const TI* __restrict__ ids, int32_t* status) {
    const int tpb = 256 / a.lpr;
    const int64_t team = (int64_t)blockIdx.x * tpb + threadIdx.x / a.lpr;
    const int64_t ch = team / a.cblk;
    const int64_t c0 = ((team - ch * a.cblk) * a.lpr + (threadIdx.x & (a.lpr - 1))) * 8;
    if (ch >= a.nchunk || c0 >= a.D) return;
    const int64_t c = EL ? 0 : min(c0, a.D - 8);
    const T* dout = reinterpret_cast<const T*>(a.dout);
    const int beg = (int)ch * a.chunk, end = min(a.N, beg + a.chunk);
    float s[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[v][j] = 0.f;
    for (int i0 = beg; i0 < end; i0 += 8) {
        int id[8];
        TI tok[8];
        Raw8<T> raw[8];
        float x[8][8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = min(i0 + u, end - 1);
            tok[u] = ids[i];
            if (EL) load_short(dout + (int64_t)i * a.ldd, a.D, x[u]);
            else raw[u] = raw8(dout + (int64_t)i * a.ldd + c);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int k = key_of((int64_t)tok[u], a.V, status);
            id[u] = i0 + u < end && k < a.V ? k : NV;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (!EL) unraw8(raw[u], x[u]);
#pragma unroll
            for (int v = 0; v < NV; ++v)  // (a branch: the lanes of a team have the same token)
                if (id[u] == v) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) s[v][j] += x[u][j];
                }
        }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
        if (v < a.V) store8(a.part + (ch * a.V + v) * a.dpad() + c, s[v]);
}

// dtable[v] = scale * sum of its chunks' parts: four columns a lane, sixteen waves a sixteenth of the chunks each
__global__ __launch_bounds__(1024) void few_rows_join_kernel(Sum a) {
    __shared__ f32x4 red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, v = blockIdx.x;
    const int64_t c = ((int64_t)blockIdx.y * 64 + lane) * 4;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (c < a.dpad()) {
        for (int k = w; k < a.nchunk; k += 128) {
            f32x4 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                x[u] = *reinterpret_cast<const f32x4*>(a.part + ((int64_t)min(k + 16 * u, a.nchunk - 1) * a.V + v) * a.dpad() + c);
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (k + 16 * u < a.nchunk) s += x[u];
        }
    }
    red[w][lane] = s;
    __syncthreads();
    if (w != 0 || c >= a.dpad()) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][lane];
    write_row4(a, v, c, s);
}

// ------------------------------------------------------------------------------------------------ plan
struct Plan {
    int form;  // 0: sorted, 1: few tokens, 2: few rows
    int bits, passes, width, items, tiles, chunk, nchunk, lpr, cblk;
    int64_t dpad;
    size_t keys, hist, seen, part, total;  // bytes / offsets of the workspace
};
// Are the rows that have a token marked?  Where one workgroup sorts, and would clear more marks than it gains by: no.
inline bool marked(int64_t N, int64_t V) { return N > kSortOne || V <= (1 << 18); }
inline Plan plan_of(int64_t N, int64_t V, int64_t D) {
    Plan p{};
    while ((V >> p.bits) != 0) ++p.bits;  // the largest key is V
    p.passes = std::max(1, (p.bits + 7) / 8);
    p.width = (p.bits + p.passes - 1) / p.passes;
    p.items = N <= (1 << 18) ? 1 : N <= (1 << 21) ? 4 : 16;  // a tile's counts are read by every workgroup: at most a few thousand tiles
    p.tiles = (int)((N + 1024 * p.items - 1) / (1024 * p.items));
    p.dpad = (D + 7) / 8 * 8;
    p.lpr = 1;
    while (p.lpr < 64 && p.lpr * 8 < D) p.lpr *= 2;
    p.cblk = (int)((D + p.lpr * 8 - 1) / (p.lpr * 8));
    // chunks of 8 to 64 tokens: about 2048 waves where there are so many tokens (65 536 tokens of 512 columns: 16 tokens a chunk
    // sum in 21.4 us and join in 14.0, 32 tokens in 20.8 and 8.1; but eight tokens take a team 2 us, whose latency only other teams
    // hide: 100 000 of 128 columns in chunks of 64 sum in 15.8 instead of 6.7)
    const int64_t waves8 = (N + 7) / 8 * p.cblk * p.lpr / 64;
    p.chunk = 8;
    while (p.chunk < 64 && waves8 * 8 / p.chunk > 2048) p.chunk *= 2;
    // The form, float32, 256 columns, replayed: 64 tokens over three or eight rows 5.0 and 5.3 us in one launch, 7.8 and 9.5 as
    // sums for each row; 128: 7.3 and 7.0, 8.9 and 10.9; 256 over nine: 14.1 in one launch, 11.0 sorted.  4096 tokens over eight
    // rows as sums 14.2, over nine sorted 16.2; 8192 over three or eight as sums 15.2 and 18.1, over nine sorted 17.5; 16 384: 20.9
    // and 24.6 as sums, 23.3 and 21.4 sorted; 65 536: 60 and 65, 40 and 31.
    p.form = N <= kFewTokens ? 1 : V <= kFewRows && N <= 8192 ? 2 : 0;
    if (p.form == 1) return p;
    if (p.form == 2) {
        // (chunks of 16 tokens or more, about 2048 waves)
        p.chunk = 16;
        while (p.chunk < 1024 && (N + 15) / 16 * p.cblk * p.lpr / 64 * 16 / p.chunk > 2048) p.chunk *= 2;
        p.nchunk = (int)((N + p.chunk - 1) / p.chunk);
        p.total = (size_t)p.nchunk * V * p.dpad * 4;
        return p;
    }
    p.nchunk = (int)((N + p.chunk - 1) / p.chunk);
    const size_t n4 = ((size_t)N * 4 + 15) / 16 * 16;
    p.keys = n4;
    const bool one = N <= kSortOne;
    p.hist = (one ? 2 : 4) * n4;
    p.seen = p.hist + (one ? 0 : (size_t)p.tiles * kBins * 4);
    p.part = p.seen + (marked(N, V) ? (size_t)(V + 15) / 16 * 16 : 0);
    p.total = p.part + (size_t)p.nchunk * 2 * p.dpad * 4;
    return p;
}

template <typename TI>
void sort_tokens(const TI* ids, int64_t N, int64_t V, const Plan& p, char* ws, int*& sid, int*& pos, uint8_t* seen,
                 int32_t* status, hipStream_t st) {
    int* k0 = (int*)ws;
    int* p0 = (int*)(ws + p.keys);
    sid = k0;
    pos = p0;
    if (N <= kSortOne) {
        const int items = N <= 1024 ? 1 : 4;
        const size_t lds = ((size_t)2 * 1024 * items + 16 * kBins + 4) * 4;
#define ONE(I)                                                                                                              \
    do {                                                                                                                    \
        auto k = sort_one_kernel<TI, I>;                                                                                    \
        if (lds > 48 * 1024) (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds); \
        hipLaunchKernelGGL(k, dim3(1), dim3(1024), lds, st, ids, (int)N, V, p.bits, p.width, sid, pos, seen, status);       \
    } while (0)
        if (items == 1) ONE(1);
        else ONE(4);
#undef ONE
        return;
    }
    int* k1 = (int*)(ws + 2 * p.keys);
    int* p1 = (int*)(ws + 3 * p.keys);
    int* hist = (int*)(ws + p.hist);
    for (int pass = 0; pass < p.passes; ++pass) {
        const int lo = pass * p.width, nb = std::min(p.width, p.bits - lo);
        int *ko = (pass & 1) ? k1 : k0, *po = (pass & 1) ? p1 : p0;
        const int *ki = (pass & 1) ? k0 : k1, *pi = (pass & 1) ? p0 : p1;
#define STEP(TK, FIRST, I, KEYS, POS)                                                                                      \
    do {                                                                                                                   \
        hipLaunchKernelGGL((sort_count_kernel<TK, FIRST, I>), dim3(p.tiles), dim3(1024), 0, st, KEYS, (int)N, V, lo, nb,   \
                           hist, seen, status);                                                                                  \
        hipLaunchKernelGGL((sort_pass_kernel<TK, FIRST, I>), dim3(p.tiles), dim3(1024), 0, st, KEYS, POS, (int)N, V, lo,   \
                           nb, p.tiles, hist, ko, po, seen);                                                                 \
    } while (0)
#define PASS(I)                                                             \
    do {                                                                    \
        if (pass == 0) STEP(TI, true, I, ids, (const int*)nullptr);         \
        else STEP(int, false, I, ki, pi);                                   \
    } while (0)
        if (p.items == 1) PASS(1);
        else if (p.items == 4) PASS(4);
        else PASS(16);
#undef PASS
#undef STEP
        sid = ko;
        pos = po;
    }
}

}  // namespace embed
}  // namespace c2

extern "C" int c2_embed_fwd(const void* table, int t_dtype, int64_t ldt, int64_t V, int64_t D, const void* ids, int idx_bytes,
                            int64_t N, float scale, void* out, int out_dtype, int64_t ldo, int32_t* status_dev, void* stream) {
    using namespace c2;
    C2_CHECK(V >= 0 && D >= 0 && N >= 0, "negative size");
    C2_CHECK(t_dtype == C2_F32 || t_dtype == C2_BF16 || t_dtype == C2_F16, "bad table dtype");
    C2_CHECK(out_dtype == C2_F32 || out_dtype == t_dtype, "out_dtype: fp32 or the table's");
    C2_CHECK(idx_bytes == 4 || idx_bytes == 8, "idx_bytes: 4 (int32) or 8 (int64)");
    if (N == 0 || D == 0) return 0;
    C2_CHECK(ids && out && ldo >= D && (V == 0 || (table && ldt >= D)), "bad arguments");
    C2_CHECK(D < (1ll << 31), "D too large");
    hipStream_t st = (hipStream_t)stream;
    const int64_t dg = (D + 7) / 8, step = std::max<int64_t>(1, (1ll << 30) / dg);  // rows of a launch: 32-bit indices
    for (int64_t n0 = 0; n0 < N; n0 += step) {
        const int64_t rows = std::min(step, N - n0);
        const unsigned count = (unsigned)(rows * dg), grid = (count + 1023) / 1024;
#define GL(T, TO, TI, EL)                                                                                                   \
    hipLaunchKernelGGL((embed::lookup_kernel<T, TO, TI, EL>), dim3(grid), dim3(256), 0, st, (const T*)table, ldt, V,         \
                       (const TI*)ids + n0, count, (unsigned)dg, D, scale, (TO*)out + n0 * ldo, ldo, status_dev)
#define GO(T, TO)                                                                                                           \
    do {                                                                                                                    \
        if (idx_bytes == 8) { if (D < 8) GL(T, TO, int64_t, true); else GL(T, TO, int64_t, false); }                         \
        else { if (D < 8) GL(T, TO, int32_t, true); else GL(T, TO, int32_t, false); }                                        \
    } while (0)
        if (t_dtype == C2_F32) GO(float, float);
        else if (t_dtype == C2_BF16) { if (out_dtype == C2_F32) GO(bf16_t, float); else GO(bf16_t, bf16_t); }
        else { if (out_dtype == C2_F32) GO(f16_t, float); else GO(f16_t, f16_t); }
#undef GO
#undef GL
    }
    C2_LAUNCH_CHECK();
    return 0;
}

extern "C" size_t c2_embed_grad_ws(int64_t N, int64_t V, int64_t D) {
    if (N <= 0 || V <= 0 || D <= 0) return 0;
    return c2::embed::plan_of(N, V, D).total;
}

extern "C" int c2_embed_grad(const void* dout, int d_dtype, int64_t ldd, const void* ids, int idx_bytes, int64_t N, int64_t V,
                             int64_t D, float scale, float* dtable, int64_t ldt, int accumulate, void* ws,
                             int32_t* status_dev, void* stream) {
    using namespace c2;
    C2_CHECK(V >= 0 && D >= 0 && N >= 0 && N <= (1ll << 26) && V <= (1ll << 27) && D <= (1ll << 23), "bad shape");
    C2_CHECK(d_dtype == C2_F32 || d_dtype == C2_BF16 || d_dtype == C2_F16, "bad gradient dtype");
    C2_CHECK(idx_bytes == 4 || idx_bytes == 8, "idx_bytes: 4 (int32) or 8 (int64)");
    C2_CHECK(scale - scale == 0.f, "scale must be finite");  // (rows without a token are sums of zero, scaled, in some forms)
    if (V == 0 || D == 0) return 0;
    C2_CHECK(dtable && ldt >= D && (N == 0 || (dout && ids && ldd >= D)), "bad arguments");
    C2_CHECK(c2_embed_grad_ws(N, V, D) == 0 || (ws && aligned16(ws)), "workspace: null, or not on 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    const embed::Plan p = embed::plan_of(N, V, D);
    if (N > 0 && p.form != 0) {
        embed::Sum a{dout, nullptr, nullptr, dtable, (float*)ws, nullptr, ldd, ldt, V, D, scale, (int)N, p.chunk, p.nchunk,
                     accumulate, p.lpr, p.cblk, 0};
        const int64_t g = p.form == 1 ? (V + embed::kRowsPerGroup - 1) / embed::kRowsPerGroup
                                      : ((int64_t)p.nchunk * p.cblk * p.lpr + 255) / 256;
        const dim3 grid((unsigned)g, p.form == 1 ? (unsigned)((D + 511) / 512) : 1u);
#define FEW(T, TI, EL)                                                                                                      \
    do {                                                                                                                    \
        if (p.form == 1)                                                                                                    \
            hipLaunchKernelGGL((embed::few_tokens_kernel<T, TI, EL>), grid, dim3(256), 0, st, a, (const TI*)ids, status_dev); \
        else if (V <= 4)                                                                                                    \
            hipLaunchKernelGGL((embed::few_rows_kernel<T, TI, EL, 4>), grid, dim3(256), 0, st, a, (const TI*)ids, status_dev); \
        else                                                                                                                \
            hipLaunchKernelGGL((embed::few_rows_kernel<T, TI, EL, 8>), grid, dim3(256), 0, st, a, (const TI*)ids, status_dev); \
    } while (0)
#define FEWT(T)                                                                          \
    do {                                                                                 \
        if (idx_bytes == 8) { if (D < 8) FEW(T, int64_t, true); else FEW(T, int64_t, false); } \
        else { if (D < 8) FEW(T, int32_t, true); else FEW(T, int32_t, false); }          \
    } while (0)
        if (d_dtype == C2_F32) FEWT(float);
        else if (d_dtype == C2_BF16) FEWT(bf16_t);
        else FEWT(f16_t);
#undef FEWT
#undef FEW
        if (p.form == 2)
            hipLaunchKernelGGL((embed::few_rows_join_kernel), dim3((unsigned)V, (unsigned)((D + 255) / 256)), dim3(1024), 0, st, a);
        C2_LAUNCH_CHECK();
        return 0;
    }
    int *sid = nullptr, *pos = nullptr;
    uint8_t* seen = N > 0 && embed::marked(N, V) && !accumulate ? (uint8_t*)ws + p.seen : nullptr;
    if (N > 0) {
        if (idx_bytes == 8) embed::sort_tokens((const int64_t*)ids, N, V, p, (char*)ws, sid, pos, seen, status_dev, st);
        else embed::sort_tokens((const int32_t*)ids, N, V, p, (char*)ws, sid, pos, seen, status_dev, st);
    }
    embed::Sum a{dout, sid, pos, dtable, N > 0 ? (float*)((char*)ws + p.part) : nullptr, seen, ldd, ldt, V, D, scale,
                 (int)N, p.chunk, p.nchunk, accumulate, p.lpr, p.cblk, 0};
    const int64_t sum_blocks = ((int64_t)p.nchunk * p.cblk * p.lpr + 255) / 256;
    const int64_t zero_blocks = accumulate ? 0 : (V + 4 * embed::kZeroRows - 1) / (4 * embed::kZeroRows);
    C2_CHECK(sum_blocks + zero_blocks < (1ll << 24), "too many blocks for one launch");
    a.sum_blocks = (int)sum_blocks;
    if (sum_blocks + zero_blocks > 0) {
        const dim3 grid((unsigned)(sum_blocks + zero_blocks));
#define SUM(T)                                                                                          \
    do {                                                                                                \
        if (D < 8) hipLaunchKernelGGL((embed::sum_kernel<T, true>), grid, dim3(256), 0, st, a);         \
        else hipLaunchKernelGGL((embed::sum_kernel<T, false>), grid, dim3(256), 0, st, a);              \
    } while (0)
        if (d_dtype == C2_F32) SUM(float);
        else if (d_dtype == C2_BF16) SUM(bf16_t);
        else SUM(f16_t);
#undef SUM
    }
    if (p.nchunk > 1)
        hipLaunchKernelGGL((embed::join_kernel), dim3((unsigned)((p.nchunk + 15) / 16), (unsigned)((D + 255) / 256)), dim3(1024), 0,
                           st, a);
    C2_LAUNCH_CHECK();
    return 0;
}
