// Distillation from a teacher's top logits, forward and backward, for gfx950.
//
// Row b: student logits s_j over V classes, the teacher's list (i_k, t_k), k < K, temperature T, weight w_b.
//   q = softmax(s / T);  p_k = softmax over the list of t_k / T, or exp(t_k / T - lse_b) when the teacher's own normaliser
//   over its whole vocabulary is given (then P = sum_k p_k <= 1; else P = 1)
//   loss   = T^2 c sum_b w_b sum_k p_k (log p_k - log q_{i_k})
//   ds_j   = T c w_b (P q_j - sum_{k: i_k = j} p_k),   c = inv_B
// With e_k = exp(d_k), d_k = (t_k - max t) / T (of the logits' difference: t / T itself may be large, and its rounding with it) and
// z = sum e_k, or d_k = t_k / T - lse and z = 1: p_k = e_k / z, and the row's sum over the list is
//   (U - W) / z - P log z + P log Z,  U = sum e_k d_k,  W = sum e_k (s_{i_k} - mS)/T,  Z = sum_j exp((s_j - mS)/T),
// so that every sum of the row (Z, z, U, W) is formed after the two maxima and one more reduction ends the row.
//
// Bound by memory: a row is read once and its gradient written once (311 MB at 4096 x 19 000 in bf16: 69-71 us, 4.5 TB/s, 0.88 of
// a large copy's rate).  Up to 32 768 classes a
// row's exponentials stay in the registers of one wave (V <= 1024) or workgroup between the two passes.  Longer rows are cut
// into segments of 8192 over many workgroups: one launch for the segments' maxima and sums, one that joins them and writes the
// gradient (it reads the row again, from the caches while a launch's rows fit them): 3 rows of 100 001 in half precision 4.4 + 6.5 us.
// The listed classes' gradients are written a second time, over the row pass's, by the thread that holds the list entry.
//
// Entries with index < 0 are absent; rows with weight 0 or an empty list cost nothing and get zero gradients whatever their
// logits hold.  An index >= V is left out and reported through the status word.
#include <algorithm>

#include "vec8.h"

namespace c2 {
namespace distill {

struct Args {
    const void* s;
    const void* idx;
    const float* top;
    const float* lse;
    const float* weight;
    void* ds;
    float* part;
    float* only;   // the loss, where one workgroup forms it (null: partial losses)
    float* loss;   // to be cleared before the partial losses are added up (null: they are added to what is there)
    int32_t* status;
    int64_t lds, ldds, ldi, ldt, B, V;
    int K, iw;
    float it;     // 1 / T
    float T;
    float inv_B;
};

// int32 or int64 indices (a.iw = 1 or 2 words) without a branch: the low and the high word, the same word twice for int32
__device__ __forceinline__ int64_t join_index(const Args& a, int lo, int hi) {
    return a.iw == 2 ? ((int64_t)hi << 32 | (unsigned)lo) : (int64_t)lo;
}
__device__ __forceinline__ int64_t list_index(const Args& a, int64_t b, int k) {
    const int* p = reinterpret_cast<const int*>(a.idx) + (b * a.ldi + k) * a.iw;
    return join_index(a, p[0], p[a.iw - 1]);
}

constexpr int kMaxList = 1024;
constexpr int kSeg = 8192;  // classes of a segment

// v_exp_f32: one unit in the last place, results below the normal range are zero
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

template <int W>  // W = 1: the rows of a workgroup's waves are independent, and only the wave itself is in step
__device__ __forceinline__ void sync_row() {
    if (W == 1) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}

// maxima / sums of N values over the W waves of a row; red: N * W floats in LDS, free on entry, free again after the next sync
template <int W, int N, bool MAX>
__device__ __forceinline__ void row_reduce(float (&v)[N], float* red) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = MAX ? wave_max(v[n]) : wave_sum(v[n]);
    if (W == 1) return;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int n = 0; n < N; ++n) red[n * W + w] = v[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        float r = red[n * W];
#pragma unroll
        for (int i = 1; i < W; ++i) r = MAX ? fmaxf(r, red[n * W + i]) : r + red[n * W + i];
        v[n] = r;
    }
}

// A teacher's logit in the list's maximum: a NaN as infinity, so that a row whose logits are all NaN is not taken for one
// without a list (the exponentials of the others are then zero, its own NaN).
__device__ __forceinline__ float in_max(float x) { return x == x ? x : INFINITY; }

// log e of a list entry (above); mt: the list's largest logit, or the teacher's normaliser
__device__ __forceinline__ float list_arg(const Args& a, float x, float mt) {
    return a.lse ? fmaf(x, a.it, -mt) : (x - mt) * a.it;
}

// The list of row b into LDS (index -1: absent) and its largest logit; t, nt: the row's threads.
__device__ __forceinline__ float load_list(const Args& a, int64_t b, int t, int nt, int* lidx, float* lval, bool report) {
    float mt = -INFINITY;
    for (int k = t; k < a.K; k += nt) {
        const int64_t i = list_index(a, b, k);
        const float v = a.top[b * a.ldt + k];
        const bool on = i >= 0 && i < a.V;
        if (report && i >= a.V && a.status) *a.status = 1;
        lidx[k] = on ? (int)i : -1;
        lval[k] = v;
        if (on) mt = fmaxf(mt, in_max(v));
    }
    return mt;
}

// Lists in LDS: [3][K4] with K4 = K rounded up to 4; places behind the list hold index -1.
__device__ __forceinline__ int list_pitch(int K) { return (K + 3) & ~3; }
__device__ __forceinline__ void end_list(int K, int t, int* lidx) {
    if (t < list_pitch(K) - K) lidx[K + t] = -1;
}

// sum of the list's e over the entries that name class j (an index may be given several times)
__device__ __forceinline__ float listed(const int* lidx, const float* lval, int K, int j) {
    typedef __attribute__((ext_vector_type(4))) int i32x4;
    float s = 0.f;
#pragma unroll 4
    for (int k = 0; k < K; k += 4) {
        const i32x4 i = *reinterpret_cast<const i32x4*>(lidx + k);
        const f32x4 e = *reinterpret_cast<const f32x4*>(lval + k);
#pragma unroll
        for (int u = 0; u < 4; ++u) s += i[u] == j ? e[u] : 0.f;
    }
    return s;
}

// Which classes does the list name more than once?  Long lists (K > 64) keep a table of their classes with counts (whole
// numbers: any order), so that only those are summed over the list: the sum for every entry took 120 us at K = 1024.  Short
// lists are summed for every entry.
struct Named {
    int *key, *count;
    int mask;  // places - 1; 0: no table
};
__device__ __forceinline__ int table_size(int K) {  // a power of two, half full at most
    return K <= 64 ? 0 : 1 << (32 - __builtin_clz(2 * K - 1));
}
__device__ __forceinline__ void clear_named(const Named& d, int t, int nt) {
    if (d.mask)
        for (int i = t; i <= d.mask; i += nt) {
            d.key[i] = -1;
            d.count[i] = 0;
        }
}
__device__ __forceinline__ void add_named(const Named& d, int j) {
    if (!d.mask) return;
    int p = (int)((unsigned)j * 2654435761u >> 8) & d.mask;
    for (;;) {  // (ends: the table is never full)
        const int old = atomicCAS(&d.key[p], -1, j);
        if (old == -1 || old == j) break;
        p = (p + 1) & d.mask;
    }
    atomicAdd(&d.count[p], 1);
}
__device__ __forceinline__ bool named_twice(const Named& d, int j) {
    if (!d.mask) return true;
    int p = (int)((unsigned)j * 2654435761u >> 8) & d.mask;
    while (d.key[p] != j) p = (p + 1) & d.mask;  // (it is there)
    return d.count[p] > 1;
}
// the gradient's second part at the class of entry k
__device__ __forceinline__ float list_part(const Named& d, const int* lidx, const float* lval, int K, int k) {
    return named_twice(d, lidx[k]) ? listed(lidx, lval, K, lidx[k]) : lval[k];
}

// A row in the registers of W waves: NC chunks of 8 classes a thread.  The last, partial chunk of a row is taken as the row's
// last eight classes: the classes it shares with its neighbour are counted once and stored twice, with the same bits (V < 8:
// EL, element by element).  A workgroup walks rows a grid apart; the next row's logits, list and scalars are requested before
// this row's gradient is stored, so that its memory latency runs under the stores.
template <typename T, typename TD, int W, int NC, bool EL, bool GRAD, int RPB>
__global__ __launch_bounds__(64 * W * RPB) void distill_row_kernel(Args a) {
    constexpr int NT = 64 * W;  // threads of a row; RPB rows a workgroup (W = 1)
    constexpr bool AHEAD = W < 16;  // (sixteen waves: 128 registers a thread hold one row)
    extern __shared__ __attribute__((aligned(16))) float dyn[];
    __shared__ float red[6 * W + RPB];
    const int t = W == 1 ? (threadIdx.x & 63) : threadIdx.x, sub = W == 1 ? (threadIdx.x >> 6) : 0;
    const int K4 = list_pitch(a.K), NP = table_size(a.K);
    float* lval = dyn + sub * (3 * K4 + 2 * NP);             // e of an entry
    float* lstu = lval + K4;                                 // the student's exponential at its class
    int* lidx = reinterpret_cast<int*>(lval + 2 * K4);
    const Named named{lidx + K4, lidx + K4 + NP, max(NP - 1, 0)};
    end_list(a.K, t, lidx);
    const float k2 = a.it * 1.4426950408889634f;
    const int V = (int)a.V;
    const int64_t step = (int64_t)gridDim.x * RPB;

    Raw8<T> raw[NC];
    float el[8];                                             // (EL)
    float w, lse, ltop;
    int lilo, lihi;
    const float* pw = a.weight ? a.weight : a.part;
    const float* plse = a.lse ? a.lse : a.part;
    const float* ptop = a.K > 0 ? a.top : a.part;
    const int* pidx = reinterpret_cast<const int*>(a.K > 0 ? a.idx : a.part);
    const int64_t pldi = a.K > 0 ? a.ldi : 0, pldt = a.K > 0 ? a.ldt : 0;
    auto fetch = [&](int64_t b) {
        const T* s = reinterpret_cast<const T*>(a.s) + b * a.lds;
        if (EL) load_row8(s, (int64_t)t * 8, a.V, el, -INFINITY);
        else {
#pragma unroll
            for (int c = 0; c < NC; ++c) raw[c] = raw8(s + min((c * NT + t) * 8, V - 8));
        }
        // (absent vectors and lists: some address that can be read, so that nothing here is conditional; `b` made a vector
        // value, or the scalars would be moved to scalar registers at once, and waited for)
        int64_t bv = b;
        asm volatile("" : "+v"(bv));
        const int k = max(0, min(t, a.K - 1));
        lilo = pidx[(bv * pldi + k) * a.iw];
        lihi = pidx[(bv * pldi + k) * a.iw + a.iw - 1];
        ltop = ptop[bv * pldt + k];
        w = pw[a.weight ? bv : 0];
        lse = plse[a.lse ? bv : 0];
    };
    float total = 0.f;
    int64_t b = (int64_t)blockIdx.x * RPB + sub;
    float v[NC][8];  // (a NaN is no maximum; its exponential makes Z, and so the row, NaN)
    float tv, rw, rlse;
    int64_t li;
    auto take = [&]() {  // what was requested, as values: at the end of the row before, where the stores behind the requests
                         // can be counted (at the loop's head they could not, and would be waited for)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (EL) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] = el[i];
            } else {
                unraw8(raw[c], v[c]);
            }
        }
        li = join_index(a, lilo, lihi);
        tv = ltop;
        rw = a.weight ? w : 1.f;
        rlse = lse;
    };
    if (AHEAD && b < a.B) {
        fetch(b);
        take();
    }
    for (; b < a.B; b += step) {
        if (!AHEAD) {
            fetch(b);
            take();
        }
        const T* s = reinterpret_cast<const T*>(a.s) + b * a.lds;
        TD* ds = reinterpret_cast<TD*>(a.ds) + b * a.ldds;  // (GRAD)
        sync_row<W>();  // the row before is done with the lists and with red
        clear_named(named, t, NT);
        // this thread's list entry (entries beyond one a thread: read here)
        const bool mine = t < a.K, on = mine && li >= 0 && li < a.V;
        if (mine && li >= a.V && a.status) *a.status = 1;
        const float sj = load1(s + (on ? li : 0));           // the student's logit there
        float m[2] = {-INFINITY, on ? in_max(tv) : -INFINITY};
        if (mine) {
            lidx[t] = on ? (int)li : -1;
            lval[t] = tv;
        }
        for (int k = t + NT; k < a.K; k += NT) {
            const int64_t i = list_index(a, b, k);
            const float x = a.top[b * a.ldt + k];
            const bool o = i >= 0 && i < a.V;
            if (i >= a.V && a.status) *a.status = 1;
            lidx[k] = o ? (int)i : -1;
            lval[k] = x;
            if (o) m[1] = fmaxf(m[1], in_max(x));
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) m[0] = fmaxf(m[0], v[c][i]);
        row_reduce<W, 2, true>(m, red);
        const bool skip = rw == 0.f || m[1] == -INFINITY;    // (uniform over the row)
        const float ms = m[0], mt = a.lse ? rlse : m[1];
        float r[4] = {0.f, 0.f, 0.f, 0.f};  // Z, z, U, W
        float P = 0.f, zn = 1.f;
        if (!skip) {
            for (int k = t; k < a.K; k += NT) {
                const int j = lidx[k];
                if (j < 0) continue;
                add_named(named, j);
                const float d = list_arg(a, lval[k], mt), e = expf(d), u = (k == t ? sj : load1(s + j)) - ms;
                if (!(e == 0.f)) {  // (0 * infinity where a class is impossible on both sides)
                    r[1] += e;
                    r[2] += e * d;
                    r[3] += e * (u * a.it);
                }
                lval[k] = e;
                lstu[k] = exp2_fast(u * k2);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] = exp2_fast((v[c][i] - ms) * k2);
                if (EL || (c + 1) * NT * 8 <= V) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) r[0] += v[c][i];
                } else {
                    const int sh = (c * NT + t) * 8 - min((c * NT + t) * 8, V - 8);  // classes that the neighbour counts
#pragma unroll
                    for (int i = 0; i < 8; ++i) r[0] += i >= sh ? v[c][i] : 0.f;
                }
            }
            row_reduce<W, 4, false>(r, red + 2 * W);
            zn = a.lse ? 1.f : r[1];
            P = a.lse || r[1] != r[1] ? r[1] : 1.f;  // (a NaN in the list: the row's)
            if (t == 0) total += rw * ((r[2] - r[3]) / zn - (a.lse ? 0.f : logf(r[1])) + P * logf(r[0]));
        }
        if (AHEAD) fetch(min(b + step, a.B - 1));
        if (GRAD) {
            const float cw = rw * a.T * a.inv_B, cq = skip ? 0.f : cw * P / r[0], cp = cw / zn;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int c0 = (c * NT + t) * 8;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] = skip ? 0.f : v[c][i] * cq;
                if (EL) store_row8(ds, c0, a.V, v[c]);
                else store8(ds + min(c0, V - 8), v[c]);  // (behind the row: its last classes again -- no branch between stores)
            }
            if (!skip) {
                sync_row<W>();  // the row pass's stores come before the listed classes'
                for (int k = t; k < a.K; k += NT)
                    if (lidx[k] >= 0) st_from_f32<TD>(ds + lidx[k], cq * lstu[k] - cp * list_part(named, lidx, lval, a.K, k));
            }
        }
        if (AHEAD) take();
    }
    if (RPB > 1) {
        __syncthreads();
        if (t == 0) red[sub] = total;
        __syncthreads();
        total = red[0];
#pragma unroll
        for (int i = 1; i < RPB; ++i) total += red[i];
    }
    if (threadIdx.x == 0) {
        total *= a.T * a.T * a.inv_B;
        if (a.only) *a.only = a.loss ? total : *a.only + total;  // the one workgroup of a small batch: the loss itself
        else a.part[blockIdx.x] = total;
        if (blockIdx.x == 0 && a.loss && !a.only) *a.loss = 0.f;
    }
}

// ---- rows in segments: ws = part [grid] | [B][S][2] segment maximum and sum | [B][K] the student's logits at the listed classes
__device__ __forceinline__ float* seg_stats(const Args& a, int64_t nseg, int64_t b) { return a.part + a.B + b * nseg * 2; }
__device__ __forceinline__ float* seg_listed(const Args& a, int64_t nseg, int64_t b) {
    return a.part + a.B + a.B * nseg * 2 + b * a.K;
}

template <typename T>
__global__ __launch_bounds__(256) void distill_seg_stats_kernel(Args a, int64_t nseg) {
    __shared__ float red[8];
    const int64_t b = blockIdx.x / nseg, g = blockIdx.x - b * nseg;
    const int t = threadIdx.x;
    if (a.weight && a.weight[b] == 0.f) return;
    const T* s = reinterpret_cast<const T*>(a.s) + b * a.lds;
    float v[4][8];
#pragma unroll
    for (int c = 0; c < 4; ++c) load_row8(s, g * kSeg + (c * 256 + t) * 8, a.V, v[c], -INFINITY);
    if (g == 0) {  // (before the second launch overwrites logits in place)
        for (int k = t; k < a.K; k += 256) {
            const int64_t i = list_index(a, b, k);
            if (i >= 0 && i < a.V) seg_listed(a, nseg, b)[k] = load1(s + i);
        }
    }
    float m[1] = {-INFINITY};
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) m[0] = fmaxf(m[0], v[c][i]);
    row_reduce<4, 1, true>(m, red);
    const float mz = m[0] == -INFINITY ? 0.f : m[0];  // (a segment of -infinity: sum 0; a NaN: sum NaN)
    const float k2 = a.it * 1.4426950408889634f;
    float z[1] = {0.f};
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) z[0] += exp2_fast((v[c][i] - mz) * k2);
    row_reduce<4, 1, false>(z, red + 4);
    if (t == 0) {
        seg_stats(a, nseg, b)[2 * g] = m[0];
        seg_stats(a, nseg, b)[2 * g + 1] = z[0];
    }
}

template <typename T, typename TD>
__global__ __launch_bounds__(256) void distill_seg_grad_kernel(Args a, int64_t nseg) {
    extern __shared__ __attribute__((aligned(16))) float dyn[];
    __shared__ float red[28];
    const int K4 = list_pitch(a.K), NP = table_size(a.K);
    float* lval = dyn;
    float* lstu = dyn + K4;
    int* lidx = reinterpret_cast<int*>(dyn + 2 * K4);
    const Named named{lidx + K4, lidx + K4 + NP, max(NP - 1, 0)};
    end_list(a.K, threadIdx.x, lidx);
    clear_named(named, threadIdx.x, 256);
    const int64_t b = blockIdx.x / nseg, g = blockIdx.x - b * nseg;
    const int t = threadIdx.x;
    if (blockIdx.x == 0 && t == 0 && a.loss) *a.loss = 0.f;
    const float w = a.weight ? a.weight[b] : 1.f;
    TD* ds = a.ds ? reinterpret_cast<TD*>(a.ds) + b * a.ldds : nullptr;
    const T* s = reinterpret_cast<const T*>(a.s) + b * a.lds;
    float v[4][8];
    if (ds && w != 0.f) {
#pragma unroll
        for (int c = 0; c < 4; ++c) load_row8(s, g * kSeg + (c * 256 + t) * 8, a.V, v[c], -INFINITY);
    }
    float m[2] = {-INFINITY, load_list(a, b, t, 256, lidx, lval, g == 0)};
    const float* st = seg_stats(a, nseg, b);
    if (w != 0.f)
        for (int64_t i = t; i < nseg; i += 256) m[0] = fmaxf(m[0], st[2 * i]);
    row_reduce<4, 2, true>(m, red);
    if (w == 0.f || m[1] == -INFINITY) {
        const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (ds) {
#pragma unroll
            for (int c = 0; c < 4; ++c) store_row8(ds, g * kSeg + (c * 256 + t) * 8, a.V, zero);
        }
        if (g == 0 && t == 0) a.part[b] = 0.f;
        return;
    }
    const float k2 = a.it * 1.4426950408889634f;
    const float ms = m[0], mt = a.lse ? a.lse[b] : m[1];
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t i = t; i < nseg; i += 256) r[0] += st[2 * i + 1] * exp2_fast((st[2 * i] - ms) * k2);
    for (int k = t; k < a.K; k += 256) {
        if (lidx[k] < 0) continue;
        add_named(named, lidx[k]);
        const float d = list_arg(a, lval[k], mt), e = expf(d), u = seg_listed(a, nseg, b)[k] - ms;
        if (!(e == 0.f)) {
            r[1] += e;
            r[2] += e * d;
            r[3] += e * (u * a.it);
        }
        lval[k] = e;
        lstu[k] = exp2_fast(u * k2);
    }
    row_reduce<4, 4, false>(r, red + 8);
    const float zn = a.lse ? 1.f : r[1], P = a.lse || r[1] != r[1] ? r[1] : 1.f;
    if (g == 0 && t == 0)
        a.part[b] = w * ((r[2] - r[3]) / zn - (a.lse ? 0.f : logf(r[1])) + P * logf(r[0])) * a.T * a.T * a.inv_B;
    if (!ds) return;
    const float cw = w * a.T * a.inv_B, cq = cw * P / r[0], cp = cw / zn;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = cq * exp2_fast((v[c][i] - ms) * k2);
        store_row8(ds, g * kSeg + (c * 256 + t) * 8, a.V, v[c]);
    }
    __syncthreads();
    for (int k = t; k < a.K; k += 256)
        if (lidx[k] >= 0 && lidx[k] / kSeg == g)
            st_from_f32<TD>(ds + lidx[k], cq * lstu[k] - cp * list_part(named, lidx, lval, a.K, k));
}

// Rows in segments?  Beyond the 32 768 classes that a workgroup keeps in registers.  (At 19 000 classes the register form is
// ahead from one row on: 9 us against 12.)
inline bool in_segments(int64_t V) { return V > 32768; }
inline int64_t n_seg(int64_t V) { return (V + kSeg - 1) / kSeg; }
// A few short rows: one workgroup of sixteen waves, which writes the loss itself -- one launch instead of two.  (A row takes a
// wave 2.5 us: at 128 rows eight rows a wave took 21 us, 32 workgroups and the second launch 6.5.)
inline bool one_group(int64_t B, int64_t V, int K) { return V <= 1024 && B <= 16 && K <= 64; }
// Workgroups (= partial losses): as many as the chip holds at once, each walks rows.
inline int n_part(int64_t B, int64_t V, int K) {
    if (in_segments(V)) return (int)B;
    if (one_group(B, V, K)) return 1;
    if (V <= 1024) return (int)std::min<int64_t>((B + 3) / 4, 256 * 6);
    return (int)std::min<int64_t>(B, 256 * (V <= 4096 ? 6 : V <= 20480 ? 2 : 1));
}

template <typename T, typename TD, bool GRAD>
int run(const Args& a, hipStream_t st) {
    size_t places = a.K <= 64 ? 0 : 1;
    while (places && places < 2 * (size_t)a.K) places *= 2;
    const size_t list = (size_t)((a.K + 3) / 4 * 4) * 12 + places * 8;  // (at most 28 KB; four rows of them 113 KB)
    if (in_segments(a.V)) {
        const int64_t ns = n_seg(a.V);
        if (a.B * ns >= (1ll << 24)) return 1;  // (a launch's grid: 2^32 threads)
        hipLaunchKernelGGL((distill_seg_stats_kernel<T>), dim3((unsigned)(a.B * ns)), dim3(256), 0, st, a, ns);
        hipLaunchKernelGGL((distill_seg_grad_kernel<T, TD>), dim3((unsigned)(a.B * ns)), dim3(256), list, st, a, ns);
        return 0;
    }
    const int grid = n_part(a.B, a.V, a.K);
#define ROWK(W, NC, EL, RPB)                                                                                                 \
    do {                                                                                                                     \
        auto k = distill_row_kernel<T, TD, W, NC, EL, GRAD, RPB>;                                                            \
        const size_t l = RPB * list;                                                                                         \
        if (l > 48 * 1024) (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)l);    \
        hipLaunchKernelGGL(k, dim3(grid), dim3(64 * W * RPB), l, st, a);                                                     \
    } while (0)
#define ROW(W, NC) ROWK(W, NC, false, 1)
#define SHORT(NC, EL)                                                                                 \
    do {                                                                                              \
        if (one_group(a.B, a.V, a.K)) ROWK(1, NC, EL, 16);                                            \
        else ROWK(1, NC, EL, 4);                                                                      \
    } while (0)
    if (a.V < 8) {
        SHORT(1, true);
        return 0;
    }
    if (a.V <= 512) SHORT(1, false);
    else if (a.V <= 1024) SHORT(2, false);
    else if (a.V <= 2048) ROW(4, 1);
    else if (a.V <= 4096) ROW(4, 2);
    else if (a.V <= 8192) ROW(8, 2);
    else if (a.V <= 12288) ROW(8, 3);
    else if (a.V <= 20480) ROW(8, 5);
    else ROW(16, 4);
#undef SHORT
#undef ROW
#undef ROWK
    return 0;
}

}  // namespace distill
}  // namespace c2

extern "C" size_t c2_distill_topk_ws(int64_t B, int64_t V, int K) {
    using namespace c2::distill;
    if (B <= 0 || V <= 0) return 0;
    if (!in_segments(V)) return (size_t)std::max(n_part(B, V, K), 4);
    return (size_t)B * (1 + 2 * (size_t)n_seg(V) + (size_t)std::max(K, 0));
}

extern "C" int c2_distill_topk_fwd_bwd(const void* logits, int l_dtype, int64_t ldl, const void* top_idx, int idx_bytes,
                                       int64_t ldi, const float* top_logits, int64_t ldt, int K, const float* teacher_lse,
                                       const float* weight, float temperature, int64_t B, int64_t V, float inv_B,
                                       float* loss_out, int loss_add, void* dlogits, int dl_dtype, int64_t lddl, float* ws,
                                       int32_t* status_dev, void* stream) {
    using namespace c2;
    C2_CHECK(B >= 0 && V >= 0 && V < (1ll << 31) && K >= 0, "bad shape");
    C2_CHECK(K <= distill::kMaxList, "at most 1024 teacher entries per row");
    C2_CHECK(l_dtype == C2_F32 || l_dtype == C2_BF16 || l_dtype == C2_F16, "bad logits dtype");
    C2_CHECK(dl_dtype == C2_F32 || dl_dtype == C2_BF16, "bad gradient dtype");
    C2_CHECK(idx_bytes == 4 || idx_bytes == 8, "idx_bytes: 4 (int32) or 8 (int64)");
    C2_CHECK(temperature > 0.f && temperature < INFINITY, "temperature must be positive and finite");
    // (its square scales the loss, log2(e) / T the exponents: below, the one loses its bits and the other is infinite)
    C2_CHECK(temperature * temperature >= 1.17549435e-38f && temperature * temperature < INFINITY,
             "temperature: its square must be a normal fp32 number");
    C2_CHECK(B > 0 && V > 0 || loss_add, "an empty batch has no loss to set: clear it and add");
    if (B == 0 || V == 0) return 0;
    C2_CHECK(logits && loss_out && ws && ldl >= V && (!dlogits || lddl >= V), "bad arguments");
    C2_CHECK(K == 0 || (top_idx && top_logits && ldi >= K && ldt >= K), "bad teacher list");
    C2_CHECK(dlogits != logits || (l_dtype == dl_dtype && ldl == lddl), "in place needs the logits' own type and pitch");
    hipStream_t st = (hipStream_t)stream;
    distill::Args a{logits, top_idx, top_logits, teacher_lse, weight, dlogits, ws, nullptr, loss_add ? nullptr : loss_out, status_dev, ldl, lddl, ldi, ldt, B, V, K, idx_bytes / 4,
                    1.f / temperature, temperature, inv_B};
    if (distill::one_group(B, V, K)) {  // (unless the loss's second stage is left to the next combine)
        const bool later = set_defer_sums(false);
        set_defer_sums(later);
        if (!later) a.only = loss_out;
    }
    int rc;
#define GO(T) rc = !dlogits ? distill::run<T, float, false>(a, st)                  \
                 : dl_dtype == C2_F32 ? distill::run<T, float, true>(a, st)       \
                                      : distill::run<T, bf16_t, true>(a, st)
    if (l_dtype == C2_F32) GO(float);
    else if (l_dtype == C2_BF16) GO(bf16_t);
    else GO(f16_t);
#undef GO
    C2_CHECK(rc == 0, "too many rows for one launch");
    if (!a.only) launch_finalize_sum(ws, distill::n_part(B, V, K), loss_out, st);
    C2_LAUNCH_CHECK();
    return 0;
}
