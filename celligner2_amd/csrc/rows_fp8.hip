// 8-bit block-scaled products with few rows (a served query, a small batch, the last few cells of a batch), for gfx950.
//
// Bound by the weight's bytes: every weight byte goes from memory to one lane's registers and from there into matrix
// instructions, v_mfma_scale_f32_16x16x128_f8f6f4 (16 rows of the weight x 16 rows of x x one scale block) for 16-bit results, or,
// widened there, four v_mfma_f32_16x16x32_bf16 for fp32 results (what either keeps: gemm_fp8.hip); nothing of it passes
// through LDS.  x is small: each workgroup brings what it needs of it (at most 384 blocks of a row, 48 KB) to
// LDS in 8 bits -- quantised there, exactly as c2_quant_fp8 does, when it comes as fp32, bf16 or half.  The first weight blocks
// of a wave are requested before x is quantised.
// A short reduction is ONE launch: a workgroup's waves are laid out NWN x NWK, 16 columns each, and NWK of them share a column
// group's reduction; the parts meet in LDS, in a fixed order.  One row, 19 000 columns, reduction 1024 (19.5 MB of weight): 5.9 us
// replayed with the weight in the caches, 7.8 (2.5 TB/s) in a run of its own.  A longer one: a workgroup of eight waves takes 128
// columns and a part of the reduction, and a second launch joins the parts.
#include <algorithm>

#include "fp8.h"

namespace c2 {
namespace fp8 {

struct RowArgs {
    const void* A;
    const uint8_t* sA;
    const uint8_t* B;
    const uint32_t* sB;
    void* Y;
    const float* bias;
    const float* alpha_dev;
    int64_t lda, ldb, ldy, K;
    int64_t slab;  // elements between the parts of Y where the workgroups share the reduction
    int M, N, nkb, a64, b64, nwk, lm;  // lm: log2 of the rows kept in LDS (M rounded up to a power of two)
    int kb_per_split;
};

constexpr int kUnits = 384;  // (scale block, row) pairs of x that a workgroup takes at most (row_plan's limits), 48 KB in LDS
constexpr int kAhead = 4;   // weight blocks of a wave on their way at once

// XT: float, bf16_t, f16_t, or uint8_t (already in 8 bits, format AF); MF: groups of 16 rows;
// PARTS: a workgroup takes a part of the reduction (else all of it, shared by its waves; MF = 1); WIDE: fp32 results
template <typename XT, int AF, typename TY, int MF, bool PARTS, bool WIDE>
__global__ __launch_bounds__(PARTS ? 512 : 1024) void few_rows_kernel(RowArgs a) {
    constexpr int U = MF == 1 ? 1 : 4;  // pieces of x that a thread has on their way (up to 16 rows have one a thread, mostly)
    extern __shared__ __attribute__((aligned(16))) char xs[];  // [block][row][128], chunk c of row r at c ^ (r / 2) % 8
    __shared__ uint8_t xe[kUnits];                             // exponent bytes [block][row]
    f32x4 (*red)[64] = reinterpret_cast<f32x4 (*)[64]>(xs);    // (at the end)
    const int m0 = PARTS ? (int)blockIdx.z * 64 : 0, M = PARTS ? min(a.M - m0, 64) : a.M;  // this workgroup's rows
    const int rows = (1 << a.lm) - 1;
    const int nthr = blockDim.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int nwn = (nthr >> 6) / a.nwk, wk = wave % a.nwk, wn = wave / a.nwk;
    const int n0 = ((int)blockIdx.x * nwn + wn) * 16;
    const int x = lane & 15, g = lane >> 4;
    const uint8_t* wrow = a.B + (int64_t)min(n0 + x, a.N - 1) * a.ldb + g * 16;
    const uint32_t* wscale = a.sB + min(n0 >> 6, a.b64 - 1) * 16 + x;
    const int wshift = ((n0 >> 4) & 3) * 8;

    // (lanes of rows behind the last one take another row's: columns of the result that nobody stores)
    const int xm = x & ((1 << a.lm) - 1), xz = (xm >> 1) & 7;
    const int kb0 = PARTS ? (int)blockIdx.y * a.kb_per_split : 0, nb = !PARTS ? a.nkb : min(a.nkb - kb0, a.kb_per_split);
    f32x4 acc[MF];
#pragma unroll
    for (int f = 0; f < MF; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    // this wave's blocks: wk, wk + nwk, ...
    u32x4 lo[kAhead], hi[kAhead];
    uint32_t ws[kAhead];
    auto request = [&](int k, int u) {
        const int kb = kb0 + k;
        const uint8_t* p = wrow + (int64_t)kb * 128;
        lo[u] = *reinterpret_cast<const u32x4*>(p);
        hi[u] = *reinterpret_cast<const u32x4*>(p + 64);
        ws[u] = wscale[(int64_t)kb * a.b64 * 16];
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
        if (wk + u * a.nwk < nb) request(wk + u * a.nwk, u);

    // x, blocks kb0 .. kb0 + nb: sixteen threads a block of a row (places behind the last row: that row again)
    if constexpr (sizeof(XT) == 1) {
        for (int i = threadIdx.x; i < nb << (a.lm + 3); i += nthr) {
            const int c = i & 7, at = i >> 3, kb = at >> a.lm, r = at & rows;
            const int64_t m = min(m0 + r, a.M - 1);
            *reinterpret_cast<u32x4*>(xs + at * 128 + ((c ^ ((r >> 1) & 7)) << 4)) = *reinterpret_cast<const u32x4*>(
                reinterpret_cast<const uint8_t*>(a.A) + m * a.lda + (int64_t)(kb0 + kb) * 128 + c * 16);
            if (c == 0) xe[at] = a.sA[scale_at(kb0 + kb, a.a64, m)];
        }
    } else {
        const int total = nb << (a.lm + 4);
        for (int i0 = 0; i0 < total; i0 += nthr * U) {  // (all lanes stay: sixteen of them find a block's largest together)
            Raw8<XT> raw[U];
            const XT* row[U];
            int64_t col[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {  // (behind the end: the last piece again; behind a row's end: its last eight)
                const int i = min(i0 + u * nthr + (int)threadIdx.x, total - 1), at = i >> 4;
                row[u] = reinterpret_cast<const XT*>(a.A) + (int64_t)min(m0 + (at & rows), a.M - 1) * a.lda;
                col[u] = (int64_t)(kb0 + (at >> a.lm)) * 128 + (i & 15) * 8;
                if (a.K >= 8) raw[u] = raw8(row[u] + min(col[u], a.K - 8));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i0 + u * nthr >= total) break;  // (uniform)
                const int i = i0 + u * nthr + threadIdx.x, t = threadIdx.x & 15, at = i >> 4, r = at & rows;
                float v[8];
                if (col[u] + 8 <= a.K) unraw8(raw[u], v);
                else load_row8(row[u], col[u], a.K, v);
                float m = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[j]));
#pragma unroll
                for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
                const int s = block_exponent<C2_E4M3>(m);
                const float inv = exp2i(-s);
                if (i < total) {
                    *reinterpret_cast<u32x2*>(xs + at * 128 + (((t >> 1) ^ ((r >> 1) & 7)) << 4) + (t & 1) * 8) =
                        u32x2{pack8<C2_E4M3>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                              pack8<C2_E4M3>(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)};
                    if (t == 0) xe[at] = (uint8_t)(s + 127);
                }
            }
        }
    }
    __syncthreads();
    for (int k0 = wk; k0 < nb; k0 += kAhead * a.nwk) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int k = k0 + u * a.nwk;
            if (k >= nb) break;  // (uniform over the wave)
            bf16x8 ww[WIDE ? 4 : 1];
            if constexpr (WIDE) {
                const float s = wide_scale(ws[u] >> wshift & 255u);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    ww[q] = widen8<C2_E4M3>(lo[u][2 * q], lo[u][2 * q + 1], s);
                    ww[2 + q] = widen8<C2_E4M3>(hi[u][2 * q], hi[u][2 * q + 1], s);
                }
            }
            const i32x8 fw = {(int)lo[u][0], (int)lo[u][1], (int)lo[u][2], (int)lo[u][3],
                              (int)hi[u][0], (int)hi[u][1], (int)hi[u][2], (int)hi[u][3]};
#pragma unroll
            for (int f = 0; f < MF; ++f) {
                const int at = (k << a.lm) + f * 16 + xm;
                const u32x4 xl = *reinterpret_cast<const u32x4*>(xs + at * 128 + ((g ^ xz) << 4));
                const u32x4 xh = *reinterpret_cast<const u32x4*>(xs + at * 128 + (((g + 4) ^ xz) << 4));
                if constexpr (WIDE) {  // (the lane's 32 bytes, eight at a time: the same reduction indices on both sides)
                    const float s = wide_scale(xe[at]);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const u32x4& v = q < 2 ? xl : xh;
                        acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ww[q], widen8<AF>(v[q % 2 * 2], v[q % 2 * 2 + 1], s), acc[f], 0, 0, 0);
                    }
                    continue;
                }
                const i32x8 fx = {(int)xl[0], (int)xl[1], (int)xl[2], (int)xl[3], (int)xh[0], (int)xh[1], (int)xh[2], (int)xh[3]};
                acc[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw, fx, acc[f], 0, AF, 0, (int)(ws[u] >> wshift), 0,
                                                                         (int)xe[at]);
            }
            if (k + kAhead * a.nwk < nb) request(k + kAhead * a.nwk, u);
        }
    }
    // lane l: row m = 16 f + l % 16 of the result, columns n0 + 4 (l / 16) + 0..3
    if constexpr (!PARTS) {
        __syncthreads();
        red[wave][lane] = acc[0];
        __syncthreads();
        if (wk != 0) return;
        for (int k = 1; k < a.nwk; ++k) acc[0] += red[wave + k][lane];
    }
    const float alpha = (WIDE ? kWideBack : 1.f) * (a.alpha_dev ? *a.alpha_dev : 1.f);
    const int n = n0 + 4 * g;
    float bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = a.bias && n + e < a.N ? a.bias[n + e] : 0.f;
    TY* y = reinterpret_cast<TY*>(a.Y) + (PARTS ? blockIdx.y * a.slab : 0) + (int64_t)(m0 + x) * a.ldy + n;
#pragma unroll
    for (int f = 0; f < MF; ++f, y += 16 * a.ldy) {
        if (f * 16 + x >= M) continue;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = alpha * acc[f][e] + bias[e];
        if (n + 4 <= a.N) {
            if constexpr (sizeof(TY) == 4) *reinterpret_cast<f32x4_a4*>(y) = f32x4{v[0], v[1], v[2], v[3]};
            else *reinterpret_cast<u32x2_a2*>(y) = u32x2{pack2<TY>(v[0], v[1]), pack2<TY>(v[2], v[3])};
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (n + e < a.N) st_from_f32<TY>(y + e, v[e]);
        }
    }
}

template <typename XT, int AF, int MF, bool PARTS>
void run_rows(const RowArgs& a, int y_dtype, bool wide, dim3 blocks, int threads, hipStream_t st) {
    // x, and room for the waves' parts
    const size_t lds = std::max((size_t)(a.kb_per_split << a.lm) * 128, PARTS ? 0 : (size_t)threads * 16);
#define ROWS(TY, WIDE) hipLaunchKernelGGL((few_rows_kernel<XT, AF, TY, MF, PARTS, WIDE>), blocks, dim3(threads), lds, st, a)
    if (y_dtype == C2_BF16) ROWS(bf16_t, false);
    else if (y_dtype == C2_F16) ROWS(f16_t, false);
    else if (wide) ROWS(float, true);
    else if constexpr (PARTS) ROWS(float, false);  // the parts of a 16-bit result
#undef ROWS
}

template <int MF, bool PARTS>
void run_types(const RowArgs& a, int x_dtype, int a_fmt, int y_dtype, bool wide, dim3 blocks, int threads, hipStream_t st) {
    if (x_dtype == C2_F32) run_rows<float, 0, MF, PARTS>(a, y_dtype, wide, blocks, threads, st);
    else if (x_dtype == C2_BF16) run_rows<bf16_t, 0, MF, PARTS>(a, y_dtype, wide, blocks, threads, st);
    else if (x_dtype == C2_F16) run_rows<f16_t, 0, MF, PARTS>(a, y_dtype, wide, blocks, threads, st);
    else if (a_fmt == C2_E4M3) run_rows<uint8_t, 0, MF, PARTS>(a, y_dtype, wide, blocks, threads, st);
    else run_rows<uint8_t, 1, MF, PARTS>(a, y_dtype, wide, blocks, threads, st);
}

// Which products are such, and how they are cut.
// In one launch: M rows times K / 128 blocks up to 128, since every workgroup quantises all of x (bf16, us, one launch against
// parts: 16 rows, 1024 columns, reduction 1024, 128 of them: 7.5, 7.8; 16 rows, 256, 19000, 2384: 46.8, 8.2; one row of that, 149:
// 13.4, 7.2); up to 64 where one part is all of it and needs no join either (16 rows, 19000, 1024: 13.7, 9.6).
// In parts: about one round of workgroups of 64 rows and 128 columns, at least two blocks each, where a workgroup's share of the
// reduction is short: 12 blocks for 32 rows, 6 for 64, and 3, in no more than one round, for 128.  Against quantising and the tiles
// of gemm_fp8.hip: 64 rows, 256 columns, reduction 1024 (2 blocks a workgroup) 8.9, 10.9; 4096, 4096 (4) 17.3, 21.6; 820, 19001 (5)
// 17.7, 21.9; 19000, 1024 (8) 17.7, 12.7; 32 rows, 1024, 19000 (5) 13.7, 17.8; 19000, 1024 (8) 11.8, 11.5; 8192, 8192 (16) 25.9, 22.7;
// 128 rows, 1024, 1024 (2) 10.0, 11.5; 4096, 1024 (2) 13.5, 15.2; 256, 19000 (3) 14.9, 16.1; 1024, 19000 (5, two rounds) 35.6, 19.5.
RowPlan row_plan(int64_t M, int64_t N, int64_t K) {
    const int64_t nkb = (K + 127) / 128, ct = (N + 127) / 128, room = M <= 64 ? 256 : 128;
    if (M > 128) return {RowPlan::kNone, 0, 0, 0};
    const int64_t s = std::max<int64_t>(1, std::min(nkb / 2, room / ct)), kb = (nkb + s - 1) / s;
    if (M <= 16 && M * nkb <= (s > 1 ? 128 : 64)) return {RowPlan::kOneLaunch, 1, (int)nkb, 0};
    if (kb > (M <= 32 ? 12 : M <= 64 ? 6 : 3) || (M > 64 && ct > room)) return {RowPlan::kNone, 0, 0, 0};
    return {RowPlan::kParts, (int)((nkb + kb - 1) / kb), (int)kb, (N + 3) / 4 * 4};
}

void launch_few_rows(const void* A, int x_dtype, int64_t lda, const uint8_t* sA, int a_fmt, const uint8_t* B, int64_t ldb,
                     const uint8_t* sB, int64_t M, int64_t N, int64_t K, void* Y, int y_dtype, int64_t ldy, const float* bias,
                     const float* alpha_dev, float* ws, hipStream_t st) {
    const int nkb = (int)((K + 127) / 128), nf = (int)((N + 15) / 16);
    RowArgs a{A, sA, B, (const uint32_t*)sB, Y, bias, alpha_dev, lda, ldb, ldy, K, 0, (int)M, (int)N, nkb, (int)((M + 63) / 64),
              (int)((N + 63) / 64), 1, 0, nkb};
    while (a.lm < 6 && (1 << a.lm) < M) ++a.lm;
    const RowPlan p = row_plan(M, N, K);
    const bool wide = y_dtype == C2_F32;
    if (p.form == RowPlan::kOneLaunch) {
        // waves that share a column group's reduction: about 4096 waves in all, two blocks of the reduction each at least; small
        // workgroups, which fill the CUs evenly
        int nwk = 1;
        while (nwk < 16 && nf * nwk < 4096 && nkb >= 4 * nwk) nwk *= 2;
        const int waves = std::max(nwk, 4), nwn = waves / nwk;
        a.nwk = nwk;
        run_types<1, false>(a, x_dtype, a_fmt, y_dtype, wide, dim3((nf + nwn - 1) / nwn), waves * 64, st);
        return;
    }
    a.kb_per_split = p.kb_per_split;
    if (p.splits > 1) {
        a.Y = ws;
        a.ldy = p.lds;
        a.slab = M * p.lds;
        a.bias = nullptr;
        a.alpha_dev = nullptr;
    }
    const dim3 grid((nf + 7) / 8, p.splits, (unsigned)((M + 63) / 64));
    const int yt = p.splits > 1 ? C2_F32 : y_dtype;
    if (M <= 16) run_types<1, true>(a, x_dtype, a_fmt, yt, wide, grid, 512, st);
    else if (M <= 32) run_types<2, true>(a, x_dtype, a_fmt, yt, wide, grid, 512, st);
    else run_types<4, true>(a, x_dtype, a_fmt, yt, wide, grid, 512, st);
    if (p.splits > 1) join_slabs(ws, M * p.lds, p.lds, p.splits, M, N, Y, y_dtype, ldy, bias, alpha_dev, st);
}

}  // namespace fp8
}  // namespace c2
