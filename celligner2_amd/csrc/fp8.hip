// 8-bit floating-point operands with one power-of-two scale per block of 128 (quantiser), for gfx950.
//
// Form.  A block is 128 neighbours along the reduction (or 128 x 128: weights).  amax = m 2^E over its FINITE elements,
// 1 <= m < 2; its scale is 2^s with the smallest s that brings amax under the format's largest number (448 = 1.75 * 2^8 for
// e4m3, 57344 = 1.75 * 2^15 for e5m2): s = E - 8 (E - 15), one more when m > 1.75; s >= -126; s = 0 for a block of zeros.
// Elements are x * 2^-s (exact: a power of two) rounded once, to nearest even, by the conversion instruction.  A power of two
// costs no accuracy in a floating format, and the matrix instruction applies it itself: v_mfma_scale_f32_16x16x128_f8f6f4
// multiplies 128 of the reduction at once and takes an exponent byte (s + 127) per row of either operand, so a block of 128 is
// one instruction and scaling costs no vector arithmetic.
//
// Operand layout.  q [rows][ldq] bytes, ldq >= cols rounded up to 128; the columns behind the last one up to that multiple
// hold zeros (written here), so that products run over whole blocks.  Scales are laid out for the product's register: byte
//   ((kb * R64 + row / 64) * 16 + row % 16) * 4 + (row / 16) % 4,   kb = block along the reduction, R64 = ceil(rows / 64):
// the dword a lane loads holds its row of the four 16-row fragments of a 64-row group, and the instruction's byte selector
// picks the fragment.  The scale of a 128 x 128 block is written to each of its rows (0.8 % of the bytes).
#include <algorithm>

#include "common.h"
#include "fp8.h"

namespace c2 {
namespace fp8 {

constexpr int64_t kMaxBlocks = 1ll << 24;  // of 256 threads: a launch's grid holds 2^32 threads at most

// Blocks of 1 x 128, row-wise only: a wave takes 512 columns of a row, 16 lanes a block, 8 elements a lane.  Bound by memory, and
// at small sizes by the launch: 4096 x 19 000 in bf16 40 us (234 MB), in fp32 66 us (389 MB), 5.9 TB/s either; 4096 x 1024 6.1 us.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int64_t cols,
                                                         int64_t nchunk, uint8_t* __restrict__ q, int64_t ldq,
                                                         uint8_t* __restrict__ scale) {
    const int lane = threadIdx.x & 63;
    const int64_t wid = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t row = wid / nchunk, c = (wid - row * nchunk) * 512 + lane * 8;
    if (row >= rows) return;
    float v[8];
    load_row8(x + row * ldx, c, cols, v);
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(v[i]));
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    const int s = block_exponent<FMT>(m);
    const float inv = exp2i(-s);
    if (c < (cols + 127) / 128 * 128) {
        u32x2 o;
        o[0] = pack8<FMT>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        o[1] = pack8<FMT>(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
        *reinterpret_cast<u32x2*>(q + row * ldq + c) = o;
        if ((lane & 15) == 0) scale[scale_at(c >> 7, (rows + 63) >> 6, row)] = (uint8_t)(s + 127);
    }
}

// A 128 x 128 tile read once: row-wise blocks (ROWS), blocks along the rows of the transposed operand (COLS), or both; SQ: one
// block for the tile.  A thread holds 8 rows x 8 columns; the transposed tile goes through LDS (16-byte stores, 128 bytes a row).
// Bound by memory: 4096 x 19 000 in bf16, both layouts, 66-70 us (311 MB: 4.5 TB/s, 0.9 of a large copy's rate); 777 x 19 001 in
// fp32 23.2 us (89 MB: 3.8 TB/s).  Rows whose ends cut a group of eight take the edge path's clamped loads: element by element
// the last column tile alone held the launch up.
template <typename T, int FMT, bool ROWS, bool COLS, bool SQ>
__global__ __launch_bounds__(256) void quant_tile_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int64_t cols,
                                                         int64_t tiles_c, uint8_t* __restrict__ q, int64_t ldq,
                                                         uint8_t* __restrict__ scale, uint8_t* __restrict__ qt,
                                                         int64_t ldqt, uint8_t* __restrict__ scale_t) {
    __shared__ float red[4][128];
    __shared__ __attribute__((aligned(16))) uint8_t tile[COLS ? 128 * 128 : 16];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, c8 = t & 15, r8 = t >> 4;
    const int64_t tr = blockIdx.x / tiles_c, tc = blockIdx.x - tr * tiles_c;
    const int64_t row0 = tr * 128, col0 = tc * 128, c = col0 + c8 * 8;
    float v[8][8];
    if (row0 + 128 <= rows && col0 + 128 <= cols) {  // an interior tile: eight loads on their way at once
        Raw8<T> raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = raw8(x + (row0 + r8 * 8 + i) * ldx + c);
#pragma unroll
        for (int i = 0; i < 8; ++i) unraw8(raw[i], v[i]);
    } else if (cols >= 8) {  // at the matrix's edge: the row's last eight elements moved to their places, zeros behind
        const int64_t cc = min(c, cols - 8);
        const int sh = (int)min(c - cc, (int64_t)8);
        Raw8<T> raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = raw8(x + min(row0 + r8 * 8 + i, rows - 1) * ldx + cc);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            unraw8(raw[i], v[i]);
#pragma unroll
            for (int b = 1; b <= 4; b <<= 1)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = (sh & b) ? (j + b < 8 ? v[i][j + b] : 0.f) : v[i][j];
            const bool in = sh < 8 && row0 + r8 * 8 + i < rows;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = in ? v[i][j] : 0.f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = min(row0 + r8 * 8 + i, rows - 1);
            load_row8(x + r * ldx, c, cols, v[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = row0 + r8 * 8 + i < rows ? v[i][j] : 0.f;
        }
    }
    float rm[8], cm[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) rm[j] = cm[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float a = finite_abs(v[i][j]);
            rm[i] = fmaxf(rm[i], a);
            cm[j] = fmaxf(cm[j], a);
        }
    if (SQ) {
        float m = rm[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) m = fmaxf(m, rm[i]);
        m = block_max<256>(m, &red[0][0]);
#pragma unroll
        for (int i = 0; i < 8; ++i) rm[i] = cm[i] = m;
    } else {
        if (ROWS) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int o = 1; o < 16; o <<= 1) rm[i] = fmaxf(rm[i], __shfl_xor(rm[i], o, 64));
        }
        if (COLS) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int o = 16; o < 64; o <<= 1) cm[j] = fmaxf(cm[j], __shfl_xor(cm[j], o, 64));
            if (lane < 16) {
#pragma unroll
                for (int j = 0; j < 8; ++j) red[wave][c8 * 8 + j] = cm[j];
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 8; ++j)
                cm[j] = fmaxf(fmaxf(red[0][c8 * 8 + j], red[1][c8 * 8 + j]), fmaxf(red[2][c8 * 8 + j], red[3][c8 * 8 + j]));
        }
    }
    if (ROWS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = row0 + r8 * 8 + i;
            const int s = block_exponent<FMT>(rm[i]);
            const float inv = exp2i(-s);
            if (r < rows) {
                u32x2 o;
                o[0] = pack8<FMT>(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
                o[1] = pack8<FMT>(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
                *reinterpret_cast<u32x2*>(q + r * ldq + c) = o;
                if (c8 == 0) scale[scale_at(tc, (rows + 63) >> 6, r)] = (uint8_t)(s + 127);
            }
        }
    }
    if (COLS) {
        // granule g (8 rows) of column k sits at granule g ^ (k / 8) of the tile's row k: the sixteen column groups of a
        // wave's write fall on sixteen different granules
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int s = block_exponent<FMT>(cm[j]);
            const float inv = exp2i(-s);
            u32x2 o;
            o[0] = pack8<FMT>(v[0][j] * inv, v[1][j] * inv, v[2][j] * inv, v[3][j] * inv);
            o[1] = pack8<FMT>(v[4][j] * inv, v[5][j] * inv, v[6][j] * inv, v[7][j] * inv);
            *reinterpret_cast<u32x2*>(tile + (c8 * 8 + j) * 128 + ((r8 ^ c8) << 3)) = o;
            if (r8 == 0 && c + j < cols) scale_t[scale_at(tr, (cols + 63) >> 6, c + j)] = (uint8_t)(s + 127);
        }
        __syncthreads();
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const int k = it * 32 + (t >> 3), p = t & 7;
            if (col0 + k < cols) {
                const u32x2 lo = *reinterpret_cast<const u32x2*>(tile + k * 128 + (((2 * p) ^ (k >> 3)) << 3));
                const u32x2 hi = *reinterpret_cast<const u32x2*>(tile + k * 128 + (((2 * p + 1) ^ (k >> 3)) << 3));
                *reinterpret_cast<u32x4*>(qt + (col0 + k) * ldqt + row0 + p * 16) = u32x4{lo[0], lo[1], hi[0], hi[1]};
            }
        }
    }
}

template <typename T, int FMT>
int quant_run(const T* x, int64_t ldx, int64_t rows, int64_t cols, int block_rows, uint8_t* q, int64_t ldq, uint8_t* scale,
              uint8_t* qt, int64_t ldqt, uint8_t* scale_t, hipStream_t st) {
    if (q && !qt && block_rows == 1) {
        const int64_t nchunk = (cols + 511) / 512, nb = (rows * nchunk + 3) / 4;
        if (nb >= kMaxBlocks) return 3;
        hipLaunchKernelGGL((quant_rows_kernel<T, FMT>), dim3((unsigned)nb), dim3(256), 0, st, x, ldx, rows, cols, nchunk, q, ldq,
                           scale);
        return 0;
    }
    const int64_t tc = (cols + 127) / 128, nb = (rows + 127) / 128 * tc;
    if (nb >= kMaxBlocks) return 3;
#define QT(R, C_, S)                                                                                                       \
    hipLaunchKernelGGL((quant_tile_kernel<T, FMT, R, C_, S>), dim3((unsigned)nb), dim3(256), 0, st, x, ldx, rows, cols, tc, q, \
                       ldq, scale, qt, ldqt, scale_t)
    if (block_rows == 128) {
        if (q && qt) QT(true, true, true);
        else if (q) QT(true, false, true);
        else QT(false, true, true);
    } else {
        if (q) QT(true, true, false);
        else QT(false, true, false);
    }
#undef QT
    return 0;
}

}  // namespace fp8
}  // namespace c2

extern "C" size_t c2_fp8_scale_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return (size_t)((cols + 127) / 128) * (size_t)((rows + 63) / 64) * 64;
}

extern "C" int c2_quant_fp8(const void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t cols, int block_rows, int fmt,
                            void* q, int64_t ldq, uint8_t* scale, void* qt, int64_t ldqt, uint8_t* scale_t, void* stream) {
    using namespace c2;
    C2_CHECK(rows >= 0 && cols >= 0, "negative size");
    C2_CHECK(block_rows == 1 || block_rows == 128, "block_rows: 1 or 128");
    C2_CHECK(fmt == C2_E4M3 || fmt == C2_E5M2, "fmt: C2_E4M3 or C2_E5M2");
    C2_CHECK(x_dtype == C2_F32 || x_dtype == C2_BF16 || x_dtype == C2_F16, "bad dtype");
    C2_CHECK(q || qt, "no output");
    if (rows == 0 || cols == 0) return 0;
    C2_CHECK(x && ldx >= cols, "bad input");
    C2_CHECK(!q || (scale && ldq >= (cols + 127) / 128 * 128 && (ldq & 15) == 0 && aligned16(q)),
             "q: rows of cols rounded up to 128 bytes, starting on 16 bytes, and scales");
    C2_CHECK(!qt || (scale_t && ldqt >= (rows + 127) / 128 * 128 && (ldqt & 15) == 0 && aligned16(qt)),
             "qt: rows of rows rounded up to 128 bytes, starting on 16 bytes, and scales");
    hipStream_t st = (hipStream_t)stream;
    int rc;
#define QR(T, F)                                                                                                          \
    rc = fp8::quant_run<T, F>((const T*)x, ldx, rows, cols, block_rows, (uint8_t*)q, ldq, scale, (uint8_t*)qt, ldqt, scale_t, st)
    if (fmt == C2_E4M3) {
        if (x_dtype == C2_F32) QR(float, C2_E4M3);
        else if (x_dtype == C2_BF16) QR(bf16_t, C2_E4M3);
        else QR(f16_t, C2_E4M3);
    } else {
        if (x_dtype == C2_F32) QR(float, C2_E5M2);
        else if (x_dtype == C2_BF16) QR(bf16_t, C2_E5M2);
        else QR(f16_t, C2_E5M2);
    }
#undef QR
    C2_CHECK(rc == 0, "too many blocks for one launch");
    C2_LAUNCH_CHECK();
    return 0;
}
