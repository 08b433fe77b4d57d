// Products of 8-bit block-scaled operands (fp8.hip):
//   Y[m][n] = alpha * sum_kb 2^(sA[m][kb] + sB[n][kb]) sum_{k in block kb} A[m][k] B[n][k]  (+ bias[n]),  fp32 accumulation.
// Forward, input gradient and weight gradient of a Linear layer are this one product (both operands row-wise along the
// reduction; the quantiser writes the transposed operand where the reduction runs over rows).
//
// 16-bit results: v_mfma_scale_f32_32x32x64_f8f6f4, two of them to a block of 128 of the reduction.  Lane l holds 32 bytes of row
// l % 32, and any assignment of the 64 reduction indices to (lane / 32, byte) is right as long as both operands use the same one:
// in step ks of a block a lane takes the 16-byte chunks 4 ks + 2 (l / 32) and the next one of its row.
// What that instruction keeps.  Measured on this chip, and the same for its 16x16x32 and 16x16x128 forms: the products of eight
// neighbours of the reduction are added in fixed point, each cut to a multiple of 2^(E - 13) with E the group's largest sum of
// exponents; the groups and the accumulator are then added in fp32.  A group of eight is so off by less than 7 * 2^-13 of its
// largest product (typically 1e-6 to 1e-4 of the result, always towards zero): far below the operands' own 2^-4 / 2^-3 and a
// 16-bit result's rounding, above fp32's.
// fp32 results: the same 32 bytes of a lane, widened in registers (fp8.h), are four v_mfma_f32_32x32x16_bf16, which keep 25 bits
// below a group's largest product and add the groups and the accumulator in fp32, to nearest (measured: over reductions of 512,
// 19 200 and 70 400 1e-7, 8e-7 and 1.6e-6 of the result's norm; fp32 arithmetic 1e-7, 6e-7 and 1.3e-6).
//
// Bound by the matrix unit where the reduction is long: 8192 x 8192 x 8192 takes 416 us, 2.64 PFLOP/s (the card's library: 2.69),
// in an unbroken row of twenty 480, where the clock gives way; the matrix unit is busy 0.70 of the time.  Short reductions are
// bound by their results: 4096 x 19 000 over 1024 takes 90-93 us (1.74 PFLOP/s), of which the five rounds' 33 MB of stores, which
// all CUs make at the same time, are a third.  fp32 results: 8192 cubed 960-975 us (1.13 PFLOP/s; the library's bf16 product
// 1.22; matrix unit busy 0.61), 1024 x 19 000 over 4096 150 us (88 with a 16-bit result), 4096 x 19 000 over 1024 183.
#include <algorithm>

#include "fp8.h"

namespace c2 {
namespace fp8 {

typedef __attribute__((address_space(3))) void lds_void;

constexpr int KB = 128;     // bytes (= elements) of a K-tile row
constexpr int GROUP_M = 8;  // tiles along M that share a panel of B

struct Args {
    const uint8_t* A;
    const uint8_t* B;
    const uint32_t* sA;
    const uint32_t* sB;
    void* Y;                // split 1: the result; else fp32 slabs [split][M][ldy]
    const float* bias;
    const float* alpha_dev;
    int64_t lda, ldb, ldy, slab;
    int M, N, nkb, kb_per_split;
    int a64, b64;           // 64-row groups of either operand's scales
    int b_off;              // the group in which B starts
};

// Item (a tile of one part of the reduction) -> split, tile: neighbours share panels of both operands.
__device__ __forceinline__ void map_item(int item, int tiles_m, int tiles_n, int& split, int& tm, int& tn) {
    const int tiles = tiles_m * tiles_n;
    split = item / tiles;
    const int t = item - split * tiles, per = GROUP_M * tiles_n, gid = t / per, first = gid * GROUP_M;
    const int gsz = min(tiles_m - first, GROUP_M), u = t - gid * per;
    tm = first + u % gsz;
    tn = u / gsz;
}

template <int N>
__device__ __forceinline__ void wait_vm() {  // all but the N newest vector-memory operations are complete
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// rows of the result: B's (first operand, e4m3), columns: A's (format AF); O*: the scale bytes
template <int AF, int OB, int OA>
__device__ __forceinline__ f32x16 mma(const i32x8& b, const i32x8& a, const f32x16& c, int sb, int sa) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, c, 0, AF, OB, sb, OA, sa);
}

// Tiles of 256 x 256 by eight waves (one workgroup a CU) and of 128 x 128 by four (two a CU).  Tried and left: 256 x 128 with
// stages of 64 bytes, two workgroups a CU (8192 cubed 514 us, 4096 x 19 000 over 1024 110); nontemporal stores of the results
// (that one 116 us for 110 in all, the three products of 4096 x 1024 x 19 000 391 for 366); workgroups started a tile's time apart.
//
// BM x BN tiles, WM x WN waves, each (BM / WM) x (BN / WN) as MI x NJ tiles of 32 x 32.  Operand tiles of 128 bytes of the
// reduction (one scale block) go to LDS by direct loads into two rings of RA and RB slots: while K-tile T is multiplied,
// B of T + RB - 1 and A of T + RA - 1 are on their way, and the wait before a tile's barrier is counted, so that they stay so.
// A slot's image is lane-linear; the chunk c (16 bytes) of row x sits at position c ^ (x / 2) % 8, which the source address
// of the load and the address of the fragment read both apply: no bank conflicts for 16 consecutive rows.  Rows behind the
// operand's last one lie outside the buffer resource and read as zeros.
// A K-tile is two steps of 64.  Right after its barrier all waves ask LDS for the first step's fragments, and multiply the
// second step of the tile BEFORE it meanwhile, which they hold in registers: the matrix unit has work under that burst.
// A workgroup walks items (tiles); the stream of loads does not stop between them: the last K-tiles' places ahead hold the
// next item's first ones, which arrive while the finished tile is stored (B's rows are the matrix unit's rows, so a lane
// holds neighbouring columns of the result).
// WIDE (fp32 results; 128 x 128 tiles, since the widened fragments of 256 x 256 do not fit the registers): a row of products is
// NJ x 4, on fragments of B widened once a step and one of A at a time.
template <int AF, typename TY, int BM, int BN, int WM, int WN, int RA, int RB, int WPE, bool WIDE>
__global__ __launch_bounds__(64 * WM * WN, WPE) void gemm_fp8_kernel(Args a, int tiles_m, int tiles_n, int items) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass knows no buffer resources, and drops the kernel's stub over them)
    constexpr int NW = WM * WN, RM = BM / WM, RN = BN / WN, MI = RM / 32, NJ = RN / 32;
    constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW;  // 1 KB pieces of an operand tile that a wave moves
    constexpr int SA = RM / 64, SB = RN / 64;          // scale words a lane needs per K-tile
    constexpr int TA = BM * KB, TB = BN * KB;
    constexpr int STORES = MI * NJ * (sizeof(TY) == 4 ? 4 : 2);  // of a wave for a whole tile, 16 bytes a lane
    constexpr int SP = 128 + 16;                       // bytes of a strip's row in LDS: no bank conflicts
    constexpr int E = 16 / sizeof(TY), SJ = 4 / sizeof(TY);  // results of a lane's store; 32-column tiles of a strip
    static_assert(RA == 3 && RB == 2, "the order of the loads and the waits below");
    static_assert(NW / 2 * 32 * SP <= TA && NW / 2 * 32 * SP <= TB && PA + STORES <= 63, "strips; the wait's counter");
    static_assert(PA >= 1 && PB >= 1 && RM % 64 == 0 && RN % 64 == 0, "tile shape");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char* const ringA = smem;
    char* const ringB = smem + RA * TA;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;

    // the items of one XCD (one L2) are neighbours: a contiguous share each, walked by its workgroups in turn
    const int xcd = blockIdx.x & 7, qi = items >> 3, ri = items & 7;
    const int share0 = xcd < ri ? xcd * (qi + 1) : ri * (qi + 1) + (xcd - ri) * qi, share1 = share0 + qi + (xcd < ri ? 1 : 0);
    const int step_items = (gridDim.x + 7 - xcd) >> 3;
    int item = share0 + (blockIdx.x >> 3);
    if (item >= share1) return;

    // lane offsets from a tile's first row
    unsigned oA[PA], oB[PB];
#pragma unroll
    for (int j = 0; j < PA; ++j) {
        const int r = 8 * (PA * wave + j) + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        oA[j] = (unsigned)(r * (int)a.lda + c * 16);
    }
#pragma unroll
    for (int j = 0; j < PB; ++j) {
        const int r = 8 * (PB * wave + j) + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        oB[j] = (unsigned)(r * (int)a.ldb + c * 16);
    }

    // an item's operands: where its rows and scales start, and how far they may be read
    struct Src {
        const uint8_t *A, *B;
        const uint32_t *sA, *sB;
        unsigned nA, nB, nsA, nsB;
        int m0, n0, nt, split;
    };
    auto clip = [](int64_t n) { return (unsigned)min(n, (int64_t)0xffffffff); };
    auto source = [&](int it) {
        Src s;
        int tm, tn;
        map_item(it, tiles_m, tiles_n, s.split, tm, tn);
        s.m0 = tm * BM;
        s.n0 = tn * BN;
        const int kb0 = s.split * a.kb_per_split;
        s.nt = min(a.nkb - kb0, a.kb_per_split);
        s.A = a.A + (int64_t)s.m0 * a.lda + (int64_t)kb0 * KB;
        s.B = a.B + (int64_t)s.n0 * a.ldb + (int64_t)kb0 * KB;
        // (from the first row's block to the end of the last row's padded length)
        s.nA = clip((int64_t)(a.M - 1 - s.m0) * a.lda + (int64_t)(a.nkb - kb0) * KB);
        s.nB = clip((int64_t)(a.N - 1 - s.n0) * a.ldb + (int64_t)(a.nkb - kb0) * KB);
        const int64_t fa = (int64_t)kb0 * a.a64 + (s.m0 + wm * RM) / 64, fb = (int64_t)kb0 * a.b64 + a.b_off + (s.n0 + wn * RN) / 64;
        const int64_t ea = (int64_t)a.nkb * a.a64, eb = (int64_t)a.nkb * a.b64;
        s.sA = a.sA + min(fa, ea - 1) * 16;  // (a wave whose rows all lie behind the last: any scales)
        s.sB = a.sB + min(fb, eb - 1) * 16;
        s.nsA = clip((ea - min(fa, ea - 1)) * 64);
        s.nsB = clip((eb - min(fb, eb - 1)) * 64);
        return s;
    };
    Src cur = source(item), nxt = cur;
    bool more = item + step_items < share1;
    if (more) nxt = source(item + step_items);

    // (buffer loads: lane offset + scalar offset of the K-tile; the compiler takes the flat form of a direct-to-LDS load for an
    // LDS access too, and drains every counter before the next use of a loaded register)
    auto buf = [](const void* p, unsigned n) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)n, 0x00020000); };
    // K-tile t of the current item; behind its last: tiles of the next item (of the last item: its last tile again, unused)
    auto loadA = [&](int t, int slot, int j) {
        const bool n = t >= cur.nt && more;
        const auto b = buf(n ? nxt.A : cur.A, n ? nxt.nA : cur.nA);
        const int k = n ? min(t - cur.nt, nxt.nt - 1) : min(t, cur.nt - 1);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (lds_void*)(ringA + slot * TA + (PA * wave + j) * 1024), 16, oA[j], k * KB, 0, 0);
    };
    auto loadB = [&](int t, int slot, int j) {
        const bool n = t >= cur.nt && more;
        const auto b = buf(n ? nxt.B : cur.B, n ? nxt.nB : cur.nB);
        const int k = n ? min(t - cur.nt, nxt.nt - 1) : min(t, cur.nt - 1);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (lds_void*)(ringB + slot * TB + (PB * wave + j) * 1024), 16, oB[j], k * KB, 0, 0);
    };

    // scales: word of (K-tile, 64-row group, row % 16); lanes of the odd 16 rows of a fragment take the next byte
    const int shift = ((lane >> 4) & 1) * 8;
    const unsigned us = (lane & 15) * 4;
    uint32_t nA[SA], nB[SB];  // requested
    int cA[SA], cB[SB], hA[SA], hB[SB];
    auto load_scales = [&](int t) {
        const bool n = t >= cur.nt && more;
        const int k = n ? t - cur.nt : min(t, cur.nt - 1);
        const auto ba = buf(n ? nxt.sA : cur.sA, n ? nxt.nsA : cur.nsA), bb = buf(n ? nxt.sB : cur.sB, n ? nxt.nsB : cur.nsB);
        // (whole offsets in the lane's register: a scalar one beyond the resource's end would not be seen as such)
        const unsigned ka = us + (unsigned)(k * a.a64) * 64, kb = us + (unsigned)(k * a.b64) * 64;
#pragma unroll
        for (int i = 0; i < SA; ++i) nA[i] = __builtin_amdgcn_raw_buffer_load_b32(ba, ka + i * 64, 0, 0);
#pragma unroll
        for (int i = 0; i < SB; ++i) nB[i] = __builtin_amdgcn_raw_buffer_load_b32(bb, kb + i * 64, 0, 0);
    };

    auto take_scales = [&]() {  // at a K-tile's end, where what came behind the request is counted (behind stores it is not)
#pragma unroll
        for (int i = 0; i < SA; ++i) {
            hA[i] = cA[i];
            cA[i] = (int)(nA[i] >> shift);
        }
#pragma unroll
        for (int i = 0; i < SB; ++i) {
            hB[i] = cB[i];
            cB[i] = (int)(nB[i] >> shift);
        }
    };

    // fragment reads: lane l holds row l % 32 of a 32-row tile, 32 bytes: chunks 4 ks + 2 (l / 32) + {0, 1}
    const int fr = lane & 31, fz = (fr >> 1) & 7;
    int fo[2][2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int u = 0; u < 2; ++u) fo[ks][u] = fr * KB + (((4 * ks + 2 * (lane >> 5) + u) ^ fz) << 4);
    auto frag = [&](const char* tile, int ks, int r0) {
        const u32x4 lo = *reinterpret_cast<const u32x4*>(tile + fo[ks][0] + r0 * KB);
        const u32x4 hi = *reinterpret_cast<const u32x4*>(tile + fo[ks][1] + r0 * KB);
        return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };

    f32x16 acc[NJ][MI];
    i32x8 a0[MI], b0[NJ], a1[MI], b1[NJ];
    // one step: NJ x MI products; piece(p) issues a share of the staging loads in front of each row of them
    auto step = [&](const i32x8 (&fa)[MI], const i32x8 (&fb)[NJ], const int (&xa)[SA], const int (&xb)[SB], auto&& piece) {
        bf16x8 wb[WIDE ? NJ : 1][4];
        if constexpr (WIDE) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const float x = wide_scale((unsigned)xb[j / 2] >> (16 * (j & 1)) & 255u);
#pragma unroll
                for (int q = 0; q < 4; ++q) wb[j][q] = widen8<C2_E4M3>((unsigned)fb[j][2 * q], (unsigned)fb[j][2 * q + 1], x);
            }
        }
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            piece(i);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (WIDE) {
                const float x = wide_scale((unsigned)xa[i / 2] >> (16 * (i & 1)) & 255u);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const bf16x8 wa = widen8<AF>((unsigned)fa[i][2 * q], (unsigned)fa[i][2 * q + 1], x);
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[j][q], wa, acc[j][i], 0, 0, 0);
                }
                continue;
            }
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int va = xa[i / 2], vb = xb[j / 2];
                if ((i & 1) == 0 && (j & 1) == 0) acc[j][i] = mma<AF, 0, 0>(fb[j], fa[i], acc[j][i], vb, va);
                if ((i & 1) == 0 && (j & 1) == 1) acc[j][i] = mma<AF, 2, 0>(fb[j], fa[i], acc[j][i], vb, va);
                if ((i & 1) == 1 && (j & 1) == 0) acc[j][i] = mma<AF, 0, 2>(fb[j], fa[i], acc[j][i], vb, va);
                if ((i & 1) == 1 && (j & 1) == 1) acc[j][i] = mma<AF, 2, 2>(fb[j], fa[i], acc[j][i], vb, va);
            }
        }
    };

    // prologue, in the order of the loop's own loads
    load_scales(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < PA; ++j) loadA(0, 0, j);
#pragma unroll
    for (int j = 0; j < PB; ++j) loadB(0, 0, j);
#pragma unroll
    for (int j = 0; j < PA; ++j) loadA(1, 1, j);

#pragma unroll
    for (int i = 0; i < SA; ++i) cA[i] = 0;
#pragma unroll
    for (int i = 0; i < SB; ++i) cB[i] = 0;
    take_scales();
    int ra = 0, rb = 0;  // slots of the K-tile that is multiplied
    bool whole = false;  // the item before was a whole tile: every wave has made STORES stores since its last load
    for (;;) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;
#pragma unroll
        for (int i = 0; i < MI; ++i) a1[i] = i32x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < NJ; ++j) b1[j] = i32x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < SA; ++i) hA[i] = 0x7f7f7f7f;
#pragma unroll
        for (int i = 0; i < SB; ++i) hB[i] = 0x7f7f7f7f;

        for (int T = 0; T < cur.nt; ++T) {
            // tile T and its scales have landed; A of T + 1 may still be on its way, and the stores of the item before behind it
            if (T == 0 && whole) wait_vm<PA + STORES>();
            else wait_vm<PA>();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            load_scales(T + 1);
            const char* tA = ringA + ra * TA + wm * RM * KB;
            const char* tB = ringB + rb * TB + wn * RN * KB;
            const int da = ra == 0 ? RA - 1 : ra - 1, db = rb == 0 ? RB - 1 : rb - 1;  // the slots of the tile before
#pragma unroll
            for (int j = 0; j < NJ; ++j) b0[j] = frag(tB, 0, j * 32);
#pragma unroll
            for (int i = 0; i < MI; ++i) a0[i] = frag(tA, 0, i * 32);
            __builtin_amdgcn_sched_barrier(0);  // the reads are on their way before the held step starts
            __builtin_amdgcn_s_setprio(1);
            step(a1, b1, hA, hB, [&](int p) {
#pragma unroll
                for (int j = p * PB / MI; j < (p + 1) * PB / MI; ++j) loadB(T + RB - 1, db, j);
            });
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int j = 0; j < NJ; ++j) b1[j] = frag(tB, 1, j * 32);
#pragma unroll
            for (int i = 0; i < MI; ++i) a1[i] = frag(tA, 1, i * 32);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            step(a0, b0, cA, cB, [&](int p) {
#pragma unroll
                for (int j = p * PA / MI; j < (p + 1) * PA / MI; ++j) loadA(T + RA - 1, da, j);
            });
            __builtin_amdgcn_s_setprio(0);
            take_scales();
            ra = ra + 1 == RA ? 0 : ra + 1;
            rb = rb + 1 == RB ? 0 : rb + 1;
        }
        // (the bias of the lane's columns, asked for under the last step: fragments and their registers are done with)
        f32x4 bias[NJ][4];
        if (a.bias) {
            const auto bb = buf(a.bias, (unsigned)a.N * 4);
            const unsigned bo = (unsigned)((lane >> 5) * 4 + cur.n0 + wn * RN) * 4;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    bias[j][q] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(bb, bo + (j * 32 + q * 8) * 4, 0, 0));
        } else {
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) bias[j][q] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        step(a1, b1, hA, hB, [&](int) {});

        // ---- the finished tile: lane l holds row m = l % 32 of a 32-column tile, columns 8 q + 4 (l / 32) + 0..3.  Strips of 32
        // rows go through LDS, to whole 128-byte row segments (16 bytes a lane): in the slots of the last K-tile, which no load is
        // on its way to (the next item's A 0, A 1 and B 0 go to the others)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();  // every wave has read the last K-tile
        asm volatile("" ::: "memory");
        int ln = lane;  // (opaque: addresses of the stores are formed here, not kept through the loop)
        asm volatile("" : "+v"(ln));
        const float alpha = (WIDE ? kWideBack : 1.f) * (a.alpha_dev ? *a.alpha_dev : 1.f);
        const int fa = ra == 0 ? RA - 1 : ra - 1, fb = rb == 0 ? RB - 1 : rb - 1;
        char* strip = (wave < NW / 2 ? ringA + fa * TA : ringB + fb * TB) + (wave & (NW / 2 - 1)) * 32 * SP;
        const int row0 = cur.m0 + wm * RM + ln / 8, col0 = cur.n0 + wn * RN + (ln % 8) * E;
        TY* out = reinterpret_cast<TY*>(a.Y) + (int64_t)cur.split * a.slab + (int64_t)row0 * a.ldy + col0;
        whole = cur.m0 + BM <= a.M && cur.n0 + BN <= a.N;  // (uniform)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int jj = 0; jj < NJ; jj += SJ) {  // SJ tiles of 32 columns make a row of 128 bytes
#pragma unroll
                for (int j = 0; j < SJ; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        f32x4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = alpha * acc[jj + j][i][4 * q + e] + bias[jj + j][q][e];
                        char* p = strip + (ln & 31) * SP + (j * 32 + q * 8 + 4 * (ln >> 5)) * (int)sizeof(TY);
                        if constexpr (sizeof(TY) == 4) *reinterpret_cast<f32x4*>(p) = v;
                        else *reinterpret_cast<u32x2*>(p) = u32x2{pack2<TY>(v[0], v[1]), pack2<TY>(v[2], v[3])};
                    }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                u32x4 x[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const u32x4*>(strip + (r * 8 + ln / 8) * SP + (ln % 8) * 16);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    TY* p = out + (int64_t)(i * 32 + r * 8) * a.ldy + jj * 32;
                    const int n = col0 + jj * 32;
                    if (whole || (row0 + i * 32 + r * 8 < a.M && n + E <= a.N)) {
                        *reinterpret_cast<u32x4_a2*>(p) = x[r];
                    } else if (row0 + i * 32 + r * 8 < a.M) {
                        const TY* v = reinterpret_cast<const TY*>(&x[r]);
#pragma unroll
                        for (int e = 0; e < E; ++e)
                            if (n + e < a.N) p[e] = v[e];
                    }
                }
            }
        if (!more) break;
        item += step_items;
        cur = nxt;
        more = item + step_items < share1;
        if (more) nxt = source(item + step_items);
    }
    // (loads behind the last K-tile may still be on their way into LDS: they end before the workgroup's memory is given away)
    wait_vm<0>();
#endif
}

// 4096 x 1024 in four parts: 14.4 us (the 67 MB that the product just wrote); 128 x 256 in 50: 4.0 us.
// Y = alpha * sum of the slabs + bias: four columns a thread, SG threads share their slabs (SG > 1 where the result alone is
// too small to keep the chip busy) and meet in LDS, in a fixed order.
template <typename TY, int SG>
__global__ __launch_bounds__(256) void join_slabs_kernel(const float* __restrict__ ws, int64_t slab, int64_t lds, int splits,
                                                         int64_t M, int N, int nq, TY* __restrict__ Y, int64_t ldy,
                                                         const float* __restrict__ bias, const float* __restrict__ alpha_dev) {
    constexpr int Q = 256 / SG;
    __shared__ f32x4 red[SG][Q];
    const int g = threadIdx.x / Q, t = threadIdx.x % Q;
    const int64_t i = (int64_t)blockIdx.x * Q + t, m = min(i / nq, M - 1);
    const int n = (int)(i % nq) * 4;
    const float* p = ws + m * lds + n;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    for (int k = g; k < splits; k += 4 * SG) {
        f32x4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = *reinterpret_cast<const f32x4*>(p + min(k + u * SG, splits - 1) * slab);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (k + u * SG < splits) s += x[u];
    }
    if (SG > 1) {
        red[g][t] = s;
        __syncthreads();
        if (g != 0) return;
#pragma unroll
        for (int k = 1; k < SG; ++k) s += red[k][t];
    }
    if (i >= M * nq) return;
    const float alpha = alpha_dev ? *alpha_dev : 1.f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (n + c < N) st_from_f32<TY>(Y + m * ldy + n + c, alpha * s[c] + (bias ? bias[n + c] : 0.f));
}

// ---- how a product is cut: tiles of 256 x 256 or 128 x 128, the reduction in `splits` parts where the tiles alone leave CUs idle; or
// 256 x 256 tiles for the columns that make whole rounds of the chip, and the best cut for the rest.  Wide (fp32 results): 128 x 128
// tiles, in parts or not.
struct Cut {
    int big, splits, kb_per_split;
    int64_t lds, slab;
};
// Estimated microseconds, from measurements on random operands: a K-tile takes a 256 x 256 workgroup 1.5 (all CUs busy), two
// 128 x 128 workgroups on one CU 1.0, a single one 0.9; starting and storing 5 and 4; the join reads its slabs at 5.3 MB/us.
// Wide: two workgroups 1.7, a single one 1.2; starting and storing 8 and 6 (2048 x 2048 over 1024 and 2048, 256 of them: 17.1 and
// 26.5; 4096 x 2048, 512: 25.1 and 38.4).
inline double cost_tiles(bool big, bool wide, int64_t items, int kb) {
    if (wide) return items <= 256 ? 1.2 * kb + 6. : (double)((items + 511) / 512) * (1.7 * kb + 8.);
    if (big) return (double)((items + 255) / 256) * (1.5 * kb + 5.);
    if (items <= 256) return 0.9 * kb + 4.;
    return (double)((items + 511) / 512) * (1.0 * kb + 4.);
}
inline int64_t n_tiles(int64_t n, int e) { return (n + e - 1) / e; }
inline Cut cut_of(int64_t M, int64_t N, int64_t K, bool wide, double& least) {
    const int nkb = (int)n_tiles(K, KB);
    Cut best{};
    best.lds = (N + 3) / 4 * 4;
    best.slab = M * best.lds;
    least = 1e300;
    for (int big = 0; big < (wide ? 1 : 2); ++big) {
        const int64_t t = big ? n_tiles(M, 256) * n_tiles(N, 256) : n_tiles(M, 128) * n_tiles(N, 128);
        // parts of at least two K-tiles, at most one round of workgroups
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(nkb / 2, 64), (big ? 256 : 512) / t));
        for (int s0 = 1; s0 <= most; ++s0) {
            const int kb = (nkb + s0 - 1) / s0, s = (nkb + kb - 1) / kb;
            double c = cost_tiles(big, wide, t * s, kb);
            if (s > 1) c += 3. + (4. * s + 2.) * (double)M * (double)N / 5.3e6;
            if (c < least) {
                least = c;
                best.big = big;
                best.splits = s;
                best.kb_per_split = kb;
            }
        }
    }
    return best;
}
struct Plan {
    int64_t n_big;  // columns of whole rounds of 256 x 256 tiles (0: none)
    Cut cut;        // of the rest
};
inline Plan plan_of(int64_t M, int64_t N, int64_t K, bool wide) {
    double whole, rest;
    Plan p{0, cut_of(M, N, K, wide, whole)};
    if (wide) return p;
    const int64_t tm = n_tiles(M, 256), full = tm * n_tiles(N, 256) / 256 * 256 / tm * 256;
    if (full > 0 && full < N) {
        const Cut r = cut_of(M, N - full, K, false, rest);
        if (cost_tiles(true, false, tm * (full / 256), (int)n_tiles(K, KB)) + rest < whole) p = {full, r};
    }
    return p;
}

template <int AF, typename TY, bool WIDE>
void launch_tiles(const Args& a, const Cut& c, hipStream_t st) {
#define TILE(BM, BN, WM, WN, PER_CU)                                                                                       \
    do {                                                                                                                   \
        const int tm = (int)n_tiles(a.M, BM), tn = (int)n_tiles(a.N, BN), items = tm * tn * c.splits;                      \
        /* a walk over several items: the loads run two K-tiles ahead, into the next item but not past it */               \
        const int grid = c.splits == 1 && a.nkb >= 2 ? std::min(items, 256 * PER_CU) : items;                              \
        auto k = gemm_fp8_kernel<AF, TY, BM, BN, WM, WN, 3, 2, 2, WIDE>;                                                       \
        constexpr int lds = (3 * BM + 2 * BN) * KB;                                                                        \
        (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds);                        \
        hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(64 * WM * WN), lds, st, a, tm, tn, items);                        \
    } while (0)
    if constexpr (!WIDE) {
        if (c.big) {
            TILE(256, 256, 2, 4, 1);
            return;
        }
    }
    TILE(128, 128, 2, 2, 2);
#undef TILE
}

template <typename TY>
void join_to(const float* ws, int64_t slab, int64_t lds, int splits, int64_t M, int64_t N, TY* Y, int64_t ldy, const float* bias,
             const float* alpha_dev, hipStream_t st) {
    const int nq = (int)(lds / 4);
    const int64_t quads = M * nq;
#define JOIN(SG)                                                                                                          \
    hipLaunchKernelGGL((join_slabs_kernel<TY, SG>), dim3((unsigned)((quads * SG + 255) / 256)), dim3(256), 0, st, ws, slab, lds, \
                       splits, M, (int)N, nq, Y, ldy, bias, alpha_dev)
    if (quads >= 65536 || splits <= 4) JOIN(1);
    else if (quads >= 16384 || splits <= 16) JOIN(4);
    else JOIN(16);
#undef JOIN
}
void join_slabs(const float* ws, int64_t slab, int64_t lds, int splits, int64_t M, int64_t N, void* Y, int y_dtype, int64_t ldy,
                const float* bias, const float* alpha_dev, hipStream_t st) {
    if (y_dtype == C2_F32) join_to(ws, slab, lds, splits, M, N, (float*)Y, ldy, bias, alpha_dev, st);
    else if (y_dtype == C2_BF16) join_to(ws, slab, lds, splits, M, N, (bf16_t*)Y, ldy, bias, alpha_dev, st);
    else join_to(ws, slab, lds, splits, M, N, (f16_t*)Y, ldy, bias, alpha_dev, st);
}

template <typename TY>
void launch(const Args& a0, const Cut& c, int a_fmt, float* ws, hipStream_t st) {
    constexpr bool WIDE = sizeof(TY) == 4;  // (the parts of a 16-bit result are what its own form makes)
    Args a = a0;
    a.kb_per_split = c.kb_per_split;
    if (c.splits > 1) {
        a.Y = ws;
        a.ldy = c.lds;
        a.slab = c.slab;
        a.bias = nullptr;
        a.alpha_dev = nullptr;
        if (a_fmt == C2_E4M3) launch_tiles<0, float, WIDE>(a, c, st);
        else launch_tiles<1, float, WIDE>(a, c, st);
        join_to<TY>(ws, c.slab, c.lds, c.splits, a0.M, a0.N, (TY*)a0.Y, a0.ldy, a0.bias, a0.alpha_dev, st);
        return;
    }
    if (a_fmt == C2_E4M3) launch_tiles<0, TY, WIDE>(a, c, st);
    else launch_tiles<1, TY, WIDE>(a, c, st);
}

template <typename TY>
void product_to(Args a, const Plan& p, int a_fmt, float* ws, hipStream_t st) {
    if (p.n_big > 0) {
        Args b = a;
        b.N = (int)p.n_big;
        launch<TY>(b, Cut{1, 1, a.nkb, 0, 0}, a_fmt, nullptr, st);
        a.B += p.n_big * a.ldb;
        a.b_off = (int)(p.n_big / 64);
        a.N -= (int)p.n_big;
        a.Y = (TY*)a.Y + p.n_big;
        if (a.bias) a.bias += p.n_big;
    }
    launch<TY>(a, p.cut, a_fmt, ws, st);
}

void product(const void* A, int64_t lda, const uint8_t* sA, int a_fmt, const void* B, int64_t ldb, const uint8_t* sB, int64_t M,
             int64_t N, int64_t K, void* Y, int y_dtype, int64_t ldy, const float* bias, const float* alpha_dev, float* ws,
             hipStream_t st) {
    const Plan p = plan_of(M, N, K, y_dtype == C2_F32);
    Args a{(const uint8_t*)A, (const uint8_t*)B, (const uint32_t*)sA, (const uint32_t*)sB, Y, bias, alpha_dev,
           lda, ldb, ldy, 0, (int)M, (int)N, (int)n_tiles(K, KB), 0, (int)n_tiles(M, 64), (int)n_tiles(N, 64), 0};
    if (y_dtype == C2_F32) product_to<float>(a, p, a_fmt, ws, st);
    else if (y_dtype == C2_BF16) product_to<bf16_t>(a, p, a_fmt, ws, st);
    else product_to<f16_t>(a, p, a_fmt, ws, st);
}
size_t product_ws(int64_t M, int64_t N, int64_t K) {
    if (in_rows(M, N, K)) {
        const RowPlan r = row_plan(M, N, K);
        return r.splits > 1 ? (size_t)r.splits * (size_t)M * (size_t)r.lds : 0;
    }
    size_t floats = 0;  // whatever the result's type
    for (const bool wide : {false, true}) {
        const Cut c = plan_of(M, N, K, wide).cut;
        if (c.splits > 1) floats = std::max(floats, (size_t)c.splits * (size_t)c.slab);
    }
    return floats;
}

// bytes of x's 8-bit copy and its scales in the workspace of c2_linear_fwd_fp8, each on 16 bytes
struct XCopy {
    int64_t ldq;
    size_t q, scale, total;
};
inline XCopy x_copy(int64_t M, int64_t K) {
    XCopy x{};
    x.ldq = (K + KB - 1) / KB * KB;
    x.q = (size_t)M * (size_t)x.ldq;
    x.scale = c2_fp8_scale_bytes(M, K);  // (both are multiples of 16)
    x.total = x.q + x.scale;
    return x;
}
inline bool sizes_ok(int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb) {  // 32-bit offsets inside a tile, tile counts
    return lda < (1ll << 22) && ldb < (1ll << 22) && ((M + 127) / 128) * ((N + 127) / 128) < (1ll << 24);
}

}  // namespace fp8
}  // namespace c2

extern "C" size_t c2_linear_fp8_ws(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return c2::fp8::product_ws(M, N, K);
}

extern "C" int c2_linear_fp8(const void* A, int64_t lda, const uint8_t* sA, int a_fmt, const void* B, int64_t ldb,
                             const uint8_t* sB, int64_t M, int64_t N, int64_t K, void* Y, int y_dtype, int64_t ldy,
                             const float* bias, const float* alpha_dev, float* ws, void* stream) {
    using namespace c2;
    C2_CHECK(M >= 0 && N >= 0 && K >= 1, "bad shape (the reduction needs at least one element)");
    C2_CHECK(M < (1ll << 30) && N < (1ll << 30) && K < (1ll << 30), "size beyond 2^30");
    C2_CHECK(a_fmt == C2_E4M3 || a_fmt == C2_E5M2, "a_fmt: C2_E4M3 or C2_E5M2");
    C2_CHECK(y_dtype == C2_F32 || y_dtype == C2_BF16 || y_dtype == C2_F16, "bad output dtype");
    if (M == 0 || N == 0) return 0;
    const int64_t kp = (K + 127) / 128 * 128;
    C2_CHECK(A && sA && B && sB && Y, "null pointer");
    C2_CHECK(lda >= kp && ldb >= kp && (lda & 15) == 0 && (ldb & 15) == 0 && aligned16(A) && aligned16(B),
             "operand rows: K rounded up to 128 bytes, starting on 16 bytes");
    C2_CHECK((reinterpret_cast<uintptr_t>(sA) & 3) == 0 && (reinterpret_cast<uintptr_t>(sB) & 3) == 0, "scales must start on 4 bytes");
    C2_CHECK(ldy >= N, "leading dimension too small");
    C2_CHECK(c2_linear_fp8_ws(M, N, K) == 0 || (ws && aligned16(ws)), "workspace: null, or not on 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    if (fp8::in_rows(M, N, K)) {
        fp8::launch_few_rows(A, fp8::kQuantised, lda, sA, a_fmt, (const uint8_t*)B, ldb, sB, M, N, K, Y, y_dtype, ldy, bias,
                             alpha_dev, ws, st);
        C2_LAUNCH_CHECK();
        return 0;
    }
    C2_CHECK(fp8::sizes_ok(M, N, K, lda, ldb), "too large for one launch");
    fp8::product(A, lda, sA, a_fmt, B, ldb, sB, M, N, K, Y, y_dtype, ldy, bias, alpha_dev, ws, st);
    C2_LAUNCH_CHECK();
    return 0;
}

extern "C" size_t c2_linear_fwd_fp8_ws(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return (c2::fp8::in_rows(M, N, K) ? 0 : c2::fp8::x_copy(M, K).total) + 4 * c2::fp8::product_ws(M, N, K);
}

extern "C" int c2_linear_fwd_fp8(const void* x, int x_dtype, int64_t ldx, const void* W, int64_t ldw, const uint8_t* sW,
                                 int64_t M, int64_t N, int64_t K, void* Y, int y_dtype, int64_t ldy, const float* bias,
                                 void* ws, void* stream) {
    using namespace c2;
    C2_CHECK(M >= 0 && N >= 0 && K >= 1, "bad shape (the reduction needs at least one element)");
    C2_CHECK(M < (1ll << 30) && N < (1ll << 30) && K < (1ll << 30), "size beyond 2^30");
    C2_CHECK(x_dtype == C2_F32 || x_dtype == C2_BF16 || x_dtype == C2_F16, "bad dtype");
    C2_CHECK(y_dtype == C2_F32 || y_dtype == C2_BF16 || y_dtype == C2_F16, "bad output dtype");
    if (M == 0 || N == 0) return 0;
    const int64_t kp = (K + 127) / 128 * 128;
    C2_CHECK(x && W && sW && Y, "null pointer");
    C2_CHECK(ldx >= K && ldy >= N, "leading dimension too small");
    C2_CHECK(ldw >= kp && (ldw & 15) == 0 && aligned16(W), "weight rows: K rounded up to 128 bytes, starting on 16 bytes");
    C2_CHECK((reinterpret_cast<uintptr_t>(sW) & 3) == 0, "scales must start on 4 bytes");
    C2_CHECK(c2_linear_fwd_fp8_ws(M, N, K) == 0 || (ws && aligned16(ws)), "workspace: null, or not on 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    if (fp8::in_rows(M, N, K)) {
        fp8::launch_few_rows(x, x_dtype, ldx, nullptr, C2_E4M3, (const uint8_t*)W, ldw, sW, M, N, K, Y, y_dtype, ldy, bias, nullptr,
                             (float*)ws, st);
        C2_LAUNCH_CHECK();
        return 0;
    }
    C2_CHECK(fp8::sizes_ok(M, N, K, kp, ldw), "too large for one launch");
    const fp8::XCopy c = fp8::x_copy(M, K);
    char* q = (char*)ws;
    uint8_t* scale = (uint8_t*)(q + c.q);
    const int rc = c2_quant_fp8(x, x_dtype, ldx, M, K, 1, C2_E4M3, q, c.ldq, scale, nullptr, 0, nullptr, stream);
    if (rc) return rc;
    fp8::product(q, c.ldq, scale, C2_E4M3, W, ldw, sW, M, N, K, Y, y_dtype, ldy, bias, nullptr, (float*)(q + c.total), st);
    C2_LAUNCH_CHECK();
    return 0;
}
