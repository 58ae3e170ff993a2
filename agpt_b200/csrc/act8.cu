// Activations kept in 8 bits for the backward, and what the backward does with them.
//
// A block is 32 neighbouring columns of a row.  It is kept as one scale byte s, standing for 2^(s - 127), and 32 codes e4m3:
//   e = the smallest exponent with max |x| <= 448 * 2^e (at least -110),  s = e + 127,  code = e4m3(x * 2^-e), to nearest, ties to even
//   (240 at most where e is 120: the next number is beyond float32)
// A scale that is a power of two makes x * 2^-e exact, so a value has one rounding, to four significant bits (at most 2^-4 of it, or half a
// step of 2^(e - 9) near zero), and a code's value is exact in bfloat16.  A value that is not zero keeps its sign and the smallest code at
// least: the mask of a ReLU can be read from the checkpoint.  A block that holds infinity or NaN is NaN as a whole: scale byte 255, codes 0x7f.
//
//   codes  uint8 [rows][columns rounded up to 32] (zeros behind the last column)
//   scales uint8 [blocks of 32 columns][rows rounded up to 16]
//
// Packing, unpacking and the ReLU's backward are bound by memory: 560k x 512 float32 209 us (6.9 TB/s) and 216 (6.7), 400k x 512 269 us (6.8).  Packing bfloat16 is half
// arithmetic, 162 us (5.4 TB/s).  Rows of no whole 16-byte pieces, or off 16-byte boundaries, go element by element: 560k x 510 344 us, 256 and 408 (374 at 512); bfloat16 351.
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/agpt_b200.h"
#include "internal.h"
#include "pdl.cuh"
#include "tc100.cuh"
#include "vec.cuh"

namespace {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ uint32_t codes2(float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 values2(uint32_t c) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)c, __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}
// the larger of two magnitudes (with some sign), NaN if one of them is
__device__ __forceinline__ float max_magnitude(float a, float b) {
    float r;
    asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// what a scale byte stands for
__device__ __forceinline__ float scale_of(uint32_t s) { return __uint_as_float(s == 255 ? 0x7fc00000u : s ? s << 23 : 0x00400000u); }

// A group of lanes has a block of PACK_ROWS consecutive rows: their loads are in flight together and their scale bytes are neighbours.  A lane has PIECES pieces of
// VEC columns, eight values where rows allow it: what a block costs once (its maximum across lanes, its exponent) is the larger part of the arithmetic, and that
// is what bounds the kernel (four values a lane: 276 us at 560k x 512, ALU pipe at 77 %).
constexpr int PACK_ROWS = 4;
template <typename T, int VEC, int PIECES, bool WHOLE>
__global__ void __launch_bounds__(256) pack_kernel(const T *__restrict__ x, int64_t ld, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales, int64_t n, int cols,
                                                    int blocks, int64_t pitch, vec::Divide by_blocks, int64_t tasks) {
    pdl_wait();
    pdl_next();
    constexpr int LANES = 32 / (VEC * PIECES), STEP = 32 / PIECES;
    const int lane = threadIdx.x % LANES;
    const int64_t task = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (task >= tasks) return;                         // whole groups leave; the shuffles below stay inside a group
    const uint32_t group = ((1u << LANES) - 1) << (threadIdx.x & 31 & ~(LANES - 1));
    const int64_t quad = vec::quotient(task, by_blocks), r0 = quad * PACK_ROWS;
    const int b = (int)(task - quad * blocks), c = b * 32 + lane * VEC;
    vec::Piece<T, VEC> piece[PACK_ROWS][PIECES];
    if (WHOLE)
#pragma unroll
        for (int u = 0; u < PACK_ROWS; u++)
#pragma unroll
            for (int j = 0; j < PIECES; j++) piece[u][j].fetch(x + (r0 + u) * ld + c + j * STEP, r0 + u < n && c + j * STEP < cols);
    uint32_t s4 = 0;
#pragma unroll
    for (int u = 0; u < PACK_ROWS; u++) {
        float v[PIECES][VEC];
#pragma unroll
        for (int j = 0; j < PIECES; j++) {
            if (WHOLE) piece[u][j].values(v[j]);
            else
#pragma unroll
                for (int i = 0; i < VEC; i++) v[j][i] = r0 + u < n && c + j * STEP + i < cols ? (float)x[(r0 + u) * ld + c + j * STEP + i] : 0.f;
        }
        float most = 0.f;                              // NaN where there is one
#pragma unroll
        for (int j = 0; j < PIECES; j++)
#pragma unroll
            for (int i = 0; i < VEC; i++) most = max_magnitude(most, v[j][i]);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) most = max_magnitude(most, __shfl_xor_sync(group, most, o));
        const uint32_t top = __float_as_uint(most) & 0x7fffffffu;
        // 2^k <= top < 2^(k+1), k = (top >> 23) - 127: top <= 448 * 2^(k-8) = 1.75 * 2^k, or one more
        const int e = max((int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u), -110);
        const bool bad = top >= 0x7f800000u;
        s4 |= (bad ? 255u : (uint32_t)(e + 127)) << (8 * u);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        uint32_t word[PIECES][VEC / 4];
#pragma unroll
        for (int j = 0; j < PIECES; j++)
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                uint32_t w = codes2(v[j][i] * down, v[j][i + 1] * down) | codes2(v[j][i + 2] * down, v[j][i + 3] * down) << 16;
                // bytes of magnitude 0 (bit 7 of the sum stays clear) whose value is not: the smallest code
                const uint32_t none = ~((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) & 0x80808080u;
                if (none) {
                    uint32_t some = 0;
#pragma unroll
                    for (int k = 0; k < 4; k++) some |= v[j][i + k] != 0.f ? 1u << (8 * k) : 0;
                    w |= none >> 7 & some;
                }
                word[j][i / 4] = w;
            }
        // 256 * 2^120 and above are no float32: what rounds there takes 240 * 2^120.  A block with infinity or NaN has 0x7f throughout.
        if (e == 120 || bad)
#pragma unroll
            for (int j = 0; j < PIECES; j++)
#pragma unroll
                for (int i = 0; i < VEC / 4; i++) {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if ((word[j][i] >> (8 * k) & 0x7f) > 0x77) word[j][i] = (word[j][i] & ~(0x7fu << (8 * k))) | 0x77u << (8 * k);
                    if (bad) word[j][i] = 0x7f7f7f7fu;
                }
        if (r0 + u < n) {
#pragma unroll
            for (int j = 0; j < PIECES; j++) {
                uint8_t *to = codes + (r0 + u) * (int64_t)blocks * 32 + c + j * STEP;
                if (VEC == 8) __stcs(reinterpret_cast<uint2 *>(to), make_uint2(word[j][0], word[j][VEC / 4 - 1]));
                else __stcs(reinterpret_cast<uint32_t *>(to), word[j][0]);
            }
        }
    }
    // rows behind the last lie inside the pitch, which is a multiple of 16
    if (lane == 0) *reinterpret_cast<uint32_t *>(scales + b * pitch + r0) = s4;
}

template <bool WHOLE>
__global__ void __launch_bounds__(256) unpack_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, float *__restrict__ out, int64_t n, int cols,
                                                      int blocks, int64_t pitch, vec::Divide by_blocks, int64_t tasks) {
    pdl_wait();
    pdl_next();
    const int lane = threadIdx.x & 7;
    const int64_t task = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
    if (task >= tasks) return;
    const int64_t quad = vec::quotient(task, by_blocks), r0 = quad * PACK_ROWS;
    const int b = (int)(task - quad * blocks), c = b * 32 + lane * 4;
    uint32_t w[PACK_ROWS];
#pragma unroll
    for (int u = 0; u < PACK_ROWS; u++) w[u] = r0 + u < n ? __ldcs(reinterpret_cast<const unsigned int *>(codes + (r0 + u) * (int64_t)blocks * 32 + c)) : 0;
    const uint32_t s4 = __ldg(reinterpret_cast<const unsigned int *>(scales + b * pitch + r0));
#pragma unroll
    for (int u = 0; u < PACK_ROWS; u++) {
        if (r0 + u >= n) break;
        const float f = scale_of(s4 >> (8 * u) & 255);
        const float2 a = values2(w[u] & 0xffff), d = values2(w[u] >> 16);
        float v[4] = {a.x * f, a.y * f, d.x * f, d.y * f};
        float *to = out + (r0 + u) * cols + c;
        if (WHOLE) {
            if (c < cols) vec::store_past<4>(to, v);
        } else
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (c + i < cols) to[i] = v[i];
    }
}

// out = grad where the kept value is above zero: the code is neither zero, nor negative, nor NaN
template <bool WHOLE>
__global__ void __launch_bounds__(256) relu_backward_kernel(const float *grad, int64_t ld, const uint8_t *__restrict__ codes, float *out, int64_t n, int cols, int blocks,
                                                             vec::Divide by_blocks, int64_t tasks) {
    pdl_wait();
    pdl_next();
    const int lane = threadIdx.x & 7;
    const int64_t task = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
    if (task >= tasks) return;
    const int64_t quad = vec::quotient(task, by_blocks), r0 = quad * PACK_ROWS;
    const int b = (int)(task - quad * blocks), c = b * 32 + lane * 4;
    uint32_t w[PACK_ROWS];
    float v[PACK_ROWS][4];
#pragma unroll
    for (int u = 0; u < PACK_ROWS; u++) {
        const bool live = r0 + u < n;
        w[u] = live ? __ldcs(reinterpret_cast<const unsigned int *>(codes + (r0 + u) * (int64_t)blocks * 32 + c)) : 0;
        if (WHOLE) {
            if (live && c < cols) vec::load<4>(grad + (r0 + u) * ld + c, v[u]);
        } else
#pragma unroll
            for (int i = 0; i < 4; i++) v[u][i] = live && c + i < cols ? grad[(r0 + u) * ld + c + i] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < PACK_ROWS; u++) {
        if (r0 + u >= n) break;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t code = w[u] >> (8 * i) & 255;
            if (code - 1 >= 0x7e) v[u][i] = 0.f;
        }
        float *to = out + (r0 + u) * cols + c;
        if (WHOLE) {
            if (c < cols) vec::store_past<4>(to, v[u]);
        } else
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (c + i < cols) to[i] = v[u][i];
    }
}

// ---- weight gradient: dW[m][N] = X^T G, db[N] = column sums of G ----------------------------------------------------------------------
// On tcgen05, float32-accurate: a kept value is exact in bfloat16, an element of G is the exact sum of three, so a product is three MMAs.  The MMA's rows are
// 128 columns of G: a converting thread owns one, walks down the rows and writes its packed pairs to tensor memory.  Up to 256 columns of X, n contiguous, come
// through shared memory, so that a split of G serves all of them.  TMA brings the raw rows; rows of G that it cannot take (off 16-byte boundaries) are copied four
// bytes at a time by the threads that convert them.  Blocks own (G tile, X columns, slice of the rows); slices are added in order.
//
// 400k rows: 512 kept columns, G of 128: 136 us (1150 TFLOP/s of MMAs); 128 kept, G of 512: 171 us (5.1 TB/s); error against float64 3e-7.  What bounds it is shared
// memory: per 64 rows of 128 x 256 the raw rows in and out, the planes and the MMAs' reads of them, each plane of G against the same codes, move 224 KB, 1750 clocks at
// 128 bytes, where the MMAs take 1536 and the memory 1100.  On the way here: accumulators drained every 64 rows by eight columns at a time 245 and 411 us, by TMA
// and 16 columns 209 and 289, every 128 rows 155 and 222 (error 1e-7 to 3e-7), eight warps on X 157 and 178, both groups on each accumulator 139 and 177, all threads on
// 128 columns of X 136 and 171.  Slower: stages of 32 rows (143 and 206), eight warps on G (146 and 207).  Later, on another GPU and side by side, 128
// kept and 512: 175 us as it was, 181 with NaN codes and infinite gradients, 183 with the bias gradient's blocks added in float64; 512 kept and 128: 140 to 142 throughout.
// Rows of G off 16-byte boundaries, 512 kept and 128: 178; 128 kept and 512: 328.
constexpr int WG_ROWS = 64, WG_X = 256, WG_G = 128, RAW_STAGES = 3;
constexpr int WG_THREADS = 768;                        // four warps that load and issue MMAs, four on G, eight on X, eight on the accumulators
constexpr uint32_t RAW_G = WG_ROWS * WG_G * 4, RAW_X = WG_ROWS * WG_X, RAW_S = 8 * WG_ROWS, PLANE = WG_ROWS * WG_X * 2;
constexpr uint32_t OFF_X = RAW_STAGES * RAW_G, OFF_P = OFF_X + RAW_STAGES * RAW_X, OFF_S = OFF_P + 2 * PLANE, OFF_BAR = OFF_S + RAW_STAGES * RAW_S;
constexpr size_t WG_SMEM = OFF_BAR + 256 + 1024;
static_assert(WG_SMEM <= 232448 && OFF_P % 1024 == 0, "shared memory");
constexpr int ACC_COLS = 128, G_COLS = 96, TMEM_COLS = 512;
constexpr int REG_ISSUE = 32, REG_G = 64, REG_X = 40, REG_ACC = 152;
static_assert(REG_ISSUE + REG_G + 2 * REG_X + 2 * REG_ACC <= 6 * 80, "setmaxnreg draws on the registers of the launch");

struct alignas(64) WeightGrad {
    CUtensorMap map_g, map_x, map_s;
    const float *grad;
    float *part, *col_part;            // [slices][m][cols], [slices][cols]: the results themselves if there is one slice
    int64_t ld, n, row_blocks;
    int m, cols, slices, x_cols, x_groups, g_tiles;
    int *status;
};

__device__ __forceinline__ void copy4(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// Two codes (bytes 0, 1 or 2, 3 of w) as bfloat16 values times 2^(scale - 127).  Sign, exponent and fraction of a code moved to their places in a bfloat16 make its
// value times 2^-120, subnormal ones included; f = 2^(scale - 7).
template <int HIGH> __device__ __forceinline__ uint32_t expand2(uint32_t w, uint32_t f) {
    uint32_t b;                                                        // each code behind eight copies of its sign
    asm("prmt.b32 %0, %1, 0, %2;" : "=r"(b) : "r"(w), "n"(HIGH ? 0xb3a2 : 0x9180));
    return mul_bf16x2(b << 4 & 0x87f087f0u, f);
}
// Codes of magnitude 0x7f are e4m3's NaN (pack writes them with scale byte 255 alone, a caller's own may have any).  Bit 7 of a byte: its code is one.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u; }
// a pair of factors, NaN for the codes that are
template <int HIGH> __device__ __forceinline__ uint32_t or_nan2(uint32_t w, uint32_t factors) {
    uint32_t m;                                                        // each byte's bit 7 over its half of the word
    asm("prmt.b32 %0, %1, 0, %2;" : "=r"(m) : "r"(nan_codes(w)), "n"(HIGH ? 0xbbaa : 0x9988));
    return factors | (m & 0x7fc07fc0u);
}

// Two floats as the packed sums of three bfloat16 each: eight bits of the fraction are cut off at a time, which is exact for every finite value (a first part that is
// rounded instead, as in tc::split3, is infinity from 0x7f7f8000 on, and its rest infinity the other way).
__device__ __forceinline__ void cut3(tc::f2 xy, uint32_t &p0, uint32_t &p1, uint32_t &p2) {
    using namespace tc;
    const f2 minus_one = 0xbf800000bf800000ull;
    uint32_t a, b;
    f2_unpack(xy, a, b);
    p0 = __byte_perm(a, b, 0x7632);
    const f2 r = f2_fma(f2_pack(a & 0xffff0000u, b & 0xffff0000u), minus_one, xy);
    f2_unpack(r, a, b);
    p1 = __byte_perm(a, b, 0x7632);
    f2_unpack(f2_fma(f2_pack(a & 0xffff0000u, b & 0xffff0000u), minus_one, r), a, b);
    p2 = __byte_perm(a, b, 0x7632);
}
// The same where infinities and NaN may be among them: these are their first part alone, so that their products are infinities and NaN as those of any float are.
__device__ __forceinline__ void cut3_any(tc::f2 xy, uint32_t &p0, uint32_t &p1, uint32_t &p2) {
    using namespace tc;
    cut3(xy, p0, p1, p2);
    uint32_t a, b;
    f2_unpack(xy, a, b);
    const bool odd_a = (a & 0x7f800000u) == 0x7f800000u, odd_b = (b & 0x7f800000u) == 0x7f800000u;
    const uint32_t keep = (odd_a ? 0 : 0xffffu) | (odd_b ? 0 : 0xffff0000u);
    p1 &= keep;
    p2 &= keep;
    // NaN whose fraction was cut off
    if (odd_a && a & 0x7fffffu) p0 |= 0x7fc0u;
    if (odd_b && b & 0x7fffffu) p0 |= 0x7fc00000u;
}

template <bool TMA_G>
__global__ void __launch_bounds__(WG_THREADS, 1) weight_kernel(const __grid_constant__ WeightGrad P) {
    using namespace tc;
    extern __shared__ __align__(1024) unsigned char dyn[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wq = warp & 3;
    const uint32_t base = smem_u32(smem), bars = base + OFF_BAR;
    volatile int &s_abort = *reinterpret_cast<volatile int *>(smem + OFF_BAR + 240);
    uint32_t &s_tmem = *reinterpret_cast<uint32_t *>(smem + OFF_BAR + 248);
    // G and X planes filled, empty; accumulators; raw rows of G and X filled, empty
    const uint32_t tF = bars, tE = tF + 16, pF = tE + 16, pE = pF + 16, cF = pE + 16, cE = cF + 16, gF = cE + 16, gE = gF + 24, xF = gE + 24, xE = xF + 24;
    const int units = P.g_tiles * P.x_groups, unit = blockIdx.x % units, slice = blockIdx.x / units;
    const int g0 = unit / P.x_groups * WG_G, x0 = unit % P.x_groups * P.x_cols;
    const int xw = min(P.x_cols, P.m - x0), halves = xw > ACC_COLS ? 2 : 1;
    const int64_t rb0 = P.row_blocks * slice / P.slices, rb1 = P.row_blocks * (slice + 1) / P.slices;

    if (tid == 0) {
        s_abort = 0;
        for (int i = 0; i < 2; i++) {
            mbar_init(tF + 8 * i, 4); mbar_init(tE + 8 * i, halves);
            mbar_init(pF + 8 * i, 8); mbar_init(pE + 8 * i, halves);
            mbar_init(cF + 8 * i, 1); mbar_init(cE + 8 * i, 8);
        }
        for (int i = 0; i < RAW_STAGES; i++) { mbar_init(gF + 8 * i, 1); mbar_init(gE + 8 * i, 4); mbar_init(xF + 8 * i, 1); mbar_init(xE + 8 * i, 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc(smem_u32(&s_tmem), TMEM_COLS);
    pdl_wait();
    pdl_next();
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = s_tmem;

    if (warp < 4) {
        regs_dec<REG_ISSUE>();
        if (warp == 2 && lane == 0) {
            // ---------------- loads ----------------
            int slot = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int64_t rb = rb0; ok && rb < rb1; rb++) {
                const int y = (int)(rb * WG_ROWS);
                if (TMA_G) {
                    if (!(ok = mbar_wait(gE + 8 * slot, ph ^ 1, &s_abort))) break;
                    mbar_expect(gF + 8 * slot, RAW_G);
                    tma_load_2d(base + slot * RAW_G, &P.map_g, g0, y, gF + 8 * slot);
                }
                if (!(ok = mbar_wait(xE + 8 * slot, ph ^ 1, &s_abort))) break;
                mbar_expect(xF + 8 * slot, (uint32_t)(WG_ROWS * P.x_cols + RAW_S));
                tma_load_2d(base + OFF_X + slot * RAW_X, &P.map_x, x0, y, xF + 8 * slot);
                tma_load_2d(base + OFF_S + slot * RAW_S, &P.map_s, y, x0 >> 5, xF + 8 * slot);
                if (++slot == RAW_STAGES) { slot = 0; ph ^= 1; }
            }
            if (!ok) {                                                 // copies in flight end before the block does
                volatile int none = 0;
                for (int i = 0; i < RAW_STAGES; i++) {
                    if (TMA_G) mbar_wait(gF + 8 * i, ph, &none);
                    mbar_wait(xF + 8 * i, ph, &none);
                }
            }
        } else if (warp < halves) {
            // ---------------- MMAs: a warp per accumulator ----------------
            const uint32_t idesc = idesc_bf16((min(ACC_COLS, xw - warp * ACC_COLS) + 15) & ~15, true);
            uint32_t i = 0;
            bool ok = true;
            for (int64_t rb = rb0; ok && rb < rb1; rb++, i++) {
                const uint32_t st = i & 1, ph = (i >> 1) & 1, turn = i >> 1, own = halves == 2 ? warp : turn & 1, uses = halves == 2 ? turn : turn >> 1;
                if (st == 0 && !(ok = warp_wait(cE + 8 * own, (uses & 1) ^ 1, &s_abort))) break;
                if (!(ok = warp_wait2(tF + 8 * st, ph, pF + 8 * st, ph, &s_abort))) break;
                fence_after();
                if (elect_one()) {
                    const uint32_t a = tmem + 2 * ACC_COLS + st * G_COLS, b = desc_lo(base + OFF_P + st * PLANE + warp * (PLANE / 2), 8192);
#pragma unroll
                    for (int q = 2; q >= 0; q--)                       // small parts first
#pragma unroll
                        for (int k = 0; k < 4; k++) mma_ts(tmem + own * ACC_COLS, a + q * 32 + k * 8, b + k * 128, desc_hi(1024), idesc, st || q < 2 || k > 0);
                    commit(tE + 8 * st);
                    commit(pE + 8 * st);
                    if (st || rb + 1 == rb1) commit(cF + 8 * own);
                }
                __syncwarp();
            }
            if (!ok && elect_one()) {                                  // MMAs in flight end before tensor memory is given back
                commit(tE);
                volatile int none = 0;
                for (int j = 0; j < 2; j++) mbar_wait(tE, j, &none);
            }
            __syncwarp();
        }
    } else if (warp < 8) {
        regs_dec<REG_G>();
        // ---------------- G: a thread has a column ----------------
        const int col = g0 + wq * 32 + lane;
        const bool live = col < P.cols;
        const uint32_t raw = base + (wq * 32 + lane) * 4, dst0 = tmem + 2 * ACC_COLS + ((uint32_t)wq << 21);
        const float *src = P.grad + (live ? col : 0);
        // without TMA a thread copies what it converts, so that nothing but the end of its own copies has to be waited for
        const auto fetch = [&](int64_t rb, int slot) {
            if (rb < rb1) {
                const int64_t r0 = rb * WG_ROWS;
                const float *p = src + r0 * P.ld;
                const uint32_t to = raw + slot * RAW_G;
                const int rows = live ? (int)min((int64_t)WG_ROWS, P.n - r0) : 0;
#pragma unroll 8
                for (int k = 0; k < WG_ROWS; k++) { copy4(to + k * 512, k < rows ? p : P.grad, k < rows ? 4 : 0); p += P.ld; }
            }
            copies_end();
        };
        if (!TMA_G) { fetch(rb0, 0); fetch(rb0 + 1, 1); }
        double csum = 0.;                                              // of row blocks, of which a slice may have thousands
        uint32_t i = 0, gp = 0;
        int slot = 0;
        for (int64_t rb = rb0; rb < rb1; rb++, i++) {
            const uint32_t st = i & 1;
            if (TMA_G) {
                if (!warp_wait2(gF + 8 * slot, gp, tE + 8 * st, ((i >> 1) & 1) ^ 1, &s_abort)) break;
            } else {
                fetch(rb + 2, slot == 0 ? 2 : slot - 1);
                copies_wait<2>();
                if (!warp_wait(tE + 8 * st, ((i >> 1) & 1) ^ 1, &s_abort)) break;
            }
            fence_after();
            const uint32_t from = raw + slot * RAW_G, dst = dst0 + st * G_COLS;
            f2 bsum = 0;
#pragma unroll 1
            for (int k0 = 0; k0 < WG_ROWS; k0 += 16) {
                uint32_t p[3][8];
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                    const f2 v = f2_pack(lds_f1(from + (k0 + k) * 512), lds_f1(from + (k0 + k + 1) * 512));
                    bsum = f2_add(bsum, v);
                    cut3(v, p[0][k >> 1], p[1][k >> 1], p[2][k >> 1]);
                }
#pragma unroll
                for (int q = 0; q < 3; q++) tmem_st8(dst + q * 32 + (k0 >> 1), p[q]);
            }
            const float2 b2 = f2_get(bsum);
            const float block_sum = b2.x + b2.y;
            csum += block_sum;
            tmem_wait_st();
            // the sum is finite, or there are infinities or NaN among the values (or it went beyond the largest float): they are cut again with an eye to these
            if (__any_sync(0xffffffffu, (__float_as_uint(block_sum) & 0x7f800000u) == 0x7f800000u)) {
#pragma unroll 1
                for (int k0 = 0; k0 < WG_ROWS; k0 += 16) {
                    uint32_t p[3][8];
#pragma unroll
                    for (int k = 0; k < 8; k++) cut3_any(f2_pack(lds_f1(from + (k0 + 2 * k) * 512), lds_f1(from + (k0 + 2 * k + 1) * 512)), p[0][k], p[1][k], p[2][k]);
#pragma unroll
                    for (int q = 0; q < 3; q++) tmem_st8(dst + q * 32 + (k0 >> 1), p[q]);
                }
                tmem_wait_st();
            }
            fence_before();
            __syncwarp();
            if (lane == 0) { if (TMA_G) mbar_arrive(gE + 8 * slot); mbar_arrive(tF + 8 * st); }
            if (++slot == RAW_STAGES) { slot = 0; gp ^= 1; }
        }
        if (!TMA_G) copies_wait<0>();
        if (P.col_part && x0 == 0 && live) P.col_part[(int64_t)slice * P.cols + col] = (float)csum;
    } else if (warp < 16) {
        regs_dec<REG_X>();
        // ---------------- X: a thread has 16 columns of four rows; of two where the block has up to 128 columns, since half of the
        // threads would have none otherwise: 400k rows of 128 by 512 take 171 us against 180 ----------------
        const int narrow = P.x_cols <= ACC_COLS, t = tid - 256, piece = t & (narrow ? 7 : 15), rows = narrow ? 2 : 4;
        const int row = (t >> (narrow ? 3 : 4)) * rows;
        const bool live = piece * 16 < P.x_cols;
        const uint32_t raw = base + OFF_X + row * P.x_cols + piece * 16, raw_s = base + OFF_S + (piece >> 1) * WG_ROWS + (row & ~3);
        // place of the first stored half piece: eight neighbouring lanes write eight different 16-byte chunks of a row
        const uint32_t swap = (piece >> 2) & 1, put = base + OFF_P + ((piece >> 2) << 13) + row * 128, at = (piece & 3) * 2 + swap, at2 = at ^ 1, row7 = row & 7;
        uint32_t i = 0, xp = 0;
        int slot = 0;
        for (int64_t rb = rb0; rb < rb1; rb++, i++) {
            const uint32_t st = i & 1;
            if (!warp_wait2(xF + 8 * slot, xp, pE + 8 * st, ((i >> 1) & 1) ^ 1, &s_abort)) break;
            if (live) {
                uint32_t sc;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(sc) : "r"(raw_s + slot * RAW_S));
                if (rb == P.row_blocks - 1) {                          // scales behind the last row may hold anything
                    const int64_t left = P.n - (rb * WG_ROWS + (row & ~3));
                    const uint32_t past = left >= 4 ? 0 : left <= 0 ? 0xffffffffu : 0xffffffffu << (8 * (int)left);
                    sc = (sc & ~past) | (0x7f7f7f7fu & past);
                }
                sc >>= 8 * (row & 3);
                // 2^(scale - 7) is a bfloat16 up to 134; above, 2^127 and a second factor (255: NaN), which NaN codes take as well
                const bool large = __vcmpgtu4(sc, 0x86868686u);
                const uint32_t from = raw + slot * RAW_X, to = put + st * PLANE;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (k >= rows) break;
                    uint32_t w[4], a[4], b[4];
                    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(from + k * P.x_cols + swap * 8));
                    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[2]), "=r"(w[3]) : "r"(from + k * P.x_cols + 8 - swap * 8));
                    const uint32_t s = sc >> (8 * k) & 255, f = (s > 134 ? 254u : s + 120) * 0x00800080u;
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        a[2 * i] = expand2<0>(w[i], f); a[2 * i + 1] = expand2<1>(w[i], f);
                        b[2 * i] = expand2<0>(w[2 + i], f); b[2 * i + 1] = expand2<1>(w[2 + i], f);
                    }
                    if (large || (nan_codes(w[0]) | nan_codes(w[1]) | nan_codes(w[2]) | nan_codes(w[3])) & 0x80808080u) {
                        const uint32_t two = s == 255 ? 0x7fc07fc0u : s > 134 ? (s - 7) * 0x00800080u : 0x3f803f80u;
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            a[2 * i] = mul_bf16x2(a[2 * i], or_nan2<0>(w[i], two)); a[2 * i + 1] = mul_bf16x2(a[2 * i + 1], or_nan2<1>(w[i], two));
                            b[2 * i] = mul_bf16x2(b[2 * i], or_nan2<0>(w[2 + i], two)); b[2 * i + 1] = mul_bf16x2(b[2 * i + 1], or_nan2<1>(w[2 + i], two));
                        }
                    }
                    sts_u4(to + k * 128 + (at ^ (row7 + k)) * 16, a);
                    sts_u4(to + k * 128 + (at2 ^ (row7 + k)) * 16, b);
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) { mbar_arrive(xE + 8 * slot); mbar_arrive(pF + 8 * st); }
            if (++slot == RAW_STAGES) { slot = 0; xp ^= 1; }
        }
    } else {
        regs_inc<REG_ACC>();
        // ---------------- accumulators: a thread has a column of G, 64 columns of X of each accumulator ----------------
        // Both groups drain each accumulator, half of its columns each, so that it is soon free for the next MMAs.
        const int group = warp >= 20, own = wq * 32 + lane;
        const uint32_t from = tmem + group * (ACC_COLS / 2) + ((uint32_t)wq << 21);
        f2 acc[2][ACC_COLS / 4];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < ACC_COLS / 4; i++) acc[h][i] = 0;
        uint32_t cp[2] = {0, 0};
        const auto drain = [&](int a, f2 (&sum)[ACC_COLS / 4], int columns) {
            if (!warp_wait(cF + 8 * a, cp[a], &s_abort)) return false;
            cp[a] ^= 1;
            fence_after();
#pragma unroll
            for (int c = 0; c < ACC_COLS / 2; c += 16)
                if (c + group * (ACC_COLS / 2) < columns) {
                    uint32_t v[16];
                    tmem_ld16(from + a * ACC_COLS + c, v);
#pragma unroll
                    for (int i = 0; i < 8; i++) sum[c / 2 + i] = f2_add(sum[c / 2 + i], f2_pack(v[2 * i], v[2 * i + 1]));
                }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(cE + 8 * a);
            return true;
        };
        const int64_t turns = (rb1 - rb0 + 1) >> 1;
        if (halves == 2) {
            for (int64_t t = 0; t < turns; t++)
                if (!drain(0, acc[0], ACC_COLS) || !drain(1, acc[1], xw - ACC_COLS)) break;
        } else {
            for (int64_t t = 0; t < turns; t += 2)
                if (!drain(0, acc[0], xw) || (t + 1 < turns && !drain(1, acc[0], xw))) break;
        }
        if (g0 + own < P.cols)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int first = h * ACC_COLS + group * (ACC_COLS / 2);
                float *to = P.part + ((int64_t)slice * P.m + x0 + first) * P.cols + g0 + own;
#pragma unroll
                for (int i = 0; i < ACC_COLS / 4; i++) {
                    const float2 v = f2_get(acc[h][i]);
                    if (first + 2 * i < xw) to[(int64_t)(2 * i) * P.cols] = v.x;
                    if (first + 2 * i + 1 < xw) to[(int64_t)(2 * i + 1) * P.cols] = v.y;
                }
            }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 0) tmem_dealloc(tmem, TMEM_COLS);
    if (tid == 0 && s_abort) atomicOr(P.status, 2);
}

// Sums of the slices in order.  A warp has 128 numbers; of many slices, the eight warps of a block have the same numbers and a run of the slices each.  The numbers are
// the weight gradient's and, behind it, the bias gradient's.  Whole calls, split / not, us: 37 slices (3000 rows, 128 by 512) 10.7 / 22.0, 18 (20,000 rows, 512 by 512) 37.0 / 40.4,
// 6 (1733 rows, 384 by 1536) 19.2 / 16.7.
constexpr int SPLIT_FROM = 16;
template <bool SPLIT>
__global__ void __launch_bounds__(256) weight_finish_kernel(const float *__restrict__ part, const float *__restrict__ col_part, int slices, int64_t size, int cols,
                                                             float *__restrict__ dw, float *__restrict__ db, int64_t weight_blocks) {
    pdl_wait();
    pdl_next();
    __shared__ float s[8][128];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const bool bias = blockIdx.x >= weight_blocks;
    const int64_t first = (blockIdx.x - (bias ? weight_blocks : 0)) * (SPLIT ? 128 : 1024) + (SPLIT ? 0 : w * 128), total = bias ? cols : size;
    const float *from = bias ? col_part : part;
    const int s0 = SPLIT ? slices * w / 8 : 0, s1 = SPLIT ? slices * (w + 1) / 8 : slices;
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    if ((total & 3) == 0) {                                            // rows of slices on 16-byte boundaries
        if (first + lane * 4 < total)
#pragma unroll 8
            for (int k = s0; k < s1; k++) {
                const float4 v = __ldcs(reinterpret_cast<const float4 *>(from + k * total + first) + lane);
                t[0] += v.x; t[1] += v.y; t[2] += v.z; t[3] += v.w;
            }
    } else {
#pragma unroll 2
        for (int k = s0; k < s1; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (first + lane * 4 + i < total) t[i] += __ldcs(from + k * total + first + lane * 4 + i);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) s[w][lane * 4 + i] = t[i];
    if (!SPLIT) {
        __syncwarp();
#pragma unroll
        for (int i = lane; i < 128; i += 32)
            if (first + i < total) (bias ? db : dw)[first + i] = s[w][i];
        return;
    }
    __syncthreads();
    const int64_t i = first + threadIdx.x;
    if (threadIdx.x < 128 && i < total) {
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) sum += s[k][threadIdx.x];
        (bias ? db : dw)[i] = sum;
    }
}

int launch_status(const char *who) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return agpt_set_error(AGPT_E_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return AGPT_OK;
}

struct Shape { int blocks; int64_t pitch, tasks; };
Shape shape_of(int64_t n, int cols) {
    Shape s;
    s.blocks = (cols + 31) / 32;
    s.pitch = (n + 15) / 16 * 16;
    s.tasks = (n + PACK_ROWS - 1) / PACK_ROWS * s.blocks;
    return s;
}
int check(const char *who, int64_t n, int cols) {
    if (n < 0 || cols <= 0) return agpt_set_error(AGPT_E_ARG, "%s: bad argument", who);
    if (cols > 1 << 20 || n > (int64_t)1 << 36 || shape_of(n, cols).tasks > (int64_t)INT32_MAX * 32) return agpt_set_error(AGPT_E_LIMIT, "%s: more than 2^20 columns or too many rows", who);
    return AGPT_OK;
}

// One block per (128 columns of the gradient, up to 256 kept columns, slice of the rows): as many slices as fill the SMs, none without rows.
struct Tiles { int x_groups, x_cols, g_tiles, slices; int64_t row_blocks; };
Tiles tiles_of(int64_t n, int m, int cols) {
    Tiles t;
    t.x_groups = (m + WG_X - 1) / WG_X;
    t.x_cols = ((m + t.x_groups - 1) / t.x_groups + 31) / 32 * 32;          // split evenly
    t.x_groups = (m + t.x_cols - 1) / t.x_cols;
    t.g_tiles = (cols + WG_G - 1) / WG_G;
    t.row_blocks = (n + WG_ROWS - 1) / WG_ROWS;
    const int64_t fill = vec::sm_count() / ((int64_t)t.x_groups * t.g_tiles);
    t.slices = (int)(fill < t.row_blocks ? fill : t.row_blocks);
    if (t.slices < 1) t.slices = 1;
    return t;
}
int64_t weight_workspace(const Tiles &t, int m, int cols) { return t.slices > 1 ? ((int64_t)t.slices * m * cols + 3) / 4 * 16 + (int64_t)t.slices * cols * 4 : 0; }

// once per device: shared memory of the kernels, and the word a wait that ran out is told to
int weight_setup(int **status) {
    static std::atomic<int *> word[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && (*status = word[dev].load())) return AGPT_OK;
    cudaError_t e = cudaFuncSetAttribute(weight_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)WG_SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(weight_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)WG_SMEM);
    if (e != cudaSuccess) return agpt_set_error(AGPT_E_CUDA, "act8_weight_grad: %s", cudaGetErrorString(e));
    const int *w = nullptr;
    if (int rc = agpt_step_gemm_status_word(&w)) return rc;
    *status = const_cast<int *>(w);
    if (dev >= 0 && dev < 64) word[dev].store(*status);
    return AGPT_OK;
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// rows x cols of `type`, boxes of box_rows x box_cols without swizzle; what lies outside reads as zero
int encode_map(CUtensorMap *m, CUtensorMapDataType type, const void *p, int64_t rows, int64_t cols, int64_t ld_bytes, int box_rows, int box_cols) {
    static std::atomic<EncodeFn> found{nullptr};
    EncodeFn fn = found.load();
    if (!fn) {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q);
        if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !f) return agpt_set_error(AGPT_E_CUDA, "cuTensorMapEncodeTiled not found");
        found.store(fn = (EncodeFn)f);
    }
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, es[2] = {1, 1};
    const CUresult r = fn(m, type, 2, const_cast<void *>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return agpt_set_error(AGPT_E_CUDA, "tensor map of %lld x %lld: error %d", (long long)rows, (long long)cols, (int)r);
    return AGPT_OK;
}

}  // namespace

extern "C" int agpt_b200_act8_pack(const void *d_x, int64_t ld, int type, uint8_t *d_codes, uint8_t *d_scales, int64_t n, int cols, void *stream) {
    if (int rc = check("act8_pack", n, cols)) return rc;
    if ((type != AGPT_KV_F32 && type != AGPT_KV_BF16) || ld < cols) return agpt_set_error(AGPT_E_ARG, "act8_pack: bad type or stride");
    if (n == 0) return AGPT_OK;
    if (!d_x || !d_codes || !d_scales || !vec::aligned(d_codes, 16) || !vec::aligned(d_scales, 16))
        return agpt_set_error(AGPT_E_ARG, "act8_pack: null or unaligned argument (codes and scales start on 16-byte boundaries)");
    const Shape s = shape_of(n, cols);
    cudaStream_t st = (cudaStream_t)stream;
    const vec::Divide by(s.blocks);
    const auto grid = [&](int lanes) { return (unsigned)((s.tasks + 256 / lanes - 1) / (256 / lanes)); };
    if (type == AGPT_KV_BF16) {
        const bool whole = cols % 8 == 0 && ld % 8 == 0 && vec::aligned(d_x, 16);
        if (whole) pdl_launch(pack_kernel<bf16, 8, 1, true>, grid(4), 256, 0, st, (const bf16 *)d_x, ld, d_codes, d_scales, n, cols, s.blocks, s.pitch, by, s.tasks);
        else pdl_launch(pack_kernel<bf16, 4, 1, false>, grid(8), 256, 0, st, (const bf16 *)d_x, ld, d_codes, d_scales, n, cols, s.blocks, s.pitch, by, s.tasks);
    } else {
        const bool whole = cols % 4 == 0 && ld % 4 == 0 && vec::aligned(d_x, 16);
        if (whole) pdl_launch(pack_kernel<float, 4, 2, true>, grid(4), 256, 0, st, (const float *)d_x, ld, d_codes, d_scales, n, cols, s.blocks, s.pitch, by, s.tasks);
        else pdl_launch(pack_kernel<float, 4, 1, false>, grid(8), 256, 0, st, (const float *)d_x, ld, d_codes, d_scales, n, cols, s.blocks, s.pitch, by, s.tasks);
    }
    return launch_status("act8_pack");
}

extern "C" int agpt_b200_act8_unpack(const uint8_t *d_codes, const uint8_t *d_scales, float *d_out, int64_t n, int cols, void *stream) {
    if (int rc = check("act8_unpack", n, cols)) return rc;
    if (n == 0) return AGPT_OK;
    if (!d_out || !d_codes || !d_scales || !vec::aligned(d_codes, 16) || !vec::aligned(d_scales, 16)) return agpt_set_error(AGPT_E_ARG, "act8_unpack: null or unaligned argument");
    const Shape s = shape_of(n, cols);
    const unsigned grid = (unsigned)((s.tasks + 31) / 32);
    const vec::Divide by(s.blocks);
    cudaStream_t st = (cudaStream_t)stream;
    if (cols % 4 == 0 && vec::aligned(d_out, 16)) pdl_launch(unpack_kernel<true>, grid, 256, 0, st, d_codes, d_scales, d_out, n, cols, s.blocks, s.pitch, by, s.tasks);
    else pdl_launch(unpack_kernel<false>, grid, 256, 0, st, d_codes, d_scales, d_out, n, cols, s.blocks, s.pitch, by, s.tasks);
    return launch_status("act8_unpack");
}

extern "C" int agpt_b200_act8_relu_backward(const float *d_grad, int64_t ld, const uint8_t *d_codes, float *d_out, int64_t n, int cols, void *stream) {
    if (int rc = check("act8_relu_backward", n, cols)) return rc;
    if (ld < cols) return agpt_set_error(AGPT_E_ARG, "act8_relu_backward: bad stride");
    if (n == 0) return AGPT_OK;
    if (!d_grad || !d_out || !d_codes || !vec::aligned(d_codes, 16)) return agpt_set_error(AGPT_E_ARG, "act8_relu_backward: null or unaligned argument");
    // where a row of grad lies elsewhere than the row of out, it could be written before it is read
    if (!(d_out == d_grad && (ld == cols || n == 1)) && vec::overlap({d_out, (int64_t)cols * 4, (int64_t)cols * 4}, {d_grad, ld * 4, (int64_t)cols * 4}, n))
        return agpt_set_error(AGPT_E_ARG, "act8_relu_backward: out overlaps grad and is not grad");
    const Shape s = shape_of(n, cols);
    const unsigned grid = (unsigned)((s.tasks + 31) / 32);
    const vec::Divide by(s.blocks);
    cudaStream_t st = (cudaStream_t)stream;
    if (cols % 4 == 0 && ld % 4 == 0 && vec::aligned(d_grad, 16) && vec::aligned(d_out, 16))
        pdl_launch(relu_backward_kernel<true>, grid, 256, 0, st, d_grad, ld, d_codes, d_out, n, cols, s.blocks, by, s.tasks);
    else pdl_launch(relu_backward_kernel<false>, grid, 256, 0, st, d_grad, ld, d_codes, d_out, n, cols, s.blocks, by, s.tasks);
    return launch_status("act8_relu_backward");
}

extern "C" int64_t agpt_b200_act8_weight_grad_workspace_bytes(int64_t n, int m, int cols) {
    if (int rc = check("act8_weight_grad_workspace_bytes", n, m)) return rc;
    if (int rc = check("act8_weight_grad_workspace_bytes", n, cols)) return rc;
    return weight_workspace(tiles_of(n, m, cols), m, cols);
}

extern "C" int agpt_b200_act8_weight_grad(const uint8_t *d_codes, const uint8_t *d_scales, const float *d_grad, int64_t ld, int64_t n, int m, int cols, float *d_weight_grad,
                                          float *d_bias_grad, void *d_workspace, int64_t workspace_bytes, void *stream) {
    if (int rc = check("act8_weight_grad", n, m)) return rc;
    if (int rc = check("act8_weight_grad", n, cols)) return rc;
    if (!d_weight_grad || ld < cols || (n && (!d_codes || !d_scales || !d_grad || !vec::aligned(d_codes, 16) || !vec::aligned(d_scales, 16))))
        return agpt_set_error(AGPT_E_ARG, "act8_weight_grad: null or unaligned argument, or bad stride");
    const Tiles t = tiles_of(n, m, cols);
    const int64_t size = (int64_t)m * cols, need = weight_workspace(t, m, cols);
    if (need && (!d_workspace || workspace_bytes < need || !vec::aligned(d_workspace, 16)))
        return agpt_set_error(AGPT_E_ARG, "act8_weight_grad: workspace too small (agpt_b200_act8_weight_grad_workspace_bytes)");
    const int64_t blocks = (int64_t)t.x_groups * t.g_tiles * t.slices;
    if (n > (int64_t)INT32_MAX - WG_ROWS || blocks > INT32_MAX || size > (int64_t)INT32_MAX * 128) return agpt_set_error(AGPT_E_LIMIT, "act8_weight_grad: more than 2^31 rows, or the weight is too large");
    cudaStream_t st = (cudaStream_t)stream;
    WeightGrad P{};
    if (int rc = weight_setup(&P.status)) return rc;
    const Shape s = shape_of(n, m);
    P.grad = d_grad;
    P.part = t.slices > 1 ? (float *)d_workspace : d_weight_grad;
    P.col_part = t.slices > 1 ? P.part + (t.slices * size + 3) / 4 * 4 : d_bias_grad;
    P.ld = ld; P.n = n; P.row_blocks = t.row_blocks;
    P.m = m; P.cols = cols; P.slices = t.slices; P.x_cols = t.x_cols; P.x_groups = t.x_groups; P.g_tiles = t.g_tiles;
    // a row stride is a multiple of 16 bytes and below 2^40; one row has none
    const bool tma = ld % 4 == 0 && vec::aligned(d_grad, 16) && ld < (int64_t)1 << 36;
    if (n) {
        if (int rc = encode_map(&P.map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, d_codes, n, s.blocks * 32, s.blocks * 32, WG_ROWS, t.x_cols)) return rc;
        if (int rc = encode_map(&P.map_s, CU_TENSOR_MAP_DATA_TYPE_UINT8, d_scales, s.blocks, s.pitch, s.pitch, 8, WG_ROWS)) return rc;
        if (tma)
            if (int rc = encode_map(&P.map_g, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, d_grad, n, cols, ld * 4, WG_ROWS, WG_G)) return rc;
    }
    if (tma) pdl_launch(weight_kernel<true>, (unsigned)blocks, WG_THREADS, WG_SMEM, st, P);
    else pdl_launch(weight_kernel<false>, (unsigned)blocks, WG_THREADS, WG_SMEM, st, P);
    if (t.slices > 1) {
        const int each = t.slices >= SPLIT_FROM ? 128 : 1024;
        const int64_t weight_blocks = (size + each - 1) / each, bias_blocks = d_bias_grad ? (cols + each - 1) / each : 0;
        pdl_launch(t.slices >= SPLIT_FROM ? weight_finish_kernel<true> : weight_finish_kernel<false>, (unsigned)(weight_blocks + bias_blocks), 256, 0, st, (const float *)P.part, (const float *)P.col_part, t.slices, size, cols, d_weight_grad,
                   d_bias_grad, weight_blocks);
    }
    return launch_status("act8_weight_grad");
}
