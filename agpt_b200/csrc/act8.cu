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
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/agpt_b200.h"
#include "internal.h"
#include "pdl.cuh"
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
// what a scale byte stands for
__device__ __forceinline__ float scale_of(uint32_t s) { return __uint_as_float(s == 255 ? 0x7fc00000u : s ? s << 23 : 0x00400000u); }

// A group of 32 / VEC lanes has a block of PACK_ROWS consecutive rows: their loads are in flight together and their scale bytes are neighbours.
constexpr int PACK_ROWS = 4;
template <typename T, int VEC, bool WHOLE>
__global__ void __launch_bounds__(256) pack_kernel(const T *__restrict__ x, int64_t ld, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales, int64_t n, int cols,
                                                    int blocks, int64_t pitch, vec::Divide by_blocks, int64_t tasks) {
    pdl_wait();
    pdl_next();
    constexpr int LANES = 32 / VEC;
    const int lane = threadIdx.x % LANES;
    const int64_t task = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (task >= tasks) return;                         // whole groups leave; the shuffles below stay inside a group
    const uint32_t group = ((LANES == 32 ? 0u : 1u << LANES) - 1) << (threadIdx.x & 31 & ~(LANES - 1));
    const int64_t quad = vec::quotient(task, by_blocks), r0 = quad * PACK_ROWS;
    const int b = (int)(task - quad * blocks), c = b * 32 + lane * VEC;
    float v[PACK_ROWS][VEC];
#pragma unroll
    for (int u = 0; u < PACK_ROWS; u++) {
        const bool live = r0 + u < n;
        if (WHOLE) {
            if (live && c < cols) vec::load<VEC>(x + (r0 + u) * ld + c, v[u]);
            else
#pragma unroll
                for (int i = 0; i < VEC; i++) v[u][i] = 0.f;
        } else
#pragma unroll
            for (int i = 0; i < VEC; i++) v[u][i] = live && c + i < cols ? (float)x[(r0 + u) * ld + c + i] : 0.f;
    }
    uint32_t s4 = 0;
#pragma unroll
    for (int u = 0; u < PACK_ROWS; u++) {
        uint32_t top = 0;                              // magnitudes in order of their bits, infinity and NaN above all
#pragma unroll
        for (int i = 0; i < VEC; i++) top = max(top, __float_as_uint(v[u][i]) & 0x7fffffffu);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(group, top, o));
        // 2^k <= top < 2^(k+1), k = (top >> 23) - 127: top <= 448 * 2^(k-8) = 1.75 * 2^k, or one more
        const int e = max((int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u), -110);
        const bool bad = top >= 0x7f800000u;
        s4 |= (bad ? 255u : (uint32_t)(e + 127)) << (8 * u);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        uint32_t word[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            uint32_t w = codes2(v[u][i] * down, v[u][i + 1] * down) | codes2(v[u][i + 2] * down, v[u][i + 3] * down) << 16;
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (v[u][i + k] != 0.f && !(w >> (8 * k) & 0x7f)) w |= 1u << (8 * k) | (v[u][i + k] < 0.f ? 0x80u << (8 * k) : 0u);
            // 256 * 2^120 and above are no float32: what rounds there takes 240 * 2^120
            if (e == 120)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if ((w >> (8 * k) & 0x7f) > 0x77) w = (w & ~(0x7fu << (8 * k))) | 0x77u << (8 * k);
            word[i / 4] = bad ? 0x7f7f7f7fu : w;
        }
        if (r0 + u < n) {
            uint8_t *to = codes + (r0 + u) * (int64_t)blocks * 32 + c;
            if (VEC == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(word[0], word[VEC / 4 - 1]);
            else *reinterpret_cast<uint32_t *>(to) = word[0];
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
            if (c < cols) vec::store<4>(to, v);
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
            if (c < cols) vec::store<4>(to, v[u]);
        } else
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (c + i < cols) to[i] = v[u][i];
    }
}

// ---- weight gradient: dW[m][N] = X^T G, db[N] = column sums of G ----------------------------------------------------------------------
// A block has 64 x 64 of dW and a slice of the rows; partial sums are added in slice order.
constexpr int WG_TILE = 64, WG_ROWS = 32;
__global__ void __launch_bounds__(256) weight_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, int64_t pitch, int blocks,
                                                      const float *__restrict__ grad, int64_t ld, int64_t n, int m, int cols, int64_t chunk, float *__restrict__ part,
                                                      float *__restrict__ col_part) {
    pdl_wait();
    pdl_next();
    __shared__ float sx[WG_ROWS][WG_TILE + 4], sg[WG_ROWS][WG_TILE + 4];
    const int m0 = blockIdx.x * WG_TILE, c0 = blockIdx.y * WG_TILE, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t r0 = (int64_t)blockIdx.z * chunk, r1 = min(r0 + chunk, n);
    float acc[4][4] = {}, sum = 0.f;
    for (int64_t r = r0; r < r1; r += WG_ROWS) {
        for (int i = threadIdx.x; i < WG_ROWS * WG_TILE; i += 256) {
            const int k = i / WG_TILE, j = i % WG_TILE;
            const bool live = r + k < r1;
            float x = 0.f;
            if (live && m0 + j < m)
                x = values2(codes[(r + k) * (int64_t)blocks * 32 + m0 + j]).x * scale_of(scales[(int64_t)((m0 + j) >> 5) * pitch + r + k]);
            sx[k][j] = x;
            sg[k][j] = live && c0 + j < cols ? grad[(r + k) * ld + c0 + j] : 0.f;
        }
        __syncthreads();
        for (int k = 0; k < WG_ROWS; k++) {
            float a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; i++) { a[i] = sx[k][ty * 4 + i]; b[i] = sg[k][tx * 4 + i]; }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] += a[i] * b[j];
        }
        if (threadIdx.x < WG_TILE)
            for (int k = 0; k < WG_ROWS; k++) sum += sg[k][threadIdx.x];
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int mm = m0 + ty * 4 + i, cc = c0 + tx * 4 + j;
            if (mm < m && cc < cols) part[((int64_t)blockIdx.z * m + mm) * cols + cc] = acc[i][j];
        }
    if (blockIdx.x == 0 && threadIdx.x < WG_TILE && c0 + threadIdx.x < cols) col_part[(int64_t)blockIdx.z * cols + c0 + threadIdx.x] = sum;
}

__global__ void __launch_bounds__(256) weight_finish_kernel(const float *__restrict__ part, const float *__restrict__ col_part, int slices, int64_t size, int cols,
                                                             float *__restrict__ dw, float *__restrict__ db) {
    pdl_wait();
    pdl_next();
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < size) {
        float t = 0.f;
#pragma unroll 8
        for (int s = 0; s < slices; s++) t += __ldcs(part + s * size + i);
        dw[i] = t;
    } else if (db && i < size + cols) {
        const int c = (int)(i - size);
        float t = 0.f;
#pragma unroll 8
        for (int s = 0; s < slices; s++) t += __ldcs(col_part + (int64_t)s * cols + c);
        db[c] = t;
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

int weight_slices(int64_t n, int m, int cols) {
    const int64_t tiles = (int64_t)((m + WG_TILE - 1) / WG_TILE) * ((cols + WG_TILE - 1) / WG_TILE);
    int64_t s = (int64_t)vec::sm_count() * 4 / tiles;
    const int64_t most = (n + WG_ROWS - 1) / WG_ROWS;
    s = s < most ? s : most;
    return (int)(s < 1 ? 1 : s);
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
        if (whole) pdl_launch(pack_kernel<bf16, 8, true>, grid(4), 256, 0, st, (const bf16 *)d_x, ld, d_codes, d_scales, n, cols, s.blocks, s.pitch, by, s.tasks);
        else pdl_launch(pack_kernel<bf16, 4, false>, grid(8), 256, 0, st, (const bf16 *)d_x, ld, d_codes, d_scales, n, cols, s.blocks, s.pitch, by, s.tasks);
    } else {
        const bool whole = cols % 4 == 0 && ld % 4 == 0 && vec::aligned(d_x, 16);
        if (whole) pdl_launch(pack_kernel<float, 4, true>, grid(8), 256, 0, st, (const float *)d_x, ld, d_codes, d_scales, n, cols, s.blocks, s.pitch, by, s.tasks);
        else pdl_launch(pack_kernel<float, 4, false>, grid(8), 256, 0, st, (const float *)d_x, ld, d_codes, d_scales, n, cols, s.blocks, s.pitch, by, s.tasks);
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
    return (int64_t)weight_slices(n, m, cols) * ((int64_t)m * cols + cols) * 4;
}

extern "C" int agpt_b200_act8_weight_grad(const uint8_t *d_codes, const uint8_t *d_scales, const float *d_grad, int64_t ld, int64_t n, int m, int cols, float *d_weight_grad,
                                          float *d_bias_grad, void *d_workspace, int64_t workspace_bytes, void *stream) {
    if (int rc = check("act8_weight_grad", n, m)) return rc;
    if (int rc = check("act8_weight_grad", n, cols)) return rc;
    if (!d_weight_grad || ld < cols || (n && (!d_codes || !d_scales || !d_grad || !vec::aligned(d_codes, 16) || !vec::aligned(d_scales, 16))))
        return agpt_set_error(AGPT_E_ARG, "act8_weight_grad: null or unaligned argument, or bad stride");
    if (!d_workspace || workspace_bytes < agpt_b200_act8_weight_grad_workspace_bytes(n, m, cols) || !vec::aligned(d_workspace, 16))
        return agpt_set_error(AGPT_E_ARG, "act8_weight_grad: workspace too small (agpt_b200_act8_weight_grad_workspace_bytes)");
    cudaStream_t st = (cudaStream_t)stream;
    const int slices = weight_slices(n, m, cols);
    const int64_t chunk = ((n + slices - 1) / slices + WG_ROWS - 1) / WG_ROWS * WG_ROWS, size = (int64_t)m * cols;
    float *part = (float *)d_workspace, *col_part = part + slices * size;
    const Shape s = shape_of(n, m);
    pdl_launch(weight_kernel, dim3((m + WG_TILE - 1) / WG_TILE, (cols + WG_TILE - 1) / WG_TILE, slices), 256, 0, st, d_codes, d_scales, s.pitch, s.blocks, d_grad, ld, n, m, cols,
               chunk, part, col_part);
    pdl_launch(weight_finish_kernel, (unsigned)((size + cols + 255) / 256), 256, 0, st, (const float *)part, (const float *)col_part, slices, size, cols, d_weight_grad, d_bias_grad);
    return launch_status("act8_weight_grad");
}
