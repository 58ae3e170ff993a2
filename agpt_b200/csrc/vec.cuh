// Accesses shared by the row operators whose rows are float32 or bfloat16: a piece of a row as floats, and back.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace vec {

// VEC neighbouring elements, VEC > 1 by one access of their size (16 bytes where a lane takes float4 or eight bfloat16)
template <int VEC> __device__ __forceinline__ void load(const float *p, float (&v)[VEC]) {
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 x = __ldcs(reinterpret_cast<const float4 *>(p + i));
            v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = __ldcs(p + i);
    }
}
__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
template <int VEC> __device__ __forceinline__ void load(const __nv_bfloat16 *p, float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        const uint4 x = __ldcs(reinterpret_cast<const uint4 *>(p));
        v[0] = low(x.x); v[1] = high(x.x); v[2] = low(x.y); v[3] = high(x.y);
        v[4] = low(x.z); v[5] = high(x.z); v[6] = low(x.w); v[7] = high(x.w);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = __bfloat162float(p[i]);
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
}

// The same in two steps, so that many loads are on their way before the first value is asked for: fetch() is one predicated load without a branch (zeros where it
// is not wanted), values() turns what came into floats.  A conversion behind a guarded load would make each load wait for the one before.
template <typename T, int VEC> struct Piece {
    static constexpr int WORDS = VEC * (int)sizeof(T) / 4, N = WORDS > 0 ? WORDS : 1;
    uint32_t w[N];
    __device__ __forceinline__ void fetch(const T *p, bool wanted) {
        if constexpr (WORDS >= 4) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4)
                asm volatile("{ .reg .pred p; setp.ne.u32 p, %5, 0; mov.b32 %0, 0; mov.b32 %1, 0; mov.b32 %2, 0; mov.b32 %3, 0; @p ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4]; }"
                             : "=&r"(w[i]), "=&r"(w[i + 1]), "=&r"(w[i + 2]), "=&r"(w[i + 3]) : "l"(reinterpret_cast<const uint32_t *>(p) + i), "r"((uint32_t)wanted));
        } else if constexpr (WORDS == 2 && VEC == 4) {
            asm volatile("{ .reg .pred p; setp.ne.u32 p, %3, 0; mov.b32 %0, 0; mov.b32 %1, 0; @p ld.global.cs.v2.u32 {%0, %1}, [%2]; }"
                         : "=&r"(w[0]), "=&r"(w[1]) : "l"(p), "r"((uint32_t)wanted));
        } else if constexpr (VEC == 1) {
            w[0] = 0;
            if constexpr (sizeof(T) == 4)
                asm volatile("{ .reg .pred p; setp.ne.u32 p, %2, 0; mov.b32 %0, 0; @p ld.global.cs.u32 %0, [%1]; }" : "=&r"(w[0]) : "l"(p), "r"((uint32_t)wanted));
            else {
                uint16_t h;
                asm volatile("{ .reg .pred p; setp.ne.u32 p, %2, 0; mov.b16 %0, 0; @p ld.global.cs.u16 %0, [%1]; }" : "=&h"(h) : "l"(p), "r"((uint32_t)wanted));
                w[0] = h;
            }
        } else {                                       // pairs off every boundary
#pragma unroll
            for (int i = 0; i < N; i++) w[i] = 0;
            if (wanted)
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    if constexpr (sizeof(T) == 4) w[i] = __ldcs(reinterpret_cast<const unsigned int *>(p) + i);
                    else w[i / 2] |= (uint32_t)__ldcs(reinterpret_cast<const unsigned short *>(p) + i) << (16 * (i & 1));
                }
        }
    }
    // the same through the caches, for rows that are read again
    __device__ __forceinline__ void fetch_kept(const T *p, bool wanted) {
        if constexpr (WORDS >= 4) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4)
                asm volatile("{ .reg .pred p; setp.ne.u32 p, %5, 0; mov.b32 %0, 0; mov.b32 %1, 0; mov.b32 %2, 0; mov.b32 %3, 0; @p ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4]; }"
                             : "=&r"(w[i]), "=&r"(w[i + 1]), "=&r"(w[i + 2]), "=&r"(w[i + 3]) : "l"(reinterpret_cast<const uint32_t *>(p) + i), "r"((uint32_t)wanted));
        } else if constexpr (sizeof(T) == 4) {
            asm volatile("{ .reg .pred p; setp.ne.u32 p, %2, 0; mov.b32 %0, 0; @p ld.global.nc.u32 %0, [%1]; }" : "=&r"(w[0]) : "l"(p), "r"((uint32_t)wanted));
        } else {
            uint16_t h;
            asm volatile("{ .reg .pred p; setp.ne.u32 p, %2, 0; mov.b16 %0, 0; @p ld.global.nc.u16 %0, [%1]; }" : "=&h"(h) : "l"(p), "r"((uint32_t)wanted));
            w[0] = h;
        }
    }
    __device__ __forceinline__ void values(float (&v)[VEC]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < VEC; i++) v[i] = __uint_as_float(w[i]);
        } else if constexpr (VEC == 1) v[0] = low(w[0]);
        else
#pragma unroll
            for (int i = 0; i < VEC; i += 2) { v[i] = low(w[i / 2]); v[i + 1] = high(w[i / 2]); }
    }
};

// n rows of `width` bytes, `pitch` bytes apart: whether two such sets share bytes (of different pitches, whether their spans do)
struct Span { const void *p; int64_t pitch, width; };
inline bool overlap(Span a, Span b, int64_t n) {
    int64_t between = (int64_t)(reinterpret_cast<uintptr_t>(b.p) - reinterpret_cast<uintptr_t>(a.p));
    if (between < 0) { const Span t = a; a = b; b = t; between = -between; }
    if (between >= (n - 1) * a.pitch + a.width) return false;
    if (n == 1 || a.pitch != b.pitch) return true;
    between %= a.pitch;
    return between < a.width || between + b.width > a.pitch;
}

inline bool aligned(const void *p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

// outputs larger than the caches: whole pieces of 16 bytes are written past them
template <int VEC> __device__ __forceinline__ void store_past(float *p, const float (&v)[VEC]) {
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) __stcs(reinterpret_cast<float4 *>(p) + i / 4, make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) p[i] = v[i];
    }
}
// one rounding to bfloat16, to nearest, of the float32 result
template <int VEC> __device__ __forceinline__ void store_past(__nv_bfloat16 *p, const float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        __stcs(reinterpret_cast<uint4 *>(p), make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])));
    } else if constexpr (VEC == 4) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) p[i] = __float2bfloat16_rn(v[i]);
    }
}

// Division of 64-bit task numbers by a launch constant: the upper half of a product with ceil(2^64 / d), exact while task * d < 2^64
struct Divide {
    uint64_t m;
    explicit Divide(uint32_t d) : m(d > 1 ? ~0ull / d + 1 : 0) {}
};
__device__ __forceinline__ int64_t quotient(int64_t a, Divide d) { return d.m ? (int64_t)__umul64hi((uint64_t)a, d.m) : a; }

inline int sm_count() {
    static int n[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return 148;
    if (!n[dev]) cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev);
    return n[dev] > 0 ? n[dev] : 148;
}

}  // namespace vec
