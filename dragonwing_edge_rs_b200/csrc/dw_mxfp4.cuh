// dw_mxfp4.cuh -- device helpers of the microscaled 4-bit format (MXFP4) and of
// the element types (f32, f16, bf16) its operators read and write.
//
// A block is 32 consecutive values of a row: one scale X = 2^e held as the byte
// e + 127 and 32 codes of 4 bits (sign, then the index of 0, 0.5, 1, 1.5, 2, 3,
// 4, 6).  e = floor(log2 max|v|) - 2, so v / X lies in (-8, 8) and the
// magnitudes above 6 saturate; the quotient is exact in f32 (a power of two) and
// rounds to the nearest code, ties to even, in one cvt.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <cstring>
#include <type_traits>

#include "dw_cuda.h"

namespace dw {

// ---- element types -----------------------------------------------------------
// Conversions are IEEE round-to-nearest-even (subnormal halves keep their value).
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two f32 rounded to T, the first in the low half: one cvt.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    uint32_t u;
    memcpy(&u, &h, 4);
    return u;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    uint32_t u;
    memcpy(&u, &h, 4);
    return u;
}

// V consecutive elements as raw words, loaded with the widest access that V
// elements allow (the caller's alignment): 32, 16, 8, 4 or 2 bytes.
template <typename T, int V>
struct Raw {
    static constexpr int kBytes = (int)sizeof(T) * V;
    static constexpr int kWords = kBytes < 4 ? 1 : kBytes / 4;
    uint32_t w[kWords];

    // Plain (coherent) loads: an operator may write an operand in place.
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (kBytes == 2) {
            w[0] = *reinterpret_cast<const unsigned short *>(p);
        } else if constexpr (kBytes == 4) {
            w[0] = *reinterpret_cast<const uint32_t *>(p);
        } else if constexpr (kBytes == 8) {
            const uint2 a = *reinterpret_cast<const uint2 *>(p);
            w[0] = a.x, w[1] = a.y;
        } else {
#pragma unroll
            for (int i = 0; i < kBytes / 16; i++) {
                const uint4 a = reinterpret_cast<const uint4 *>(p)[i];
                w[4 * i] = a.x, w[4 * i + 1] = a.y, w[4 * i + 2] = a.z, w[4 * i + 3] = a.w;
            }
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; i++) w[i] = 0;
    }
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (kBytes == 2) {
            *reinterpret_cast<unsigned short *>(p) = (unsigned short)w[0];
        } else if constexpr (kBytes == 4) {
            *reinterpret_cast<uint32_t *>(p) = w[0];
        } else if constexpr (kBytes == 8) {
            *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < kBytes / 16; i++)
                reinterpret_cast<uint4 *>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else {
            if constexpr (std::is_same_v<T, __nv_bfloat16>)  // a bf16 is the upper half of its f32
                return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
            const unsigned short h = (unsigned short)(w[i >> 1] >> (16 * (i & 1)));
            T t;
            memcpy(&t, &h, 2);
            return to_f32(t);
        }
    }
    __device__ __forceinline__ void set(const float (&v)[V]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; i++) w[i] = __float_as_uint(v[i]);
        } else if constexpr (V == 1) {
            const T t = from_f32<T>(v[0]);
            unsigned short h;
            memcpy(&h, &t, 2);
            w[0] = h;
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; i++) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
        }
    }
};

// 8 elements in one access: 16 bytes, or 32 aligned ones.
template <typename T>
__device__ __forceinline__ void load_wide(Raw<T, 8> &r, const T *p) {
    if constexpr (sizeof(T) == 4)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
                       "=r"(r.w[7])
                     : "l"(p));
    else
        r.load(p);
}
template <typename T>
__device__ __forceinline__ void store_wide(const Raw<T, 8> &r, T *p) {
    if constexpr (sizeof(T) == 4)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]),
                     "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7])
                     : "memory");
    else
        r.store(p);
}

// ---- the format --------------------------------------------------------------
__host__ __device__ inline size_t mx_blocks(size_t k) { return (k + 31) / 32; }      // scales of a row
__host__ __device__ inline size_t mx_tiles(size_t k) { return (mx_blocks(k) + 3) / 4; }  // scale tiles along a row
// Byte of the scale of (row, block): tiles of 128 rows x 4 blocks, 512 bytes each;
// inside a tile 16 bytes for each r % 32, holding r / 32 = 0..3 of 4 blocks each.
// A tile is what one 32x128b tcgen05.cp brings into tensor memory, so the product
// copies scales unchanged.
__host__ __device__ inline size_t mx_scale_at(size_t row, size_t block, size_t tiles) {
    return ((row >> 7) * tiles + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// The scale byte for a block whose largest |v| has the f32 bits `amax` (sign bit
// clear; NaN compares above infinity).  Blocks holding a NaN or an infinity get
// the NaN scale 0xFF; e is clamped to -127 (amax below 2^-124, zeros included).
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
    if (amax >= 0x7F800000u) return 0xFFu;
    return (uint32_t)max((int)(amax >> 23) - 2, 0);
}

// The f32 bits of the largest |v| (a NaN where there is one), three to an instruction.
template <int N>
__device__ __forceinline__ uint32_t mx_amax(const float (&v)[N]) {
    float m = fabsf(v[0]);
    if constexpr (N % 2 == 0) asm("max.NaN.abs.f32 %0, %1, %2, %2;" : "=f"(m) : "f"(v[0]), "f"(v[N - 1]));
#pragma unroll
    for (int i = 1; i + 1 < N; i += 2) asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(m), "f"(v[i]), "f"(v[i + 1]));
    return __float_as_uint(m);
}

// 1 / X (scale byte <= 252; 0 for the NaN scale, whose codes are 0).
__device__ __forceinline__ float mx_inv_scale(uint32_t byte) {
    return byte == 0xFFu ? 0.0f : __uint_as_float((254u - byte) << 23);
}

// X, exact: 2^-127 is subnormal; 0xFF is NaN.
__device__ __forceinline__ float mx_scale(uint32_t byte) {
    if (byte == 0xFFu) return __uint_as_float(0x7FC00000u);
    return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// Codes of 8 / 2 values already divided by X (low nibble first).
__device__ __forceinline__ uint32_t mx_codes8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
__device__ __forceinline__ uint32_t mx_codes2(float a, float b) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "mov.b32 %0, {b0, b0, b0, b0};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b));
    return r & 0xFFu;
}

// The 8 values of 4 code bytes (before the scale), exact.
__device__ __forceinline__ void mx_decode8(uint32_t c, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(c));
#pragma unroll
    for (int i = 0; i < 4; i++) {
        __half2 t;
        memcpy(&t, &h[i], 4);
        const float2 f = __half22float2(t);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}

// The value of the code in the low four bits.
__device__ __forceinline__ float mx_decode1(uint32_t c) {
    uint32_t h;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t}"
        : "=r"(h)
        : "r"(c));
    __half2 t;
    memcpy(&t, &h, 4);
    return __low2float(t);
}

// 32 values of one thread -> 16 code bytes and the scale byte.
__device__ __forceinline__ uint32_t mx_quantize32(const float (&v)[32], uint4 &codes) {
    const uint32_t s = mx_scale_byte(mx_amax(v));
    const float inv = mx_inv_scale(s);
    uint32_t c[4];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = v[8 * q + i] * inv;
        c[q] = mx_codes8(t);
    }
    codes = s == 0xFFu ? make_uint4(0, 0, 0, 0) : make_uint4(c[0], c[1], c[2], c[3]);
    return s;
}

}  // namespace dw
