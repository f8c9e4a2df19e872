// mxfp4.cu -- quantisation to microscaled 4-bit floating point, back, and the
// layout of row-major scales (format: dw_mxfp4.cuh).  Bandwidth-bound streaming
// kernels.

#include <algorithm>

#include "dw_device.cuh"
#include "dw_launch.h"
#include "dw_mxfp4.cuh"

namespace dw {
namespace {

constexpr int kThreads = 256;

// 16 threads take 128 values of a row, 8 each: four blocks.  A thread does so for four
// rows, 32 apart, whose scales are 16 neighbouring bytes of a tile: four independent
// loads in flight, and its addresses and bounds worked out once.  A thread block is
// `ux` such units across and kThreads / (16 * ux) rows of a 32-row group down.  Both
// kernels are near the issue rate, not only the memory's (8192 x 4096 f16 took 19.3 us
// to quantise at 135 instructions for 8 values, 15.6 at 110, 13.7 at 80).  With other
// inputs each time, out of L2, that takes 15.2 us, by stores of single scale bytes 15.6;
// its bytes take 13.2 at the copy rate.
constexpr int kRows = 4;

struct Shape {
    size_t rows, k, pitch;  // pitch: elements from row to row
    size_t nb, tiles;
    int lux;                // log2(ux)
    bool vec;               // rows start on 16-byte boundaries (f32: 32-byte)
};

struct Place {
    size_t row, col;  // of the first row's 8 values
    size_t scale;     // byte of the unit's 16 scales: four words, one for each row, of four blocks
    int rows;         // how many of the four rows there are
    bool whole;       // 8 values, loaded or stored at once
    __device__ __forceinline__ explicit Place(const Shape &p) {
        const uint32_t u = (threadIdx.x >> 4) & ((1u << p.lux) - 1);
        const int lr = 4 - p.lux;  // log2(rows of a thread block)
        const uint32_t r32 = ((blockIdx.x & ((32u >> lr) - 1)) << lr) + (threadIdx.x >> (4 + p.lux));
        const size_t unit = ((size_t)blockIdx.y << p.lux) + u, tile = blockIdx.x >> (5 - lr);
        col = (unit << 7) + (threadIdx.x & 15) * 8;
        row = tile * 128 + r32;
        scale = (tile * p.tiles + unit) * 512 + r32 * 16;
        rows = row >= p.rows ? 0 : (int)min((p.rows - row + 31) >> 5, (size_t)kRows);
        whole = p.vec && col + 8 <= p.k;
    }
};

// The bits of the largest |v| of 8 values, as f32.
template <typename T>
__device__ __forceinline__ uint32_t amax8(const Raw<T, 8> &r) {
    if constexpr (sizeof(T) == 4) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = r.get(i);
        return mx_amax(v);
    } else {
        // two to a word: magnitudes order like their bits
        uint32_t m = __vmaxu2(__vmaxu2(r.w[0] & 0x7FFF7FFFu, r.w[1] & 0x7FFF7FFFu),
                              __vmaxu2(r.w[2] & 0x7FFF7FFFu, r.w[3] & 0x7FFF7FFFu));
        m = max(m & 0xFFFFu, m >> 16);
        if constexpr (std::is_same_v<T, __nv_bfloat16>) return m << 16;
        return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
    }
}

// 8 elements from anywhere: the widest accesses that the address allows; 16-bit elements
// at an odd place from the five words around them, where these lie in [first, last)
// (8192 x 4095 f16 22.9 us with its rows at every phase, 8192 x 4096 15.3).
template <typename T>
__device__ __forceinline__ void load_any(Raw<T, 8> &r, const T *src, const T *first, const T *last) {
    const uint32_t a = (uint32_t)(uintptr_t)src & 15;
    constexpr int kWords = Raw<T, 8>::kWords;
    if (a == 0) {
        r.load(src);
    } else if ((a & 7) == 0) {
#pragma unroll
        for (int i = 0; i < kWords / 2; i++) {
            const uint2 w = reinterpret_cast<const uint2 *>(src)[i];
            r.w[2 * i] = w.x, r.w[2 * i + 1] = w.y;
        }
    } else if ((a & 3) == 0) {
#pragma unroll
        for (int i = 0; i < kWords; i++) r.w[i] = reinterpret_cast<const uint32_t *>(src)[i];
    } else if (sizeof(T) == 2 && src > first && src + 9 <= last) {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(src - 1);
        uint32_t lo = w[0];
#pragma unroll
        for (int i = 0; i < kWords; i++) {
            const uint32_t hi = w[i + 1];
            r.w[i] = __funnelshift_r(lo, hi, 16);
            lo = hi;
        }
    } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = to_f32(src[i]);
        r.set(v);
    }
}

// 8 values divided by X, as f32.  The 16-bit types are scaled in their own type, two at
// a time: a power of two changes no digit (what falls below the smallest f16 would round
// to code 0), unless it is beyond f16 (then `inv` > 2^15 and f32 does it).
template <typename T>
__device__ __forceinline__ void scale8(const Raw<T, 8> &r, float inv, float (&v)[8]) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        const __nv_bfloat162 f = __float2bfloat162_rn(inv);
        Raw<T, 8> t;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            __nv_bfloat162 h;
            memcpy(&h, &r.w[i], 4);
            h = __hmul2(h, f);
            memcpy(&t.w[i], &h, 4);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = t.get(i);
    } else if constexpr (sizeof(T) == 2) {
        if (inv <= 32768.0f) {
            const __half2 f = __float2half2_rn(inv);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                __half2 h;
                memcpy(&h, &r.w[i], 4);
                const float2 g = __half22float2(__hmul2(h, f));
                v[2 * i] = g.x, v[2 * i + 1] = g.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = r.get(i) * inv;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = r.get(i) * inv;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_quantize_mxfp4(const T *x, uint8_t *q, uint8_t *s,
                                                             const __grid_constant__ Shape p) {
    pdl_wait();
    pdl_trigger();
    const Place at(p);
    const T *src = x + at.row * p.pitch + at.col;
    Raw<T, 8> raw[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++, src += 32 * p.pitch) {
        raw[i].zero();
        if (i >= at.rows || at.col >= p.k) continue;
        if (at.whole) {
            load_wide(raw[i], src);
        } else if (at.col + 8 <= p.k) {
            load_any(raw[i], src, x, x + (p.rows - 1) * p.pitch + p.k);
        } else {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = at.col + j < p.k ? to_f32(src[j]) : 0.0f;
            raw[i].set(v);
        }
    }
    uint8_t *dst = q + (at.row * p.nb * 32 + at.col) / 2;
    s += at.scale;  // the unit's
    const bool codes_here = at.col < p.nb * 32;
    const int lane16 = threadIdx.x & 15;
    uint32_t scales = 0;  // of block lane16 / 4 and row lane16 % 4
#pragma unroll
    for (int i = 0; i < kRows; i++, dst += p.nb * 512) {
        uint32_t amax = amax8(raw[i]);
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const uint32_t sb = mx_scale_byte(amax);
        float v[8];
        scale8(raw[i], mx_inv_scale(sb), v);
        const uint32_t codes = sb == 0xFFu ? 0u : mx_codes8(v);
        if ((lane16 & 3) == i) scales = sb;
        if (i < at.rows && codes_here) *reinterpret_cast<uint32_t *>(dst) = codes;
    }
    // the unit's 16 scales: a row's four are a word, which the thread of that row stores
    scales <<= 8 * (lane16 >> 2);
    scales |= __shfl_xor_sync(0xffffffffu, scales, 4);
    scales |= __shfl_xor_sync(0xffffffffu, scales, 8);
    if (lane16 < at.rows && at.col < p.tiles * 128) *reinterpret_cast<uint32_t *>(s + 4 * lane16) = scales;
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) k_dequantize_mxfp4(const uint8_t *q, const uint8_t *s, T *y,
                                                               const __grid_constant__ Shape p) {
    pdl_wait();
    pdl_trigger();
    const Place at(p);
    if (kVec && at.col >= p.k) return;
    const uint8_t *src = q + (at.row * p.nb * 32 + at.col) / 2;
    s += at.scale;
    uint32_t codes[kRows], sb[kRows] = {};
    if (at.rows && at.col < p.k) {
        const uint4 w = *reinterpret_cast<const uint4 *>(s);
        sb[0] = w.x, sb[1] = w.y, sb[2] = w.z, sb[3] = w.w;
    }
#pragma unroll
    for (int i = 0; i < kRows; i++, src += p.nb * 512) {
        codes[i] = 0;
        if (i >= at.rows || at.col >= p.k) continue;
        codes[i] = *reinterpret_cast<const uint32_t *>(src);
    }
#pragma unroll
    for (int i = 0; i < kRows; i++) sb[i] = (sb[i] >> (8 * ((threadIdx.x & 15) >> 2))) & 0xFFu;
    if constexpr (!kVec) {
        // rows that start anywhere: the 16 threads of a unit write 16 neighbours at a time
        // (each its own 8, one by one, took 5.8 instead of 2.6 us for 1000 x 1010 f32).  Two
        // shuffles and a store an element: 8192 x 4095 f16 28.2 us, 8192 x 4096 15.0.
        const int lane16 = threadIdx.x & 15;
        const size_t col0 = at.col - lane16 * 8;
        T *dst = y + at.row * p.k + col0 + lane16;
#pragma unroll
        for (int i = 0; i < kRows; i++, dst += 32 * p.k)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t c = __shfl_sync(0xffffffffu, codes[i], 2 * j + (lane16 >> 3), 16);
                const uint32_t b = __shfl_sync(0xffffffffu, sb[i], 2 * j, 16);
                const float v = mx_decode1(c >> (4 * (lane16 & 7))) * mx_scale(b);
                if (i < at.rows && col0 + 16 * j + lane16 < p.k) dst[16 * j] = from_f32<T>(v);
            }
        return;
    }
    T *dst = y + at.row * p.k + at.col;
#pragma unroll
    for (int i = 0; i < kRows; i++, dst += 32 * p.k) {
        if (i >= at.rows) continue;
        float v[8];
        mx_decode8(codes[i], v);
        const float X = mx_scale(sb[i]);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] *= X;
        Raw<T, 8> r;  // all 8 lie in the row: k is a multiple of 8 here
        r.set(v);
        store_wide(r, dst);
    }
}

// Row-major scales [rows][nb] -> tiles; the places of a tile past the last block
// get byte 0 (rows past the last are left as they are).  One thread per (row, tile), four
// byte loads each: 11008 x 4096 3.9 us against 0.4 for its bytes, once for a weight.
__global__ void __launch_bounds__(kThreads) k_pack_scales(const uint8_t *in, uint8_t *s, size_t rows, size_t nb,
                                                          size_t tiles) {
    pdl_wait();
    pdl_trigger();
    const size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= rows * tiles) return;
    const size_t row = i / tiles, t = i - row * tiles;
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (t * 4 + j < nb) w |= (uint32_t)in[row * nb + t * 4 + j] << (8 * j);
    *reinterpret_cast<uint32_t *>(s + mx_scale_at(row, t * 4, tiles)) = w;
}

// The grid of the streaming kernels: x over 128-row tiles and groups of their 32 rows, y
// over groups of units.
bool make_shape(size_t rows, size_t k, size_t pitch, bool vec, Shape *p, dim3 *grid) {
    p->rows = rows, p->k = k, p->pitch = pitch, p->vec = vec;
    p->nb = mx_blocks(k), p->tiles = mx_tiles(k);
    p->lux = 0;
    while (p->lux < 4 && ((size_t)1 << p->lux) < p->tiles) p->lux++;
    const size_t per_block = kThreads >> (4 + p->lux);  // rows of a thread block, of a group's 32
    // (one tile needs only the groups that it has rows in)
    const size_t gx = rows <= 32 ? (rows + per_block - 1) / per_block : (rows + 127) / 128 * (32 / per_block);
    const size_t gy = (p->tiles + ((size_t)1 << p->lux) - 1) >> p->lux;
    if (gx > 0x7fffffffu || gy > 65535u) return false;
    *grid = dim3((unsigned)gx, (unsigned)gy);
    return true;
}

template <typename T>
dw_status quantize(dw_backend *be, const void *x, size_t rows, size_t k, size_t pitch, uint8_t *q, uint8_t *s) {
    Shape p;
    dim3 grid;
    constexpr size_t kWide = sizeof(T) * 8;
    const bool vec = (uintptr_t)x % kWide == 0 && pitch * sizeof(T) % kWide == 0;
    if (!make_shape(rows, k, pitch, vec, &p, &grid))
        return dw_fail(be, DW_ERR_UNSUPPORTED, "quantize_mxfp4: %zu x %zu is too large", rows, k);
    return launch_dependent(be, "quantize_mxfp4", k_quantize_mxfp4<T>, grid, kThreads, 0, 0, (const T *)x, q, s, p);
}

template <typename T>
dw_status dequantize(dw_backend *be, const uint8_t *q, const uint8_t *s, size_t rows, size_t k, void *y) {
    Shape p;
    dim3 grid;
    constexpr size_t kWide = sizeof(T) * 8;
    const bool vec = (uintptr_t)y % kWide == 0 && k * sizeof(T) % kWide == 0;
    if (!make_shape(rows, k, k, vec, &p, &grid))
        return dw_fail(be, DW_ERR_UNSUPPORTED, "dequantize_mxfp4: %zu x %zu is too large", rows, k);
    return launch_dependent(be, "dequantize_mxfp4", vec ? k_dequantize_mxfp4<T, true> : k_dequantize_mxfp4<T, false>, grid, kThreads, 0, 0, q, s, (T *)y, p);
}

}  // namespace

dw_status launch_quantize_mxfp4(dw_backend *be, const void *x, int dtype, size_t rows, size_t k, size_t pitch, uint8_t *q,
                                uint8_t *s) {
    switch (dtype) {
        case DW_F32: return quantize<float>(be, x, rows, k, pitch, q, s);
        case DW_F16: return quantize<__half>(be, x, rows, k, pitch, q, s);
        default: return quantize<__nv_bfloat16>(be, x, rows, k, pitch, q, s);
    }
}

dw_status launch_dequantize_mxfp4(dw_backend *be, const uint8_t *q, const uint8_t *s, size_t rows, size_t k, void *y,
                                  int dtype) {
    switch (dtype) {
        case DW_F32: return dequantize<float>(be, q, s, rows, k, y);
        case DW_F16: return dequantize<__half>(be, q, s, rows, k, y);
        default: return dequantize<__nv_bfloat16>(be, q, s, rows, k, y);
    }
}

dw_status launch_pack_scales_mxfp4(dw_backend *be, const uint8_t *in, size_t rows, size_t k, uint8_t *s) {
    const size_t nb = mx_blocks(k), tiles = mx_tiles(k), blocks = (rows * tiles + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffu) return dw_fail(be, DW_ERR_UNSUPPORTED, "pack_scales_mxfp4: %zu x %zu is too large", rows, k);
    return launch_dependent(be, "pack_scales_mxfp4", k_pack_scales, (unsigned)blocks, kThreads, 0, 0, in, s, rows, nb, tiles);
}

}  // namespace dw
