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

// 16 threads take one unit: 128 values of a row, 8 each, four blocks, four
// scale bytes of one tile.  A thread block is `ux` units across and
// kThreads / (16 * ux) rows down, and does kRows such groups of rows, so that
// each thread has kRows independent loads in flight.
struct Shape {
    size_t rows, k, pitch;  // pitch: elements from row to row
    size_t nb, tiles;
    int lux;                // log2(ux)
    bool vec;               // rows start on 16-byte boundaries
};

template <typename T, int kRows>
__global__ void __launch_bounds__(kThreads) k_quantize_mxfp4(const T *__restrict__ x, uint8_t *__restrict__ q,
                                                             uint8_t *__restrict__ s, Shape p) {
    const int lane16 = threadIdx.x & 15;
    const int u = (threadIdx.x >> 4) & ((1 << p.lux) - 1);
    const int ry = threadIdx.x >> (4 + p.lux);
    const int rows_blk = kThreads >> (4 + p.lux);
    const size_t unit = ((size_t)blockIdx.y << p.lux) + u;
    const size_t col = unit * 128 + lane16 * 8;
    const size_t row0 = (size_t)blockIdx.x * rows_blk * kRows + ry;
    pdl_wait();
    pdl_trigger();
    Raw<T, 8> raw[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++) {
        const size_t row = row0 + (size_t)i * rows_blk;
        raw[i].zero();
        if (row >= p.rows || col >= p.k) continue;
        const T *src = x + row * p.pitch + col;
        if (p.vec && col + 8 <= p.k) {
            raw[i].load(src);
        } else {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = col + j < p.k ? to_f32(src[j]) : 0.0f;
            raw[i].set(v);
        }
    }
#pragma unroll
    for (int i = 0; i < kRows; i++) {
        const size_t row = row0 + (size_t)i * rows_blk;
        float v[8];
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[j] = raw[i].get(j);
            amax = max(amax, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        }
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const uint32_t sb = mx_scale_byte(amax);
        const float inv = mx_inv_scale(sb);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] *= inv;
        const uint32_t codes = sb == 0xFFu ? 0u : mx_codes8(v);
        // the unit's four scale bytes, gathered from threads 0, 4, 8, 12 of the 16
        uint32_t sw = sb << (8 * (lane16 >> 2));
        sw |= __shfl_xor_sync(0xffffffffu, sw, 4);
        sw |= __shfl_xor_sync(0xffffffffu, sw, 8);
        if (row >= p.rows || unit >= p.tiles) continue;
        if (col < p.nb * 32) *reinterpret_cast<uint32_t *>(q + (row * p.nb * 32 + col) / 2) = codes;
        if (lane16 == 0) *reinterpret_cast<uint32_t *>(s + mx_scale_at(row, unit * 4, p.tiles)) = sw;
    }
}

template <typename T, int kRows>
__global__ void __launch_bounds__(kThreads) k_dequantize_mxfp4(const uint8_t *__restrict__ q, const uint8_t *__restrict__ s,
                                                               T *__restrict__ y, Shape p) {
    const int lane16 = threadIdx.x & 15;
    const int u = (threadIdx.x >> 4) & ((1 << p.lux) - 1);
    const int ry = threadIdx.x >> (4 + p.lux);
    const int rows_blk = kThreads >> (4 + p.lux);
    const size_t unit = ((size_t)blockIdx.y << p.lux) + u;
    const size_t col = unit * 128 + lane16 * 8;
    const size_t row0 = (size_t)blockIdx.x * rows_blk * kRows + ry;
    pdl_wait();
    pdl_trigger();
    uint32_t codes[kRows], sb[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++) {
        const size_t row = row0 + (size_t)i * rows_blk;
        codes[i] = sb[i] = 0;
        if (row >= p.rows || col >= p.k) continue;
        codes[i] = __ldg(reinterpret_cast<const uint32_t *>(q + (row * p.nb * 32 + col) / 2));
        sb[i] = __ldg(s + mx_scale_at(row, col / 32, p.tiles));
    }
#pragma unroll
    for (int i = 0; i < kRows; i++) {
        const size_t row = row0 + (size_t)i * rows_blk;
        if (row >= p.rows || col >= p.k) continue;
        float v[8];
        mx_decode8(codes[i], v);
        const float X = mx_scale(sb[i]);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] *= X;
        T *dst = y + row * p.k + col;
        if (p.vec && col + 8 <= p.k) {
            Raw<T, 8> r;
            r.set(v);
            r.store(dst);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (col + j < p.k) dst[j] = from_f32<T>(v[j]);
        }
    }
}

// Row-major scales [rows][nb] -> tiles; the places of a tile past the last block
// get byte 0 (rows past the last are left as they are).  One thread per (row, tile).
__global__ void __launch_bounds__(kThreads) k_pack_scales(const uint8_t *__restrict__ in, uint8_t *__restrict__ s,
                                                          size_t rows, size_t nb, size_t tiles) {
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

constexpr int kRowsPer = 2;

// The grid of the streaming kernels: x over groups of rows, y over groups of units.
bool make_shape(size_t rows, size_t k, size_t pitch, bool vec, Shape *p, dim3 *grid) {
    p->rows = rows, p->k = k, p->pitch = pitch, p->vec = vec;
    p->nb = mx_blocks(k), p->tiles = mx_tiles(k);
    p->lux = 0;
    while (p->lux < 4 && ((size_t)1 << p->lux) < p->tiles) p->lux++;
    const size_t rows_blk = (size_t)(kThreads >> (4 + p->lux)) * kRowsPer;
    const size_t gx = (rows + rows_blk - 1) / rows_blk, gy = (p->tiles + ((size_t)1 << p->lux) - 1) >> p->lux;
    if (gx > 0x7fffffffu || gy > 65535u) return false;
    *grid = dim3((unsigned)gx, (unsigned)gy);
    return true;
}

template <typename T>
dw_status quantize(dw_backend *be, const void *x, size_t rows, size_t k, size_t pitch, uint8_t *q, uint8_t *s) {
    Shape p;
    dim3 grid;
    const bool vec = ((uintptr_t)x & 15) == 0 && pitch * sizeof(T) % 16 == 0;
    if (!make_shape(rows, k, pitch, vec, &p, &grid))
        return dw_fail(be, DW_ERR_UNSUPPORTED, "quantize_mxfp4: %zu x %zu is too large", rows, k);
    return launch_dependent(be, "quantize_mxfp4", k_quantize_mxfp4<T, kRowsPer>, grid, kThreads, 0, 0, (const T *)x, q, s, p);
}

template <typename T>
dw_status dequantize(dw_backend *be, const uint8_t *q, const uint8_t *s, size_t rows, size_t k, void *y) {
    Shape p;
    dim3 grid;
    const bool vec = ((uintptr_t)y & 15) == 0 && k * sizeof(T) % 16 == 0;
    if (!make_shape(rows, k, k, vec, &p, &grid))
        return dw_fail(be, DW_ERR_UNSUPPORTED, "dequantize_mxfp4: %zu x %zu is too large", rows, k);
    return launch_dependent(be, "dequantize_mxfp4", k_dequantize_mxfp4<T, kRowsPer>, grid, kThreads, 0, 0, q, s, (T *)y, p);
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
