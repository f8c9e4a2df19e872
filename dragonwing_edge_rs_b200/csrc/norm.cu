// norm.cu -- RMS and layer norms around a residual block, fused with the block's
// gate and residual scale and, where asked, with the MXFP4 quantisation of the
// result:
//   n   = post(x)                          x: the block's output
//   out = R(res + res_scale * gate * n)    R: rounding to res's type
//   y   = pre(out)                         the next block's input
// with rms(v) = v / sqrt(mean(v^2) + eps) * w + b and layer(v) the same on
// v - mean(v).  Without a residual y = pre(x).  All arithmetic is f32.
//
// Bandwidth-bound: x, res and gate are read once, out and y written once.  A row
// is held in registers between its reductions.

#include <algorithm>

#include "dw_device.cuh"
#include "dw_mxfp4.cuh"

namespace dw {
namespace {

constexpr int kMaxT = 512;  // threads of a row
constexpr int kMaxE = 32;   // elements of a thread

struct Params {
    const void *x, *gate, *res;
    const float *w0, *b0, *w1, *b1;
    void *out, *y;
    uint8_t *q, *s;
    size_t rows, c, x_pitch, res_pitch, y_pitch, gate_rows, nb, tiles;
    int pre, post, y_dtype;  // y_dtype: DW_F32..DW_BF16, -1: none, -2: MXFP4
    float eps, inv_c, res_scale;
    bool has_res;
};

// Sum over the threads of a row.  `slot` alternates over four buffers, so a
// buffer is written again only after three more barriers.
__device__ __forceinline__ float row_sum(float v, float (*red)[32], int &slot) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (blockDim.x == 32) return v;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) red[slot][warp] = v;
    __syncthreads();
    v = lane < warps ? red[slot][lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    slot = (slot + 1) & 3;
    return v;
}

template <int V>
__device__ __forceinline__ void load_f32(const float *p, float (&v)[V]) {
    Raw<float, V> r;
    r.load(p);
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = r.get(i);
}

// v[j][i] -> its norm, in place.  Elements past the row are 0 and stay out of the
// statistics (`live`: element group j lies in the row).
template <int V, int N>
__device__ __forceinline__ void normalise(float (&v)[N][V], const bool (&live)[N], int kind, const float *w, const float *b,
                                          const Params &p, float (*red)[32], int &slot) {
    const int T = blockDim.x, tid = threadIdx.x;
    if (kind == DW_NORM_LAYER) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int i = 0; i < V; i++) sum += v[j][i];
        const float mean = row_sum(sum, red, slot) * p.inv_c;
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int i = 0; i < V; i++) v[j][i] = live[j] ? v[j][i] - mean : 0.0f;
    }
    float sq = 0.0f;
#pragma unroll
    for (int j = 0; j < N; j++)
#pragma unroll
        for (int i = 0; i < V; i++) sq = fmaf(v[j][i], v[j][i], sq);
    const float rstd = __frsqrt_rn(fmaf(row_sum(sq, red, slot), p.inv_c, p.eps));
#pragma unroll
    for (int j = 0; j < N; j++) {
        if (!live[j]) continue;
        const size_t at = ((size_t)j * T + tid) * V;
        float wv[V], bv[V];
        if (w) load_f32<V>(w + at, wv);
        if (b) load_f32<V>(b + at, bv);
#pragma unroll
        for (int i = 0; i < V; i++) {
            v[j][i] *= rstd;
            if (w) v[j][i] *= wv[i];
            if (b) v[j][i] += bv[i];
        }
    }
}

// One group of V values as MXFP4: 32 / V neighbouring threads hold a block.
template <int V>
__device__ __forceinline__ void put_mxfp4(const float (&v)[V], size_t at, size_t row, const Params &p) {
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < V; i++) amax = max(amax, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
    for (int o = 1; o < 32 / V; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const uint32_t sb = mx_scale_byte(amax);
    const float inv = mx_inv_scale(sb);
    const size_t block = at / 32;
    uint8_t *dst = p.q + (row * p.nb * 32 + at) / 2;
    if constexpr (V == 8) {
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = v[i] * inv;
        if (block < p.nb) *reinterpret_cast<uint32_t *>(dst) = sb == 0xFFu ? 0u : mx_codes8(t);
    } else if constexpr (V == 2) {
        if (block < p.nb) *dst = sb == 0xFFu ? (uint8_t)0 : (uint8_t)mx_codes2(v[0] * inv, v[1] * inv);
    } else {
        const float next = __shfl_down_sync(0xffffffffu, v[0], 1);
        if ((threadIdx.x & 1) == 0 && block < p.nb) *dst = sb == 0xFFu ? (uint8_t)0 : (uint8_t)mx_codes2(v[0] * inv, next * inv);
    }
    if ((at & 31) == 0 && block < p.tiles * 4) p.s[mx_scale_at(row, block, p.tiles)] = (uint8_t)sb;
}

template <typename T, int V>
__device__ __forceinline__ void put(void *y, size_t at, const float (&v)[V]) {
    Raw<T, V> r;
    r.set(v);
    r.store((T *)y + at);
}

// blockDim = (threads of a row, rows); element group j of thread t starts at
// column (j * threads + t) * V.
template <typename X, typename R, int V, int N>
__global__ void __launch_bounds__(kMaxT) k_norm(const __grid_constant__ Params p) {
    __shared__ float red[4][32];
    int slot = 0;
    const int T = blockDim.x, tid = threadIdx.x;
    for (size_t row = (size_t)blockIdx.x * blockDim.y + threadIdx.y; row < p.rows; row += (size_t)gridDim.x * blockDim.y) {
        Raw<X, V> xr[N], gr[N];
        Raw<R, V> rr[N];
        bool live[N];
        const X *x = (const X *)p.x + row * p.x_pitch;
        const R *res = (const R *)p.res + row * p.res_pitch;
        const X *gate = (const X *)p.gate + (p.gate_rows ? row / p.gate_rows : 0) * p.c;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const size_t at = ((size_t)j * T + tid) * V;
            live[j] = at < p.c;
            xr[j].zero(), rr[j].zero(), gr[j].zero();
            if (live[j]) {
                xr[j].load(x + at);
                if (p.has_res) rr[j].load(res + at);
                if (p.gate) gr[j].load(gate + at);
            }
        }
        float v[N][V];
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int i = 0; i < V; i++) v[j][i] = xr[j].get(i);
        if (p.has_res) {
            if (p.post != DW_NORM_NONE) normalise<V, N>(v, live, p.post, p.w0, p.b0, p, red, slot);
#pragma unroll
            for (int j = 0; j < N; j++) {
                if (!live[j]) continue;
                float o[V];
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float n = p.gate ? v[j][i] * gr[j].get(i) : v[j][i];
                    o[i] = fmaf(p.res_scale, n, rr[j].get(i));
                }
                Raw<R, V> r;
                r.set(o);
                r.store((R *)p.out + row * p.res_pitch + ((size_t)j * T + tid) * V);
#pragma unroll
                for (int i = 0; i < V; i++) v[j][i] = r.get(i);
            }
        }
        if (p.y_dtype == -1) continue;
        if (p.pre != DW_NORM_NONE) normalise<V, N>(v, live, p.pre, p.w1, p.b1, p, red, slot);
#pragma unroll
        for (int j = 0; j < N; j++) {
            const size_t at = ((size_t)j * T + tid) * V;
            if (p.y_dtype == -2) {
                put_mxfp4<V>(v[j], at, row, p);
                continue;
            }
            if (!live[j]) continue;
            const size_t to = row * p.y_pitch + at;
            if (p.y_dtype == DW_F32)
                put<float, V>(p.y, to, v[j]);
            else if (p.y_dtype == DW_F16)
                put<__half, V>(p.y, to, v[j]);
            else
                put<__nv_bfloat16, V>(p.y, to, v[j]);
        }
    }
}

// Rows too long for registers: one thread block a row, elements read again for
// each reduction (from L2) and `out` read back by the thread that wrote it.
template <typename X, typename R>
__global__ void __launch_bounds__(kMaxT) k_norm_long(const __grid_constant__ Params p) {
    __shared__ float red[4][32];
    int slot = 0;
    const size_t row = blockIdx.x;
    const size_t T = blockDim.x, end = p.tiles * 128;
    const X *x = (const X *)p.x + row * p.x_pitch;
    const R *res = (const R *)p.res + row * p.res_pitch;
    const X *gate = (const X *)p.gate + (p.gate_rows ? row / p.gate_rows : 0) * p.c;
    R *out = (R *)p.out + row * p.res_pitch;
    auto stats = [&](auto at, int kind, float &mean, float &rstd) {
        mean = 0.0f, rstd = 1.0f;
        if (kind == DW_NORM_NONE) return;
        if (kind == DW_NORM_LAYER) {
            float sum = 0.0f;
            for (size_t i = threadIdx.x; i < p.c; i += T) sum += at(i);
            mean = row_sum(sum, red, slot) * p.inv_c;
        }
        float sq = 0.0f;
        for (size_t i = threadIdx.x; i < p.c; i += T) {
            const float d = at(i) - mean;
            sq = fmaf(d, d, sq);
        }
        rstd = __frsqrt_rn(fmaf(row_sum(sq, red, slot), p.inv_c, p.eps));
    };
    auto scaled = [&](float v, size_t i, float mean, float rstd, const float *w, const float *b) {
        v = (v - mean) * rstd;
        if (w) v *= w[i];
        if (b) v += b[i];
        return v;
    };
    auto from_x = [&](size_t i) { return to_f32(x[i]); };
    auto from_out = [&](size_t i) { return to_f32(out[i]); };
    float mean, rstd;
    if (p.has_res) {
        stats(from_x, p.post, mean, rstd);
        for (size_t i = threadIdx.x; i < p.c; i += T) {
            float n = from_x(i);
            if (p.post != DW_NORM_NONE) n = scaled(n, i, mean, rstd, p.w0, p.b0);
            if (p.gate) n *= to_f32(gate[i]);
            out[i] = from_f32<R>(fmaf(p.res_scale, n, to_f32(res[i])));
        }
        if (p.y_dtype == -1) return;
        stats(from_out, p.pre, mean, rstd);
    } else {
        stats(from_x, p.pre, mean, rstd);
    }
    for (size_t i = threadIdx.x; i < end; i += T) {  // whole warps: MXFP4 blocks are a warp's 32 elements
        float v[1] = {0.0f};
        if (i < p.c) {
            v[0] = p.has_res ? from_out(i) : from_x(i);
            if (p.pre != DW_NORM_NONE) v[0] = scaled(v[0], i, mean, rstd, p.w1, p.b1);
        }
        if (p.y_dtype == -2) {
            put_mxfp4<1>(v, i, row, p);
        } else if (i < p.c) {
            const size_t to = row * p.y_pitch + i;
            if (p.y_dtype == DW_F32)
                put<float, 1>(p.y, to, v);
            else if (p.y_dtype == DW_F16)
                put<__half, 1>(p.y, to, v);
            else
                put<__nv_bfloat16, 1>(p.y, to, v);
        }
    }
}

template <typename X, typename R>
dw_status run(dw_backend *be, const Params &p) {
    // V: the most elements (8, 2, 1) that every row of every operand has aligned
    auto fits = [&](int V) {
        if (p.c % V) return false;
        auto ok = [&](const void *ptr, size_t es, size_t pitch) {
            const size_t a = std::min<size_t>(16, es * V);
            return !ptr || ((uintptr_t)ptr % a == 0 && pitch * es % a == 0);
        };
        const size_t ys = p.y_dtype == DW_F32 ? 4 : 2;
        return ok(p.x, sizeof(X), p.x_pitch) && ok(p.gate, sizeof(X), p.c) && ok(p.res, sizeof(R), p.res_pitch) &&
               ok(p.out, sizeof(R), p.res_pitch) && ok(p.y, ys, p.y_pitch) && ok(p.w0, 4, 0) && ok(p.b0, 4, 0) &&
               ok(p.w1, 4, 0) && ok(p.b1, 4, 0);
    };
    if (p.rows > 0x7fffffffu) return dw_fail(be, DW_ERR_UNSUPPORTED, "norm: more than 2^31 - 1 rows");
    if (p.c > (size_t)kMaxT * kMaxE) {
        k_norm_long<X, R><<<(unsigned)p.rows, kMaxT, 0, be->stream>>>(p);
        return dw_after_launch(be, "norm (long rows)");
    }
    // E: elements of a thread; T: threads of a row (a power of two from 32 to 512)
    int E = 8, T = 32;
    while ((size_t)T * E < p.c && T < kMaxT) T *= 2;
    while ((size_t)T * E < p.c) E *= 2;
    const int rows_blk = T == 32 ? 8 : 1;
    const size_t blocks = (p.rows + rows_blk - 1) / rows_blk;
    const dim3 block(T, rows_blk);
    auto go = [&](auto kernel) {
        kernel<<<(unsigned)blocks, block, 0, be->stream>>>(p);
        return dw_after_launch(be, "norm");
    };
    if (fits(8)) {
        if (E == 8) return go(k_norm<X, R, 8, 1>);
        if (E == 16) return go(k_norm<X, R, 8, 2>);
        return go(k_norm<X, R, 8, 4>);
    }
    if (fits(2)) {
        if (E == 8) return go(k_norm<X, R, 2, 4>);
        if (E == 16) return go(k_norm<X, R, 2, 8>);
        return go(k_norm<X, R, 2, 16>);
    }
    if (E == 8) return go(k_norm<X, R, 1, 8>);
    if (E == 16) return go(k_norm<X, R, 1, 16>);
    return go(k_norm<X, R, 1, 32>);
}

}  // namespace

dw_status launch_norm(dw_backend *be, const dw_norm_desc &d, const NormArgs &a) {
    Params p{};
    p.x = a.x, p.gate = a.gate, p.res = a.res, p.out = a.out, p.y = a.y, p.q = a.q, p.s = a.s;
    p.w0 = a.w_post, p.b0 = a.b_post, p.w1 = a.w_pre, p.b1 = a.b_pre;
    p.rows = d.rows, p.c = d.c, p.gate_rows = d.gate_rows;
    p.x_pitch = d.x_pitch ? d.x_pitch : d.c, p.res_pitch = d.res_pitch ? d.res_pitch : d.c;
    p.y_pitch = d.y_pitch ? d.y_pitch : d.c;
    p.nb = mx_blocks(d.c), p.tiles = mx_tiles(d.c);
    p.pre = d.pre, p.post = d.post;
    p.y_dtype = a.q ? -2 : a.y ? d.y_dtype : -1;
    p.eps = d.eps, p.inv_c = 1.0f / (float)d.c, p.res_scale = d.res_scale;
    p.has_res = a.res != nullptr;
    if (d.x_dtype == DW_F32) return run<float, float>(be, p);
    if (d.x_dtype == DW_F16)
        return p.has_res && d.res_dtype == DW_F32 ? run<__half, float>(be, p) : run<__half, __half>(be, p);
    return p.has_res && d.res_dtype == DW_F32 ? run<__nv_bfloat16, float>(be, p) : run<__nv_bfloat16, __nv_bfloat16>(be, p);
}

}  // namespace dw
