// heads.cu -- the heads of a projection's rows on their way to attention: norms of query and
// key heads with the position rotation, keys and values appended to the paged 8-bit cache, and
// cached values read back.
//   norm     rms(x) = x / sqrt(mean(x^2) + eps) * w over a head, layer(x) the same on x - mean(x)
//   rotate   (a, b) -> (a cos t - b sin t, a sin t + b cos t), t = position * freq, in pairs
//   append   X = 2^e, e the smallest with max|v| <= 448 X over the block; code = e4m3(v / X)
// Angles: a frequency is a 64-bit fraction of a turn, so position * frequency modulo a turn is
// one integer product, exact however far the position.
//
// All are bound by the bytes of the rows, in short calls by latency.

#include <algorithm>

#include "dw_kv.cuh"
#include "dw_launch.h"
#include "dw_mxfp4.cuh"

namespace dw {
namespace {

constexpr int kThreads = 256;

struct HeadParams {
    const void *q, *k, *v;
    void *q_out, *k_out;
    size_t q_pitch, k_pitch, v_pitch, qo_pitch, ko_pitch;
    const float *w_q, *w_k;
    const uint64_t *rope;
    const int32_t *positions;
    uint32_t tokens;
    int hq, hk, d, rot, norm;
    float eps, inv_d;
    int group, chunk, chunks;  // lanes of a head, head groups of a warp, warps of a row
    bool neighbours, vec;
};

__device__ __forceinline__ void turn_f32(uint64_t freq, int64_t position, float &c, float &s) {
    const int64_t t = (int64_t)(freq * (uint64_t)position);  // half turns * 2^63
    sincospif((float)(int32_t)(t >> 32) * 0x1p-31f, &s, &c);
}
__device__ __forceinline__ void turn_f64(uint64_t freq, int64_t position, double &c, double &s) {
    const int64_t t = (int64_t)(freq * (uint64_t)position);
    sincospi((double)t * 0x1p-63, &s, &c);
}

// Where slot `c` of a head has its 2 E values: E from `a` on and E from `b` on; whether they
// turn, then by the pairs c * E + i.  Halves: pair i is (a + i, b + i); neighbours: the 2 E
// values lie together and pair i is values 2 i and 2 i + 1 of them.
template <int E>
struct Slot {
    int a, b;
    bool turns;
    __device__ __forceinline__ Slot(int c, int rot, bool neighbours) {
        const int n = rot / (2 * E);
        turns = c < n;
        if (turns && !neighbours)
            a = c * E, b = rot / 2 + c * E;
        else
            a = 2 * c * E, b = a + E;
    }
};
template <int E, typename F>
__device__ __forceinline__ void rotate(F (&v)[2 * E], const F (&c)[E], const F (&s)[E], bool neighbours) {
    auto turn = [](F &a, F &b, F cos, F sin) {
        const F x = a, y = b;
        a = x * cos - y * sin;
        b = x * sin + y * cos;
    };
    if (neighbours) {
#pragma unroll
        for (int i = 0; i < E; i++) turn(v[2 * i], v[2 * i + 1], c[i], s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < E; i++) turn(v[i], v[E + i], c[i], s[i]);
    }
}

// Head groups [first, first + chunk) of one row by one warp: a group is 32 / `group` heads, a
// lane has J slots of a head.
template <typename T, int E, int J>
__device__ __forceinline__ void norm_rope_row(const HeadParams &p, size_t row, int64_t position, int first) {
    const int lane = threadIdx.x & 31, sub = lane & (p.group - 1), per = 32 / p.group;
    const int heads = p.hq + p.hk;
    float cs[J][E], sn[J][E], w[J][2 * E];
    int a[J], b[J];
    bool live[J], turns[J];
#pragma unroll
    for (int j = 0; j < J; j++) {
        const int c = sub + j * p.group;
        const Slot<E> slot(c, p.rot, p.neighbours);
        live[j] = 2 * E * c < p.d;
        a[j] = slot.a, b[j] = slot.b, turns[j] = slot.turns && live[j];
#pragma unroll
        for (int i = 0; i < E; i++)
            if (turns[j]) turn_f32(p.rope[c * E + i], position, cs[j][i], sn[j][i]);
    }
    auto source = [&](int h) {
        return h < p.hq ? (const T *)p.q + row * p.q_pitch + (size_t)h * p.d : (const T *)p.k + row * p.k_pitch + (size_t)(h - p.hq) * p.d;
    };
    Raw<T, E> ra[J], rb[J];
    auto load = [&](int h) {
        if (h >= heads) return;
        const T *x = source(h);
#pragma unroll
        for (int j = 0; j < J; j++)
            if (live[j]) ra[j].load(x + a[j]), rb[j].load(x + b[j]);
    };
    int h = first * per + lane / p.group, weights = -1;
    const int end = min((first + p.chunk) * per, (heads + per - 1) / per * per);
    load(h);
    for (; h < end; h += per) {
        float v[J][2 * E];
        const bool there = h < heads;
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int i = 0; i < E; i++) {
                v[j][i] = there && live[j] ? ra[j].get(i) : 0.0f;
                v[j][E + i] = there && live[j] ? rb[j].get(i) : 0.0f;
            }
        if (h + per < end) load(h + per);
        if (p.norm != DW_NORM_NONE) {
            const int kind = h < p.hq ? 0 : 1;
            if (kind != weights) {
                const float *from = kind ? p.w_k : p.w_q;
                weights = kind;
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int i = 0; i < E; i++) {
                        w[j][i] = from && live[j] ? from[a[j] + i] : 1.0f;
                        w[j][E + i] = from && live[j] ? from[b[j] + i] : 1.0f;
                    }
            }
            auto sum = [&](float x) {
#pragma unroll
                for (int o = 16; o; o >>= 1)
                    if (o < p.group) x += __shfl_xor_sync(0xffffffffu, x, o);
                return x;
            };
            if (p.norm == DW_NORM_LAYER) {
                float m = 0.0f;
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int i = 0; i < 2 * E; i++) m += v[j][i];
                m = sum(m) * p.inv_d;
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int i = 0; i < 2 * E; i++) v[j][i] = live[j] ? v[j][i] - m : 0.0f;
            }
            float sq = 0.0f;
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < 2 * E; i++) sq = fmaf(v[j][i], v[j][i], sq);
            const float rstd = __frsqrt_rn(fmaf(sum(sq), p.inv_d, p.eps));
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < 2 * E; i++) v[j][i] *= rstd * w[j][i];
        }
        if (!there) continue;
        T *out = h < p.hq ? (T *)p.q_out + row * p.qo_pitch + (size_t)h * p.d : (T *)p.k_out + row * p.ko_pitch + (size_t)(h - p.hq) * p.d;
#pragma unroll
        for (int j = 0; j < J; j++) {
            if (!live[j]) continue;
            if (turns[j]) rotate<E, float>(v[j], cs[j], sn[j], p.neighbours);
            float lo[E], hi[E];
#pragma unroll
            for (int i = 0; i < E; i++) lo[i] = v[j][i], hi[i] = v[j][E + i];
            Raw<T, E> r;
            r.set(lo);
            r.store(out + a[j]);
            r.set(hi);
            r.store(out + b[j]);
        }
    }
}

template <typename T, int E, int J>
__global__ void __launch_bounds__(kThreads) k_norm_rope(const __grid_constant__ HeadParams p) {
    pdl_wait();
    pdl_trigger();
    const size_t unit = (size_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32, row = unit / p.chunks;
    if (row >= p.tokens) return;
    norm_rope_row<T, E, J>(p, row, p.positions ? p.positions[row] : 0, (int)(unit % p.chunks) * p.chunk);
}

// ---- append ------------------------------------------------------------------------
// A block of threads has one head of one page that rows are written to, a warp eight of its
// tokens, a lane 2 E = d / 32 values of each.  Keys are computed in f64 and kept as f32 rounded
// to odd (a last bit of 1 where anything was cut off), which rounds to e4m3 as the f64 would:
// the cached codes are the definition's own, whatever hardware or order computed them.  A
// warp's tokens follow each other, so the angles after the first come by one complex product
// each.  The blocks behind those of the pages norm and turn query rows.
constexpr int kWarpTokens = 8;

__device__ __forceinline__ float round_to_odd(double v) {
    const float f = __double2float_rz(v);
    return __uint_as_float(__float_as_uint(f) | (uint32_t)((__double2loint(v) & 0x1FFFFFFF) != 0));
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T, int E>
__device__ __forceinline__ void load_values(const T *p, bool vec, float (&v)[E]) {
    if (vec) {
        Raw<T, E> r;
        r.load(p);
#pragma unroll
        for (int i = 0; i < E; i++) v[i] = r.get(i);
    } else {
#pragma unroll
        for (int i = 0; i < E; i++) v[i] = to_f32(p[i]);
    }
}

// E codes (1, 2 or 4) to aligned places.
template <int E>
__device__ __forceinline__ void store_codes(uint8_t *p, const float (&v)[E]) {
    if constexpr (E == 1)
        *p = (uint8_t)e4m3_codes2(v[0], 0.0f);
    else if constexpr (E == 2)
        *reinterpret_cast<uint16_t *>(p) = (uint16_t)e4m3_codes2(v[0], v[1]);
    else
        *reinterpret_cast<uint32_t *>(p) = e4m3_codes2(v[0], v[1]) | e4m3_codes2(v[2], v[3]) << 16;
}

// The 2 E codes of a lane, times f, rounded again.
template <int E>
__device__ __forceinline__ void rescale_codes(uint8_t *p, float f) {
    if constexpr (E == 1) {
        const uint16_t c = *reinterpret_cast<const uint16_t *>(p);
        const float2 v = e4m3_to_f32x2(c);
        *reinterpret_cast<uint16_t *>(p) = (uint16_t)e4m3_codes2(v.x * f, v.y * f);
    } else {
        const uint32_t c = *reinterpret_cast<const uint32_t *>(p);
        const float2 v = e4m3_to_f32x2((uint16_t)c), u = e4m3_to_f32x2((uint16_t)(c >> 16));
        *reinterpret_cast<uint32_t *>(p) = e4m3_codes2(v.x * f, v.y * f) | e4m3_codes2(u.x * f, u.y * f) << 16;
    }
}

template <typename T, int E, int QE, int QJ>
__global__ void __launch_bounds__(512)
    k_append(const __grid_constant__ HeadParams p, const __grid_constant__ KvCache c, const __grid_constant__ Seqs q,
             const uint32_t page_blocks, int32_t *err) {
    __shared__ uint32_t top[2][16];
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, warps = blockDim.x / 32;
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x >= page_blocks) {
        const size_t unit = (size_t)(blockIdx.x - page_blocks) * warps + warp;
        const int64_t row = (int64_t)(unit / p.chunks);
        if (row >= p.tokens) return;
        int64_t place;
        const uint32_t s = seq_of_item(q, row, 1, 1, 0, place);
        const SeqRange r = seq_range(q, s, c.page, err);
        if (place < 0 || place >= r.n) return;
        HeadParams pq = p;
        pq.hk = 0;
        norm_rope_row<T, QE, QJ>(pq, (size_t)row, r.position((int)row), (int)(unit % p.chunks) * p.chunk);
        return;
    }
    const int head = (int)(blockIdx.x % p.hk);
    int64_t place;
    const uint32_t s = seq_of_item(q, blockIdx.x / p.hk, 1, c.page, 2, place);
    const SeqRange r = seq_range(q, s, c.page, err);
    const int first = max(r.len - r.n, 0);  // the sequence's first new token
    const int64_t begin = (first / c.page + place) * c.page;
    if (place < 0 || first >= r.len || begin >= r.len) return;
    const int t0 = max(first, (int)begin), t1 = (int)min((int64_t)r.len, begin + c.page);
    const uint32_t page = seq_page(q, c, s, (uint32_t)(begin / c.page), err);
    uint8_t *const scale = c.s + kv_block(c, page, head) * 2;
    const bool has_old = t0 > begin;
    const int k_old = has_old ? kv_exponent(scale[0]) : kKvMinExp, v_old = has_old ? kv_exponent(scale[1]) : kKvMinExp;
    uint8_t *const kc = kv_codes(c.k, c, page, head), *const vc = kv_codes(c.v, c, page, head);

    const int w0 = (int)begin + warp * kWarpTokens;  // the warp's first token
    const Slot<E> slot(lane, p.rot, p.neighbours);
    const T *const kp = (const T *)p.k + (size_t)head * p.d, *const vp = (const T *)p.v + (size_t)head * p.d;
    float kv[kWarpTokens][2 * E], vv[kWarpTokens][2 * E];
#pragma unroll
    for (int i = 0; i < kWarpTokens; i++) {
        const int t = w0 + i;
        if (t < t0 || t >= t1) continue;
        const size_t row = (size_t)r.row0 + (t - (r.len - r.n));
        float lo[E], hi[E];
        load_values<T, E>(kp + row * p.k_pitch + slot.a, p.vec, lo);
        load_values<T, E>(kp + row * p.k_pitch + slot.b, p.vec, hi);
#pragma unroll
        for (int j = 0; j < E; j++) kv[i][j] = lo[j], kv[i][E + j] = hi[j];
        load_values<T, E>(vp + row * p.v_pitch + 2 * E * lane, p.vec, lo);
        load_values<T, E>(vp + row * p.v_pitch + 2 * E * lane + E, p.vec, hi);
#pragma unroll
        for (int j = 0; j < E; j++) vv[i][j] = lo[j], vv[i][E + j] = hi[j];
    }
    double cs[E], sn[E], cs1[E], sn1[E], w[2 * E];
#pragma unroll
    for (int j = 0; j < E; j++) {
        const bool weighs = p.norm != DW_NORM_NONE && p.w_k;
        w[j] = weighs ? (double)p.w_k[slot.a + j] : 1.0, w[E + j] = weighs ? (double)p.w_k[slot.b + j] : 1.0;
        cs[j] = cs1[j] = 1.0, sn[j] = sn1[j] = 0.0;
        if (slot.turns && w0 < t1 && w0 + kWarpTokens > t0) {
            const uint64_t f = p.rope[lane * E + j];
            turn_f64(f, max(w0, t0), cs[j], sn[j]);
            if (min(w0 + kWarpTokens, t1) - max(w0, t0) > 1) turn_f64(f, 1, cs1[j], sn1[j]);
        }
    }
    float kmax = 0.0f, vmax = 0.0f;
    uint32_t poison = 0;
#pragma unroll
    for (int i = 0; i < kWarpTokens; i++) {
        const int t = w0 + i;
        if (t < t0 || t >= t1) continue;
        double x[2 * E];
#pragma unroll
        for (int j = 0; j < 2 * E; j++) x[j] = kv[i][j];
        if (p.norm != DW_NORM_NONE) {
            if (p.norm == DW_NORM_LAYER) {
                double m = 0.0;
#pragma unroll
                for (int j = 0; j < 2 * E; j++) m += x[j];
                m = warp_sum(m) / p.d;
#pragma unroll
                for (int j = 0; j < 2 * E; j++) x[j] -= m;
            }
            double sq = 0.0;
#pragma unroll
            for (int j = 0; j < 2 * E; j++) sq = fma(x[j], x[j], sq);
            const double rstd = 1.0 / sqrt(warp_sum(sq) / p.d + (double)p.eps);
#pragma unroll
            for (int j = 0; j < 2 * E; j++) x[j] *= rstd * w[j];
        }
        if (slot.turns) rotate<E, double>(x, cs, sn, p.neighbours);
        bool ok = true;
        float km = 0.0f, vm = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * E; j++) {
            ok = ok && isfinite(x[j]) && isfinite(vv[i][j]);
            kv[i][j] = round_to_odd(x[j]);
            km = fmaxf(km, fabsf(kv[i][j])), vm = fmaxf(vm, fabsf(vv[i][j]));
        }
        if (__all_sync(0xffffffffu, ok))
            kmax = fmaxf(kmax, km), vmax = fmaxf(vmax, vm);
        else
            poison |= 1u << i;
#pragma unroll
        for (int j = 0; j < E; j++) {  // the next token's angle
            const double cn = cs[j] * cs1[j] - sn[j] * sn1[j];
            sn[j] = sn[j] * cs1[j] + cs[j] * sn1[j];
            cs[j] = cn;
        }
    }
    kmax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(kmax)));
    vmax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(vmax)));
    if (lane == 0) top[0][warp] = __float_as_uint(kmax), top[1][warp] = __float_as_uint(vmax);
    __syncthreads();
    uint32_t km = 0, vm = 0;
    for (int i = 0; i < warps; i++) km = max(km, top[0][i]), vm = max(vm, top[1][i]);
    const int ke = max(kv_scale_exponent(__uint_as_float(km)), k_old), ve = max(kv_scale_exponent(__uint_as_float(vm)), v_old);
    const float k_inv = kv_pow2(-ke), v_inv = kv_pow2(-ve);
    if (threadIdx.x == 0) scale[0] = (uint8_t)(ke + 127), scale[1] = (uint8_t)(ve + 127);
#pragma unroll
    for (int i = 0; i < kWarpTokens; i++) {
        const int t = w0 + i;
        uint8_t *const kr = kc + (t - (int)begin) * p.d, *const vr = vc + (t - (int)begin) * p.d;
        if (t < t0) {
            if (ke != k_old) rescale_codes<E>(kr + 2 * E * lane, kv_pow2(k_old - ke));
            if (ve != v_old) rescale_codes<E>(vr + 2 * E * lane, kv_pow2(v_old - ve));
        } else if (t < t1) {
            const bool bad = poison >> i & 1;
            float lo[E], hi[E], all[2 * E];
#pragma unroll
            for (int j = 0; j < E; j++) {
                lo[j] = bad ? __uint_as_float(0x7FC00000u) : kv[i][j] * k_inv;
                hi[j] = bad ? __uint_as_float(0x7FC00000u) : kv[i][E + j] * k_inv;
            }
#pragma unroll
            for (int j = 0; j < 2 * E; j++) all[j] = bad ? 0.0f : vv[i][j] * v_inv;
            store_codes<E>(kr + slot.a, lo);
            store_codes<E>(kr + slot.b, hi);
            store_codes<2 * E>(vr + 2 * E * lane, all);
        }
    }
}

// ---- read --------------------------------------------------------------------------
// A warp has a row's keys or values, a lane 8 values at a time.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_read(const __grid_constant__ KvCache c, const __grid_constant__ Seqs q, T *k_out, T *v_out, size_t k_pitch, size_t v_pitch,
           const bool vec, int32_t *err) {
    const int lane = threadIdx.x & 31;
    const size_t unit = (size_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
    pdl_wait();
    pdl_trigger();
    const int64_t row = (int64_t)(unit / 2);
    const bool values = unit & 1;
    T *out = values ? v_out : k_out;
    if (row >= q.tokens || !out) return;
    int64_t place;
    const uint32_t s = seq_of_item(q, row, 1, 1, 0, place);
    const SeqRange r = seq_range(q, s, c.page, err);
    if (place < 0 || place >= r.n) return;
    out += (size_t)row * (values ? v_pitch : k_pitch);
    const int t = r.position((int)row);
    const uint32_t page = t < 0 ? 0 : seq_page(q, c, s, (uint32_t)t / (uint32_t)c.page, err);
    for (int i = lane * 8; i < c.heads * c.d; i += 256) {
        const int head = i / c.d;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 0.0f;
        if (t >= 0) {
            const uint8_t *codes = kv_codes(values ? c.v : c.k, c, page, head) + (t % c.page) * c.d + i % c.d;
            const float x = kv_pow2(kv_exponent(c.s[kv_block(c, page, head) * 2 + values]));
            const uint2 w = *reinterpret_cast<const uint2 *>(codes);
            const uint32_t ws[2] = {w.x, w.y};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = e4m3_to_f32x2((uint16_t)(ws[j / 2] >> (16 * (j % 2))));
                v[2 * j] = f.x * x, v[2 * j + 1] = f.y * x;
            }
        }
        if (vec) {
            Raw<T, 8> o;
            o.set(v);
            o.store(out + i);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) out[i + j] = from_f32<T>(v[j]);
        }
    }
}

bool aligned(const HeadRows &h, size_t es, size_t a) { return !h.ptr || ((uintptr_t)h.ptr % a == 0 && h.pitch * es % a == 0); }

HeadParams params(const dw_head_desc &d, size_t tokens, const HeadArgs &a) {
    HeadParams p{};
    p.q = a.q.ptr, p.k = a.k.ptr, p.v = a.v.ptr, p.q_out = a.q_out.ptr, p.k_out = a.k_out.ptr;
    p.q_pitch = a.q.pitch, p.k_pitch = a.k.pitch, p.v_pitch = a.v.pitch, p.qo_pitch = a.q_out.pitch, p.ko_pitch = a.k_out.pitch;
    p.w_q = a.w_q, p.w_k = a.w_k, p.rope = a.rope, p.positions = a.positions;
    p.tokens = (uint32_t)tokens;
    p.hq = a.q.ptr ? d.q_heads : 0, p.hk = a.k.ptr ? d.kv_heads : 0;
    p.d = d.head_dim, p.rot = d.rot_dim, p.norm = d.norm;
    p.eps = d.eps, p.inv_d = 1.0f / (float)d.head_dim, p.neighbours = d.neighbours != 0;
    return p;
}

// The lanes of a head with E values in a piece and J slots a lane, and how the heads of a row
// are shared out: few rows give each warp one group of heads, many rows all of a row's, so that
// its angles are computed once.
void split(const dw_backend *be, HeadParams &p, int heads, int E, int J) {
    p.group = 1;
    while (p.group * 2 * E * J < p.d) p.group *= 2;
    const int per = 32 / p.group, groups = (heads + per - 1) / per;
    const size_t warps = (size_t)be->sm_count * 32;  // that the GPU holds at about this many registers
    p.chunk = (int)std::max<size_t>(1, std::min<size_t>(groups, (size_t)p.tokens * groups / warps));
    p.chunks = (groups + p.chunk - 1) / p.chunk;
}

template <typename T>
constexpr int kWide = 16 / (int)sizeof(T);  // values of a 16-byte access

// Whether 16-byte accesses hold whole slots.
template <typename T>
bool wide(const HeadParams &p, std::initializer_list<HeadRows> rows) {
    constexpr int E = kWide<T>;
    bool ok = p.d % (2 * E) == 0 && p.rot % (2 * E) == 0 && p.d / (2 * E) <= 32;
    for (const HeadRows &r : rows) ok = ok && aligned(r, sizeof(T), 16);
    return ok;
}

template <typename T>
dw_status norm_rope(dw_backend *be, HeadParams p, const HeadArgs &a) {
    const int heads = p.hq + p.hk;
    auto go = [&](auto kernel, int E, int J) {
        split(be, p, heads, E, J);
        const size_t blocks = ((size_t)p.tokens * p.chunks + kThreads / 32 - 1) / (kThreads / 32);
        if (blocks > 0x7fffffffu) return dw_fail(be, DW_ERR_UNSUPPORTED, "norm_rope: too many rows");
        return launch_dependent(be, "norm_rope", kernel, (unsigned)blocks, kThreads, 0, 0, p);
    };
    if (wide<T>(p, {a.q, a.k, a.q_out, a.k_out})) return go(k_norm_rope<T, kWide<T>, 1>, kWide<T>, 1);
    if (p.d <= 128) return go(k_norm_rope<T, 1, 2>, 1, 2);
    return go(k_norm_rope<T, 1, 8>, 1, 8);
}

template <typename T, int E>
dw_status append(dw_backend *be, HeadParams p, const KvCache &c, const Seqs &s, const HeadArgs &a) {
    p.vec = aligned(a.k, sizeof(T), E * sizeof(T)) && aligned(a.v, sizeof(T), E * sizeof(T));
    const unsigned threads = (unsigned)(c.page / kWarpTokens * 32);
    const size_t pages = seq_items(s.tokens, s.seqs, 1, c.page, 2) * p.hk;
    auto go = [&](auto kernel, int QE, int QJ) {
        size_t blocks = pages;
        p.chunks = 1;
        if (p.hq) {
            split(be, p, p.hq, QE, QJ);
            blocks += ((size_t)p.tokens * p.chunks + threads / 32 - 1) / (threads / 32);
        }
        if (blocks > 0x7fffffffu) return dw_fail(be, DW_ERR_UNSUPPORTED, "append_kv: too many rows");
        return launch_dependent(be, "append_kv", kernel, (unsigned)blocks, threads, 0, 0, p, c, s, (uint32_t)pages, be->dev_err);
    };
    if (wide<T>(p, {a.q, a.q_out})) return go(k_append<T, E, kWide<T>, 1>, kWide<T>, 1);
    return go(k_append<T, E, 1, E>, 1, E);
}

}  // namespace

dw_status launch_norm_rope(dw_backend *be, const dw_head_desc &d, size_t tokens, const HeadArgs &a) {
    const HeadParams p = params(d, tokens, a);
    if (d.dtype == DW_F32) return norm_rope<float>(be, p, a);
    if (d.dtype == DW_F16) return norm_rope<__half>(be, p, a);
    return norm_rope<__nv_bfloat16>(be, p, a);
}

dw_status launch_append_kv(dw_backend *be, const dw_head_desc &d, const KvCache &c, const Seqs &s, const HeadArgs &a) {
    const HeadParams p = params(d, s.tokens, a);
    auto with = [&](auto t) {
        using T = decltype(t);
        return c.d == 64 ? append<T, 1>(be, p, c, s, a) : append<T, 2>(be, p, c, s, a);
    };
    if (d.dtype == DW_F32) return with(float{});
    if (d.dtype == DW_F16) return with(__half{});
    return with(__nv_bfloat16{});
}

dw_status launch_read_kv(dw_backend *be, const KvCache &c, const Seqs &s, int dtype, const HeadRows &k, const HeadRows &v) {
    const size_t blocks = ((size_t)s.tokens * 2 + kThreads / 32 - 1) / (kThreads / 32);
    auto go = [&](auto t) {
        using T = decltype(t);
        const bool vec = aligned(k, sizeof(T), 16) && aligned(v, sizeof(T), 16);
        return launch_dependent(be, "read_kv", k_read<T>, (unsigned)blocks, kThreads, 0, 0, c, s, (T *)k.ptr, (T *)v.ptr, k.pitch, v.pitch,
                                vec, be->dev_err);
    };
    if (dtype == DW_F32) return go(float{});
    if (dtype == DW_F16) return go(__half{});
    return go(__nv_bfloat16{});
}

}  // namespace dw
