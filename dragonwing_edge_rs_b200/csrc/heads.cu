// heads.cu -- the heads of a projection's rows on their way to attention: norms of query and
// key heads with the position rotation, keys and values appended to the paged 8-bit cache, and
// cached values read back.
//   norm     rms(x) = x / sqrt(mean(x^2) + eps) * w over a head, layer(x) the same on x - mean(x)
//   rotate   (a, b) -> (a cos t - b sin t, a sin t + b cos t), t = position * freq, in pairs
//   append   X = 2^e, e the smallest with max|v| <= 448 X over the block; code = e4m3(v / X)
// Angles: a frequency is a 64-bit fraction of a turn, so position * frequency modulo a turn is
// one integer product, exact however far the position.
//
// Rotations and reads of many rows are bound by their bytes and the loads in flight, appends by
// the chain from a page's lookup to its codes, short calls by latency.

#include <algorithm>
#include <type_traits>

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
    bool neighbours, whole;  // whole: heads turn whole
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
    }
    // Two groups' values are on their way while one is computed (8192 x 40 heads of 128, 64 of them
    // turned: bf16 50.9 us, f32 71.4; 16-bit rows are bound by the instructions).
    struct Group {
        Raw<T, E> a[J], b[J];
    } g0, g1;
    auto load = [&](Group &x, int h) {
        if (h >= heads) return;
        const T *from = h < p.hq ? (const T *)p.q + row * p.q_pitch + (size_t)h * p.d : (const T *)p.k + row * p.k_pitch + (size_t)(h - p.hq) * p.d;
#pragma unroll
        for (int j = 0; j < J; j++)
            if (live[j]) x.a[j].load(from + a[j]), x.b[j].load(from + b[j]);
    };
    int h = first * per + lane / p.group, weights = -1;
    const int end = min((first + p.chunk) * per, (heads + per - 1) / per * per);
    load(g0, h);
    if (h + per < end) load(g1, h + per);
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int i = 0; i < E; i++)
            if (turns[j]) turn_f32(p.rope[(sub + j * p.group) * E + i], position, cs[j][i], sn[j][i]);
    auto sum = [&](float x) {
#pragma unroll
        for (int o = 16; o; o >>= 1)
            if (o < p.group) x += __shfl_xor_sync(0xffffffffu, x, o);
        return x;
    };
    auto one = [&](Group &x) {
        float v[J][2 * E];
        const bool there = h < heads;
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int i = 0; i < E; i++) {
                v[j][i] = there && live[j] ? x.a[j].get(i) : 0.0f;
                v[j][E + i] = there && live[j] ? x.b[j].get(i) : 0.0f;
            }
        if (h + 2 * per < end) load(x, h + 2 * per);
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
        if (there) {
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
        h += per;
    };
    while (h < end) {
        one(g0);
        if (h < end) one(g1);
    }
}

constexpr int kAhead = 4;

// The same for heads that turn whole and fill their lanes (d = 2 E * 32 / kPer; kPer heads a
// group): a lane keeps the products of weights and angles, so that a value is
// rstd * (a * (w_a cos) - b * (w_b sin)), and finds one in kPer of its angles, the others by
// exchange with the lanes that have the same pairs of the group's other heads.
template <typename T, int E, int kPer>
__device__ __forceinline__ void rope_row(const HeadParams &p, size_t row, int64_t position, int first) {
    constexpr int kGroup = 32 / kPer, kMine = E > kPer ? E / kPer : 1, kD = 2 * E * kGroup;
    const int lane = threadIdx.x & 31, sub = lane % kGroup, in = lane / kGroup;
    const int qg = (p.hq + kPer - 1) / kPer, kg = (p.hk + kPer - 1) / kPer, end = min(first + p.chunk, qg + kg);
    const bool nb = p.neighbours;
    const int a = nb ? 2 * E * sub : E * sub, b = nb ? a + E : kD / 2 + E * sub;
    struct Group {
        Raw<T, E> a, b;
    } groups[kAhead];
    // group g of the row: its heads of q, or of k
    auto place = [&](const void *q, size_t q_pitch, const void *k, size_t k_pitch, int g, bool &there) {
        const bool key = g >= qg;
        const int h = (key ? g - qg : g) * kPer + in, heads = key ? p.hk : p.hq;
        there = h < heads;
        return (T *)(key ? k : q) + row * (key ? k_pitch : q_pitch) + (size_t)min(h, heads - 1) * kD;
    };
    auto load = [&](Group &x, int g) {
        bool there;
        const T *from = place(p.q, p.q_pitch, p.k, p.k_pitch, g, there);
        x.a.load(from + a), x.b.load(from + b);
    };
#pragma unroll
    for (int n = 0; n < kAhead; n++)
        if (first + n < end) load(groups[n], first + n);
    float mc[kMine], ms[kMine], cs[E], sn[E];
#pragma unroll
    for (int m = 0; m < kMine; m++)
        if (in + m * kPer < E) turn_f32(p.rope[sub * E + in + m * kPer], position, mc[m], ms[m]);
#pragma unroll
    for (int i = 0; i < E; i++) {
        cs[i] = __shfl_sync(0xffffffffu, mc[i / kPer], i % kPer * kGroup + sub);
        sn[i] = __shfl_sync(0xffffffffu, ms[i / kPer], i % kPer * kGroup + sub);
    }
    // halves: pair i is values i and E + i of a lane; neighbours: values 2 i and 2 i + 1
    auto A = [&](const float (&v)[2 * E], int i) { return nb ? v[2 * i] : v[i]; };
    auto B = [&](const float (&v)[2 * E], int i) { return nb ? v[2 * i + 1] : v[E + i]; };
    float ac[E], bs[E], as[E], bc[E];
    auto weigh = [&](const float *weights) {
        float w[2 * E];
#pragma unroll
        for (int i = 0; i < E; i++) w[i] = weights ? weights[a + i] : 1.0f, w[E + i] = weights ? weights[b + i] : 1.0f;
#pragma unroll
        for (int i = 0; i < E; i++) {
            ac[i] = A(w, i) * cs[i], as[i] = A(w, i) * sn[i];
            bc[i] = B(w, i) * cs[i], bs[i] = -(B(w, i) * sn[i]);
        }
    };
    auto sum = [&](float x) {
#pragma unroll
        for (int o = 1; o < kGroup; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        return x;
    };
    auto one = [&](Group &x, int g) {
        float v[2 * E];
#pragma unroll
        for (int i = 0; i < E; i++) v[i] = x.a.get(i), v[E + i] = x.b.get(i);
        if (g + kAhead < end) load(x, g + kAhead);
        if (p.norm != DW_NORM_NONE) {
            if (p.norm == DW_NORM_LAYER) {
                float m = 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * E; i++) m += v[i];
                m = sum(m) * p.inv_d;
#pragma unroll
                for (int i = 0; i < 2 * E; i++) v[i] -= m;
            }
            float2 sq = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < 2 * E; i += 2) sq = __ffma2_rn(make_float2(v[i], v[i + 1]), make_float2(v[i], v[i + 1]), sq);
            const float rstd = __frsqrt_rn(fmaf(sum(sq.x + sq.y), p.inv_d, p.eps));
#pragma unroll
            for (int i = 0; i < 2 * E; i += 2) {
                const float2 r = __fmul2_rn(make_float2(v[i], v[i + 1]), make_float2(rstd, rstd));
                v[i] = r.x, v[i + 1] = r.y;
            }
        }
        float y[2 * E];
        auto turn = [&](auto near) {  // two pairs to an instruction
            constexpr bool kNear = decltype(near)::value;
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                const int a0 = kNear ? 2 * i : i, a1 = kNear ? 2 * i + 2 : i + 1, b0 = kNear ? 2 * i + 1 : E + i, b1 = kNear ? 2 * i + 3 : E + i + 1;
                const float2 va = make_float2(v[a0], v[a1]), vb = make_float2(v[b0], v[b1]);
                const float2 ya = __ffma2_rn(va, make_float2(ac[i], ac[i + 1]), __fmul2_rn(vb, make_float2(bs[i], bs[i + 1])));
                const float2 yb = __ffma2_rn(va, make_float2(as[i], as[i + 1]), __fmul2_rn(vb, make_float2(bc[i], bc[i + 1])));
                y[a0] = ya.x, y[a1] = ya.y, y[b0] = yb.x, y[b1] = yb.y;
            }
        };
        if (nb)
            turn(std::true_type{});
        else
            turn(std::false_type{});
        bool there;
        T *out = place(p.q_out, p.qo_pitch, p.k_out, p.ko_pitch, g, there);
        if (!there) return;
        float lo[E], hi[E];
#pragma unroll
        for (int i = 0; i < E; i++) lo[i] = y[i], hi[i] = y[E + i];
        Raw<T, E> r;
        r.set(lo);
        r.store(out + a);
        r.set(hi);
        r.store(out + b);
    };
    weigh(first < qg ? p.w_q : p.w_k);
    for (int base = first; base < end; base += kAhead) {
#pragma unroll
        for (int n = 0; n < kAhead; n++) {
            const int g = base + n;
            if (g >= end) break;
            if (g == qg && g != first) weigh(p.w_k);
            one(groups[n], g);
        }
    }
}

template <typename T, int E, int kPer>
__global__ void __launch_bounds__(kThreads) k_rope(const __grid_constant__ HeadParams p) {
    pdl_wait();
    pdl_trigger();
    const size_t unit = (size_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32, row = unit / p.chunks;
    if (row >= p.tokens) return;
    rope_row<T, E, kPer>(p, row, p.positions[row], (int)(unit % p.chunks) * p.chunk);
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
// tokens, a lane 2 E = d / 32 values of each.  Keys are computed in f64 and kept, in shared
// memory, as f32 rounded to odd (a last bit of 1 where anything was cut off), which rounds to
// e4m3 as the f64 would: the cached codes are the definition's own, whatever hardware or order
// computed them.  (f32 with a bound, and f64 where that leaves two codes open, took longer: the
// bound has to hold for the pair, and one token in five had a value too small beside its
// partner.)  A warp's tokens follow each other, so the angles after the first come by one
// complex product each.  The blocks behind those of the pages norm and turn query rows.  (4096
// tokens, 8 heads of 128 bf16, three sets of inputs in turn: 18.4 us, 25 MB; with 32 query heads
// 31.9, 92 MB.)
constexpr int kWarpTokens = 8;

__device__ __forceinline__ float round_to_odd(double v) {
    const float f = __double2float_rz(v);
    return __uint_as_float(__float_as_uint(f) | (uint32_t)((__double2loint(v) & 0x1FFFFFFF) != 0));
}

template <typename T, int E, bool kVec>
__device__ __forceinline__ void load_values(const T *p, float (&v)[E]) {
    if constexpr (kVec) {
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

// The place of item w of rows whose sequences have as many each.
__device__ __forceinline__ uint32_t seq_and_place(const Seqs &q, uint32_t w, uint32_t each, int per, int size, int extra, int64_t &place) {
    if (q.starts) return seq_of_item(q, w, per, size, extra, place);
    place = w % each;
    return w / each;
}

template <typename T, int E, int QE, int QJ, bool kVec>
__global__ void __launch_bounds__(512)
    k_append(const __grid_constant__ HeadParams p, const __grid_constant__ KvCache c, const __grid_constant__ Seqs q,
             const uint32_t page_blocks, const uint32_t each_rows, const uint32_t each_pages, int32_t *err) {
    extern __shared__ float keys[];  // [page][d], as lanes have them
    __shared__ uint32_t top[2][16];
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, warps = blockDim.x / 32;
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x >= page_blocks) {
        const size_t unit = (size_t)(blockIdx.x - page_blocks) * warps + warp;
        const size_t row = unit / p.chunks;
        if (row >= p.tokens) return;
        int64_t place;
        const uint32_t s = seq_and_place(q, (uint32_t)row, each_rows, 1, 1, 0, place);
        const SeqRange r = seq_range(q, s, c.page, err, -1);
        if (place < 0 || place >= r.n) return;
        HeadParams pq = p;
        pq.hk = 0;
        const int from = (int)(unit % p.chunks) * p.chunk;
        if constexpr (QJ == 0)
            rope_row<T, QE, QE / E>(pq, row, r.position((int)row), from);
        else
            norm_rope_row<T, QE, QJ>(pq, row, r.position((int)row), from);
        return;
    }
    const int head = (int)(blockIdx.x % p.hk);
    int64_t place;
    const uint32_t s = seq_and_place(q, blockIdx.x / p.hk, each_pages, 1, c.page, 2, place);
    const SeqRange r = seq_range(q, s, c.page, err, blockIdx.x / p.hk);
    const int shift = 31 - __clz(c.page);   // pages hold a power of two of tokens
    const int first = max(r.len - r.n, 0);  // the sequence's first new token
    const int64_t begin = ((first >> shift) + place) << shift;
    if (place < 0 || first >= r.len || begin >= r.len) return;
    const uint32_t named = (uint32_t)q.table[(size_t)s * q.width + (uint32_t)(begin >> shift)], page = min(named, c.pages - 1);
    // Nothing is written for a sequence whose length, starts or page lie outside: what they were
    // brought to belongs to other sequences, or to other tokens of this one.  (The same for all
    // threads of the block.)
    if (named >= c.pages) record_error(err, DW_DEV_BAD_ARG, 62, (int)s);
    if (named >= c.pages || !r.ok || !seq_apart(q, s)) return;
    const int t0 = max(first, (int)begin), t1 = (int)min((int64_t)r.len, begin + c.page);
    const int w0 = (int)begin + warp * kWarpTokens;  // the warp's first token
    const Slot<E> slot(lane, p.rot, p.neighbours);
    const T *const kp = (const T *)p.k + (size_t)head * p.d, *const vp = (const T *)p.v + (size_t)head * p.d;
    uint8_t *const scale = c.s + kv_block(c, page, head) * 2;
    const bool has_old = t0 > begin;
    const int k_old = has_old ? kv_exponent(scale[0]) : kKvMinExp, v_old = has_old ? kv_exponent(scale[1]) : kKvMinExp;
    uint8_t *const kc = kv_codes(c.k, c, page, head), *const vc = kv_codes(c.v, c, page, head);
    const int from = max(w0, t0), to = min(w0 + kWarpTokens, t1);
    // the lane's places in the rows of the warp's first token
    const size_t row = (size_t)r.row0 + (from - (r.len - r.n));
    const T *const ka = kp + row * p.k_pitch + slot.a, *const va = vp + row * p.v_pitch + 2 * E * lane;
    const int half = slot.b - slot.a;
    float kmax = 0.0f, vmax = 0.0f;
    uint32_t poison = 0;
    if (from < to) {
        double cs[E], sn[E], cs1[E], sn1[E];
        double w[2 * E];
        const double inv_d = 1.0 / (64 * E);  // a power of two
        const bool weighs = p.w_k;
#pragma unroll
        for (int j = 0; j < E; j++) {
            w[j] = weighs ? p.w_k[slot.a + j] : 1.0f, w[E + j] = weighs ? p.w_k[slot.b + j] : 1.0f;
            cs[j] = cs1[j] = 1.0, sn[j] = sn1[j] = 0.0;
            if (slot.turns) {
                const int pair = lane * E + j, pairs = p.rot / 2;
                turn_f64(p.rope[pair], from, cs[j], sn[j]);
                const double *const step = reinterpret_cast<const double *>(p.rope + pairs);
                cs1[j] = step[pair], sn1[j] = step[pairs + pair];
            }
        }
        auto some = [&](const int t4, auto count) {
            constexpr int kBatch = decltype(count)::value;
            float kv[kBatch][2 * E], vv[kBatch][2 * E];
#pragma unroll
            for (int i = 0; i < kBatch; i++) {
                const uint32_t n = (uint32_t)(min(t4 + i, to - 1) - from);
                const T *const k = ka + n * p.k_pitch;
                float lo[E], hi[E];
                load_values<T, E, kVec>(k, lo);
                load_values<T, E, kVec>(k + half, hi);
#pragma unroll
                for (int j = 0; j < E; j++) kv[i][j] = lo[j], kv[i][E + j] = hi[j];
                load_values<T, 2 * E, kVec>(va + n * p.v_pitch, vv[i]);
            }
            // the batch's tokens side by side (one after the other each waited for its own sums; what
            // lies behind the last is computed too, and left)
            double x[kBatch][2 * E];
#pragma unroll
            for (int i = 0; i < kBatch; i++)
#pragma unroll
                for (int j = 0; j < 2 * E; j++) x[i][j] = kv[i][j];
            if (p.norm != DW_NORM_NONE) {
                double sum[kBatch];
                auto sums = [&]() {
#pragma unroll
                    for (int o = 16; o; o >>= 1)
#pragma unroll
                        for (int i = 0; i < kBatch; i++) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
                };
                if (p.norm == DW_NORM_LAYER) {
#pragma unroll
                    for (int i = 0; i < kBatch; i++) {
                        sum[i] = 0.0;
#pragma unroll
                        for (int j = 0; j < 2 * E; j++) sum[i] += x[i][j];
                    }
                    sums();
#pragma unroll
                    for (int i = 0; i < kBatch; i++)
#pragma unroll
                        for (int j = 0; j < 2 * E; j++) x[i][j] -= sum[i] * inv_d;
                }
#pragma unroll
                for (int i = 0; i < kBatch; i++) {
                    sum[i] = 0.0;
#pragma unroll
                    for (int j = 0; j < 2 * E; j++) sum[i] = fma(x[i][j], x[i][j], sum[i]);
                }
                sums();
#pragma unroll
                for (int i = 0; i < kBatch; i++) {
                    const double rstd = rsqrt(fma(sum[i], inv_d, (double)p.eps));
#pragma unroll
                    for (int j = 0; j < 2 * E; j++) x[i][j] *= rstd * w[j];
                }
            }
#pragma unroll
            for (int i = 0; i < kBatch; i++) {
                const int t = min(t4 + i, to - 1);
                const bool in = t4 + i < to;
                if (slot.turns) rotate<E, double>(x[i], cs, sn, p.neighbours);
                bool ok = true;
                float km = 0.0f, vm = 0.0f, y[2 * E];
#pragma unroll
                for (int j = 0; j < 2 * E; j++) {
                    ok = ok && isfinite(x[i][j]) && isfinite(vv[i][j]);
                    y[j] = round_to_odd(x[i][j]);
                    km = fmaxf(km, fabsf(y[j])), vm = fmaxf(vm, fabsf(vv[i][j]));
                }
                const bool number = __all_sync(0xffffffffu, ok);
                if (in && number) kmax = fmaxf(kmax, km), vmax = fmaxf(vmax, vm);
                if (in && !number) poison |= 1u << (t - w0);
                float *const place = keys + (uint32_t)(t - (int)begin) * (64 * E) + lane * 2 * E;
#pragma unroll
                for (int j = 0; j < 2 * E; j++)
                    if (in) place[j] = y[j];
#pragma unroll
                for (int j = 0; j < E; j++) {  // the next token's angle
                    const double cn = cs[j] * cs1[j] - sn[j] * sn1[j];
                    sn[j] = sn[j] * cs1[j] + cs[j] * sn1[j];
                    cs[j] = cn;
                }
            }
        };
        if (to - from == 1) {
            some(from, std::integral_constant<int, 1>{});
        } else {
#pragma unroll 1
            for (int t4 = from; t4 < to; t4 += 4) some(t4, std::integral_constant<int, 4>{});
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
    if (ke != k_old || ve != v_old)  // the codes that the block holds are rounded again
        for (int t = w0; t < min(w0 + kWarpTokens, t0); t++) {
            uint8_t *const kr = kc + (t - (int)begin) * p.d, *const vr = vc + (t - (int)begin) * p.d;
            if (ke != k_old) rescale_codes<E>(kr + 2 * E * lane, kv_pow2(k_old - ke));
            if (ve != v_old) rescale_codes<E>(vr + 2 * E * lane, kv_pow2(v_old - ve));
        }
#pragma unroll 4
    for (int t = from; t < to; t++) {
        const uint32_t in = (uint32_t)(t - (int)begin) * (64 * E);
        uint8_t *const kr = kc + in, *const vr = vc + in;
        const bool bad = poison >> (t - w0) & 1;
        const float *const place = keys + in + lane * 2 * E;
        float lo[E], hi[E], all[2 * E];
#pragma unroll
        for (int j = 0; j < E; j++) {
            lo[j] = bad ? __uint_as_float(0x7FC00000u) : place[j] * k_inv;
            hi[j] = bad ? __uint_as_float(0x7FC00000u) : place[E + j] * k_inv;
        }
        load_values<T, 2 * E, kVec>(va + (uint32_t)(t - from) * p.v_pitch, all);
#pragma unroll
        for (int j = 0; j < 2 * E; j++) all[j] = bad ? 0.0f : all[j] * v_inv;
        store_codes<E>(kr + slot.a, lo);
        store_codes<E>(kr + slot.b, hi);
        store_codes<2 * E>(vr + 2 * E * lane, all);
    }
}

// ---- read --------------------------------------------------------------------------
// A warp has a row's keys or values, a lane 16 of them at a time (4096 rows of 8 heads of 128 bf16
// 7.2 us, 25 MB: a row's lookups and its loads, one after the other).
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_read(const __grid_constant__ KvCache c, const __grid_constant__ Seqs q, const uint32_t each_rows, T *k_out, T *v_out, size_t k_pitch,
           size_t v_pitch, const bool vec, int32_t *err) {
    const int lane = threadIdx.x & 31;
    const size_t unit = (size_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
    pdl_wait();
    pdl_trigger();
    const size_t row = unit / 2;
    const bool values = unit & 1;
    T *out = values ? v_out : k_out;
    if (row >= q.tokens || !out) return;
    int64_t place;
    const uint32_t s = seq_and_place(q, (uint32_t)row, each_rows, 1, 1, 0, place);
    const SeqRange r = seq_range(q, s, c.page, err, -1);
    for (size_t i = row * 32 + lane; q.starts && i < q.seqs; i += (size_t)q.tokens * 32)
        if (bad_start(q, (int64_t)i)) record_error(err, DW_DEV_BAD_ARG, 61, (int)i);
    if (place < 0 || place >= r.n) return;
    out += row * (values ? v_pitch : k_pitch);
    const int t = r.position((int)row), shift = 31 - __clz(c.page), d_shift = 31 - __clz(c.d);  // powers of two
    const uint32_t page = t < 0 ? 0 : seq_page(q, c, s, (uint32_t)t >> shift, err);
    const uint8_t *const codes = (values ? c.v : c.k) + ((kv_block(c, page, 0) << shift) + (t & (c.page - 1))) * c.d;
    const uint8_t *const scales = c.s + kv_block(c, page, 0) * 2 + values;
#pragma unroll 2
    for (int i = lane * 16; i < c.heads << d_shift; i += 512) {
        const int head = i >> d_shift;
        uint4 w = make_uint4(0, 0, 0, 0);
        float x = 0.0f;
        if (t >= 0) {
            w = *reinterpret_cast<const uint4 *>(codes + ((size_t)head << (shift + d_shift)) + (i & (c.d - 1)));
            x = kv_pow2(kv_exponent(scales[2 * head]));
        }
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = e4m3_to_f32x2((uint16_t)(ws[2 * h + j / 2] >> (16 * (j % 2))));
                v[2 * j] = f.x * x, v[2 * j + 1] = f.y * x;
            }
            if (vec) {
                Raw<T, 8> o;
                o.set(v);
                o.store(out + i + 8 * h);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) out[i + 8 * h + j] = from_f32<T>(v[j]);
            }
        }
    }
}

bool aligned(const HeadRows &h, size_t es, size_t a) { return !h.ptr || ((uintptr_t)h.ptr % a == 0 && h.pitch * es % a == 0); }

HeadParams params(const dw_head_desc &d, size_t tokens, const HeadArgs &a) {
    HeadParams p{};
    p.q = a.q.ptr, p.k = a.k.ptr, p.v = a.v.ptr, p.q_out = a.q_out.ptr, p.k_out = a.k_out.ptr;
    p.q_pitch = a.q.pitch, p.k_pitch = a.k.pitch, p.v_pitch = a.v.pitch, p.qo_pitch = a.q_out.pitch, p.ko_pitch = a.k_out.pitch;
    if (d.norm != DW_NORM_NONE) p.w_q = a.w_q, p.w_k = a.w_k;  // (without a norm nothing weighs)
    p.rope = a.rope, p.positions = a.positions;
    p.tokens = (uint32_t)tokens;
    p.hq = a.q.ptr ? d.q_heads : 0, p.hk = a.k.ptr ? d.kv_heads : 0;
    p.d = d.head_dim, p.rot = d.rot_dim, p.norm = d.norm;
    p.eps = d.eps, p.inv_d = 1.0f / (float)d.head_dim, p.neighbours = d.neighbours != 0;
    p.whole = d.rot_dim == d.head_dim;
    return p;
}

// The lanes of a head with E values in a piece and J slots a lane, and how the heads of a row
// are shared out: a warp has all of a row's, so that its angles are computed once, unless the
// rows are fewer than the warps that the GPU holds at about this many registers (ten groups,
// all by one warp and one a warp: 1 row 6.0 and 2.3 us, 256 rows 7.2 and 4.3, shared by this
// rule 3.6, 1024 rows 7.3, 9.9 and 5.7, 2048 rows 8.9 and 17).
void split(const dw_backend *be, HeadParams &p, int E, int J) {
    p.group = 1;
    while (p.group * 2 * E * J < p.d) p.group *= 2;
    const int per = 32 / p.group, groups = (p.hq + per - 1) / per + (p.hk + per - 1) / per;
    const int parts = (int)std::min<size_t>(groups, std::max<size_t>(1, (size_t)be->sm_count * 16 / p.tokens));
    p.chunk = (groups + parts - 1) / parts;
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
    auto go = [&](auto kernel, int E, int J) {
        split(be, p, E, J);
        const size_t blocks = ((size_t)p.tokens * p.chunks + kThreads / 32 - 1) / (kThreads / 32);
        if (blocks > 0x7fffffffu) return dw_fail(be, DW_ERR_UNSUPPORTED, "norm_rope: too many rows");
        return launch_dependent(be, "norm_rope", kernel, (unsigned)blocks, kThreads, 0, 0, p);
    };
    if (wide<T>(p, {a.q, a.k, a.q_out, a.k_out})) {
        constexpr int E = kWide<T>;
        if (p.whole && p.d == 16 * E) return go(k_rope<T, E, 4>, E, 1);
        if (p.whole && p.d == 8 * E) return go(k_rope<T, E, 8>, E, 1);
        if (p.whole && p.d == 32 * E) return go(k_rope<T, E, 2>, E, 1);
    }
    if (wide<T>(p, {a.q, a.k, a.q_out, a.k_out})) return go(k_norm_rope<T, kWide<T>, 1>, kWide<T>, 1);
    if (p.d <= 128) return go(k_norm_rope<T, 1, 2>, 1, 2);
    return go(k_norm_rope<T, 1, 8>, 1, 8);
}

template <typename T, int E>
dw_status append(dw_backend *be, HeadParams p, const KvCache &c, const Seqs &s, const HeadArgs &a) {
    const bool vec = aligned(a.k, sizeof(T), E * sizeof(T)) && aligned(a.v, sizeof(T), 2 * E * sizeof(T));
    const unsigned threads = (unsigned)(c.page / kWarpTokens * 32);
    const size_t n = s.tokens / s.seqs, each = seq_items_each(n, 1, c.page, 2);
    const size_t pages = (s.starts ? seq_items(s.tokens, s.seqs, 1, c.page, 2) : each * s.seqs) * p.hk;
    auto go = [&](auto kernel, int QE, int QJ) {
        size_t blocks = pages;
        p.chunks = 1;
        if (p.hq) {
            HeadParams queries = p;
            queries.hk = 0;
            split(be, queries, QE, QJ ? QJ : 1);
            p.group = queries.group, p.chunk = queries.chunk, p.chunks = queries.chunks;
            blocks += ((size_t)p.tokens * p.chunks + threads / 32 - 1) / (threads / 32);
        }
        if (blocks > 0x7fffffffu) return dw_fail(be, DW_ERR_UNSUPPORTED, "append_kv: too many rows");
        const size_t smem = (size_t)c.page * c.d * 4;
        if (smem > 48 * 1024)
            if (dw_status st = dw_cuda_check(be, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                                             "append_kv attributes");
                st != DW_OK)
                return st;
        return launch_dependent(be, "append_kv", kernel, (unsigned)blocks, threads, smem, 0, p, c, s, (uint32_t)pages, (uint32_t)n,
                                (uint32_t)each, be->dev_err);
    };
    if (vec && wide<T>(p, {a.q, a.q_out}) && p.whole) return go(k_append<T, E, kWide<T>, 0, true>, kWide<T>, 1);
    if (vec && wide<T>(p, {a.q, a.q_out})) return go(k_append<T, E, kWide<T>, 1, true>, kWide<T>, 1);
    return go(k_append<T, E, 1, E, false>, 1, E);
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
        return launch_dependent(be, "read_kv", k_read<T>, (unsigned)blocks, kThreads, 0, 0, c, s, s.tokens / s.seqs, (T *)k.ptr, (T *)v.ptr, k.pitch, v.pitch,
                                vec, be->dev_err);
    };
    if (dtype == DW_F32) return go(float{});
    if (dtype == DW_F16) return go(__half{});
    return go(__nv_bfloat16{});
}

}  // namespace dw

// What the kernels of sequences are launched over, on the host.
extern "C" DW_API size_t dw_debug_seq_items(const int32_t *starts, size_t seqs, size_t tokens, int per, int size, int extra, uint32_t *seq,
                                            int64_t *place) {
    if (!seqs || per <= 0 || size <= 0 || extra < 0) return 0;
    const size_t each = dw::seq_items_each(tokens / seqs, per, size, extra);
    const size_t n = starts ? dw::seq_items(tokens, seqs, per, size, extra) : each * seqs;
    for (size_t w = 0; seq && place && w < n; w++) {
        if (!starts) {
            seq[w] = (uint32_t)(w / each), place[w] = (int64_t)(w % each);
            continue;
        }
        seq[w] = dw::find_item(
            (uint32_t)seqs, (int64_t)w, [&](uint32_t s) { return dw::seq_first_item(starts[s], s, per, size, extra); },
            [](auto f) {
                uint32_t m = 0;
                for (uint32_t i = 0; i < 32; i++) m |= (uint32_t)f(i) << i;
                return m;
            },
            place[w]);
    }
    return n;
}
