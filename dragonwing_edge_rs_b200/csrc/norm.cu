// norm.cu -- RMS and layer norms around a residual block, fused with the block's
// gate and residual scale and, where asked, with the MXFP4 quantisation of the
// result:
//   n   = post(x)                          x: the block's output
//   out = R(res + res_scale * gate * n)    R: rounding to res's type
//   y   = pre(out)                         the next block's input
// with rms(v) = v / sqrt(mean(v^2) + eps) * w + b and layer(v) the same on
// v - mean(v).  Without a residual y = pre(x).  All arithmetic is f32.
//
// Bandwidth-bound: x, res and gate are read once, out and y written once.  Three forms:
// persistent blocks that stream many rows through a ring (8192 x 4096 bf16 with both
// norms 45.6 us, 5.9 TB/s; near the issue rate too), a block
// a row in registers for few (1 x 4096 2.3 us, latency), and a re-reading one for rows
// over 16384.  Times here and below are of launches in a row in short runs; the lower
// clock of a sustained loop costs some 10% (50 us).  Those beside a choice compare its two
// sides at the time it was made.

#include <algorithm>

#include "dw_device.cuh"
#include "dw_launch.h"
#include "dw_mxfp4.cuh"
#include "dw_ptx.cuh"

namespace dw {
namespace {

constexpr int kMaxT = 512;  // threads of a row
constexpr int kMaxE = 32;   // elements of a thread
constexpr size_t kSmemBudget = 216 * 1024;  // of an SM's shared memory for weights and rows to come

struct Params {
    const void *x, *gate, *res;
    const float *w0, *b0, *w1, *b1;
    void *out, *y;
    uint8_t *q, *s;
    size_t rows, c, x_pitch, res_pitch, y_pitch, nb, tiles;
    uint32_t gate_rows;
    int pre, post, y_dtype;  // y_dtype: DW_F32..DW_BF16, -1: none, -2: MXFP4
    float eps, inv_c, res_scale;
    bool has_res;
};

// Sum over the T threads of a row (a power of two; rows of T <= 32 lie in one warp,
// longer ones take whole warps, and all threads of the block call together).
// `slot` alternates over four buffers, so a buffer is written again only after
// three more barriers.  kBar: the threads that call and meet at barrier `bar`, where these
// are not the whole block (`thread`: the place among them).
template <int kBar = 0>
__device__ __forceinline__ float row_sum(float v, int T, float (*red)[16], int &slot, int thread = 0, int bar = 0) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
        if (o < T) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (T <= 32) return v;
    if (!kBar) thread = threadIdx.y * blockDim.x + threadIdx.x;
    const int lane = thread & 31, warp = thread >> 5;
    const int warps = T >> 5, first = warp & ~(warps - 1);
    if (lane == 0) red[slot][warp] = v;
    if (kBar)
        named_barrier_sync(bar, kBar);
    else
        __syncthreads();
    const float *part = &red[slot][first];  // every thread adds the warps' sums, in the same order
    v = part[0] + part[1];
    if (T >= 128) v += part[2] + part[3];
    if (T >= 256) {
        const float4 q = *reinterpret_cast<const float4 *>(part + 4);
        v += (q.x + q.y) + (q.z + q.w);
    }
    if (T >= 512) {
        const float4 q = *reinterpret_cast<const float4 *>(part + 8), r = *reinterpret_cast<const float4 *>(part + 12);
        v += ((q.x + q.y) + (q.z + q.w)) + ((r.x + r.y) + (r.z + r.w));
    }
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

// Element-wise f32 over V values, two to an instruction where V is even (the streaming
// kernel is half issue-bound).
template <int V>
__device__ __forceinline__ void mul_all(float (&a)[V], const float (&b)[V]) {
    if constexpr (V % 2 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float2 r = __fmul2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
            a[i] = r.x, a[i + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) a[i] *= b[i];
    }
}
template <int V>
__device__ __forceinline__ void scale_all(float (&a)[V], float s) {
    if constexpr (V % 2 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float2 r = __fmul2_rn(make_float2(a[i], a[i + 1]), make_float2(s, s));
            a[i] = r.x, a[i + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) a[i] *= s;
    }
}
// c += a * b
template <int V>
__device__ __forceinline__ void fma_all(const float (&a)[V], const float (&b)[V], float (&c)[V]) {
    if constexpr (V % 2 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float2 r = __ffma2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), make_float2(c[i], c[i + 1]));
            c[i] = r.x, c[i + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) c[i] = fmaf(a[i], b[i], c[i]);
    }
}

// v[j][i] -> its norm, in place.  Elements past the row are 0 and stay out of the
// statistics (`live`: element group j lies in the row).  weight(j, wv) and bias(j,
// bv) give a group's weights and return whether there are any.
template <int V, int N, typename W, typename B>
__device__ __forceinline__ void normalise(float (&v)[N][V], const bool (&live)[N], int kind, int T, const Params &p,
                                          float (*red)[16], int &slot, W weight, B bias) {
    if (kind == DW_NORM_LAYER) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int i = 0; i < V; i++) sum += v[j][i];
        const float mean = row_sum(sum, T, red, slot) * p.inv_c;
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
    const float rstd = __frsqrt_rn(fmaf(row_sum(sq, T, red, slot), p.inv_c, p.eps));
#pragma unroll
    for (int j = 0; j < N; j++) {
        if (!live[j]) continue;
        float t[V];
#pragma unroll
        for (int i = 0; i < V; i++) v[j][i] *= rstd;
        if (weight(j, t)) {
#pragma unroll
            for (int i = 0; i < V; i++) v[j][i] *= t[i];
        }
        if (bias(j, t)) {
#pragma unroll
            for (int i = 0; i < V; i++) v[j][i] += t[i];
        }
    }
}

// One group of V values, from column `at` on, as MXFP4: 32 / V neighbouring threads hold a
// block.  q, s: the codes of the row, its place in the first scale tile.
template <int V, typename I>
__device__ __forceinline__ void put_mxfp4(float (&v)[V], I at, uint8_t *q, uint8_t *s, bool there, const Params &p) {
    uint32_t amax = mx_amax(v);
#pragma unroll
    for (int o = 1; o < 32 / V; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const uint32_t sb = mx_scale_byte(amax);
    const I block = at / 32;
    q += at / 2;
    const float next = V == 1 ? __shfl_down_sync(0xffffffffu, v[0], 1) : 0.0f;
    if (!there || block >= p.nb) return;
    const float inv = mx_inv_scale(sb);
    scale_all<V>(v, inv);
    if constexpr (V == 8) {
        *reinterpret_cast<uint32_t *>(q) = sb == 0xFFu ? 0u : mx_codes8(v);
    } else if constexpr (V == 2) {
        *q = sb == 0xFFu ? (uint8_t)0 : (uint8_t)mx_codes2(v[0], v[1]);
    } else {
        if ((threadIdx.x & 1) == 0) *q = sb == 0xFFu ? (uint8_t)0 : (uint8_t)mx_codes2(v[0], next * inv);
    }
    if ((at & 31) == 0) {
        s[(size_t)(block / 4) * 512 + block % 4] = (uint8_t)sb;
        if (block + 1 == p.nb)  // the places of the tile past the last block
            for (size_t b = p.nb; b < p.tiles * 4; b++) s[b / 4 * 512 + b % 4] = 0;
    }
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
__global__ void __launch_bounds__(kMaxT, V * N <= 8 ? 2 : 1) k_norm(const __grid_constant__ Params p) {
    __shared__ __align__(16) float red[4][16];
    int slot = 0;
    const int T = blockDim.x, tid = threadIdx.x;
    auto from = [&](const float *w) {
        return [w, T, tid](int j, float (&t)[V]) {
            if (w) load_f32<V>(w + ((size_t)j * T + tid) * V, t);
            return w != nullptr;
        };
    };
    pdl_wait();
    pdl_trigger();
    for (size_t row = (size_t)blockIdx.x * blockDim.y + threadIdx.y; row < p.rows; row += (size_t)gridDim.x * blockDim.y) {
        Raw<X, V> xr[N], gr[N];
        Raw<R, V> rr[N];
        bool live[N];
        const X *x = (const X *)p.x + row * p.x_pitch;
        const R *res = (const R *)p.res + row * p.res_pitch;
        const X *gate = (const X *)p.gate + (size_t)(p.gate_rows ? (uint32_t)row / p.gate_rows : 0) * p.c;
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
            if (p.post != DW_NORM_NONE) normalise<V, N>(v, live, p.post, T, p, red, slot, from(p.w0), from(p.b0));
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
        if (p.pre != DW_NORM_NONE) normalise<V, N>(v, live, p.pre, T, p, red, slot, from(p.w1), from(p.b1));
#pragma unroll
        for (int j = 0; j < N; j++) {
            const size_t at = ((size_t)j * T + tid) * V;
            if (p.y_dtype == -2) {
                put_mxfp4<V>(v[j], (uint32_t)at, p.q + row * p.nb * 16, p.s + mx_scale_at(row, 0, p.tiles), true, p);
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

// Many rows: one persistent thread block an SM, of up to three teams that share the weights
// in shared memory and otherwise go their own ways (a block for each, with weights of its
// own, left less room for rows: 8192 x 4096 bf16 with both norms 48.1 against 44.4 us).  A
// team's steps of G = kThreads / T rows come by bulk copies that a warp of its own issues
// (kThreads others compute): a ring of stages holds the x, residual and gate rows of the
// steps to come, so the loads in flight do not depend on how many rows the registers hold.
// Bulk copies move whole 16-byte pieces: a row that starts or ends inside one is copied with
// its surroundings (its neighbours' elements), except where that would leave the tensor.
constexpr int kStreamStages = 2;

// Bytes of a stage: per tensor G rows, one after the other as in memory (`packed`: one
// copy), or each in a place of its own.
struct StreamRows {
    uint32_t bytes, stride, region;
    __host__ __device__ StreamRows(size_t c, size_t es, int G, bool packed, bool present)
        : bytes(present ? (uint32_t)(c * es) : 0u),
          stride(!present ? 0u : packed ? bytes : (bytes + 31) & ~15u),
          region(!present ? 0u : (G * stride + 31) & ~15u) {}
};

// The part of [src, src + bytes) that bulk copies bring, with what surrounds it.
struct Span {
    uintptr_t from, to, base;  // base: the 16-byte piece of src
    __device__ __forceinline__ Span(const uint8_t *src, uint32_t bytes, const uint8_t *first, const uint8_t *last) {
        const uintptr_t a = (uintptr_t)src, e = a + bytes;
        base = a & ~(uintptr_t)15;
        from = base < (uintptr_t)first ? base + 16 : base;
        to = (e + 15) & ~(uintptr_t)15;
        if (to > (uintptr_t)last) to -= 16;
        if (to < from) to = from;
    }
    __device__ __forceinline__ uint32_t bytes() const { return (uint32_t)(to - from); }
    // The bytes at the tensor's ends that it leaves out (fewer than 16 at each): by the calling
    // thread's own stores, which later bulk copies into the same place have to come after.
    __device__ __forceinline__ void edges(uint8_t *dst, const uint8_t *src, uint32_t bytes) const {
        const uintptr_t a = (uintptr_t)src, e = a + bytes;
        if (from <= a && to >= e) return;
        for (uintptr_t q = a; q < e && q < from; q++) dst[q - base] = *(const uint8_t *)q;
        for (uintptr_t q = to > a ? to : a; q < e; q++) dst[q - base] = *(const uint8_t *)q;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
};

// The most teams of a block that its registers hold.  (Short accesses wait long enough for
// three to pay for some spills: 8192 x 4095 bf16 154 -> 137 us, 4096 x 3002 to MXFP4 67 -> 59,
// 8192 x 4094 101 -> 102.)
template <typename R, int V, int N, int kThreads>
constexpr int stream_teams() {
    return kThreads > 256 ? 1 : V * N > 16 || (V == 8 && N > 1 && sizeof(R) == 4) ? 2 : 3;
}

template <typename X, typename R, int V, int N, int kThreads, bool kFull>
__global__ void __launch_bounds__((kThreads + 32) * stream_teams<R, V, N, kThreads>(), 1)
    k_norm_stream(const __grid_constant__ Params p, const int T, const int stages, uint64_t wait_cap_ns, int32_t *err) {
    constexpr int kTeams = stream_teams<R, V, N, kThreads>();
    extern __shared__ __align__(128) uint8_t shared[];
    __shared__ __align__(16) float red[kTeams][4][16];
    __shared__ uint64_t full_bars[kTeams][kStreamStages], empty_bars[kTeams][kStreamStages];
    __shared__ int abort_word;
    const int teams = blockDim.x / (kThreads + 32), team = threadIdx.x / (kThreads + 32), thread = threadIdx.x % (kThreads + 32);
    uint64_t *const full_bar = full_bars[team], *const empty_bar = empty_bars[team];
    volatile int *abort_flag = &abort_word;
    int slot = 0;
    const int lane = thread & 31;
    const int G = kThreads / T, g = thread / T, tid = thread & (T - 1);
    const size_t steps = (p.rows + G - 1) / G;
    // a gate row of the rows themselves comes with them
    const bool row_gate = p.gate && p.gate_rows, packed_x = p.x_pitch == p.c, packed_r = p.res_pitch == p.c;
    const StreamRows lx(p.c, sizeof(X), G, packed_x, true), lr(p.c, sizeof(R), G, packed_r, p.has_res),
        lg(p.c, sizeof(X), G, false, row_gate);
    const uint32_t stage_bytes = lx.region + lr.region + lg.region;
    uint8_t *const ring = shared + team * stages * stage_bytes;
    const uint32_t base = smem_u32(ring);
    const uint8_t *const x0 = (const uint8_t *)p.x, *const r0 = (const uint8_t *)p.res, *const g0 = (const uint8_t *)p.gate;
    const size_t x_pitch = p.x_pitch * sizeof(X), r_pitch = p.res_pitch * sizeof(R);
    if (thread == 0) {
        for (int s = 0; s < stages; s++) mbar_init(smem_u32(&full_bar[s]), 1), mbar_init(smem_u32(&empty_bar[s]), kThreads / 32);
        if (team == 0) abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    // Waits for a phase; after an expired wait nothing waits any more and what is left runs
    // through on what the ring holds.
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (mbar_try_wait(smem_u32(bar), parity)) return;
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait_sleep(smem_u32(bar), parity, 20000u) && !*abort_flag)
            if (globaltimer_ns() - t0 > wait_cap_ns) {
                *abort_flag = 1;
                record_error(err, DW_DEV_WAIT_EXPIRED, 41, (int)parity);
            }
    };
    pdl_wait();
    pdl_trigger();
    // every block's first team before any second one
    const size_t step0 = (size_t)team * gridDim.x + blockIdx.x, step_stride = (size_t)teams * gridDim.x;
    if (thread >= kThreads) {
        int s = 0, issued = 0;
        uint32_t ph = 0;
        for (size_t step = step0; step < steps && !*abort_flag; step += step_stride) {
            if (issued >= stages) wait(&empty_bar[s], ph ^ 1u);
            __syncwarp();
            if (__any_sync(0xffffffffu, *abort_flag)) break;
            const size_t row0 = step * G;
            const uint32_t rows = (uint32_t)min((size_t)G, p.rows - row0), bar = smem_u32(&full_bar[s]);
            // the copies of the step, each to one lane
            auto copies = [&](auto each) {
                auto tensor = [&](const StreamRows &l, const uint8_t *t, size_t pitch, bool packed, uint32_t at, int first_lane) {
                    const uint8_t *last = t + (p.rows - 1) * pitch + l.bytes;
                    if (packed) {
                        if (lane == first_lane) each(t + row0 * pitch, rows * l.bytes, t, last, at);
                    } else {
                        for (uint32_t r = lane; r < rows; r += 32) each(t + (row0 + r) * pitch, l.bytes, t, last, at + r * l.stride);
                    }
                };
                tensor(lx, x0, x_pitch, packed_x, s * stage_bytes, 0);
                if (p.has_res) tensor(lr, r0, r_pitch, packed_r, s * stage_bytes + lx.region, 1);
                if (row_gate) {
                    const uint8_t *last = g0 + (size_t)((uint32_t)(p.rows - 1) / p.gate_rows + 1) * lg.bytes;
                    for (uint32_t r = lane; r < rows; r += 32)
                        each(g0 + (size_t)((uint32_t)(row0 + r) / p.gate_rows) * lg.bytes, lg.bytes, g0, last,
                             s * stage_bytes + lx.region + lr.region + r * lg.stride);
                }
            };
            if constexpr (V == 8) {  // whole pieces
                if (lane == 0) mbar_expect_tx(bar, rows * (lx.bytes + lr.bytes + lg.bytes));
                __syncwarp();
                copies([&](const uint8_t *src, uint32_t n, const uint8_t *, const uint8_t *, uint32_t at) {
                    bulk_load(base + at, src, n, bar);
                });
            } else {
                uint32_t bytes = 0;
                copies([&](const uint8_t *src, uint32_t n, const uint8_t *first, const uint8_t *last, uint32_t at) {
                    const Span span(src, n, first, last);
                    bytes += span.bytes();
                    span.edges(ring + at, src, n);
                });
                bytes = __reduce_add_sync(0xffffffffu, bytes);
                __syncwarp();  // every lane's edges come before the arrive (the sum orders no memory)
                if (lane == 0) mbar_expect_tx(bar, bytes);
                __syncwarp();
                copies([&](const uint8_t *src, uint32_t n, const uint8_t *first, const uint8_t *last, uint32_t at) {
                    const Span span(src, n, first, last);
                    if (span.bytes()) bulk_load(base + at + (uint32_t)(span.from - span.base), (const void *)span.from, span.bytes(), bar);
                });
            }
            issued++;
            if (++s == stages) s = 0, ph ^= 1;
        }
        // the last copies into each stage have landed before the block ends
        for (int i = 0; i < min(issued, stages); i++) {
            if (--s < 0) s = stages - 1, ph ^= 1;
            const uint64_t t0 = globaltimer_ns();
            while (!mbar_try_wait_sleep(smem_u32(&full_bar[s]), ph, 20000u) && globaltimer_ns() - t0 < wait_cap_ns) {
            }
        }
        return;
    }
    // c0: what the normalised x of a column is multiplied by (weight, residual scale and,
    // where all rows share it, the gate); w1: the weight of the next norm (both in shared
    // memory, 16 bytes of a thread beside its neighbour's: registers go to a third team
    // instead)
    float *c0 = reinterpret_cast<float *>(shared + (size_t)teams * stages * stage_bytes), *w1 = c0 + N * T * V;
    bool live[N];
    auto column = [&](int j) { return (uint32_t)(j * T + tid) * V; };
    auto kept = [&](const float *from, int j, float (&t)[V]) {
        if constexpr (V == 8) {
            const float4 *f = reinterpret_cast<const float4 *>(from);
            const float4 a = f[2 * j * T + tid], b = f[(2 * j + 1) * T + tid];
            t[0] = a.x, t[1] = a.y, t[2] = a.z, t[3] = a.w, t[4] = b.x, t[5] = b.y, t[6] = b.z, t[7] = b.w;
        } else {
            load_f32<V>(from + column(j), t);
        }
    };
    auto keep = [&](float *to, int j, const float (&t)[V]) {
        if constexpr (V == 8) {
            float4 *f = reinterpret_cast<float4 *>(to);
            f[2 * j * T + tid] = make_float4(t[0], t[1], t[2], t[3]), f[(2 * j + 1) * T + tid] = make_float4(t[4], t[5], t[6], t[7]);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) to[column(j) + i] = t[i];
        }
    };
#pragma unroll
    for (int j = 0; j < N; j++) {
        live[j] = kFull || column(j) < p.c;
        if (!live[j] || g || j % teams != team) continue;  // the teams share the columns
        float t[V];
        if (p.has_res) {
#pragma unroll
            for (int i = 0; i < V; i++) t[i] = p.res_scale;
            if (p.gate && !row_gate) {
                Raw<X, V> x;
                x.load((const X *)p.gate + column(j));
#pragma unroll
                for (int i = 0; i < V; i++) t[i] *= x.get(i);
            }
            if (p.w0 && p.post != DW_NORM_NONE) {
                float w[V];
                load_f32<V>(p.w0 + column(j), w);
#pragma unroll
                for (int i = 0; i < V; i++) t[i] *= w[i];
            }
            keep(c0, j, t);
        }
#pragma unroll
        for (int i = 0; i < V; i++) t[i] = 1.0f;
        if (p.w1) load_f32<V>(p.w1 + column(j), t);
        keep(w1, j, t);
    }
    named_barrier_sync(1 + kTeams, teams * kThreads);
    // (mean, 1 / root) of v over the row; elements past the row are 0
    auto statistics = [&](float (&v)[N][V], int kind) {
        if (kind == DW_NORM_LAYER) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < N; j++)
#pragma unroll
                for (int i = 0; i < V; i++) sum += v[j][i];
            const float mean = row_sum<kThreads>(sum, T, red[team], slot, thread, 1 + team) * p.inv_c;
#pragma unroll
            for (int j = 0; j < N; j++)
#pragma unroll
                for (int i = 0; i < V; i++) v[j][i] = live[j] ? v[j][i] - mean : 0.0f;
        }
        float part[V], sq = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) part[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < N; j++) fma_all<V>(v[j], v[j], part);
#pragma unroll
        for (int i = 0; i < V; i++) sq += part[i];
        return __frsqrt_rn(fmaf(row_sum<kThreads>(sq, T, red[team], slot, thread, 1 + team), p.inv_c, p.eps));
    };
    int s = 0;
    uint32_t ph = 0;
    for (size_t step = step0; step < steps; step += step_stride) {
        wait(&full_bar[s], ph);
        const size_t row = step * G + g, row0 = packed_x ? step * G : row, rrow0 = packed_r ? step * G : row;
        const bool there = row < p.rows;
        // rows of the last step past the end hold what the stage held: they stay in
        // their own threads and nothing of them is stored
        const uint8_t *stage = ring + s * stage_bytes;
        const X *xs = reinterpret_cast<const X *>(stage + g * lx.stride + (((uintptr_t)x0 + row0 * x_pitch) & 15));
        const R *rs = reinterpret_cast<const R *>(stage + lx.region + g * lr.stride + (((uintptr_t)r0 + rrow0 * r_pitch) & 15));
        const X *gs = reinterpret_cast<const X *>(stage + lx.region + lr.region + g * lg.stride +
                                                  (((uintptr_t)g0 + (size_t)(row_gate ? (uint32_t)row / p.gate_rows : 0) * lx.bytes) & 15));
        auto release = [&]() {  // the warp has read the stage
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&empty_bar[s]));
            if (++s == stages) s = 0, ph ^= 1;
        };
        float v[N][V];
        // 16-byte accesses: the residual and gate rows go to registers too and the stage is
        // free at once; shorter ones: they are read where they are used
        Raw<R, V> rr[V == 8 ? N : 1];
        Raw<X, V> gr[V == 8 ? N : 1];
#pragma unroll
        for (int j = 0; j < N; j++) {
            Raw<X, V> xr;
            xr.zero();
            if (V == 8 && !kFull) rr[V == 8 ? j : 0].zero();
            if (live[j]) {
                xr.load(xs + column(j));
                if (V == 8 && p.has_res) rr[V == 8 ? j : 0].load(rs + column(j));
                if (V == 8 && row_gate) gr[V == 8 ? j : 0].load(gs + column(j));
            }
#pragma unroll
            for (int i = 0; i < V; i++) v[j][i] = xr.get(i);
        }
        if (V == 8 || !p.has_res) release();
        if (p.has_res) {
            const float rstd = p.post != DW_NORM_NONE ? statistics(v, p.post) : 1.0f;
            R *out = (R *)p.out + row * p.res_pitch;
            // the gate of the row or the bias: branches around whole loops (inside, each
            // element would carry their predicated instructions)
            auto join = [&](auto coefficient, auto bias) {
#pragma unroll
                for (int j = 0; j < N; j++) {
                    if (!live[j]) continue;
                    float o[V], t[V];
                    kept(c0, j, t);
                    coefficient(j, t);
                    Raw<R, V> res = rr[V == 8 ? j : 0];
                    if constexpr (V < 8) res.load(rs + column(j));
#pragma unroll
                    for (int i = 0; i < V; i++) o[i] = res.get(i);
                    scale_all<V>(v[j], rstd);
                    fma_all<V>(v[j], t, o);
                    bias(j, o);
                    Raw<R, V> r;
                    r.set(o);
                    if (there) r.store(out + column(j));
#pragma unroll
                    for (int i = 0; i < V; i++) v[j][i] = r.get(i);
                }
            };
            auto nothing = [](int, float (&)[V]) {};
            if (!row_gate && !(p.b0 && p.post != DW_NORM_NONE)) {
                join(nothing, nothing);
            } else {
                join(
                    [&](int j, float (&t)[V]) {
                        if (!row_gate) return;
                        Raw<X, V> g = gr[V == 8 ? j : 0];
                        if constexpr (V < 8) g.load(gs + column(j));
#pragma unroll
                        for (int i = 0; i < V; i++) t[i] *= g.get(i);
                    },
                    [&](int j, float (&o)[V]) {  // + res_scale * gate * b
                        if (!p.b0 || p.post == DW_NORM_NONE) return;
                        float b[V];
                        load_f32<V>(p.b0 + column(j), b);
                        Raw<X, V> g = gr[V == 8 ? j : 0];
                        if (V < 8 && row_gate) g.load(gs + column(j));
                        if (p.gate && !row_gate) g.load((const X *)p.gate + column(j));
#pragma unroll
                        for (int i = 0; i < V; i++) o[i] = fmaf(b[i], p.gate ? p.res_scale * g.get(i) : p.res_scale, o[i]);
                    });
            }
        }
        if (V < 8 && p.has_res) release();
        if (p.y_dtype == -1) continue;
        if (p.pre != DW_NORM_NONE) {
            const float rstd = statistics(v, p.pre);
#pragma unroll
            for (int j = 0; j < N; j++) {
                if (!live[j]) continue;
                float t[V];
                kept(w1, j, t);
                scale_all<V>(v[j], rstd);
                mul_all<V>(v[j], t);
            }
            if (p.b1) {
#pragma unroll
                for (int j = 0; j < N; j++) {
                    if (!live[j]) continue;
                    float t[V];
                    load_f32<V>(p.b1 + column(j), t);
#pragma unroll
                    for (int i = 0; i < V; i++) v[j][i] += t[i];
                }
            }
        }
        if (p.y_dtype == -2) {
            uint8_t *q = p.q + row * p.nb * 16, *sr = p.s + mx_scale_at(row, 0, p.tiles);
#pragma unroll
            for (int j = 0; j < N; j++) put_mxfp4<V>(v[j], column(j), q, sr, there, p);
        } else if (there) {
            auto store = [&](auto *y) {
                y += row * p.y_pitch;
#pragma unroll
                for (int j = 0; j < N; j++)
                    if (live[j]) put<std::remove_pointer_t<decltype(y)>, V>(y, column(j), v[j]);
            };
            if (p.y_dtype == DW_F32)
                store((float *)p.y);
            else if (p.y_dtype == DW_F16)
                store((__half *)p.y);
            else
                store((__nv_bfloat16 *)p.y);
        }
    }
}

// Rows too long for registers: one thread block a row, elements read again for
// each reduction (from L2) and `out` read back by the thread that wrote it.  Bound by its
// single-element accesses, and by the SMs that few rows leave idle (both norms, bf16:
// 64 x 40000 75 us against 3.2 for its bytes, 8192 x 20000 1038 against 203).
template <typename X, typename R>
__global__ void __launch_bounds__(kMaxT) k_norm_long(const __grid_constant__ Params p) {
    __shared__ __align__(16) float red[4][16];
    int slot = 0;
    const size_t row = blockIdx.x;
    const size_t T = blockDim.x, end = p.nb * 32;
    const X *x = (const X *)p.x + row * p.x_pitch;
    const R *res = (const R *)p.res + row * p.res_pitch;
    const X *gate = (const X *)p.gate + (size_t)(p.gate_rows ? (uint32_t)row / p.gate_rows : 0) * p.c;
    R *out = (R *)p.out + row * p.res_pitch;
    pdl_wait();
    pdl_trigger();
    auto stats = [&](auto at, int kind, float &mean, float &rstd) {
        mean = 0.0f, rstd = 1.0f;
        if (kind == DW_NORM_NONE) return;
        if (kind == DW_NORM_LAYER) {
            float sum = 0.0f;
            for (size_t i = threadIdx.x; i < p.c; i += T) sum += at(i);
            mean = row_sum(sum, (int)T, red, slot) * p.inv_c;
        }
        float sq = 0.0f;
        for (size_t i = threadIdx.x; i < p.c; i += T) {
            const float d = at(i) - mean;
            sq = fmaf(d, d, sq);
        }
        rstd = __frsqrt_rn(fmaf(row_sum(sq, (int)T, red, slot), p.inv_c, p.eps));
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
            put_mxfp4<1>(v, i, p.q + row * p.nb * 16, p.s + mx_scale_at(row, 0, p.tiles), true, p);
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

template <typename X, typename R, int V, int N, int kThreads, bool kFull = false>
bool stream_as(dw_backend *be, const Params &p, int T, dw_status *st) {
    auto kernel = k_norm_stream<X, R, V, N, kThreads, kFull>;
    const int G = kThreads / T;
    const size_t stage = StreamRows(p.c, sizeof(X), G, p.x_pitch == p.c, true).region +
                         StreamRows(p.c, sizeof(R), G, p.res_pitch == p.c, p.has_res).region +
                         StreamRows(p.c, sizeof(X), G, false, p.gate && p.gate_rows).region;
    const size_t weights = (size_t)T * N * V * 4 * 2;
    // Teams as registers and the ring allow, with two stages each where there is room: one
    // fills while the other's values go to registers.  More copies in flight only get in
    // each other's way (8192 x 4096 bf16, both norms, three teams: 1, 2, 3, 8 stages 47.5,
    // 44.4, 46.0, 46.8 us; two teams 52.4), and so does a third team where little is
    // computed: a whole row of 16-bit results from a residual and one norm (47.8 against
    // 43.3 us with two; to MXFP4 47.0 against 54.7, rows of 4000 44.4 against 51.1).
    const bool light = kFull && p.has_res && p.post == DW_NORM_NONE && p.pre != DW_NORM_LAYER && p.y_dtype != -2;
    constexpr int kTeams = stream_teams<R, V, N, kThreads>();
    const size_t room = kSmemBudget < weights ? 0 : kSmemBudget - weights, held = room / stage;
    if (!held) return false;
    const int teams = (int)std::min<size_t>(held, light ? std::min(kTeams, 2) : kTeams);
    const int stages = (int)std::min<size_t>(held / teams, kStreamStages);
    const size_t steps = (p.rows + G - 1) / (size_t)G;
    // With few steps nothing is there to fetch ahead (1000 x 1010 f32, 250 steps: 9.0 against
    // 6.8 us by a block a row; 296 x 4096 bf16 4.3 against 3.9, 400 rows 4.6 against 6.7).
    // Of longer rows an SM holds only one such block (148 x 5120 4.7 against 4.1 us, 200 rows
    // 4.9 against 7.0).
    const bool few = V == 8 && p.c > 4096 ? p.rows <= (size_t)be->sm_count : steps < (size_t)be->sm_count * 2;
    if (few) return false;
    static bool attr_set[16] = {};
    if (be->device < 16 && !attr_set[be->device]) {
        *st = dw_cuda_check(
            be, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBudget), "norm attributes");
        if (*st != DW_OK) return true;
        attr_set[be->device] = true;
    }
    const unsigned grid = (unsigned)std::min<size_t>(steps, (size_t)be->sm_count);
    *st = launch_dependent(be, "norm", kernel, grid, (kThreads + 32) * teams, teams * stages * stage + weights, 0, p, T, stages,
                           be->wait_cap_ns, be->dev_err);
    return true;
}

// Launches the streaming form with accesses of V elements; false where a row is too long
// or the rows too few for it.
template <typename X, typename R>
bool stream(dw_backend *be, const Params &p, int V, dw_status *st) {
    if (V == 8) {
        int T = 8;
        while ((size_t)T * (T < 32 ? 8 : 16) < p.c && T < 256) T *= 2;
        if ((size_t)T * 8 >= p.c) return stream_as<X, R, 8, 1, 256>(be, p, T, st);
        if ((size_t)T * 16 == p.c) return stream_as<X, R, 8, 2, 256, true>(be, p, T, st);
        if ((size_t)T * 16 >= p.c) return stream_as<X, R, 8, 2, 256>(be, p, T, st);
        // 4096 x 5120 and 4096 x 7168 bf16, both norms: 36.9 and 47.4 us, by rows of 512 threads 56.5
        // and 59.3; 4096 x 8192 51.8, by 256 threads of 32 elements 51.8 and with one norm 48.4 against 43.9
        if ((size_t)256 * 24 >= p.c) return stream_as<X, R, 8, 3, 256>(be, p, 256, st);
        if ((size_t)512 * 16 == p.c) return stream_as<X, R, 8, 2, 512, true>(be, p, 512, st);
        if ((size_t)256 * 32 >= p.c) {
            // two rows at once, where the ring has two stages of them (with f32 residuals it has one:
            // 4096 x 7168 f32 109 against 87 us; R alone decides, so that a norm of `out` has its split)
            if constexpr (sizeof(R) == 4) return stream_as<X, R, 8, 2, 512>(be, p, 512, st);
            return stream_as<X, R, 8, 4, 512>(be, p, 256, st);
        }
        // (2048 x 11008 f32 68.6 us, with the registers and weights of 32 elements a thread 94.8)
        if ((size_t)512 * 24 >= p.c) return stream_as<X, R, 8, 3, 512>(be, p, 512, st);
        return stream_as<X, R, 8, 4, 512>(be, p, 512, st);
    }
    // an MXFP4 block is 32 / V threads (here as above the same split for every y: the same sums)
    int T = 32 / V;
    while ((size_t)T * 16 < p.c && T < 256) T *= 2;
    if (V == 2) {
        if (p.c <= 64) return stream_as<X, R, 2, 2, 256>(be, p, T, st);
        if ((size_t)T * 16 >= p.c) return stream_as<X, R, 2, 8, 256>(be, p, T, st);
        if ((size_t)512 * 16 >= p.c) return stream_as<X, R, 2, 8, 512>(be, p, 512, st);
        return stream_as<X, R, 2, 16, 512>(be, p, 512, st);
    }
    if (p.c <= 128) return stream_as<X, R, 1, 4, 256>(be, p, T, st);
    if ((size_t)T * 16 >= p.c) return stream_as<X, R, 1, 16, 256>(be, p, T, st);
    if ((size_t)512 * 16 >= p.c) return stream_as<X, R, 1, 16, 512>(be, p, 512, st);
    return stream_as<X, R, 1, 32, 512>(be, p, 512, st);
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
        return launch_dependent(be, "norm (long rows)", k_norm_long<X, R>, (unsigned)p.rows, kMaxT, 0, 0, p);
    }
    dw_status st;
    const int V = fits(8) ? 8 : fits(2) ? 2 : 1;
    if (stream<X, R>(be, p, V, &st)) return st;
    // E: elements of a thread; T: threads of a row (a power of two from 32 to 512)
    int E = 8, T = 32;
    while ((size_t)T * E < p.c && T < kMaxT) T *= 2;
    while ((size_t)T * E < p.c) E *= 2;
    const int rows_blk = T == 32 ? 8 : 1;
    const size_t blocks = (p.rows + rows_blk - 1) / rows_blk;
    const dim3 block(T, rows_blk);
    auto go = [&](auto kernel) {
        return launch_dependent(be, "norm", kernel, (unsigned)blocks, block, 0, 0, p);
    };
    if (V == 8) {
        if (E == 8) return go(k_norm<X, R, 8, 1>);
        if (E == 16) return go(k_norm<X, R, 8, 2>);
        return go(k_norm<X, R, 8, 4>);
    }
    if (V == 2) {
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
    p.rows = d.rows, p.c = d.c, p.gate_rows = (uint32_t)std::min(d.gate_rows, d.rows);
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
