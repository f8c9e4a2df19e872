// attention.cu -- attention over the paged 8-bit cache for few query rows (single tokens,
// drafted tokens, any batch that has few rows for each sequence):
//   out = sum_j softmax_j(scale * q . k_j) v_j
// A block's keys are codes times 2^ek, its values codes times 2^ev.  With t_j = log2(e) scale
// q . k_j + ev_j and M = max t_j over the tokens so far,
//   w_j = 2^(t_j - M + 14),  out = sum_j w_j code_j / sum_j w_j 2^(-ev_j):
// the value scale rides in the exponent, so the products see codes alone, and 14 puts the
// largest w at 2^14, which leaves the small ones of a long softmax 38 binary places in f16.
// The 11 bits that a w keeps are the one rounding beyond f32 (codes and f16 queries are exact
// in f16; a bf16 query row is taken times a power of two that puts its largest value near 2^15).
//
// A warp owns 16 (or 32) rows, token by token the heads of a group that share a cache head, and
// goes through tiles of 32 tokens that its own TMA copies bring into its own ring of stages: no
// barrier but the copies' own before the end.  Codes become f16 in registers on the way into
// mma.sync (m16n8k16), in the layout that the copies' swizzle makes free of bank conflicts.  The
// warps of a CTA and the CTAs of a cluster share a sequence's tiles in turn and join their sums
// through shared memory, in a fixed order.  Bound by the cache's bytes.

#include <algorithm>
#include <type_traits>

#include "dw_attend.cuh"
#include "dw_launch.h"
#include "dw_mxfp4.cuh"
#include "dw_ptx.cuh"

namespace dw {
namespace {

constexpr int kTile = 32;  // tokens of a tile
constexpr int kWarps = 4;
constexpr int kStages = 2;
constexpr float kHead = 14.0f;  // exponent of the largest weight

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync_relaxed() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(const void *p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ float ld_peer(const float *p, uint32_t rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_peer4(const float *p, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(peer_addr(p, rank))
                 : "memory");
    return v;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Column c of eight, as a place among the eight rows (or pieces) that it reads: rows of two
// neighbouring columns lie four apart, which the copies' swizzle turns into other banks.
__device__ __forceinline__ int spread(int c) { return (c & 1) * 4 + (c >> 1); }

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kWarps * 32)
    k_attend_rows(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                  const __grid_constant__ AttendParams p, const __grid_constant__ KvCache c, const __grid_constant__ Seqs sq) {
    constexpr int R = 16 * MT, KS = D / 16, kBytes = kTile * D;  // rows, steps of a logit, bytes of a tile's keys
    constexpr int NT = D / 8, kPieces = D / 64;                  // column tiles of the output; 16-byte pieces of a lane's keys
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ uint64_t full[kWarps][kStages];
    __shared__ uint32_t scales[kWarps][kStages];
    __shared__ float part_m[kWarps][R], part_l[kWarps][R], all_m[R], all_l[R];
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, quad = lane & 3;
    uint8_t *const smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint8_t *const ring = smem + warp * kStages * 2 * kBytes;
    const uint32_t S = cluster_size(), rank = cluster_rank();
    if (lane == 0) {
        for (int i = 0; i < kStages; i++) mbar_init(smem_u32(&full[warp][i]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    pdl_wait();
    pdl_trigger();
    // which rows of which sequence, which head
    const uint32_t unit = blockIdx.x / S, item = unit / (uint32_t)c.heads;
    const int head = (int)(unit % (uint32_t)c.heads);
    int64_t place;
    uint32_t s;
    if (p.per_seq) {
        s = item / (uint32_t)p.per_seq, place = item % (uint32_t)p.per_seq;
    } else {
        s = seq_of_item(sq, item, p.group, R, 1, place);
    }
    const SeqRange r = seq_range(sq, s, c.page, p.err);
    const int rows_all = r.n * p.group, first = (int)min(place * R, (int64_t)0x7fffffff);
    if (place < 0 || first >= rows_all) return;
    const int rows = min(R, rows_all - first), token_a = first / p.group, token_b = (first + rows - 1) / p.group;
    const int lo = row_bounds(p, r, token_a).lo, hi = row_bounds(p, r, token_b).hi;
    // tokens that every row sees: tiles inside need no mask
    const int lo_all = row_bounds(p, r, token_b).lo, hi_all = row_bounds(p, r, token_a).hi;
    const int tile0 = lo / kTile, tiles = hi > lo ? (hi + kTile - 1) / kTile - tile0 : 0;
    const int step = (int)S * kWarps, gid = (int)rank * kWarps + warp;
    const int mine = tiles > gid ? (tiles - gid + step - 1) / step : 0;  // tiles of this warp

    // The pages of 32 of the warp's tiles and their scale bytes, a tile a lane (two pages where
    // they hold 16 tokens); those of the next 32 are loaded on the way, the pages and then the
    // scales, each well before it is used.
    const bool two = c.page < kTile;
    struct Pages {
        uint32_t page[2], scale[2];
    } now{}, next{};
    auto fetch_pages = [&](Pages &b, int base) {
        const int i = base + lane, t = (tile0 + gid + i * step) * kTile;
        if (i >= mine) return;
        b.page[0] = seq_page(sq, c, s, (uint32_t)t / (uint32_t)c.page, p.err);
        b.page[1] = two && t + 16 < r.len ? seq_page(sq, c, s, (uint32_t)(t + 16) / (uint32_t)c.page, p.err) : b.page[0];
    };
    auto fetch_scales = [&](Pages &b, int base) {
        if (base + lane >= mine) return;
#pragma unroll
        for (int h = 0; h < 2; h++) b.scale[h] = *reinterpret_cast<const uint16_t *>(c.s + kv_block(c, b.page[h], head) * 2);
    };
    const int box = two ? 16 : kTile;
    auto issue = [&](int i) {  // the copies of the warp's tile i, and its scales' place
        const int t = (tile0 + gid + i * step) * kTile, stage = i % kStages;
        if ((i & 31) == 0 && i) now = next;
        const uint32_t pg0 = __shfl_sync(0xffffffffu, now.page[0], i & 31), pg1 = __shfl_sync(0xffffffffu, now.page[1], i & 31);
        if (lane == 0) {
            const uint32_t bar = smem_u32(&full[warp][stage]), dst = smem_u32(ring + stage * 2 * kBytes);
            const bool second = two && t + 16 < r.len;
            mbar_expect_tx(bar, 2 * (second || !two ? kBytes : kBytes / 2));
            const int row0 = (int)(((size_t)pg0 * c.heads + head) * c.page) + t % c.page;
            tma_load_2d(dst, &tmap_k, bar, 0, row0);
            tma_load_2d(dst + kBytes, &tmap_v, bar, 0, row0);
            if (second) {
                const int row1 = (int)(((size_t)pg1 * c.heads + head) * c.page);
                tma_load_2d(dst + box * D, &tmap_k, bar, 0, row1);
                tma_load_2d(dst + kBytes + box * D, &tmap_v, bar, 0, row1);
            }
        }
        if (lane == (i & 31)) scales[warp][stage] = now.scale[0] | now.scale[1] << 16;
        if ((i & 31) == 8) fetch_pages(next, (i & ~31) + 32);
        if ((i & 31) == 20) fetch_scales(next, (i & ~31) + 32);
    };
    fetch_pages(now, 0);
    fetch_scales(now, 0);
    for (int i = 0; i < min(kStages, mine); i++) issue(i);

    // queries: step ks = 4 i + w of a logit takes the key values 16 (quad + 4 i) + 4 w .. + 3 of a lane
    uint32_t qf[MT][KS][4];
    float a_row[MT][2];  // what a logit of a row is multiplied by, but for its block's scale
    int my_lo[MT][2], my_hi[MT][2];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int row = m * 16 + h * 8 + g, at = first + row;
            const bool there = row < rows;
            const int token = there ? at / p.group : token_a;
            const Bounds b = row_bounds(p, r, token);
            my_lo[m][h] = b.lo, my_hi[m][h] = there ? b.hi : 0;
            const T *src = (const T *)p.q + (size_t)(r.row0 + token) * p.q_pitch + (size_t)(head * p.group + at % p.group) * D;
            float v[kPieces][16], top = 0.0f;
#pragma unroll
            for (int i = 0; i < kPieces; i++)
#pragma unroll
                for (int e = 0; e < 16; e += 8) {
                    Raw<T, 8> x;
                    x.zero();
                    const T *from = src + 16 * (quad + 4 * i) + e;
                    if (there && p.vec)
                        x.load(from);
                    else if (there) {
                        float u[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) u[j] = to_f32(from[j]);
                        x.set(u);
                    }
#pragma unroll
                    for (int j = 0; j < 8; j++) v[i][e + j] = x.get(j), top = fmaxf(top, fabsf(v[i][e + j]));
                }
            int e = 0;
            if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                e = query_exponent(top);
            }
            const float down = kv_pow2(-e);
            a_row[m][h] = p.scale_log2 * kv_pow2(e);
#pragma unroll
            for (int i = 0; i < kPieces; i++)
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    qf[m][4 * i + w][h] = pack2<__half>(v[i][4 * w] * down, v[i][4 * w + 1] * down);
                    qf[m][4 * i + w][2 + h] = pack2<__half>(v[i][4 * w + 2] * down, v[i][4 * w + 3] * down);
                }
        }

    float o[MT][NT][4], M[MT][2], L[MT][2];
#pragma unroll
    for (int m = 0; m < MT; m++) {
#pragma unroll
        for (int h = 0; h < 2; h++) M[m][h] = -INFINITY, L[m][h] = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[m][n][e] = 0.0f;
    }

    // Waits, with a limit, for the copies of the warp's tile i.
    auto landed = [&](int i) {
        const uint32_t bar = smem_u32(&full[warp][i % kStages]), parity = (uint32_t)(i / kStages) & 1;
        bool done = mbar_try_wait(bar, parity);
        if (__all_sync(0xffffffffu, done)) return true;
        const uint64_t t0 = globaltimer_ns();
        while (!__all_sync(0xffffffffu, done)) {
            if (!done) done = mbar_try_wait_sleep(bar, parity, 20000u);
            if (__any_sync(0xffffffffu, globaltimer_ns() - t0 > p.wait_cap_ns)) return false;
        }
        return true;
    };
    __syncwarp();
    for (int i = 0; i < mine; i++) {
        const int stage = i % kStages, t = (tile0 + gid + i * step) * kTile;
        if (!landed(i)) {
            if (lane == 0) record_error(p.err, DW_DEV_WAIT_EXPIRED, 51, i);
            for (int j = i; j < min(i + kStages, mine); j++) landed(j);  // nothing more is issued
            break;
        }
        const uint8_t *ks = ring + stage * 2 * kBytes, *vs = ks + kBytes;
        const uint32_t sc = scales[warp][stage];  // of the tile's (up to two) blocks
        // ---- logits
        float x[MT][4][4];
#pragma unroll
        for (int n = 0; n < 4; n++) {
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int e = 0; e < 4; e++) x[m][n][e] = 0.0f;
            const int row = 8 * n + spread(g);
#pragma unroll
            for (int j = 0; j < kPieces; j++) {
                const int piece = D == 128 ? (quad + 4 * j) ^ (row & 7) : quad ^ ((row >> 1) & 3);
                const uint4 k = *reinterpret_cast<const uint4 *>(ks + row * D + piece * 16);
                const uint32_t kw[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const uint32_t b0 = e4m3_to_f16x2((uint16_t)kw[w]), b1 = e4m3_to_f16x2((uint16_t)(kw[w] >> 16));
#pragma unroll
                    for (int m = 0; m < MT; m++) mma_f16(x[m][n], qf[m][4 * j + w], b0, b1);
                }
            }
        }
        // ---- weights
        const int ve[2] = {kv_exponent(sc >> 8 & 255), kv_exponent(sc >> 24)};
        const float ka[2] = {kv_pow2(kv_exponent(sc & 255)), kv_pow2(kv_exponent(sc >> 16 & 255))};
        const bool masked = t < lo_all || t + kTile > hi_all;
        uint32_t pf[MT][4][2];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const float a = a_row[m][h] * ka[n / 2], b = (float)ve[n / 2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float &v = x[m][n][2 * h + e];
                        v = fmaf(v, a, b);
                        if (masked) {
                            const int at = t + 8 * n + quad + 4 * e;  // columns 2 quad, 2 quad + 1
                            if (at < my_lo[m][h] || at >= my_hi[m][h]) v = -INFINITY;
                        }
                        top = fmaxf(top, v);
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float now_m = fmaxf(M[m][h], top);
                if (now_m != M[m][h]) {
                    const float f = carry(M[m][h], now_m);
                    M[m][h] = now_m;
                    L[m][h] *= f;
#pragma unroll
                    for (int n = 0; n < NT; n++) o[m][n][2 * h] *= f, o[m][n][2 * h + 1] *= f;
                }
                const float base = (now_m == -INFINITY ? 0.0f : -now_m) + kHead;
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    float sum = 0.0f;
#pragma unroll
                    for (int n = 2 * b; n < 2 * b + 2; n++) {
                        const float w0 = ex2_approx(x[m][n][2 * h] + base), w1 = ex2_approx(x[m][n][2 * h + 1] + base);
                        sum += w0 + w1;
                        pf[m][n][h] = pack2<__half>(w0, w1);
                    }
                    L[m][h] = fmaf(sum, kv_pow2(-ve[b]), L[m][h]);
                }
            }
        // ---- values
        const bool tail = t + kTile > r.len;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            uint32_t v[4][D / 32];  // rows quad, quad + 4, quad + 8, quad + 12 of 16: the lane's D / 8 values
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int row = 16 * j + 4 * e + quad;
                if constexpr (D == 128) {
                    const uint4 u = *reinterpret_cast<const uint4 *>(vs + row * D + (spread(g) ^ (row & 7)) * 16);
                    v[e][0] = u.x, v[e][1] = u.y, v[e][2] = u.z, v[e][3] = u.w;
                } else {
                    const int piece = (2 * ((g >> 1) & 1) + (g >> 2)) ^ ((row >> 1) & 3);
                    const uint2 u = *reinterpret_cast<const uint2 *>(vs + row * D + piece * 16 + (g & 1) * 8);
                    v[e][0] = u.x, v[e][1] = u.y;
                }
                if (tail && t + row >= r.len) {  // no token: whatever the page holds there
#pragma unroll
                    for (int w = 0; w < D / 32; w++) v[e][w] = 0;
                }
            }
#pragma unroll
            for (int w = 0; w < D / 32; w++) {
                const uint32_t b[2][2] = {{__byte_perm(v[0][w], v[1][w], 0x5140), __byte_perm(v[0][w], v[1][w], 0x7362)},
                                          {__byte_perm(v[2][w], v[3][w], 0x5140), __byte_perm(v[2][w], v[3][w], 0x7362)}};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t b0 = e4m3_to_f16x2((uint16_t)(b[0][e / 2] >> (16 * (e % 2))));
                    const uint32_t b1 = e4m3_to_f16x2((uint16_t)(b[1][e / 2] >> (16 * (e % 2))));
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        const uint32_t a[4] = {pf[m][2 * j][0], pf[m][2 * j][1], pf[m][2 * j + 1][0], pf[m][2 * j + 1][1]};
                        mma_f16(o[m][4 * w + e], a, b0, b1);
                    }
                }
            }
        }
        __syncwarp();  // the stage has been read
        if (i + kStages < mine) issue(i + kStages);
    }

    // ---- join: the warps' sums, then those of the cluster's CTAs.  A warp leaves its sums in its
    // ring (its copies have all landed).
    float *const part = reinterpret_cast<float *>(ring);  // [R][D]
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float l = L[m][h];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            const int row = m * 16 + h * 8 + g;
            if (quad == 0) part_m[warp][row] = M[m][h], part_l[warp][row] = l;
            // column 2 quad + e of output tile n is value n of the lane's piece
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int col = 2 * quad + e;
                const int at = D == 128 ? spread(col) * 16 : (2 * ((col >> 1) & 1) + (col >> 2)) * 16 + (col & 1) * 8;
#pragma unroll
                for (int n = 0; n < NT; n += 4)
                    *reinterpret_cast<float4 *>(part + row * D + at + n) =
                        make_float4(o[m][n][2 * h + e], o[m][n + 1][2 * h + e], o[m][n + 2][2 * h + e], o[m][n + 3][2 * h + e]);
            }
        }
    __syncthreads();
    constexpr int kQuads = D / 4;
    auto store = [&](int row, int at, float4 v, float l) {
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
        const int token = (first + row) / p.group, h = head * p.group + (first + row) % p.group;
        T *dst = (T *)p.out + (size_t)(r.row0 + token) * p.out_pitch + (size_t)h * D + at;
        const float y[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
        if (p.vec) {
            Raw<T, 4> x;
            x.set(y);
            x.store(dst);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) dst[i] = from_f32<T>(y[i]);
        }
    };
    float *const part0 = reinterpret_cast<float *>(smem);
    constexpr int kRing = kStages * 2 * kBytes / 4;  // floats of a warp's ring
    for (int i = threadIdx.x; i < rows * kQuads; i += kWarps * 32) {
        const int row = i / kQuads, at = i % kQuads * 4;
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) m = fmaxf(m, part_m[w][row]);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float f = carry(part_m[w][row], m);
            const float4 u = *reinterpret_cast<const float4 *>(part0 + w * kRing + row * D + at);
            l = fmaf(part_l[w][row], f, l);
            v.x = fmaf(u.x, f, v.x), v.y = fmaf(u.y, f, v.y), v.z = fmaf(u.z, f, v.z), v.w = fmaf(u.w, f, v.w);
        }
        if (S == 1) {
            store(row, at, v, l);
        } else {
            *reinterpret_cast<float4 *>(part0 + row * D + at) = v;
            if (at == 0) all_m[row] = m, all_l[row] = l;
        }
    }
    if (S == 1) return;
    cluster_sync();
    for (int i = (int)rank * kWarps * 32 + threadIdx.x; i < rows * kQuads; i += (int)S * kWarps * 32) {
        const int row = i / kQuads, at = i % kQuads * 4;
        float m = -INFINITY, l = 0.0f;
        for (uint32_t k = 0; k < S; k++) m = fmaxf(m, ld_peer(all_m + row, k));
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t k = 0; k < S; k++) {
            const float f = carry(ld_peer(all_m + row, k), m);
            const float4 u = ld_peer4(part0 + row * D + at, k);
            l = fmaf(ld_peer(all_l + row, k), f, l);
            v.x = fmaf(u.x, f, v.x), v.y = fmaf(u.y, f, v.y), v.z = fmaf(u.z, f, v.z), v.w = fmaf(u.w, f, v.w);
        }
        store(row, at, v, l);
    }
    cluster_sync_relaxed();  // no CTA leaves while its sums may be read
}

// Codes as a 2-D byte tensor [tokens of all pages and heads][d]; a box is `rows` tokens.
bool code_map(dw_backend *be, CUtensorMap *map, const uint8_t *codes, const KvCache &c, int rows) {
    cuuint64_t dims[2] = {(cuuint64_t)c.d, (cuuint64_t)c.pages * c.heads * c.page};
    cuuint64_t strides[1] = {(cuuint64_t)c.d};
    cuuint32_t box[2] = {(cuuint32_t)c.d, (cuuint32_t)rows};
    cuuint32_t estr[2] = {1, 1};
    return be->encode_tiled && be->encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(codes), dims, strides, box,
                                                estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                                c.d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
dw_status attend_rows(dw_backend *be, AttendParams p, const KvCache &c, const Seqs &s) {
    constexpr int R = 16;
    auto kernel = k_attend_rows<T, D, 1>;
    constexpr size_t smem = 1024 + (size_t)kWarps * kStages * 2 * kTile * D;
    const size_t n = s.tokens / s.seqs;
    p.per_seq = s.starts ? 0 : (int)((n * p.group + R - 1) / R);
    const size_t items = s.starts ? seq_items(s.tokens, s.seqs, p.group, R, 1) : (size_t)p.per_seq * s.seqs, units = items * c.heads;
    p.items = (uint32_t)items;
    // CTAs that share a block's tiles: as many as the GPU holds at once, each with a tile a warp at least
    const size_t most = ((size_t)s.width * c.page + kTile - 1) / kTile;
    unsigned S = 1;
    while (S < 8 && units * 2 * S <= (size_t)be->sm_count * 2 && (size_t)2 * S * kWarps <= most) S *= 2;
    if (units * S > 0x7fffffffu) return dw_fail(be, DW_ERR_UNSUPPORTED, "attention_kv8: too many rows");
    CUtensorMap tk, tv;
    const int box = std::min(c.page, kTile);
    if (!code_map(be, &tk, c.k, c, box) || !code_map(be, &tv, c.v, c, box))
        return dw_fail(be, DW_ERR_DEVICE, "attention_kv8: tensor map rejected");
    static bool attr_set[16] = {};
    if (be->device < 16 && !attr_set[be->device]) {
        dw_status st = dw_cuda_check(be, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                                     "attention_kv8 attributes");
        if (st != DW_OK) return st;
        attr_set[be->device] = true;
    }
    return launch_dependent(be, "attention_kv8", kernel, (unsigned)(units * S), kWarps * 32, smem, S, tk, tv, p, c, s);
}

}  // namespace

dw_status launch_attention_kv8(dw_backend *be, const dw_attention_desc &d, const KvCache &c, const Seqs &s, const HeadRows &q,
                               const HeadRows &out) {
    AttendParams p{};
    p.q = q.ptr, p.out = out.ptr, p.q_pitch = q.pitch, p.out_pitch = out.pitch;
    p.group = d.q_heads / c.heads;
    p.scale_log2 = d.scale * 1.44269504088896340736f;
    p.causal = d.causal, p.window = d.causal ? d.window : 0;
    auto fits = [](const HeadRows &h) { return (uintptr_t)h.ptr % 16 == 0 && h.pitch % 8 == 0; };
    p.vec = fits(q) && fits(out);
    p.wait_cap_ns = be->wait_cap_ns, p.err = be->dev_err;
    auto with = [&](auto t) {
        using T = decltype(t);
        if (s.tokens / s.seqs * p.group > 64) return c.d == 64 ? attend_prompt<T, 64>(be, p, c, s) : attend_prompt<T, 128>(be, p, c, s);
        return c.d == 64 ? attend_rows<T, 64>(be, p, c, s) : attend_rows<T, 128>(be, p, c, s);
    };
    return d.dtype == DW_F16 ? with(__half{}) : with(__nv_bfloat16{});
}

}  // namespace dw
