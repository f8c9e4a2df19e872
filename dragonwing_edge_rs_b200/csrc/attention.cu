// attention.cu -- attention over the paged 8-bit cache for few query rows (single tokens,
// drafted tokens, any batch that has few rows for each sequence):
//   out = sum_j softmax_j(scale * q . k_j) v_j
// A block's keys are codes times 2^ek, its values codes times 2^ev.  With t_j = log2(e) scale
// q . k_j + ev_j and M = max t_j over the tokens so far,
//   w_j = 2^(t_j - M + 11),  out = sum_j w_j code_j / sum_j w_j 2^(-ev_j):
// the value scale rides in the exponent, so the products see codes alone.  M lags: it moves, to
// a whole number, where a row's true maximum is more than 2^4 above, so the largest w stays
// below 2^15, inside f16, and the smallest keep 31 binary places and more below it.
// The 11 bits that a w is cut to, in both sums, are the one loss beyond f32 (codes and f16 queries are exact
// in f16; a bf16 query row is taken times a power of two that puts its largest value near 2^15).
//
// A warp owns 8 NT rows, token by token the heads of a group that share a cache head, and
// goes through tiles of 32 tokens that its own asynchronous copies bring into its own ring of
// stages: no barrier before the end (a TMA copy of a tile and its barrier took a warp 600 of
// 2200 cycles to issue; 16 copies of 16 bytes a lane take 100).  Codes become f16 in registers on the way into
// mma.sync (m16n8k16).  Tokens, and then values, take the 16-row side and the rows the 8-column
// side (S^T = K Q^T, O^T = V^T P^T): with rows on the 16 side a group of four wasted three
// quarters of the products.  The copies swizzle the rows, so that all reads are free of bank conflicts.  The
// warps of a CTA and the CTAs of a cluster share a sequence's tiles in turn and join their sums
// through shared memory, in a fixed order.  Bound by the cache's bytes where these are many (one token of
// each of 64 sequences of up to 8192, 539 MB, in 95 us: 5670 GB/s), by the longest sequence and a fixed
// 8 us where they are few (one token over 4000: 8.4 us).

#include <algorithm>
#include <type_traits>

#include "dw_attend.cuh"
#include "dw_launch.h"
#include "dw_mxfp4.cuh"
#include "dw_ptx.cuh"

namespace dw {
namespace {

constexpr int kTile = 32;  // tokens of a tile
constexpr int kStages = 2;
constexpr float kHead = 11.0f, kLag = 4.0f;

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Column c of eight, as a place among the eight rows (or pieces) that it reads: rows of two
// neighbouring columns lie four apart, which the rows' swizzle turns into other banks.
__device__ __forceinline__ int spread(int c) { return (c & 1) * 4 + (c >> 1); }

// 8 x 8 f16 of a warp, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <typename T, int D, int NT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kWarps == 8 ? 1 : NT == 1 ? 3 : 2)
    k_attend_rows(const __grid_constant__ AttendParams p, const __grid_constant__ KvCache c, const __grid_constant__ Seqs sq) {
    constexpr int R = 8 * NT, KS = D / 16, kBytes = kTile * D;  // rows, steps of a logit, bytes of a tile's keys
    constexpr int VT = D / 16, kPieces = D / 64;                // row tiles of the output; 16-byte pieces of a lane's keys
    constexpr int kRing = kStages * 2 * kBytes;
    static_assert(R * D * 4 <= kRing, "a warp's sums lie over its ring");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ uint32_t scales[kWarps][kStages];
    __shared__ float part_m[kWarps][R], part_l[kWarps][R], all_m[R], all_l[R];
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, quad = lane & 3;
    uint8_t *const ring = smem_raw + warp * kRing;
    const uint32_t S = cluster_size(), rank = cluster_rank();
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
        if (head == 0 && warp == 0 && bad_start(sq, (int64_t)item * 32 + lane)) record_error(p.err, DW_DEV_BAD_ARG, 61, (int)s);
    }
    // (without a window the first tiles' pages are looked up before the length is known)
    const bool two = c.page < kTile;
    constexpr uint32_t kGone = ~0u;
    const int shift = 31 - __clz(c.page);  // pages hold a power of two of tokens
    const int step = (int)S * kWarps, gid = (int)rank * kWarps + warp;
    uint32_t guess[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t index = (uint32_t)((gid + lane * step) * kTile + 16 * h) >> shift;
        guess[h] = !p.window && index < sq.width ? (uint32_t)sq.table[(size_t)s * sq.width + index] : 0u;
    }
    int row0;
    const int rows_all = seq_rows(sq, s, row0, p.err) * p.group, first = (int)min(place * R, (int64_t)0x7fffffff);
    if (place < 0 || first >= rows_all) return;
    const int rows = min(R, rows_all - first);
    // the query rows: a lane has the values 16 (quad + 4 j) .. + 15 of row g of eight
    Raw<T, 8> qx[NT][2 * kPieces];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int at = first + min(n * 8 + g, rows - 1);
        const T *src = (const T *)p.q + (size_t)(row0 + at / p.group) * p.q_pitch + (size_t)(head * p.group + at % p.group) * D;
        if (p.vec) {
#pragma unroll
            for (int j = 0; j < 2 * kPieces; j++) qx[n][j].load(src + 16 * (quad + 4 * (j / 2)) + 8 * (j & 1));
        } else {
#pragma unroll
            for (int j = 0; j < 2 * kPieces; j++) {
                float u[8];
#pragma unroll
                for (int e = 0; e < 8; e++) u[e] = to_f32(src[16 * (quad + 4 * (j / 2)) + 8 * (j & 1) + e]);
                qx[n][j].set(u);
            }
        }
    }
    const SeqRange r = seq_range(sq, s, c.page, p.err, -1);
    const int token_a = first / p.group, token_b = (first + rows - 1) / p.group;
    const int lo = row_bounds(p, r, token_a).lo, hi = row_bounds(p, r, token_b).hi;
    // tokens that every row sees: tiles inside need no mask
    const int lo_all = row_bounds(p, r, token_b).lo, hi_all = row_bounds(p, r, token_a).hi;
    const int tile0 = lo / kTile, tiles = hi > lo ? (hi + kTile - 1) / kTile - tile0 : 0;
    const int mine = tiles > gid ? (tiles - gid + step - 1) / step : 0;  // tiles of this warp

    // Where 32 of the warp's tiles lie (a tile a lane, two pages where they hold 16 tokens) and
    // their scale bytes; those of the next 32 are loaded on the way, the pages and then the
    // scales, each well before it is used.
    struct Pages {
        uint32_t page[2];
        uint32_t row[2];  // of the codes, where 16 tokens begin
        uint32_t scale;
    } now{}, next{};
    auto places = [&](Pages &b, int t) {
#pragma unroll
        for (int h = 0; h < 2; h++)
            b.row[h] = ((b.page[h] * (uint32_t)c.heads + (uint32_t)head) << shift) + (uint32_t)((t + 16 * h) & (c.page - 1));
    };
    auto fetch_pages = [&](Pages &b, int base) {
        const int i = base + lane, t = (tile0 + gid + i * step) * kTile;
        if (i >= mine) return;
        // (a page whose tokens lie before the window may have been given away: zeros in its place)
        const bool gone = two && t + 16 <= lo;
        b.page[0] = seq_page(sq, c, s, (uint32_t)(gone ? t + 16 : t) >> shift, p.err);
        b.page[1] = two && !gone && t + 16 < r.len ? seq_page(sq, c, s, (uint32_t)(t + 16) >> shift, p.err) : b.page[0];
        places(b, t);
        if (gone) b.row[0] = kGone;
    };
    auto fetch_scales = [&](Pages &b, int base) {
        if (base + lane >= mine) return;
        const uint16_t *from = reinterpret_cast<const uint16_t *>(c.s);
        b.scale = from[kv_block(c, b.page[0], head)] | (uint32_t)from[kv_block(c, b.page[1], head)] << 16;
    };
    // The copies of the warp's tile i (nothing behind the last: every turn makes a group), and its
    // scales' place.  Lane l of copy k has piece l % kLine of row kLines k + l / kLine; a piece lies
    // where its place in the 128-byte line, xor the line modulo 8 (of 64-byte rows: the pair of rows
    // modulo 4), says.
    constexpr int kLine = D / 16, kLines = 32 / kLine;  // 16-byte pieces of a row, rows of a copy
    const int c_row = lane / kLine, c_piece = lane % kLine;
    uint32_t c_to[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int row = k * kLines + c_row;
        c_to[k] = smem_u32(ring) + row * D + (D == 128 ? c_piece ^ (row & 7) : c_piece ^ ((row >> 1) & 3)) * 16;
    }
    auto issue = [&](int i) {
        if (i < mine) {
            const uint32_t stage = (uint32_t)(i % kStages) * 2 * kBytes;
            if ((i & 31) == 0 && i) now = next;
            const uint32_t at0 = __shfl_sync(0xffffffffu, now.row[0], i & 31), at1 = __shfl_sync(0xffffffffu, now.row[1], i & 31);
            const size_t from[2] = {(size_t)(at0 == kGone ? at1 : at0) * D + lane * 16, (size_t)at1 * D + lane * 16};
            const uint32_t bytes[2] = {at0 == kGone ? 0u : 16u, 16u};  // read; the rest of 16 is zeros
#pragma unroll
            for (int k = 0; k < kTile / kLines; k++) {
                constexpr int kHalfCopies = kTile / kLines / 2;
                const size_t at = from[k / kHalfCopies] + (k % kHalfCopies) * 512;
                const uint32_t to = c_to[k & 1] + stage + (k & ~1) * 512;
                const uint32_t n = bytes[k / kHalfCopies];
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(c.k + at), "r"(n) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + kBytes), "l"(c.v + at), "r"(n) : "memory");
            }
            if (lane == (i & 31)) scales[warp][i % kStages] = now.scale;
            if ((i & 31) == 8) fetch_pages(next, (i & ~31) + 32);
            if ((i & 31) == 20) fetch_scales(next, (i & ~31) + 32);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (p.window) {
        fetch_pages(now, 0);
    } else if (lane < mine) {
        const int t = (gid + lane * step) * kTile;
        const bool second = two && t + 16 < r.len;
        if (guess[0] >= c.pages || (second && guess[1] >= c.pages)) record_error(p.err, DW_DEV_BAD_ARG, 62, (int)s);
        now.page[0] = min(guess[0], c.pages - 1), now.page[1] = second ? min(guess[1], c.pages - 1) : now.page[0];
        places(now, t);
    }
    fetch_scales(now, 0);
    for (int i = 0; i < kStages; i++) issue(i);

    // queries: step ks = 4 j + w of a logit takes the values 16 (quad + 4 j) + 4 w .. + 3 of a lane
    uint32_t qf[NT][KS][2];
    float a_row[NT][2];  // of rows 2 quad and 2 quad + 1: what a logit is multiplied by, but for its block's scale
    int my_lo[NT][2], my_hi[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const Raw<T, 8>(&x)[2 * kPieces] = qx[n];
        float a = p.scale_log2, down = 1.0f;
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < 2 * kPieces; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[j].get(e)));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = query_exponent(top);
            down = kv_pow2(-e), a *= kv_pow2(e);
        }
#pragma unroll
        for (int j = 0; j < 2 * kPieces; j++)
#pragma unroll
            for (int w = 0; w < 2; w++) {
                qf[n][2 * j + w][0] = pack2<__half>(x[j].get(4 * w) * down, x[j].get(4 * w + 1) * down);
                qf[n][2 * j + w][1] = pack2<__half>(x[j].get(4 * w + 2) * down, x[j].get(4 * w + 3) * down);
            }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int mine_row = n * 8 + 2 * quad + h;
            const Bounds b = row_bounds(p, r, (first + min(mine_row, rows - 1)) / p.group);
            my_lo[n][h] = b.lo, my_hi[n][h] = mine_row < rows ? b.hi : 0;
            a_row[n][h] = __shfl_sync(0xffffffffu, a, 4 * (2 * quad + h));
        }
    }

    float o[NT][VT][4], M[NT][2], L[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int h = 0; h < 2; h++) M[n][h] = -INFINITY, L[n][h] = 0.0f;
#pragma unroll
        for (int v = 0; v < VT; v++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[n][v][e] = 0.0f;
    }

    for (int i = 0; i < mine; i++) {
        const int stage = i % kStages, t = (tile0 + gid + i * step) * kTile;
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();  // every lane's copies of the tile are there
        const uint8_t *ks = ring + stage * 2 * kBytes, *vs = ks + kBytes;
        const uint32_t sc = scales[warp][stage];  // of the tile's (up to two) blocks
        // ---- logits: 16 tokens a row tile, row c of eight the token spread(c)
        float x[NT][2][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int e = 0; e < 4; e++) x[n][m][e] = 0.0f;
#pragma unroll
        for (int j = 0; j < kPieces; j++) {
            uint32_t kw[4][4];
#pragma unroll
            for (int b = 0; b < 4; b++) {  // eight tokens
                const int row = 8 * b + spread(g);
                const int piece = D == 128 ? (quad + 4 * j) ^ (row & 7) : quad ^ ((row >> 1) & 3);
                const uint4 k = *reinterpret_cast<const uint4 *>(ks + row * D + piece * 16);
                kw[b][0] = k.x, kw[b][1] = k.y, kw[b][2] = k.z, kw[b][3] = k.w;
            }
#pragma unroll
            for (int w = 0; w < 4; w++)
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    const uint32_t a[4] = {e4m3_to_f16x2((uint16_t)kw[2 * m][w]), e4m3_to_f16x2((uint16_t)kw[2 * m + 1][w]),
                                           e4m3_to_f16x2((uint16_t)(kw[2 * m][w] >> 16)), e4m3_to_f16x2((uint16_t)(kw[2 * m + 1][w] >> 16))};
#pragma unroll
                    for (int n = 0; n < NT; n++) mma_f16(x[n][m], a, qf[n][4 * j + w][0], qf[n][4 * j + w][1]);
                }
        }
        // ---- weights
        const int ve[2] = {kv_exponent(sc >> 8 & 255), kv_exponent(sc >> 24)};
        const float ka[2] = {kv_pow2(kv_exponent(sc & 255)), kv_pow2(kv_exponent(sc >> 16 & 255))};
        const bool masked = t < lo_all || t + kTile > hi_all;
        uint32_t pf[NT][4];  // f16 weights of eight tokens (values of a row together)
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float top[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                top[h] = -INFINITY;
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    float &v = x[n][b / 2][2 * (b & 1) + h];
                    v = fmaf(v, a_row[n][h] * ka[b / 2], (float)ve[b / 2]);
                    if (masked) {
                        const int at = t + 8 * b + spread(g);
                        if (at < my_lo[n][h] || at >= my_hi[n][h]) v = -INFINITY;
                    }
                    top[h] = fmaxf(top[h], v);
                }
            }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1)
#pragma unroll
                for (int h = 0; h < 2; h++) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], d));
            if (__any_sync(0xffffffffu, top[0] > M[n][0] + kLag || top[1] > M[n][1] + kLag)) {
                // M moves, to a whole number: what is scaled stays exact
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float to = top[h] > M[n][h] + kLag ? ceilf(top[h]) : M[n][h], f = carry(M[n][h], to);
                    M[n][h] = to;
                    L[n][h] *= f;
#pragma unroll
                    for (int v = 0; v < VT; v++) o[n][v][h] *= f, o[n][v][2 + h] *= f;
                }
            }
            float base[2];
#pragma unroll
            for (int h = 0; h < 2; h++) base[h] = (M[n][h] == -INFINITY ? 0.0f : -M[n][h]) + kHead;
            float2 sum[2] = {};
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const float2 w = eleven_bits(ex2_approx(x[n][b / 2][2 * (b & 1)] + base[0]), ex2_approx(x[n][b / 2][2 * (b & 1) + 1] + base[1]));
                sum[b / 2] = __fadd2_rn(sum[b / 2], w);
                pf[n][b] = transposed(pack2<__half>(w.x, w.y));
            }
            L[n][0] = fmaf(sum[0].x, kv_pow2(-ve[0]), fmaf(sum[1].x, kv_pow2(-ve[1]), L[n][0]));
            L[n][1] = fmaf(sum[0].y, kv_pow2(-ve[0]), fmaf(sum[1].y, kv_pow2(-ve[1]), L[n][1]));
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
            for (int w = 0; w < D / 32; w++)
#pragma unroll
                for (int e = 0; e < 2; e++) {  // the lane's values 4 w + 2 e and the next, of two tokens each
                    const uint32_t b0 = __byte_perm(v[0][w], v[1][w], e ? 0x7362 : 0x5140);
                    const uint32_t b1 = __byte_perm(v[2][w], v[3][w], e ? 0x7362 : 0x5140);
                    const uint32_t a[4] = {e4m3_to_f16x2((uint16_t)b0), e4m3_to_f16x2((uint16_t)(b0 >> 16)), e4m3_to_f16x2((uint16_t)b1),
                                           e4m3_to_f16x2((uint16_t)(b1 >> 16))};
#pragma unroll
                    for (int n = 0; n < NT; n++) mma_f16(o[n][2 * w + e], a, pf[n][2 * j], pf[n][2 * j + 1]);
                }
        }
        __syncwarp();  // the stage has been read
        issue(i + kStages);
    }

    // ---- join: the warps' sums, then those of the cluster's CTAs.  A warp leaves its sums in its
    // ring (its copies have all landed).
    float *const part = reinterpret_cast<float *>(ring);  // [R][D]
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float l = L[n][h];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
            const int row = n * 8 + 2 * quad + h;
            if (g == 0) part_m[warp][row] = M[n][h], part_l[warp][row] = l;
            const int at = D == 128 ? spread(g) * 16 : (2 * ((g >> 1) & 1) + (g >> 2)) * 16 + (g & 1) * 8;
#pragma unroll
            for (int v = 0; v < VT; v += 2)
                *reinterpret_cast<float4 *>(part + row * D + at + 2 * v) =
                    make_float4(o[n][v][h], o[n][v][2 + h], o[n][v + 1][h], o[n][v + 1][2 + h]);
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
    float *const part0 = reinterpret_cast<float *>(smem_raw);
    for (int i = threadIdx.x; i < rows * kQuads; i += kWarps * 32) {
        const int row = i / kQuads, at = i % kQuads * 4;
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) m = fmaxf(m, part_m[w][row]);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float f = carry(part_m[w][row], m);
            const float4 u = *reinterpret_cast<const float4 *>(part0 + w * (kRing / 4) + row * D + at);
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
        float l;
        const float4 v = join_sums(all_m + row, all_l + row, part0 + row * D + at, S, l);
        store(row, at, v, l);
    }
    cluster_sync_relaxed();  // no CTA leaves while its sums may be read
}

template <typename T, int D, int NT, int kWarps>
dw_status launch_rows(dw_backend *be, const AttendParams &p, const KvCache &c, const Seqs &s, size_t units, unsigned S) {
    auto kernel = k_attend_rows<T, D, NT, kWarps>;
    constexpr size_t smem = (size_t)kWarps * kStages * 2 * kTile * D;
    static bool attr_set[16] = {};
    if (be->device < 16 && !attr_set[be->device]) {
        dw_status st = dw_cuda_check(be, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                                     "attention_kv8 attributes");
        if (st != DW_OK) return st;
        attr_set[be->device] = true;
    }
    return launch_dependent(be, "attention_kv8", kernel, (unsigned)(units * S), kWarps * 32, smem, S, p, c, s);
}

template <typename T, int D, int NT>
dw_status attend_rows(dw_backend *be, AttendParams p, const KvCache &c, const Seqs &s) {
    constexpr int R = 8 * NT;
    const size_t n = s.tokens / s.seqs, sms = (size_t)be->sm_count;
    p.per_seq = s.starts ? 0 : (int)seq_items_each(n, p.group, R, 1);
    const size_t items = s.starts ? seq_items(s.tokens, s.seqs, p.group, R, 1) : (size_t)p.per_seq * s.seqs, units = items * c.heads;
    if (units * kMaxShare > 0x7fffffffu) return dw_fail(be, DW_ERR_UNSUPPORTED, "attention_kv8: too many rows");
    p.items = (uint32_t)items;
    // S CTAs share a unit's tiles (`most`: as many as the longest sequence can have).  While an SM for each unit is
    // there: CTAs of eight warps, as many as SMs, each with a tile a warp at least (one row, 8 heads: over 8000
    // tokens S = 1, 2, 4, 8 38, 23, 15, 11 us; 8 sequences of 4000 22, 16.6, 23, 39, by four warps 28, 19, 20,
    // 25; 16 sequences 25, 32, 42, 70, by four warps 30, 32, 37, 38).
    // With few rows the same up to two units an SM (32 sequences of up to 2000 22.4, of 2000 29.9; by four warps
    // 26.3 and 30.5, two sharing 21.9 and 35.9); with more they fall behind (32 sequences of 2000, 16 rows each 37,
    // by four warps 31).
    // More units: CTAs of four warps, several an SM.  With few rows they share too, for the balance of long and
    // short sequences, while a warp keeps twelve tiles of the longest (64 sequences of up to 8192: 106, 95, 94, 126
    // us, by eight warps 98, 107, 153, 270).
    const size_t most = ((size_t)s.width * c.page + kTile - 1) / kTile;
    unsigned S = 1;
    if (units <= (NT == 1 ? 2 : 1) * sms) {
        while (S < kMaxShare && units * 2 * S <= sms && (size_t)2 * S * 8 <= most) S *= 2;
        return launch_rows<T, D, NT, 8>(be, p, c, s, units, S);
    }
    while (NT == 1 && S < kMaxShare && units * 2 * S <= 15 * sms && 2 * S * 4 * 12 <= most) S *= 2;
    return launch_rows<T, D, NT, 4>(be, p, c, s, units, S);
}

template <typename T, int D>
dw_status attend(dw_backend *be, const AttendParams &p, const KvCache &c, const Seqs &s) {
    const size_t rows = (s.tokens + s.seqs - 1) / s.seqs * p.group;  // of a sequence, on average
    // Up to 24 rows a warp has them all.  With more the cache would be read again for every 24; the
    // kernel of many rows has 256 in a CTA, at the price of one CTA an SM and a longer start, and of
    // the products of 128 rows, however few there are (8 heads, us, this one's first: 20 rows of 16
    // sequences of up to 4000 tokens 40 and 75; 24 rows over 8000 tokens 19 and 22; 32 rows 35 and 22;
    // 64 rows of 16 sequences of 1000 42 and 26; 256 rows over 8000 72 and 33).  Between 24 and 48 it
    // gains only where CTAs are few and share the tokens (40 rows of 16 sequences of 4000 72 and
    // 83; 48 rows of 64 of 1000 87 and 92, of one of 8000 36 and 22).
    if (rows > 48 || (rows > 24 && s.seqs * c.heads * 2 <= (size_t)be->sm_count)) return attend_prompt<T, D>(be, p, c, s);
    // (The average: a call's starts are known on the device alone.  Sequences of very different rows
    // lose by it: 1024 rows behind 3000 tokens beside 63 single tokens 375 us, in calls of their own 85 and
    // 95; a prompt of 512 beside 255 single tokens 161, of their own 20 and 90.)
    // (fewer rows than it has places cost a warp products and registers: one row of 64 sequences of up
    // to 8192 tokens 94 us by 8 places, 129 by 16, 182 by 24; 8 rows over 8000 tokens 11.1, 13.9, 18.2)
    if (rows <= 8) return attend_rows<T, D, 1>(be, p, c, s);
    return rows <= 16 ? attend_rows<T, D, 2>(be, p, c, s) : attend_rows<T, D, 3>(be, p, c, s);
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
        return c.d == 64 ? attend<T, 64>(be, p, c, s) : attend<T, 128>(be, p, c, s);
    };
    return d.dtype == DW_F16 ? with(__half{}) : with(__nv_bfloat16{});
}

}  // namespace dw
