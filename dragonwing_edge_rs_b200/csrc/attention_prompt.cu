// attention_prompt.cu -- attention over the paged 8-bit cache for many query rows (prompts and
// pieces of them), on the tcgen05 tensor cores.  The mathematics is attention.cu's: weights
// w_j = 2^(t_j - M + 7) with t_j = log2(e) scale q . k_j + ev_j, out = sum w_j code_j /
// sum w_j 2^(-ev_j).  M is a maximum that lags: it moves (and what is summed so far is scaled)
// only where a row's true one is more than 2^8 above, so w stays below 2^15, inside f16, and the
// sums are rarely touched.
//
// A CTA has 256 rows (two tiles of 128: token by token the heads of a group) and goes through
// tiles of 64 tokens:
//   converters (4 warps)   codes of keys and values, from global memory through registers, as
//                          f16 into shared memory (128-byte swizzled rows of 64 values);
//   2 issuing warps        (one for each row tile: what one waits for, the other's products fill)
//                          S = Q K^T (128 x 64 x d) into tensor memory, O += P V with P from
//                          tensor memory and V as it lies (tokens x values);
//   2 x 4 softmax warps    a thread a row: S -> weights (f16, over S) and their sum.
// Where units (a CTA's rows and a cache head) are few, the CTAs of a cluster share their tokens.
// Tensor memory holds O of both row tiles (256 columns) and two S of each: the next logits are
// there when a tile's weights are done.  (Tiles of 128 tokens leave room for one S of each; a
// row tile then waited for its own products, 1450 of 4700 cycles.)
// Bound by the weights' arithmetic and by shared memory, which products and converters share (a
// 4096-token prompt, 32 heads over 8 of 128, 137 GFLOP, in 172 us: 800 TFLOP/s).

#include <algorithm>
#include <type_traits>

#include "dw_attend.cuh"
#include "dw_launch.h"
#include "dw_mxfp4.cuh"
#include "dw_ptx.cuh"
#include "dw_tcgen05.cuh"

namespace dw {
namespace {

constexpr int kRows = 256, kTile = 64;  // query rows of a CTA, tokens of a tile
constexpr int kGroups = kTile / 16;     // of tokens that share scales
constexpr int kThreads = 512;
constexpr int kStages = 4;   // of keys and of values
constexpr float kHead = 7.0f, kLag = 8.0f;

__device__ __forceinline__ bool wait_phase(uint64_t *barrier, uint32_t parity, const AttendParams &p, volatile int *abort_flag, int site) {
    const uint32_t bar = smem_u32(barrier);
    // nearly every wait ends here, without a look at the clock (a wait with a time to sleep wakes
    // up late)
#pragma unroll 1
    for (int i = 0; i < 4096; i++)
        if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
    for (;;) {
        if (mbar_try_wait_sleep(bar, parity, 20000u)) return true;
        if (*abort_flag) return false;
        if (globaltimer_ns() - t0 > p.wait_cap_ns) {
            *abort_flag = 1;
            record_error(p.err, DW_DEV_WAIT_EXPIRED, site, (int)parity);
            return false;
        }
    }
}
// The same for a whole warp, with one answer.
__device__ __forceinline__ bool wait_warp(uint64_t *barrier, uint32_t parity, const AttendParams &p, volatile int *abort_flag, int site) {
    return __all_sync(0xffffffffu, wait_phase(barrier, parity, p, abort_flag, site));
}

// One product of 128 x N x 16, by an elected lane: both operands in shared memory, or the first
// in tensor memory.
__device__ __forceinline__ void mma_ss(uint32_t elected, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t elected, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t elected, uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(elected)
        : "memory");
}

__device__ __forceinline__ void tm_ld32(uint32_t taddr, float (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
          "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
          "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A row's columns of tensor memory times f, 16 at a time.  (Inlined, and with few registers: as a
// call it cost every tile its moves, 21 us more for a 4096-token prompt.)
__device__ __forceinline__ void scale_columns(uint32_t taddr, int count, float f) {
#pragma unroll 1
    for (int q = 0; q < count; q += 16) {
        uint32_t x[16];
        tm_ld16(taddr + q, x);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
        tm_st16(taddr + q, x);
    }
}

// Values x tokens as they lie (rows of 64 values are tokens): the second operand's descriptor
// where its columns, not its depth, run along the rows.  128-byte swizzle, 8 rows every 1024
// bytes; the next 64 columns `next` bytes on.
__device__ __forceinline__ uint64_t desc_rows(uint32_t addr, uint32_t next) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Byte of the 16-byte piece `chunk` (0..7) of row r in a tile of swizzled 128-byte rows.
__device__ __forceinline__ uint32_t swizzled(int r, int chunk) { return (uint32_t)(r * 128 + ((chunk ^ (r & 7)) << 4)); }

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    k_attend_prompt(const __grid_constant__ AttendParams p, const __grid_constant__ KvCache c, const __grid_constant__ Seqs sq) {
    constexpr int kHalves = D / 64;                   // swizzled tiles of 64 values
    constexpr uint32_t kHalf = kTile * 128, kOperand = kHalves * kHalf;    // bytes of one, of a tile's keys or values
    constexpr uint32_t kQHalf = 128 * 128, kQOperand = kHalves * kQHalf;   // the same of a row tile's queries
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ uint64_t q_full[2], s_full[2][2], p_full[2][2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], drain[2];
    __shared__ float4 scales[8][kGroups];  // of eight tiles: 2^ek, ev, 2^-ev
    __shared__ float row_scale[kRows], all_m[kRows], all_l[kRows];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    uint8_t *const base = smem_raw + (smem - smem_u32(smem_raw));
    const uint32_t q_at = 0, k_at = 2 * kQOperand, v_at = k_at + kStages * kOperand;

    pdl_wait();
    // which rows of which sequence, which head: those that see most first
    const uint32_t S = cluster_size(), rank = cluster_rank(), block = blockIdx.x / S;
    const uint32_t unit = block / (uint32_t)c.heads;
    const int head = (int)(block % (uint32_t)c.heads);
    int64_t place;
    uint32_t s;
    if (p.per_seq) {
        s = unit % sq.seqs, place = p.per_seq - 1 - (int)(unit / sq.seqs);
    } else {
        s = seq_of_item(sq, p.items - 1 - unit, p.group, kRows, 1, place);
    }
    const SeqRange r = seq_range(sq, s, c.page, p.err, p.items - 1 - unit);
    const int rows_all = r.n * p.group, first = (int)min(place * kRows, (int64_t)0x7fffffff);
    if (place < 0 || first >= rows_all) {
        pdl_trigger();
        return;
    }
    const int rows = min(kRows, rows_all - first);
    auto token_of = [&](int row) { return (first + row) / p.group; };
    const int lo = row_bounds(p, r, token_of(0)).lo;
    int tile0 = lo / kTile;
    // tiles of either row tile: up to the last token that its last row sees
    int tiles[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int hi = rows > t * 128 ? row_bounds(p, r, token_of(min(rows, t * 128 + 128) - 1)).hi : 0;
        tiles[t] = max(0, (hi + kTile - 1) / kTile - tile0);
    }
    if (S > 1) {  // this CTA's share of them
        const int share = (max(tiles[0], tiles[1]) + (int)S - 1) / (int)S, from = (int)rank * share;
        tile0 += from;
#pragma unroll
        for (int t = 0; t < 2; t++) tiles[t] = min(max(tiles[t] - from, 0), share);
    }
    const int all = max(tiles[0], tiles[1]);

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(smem_u32(&q_full[i]), 4), mbar_init(smem_u32(&s_full[i][0]), 1), mbar_init(smem_u32(&s_full[i][1]), 1);
            mbar_init(smem_u32(&p_full[i][0]), 4), mbar_init(smem_u32(&p_full[i][1]), 4), mbar_init(smem_u32(&drain[i]), 1);
        }
        for (int i = 0; i < kStages; i++) {
            mbar_init(smem_u32(&k_full[i]), 4), mbar_init(smem_u32(&k_empty[i]), 2);
            mbar_init(smem_u32(&v_full[i]), 4), mbar_init(smem_u32(&v_empty[i]), 2);
        }
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);  // two S of 64 columns of each row tile, then O

    // a softmax thread's row: sums, maximum (as the last phase needs them)
    float M = -INFINITY, L = 0.0f;
    bool ok = true;
    if (warp >= 12) {
        // ---- converters: a thread has 16 codes of each half of a row in each of two groups of 32 rows
        const int tid = threadIdx.x - 384, part = tid & 3, sub = tid >> 2;
        constexpr int kG = kTile / 32, kN = kG * kHalves;
        const int shift = 31 - __clz(c.page);  // pages hold a power of two of tokens
        // Codes are loaded two tiles ahead, and a row's page looked up a tile before that: a load takes
        // some 800 cycles, a lookup as many before it.
        struct Pages {
            uint32_t row[kG], group;  // of the thread's rows; of group tid
        } ahead{};
        struct Codes {
            uint4 k[kN], v[kN];
            uint32_t scales;  // of group tid
        } x0, x1;
        bool bad = false;
        const int begin = lo & -c.page;  // pages that end before the window may have been given away
        auto lookup = [&](int t) {  // the page of token t, in bounds in any case
            if (t >= r.len || t < begin) return 0u;
            const uint32_t id = (uint32_t)sq.table[(size_t)s * sq.width + (uint32_t)(t >> shift)];
            bad |= id >= c.pages;
            return id;
        };
        auto find = [&](Pages &g, int tile) {
            const int t = (tile0 + tile) * kTile;
#pragma unroll
            for (int i = 0; i < kG; i++) g.row[i] = lookup(t + i * 32 + sub);
            if (tid < kGroups) g.group = lookup(t + tid * 16);
        };
        auto load = [&](uint4 (&x)[kN], const uint8_t *codes, const Pages &pg, int tile) {
#pragma unroll
            for (int g = 0; g < kG; g++) {
                const int t = (tile0 + tile) * kTile + g * 32 + sub;
                const uint32_t row = ((min(pg.row[g], c.pages - 1) * (uint32_t)c.heads + (uint32_t)head) << shift) + (uint32_t)(t & (c.page - 1));
                const uint4 *from = reinterpret_cast<const uint4 *>(codes + (size_t)row * D) + part;
#pragma unroll
                for (int h = 0; h < kHalves; h++)  // no token, or none that a row sees: zeros, whatever the page holds there
                    x[g * kHalves + h] = t < r.len && t >= begin ? from[4 * h] : make_uint4(0, 0, 0, 0);
            }
        };
        auto load_scales = [&](Codes &x, const Pages &pg) {
            if (tid < kGroups) x.scales = *reinterpret_cast<const uint16_t *>(c.s + kv_block(c, min(pg.group, c.pages - 1), head) * 2);
        };
        auto store = [&](const uint4 (&x)[kN], uint32_t at) {
            // (row & 7 is the same in every group)
            const uint32_t to = smem + at + swizzled(sub, 2 * part), to1 = smem + at + swizzled(sub, 2 * part + 1);
#pragma unroll
            for (int g = 0; g < kG; g++)
#pragma unroll
                for (int h = 0; h < kHalves; h++) {
                    const uint4 u = x[g * kHalves + h];
                    sts_v4(to + h * kHalf + g * 4096, make_uint4(e4m3_to_f16x2((uint16_t)u.x), e4m3_to_f16x2((uint16_t)(u.x >> 16)),
                                                                 e4m3_to_f16x2((uint16_t)u.y), e4m3_to_f16x2((uint16_t)(u.y >> 16))));
                    sts_v4(to1 + h * kHalf + g * 4096, make_uint4(e4m3_to_f16x2((uint16_t)u.z), e4m3_to_f16x2((uint16_t)(u.z >> 16)),
                                                                  e4m3_to_f16x2((uint16_t)u.w), e4m3_to_f16x2((uint16_t)(u.w >> 16))));
                }
        };
        auto done = [&](uint64_t *bar) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(bar));
        };
        Pages second{};
        if (all) find(ahead, 0);
        if (all > 1) find(second, 1);
        if (all) load(x0.k, c.k, ahead, 0), load_scales(x0, ahead), load(x0.v, c.v, ahead, 0);
        if (all > 1) load(x1.k, c.k, second, 1), load_scales(x1, second), load(x1.v, c.v, second, 1);
        if (all > 2) find(ahead, 2);
        auto convert = [&](int j, Codes &x) {
            const int st = j % kStages;
            const uint32_t ph = (uint32_t)(j / kStages) & 1;
            if (j >= kStages && !wait_warp(&k_empty[st], ph ^ 1, p, abort_flag, 71)) return false;
            store(x.k, k_at + st * kOperand);
            if (tid < kGroups) {
                const int ve = kv_exponent(x.scales >> 8);
                scales[j & 7][tid] = make_float4(kv_pow2(kv_exponent(x.scales & 255)), (float)ve, kv_pow2(-ve), 0.0f);
            }
            done(&k_full[st]);
            const Pages now = ahead;
            if (j + 2 < all) load(x.k, c.k, now, j + 2), load_scales(x, now);
            if (j + 3 < all) find(ahead, j + 3);
            if (j >= kStages && !wait_warp(&v_empty[st], ph ^ 1, p, abort_flag, 72)) return false;
            store(x.v, v_at + st * kOperand);
            done(&v_full[st]);
            if (j + 2 < all) load(x.v, c.v, now, j + 2);
            return true;
        };
        for (int j = 0; j < all; j += 2)
            if (!convert(j, x0) || (j + 1 < all && !convert(j + 1, x1))) break;
        if (bad) record_error(p.err, DW_DEV_BAD_ARG, 62, (int)s);
    } else if (warp < 2) {
        // ---- products of row tile t: S of tile j + 2 goes to the place of what the weights of tile j were made of
        const int t = warp;
        const uint32_t elected = elect_one();
        constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(kTile >> 3) << 17) | (8u << 24);
        constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);
        constexpr uint64_t hi = ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
        auto phase = [](int j) { return (uint32_t)(j / kStages) & 1; };
        ok = !tiles[t] || wait_warp(&q_full[t], 0, p, abort_flag, 73);
        for (int j = -2; j < all && ok; j++) {
            const int k = j + 2;
            const bool sums = j >= 0 && j < tiles[t], logits = k < tiles[t];
            // (stages of tiles that only the other row tile needs are waited for and given back too)
            if (j >= 0) ok = wait_warp(&v_full[j % kStages], phase(j), p, abort_flag, 75);
            if (k < all && ok) ok = wait_warp(&k_full[k % kStages], phase(k), p, abort_flag, 74);
            if (sums && ok) ok = wait_warp(&p_full[t][j & 1], (uint32_t)(j >> 1) & 1, p, abort_flag, 76);
            if (!ok) break;
            tc_fence_after();
            const uint32_t s_tm = tmem + (2 * t + (j & 1)) * kTile;
            if (sums) {
                const uint32_t b = smem + v_at + (j % kStages) * kOperand;
#pragma unroll
                for (int i = 0; i < kTile / 16; i++)
                    mma_ts(elected, tmem + 256 + t * D, s_tm + i * 8, desc_rows(b + i * 2048, kHalf), idesc_o, (j || i) ? 1u : 0u);
            }
            if (logits) {
                const uint32_t a = smem + q_at + t * kQOperand, b = smem + k_at + (k % kStages) * kOperand;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    const uint32_t in = (uint32_t)(i % 4) * 32;
                    mma_ss(elected, s_tm, smem_desc(a + (i / 4) * kQHalf + in, hi), smem_desc(b + (i / 4) * kHalf + in, hi), idesc_s, i ? 1u : 0u);
                }
            }
            // also without logits (behind the last tile): the sums up to tile j are done then
            if (k < tiles[t] + 2) commit(elected, &s_full[t][j & 1]);
            if (j >= 0) commit(elected, &v_empty[j % kStages]);
            if (k < all) commit(elected, &k_empty[k % kStages]);
        }
        // products in flight end before the tensor memory is given back
        commit(elected, &drain[t]);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait_sleep(smem_u32(&drain[t]), 0, 20000u) && globaltimer_ns() - t0 < p.wait_cap_ns) {
        }
    } else if (warp >= 4) {
        // ---- softmax: a thread has a row
        const int t = (warp - 4) >> 2, row = t * 128 + (warp & 3) * 32 + lane;
        const bool there = row < rows;
        const int at = first + min(row, rows - 1), token = at / p.group;  // (behind the last: as the last, and not stored)
        const Bounds b = row_bounds(p, r, token);
        float a_row = p.scale_log2;
        // The warp's 32 query rows, in f16, to shared memory: kPer lanes a row, eight rows of a lane
        // in flight (a row a thread, its pieces one after the other, took 13000 cycles).
        if (tiles[t]) {
            constexpr int kPer = D / 8, kStep = 32 / kPer;
            const int piece = lane % kPer, row0 = t * 128 + (warp & 3) * 32 + lane / kPer;
            int token = (first + row0) / p.group, in = (first + row0) % p.group;  // of the lane's next row
            const T *src = nullptr;
            auto source = [&](int row) {  // of its rows in turn; behind the last, the last one's
                if (row < rows) src = (const T *)p.q + (size_t)(r.row0 + token) * p.q_pitch + (size_t)(head * p.group + in) * D + 8 * piece;
                in += kStep;
                while (in >= p.group) in -= p.group, token++;
                return src;
            };
            src = (const T *)p.q + (size_t)(r.row0 + token_of(0)) * p.q_pitch + (size_t)(head * p.group + first % p.group) * D + 8 * piece;
            // all of a lane's pieces at once to their places (by way of registers, four or eight in flight,
            // they took 7000 cycles), bf16 rows turned into f16 there
            auto place = [&](int row) { return smem + q_at + t * kQOperand + (piece / 8) * kQHalf + swizzled(row & 127, piece & 7); };
#pragma unroll 4
            for (int i = 0; i < kPer; i++) {
                const int row = row0 + i * kStep;
                const T *from = source(row);
                if (p.vec) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(place(row)), "l"(from) : "memory");
                } else {
                    Raw<T, 8> x;
                    float u[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) u[e] = to_f32(from[e]);
                    x.set(u);
                    sts_v4(place(row), make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]));
                }
            }
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
            if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll 1
                for (int i0 = 0; i0 < kPer; i0 += 4) {
                    Raw<T, 8> x[4];
                    float top[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint4 v = lds_v4(place(row0 + (i0 + i) * kStep));
                        x[i].w[0] = v.x, x[i].w[1] = v.y, x[i].w[2] = v.z, x[i].w[3] = v.w, top[i] = 0.0f;
#pragma unroll
                        for (int e = 0; e < 8; e++) top[i] = fmaxf(top[i], fabsf(x[i].get(e)));
                    }
#pragma unroll
                    for (int o = kPer / 2; o; o >>= 1)
#pragma unroll
                        for (int i = 0; i < 4; i++) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int row = row0 + (i0 + i) * kStep, e = query_exponent(top[i]);
                        const float down = kv_pow2(-e);
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) w[k] = pack2<__half>(x[i].get(2 * k) * down, x[i].get(2 * k + 1) * down);
                        sts_v4(place(row), make_uint4(w[0], w[1], w[2], w[3]));
                        if (piece == 0) row_scale[row] = kv_pow2(e);
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&q_full[t]));
            if constexpr (std::is_same_v<T, __nv_bfloat16>) a_row *= row_scale[row];
        }
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s0_tm = tmem + 2 * t * kTile + lanes, o_tm = tmem + 256 + t * D + lanes;
        // tokens that all of the warp's rows see, and those that any does
        const int lo_all = __reduce_max_sync(0xffffffffu, b.lo), hi_all = __reduce_min_sync(0xffffffffu, b.hi);
        for (int j = 0; j < tiles[t]; j++) {
            const int t0 = (tile0 + j) * kTile;
            if (!wait_warp(&s_full[t][j & 1], (uint32_t)(j >> 1) & 1, p, abort_flag, 77)) {
                ok = false;
                break;
            }
            tc_fence_after();
            {
                const uint32_t s_tm = s0_tm + (j & 1) * kTile;
                float x[kTile / 32][32];
#pragma unroll
                for (int q = 0; q < kTile / 32; q++) tm_ld32(s_tm + q * 32, x[q]);
                float4 sc[kGroups];
#pragma unroll
                for (int g = 0; g < kGroups; g++) {
                    sc[g] = scales[j & 7][g];
                    sc[g].x = fmaxf(sc[g].x * a_row, 1e-37f);  // above 0: -inf, which hides a token, stays -inf
                }
                tc_wait_ld();
                if (t0 < lo_all || t0 + kTile > hi_all) {  // a tile that some row sees in part
                    auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
#pragma unroll
                    for (int q = 0; q < kTile / 32; q++) {
                        const uint32_t seen = below(b.hi - t0 - 32 * q) & ~below(b.lo - t0 - 32 * q);
#pragma unroll
                        for (int i = 0; i < 32; i++) x[q][i] = seen >> i & 1 ? x[q][i] : -INFINITY;
                    }
                }
                // the largest exponent; NaN where there is one (M then becomes NaN, and all that the row sums)
                float top = -INFINITY;
#pragma unroll
                for (int g = 0; g < kGroups; g++) {
                    const float *v = x[g / 2] + 16 * (g & 1);
                    float m = max_nan(v[0], v[1], v[2]), n = max_nan(v[3], v[4], v[5]);
#pragma unroll
                    for (int i = 6; i < 14; i += 4) m = max_nan(m, v[i], v[i + 1]), n = max_nan(n, v[i + 2], v[i + 3]);
                    m = max_nan(m, v[14], v[15]);
                    top = max_nan(top, top, fmaf(max_nan(m, n, n), sc[g].x, sc[g].y));
                }
                if (__any_sync(0xffffffffu, !(top <= M + kLag))) {
                    // M moves, to a whole number: what is scaled stays exact
                    const float next = top <= M + kLag ? M : ceilf(top), f = carry(M, next);
                    M = next;
                    L *= f;
                    if (j) {
                        // the sums up to tile j - 1 are done when the logits of tile j + 1 are there
                        ok = wait_warp(&s_full[t][(j + 1) & 1], (uint32_t)((j + 1) >> 1) & 1, p, abort_flag, 79);
                        tc_fence_after();
                        scale_columns(o_tm, D, f);
                    }
                }
                const float head_room = (M == -INFINITY ? 0.0f : -M) + kHead;
#pragma unroll
                for (int q = 0; q < kTile / 32; q++) {
                    uint32_t w[16];
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        const float a = sc[2 * q + g].x, add = sc[2 * q + g].y + head_room;
                        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                        for (int i = 16 * g; i < 16 * g + 16; i += 2) {
                            float2 y = __ffma2_rn(make_float2(x[q][i], x[q][i + 1]), make_float2(a, a), make_float2(add, add));
                            y = eleven_bits(ex2_approx(y.x), ex2_approx(y.y));
                            sum = __fadd2_rn(sum, y);
                            w[i / 2] = pack2<__half>(y.x, y.y);
                        }
                        L = fmaf(sum.x + sum.y, sc[2 * q + g].z, L);
                    }
                    tm_st16(s_tm + q * 16, w);
                }
            }
            if (!ok) break;
            tm_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&p_full[t][j & 1]));
        }
        if (tiles[t] && ok) ok = wait_warp(&s_full[t][(tiles[t] + 1) & 1], (uint32_t)((tiles[t] + 1) >> 1) & 1, p, abort_flag, 78);
        if (ok && rows > t * 128 + (warp & 3) * 32 && S == 1) {
            tc_fence_after();
            const float f = L == 0.0f ? 0.0f : 1.0f / L;
            T *dst = (T *)p.out + (size_t)(r.row0 + token) * p.out_pitch + (size_t)(head * p.group + at % p.group) * D;
#pragma unroll
            for (int q = 0; q < D / 32; q++) {
                float x[32];
                if (tiles[t]) {
                    tm_ld32(o_tm + q * 32, x);
                    tc_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) x[i] = 0.0f;
                }
                if (!there) continue;
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = x[i + e] * f;
                    if (p.vec) {
                        Raw<T, 8> o;
                        o.set(y);
                        o.store(dst + q * 32 + i);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e++) dst[q * 32 + i + e] = from_f32<T>(y[e]);
                    }
                }
            }
        }
    }
    if (S > 1) {
        // ---- join: each CTA leaves its sums in shared memory, over its queries and stages
        float *const part = reinterpret_cast<float *>(base);  // [256][D], a row's 16-byte pieces xor the row modulo 8
        auto piece_at = [&](int row, int piece) { return part + row * D + (piece ^ (row & 7)) * 4; };
        __syncwarp();
        __syncthreads();  // all products are done
        if (warp >= 4 && warp < 12) {
            const int t = (warp - 4) >> 2, row = t * 128 + (warp & 3) * 32 + lane;
            all_m[row] = M, all_l[row] = L;
            tc_fence_after();
            if (tiles[t]) {
#pragma unroll
                for (int q = 0; q < D / 32; q++) {
                    float x[32];
                    tm_ld32(tmem + 256 + t * D + ((uint32_t)((warp & 3) * 32) << 16) + q * 32, x);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        *reinterpret_cast<float4 *>(piece_at(row, q * 8 + i)) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                }
            } else {
#pragma unroll 4
                for (int i = 0; i < D / 4; i++) *reinterpret_cast<float4 *>(piece_at(row, i)) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
        cluster_sync();
        for (int i = (int)rank * kThreads + threadIdx.x; i < rows * (D / 4); i += (int)S * kThreads) {
            const int row = i / (D / 4), piece = i % (D / 4);
            float l;
            const float4 v = join_sums(all_m + row, all_l + row, piece_at(row, piece), S, l);
            const float f = l == 0.0f ? 0.0f : 1.0f / l, y[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
            const int at = first + row;
            T *dst = (T *)p.out + (size_t)(r.row0 + at / p.group) * p.out_pitch + (size_t)(head * p.group + at % p.group) * D + piece * 4;
            if (p.vec) {
                Raw<T, 4> o;
                o.set(y);
                o.store(dst);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) dst[e] = from_f32<T>(y[e]);
            }
        }
        cluster_sync_relaxed();  // no CTA leaves while its sums may be read
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace

template <typename T, int D>
dw_status attend_prompt(dw_backend *be, AttendParams p, const KvCache &c, const Seqs &s) {
    auto kernel = k_attend_prompt<T, D>;
    constexpr size_t smem = 1024 + (size_t)(2 * 128 + 2 * kStages * kTile) * D * 2;
    const size_t n = s.tokens / s.seqs;
    p.per_seq = s.starts ? 0 : (int)seq_items_each(n, p.group, kRows, 1);
    const size_t items = s.starts ? seq_items(s.tokens, s.seqs, p.group, kRows, 1) : (size_t)p.per_seq * s.seqs;
    if (items * c.heads > 0x7fffffffu) return dw_fail(be, DW_ERR_UNSUPPORTED, "attention_kv8: too many rows");
    p.items = (uint32_t)items;
    static bool attr_set[16] = {};
    if (be->device < 16 && !attr_set[be->device]) {
        dw_status st = dw_cuda_check(be, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                                     "attention_kv8 attributes");
        if (st != DW_OK) return st;
        attr_set[be->device] = true;
    }
    // S CTAs share a unit's tiles while an SM each is there and four tiles each (256 rows over 8000 tokens, 8
    // heads: S = 1, 2, 4, 8 145, 83, 47, 33 us; 300 rows and tokens: with shares of two tiles 16.3, without 14.5)
    const size_t units = items * c.heads, most = ((size_t)s.width * c.page + kTile - 1) / kTile;
    unsigned S = 1;
    while (S < kMaxShare && units * 2 * S <= (size_t)be->sm_count && 2 * S * 4 <= most) S *= 2;
    return launch_dependent(be, "attention_kv8 (prompt)", kernel, (unsigned)(units * S), kThreads, smem, S, p, c, s);
}

template dw_status attend_prompt<__half, 64>(dw_backend *, AttendParams, const KvCache &, const Seqs &);
template dw_status attend_prompt<__half, 128>(dw_backend *, AttendParams, const KvCache &, const Seqs &);
template dw_status attend_prompt<__nv_bfloat16, 64>(dw_backend *, AttendParams, const KvCache &, const Seqs &);
template dw_status attend_prompt<__nv_bfloat16, 128>(dw_backend *, AttendParams, const KvCache &, const Seqs &);

}  // namespace dw
