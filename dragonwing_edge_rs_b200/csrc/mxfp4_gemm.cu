// mxfp4_gemm.cu -- the product of two MXFP4 operands on the tcgen05 tensor cores
// (kind::mxf4, block scales in tensor memory), with bias, activation and the
// rounding or MXFP4 quantisation of the result fused into the epilogue:
//   y[m, n] = act(sum_k A[m, k] * B[n, k] + bias[n])
// Products and sums are the tensor core's (f32 accumulators); bias and activation
// are f32.
//
// Two kernels, one for many rows of A (pairs of CTAs, cta_group::2) and one for few (the
// weights on the 128-row side), built alike and warp-specialised:
//   warp 0    producer: TMA boxes of codes (128 bytes a row, 128-byte swizzle) and of
//             scale tiles into a ring of stages;
//   warp 2    tcgen05.cp of a stage's scale tiles into that stage's scale columns of
//             tensor memory;
//   warp 1    the products of a stage, tcgen05.mma.kind::mxf4 of 64 codes each;
//   the rest  epilogue: accumulators -> bias, activation, rounding or requantisation.
// What bounds them (B200): with many rows each SM's intake from L2 -- a stage of 512 codes
// is 70 KB for 256 x 256 outputs (0.63 us; 0.54 us at the tensor rate) and 52 KB for
// 256 x 128 (0.36 us) -- and beyond one round of tiles the power limit; 8192^3 runs at
// 5.4 to 5.7 PFLOP/s (193 to 205 us), 4096^3 at 4.4 (31 us), in a sustained loop at 3.8
// (36 us).  With few rows the weights' bytes and about 2.3 us of
// launch, first copies and hand-offs: 11008 x 4096 (24 MB) 5.5 us from L2, 7.6 from HBM.
// What a step of it cost and saved stands beside each part: launches in a row in short
// runs, measured when the step was made.
//
// Every mbarrier wait is bounded; on expiry the CTA records the failure, waits
// (bounded) for its own copies and products in flight, frees its tensor memory
// and exits.

#include <algorithm>

#include "dw_device.cuh"
#include "dw_launch.h"
#include "dw_mxfp4.cuh"
#include "dw_ptx.cuh"
#include "dw_tcgen05.cuh"

namespace dw {
namespace {

constexpr int kBM = 128;
constexpr int kBKBytes = 128;  // a K block: 256 codes
constexpr size_t kSmemLimit = 227 * 1024;  // of a CTA
constexpr size_t kSmemSm = 228 * 1024;     // of an SM

struct GemmParams {
    const float *bias;
    void *y;
    uint8_t *y_s;
    size_t m, n;
    int tiles_k;      // scale tiles (128 codes) along K
    size_t out_nb, out_tiles;  // MXFP4 result: blocks and scale tiles along n
    int k_blocks;     // 512-wide K blocks
    int tiles_m, tiles;
    int stages, act;
    bool vec, bias_vec;  // rows of y, the bias start on 16-byte boundaries
    uint64_t wait_cap_ns;
    int32_t *err;
};

// Bounded wait for a phase: polls first (most waits are short), then suspends; false
// once the CTA is aborting or the cap expired.
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, uint64_t cap_ns, int32_t *err,
                                           volatile int *abort_flag, int site) {
#pragma unroll 1
    for (int i = 0; i < 8; i++)
        if (mbar_test_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
    for (;;) {
        if (mbar_try_wait_sleep(bar, parity, 20000u)) return true;
        if (*abort_flag) return false;
        if (globaltimer_ns() - t0 > cap_ns) {
            *abort_flag = 1;
            record_error(err, DW_DEV_WAIT_EXPIRED, site, (int)parity);
            return false;
        }
    }
}

// The same for a whole warp, with one answer.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, uint64_t cap_ns, int32_t *err, volatile int *abort_flag,
                                          int site) {
#pragma unroll 1
    for (int i = 0; i < 1024; i++)
        if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, wait_phase(bar, parity, cap_ns, err, abort_flag, site));
}

// Waits for a phase that the CTA's own work in flight completes, whatever happened before.
__device__ __forceinline__ void drain_phase(uint32_t bar, uint32_t parity, uint64_t cap_ns) {
    const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
    while (!mbar_try_wait_sleep(bar, parity, 20000u))
        if (globaltimer_ns() - t0 > cap_ns) return;
}

// The warps that feed the tensor core run their loops with all lanes, on warp-uniform
// values, and predicate each issue on one elected lane: operands then come from
// uniform registers.  (A loop inside `if (lane == 0)` issues an MMA only every ~110
// cycles and a scale copy every ~80: 4096^3 took 34 us so, 30.7 this way.)
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// 512 bytes (32 rows of 16) -> 4 columns of all four lane quarters of tensor memory
// (of both CTAs of a pair).
template <int kCtas>
__device__ __forceinline__ void tc_cp_scales(uint32_t elected, uint32_t taddr, uint64_t desc) {
    if constexpr (kCtas == 1)
        asm volatile(
            "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr),
            "l"(desc), "r"(elected)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr),
            "l"(desc), "r"(elected)
            : "memory");
}

// One product of 128 (256 by a pair) x N x 64 with block scales (two 32-wide blocks a row).
template <int kCtas>
__device__ __forceinline__ void tc_mma_mxf4(uint32_t elected, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                            uint32_t sfb, uint32_t accumulate) {
    if constexpr (kCtas == 1)
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(elected)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t"
            "@q tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(elected)
            : "memory");
}

__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}

// silu(v) = v / (1 + e^-v) by ex2.approx and rcp.approx: a relative error of a few
// 2^-24 plus |v| * 2^-24 (the exponent's rounding).  e^-v = inf gives v * 0 = -0.
// A NaN stays one through either (a plain fmaxf would make it 0).
__device__ __forceinline__ float activate(float v, int act) {
    if (act == DW_EPI_RELU) {
        float r;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(0.0f));
        return r;
    }
    if (act == DW_EPI_SILU) {
        float r;
        asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + __expf(-v)));
        return v * r;
    }
    return v;
}

// Instruction descriptor of kind::mxf4: A, B e2m1 (1 at bits 7-9 and 10-12), N >> 3
// at bits 17-22, scales ue8m0 (bit 23), M >> 4 at bits 24-28; the scale byte pair
// that a 64-wide step reads: bits 29-30 (A) and 4-5 (B).
constexpr uint32_t mx_idesc(int m, int n, int pair) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24) |
           ((uint32_t)(2 * pair) << 29) | ((uint32_t)(2 * pair) << 4);
}

// Bias and activation of 32 columns of a row.
__device__ __forceinline__ void finish32(float (&v)[32], size_t col, const GemmParams &p) {
    if (p.bias) {
        if (col + 32 <= p.n && p.bias_vec) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float4 b = reinterpret_cast<const float4 *>(p.bias + col)[i];
                v[4 * i] += b.x, v[4 * i + 1] += b.y, v[4 * i + 2] += b.z, v[4 * i + 3] += b.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; i++)
                if (col + i < p.n) v[i] += p.bias[col + i];
        }
    }
    if (p.act == DW_EPI_RELU) {
#pragma unroll
        for (int i = 0; i < 32; i++) v[i] = activate(v[i], DW_EPI_RELU);
    } else if (p.act == DW_EPI_SILU) {
#pragma unroll
        for (int i = 0; i < 32; i++) v[i] = activate(v[i], DW_EPI_SILU);
    }
}

// 64 bytes of each of 32 consecutive rows (lane = row) -> y.  Four lanes exchange
// 16-byte pieces first, so that a store covers 8 rows of 64 bytes instead of 32 of 16
// (one line a row: the epilogue of a 256 x 256 tile took 4 us of stores).
template <typename T>
__device__ __forceinline__ void store64(uint32_t (&w)[16], size_t row, size_t col, const GemmParams &p) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int s = 1; s < 4; s <<= 1)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            if (c & s) continue;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t a = w[4 * c + i], b = w[4 * (c | s) + i];
                const uint32_t got = __shfl_xor_sync(0xffffffffu, lane & s ? a : b, s);
                if (lane & s)
                    w[4 * c + i] = got;
                else
                    w[4 * (c | s) + i] = got;
            }
        }
    const size_t row0 = row - (lane & 3);
    T *dst = (T *)p.y + row0 * p.n + col + (lane & 3) * (16 / sizeof(T));
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (row0 + k < p.m) *reinterpret_cast<uint4 *>(dst + k * p.n) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
}

// What the epilogue stores: 0 f32, 1 f16, 2 bf16, 3 MXFP4.  Rows of y that do not start on
// 16 bytes are written one element a lane, a row a lane (4096 x 4001 x 4096 f16 186 us,
// 4096 x 4000 x 4096 31).
template <int kOut>
__device__ __forceinline__ void put32(float (&v)[32], size_t row, size_t col, const GemmParams &p, uint32_t &scale) {
    if constexpr (kOut == 3) {
        if (col + 32 > p.n) {
#pragma unroll
            for (int i = 0; i < 32; i++)
                if (col + i >= p.n) v[i] = 0.0f;
        }
        uint4 codes;
        scale = mx_quantize32(v, codes);
        if (row < p.m && col / 32 < p.out_nb) *reinterpret_cast<uint4 *>((uint8_t *)p.y + (row * p.out_nb + col / 32) * 16) = codes;
    } else {
        using T = std::conditional_t<kOut == 0, float, std::conditional_t<kOut == 1, __half, __nv_bfloat16>>;
        if (p.vec && col + 32 <= p.n) {
            constexpr int kPer = 64 / sizeof(T);  // columns of 64 bytes
#pragma unroll
            for (int h = 0; h < 32 / kPer; h++) {
                uint32_t w[16];
                if constexpr (kOut == 0) {
#pragma unroll
                    for (int i = 0; i < 16; i++) w[i] = __float_as_uint(v[16 * h + i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
                }
                store64<T>(w, row, col + h * kPer, p);
            }
        } else if (row < p.m) {
            T *dst = (T *)p.y + row * p.n + col;
#pragma unroll
            for (int i = 0; i < 32; i++)
                if (col + i < p.n) dst[i] = from_f32<T>(v[i]);
        }
    }
}

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
// The same without ordering memory: nobody leaves (or reuses) before all are here.
__device__ __forceinline__ void cluster_sync_relaxed() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The scale bytes of kN (1 or 2) blocks of a row, the last of a row with the zeros of
// the tile's places past it.
template <int kN>
__device__ __forceinline__ void put_scales(uint32_t scales, size_t row, size_t block, const GemmParams &p) {
    if (row >= p.m) return;
    uint8_t *s = p.y_s + mx_scale_at(row, block, p.out_tiles);
    if constexpr (kN == 2)
        *reinterpret_cast<uint16_t *>(s) = (uint16_t)scales;
    else
        *s = (uint8_t)scales;
    if (block + kN >= p.out_nb)
        for (size_t b = block + kN; b < p.out_tiles * 4; b++) p.y_s[mx_scale_at(row, b, p.out_tiles)] = 0;
}

// ---- many rows -----------------------------------------------------------------
// A pair of CTAs (cta_group::2) computes a 256 x BN tile: each holds 128 rows of A,
// half of B's rows, the scales of its rows of A and those of all BN rows of B, so a
// K block costs each SM's L2 port (128 + BN / 2) * 128 bytes of codes for
// 256 * BN * 256 products of the pair.  The leader issues for both, and both CTAs' copies
// complete on its barrier (a relay by the peer, releasing and acquiring at cluster scope,
// took 64 us for 4096^3; this 40).  The epilogue takes its accumulators into registers
// at once and gives the tensor memory back before it converts and stores.
//
// Pairs of one cluster can share a tile's K (then it is the cluster's only tile): each
// leaves its partial tile in shared memory, over the ring, and adds up its share of the
// columns in the order of the pairs.
constexpr int kEpiWarps = 16;
constexpr int kGemmThreads = 128 + 32 * kEpiWarps;
constexpr int kMaxStages = 8;

__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Copies into this CTA that complete on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
        "[%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
        "[%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
__device__ __forceinline__ void tc_commit1(uint32_t elected, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
        "r"(elected)
        : "memory");
}
// Commits of the pair: to the leader's barrier, or to the same barrier of both CTAs.
__device__ __forceinline__ void tc_commit2(uint32_t elected, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
        "r"(elected)
        : "memory");
}
__device__ __forceinline__ void tc_commit2_both(uint32_t elected, uint32_t bar, uint16_t ctas) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
        "h"(ctas), "r"(elected)
        : "memory");
}

template <int BN, int kOut>
__global__ void __launch_bounds__(kGemmThreads, 1)
    k_mxfp4_gemm(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                 const __grid_constant__ CUtensorMap tmap_sa, const __grid_constant__ CUtensorMap tmap_sb,
                 const __grid_constant__ GemmParams p) {
    // a stage: 512 codes of a row in two swizzled boxes of 128 bytes, four scale tiles
    constexpr uint32_t kA = kBM * kBKBytes, kB = BN / 2 * kBKBytes, kSA = 2048, kSB = (BN / 128) * 2048;
    constexpr uint32_t kStage = 2 * (kA + kB) + kSA + kSB;
    constexpr uint32_t kScaleCols = 16 + BN / 8;  // tensor-memory columns of a stage's scales
    constexpr int kAcc = 256 / BN;                // accumulator buffers
    constexpr int kCols = BN / 4;                 // columns of an epilogue warp
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    __shared__ uint64_t full_bar[kMaxStages], sf_bar[kMaxStages], empty_bar[kMaxStages];
    __shared__ uint64_t tfull_bar[kAcc], tempty_bar[kAcc], drain_bar[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    // CTAs of the cluster: pairs that share a tile's K (one pair: all of it, and the
    // pairs of the grid loop over the tiles)
    const uint32_t cta = cluster_rank(), rank = cta & 1, lead = cta & ~1u, S = cluster_size() >> 1, part_k = cta >> 1;
    const int pair = (int)(blockIdx.x / (2 * S)), pairs = (int)(gridDim.x / (2 * S));
    const int kb0 = (int)((long long)p.k_blocks * part_k / S), kb1 = (int)((long long)p.k_blocks * (part_k + 1) / S);
    const uint16_t both = (uint16_t)(3u << lead);

    if (threadIdx.x == 32 * 3) {
        prefetch_map(&tmap_a), prefetch_map(&tmap_b), prefetch_map(&tmap_sa), prefetch_map(&tmap_sb);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; s++) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&sf_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        for (int a = 0; a < kAcc; a++) {
            mbar_init(smem_u32(&tfull_bar[a]), 1);
            mbar_init(smem_u32(&tempty_bar[a]), 2 * kEpiWarps);
        }
        mbar_init(smem_u32(&drain_bar[0]), 1);
        mbar_init(smem_u32(&drain_bar[1]), 1);
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    pdl_wait();  // in every warp: the bounded waits count from here
    pdl_trigger();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
    const uint32_t sf_cols = tmem + 256;  // scales after the accumulators
    float *partial = reinterpret_cast<float *>(smem_raw + (smem - smem_u32(smem_raw)));  // [BN][128]

    if (warp == 0) {
        const uint32_t elected = elect_one();
        int s = 0, issued = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int tile = pair; ok && tile < p.tiles; tile += pairs) {
            const int tm = (tile % p.tiles_m) * 2 + (int)rank, tn = tile / p.tiles_m;  // 128-row tile of A, BN-row tile of B
            const int a_row = tm * kBM, b_row = tn * BN + (int)rank * (BN / 2);
            for (int kb = kb0; kb < kb1; kb++) {
                if (issued >= p.stages && !wait_warp(smem_u32(&empty_bar[s]), ph ^ 1u, p.wait_cap_ns, p.err, abort_flag, 21)) {
                    ok = false;
                    break;
                }
                // both CTAs' copies complete on the leader's barrier
                const uint32_t bar = peer_addr(smem_u32(&full_bar[s]), lead), base = smem + s * kStage;
                const uint32_t sf = base + 2 * (kA + kB);
                if (elected) {
                    if (rank == 0) mbar_expect_tx(smem_u32(&full_bar[s]), 2 * kStage);
                    tma_load_2d_pair(base, &tmap_a, bar, 2 * kb * kBKBytes, a_row);
                    tma_load_2d_pair(base + 2 * kA, &tmap_b, bar, 2 * kb * kBKBytes, b_row);
                    tma_load_3d_pair(sf, &tmap_sa, bar, 0, 4 * kb, tm);
                    tma_load_3d_pair(sf + kSA, &tmap_sb, bar, 0, 4 * kb, tn * (BN / 128));
                    tma_load_2d_pair(base + kA, &tmap_a, bar, (2 * kb + 1) * kBKBytes, a_row);
                    tma_load_2d_pair(base + 2 * kA + kB, &tmap_b, bar, (2 * kb + 1) * kBKBytes, b_row);
                }
                issued++;
                if (++s == p.stages) s = 0, ph ^= 1;
            }
        }
        // the last copies into each stage have landed before the pair ends
        for (int i = 0; rank == 0 && i < min(issued, p.stages); i++) {
            if (--s < 0) s = p.stages - 1, ph ^= 1;
            drain_phase(smem_u32(&full_bar[s]), ph, p.wait_cap_ns);
        }
    } else if (warp == 2 && rank == 0) {
        // each stage's scales into both CTAs' tensor memory, ahead of the products (a
        // thread of its own: copies that the issuing thread puts between its products
        // hold these up, 0.58 instead of 0.40 us per 256 x 256 x 256)
        const uint32_t elected = elect_one();
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int tile = pair; ok && tile < p.tiles; tile += pairs) {
            for (int kb = kb0; kb < kb1; kb++) {
                if (!wait_warp(smem_u32(&full_bar[s]), ph, p.wait_cap_ns, p.err, abort_flag, 22)) {
                    ok = false;
                    break;
                }
                const uint32_t sf = smem + s * kStage + 2 * (kA + kB);
                const uint32_t sfa = sf_cols + s * kScaleCols, sfb = sfa + 16;
                const int chunks = min(4, p.tiles_k - 4 * kb);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    if (c >= chunks) break;
                    tc_cp_scales<2>(elected, sfa + c * 4, smem_desc_noswz(sf + c * 512, 16, 128));
#pragma unroll
                    for (int j = 0; j < BN / 128; j++)
                        tc_cp_scales<2>(elected, sfb + c * (BN / 32) + j * 4, smem_desc_noswz(sf + kSA + j * 2048 + c * 512, 16, 128));
                }
                tc_commit2(elected, smem_u32(&sf_bar[s]));
                if (++s == p.stages) s = 0, ph ^= 1;
            }
        }
        tc_commit2(elected, smem_u32(&drain_bar[1]));
        drain_phase(smem_u32(&drain_bar[1]), 0, p.wait_cap_ns);
    } else if (warp == 1 && rank == 0) {
        // a commit costs the tensor pipe about 0.1 us, so a stage is 512 wide: eight products
        const uint32_t elected = elect_one();
        const uint64_t hi = ((uint64_t)((8 * kBKBytes) >> 4) << 32) | (1ull << 46) | (2ull << 61);
        int s = 0, acc = 0;
        uint32_t ph = 0, aph = 0;
        bool ok = true;
        for (int tile = pair; ok && tile < p.tiles; tile += pairs) {
            if (!wait_warp(smem_u32(&tempty_bar[acc]), aph ^ 1u, p.wait_cap_ns, p.err, abort_flag, 23)) break;
            const uint32_t d = tmem + acc * BN;
            for (int kb = kb0; kb < kb1; kb++) {
                if (!wait_warp(smem_u32(&sf_bar[s]), ph, p.wait_cap_ns, p.err, abort_flag, 24)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t base = smem + s * kStage;
                const uint32_t sfa = sf_cols + s * kScaleCols, sfb = sfa + 16;
                const int chunks = min(4, p.tiles_k - 4 * kb);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    if (c >= chunks) break;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t off = (uint32_t)((c & 1) * 2 + h) * 32;
                        tc_mma_mxf4<2>(elected, d, smem_desc(base + (c >> 1) * kA + off, hi),
                                       smem_desc(base + 2 * kA + (c >> 1) * kB + off, hi), mx_idesc(2 * kBM, BN, h), sfa + c * 4,
                                       sfb + c * (BN / 32), (kb > kb0 || c || h) ? 1u : 0u);
                    }
                }
                tc_commit2_both(elected, smem_u32(&empty_bar[s]), both);
                if (++s == p.stages) s = 0, ph ^= 1;
            }
            if (!ok) break;
            tc_commit2_both(elected, smem_u32(&tfull_bar[acc]), both);
            if (++acc == kAcc) acc = 0, aph ^= 1;
        }
        tc_commit2(elected, smem_u32(&drain_bar[0]));
        drain_phase(smem_u32(&drain_bar[0]), 0, p.wait_cap_ns);
    } else if (warp >= 4) {
        const int quarter = warp & 3;  // tensor-memory lanes this warp may read
        const int part = (warp - 4) >> 2;
        int acc = 0;
        uint32_t aph = 0;
        for (int tile = pair; tile < p.tiles; tile += pairs) {
            const int tm = tile % p.tiles_m, tn = tile / p.tiles_m;
            if (!__all_sync(0xffffffffu, wait_phase(smem_u32(&tfull_bar[acc]), aph, p.wait_cap_ns, p.err, abort_flag, 26))) break;
            tc_fence_after();
            const size_t row = ((size_t)tm * 2 + rank) * kBM + quarter * 32 + lane;
            const size_t col0 = (size_t)tn * BN + part * kCols;
            const uint32_t base = tmem + acc * BN + part * kCols + ((uint32_t)(quarter * 32) << 16);
            uint32_t r[kCols / 32][32];
#pragma unroll
            for (int g = 0; g < kCols / 32; g++) tc_ld32(base + g * 32, r[g]);
            tc_wait_ld();
            if (BN == 128 && S > 1) {  // the cluster's only tile: the partial sums, over the ring (all of it has been read)
#pragma unroll
                for (int g = 0; g < kCols / 32; g++)
#pragma unroll
                    for (int i = 0; i < 32; i++) partial[(part * kCols + g * 32 + i) * 128 + quarter * 32 + lane] = __uint_as_float(r[g][i]);
                break;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(peer_addr(smem_u32(&tempty_bar[acc]), lead));
            if (++acc == kAcc) acc = 0, aph ^= 1;
            if (col0 >= p.n) continue;
            uint32_t scales = 0;
#pragma unroll
            for (int g = 0; g < kCols / 32; g++) {
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[g][i]);
                const size_t col = col0 + g * 32;
                finish32(v, col, p);
                uint32_t sb = 0;
                put32<kOut>(v, row, col, p, sb);
                scales |= sb << (8 * g);
            }
            if constexpr (kOut == 3) put_scales<kCols / 32>(scales, row, col0 / 32, p);
        }
    }
    __syncwarp();
    tc_fence_before();
    if (BN != 128 || S == 1) {
        cluster_sync_relaxed();  // all products and copies are done
    } else {
        cluster_sync();  // the same, and the partial sums lie ready
        // each pair adds up BN / S columns of the partial tiles, in the order of the pairs
        const int w = warp - 4, quarter = w & 3, group = w >> 2;
        if (w >= 0 && group < (int)(BN / 32 / S) && *abort_flag == 0) {
            const int tm = pair % p.tiles_m, tn = pair / p.tiles_m;
            const int c0 = (int)(part_k * (BN / S)) + group * 32;
            const size_t row = ((size_t)tm * 2 + rank) * kBM + quarter * 32 + lane, col = (size_t)tn * BN + c0;
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; i++) v[i] = 0.0f;
            for (uint32_t q = 0; q < S; q++) {
                const uint32_t from = peer_addr(smem_u32(partial + c0 * 128 + quarter * 32 + lane), 2 * q + rank);
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    float u;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(u) : "r"(from + i * 512) : "memory");
                    v[i] += u;
                }
            }
            if (col < p.n) {
                finish32(v, col, p);
                uint32_t sb = 0;
                put32<kOut>(v, row, col, p, sb);
                if constexpr (kOut == 3) put_scales<1>(sb, row, col / 32, p);
            }
        }
        cluster_sync_relaxed();  // no CTA leaves while its partial sums may be read
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ---- few rows ------------------------------------------------------------------
// The weights take the tensor core's 128-row side and the m rows of A its column
// side (bn = 16, 32, 64 or 128 of them), so a tile's result is 128 outputs x bn
// rows.  K is split over the CTAs of a cluster, which leave their partial tiles in
// shared memory, and each of them adds up every S-th row of A in the order of the
// ranks: no workspace, no atomics, the same bits each time.
struct SkinnyParams {
    const float *bias;
    void *y;
    uint8_t *y_s;
    size_t m, n;
    size_t out_nb, out_tiles;
    int tiles_k, k_blocks, bn, stages, act, out;  // out: DW_F32 .. DW_BF16, 3: MXFP4
    uint32_t stage_bytes, idesc[2], tmem_cols;
    bool vec;  // y is aligned for stores of four outputs
    uint64_t wait_cap_ns;
    int32_t *err;
};

constexpr int kSkinnyThreads = 256;
constexpr int kSkinnyStages = 8;

__device__ __forceinline__ float4 ld_peer4(uint32_t addr, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(peer_addr(addr, rank))
                 : "memory");
    return v;
}

__global__ void __launch_bounds__(kSkinnyThreads)
    k_mxfp4_skinny(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a,
                   const __grid_constant__ CUtensorMap tmap_sw, const __grid_constant__ CUtensorMap tmap_sa,
                   const __grid_constant__ SkinnyParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    float *part = reinterpret_cast<float *>(smem_raw + (smem - smem_u32(smem_raw)));  // [bn][128], over the ring
    __shared__ uint64_t full_bar[kSkinnyStages], sf_bar[kSkinnyStages], empty_bar[kSkinnyStages], done_bar, drain_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), S = cluster_size();
    const size_t n0 = (size_t)blockIdx.y * 128;
    const int kb0 = (int)((long long)p.k_blocks * rank / S), kb1 = (int)((long long)p.k_blocks * (rank + 1) / S);
    const uint32_t w_bytes = kBM * kBKBytes, a_bytes = (uint32_t)p.bn * kBKBytes;

    if (threadIdx.x == 32 * 3) {
        prefetch_map(&tmap_w), prefetch_map(&tmap_a), prefetch_map(&tmap_sw), prefetch_map(&tmap_sa);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; s++) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&sf_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        mbar_init(smem_u32(&done_bar), 1);
        mbar_init(smem_u32(&drain_bar), 1);
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(p.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_wait();  // in every warp: the bounded waits count from here
    pdl_trigger();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
    const uint32_t sf_cols = tmem + (uint32_t)p.bn;  // 16 columns a stage after the accumulators
    const uint64_t hi = ((uint64_t)((8 * kBKBytes) >> 4) << 32) | (1ull << 46) | (2ull << 61);

    if (warp == 0) {
        const uint32_t elected = elect_one();
        int s = 0, issued = 0;
        uint32_t ph = 0;
        for (int kb = kb0; kb < kb1; kb++) {
            if (issued >= p.stages && !wait_warp(smem_u32(&empty_bar[s]), ph ^ 1u, p.wait_cap_ns, p.err, abort_flag, 31)) break;
            const uint32_t bar = smem_u32(&full_bar[s]), base = smem + s * p.stage_bytes;
            if (elected) {
                mbar_expect_tx(bar, p.stage_bytes);
                tma_load_2d(base, &tmap_w, bar, kb * kBKBytes, (int)n0);
                tma_load_3d(base + w_bytes, &tmap_sw, bar, 0, 2 * kb, (int)blockIdx.y);
                tma_load_2d(base + w_bytes + 1024, &tmap_a, bar, kb * kBKBytes, 0);
                tma_load_3d(base + w_bytes + 1024 + a_bytes, &tmap_sa, bar, 0, 2 * kb, 0);
            }
            issued++;
            if (++s == p.stages) s = 0, ph ^= 1;
        }
        for (int i = 0; i < min(issued, p.stages); i++) {
            if (--s < 0) s = p.stages - 1, ph ^= 1;
            drain_phase(smem_u32(&full_bar[s]), ph, p.wait_cap_ns);
        }
    } else if (warp == 2) {
        // scales of each stage into tensor memory, ahead of the products
        const uint32_t elected = elect_one();
        int s = 0;
        uint32_t ph = 0;
        for (int kb = kb0; kb < kb1; kb++) {
            if (!wait_warp(smem_u32(&full_bar[s]), ph, p.wait_cap_ns, p.err, abort_flag, 32)) break;
            const uint32_t base = smem + s * p.stage_bytes + w_bytes;
            const int chunks = min(2, p.tiles_k - 2 * kb);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                if (c >= chunks) break;
                tc_cp_scales<1>(elected, sf_cols + s * 16 + c * 4, smem_desc_noswz(base + c * 512, 16, 128));
                tc_cp_scales<1>(elected, sf_cols + s * 16 + 8 + c * 4, smem_desc_noswz(base + 1024 + a_bytes + c * 512, 16, 128));
            }
            tc_commit1(elected, smem_u32(&sf_bar[s]));
            if (++s == p.stages) s = 0, ph ^= 1;
        }
        tc_commit1(elected, smem_u32(&drain_bar));
        drain_phase(smem_u32(&drain_bar), 0, p.wait_cap_ns);
    } else if (warp == 1) {
        const uint32_t elected = elect_one();
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; kb++) {
            if (!wait_warp(smem_u32(&sf_bar[s]), ph, p.wait_cap_ns, p.err, abort_flag, 33)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t base = smem + s * p.stage_bytes;
            const int chunks = min(2, p.tiles_k - 2 * kb);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                if (c >= chunks) break;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t off = (uint32_t)(c * 2 + h) * 32;
                    tc_mma_mxf4<1>(elected, tmem, smem_desc(base + off, hi), smem_desc(base + w_bytes + 1024 + off, hi), p.idesc[h],
                                   sf_cols + s * 16 + c * 4, sf_cols + s * 16 + 8 + c * 4, (kb > kb0 || c || h) ? 1u : 0u);
                }
            }
            tc_commit1(elected, smem_u32(&empty_bar[s]));
            if (++s == p.stages) s = 0, ph ^= 1;
        }
        tc_commit1(elected, smem_u32(&done_bar));
        if (!ok) drain_phase(smem_u32(&done_bar), 0, p.wait_cap_ns);
    }
    __syncwarp();
    if (warp >= 4) {
        // accumulators -> part[row of A][output]
        const int quarter = warp & 3;
        if (__all_sync(0xffffffffu, wait_phase(smem_u32(&done_bar), 0, p.wait_cap_ns, p.err, abort_flag, 34))) {
            tc_fence_after();
            const uint32_t base = tmem + ((uint32_t)(quarter * 32) << 16);
            const int cols = (int)p.m;
            for (int c0 = 0; c0 < cols; c0 += 16) {
                int32_t r[16];
                tc_ld16(base + c0, r);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (c0 + i < cols) part[(c0 + i) * 128 + quarter * 32 + lane] = __int_as_float(r[i]);
            }
        }
    }
    tc_fence_before();
    if (S > 1)
        cluster_sync();
    else
        __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
    }
    if (*abort_flag == 0) {
        // a warp takes a row of A, a lane four neighbouring outputs
        const size_t col = n0 + 4 * lane;
        float bias[4];
#pragma unroll
        for (int i = 0; i < 4; i++) bias[i] = p.bias && col + i < p.n ? p.bias[col + i] : 0.0f;
        const int rows = (int)p.m;
        for (int j = (int)rank + (int)S * warp; j < rows; j += (kSkinnyThreads / 32) * (int)S) {
            const uint32_t addr = smem_u32(part + j * 128 + 4 * lane);
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            float4 u[8];
#pragma unroll
            for (uint32_t r = 0; r < 8; r++)
                if (r < S) u[r] = ld_peer4(addr, r);
#pragma unroll
            for (uint32_t r = 0; r < 8; r++)
                if (r < S) v[0] += u[r].x, v[1] += u[r].y, v[2] += u[r].z, v[3] += u[r].w;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = activate(v[i] + bias[i], p.act);
            const size_t row = j;
            if (p.out == 3) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (col + i >= p.n) v[i] = 0.0f;
                uint32_t amax = mx_amax(v);
#pragma unroll
                for (int o = 4; o; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                const uint32_t sb = mx_scale_byte(amax);
                const float inv = mx_inv_scale(sb);
                const size_t block = col / 32;
                const uint32_t codes = mx_codes2(v[0] * inv, v[1] * inv) | (mx_codes2(v[2] * inv, v[3] * inv) << 8);
                if (block < p.out_nb)
                    *reinterpret_cast<uint16_t *>((uint8_t *)p.y + (row * p.out_nb * 32 + col) / 2) = sb == 0xFFu ? 0 : (uint16_t)codes;
                if ((lane & 7) == 0 && block < p.out_tiles * 4) p.y_s[mx_scale_at(row, block, p.out_tiles)] = (uint8_t)sb;
            } else {
                auto store = [&](auto *y) {
                    using T = std::remove_pointer_t<decltype(y)>;
                    y += row * p.n + col;
                    if (p.vec && col + 4 <= p.n) {
                        Raw<T, 4> r;
                        r.set(v);
                        r.store(y);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (col + i < p.n) y[i] = from_f32<T>(v[i]);
                    }
                };
                if (p.out == DW_F32)
                    store((float *)p.y);
                else if (p.out == DW_F16)
                    store((__half *)p.y);
                else
                    store((__nv_bfloat16 *)p.y);
            }
        }
    }
    if (S > 1) cluster_sync_relaxed();  // no CTA leaves while its partials may be read
}

// Codes as a 2-D byte tensor [rows][bytes of a row]; a box is 128 bytes of `box_rows` rows.
bool code_map(dw_backend *be, CUtensorMap *map, const uint8_t *q, size_t rows, size_t k, int box_rows) {
    cuuint64_t dims[2] = {(cuuint64_t)mx_blocks(k) * 16, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)mx_blocks(k) * 16};
    cuuint32_t box[2] = {(cuuint32_t)kBKBytes, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return be->encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(q), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Scales as a 3-D tensor [row tiles][tiles along K][512 bytes]; a box is
// `k_tiles` tiles along K of `row_tiles` row tiles.
bool scale_map(dw_backend *be, CUtensorMap *map, const uint8_t *s, size_t rows, size_t k, int k_tiles, int row_tiles) {
    cuuint64_t dims[3] = {128, (cuuint64_t)mx_tiles(k), (cuuint64_t)((rows + 127) / 128)};
    cuuint64_t strides[2] = {512, (cuuint64_t)mx_tiles(k) * 512};
    cuuint32_t box[3] = {128, (cuuint32_t)k_tiles, (cuuint32_t)row_tiles};
    cuuint32_t estr[3] = {1, 1, 1};
    return be->encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<uint8_t *>(s), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, int kOut>
dw_status launch(dw_backend *be, const MxGemmArgs &a, int S) {
    constexpr size_t kStage = 2 * (kBM + BN / 2) * kBKBytes + 2048 + (BN / 128) * 2048;
    GemmParams p{};
    p.bias = a.bias, p.y = a.y, p.y_s = a.y_s;
    p.m = a.m, p.n = a.n;
    p.tiles_k = (int)mx_tiles(a.k);
    p.out_nb = mx_blocks(a.n), p.out_tiles = mx_tiles(a.n);
    p.k_blocks = (int)((a.k + 511) / 512);
    const size_t tm = (a.m + 2 * kBM - 1) / (2 * kBM), tn = (a.n + BN - 1) / BN;
    if (tm * tn > 0x7fff0000u) return dw_fail(be, DW_ERR_UNSUPPORTED, "gemm_mxfp4: %zu x %zu is too large", a.m, a.n);
    p.tiles_m = (int)tm, p.tiles = (int)(tm * tn);
    p.act = a.act;
    const size_t es = kOut == 0 ? 4 : 2;
    p.vec = ((uintptr_t)a.y & 15) == 0 && a.n * es % 16 == 0;
    p.bias_vec = ((uintptr_t)a.bias & 15) == 0;
    p.wait_cap_ns = be->wait_cap_ns, p.err = be->dev_err;
    p.stages = (int)std::min<size_t>(kMaxStages, (kSmemLimit - 4096) / kStage);
    // at least 116 KiB: one CTA per SM owns the tensor memory
    // and the partial tile of a split K lies over the ring
    const size_t smem = std::max<size_t>(1024 + std::max<size_t>(p.stages * kStage, BN * 512), 116 * 1024);
    CUtensorMap ta, tb, tsa, tsb;
    if (!be->encode_tiled || !code_map(be, &ta, a.a_q, a.m, a.k, kBM) || !code_map(be, &tb, a.b_q, a.n, a.k, BN / 2) ||
        !scale_map(be, &tsa, a.a_s, a.m, a.k, 4, 1) || !scale_map(be, &tsb, a.b_s, a.n, a.k, 4, BN / 128))
        return dw_fail(be, DW_ERR_DEVICE, "gemm_mxfp4: tensor map rejected");
    auto kernel = k_mxfp4_gemm<BN, kOut>;
    static bool attr_set[16] = {};
    if (be->device < 16 && !attr_set[be->device]) {
        dw_status st = dw_cuda_check(
            be, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kSmemLimit - 2048)),
            "gemm_mxfp4 attributes");
        if (st != DW_OK) return st;
        attr_set[be->device] = true;
    }
    return launch_dependent(be, "gemm_mxfp4", kernel, 2 * S * (S > 1 ? p.tiles : std::min(p.tiles, be->sm_count / 2)), kGemmThreads,
                            smem, 2 * S, ta, tb, tsa, tsb, p);
}

dw_status launch_skinny(dw_backend *be, const MxGemmArgs &a) {
    SkinnyParams p{};
    p.bias = a.bias, p.y = a.y, p.y_s = a.y_s;
    p.m = a.m, p.n = a.n;
    p.tiles_k = (int)mx_tiles(a.k);
    p.out_nb = mx_blocks(a.n), p.out_tiles = mx_tiles(a.n);
    p.k_blocks = (int)((a.k + 255) / 256);
    p.bn = a.m <= 16 ? 16 : a.m <= 32 ? 32 : a.m <= 64 ? 64 : 128;
    p.act = a.act, p.out = a.y_s ? 3 : a.y_dtype;
    p.vec = a.n % 4 == 0 && (uintptr_t)a.y % (a.y_dtype == DW_F32 ? 16 : 8) == 0;
    p.stage_bytes = kBM * kBKBytes + 1024 + p.bn * kBKBytes + 1024;
    for (int h = 0; h < 2; h++) p.idesc[h] = mx_idesc(128, p.bn, h);
    const int per_sm = p.bn <= 64 ? 2 : 1;  // CTAs whose rings an SM holds
    p.wait_cap_ns = be->wait_cap_ns, p.err = be->dev_err;
    const size_t tn = (a.n + 127) / 128;
    // CTAs that share a tile's K: about one an SM (4096 outputs, K 4096, one row: S = 1, 2,
    // 4, 8 took 5.5, 4.4, 4.2, 4.6 us; 11008 outputs S = 1, 2, 4: 6.2, 6.2, 8.1), each with
    // a K block at least; clusters of 8 CTAs that fill an SM each do not fit 16 at a time
    unsigned S = 1;
    const unsigned most = per_sm == 2 ? 8 : 4;
    while (S < most && 2 * S * tn <= (size_t)be->sm_count * 4 / 3 && 2 * (int)S <= p.k_blocks) S *= 2;
    // The ring: no longer than a CTA's K blocks, and of at most three stages where the CTAs
    // outnumber the SMs and have few blocks each: a third of them then fits beside two others,
    // or the next launch's (11008 outputs, K 4096, one row 6.4 -> 5.5 us; 65536 outputs, K 256,
    // where a ring of three stages would hold two that nothing fills: 5.2 -> 4.5 us)
    const int own = (p.k_blocks + (int)S - 1) / (int)S;
    p.stages = (int)std::min<size_t>(kSkinnyStages, ((kSmemLimit - 8192) / per_sm - 2048) / p.stage_bytes);
    p.stages = std::min(p.stages, p.bn <= 32 && S * tn > (size_t)be->sm_count && own <= 8 ? std::min(own, 3) : own);
    // Tensor memory: accumulators and 16 columns a stage.  A CTA takes no larger share of an
    // SM's 512 columns than of its shared memory, so those that fit together, of this launch
    // and others, find columns: none waits for another's, which might itself wait for a
    // CTA of the waiting one's cluster.
    p.tmem_cols = 32;
    while ((int)p.tmem_cols < p.bn + 16 * p.stages) p.tmem_cols *= 2;
    const size_t smem = std::max(1024 + std::max<size_t>(p.stages * p.stage_bytes, (size_t)p.bn * 512),
                                 kSmemSm * p.tmem_cols / 512);
    CUtensorMap tw, ta, tsw, tsa;
    if (!be->encode_tiled || !code_map(be, &tw, a.b_q, a.n, a.k, kBM) || !code_map(be, &ta, a.a_q, a.m, a.k, p.bn) ||
        !scale_map(be, &tsw, a.b_s, a.n, a.k, 2, 1) || !scale_map(be, &tsa, a.a_s, a.m, a.k, 2, 1))
        return dw_fail(be, DW_ERR_DEVICE, "gemm_mxfp4: tensor map rejected");
    static bool attr_set[16] = {};
    if (be->device < 16 && !attr_set[be->device]) {
        dw_status st = dw_cuda_check(be,
                                     cudaFuncSetAttribute(k_mxfp4_skinny, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                          (int)(kSmemLimit - 2048)),
                                     "gemm_mxfp4 attributes");
        if (st != DW_OK) return st;
        attr_set[be->device] = true;
    }
    return launch_dependent(be, "gemm_mxfp4", k_mxfp4_skinny, dim3(S, (unsigned)tn), kSkinnyThreads, smem, S, tw, ta,
                            tsw, tsa, p);
}

}  // namespace

// Which kernel, tile and split of K (times on B200, launches in a row on the same operands
// unless said, us; between the shapes named the rules are not measured):
//   few rows: up to 64 (m 64, n 11008, k 4096: 7.7 against 9.5), or up to 128 where the
//     pairs would have few tiles of a long K (m 128, k 4096: n 1000 5.8 against 7.0, n 4096
//     6.9 against 6.5; k 11008, n 4096: 8.9 against 10.3);
//   256 x 256 tiles once they fill the pairs (other operands each time: 4096^3 30.6 against
//     32.8, 2048 x 4096 x 4096 17.7 against 19.0), 256 x 128 below, whose accumulators are
//     double-buffered and whose last round is shorter (256 x 11008 x 4096 12.2 against 13.4);
//   two pairs for each tile's K when both fit at once and K is long (256 x 4096 x 11008
//     10.4 against 11.0; with k 4096 7.8 against 6.6).
dw_status launch_gemm_mxfp4(dw_backend *be, const MxGemmArgs &a) {
    const size_t pairs = (size_t)be->sm_count / 2, rows = (a.m + 255) / 256, k_blocks = (a.k + 511) / 512;
    const bool few = a.n <= 65535ull * 128;  // outputs that the few-rows grid holds
    if (few && (a.m <= 64 || (a.m <= 128 && a.n <= 4096 && a.k > 4096) || (a.m <= 128 && a.n <= 1024 && a.k >= 2048)))
        return launch_skinny(be, a);
    const bool wide = rows * ((a.n + 255) / 256) >= pairs;
    const int S = !wide && rows * ((a.n + 127) / 128) <= pairs / 2 - 1 && k_blocks >= 16 ? 2 : 1;
    switch ((wide ? 4 : 0) + (a.y_s ? 3 : a.y_dtype)) {
        case 0: return launch<128, 0>(be, a, S);
        case 1: return launch<128, 1>(be, a, S);
        case 2: return launch<128, 2>(be, a, S);
        case 3: return launch<128, 3>(be, a, S);
        case 4: return launch<256, 0>(be, a, S);
        case 5: return launch<256, 1>(be, a, S);
        case 6: return launch<256, 2>(be, a, S);
        default: return launch<256, 3>(be, a, S);
    }
}

}  // namespace dw
