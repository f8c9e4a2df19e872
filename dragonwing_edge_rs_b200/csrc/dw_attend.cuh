// dw_attend.cuh -- what the attention kernels share: their arguments and the tokens a row sees.
#pragma once

#include <cstdint>

#include "dw_kv.cuh"
#include "dw_ptx.cuh"

namespace dw {

struct AttendParams {
    const void *q;
    void *out;
    size_t q_pitch, out_pitch;
    int group;         // query heads of a cache head
    int per_seq;       // blocks of rows of a sequence where all have as many; 0: by their starts
    uint32_t items;    // blocks of rows of all sequences
    float scale_log2;  // scale * log2(e)
    int causal, window;
    bool vec;          // rows allow 16-byte accesses
    uint64_t wait_cap_ns;
    int32_t *err;
};

struct Bounds {
    int lo, hi;
};
// The tokens that row `token` of a sequence's rows sees: [lo, hi).
__device__ __forceinline__ Bounds row_bounds(const AttendParams &p, const SeqRange &r, int token) {
    const int pos = r.len - r.n + token;
    Bounds b{0, r.len};
    if (p.causal) {
        b.hi = max(0, min(r.len, pos + 1));
        if (p.window) b.lo = max(0, pos + 1 - p.window);
    }
    return b;
}

// (x, y) -> the sums' factor where the maximum goes from x to y (-inf: nothing so far).
__device__ __forceinline__ float carry(float x, float y) { return x == y ? 1.0f : ex2_approx(x - y); }

// Weights cut to the 11 bits that f16 keeps, but with f32's exponents (a block of small values has
// weights far below f16's range that count in the sum of weights).  Both sums take these, so only
// what the cuts differ by between a row's tokens is an error, as much as of a rounding to nearest, and
// a row of one token is exact; with the uncut ones in the sum of weights it was half as much again.
// (f16 itself, for the products: weights times their block's scale, 2^ev, keep the 11 bits down to 2^-20
// of a row's largest, fewer down to 2^-31 and are 0 below, where they still count in the sum of weights.
// A block of so much larger values that has zeros in a channel therefore hides the others there.)
__device__ __forceinline__ float2 eleven_bits(float x, float y) {
    return make_float2(__uint_as_float(__float_as_uint(x) & ~0x1FFFu), __uint_as_float(__float_as_uint(y) & ~0x1FFFu));
}

// A bf16 query row goes to f16 times 2^-e, which puts its largest magnitude `top` into
// [2^14, 2^15): nothing overflows and what falls below f16's smallest step is 2^-39 of it.
__device__ __forceinline__ int query_exponent(float top) {
    return min(max((int)(__float_as_uint(top) >> 23) - 127 - 14, -126), 126);
}

// ---- sums of several CTAs -----------------------------------------------------------
// The CTAs of a cluster go through shares of a sequence's tokens and join their sums through
// shared memory, in the order of their ranks.
constexpr unsigned kMaxShare = 8;

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
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync_relaxed() {
    __syncwarp();
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


// Four values of a row's sum, and what to divide them by, over all CTAs: each has a maximum, the
// sum of the weights and sums of the values at these places.  (All loads at once: one after the
// other they took 2000 cycles.)
__device__ __forceinline__ float4 join_sums(const float *m_at, const float *l_at, const float *v_at, uint32_t S, float &l) {
    float pm[kMaxShare], pl[kMaxShare], m = -INFINITY;
    float4 pv[kMaxShare], v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (uint32_t k = 0; k < kMaxShare; k++)
        if (k < S) pm[k] = ld_peer(m_at, k), pl[k] = ld_peer(l_at, k), pv[k] = ld_peer4(v_at, k);
#pragma unroll
    for (uint32_t k = 0; k < kMaxShare; k++)
        if (k < S) m = fmaxf(m, pm[k]);
    l = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < kMaxShare; k++) {
        if (k >= S) continue;
        const float f = carry(pm[k], m);
        l = fmaf(pl[k], f, l);
        v.x = fmaf(pv[k].x, f, v.x), v.y = fmaf(pv[k].y, f, v.y), v.z = fmaf(pv[k].z, f, v.z), v.w = fmaf(pv[k].w, f, v.w);
    }
    return v;
}

// attention_prompt.cu
template <typename T, int D>
dw_status attend_prompt(dw_backend *be, AttendParams p, const KvCache &c, const Seqs &s);

}  // namespace dw
