// dw_attend.cuh -- what the attention kernels share: their arguments and the tokens a row sees.
#pragma once

#include <cstdint>

#include "dw_kv.cuh"

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

// A bf16 query row goes to f16 times 2^-e, which puts its largest magnitude `top` into
// [2^14, 2^15): nothing overflows and what falls below f16's smallest step is 2^-39 of it.
__device__ __forceinline__ int query_exponent(float top) {
    return min(max((int)(__float_as_uint(top) >> 23) - 127 - 14, -126), 126);
}

// attention_prompt.cu
template <typename T, int D>
dw_status attend_prompt(dw_backend *be, AttendParams p, const KvCache &c, const Seqs &s);

}  // namespace dw
