// dw_kv.cuh -- device helpers of the paged 8-bit key/value cache: which rows and tokens a
// sequence has, where its pages lie, and the e4m3 codes.
//
// A block (a page's tokens of one head) has one scale X = 2^e for its keys and one for its
// values, held as the byte e + 127, e in [-64, 63].  The bounds keep every exponent that
// attention forms from two of them inside f32.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#include "dw_device.cuh"

namespace dw {

constexpr int kKvMinExp = -64, kKvMaxExp = 63;

__device__ __forceinline__ size_t kv_block(const KvCache &c, uint32_t page, int head) { return (size_t)page * c.heads + head; }
__device__ __forceinline__ uint8_t *kv_codes(uint8_t *codes, const KvCache &c, uint32_t page, int head) {
    return codes + kv_block(c, page, head) * (size_t)(c.page * c.d);
}
// A scale byte's exponent, whatever the byte.
__device__ __forceinline__ int kv_exponent(uint32_t byte) { return min(max((int)byte - 127, kKvMinExp), kKvMaxExp); }
__device__ __forceinline__ float kv_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The smallest e with amax <= 448 * 2^e; amax >= 0 finite, as f32 rounded to odd or exact
// (448 * 2^e has an even last bit, so the rounding does not move a value past it).
__device__ __forceinline__ int kv_scale_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);  // 448 = 1.75 * 2^8
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u);
    return min(max(e, kKvMinExp), kKvMaxExp);
}

// Two f32 -> e4m3 codes (the first in the low byte), to nearest even, 448 at most, NaN 0x7F.
__device__ __forceinline__ uint32_t e4m3_codes2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(a), "f"(b));
    return r;
}
// The two codes of a half word as f16 values (exact).
__device__ __forceinline__ uint32_t e4m3_to_f16x2(uint16_t c) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
    return r;
}
__device__ __forceinline__ float2 e4m3_to_f32x2(uint16_t c) {
    const uint32_t r = e4m3_to_f16x2(c);
    __half2 h;
    memcpy(&h, &r, 4);
    return __half22float2(h);
}

// ---- sequences -----------------------------------------------------------------
struct SeqRange {
    int row0, n;  // its rows
    int len;      // its tokens in the cache
    bool ok;      // neither had to be brought into bounds
    __device__ __forceinline__ int position(int row) const { return len - n + (row - row0); }
};

__device__ __forceinline__ int seq_start(const Seqs &q, uint32_t s) {
    if (!q.starts) return (int)(s * (q.tokens / q.seqs));
    return min(max(q.starts[s], 0), (int)q.tokens);
}

// The rows of a sequence, its starts checked (ok: not changed where they are in order).
__device__ __forceinline__ int seq_rows(const Seqs &q, uint32_t s, int &row0, int32_t *err, bool &ok) {
    row0 = seq_start(q, s);
    const int end = seq_start(q, s + 1);
    if (q.starts && (end < row0 || q.starts[s] != row0 || q.starts[s + 1] != end)) {
        record_error(err, DW_DEV_BAD_ARG, 61, (int)s);
        ok = false;
    }
    return max(end - row0, 0);
}
__device__ __forceinline__ int seq_rows(const Seqs &q, uint32_t s, int &row0, int32_t *err) {
    bool ok = true;
    return seq_rows(q, s, row0, err, ok);
}
// Whether the starts around a sequence's own leave its rows to it alone: where starts descend, the
// sequences on both sides may claim the same rows, and which of them is wrong is not known.
__device__ __forceinline__ bool seq_apart(const Seqs &q, uint32_t s) {
    if (!q.starts) return true;
    return (s == 0 || q.starts[s - 1] <= q.starts[s]) && (s + 2 > q.seqs || q.starts[s + 1] <= q.starts[s + 2]);
}

__device__ __forceinline__ bool bad_start(const Seqs &q, int64_t s) {
    if (!q.starts || s >= q.seqs) return false;
    const int a = q.starts[s], b = q.starts[s + 1];
    return a < 0 || a > b || (uint32_t)b > q.tokens;
}

// Where starts descend, the search for an item's sequence comes to some sequences by no item, so the
// items look through all starts as well: the lanes of item w at the 32 of its share (items are as
// many as sequences at least; below 0: no share).
__device__ __forceinline__ SeqRange seq_range(const Seqs &q, uint32_t s, int page, int32_t *err, int64_t w) {
    SeqRange r;
    r.ok = true;
    const int most = (int)min((uint64_t)q.width * page, (uint64_t)0x7fffff00u), len = q.lens[s];
    const bool bad = w >= 0 && bad_start(q, w * 32 + (threadIdx.x & 31));
    r.n = seq_rows(q, s, r.row0, err, r.ok);
    r.len = min(max(len, 0), most);
    r.ok = r.ok && len == r.len;
    if (len != r.len || bad) record_error(err, DW_DEV_BAD_ARG, 61, (int)s);
    return r;
}

// Items of work, cut from each sequence's rows: sequence s owns the items from start(s) *
// per / size + extra * s on, which are at least floor(n * per / size) + extra.  A call launches
// as many as its totals allow (they are known on the host, the sequences' own are not);
// items that a sequence has too many are empty.
__host__ __device__ inline size_t seq_items(size_t tokens, size_t seqs, int per, int size, int extra) {
    return tokens * per / size + extra * seqs;
}
__host__ __device__ inline int64_t seq_first_item(int64_t start, uint32_t s, int per, int size, int extra) {
    return start * per / size + (int64_t)extra * s;
}
// Those of each sequence where all have n rows: blocks of `size` of n * per rows, or with extra = 2 the
// pages of `size` tokens that n rows can lie in, from anywhere in the first.
__host__ __device__ inline size_t seq_items_each(size_t n, int per, int size, int extra) {
    return extra == 2 ? (n + size - 2) / size + 1 : (n * per + size - 1) / size;
}
// The sequence of item w, by the items that sequences begin with, and its place there (below 0: of no
// sequence).  vote(f): the bits of f(0) .. f(31).
template <typename First, typename Vote>
__host__ __device__ __forceinline__ uint32_t find_item(uint32_t seqs, int64_t w, First first, Vote vote, int64_t &place) {
    uint32_t lo = 0, count = seqs;
    while (count > 1) {  // the last of 32 evenly spaced ones that does not start behind w
        const uint32_t step = (count + 31) / 32;
        const uint32_t mask = vote([&](uint32_t i) { return i * step < count && first(lo + i * step) <= w; }) | 1u;
#ifdef __CUDA_ARCH__
        const uint32_t k = 31 - __clz(mask);
#else
        const uint32_t k = 31 - __builtin_clz(mask);
#endif
        lo += k * step;
        count = count - k * step < step ? count - k * step : step;
    }
    place = w - first(lo);
    return lo;
}
// The same of a call's sequences; a whole warp calls.
__device__ __forceinline__ uint32_t seq_of_item(const Seqs &q, int64_t w, int per, int size, int extra, int64_t &place) {
    const uint32_t lane = threadIdx.x & 31;
    return find_item(
        q.seqs, w, [&](uint32_t s) { return seq_first_item(seq_start(q, s), s, per, size, extra); },
        [&](auto f) { return __ballot_sync(0xffffffffu, f(lane)); }, place);
}

// A sequence's page `index` (its tokens from index * page on) to read from, in bounds in any case.
__device__ __forceinline__ uint32_t seq_page(const Seqs &q, const KvCache &c, uint32_t s, uint32_t index, int32_t *err) {
    const uint32_t id = (uint32_t)q.table[(size_t)s * q.width + index];
    if (id < c.pages) return id;
    record_error(err, DW_DEV_BAD_ARG, 62, (int)s);
    return 0;
}

}  // namespace dw
