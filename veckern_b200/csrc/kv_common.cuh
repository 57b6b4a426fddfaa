// Shared by the kernels of the paged key/value cache: the views that they get by value, the sequences' bounds, and the
// 16-bit types' conversions.
//
// What a call reads from device memory (offsets, lengths, page numbers) is never trusted: a sequence's bounds are
// clamped to the call's sizes and a page number outside the cache is not followed. Both set ERR_LAYOUT.
//
// These kernels start while the kernel before them on the stream still runs, and wait for its results inside. What that one
// may have written (anything: lengths from an eviction, rows from an attention, scores, lse) must not be read through the
// read-only path, which is for memory that nobody writes while the kernel lives: __ldca, which stays behind the wait, and no
// __ldg.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "vk_device.cuh"

namespace vk {

enum : int { ERR_WORKSPACE = 8 };  // status bit: the call's workspace is one that a wait that ran out has left as it was

struct KvPages {
    uint16_t* k;  // elements of the cache's 16-bit type
    uint16_t* v;
    int64_t ks[3], vs[3];  // strides in elements: page, slot, head
    int64_t pages;
    int page_shift;  // page size = 1 << page_shift
    int heads, dim;
    int* status;
};

struct KvBatch {
    const int32_t* offsets;
    const int32_t* table;
    const int32_t* lens;
    int64_t table_stride;
    int64_t tokens;
    int batch;
    int width;
};

struct KvSeq {
    int64_t first;  // row of its first new token
    int count;      // new tokens
    int len;        // slots, new tokens included
};

// The checks come behind all loads, which then wait for one another's latency only.
__device__ __forceinline__ int kv_len_checked(const KvPages& c, const KvBatch& bt, int len) {
    const int64_t most = (int64_t)bt.width << c.page_shift;
    if (len < 0 || len > most) {
        atomicOr(c.status, ERR_LAYOUT);
        len = len < 0 ? 0 : (int)most;
    }
    return len;
}
__device__ __forceinline__ int kv_len(const KvPages& c, const KvBatch& bt, int b) {
    return kv_len_checked(c, bt, __ldca(bt.lens + b));
}

__device__ __forceinline__ KvSeq kv_seq(const KvPages& c, const KvBatch& bt, int b) {
    int64_t lo = __ldca(bt.offsets + b), hi = __ldca(bt.offsets + b + 1);
    const int len = __ldca(bt.lens + b);
    if (lo < 0 || hi < lo || hi > bt.tokens) {
        atomicOr(c.status, ERR_LAYOUT);
        lo = min(max(lo, int64_t(0)), bt.tokens);
        hi = min(max(hi, lo), bt.tokens);
    }
    return {lo, (int)(hi - lo), kv_len_checked(c, bt, len)};
}

// The table's entry for a slot (slot < the sequence's length), and the page that it names, or -1.
__device__ __forceinline__ int kv_entry(const KvPages& c, const int32_t* table, int slot) {
    return __ldca(table + (slot >> c.page_shift));
}
__device__ __forceinline__ int64_t kv_page_checked(const KvPages& c, int page) {
    if ((uint64_t)(int64_t)page >= (uint64_t)c.pages) {
        atomicOr(c.status, ERR_LAYOUT);
        return -1;
    }
    return page;
}
__device__ __forceinline__ int64_t kv_page(const KvPages& c, const int32_t* table, int slot) {
    return kv_page_checked(c, kv_entry(c, table, slot));
}

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
    if constexpr (std::is_same_v<T, __half>) return __half2float(x);
    else return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
    if constexpr (std::is_same_v<T, __half>) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}

// Sequence of a token row: the last b whose offset is at most it (offsets ascend; empty sequences share one).
__device__ __forceinline__ int kv_find(const KvBatch& bt, int64_t row) {
    int lo = 0, hi = bt.batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldca(bt.offsets + mid) <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Division of 0 <= x < 2^31 by a number that a whole call shares: a multiplication by 2^(32 + shift) / by, rounded up
// (Granlund and Montgomery, "Division by invariant integers using multiplication").
struct Divisor {
    uint32_t by, mul;
    int shift;
    __host__ static Divisor of(uint32_t by) {
        int shift = 0;
        while ((uint64_t(1) << shift) < by) ++shift;
        // 2^shift >= by: the quotient fits 33 bits, its leading bit is left out and added back as x itself
        const uint64_t m = ((uint64_t(1) << 32) * ((uint64_t(1) << shift) - by)) / by + 1;
        return {by, (uint32_t)m, shift};
    }
    __host__ __device__ __forceinline__ uint32_t operator()(uint32_t x) const {
#ifdef __CUDA_ARCH__
        const uint32_t high = __umulhi(x, mul);
#else
        const uint32_t high = (uint32_t)((uint64_t)x * mul >> 32);
#endif
        return (uint32_t)(((uint64_t)high + x) >> shift);
    }
};

struct KvAttend {
    const uint16_t* q;
    uint16_t* out;
    float* lse;     // [tokens][heads]
    float* scores;  // may be null
    int64_t qs[2], os[2], ss[2];
    int64_t scores_width;
    int heads, group;  // query heads; query heads per kv head
    int tokens;        // of a chunk's row tile
    Divisor by_group, by_tokens, by_pair;  // group, tokens, 2 tokens
    int max_q;
    int causal;
    float scale;
    long long wait_limit;  // cycles
};

}  // namespace vk
