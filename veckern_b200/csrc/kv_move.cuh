// The cache's kernels that move keys and values: append and evict.
#pragma once
#include "kv_common.cuh"

namespace vk {

// One thread per 16 bytes of a new token's head. Every byte is read and written once: bound by memory, by the launch
// for a step's few tokens.
__global__ void __launch_bounds__(256) kv_append_kernel(KvPages c, KvBatch bt, const uint16_t* k, const uint16_t* v,
                                                        int64_t k_tok, int64_t k_head, int64_t v_tok, int64_t v_head) {
    const int parts = c.dim >> 3;
    const int64_t all = bt.tokens * c.heads * parts;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x) {
        const int part = (int)(i % parts);
        const int64_t r = i / parts;
        const int head = (int)(r % c.heads);
        const int64_t tok = r / c.heads;
        const int b = kv_find(bt, tok);
        const KvSeq s = kv_seq(c, bt, b);
        if (tok < s.first || tok >= s.first + s.count) continue;  // rows outside every sequence
        const int slot = s.len - s.count + (int)(tok - s.first);
        if (slot < 0) {
            atomicOr(c.status, ERR_LAYOUT);
            continue;
        }
        const int64_t page = kv_page(c, bt.table + b * bt.table_stride, slot);
        if (page < 0) continue;
        const int in = slot & ((1 << c.page_shift) - 1);
        const uint4 kk = __ldg(reinterpret_cast<const uint4*>(k + tok * k_tok + head * k_head) + part);
        const uint4 vv = __ldg(reinterpret_cast<const uint4*>(v + tok * v_tok + head * v_head) + part);
        reinterpret_cast<uint4*>(c.k + page * c.ks[0] + in * c.ks[1] + head * c.ks[2])[part] = kk;
        reinterpret_cast<uint4*>(c.v + page * c.vs[0] + in * c.vs[1] + head * c.vs[2])[part] = vv;
    }
}

struct KvEvict {
    const int32_t* new_table;
    int64_t new_stride;
    int new_width;
    int keep, recent;
    const float* scores;
    int64_t ss[2];
    int64_t width;
    float* new_scores;
    int32_t* kept;
    int32_t* new_lens;
};

// Order of scores as unsigned integers: larger score, larger integer; NaN below everything, -0 as +0.
__device__ __forceinline__ uint32_t kv_rank(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int SELECT_THREADS = 1024;

// One block per (sequence, kv head) finds the slots to keep: the k - r largest ranks among the first n - r slots by a
// radix selection of four 8-bit digits (each pass counts the digit's values among the slots that match the digits
// found so far), then all kept slots in order.
__global__ void __launch_bounds__(SELECT_THREADS) kv_select_kernel(KvPages c, KvBatch bt, KvEvict e) {
    __shared__ int hist[256];
    __shared__ int warp_gt[32], warp_eq[32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int b = blockIdx.y, head = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = kv_len(c, bt, b);
    const int k = min(n, e.keep), r = min(e.recent, k), m = k - r, cand = n - r;
    const float* sc = e.scores + b * e.ss[0] + head * e.ss[1];
    int32_t* kept = e.kept + ((int64_t)b * c.heads + head) * e.keep;
    float* ns = e.new_scores + ((int64_t)b * c.heads + head) * e.width;
    auto score = [&](int slot) { return slot < e.width ? sc[slot] : 0.0f; };
    if (head == 0 && tid == 0) e.new_lens[b] = k;
    uint32_t prefix = 0, mask = 0;
    int need = m;  // still to be found among the slots that match the prefix
    if (m > 0 && m < cand) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < cand; i += SELECT_THREADS) {
                const uint32_t u = kv_rank(score(i));
                if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int left = need, d = 255;
                while (d > 0 && left > hist[d]) left -= hist[d--];
                s_prefix = prefix | ((uint32_t)d << shift);
                s_need = left;
            }
            __syncthreads();
            prefix = s_prefix;
            need = s_need;
            mask |= 255u << shift;
        }
    } else if (m == cand) {
        need = cand;  // everything ties with, or beats, rank 0
    } else {
        prefix = 0xffffffffu;  // m == 0: no rank is above this one, and none that ties is taken
    }
    // each warp takes a contiguous range of slots: count, then emit behind the ranges before it
    const int span = ((cand + 31) / 32 + 31) / 32 * 32, lo = min(cand, warp * span), hi = min(cand, lo + span);
    int gt = 0, eq = 0;
    for (int i = lo; i < hi; i += 32) {
        const uint32_t u = i + lane < hi ? kv_rank(score(i + lane)) : 0u;
        gt += __popc(__ballot_sync(FULL, i + lane < hi && u > prefix));
        eq += __popc(__ballot_sync(FULL, i + lane < hi && u == prefix));
    }
    if (lane == 0) {
        warp_gt[warp] = gt;
        warp_eq[warp] = eq;
    }
    __syncthreads();
    int before_gt = 0, before_eq = 0;
    for (int w = 0; w < warp; ++w) {
        before_gt += warp_gt[w];
        before_eq += warp_eq[w];
    }
    for (int i = lo; i < hi; i += 32) {
        const int slot = i + lane;
        const float x = slot < hi ? score(slot) : 0.0f;
        const uint32_t u = kv_rank(x);
        const unsigned mg = __ballot_sync(FULL, slot < hi && u > prefix);
        const unsigned me = __ballot_sync(FULL, slot < hi && u == prefix);
        const unsigned below = (1u << lane) - 1u;
        const int eq_before = before_eq + __popc(me & below);
        const bool mine = (mg >> lane & 1u) || ((me >> lane & 1u) && eq_before < need);
        if (mine) {
            const int at = before_gt + __popc(mg & below) + min(eq_before, need);
            kept[at] = slot;
            if (at < e.width) ns[at] = x;
        }
        before_gt += __popc(mg);
        before_eq += __popc(me);
    }
    for (int i = tid; i < r; i += SELECT_THREADS) {
        kept[m + i] = cand + i;
        if (m + i < e.width) ns[m + i] = score(cand + i);
    }
    for (int i = k + tid; i < e.keep; i += SELECT_THREADS) kept[i] = -1;
    for (int64_t i = k + tid; i < e.width; i += SELECT_THREADS) ns[i] = 0.0f;
}

// Copies the kept slots' keys and values; one thread per 16 bytes.
__global__ void __launch_bounds__(256) kv_compact_kernel(KvPages c, KvBatch bt, KvEvict e) {
    const int parts = c.dim >> 3, b = blockIdx.z, head = blockIdx.y;
    const int k = min(kv_len(c, bt, b), e.keep);
    const int32_t* kept = e.kept + ((int64_t)b * c.heads + head) * e.keep;
    const int64_t most = (int64_t)e.new_width << c.page_shift;
    const int in = (1 << c.page_shift) - 1;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (int64_t)k * parts;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int to = (int)(i / parts), part = (int)(i % parts);
        const int from = kept[to];
        if (to >= most) {
            atomicOr(c.status, ERR_LAYOUT);
            continue;
        }
        const int64_t p0 = kv_page(c, bt.table + b * bt.table_stride, from);
        const int64_t p1 = kv_page(c, e.new_table + b * e.new_stride, to);
        if (p0 < 0 || p1 < 0) continue;
        const uint4 kk = reinterpret_cast<const uint4*>(c.k + p0 * c.ks[0] + (from & in) * c.ks[1] + head * c.ks[2])[part];
        const uint4 vv = reinterpret_cast<const uint4*>(c.v + p0 * c.vs[0] + (from & in) * c.vs[1] + head * c.vs[2])[part];
        reinterpret_cast<uint4*>(c.k + p1 * c.ks[0] + (to & in) * c.ks[1] + head * c.ks[2])[part] = kk;
        reinterpret_cast<uint4*>(c.v + p1 * c.vs[0] + (to & in) * c.vs[1] + head * c.vs[2])[part] = vv;
    }
}

}  // namespace vk
