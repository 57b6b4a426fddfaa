// The cache's kernels that move keys and values: append and evict.
#pragma once
#include <cooperative_groups.h>

#include "kv_common.cuh"

namespace vk {

// Takes the reported bits out of the status word and no others: a kernel of another stream may set some meanwhile.
__global__ void kv_reported_kernel(int* status, int bits) { atomicAnd(status, ~bits); }

// One thread per 16 bytes of a new token's head. Every byte is read and written once: bound by memory (9 prompts of up to
// 2,011 tokens, 8 kv heads of 128, 104 MB: 20.9 us, 5.0 TB/s among calls on other data, 18.9 when one call is repeated), by
// the launch for a step's few tokens (2.5 us in a graph).
__global__ void __launch_bounds__(256) kv_append_kernel(KvPages c, KvBatch bt, const uint16_t* k, const uint16_t* v,
                                                        int64_t k_tok, int64_t k_head, int64_t v_tok, int64_t v_head) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
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
        const uint4 kk = __ldca(reinterpret_cast<const uint4*>(k + tok * k_tok + head * k_head) + part);
        const uint4 vv = __ldca(reinterpret_cast<const uint4*>(v + tok * v_tok + head * v_head) + part);
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

// Selection: a cluster of CTAs for each (sequence, kv head) finds the slots to keep.
//
// Each CTA holds an equal, contiguous slice of the slots' ranks in shared memory, read from memory once. The rank of the
// (k - r)-th largest among the first n - r slots is found digit by digit (11, 11 and 10 bits from the top): every CTA
// counts the digit's values among its ranks that match the digits so far, the cluster's counts are added up through
// distributed shared memory, by every CTA for itself. A first digit of 11 bits tells scores apart within an octave, so
// that a warp's counting meets few equal addresses. Ranks above the found one are kept, and of those equal to it the
// first ones; where a CTA's kept slots go follows from the counts of the CTAs before it.
//
// Bound by latency: up to eight cluster-wide steps, and a slice's passes through shared memory. Up to 16 CTAs per
// (sequence, kv head), so that a long sequence's passes are short. Measured, 8 kv heads, cold caches: 1,087 slots 11 us, 131,072
// slots 28 us (one block of 1,024 threads per head: 29 and 265).
constexpr int SELECT_THREADS = 512;
constexpr int SELECT_BINS = 2048;
constexpr int SELECT_HELD = 16384;  // ranks that a CTA keeps in shared memory; a larger slice is read again instead
constexpr int SELECT_CLUSTER = 16;

// The score of a rank (a NaN and a zero without their signs).
__device__ __forceinline__ float kv_score(uint32_t u) {
    return u == 0u ? __int_as_float(0x7fffffff) : __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

template <int C>
__global__ void __launch_bounds__(SELECT_THREADS, 2) kv_select_kernel(KvPages c, KvBatch bt, KvEvict e) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    extern __shared__ __align__(1024) uint8_t ring[];
    int* hist = reinterpret_cast<int*>(ring);  // [digit][SELECT_BINS], sums of the cluster, one share of all CTAs' counts
    uint32_t* held = reinterpret_cast<uint32_t*>(hist + 5 * SELECT_BINS);  // [min(slice, SELECT_HELD)]
    __shared__ int warp_a[SELECT_THREADS / 32], warp_b[SELECT_THREADS / 32];
    __shared__ int found_digit, found_need, mine_gt, mine_eq;
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int WARPS = SELECT_THREADS / 32;
    const int b = blockIdx.z, head = blockIdx.y;
    const int n = kv_len(c, bt, b);
    const int k = min(n, e.keep), r = min(e.recent, k), m = k - r, cand = n - r;
    const float* sc = e.scores + b * e.ss[0] + head * e.ss[1];
    int32_t* kept = e.kept + ((int64_t)b * c.heads + head) * e.keep;
    float* ns = e.new_scores + ((int64_t)b * c.heads + head) * e.width;
    auto score = [&](int64_t slot) { return slot < e.width ? __ldca(sc + slot) : 0.0f; };
    if (head == 0 && rank == 0 && tid == 0) e.new_lens[b] = k;
    const int slice = (cand + C - 1) / C, from = min(cand, rank * slice), size = min(cand, from + slice) - from;
    const bool fits = slice <= SELECT_HELD;
    for (int i = tid; i < 3 * SELECT_BINS; i += SELECT_THREADS) hist[i] = 0;
    if (fits) {
        // of the slice, slots that have a score; the loads behind them are of the last one again, so that none of a batch
        // waits for a branch
        const int have = (int)min((int64_t)size, max(e.width - from, int64_t(0)));
        const float* mine = sc + from;
        for (int i0 = tid; i0 < size; i0 += 8 * SELECT_THREADS) {
            float x[8] = {};
            if (have > 0)
#pragma unroll
                for (int u = 0; u < 8; ++u) x[u] = __ldca(mine + min(i0 + u * SELECT_THREADS, have - 1));
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = i0 + u * SELECT_THREADS;
                if (i < size) held[i] = kv_rank(i < have ? x[u] : 0.0f);
            }
        }
    }
    __syncthreads();
    auto cluster_sync = [&] {
        if constexpr (C > 1) cluster.sync();
        else __syncthreads();
    };
    auto rank_of = [&](int i) { return fits ? held[i] : kv_rank(score(from + i)); };
    // sum over the threads before this one, and the block's total
    auto scan = [&](int x, int* total) {
        int incl = x;
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(FULL, incl, o);
            if (lane >= o) incl += y;
        }
        __syncthreads();
        if (lane == 31) warp_a[warp] = incl;
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) before += warp_a[w];
            all += warp_a[w];
        }
        *total = all;
        return before + incl - x;
    };
    // m == cand: everything is at or above rank 0. m == 0: no rank is above this one, and none equal to it is wanted.
    uint32_t cut = m == cand ? 0u : 0xffffffffu;
    int need = m == cand ? cand : 0;  // slots of rank `cut` to keep
    if (m > 0 && m < cand) {  // the same for the whole cluster
        cut = 0;
        need = m;
        uint32_t mask = 0;
        constexpr int SHIFT[3] = {21, 10, 0};
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = SHIFT[pass];
            constexpr int PER = SELECT_BINS / SELECT_THREADS;
            const uint32_t low = pass == 2 ? 1023u : 2047u;
            int* h = hist + pass * SELECT_BINS;
            for (int i = tid; i < size; i += SELECT_THREADS) {
                const uint32_t u = rank_of(i);
                if ((u & mask) == cut) atomicAdd(h + (u >> shift & low), 1);
            }
            cluster_sync();
            // thread t takes PER digits, from the largest down
            const int first = SELECT_BINS - PER * (tid + 1);
            int sum[PER] = {};
            if constexpr (C < 8) {
#pragma unroll
                for (int o = 0; o < C; ++o) {
                    const int4 x = *reinterpret_cast<const int4*>(cluster.map_shared_rank(h, o) + first);
                    sum[0] += x.w, sum[1] += x.z, sum[2] += x.y, sum[3] += x.x;
                }
            } else {
                // Every CTA adding up everything reads C x 8 KB from the others, and distant shared memory is slow: of a
                // larger cluster each CTA adds up its share of the digits and hands the sums to all.
                constexpr int GROUPS = SELECT_BINS / 4 / C;  // of four digits, in a share
                const int o = tid / GROUPS, group = tid % GROUPS, at = rank * 4 * GROUPS + 4 * group;
                int4* const share = reinterpret_cast<int4*>(hist + 4 * SELECT_BINS);  // [CTA][group]
                share[tid] = *reinterpret_cast<const int4*>(cluster.map_shared_rank(h, o) + at);
                __syncthreads();
                int4 all = make_int4(0, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    const int4 x = share[i * GROUPS + group];
                    all.x += x.x, all.y += x.y, all.z += x.z, all.w += x.w;
                }
                int* const totals = hist + 3 * SELECT_BINS;
                *reinterpret_cast<int4*>(cluster.map_shared_rank(totals, o) + at) = all;
                cluster.sync();
                const int4 x = *reinterpret_cast<const int4*>(totals + first);
                sum[0] = x.w, sum[1] = x.z, sum[2] = x.y, sum[3] = x.x;
            }
            static_assert(PER == 4, "an int4 per thread and CTA");
            int total;
            int before = scan(sum[0] + sum[1] + sum[2] + sum[3], &total);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (before < need && need <= before + sum[i]) {
                    found_digit = first + PER - 1 - i;
                    found_need = need - before;
                }
                before += sum[i];
            }
            __syncthreads();
            cut |= (uint32_t)found_digit << shift;
            need = found_need;
            mask |= low << shift;
        }
    }
    // each warp takes a contiguous range of the slice: count, then emit behind the ranges and CTAs before it
    const int span = ((size + WARPS - 1) / WARPS + 31) / 32 * 32, lo = min(size, warp * span), hi = min(size, lo + span);
    int gt = 0, eq = 0;
#pragma unroll 4
    for (int i = lo + lane; i < hi; i += 32) {
        const uint32_t u = rank_of(i);
        gt += u > cut;
        eq += u == cut;
    }
    gt = __reduce_add_sync(FULL, gt);
    eq = __reduce_add_sync(FULL, eq);
    __syncthreads();
    if (lane == 0) {
        warp_a[warp] = gt;
        warp_b[warp] = eq;
    }
    __syncthreads();
    int before_gt = 0, before_eq = 0, all_gt = 0, all_eq = 0;
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before_gt += warp_a[w], before_eq += warp_b[w];
        all_gt += warp_a[w], all_eq += warp_b[w];
    }
    int cta_gt = 0, cta_eq = 0;  // of the CTAs before this one: one lane each
    if constexpr (C > 1) {
        if (tid == 0) mine_gt = all_gt, mine_eq = all_eq;
        cluster.sync();
        if (lane < rank) {
            cta_gt = *cluster.map_shared_rank(&mine_gt, lane);
            cta_eq = *cluster.map_shared_rank(&mine_eq, lane);
        }
        cta_gt = __reduce_add_sync(FULL, cta_gt);
        cta_eq = __reduce_add_sync(FULL, cta_eq);
        cluster.sync();  // nobody reads this CTA's shared memory from here on
    }
    before_gt += cta_gt, before_eq += cta_eq;
    const unsigned below = (1u << lane) - 1u;
    const int width = (int)min(e.width, (int64_t)INT32_MAX);
    int at0 = before_gt + min(before_eq, need);
    for (int i0 = lo; i0 < hi; i0 += 128) {  // four groups of 32 at a time, their ranks fetched together
        uint32_t u[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) u[w] = i0 + 32 * w + lane < hi ? rank_of(i0 + 32 * w + lane) : 0u;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int i = i0 + 32 * w + lane;
            unsigned keep = __ballot_sync(FULL, i < hi && u[w] > cut);
            const unsigned me = __ballot_sync(FULL, i < hi && u[w] == cut);
            if (me) {  // the first ones of those that tie
                keep |= __ballot_sync(FULL, (me >> lane & 1u) && before_eq + __popc(me & below) < need);
                before_eq += __popc(me);
            }
            if (keep >> lane & 1u) {
                const int at = at0 + __popc(keep & below);
                kept[at] = from + i;
                if (at < width) ns[at] = kv_score(u[w]);
            }
            at0 += __popc(keep);
        }
    }
    // a share of the latest slots, and what lies behind the kept ones
    for (int i = rank * SELECT_THREADS + tid; i < r; i += C * SELECT_THREADS) {
        kept[m + i] = cand + i;
        if (m + i < e.width) ns[m + i] = score(cand + i);
    }
    for (int64_t i = k + rank * SELECT_THREADS + tid; i < e.keep; i += C * SELECT_THREADS) kept[i] = -1;
    for (int64_t i = k + rank * SELECT_THREADS + tid; i < e.width; i += C * SELECT_THREADS) ns[i] = 0.0f;
}

// Copies the kept slots' keys and values, 16 bytes of each per thread and step. A grid of its own: the selection's few
// CTAs have too few loads in flight for it (131,072 slots cut to 16,384, 8 kv heads: 128 us in one kernel, 93
// in two when that was tried, 52 since the selection got faster). Measured: 16 sequences of up to 8,192 slots cut to half,
// 8 kv heads of 128, 529 MB: 87 us, 6.1 TB/s.
__global__ void __launch_bounds__(256) kv_compact_kernel(KvPages c, KvBatch bt, KvEvict e) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int parts = c.dim >> 3, b = blockIdx.z, head = blockIdx.y;
    const int k = min(kv_len(c, bt, b), e.keep);
    const int32_t* kept = e.kept + ((int64_t)b * c.heads + head) * e.keep;
    const int64_t most = (int64_t)e.new_width << c.page_shift;
    const int in = (1 << c.page_shift) - 1;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (int64_t)k * parts;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int to = (int)(i / parts), part = (int)(i % parts);
        if (to >= most) {
            atomicOr(c.status, ERR_LAYOUT);
            continue;
        }
        const int from = __ldca(kept + to), entry1 = kv_entry(c, e.new_table + b * e.new_stride, to);
        const int entry0 = kv_entry(c, bt.table + b * bt.table_stride, from);
        const int64_t p0 = kv_page_checked(c, entry0), p1 = kv_page_checked(c, entry1);
        if (p0 < 0 || p1 < 0) continue;
        const uint4 kk =
            __ldca(reinterpret_cast<const uint4*>(c.k + p0 * c.ks[0] + (from & in) * c.ks[1] + head * c.ks[2]) + part);
        const uint4 vv =
            __ldca(reinterpret_cast<const uint4*>(c.v + p0 * c.vs[0] + (from & in) * c.vs[1] + head * c.vs[2]) + part);
        reinterpret_cast<uint4*>(c.k + p1 * c.ks[0] + (to & in) * c.ks[1] + head * c.ks[2])[part] = kk;
        reinterpret_cast<uint4*>(c.v + p1 * c.vs[0] + (to & in) * c.vs[1] + head * c.vs[2])[part] = vv;
    }
}

}  // namespace vk
