// Weights that the rows of a chunk gave each slot: scores[slot] += sum over rows of exp(s - lse of the row).
//
// The attention kernel cannot add them up itself, since a row's total is only known at its end; what it would have to
// keep (rows x slots) is larger than what it takes to compute the products again. Here the slots are the accumulator's
// lanes: S^T = K Q^T puts a slot's products with 128 rows into one thread's columns, so that its weights are summed in
// registers, without a shuffle or an atomic, and every row's lse is read by all threads alike from shared memory.
//
// A unit is a pair of slot tiles (2 x 128) against one row tile; two warpgroups share a slot tile, half of the rows each
// (four warps per scheduler; with two their latencies were not covered: 88 us where four take 70). Units run row tile by
// row tile within a pair, the pair's keys stay in shared memory and the rows stream; the units of all (sequence, kv head,
// pair)s are laid end to end and shared out equally, and cut pairs are finished from parts, as in the step kernel.
//
// The least it could take: one exponential per (row, slot), 16 a clock and SM on the special function units (1,024 cycles per
// 128 x 128 tile against 512 for its product at a head size of 128). Measured: 2,048 tokens over 16,384 slots, 16 heads over 8
// of 128: 180 us, 61 % of that rate. What holds it back is the rest of a tile: of 173 us then, 122 were left without the
// exponentials (loads from tensor memory, additions, a barrier per row tile for the rows' lse), 159 without the products.
#pragma once
#include "kv_chunk.cuh"

namespace vk {

constexpr int WEIGHTS_PAIR = 2 * CHUNK_SLOTS;  // slots of a pair
constexpr float WEIGHTS_PART_COST = 0.15f;       // of a unit
// Row tiles in flight. At a head size of 64 more than are needed: with over half of an SM's shared memory no two of these
// CTAs meet on an SM, where one would wait for the other's tensor memory while both wait for parts of CTAs elsewhere.
template <int DP>
constexpr int WEIGHTS_RING = DP == 128 ? 4 : 8;
constexpr int WEIGHTS_THREADS = 576;  // four warpgroups that add up, the MMA warp, the loading warp
template <int DP>
constexpr int weights_smem() {
    return (2 + WEIGHTS_RING<DP>) * CHUNK_SLOT<DP> + 4 * 2 * 64 * 4 + 2 * 2 * 128 * 4 + 512;
}
static_assert(2 * weights_smem<64>() > 233472 && 2 * weights_smem<128>() > 233472, "one CTA per SM");

struct WeightsShape {
    const KvAttend& a;
    int tokens;  // of a row tile
    __device__ __forceinline__ bool takes(const KvSeq& s) const {
        return s.count > 0 && s.len > 0;
    }
    __device__ __forceinline__ int pairs(const KvSeq& s) const {
        return (int)((min((int64_t)s.len, a.scores_width) + WEIGHTS_PAIR - 1) / WEIGHTS_PAIR);
    }
    __device__ __forceinline__ int row_tiles(const KvSeq& s) const { return (int)a.by_tokens(s.count + tokens - 1); }
    // the first row tile with a row that sees the pair's first slot
    __device__ __forceinline__ int first(const KvSeq& s, int pair) const {
        const int x = pair * WEIGHTS_PAIR - (s.len - s.count);
        return a.causal && x > 0 ? (int)a.by_tokens(x) : 0;
    }
    // units of the pairs before `pair`
    __device__ __forceinline__ int before(const KvSeq& s, int pair) const {
        int sum = pair * row_tiles(s);
        if (a.causal) {
            const int ahead = s.len - s.count;
            const int p0 = ahead < 0 ? 0 : min(pair, (ahead + WEIGHTS_PAIR - 1) / WEIGHTS_PAIR);
            sum -= (int)floor_sum(pair - p0, tokens, WEIGHTS_PAIR, p0 * WEIGHTS_PAIR - ahead);
        }
        return sum;
    }
};

// A CTA's next segment: consecutive row tiles of one (sequence, kv head, pair).
struct WeightsSegment {
    KvSeq s;
    int b, head, pair, q0, count;
    bool leaves;                // begins behind the pair's first unit
    int rest;                   // units of the pair behind it
    bool both;                  // the second tile has slots
};
struct WeightsWalk {
    const KvPages& c;
    const KvBatch& bt;
    const WeightsShape& shape;
    KvShare share;
    int head, pair, skip;
    bool located;
    __device__ __forceinline__ bool next(WeightsSegment* g) {
        if (share.left <= 0) return false;
        KvSeq s = kv_seq(c, bt, share.b);
        while (!shape.takes(s) || head >= c.heads) {
            s = kv_seq(c, bt, ++share.b);
            head = pair = skip = 0;
        }
        const int all = shape.pairs(s);
        if (!located) {
            const int per = shape.before(s, all);
            int off = share.off;
            for (head = 0; off >= per; ++head) off -= per;
            pair = locate_pair(all, off, [&](int p) { return shape.before(s, p); });
            skip = off - shape.before(s, pair);
            located = true;
        }
        const int tiles = shape.row_tiles(s) - shape.first(s, pair);
        g->s = s;
        g->b = share.b;
        g->head = head;
        g->pair = pair;
        g->q0 = shape.first(s, pair) + skip;
        g->count = min(tiles - skip, share.left);
        g->leaves = skip > 0;
        g->rest = tiles - skip - g->count;
        g->both = min((int64_t)s.len, shape.a.scores_width) > (int64_t)pair * WEIGHTS_PAIR + CHUNK_SLOTS;
        share.left -= g->count;
        skip = 0;
        if (++pair == all) pair = 0, ++head;
        return true;
    }
};

template <typename T, int DP>
__global__ void __launch_bounds__(WEIGHTS_THREADS, 1)
    kv_weights_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, KvPages c,
                      KvBatch bt, KvAttend a, KvParts parts) {
    constexpr int HALVES = DP / 64, KS = DP / 16, RING = WEIGHTS_RING<DP>, SLOT = CHUNK_SLOT<DP>;
    extern __shared__ __align__(1024) uint8_t ring[];  // the swizzle goes by address bits: 1024-byte aligned
    uint8_t* smem_k = ring + RING * SLOT;              // the pair's two tiles
    float* s_lse = reinterpret_cast<float*>(smem_k + 2 * SLOT);  // [warpgroup][2][64]: minus a row's lse, base 2
    float* s_sum = s_lse + 4 * 2 * 64;                           // [2][slot tile][128]: of the second half of the rows
    uint64_t* q_full = reinterpret_cast<uint64_t*>(s_sum + 2 * 2 * 128);
    uint64_t* q_empty = q_full + RING;
    uint64_t* k_full = q_empty + RING;
    uint64_t* k_empty = k_full + 1;
    uint64_t* s_full = k_empty + 1;  // [slot tile][2]
    uint64_t* s_empty = s_full + 4;
    uint64_t* mma_done = s_empty + 4;
    int* scratch = reinterpret_cast<int*>(mma_done + 1);
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(scratch + KV_SHARE_SCRATCH);
    const int warp = __shfl_sync(FULL, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        prefetch_map(&map_q);
        prefetch_map(&map_k);
        for (int i = 0; i < RING; ++i) {
            mbar_init(q_full + i, 1);
            mbar_init(q_empty + i, 1);
        }
        mbar_init(k_full, 1);
        mbar_init(k_empty, 1);
        mbar_init(mma_done, 1);
        for (int i = 0; i < 4; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(s_empty + i, 8);
        }
        fence_mbar_init();
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (a.tokens * a.group < CHUNK_ROWS) {  // the other rows are never loaded: their products must not be NaN
        for (int i = threadIdx.x; i < RING * SLOT / 16; i += WEIGHTS_THREADS)
            reinterpret_cast<uint4*>(ring)[i] = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
    }
    tmem_fence_before();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const WeightsShape shape{a, a.tokens};
    KvShare share = kv_share<WEIGHTS_THREADS>(c, bt, parts, scratch, WEIGHTS_PART_COST, [&](const KvSeq& s, int* longest) {
        if (!shape.takes(s)) return 0;
        *longest = max(*longest, shape.row_tiles(s));
        return shape.before(s, shape.pairs(s)) * c.heads;
    });
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    tmem_fence_after();
    const uint32_t tm = __shfl_sync(FULL, *tmem_at, 0);
    KvWait wait{c.status, parts.bad, a.wait_limit};
    WeightsWalk walk{c, bt, shape, share, 0, 0, 0, false};
    WeightsSegment g;
    if (warp == 17) {
        int slot = 0, loaded = 0, k_fills = 0;
        uint32_t phase = 0, k_phase = 0;
        const int box_shift = min(c.page_shift, 6), boxes = CHUNK_SLOTS >> box_shift;
        const uint32_t me = elect_lane();
        while (!wait.dead && walk.next(&g)) {
            const int32_t* table = bt.table + g.b * bt.table_stride;
            wait.together(k_empty, k_phase ^ 1);
            if (wait.dead) break;
            k_phase ^= 1;
            ++k_fills;
            TilePages tp[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int first = g.pair * WEIGHTS_PAIR + u * CHUNK_SLOTS, n = u == 0 || g.both ? boxes : 0;
                tp[u] = tile_pages(c, tile_entries(c, table, first, n, box_shift, g.s.len), first, n, box_shift, g.s.len);
            }
            if (lane == 0) mbar_arrive_expect_tx(k_full, (tp[0].count + tp[1].count) * HALVES * (128 << box_shift));
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 2; ++u)
                for (int i = 0; i < tp[u].count; ++i) {
                    const int page = __shfl_sync(FULL, tp[u].page, i), from = i << box_shift;
                    const int in = (g.pair * WEIGHTS_PAIR + u * CHUNK_SLOTS + from) & ((1 << c.page_shift) - 1);
#pragma unroll
                    for (int half = 0; half < HALVES; ++half)
                        tma_page(smem_k + u * SLOT + half * (CHUNK_SLOTS * 128) + from * 128, &map_k, half * 64, in, g.head,
                                 page, k_full, me);
                }
            for (int q = g.q0; q < g.q0 + g.count; ++q) {
                wait.together(q_empty + slot, phase ^ 1);
                if (wait.dead) break;
                ++loaded;
                if (lane == 0) {
                    mbar_arrive_expect_tx(q_full + slot, HALVES * shape.tokens * a.group * 128);
                    for (int h = 0; h < HALVES; ++h)
                        tma_rows(ring + slot * SLOT + h * (CHUNK_ROWS * 128), &map_q, h * 64, g.head * a.group,
                                 (int)g.s.first + q * shape.tokens, q_full + slot);
                }
                __syncwarp();
                if (++slot == RING) slot = 0, phase ^= 1;
            }
        }
        if (lane == 0) {
            wait.drain(k_full, k_fills);
            for (int i = 0; i < RING; ++i) wait.drain(q_full + i, loaded / RING + (i < loaded % RING));
        }
    } else if (warp == 16) {
        const uint32_t idesc = umma_idesc<T>(CHUNK_ROWS, false, a.scale < 0.f);
        const uint32_t k_low = umma_low(smem_u32(smem_k), 16), q_low = umma_low(smem_u32(ring), 16);
        int slot = 0, used[2] = {0, 0};  // row tiles that went to each warpgroup's two buffers
        uint32_t phase = 0, k_phase = 0;
        const uint32_t me = elect_lane();
        const int ks = (c.dim + 15) / 16;  // steps of 16 elements; the padding's products are left out
        while (walk.next(&g)) {
            const bool both = __shfl_sync(FULL, g.both, 0);
            const int count = __shfl_sync(FULL, g.count, 0);
            wait(k_full, k_phase);
            k_phase ^= 1;
            for (int q = 0; q < count; ++q) {
                wait(q_full + slot, phase);
                const uint32_t rows = q_low + slot * (SLOT / 16);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (i == 1 && !both) continue;
                    const int buf = used[i] & 1;
                    const uint32_t at = tm + (2 * i + buf) * 128, k = k_low + i * (SLOT / 16);
                    wait(s_empty + 2 * i + buf, (used[i] >> 1 & 1) ^ 1);
                    tmem_fence_after();
                    ++used[i];
#pragma unroll
                    for (int e = 0; e < KS; ++e) {
                        const uint32_t off = (e >> 2) * (CHUNK_ROWS * 8) + (e & 3) * 2;
                        if (e < ks) umma_ss(at, k + off, rows + off, idesc, e > 0, me);
                    }
                    umma_commit(s_full + 2 * i + buf, me);
                }
                umma_commit(q_empty + slot, wait.live(me));
                if (++slot == RING) slot = 0, phase ^= 1;
            }
            umma_commit(k_empty, wait.live(me));
        }
        umma_commit(mma_done, me);
        if (lane == 0) wait.drain(mma_done, 1);
    } else {
        const int wg = warp >> 2, i = wg & 1, half = wg >> 1, r = (warp & 3) * 32 + lane;
        const int row = half * 64 + (r & 63), row_token = (int)a.by_group(row);  // whose lse this thread fetches
        const uint32_t lanes = tm + ((uint32_t)((warp & 3) * 32) << 16) + i * 256 + half * 64;
        float* lse = s_lse + wg * 128;
        const float scale = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-37f);
        const Pair scale2 = pair_of(scale, scale);
        int used = 0, turn = 0;
        while (walk.next(&g)) {
            if (i == 1 && !g.both) continue;
            const int j = g.pair * WEIGHTS_PAIR + i * CHUNK_SLOTS + r;
            // no row, or one that saw nothing: weight 0
            auto minus_lse = [&](int q) {
                const int token = q * shape.tokens + row_token;
                if (row >= shape.tokens * a.group || token >= g.s.count) return -INFINITY;
                const float v = __ldca(a.lse + (g.s.first + token) * a.heads + g.head * a.group + row - row_token * a.group);
                return v == -INFINITY ? -INFINITY : -v * 1.4426950408889634f;
            };
            Pair sum[2] = {pair_of(0.f, 0.f), pair_of(0.f, 0.f)};
            float next = minus_lse(g.q0);
            for (int q = g.q0; q < g.q0 + g.count; ++q) {
                const int buf = used & 1;
                if (r < 64) lse[buf * 64 + r] = next;
                if (q + 1 < g.q0 + g.count) next = minus_lse(q + 1);
                bar_sync(1 + wg, 128);
                wait(s_full + 2 * i + buf, used >> 1 & 1);
                ++used;
                tmem_fence_after();
                // rows that see this slot: from `from` on; the tile's rows end at `to`; counted from this half's first
                const int to = min(shape.tokens, g.s.count - q * shape.tokens) * a.group - half * 64;
                const int from =
                    (a.causal ? max(0, j - (g.s.len - g.s.count) - q * shape.tokens) * a.group : 0) - half * 64;
                const bool masked = __any_sync(FULL, from > 0) || to < min(64, shape.tokens * a.group - half * 64);
                const float4* l4 = reinterpret_cast<const float4*>(lse + buf * 64);
#pragma unroll
                for (int h = 0; h < 64; h += 32) {
                    float x[32];
                    tmem_ld32(lanes + buf * 128 + h, x);
                    tmem_wait_ld();
                    if (h == 32) {
                        tmem_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(s_empty + 2 * i + buf);
                    }
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) x[e] = h + e >= from && h + e < to ? x[e] : -INFINITY;
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float4 y = l4[h / 4 + e];
                        const float2 u = floats(fma2(pair_of(x[4 * e], x[4 * e + 1]), scale2, pair_of(y.x, y.y)));
                        const float2 w = floats(fma2(pair_of(x[4 * e + 2], x[4 * e + 3]), scale2, pair_of(y.z, y.w)));
                        sum[0] = sum[0] + pair_of(ex2(u.x), ex2(u.y));
                        sum[1] = sum[1] + pair_of(ex2(w.x), ex2(w.y));
                    }
                }
            }
            const float2 both = floats(sum[0] + sum[1]);
            float total = both.x + both.y;
            // The second half's warpgroup hands its sum over, into the other buffer each time: it cannot be two ahead.
            float* other = s_sum + (turn & 1) * 256 + i * 128 + r;
            turn ^= 1;
            if (half == 1) *other = total;
            bar_sync(5 + i, 256);
            if (half == 1) continue;
            total += *other;
            const int part = 2 * walk.share.me + i;
            if (g.leaves) {
                parts.o[(int64_t)part * CHUNK_SLOTS + r] = total;
                bar_sync(1 + wg, 128);
                if (r == 0) part_publish(parts, part);
            } else {
                const int follow = walk.share.followers(g.rest);
                if (follow) {
                    for (int k = r; k < follow; k += 128) part_await(parts, part + 2 + 2 * k, wait);
                    bar_sync(1 + wg, 128);
                    for (int k0 = 0; k0 < follow; k0 += 8) {  // eight in flight; the last ones again, for nothing
                        float x[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            x[k] = __ldcg(parts.o + (int64_t)(part + 2 + 2 * min(k0 + k, follow - 1)) * CHUNK_SLOTS + r);
#pragma unroll
                        for (int k = 0; k < 8; ++k) total += k0 + k < follow ? x[k] : 0.f;
                    }
                    for (int k = r; k < follow; k += 128) parts.ready[part + 2 + 2 * k] = 0;
                }
                if (j < min((int64_t)g.s.len, a.scores_width)) a.scores[g.b * a.ss[0] + g.head * a.ss[1] + j] += total;
            }
        }
    }
    __syncthreads();
    if (warp == 16) {
        __syncwarp();
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm) : "memory");
    }
}

}  // namespace vk
