// Attention of a chunk of new tokens over the paged cache on the 5th-generation tensor cores.
//
// A kv head's rows (tokens x its query heads, token by token) come in tiles of 128, the tensor memory's lanes: with 5
// query heads to a kv head a tile holds 25 tokens, 125 rows. A unit of work is a pair of row tiles against 128 slots; the
// units of all (sequence, kv head, pair)s are laid end to end and every CTA takes an equal share, so that neither the
// causal mask nor ragged lengths nor few rows over a long cache leave SMs idle; cut pairs are joined from parts
// (kv_join_kernel).
//
// Per unit and row tile: scores S = Q K^T (tcgen05.mma, both operands in shared memory) into tensor memory; a warpgroup,
// one row per thread, takes the maximum, exponentials and their sum, and puts the weights P as 16-bit values where S was;
// O += P V with P from tensor memory. While one tile's warpgroup works, the tensor cores do the other tile's products.
// O stays in tensor memory; it is rescaled only when a row's maximum has grown by more than 2^8 since the reference that
// its weights use, which the sums allow (weights up to 256 in 16 bits keep their relative precision).
//
// Bound: 4 x 128 x 128 x head size operations per tile and unit on the tensor cores, and 128 x 128 exponentials on the
// 16-a-clock special function units, which is the same time (1,024 cycles) at a head size of 128.
#pragma once
#include "kv_step.cuh"

namespace vk {

constexpr int CHUNK_ROWS = 128;                 // rows of a tile
constexpr int CHUNK_SLOTS = 128;                // slots of a unit
constexpr int CHUNK_THREADS = 384;              // two softmax warpgroups; one with the MMA warp and the loading warp
constexpr int CHUNK_PART_ROWS = 2 * CHUNK_ROWS;
template <int DP>
constexpr int CHUNK_Q = 2 * CHUNK_ROWS * DP * 2;   // bytes of the two query tiles
template <int DP>
constexpr int CHUNK_SLOT = CHUNK_SLOTS * DP * 2;   // bytes of a tile of keys or values
template <int DP>
constexpr int CHUNK_RING = DP == 128 ? 5 : 10;     // tiles in flight, keys and values alternating
template <int DP>
constexpr int chunk_smem() {
    return CHUNK_Q<DP> + CHUNK_RING<DP> * CHUNK_SLOT<DP> + 512;
}

// A row tile's box of the queries (64 elements of a kv head's query heads, for a tile's tokens) into shared memory.
__device__ __forceinline__ void tma_rows(void* dst, const CUtensorMap* map, int d, int head, int token, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(d), "r"(head), "r"(token), "r"(smem_u32(bar))
        : "memory");
}

// ---- tcgen05
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
    // 128-byte swizzle (2 << 61), descriptor version 1; byte offsets in units of 16
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
template <typename T>
__device__ __forceinline__ uint32_t umma_idesc(int n, bool b_by_rows, bool negate) {
    const uint32_t type = std::is_same_v<T, __half> ? 0u : 1u;
    return 1u << 4 | type << 7 | type << 10 | (negate ? 1u << 13 : 0u) | (b_by_rows ? 1u << 16 : 0u) |
           (uint32_t)(n >> 3) << 17 | (uint32_t)(CHUNK_ROWS >> 4) << 24;
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
// The barrier gets an arrival when all products that this thread issued so far are done.
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define VK_R8(x, i) "=f"((x)[i]), "=f"((x)[i + 1]), "=f"((x)[i + 2]), "=f"((x)[i + 3]), "=f"((x)[i + 4]), \
                    "=f"((x)[i + 5]), "=f"((x)[i + 6]), "=f"((x)[i + 7])
#define VK_W8(x, i) "r"((x)[i]), "r"((x)[i + 1]), "r"((x)[i + 2]), "r"((x)[i + 3]), "r"((x)[i + 4]), \
                    "r"((x)[i + 5]), "r"((x)[i + 6]), "r"((x)[i + 7])
// 32 columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t at, float* x) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : VK_R8(x, 0), VK_R8(x, 8), VK_R8(x, 16), VK_R8(x, 24)
        : "r"(at));
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t* x) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
        VK_W8(x, 0), VK_W8(x, 8), VK_W8(x, 16), VK_W8(x, 24)
        : "memory");
}

// ---- the order of units
// sum of floor((a i + b) / m) over 0 <= i < n, by Euclid's steps on (m, a); a, b >= 0
__device__ __forceinline__ int64_t floor_sum(int64_t n, int64_t m, int64_t a, int64_t b) {
    int64_t sum = 0;
    while (n > 0) {
        sum += n * (n - 1) / 2 * (a / m) + n * (b / m);
        a %= m;
        b %= m;
        const int64_t y = a * n + b;
        if (y < m) break;
        n = y / m;
        b = y % m;
        const int64_t t = m;
        m = a;
        a = t;
    }
    return sum;
}

struct ChunkShape {
    int group, causal;
    int tokens;  // of a row tile
    __device__ __forceinline__ bool takes(const KvSeq& s) const { return s.count > 0 && !step_takes(s, group); }
    __device__ __forceinline__ int pairs(const KvSeq& s) const { return (s.count + 2 * tokens - 1) / (2 * tokens); }
    // slots that the pair's last row sees
    __device__ __forceinline__ int limit(const KvSeq& s, int pair) const {
        return causal ? max(0, s.len - s.count + min(s.count, (pair + 1) * 2 * tokens)) : s.len;
    }
    __device__ __forceinline__ int tiles(const KvSeq& s, int pair) const {
        return max(1, (limit(s, pair) + CHUNK_SLOTS - 1) / CHUNK_SLOTS);
    }
    // units of the pairs before `pair`
    __device__ __forceinline__ int64_t before(const KvSeq& s, int pair) const {
        if (!causal) return (int64_t)pair * tiles(s, 0);
        const int all = pairs(s), n = min(pair, all - 1), per = 2 * tokens;
        const int64_t a = (int64_t)s.len - s.count;
        const int one = a > CHUNK_SLOTS ? 0 : (int)min((int64_t)n, (CHUNK_SLOTS - a) / per);  // pairs of one unit
        const int64_t sum = one + floor_sum(n - one, CHUNK_SLOTS, per, a + (int64_t)(one + 1) * per + CHUNK_SLOTS - 1);
        return pair < all ? sum : sum + tiles(s, all - 1);
    }
};

// A CTA's next segment: consecutive units of one (sequence, kv head, pair).
struct ChunkSegment {
    KvSeq s;
    int b, head, pair, t0, count, tiles;
    int token0;  // of the pair's first row
    bool both;   // the second tile has rows
};
struct ChunkWalk {
    const KvPages& c;
    const KvBatch& bt;
    const ChunkShape& shape;
    KvShare share;
    int head, pair, t0;
    bool located;
    __device__ __forceinline__ bool next(ChunkSegment* g) {
        if (share.left <= 0) return false;
        KvSeq s = kv_seq(c, bt, share.b);
        while (!shape.takes(s) || head >= c.heads) {
            s = kv_seq(c, bt, ++share.b);
            head = pair = t0 = 0;
        }
        const int all = shape.pairs(s);
        if (!located) {  // the position of the share's first unit within its sequence
            const int64_t per = shape.before(s, all);
            head = (int)(share.off / per);
            const int64_t off = share.off % per;
            int lo = 0, hi = all - 1;  // the last pair that begins at or before off
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (shape.before(s, mid) <= off) lo = mid;
                else hi = mid - 1;
            }
            pair = lo;
            t0 = (int)(off - shape.before(s, lo));
            located = true;
        }
        g->s = s;
        g->b = share.b;
        g->head = head;
        g->pair = pair;
        g->t0 = t0;
        g->tiles = shape.tiles(s, pair);
        g->count = (int)min((int64_t)(g->tiles - t0), share.left);
        g->token0 = pair * 2 * shape.tokens;
        g->both = s.count > g->token0 + shape.tokens;
        share.left -= g->count;
        t0 = 0;
        if (++pair == all) pair = 0, ++head;
        return true;
    }
};

template <typename T, int DP>
__global__ void __launch_bounds__(CHUNK_THREADS, 1)
    kv_chunk_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, KvPages c, KvBatch bt, KvAttend a, KvParts parts) {
    constexpr int HALVES = DP / 64, KS = DP / 16, RING = CHUNK_RING<DP>, SLOT = CHUNK_SLOT<DP>;
    constexpr uint32_t TM_S = 0, TM_O = 256;  // columns: S (and P) of the two tiles, O of the two
    extern __shared__ __align__(1024) uint8_t ring[];  // the swizzle goes by address bits: 1024-byte aligned
    uint8_t* smem_q = ring + RING * SLOT;
    uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem_q + CHUNK_Q<DP>);
    uint64_t* kv_empty = kv_full + RING;
    uint64_t* q_full = kv_empty + RING;
    uint64_t* q_empty = q_full + 1;
    uint64_t* s_full = q_empty + 1;  // [2]
    uint64_t* p_full = s_full + 2;
    uint64_t* o_full = p_full + 2;
    int64_t* scratch = reinterpret_cast<int64_t*>(o_full + 2);  // THREADS / 32 + 2
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(scratch + CHUNK_THREADS / 32 + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < RING; ++i) {
            mbar_init(kv_full + i, 1);
            mbar_init(kv_empty + i, 1);
        }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 128);
            mbar_init(o_full + i, 1);
        }
        fence_mbar_init();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // query rows past a tile's tokens are never loaded
    for (int i = threadIdx.x; i < CHUNK_Q<DP> / 16; i += CHUNK_THREADS)
        reinterpret_cast<uint4*>(smem_q)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
    tmem_fence_before();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const ChunkShape shape{a.group, a.causal, CHUNK_ROWS / a.group};
    KvShare share = kv_share<CHUNK_THREADS>(c, bt, scratch, [&](const KvSeq& s) -> int64_t {
        return shape.takes(s) ? shape.before(s, shape.pairs(s)) * c.heads : 0;
    });
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x < 2) parts.at[2 * blockIdx.x + threadIdx.x].w = PART_NONE;
    __syncthreads();
    tmem_fence_after();
    const uint32_t tm = *tmem_at;
    KvWait wait{c.status};
    ChunkWalk walk{c, bt, shape, share, 0, 0, 0, false};
    ChunkSegment g;
    int slot = 0;  // of the ring
    uint32_t phase = 0;
    const int box_shift = min(c.page_shift, 6);
    // 384 threads start with 168 registers: 2 x 128 x 216 + 128 x 72 is the same sum
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 9) {
            int loaded = 0;
            uint32_t q_phase = 0;
            while (walk.next(&g)) {
                wait(q_empty, q_phase ^ 1);
                if (lane == 0) {
                    const int n = g.both ? 2 : 1;
                    mbar_arrive_expect_tx(q_full, n * HALVES * shape.tokens * a.group * 128);
                    for (int i = 0; i < n; ++i)
                        for (int h = 0; h < HALVES; ++h)
                            tma_rows(smem_q + (i * HALVES + h) * (CHUNK_ROWS * 128), &map_q, h * 64, g.head * a.group,
                                     (int)g.s.first + g.token0 + i * shape.tokens, q_full);
                }
                q_phase ^= 1;
                const int32_t* table = bt.table + g.b * bt.table_stride;
                const int boxes = CHUNK_SLOTS >> box_shift, i = lane % boxes, half = lane / boxes;
                for (int t = g.t0; t < g.t0 + g.count; ++t) {
                    const int at = t * CHUNK_SLOTS + (i << box_shift);
                    const bool live = half < HALVES && at < g.s.len;
                    int page = 0;
                    if (live) {
                        page = (int)kv_page(c, table, at);
                        if (page < 0) page = (int)c.pages;  // past the map: reads as zero
                    }
                    const int n = __popc(__ballot_sync(FULL, live));
                    for (int side = 0; side < 2; ++side) {
                        wait(kv_empty + slot, phase ^ 1);
                        if (lane == 0) mbar_arrive_expect_tx(kv_full + slot, n * (128 << box_shift));
                        __syncwarp();
                        if (live)
                            tma_page(ring + slot * SLOT + half * (CHUNK_SLOTS * 128) + (i << box_shift) * 128,
                                     side ? &map_v : &map_k, half * 64, at & ((1 << c.page_shift) - 1), g.head, page,
                                     kv_full + slot);
                        ++loaded;
                        if (++slot == RING) slot = 0, phase ^= 1;
                    }
                }
            }
            // A wait that ran out may have left copies in flight into this CTA's memory: see them land before it ends.
            if (wait.dead && lane == 0)
                for (int i = 0; i < RING; ++i) {
                    const int fills = loaded / RING + (i < loaded % RING);
                    if (fills && !mbar_wait_bounded(kv_full + i, (fills - 1) & 1, 2 * KV_WAIT_BUDGET))
                        atomicOr(c.status, ERR_DRAIN_TIMEOUT);
                }
        } else if (warp == 8) {
            uint32_t q_phase = 0, p_phase[2] = {0, 0};
            while (walk.next(&g)) {
                const uint32_t idesc_s = umma_idesc<T>(CHUNK_SLOTS, false, a.scale < 0.f);
                const uint32_t idesc_o = umma_idesc<T>(DP, true, false);
                auto scores = [&](int i) {  // S_i = Q_i K^T, K in the current ring slot
                    if (lane == 0) {
                        const uint32_t q = smem_u32(smem_q) + i * HALVES * (CHUNK_ROWS * 128), k = smem_u32(ring + slot * SLOT);
#pragma unroll
                        for (int e = 0; e < KS; ++e) {
                            const uint32_t off = (e >> 2) * (CHUNK_ROWS * 128) + (e & 3) * 32;
                            umma_ss(tm + TM_S + i * 128, umma_desc(q + off, 16, 1024), umma_desc(k + off, 16, 1024), idesc_s,
                                    e > 0);
                        }
                        umma_commit(s_full + i);
                    }
                    __syncwarp();
                };
                auto advance = [&] {
                    if (++slot == RING) slot = 0, phase ^= 1;
                };
                wait(q_full, q_phase);
                q_phase ^= 1;
                wait(kv_full + slot, phase);
                tmem_fence_after();
                scores(0);
                if (g.both) scores(1);
                if (lane == 0) {
                    umma_commit(kv_empty + slot);
                    if (g.count == 1) umma_commit(q_empty);
                }
                __syncwarp();
                advance();
                for (int t = g.t0; t < g.t0 + g.count; ++t) {
                    // values of tile t in the current slot, keys of tile t + 1 in the next one
                    const int v_slot = slot;
                    const int held = min(CHUNK_SLOTS, g.s.len - t * CHUNK_SLOTS);  // slots of the sequence in this tile
                    wait(kv_full + slot, phase);
                    if (held < CHUNK_SLOTS && (held & 15) && held > 0) {
                        // The page's slots past the sequence hold anything: none may meet a weight of zero. The product stops
                        // at the 16 slots that hold the last one; their rest is cleared.
                        for (int r = held; r < (held + 15) / 16 * 16; ++r)
                            if (lane < 8 * HALVES)
                                *reinterpret_cast<uint4*>(ring + v_slot * SLOT + (lane >> 3) * (CHUNK_SLOTS * 128) + r * 128 +
                                                          (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    const int steps = max(1, (min(held, CHUNK_SLOTS) + 15) / 16);
                    const bool more = t + 1 < g.t0 + g.count;
                    advance();
                    for (int i = 0; i < (g.both ? 2 : 1); ++i) {
                        wait(p_full + i, p_phase[i]);
                        p_phase[i] ^= 1;
                        tmem_fence_after();
                        if (lane == 0 && held > 0) {
                            const uint32_t v = smem_u32(ring + v_slot * SLOT);
                            for (int e = 0; e < steps; ++e)
                                umma_ts(tm + TM_O + i * 128, tm + TM_S + i * 128 + e * 8,
                                        umma_desc(v + e * 2048, CHUNK_SLOTS * 128, 1024), idesc_o, t > g.t0 || e > 0);
                        }
                        __syncwarp();
                        if (more) {
                            if (i == 0) {
                                wait(kv_full + slot, phase);
                                tmem_fence_after();
                            }
                            scores(i);
                        } else if (lane == 0) {
                            umma_commit(o_full + i);
                        }
                    }
                    if (lane == 0) umma_commit(kv_empty + v_slot);
                    if (more) {
                        if (lane == 0) {
                            umma_commit(kv_empty + slot);
                            if (t + 2 == g.t0 + g.count) umma_commit(q_empty);
                        }
                        advance();
                    }
                    __syncwarp();
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        uint32_t s_phase = 0, o_phase = 0;
        bool first_segment = true;
        while (walk.next(&g)) {
            const int i = warp >> 2, r = (warp & 3) * 32 + lane;
            const uint32_t lanes = tm + ((uint32_t)((warp & 3) * 32) << 16);
            const uint32_t tm_s = lanes + TM_S + i * 128, tm_o = lanes + TM_O + i * 128;
            const int token = g.token0 + i * shape.tokens + r / a.group;
            const bool live = r < shape.tokens * a.group && token < g.s.count;
            const int lim = live ? max(0, row_limit(g.s, a.causal, token)) : 0;
            const int open = max(0, min(g.s.len, row_limit(g.s, a.causal, g.token0 + i * shape.tokens)));  // every row sees these
            // base 2; a scale of zero keeps -inf what it is
            const float scale = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-37f);
            float m = -INFINITY, l = 0.f;
            if (i == 0 || g.both) {
                for (int t = g.t0; t < g.t0 + g.count; ++t) {
                    float x[CHUNK_SLOTS];
                    wait(s_full + i, s_phase);
                    s_phase ^= 1;
                    tmem_fence_after();
#pragma unroll
                    for (int e = 0; e < 4; ++e) tmem_ld32(tm_s + 32 * e, x + 32 * e);
                    tmem_wait_ld();
                    if ((t + 1) * CHUNK_SLOTS > open) {
                        const int see = lim - t * CHUNK_SLOTS;
#pragma unroll
                        for (int e = 0; e < CHUNK_SLOTS; ++e) x[e] = e < see ? x[e] : -INFINITY;
                    }
                    float top4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                    for (int e = 4; e < CHUNK_SLOTS; ++e) top4[e & 3] = fmaxf(top4[e & 3], x[e]);
                    const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
                    const bool grow = (top - m) * scale > 8.f;  // m = -inf: unless all is masked
                    if (t == g.t0) {
                        m = top;
                    } else if (__any_sync(FULL, grow)) {
                        const float f = grow ? (m == -INFINITY ? 0.f : ex2((m - top) * scale)) : 1.f;
                        if (grow) m = top;
                        l *= f;
#pragma unroll 1
                        for (int e = 0; e < DP; e += 32) {
                            float o[32];
                            tmem_ld32(tm_o + e, o);
                            tmem_wait_ld();
                            uint32_t w[32];
#pragma unroll
                            for (int k = 0; k < 32; ++k) w[k] = __float_as_uint(o[k] * f);
                            tmem_st32(tm_o + e, w);
                        }
                    }
                    const float ref = m == -INFINITY ? 0.f : m * scale;
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
                    uint32_t p[CHUNK_SLOTS / 2];
#pragma unroll
                    for (int e = 0; e < CHUNK_SLOTS; e += 2) {
                        const float y0 = ex2(fmaf(x[e], scale, -ref)), y1 = ex2(fmaf(x[e + 1], scale, -ref));
                        sum[e & 3] += y0;
                        sum[(e & 3) + 1] += y1;
                        p[e / 2] = pack2<T>(y0, y1);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tmem_st32(tm_s, p);
                    tmem_st32(tm_s + 32, p + 32);
                    tmem_wait_st();
                    tmem_fence_before();
                    mbar_arrive(p_full + i);
                }
                wait(o_full + i, o_phase);
                o_phase ^= 1;
                tmem_fence_after();
                const bool whole = g.count == g.tiles;
                const bool none = g.t0 * CHUNK_SLOTS >= g.s.len;  // no product was made: O holds anything
                const int64_t part = 2 * (int64_t)blockIdx.x + (first_segment ? 0 : 1);
                const int h = g.head * a.group + r % a.group;
                const int64_t tok = g.s.first + token;
                const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
#pragma unroll 1
                for (int e = 0; e < DP; e += 32) {
                    float o[32];
                    tmem_ld32(tm_o + e, o);
                    tmem_wait_ld();
                    if (none)
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = 0.f;
                    if (live && whole) {
                        uint4* out = reinterpret_cast<uint4*>(a.out + tok * a.os[0] + h * a.os[1] + e);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (e + 8 * k < c.dim)
                                out[k] = make_uint4(pack2<T>(o[8 * k] * inv, o[8 * k + 1] * inv),
                                                    pack2<T>(o[8 * k + 2] * inv, o[8 * k + 3] * inv),
                                                    pack2<T>(o[8 * k + 4] * inv, o[8 * k + 5] * inv),
                                                    pack2<T>(o[8 * k + 6] * inv, o[8 * k + 7] * inv));
                    } else if (live) {
                        float4* po = reinterpret_cast<float4*>(parts.o + (part * CHUNK_PART_ROWS + i * CHUNK_ROWS + r) * DP + e);
#pragma unroll
                        for (int k = 0; k < 8; ++k) po[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                    }
                }
                const float top = m == -INFINITY ? -INFINITY : m * scale;
                if (live && whole) a.lse[tok * a.heads + h] = (top + log2f(l)) * 0.6931471805599453f;
                else if (live) parts.ml[part * CHUNK_PART_ROWS + i * CHUNK_ROWS + r] = make_float2(top, l);
                if (!whole && threadIdx.x == 0)
                    parts.at[part] = make_int4(g.b, g.head, g.pair, PART_HELD | (g.t0 == 0 ? PART_FIRST : 0) |
                                                                        (g.t0 + g.count == g.tiles ? PART_LAST : 0));
                tmem_fence_before();
            }
            first_segment = false;
        }
    }
    __syncthreads();
    if (warp == 8) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm) : "memory");
    }
}

}  // namespace vk
