// Attention of a chunk of new tokens over the paged cache on the 5th-generation tensor cores.
//
// A kv head's rows (tokens x its query heads, token by token) come in tiles of 128, the tensor memory's lanes: with 5
// query heads to a kv head a tile holds 25 tokens, 125 rows. A unit of work is a pair of row tiles against 128 slots or,
// where a sequence's last pair has one tile only, that tile against 2 x 128 slots; the units of all (sequence, kv head,
// pair)s are laid end to end and every CTA takes an equal share, so that neither the causal mask nor ragged lengths nor
// few rows over a long cache leave SMs idle; cut pairs are finished from parts as in the step kernel.
//
// Per unit and tile: scores S = Q K^T (tcgen05.mma, both operands in shared memory) into tensor memory; a warpgroup, one
// row per thread, takes the maximum, exponentials and their sum, and puts the weights P as 16-bit values where S was;
// O += P V with P from tensor memory. While one tile's warpgroup works, the tensor cores do the other tile's products.
// O stays in tensor memory; it is rescaled only when a row's maximum has grown by more than 2^8 since the reference that
// its weights use, which the sums allow (weights up to 256 in 16 bits keep their relative precision).
//
// Bound: 4 x 128 x 128 x head size operations per tile and unit on the tensor cores (1,024 cycles at a head size of 128)
// and 128 x 128 exponentials on the special function units (1,024 cycles as well). Tensor memory holds S and O of two
// tiles and no more, so a tile's products wait for its weights and the other way round: a unit takes as long as one tile's
// weights (1,400 cycles), its products (1,200) and the hand-overs between them (800), while the other tile fills the gaps.
// Measured (4,096 tokens over 16,384 slots, 32 heads over 8, head size 128): 860-873 us, 1,100-1,120 TFLOP/s, in a run of
// many, where power holds the clock down; 738 us, 1,300 TFLOP/s, for eight calls from rest. Tensor pipe and special function
// units are each busy for 64 % of it. What did not pay, measured from rest against the 752 us of the time: a part of the
// exponentials by a polynomial (1 in 8: 758 us, 2 in 8: 777), the weights handed over in two halves (770), a warp of its own
// for each tile's products (920; taking turns 781).
//
// The weights are rounded to the cache's 16-bit type, as in the step kernel; scores, references, sums and O are 32-bit. Which
// rows of a warp move their reference together depends on the tile's rows, so that a row's last bit may depend on its
// neighbours; equal calls give equal bits.
#pragma once
#include "kv_step.cuh"

namespace vk {

constexpr int CHUNK_ROWS = 128;                 // rows of a tile
constexpr int CHUNK_SLOTS = 128;                // slots of a unit
constexpr float CHUNK_PART_COST = 0.8f;         // of a unit
constexpr int CHUNK_THREADS = 384;              // two softmax warpgroups; one with the MMA warp and the loading warp
template <int DP>
constexpr int CHUNK_Q = 2 * CHUNK_ROWS * DP * 2;   // bytes of the two query tiles
template <int DP>
constexpr int CHUNK_SLOT = CHUNK_SLOTS * DP * 2;   // bytes of a tile of keys or values
template <int DP>
constexpr int CHUNK_RING = DP == 128 ? 5 : 10;     // tiles in flight, keys and values alternating
template <int DP>
constexpr int chunk_smem() {
    return CHUNK_Q<DP> + CHUNK_RING<DP> * CHUNK_SLOT<DP> + 2 * CHUNK_ROWS * 8 + 512;
}

// A row tile's box of the queries (64 elements of a kv head's query heads, for a tile's tokens) into shared memory.
__device__ __forceinline__ void tma_rows(void* dst, const CUtensorMap* map, int d, int head, int token, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(d), "r"(head), "r"(token), "r"(smem_u32(bar))
        : "memory");
}

static_assert(2 * chunk_smem<64>() > 233472 && 2 * chunk_smem<128>() > 233472, "one CTA per SM: each takes all tensor memory");

// ---- tcgen05
// A descriptor's low word holds the operand's address and leading offset in units of 16 bytes, so that the next step's
// operand is one 32-bit addition away; the high word is constant: 8-row groups 1,024 bytes apart, descriptor version 1,
// 128-byte swizzle.
//
// The instructions below are reached by a whole warp and take effect for the lane that `me` is nonzero in. Issued inside
// a branch of that lane instead, every operand was moved from the lane's to the warp's registers anew, about 100 cycles
// per product: the warp that issues them was the kernel's bound (4,096 tokens over 16,384 slots, 32 heads over 8:
// 1,105 us then, 770 when this came). `me` is what elect.sync gave: with the first lane's, computed, the case took 982 us in
// a run of many, 860 with this.
constexpr uint32_t UMMA_HIGH = 1024u >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t umma_low(uint32_t addr, uint32_t lead) { return addr >> 4 | (lead >> 4) << 16; }
template <typename T>
__device__ __forceinline__ uint32_t umma_idesc(int n, bool b_by_rows, bool negate) {
    const uint32_t type = std::is_same_v<T, __half> ? 0u : 1u;
    return 1u << 4 | type << 7 | type << 10 | (negate ? 1u << 13 : 0u) | (b_by_rows ? 1u << 16 : 0u) |
           (uint32_t)(n >> 3) << 17 | (uint32_t)(CHUNK_ROWS >> 4) << 24;
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add, uint32_t me) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
        "mov.b64 da, {%1, %6};\n\tmov.b64 db, {%2, %6};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(me), "n"(UMMA_HIGH)
        : "memory");
}
// A from tensor memory.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add, uint32_t me) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
        "mov.b64 db, {%2, %6};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(me), "n"(UMMA_HIGH)
        : "memory");
}
// The barrier gets an arrival when all products that this lane issued so far are done.
__device__ __forceinline__ void umma_commit(uint64_t* bar, uint32_t me) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(me)
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
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* x) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
        VK_W8(x, 0), VK_W8(x, 8)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t* x) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
        VK_W8(x, 0), VK_W8(x, 8), VK_W8(x, 16), VK_W8(x, 24)
        : "memory");
}

// ---- two 32-bit values at a time
struct Pair {
    unsigned long long v;
};
__device__ __forceinline__ Pair pair_of(float x, float y) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(x), "f"(y));
    return p;
}
__device__ __forceinline__ float2 floats(Pair p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
    return f;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
    Pair p;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
    return p;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair p;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return p;
}
// ---- the order of units
// sum of floor((a i + b) / m) over 0 <= i < n, by Euclid's steps on (m, a): taking out the whole parts of a / m and b / m
// leaves a sum of the same kind with a and m exchanged (such sums: Graham, Knuth and Patashnik, "Concrete Mathematics",
// section 3.5). The sum is below 2^31 (the host has checked the units), so that arithmetic modulo 2^32 gives it; a n + b after
// the first reduction is below m (n + 1).
__device__ __forceinline__ uint32_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
    uint32_t sum = 0;
    while (n > 0) {
        const uint32_t qa = a / m, qb = b / m;
        sum += ((n & 1) ? n * ((n - 1) / 2) : n / 2 * (n - 1)) * qa + n * qb;
        a -= qa * m;
        b -= qb * m;
        const uint32_t y = a * n + b;
        if (y < m) break;
        n = y / m;
        b = y - n * m;
        const uint32_t t = m;
        m = a;
        a = t;
    }
    return sum;
}

// The last of `all` pairs with before(pair) <= off, by a whole warp: 32 candidates at a time.
template <class Before>
__device__ __forceinline__ int locate_pair(int all, int off, Before&& before) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = all;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const unsigned fits = __ballot_sync(FULL, at < hi && before(min(at, hi - 1)) <= off);
        lo += (31 - __clz(fits)) * step;  // lane 0's candidate always fits
        hi = min(hi, lo + step);
    }
    return lo;
}

struct ChunkShape {
    const KvAttend& a;
    int tokens;  // of a row tile
    __device__ __forceinline__ bool takes(const KvSeq& s) const { return s.count > 0; }
    __device__ __forceinline__ int pairs(const KvSeq& s) const { return (int)a.by_pair(s.count + 2 * tokens - 1); }
    // a sequence's last pair may have one tile only
    __device__ __forceinline__ bool lone(const KvSeq& s, int pair) const { return s.count <= (2 * pair + 1) * tokens; }
    // slots that the pair's last row sees
    __device__ __forceinline__ int limit(const KvSeq& s, int pair) const {
        return a.causal ? max(0, s.len - s.count + min(s.count, (pair + 1) * 2 * tokens)) : s.len;
    }
    __device__ __forceinline__ int units(const KvSeq& s, int pair) const {
        const int n = lone(s, pair) ? 2 * CHUNK_SLOTS : CHUNK_SLOTS;
        return max(1, (limit(s, pair) + n - 1) / n);
    }
    // units of the pairs before `pair`
    __device__ __forceinline__ int before(const KvSeq& s, int pair) const {
        const int all = pairs(s), n = min(pair, all - 1), per = 2 * tokens;
        const int ahead = s.len - s.count;  // more than -2^31: both are counts
        int sum;
        if (!a.causal) {
            sum = n * max(1, (s.len + CHUNK_SLOTS - 1) / CHUNK_SLOTS);
        } else {
            const int one = ahead > CHUNK_SLOTS ? 0 : min(n, (int)a.by_pair(CHUNK_SLOTS - ahead));  // pairs of one unit
            sum = one + (int)floor_sum(n - one, CHUNK_SLOTS, per, ahead + (one + 1) * per + CHUNK_SLOTS - 1);
        }
        return pair < all ? sum : sum + units(s, all - 1);
    }
};

// A CTA's next segment: consecutive units of one (sequence, kv head, pair).
struct ChunkSegment {
    KvSeq s;
    int b, head, t0, count, units;
    int token0;  // of the pair's first row
    bool lone;
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
            const int per = shape.before(s, all);
            int off = share.off;
            for (head = 0; off >= per; ++head) off -= per;
            pair = locate_pair(all, off, [&](int p) { return shape.before(s, p); });
            t0 = off - shape.before(s, pair);
            located = true;
        }
        g->s = s;
        g->b = share.b;
        g->head = head;
        g->t0 = t0;
        g->units = shape.units(s, pair);
        g->count = min(g->units - t0, share.left);
        g->token0 = pair * 2 * shape.tokens;
        g->lone = shape.lone(s, pair);
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
    float2* lone_ml = reinterpret_cast<float2*>(smem_q + CHUNK_Q<DP>);  // [warpgroup][row] of a lone tile
    uint64_t* kv_full = reinterpret_cast<uint64_t*>(lone_ml + 2 * CHUNK_ROWS);
    uint64_t* kv_empty = kv_full + RING;
    uint64_t* q_full = kv_empty + RING;
    uint64_t* q_empty = q_full + 1;
    uint64_t* s_full = q_empty + 1;  // [tile]
    uint64_t* p_full = s_full + 2;
    uint64_t* o_full = p_full + 2;
    uint64_t* mma_done = o_full + 2;
    int* scratch = reinterpret_cast<int*>(mma_done + 1);
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(scratch + KV_SHARE_SCRATCH);
    const int warp = __shfl_sync(FULL, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        prefetch_map(&map_q);
        prefetch_map(&map_k);
        prefetch_map(&map_v);
        for (int i = 0; i < RING; ++i) {
            mbar_init(kv_full + i, 1);
            mbar_init(kv_empty + i, 1);
        }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(mma_done, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 4);
            mbar_init(o_full + i, 1);
        }
        fence_mbar_init();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (a.tokens * a.group < CHUNK_ROWS) {  // the other rows are never loaded
        for (int i = threadIdx.x; i < CHUNK_Q<DP> / 16; i += CHUNK_THREADS)
            reinterpret_cast<uint4*>(smem_q)[i] = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
    }
    tmem_fence_before();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const ChunkShape shape{a, a.tokens};
    KvShare share = kv_share<CHUNK_THREADS>(c, bt, parts, scratch, CHUNK_PART_COST, [&](const KvSeq& s, int* longest) {
        if (!shape.takes(s)) return 0;
        const int pairs = shape.pairs(s);
        *longest = max(*longest, max(shape.units(s, pairs - 1), shape.units(s, max(0, pairs - 2))));
        return shape.before(s, pairs) * c.heads;
    });
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    tmem_fence_after();
    const uint32_t tm = __shfl_sync(FULL, *tmem_at, 0);
    KvWait wait{c.status, parts.bad, a.wait_limit};
    ChunkWalk walk{c, bt, shape, share, 0, 0, 0, false};
    ChunkSegment g;
    // 384 threads start with 168 registers: 2 x 128 x 200 + 128 x 104 is the same sum
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        // The ring's n-th fill; a segment's tiles come as keys, values, keys, values.
        int fill = 0;
        auto at = [&](int n) { return n % RING; };
        auto parity = [&](int n) -> uint32_t { return n / RING & 1; };
        if (warp == 9) {
            uint32_t q_phase = 0;
            int q_fills = 0;
            const int box_shift = min(c.page_shift, 6);
            const int boxes = CHUNK_SLOTS >> box_shift;
            const uint32_t me = elect_lane();
            while (!wait.dead && walk.next(&g)) {
                wait.together(q_empty, q_phase ^ 1);
                if (wait.dead) break;
                q_phase ^= 1;
                ++q_fills;
                if (lane == 0) {
                    const int n = g.lone ? 1 : 2;
                    mbar_arrive_expect_tx(q_full, n * HALVES * shape.tokens * a.group * 128);
                    for (int k = 0; k < n; ++k)
                        for (int h = 0; h < HALVES; ++h)
                            tma_rows(smem_q + (k * HALVES + h) * (CHUNK_ROWS * 128), &map_q, h * 64, g.head * a.group,
                                     (int)g.s.first + g.token0 + k * shape.tokens, q_full);
                }
                const int32_t* table = bt.table + g.b * bt.table_stride;
                const int per = g.lone ? 2 : 1;
                const int end = (g.t0 + g.count) * per;
                int entry = tile_entries(c, table, g.t0 * per * CHUNK_SLOTS, boxes, box_shift, g.s.len);
                for (int t = g.t0 * per; t < end && !wait.dead; ++t) {
                    const TilePages tp = tile_pages(c, entry, t * CHUNK_SLOTS, boxes, box_shift, g.s.len);
                    if (t + 1 < end) entry = tile_entries(c, table, (t + 1) * CHUNK_SLOTS, boxes, box_shift, g.s.len);
                    // rolled: this warp's registers are few, and what it spills the other one waits for
#pragma unroll 1
                    for (int side = 0; side < 2; ++side, ++fill) {
                        const int slot = at(fill);
                        wait.together(kv_empty + slot, parity(fill) ^ 1);
                        if (wait.dead) break;
                        if (lane == 0) mbar_arrive_expect_tx(kv_full + slot, tp.count * HALVES * (128 << box_shift));
                        __syncwarp();
                        uint8_t* dst = ring + slot * SLOT;
#pragma unroll 2
                        for (int i = 0; i < tp.count; ++i) {
                            const int page = __shfl_sync(FULL, tp.page, i), from = i << box_shift;
                            const int in = (t * CHUNK_SLOTS + from) & ((1 << c.page_shift) - 1);
#pragma unroll
                            for (int half = 0; half < HALVES; ++half)
                                tma_page(dst + half * (CHUNK_SLOTS * 128) + from * 128, side ? &map_v : &map_k, half * 64, in,
                                         g.head, page, kv_full + slot, me);
                        }
                    }
                }
            }
            if (lane == 0) {
                wait.drain(q_full, q_fills);
                for (int i = 0; i < RING; ++i) wait.drain(kv_full + i, fill / RING + (i < fill % RING));
            }
        } else if (warp == 8) {
            uint32_t q_phase = 0, p_phase = 0;  // p_phase: bit per tile
            const uint32_t me = elect_lane();
            const int ks = (c.dim + 15) / 16;  // steps of 16 elements; the padding's products are left out
            const uint32_t idesc_s = umma_idesc<T>(CHUNK_SLOTS, false, a.scale < 0.f);
            const uint32_t idesc_o = umma_idesc<T>(ks * 16, true, false);
            const uint32_t q_low = umma_low(smem_u32(smem_q), 16), k_low = umma_low(smem_u32(ring), 16);
            const uint32_t v_low = umma_low(smem_u32(ring), CHUNK_SLOTS * 128);
            while (walk.next(&g)) {
                const bool lone = __shfl_sync(FULL, g.lone, 0);
                const int count = __shfl_sync(FULL, g.count, 0), step = lone ? 4 : 2;
                // keys of tile i's part of unit u of this segment, and its values the fill after it
                auto key_fill = [&](int u, int i) { return fill + u * step + (lone ? 2 * i : 0); };
                auto scores = [&](int u, int i) {  // S_i = Q_i K^T
                    const int n = key_fill(u, i), slot = at(n);
                    const uint32_t q = q_low + (lone ? 0 : i * HALVES * (CHUNK_ROWS * 8)), k = k_low + slot * (SLOT / 16);
                    if (lone || i == 0) wait(kv_full + slot, parity(n));
                    tmem_fence_after();
                    if (ks == KS) {
#pragma unroll
                        for (int e = 0; e < KS; ++e) {
                            const uint32_t off = (e >> 2) * (CHUNK_ROWS * 8) + (e & 3) * 2;
                            umma_ss(tm + TM_S + i * 128, q + off, k + off, idesc_s, e > 0, me);
                        }
                    } else {
#pragma unroll 1
                        for (int e = 0; e < ks; ++e) {
                            const uint32_t off = (e >> 2) * (CHUNK_ROWS * 8) + (e & 3) * 2;
                            umma_ss(tm + TM_S + i * 128, q + off, k + off, idesc_s, e > 0, me);
                        }
                    }
                    umma_commit(s_full + i, me);
                    if (lone || i == 1) umma_commit(kv_empty + slot, wait.live(me));
                };
                wait(q_full, q_phase);
                q_phase ^= 1;
                scores(0, 0);
                scores(0, 1);
                if (count == 1) umma_commit(q_empty, wait.live(me));
                for (int u = 0; u < count; ++u) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int n = key_fill(u, i) + 1, slot = at(n);
                        // slots of the sequence in this tile
                        const int held = __shfl_sync(FULL, g.s.len - (lone ? 2 * (g.t0 + u) + i : g.t0 + u) * CHUNK_SLOTS, 0);
                        const uint32_t v = v_low + slot * (SLOT / 16), p = tm + TM_S + i * 128, o = tm + TM_O + i * 128;
                        if (lone || i == 0) wait(kv_full + slot, parity(n));
                        if (held > 0 && held < CHUNK_SLOTS && (held & 15) && (lone || i == 0)) {
                            // The page's slots past the sequence hold anything: none may meet a weight of zero. The
                            // product stops at the 16 slots that hold the last one; their rest is cleared.
                            for (int r = held; r < (held + 15) / 16 * 16; ++r)
                                if (lane < 8 * HALVES)
                                    *reinterpret_cast<uint4*>(ring + slot * SLOT + (lane >> 3) * (CHUNK_SLOTS * 128) +
                                                              r * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                            fence_proxy_async_smem();
                            __syncwarp();
                        }
                        wait(p_full + i, p_phase >> i & 1);
                        tmem_fence_after();
                        if (held >= CHUNK_SLOTS) {
#pragma unroll
                            for (int e = 0; e < CHUNK_SLOTS / 16; ++e)
                                umma_ts(o, p + e * 8, v + e * 128, idesc_o, u > 0 || e > 0, me);
                        } else {
#pragma unroll 1
                            for (int e = 0; 16 * e < held; ++e)
                                umma_ts(o, p + e * 8, v + e * 128, idesc_o, u > 0 || e > 0, me);
                        }
                        p_phase ^= 1u << i;
                        if (lone || i == 1) umma_commit(kv_empty + slot, wait.live(me));
                        if (u + 1 < count) scores(u + 1, i);
                        else umma_commit(o_full + i, me);
                    }
                    if (u + 2 == count) umma_commit(q_empty, wait.live(me));
                }
                fill += count * step;
            }
            umma_commit(mma_done, me);
            if (lane == 0) wait.drain(mma_done, 1);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int i = warp >> 2, r = (warp & 3) * 32 + lane;  // tile and row
        const int r_token = (int)a.by_group(r);
        const uint32_t lanes = tm + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t tm_s = lanes + TM_S + i * 128, tm_o = lanes + TM_O + i * 128;
        // base 2; a scale of zero keeps -inf what it is
        const float scale = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-37f);
        uint32_t s_phase = 0, o_phase = 0;
        while (walk.next(&g)) {
            const int token1 = g.token0 + (g.lone ? 0 : i * shape.tokens);  // of the tile's first row
            const int token = token1 + r_token;
            const bool live = r < shape.tokens * a.group && token < g.s.count;
            const int lim = live ? max(0, row_limit(g.s, a.causal, token)) : 0;
            const int open = max(0, min(g.s.len, row_limit(g.s, a.causal, token1)));  // slots that every row sees
            float ref = 0.f, l = 0.f;  // base 2
            for (int t = g.t0; t < g.t0 + g.count; ++t) {
                const int slot0 = (g.lone ? 2 * t + i : t) * CHUNK_SLOTS;
                float x[CHUNK_SLOTS];
                wait(s_full + i, s_phase);
                s_phase ^= 1;
                tmem_fence_after();
#pragma unroll
                for (int e = 0; e < 4; ++e) tmem_ld32(tm_s + 32 * e, x + 32 * e);
                tmem_wait_ld();
                const bool masked = slot0 + CHUNK_SLOTS > open;
                if (masked) {
                    const int see = lim - slot0;
#pragma unroll
                    for (int e = 0; e < CHUNK_SLOTS; ++e) x[e] = e < see ? x[e] : -INFINITY;
                }
                // Weights are taken against the reference so far. Their sum says whether one may have outgrown 2^8; only
                // then, and in a segment's first tile, is the maximum looked for and the reference moved. (A row that
                // sees nothing of its first tile sees nothing of the later ones.)
                const Pair scale2 = pair_of(scale, scale);
                float sum = 0.f;
                auto weights = [&] {
                    const Pair ref2 = pair_of(-ref, -ref);
                    Pair part[2] = {pair_of(0.f, 0.f), pair_of(0.f, 0.f)};
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        uint32_t p[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int k = 32 * h + 2 * e;
                            const Pair y = fma2(pair_of(x[k], x[k + 1]), scale2, ref2);
                            const float2 z = floats(y), w = make_float2(ex2(z.x), ex2(z.y));
                            part[e & 1] = part[e & 1] + pair_of(w.x, w.y);
                            p[e] = pack2<T>(w.x, w.y);
                        }
                        tmem_st16(tm_s + 16 * h, p);
                    }
                    const float2 w = floats(part[0] + part[1]);
                    sum = w.x + w.y;
                };
                if (t > g.t0) weights();
                if (t == g.t0 || __any_sync(FULL, sum > 256.f)) {
                    float top = fmaxf(x[0], x[1]), top_b = fmaxf(x[2], x[3]);
#pragma unroll
                    for (int e = 4; e < CHUNK_SLOTS; e += 4) {
                        top = fmaxf(fmaxf(top, x[e]), x[e + 1]);
                        top_b = fmaxf(fmaxf(top_b, x[e + 2]), x[e + 3]);
                    }
                    top = fmaxf(top, top_b) * scale;
                    if (t == g.t0) {
                        ref = top == -INFINITY ? 0.f : top;
                    } else {
                        const float f = top > ref ? ex2(ref - top) : 1.f;
                        ref = fmaxf(ref, top);
                        l *= f;
#pragma unroll 1
                        for (int e = 0; e < c.dim; e += 32) {
                            float o[32];
                            __syncwarp();
                            tmem_ld32(tm_o + e, o);
                            tmem_wait_ld();
                            uint32_t w[32];
#pragma unroll
                            for (int k = 0; k < 32; ++k) w[k] = __float_as_uint(o[k] * f);
                            tmem_st32(tm_o + e, w);
                        }
                    }
                    weights();
                }
                l += sum;
                tmem_wait_st();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + i);
            }
            wait(o_full + i, o_phase);
            o_phase ^= 1;
            tmem_fence_after();
            // base 2 from here on. A tile past the sequence met no product: its O holds anything.
            float top = l == 0.f ? -INFINITY : ref, total = l, f_mine = 1.f, f_other = 0.f;
            if (g.lone) {  // each warpgroup joins the two for half of the elements
                const float mine = top;
                lone_ml[i * CHUNK_ROWS + r] = make_float2(top, total);
                tmem_fence_before();
                bar_sync(3, 256);
                tmem_fence_after();
                const float2 ml = lone_ml[(i ^ 1) * CHUNK_ROWS + r];
                top = fmaxf(top, ml.x);
                f_mine = part_factor(mine, top);
                f_other = part_factor(ml.x, top);
                total = total * f_mine + ml.y * f_other;
            }
            const int64_t slot_a = (int64_t)g.t0 * (g.lone ? 2 : 1) * CHUNK_SLOTS;  // of the first unit's tiles
            const bool none_mine = slot_a + (g.lone ? i * CHUNK_SLOTS : 0) >= g.s.len;
            const bool none_other = !g.lone || slot_a + (i ^ 1) * CHUNK_SLOTS >= g.s.len;
            const int e_from = g.lone ? i * (DP / 2) : 0, e_to = g.lone && i == 0 ? min(c.dim, DP / 2) : c.dim;
            const bool leaves = g.t0 > 0;                                                       // a part for an earlier CTA
            const int follow = leaves ? 0 : walk.share.followers(g.units - g.count);  // CTAs with the rest of this one
            auto part_of = [&](int k) -> int64_t { return 2 * (int64_t)(walk.share.me + k) + i; };
            if (follow) {
                for (int k = r; k < follow; k += 128) part_await(parts, (int)part_of(1 + k), wait);
                bar_sync(1 + i, 128);
                float f = 1.f;
                for (int k0 = 0; k0 < follow; k0 += 8) {  // eight in flight; the last ones again, for nothing
                    float2 ml[8];
                    float next = top;
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        ml[k] = __ldcg(parts.ml + part_of(1 + min(k0 + k, follow - 1)) * CHUNK_ROWS + r);
#pragma unroll
                    for (int k = 0; k < 8; ++k) next = fmaxf(next, ml[k].x);
                    const float g0 = part_factor(top, next);
                    f *= g0;
                    total *= g0;
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k0 + k < follow) total += ml[k].y * part_factor(ml[k].x, next);
                    top = next;
                }
                f_mine *= f;
                f_other *= f;
            }
            const int h = g.head * a.group + r - r_token * a.group;
            const int64_t tok = g.s.first + token;
            const float inv = total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;
#pragma unroll 1
            for (int e = e_from; e < e_to; e += 32) {
                float o[32];
                __syncwarp();  // lanes without a row come from another path
                tmem_ld32(tm_o + e, o);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = none_mine ? 0.f : o[k] * f_mine;
                if (!none_other) {
                    float x[32];
                    tmem_ld32(lanes + TM_O + (i ^ 1) * 128 + e, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] += x[k] * f_other;
                }
                // parts: [four columns][row], so that a warp's accesses are contiguous
                for (int k = 0; k < follow; k += 3) {  // three in flight; the last ones again, for nothing
                    float4 y[3][8];
                    float f[3];
#pragma unroll
                    for (int u = 0; u < 3; ++u) {
                        const int64_t part = part_of(1 + min(k + u, follow - 1));
                        const float4* po =
                            reinterpret_cast<const float4*>(parts.o) + (part * (DP / 4) + e / 4) * CHUNK_ROWS + r;
                        f[u] = __ldcg(parts.ml + part * CHUNK_ROWS + r).x;
#pragma unroll
                        for (int w = 0; w < 8; ++w) y[u][w] = __ldcg(po + w * CHUNK_ROWS);
                    }
#pragma unroll
                    for (int u = 0; u < 3; ++u) {
                        f[u] = k + u < follow ? part_factor(f[u], top) : 0.f;
                        if (f[u] == 0.f) continue;
#pragma unroll
                        for (int w = 0; w < 8; ++w) {
                            o[4 * w] += y[u][w].x * f[u], o[4 * w + 1] += y[u][w].y * f[u];
                            o[4 * w + 2] += y[u][w].z * f[u], o[4 * w + 3] += y[u][w].w * f[u];
                        }
                    }
                }
                if (leaves) {
                    float4* po = reinterpret_cast<float4*>(parts.o) + (part_of(0) * (DP / 4) + e / 4) * CHUNK_ROWS + r;
#pragma unroll
                    for (int w = 0; w < 8; ++w)
                        po[w * CHUNK_ROWS] = make_float4(o[4 * w], o[4 * w + 1], o[4 * w + 2], o[4 * w + 3]);
                } else if (live) {
                    uint4* out = reinterpret_cast<uint4*>(a.out + tok * a.os[0] + h * a.os[1] + e);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (e + 8 * k < c.dim)
                            out[k] = make_uint4(pack2<T>(o[8 * k] * inv, o[8 * k + 1] * inv),
                                                pack2<T>(o[8 * k + 2] * inv, o[8 * k + 3] * inv),
                                                pack2<T>(o[8 * k + 4] * inv, o[8 * k + 5] * inv),
                                                pack2<T>(o[8 * k + 6] * inv, o[8 * k + 7] * inv));
                }
            }
            tmem_fence_before();
            if (g.lone) bar_sync(3, 256);  // both have read the two sums
            if (leaves) {
                parts.ml[part_of(0) * CHUNK_ROWS + r] = make_float2(top, total);
                bar_sync(1 + i, 128);
                if (r == 0) part_publish(parts, (int)part_of(0));
            } else {
                if (live && !(g.lone && i == 1)) a.lse[tok * a.heads + h] = (top + log2f(total)) * 0.6931471805599453f;
                if (follow) {
                    bar_sync(1 + i, 128);
                    for (int k = r; k < follow; k += 128) parts.ready[part_of(1 + k)] = 0;
                }
            }
        }
    }
    __syncthreads();
    if (warp == 8) {
        __syncwarp();
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm) : "memory");
    }
}

}  // namespace vk
