// Attention of a sequence's few new tokens over the paged cache (at most 16 rows = tokens x query heads of a kv head:
// decoding steps, drafted tokens), and how a call's work is shared out.
//
// Every slot's key and value (4 x head_dim bytes per kv head) is read once and meets at most 16 rows, so the kernel is
// bound by memory. One CTA per 64-slot tile would leave SMs idle on short batches and unbalanced on ragged ones:
// instead all (sequence, kv head, tile) units are laid end to end and every CTA takes an equal, contiguous share. A
// sequence's head that a CTA holds whole is finished in place. One that is cut is finished by the CTA that holds its
// beginning, which comes to it last and finds the parts of the CTAs that follow (unnormalised sums with their maximum
// and total; they come to theirs first) in the workspace. It adds them up in order: results do not depend on timing.
// Shares are handed out from the last to the first, in the order in which CTAs start: who waits for a part waits for a CTA
// that runs already and that waits for nobody before it has made the part, whatever else has the rest of the SMs.
//
// Inside a CTA one warp keeps a ring of tiles filled by TMA (one box per page and 64 head elements, in the 128-byte
// swizzle that ldmatrix reads without conflicts); four warps take 16 slots of each tile, with their own running maximum
// and sum, on mma.sync m16n8k16: at 16 rows the tensor work is under a fifth of its rate while memory is saturated, and
// the operands stay in registers from the scores to the values, which tcgen05's 128-row tiles would not allow.
//
// The weights are rounded to the cache's 16-bit type before they meet the values, since the products take operands of one
// type; sums, maxima, totals and kept scores stay in 32 bits. Their error, 2^-9 of a weight at most, lies under the result's
// own rounding to that type.
//
// Measured: 32 sequences of up to 8,192 slots, 32 heads over 8 of 128: 118-121 us, 6.0-6.2 TB/s; one token over 1,000
// slots: 10.9 us in a graph, of which reading is one and the atomic that orders the shares 0.7. Two CTAs share an SM (at a
// head size of 64, 8 x 5 tokens over 4,001 slots: three make no difference, four take 25.8 us where two take 17.4).
#pragma once
#include <cuda.h>

#include "kv_common.cuh"

namespace vk {

constexpr int STEP_TILE = 64;  // slots of a tile
constexpr float STEP_PART_COST = 0.5f;  // of a tile
constexpr int STEP_ROWS = 16;  // most rows of a sequence's kv head
constexpr int STEP_WARPS = 4;  // consumers; one more warp loads
constexpr int STEP_THREADS = 32 * (STEP_WARPS + 1);
constexpr int STEP_RING = 96 * 1024;  // bytes in flight per CTA; two CTAs share an SM
constexpr long long KV_WAIT_LIMIT = 4000000000LL;         // cycles: about two seconds
constexpr long long KV_DRAIN_LIMIT = 2 * KV_WAIT_LIMIT;  // of a wait for what is in flight when a CTA gives up

// What a call keeps in its workspace. A CTA leaves at most one part of each of its row tiles: of its first segment, when
// that does not begin its (sequence, kv head, rows); ready[part] tells the CTA that waits for it and is zero again when
// the call is done.
struct KvParts {
    uint32_t* ready;
    uint32_t* started;  // CTAs of the running kernel that have begun; the last one makes it zero again
    uint32_t* bad;      // not zero: a wait ran out in a call with this workspace, so that the flags may be anything
    float* o;    // [part]: unnormalised sums
    float2* ml;  // [part][row]: maximum (base 2) and sum
    float* s;    // [sequence][kv head][slot][s_rows]: scaled scores (base 2) of the step path, for the weights
    int64_t s_slots;  // slots that have a score and may be a sequence's
    int s_rows;  // rows rounded up to 4, 8 or 16
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t me;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(me));
    return me;
}
// A 2-d box of a page (box slots x 64 elements of one head) into shared memory. Reached by a whole warp with equal
// arguments, copied once, by the lane whose `me` is nonzero: from lanes with arguments of their own a copy takes over 100
// cycles each (2,048 tokens over 8,192 slots, 32 heads over 8 of 128, pages of 8 slots: 271 us then, 197 when this came, 207
// now).
__device__ __forceinline__ void tma_page(void* dst, const CUtensorMap* map, int d, int slot, int head, int page,
                                         uint64_t* bar, uint32_t me) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %7, 0;\n\t"
        "@q cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n\t"
        "}" ::"r"(smem_u32(dst)),
        "l"(map), "r"(d), "r"(slot), "r"(head), "r"(page), "r"(smem_u32(bar)), "r"(me)
        : "memory");
}
// The table's entries for a tile's boxes, lane i the i-th box's; loaded a tile ahead, since a load does not move over the waits
// and copies in between.
__device__ __forceinline__ int tile_entries(const KvPages& c, const int32_t* table, int first, int boxes, int box_shift,
                                            int len) {
    const int lane = threadIdx.x & 31, slot = first + (lane << box_shift);
    return lane < boxes && slot < len ? kv_entry(c, table, slot) : 0;
}
// The pages of these boxes (a page that does not exist lies past the map: it reads as zero), and the number of boxes that the
// sequence reaches.
struct TilePages {
    int page, count;
};
__device__ __forceinline__ TilePages tile_pages(const KvPages& c, int entry, int first, int boxes, int box_shift, int len) {
    const int lane = threadIdx.x & 31, slot = first + (lane << box_shift);
    const bool live = lane < boxes && slot < len;
    int page = 0;
    if (live) {
        page = (int)kv_page_checked(c, entry);
        if (page < 0) page = (int)c.pages;
    }
    return {page, __popc(__ballot_sync(FULL, live))};
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Bounded waits of one thread or warp: after the first that runs out, the later ones return at once, so that the CTA
// unwinds; what it computes then is void and the status word says so. The workspace is marked too: later calls with it, of
// other caches as well, report that theirs is void until it has been cleared. Called by whole warps, which leave it
// together: what follows is often an instruction that all lanes have to execute as one.
//
// A thread that gave up hands no memory back to be filled again and fills none, so that a barrier has one fill in flight at
// most, which its phase tells. The warp that starts copies or products waits for its last ones before it ends, whatever the
// others do: none outlives the CTA.
struct KvWait {
    int* status;
    uint32_t* bad;
    long long limit;
    bool dead = false;
    __device__ __forceinline__ void ran_out() {
        dead = true;
        atomicOr(status, ERR_WAIT_TIMEOUT);
        *reinterpret_cast<volatile uint32_t*>(bad) = 1u;
    }
    __device__ __forceinline__ void operator()(uint64_t* bar, uint32_t parity) {
        if (!mbar_try_wait(bar, parity) && !dead && !mbar_wait_bounded(bar, parity, limit)) ran_out();
        __syncwarp();
    }
    // The same, and all lanes of the warp give up if one does. For warps that fill memory: they copy with the elected lane's
    // predicate as it is (one computed from it made every copy slower: 8 x 5 tokens over 4,001 slots 20.6 us where this takes
    // 19.1), under a branch of the whole warp.
    __device__ __forceinline__ void together(uint64_t* bar, uint32_t parity) {
        if (__all_sync(FULL, mbar_try_wait(bar, parity)) || dead) return;
        if (!__all_sync(FULL, mbar_wait_bounded(bar, parity, limit))) ran_out();
    }
    // `me` (whether this lane acts for its warp), unless the lane gave up.
    __device__ __forceinline__ uint32_t live(uint32_t me) const { return dead ? 0u : me; }
    // Waits for the last fill of a barrier that has had `fills` of them.
    __device__ __forceinline__ void drain(uint64_t* bar, int fills) const {
        if (fills && !mbar_wait_bounded(bar, (fills - 1) & 1, KV_DRAIN_LIMIT)) atomicOr(status, ERR_DRAIN_TIMEOUT);
    }
};

// A barrier of `threads` threads, whole warps. Their lanes meet first: what comes before is often a loop or a branch that they
// leave one by one, and all lanes of a warp have to execute the barrier as one.
__device__ __forceinline__ void bar_sync(int id, int threads) {
    __syncwarp();
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Part `i` is written (by threads that a barrier has joined since): tell the CTA that adds it up.
__device__ __forceinline__ void part_publish(const KvParts& parts, int i) {
    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(parts.ready + i), "r"(1u) : "memory");
}
// Waits, with a limit, for part i. Its CTA has started, comes to it before anything else and waits for nobody to make it.
__device__ __forceinline__ void part_await(const KvParts& parts, int i, KvWait& wait) {
    uint32_t there = 0;
    const long long t0 = clock64();
    while (!wait.dead) {
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(there) : "l"(parts.ready + i) : "memory");
        if (there) break;
        if (clock64() - t0 > wait.limit) wait.ran_out();
    }
}
__device__ __forceinline__ float part_factor(float m, float top) { return m == -INFINITY ? 0.f : ex2(m - top); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, __half>)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two values rounded to the 16-bit type, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (std::is_same_v<T, __half>) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The share of one CTA: a walk over units laid end to end, sequence by sequence. Count(s) is the number of units of a
// sequence; the caller splits a sequence's units into its heads and tiles. The host has checked that the units of sequences
// whose tokens are the call's, each once, are fewer than 2^31 - 1 together. Offsets that do not ascend can make them more:
// sums stop there, and such a call is reported and does nothing.
struct KvShare {
    int me;    // which share; none from `ctas` on
    int b;     // sequence of the next unit
    int off;   // unit within it
    int left;  // units of this CTA that are not taken yet
    int each;  // units of a CTA; the first `more` of them have one more
    int more;
    int ctas;  // CTAs with a share
    __device__ __forceinline__ int first(int cta) const { return each * cta + min(cta, more); }
    // CTAs that hold the next `rest` units after this CTA's share
    __device__ __forceinline__ int followers(int rest) const {
        const int next = me + 1, end = first(next) + rest;
        int n = 0;
        while (next + n < ctas && first(next + n) < end) ++n;
        return n;
    }
};

constexpr int KV_SHARE_SCRATCH = 40;
// Count(s, &longest) also raises `longest` to the units of the sequence's longest segment. A segment of L units that is cut
// every m units takes m of a unit's time and L / m of a part's: least with m = sqrt(L part / unit), which is the least that
// a CTA gets (part_cost: part / unit), except where all units together are fewer.
template <int THREADS, class Count>
__device__ __forceinline__ KvShare kv_share(const KvPages& c, const KvBatch& bt, const KvParts& parts, int* scratch,
                                            float part_cost, Count&& count) {
    // scratch: KV_SHARE_SCRATCH values of shared memory. Thread t sums a contiguous range of the sequences. No CTA without a
    // share lies between others: the parts of a cut segment belong to consecutive CTAs.
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    constexpr int WARPS = THREADS / 32, PLACE = KV_SHARE_SCRATCH - 1;
    static_assert(2 * WARPS + 2 <= PLACE, "scratch");
    if (t == THREADS - 1) {  // beside the others' loads
        const uint32_t bad = *reinterpret_cast<const volatile uint32_t*>(parts.bad);
        scratch[PLACE] = (int)atomicInc(parts.started, gridDim.x - 1);
        if (bad) atomicOr(c.status, ERR_WORKSPACE);
    }
    const int span = (bt.batch + THREADS - 1) / THREADS;
    const int b0 = min(bt.batch, t * span), b1 = min(bt.batch, b0 + span);
    constexpr uint32_t MOST = 0x7fffffff;
    uint32_t sum = 0;
    int longest = 0;
    for (int b = b0; b < b1; ++b) sum = min(sum + (uint32_t)count(kv_seq(c, bt, b), &longest), MOST);
    longest = __reduce_max_sync(FULL, longest);
    uint32_t incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(FULL, incl, o);
        if (lane >= o) incl = min(incl + x, MOST);
    }
    if (lane == 31) {
        scratch[warp] = (int)incl;
        scratch[WARPS + warp] = longest;
    }
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += (uint32_t)scratch[w];
        all = min(all + (uint32_t)scratch[w], MOST);
        longest = max(longest, scratch[WARPS + w]);
    }
    if (all == MOST && t == 0) atomicOr(c.status, ERR_LAYOUT);
    const int total = all == MOST ? 0 : (int)all;
    const int least = max(1, (int)(sqrtf(longest * part_cost) + 0.5f));
    KvShare s;
    s.ctas = min((int)gridDim.x, (total + least - 1) / least);
    const uint32_t shares = max(s.ctas, 1);
    s.each = (int)((uint32_t)total / shares);
    s.more = total - s.each * (int)shares;
    const int place = scratch[PLACE];
    s.me = place < s.ctas ? s.ctas - 1 - place : s.ctas;
    const int first = s.first(s.me);
    s.left = s.me < s.ctas ? s.first(s.me + 1) - first : 0;
    before += incl - sum;  // exact where there are shares
    if (s.left > 0 && (uint32_t)first >= before && (uint32_t)first < before + sum) {
        int off = first - (int)before, b = b0;
        if (b1 - b0 > 1)
            for (;; ++b) {
                const int n = count(kv_seq(c, bt, b), &longest);
                if (off < n) break;
                off -= n;
            }
        scratch[2 * WARPS] = b;
        scratch[2 * WARPS + 1] = off;
    }
    __syncthreads();
    s.b = scratch[2 * WARPS];
    s.off = scratch[2 * WARPS + 1];
    return s;
}

// Lowest slot that some row does not see: n for every row, or the first row's limit under the causal mask.
__device__ __forceinline__ int row_limit(const KvSeq& s, int causal, int token) {
    return causal ? s.len - s.count + token + 1 : s.len;
}

// The host launches this kernel where the caller's bound says that no sequence has more rows; one that has all the same
// is left out and reported.
__device__ __forceinline__ bool step_takes(const KvSeq& s, int group, int rows) {
    return s.count > 0 && s.count * (int64_t)group <= rows;
}

template <int DP>
constexpr int STEP_STAGE = STEP_TILE * DP * 2 * 2;  // bytes of a tile's keys and values
template <int DP>
constexpr int step_smem() {
    return STEP_RING + STEP_WARPS * 8 * DP * 4 + STEP_WARPS * STEP_ROWS * 8 + 256;
}

// DP: head size padded to 64 or 128 (the boxes' columns past the head read as zero). R: rows rounded up to 8 or 16; of
// m16n8k16's rows the upper eight are not worked on when R is 8.
template <typename T, int DP, int R, bool SCORES>
__global__ void __launch_bounds__(STEP_THREADS, 2)
    kv_step_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, KvPages c,
                   KvBatch bt, KvAttend a, KvParts parts) {
    constexpr int STAGE = STEP_STAGE<DP>, STAGES = STEP_RING / STAGE, HALVES = DP / 64, KS = DP / 16;
    extern __shared__ __align__(1024) uint8_t ring[];  // the swizzle goes by address bits: 1024-byte aligned
    float* sum_o = reinterpret_cast<float*>(ring + STEP_RING);                              // [warp][8][DP]
    float2* sum_ml = reinterpret_cast<float2*>(sum_o + STEP_WARPS * 8 * DP);                // [warp][16]
    uint64_t* full = reinterpret_cast<uint64_t*>(sum_ml + STEP_WARPS * STEP_ROWS);
    uint64_t* empty = full + STAGES;
    int* scratch = reinterpret_cast<int*>(empty + STAGES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        prefetch_map(&map_k);
        prefetch_map(&map_v);
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, STEP_WARPS);
        }
        fence_mbar_init();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    auto tiles_of = [&](const KvSeq& s) { return max(1, (s.len + STEP_TILE - 1) / STEP_TILE); };
    const int most = SCORES ? parts.s_rows : R;  // rows
    auto units_of = [&](const KvSeq& s, int* longest) {
        if (s.count > 0 && !step_takes(s, a.group, most)) atomicOr(c.status, ERR_LAYOUT);
        if (!step_takes(s, a.group, most)) return 0;
        *longest = max(*longest, tiles_of(s));
        return tiles_of(s) * c.heads;
    };
    KvShare share = kv_share<STEP_THREADS>(c, bt, parts, scratch, STEP_PART_COST, units_of);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    KvWait wait{c.status, parts.bad, a.wait_limit};
    int stage = 0;
    uint32_t phase = 0;
    const int box_shift = min(c.page_shift, 6), boxes = STEP_TILE >> box_shift;
    int loaded = 0;
    while (share.left > 0) {
        const KvSeq s = kv_seq(c, bt, share.b);
        const int tiles = tiles_of(s);
        if (!step_takes(s, a.group, most) || share.off >= tiles * c.heads) {
            ++share.b;
            share.off = 0;
            continue;
        }
        const int head = (int)((uint32_t)share.off / (uint32_t)tiles), t0 = share.off - head * tiles;
        const int count = min(tiles - t0, share.left);
        share.off += count;
        share.left -= count;
        const int32_t* table = bt.table + share.b * bt.table_stride;
        if (warp == STEP_WARPS) {
            const uint32_t me = elect_lane();
            int entry = tile_entries(c, table, t0 * STEP_TILE, boxes, box_shift, s.len);
            for (int t = t0; t < t0 + count; ++t) {
                const TilePages tp = tile_pages(c, entry, t * STEP_TILE, boxes, box_shift, s.len);
                if (t + 1 < t0 + count) entry = tile_entries(c, table, (t + 1) * STEP_TILE, boxes, box_shift, s.len);
                wait.together(empty + stage, phase ^ 1);
                if (wait.dead) {
                    share.left = 0;
                    break;
                }
                if (lane == 0) mbar_arrive_expect_tx(full + stage, tp.count * 2 * HALVES * (128 << box_shift));
                __syncwarp();
                uint8_t* dst = ring + stage * STAGE;
                for (int i = 0; i < tp.count; ++i) {
                    const int page = __shfl_sync(FULL, tp.page, i), at = i << box_shift;
                    const int slot = (t * STEP_TILE + at) & ((1 << c.page_shift) - 1);
#pragma unroll
                    for (int part = 0; part < 2 * HALVES; ++part)
                        tma_page(dst + part * (STEP_TILE * 128) + at * 128, part < HALVES ? &map_k : &map_v,
                                 part % HALVES * 64, slot, head, page, full + stage, me);
                }
                ++loaded;
                if (++stage == STAGES) stage = 0, phase ^= 1;
            }
        } else {
            const int g = lane >> 2, q2 = (lane & 3) * 2, rows = s.count * a.group;
            uint32_t q[KS][4];
            int lim[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int r = g + 8 * u;
                const bool live = r < rows && (u == 0 || R == 16);
                lim[u] = live ? row_limit(s, a.causal, r / a.group) : 0;
                const uint16_t* row = a.q + (s.first + (live ? r / a.group : 0)) * a.qs[0] +
                                      (head * a.group + (live ? r % a.group : 0)) * a.qs[1];
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int d = 16 * k + 8 * e + q2;
                        uint32_t x = 0u;
                        if (u == 0 || R == 16) x = __ldca(reinterpret_cast<const unsigned int*>(row + (d < c.dim ? d : 0)));
                        q[k][u + 2 * e] = live && d < c.dim ? x : 0u;
                    }
            }
            const float scale = a.scale * 1.4426950408889634f;
            const int open = min(s.len, row_limit(s, a.causal, 0));  // slots that every row sees
            const int kept = SCORES ? (int)min((int64_t)s.len, parts.s_slots) : 0;
            float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
            for (int t = t0; t < t0 + count; ++t) {
                const int slot0 = t * STEP_TILE + warp * 16;
                wait(full + stage, phase);
                if (slot0 < s.len) {
                    const uint32_t base = smem_u32(ring + stage * STAGE);
                    const bool ends = slot0 + 16 > s.len;
                    if (ends) {  // the page's slots past the sequence hold anything: their values must not meet a zero
                        uint8_t* v = ring + stage * STAGE + HALVES * (STEP_TILE * 128);
                        for (int i = (s.len - slot0) * 8 + lane; i < 16 * 8; i += 32)
#pragma unroll
                            for (int hf = 0; hf < HALVES; ++hf)
                                *reinterpret_cast<uint4*>(v + hf * (STEP_TILE * 128) + warp * 2048 + i * 16) =
                                    make_uint4(0u, 0u, 0u, 0u);
                        __syncwarp();
                    }
                    float x[2][4] = {};
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        // matrices: slots 0-7 and 8-15, each with elements 0-7 and 8-15 of this step's 16
                        const int slot = warp * 16 + (lane & 7) + ((lane >> 4) << 3), ch = (k & 3) * 2 + ((lane >> 3) & 1);
                        uint32_t b[4];
                        ldsm4(base + (k >> 2) * (STEP_TILE * 128) + slot * 128 + ((ch ^ (slot & 7)) << 4), b);
                        mma16<T>(x[0], q[k], b[0], b[1]);
                        mma16<T>(x[1], q[k], b[2], b[3]);
                    }
                    const bool masked = slot0 + 16 > open;
#pragma unroll
                    for (int u = 0; u < (R == 16 ? 2 : 1); ++u) {
                        float top = -INFINITY;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float& y = x[e >> 1][2 * u + (e & 1)];
                            y *= scale;
                            if (masked && slot0 + (e >> 1) * 8 + q2 + (e & 1) >= lim[u]) y = -INFINITY;
                            top = fmaxf(top, y);
                        }
                        if constexpr (SCORES) {
                            const int64_t first = ((int64_t)share.b * c.heads + head) * parts.s_slots + slot0 + q2;
                            float* sp = parts.s + first * parts.s_rows + g + 8 * u;
                            // kept where the sequence and the workspace have the slot
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int j = (e >> 1) * 8 + (e & 1);
                                if (slot0 + q2 + j < kept && g + 8 * u < parts.s_rows)
                                    sp[j * parts.s_rows] = x[e >> 1][2 * u + (e & 1)];
                            }
                        }
                        top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
                        const float next = fmaxf(m[u], top);
                        const float ref = next == -INFINITY ? 0.f : next;
                        if (__any_sync(FULL, next != m[u])) {
                            const float f = ex2(m[u] - ref);
                            l[u] *= f;
#pragma unroll
                            for (int i = 0; i < DP / 8; ++i) {
                                o[i][2 * u] *= f;
                                o[i][2 * u + 1] *= f;
                            }
                            m[u] = next;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float& y = x[e >> 1][2 * u + (e & 1)];
                            y = ex2(y - ref);
                            l[u] += y;
                        }
                    }
                    // the accumulator's layout of the weights is the operand's: 16 rows x 16 slots
                    const uint32_t p[4] = {pack2<T>(x[0][0], x[0][1]), R == 16 ? pack2<T>(x[0][2], x[0][3]) : 0u,
                                           pack2<T>(x[1][0], x[1][1]), R == 16 ? pack2<T>(x[1][2], x[1][3]) : 0u};
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i) {
                        const int slot = warp * 16 + (lane & 15), ch = (i & 3) * 2 + (lane >> 4);
                        uint32_t b[4];
                        ldsm4t(base + (HALVES + (i >> 2)) * (STEP_TILE * 128) + slot * 128 + ((ch ^ (slot & 7)) << 4), b);
                        mma16<T>(o[2 * i], p, b[0], b[1]);
                        mma16<T>(o[2 * i + 1], p, b[2], b[3]);
                    }
                    if (ends) fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0 && !wait.dead) mbar_arrive(empty + stage);
                if (++stage == STAGES) stage = 0, phase ^= 1;
            }
            // Join the four warps, eight rows at a time.
            const bool leaves = t0 > 0;                                             // a part for an earlier CTA
            const int follow = leaves ? 0 : share.followers(tiles - count);  // CTAs with the rest of this one
            for (int i = threadIdx.x; i < follow; i += 32 * STEP_WARPS) part_await(parts, share.me + 1 + i, wait);
#pragma unroll
            for (int u = 0; u < R / 8; ++u) {
                l[u] += __shfl_xor_sync(FULL, l[u], 1);
                l[u] += __shfl_xor_sync(FULL, l[u], 2);
                if ((lane & 3) == 0) sum_ml[warp * STEP_ROWS + 8 * u + g] = make_float2(m[u], l[u]);
            }
            // Thread (row, eight elements), for a head size of 64 the first half of the threads.
            constexpr int U = R / 8;
            const int r8 = threadIdx.x / (DP / 8), d = threadIdx.x % (DP / 8) * 8;
            const bool works = r8 < 8;
            float top[U], total[U] = {}, v[U][8] = {};
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < DP / 8; ++i)
                    *reinterpret_cast<float2*>(sum_o + (warp * 8 + g) * DP + 8 * i + q2) =
                        make_float2(o[i][2 * u], o[i][2 * u + 1]);
                bar_sync(1, 32 * STEP_WARPS);
                top[u] = -INFINITY;
                if (works) {
                    const int r = 8 * u + r8;
#pragma unroll
                    for (int w = 0; w < STEP_WARPS; ++w) top[u] = fmaxf(top[u], sum_ml[w * STEP_ROWS + r].x);
#pragma unroll
                    for (int w = 0; w < STEP_WARPS; ++w) {
                        const float2 ml = sum_ml[w * STEP_ROWS + r];
                        const float f = part_factor(ml.x, top[u]);
                        total[u] += f * ml.y;
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[u][e] += f * sum_o[(w * 8 + r8) * DP + d + e];
                    }
                }
                bar_sync(1, 32 * STEP_WARPS);
            }
            if (works && leaves) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t p = (int64_t)share.me * STEP_ROWS + 8 * u + r8;
                    float4* po = reinterpret_cast<float4*>(parts.o + p * DP + d);
                    po[0] = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
                    po[1] = make_float4(v[u][4], v[u][5], v[u][6], v[u][7]);
                    if (d == 0) parts.ml[p] = make_float2(top[u], total[u]);
                }
            } else if (works) {
                constexpr int FLY = 8 / U;  // parts in flight; the last ones again, for nothing
                for (int k0 = 0; k0 < follow; k0 += FLY) {
                    float2 ml[FLY][U];
                    float4 x[FLY][U], y[FLY][U];
#pragma unroll
                    for (int k = 0; k < FLY; ++k)
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            const int64_t p = (int64_t)(share.me + 1 + min(k0 + k, follow - 1)) * STEP_ROWS + 8 * u + r8;
                            const float4* po = reinterpret_cast<const float4*>(parts.o + p * DP + d);
                            ml[k][u] = __ldcg(parts.ml + p);
                            x[k][u] = __ldcg(po);
                            y[k][u] = __ldcg(po + 1);
                        }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        float next = top[u];
#pragma unroll
                        for (int k = 0; k < FLY; ++k) next = fmaxf(next, ml[k][u].x);
                        const float f = part_factor(top[u], next);
                        total[u] *= f;
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[u][e] *= f;
#pragma unroll
                        for (int k = 0; k < FLY; ++k) {
                            const float h = k0 + k < follow ? part_factor(ml[k][u].x, next) : 0.f;
                            if (h == 0.f) continue;
                            total[u] += ml[k][u].y * h;
                            v[u][0] += x[k][u].x * h, v[u][1] += x[k][u].y * h, v[u][2] += x[k][u].z * h;
                            v[u][3] += x[k][u].w * h, v[u][4] += y[k][u].x * h, v[u][5] += y[k][u].y * h;
                            v[u][6] += y[k][u].z * h, v[u][7] += y[k][u].w * h;
                        }
                        top[u] = next;
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int r = 8 * u + r8;
                    if (r >= rows) continue;
                    const int64_t tok = s.first + r / a.group;
                    const int h = head * a.group + r % a.group;
                    const float inv = total[u] > 0.f ? 1.f / total[u] : total[u] == 0.f ? 0.f : total[u];
                    if (d < c.dim)
                        *reinterpret_cast<uint4*>(a.out + tok * a.os[0] + h * a.os[1] + d) =
                            make_uint4(pack2<T>(v[u][0] * inv, v[u][1] * inv), pack2<T>(v[u][2] * inv, v[u][3] * inv),
                                       pack2<T>(v[u][4] * inv, v[u][5] * inv), pack2<T>(v[u][6] * inv, v[u][7] * inv));
                    if (d == 0) a.lse[tok * a.heads + h] = (top[u] + log2f(total[u])) * 0.6931471805599453f;
                }
            }
            if (leaves || follow) bar_sync(1, 32 * STEP_WARPS);
            if (leaves && threadIdx.x == 0) part_publish(parts, share.me);
            for (int i = threadIdx.x; i < follow; i += 32 * STEP_WARPS) parts.ready[share.me + 1 + i] = 0;
        }
    }
    if (warp == STEP_WARPS && lane == 0)
        for (int i = 0; i < STAGES; ++i) wait.drain(full + i, loaded / STAGES + (i < loaded % STAGES));
}

// Weights that the rows of the step path gave each slot, from the scores that the step kernel left: R of them per slot,
// four slots per thread. Bound by memory, which the step kernel's 4 R bytes per slot and kv head make a twelfth more for
// four rows of 128 elements; keeping them is cheaper than reading the keys again (half of the cache's bytes).
constexpr int STEP_WEIGHTS_SLOTS = 1024;  // of a block
template <int R>
__global__ void __launch_bounds__(256) kv_step_weights_kernel(KvPages c, KvBatch bt, KvAttend a, KvParts parts) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ float s_lse[R];
    const int b = blockIdx.z, head = blockIdx.y;
    const KvSeq s = kv_seq(c, bt, b);
    const int64_t end = min((int64_t)s.len, a.scores_width);
    if (!step_takes(s, a.group, R) || (int64_t)blockIdx.x * STEP_WEIGHTS_SLOTS >= end) return;
    const int rows = s.count * a.group;
    if (threadIdx.x < R) {
        const int r = threadIdx.x;
        float x = INFINITY;  // no row, or one that saw nothing: weight 0
        if (r < rows) {
            const float v = a.lse[(s.first + r / a.group) * a.heads + head * a.group + r % a.group];
            x = v == -INFINITY ? INFINITY : v * 1.4426950408889634f;
        }
        s_lse[r] = x;
    }
    __syncthreads();
    const float4* sp = reinterpret_cast<const float4*>(parts.s + ((int64_t)b * c.heads + head) * parts.s_slots * R);
    float* out = a.scores + b * a.ss[0] + head * a.ss[1];
    for (int64_t j0 = (int64_t)blockIdx.x * STEP_WEIGHTS_SLOTS + threadIdx.x; j0 < end;
         j0 += (int64_t)gridDim.x * STEP_WEIGHTS_SLOTS) {
        float4 x[4][R / 4];
        float before[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t j = min(j0 + u * 256, end - 1);
            before[u] = out[j];
#pragma unroll
            for (int i = 0; i < R / 4; ++i) x[u][i] = __ldca(sp + j * (R / 4) + i);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < R / 4; ++i) {
                // rows that are not there left anything
                if (4 * i < rows) sum += ex2(x[u][i].x - s_lse[4 * i]);
                if (4 * i + 1 < rows) sum += ex2(x[u][i].y - s_lse[4 * i + 1]);
                if (4 * i + 2 < rows) sum += ex2(x[u][i].z - s_lse[4 * i + 2]);
                if (4 * i + 3 < rows) sum += ex2(x[u][i].w - s_lse[4 * i + 3]);
            }
            if (j0 + u * 256 < end) out[j0 + u * 256] = before[u] + sum;
        }
    }
}

}  // namespace vk
