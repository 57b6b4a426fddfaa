// C ABI of the paged key/value cache (vk_kv_*): checks of arguments, the cache's handle, and the launches.
#include <atomic>
#include <new>
#include <type_traits>
#include <utility>

#include <cudaTypedefs.h>

#include "kv_move.cuh"
#include "kv_weights.cuh"
#include "status.h"

struct vk_kv {
    vk_kv_desc_t desc{};
    int page_shift = 0;
    int sm_count = 0;
    int* status = nullptr;
    std::atomic<int64_t> wait_limit{vk::KV_WAIT_LIMIT};
    CUtensorMap map_k, map_v;
    ~vk_kv() {
        if (status) cudaFree(status);
    }
};

namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

vk::KvPages pages_of(const vk_kv* kv) {
    vk::KvPages c{};
    c.k = static_cast<uint16_t*>(kv->desc.k);
    c.v = static_cast<uint16_t*>(kv->desc.v);
    for (int i = 0; i < 3; ++i) {
        c.ks[i] = kv->desc.k_stride[i];
        c.vs[i] = kv->desc.v_stride[i];
    }
    c.pages = kv->desc.pages;
    c.page_shift = kv->page_shift;
    c.heads = kv->desc.kv_heads;
    c.dim = kv->desc.head_dim;
    c.status = kv->status;
    return c;
}

// Checks a call's handle and sequences; *out is the kernels' view of them.
int check_batch(const vk_kv* kv, const vk_kv_batch_t* bt, bool offsets, vk::KvBatch* out) {
    if (!kv) return fail(VK_ERR_INVALID, "cache must not be NULL");
    if (!bt) return fail(VK_ERR_INVALID, "batch must not be NULL");
    if (bt->batch < 0 || bt->batch > 65535) return fail(VK_ERR_INVALID, "batch must be in [0, 65535]");
    // the kernels round counts of tokens up to pairs of row tiles in 32 bits
    if (bt->tokens < 0 || bt->tokens > INT32_MAX - 1024) return fail(VK_ERR_INVALID, "tokens must be in [0, 2^31 - 1024)");
    if (bt->table_width < 0 || bt->table_stride < 0 ||
        ((int64_t)bt->table_width << kv->page_shift) > INT32_MAX - 1024)
        return fail(VK_ERR_INVALID, "table_width must be >= 0 and cover less than 2^31 slots");
    if (bt->batch > 0 && ((offsets && !bt->offsets) || !bt->lens || (bt->table_width > 0 && !bt->table)))
        return fail(VK_ERR_INVALID, "offsets, lens and table must not be NULL");
    out->offsets = bt->offsets;
    out->table = bt->table;
    out->lens = bt->lens;
    out->table_stride = bt->table_stride;
    out->tokens = bt->tokens;
    out->batch = bt->batch;
    out->width = bt->table_width;
    return VK_OK;
}

int check_rows(const char* what, const void* p, const int64_t* stride) {
    if (!p) return fail(VK_ERR_INVALID, "%s must not be NULL", what);
    if (!aligned16(p)) return fail(VK_ERR_INVALID, "%s must be 16-byte aligned", what);
    if (!stride || stride[0] < 0 || stride[1] < 0 || stride[0] % 8 || stride[1] % 8)
        return fail(VK_ERR_INVALID, "%s: strides must be multiples of 8 elements", what);
    return VK_OK;
}

// Whether rows of `len` elements at i * s0 + j * s1, i < n0, j < n1, may share elements. (Rows that two strides interleave
// without a common element count as sharing some: nobody lays out results like that.)
bool rows_overlap(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t len) {
    if (n0 <= 1) n0 = n1, s0 = s1, n1 = 1;
    if (n0 <= 1 || len == 0) return false;
    if (n1 <= 1) return s0 < len;
    if (s0 > s1) std::swap(s0, s1), std::swap(n0, n1);
    return s0 < len || s1 < (__int128)s0 * (n0 - 1) + len;
}

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// How a call's attention is laid out: which kernel, its CTAs, and the workspace.
//
// Where every sequence has at most 16 rows (tokens x query heads of a kv head) the step kernel reads the cache at the
// memory's rate on mma.sync; with a longer sequence in the call the chunk kernel takes them all. Its tile of 128 rows is
// mostly empty for a short sequence, but it reads 2 x 128 slots per 3,300 cycles and SM, which is the memory's rate too, so
// that a launch for the short ones of a mixed call would cost more than it saves. Both sides, the same call with the bound
// and without it (32 heads over 8 of 128): 32 sequences of up to 8,192 slots 120 and 132 us, 4 of up to 50,021 102 and 105;
// 8 x 5 tokens over up to 4,001 slots (24 heads over 8 of 64) 17.2 and 24.1. With weights a chunk's products are computed
// twice, where the step kernel keeps them: 141 and 291, 122 and 150, 28 and 50.
struct AttendPlan {
    bool step;
    int rows, s_rows;  // of the step path, rounded up to 8 or 16; to 4, 8 or 16
    int ctas;
    int64_t s_slots;
    size_t ready, started, bad, o, ml, s, bytes;  // offsets
};

AttendPlan plan_attend(const vk_kv* kv, const vk::KvBatch& bt, int group, int max_q, int64_t scores_width) {
    AttendPlan p{};
    const int64_t rows = (int64_t)max_q * group;
    p.step = rows <= vk::STEP_ROWS;
    p.rows = rows <= 8 ? 8 : 16;
    p.s_rows = rows <= 4 ? 4 : p.rows;
    p.ctas = p.step ? 2 * kv->sm_count : kv->sm_count;
    const int dp = kv->desc.head_dim <= 64 ? 64 : 128;
    // of the step path's kept scores: a table may be far wider than its sequences and their scores
    p.s_slots = std::min((int64_t)bt.width << kv->page_shift, scores_width);
    // What has to be zero before a call lies at the start, whatever the sizes.
    const size_t rows_of_parts = (size_t)p.ctas * (p.step ? vk::STEP_ROWS : 2 * vk::CHUNK_ROWS);
    p.started = VK_KV_WORKSPACE_ZEROED - sizeof(uint32_t);
    p.bad = p.started - sizeof(uint32_t);
    p.o = VK_KV_WORKSPACE_ZEROED;
    p.ml = p.o + align256(rows_of_parts * dp * sizeof(float));
    p.s = p.ml + align256(rows_of_parts * sizeof(float2));
    p.bytes = p.s;
    if (p.step) p.bytes += align256((size_t)bt.batch * kv->desc.kv_heads * p.s_slots * p.s_rows * sizeof(float));
    return p;
}

// Once per kernel and device: the dynamic shared memory that it may take, clusters of more than 8.
template <auto* Fn>
int prepare_kernel(int device, size_t smem, bool large_clusters = false) {
    static std::atomic<uint64_t> done{0};  // a bit per device; from the 65th on the calls are made again
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if (done.load(std::memory_order_acquire) & bit) return VK_OK;
    VK_TRY_CUDA(cudaFuncSetAttribute(Fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (large_clusters) VK_TRY_CUDA(cudaFuncSetAttribute(Fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    done.fetch_or(bit, std::memory_order_release);
    return VK_OK;
}

// Launches fn so that it may start while the kernel before it on the stream ends; it waits for that one's results itself.
template <class... Args>
int launch_behind(void (*fn)(Args...), dim3 grid, int threads, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    VK_TRY_CUDA(cudaLaunchKernelEx(&cfg, fn, args...));
    return VK_OK;
}

template <typename T, int DP, int R, bool SCORES>
int launch_step_as(const vk_kv* kv, const vk::KvPages& c, const vk::KvBatch& bt, const vk::KvAttend& a,
                   const vk::KvParts& parts, int ctas, cudaStream_t st) {
    constexpr auto fn = &vk::kv_step_kernel<T, DP, R, SCORES>;
    constexpr int smem = vk::step_smem<DP>();
    VK_TRY(prepare_kernel<fn>(kv->desc.device, smem));
    VK_TRY(launch_behind(fn, dim3(ctas), vk::STEP_THREADS, smem, st, kv->map_k, kv->map_v, c, bt, a, parts));
    if constexpr (SCORES) {
        if (parts.s_slots > 0) {
            const auto weights = parts.s_rows == 4   ? &vk::kv_step_weights_kernel<4>
                                 : parts.s_rows == 8 ? &vk::kv_step_weights_kernel<8>
                                                     : &vk::kv_step_weights_kernel<16>;
            const int64_t blocks = std::min<int64_t>(ceil_div(parts.s_slots, vk::STEP_WEIGHTS_SLOTS), 4096);
            VK_TRY(launch_behind(weights, dim3((unsigned)blocks, c.heads, bt.batch), 256, 0, st, c, bt, a, parts));
        }
    }
    return VK_OK;
}

template <typename T, int DP>
int launch_step(const vk_kv* kv, const vk::KvPages& c, const vk::KvBatch& bt, const vk::KvAttend& a,
                const vk::KvParts& parts, const AttendPlan& p, cudaStream_t st) {
    if (p.rows == 8)
        return a.scores ? launch_step_as<T, DP, 8, true>(kv, c, bt, a, parts, p.ctas, st)
                        : launch_step_as<T, DP, 8, false>(kv, c, bt, a, parts, p.ctas, st);
    return a.scores ? launch_step_as<T, DP, 16, true>(kv, c, bt, a, parts, p.ctas, st)
                    : launch_step_as<T, DP, 16, false>(kv, c, bt, a, parts, p.ctas, st);
}

int encoder(PFN_cuTensorMapEncodeTiled_v12000* out) {
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> known{nullptr};
    PFN_cuTensorMapEncodeTiled_v12000 encode = known.load();
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        VK_TRY_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found));
        if (!fn || found != cudaDriverEntryPointSuccess)
            return fail(VK_ERR_UNSUPPORTED, "the driver has no cuTensorMapEncodeTiled");
        encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
        known.store(encode);
    }
    *out = encode;
    return VK_OK;
}

template <int C>
int launch_select(int device, size_t smem, const vk::KvPages& c, const vk::KvBatch& bt, const vk::KvEvict& e,
                  cudaStream_t st) {
    constexpr auto fn = &vk::kv_select_kernel<C>;
    VK_TRY(prepare_kernel<fn>(device, 5 * vk::SELECT_BINS * sizeof(int) + vk::SELECT_HELD * sizeof(uint32_t), true));
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(C, c.heads, bt.batch);
    cfg.blockDim = dim3(vk::SELECT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    VK_TRY_CUDA(cudaLaunchKernelEx(&cfg, fn, c, bt, e));
    return VK_OK;
}

// The tensor map of the keys' or values' pages: (element, slot, head, page), boxes of 64 elements of up to 64 slots.
int encode_map(const vk_kv_desc_t& d, void* base, const int64_t* stride, CUtensorMap* map) {
    PFN_cuTensorMapEncodeTiled_v12000 encode;
    VK_TRY(encoder(&encode));
    const cuuint64_t dims[4] = {(cuuint64_t)d.head_dim, (cuuint64_t)d.page_size, (cuuint64_t)d.kv_heads,
                                (cuuint64_t)d.pages};
    // a dimension of one entry is never stepped along: any valid stride does
    const cuuint64_t strides[3] = {(cuuint64_t)stride[1] * 2, d.kv_heads > 1 ? (cuuint64_t)stride[2] * 2 : 16,
                                   d.pages > 1 ? (cuuint64_t)stride[0] * 2 : 16};
    const cuuint32_t box[4] = {64, (cuuint32_t)std::min(d.page_size, vk::STEP_TILE), 1, 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, base, dims, strides, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(VK_ERR_INVALID, "the pages' sizes and strides do not make a tensor map (%d)", (int)r);
    return VK_OK;
}

// The tensor map of a chunk's query rows: (element, head, token), boxes of one row tile's tokens and kv head.
int encode_rows(const vk::KvAttend& a, int dim, int64_t tokens, CUtensorMap* map) {
    PFN_cuTensorMapEncodeTiled_v12000 encode;
    VK_TRY(encoder(&encode));
    const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)a.heads, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {a.heads > 1 ? (cuuint64_t)a.qs[1] * 2 : 16, tokens > 1 ? (cuuint64_t)a.qs[0] * 2 : 16};
    const cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(vk::CHUNK_ROWS / a.group)}, step[3] = {1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<uint16_t*>(a.q), dims, strides, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(VK_ERR_INVALID, "q's sizes and strides do not make a tensor map (%d)", (int)r);
    return VK_OK;
}

template <typename T, int DP>
int launch_chunk(const vk_kv* kv, const vk::KvPages& c, const vk::KvBatch& bt, const vk::KvAttend& a,
                 const vk::KvParts& parts, const AttendPlan& p, cudaStream_t st) {
    CUtensorMap map_q;
    VK_TRY(encode_rows(a, c.dim, bt.tokens, &map_q));
    constexpr auto fn = &vk::kv_chunk_kernel<T, DP>;
    constexpr int smem = vk::chunk_smem<DP>();
    VK_TRY(prepare_kernel<fn>(kv->desc.device, smem));
    VK_TRY(launch_behind(fn, dim3(p.ctas), vk::CHUNK_THREADS, smem, st, map_q, kv->map_k, kv->map_v, c, bt, a, parts));
    if (!a.scores || a.scores_width == 0) return VK_OK;
    constexpr auto weights = &vk::kv_weights_kernel<T, DP>;
    constexpr int weights_smem = vk::weights_smem<DP>();
    VK_TRY(prepare_kernel<weights>(kv->desc.device, weights_smem));
    return launch_behind(weights, dim3(p.ctas), vk::WEIGHTS_THREADS, weights_smem, st, map_q, kv->map_k, c, bt, a, parts);
}

template <typename T>
int launch_attend(const vk_kv* kv, const vk::KvBatch& bt, const vk::KvAttend& a, void* workspace, const AttendPlan& p,
                  cudaStream_t st) {
    const vk::KvPages c = pages_of(kv);
    uint8_t* w = static_cast<uint8_t*>(workspace);
    vk::KvParts parts{};
    parts.ready = reinterpret_cast<uint32_t*>(w + p.ready);
    parts.started = reinterpret_cast<uint32_t*>(w + p.started);
    parts.bad = reinterpret_cast<uint32_t*>(w + p.bad);
    parts.o = reinterpret_cast<float*>(w + p.o);
    parts.ml = reinterpret_cast<float2*>(w + p.ml);
    parts.s = reinterpret_cast<float*>(w + p.s);
    parts.s_slots = p.s_slots;
    parts.s_rows = p.s_rows;
    if (p.step)
        return c.dim <= 64 ? launch_step<T, 64>(kv, c, bt, a, parts, p, st) : launch_step<T, 128>(kv, c, bt, a, parts, p, st);
    return c.dim <= 64 ? launch_chunk<T, 64>(kv, c, bt, a, parts, p, st) : launch_chunk<T, 128>(kv, c, bt, a, parts, p, st);
}

// Checks what attention's launches and its workspace's size depend on.
int check_attend(const vk_kv* kv, const vk_kv_attend_t* args) {
    if (!args) return fail(VK_ERR_INVALID, "args must not be NULL");
    const int g = kv->desc.kv_heads;
    if (args->heads < g || args->heads % g || args->heads / g > 128)
        return fail(VK_ERR_INVALID, "heads must be a multiple of kv_heads (%d), at most 128 times it", g);
    if (args->max_q < 0) return fail(VK_ERR_INVALID, "max_q must be >= 0");
    return VK_OK;
}
int max_q_of(const vk_kv_attend_t* args, int64_t tokens) {
    return args->max_q > 0 ? (int)std::min<int64_t>(args->max_q, tokens) : (int)tokens;
}

// While it lives, this thread's calls neither join a capture of a stream nor end one, whatever its mode.
struct BesideCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    BesideCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~BesideCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// A stream of the device that the entries below keep to themselves (made once; making one takes about 300 us).
int own_stream(int device, cudaStream_t* out) {
    static std::atomic<cudaStream_t> known[64]{};
    if (device < 0 || device >= 64) return fail(VK_ERR_UNSUPPORTED, "device %d", device);
    cudaStream_t st = known[device].load(std::memory_order_acquire);
    if (!st) {
        cudaStream_t made = nullptr;
        VK_TRY_CUDA(cudaStreamCreateWithFlags(&made, cudaStreamNonBlocking));
        if (known[device].compare_exchange_strong(st, made)) st = made;
        else cudaStreamDestroy(made);  // another thread was first
    }
    *out = st;
    return VK_OK;
}

// Clears memory that is not in use, and waits for it, without waiting for anybody's work: the default stream, on which
// cudaMemset runs, is not ordered with streams that do not block on it.
int clear_now(int device, void* p, size_t bytes) {
    cudaStream_t st;
    VK_TRY(own_stream(device, &st));
    VK_TRY_CUDA(cudaMemsetAsync(p, 0, bytes, st));
    VK_TRY_CUDA(cudaStreamSynchronize(st));
    return VK_OK;
}

}  // namespace

extern "C" {

int vk_kv_create(const vk_kv_desc_t* d, vk_kv_t** out) {
    if (!d || !out) return fail(VK_ERR_INVALID, "desc and out must not be NULL");
    *out = nullptr;
    if (d->dtype != VK_KV_F16 && d->dtype != VK_KV_BF16)
        return fail(VK_ERR_INVALID, "dtype must be VK_KV_F16 or VK_KV_BF16");
    if (d->page_size < 8 || d->page_size > 1024 || (d->page_size & (d->page_size - 1)))
        return fail(VK_ERR_INVALID, "page_size must be a power of two in [8, 1024]");
    if (d->head_dim < 8 || d->head_dim > 128 || d->head_dim % 8)
        return fail(VK_ERR_INVALID, "head_dim must be a multiple of 8 in [8, 128]");
    if (d->kv_heads < 1 || d->kv_heads > 65535) return fail(VK_ERR_INVALID, "kv_heads must be in [1, 65535]");
    if (d->pages < 1 || d->pages > INT32_MAX) return fail(VK_ERR_INVALID, "pages must be in [1, 2^31)");
    for (int side = 0; side < 2; ++side) {
        const void* p = side ? d->v : d->k;
        const int64_t* s = side ? d->v_stride : d->k_stride;
        const char* what = side ? "v" : "k";
        if (!p || !aligned16(p)) return fail(VK_ERR_INVALID, "%s must be a 16-byte aligned device address", what);
        for (int i = 0; i < 3; ++i)
            if (s[i] < 0 || s[i] % 8 || s[i] >= (int64_t(1) << 38))
                return fail(VK_ERR_INVALID, "%s: strides must be multiples of 8 elements below 2^38", what);
    }
    DeviceGuard guard(d->device);
    if (guard.err != cudaSuccess) return fail(VK_ERR_CUDA, "cudaSetDevice: %s", cudaGetErrorString(guard.err));
    vk_kv* kv = new (std::nothrow) vk_kv;
    if (!kv) return fail(VK_ERR_NOMEM, "out of host memory");
    kv->desc = *d;
    while ((1 << kv->page_shift) < d->page_size) ++kv->page_shift;
    cudaError_t e = cudaDeviceGetAttribute(&kv->sm_count, cudaDevAttrMultiProcessorCount, d->device);
    if (e == cudaSuccess) e = cudaMalloc(&kv->status, sizeof(int));
    if (e != cudaSuccess) {
        delete kv;
        return fail(e == cudaErrorMemoryAllocation ? VK_ERR_NOMEM : VK_ERR_CUDA, "vk_kv_create: %s",
                    cudaGetErrorString(e));
    }
    int r = clear_now(d->device, kv->status, sizeof(int));
    if (r == VK_OK) r = encode_map(*d, d->k, d->k_stride, &kv->map_k);
    if (r == VK_OK) r = encode_map(*d, d->v, d->v_stride, &kv->map_v);
    if (r != VK_OK) {
        delete kv;
        return r;
    }
    *out = kv;
    return VK_OK;
}

int vk_kv_destroy(vk_kv_t* kv) {
    if (!kv) return VK_OK;
    DeviceGuard guard(kv->desc.device);
    delete kv;
    return VK_OK;
}

int vk_kv_sync(vk_kv_t* kv, void* stream) {
    if (!kv) return fail(VK_ERR_INVALID, "cache must not be NULL");
    DeviceGuard guard(kv->desc.device);
    if (guard.err != cudaSuccess) return fail(VK_ERR_CUDA, "cudaSetDevice: %s", cudaGetErrorString(guard.err));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int status = 0;
    VK_TRY_CUDA(cudaMemcpyAsync(&status, kv->status, sizeof(int), cudaMemcpyDeviceToHost, st));
    VK_TRY_CUDA(cudaStreamSynchronize(st));
    if (!status) return VK_OK;
    vk::kv_reported_kernel<<<1, 1, 0, st>>>(kv->status, status);
    VK_TRY_CUDA(cudaGetLastError());
    VK_TRY_CUDA(cudaStreamSynchronize(st));
    if (status & (vk::ERR_WAIT_TIMEOUT | vk::ERR_DRAIN_TIMEOUT))
        return fail(VK_ERR_DEVICE, "a bounded wait ran out in a cache kernel (status %d)", status);
    if (status & vk::ERR_WORKSPACE)
        return fail(VK_ERR_DEVICE, "a call's workspace was not cleared after a bounded wait had run out in another call");
    return fail(VK_ERR_INVALID,
                "a page number, length or offset was out of range: attention read the slots of such a page as zeros, nothing "
                "was written to them, and rows of such offsets may be missing");
}

int vk_kv_wait_limit(vk_kv_t* kv, int64_t cycles) {
    if (!kv) return fail(VK_ERR_INVALID, "cache must not be NULL");
    if (cycles < 0) return fail(VK_ERR_INVALID, "cycles must be >= 0");
    kv->wait_limit.store(cycles ? std::min<int64_t>(cycles, vk::KV_WAIT_LIMIT) : vk::KV_WAIT_LIMIT, std::memory_order_relaxed);
    return VK_OK;
}

int vk_kv_append(vk_kv_t* kv, const vk_kv_batch_t* batch, const void* k, const int64_t* k_stride, const void* v,
                 const int64_t* v_stride, void* stream) {
    vk::KvBatch bt{};
    VK_TRY(check_batch(kv, batch, true, &bt));
    if (bt.tokens == 0 || bt.batch == 0) return VK_OK;
    VK_TRY(check_rows("k", k, k_stride));
    VK_TRY(check_rows("v", v, v_stride));
    DeviceGuard guard(kv->desc.device);
    if (guard.err != cudaSuccess) return fail(VK_ERR_CUDA, "cudaSetDevice: %s", cudaGetErrorString(guard.err));
    const int64_t threads = bt.tokens * kv->desc.kv_heads * (kv->desc.head_dim / 8);
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(threads, 256), (int64_t)kv->sm_count * 32);
    return launch_behind(&vk::kv_append_kernel, dim3(grid), 256, 0, static_cast<cudaStream_t>(stream), pages_of(kv), bt,
                         static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), k_stride[0], k_stride[1],
                         v_stride[0], v_stride[1]);
}

int vk_kv_attend(vk_kv_t* kv, const vk_kv_batch_t* batch, const vk_kv_attend_t* args, void* stream) {
    vk::KvBatch bt{};
    VK_TRY(check_batch(kv, batch, true, &bt));
    VK_TRY(check_attend(kv, args));
    const int g = kv->desc.kv_heads;
    if (!(args->scale == args->scale) || args->scale - args->scale != 0.0f)
        return fail(VK_ERR_INVALID, "scale must be finite");
    if (args->scores && (args->scores_width < 0 || args->scores_stride[0] < 0 || args->scores_stride[1] < 0))
        return fail(VK_ERR_INVALID, "scores: width and strides must be >= 0");
    if (bt.tokens == 0 || bt.batch == 0) return VK_OK;
    VK_TRY(check_rows("q", args->q, args->q_stride));
    VK_TRY(check_rows("out", args->out, args->out_stride));
    if (!args->lse) return fail(VK_ERR_INVALID, "lse must not be NULL");
    if (rows_overlap(bt.tokens, args->out_stride[0], args->heads, args->out_stride[1], kv->desc.head_dim))
        return fail(VK_ERR_INVALID, "out: rows overlap");
    if (args->scores &&
        rows_overlap(bt.batch, args->scores_stride[0], g, args->scores_stride[1], args->scores_width))
        return fail(VK_ERR_INVALID, "scores: rows overlap; each sequence and kv head is added to its own");
    DeviceGuard guard(kv->desc.device);
    if (guard.err != cudaSuccess) return fail(VK_ERR_CUDA, "cudaSetDevice: %s", cudaGetErrorString(guard.err));
    vk::KvAttend a{};
    a.q = static_cast<const uint16_t*>(args->q);
    a.out = static_cast<uint16_t*>(args->out);
    a.lse = args->lse;
    a.scores = args->scores;
    for (int i = 0; i < 2; ++i) {
        a.qs[i] = args->q_stride[i];
        a.os[i] = args->out_stride[i];
        a.ss[i] = args->scores_stride[i];
    }
    a.scores_width = args->scores_width;
    a.heads = args->heads;
    a.group = args->heads / g;
    a.tokens = vk::CHUNK_ROWS / a.group;
    a.by_group = vk::Divisor::of(a.group);
    a.by_tokens = vk::Divisor::of(a.tokens);
    a.by_pair = vk::Divisor::of(2 * a.tokens);
    a.max_q = max_q_of(args, bt.tokens);
    a.causal = args->causal != 0;
    a.scale = args->scale;
    a.wait_limit = kv->wait_limit.load(std::memory_order_relaxed);
    // The kernels count their units of work (tiles and pairs of tiles, of every kv head) in 32 bits.
    const int64_t tiles = ceil_div((int64_t)bt.width << kv->page_shift, vk::STEP_TILE) + 1;
    if (tiles * g * ((double)bt.tokens * a.group / vk::CHUNK_ROWS + 2.0 * bt.batch) >= 2147483647.0)
        return fail(VK_ERR_UNSUPPORTED, "too many tiles (tables of %d pages, %lld tokens); use fewer sequences per call",
                    bt.width, (long long)bt.tokens);
    const AttendPlan plan = plan_attend(kv, bt, a.group, a.max_q, a.scores ? a.scores_width : 0);
    if (args->workspace_bytes < plan.bytes || !args->workspace || reinterpret_cast<uintptr_t>(args->workspace) % 256)
        return fail(VK_ERR_INVALID, "workspace must be 256-byte aligned and hold %zu bytes (vk_kv_attend_workspace)",
                    plan.bytes);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return kv->desc.dtype == VK_KV_F16 ? launch_attend<__half>(kv, bt, a, args->workspace, plan, st)
                                       : launch_attend<__nv_bfloat16>(kv, bt, a, args->workspace, plan, st);
}

int vk_kv_attend_workspace(const vk_kv_t* kv, const vk_kv_batch_t* batch, const vk_kv_attend_t* args, size_t* bytes) {
    vk::KvBatch bt{};
    if (!kv || !batch || !bytes) return fail(VK_ERR_INVALID, "cache, batch and bytes must not be NULL");
    vk_kv_batch_t sizes = *batch;  // pointers are not read
    static const int32_t none = 0;
    sizes.offsets = sizes.table = sizes.lens = &none;
    VK_TRY(check_batch(kv, &sizes, true, &bt));
    VK_TRY(check_attend(kv, args));
    if (args->scores && args->scores_width < 0) return fail(VK_ERR_INVALID, "scores: width must be >= 0");
    *bytes = plan_attend(kv, bt, args->heads / kv->desc.kv_heads, max_q_of(args, bt.tokens),
                         args->scores ? args->scores_width : 0)
                 .bytes;
    return VK_OK;
}

int vk_kv_workspace_create(int device, size_t bytes, void** out) {
    if (!out) return fail(VK_ERR_INVALID, "out must not be NULL");
    *out = nullptr;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return fail(VK_ERR_CUDA, "cudaSetDevice: %s", cudaGetErrorString(guard.err));
    BesideCapture beside;
    void* p = nullptr;
    VK_TRY_CUDA(cudaMalloc(&p, std::max<size_t>(bytes, VK_KV_WORKSPACE_ZEROED)));
    const int r = clear_now(device, p, VK_KV_WORKSPACE_ZEROED);
    if (r != VK_OK) {
        cudaFree(p);
        return r;
    }
    *out = p;
    return VK_OK;
}

int vk_kv_workspace_clear(int device, void* workspace) {
    if (!workspace) return fail(VK_ERR_INVALID, "workspace must not be NULL");
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return fail(VK_ERR_CUDA, "cudaSetDevice: %s", cudaGetErrorString(guard.err));
    BesideCapture beside;
    return clear_now(device, workspace, VK_KV_WORKSPACE_ZEROED);
}

int vk_kv_workspace_destroy(int device, void* workspace) {
    if (!workspace) return VK_OK;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return fail(VK_ERR_CUDA, "cudaSetDevice: %s", cudaGetErrorString(guard.err));
    VK_TRY_CUDA(cudaFree(workspace));
    return VK_OK;
}

int vk_kv_evict(vk_kv_t* kv, const vk_kv_batch_t* batch, const vk_kv_evict_t* args, void* stream) {
    vk::KvBatch bt{};
    VK_TRY(check_batch(kv, batch, false, &bt));
    if (!args) return fail(VK_ERR_INVALID, "args must not be NULL");
    if (args->keep < 0 || args->recent < 0 || args->recent > args->keep)
        return fail(VK_ERR_INVALID, "keep and recent must satisfy 0 <= recent <= keep");
    if (args->new_table_width < 0 || args->new_table_stride < 0 ||
        ((int64_t)args->new_table_width << kv->page_shift) > INT32_MAX - 1024)
        return fail(VK_ERR_INVALID, "new_table_width must be >= 0 and cover less than 2^31 slots");
    if (args->scores_width < 0 || args->scores_stride[0] < 0 || args->scores_stride[1] < 0)
        return fail(VK_ERR_INVALID, "scores: width and strides must be >= 0");
    if (bt.batch == 0) return VK_OK;
    if ((args->scores_width > 0 && (!args->scores || !args->new_scores)) || !args->new_lens ||
        (args->keep > 0 && (!args->kept || (args->new_table_width > 0 && !args->new_table))))
        return fail(VK_ERR_INVALID, "scores, new_scores, kept, new_lens and new_table must not be NULL");
    DeviceGuard guard(kv->desc.device);
    if (guard.err != cudaSuccess) return fail(VK_ERR_CUDA, "cudaSetDevice: %s", cudaGetErrorString(guard.err));
    vk::KvEvict e{};
    e.new_table = args->new_table;
    e.new_stride = args->new_table_stride;
    e.new_width = args->new_table_width;
    e.keep = args->keep;
    e.recent = args->recent;
    e.scores = args->scores;
    e.ss[0] = args->scores_stride[0];
    e.ss[1] = args->scores_stride[1];
    e.width = args->scores_width;
    e.new_scores = args->new_scores;
    e.kept = args->kept;
    e.new_lens = args->new_lens;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const vk::KvPages c = pages_of(kv);
    // CTAs per (sequence, kv head): slices of 2,048 slots or fewer while there are SMs for them; a power of two.
    const int64_t slots = (int64_t)bt.width << c.page_shift, groups = (int64_t)bt.batch * c.heads;
    const int64_t want = ceil_div(slots, 2048);
    int ctas = 1;
    while (ctas < vk::SELECT_CLUSTER && ctas < want && (2 * ctas * groups <= kv->sm_count || slots / ctas > 16384)) ctas *= 2;
    const size_t smem = 5 * vk::SELECT_BINS * sizeof(int) +
                        (size_t)std::min<int64_t>(ceil_div(slots, ctas), vk::SELECT_HELD) * sizeof(uint32_t);
    VK_TRY((ctas == 1   ? launch_select<1>(kv->desc.device, smem, c, bt, e, st)
            : ctas == 2 ? launch_select<2>(kv->desc.device, smem, c, bt, e, st)
            : ctas == 4 ? launch_select<4>(kv->desc.device, smem, c, bt, e, st)
            : ctas == 8 ? launch_select<8>(kv->desc.device, smem, c, bt, e, st)
                        : launch_select<vk::SELECT_CLUSTER>(kv->desc.device, smem, c, bt, e, st)));
    if (e.keep > 0) {
        const int64_t most = std::min<int64_t>(e.keep, slots);  // slots that can be kept
        const unsigned tiles = (unsigned)std::min<int64_t>(ceil_div(most * (c.dim / 8), 256), 4096);
        if (tiles) VK_TRY(launch_behind(&vk::kv_compact_kernel, dim3(tiles, c.heads, bt.batch), 256, 0, st, c, bt, e));
    }
    return VK_OK;
}

}  // extern "C"
