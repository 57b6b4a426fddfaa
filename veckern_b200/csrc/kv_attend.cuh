// Weights that a chunk's rows gave each slot.
#pragma once
#include "kv_chunk.cuh"

namespace vk {

// q . k with lane l holding elements 4l .. 4l + 3 (zero past the head's size).
template <typename T>
__device__ __forceinline__ void load4(const uint16_t* p, int dim, float (&x)[4]) {
    const int lane = threadIdx.x & 31;
    const T* t = reinterpret_cast<const T*>(p);
    for (int i = 0; i < 4; ++i) x[i] = 4 * lane + i < dim ? to_f32(t[4 * lane + i]) : 0.0f;
}

__device__ __forceinline__ float dot4(const float (&a)[4], const float (&b)[4]) {
    float s = a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3];
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(FULL, s, o);
    return s;
}

// One warp per (sequence, kv head, slot): the weights that every row gave it.
template <typename T>
__global__ void __launch_bounds__(256) kv_weights_kernel(KvPages c, KvBatch bt, KvAttend a) {
    const int b = blockIdx.z, kvh = blockIdx.y, j = blockIdx.x * 8 + (threadIdx.x >> 5);
    const KvSeq s = kv_seq(c, bt, b);
    if (j >= s.len || j >= a.scores_width || step_takes(s, a.group)) return;
    const int64_t page = kv_page(c, bt.table + b * bt.table_stride, j);
    if (page < 0) return;
    float k[4], sum = 0.f;
    load4<T>(c.k + page * c.ks[0] + (j & ((1 << c.page_shift) - 1)) * c.ks[1] + kvh * c.ks[2], c.dim, k);
    for (int t = a.causal ? max(0, j - (s.len - s.count)) : 0; t < s.count; ++t)
        for (int g = 0; g < a.group; ++g) {
            const int64_t tok = s.first + t;
            const int h = kvh * a.group + g;
            float q[4];
            load4<T>(a.q + tok * a.qs[0] + h * a.qs[1], c.dim, q);
            sum += expf(dot4(q, k) * a.scale - a.lse[tok * a.heads + h]);
        }
    if ((threadIdx.x & 31) == 0) a.scores[b * a.ss[0] + kvh * a.ss[1] + j] += sum;
}

}  // namespace vk
