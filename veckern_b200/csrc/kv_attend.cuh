// Attention over the paged cache, one block per (new token, query head).
#pragma once
#include "kv_step.cuh"

namespace vk {

constexpr int ROW_WARPS = 4;

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

// Each warp takes every fourth slot with its own running maximum and sum; the warps are joined at the end.
template <typename T>
__global__ void __launch_bounds__(32 * ROW_WARPS) kv_attend_kernel(KvPages c, KvBatch bt, KvAttend a) {
    __shared__ float s_m[ROW_WARPS], s_l[ROW_WARPS], s_o[ROW_WARPS][128];
    const int64_t tok = blockIdx.x;
    const int h = blockIdx.y, kvh = h / a.group, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = kv_find(bt, tok);
    const KvSeq s = kv_seq(c, bt, b);
    if (tok < s.first || tok >= s.first + s.count || step_takes(s, a.group)) return;
    const int32_t* table = bt.table + b * bt.table_stride;
    const int end = a.causal ? max(0, s.len - s.count + (int)(tok - s.first) + 1) : s.len;
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    load4<T>(a.q + tok * a.qs[0] + h * a.qs[1], c.dim, q);
    const int in = (1 << c.page_shift) - 1;
    for (int j = warp; j < end; j += ROW_WARPS) {
        const int64_t page = kv_page(c, table, j);
        if (page < 0) continue;
        float k[4], v[4];
        load4<T>(c.k + page * c.ks[0] + (j & in) * c.ks[1] + kvh * c.ks[2], c.dim, k);
        load4<T>(c.v + page * c.vs[0] + (j & in) * c.vs[1] + kvh * c.vs[2], c.dim, v);
        const float x = dot4(q, k) * a.scale;
        const float top = fmaxf(m, x), f = expf(m - top), p = expf(x - top);
        for (int i = 0; i < 4; ++i) o[i] = o[i] * f + p * v[i];
        l = l * f + p;
        m = top;
    }
    s_m[warp] = m;
    s_l[warp] = l;
    for (int i = 0; i < 4; ++i) s_o[warp][4 * lane + i] = o[i];
    __syncthreads();
    float top = -INFINITY, total = 0.f;
    for (int w = 0; w < ROW_WARPS; ++w) top = fmaxf(top, s_m[w]);
    for (int w = 0; w < ROW_WARPS; ++w) total += s_l[w] > 0.f ? s_l[w] * expf(s_m[w] - top) : 0.f;
    const int d = threadIdx.x;
    if (d < c.dim) {
        float x = 0.f;
        for (int w = 0; w < ROW_WARPS; ++w) x += s_l[w] > 0.f ? s_o[w][d] * expf(s_m[w] - top) : 0.f;
        reinterpret_cast<T*>(a.out + tok * a.os[0] + h * a.os[1])[d] = from_f32<T>(total > 0.f ? x / total : 0.f);
    }
    if (d == 0) a.lse[tok * a.heads + h] = total > 0.f ? top + logf(total) : -INFINITY;
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
