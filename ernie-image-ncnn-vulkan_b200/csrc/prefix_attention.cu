// Attention of a batch whose sequences share a prefix, over the paged K/V cache.
#include "decode.h"

namespace ernie_b200
{
namespace
{
constexpr int kWarps = 4;

__device__ __forceinline__ float warp_total(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store(float *p, float v) { *p = v; }
__device__ __forceinline__ void store(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// One CTA per slot and query head; its warps take the keys in turn, lanes the dimensions, and each warp
// keeps its running maximum, sum and weighted values, joined at the end.
template <class T, int D> __global__ void __launch_bounds__(kWarps * 32) attend_kernel(PrefixAttentionArgs a)
{
    constexpr int N = D / 32;
    __shared__ float wm[kWarps], wl[kWarps], wo[kWarps][D];
    const int slot = blockIdx.x, head = blockIdx.y, s = slot / a.batch.queries, i = slot - s * a.batch.queries;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const SequenceView view = sequence_view(a.batch, a.kv.page_shift, s);
    if (i >= view.count) return;
    const int own = max(0, view.len - view.count + i + 1), kv_head = head / (a.heads / a.kv.kv_heads);
    const int *own_table = a.batch.tables + static_cast<size_t>(s) * a.batch.max_pages;
    const int *prefix_table = a.batch.max_prefix_pages ? a.batch.prefix_tables + static_cast<size_t>(s / (a.batch.sequences / a.batch.groups)) * a.batch.max_prefix_pages : nullptr;
    const T *q = static_cast<const T *>(a.q) + (static_cast<size_t>(slot) * a.heads + head) * D;
    float x[N], o[N] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) x[n] = to_float(q[lane + 32 * n]) * rsqrtf(static_cast<float>(D));
    for (int key = warp; key < view.prefix_len + own; key += kWarps)
    {
        const bool shared = key < view.prefix_len;
        const int at = shared ? key : key - view.prefix_len;
        const int page = (shared ? prefix_table : own_table)[at >> a.kv.page_shift];
        const bool good = page >= 0 && page < a.kv.pages;
        if (!good) report_range(a.batch.error_flag);
        const size_t row = ((static_cast<size_t>(good ? page : 0) * a.kv.kv_heads + kv_head) << a.kv.page_shift) + (at & ((1 << a.kv.page_shift) - 1));
        const T *k = static_cast<const T *>(a.kv.k) + row * D, *v = static_cast<const T *>(a.kv.v) + row * D;
        float d = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) d = fmaf(x[n], good ? to_float(k[lane + 32 * n]) : 0.f, d);
        d = warp_total(d);
        const float m_new = fmaxf(m, d);
        if (m_new == -INFINITY) continue;
        const float alpha = __expf(m - m_new), p = __expf(d - m_new);
        l = l * alpha + p;
#pragma unroll
        for (int n = 0; n < N; ++n) o[n] = fmaf(p, good ? to_float(v[lane + 32 * n]) : 0.f, o[n] * alpha);
        m = m_new;
    }
    if (lane == 0)
    {
        wm[warp] = m;
        wl[warp] = l;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) wo[warp][lane + 32 * n] = o[n];
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kWarps * 32)
    {
        float top = -INFINITY, sum = 0.f, acc = 0.f;
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, wm[w]);
        for (int w = 0; w < kWarps; ++w)
        {
            if (wm[w] == -INFINITY) continue;
            const float f = __expf(wm[w] - top);
            sum += wl[w] * f;
            acc += wo[w][d] * f;
        }
        store(static_cast<T *>(a.out) + (static_cast<size_t>(slot) * a.heads + head) * D + d, sum > 0.f ? acc / sum : 0.f);
    }
}
} // namespace

size_t prefix_attention_workspace(const PagedLayer &, const PagedBatch &, int, int) { return 16; }
int prepare_prefix_attention_kernels() { return cudaSuccess; }

int launch_prefix_attention(const PrefixAttentionArgs &a, int, cudaStream_t stream)
{
    const dim3 grid(a.batch.sequences * a.batch.queries, a.heads);
    if (a.kv.bf16)
    {
        if (a.kv.dim == 64) attend_kernel<__nv_bfloat16, 64><<<grid, kWarps * 32, 0, stream>>>(a);
        else attend_kernel<__nv_bfloat16, 128><<<grid, kWarps * 32, 0, stream>>>(a);
    }
    else if (a.kv.dim == 64) attend_kernel<float, 64><<<grid, kWarps * 32, 0, stream>>>(a);
    else attend_kernel<float, 128><<<grid, kWarps * 32, 0, stream>>>(a);
    return cudaGetLastError();
}
} // namespace ernie_b200
