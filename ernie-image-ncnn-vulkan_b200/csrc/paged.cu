// The paged K/V cache of batched decoding: new tokens' keys and values rotated into their pages, and the
// cached state of beams rearranged after a selection.
#include "decode.h"

namespace ernie_b200
{
namespace
{
template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// One CTA per slot (a token, or nothing), one thread per pair (d, d + dim/2) of a head.
template <class In, class Out> __global__ void append_kernel(AppendArgs a)
{
    const int slot = blockIdx.x, s = slot / a.batch.queries, i = slot - s * a.batch.queries;
    const SequenceView view = sequence_view(a.batch, a.kv.page_shift, s);
    if (i >= view.count) return;
    const int place = view.len - view.count + i; // in the sequence's own pages
    const long long position = static_cast<long long>(view.prefix_len) + place;
    if (position < 0 || position >= a.rope_rows)
    {
        report_range(a.batch.error_flag);
        return;
    }
    const int dim = a.kv.dim, half = dim / 2;
    int page = -1;
    if (place >= 0)
    {
        page = a.batch.tables[static_cast<size_t>(s) * a.batch.max_pages + (place >> a.kv.page_shift)];
        if (page < 0 || page >= a.kv.pages)
        {
            report_range(a.batch.error_flag);
            page = -1;
        }
    }
    const In *x = static_cast<const In *>(a.qkv) + static_cast<size_t>(slot) * a.ld;
    const float *c = a.cos + position * dim, *sn = a.sin + position * dim;
    const int width = a.heads + 2 * a.kv.kv_heads;
    for (int t = threadIdx.x; t < width * half; t += blockDim.x)
    {
        const int head = t / half, d = t - head * half;
        float lo = to_float(x[head * dim + d]), hi = to_float(x[head * dim + d + half]);
        if (head < a.heads + a.kv.kv_heads)
        {
            const float first = lo, second = hi;
            lo = __fsub_rn(__fmul_rn(first, c[d]), __fmul_rn(second, sn[d]));
            hi = __fadd_rn(__fmul_rn(second, c[d + half]), __fmul_rn(first, sn[d + half]));
        }
        Out *dst;
        if (head < a.heads) dst = static_cast<Out *>(a.q_out) + (static_cast<size_t>(slot) * a.heads + head) * dim;
        else
        {
            if (page < 0) continue;
            const bool key = head < a.heads + a.kv.kv_heads;
            const int kv_head = head - a.heads - (key ? 0 : a.kv.kv_heads);
            const size_t row = ((static_cast<size_t>(page) * a.kv.kv_heads + kv_head) << a.kv.page_shift) +
                               (place & ((1 << a.kv.page_shift) - 1));
            dst = static_cast<Out *>(key ? a.kv.k : a.kv.v) + row * dim;
        }
        dst[d] = from_float<Out>(lo);
        dst[d + half] = from_float<Out>(hi);
    }
}

// What each place of a group takes over, worked out from the parents by one warp (lane = place).
struct GroupMoves
{
    int parent[kMaxBeams]; // -1: none
    int takes[kMaxBeams];  // the old place whose pages the place gets
    int copies[kMaxBeams]; // whether the parent's tokens have to be copied into them
};

__device__ __forceinline__ void group_moves(const int *parents, int beams, int *error_flag, GroupMoves &m)
{
    const unsigned full = 0xffffffffu;
    const int lane = threadIdx.x & 31;
    int p = lane < beams ? parents[lane] : -1;
    if (lane < beams && (p < -1 || p >= beams))
    {
        report_range(error_flag);
        p = -1;
    }
    // lane as a parent: its children, and of them the heir
    unsigned children = 0;
    for (int i = 0; i < beams; ++i)
        if (__shfl_sync(full, p, i) == lane) children |= 1u << i;
    const int heir = !children ? -1 : (children >> lane & 1u) ? lane : __ffs(children) - 1;
    const int parents_heir = __shfl_sync(full, heir, p < 0 ? 0 : p);
    const bool inherits = lane < beams && p >= 0 && parents_heir == lane;
    const unsigned others = __ballot_sync(full, lane < beams && !inherits);
    const unsigned childless = __ballot_sync(full, lane < beams && !children);
    int takes = p;
    if (lane < beams && !inherits)
    {
        const int nth = __popc(others & ((1u << lane) - 1u));
        takes = static_cast<int>(__fns(childless, 0, nth + 1)); // as many childless places as places without inheritance
    }
    if (lane < beams)
    {
        m.parent[lane] = p;
        m.takes[lane] = takes;
        m.copies[lane] = !inherits && p >= 0;
    }
}

// grid (groups, y): the CTAs of a group share its copies; each works out the moves for itself.
__global__ void reorder_kernel(ReorderArgs a, int element_bytes)
{
    __shared__ GroupMoves m;
    const int group = blockIdx.x;
    const size_t base = static_cast<size_t>(group) * a.beams;
    if (threadIdx.x < 32) group_moves(a.parents + base, a.beams, a.error_flag, m);
    __syncthreads();
    const size_t layer_bytes = a.kv.layer_elements() * element_bytes;
    const size_t row_bytes = static_cast<size_t>(a.kv.dim) * element_bytes;
    const size_t head_bytes = row_bytes << a.kv.page_shift;
    const int page_size = 1 << a.kv.page_shift;
    for (int i = 0; i < a.beams; ++i)
    {
        const int p = m.parent[i];
        const int len = p < 0 ? 0 : clamped_length(a.lens[base + p], a.max_pages, a.kv.page_shift, a.error_flag);
        if (blockIdx.y == 0)
        {
            const int *row = a.tables + (base + m.takes[i]) * a.max_pages;
            for (int t = threadIdx.x; t < a.max_pages; t += blockDim.x) a.new_tables[(base + i) * a.max_pages + t] = row[t];
            if (threadIdx.x == 0) a.new_lens[base + i] = len;
        }
        if (!m.copies[i]) continue;
        const int *from = a.tables + (base + p) * a.max_pages, *into = a.tables + (base + m.takes[i]) * a.max_pages;
        const int pages = (len + page_size - 1) >> a.kv.page_shift;
        for (int u = blockIdx.y; u < pages * a.layers; u += gridDim.y)
        {
            const int layer = u / pages, t = u - layer * pages;
            const int source = from[t], target = into[t];
            if (source < 0 || source >= a.kv.pages || target < 0 || target >= a.kv.pages)
            {
                report_range(a.error_flag);
                continue;
            }
            const int tokens = min(page_size, len - (t << a.kv.page_shift));
            const int vectors = static_cast<int>(tokens * row_bytes / 16);
            for (int w = threadIdx.x; w < vectors * a.kv.kv_heads; w += blockDim.x)
            {
                const int head = w / vectors, at = w - head * vectors;
                const size_t src = layer * layer_bytes + (static_cast<size_t>(source) * a.kv.kv_heads + head) * head_bytes + at * 16;
                const size_t dst = layer * layer_bytes + (static_cast<size_t>(target) * a.kv.kv_heads + head) * head_bytes + at * 16;
                *reinterpret_cast<uint4 *>(static_cast<char *>(a.kv.k) + dst) = *reinterpret_cast<const uint4 *>(static_cast<const char *>(a.kv.k) + src);
                *reinterpret_cast<uint4 *>(static_cast<char *>(a.kv.v) + dst) = *reinterpret_cast<const uint4 *>(static_cast<const char *>(a.kv.v) + src);
            }
        }
    }
}
} // namespace

int launch_paged_append(const AppendArgs &a, cudaStream_t stream)
{
    const int slots = a.batch.sequences * a.batch.queries;
    if (a.qkv_bf16)
    {
        if (a.kv.bf16) append_kernel<__nv_bfloat16, __nv_bfloat16><<<slots, 256, 0, stream>>>(a);
        else append_kernel<__nv_bfloat16, float><<<slots, 256, 0, stream>>>(a);
    }
    else if (a.kv.bf16) append_kernel<float, __nv_bfloat16><<<slots, 256, 0, stream>>>(a);
    else append_kernel<float, float><<<slots, 256, 0, stream>>>(a);
    return cudaGetLastError();
}

int launch_beam_reorder(const ReorderArgs &a, int sms, cudaStream_t stream)
{
    const int share = (sms * 4 + a.groups - 1) / a.groups;
    reorder_kernel<<<dim3(a.groups, share), 256, 0, stream>>>(a, a.kv.bf16 ? 2 : 4);
    return cudaGetLastError();
}
} // namespace ernie_b200
