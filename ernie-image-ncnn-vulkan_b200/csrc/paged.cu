// The paged K/V cache of batched decoding: new tokens' keys and values rotated into their pages, and the
// cached state of beams rearranged after a selection.
#include "decode.h"
#include "ptx.cuh"

namespace ernie_b200
{
namespace
{
template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Four or eight consecutive values in FP32.
template <class T, int N> __device__ __forceinline__ void load_values(const T *p, bool vectors, float (&v)[N])
{
    if (!vectors)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_float(p[i]);
    }
    else if constexpr (sizeof(T) == 4)
    {
#pragma unroll
        for (int i = 0; i < N; i += 4)
        {
            const float4 x = __ldcs(reinterpret_cast<const float4 *>(p + i));
            v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
        }
    }
    else
    {
        static_assert(sizeof(T) == 4 || N == 8, "a 16-byte vector");
        const uint4 x = __ldcs(reinterpret_cast<const uint4 *>(p));
        const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
        {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}

template <int N> __device__ __forceinline__ void store_values(float *p, const float (&v)[N])
{
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
template <int N> __device__ __forceinline__ void store_values(__nv_bfloat16 *p, const float (&v)[N])
{
    unsigned w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
    {
        const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const unsigned *>(&x);
    }
    if constexpr (N == 8) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
}

constexpr int kAppendThreads = 256;

// A CTA per slot (a token, or nothing) and share of its heads. A thread holds N dims of a head's lower half
// and their partners in the upper one (16 bytes of the projection each) of every head of its row of threads,
// with one read of their cos and sin; the first heads' loads are issued before the token's place is known.
// The bound is the traffic: projection in, queries, keys and values out.
template <class In, class Out, int D> __global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs a, int vectors)
{
    constexpr int N = sizeof(In) == 2 ? 8 : 4, kHalf = D / 2, kLanes = kHalf / N, kHeads = kAppendThreads / kLanes;
    constexpr int kAhead = 3; // heads of a thread whose loads are in flight together
    grid_dependency_wait();
    grid_dependents_launch();
    const int slot = blockIdx.x, s = slot / a.batch.queries, i = slot - s * a.batch.queries;
    const int d = (threadIdx.x % kLanes) * N, first = blockIdx.y * kHeads + threadIdx.x / kLanes, step = gridDim.y * kHeads;
    const int rotated = a.heads + a.kv.kv_heads, width = rotated + a.kv.kv_heads;
    const In *x = static_cast<const In *>(a.qkv) + static_cast<size_t>(slot) * a.ld + d;
    float lo[kAhead][N], hi[kAhead][N];
    auto fetch = [&](int head) {
#pragma unroll
        for (int t = 0; t < kAhead; ++t)
        {
            if (head + t * step >= width) break;
            load_values<In, N>(x + (head + t * step) * D, vectors, lo[t]);
            load_values<In, N>(x + (head + t * step) * D + kHalf, vectors, hi[t]);
        }
    };
    if (first < width) fetch(first);
    const SequenceView view = sequence_view(a.batch, a.kv.page_shift, s);
    if (i >= view.count) return;
    const int place = view.len - view.count + i; // in the sequence's own pages
    const int position = view.prefix_len + place;
    if (position < 0 || position >= a.rope_rows)
    {
        report_range(a.batch.error_flag);
        return;
    }
    int page = place >= 0 ? a.batch.tables[static_cast<size_t>(s) * a.batch.max_pages + (place >> a.kv.page_shift)] : -1;
    float cos_lo[N], cos_hi[N], sin_lo[N], sin_hi[N];
    const size_t angle = static_cast<size_t>(position) * D + d;
#pragma unroll
    for (int e = 0; e < N; e += 4)
    {
        *reinterpret_cast<float4 *>(cos_lo + e) = *reinterpret_cast<const float4 *>(a.cos + angle + e);
        *reinterpret_cast<float4 *>(cos_hi + e) = *reinterpret_cast<const float4 *>(a.cos + angle + kHalf + e);
        *reinterpret_cast<float4 *>(sin_lo + e) = *reinterpret_cast<const float4 *>(a.sin + angle + e);
        *reinterpret_cast<float4 *>(sin_hi + e) = *reinterpret_cast<const float4 *>(a.sin + angle + kHalf + e);
    }
    if (place >= 0 && (page < 0 || page >= a.kv.pages))
    {
        report_range(a.batch.error_flag);
        page = -1;
    }
    for (int head = first; head < width; head += kAhead * step)
    {
        if (head != first) fetch(head);
#pragma unroll
        for (int t = 0; t < kAhead; ++t)
        {
            const int h = head + t * step;
            if (h >= width) break;
            if (h < rotated)
            {
#pragma unroll
                for (int e = 0; e < N; ++e)
                {
                    const float low = lo[t][e], high = hi[t][e];
                    lo[t][e] = __fsub_rn(__fmul_rn(low, cos_lo[e]), __fmul_rn(high, sin_lo[e]));
                    hi[t][e] = __fadd_rn(__fmul_rn(high, cos_hi[e]), __fmul_rn(low, sin_hi[e]));
                }
            }
            Out *dst;
            if (h < a.heads) dst = static_cast<Out *>(a.q_out) + (static_cast<size_t>(slot) * a.heads + h) * D;
            else
            {
                if (page < 0) continue;
                const int kv_head = h - (h < rotated ? a.heads : rotated);
                const size_t row = ((static_cast<size_t>(page) * a.kv.kv_heads + kv_head) << a.kv.page_shift) +
                                   (place & ((1 << a.kv.page_shift) - 1));
                dst = static_cast<Out *>(h < rotated ? a.kv.k : a.kv.v) + row * D;
            }
            store_values<N>(dst + d, lo[t]);
            store_values<N>(dst + d + kHalf, hi[t]);
        }
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

constexpr int kCopyWarps = 8, kCopyAhead = 8; // 16-byte loads of a lane in flight

// A warp's copy of `vectors` 16-byte vectors of K and V.
__device__ __forceinline__ void copy_rows(const uint4 *k_from, uint4 *k_into, const uint4 *v_from, uint4 *v_into, int vectors, int lane)
{
    for (int at = lane; at < vectors; at += 32 * kCopyAhead / 2)
    {
        uint4 k[kCopyAhead / 2], v[kCopyAhead / 2];
#pragma unroll
        for (int i = 0; i < kCopyAhead / 2; ++i)
            if (at + 32 * i < vectors)
            {
                k[i] = __ldcs(k_from + at + 32 * i);
                v[i] = __ldcs(v_from + at + 32 * i);
            }
#pragma unroll
        for (int i = 0; i < kCopyAhead / 2; ++i)
            if (at + 32 * i < vectors)
            {
                __stcs(k_into + at + 32 * i, k[i]);
                __stcs(v_into + at + 32 * i, v[i]);
            }
    }
}

// grid (groups, y): the warps of a group's CTAs share its copies, a layer's head of a page at a time; each CTA
// works out the moves for itself, the first one writes the new rows. Sources are pages that pass to an heir,
// targets those of childless places, so no page is both and the copies need no order.
__global__ void __launch_bounds__(kCopyWarps * 32) reorder_kernel(const __grid_constant__ ReorderArgs a, int element_shift)
{
    __shared__ GroupMoves m;
    __shared__ int lens[kMaxBeams], first_page[kMaxBeams + 1]; // of the copied places' pages, one after the other
    grid_dependency_wait();
    grid_dependents_launch();
    const int group = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const size_t base = static_cast<size_t>(group) * a.beams;
    const int page_size = 1 << a.kv.page_shift;
    if (warp == 0)
    {
        group_moves(a.parents + base, a.beams, a.error_flag, m);
        __syncwarp();
        int len = 0, pages = 0;
        if (lane < a.beams)
        {
            const int p = m.parent[lane];
            if (p >= 0) len = clamped_length(a.lens[base + p], a.max_pages, a.kv.page_shift, a.error_flag);
            if (m.copies[lane]) pages = (len + page_size - 1) >> a.kv.page_shift;
        }
        lens[lane] = len;
        int scan = pages;
#pragma unroll
        for (int step = 1; step < 32; step *= 2)
        {
            const int other = __shfl_up_sync(0xffffffffu, scan, step);
            if (lane >= step) scan += other;
        }
        first_page[lane + 1] = scan;
        if (lane == 0) first_page[0] = 0;
    }
    __syncthreads();
    if (blockIdx.y == 0)
    {
        for (int t = threadIdx.x; t < a.beams * a.max_pages; t += blockDim.x)
        {
            const int i = t / a.max_pages;
            a.new_tables[base * a.max_pages + t] = a.tables[(base + m.takes[i]) * a.max_pages + t - i * a.max_pages];
        }
        if (threadIdx.x < a.beams) a.new_lens[base + threadIdx.x] = lens[threadIdx.x];
    }
    const int pages = first_page[kMaxBeams], stride = gridDim.y * kCopyWarps;
    const size_t row_vectors = (static_cast<size_t>(a.kv.dim) << element_shift) / 16, head_vectors = row_vectors << a.kv.page_shift;
    const size_t layer_vectors = head_vectors * a.kv.kv_heads * a.kv.pages;
    // a step copies page t of the copies for head h of all the layers' heads
    if (pages == 0) return;
    const int heads = a.kv.kv_heads * a.layers, begin = blockIdx.y * kCopyWarps + warp, more_h = stride / pages, more_t = stride - more_h * pages;
    for (int h = begin / pages, t = begin - h * pages; h < heads; h += more_h + (t + more_t >= pages), t += more_t - (t + more_t >= pages ? pages : 0))
    {
        const int layer = h / a.kv.kv_heads, head = h - layer * a.kv.kv_heads;
        const int i = __popc(__ballot_sync(0xffffffffu, first_page[lane + 1] <= t)); // the place that page belongs to
        const int page = t - first_page[i];
        const int source = a.tables[(base + m.parent[i]) * a.max_pages + page], target = a.tables[(base + m.takes[i]) * a.max_pages + page];
        if (source < 0 || source >= a.kv.pages || target < 0 || target >= a.kv.pages)
        {
            if (lane == 0) report_range(a.error_flag);
            continue;
        }
        const int vectors = min(page_size, lens[i] - (page << a.kv.page_shift)) * static_cast<int>(row_vectors);
        const size_t from = layer * layer_vectors + (static_cast<size_t>(source) * a.kv.kv_heads + head) * head_vectors;
        const size_t into = layer * layer_vectors + (static_cast<size_t>(target) * a.kv.kv_heads + head) * head_vectors;
        copy_rows(static_cast<const uint4 *>(a.kv.k) + from, static_cast<uint4 *>(a.kv.k) + into, static_cast<const uint4 *>(a.kv.v) + from,
                  static_cast<uint4 *>(a.kv.v) + into, vectors, lane);
    }
}

template <class In, class Out> int launch_append(const AppendArgs &a, int sms, cudaStream_t stream)
{
    constexpr int kValues = sizeof(In) == 2 ? 8 : 4;
    const int slots = a.batch.sequences * a.batch.queries, width = a.heads + 2 * a.kv.kv_heads;
    const int at_once = kAppendThreads / (a.kv.dim / 2 / kValues), passes = (width + at_once - 1) / at_once;
    // few slots: their heads over several CTAs (one decode step of five beams: three CTAs a slot)
    const int share = slots >= 2 * sms ? 1 : passes < 64 ? passes : 64;
    const int vectors = reinterpret_cast<uintptr_t>(a.qkv) % 16 == 0 && a.ld % (16 / static_cast<int>(sizeof(In))) == 0;
    const dim3 grid(slots, share);
    if (a.kv.dim == 64) return launch_dependent(append_kernel<In, Out, 64>, grid, kAppendThreads, stream, a, vectors);
    return launch_dependent(append_kernel<In, Out, 128>, grid, kAppendThreads, stream, a, vectors);
}
} // namespace

int launch_paged_append(const AppendArgs &a, int sms, cudaStream_t stream)
{
    if (a.qkv_bf16) return a.kv.bf16 ? launch_append<__nv_bfloat16, __nv_bfloat16>(a, sms, stream) : launch_append<__nv_bfloat16, float>(a, sms, stream);
    return a.kv.bf16 ? launch_append<float, __nv_bfloat16>(a, sms, stream) : launch_append<float, float>(a, sms, stream);
}

int launch_beam_reorder(const ReorderArgs &a, int sms, cudaStream_t stream)
{
    // eight CTAs of eight warps per SM, shared by the groups
    const int share = (sms * 8 + a.groups - 1) / a.groups;
    return launch_dependent(reorder_kernel, dim3(a.groups, share), kCopyWarps * 32, stream, a, a.kv.bf16 ? 1 : 2);
}
} // namespace ernie_b200
