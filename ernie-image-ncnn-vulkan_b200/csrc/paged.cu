// The paged K/V cache of batched decoding: new tokens' keys and values rotated into their pages, and the
// cached state of beams rearranged after a selection.
#include "decode.h"
#include "ptx.cuh"

namespace ernie_b200
{
namespace
{
// Four consecutive values, as they come: 16 bytes of FP32, 8 of BF16.
template <class T> struct Four;
template <> struct Four<float>
{
    float4 x;
    __device__ __forceinline__ void load(const float *p, bool vectors)
    {
        if (vectors) x = __ldcs(reinterpret_cast<const float4 *>(p));
        else x = make_float4(p[0], p[1], p[2], p[3]);
    }
    __device__ __forceinline__ float4 get() const { return x; }
};
template <> struct Four<__nv_bfloat16>
{
    uint2 x;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p, bool vectors)
    {
        const unsigned short *q = reinterpret_cast<const unsigned short *>(p);
        if (vectors) x = __ldcs(reinterpret_cast<const uint2 *>(p));
        else x = make_uint2(q[0] | static_cast<unsigned>(q[1]) << 16, q[2] | static_cast<unsigned>(q[3]) << 16);
    }
    __device__ __forceinline__ float4 get() const
    {
        return make_float4(__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xffff0000u));
    }
};

__device__ __forceinline__ void store_four(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void store_four(__nv_bfloat16 *p, float4 v)
{
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
}

// x c - y s and y c + x s without contraction
__device__ __forceinline__ float4 turn_low(float4 x, float4 y, float4 c, float4 s)
{
    return make_float4(__fsub_rn(__fmul_rn(x.x, c.x), __fmul_rn(y.x, s.x)), __fsub_rn(__fmul_rn(x.y, c.y), __fmul_rn(y.y, s.y)),
                       __fsub_rn(__fmul_rn(x.z, c.z), __fmul_rn(y.z, s.z)), __fsub_rn(__fmul_rn(x.w, c.w), __fmul_rn(y.w, s.w)));
}
__device__ __forceinline__ float4 turn_high(float4 x, float4 y, float4 c, float4 s)
{
    return make_float4(__fadd_rn(__fmul_rn(y.x, c.x), __fmul_rn(x.x, s.x)), __fadd_rn(__fmul_rn(y.y, c.y), __fmul_rn(x.y, s.y)),
                       __fadd_rn(__fmul_rn(y.z, c.z), __fmul_rn(x.z, s.z)), __fadd_rn(__fmul_rn(y.w, c.w), __fmul_rn(x.w, s.w)));
}

constexpr int kAppendThreads = 128;
constexpr int kAppendAhead = 6; // heads of a thread whose loads are in flight together
template <class In> constexpr int kAppendCtas = sizeof(In) == 2 ? 8 : 5; // of an SM

// A CTA per slot (a token, or nothing) and share of its heads. A thread holds four dims of a head's lower half
// and their partners in the upper one, of every head of its row of threads, with one read of their cos and sin;
// the first heads' loads are issued before the token's place is known. The bound is the traffic: projection in,
// queries, keys and values out. A slot is a chain of some 3 us (lengths, page and angles, stores) around 24 KB,
// so an SM needs many slots at a time: small CTAs with six heads to a thread. (16000 tokens of 48 heads from
// BF16 to BF16, 410 MB: 80 to 84 us, 4.9 to 5.1 TB/s; 140 us with eight dims to a thread at 114 registers, 94 us with 256
// threads and three heads each, 96 us with these walking over the slots and the next one's loads in flight.)
template <class In, class Out, int D>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas<In>) append_kernel(const __grid_constant__ AppendArgs a, int vectors)
{
    constexpr int kHalf = D / 2, kLanes = kHalf / 4, kHeads = kAppendThreads / kLanes;
    grid_dependency_wait();
    grid_dependents_launch();
    const int slot = blockIdx.x, s = slot / a.batch.queries, i = slot - s * a.batch.queries;
    const int d = (threadIdx.x % kLanes) * 4, first = blockIdx.y * kHeads + threadIdx.x / kLanes, step = gridDim.y * kHeads;
    const int rotated = a.heads + a.kv.kv_heads, width = rotated + a.kv.kv_heads;
    const In *x = static_cast<const In *>(a.qkv) + static_cast<size_t>(slot) * a.ld + d;
    Four<In> lo[kAppendAhead], hi[kAppendAhead];
    auto fetch = [&](int head) {
#pragma unroll
        for (int t = 0; t < kAppendAhead; ++t)
            if (head + t * step < width)
            {
                lo[t].load(x + (head + t * step) * D, vectors);
                hi[t].load(x + (head + t * step) * D + kHalf, vectors);
            }
    };
    fetch(first);
    const int len = a.batch.lens[s];
    const SequenceView view = sequence_view(a.batch, a.kv.page_shift, s);
    if (i >= view.count) return;
    // in the sequence's own pages; a length past the table counts as it is here, so that no new token takes an old one's place
    const int place = max(len, view.len) - view.count + i;
    const bool held = place >= 0 && place < static_cast<long long>(a.batch.max_pages) << a.kv.page_shift;
    const long long position = static_cast<long long>(view.prefix_len) + place;
    if (position < 0 || position >= a.rope_rows)
    {
        report_range(a.batch.error_flag);
        return;
    }
    int page = held ? a.batch.tables[static_cast<size_t>(s) * a.batch.max_pages + (place >> a.kv.page_shift)] : -1;
    const float *cos = a.cos + static_cast<size_t>(position) * D + d, *sin = a.sin + static_cast<size_t>(position) * D + d;
    const float4 cos_lo = *reinterpret_cast<const float4 *>(cos), cos_hi = *reinterpret_cast<const float4 *>(cos + kHalf);
    const float4 sin_lo = *reinterpret_cast<const float4 *>(sin), sin_hi = *reinterpret_cast<const float4 *>(sin + kHalf);
    if (held && (page < 0 || page >= a.kv.pages))
    {
        report_range(a.batch.error_flag);
        page = -1;
    }
    for (int head = first; head < width; head += kAppendAhead * step)
    {
        if (head != first) fetch(head);
#pragma unroll
        for (int t = 0; t < kAppendAhead; ++t)
        {
            const int h = head + t * step;
            if (h >= width) break;
            const float4 low = lo[t].get(), high = hi[t].get();
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
            store_four(dst + d, h < rotated ? turn_low(low, high, cos_lo, sin_lo) : low);
            store_four(dst + d + kHalf, h < rotated ? turn_high(low, high, cos_hi, sin_hi) : high);
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
// targets those of childless places, so no page is both and the copies need no order. The bound is the traffic: the
// copies of 12 groups of 4 beams over 26 layers, 479 MB read and written, take 79 to 83 us, 5.8 to 6.1 TB/s.
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
    const int slots = a.batch.sequences * a.batch.queries, width = a.heads + 2 * a.kv.kv_heads;
    const int at_once = kAppendThreads / (a.kv.dim / 8), passes = (width + at_once - 1) / at_once;
    // few slots: their heads over several CTAs (48 heads of 128: six). 100 slots 5.0 us, whole ones 5.2; 300 slots
    // 5.2 and 5.1; 600 slots 8.5 and 5.2
    const int share = slots >= 2 * sms ? 1 : passes < 64 ? passes : 64;
    const int vectors = reinterpret_cast<uintptr_t>(a.qkv) % (4 * sizeof(In)) == 0 && a.ld % 4 == 0;
    const dim3 grid(slots, share);
    if (a.kv.dim == 64) return launch_dependent(append_kernel<In, Out, 64>, grid, kAppendThreads, 0, stream, a, vectors);
    return launch_dependent(append_kernel<In, Out, 128>, grid, kAppendThreads, 0, stream, a, vectors);
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
    return launch_dependent(reorder_kernel, dim3(a.groups, share), kCopyWarps * 32, 0, stream, a, a.kv.bf16 ? 1 : 2);
}
} // namespace ernie_b200
