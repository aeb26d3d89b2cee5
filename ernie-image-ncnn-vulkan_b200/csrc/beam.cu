// Beam selection: of each group's beams x vocabulary continuations the best `beams`, by
// score + logit - log sum exp(logits).
//
// The logits are read once. Within a row the order of the totals is the order of the logits, so a CTA that
// owns a stretch of a row needs only the stretch's maximum m, its sum of exp(x - m) and its `beams` largest
// logits; a second kernel joins the stretches of each row (lse = m + log sum s_c exp(m_c - m), in 64 bits)
// and merges the rows' sorted lists. The bound is the logits' traffic: a thread holds 32 logits of a tile and
// has the next tile's loads in flight meanwhile, keeps its own maximum and sum, and the CTA's threads meet
// once per tile to ask whether any logit beats the list, which after the first tile is rare.
#include "decode.h"
#include "ptx.cuh"

namespace ernie_b200
{
namespace
{
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxChunks = 64;   // stretches of a row: two lists per lane of the joining warp
constexpr int kListEntries = 4096; // of a group's lists in the joining CTA's shared memory
constexpr int kCandidates = 512; // of a tile, before the exact ranking
constexpr int kTilesAhead = 4;   // tiles of a stretch where there are plenty

struct Plan
{
    int per_thread; // logits of a tile that a thread holds
    int chunks, tiles_per_chunk;
};

// Large tiles (8192 logits) when they give every SM two CTAs, smaller ones otherwise; with many tiles a CTA
// takes four in a row, so that three of four loads are covered by work.
Plan plan_of(long long rows, int vocab, int beams, int sms)
{
    Plan p;
    const long long span = static_cast<long long>(vocab) + 8; // a row may begin inside a vector
    for (p.per_thread = 32; p.per_thread > 8; p.per_thread /= 2)
        if (rows * ((span + p.per_thread * kThreads - 1) / (p.per_thread * kThreads)) >= 2 * sms) break;
    const long long tile = static_cast<long long>(p.per_thread) * kThreads, tiles = (span + tile - 1) / tile;
    long long most = kListEntries / (beams * beams);
    most = most < kMaxChunks ? most : kMaxChunks;
    p.tiles_per_chunk = static_cast<int>((tiles + most - 1) / most);
    if (p.tiles_per_chunk < kTilesAhead && rows * tiles >= 2ll * sms * 2 * kTilesAhead) p.tiles_per_chunk = kTilesAhead;
    p.chunks = static_cast<int>((tiles + p.tiles_per_chunk - 1) / p.tiles_per_chunk);
    return p;
}

// What a stretch leaves behind: [rows][chunks] of each.
struct Parts
{
    float *top, *sum;  // sum is NaN where the stretch holds a NaN or a +inf
    float *value;      // [beams] logits, descending, equal ones by token; -inf past the last
    int *token;
};

size_t rounded(size_t bytes) { return (bytes + 15) / 16 * 16; }

Parts parts_of(void *workspace, long long rows, int beams, const Plan &p)
{
    const size_t n = static_cast<size_t>(rows) * p.chunks;
    char *at = static_cast<char *>(workspace);
    Parts parts;
    parts.top = reinterpret_cast<float *>(at);
    parts.sum = reinterpret_cast<float *>(at += rounded(n * 4));
    parts.value = reinterpret_cast<float *>(at += rounded(n * 4));
    parts.token = reinterpret_cast<int *>(at += rounded(n * beams * 4));
    return parts;
}

__device__ __forceinline__ bool better(float av, int ai, float bv, int bi) { return av > bv || (av == bv && ai < bi); }

// A row is looked at only if it can offer tokens.
__device__ __forceinline__ bool row_offers(const BeamSelectArgs &a, long long row)
{
    return !a.finished[row] && isfinite(a.scores[row]);
}

template <class T> struct Vector;
template <> struct Vector<float>
{
    static constexpr int kSize = 4;
    static __device__ __forceinline__ void load(const float *p, float *v)
    {
        const float4 x = __ldcs(reinterpret_cast<const float4 *>(p));
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    }
    static __device__ __forceinline__ float one(const float *p) { return *p; }
};
template <> struct Vector<__nv_bfloat16>
{
    static constexpr int kSize = 8;
    static __device__ __forceinline__ void load(const __nv_bfloat16 *p, float *v)
    {
        const uint4 x = __ldcs(reinterpret_cast<const uint4 *>(p));
        const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ float one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
};

// A thread's logits of the tile that starts at `base` (an index of the row, on a 16-byte boundary).
template <class T, int E> __device__ __forceinline__ void load_tile(const T *x, long long base, int vocab, float (&v)[E])
{
    constexpr int V = Vector<T>::kSize;
#pragma unroll
    for (int j = 0; j < E / V; ++j)
    {
        const long long at = base + static_cast<long long>(j * kThreads + threadIdx.x) * V;
        if (at >= 0 && at + V <= vocab) Vector<T>::load(x + at, v + j * V);
        else
#pragma unroll
            for (int e = 0; e < V; ++e) v[j * V + e] = at + e >= 0 && at + e < vocab ? Vector<T>::one(x + at + e) : -INFINITY;
    }
}

template <class T, int E> __global__ void __launch_bounds__(kThreads, 2) stretch_kernel(BeamSelectArgs a, Plan plan, Parts parts)
{
    constexpr int V = Vector<T>::kSize;
    __shared__ float warp_value[kWarps], list_value[kMaxBeams], cand_value[kCandidates];
    __shared__ float warp_sum[kWarps];
    __shared__ int list_token[kMaxBeams], cand_token[kCandidates], found;
    grid_dependency_wait();
    grid_dependents_launch();
    const long long row = blockIdx.x / plan.chunks;
    const int chunk = static_cast<int>(blockIdx.x - row * plan.chunks);
    if (!row_offers(a, row)) return;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, k = a.beams;
    const T *x = static_cast<const T *>(a.logits) + row * a.ld;
    // vectors start at 16-byte boundaries: index 0 of the row is element `shift` of the first one
    const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
    long long base = static_cast<long long>(chunk) * plan.tiles_per_chunk * (E * kThreads) - shift;
    const long long end = min(static_cast<long long>(a.vocab), base + static_cast<long long>(plan.tiles_per_chunk) * (E * kThreads));
    if (tid < kMaxBeams)
    {
        list_value[tid] = -INFINITY;
        list_token[tid] = -1;
    }
    if (tid == 0) found = 0;
    auto token_at = [&](int e) { return static_cast<int>(base + static_cast<long long>((e / V) * kThreads + tid) * V + e % V); };
    float top = -INFINITY, sum = 0.f; // the thread's own
    bool bad = false;
    float bound = -INFINITY; // the list's last entry
    float next[E];
    load_tile<T, E>(x, base, a.vocab, next);
    __syncthreads();
    for (bool first = true; base < end; base += E * kThreads, first = false)
    {
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = next[e];
        if (base + E * kThreads < end) load_tile<T, E>(x, base + E * kThreads, a.vocab, next);
        float mine = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e)
        {
            mine = fmaxf(mine, v[e]);
            bad |= !(v[e] < INFINITY);
        }
        if (mine > top)
        {
            sum *= __expf(top - mine); // 0 while nothing has been seen
            top = mine;
        }
        if (top > -INFINITY)
        {
            float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < E; ++e) s[e & 3] += __expf(v[e] - top);
            sum += (s[0] + s[1]) + (s[2] + s[3]);
        }
        // Later tokens have to beat the list's last one; the first tile finds its own bound: of a warp's lane
        // maxima in descending order the k-th bounds the warp's k-th largest logit from below.
        bool wanted = mine > bound;
        if (first)
        {
            float sorted = mine;
#pragma unroll
            for (int size = 2; size <= 32; size *= 2)
#pragma unroll
                for (int step = size / 2; step > 0; step /= 2)
                {
                    const float other = __shfl_xor_sync(0xffffffffu, sorted, step);
                    const bool high = ((lane & step) == 0) == ((lane & size) == 0);
                    sorted = high ? fmaxf(sorted, other) : fminf(sorted, other);
                }
            sorted = __shfl_sync(0xffffffffu, sorted, k - 1);
            if (lane == 0) warp_value[warp] = sorted;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWarps; ++w) bound = fmaxf(bound, warp_value[w]);
            wanted = mine >= bound && mine > -INFINITY;
        }
        if (!__syncthreads_or(wanted)) continue;
        if (wanted)
        {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if ((first ? v[e] >= bound : v[e] > bound) && v[e] > -INFINITY)
                {
                    const int n = atomicAdd(&found, 1);
                    if (n < kCandidates)
                    {
                        cand_value[n] = v[e];
                        cand_token[n] = token_at(e);
                    }
                }
        }
        if (!first && tid < k && list_value[tid] > -INFINITY)
        {
            const int n = atomicAdd(&found, 1);
            if (n < kCandidates)
            {
                cand_value[n] = list_value[tid];
                cand_token[n] = list_token[tid];
            }
        }
        __syncthreads();
        const int n = found;
        if (n <= kCandidates)
        {
            if (tid < k) list_value[tid] = -INFINITY, list_token[tid] = -1;
            __syncthreads();
            for (int c = tid; c < n; c += kThreads)
            {
                const float cv = cand_value[c];
                const int ci = cand_token[c];
                int rank = 0;
                for (int o = 0; o < n; ++o) rank += better(cand_value[o], cand_token[o], cv, ci);
                if (rank < k)
                {
                    list_value[rank] = cv;
                    list_token[rank] = ci;
                }
            }
        }
        else
        {
            // many equal logits at the bound: the list entry by entry, each the best one after the last
            const float old_value = tid < k ? list_value[tid] : -INFINITY;
            const int old_token = tid < k ? list_token[tid] : -1;
            float last_value = INFINITY;
            int last_token = -1;
            for (int r = 0; r < k; ++r)
            {
                float bv = -INFINITY;
                int bi = INT32_MAX;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (better(last_value, last_token, v[e], token_at(e)) && better(v[e], token_at(e), bv, bi)) bv = v[e], bi = token_at(e);
                if (better(last_value, last_token, old_value, old_token) && better(old_value, old_token, bv, bi) && old_token >= 0)
                    bv = old_value, bi = old_token;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
                {
                    const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
                    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
                    if (better(ov, oi, bv, bi)) bv = ov, bi = oi;
                }
                __syncthreads();
                if (lane == 0)
                {
                    cand_value[warp] = bv;
                    cand_token[warp] = bi;
                }
                __syncthreads();
                for (int w = 0; w < kWarps; ++w)
                    if (better(cand_value[w], cand_token[w], bv, bi)) bv = cand_value[w], bi = cand_token[w];
                last_value = bv;
                last_token = bi;
                if (tid == 0)
                {
                    list_value[r] = bv;
                    list_token[r] = bv > -INFINITY ? bi : -1;
                }
            }
        }
        __syncthreads();
        bound = list_value[k - 1];
        if (tid == 0) found = 0;
    }
    // the threads' maxima and sums
    float most = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) warp_value[warp] = most;
    const bool poisoned = __syncthreads_or(bad);
    most = warp_value[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) most = fmaxf(most, warp_value[w]);
    sum = top > -INFINITY ? sum * __expf(top - most) : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    const size_t out = blockIdx.x;
    if (tid == 0)
    {
        float s = 0.f;
        for (int w = 0; w < kWarps; ++w) s += warp_sum[w];
        parts.top[out] = most;
        parts.sum[out] = poisoned ? NAN : s;
    }
    if (tid < k)
    {
        parts.value[out * k + tid] = list_value[tid];
        parts.token[out * k + tid] = list_token[tid];
    }
}

// FP32 bits in an order of unsigned integers (the two zeros equal).
__device__ __forceinline__ unsigned ordered(float v)
{
    const unsigned u = __float_as_uint(v + 0.f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// One CTA per group, a warp per beam: the beam's list from its stretches' lists, then one warp merges the
// beams' lists (lane = beam).
__global__ void merge_kernel(BeamSelectArgs a, Plan plan, Parts parts)
{
    __shared__ double total[kMaxBeams][kMaxBeams];
    __shared__ int token[kMaxBeams][kMaxBeams], done[kMaxBeams];
    __shared__ float entry_value[kListEntries];
    __shared__ int entry_token[kListEntries];
    const unsigned full = 0xffffffffu;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, k = a.beams;
    const long long base = static_cast<long long>(blockIdx.x) * k, row = base + warp;
    const float score = a.scores[row];
    const bool finished = a.finished[row] != 0, offers = row_offers(a, row);
    grid_dependency_wait();
    grid_dependents_launch();
    if (lane < k) total[warp][lane] = -INFINITY;
    __syncwarp();
    if (lane == 0) done[warp] = finished;
    if (finished)
    {
        if (lane == 0 && isfinite(score))
        {
            total[warp][0] = score;
            token[warp][0] = a.end_token;
        }
    }
    else if (offers)
    {
        // the lists into shared memory, the statistics into registers, all at once
        const int entries = plan.chunks * k;
        float *values = entry_value + warp * entries;
        int *tokens = entry_token + warp * entries;
        for (int e = lane; e < entries; e += 32)
        {
            values[e] = parts.value[row * entries + e];
            tokens[e] = parts.token[row * entries + e];
        }
        float part_top[2], part_sum[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            const int c = lane + 32 * h;
            part_top[h] = c < plan.chunks ? parts.top[row * plan.chunks + c] : -INFINITY;
            part_sum[h] = c < plan.chunks ? parts.sum[row * plan.chunks + c] : 0.f;
        }
        __syncwarp();
        float top = fmaxf(part_top[0], part_top[1]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(full, top, o));
        double sum = 0.0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            if (part_sum[h] != part_sum[h]) sum = NAN;
            else if (part_top[h] > -INFINITY) sum += static_cast<double>(part_sum[h]) * exp(static_cast<double>(part_top[h]) - top);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(full, sum, o);
        const double lse = static_cast<double>(top) + log(sum);
        if (isfinite(lse))
        {
            // lane's lists: stretches lane and lane + 32, each with the place of its next entry
            int at[2] = {0, 0};
            for (int r = 0; r < k; ++r)
            {
                float bv = -INFINITY;
                int bi = INT32_MAX, from = 0;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                {
                    const int c = lane + 32 * h;
                    if (c >= plan.chunks || at[h] >= k) continue;
                    const float v = values[c * k + at[h]];
                    const int i = tokens[c * k + at[h]];
                    if (v > -INFINITY && better(v, i, bv, bi)) bv = v, bi = i, from = h;
                }
                const unsigned key = ordered(bv), most = __reduce_max_sync(full, key);
                const int best = static_cast<int>(__reduce_min_sync(full, key == most ? static_cast<unsigned>(bi) : 0x7fffffffu));
                if (best == INT32_MAX) break;
                if (bi == best) ++at[from];
                const float v = __shfl_sync(full, bv, __ffs(__ballot_sync(full, bi == best)) - 1);
                if (lane == 0)
                {
                    total[warp][r] = static_cast<double>(score) + (static_cast<double>(v) - lse);
                    token[warp][r] = best;
                }
            }
        }
    }
    __syncthreads();
    if (warp != 0) return;
    int at = 0, parent = -1, chosen = -1, ended = 1;
    float value = -INFINITY;
    for (int r = 0; r < k; ++r)
    {
        double best = lane < k && at < k ? total[lane][at] : -INFINITY;
        int who = lane;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
        {
            const double other = __shfl_xor_sync(full, best, o);
            const int other_who = __shfl_xor_sync(full, who, o);
            if (other > best || (other == best && other_who < who)) best = other, who = other_who;
        }
        if (best == -INFINITY) break;
        const int taken = __shfl_sync(full, at, who);
        if (lane == who) ++at;
        if (lane == r)
        {
            parent = who;
            chosen = token[who][taken];
            value = static_cast<float>(best);
            ended = done[who] || (a.end_token >= 0 && chosen == a.end_token);
        }
    }
    if (lane < k)
    {
        a.parents[base + lane] = parent;
        a.tokens[base + lane] = chosen;
        a.new_scores[base + lane] = value;
        a.new_finished[base + lane] = ended;
    }
}

template <class T> cudaError_t launch_stretches(const BeamSelectArgs &a, const Plan &p, const Parts &parts, unsigned ctas, cudaStream_t stream)
{
    if (p.per_thread == 32) return launch_dependent(stretch_kernel<T, 32>, ctas, kThreads, stream, a, p, parts);
    if (p.per_thread == 16) return launch_dependent(stretch_kernel<T, 16>, ctas, kThreads, stream, a, p, parts);
    return launch_dependent(stretch_kernel<T, 8>, ctas, kThreads, stream, a, p, parts);
}
} // namespace

size_t beam_select_workspace(int groups, int beams, int vocab, int sms)
{
    const long long rows = static_cast<long long>(groups) * beams;
    const Plan p = plan_of(rows, vocab, beams, sms);
    const size_t n = static_cast<size_t>(rows) * p.chunks;
    return 2 * rounded(n * 4) + 2 * rounded(n * beams * 4);
}

int launch_beam_select(const BeamSelectArgs &a, int sms, cudaStream_t stream)
{
    const long long rows = static_cast<long long>(a.groups) * a.beams;
    const Plan p = plan_of(rows, a.vocab, a.beams, sms);
    if (rows * p.chunks > INT32_MAX) return cudaErrorInvalidValue;
    const Parts parts = parts_of(a.workspace, rows, a.beams, p);
    const unsigned ctas = static_cast<unsigned>(rows * p.chunks);
    const cudaError_t e = a.bf16 ? launch_stretches<__nv_bfloat16>(a, p, parts, ctas, stream) : launch_stretches<float>(a, p, parts, ctas, stream);
    if (e != cudaSuccess) return e;
    return launch_dependent(merge_kernel, a.groups, 32 * a.beams, stream, a, p, parts);
}
} // namespace ernie_b200
