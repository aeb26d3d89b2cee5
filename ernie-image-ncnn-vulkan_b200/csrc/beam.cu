// Beam selection: of each group's beams x vocabulary continuations the best `beams`, by
// score + logit - log sum exp(logits).
//
// The logits are read once. Within a row the order of the totals is the order of the logits, so whoever owns a
// stretch of a row needs only the sum of its exponentials and its `beams` largest logits. A stretch belongs to
// a warp, which never waits for another one: a lane holds eight 16-byte vectors of a tile and has the next
// tile's in flight meanwhile (the bound is the logits' traffic), keeps its own reference and sum, and the
// warp's list of the best lies sorted across its lanes, one each. Of a tile only what beats the list's last
// entry is looked at one by one, which after a few tiles is rare; so stretches are as long as keeps every warp
// busy. (64 x 8 rows of 131072 logits, 268 MB: 58 us, 4.6 TB/s; 157 us with eight warps on one list that meet
// several times a tile, 78 us with four times as many stretches, 76 to 87 us with warps that read each other's
// lists for a higher bound. 64 rows of random, falling, equal and rising logits: 18, 16, 18 and 35 us.)
// A second kernel joins the stretches of each row and merges the rows' lists.
//
// Sums: a lane's reference is c = x L rounded, for its largest logit x so far and L = log2(e) rounded, and its
// sum that of 2^(x L - c), one FMA and one exponential each. With S and C joined in 64 bits the logarithm of
// the row's sum is (C + log2 S) / L: the roundings of c and, to first order, of L cancel. That needs x L - c to be
// small, which the rounding of c itself exceeds for huge x; so c is kept within +-2^20, where it is off by 2^-4 at
// most. Any c serves as long as nothing over- or underflows, so a lane that holds masked logits only (the type's
// lowest value) adds its zeros to the row's sum as it should; a row whose common reference is at the limit, be it
// masked as a whole or of logits near a million, is summed up again relative to its largest logit.
#include "decode.h"
#include "ptx.cuh"
#include <cfloat>
#include <climits>

namespace ernie_b200
{
namespace
{
constexpr int kVectors = 8;        // 16-byte vectors of a tile that a lane holds
constexpr int kMaxStretches = 64;  // of a row: two lists per lane of the joining warp
constexpr int kListEntries = 4096; // of a group's lists in the joining CTA's shared memory
constexpr int kRing = 3;           // tiles of a warp in shared memory: one in work, two in flight
constexpr int kResident = 16; // warps per SM
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSteady = 1048576.f; // the references' limit

struct Plan
{
    int stretches, tiles; // of a row, of a stretch
};

// Up to kResident warps per SM work at a time; `skew` logits of a row's first vector may lie before the row. A row is
// cut so that the rounds of warps times a stretch's tiles are fewest, a stretch's start counted as six tiles.
Plan plan_of(long long rows, int vocab, int skew, int beams, bool bf16, int sms)
{
    const long long tile = 32 * kVectors * (bf16 ? 8 : 4), tiles = (static_cast<long long>(vocab) + skew + tile - 1) / tile;
    long long most = kListEntries / (beams * beams), best = LLONG_MAX;
    if (most > kMaxStretches) most = kMaxStretches;
    Plan p = {1, 1};
    for (long long s = 1; s <= most && s <= tiles; ++s)
    {
        const long long each = (tiles + s - 1) / s, rounds = (rows * s + kResident * sms - 1) / (kResident * sms), cost = rounds * (each + 6);
        if (cost >= best) continue;
        best = cost;
        p.tiles = static_cast<int>(each);
        p.stretches = static_cast<int>((tiles + each - 1) / each);
    }
    return p;
}

// What a stretch leaves behind: [rows][stretches] of each.
struct Parts
{
    float *reference, *sum; // sum is NaN where the stretch holds a NaN or a +inf
    float *value;      // [beams] logits, descending, equal ones by token; -inf past the last
    int *token;
};

size_t rounded(size_t bytes) { return (bytes + 15) / 16 * 16; }

Parts parts_of(void *workspace, long long rows, int beams, const Plan &p)
{
    const size_t n = static_cast<size_t>(rows) * p.stretches;
    char *at = static_cast<char *>(workspace);
    Parts parts;
    parts.reference = reinterpret_cast<float *>(at);
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

// Sixteen bytes of logits.
template <class T> struct Vector;
template <> struct Vector<float>
{
    static constexpr int kSize = 4;
    static __device__ __forceinline__ float get(const uint4 &x, int i)
    {
        return __uint_as_float(i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w);
    }
    static __device__ __forceinline__ float value(float v) { return v; }
};
template <> struct Vector<__nv_bfloat16>
{
    static constexpr int kSize = 8;
    static __device__ __forceinline__ float get(const uint4 &x, int i)
    {
        const unsigned w = i < 2 ? x.x : i < 4 ? x.y : i < 6 ? x.z : x.w;
        return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    }
    static __device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }
};

// Copies the lane's vectors of the tile that starts at `base` (an index of the row, on a 16-byte boundary) to
// `ring`, where only this lane reads them; -inf outside the row. The copies run on until waited for.
template <class T> __device__ __forceinline__ void fill_tile(const T *x, long long base, int vocab, int lane, uint4 *ring)
{
    constexpr int V = Vector<T>::kSize;
#pragma unroll
    for (int j = 0; j < kVectors; ++j)
    {
        const long long at = base + (j * 32 + lane) * V;
        uint4 *slot = ring + j * 32 + lane;
        if (at >= 0 && at + V <= vocab)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(slot)), "l"(x + at) : "memory");
        else
        {
            unsigned w[4] = {};
#pragma unroll
            for (int e = 0; e < V; ++e)
            {
                const bool inside = at + e >= 0 && at + e < vocab;
                if constexpr (V == 4) w[e] = inside ? __float_as_uint(x[at + e]) : 0xff800000u;
                else w[e / 2] |= (inside ? static_cast<unsigned>(__bfloat16_as_ushort(x[at + e])) : 0xff80u) << (16 * (e & 1));
            }
            *slot = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}
__device__ __forceinline__ void close_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the newest kRing - 2 groups of copies have arrived.
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory"); }

// FP32 bits in an order of unsigned integers (the two zeros equal), and back.
__device__ __forceinline__ unsigned ordered(float v)
{
    const unsigned u = __float_as_uint(v + 0.f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(unsigned u) { return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xffffffffu)); }

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A CTA is one warp, so that the SMs' shares of the stretches differ by one (256 threads: 60.3 for 59.0 us).
template <class T> __global__ void __launch_bounds__(32, kResident) stretch_kernel(const __grid_constant__ BeamSelectArgs a, Plan plan, Parts parts)
{
    constexpr int V = Vector<T>::kSize;
    constexpr unsigned full = 0xffffffffu;
    grid_dependency_wait();
    grid_dependents_launch();
    const int lane = threadIdx.x, k = a.beams;
    const long long out = blockIdx.x, row = out / plan.stretches;
    if (!row_offers(a, row)) return;
    const T *x = static_cast<const T *>(a.logits) + row * a.ld;
    // vectors start at 16-byte boundaries: index 0 of the row is element `skew` of the first one
    const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
    constexpr int kTileSize = 32 * kVectors * V;
    long long base = (out - row * plan.stretches) * plan.tiles * kTileSize - skew;
    const long long end = min(static_cast<long long>(a.vocab), base + static_cast<long long>(plan.tiles) * kTileSize);
    float c = -INFINITY, sum = 0.f, top = -INFINITY; // the lane's reference, sum and largest logit
    float value = -INFINITY, last_value = -INFINITY; // the list: lane i holds the i-th best; its last entry
    int token = INT_MAX;
    bool listed = false; // whether the list has its beginning
    __shared__ uint4 ring[kRing * kVectors * 32];
#pragma unroll
    for (int t = 0; t < kRing - 1; ++t)
    {
        if (base + t * kTileSize < end) fill_tile<T>(x, base + t * kTileSize, a.vocab, lane, ring + t * (kVectors * 32));
        close_copies();
    }
    int slot = 0;
    for (; base < end; base += kTileSize, slot = slot == kRing - 1 ? 0 : slot + 1)
    {
        wait_copies();
        __syncwarp(); // any lane may look at another's logits from here on
        uint4 v[kVectors];
#pragma unroll
        for (int j = 0; j < kVectors; ++j) v[j] = ring[slot * (kVectors * 32) + j * 32 + lane];
        // the tile before this one has left its slot
        const int free = slot == 0 ? kRing - 1 : slot - 1;
        if (base + (kRing - 1) * kTileSize < end) fill_tile<T>(x, base + (kRing - 1) * kTileSize, a.vocab, lane, ring + free * (kVectors * 32));
        close_copies();
        float mine[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
#pragma unroll
            for (int e = 0; e < V; e += 2) mine[(e / 2) & 3] = max3(mine[(e / 2) & 3], Vector<T>::get(v[j], e), Vector<T>::get(v[j], e + 1));
        const float best = fmaxf(max3(mine[0], mine[1], mine[2]), mine[3]);
        if (best > top)
        {
            const float raised = fminf(fmaxf(best * kLog2e, -kSteady), kSteady);
            sum *= exp2_fast(c - raised); // 0 while nothing has been seen
            c = raised;
            top = best;
        }
        if (top > -INFINITY)
        {
            float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) s[e & 3] += exp2_fast(fmaf(Vector<T>::get(v[j], e), kLog2e, -c));
            sum += (s[0] + s[1]) + (s[2] + s[3]);
        }
        else
        {
            // nothing but -inf, or NaN, which the maximum passes over
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (Vector<T>::get(v[j], e) != Vector<T>::get(v[j], e)) sum = NAN;
        }
        // Tokens have to beat the list's last one. The first tile's lanes' largest logits, sorted, are the list's
        // beginning; there, and where more than k lanes have a candidate (logits that rise along the row), the k-th
        // of them bounds the k-th largest of the tile from below.
        float limit = last_value > -INFINITY ? from_ordered(ordered(last_value) + 1) : -FLT_MAX;
        const unsigned hopeful = __ballot_sync(full, best >= limit);
        if (!hopeful) continue;
        int best_place = 0; // of the lane's largest logit, the first of equal ones
#pragma unroll
        for (int j = kVectors - 1; j >= 0; --j)
#pragma unroll
            for (int e = V - 1; e >= 0; --e)
                if (Vector<T>::get(v[j], e) == best) best_place = j * 32 * V + e;
        const int best_token = static_cast<int>(base + lane * V + best_place);
        const bool first = !listed;
        if (first || __popc(hopeful) > k)
        {
            float sorted_value = best;
            int sorted_token = best > -INFINITY ? best_token : INT_MAX;
#pragma unroll
            for (int size = 2; size <= 32; size *= 2)
#pragma unroll
                for (int step = size / 2; step > 0; step /= 2)
                {
                    const float other_value = __shfl_xor_sync(full, sorted_value, step);
                    const int other_token = __shfl_xor_sync(full, sorted_token, step);
                    const bool high = ((lane & step) == 0) == ((lane & size) == 0);
                    if (high == better(other_value, other_token, sorted_value, sorted_token)) sorted_value = other_value, sorted_token = other_token;
                }
            limit = fmaxf(limit, __shfl_sync(full, sorted_value, k - 1));
            if (first)
            {
                listed = true;
                value = sorted_value;
                token = sorted_token;
            }
        }
        int count = 0;
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) count += Vector<T>::get(v[j], e) >= limit;
        auto insert = [&](float new_value, int new_token) {
            // the entries before it are a prefix of the lanes
            const int place = __popc(__ballot_sync(full, better(value, token, new_value, new_token)));
            const float moved_value = __shfl_up_sync(full, value, 1);
            const int moved_token = __shfl_up_sync(full, token, 1);
            if (lane == place) value = new_value, token = new_token;
            else if (lane > place) value = moved_value, token = moved_token;
        };
        if (!first)
            for (unsigned holders = __ballot_sync(full, count == 1); holders; holders &= holders - 1)
            {
                const int from = __ffs(holders) - 1;
                insert(__shfl_sync(full, best, from), __shfl_sync(full, best_token, from));
            }
        // lanes that hold several: the warp looks through such a lane's logits together
        for (unsigned holders = __ballot_sync(full, count > 1); holders; holders &= holders - 1)
        {
            const int from = __ffs(holders) - 1, held = first ? __shfl_sync(full, best_token, from) : -1;
#pragma unroll 1
            for (int i = lane; i < kVectors * V; i += 32)
            {
                const int j = i / V, e = i % V;
                const float x = Vector<T>::value(reinterpret_cast<const T *>(ring + slot * (kVectors * 32) + j * 32 + from)[e]);
                const int x_token = static_cast<int>(base + (j * 32 + from) * V + e);
                const bool beats = better(x, x_token, __shfl_sync(full, value, k - 1), __shfl_sync(full, token, k - 1));
                for (unsigned found = __ballot_sync(full, x >= limit && x_token != held && beats); found; found &= found - 1)
                {
                    const int one = __ffs(found) - 1;
                    const float new_value = __shfl_sync(full, x, one);
                    const int new_token = __shfl_sync(full, x_token, one);
                    if (__any_sync(full, lane == k - 1 && better(new_value, new_token, value, token))) insert(new_value, new_token);
                }
            }
        }
        last_value = __shfl_sync(full, value, k - 1);
    }
    // the lanes' references and sums
    float reference = c;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) reference = fmaxf(reference, __shfl_xor_sync(full, reference, o));
    if (top > -INFINITY) sum *= exp2_fast(c - reference); // (an infinite sum stands at the limit, by a factor of one)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(full, sum, o);
    if (lane == 0)
    {
        parts.reference[out] = reference;
        parts.sum[out] = sum;
    }
    if (lane < k)
    {
        parts.value[out * k + lane] = value;
        parts.token[out * k + lane] = token;
    }
}

// By a warp: the largest logit of the stretches' lists, and the sum of exp(logit - top) over the row.
__device__ __forceinline__ float row_top(const float *values, int stretches, int beams)
{
    float top = -INFINITY;
    for (int c = threadIdx.x % 32; c < stretches; c += 32) top = fmaxf(top, values[c * beams]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    return top;
}
__device__ __noinline__ double row_sum(const BeamSelectArgs &a, long long row, float top)
{
    double sum = 0.0;
#pragma unroll 8
    for (int t = threadIdx.x % 32; t < a.vocab; t += 32)
    {
        const long long at = row * a.ld + t;
        const float x = a.bf16 ? __uint_as_float(static_cast<unsigned>(static_cast<const unsigned short *>(a.logits)[at]) << 16)
                               : static_cast<const float *>(a.logits)[at];
        sum += exp2f((x - top) * kLog2e);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// One CTA per group, a warp per beam: the beam's list from its stretches' lists, then each continuation's place
// among all the beams'.
__global__ void merge_kernel(BeamSelectArgs a, Plan plan, Parts parts)
{
    __shared__ double total[kMaxBeams][kMaxBeams];
    __shared__ int token[kMaxBeams][kMaxBeams], count[kMaxBeams];
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
        const int entries = plan.stretches * k;
        float *values = entry_value + warp * entries;
        int *tokens = entry_token + warp * entries;
        for (int e = lane; e < entries; e += 32)
        {
            values[e] = parts.value[row * entries + e];
            tokens[e] = parts.token[row * entries + e];
        }
        float part_reference[2], part_sum[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            const int c = lane + 32 * h;
            part_reference[h] = c < plan.stretches ? parts.reference[row * plan.stretches + c] : -INFINITY;
            part_sum[h] = c < plan.stretches ? parts.sum[row * plan.stretches + c] : 0.f;
        }
        __syncwarp();
        float reference = fmaxf(part_reference[0], part_reference[1]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) reference = fmaxf(reference, __shfl_xor_sync(full, reference, o));
        double sum = 0.0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            if (part_sum[h] != part_sum[h]) sum = NAN;
            else if (part_reference[h] > -INFINITY) sum += static_cast<double>(part_sum[h]) * exp2f(part_reference[h] - reference);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(full, sum, o);
        // the logarithm of the row's sum is base + log_sum
        double base = 0.0, log_sum = (static_cast<double>(reference) + log2(sum)) / static_cast<double>(kLog2e);
        if (!(fabsf(reference) < kSteady) && sum == sum)
        {
            const float top = row_top(values, plan.stretches, k);
            base = top;
            log_sum = isfinite(top) ? log(row_sum(a, row, top)) : NAN; // only -inf, or a +inf
        }
        if (isfinite(log_sum))
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
                    if (c >= plan.stretches || at[h] >= k) continue;
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
                    total[warp][r] = static_cast<double>(score) + ((static_cast<double>(v) - base) - log_sum);
                    token[warp][r] = best;
                }
            }
        }
    }
    __syncthreads();
    // A continuation's place is the number of better ones: those before it in its beam's list, and of every other beam
    // the first few. Nothing past the last place is followed.
    const double mine = lane < k ? total[warp][lane] : -INFINITY;
    const int offered = __popc(__ballot_sync(full, mine > -INFINITY));
    if (lane == 0) count[warp] = offered;
    if (lane < offered)
    {
        int place = lane;
        for (int b = 0; b < k; ++b)
            for (int j = 0; b != warp && j < k && place < k; ++j, ++place)
            {
                const double other = total[b][j];
                if (!(other > mine || (other == mine && b < warp && other > -INFINITY))) break;
            }
        if (place < k)
        {
            const int chosen = token[warp][lane];
            a.parents[base + place] = warp;
            a.tokens[base + place] = chosen;
            a.new_scores[base + place] = static_cast<float>(mine);
            a.new_finished[base + place] = finished || (a.end_token >= 0 && chosen == a.end_token);
        }
    }
    __syncthreads();
    if (warp != 0) return;
    const int every = __reduce_add_sync(full, lane < k ? count[lane] : 0);
    if (lane < k && lane >= every)
    {
        a.parents[base + lane] = -1;
        a.tokens[base + lane] = -1;
        a.new_scores[base + lane] = -INFINITY;
        a.new_finished[base + lane] = 1;
    }
}

size_t parts_bytes(long long rows, int beams, const Plan &p)
{
    const size_t n = static_cast<size_t>(rows) * p.stretches;
    return 2 * rounded(n * 4) + 2 * rounded(n * beams * 4);
}
} // namespace

size_t beam_select_workspace(int groups, int beams, int vocab, int sms)
{
    // whatever the logits' type and alignment turn out to be
    const long long rows = static_cast<long long>(groups) * beams;
    size_t most = 0;
    for (const bool bf16 : {false, true})
        for (const int skew : {0, bf16 ? 7 : 3})
        {
            const size_t bytes = parts_bytes(rows, beams, plan_of(rows, vocab, skew, beams, bf16, sms));
            if (bytes > most) most = bytes;
        }
    return most;
}

int prepare_beam_kernels()
{
    // the SMs' split between shared memory and L1 stays as it is between the two kernels
    cudaError_t e = cudaFuncSetAttribute(merge_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(stretch_kernel<float>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(stretch_kernel<__nv_bfloat16>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    return e;
}

int launch_beam_select(const BeamSelectArgs &a, int sms, cudaStream_t stream)
{
    const long long rows = static_cast<long long>(a.groups) * a.beams;
    const int vector = a.bf16 ? 8 : 4;
    const bool aligned = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && (rows == 1 || a.ld % vector == 0);
    const Plan p = plan_of(rows, a.vocab, aligned ? 0 : vector - 1, a.beams, a.bf16, sms);
    const long long ctas = rows * p.stretches;
    if (ctas > INT32_MAX) return cudaErrorInvalidValue;
    const Parts parts = parts_of(a.workspace, rows, a.beams, p);
    const unsigned grid = static_cast<unsigned>(ctas);
    const cudaError_t e = a.bf16 ? launch_dependent(stretch_kernel<__nv_bfloat16>, grid, 32, 0, stream, a, p, parts)
                                 : launch_dependent(stretch_kernel<float>, grid, 32, 0, stream, a, p, parts);
    if (e != cudaSuccess) return e;
    return launch_dependent(merge_kernel, a.groups, 32 * a.beams, 0, stream, a, p, parts);
}
} // namespace ernie_b200
