// Attention of a batch whose sequences share prefixes, over the paged K/V cache:
//   out = softmax(q k^T / sqrt(D)) v over [the group's prefix | the sequence's own tokens up to the row's place].
//
// The softmax over both stretches is joined from partial results: a stretch of keys leaves, per row, its
// maximum m, l = sum 2^(s - m) and o = sum 2^(s - m) v (scores s in units of log2), and the join weighs them by
// 2^(m - max m). Two lists of items are worked on at the same time by one grid, one CTA per SM:
//   prefix  (group, block of rows, K/V head): every row of the group against the group's prefix, which is
//           read once per block of rows however many sequences share it;
//   own     (sequence, block of rows, K/V head): a sequence's rows against its own tokens.
// A row is a query head of a slot: the heads/kv_heads query heads that share a K/V head are rows of one item.
// An item's keys are cut into units, and each list's units are dealt out evenly, in order, to that list's
// workers (a fixed cost of every item counted in), so that an item may span several workers and a worker
// several items; an item's share of a worker is a part. Along the order both the item and the worker only ever
// step up, so item + worker numbers the parts without gaps or clashes, and an item's parts lie side by side. The
// lists share the CTAs by their estimated cost. All of this is worked out on the device, by every CTA for itself,
// from the lengths of this very call.
//
// Where a ragged batch's group has more slots than one block holds, the rows of its prefix items are those of its
// tokens instead of its slots, found through the sums of the sequences' counts: 64 sequences of which one brings
// 32 new tokens and the others one each go over the prefix with 95 tokens, not with 2048 slots.
//
// A list is worked on in one of two ways, chosen on the host by the rows of an item:
//   stream  few rows, or an FP32 cache. A worker is a warp: 16 rows and its own TMA ring of K/V slots. The
//           bound is the K/V traffic, and eight independent warps per SM hide each other's latencies without
//           ever meeting (an SM streams 60 to 65 GB/s of a BF16 cache, 100 of them the memory's 6.3 TB/s). BF16
//           uses mma.sync m16n8 tiles, FP32 packed FMAs (three products of TF32 parts on the tensor cores took
//           2.4 times as long and lost two bits).
//   tile    many rows of a BF16 cache. A worker is a CTA: 256 rows (two tiles of 128) share each K/V tile on
//           the tensor cores (tcgen05.mma, accumulators in TMEM), one row per softmax thread. A unit of 256
//           rows and 128 keys takes about 3350 cycles. Shared memory's 128 bytes per cycle bound it: four
//           products that read 64 KB each, 64 KB of weights stored, 64 KB of keys and values loaded, 3070
//           cycles (the exponentials alone would take 2048).
// 256 sequences of 1024 own tokens behind 16384 shared ones (32 query heads over 8, BF16) take 147 to 170 us (power),
// 64 of 512 behind 4096 30, 12 groups of 8 with 300 behind 1800 in FP32 103.
// A second kernel joins the parts of each row.
#include "attend_layout.h"
#include "decode.h"
#include "ptx.cuh"
#include <cudaTypedefs.h>

namespace ernie_b200
{
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

namespace
{
constexpr int kThreads = 384; // three warpgroups: control, and twice four working warps
constexpr int kWorkers = 8;   // streaming warps of a CTA
constexpr int kTile = 128;    // rows and keys of a tile
static_assert(kTile == kWeightRows, "weights' tile");
// 128 x 72 + 256 x 216 registers are the launch's 384 x 168 (with 88 and 208 the tiles' unit loop spills: 16 sequences of
// 16 to 32 rows behind 2000 tokens 44.7 us for 42.3, 256 behind 16384 165 for 158).
constexpr int kRegsControl = 72, kRegsWork = 216, kMinLaunchRegs = 168;
static_assert(128 * kRegsControl + 256 * kRegsWork <= kThreads * kMinLaunchRegs, "register split");

// Division of numbers below 2^31 by a divisor that the host knows, n / d = (hi32(n m) + n) >> shift: Granlund and
// Montgomery, "Division by invariant integers using multiplication", 1994.
struct Divisor
{
    unsigned m, shift;
};
Divisor divisor(unsigned d)
{
    Divisor r = {0, 0};
    while ((1ull << r.shift) < d) ++r.shift;
    r.m = static_cast<unsigned>(((1ull << 32) * ((1ull << r.shift) - d)) / d + 1);
    return r;
}
__device__ __forceinline__ int divide(int n, Divisor d) { return static_cast<int>((__umulhi(n, d.m) + n) >> d.shift); }

// One of the two lists, as the host lays it out.
struct List
{
    int owners;     // groups or sequences
    int rows;       // of an owner and K/V head
    int slots;      // of an owner
    int block;      // rows of an item, and its log2
    int block_shift;
    int blocks;     // items of an owner and K/V head
    int part_rows;  // rows that a part stores
    int tile;       // 1: on the tensor cores' tiles, 0: streamed
    int unit_shift; // log2 of a unit's keys
    int lead;       // an item's fixed cost, in units
    int cost;       // of a unit on an SM, relative
    int workers;    // that the list may be dealt out to
    float *o;       // [items + workers][part_rows][D]
    float2 *ml;     // [items + workers][part_rows]
    int2 *meta;     // [items]: the workers of the first and the last part
};

struct AttendArgs
{
    PrefixAttentionArgs a;
    List list[2]; // prefix, own
    int ctas;
    int share;    // query heads of a K/V head
    Divisor by_share, by_queries, by_heads, by_group; // query heads of a K/V head, slots of a sequence, query heads, slots of a group
    float scale;  // log2(e) / sqrt(D)
    int granule;  // keys of a TMA box
    int per;      // sequences of a group
    int *earlier; // [sequences + 1]: tokens of the sequences before one
};
// kTokens: the prefix items' rows are those of the tokens, otherwise those of the slots.
template <bool kTokens> struct Args : AttendArgs
{
};

template <class T, int D> struct Layout
{
    static constexpr int kSlotKeys = sizeof(T) == 2 ? 16 : 8;                      // one step of a streaming warp
    static constexpr int kColumns = D * static_cast<int>(sizeof(T)) / 128;         // 128-byte column blocks of a row
    static constexpr int kSlotBytes = kSlotKeys * D * static_cast<int>(sizeof(T)); // a slot: a step's K or its V
    static constexpr int kRing = D == 128 ? 7 : 11;                                // slots of a warp
    static constexpr int kStreamBytes = kWorkers * kRing * kSlotBytes;
    static constexpr int kTileBytes = kTile * D * 2;       // a Q, K or V tile
    static constexpr int kWeightBytes = kTile * kTile * 2; // a P tile
    static constexpr int kTileModeBytes = 5 * kTileBytes + 2 * kWeightBytes;
    static constexpr int kBody = kStreamBytes > kTileModeBytes ? kStreamBytes : kTileModeBytes;
    static constexpr int kSmemBytes = kBody + 1024 + 2048; // alignment; barriers and the plan
};

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The same, kept in its place among waits and arrivals.
__device__ __forceinline__ float exp2_here(float x)
{
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ float4 ld_shared_v4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ void ldmatrix(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void ldmatrix_trans(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Whether the phase with the given parity has completed, without waiting (try_wait may suspend the thread).
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity)
{
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return done != 0;
}

// Loads of own tokens, which nobody else reads, leave L2 first, so that a prefix stays for its other blocks of rows
// (256 sequences behind 16384 tokens, two thirds of the traffic own tokens: 837 MB read of 609 MB, 161 us; with the
// hint 156).
__device__ __forceinline__ uint64_t cache_policy(int which)
{
    uint64_t policy;
    if (which == 0) asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
    else asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ void tma_load_2d_hint(uint32_t smem_dst, const CUtensorMap *map, uint32_t bar, int x, int y, uint64_t policy)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(smem_dst),
                 "l"(map), "r"(bar), "r"(x), "r"(y), "l"(policy)
                 : "memory");
}

// A whole warp's bounded wait, with one answer for all its lanes.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

// ---------------------------------------------------------------- the plan
struct Keys
{
    int keys; // that the rows of an item see at most
    int rows; // of a group and K/V head, if they are its tokens'
    OwnView own;
};

template <bool X> __device__ __forceinline__ Keys item_keys(const Args<X> &p, int which, int owner, int block)
{
    const PagedBatch &b = p.a.batch;
    Keys k = {0, 0, {0, 0}};
    if (which == 0)
    {
        if constexpr (X) k.rows = (p.earlier[(owner + 1) * p.per] - p.earlier[owner * p.per]) * p.share;
        k.keys = clamped_length(b.prefix_lens[owner], b.max_prefix_pages, p.a.kv.page_shift, b.error_flag);
        if constexpr (X)
            if (block << p.list[0].block_shift >= k.rows) k.keys = 0;
        return k;
    }
    k.own = own_view(b, p.a.kv.page_shift, owner);
    const int first = block << p.list[1].block_shift, rows = min(first + p.list[1].block, k.own.count * p.share);
    if (rows > first) k.keys = max(0, k.own.len - k.own.count + divide(rows - 1, p.by_share) + 1);
    return k;
}

template <bool X> __device__ __forceinline__ int rows_of(const Args<X> &p, int which, const Keys &item)
{
    return X && which == 0 ? item.rows : p.list[which].rows;
}

__device__ __forceinline__ int units_of(const List &l, int keys)
{
    return (keys >> l.unit_shift) + ((keys & ((1 << l.unit_shift) - 1)) != 0);
}

// An item takes so many steps of the order: its fixed cost first, during which nothing is computed, so that
// many short items weigh what they take, then its units.
__device__ __forceinline__ int steps_of(const List &l, int keys)
{
    const int units = units_of(l, keys);
    return units ? units + l.lead : 0;
}

// The CTA's list (-1: nothing to do) and how it is dealt out: `each` steps to a worker, one more to the first
// `more` of them.
struct Plan
{
    int which, cta, ctas, workers, each, more;
    __device__ int first_step(int worker) const { return worker * each + min(worker, more); }
};

// Where a worker begins: so many steps after the first one of the owners that a thread has summed up.
struct PlanShared
{
    int warp_sum[2][kThreads / 32];
    int2 begin[kWorkers]; // that thread's first owner, steps
};

// A worker's walk over its steps.
struct Walk
{
    int worker, at, end;          // next step and the worker's end
    int owner, block, head, step; // the next step's item and its number within the item
};

struct Part
{
    int owner, block, head;
    Keys item;
    int first_unit, units; // of the part
    bool last;             // the item's last part
    int place;             // of its results
};

// The next part of the walk; false at its end. All threads of a worker take the same steps.
template <bool X> __device__ __forceinline__ bool next_part(const Args<X> &p, int which, Walk &w, Part &part)
{
    const List &l = p.list[which];
    while (w.at < w.end && w.owner < l.owners) // (the owners run out first only if the lengths change under the call)
    {
        part.item = item_keys(p, which, w.owner, w.block);
        const int steps = steps_of(l, part.item.keys);
        if (w.step >= steps) // nothing here
        {
            w.step = 0;
            w.head = 0;
            if (++w.block == l.blocks) w.block = 0, ++w.owner;
            continue;
        }
        const int end = min(steps, w.step + (w.end - w.at));
        part.owner = w.owner;
        part.block = w.block;
        part.head = w.head;
        part.first_unit = max(0, w.step - l.lead);
        part.units = max(0, end - l.lead) - part.first_unit;
        part.last = end == steps;
        part.place = (w.owner * l.blocks + w.block) * p.a.kv.kv_heads + w.head + w.worker;
        w.at += end - w.step;
        w.step = end;
        if (part.last)
        {
            w.step = 0;
            if (++w.head == p.a.kv.kv_heads)
            {
                w.head = 0;
                if (++w.block == l.blocks) w.block = 0, ++w.owner;
            }
        }
        if (part.units) return true;
    }
    return false;
}

__device__ __forceinline__ void write_meta(const List &l, const Walk &w, const Part &part)
{
    int *meta = reinterpret_cast<int *>(l.meta + (part.place - w.worker));
    if (part.first_unit == 0) meta[0] = w.worker;
    if (part.last) meta[1] = w.worker;
}

// The walk of worker `local` of the CTA (tile: 0, the CTA itself).
template <bool X> __device__ __forceinline__ Walk walk_of(const Args<X> &p, const Plan &plan, const PlanShared &s, int local)
{
    const List &l = p.list[plan.which];
    Walk w = {local * plan.ctas + plan.cta, 0, 0, 0, 0, 0, 0}; // neighbours in the order go to different SMs
    if (w.worker >= plan.workers) return w;
    w.at = plan.first_step(w.worker);
    w.end = plan.first_step(w.worker + 1);
    const int2 begin = s.begin[local];
    w.owner = begin.x;
    int left = begin.y;
    while (w.owner < l.owners)
    {
        const int steps = steps_of(l, item_keys(p, plan.which, w.owner, w.block).keys);
        if (left < steps * p.a.kv.kv_heads)
        {
            for (; left >= steps; left -= steps) ++w.head;
            w.step = left;
            break;
        }
        left -= steps * p.a.kv.kv_heads;
        if (++w.block == l.blocks) w.block = 0, ++w.owner;
    }
    return w;
}

__device__ __forceinline__ int scan_warp(int x)
{
#pragma unroll
    for (int step = 1; step < 32; step *= 2)
    {
        const int other = __shfl_up_sync(0xffffffffu, x, step);
        if (threadIdx.x % 32 >= step) x += other;
    }
    return x;
}

// All threads: sums up to and including the thread's own.
__device__ __forceinline__ int scan_block(int x, int *warp_sum)
{
    const int warp = threadIdx.x / 32;
    int scan = scan_warp(x);
    if (threadIdx.x % 32 == 31) warp_sum[warp] = scan;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kThreads / 32; ++j)
        if (j < warp) scan += warp_sum[j];
    return scan;
}

// All threads: the lists' steps, dealt out.
template <bool X> __device__ __forceinline__ Plan make_plan(const Args<X> &p, PlanShared &s)
{
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, heads = p.a.kv.kv_heads;
    int mine[2], before[2], chunk[2];
#pragma unroll
    for (int n = 0; n < 2; ++n)
    {
        const int i = X ? 1 - n : n;
        const List &l = p.list[i];
        chunk[i] = l.owners <= kThreads ? 1 : (l.owners + kThreads - 1) / kThreads;
        const int first = tid * chunk[i], end = min(l.owners, first + chunk[i]);
        int sum = 0, tokens = 0;
        for (int o = first; o < end; ++o)
        {
            for (int b = 0; b < l.blocks; ++b) sum += steps_of(l, item_keys(p, i, o, b).keys);
            if (X && i == 1) tokens += own_view(p.a.batch, p.a.kv.page_shift, o).count;
        }
        mine[i] = sum * heads;
        if (X && i == 1)
        {
            // every CTA writes the same sums, and reads its own
            int at = scan_block(tokens, s.warp_sum[0]) - tokens;
            for (int o = first; o < end; ++o)
            {
                p.earlier[o] = at;
                at += own_view(p.a.batch, p.a.kv.page_shift, o).count;
                if (o == l.owners - 1) p.earlier[l.owners] = at;
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
    {
        const int scan = scan_warp(mine[i]);
        before[i] = scan - mine[i];
        if (lane == 31) s.warp_sum[i][warp] = scan;
    }
    __syncthreads();
    int total[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < kThreads / 32; ++j)
        {
            const int sum = s.warp_sum[i][j];
            if (j < warp) before[i] += sum;
            total[i] += sum;
        }
    Plan plan = {-1, 0, 0, 0, 0, 0};
    if (total[0] + total[1] == 0) return plan;
    // the lists' CTAs: by cost, at least one for a list with work, no more than it has steps
    const float cost0 = static_cast<float>(total[0]) * p.list[0].cost, cost1 = static_cast<float>(total[1]) * p.list[1].cost;
    int n0 = static_cast<int>(p.ctas * __fdividef(cost0, cost0 + cost1) + 0.5f);
    n0 = total[0] == 0 ? 0 : total[1] == 0 ? p.ctas : max(1, min(p.ctas - 1, n0));
    if (n0 > total[0]) n0 = total[0];
    const int n1 = min(total[1], p.ctas - n0);
    if (n0 + n1 < p.ctas) n0 = min(total[0], p.ctas - n1);
    const int cta = blockIdx.x;
    if (cta >= n0 + n1) return plan;
    plan.which = cta < n0 ? 0 : 1;
    plan.cta = plan.which ? cta - n0 : cta;
    plan.ctas = plan.which ? n1 : n0;
    const List &l = p.list[plan.which];
    const int steps = plan.which ? total[1] : total[0];
    plan.workers = l.tile ? plan.ctas : min(steps, plan.ctas * kWorkers);
    plan.each = steps / plan.workers;
    plan.more = steps - plan.each * plan.workers;
    const int ahead = plan.which ? before[1] : before[0], held = plan.which ? mine[1] : mine[0];
    const int owner = tid * (plan.which ? chunk[1] : chunk[0]);
#pragma unroll
    for (int local = 0; local < kWorkers; ++local)
    {
        const int worker = local * plan.ctas + plan.cta, left = plan.first_step(worker) - ahead;
        if (worker < plan.workers && left >= 0 && left < held) s.begin[local] = make_int2(owner, left);
    }
    __syncthreads();
    return plan;
}

// ---------------------------------------------------------------- rows
struct Row
{
    int query; // row of q and out
    int keys;  // that the row sees of the item's; 0 without a token
};

template <bool X> __device__ __forceinline__ Row row_of(const Args<X> &p, int which, const Part &part, int row)
{
    const PagedBatch &b = p.a.batch;
    const List &l = p.list[which];
    const int r = (part.block << l.block_shift) + row;
    Row out = {0, 0};
    if (row >= l.block || r >= rows_of(p, which, part.item)) return out;
    const int at = divide(r, p.by_share), head = part.head * p.share + r - at * p.share;
    int slot = part.owner * l.slots + at;
    if (X && which == 0)
    {
        // the last sequence with no more than `token` tokens before it holds that one
        int s = part.owner * p.per, more = p.per;
        const int token = p.earlier[s] + at;
        while (more > 1)
        {
            const int half = more >> 1;
            if (p.earlier[s + half] <= token) s += half, more -= half;
            else more = half;
        }
        slot = s * b.queries + token - p.earlier[s];
        out.keys = part.item.keys;
    }
    else if (which == 0)
    {
        const int s = divide(slot, p.by_queries);
        if (b.counts && slot - s * b.queries >= b.counts[s]) return out;
        out.keys = part.item.keys;
    }
    else
    {
        if (at >= part.item.own.count) return out;
        out.keys = max(0, part.item.own.len - part.item.own.count + at + 1);
    }
    out.query = slot * p.a.heads + head;
    return out;
}

// First row of the pool that holds key `key` of the part's item, or the row past the end (TMA reads zeros
// there) for a key past the item's or a bad page, which `bad` remembers: nothing here waits for the table.
template <bool X> __device__ __forceinline__ int pool_row(const Args<X> &p, int which, const Part &part, int key, bool &bad)
{
    const PagedLayer &kv = p.a.kv;
    const int outside = (kv.pages * kv.kv_heads) << kv.page_shift;
    if (key >= part.item.keys) return outside;
    const PagedBatch &b = p.a.batch;
    const int *table = which == 0 ? b.prefix_tables + static_cast<size_t>(part.owner) * b.max_prefix_pages
                                  : b.tables + static_cast<size_t>(part.owner) * b.max_pages;
    const int page = table[key >> kv.page_shift];
    const bool good = static_cast<unsigned>(page) < static_cast<unsigned>(kv.pages);
    bad |= !good;
    const int row = ((page * kv.kv_heads + part.head) << kv.page_shift) + (key & ((1 << kv.page_shift) - 1));
    return good ? row : outside;
}

// ---------------------------------------------------------------- stream
// A slot holds K or V of kSlotKeys keys, 128-byte rows in swizzled column blocks. A warp's ring takes K and V of
// a step in turn, so that K's slot is free again once the scores are done.

// BF16: a warp's 16 rows in mma.sync fragments: rows lane/4 and lane/4 + 8; a lane's columns are
// 2 (lane % 4) and the next of every eight.
template <int D> struct Rows16
{
    static constexpr int kKeys = 16, kTiles = 2; // of a step; score tiles of eight keys
    uint32_t q[D / 16][4];
    __device__ __forceinline__ void load(const AttendArgs &p, const Row &r0, const Row &r1, int lane)
    {
        const __nv_bfloat16 *base = static_cast<const __nv_bfloat16 *>(p.a.q) + 2 * (lane & 3);
        const __nv_bfloat16 *x0 = base + static_cast<size_t>(r0.query) * D, *x1 = base + static_cast<size_t>(r1.query) * D;
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
        {
            q[s][0] = r0.keys ? *reinterpret_cast<const uint32_t *>(x0 + 16 * s) : 0u;
            q[s][1] = r1.keys ? *reinterpret_cast<const uint32_t *>(x1 + 16 * s) : 0u;
            q[s][2] = r0.keys ? *reinterpret_cast<const uint32_t *>(x0 + 16 * s + 8) : 0u;
            q[s][3] = r1.keys ? *reinterpret_cast<const uint32_t *>(x1 + 16 * s + 8) : 0u;
        }
    }
    // two chains per score tile, so that a step waits for half as many products in a row
    __device__ __forceinline__ void scores(uint32_t k, int lane, float (&s)[kTiles][4]) const
    {
        const int key = (lane >> 4) * 8 + (lane & 7), half = (lane >> 3) & 1;
        float odd[kTiles][4] = {};
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
        {
            uint32_t b[4];
            const int chunk = 2 * i + half;
            ldmatrix(k + (chunk >> 3) * (kKeys * 128) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4), b);
            mma_bf16((i & 1 ? odd : s)[0], q[i], b[0], b[1]);
            mma_bf16((i & 1 ? odd : s)[1], q[i], b[2], b[3]);
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[t][j] += odd[t][j];
    }
    // o += p v, of the step's keys the first `valid`
    __device__ __forceinline__ void weigh(uint32_t v, int lane, const float (&s)[kTiles][4], int valid, float (&o)[D / 8][4]) const
    {
        const uint32_t a[4] = {pack2(s[0][0], s[0][1]), pack2(s[0][2], s[0][3]), pack2(s[1][0], s[1][1]), pack2(s[1][2], s[1][3])};
        const int key = ((lane >> 3) & 1) * 8 + (lane & 7), half = lane >> 4;
        uint32_t keep[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            const int first = 8 * h + 2 * (lane & 3);
            keep[h] = (first < valid ? 0xffffu : 0u) | (first + 1 < valid ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
        {
            uint32_t b[4];
            const int chunk = 2 * i + half;
            ldmatrix_trans(v + (chunk >> 3) * (kKeys * 128) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4), b);
            if (valid < kKeys) // what lies past the last key may be anything, NaN too
            {
                b[0] &= keep[0], b[1] &= keep[1], b[2] &= keep[0], b[3] &= keep[1];
            }
            mma_bf16(o[2 * i], a, b[0], b[1]);
            mma_bf16(o[2 * i + 1], a, b[2], b[3]);
        }
    }
};

template <class T, int D> struct Ring
{
    using L = Layout<T, D>;
    uint32_t slots, bars; // of the CTA
    __device__ uint32_t slot(int worker, unsigned n) const { return slots + (worker * L::kRing + n % L::kRing) * L::kSlotBytes; }
    __device__ uint32_t full(int worker, unsigned n) const { return bars + 8 * (worker * L::kRing + n % L::kRing); }
    __device__ uint32_t empty(int worker, unsigned n) const { return full(worker, n) + 8 * kWorkers * L::kRing; }
    static __device__ uint32_t round(unsigned n) { return (n / L::kRing) & 1u; }
};

// Steps of a part.
template <class T, int D> __device__ __forceinline__ int steps_of_part(const Part &part, int unit_shift)
{
    constexpr int keys = Layout<T, D>::kSlotKeys;
    const int end = min(static_cast<long long>(part.item.keys), static_cast<long long>(part.first_unit + part.units) << unit_shift);
    return (end - (part.first_unit << unit_shift) + keys - 1) / keys;
}

// Four producer warps, each feeding two workers: eight lanes for a worker's K and eight for its V, which run ahead
// by themselves; a lane issues one box of every slot of theirs.
template <class T, int D, bool X>
__device__ __forceinline__ void stream_produce(const Args<X> &p, const Plan &plan, const PlanShared &shared, const CUtensorMap *map_k,
                                               const CUtensorMap *map_v, const Ring<T, D> &ring)
{
    using L = Layout<T, D>;
    const int lane = threadIdx.x & 31, sub = lane & 7, leader = lane & 24, worker = (threadIdx.x / 32) * 2 + (lane >> 4);
    const int shift = p.list[plan.which].unit_shift;
    const unsigned mine = 0xffu << leader;
    const CUtensorMap *map = lane & 8 ? map_v : map_k;
    const bool fine = p.granule < L::kSlotKeys; // two boxes of eight keys to a column block
    const int granule = fine ? sub & 1 : 0, column = fine ? sub >> 1 : sub, granule_shift = fine ? 3 : 31 - __clz(L::kSlotKeys);
    const bool has_box = column < L::kColumns;
    const int first_column = column * (128 / static_cast<int>(sizeof(T)));
    const uint32_t into = column * (L::kSlotKeys * 128) + granule * (8 * 128);
    const uint64_t policy = cache_policy(plan.which);
    Walk w = walk_of(p, plan, shared, worker);
    unsigned n = (lane & 8) >> 3; // the next slot: even ones K's, odd ones V's
    int left = 0, key = 0, row = 0;
    bool bad = false;
    Part part;
    bool more = next_part(p, plan.which, w, part);
    if (more)
    {
        left = steps_of_part<T, D>(part, shift);
        key = part.first_unit << shift;
        row = has_box ? pool_row(p, plan.which, part, key + granule * 8, bad) : 0;
    }
    long long since = clock64();
    while (__any_sync(0xffffffffu, more))
    {
        const bool free = __shfl_sync(0xffffffffu, static_cast<int>(mbar_test(ring.empty(worker, n), ring.round(n) ^ 1u)), leader);
        // no ring has room: out of the workers' issue slots for a while (a step lasts several times as long)
        if (!__any_sync(0xffffffffu, more && free)) __nanosleep(32);
        if (more && free)
        {
            const int kept = min(L::kSlotKeys >> granule_shift, (part.item.keys - key + (1 << granule_shift) - 1) >> granule_shift); // granules with keys
            if (lane == leader) mbar_arrive_expect_tx(ring.full(worker, n), (kept * L::kColumns * 128) << granule_shift);
            __syncwarp(mine);
            if (has_box && granule < kept) tma_load_2d_hint(ring.slot(worker, n) + into, map, ring.full(worker, n), first_column, row, policy);
            n += 2;
            key += L::kSlotKeys;
            if (--left == 0)
            {
                more = next_part(p, plan.which, w, part);
                if (more)
                {
                    left = steps_of_part<T, D>(part, shift);
                    key = part.first_unit << shift;
                }
            }
            if (more && has_box) row = pool_row(p, plan.which, part, key + granule * 8, bad);
            since = clock64();
        }
        else if (more && clock64() - since > kWaitLimitCycles)
        {
            if (lane == leader) atomicExch(p.a.batch.error_flag, kErrAttendUnfinished);
            more = false;
        }
        __syncwarp();
        more = __shfl_sync(0xffffffffu, static_cast<int>(more), leader);
    }
    if (bad) report_range(p.a.batch.error_flag);
}

template <int D, bool X>
__device__ __forceinline__ void stream_work(const Args<X> &p, const Plan &plan, const PlanShared &shared, const Ring<__nv_bfloat16, D> &ring)
{
    using T = __nv_bfloat16;
    using L = Layout<T, D>;
    using R = Rows16<D>;
    const List &l = p.list[plan.which];
    const int worker = threadIdx.x / 32 - 4, lane = threadIdx.x & 31, r0 = lane >> 2, r1 = r0 + 8;
    Walk w = walk_of(p, plan, shared, worker);
    unsigned n = 0; // slots so far: K and V of a step in turn
    Part part;
    while (next_part(p, plan.which, w, part))
    {
        if (lane == 0) write_meta(l, w, part);
        const Row first = row_of(p, plan.which, part, r0), second = row_of(p, plan.which, part, r1);
        R x;
        x.load(p, first, second, lane);
        // below this key every row with a token sees every key
        const int all_see = __reduce_min_sync(0xffffffffu, min(first.keys ? first.keys : INT_MAX, second.keys ? second.keys : INT_MAX));
        float o[D / 8][4], m0 = -INFINITY, m1 = -INFINITY, c0 = 0.f, c1 = 0.f, l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
        const int steps = steps_of_part<T, D>(part, l.unit_shift);
        int key0 = part.first_unit << l.unit_shift;
        for (int u = 0; u < steps; ++u, n += 2, key0 += L::kSlotKeys)
        {
            if (!warp_wait(ring.full(worker, n), ring.round(n)))
            {
                if (lane == 0) atomicExch(p.a.batch.error_flag, kErrAttendUnfinished);
                return;
            }
            const bool v_there = mbar_test(ring.full(worker, n + 1), ring.round(n + 1));
            float s[R::kTiles][4] = {};
            x.scores(ring.slot(worker, n), lane, s);
            __syncwarp();
            if (lane == 0) mbar_arrive(ring.empty(worker, n));
            if (key0 + L::kSlotKeys > all_see)
            {
#pragma unroll
                for (int t = 0; t < R::kTiles; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (key0 + 8 * t + 2 * (lane & 3) + (j & 1) >= (j < 2 ? first.keys : second.keys)) s[t][j] = -INFINITY;
            }
            float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
            for (int t = 0; t < R::kTiles; ++t)
            {
                t0 = max3(t0, s[t][0], s[t][1]);
                t1 = max3(t1, s[t][2], s[t][3]);
            }
            // the maximum is raised only when a score passes it by 2^8: until then sums and values share the
            // old one. (Nothing compares above while both are -inf: the difference is NaN.)
            if (__any_sync(0xffffffffu, (t0 - m0) * p.scale > 8.f || (t1 - m1) * p.scale > 8.f))
            {
                t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
                t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
                t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
                t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
                const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
                const float f0 = n0 == m0 ? 1.f : exp2_fast((m0 - n0) * p.scale), f1 = n1 == m1 ? 1.f : exp2_fast((m1 - n1) * p.scale);
                m0 = n0;
                m1 = n1;
                c0 = m0 == -INFINITY ? 0.f : -m0 * p.scale;
                c1 = m1 == -INFINITY ? 0.f : -m1 * p.scale;
                l0 *= f0;
                l1 *= f1;
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                {
                    o[i][0] *= f0;
                    o[i][1] *= f0;
                    o[i][2] *= f1;
                    o[i][3] *= f1;
                }
            }
#pragma unroll
            for (int t = 0; t < R::kTiles; ++t)
            {
                s[t][0] = exp2_fast(fmaf(s[t][0], p.scale, c0));
                s[t][1] = exp2_fast(fmaf(s[t][1], p.scale, c0));
                s[t][2] = exp2_fast(fmaf(s[t][2], p.scale, c1));
                s[t][3] = exp2_fast(fmaf(s[t][3], p.scale, c1));
                l0 += s[t][0] + s[t][1];
                l1 += s[t][2] + s[t][3];
            }
            if (!__all_sync(0xffffffffu, v_there) && !warp_wait(ring.full(worker, n + 1), ring.round(n + 1)))
            {
                if (lane == 0) atomicExch(p.a.batch.error_flag, kErrAttendUnfinished);
                return;
            }
            x.weigh(ring.slot(worker, n + 1), lane, s, part.item.keys - key0, o);
            __syncwarp();
            if (lane == 0) mbar_arrive(ring.empty(worker, n + 1));
        }
        // a lane's sums cover its columns only
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        const int rows = min(l.block, rows_of(p, plan.which, part.item) - part.block * l.block); // of the item
        const size_t place = static_cast<size_t>(part.place) * l.part_rows;
        float *dst = l.o + place * D + 2 * (lane & 3);
        float2 *ml = l.ml + place;
        if ((lane & 3) == 0)
        {
            if (r0 < rows) ml[r0] = make_float2(m0 * p.scale, l0);
            if (r1 < rows) ml[r1] = make_float2(m1 * p.scale, l1);
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
        {
            if (r0 < rows) *reinterpret_cast<float2 *>(dst + r0 * D + 8 * i) = make_float2(o[i][0], o[i][1]);
            if (r1 < rows) *reinterpret_cast<float2 *>(dst + r1 * D + 8 * i) = make_float2(o[i][2], o[i][3]);
        }
    }
}

// FP32: R rows of a warp, in two halves of 16 lanes; a lane holds every sixteenth group of four dims of the
// queries and values of its half's rows, two dims to a packed FMA. A step takes four keys: partial scores of
// all rows, then a scatter of their sums over the 16 lanes (key lane/4 % 4 and a quarter of the rows each),
// the weights of a slot's eight keys there, and their way back by shuffles. Shared memory and shuffles deliver a
// value per lane and cycle, so a value of K or V has to serve many rows: eight rows to a lane take 250 of those
// cycles for a slot, one row to a lane 1024. What bounds it then is latency, with two warps to a scheduler: of the
// 103 us that 12 groups of 8 sequences take (254 MB) the FMA pipe works 43 (sums over single dims: 144 us; rows
// paired in the packed FMAs: 141 us; a round of weights for every four keys: 115 us).
template <int D, int R, bool X>
__device__ __forceinline__ void stream_work_f32(const Args<X> &p, const Plan &plan, const PlanShared &shared, const Ring<float, D> &ring)
{
    using L = Layout<float, D>;
    constexpr int kSlotKeys = L::kSlotKeys, kKeys = 4, kSteps = kSlotKeys / kKeys, kRows = R / 2, kGroups = D / 64, kPairs = 2 * kGroups;
    constexpr int kHeld = kRows >= 4 ? kRows / 4 : 1; // rows whose weights a lane works out
    const List &l = p.list[plan.which];
    const int worker = threadIdx.x / 32 - 4, lane = threadIdx.x & 31, half = lane & 16, share = lane & 15, first_row = half ? kRows : 0;
    const int my_key = share >> 2, my_row = kRows >= 4 ? (share & 3) * kHeld : (share >> 1) & 1;
    // the lane of key 0 that holds a row
    auto holder = [&](int row) { return half + (kRows >= 4 ? row / kHeld : row * 2); };
    Walk w = walk_of(p, plan, shared, worker);
    unsigned n = 0; // slots so far: K and V of a step in turn
    Part part;
    while (next_part(p, plan.which, w, part))
    {
        if (lane == 0) write_meta(l, w, part);
        float2 q[kRows][kPairs], o[kRows][kPairs]; // two neighbouring dims each
        int all_see = INT_MAX;
#pragma unroll
        for (int i = 0; i < kRows; ++i)
        {
            const Row row = row_of(p, plan.which, part, first_row + i);
            const float4 *query = reinterpret_cast<const float4 *>(static_cast<const float *>(p.a.q) + static_cast<size_t>(row.query) * D) + share;
            if (row.keys) all_see = min(all_see, row.keys);
#pragma unroll
            for (int j = 0; j < kGroups; ++j)
            {
                const float4 x = row.keys ? query[j * 16] : make_float4(0.f, 0.f, 0.f, 0.f);
                q[i][2 * j] = make_float2(x.x, x.y);
                q[i][2 * j + 1] = make_float2(x.z, x.w);
            }
        }
        all_see = __reduce_min_sync(0xffffffffu, all_see);
        int seen[kHeld];
        float m[kHeld], c[kHeld], sum[kHeld];
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
        {
            seen[i] = row_of(p, plan.which, part, first_row + my_row + i).keys;
            m[i] = -INFINITY;
            c[i] = sum[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int d = 0; d < kPairs; ++d) o[i][d] = make_float2(0.f, 0.f);
        const int steps = steps_of_part<float, D>(part, l.unit_shift);
        int key0 = part.first_unit << l.unit_shift;
        for (int u = 0; u < steps; ++u, n += 2)
        {
            if (!warp_wait(ring.full(worker, n), ring.round(n)))
            {
                if (lane == 0) atomicExch(p.a.batch.error_flag, kErrAttendUnfinished);
                return;
            }
            const bool v_there = mbar_test(ring.full(worker, n + 1), ring.round(n + 1));
            const int valid = part.item.keys - key0; // what lies past the last key may be anything, NaN too
            const uint32_t k = ring.slot(worker, n), v = ring.slot(worker, n + 1);
            // dims 64 j + 4 share .. + 3 of key i of the slot: column block, the key's row and its swizzle in one
            // exclusive or (slots are 1024-byte aligned)
            const uint32_t lane_part = (share >> 3) * (kSlotKeys * 128) + ((share & 7) << 4);
            auto at = [&](uint32_t slot, int j, int i) { return ((slot + lane_part) ^ (i * 144)) + j * (2 * kSlotKeys * 128); };
            float w8[kSteps][kHeld]; // scores, then weights: of key 4 t + my_key
#pragma unroll
            for (int t = 0; t < kSteps; ++t)
            {
                // partial sums over the lane's dims, value i * kRows + row; two keys at a time, for the registers
                float s[kKeys * kRows];
#pragma unroll
                for (int i = 0; i < kKeys; i += 2)
                {
                    float2 s2[2][kRows];
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                    {
#pragma unroll
                        for (int r = 0; r < kRows; ++r) s2[e][r] = make_float2(0.f, 0.f);
#pragma unroll
                        for (int j = 0; j < kGroups; ++j)
                        {
                            const float4 x = ld_shared_v4(at(k, j, t * kKeys + i + e));
#pragma unroll
                            for (int r = 0; r < kRows; ++r)
                            {
                                s2[e][r] = __ffma2_rn(q[r][2 * j], make_float2(x.x, x.y), s2[e][r]);
                                s2[e][r] = __ffma2_rn(q[r][2 * j + 1], make_float2(x.z, x.w), s2[e][r]);
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int r = 0; r < kRows; ++r) s[(i + e) * kRows + r] = s2[e][r].x + s2[e][r].y;
                }
                // their sums over the half's lanes, scattered
                int values = kKeys * kRows;
#pragma unroll
                for (int step = 8; step > 0; step /= 2)
                {
                    if (values > 1)
                    {
                        values /= 2;
#pragma unroll
                        for (int i = 0; i < kKeys * kRows / 2; ++i)
                        {
                            if (i >= values) break;
                            const float low = s[i], high = s[i + values];
                            const bool upper = (share & step) != 0;
                            s[i] = (upper ? high : low) + __shfl_xor_sync(0xffffffffu, upper ? low : high, step);
                        }
                    }
                    else
                        s[0] += __shfl_xor_sync(0xffffffffu, s[0], step);
                }
#pragma unroll
                for (int i = 0; i < kHeld; ++i) w8[t][i] = s[i];
            }
            if (key0 + kSlotKeys > all_see)
            {
#pragma unroll
                for (int t = 0; t < kSteps; ++t)
#pragma unroll
                    for (int i = 0; i < kHeld; ++i)
                        if (key0 + t * kKeys + my_key >= seen[i]) w8[t][i] = -INFINITY;
            }
            bool raise = false;
#pragma unroll
            for (int i = 0; i < kHeld; ++i) raise |= (fmaxf(w8[0][i], w8[1][i]) - m[i]) * p.scale > 8.f;
            // the maximum is raised only when a score passes it by 2^8, as for BF16
            if (__any_sync(0xffffffffu, raise))
            {
                float f[kHeld];
#pragma unroll
                for (int i = 0; i < kHeld; ++i)
                {
                    float top = fmaxf(w8[0][i], w8[1][i]);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, m[i]);
                    f[i] = top == m[i] ? 1.f : exp2_fast((m[i] - top) * p.scale);
                    m[i] = top;
                    c[i] = top == -INFINITY ? 0.f : -top * p.scale;
                    sum[i] *= f[i];
                }
#pragma unroll
                for (int r = 0; r < kRows; ++r)
                {
                    const float g = __shfl_sync(0xffffffffu, f[r % kHeld], holder(r));
#pragma unroll
                    for (int d = 0; d < kPairs; ++d) o[r][d] = make_float2(o[r][d].x * g, o[r][d].y * g);
                }
            }
#pragma unroll
            for (int t = 0; t < kSteps; ++t)
#pragma unroll
                for (int i = 0; i < kHeld; ++i)
                {
                    w8[t][i] = exp2_fast(fmaf(w8[t][i], p.scale, c[i]));
                    sum[i] += w8[t][i];
                }
            if (!__all_sync(0xffffffffu, v_there) && !warp_wait(ring.full(worker, n + 1), ring.round(n + 1)))
            {
                if (lane == 0) atomicExch(p.a.batch.error_flag, kErrAttendUnfinished);
                return;
            }
#pragma unroll
            for (int i = 0; i < kSlotKeys; ++i)
            {
                float weight[kRows];
#pragma unroll
                for (int r = 0; r < kRows; ++r) weight[r] = __shfl_sync(0xffffffffu, w8[i / kKeys][r % kHeld], holder(r) + 4 * (i % kKeys));
                if (i >= valid) break;
#pragma unroll
                for (int j = 0; j < kGroups; ++j)
                {
                    const float4 x = ld_shared_v4(at(v, j, i));
#pragma unroll
                    for (int r = 0; r < kRows; ++r)
                    {
                        o[r][2 * j] = __ffma2_rn(make_float2(weight[r], weight[r]), make_float2(x.x, x.y), o[r][2 * j]);
                        o[r][2 * j + 1] = __ffma2_rn(make_float2(weight[r], weight[r]), make_float2(x.z, x.w), o[r][2 * j + 1]);
                    }
                }
            }
            key0 += kSlotKeys;
            __syncwarp();
            if (lane < 2) mbar_arrive(ring.empty(worker, n + lane));
        }
        const int rows = min(l.block, rows_of(p, plan.which, part.item) - part.block * l.block); // of the item
        const size_t place = static_cast<size_t>(part.place) * l.part_rows;
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
        {
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 4);
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 8);
            const int row = first_row + my_row + i;
            if (my_key == 0 && lane == holder(my_row) && row < rows) l.ml[place + row] = make_float2(m[i] * p.scale, sum[i]);
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i)
        {
            if (first_row + i >= rows) break;
            float4 *dst = reinterpret_cast<float4 *>(l.o + (place + first_row + i) * D) + share;
#pragma unroll
            for (int j = 0; j < kGroups; ++j)
            {
                dst[j * 16] = make_float4(o[i][2 * j].x, o[i][2 * j].y, o[i][2 * j + 1].x, o[i][2 * j + 1].y);
            }
        }
    }
}

// ---------------------------------------------------------------- tile (BF16)
// Shared memory: Q_A, Q_B, three tiles that K and V pass through, P_A, P_B. TMEM: S_A 0, S_B 128, O_A 256,
// O_B 384. As in the block attention, softmax copies S_g to registers and frees it, so that S_g of the next
// unit is computed meanwhile, and rescales O_g only when a row's maximum has grown by more than 2^8.
// K and V tiles are loaded in the order K0 K1 V0 K2 V1 K3 V2 ..., in which they are also used: load i goes to
// tile i % 3 once load i - 3 has been used, which is a whole unit ahead of its own use for K and V alike
// (with two buffers for K and one for V, V came 0.6 us late in every unit).
// The two tiles of rows take turns at the exponentials, each with the SM's 16 per clock to itself, and have an
// issuing warp of their own, so that neither waits for the other's scores or weights: in step they would
// compete for the exponentials and then leave them idle together.
template <int D> struct TileSmem
{
    using L = Layout<__nv_bfloat16, D>;
    uint32_t base, bars;
    __device__ uint32_t q(int g) const { return base + g * L::kTileBytes; }
    __device__ uint32_t kv(unsigned load) const { return base + (2 + load % 3) * L::kTileBytes; }
    __device__ uint32_t p(int g) const { return base + 5 * L::kTileBytes + g * L::kWeightBytes; }
    __device__ uint32_t full(unsigned load) const { return bars + 8u * (load % 3); }
    __device__ uint32_t empty(unsigned load) const { return bars + 8u * (3 + load % 3); }
    static __device__ uint32_t round(unsigned load) { return (load / 3) & 1u; }
    static __device__ unsigned k_load(unsigned unit) { return unit ? 2 * unit - 1 : 0; }
    static __device__ unsigned v_load(unsigned unit) { return 2 * unit + 2; }
    __device__ uint32_t q_full(int g) const { return bars + 8u * (6 + g); }
    __device__ uint32_t s_full(int g) const { return bars + 8u * (8 + g); }
    __device__ uint32_t s_free(int g) const { return bars + 8u * (10 + g); }
    __device__ uint32_t p_full(int g) const { return bars + 8u * (12 + g); }
    __device__ uint32_t pv_done(int g) const { return bars + 8u * (14 + g); }
    __device__ uint32_t done() const { return bars + 8u * 16; }
    __device__ uint32_t turn(int g) const { return bars + 8u * (17 + g); }
    __device__ uint32_t tmem_slot() const { return bars + 8u * 19; }
    static constexpr int kBarriers = 19;
    // both issuers empty a K/V tile; the four softmax warps of a tile of rows arrive together
    static __device__ uint32_t arrivals(int barrier)
    {
        return barrier < 3 ? 1 : barrier < 6 ? 2 : barrier < 8 ? 4 : barrier < 10 ? 1 : barrier < 14 ? 4 : barrier < 16 ? 1 : barrier == 16 ? 8 : 4;
    }
};

// Descriptor of V [key][dim] as the second operand (dims x keys, dims contiguous): 128-byte rows of 64 dims,
// 8-key groups 1024 bytes apart, the other 64 dims a column block of 128 keys further on.
__device__ __forceinline__ uint64_t value_desc(uint32_t addr)
{
    uint64_t desc = 0;
    desc |= static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
    desc |= static_cast<uint64_t>((kTile * 128) >> 4) << 16;
    desc |= static_cast<uint64_t>(1024u >> 4) << 32;
    desc |= static_cast<uint64_t>(1u) << 46;
    desc |= static_cast<uint64_t>(2u) << 61;
    return desc;
}

// The K and V tiles of the CTA's units; a lane per box.
template <int D, bool X>
__device__ __forceinline__ void tile_produce(const Args<X> &p, int which, Walk w, const CUtensorMap *map_k, const CUtensorMap *map_v,
                                             const TileSmem<D> &sm)
{
    using L = Layout<__nv_bfloat16, D>;
    const int lane = threadIdx.x & 31, granules = kTile / p.granule, granule = lane % 16, column = lane / 16;
    const bool active = granule < granules && column < L::kColumns;
    const uint32_t into = column * (kTile * 128) + granule * p.granule * 128;
    const uint64_t policy = cache_policy(which);
    Part part;
    int u = 0, key = 0;
    bool bad = false, ok = true;
    part.units = 0;
    // the pool's row of the lane's box of the next unit
    auto fetch = [&](int &row) {
        if (u == part.units)
        {
            if (!next_part(p, which, w, part)) return false;
            u = 0;
            key = part.first_unit * kTile + granule * p.granule;
        }
        row = active ? pool_row(p, which, part, key, bad) : 0;
        key += kTile;
        ++u;
        return true;
    };
    auto load = [&](unsigned i, const CUtensorMap *map, int row) {
        if (ok) ok = warp_wait(sm.empty(i), TileSmem<D>::round(i) ^ 1u);
        if (!ok) return;
        if (lane == 0) mbar_arrive_expect_tx(sm.full(i), L::kTileBytes);
        __syncwarp();
        if (active) tma_load_2d_hint(sm.kv(i) + into, map, sm.full(i), column * 64, row, policy);
    };
    int row = 0, next = 0, after = 0; // of units n, n + 1 and n + 2
    bool have = fetch(row), have_next = have && fetch(next);
    if (have) load(0, map_k, row);
    for (unsigned n = 0; have && ok; ++n)
    {
        const bool have_after = have_next && fetch(after);
        if (have_next) load(sm.k_load(n + 1), map_k, next);
        load(sm.v_load(n), map_v, row);
        row = next;
        next = after;
        have = have_next;
        have_next = have_after;
    }
    if (bad) report_range(p.a.batch.error_flag);
    if (!ok && lane == 0) atomicExch(p.a.batch.error_flag, kErrAttendUnfinished);
}

// The products of tile g of rows, by one thread.
template <int D, bool X> __device__ __forceinline__ void tile_multiply(const Args<X> &p, int which, Walk w, const TileSmem<D> &sm, uint32_t tmem, int g)
{
    const List &l = p.list[which];
    constexpr uint32_t score_desc = idesc_bf16(128, 128);
    constexpr uint32_t value_idesc = idesc_bf16(128, D) | (1u << 16); // second operand with contiguous dims
    unsigned n = 0, seen = 0, parts = 0; // units; units and parts of this tile of rows
    bool ok = true;
    auto arrived = [&](unsigned load) { return ok = ok && mbar_wait(sm.full(load), sm.round(load)); };
    auto issue_s = [&](unsigned unit) {
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
        {
            const uint64_t ad = smem_desc_sw128(sm.q(g) + (i >> 2) * (kTile * 128)) + 2u * (i & 3);
            const uint64_t bd = smem_desc_sw128(sm.kv(sm.k_load(unit)) + (i >> 2) * (kTile * 128)) + 2u * (i & 3);
            umma_bf16(tmem + g * 128, ad, bd, score_desc, i > 0 ? 1u : 0u);
        }
        umma_commit(sm.s_full(g));
        umma_commit(sm.empty(sm.k_load(unit)));
    };
    Part part;
    while (ok && next_part(p, which, w, part))
    {
        if (min(l.block, rows_of(p, which, part.item) - part.block * l.block) <= g * kTile)
        {
            // no rows in this tile: the other one's K and V pass by
            for (int u = 0; u < part.units; ++u, ++n)
            {
                if (arrived(sm.k_load(n))) mbar_arrive(sm.empty(sm.k_load(n)));
                if (arrived(sm.v_load(n))) mbar_arrive(sm.empty(sm.v_load(n)));
            }
            continue;
        }
        ok = mbar_wait(sm.q_full(g), parts++ & 1u);
        if (arrived(sm.k_load(n))) issue_s(n);
        for (int u = 0; u < part.units && ok; ++u, ++n, ++seen)
        {
            if (u + 1 < part.units)
            {
                if (!arrived(sm.k_load(n + 1)) || !(ok = mbar_wait(sm.s_free(g), seen & 1u))) break;
                issue_s(n + 1);
            }
            if (!arrived(sm.v_load(n)) || !(ok = mbar_wait(sm.p_full(g), seen & 1u))) break;
            tc_fence_after();
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i)
            {
                const uint64_t ad = smem_desc_sw128(sm.p(g) + (i >> 2) * (kTile * 128)) + 2u * (i & 3);
                umma_bf16(tmem + 256 + g * 128, ad, value_desc(sm.kv(sm.v_load(n)) + i * 2048), value_idesc, (u > 0 || i > 0) ? 1u : 0u);
            }
            umma_commit(sm.pv_done(g));
            umma_commit(sm.empty(sm.v_load(n)));
        }
    }
    if (!ok) atomicExch(p.a.batch.error_flag, kErrAttendUnfinished);
}

template <int D, bool X>
__device__ __forceinline__ void tile_softmax(const Args<X> &p, int which, Walk w, const TileSmem<D> &sm, uint32_t tmem)
{
    const List &l = p.list[which];
    const int warp = threadIdx.x / 32 - 4, lane = threadIdx.x & 31, g = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16), s_at = lanes + g * 128, o_at = lanes + 256 + g * 128;
    const float c = p.scale;
    unsigned seen = 0, turns = 0; // units of this tile of rows; of them with the other tile at work too
    bool ok = true;
    unsigned n = 0; // units of the CTA
    constexpr int kLanes = D / 8, kRowsAtOnce = 32 / kLanes; // of a row of queries, 16 bytes per lane
    Part part;
    Row row;
    int rows; // of the part's item
    // the next part with rows in this tile, and its queries: the warp's 32 rows on their way to the tile
    auto advance = [&]() {
        while (next_part(p, which, w, part))
        {
            if (warp == 0 && lane == 0) write_meta(l, w, part);
            rows = min(l.block, rows_of(p, which, part.item) - part.block * l.block);
            if (g * kTile < rows)
            {
                row = row_of(p, which, part, g * kTile + r);
                const int chunk = lane % kLanes;
                const uint4 *q = static_cast<const uint4 *>(p.a.q) + chunk;
#pragma unroll
                for (int i = 0; i < 32 / kRowsAtOnce; ++i)
                {
                    const int from = i * kRowsAtOnce + lane / kLanes, at = quarter * 32 + from;
                    const int query = __shfl_sync(0xffffffffu, row.query, from), keys = __shfl_sync(0xffffffffu, row.keys, from);
                    const uint32_t dst = sm.q(g) + (chunk >> 3) * (kTile * 128) + at * 128 + (((chunk & 7) ^ (at & 7)) << 4);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(q + static_cast<size_t>(query) * kLanes), "r"(keys ? 16 : 0)
                                 : "memory"); // zeros for a row without a token
                }
                return true;
            }
            n += part.units;
        }
        return false;
    };
    // The next part's queries are fetched while the last product runs, and are in place before the last part's results
    // leave, so that its first scores are computed meanwhile.
    const int at = g * kTile + r;
    int done_rows = 0;                // of the part before
    size_t place = 0;                 // of its results
    float m = -INFINITY, sum = 0.f;
    for (bool first = true;; first = false)
    {
        const bool have = ok && advance();
        if (!first)
        {
            if (ok) ok = warp_wait(sm.pv_done(g), (seen - 1) & 1u);
            if (!ok)
            {
                if (lane == 0) atomicExch(p.a.batch.error_flag, kErrAttendUnfinished);
                break;
            }
            tc_fence_after();
        }
        if (have)
        {
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(sm.q_full(g));
        }
        if (!first)
        {
            if (at < done_rows) l.ml[place + at] = make_float2(m * c, sum);
            // a warp's 32 rows through their own places in the P tile, 64 columns at a time, so that a store is whole rows
            float *dst = l.o + (place + g * kTile + quarter * 32) * D;
#pragma unroll
            for (int h = 0; h < D / 64; ++h)
            {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                {
                    float o[32];
                    tmem_load_32(o_at + h * 64 + i * 32, o);
#pragma unroll
                    for (int t = 0; t < 8; ++t)
                        st_shared_v4(sm.p(g) + weight_chunk(r, i * 8 + t), __float_as_uint(o[4 * t]), __float_as_uint(o[4 * t + 1]),
                                     __float_as_uint(o[4 * t + 2]), __float_as_uint(o[4 * t + 3]));
                }
                __syncwarp();
#pragma unroll 8
                for (int i = 0; i < 32; i += 2)
                {
                    const int from = i + (lane >> 4);
                    const float4 v = ld_shared_v4(sm.p(g) + weight_chunk(quarter * 32 + from, lane & 15));
                    if (g * kTile + quarter * 32 + from < done_rows) *reinterpret_cast<float4 *>(dst + from * D + h * 64 + (lane & 15) * 4) = v;
                }
                __syncwarp();
            }
            tc_fence_before();
        }
        if (!have) break;
        m = -INFINITY;
        sum = 0.f;
        for (int u = 0; u < part.units && ok; ++u, ++seen)
        {
            if (!(ok = warp_wait(sm.s_full(g), seen & 1u))) break;
            tc_fence_after();
            float x[128];
            tmem_load_128(s_at, x);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(sm.s_free(g));
            const int key0 = (part.first_unit + u) * kTile, visible = row.keys - key0;
            if (visible < kTile)
            {
#pragma unroll
                for (int k = 0; k < 128; ++k)
                    if (k >= visible) x[k] = -INFINITY;
            }
            float mx[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) mx[k] = x[k];
#pragma unroll
            for (int k = 8; k < 128; k += 2) mx[(k >> 1) & 7] = max3(mx[(k >> 1) & 7], x[k], x[k + 1]);
            const float top = fmaxf(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], max3(mx[5], mx[6], mx[7])));
            // PV_g of the last unit still reads P_g and adds to O_g: a rescale waits for it, otherwise the weights
            // are worked out meanwhile and only their stores wait
            bool waited = u == 0;
            if (u == 0) m = top;
            else if (__any_sync(0xffffffffu, (top - m) * c > 8.f)) // NaN while neither is finite: no
            {
                if (!(ok = warp_wait(sm.pv_done(g), (seen - 1) & 1u))) break;
                tc_fence_after();
                waited = true;
                const float raised = fmaxf(m, top), alpha = raised == m ? 1.f : exp2_fast((m - raised) * c);
#pragma unroll
                for (int i = 0; i < D / 32; ++i)
                {
                    float o[32];
                    tmem_load_32(o_at + i * 32, o);
#pragma unroll
                    for (int t = 0; t < 32; ++t) o[t] *= alpha;
                    tmem_store_32(o_at + i * 32, o);
                }
                tmem_store_wait();
                sum *= alpha;
                m = raised;
            }
            const float offset = m == -INFINITY ? 0.f : -m * c;
            const float2 scale2 = make_float2(c, c), offset2 = make_float2(offset, offset);
            float2 part_sum[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            uint32_t packed[64];
            const bool both = rows > kTile;
            if (both && !(ok = warp_wait(sm.turn(g), (turns & 1u) ^ (g ? 0u : 1u)))) break;
#pragma unroll
            for (int k = 0; k < 128; k += 2)
            {
                const float2 arg = __ffma2_rn(make_float2(x[k], x[k + 1]), scale2, offset2);
                const float e0 = exp2_here(arg.x), e1 = exp2_here(arg.y);
                part_sum[(k >> 1) & 3] = __fadd2_rn(part_sum[(k >> 1) & 3], make_float2(e0, e1));
                packed[k >> 1] = pack2(e0, e1);
            }
            if (both)
            {
                __syncwarp();
                if (lane == 0) mbar_arrive(sm.turn(1 - g));
                ++turns;
            }
            if (!waited)
            {
                if (!(ok = warp_wait(sm.pv_done(g), (seen - 1) & 1u))) break;
                tc_fence_after();
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
                st_shared_v4(sm.p(g) + weight_chunk(r, i), packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]);
            const float2 s4 = __fadd2_rn(__fadd2_rn(part_sum[0], part_sum[1]), __fadd2_rn(part_sum[2], part_sum[3]));
            sum += s4.x + s4.y;
            // values past the item's last key may be anything, NaN too: zeros, by both tiles' threads alike
            if (key0 + kTile > part.item.keys)
            {
                const unsigned load = sm.v_load(n + u);
                if (!(ok = warp_wait(sm.full(load), sm.round(load)))) break;
                if (key0 + r >= part.item.keys)
                {
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) st_shared_v4(sm.kv(load) + (i >> 3) * (kTile * 128) + r * 128 + (i & 7) * 16, 0, 0, 0, 0);
                }
            }
            fence_async_smem();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(sm.p_full(g));
        }
        n += part.units;
        done_rows = rows;
        place = static_cast<size_t>(part.place) * l.part_rows;
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(sm.done());
}

// ---------------------------------------------------------------- the kernel
template <class T, int D, bool X>
__global__ void __launch_bounds__(kThreads, 1)
    attend_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Args<X> p)
{
    using L = Layout<T, D>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *base_ptr = smem_raw + (base - raw);
    const uint32_t bars = base + L::kBody;
    PlanShared &shared = *reinterpret_cast<PlanShared *>(base_ptr + L::kBody + 1776);
    static_assert(sizeof(PlanShared) <= 2048 - 1776, "plan");
    const int warp = threadIdx.x / 32;
    const TileSmem<D> sm{base, bars + 2 * kWorkers * L::kRing * 8};
    const Ring<T, D> ring{base, bars};
    static_assert(2 * kWorkers * L::kRing + TileSmem<D>::kBarriers <= kThreads, "a thread per barrier");
    static_assert(2 * kWorkers * L::kRing * 8 + TileSmem<D>::kBarriers * 8 + 8 <= 1776, "barriers");
    {
        // both ways' barriers
        const int t = threadIdx.x - 2 * kWorkers * L::kRing;
        if (t < 0) mbar_init(bars + 8 * threadIdx.x, 1);
        else if (t < TileSmem<D>::kBarriers)
            mbar_init(sm.bars + 8 * t, TileSmem<D>::arrivals(t));
        fence_barrier_init();
        if (threadIdx.x == kThreads - 1)
        {
            prefetch_tensormap(&map_k);
            prefetch_tensormap(&map_v);
        }
    }
    grid_dependency_wait(); // the lengths, tables, queries and the cache are written from here on
    grid_dependents_launch();
    const Plan plan = make_plan(p, shared);
    if (plan.which < 0) return;
    const bool tile = p.list[plan.which].tile != 0;
    if (tile && warp == 1)
    {
        tmem_alloc(sm.tmem_slot(), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp < 4)
    {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
        if constexpr (sizeof(T) == 2)
        {
            if (tile)
            {
                const Walk w = walk_of(p, plan, shared, 0);
                if (warp == 0) tile_produce<D>(p, plan.which, w, &map_k, &map_v, sm);
                else if (warp <= 2)
                {
                    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(base_ptr + (sm.tmem_slot() - base));
                    if ((threadIdx.x & 31) == 0) tile_multiply<D>(p, plan.which, w, sm, tmem, warp - 1);
                    __syncwarp();
                    if (warp == 2) return;
                    if (!warp_wait(sm.done(), 0) && (threadIdx.x & 31) == 0) atomicExch(p.a.batch.error_flag, kErrAttendUnfinished);
                    tc_fence_after();
                    tmem_dealloc(tmem, 512);
                }
                return;
            }
        }
        stream_produce<T, D>(p, plan, shared, &map_k, &map_v, ring);
    }
    else
    {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsWork));
        if constexpr (sizeof(T) == 2)
        {
            if (tile)
            {
                const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(base_ptr + (sm.tmem_slot() - base));
                tile_softmax<D>(p, plan.which, walk_of(p, plan, shared, 0), sm, tmem);
                return;
            }
        }
        if constexpr (sizeof(T) == 2) stream_work<D>(p, plan, shared, ring);
        else
        {
            const int rows = p.list[plan.which].part_rows;
            if (rows > 8) stream_work_f32<D, 16>(p, plan, shared, ring);
            else if (rows > 4) stream_work_f32<D, 8>(p, plan, shared, ring);
            else stream_work_f32<D, 4>(p, plan, shared, ring);
        }
    }
}

// ---------------------------------------------------------------- the join
// R rows per warp (consecutive rows of q and out): 32 / R lanes work out a row's weights, eight parts at a
// time, and all 32 its weighted sum of values, A parts' loads in flight together. Few rows: one per warp with
// eight loads ahead, since a row may have many parts. Many: four per warp, so that they are all on the SMs at
// once with their places worked out before the attention ends (16384 rows one by one took three rounds, 10 us).
constexpr int kJoinWarps = 8;

template <class T, int D, int R, int A, bool X>
__global__ void __launch_bounds__(kJoinWarps * 32, R == 1 ? 1 : 4) join_kernel(const __grid_constant__ Args<X> p)
{
    constexpr int N = D / 32, kLanes = 32 / R, kBatch = 8; // values of a lane; lanes of a row; parts weighed together
    static_assert(kLanes >= kBatch && kBatch % A == 0, "parts of a batch");
    const unsigned full = 0xffffffffu;
    const int lane = threadIdx.x & 31, first_row = (blockIdx.x * kJoinWarps + threadIdx.x / 32) * R;
    const PagedBatch &b = p.a.batch;
    const int rows = b.sequences * b.queries * p.a.heads;
    // The lane's row. The lengths are older than the kernel before this one, which waited for them before it let
    // this one start.
    const int at = first_row + lane / kLanes;
    const int slot = at < rows ? divide(at, p.by_heads) : 0, head = at < rows ? at - slot * p.a.heads : 0;
    const int s = divide(slot, p.by_queries), i = slot - s * b.queries;
    const int kv_head = divide(head, p.by_share), group = divide(slot, p.by_group);
    SequenceView view;
    view.prefix_len = b.max_prefix_pages ? b.prefix_lens[group] : 0;
    static_cast<OwnView &>(view) = own_view(b, p.a.kv.page_shift, s);
    if (b.max_prefix_pages) view.prefix_len = clamped_length(view.prefix_len, b.max_prefix_pages, p.a.kv.page_shift, b.error_flag);
    const bool wanted = at < rows && i < view.count;
    int item[2] = {-1, -1}, within[2] = {0, 0};
    if constexpr (X) // the sums of the counts are the attention's
    {
        grid_dependency_wait();
        grid_dependents_launch();
    }
    const int before = X ? p.earlier[s] - p.earlier[group * p.per] : slot - group * p.list[0].slots - i;
#pragma unroll
    for (int which = 0; which < 2; ++which)
    {
        const List &l = p.list[which];
        if (!wanted || (which == 0 ? view.prefix_len == 0 : view.len - view.count + i + 1 <= 0)) continue;
        const int owner = which == 0 ? group : s;
        const int r = (which == 0 ? before + i : i) * p.share + head - kv_head * p.share, block = r >> l.block_shift;
        item[which] = (owner * l.blocks + block) * p.a.kv.kv_heads + kv_head;
        within[which] = r - block * l.block;
    }
    if constexpr (!X)
    {
        grid_dependency_wait();
        grid_dependents_launch();
    }
    if (first_row >= rows) return;
    int parts[2] = {0, 0}, first[2] = {0, 0}; // of the lane's row, and the first part's place
#pragma unroll
    for (int which = 0; which < 2; ++which)
    {
        if (item[which] < 0) continue;
        const int2 meta = p.list[which].meta[item[which]];
        const PartRange range = parts_between(meta.x, meta.y, p.list[which].workers);
        if (range.count == 0) atomicExch(b.error_flag, kErrAttendUnfinished); // a worker gave up
        parts[which] = range.count;
        first[which] = item[which] + range.first;
    }
    const int total = parts[0] + parts[1], most_parts = __reduce_max_sync(full, total);
    float top = -INFINITY, sum = 0.f, o[R][N] = {};
    for (int base = 0; base < most_parts; base += kBatch)
    {
        const int j = base + lane % kLanes;
        float2 ml = make_float2(-INFINITY, 0.f);
        if (lane % kLanes < kBatch && j < total)
        {
            const int which = j < parts[0] ? 0 : 1;
            const List &l = p.list[which];
            ml = l.ml[static_cast<size_t>(which ? first[1] + j - parts[0] : first[0] + j) * l.part_rows + (which ? within[1] : within[0])];
        }
        float weight = 0.f, rescale = 1.f;
#pragma unroll
        for (int k0 = 0; k0 < kBatch; k0 += A)
        {
            if (base + k0 >= most_parts) break;
            float x[R][A][N];
#pragma unroll
            for (int r = 0; r < R; ++r)
            {
                const int parts0 = __shfl_sync(full, parts[0], r * kLanes), total_r = __shfl_sync(full, total, r * kLanes);
                const int first0 = __shfl_sync(full, first[0], r * kLanes), first1 = __shfl_sync(full, first[1], r * kLanes);
                const int within0 = __shfl_sync(full, within[0], r * kLanes), within1 = __shfl_sync(full, within[1], r * kLanes);
#pragma unroll
                for (int k = 0; k < A; ++k)
                {
                    const int jj = base + k0 + k;
                    const bool shared = jj < parts0;
                    const List &l = p.list[shared ? 0 : 1];
                    const float *src = l.o + (static_cast<size_t>(shared ? first0 + jj : first1 + jj - parts0) * l.part_rows + (shared ? within0 : within1)) * D + lane * N;
#pragma unroll
                    for (int d = 0; d < N; ++d) x[r][k][d] = 0.f;
                    if (jj < total_r)
                    {
                        if constexpr (N == 4)
                        {
                            const float4 t = *reinterpret_cast<const float4 *>(src);
                            x[r][k][0] = t.x, x[r][k][1] = t.y, x[r][k][2] = t.z, x[r][k][3] = t.w;
                        }
                        else
                        {
                            const float2 t = *reinterpret_cast<const float2 *>(src);
                            x[r][k][0] = t.x, x[r][k][1] = t.y;
                        }
                    }
                }
            }
            if (k0 == 0) // the batch's weights, while the values are on their way
            {
                float most = ml.x;
#pragma unroll
                for (int step = kLanes / 2; step > 0; step >>= 1) most = fmaxf(most, __shfl_xor_sync(full, most, step));
                most = fmaxf(most, top);
                rescale = top == most ? 1.f : exp2_fast(top - most);
                weight = ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - most);
                float part_sum = weight * ml.y;
#pragma unroll
                for (int step = kLanes / 2; step > 0; step >>= 1) part_sum += __shfl_xor_sync(full, part_sum, step);
                sum = sum * rescale + part_sum;
                top = most;
#pragma unroll
                for (int r = 0; r < R; ++r)
                {
                    const float f = __shfl_sync(full, rescale, r * kLanes);
#pragma unroll
                    for (int d = 0; d < N; ++d) o[r][d] *= f;
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int k = 0; k < A; ++k)
                {
                    const float f = __shfl_sync(full, weight, r * kLanes + k0 + k);
#pragma unroll
                    for (int d = 0; d < N; ++d) o[r][d] = fmaf(f, x[r][k][d], o[r][d]);
                }
        }
    }
    const float inverse = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
    {
        const float f = __shfl_sync(full, inverse, r * kLanes);
        if (!__shfl_sync(full, static_cast<int>(wanted), r * kLanes)) continue;
        T *dst = static_cast<T *>(p.a.out) + static_cast<size_t>(first_row + r) * D + lane * N;
        if constexpr (sizeof(T) == 4)
        {
            if constexpr (N == 4) *reinterpret_cast<float4 *>(dst) = make_float4(o[r][0] * f, o[r][1] * f, o[r][2] * f, o[r][3] * f);
            else *reinterpret_cast<float2 *>(dst) = make_float2(o[r][0] * f, o[r][1] * f);
        }
        else if constexpr (N == 4)
            *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2(o[r][0] * f, o[r][1] * f), pack2(o[r][2] * f, o[r][3] * f));
        else
            *reinterpret_cast<uint32_t *>(dst) = pack2(o[r][0] * f, o[r][1] * f);
    }
}

// ---------------------------------------------------------------- host
// More rows of an owner and K/V head than this go to the tensor cores' tiles. With 8 K/V heads of 128 (one group
// behind 2048 tokens / eight such groups / one behind 16384), in us, streamed and in tiles: 24 rows 22 / 22 / 34 and
// 17 / 33 / 29; 40 rows 23 / 26 / 36 and 17 / 34 / 29; 80 rows 21 / 45 / 44 and 18 / 38 / 30; 200 rows 24 / 91 / 86
// and 20 / 55 / 38.
constexpr int kTileRows = 32;

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

// Within one block, slots without a token cost nothing. The sums take 1 to 4 us of a call whose slots are all filled: 64
// sequences of 32 slots behind 4096 tokens 172 us by slots and 176 by tokens; with one slot each, 256 behind 8192 77 and
// 77, five behind 300 11.5 and 12.8, 12 groups of eight (FP32) 103 and 105. They save what is empty: of the 64 one with 32
// tokens and the others with one each 179 and 58, 16 of 0 to 32 tokens behind 2000 46 and 37, every other one of the 256
// idle 74 and 46. So sequences of one slot go by slots while a group has few rows.
bool by_tokens(const AttendArgs &p, const PagedBatch &b)
{
    return b.counts && p.list[0].owners && p.list[0].blocks > 1 && (b.queries > 1 || p.list[0].rows > 256);
}

// Lays out the lists and the workspace; returns its size.
size_t lay_out(const PagedLayer &kv, const PagedBatch &b, int heads, int ctas, void *workspace, AttendArgs &p)
{
    p.ctas = ctas;
    p.share = heads / kv.kv_heads;
    p.by_share = divisor(p.share);
    p.by_queries = divisor(b.queries);
    p.by_heads = divisor(heads);
    p.by_group = divisor(b.sequences / b.groups * b.queries);
    char *base = static_cast<char *>(workspace);
    size_t at = 0;
    for (int i = 0; i < 2; ++i)
    {
        List &l = p.list[i];
        l.owners = i == 0 ? (b.max_prefix_pages ? b.groups : 0) : b.sequences;
        l.slots = (i == 0 ? b.sequences / b.groups : 1) * b.queries;
        l.rows = l.slots * p.share;
        l.tile = kv.bf16 && l.rows > kTileRows;
        l.block_shift = l.tile ? 8 : 4;
        l.block = 1 << l.block_shift;
        l.blocks = (l.rows + l.block - 1) / l.block;
        l.part_rows = l.rows < l.block ? l.rows : l.block;
        l.unit_shift = l.tile ? 7 : 5;
        // nanoseconds of an SM: a tile's unit with one and with two tiles of rows; a streamed unit as fast as an SM
        // takes them when the memory is not the limit. An item's fixed cost: queries in, partial results out (streamed
        // items at three units: 64 sequences behind 4096 tokens 31.1 us for 30.1, FP32 groups 110 for 102)
        l.cost = l.tile ? (l.rows > kTile ? 1900 : 1100) : (kv.bf16 ? 180 : l.rows > 8 ? 850 : l.rows > 4 ? 500 : 350) * kv.dim / 128;
        l.lead = l.tile ? (l.rows > kTile ? 4 : 6) : 1;
        const size_t items = static_cast<size_t>(l.owners) * l.blocks * kv.kv_heads;
        l.workers = ctas * (l.tile ? 1 : kWorkers);
        const size_t parts = l.owners ? items + l.workers : 0;
        l.o = reinterpret_cast<float *>(base + at);
        at += rounded(parts * l.part_rows * kv.dim * sizeof(float));
        l.ml = reinterpret_cast<float2 *>(base + at);
        at += rounded(parts * l.part_rows * sizeof(float2));
        l.meta = reinterpret_cast<int2 *>(base + at);
        at += rounded(items * sizeof(int2));
    }
    p.per = b.sequences / b.groups;
    p.earlier = nullptr;
    if (by_tokens(p, b))
    {
        p.earlier = reinterpret_cast<int *>(base + at);
        at += rounded((static_cast<size_t>(b.sequences) + 1) * sizeof(int));
    }
    return at;
}

bool map_pool(CUtensorMap *map, const void *pool, const PagedLayer &kv, int granule)
{
    const auto encode = tensor_map_encoder();
    if (!encode) return false;
    const cuuint64_t element = kv.bf16 ? 2 : 4;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(kv.dim), (static_cast<cuuint64_t>(kv.pages) * kv.kv_heads) << kv.page_shift};
    const cuuint64_t strides[1] = {kv.dim * element};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / element), static_cast<cuuint32_t>(granule)};
    const cuuint32_t element_strides[2] = {1, 1};
    return encode(map, kv.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void *>(pool), dims,
                  strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int D, bool X> int launch(const AttendArgs &args, const CUtensorMap &map_k, const CUtensorMap &map_v, cudaStream_t stream)
{
    Args<X> p;
    static_cast<AttendArgs &>(p) = args;
    const cudaError_t e = launch_dependent(attend_kernel<T, D, X>, p.ctas, kThreads, Layout<T, D>::kSmemBytes, stream, map_k, map_v, p);
    if (e != cudaSuccess) return e;
    const long long rows = static_cast<long long>(p.a.batch.sequences) * p.a.batch.queries * p.a.heads;
    const bool many = rows > 32ll * p.ctas; // one row per warp fills the SMs once up to here
    const long long per_cta = kJoinWarps * (many ? 4 : 1);
    const dim3 grid(static_cast<unsigned>((rows + per_cta - 1) / per_cta));
    return launch_dependent(many ? join_kernel<T, D, 4, 2, X> : join_kernel<T, D, 1, 8, X>, grid, kJoinWarps * 32, 0, stream, p);
}

template <class T, int D> int launch(const PrefixAttentionArgs &a, int sms, cudaStream_t stream)
{
    AttendArgs p;
    p.a = a;
    lay_out(a.kv, a.batch, a.heads, sms, a.workspace, p);
    p.scale = 1.4426950408889634f / sqrtf(static_cast<float>(D));
    p.granule = 1 << a.kv.page_shift;
    if (p.granule > Layout<T, D>::kSlotKeys) p.granule = Layout<T, D>::kSlotKeys;
    CUtensorMap map_k, map_v;
    if (!map_pool(&map_k, a.kv.k, a.kv, p.granule) || !map_pool(&map_v, a.kv.v, a.kv, p.granule)) return cudaErrorInvalidValue;
    return p.earlier ? launch<T, D, true>(p, map_k, map_v, stream) : launch<T, D, false>(p, map_k, map_v, stream);
}

template <class T, int D, bool X> cudaError_t prepare()
{
    cudaFuncAttributes attr;
    const cudaError_t e = cudaFuncGetAttributes(&attr, attend_kernel<T, D, X>);
    if (e != cudaSuccess) return e;
    // the register split needs this many registers per thread at launch
    if (attr.numRegs < kMinLaunchRegs) return cudaErrorInvalidConfiguration;
    static_assert(Layout<T, D>::kSmemBytes <= 232448, "shared memory of a CTA");
    // the join keeps the SMs' split between shared memory and L1: changing it between the two kernels of every
    // call drains the SMs
    cudaError_t c = cudaFuncSetAttribute(join_kernel<T, D, 1, 8, X>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (c == cudaSuccess) c = cudaFuncSetAttribute(join_kernel<T, D, 4, 2, X>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (c != cudaSuccess) return c;
    return cudaFuncSetAttribute(attend_kernel<T, D, X>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<T, D>::kSmemBytes);
}

template <class T, int D> cudaError_t prepare()
{
    const cudaError_t e = prepare<T, D, false>();
    return e == cudaSuccess ? prepare<T, D, true>() : e;
}
} // namespace

size_t prefix_attention_workspace(const PagedLayer &kv, const PagedBatch &batch, int heads, int sms)
{
    AttendArgs p;
    return lay_out(kv, batch, heads, sms, nullptr, p);
}

bool prefix_attention_countable(const PagedLayer &kv, const PagedBatch &batch, int heads)
{
    AttendArgs p;
    lay_out(kv, batch, heads, 1, nullptr, p);
    double steps = 0;
    for (int i = 0; i < 2; ++i)
    {
        const List &l = p.list[i];
        const double keys = static_cast<double>(i == 0 ? batch.max_prefix_pages : batch.max_pages) * (1 << kv.page_shift);
        steps += (keys / (1 << l.unit_shift) + 1 + l.lead) * l.owners * l.blocks * kv.kv_heads;
    }
    return steps < 1e9;
}

int prepare_prefix_attention_kernels()
{
    cudaError_t e = prepare<__nv_bfloat16, 128>();
    if (e == cudaSuccess) e = prepare<__nv_bfloat16, 64>();
    if (e == cudaSuccess) e = prepare<float, 128>();
    if (e == cudaSuccess) e = prepare<float, 64>();
    return e;
}

int launch_prefix_attention(const PrefixAttentionArgs &a, int sms, cudaStream_t stream)
{
    if (a.kv.bf16) return a.kv.dim == 64 ? launch<__nv_bfloat16, 64>(a, sms, stream) : launch<__nv_bfloat16, 128>(a, sms, stream);
    return a.kv.dim == 64 ? launch<float, 64>(a, sms, stream) : launch<float, 128>(a, sms, stream);
}
} // namespace ernie_b200
