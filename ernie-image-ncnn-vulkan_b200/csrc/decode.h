// Batched decoding over a paged K/V cache: the views that the kernels take and the launch interface
// (paged.cu, prefix_attention.cu, beam.cu). Every index that comes from device memory is checked against
// its bound before it is followed; a bad one records kErrPagedRange in the context's status word.
#pragma once
#include "kernels.h"
#include <utility>

namespace ernie_b200
{
constexpr int kErrPagedRange = 41, kErrAttendUnfinished = 42;

// K and V of one layer: [pages][kv_heads][page_size][dim] of T.
struct PagedLayer
{
    void *k = nullptr, *v = nullptr;
    int pages = 0, page_shift = 0, kv_heads = 0, dim = 0;
    int bf16 = 0;
    __host__ __device__ size_t layer_elements() const { return (static_cast<size_t>(pages) * kv_heads * dim) << page_shift; }
};

struct PagedBatch
{
    int sequences = 0, queries = 0, groups = 1, max_pages = 0, max_prefix_pages = 0;
    const int *tables = nullptr, *lens = nullptr, *counts = nullptr, *prefix_tables = nullptr, *prefix_lens = nullptr;
    int *error_flag = nullptr;
};

#ifdef __CUDACC__
// A kernel that waits for the one before it by itself (griddepcontrol.wait), so that its launch and set-up
// overlap that one's end.
template <class... Params, class... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream, Args &&...args)
{
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

__device__ __forceinline__ void report_range(int *flag)
{
    if (flag) atomicExch(flag, kErrPagedRange);
}

// A length clamped to what its table holds.
__device__ __forceinline__ int clamped_length(int len, int max_pages, int page_shift, int *flag)
{
    const long long most = static_cast<long long>(max_pages) << page_shift;
    if (len >= 0 && len <= most) return len;
    report_range(flag);
    return len < 0 ? 0 : static_cast<int>(most);
}

struct OwnView
{
    int len;   // own tokens
    int count; // of them new
};

// All loads come before the first check, so that they wait for one another once.
__device__ __forceinline__ OwnView own_view(const PagedBatch &b, int page_shift, int s)
{
    OwnView v;
    v.len = b.lens[s];
    v.count = b.counts ? b.counts[s] : b.queries;
    v.len = clamped_length(v.len, b.max_pages, page_shift, b.error_flag);
    if (v.count < 0 || v.count > b.queries)
    {
        report_range(b.error_flag);
        v.count = v.count < 0 ? 0 : b.queries;
    }
    return v;
}

struct SequenceView : OwnView
{
    int prefix_len;
};

__device__ __forceinline__ SequenceView sequence_view(const PagedBatch &b, int page_shift, int s)
{
    SequenceView v;
    v.prefix_len = b.max_prefix_pages ? b.prefix_lens[s / (b.sequences / b.groups)] : 0;
    static_cast<OwnView &>(v) = own_view(b, page_shift, s);
    if (b.max_prefix_pages) v.prefix_len = clamped_length(v.prefix_len, b.max_prefix_pages, page_shift, b.error_flag);
    return v;
}
#endif

struct AppendArgs
{
    PagedLayer kv;
    PagedBatch batch;
    const void *qkv = nullptr;
    int qkv_bf16 = 0;
    long long ld = 0;
    int heads = 0;
    const float *cos = nullptr, *sin = nullptr;
    int rope_rows = 0;
    void *q_out = nullptr;
};
int launch_paged_append(const AppendArgs &args, int sms, cudaStream_t stream);

struct ReorderArgs
{
    PagedLayer kv; // layer 0; `layers` follow one another
    int layers = 0, groups = 0, beams = 0, max_pages = 0;
    const int *parents = nullptr, *tables = nullptr, *lens = nullptr;
    int *new_tables = nullptr, *new_lens = nullptr;
    int *error_flag = nullptr;
};
constexpr int kMaxBeams = 32;
int launch_beam_reorder(const ReorderArgs &args, int sms, cudaStream_t stream);

struct PrefixAttentionArgs
{
    PagedLayer kv;
    PagedBatch batch;
    const void *q = nullptr;
    int heads = 0;
    void *out = nullptr;
    void *workspace = nullptr;
};
size_t prefix_attention_workspace(const PagedLayer &kv, const PagedBatch &batch, int heads, int sms);
// Whether the kernel's 32-bit counts of work can hold the longest lengths that the tables allow.
bool prefix_attention_countable(const PagedLayer &kv, const PagedBatch &batch, int heads);
int launch_prefix_attention(const PrefixAttentionArgs &args, int sms, cudaStream_t stream);
int prepare_prefix_attention_kernels();

struct BeamSelectArgs
{
    const void *logits = nullptr;
    int bf16 = 0;
    long long ld = 0;
    int groups = 0, beams = 0, vocab = 0, end_token = -1;
    const float *scores = nullptr;
    const int *finished = nullptr;
    int *parents = nullptr, *tokens = nullptr;
    float *new_scores = nullptr;
    int *new_finished = nullptr;
    void *workspace = nullptr;
};
size_t beam_select_workspace(int groups, int beams, int vocab, int sms);
int prepare_beam_kernels();
int launch_beam_select(const BeamSelectArgs &args, int sms, cudaStream_t stream);
} // namespace ernie_b200
