// C ABI of batched decoding behind shared prefixes (include/ernie_cuda.h): argument checks and launches.
// The arguments are checked before the context is looked at, so that every refusal of shapes and pointers
// is the same with or without a device.
#include "capi_internal.h"
#include "decode.h"
#include <cstdint>

using namespace ernie_b200;
using namespace ernie_b200::capi;

static_assert(kErrPagedRange == ERNIE_CUDA_STATUS_PAGED_RANGE && kErrAttendUnfinished == ERNIE_CUDA_STATUS_ATTENTION_UNFINISHED, "statuses");

namespace
{
constexpr long long kMaxSlots = 1 << 24; // sequences * queries
constexpr int kMaxHeads = 1024;
constexpr long long kMaxCount = INT32_MAX - 1024; // of what 32-bit indices count: the last one steps past the end by a tile or a CTA's threads

bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

bool overlap(const void *a, size_t a_bytes, const void *b, size_t b_bytes)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + b_bytes && y < x + a_bytes;
}

int check_precision(int precision)
{
    if (precision != ERNIE_PRECISION_BF16 && precision != ERNIE_PRECISION_FP32)
        return fail(ERNIE_CUDA_ERROR, "Unknown precision");
    return ERNIE_CUDA_OK;
}

// What a call writes may not lie in the cache that it works on.
int check_outside(const ernie_cuda_paged_kv *kv, const PagedLayer &layer, const void *p, size_t bytes)
{
    const size_t pool = layer.layer_elements() * (layer.bf16 ? 2 : 4) * kv->layers;
    if (overlap(kv->k, pool, p, bytes) || overlap(kv->v, pool, p, bytes))
        return fail(ERNIE_CUDA_ERROR, "A result or the workspace overlaps the paged cache");
    return ERNIE_CUDA_OK;
}

int check_kv(const ernie_cuda_paged_kv *kv, int layer, PagedLayer &out)
{
    if (!kv || !kv->k || !kv->v) return fail(ERNIE_CUDA_ERROR, "null argument");
    ERNIE_TRY(check_precision(kv->precision));
    int shift = 0;
    while (shift < 7 && (1 << shift) < kv->page_size) ++shift;
    if (shift < 3 || kv->page_size != 1 << shift)
        return fail(ERNIE_CUDA_ERROR, "Page size must be 8, 16, 32, 64 or 128");
    if (kv->head_dim != 64 && kv->head_dim != 128) return fail(ERNIE_CUDA_ERROR, "Head dimension must be 64 or 128");
    if (kv->layers < 1 || kv->layers > 65536 || kv->pages < 1 || kv->kv_heads < 1 || kv->kv_heads > kMaxHeads ||
        ((static_cast<long long>(kv->pages) * kv->kv_heads) << shift) > INT32_MAX)
        return fail(ERNIE_CUDA_ERROR, "Invalid paged cache shape");
    if (layer < 0 || layer >= kv->layers) return fail(ERNIE_CUDA_ERROR, "Layer outside the paged cache");
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return fail(ERNIE_CUDA_ERROR, "The paged cache must be 16-byte aligned");
    out.pages = kv->pages;
    out.page_shift = shift;
    out.kv_heads = kv->kv_heads;
    out.dim = kv->head_dim;
    out.bf16 = kv->precision == ERNIE_PRECISION_BF16;
    const size_t bytes = out.layer_elements() * (out.bf16 ? 2 : 4);
    if (overlap(kv->k, bytes * kv->layers, kv->v, bytes * kv->layers))
        return fail(ERNIE_CUDA_ERROR, "The cache's keys and values overlap");
    out.k = static_cast<char *>(kv->k) + bytes * layer;
    out.v = static_cast<char *>(kv->v) + bytes * layer;
    return ERNIE_CUDA_OK;
}

int check_batch(const ernie_cuda_paged_batch *b, PagedBatch &out)
{
    if (!b || !b->tables || !b->lens) return fail(ERNIE_CUDA_ERROR, "null argument");
    if (b->sequences < 1 || b->queries < 1 || static_cast<long long>(b->sequences) * b->queries > kMaxSlots ||
        b->max_pages < 1 || b->max_prefix_pages < 0)
        return fail(ERNIE_CUDA_ERROR, "Invalid batch shape");
    if (b->groups < 1 || b->sequences % b->groups)
        return fail(ERNIE_CUDA_ERROR, "The groups must divide the sequences");
    if ((b->max_prefix_pages > 0) != (b->prefix_tables != nullptr) || (b->max_prefix_pages > 0) != (b->prefix_lens != nullptr))
        return fail(ERNIE_CUDA_ERROR, "A prefix needs its tables, lengths and page count together");
    if (!aligned(b->tables, 4) || !aligned(b->lens, 4) || !aligned(b->counts, 4) || !aligned(b->prefix_tables, 4) ||
        !aligned(b->prefix_lens, 4))
        return fail(ERNIE_CUDA_ERROR, "Tables and lengths must be 4-byte aligned");
    out.sequences = b->sequences;
    out.queries = b->queries;
    out.groups = b->groups;
    out.max_pages = b->max_pages;
    out.max_prefix_pages = b->max_prefix_pages;
    out.tables = b->tables;
    out.lens = b->lens;
    out.counts = b->counts;
    out.prefix_tables = b->prefix_tables;
    out.prefix_lens = b->prefix_lens;
    return ERNIE_CUDA_OK;
}

int check_heads(int heads, const PagedLayer &kv)
{
    if (heads < 1 || heads > kMaxHeads || heads % kv.kv_heads)
        return fail(ERNIE_CUDA_ERROR, "The query heads must be a multiple of the K/V heads, at most 1024");
    return ERNIE_CUDA_OK;
}

int check_rows(const PagedBatch &b, int heads)
{
    if (static_cast<long long>(b.sequences) * b.queries * heads > kMaxCount)
        return fail(ERNIE_CUDA_ERROR, "2^31 query rows in one call, or nearly");
    return ERNIE_CUDA_OK;
}

int check_work(const PagedBatch &b, const PagedLayer &kv, int heads)
{
    if (!prefix_attention_countable(kv, b, heads))
        return fail(ERNIE_CUDA_ERROR, "The batch's tables hold too many tokens for one attention call");
    return ERNIE_CUDA_OK;
}

// Positions and lengths are 32-bit numbers.
int check_tokens(const PagedBatch &b, const PagedLayer &kv)
{
    const long long own = static_cast<long long>(b.max_pages) << kv.page_shift;
    const long long shared = static_cast<long long>(b.max_prefix_pages) << kv.page_shift;
    if (own + shared > kMaxCount) return fail(ERNIE_CUDA_ERROR, "Tables span 2^31 tokens, or nearly");
    return ERNIE_CUDA_OK;
}

int check_beams(int groups, int beams, int vocab)
{
    if (groups < 1 || beams < 1 || beams > kMaxBeams || vocab < 1)
        return fail(ERNIE_CUDA_ERROR, "Beam search needs groups, 1..32 beams and a vocabulary");
    if (static_cast<long long>(groups) * beams > kMaxSlots) return fail(ERNIE_CUDA_ERROR, "Too many beams in one call");
    if (vocab > kMaxCount) return fail(ERNIE_CUDA_ERROR, "A vocabulary of 2^31 tokens, or nearly");
    return ERNIE_CUDA_OK;
}
} // namespace

extern "C" int ernie_cuda_paged_append(ernie_cuda_context *ctx, const ernie_cuda_paged_kv *kv, int layer,
                                       const ernie_cuda_paged_batch *batch, const void *qkv, int precision, int64_t ld,
                                       int heads, const float *cos, const float *sin, int rope_rows, void *q_out)
{
    AppendArgs a;
    ERNIE_TRY(check_kv(kv, layer, a.kv));
    ERNIE_TRY(check_batch(batch, a.batch));
    ERNIE_TRY(check_tokens(a.batch, a.kv));
    ERNIE_TRY(check_precision(precision));
    ERNIE_TRY(check_heads(heads, a.kv));
    if (!qkv || !cos || !sin || !q_out) return fail(ERNIE_CUDA_ERROR, "null argument");
    const long long width = static_cast<long long>(heads + 2 * a.kv.kv_heads) * a.kv.dim;
    if (ld < width || ld > INT32_MAX) return fail(ERNIE_CUDA_ERROR, "The projection's row stride is below its width or above 2^31");
    if (rope_rows < 1) return fail(ERNIE_CUDA_ERROR, "The rotation needs its table of positions");
    const size_t element = precision == ERNIE_PRECISION_BF16 ? 2 : 4;
    if (!aligned(qkv, element) || !aligned(cos, 16) || !aligned(sin, 16) || !aligned(q_out, 16))
        return fail(ERNIE_CUDA_ERROR, "cos, sin and the queries must be 16-byte aligned");
    const size_t slots = static_cast<size_t>(a.batch.sequences) * a.batch.queries;
    if (overlap(qkv, ((slots - 1) * ld + width) * element, q_out, slots * heads * a.kv.dim * (a.kv.bf16 ? 2 : 4)))
        return fail(ERNIE_CUDA_ERROR, "The queries may not overlap the projection");
    ERNIE_TRY(check_outside(kv, a.kv, q_out, slots * heads * a.kv.dim * (a.kv.bf16 ? 2 : 4)));
    if (!ctx) return fail(ERNIE_CUDA_ERROR, "null context");
    a.qkv = qkv;
    a.qkv_bf16 = precision == ERNIE_PRECISION_BF16;
    a.ld = ld;
    a.heads = heads;
    a.cos = cos;
    a.sin = sin;
    a.rope_rows = rope_rows;
    a.q_out = q_out;
    a.batch.error_flag = ctx->error_flag;
    DeviceGuard guard(ctx->device);
    return from_launch(launch_paged_append(a, ctx->num_sms, ctx->stream), "Paged append");
}

extern "C" int ernie_cuda_prefix_attention_workspace(ernie_cuda_context *ctx, const ernie_cuda_paged_kv *kv,
                                                     const ernie_cuda_paged_batch *batch, int heads, size_t *bytes)
{
    if (!bytes) return fail(ERNIE_CUDA_ERROR, "null argument");
    *bytes = 0;
    PagedLayer layer;
    PagedBatch b;
    ERNIE_TRY(check_kv(kv, 0, layer));
    ERNIE_TRY(check_batch(batch, b));
    ERNIE_TRY(check_tokens(b, layer));
    ERNIE_TRY(check_heads(heads, layer));
    ERNIE_TRY(check_rows(b, heads));
    ERNIE_TRY(check_work(b, layer, heads));
    if (!ctx) return fail(ERNIE_CUDA_ERROR, "null context");
    *bytes = prefix_attention_workspace(layer, b, heads, ctx->num_sms);
    return ERNIE_CUDA_OK;
}

extern "C" int ernie_cuda_prefix_attention(ernie_cuda_context *ctx, const ernie_cuda_paged_kv *kv, int layer,
                                           const ernie_cuda_paged_batch *batch, const void *q, int heads, void *out,
                                           void *workspace, size_t workspace_bytes)
{
    PrefixAttentionArgs a;
    ERNIE_TRY(check_kv(kv, layer, a.kv));
    ERNIE_TRY(check_batch(batch, a.batch));
    ERNIE_TRY(check_tokens(a.batch, a.kv));
    ERNIE_TRY(check_heads(heads, a.kv));
    ERNIE_TRY(check_rows(a.batch, heads));
    ERNIE_TRY(check_work(a.batch, a.kv, heads));
    if (!q || !out || !workspace) return fail(ERNIE_CUDA_ERROR, "null argument");
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 16))
        return fail(ERNIE_CUDA_ERROR, "Queries, output and workspace must be 16-byte aligned");
    const size_t bytes = static_cast<size_t>(a.batch.sequences) * a.batch.queries * heads * a.kv.dim * (a.kv.bf16 ? 2 : 4);
    if (overlap(q, bytes, out, bytes) || overlap(workspace, workspace_bytes, out, bytes) || overlap(workspace, workspace_bytes, q, bytes))
        return fail(ERNIE_CUDA_ERROR, "Queries, output and workspace may not overlap");
    ERNIE_TRY(check_outside(kv, a.kv, out, bytes));
    ERNIE_TRY(check_outside(kv, a.kv, workspace, workspace_bytes));
    if (!ctx) return fail(ERNIE_CUDA_ERROR, "null context");
    if (workspace_bytes < prefix_attention_workspace(a.kv, a.batch, heads, ctx->num_sms))
        return fail(ERNIE_CUDA_ERROR, "The attention's workspace is too small");
    a.q = q;
    a.heads = heads;
    a.out = out;
    a.workspace = workspace;
    a.batch.error_flag = ctx->error_flag;
    DeviceGuard guard(ctx->device);
    return from_launch(launch_prefix_attention(a, ctx->num_sms, ctx->stream), "Prefix attention");
}

extern "C" int ernie_cuda_beam_select_workspace(ernie_cuda_context *ctx, int groups, int beams, int vocab, size_t *bytes)
{
    if (!bytes) return fail(ERNIE_CUDA_ERROR, "null argument");
    *bytes = 0;
    ERNIE_TRY(check_beams(groups, beams, vocab));
    if (!ctx) return fail(ERNIE_CUDA_ERROR, "null context");
    *bytes = beam_select_workspace(groups, beams, vocab, ctx->num_sms);
    return ERNIE_CUDA_OK;
}

extern "C" int ernie_cuda_beam_select(ernie_cuda_context *ctx, const void *logits, int precision, int64_t ld, int groups,
                                      int beams, int vocab, int end_token, const float *scores, const int32_t *finished,
                                      int32_t *parents, int32_t *tokens, float *new_scores, int32_t *new_finished,
                                      void *workspace, size_t workspace_bytes)
{
    ERNIE_TRY(check_beams(groups, beams, vocab));
    ERNIE_TRY(check_precision(precision));
    if (!logits || !scores || !finished || !parents || !tokens || !new_scores || !new_finished || !workspace)
        return fail(ERNIE_CUDA_ERROR, "null argument");
    if (ld < vocab) return fail(ERNIE_CUDA_ERROR, "The logits' row stride is below the vocabulary");
    if (end_token >= vocab) return fail(ERNIE_CUDA_ERROR, "The end token is outside the vocabulary");
    if (!aligned(logits, precision == ERNIE_PRECISION_BF16 ? 2 : 4) || !aligned(scores, 4) || !aligned(finished, 4) ||
        !aligned(parents, 4) || !aligned(tokens, 4) || !aligned(new_scores, 4) || !aligned(new_finished, 4) ||
        !aligned(workspace, 16))
        return fail(ERNIE_CUDA_ERROR, "Beam selection's arrays are not aligned to their elements, or its workspace to 16 bytes");
    {
        // every output and the workspace lie apart from all else, but for the new state in place of the old one
        const size_t list = static_cast<size_t>(groups) * beams * 4, element = precision == ERNIE_PRECISION_BF16 ? 2 : 4;
        const size_t table = ((static_cast<size_t>(groups) * beams - 1) * ld + vocab) * element;
        const void *arrays[8] = {parents, tokens, new_scores, new_finished, workspace, scores, finished, logits};
        const size_t sizes[8] = {list, list, list, list, workspace_bytes, list, list, table};
        for (int i = 0; i < 5; ++i)
            for (int j = i + 1; j < 8; ++j)
            {
                const bool in_place = (i == 2 && j == 5) || (i == 3 && j == 6);
                if (!(in_place && arrays[i] == arrays[j]) && overlap(arrays[i], sizes[i], arrays[j], sizes[j]))
                    return fail(ERNIE_CUDA_ERROR, "Beam selection's arrays overlap");
            }
    }
    if (!ctx) return fail(ERNIE_CUDA_ERROR, "null context");
    if (workspace_bytes < beam_select_workspace(groups, beams, vocab, ctx->num_sms))
        return fail(ERNIE_CUDA_ERROR, "The selection's workspace is too small");
    BeamSelectArgs a;
    a.logits = logits;
    a.bf16 = precision == ERNIE_PRECISION_BF16;
    a.ld = ld;
    a.groups = groups;
    a.beams = beams;
    a.vocab = vocab;
    a.end_token = end_token;
    a.scores = scores;
    a.finished = finished;
    a.parents = parents;
    a.tokens = tokens;
    a.new_scores = new_scores;
    a.new_finished = new_finished;
    a.workspace = workspace;
    DeviceGuard guard(ctx->device);
    return from_launch(launch_beam_select(a, ctx->num_sms, ctx->stream), "Beam selection");
}

extern "C" int ernie_cuda_beam_reorder(ernie_cuda_context *ctx, const ernie_cuda_paged_kv *kv, int groups, int beams,
                                       const int32_t *parents, const int32_t *tables, int max_pages, const int32_t *lens,
                                       int32_t *new_tables, int32_t *new_lens)
{
    ReorderArgs a;
    ERNIE_TRY(check_kv(kv, 0, a.kv));
    ERNIE_TRY(check_beams(groups, beams, 1));
    if (!parents || !tables || !lens || !new_tables || !new_lens) return fail(ERNIE_CUDA_ERROR, "null argument");
    if (max_pages < 1 || (static_cast<long long>(max_pages) << a.kv.page_shift) > kMaxCount ||
        static_cast<long long>(max_pages) * beams > kMaxCount)
        return fail(ERNIE_CUDA_ERROR, "Invalid page table width");
    if (!aligned(parents, 4) || !aligned(tables, 4) || !aligned(lens, 4) || !aligned(new_tables, 4) || !aligned(new_lens, 4))
        return fail(ERNIE_CUDA_ERROR, "Tables, lengths and parents must be 4-byte aligned");
    const size_t rows = static_cast<size_t>(groups) * beams, table = rows * max_pages * 4, list = rows * 4;
    const void *in[3] = {tables, lens, parents};
    const size_t in_bytes[3] = {table, list, list};
    for (int i = 0; i < 3; ++i)
        if (overlap(in[i], in_bytes[i], new_tables, table) || overlap(in[i], in_bytes[i], new_lens, list))
            return fail(ERNIE_CUDA_ERROR, "The new tables and lengths may not overlap the old ones or the parents");
    if (overlap(new_tables, table, new_lens, list)) return fail(ERNIE_CUDA_ERROR, "The new tables and lengths overlap");
    ERNIE_TRY(check_outside(kv, a.kv, new_tables, table));
    ERNIE_TRY(check_outside(kv, a.kv, new_lens, list));
    if (!ctx) return fail(ERNIE_CUDA_ERROR, "null context");
    a.layers = kv->layers;
    a.groups = groups;
    a.beams = beams;
    a.max_pages = max_pages;
    a.parents = parents;
    a.tables = tables;
    a.lens = lens;
    a.new_tables = new_tables;
    a.new_lens = new_lens;
    a.error_flag = ctx->error_flag;
    DeviceGuard guard(ctx->device);
    return from_launch(launch_beam_reorder(a, ctx->num_sms, ctx->stream), "Beam reorder");
}
