"""Batched decoding behind shared prefixes on a B200 against the float64 oracle (oracle/decode.py).

Tolerances count roundings (u = 2^-24 for FP32, h = 2^-8 for BF16, half a step each):
 * append: two products and their sum, 3 u of the products' magnitudes, and one rounding to the cache's type;
 * attention: a score of D products, each exact to 4 u (an FP32 operand may be split into parts whose smallest
   cross product is left out) and summed in FP32, is off by at most e = (D + 4) u sum|q||k| / sqrt(D); the weights
   by 2 expm1(2 e) + 16 u relative (exponential, rescaling), their sums over n keys by (n + 16) u each, all relative
   to sum p|v|; with a BF16 cache the weights are rounded once (h of sum p|v|) and the result once (h);
 * selection: a row's sum of exponentials is added up in chains of at most 16 + 5 + 8 + 64 terms with an exponential
   of relative error 8 u: 101 u of the logarithm, and one rounding of the total.
"""
import numpy as np
import pytest

import decode as od
import ernie_cuda as ec
import oracle as o

pytestmark = pytest.mark.gpu
U, H = 2.0 ** -24, 2.0 ** -8


def bf16_bits(x):
    """Round-to-nearest-even FP32 -> BF16 bits (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


class Device:
    """Arrays on the device in one of the two types; freed together."""

    def __init__(self, ctx):
        self.ctx, self.buffers, self.shapes = ctx, {}, {}

    def put(self, name, array, precision=None, offset=0):
        """Uploads `array` (as BF16 bits for ec.BF16) `offset` bytes into a buffer; returns its address."""
        raw = bf16_bits(array) if precision == ec.BF16 else np.ascontiguousarray(array)
        raw = raw.astype(np.float32) if precision == ec.FP32 else raw
        data = np.zeros(raw.nbytes + offset, np.uint8)
        data[offset:] = raw.reshape(-1).view(np.uint8)
        self.buffers[name] = self.ctx.to_device(data)
        self.shapes[name] = (raw.shape, raw.dtype, offset)
        return self.buffers[name].ptr + offset

    def raw(self, name):
        shape, dtype, offset = self.shapes[name]
        data = self.buffers[name].download((self.buffers[name].nbytes,), np.uint8)
        return data[offset:].view(dtype).reshape(shape)

    def get(self, name):
        raw = self.raw(name)
        return o.bf16_to_f32(raw.reshape(-1)).reshape(raw.shape) if raw.dtype == np.uint16 else raw

    def free(self):
        for b in self.buffers.values():
            b.free()


@pytest.fixture
def dev(ctx):
    d = Device(ctx)
    yield d
    ctx.synchronize()
    d.free()


def values(rng, shape, precision, scale=1.0):
    """FP32 values that the type holds exactly."""
    x = (rng.standard_normal(shape) * scale).astype(np.float32)
    return o.bf16_to_f32(bf16_bits(x).reshape(-1)).reshape(shape) if precision == ec.BF16 else x


def split_pages(rng, rows, extra=2):
    """Tables with rows[i] entries each (-7 past them) from one shuffled pool; the pool's size."""
    total = int(sum(rows)) + extra
    order, at, width = rng.permutation(total), 0, max(1, max(rows))
    tables = np.full((len(rows), width), -7, np.int32)
    for i, n in enumerate(rows):
        tables[i, :n] = order[at:at + n]
        at += n
    return tables, total


# ------------------------------------------------------------------ append
APPENDS = [
    # sequences, queries, heads, kv heads, dim, page, in, cache, padding of a row, offset in bytes, prefix groups
    (1, 1, 32, 8, 128, 16, ec.FP32, ec.BF16, 0, 0, 0),
    (5, 1, 32, 8, 128, 16, ec.FP32, ec.FP32, 0, 0, 1),
    (6, 7, 6, 2, 64, 8, ec.BF16, ec.BF16, 0, 0, 3),
    (3, 33, 7, 1, 128, 32, ec.FP32, ec.BF16, 3, 4, 1),
    (4, 20, 5, 5, 64, 64, ec.BF16, ec.FP32, 5, 2, 2),
    (2, 150, 12, 6, 128, 128, ec.BF16, ec.BF16, 8, 16, 1),
    (2, 40, 20, 4, 128, 16, ec.FP32, ec.FP32, 4, 16, 0),
]


@pytest.mark.parametrize("case", APPENDS, ids=str)
def test_append(ctx, dev, case):
    sequences, queries, heads, kv_heads, dim, page, source, cache, pad, offset, groups = case
    rng = np.random.default_rng(sum(int(x) for x in case))
    counts = rng.integers(0, queries + 1, sequences).astype(np.int32)
    counts[-1] = queries
    lens = (counts + rng.integers(0, 40, sequences)).astype(np.int32)
    tables, pages = split_pages(rng, [-(-int(n) // page) for n in lens])
    prefix_lens = rng.integers(0, 60, groups).astype(np.int32) if groups else None
    k, v = (values(rng, (2, pages, kv_heads, page, dim), cache) for _ in range(2))
    q = values(rng, (sequences * queries, heads, dim), cache)
    width = (heads + 2 * kv_heads) * dim
    qkv = values(rng, (sequences * queries, width + pad), source)
    rows = 260
    cos, sin = rng.uniform(-1, 1, (2, rows, dim)).astype(np.float32)
    kv = ec.PagedKv(dev.put("k", k, cache), dev.put("v", v, cache), 2, pages, page, kv_heads, dim, cache)
    prefix = dict(groups=groups, prefix_tables=dev.put("pt", np.zeros((groups, 8), np.int32)), max_prefix_pages=8,
                  prefix_lens=dev.put("pl", prefix_lens)) if groups else {}
    if groups:
        prefix_lens = np.minimum(prefix_lens, 8 * page)
    batch = ec.PagedBatch(sequences, queries, dev.put("t", tables), tables.shape[1], dev.put("n", lens),
                          dev.put("c", counts), **prefix)
    ctx.paged_append(kv, 1, batch, dev.put("x", qkv, source, offset), source, width + pad, heads, dev.put("cos", cos),
                     dev.put("sin", sin), rows, dev.put("q", q, cache))
    ctx.synchronize()
    rk, rv, rq = k.astype(np.float64), v.astype(np.float64), q.astype(np.float64)
    scales = od.append(rk, rv, 1, rq, tables, lens, counts, qkv, cos, sin, prefix_lens)
    for name, ref, old, scale in (("q", rq, q, scales[0]), ("k", rk, k, scales[1]), ("v", rv, v, scales[2])):
        got = dev.get(name).astype(np.float64)
        same = ref == old
        assert np.array_equal(got[same], old[same].astype(np.float64)), name
        limit = 3 * U * scale + (H if cache == ec.BF16 else 0.0) * (np.abs(ref) + 3 * U * scale)
        assert (np.abs(got - ref) <= limit).all(), (name, float(np.abs(got - ref).max()))
    if cache == source or cache == ec.FP32:  # values only move
        assert np.array_equal(dev.get("v").astype(np.float64), rv)


def test_append_range_reports(ctx, dev):
    """Bad pages, positions, lengths and counts: nothing stored for them, the rest as usual, status 41."""
    rng = np.random.default_rng(3)
    k, v = np.zeros((2, 1, 6, 2, 8, 64), np.float32)
    cos, sin = np.ones((20, 64), np.float32), np.zeros((20, 64), np.float32)
    kv = ec.PagedKv(dev.put("k", k), dev.put("v", v), 1, 6, 8, 2, 64, ec.FP32)
    #         good    page below 0    page past the pool    position past the table of rotations
    tables = np.array([[3, 1, 1], [-1, 2, 2], [6, 4, 4], [0, 5, 5]], np.int32)
    lens = np.array([1, 4, 2, 21], np.int32)
    q = dev.put("q", np.full((4, 2, 64), 9.0, np.float32))
    batch = ec.PagedBatch(4, 1, dev.put("t", tables), 3, dev.put("n", lens))
    wide = values(rng, (4, 6 * 64), ec.FP32)
    ctx.paged_append(kv, 0, batch, dev.put("w", wide), ec.FP32, 384, 2, dev.put("c", cos), dev.put("s", sin), 20, q)
    with pytest.raises(ec.CudaError, match="status 41"):
        ctx.synchronize()
    got = dev.get("k")
    assert np.array_equal(got[0, 3, :, 0], wide[0, 128:256].reshape(2, 64))
    got[0, 3, :, 0] = 0
    assert not got.any()
    assert np.array_equal(dev.get("q")[:3], wide[:3, :128].reshape(3, 2, 64)) and (dev.get("q")[3] == 9.0).all()
    # lengths below zero and past the table, counts out of range: clamped, reported, no store outside
    for bad_lens, bad_counts in (([-5, 1, 1, 1], [1, 1, 1, 1]), ([1, 1, 1, 1], [2, 0, 0, 0]), ([1, 1, 1, 1], [-1, 0, 0, 0]),
                                 ([25, 1, 1, 1], [0, 0, 0, 0])):
        dev2 = Device(ctx)
        good = np.array([[0, 1, 2], [3, 3, 3], [4, 4, 4], [5, 5, 5]], np.int32)
        batch = ec.PagedBatch(4, 1, dev2.put("t", good), 3, dev2.put("n", np.array(bad_lens, np.int32)),
                              dev2.put("m", np.array(bad_counts, np.int32)))
        ctx.paged_append(kv, 0, batch, dev.buffers["w"], ec.FP32, 384, 2, dev.buffers["c"], dev.buffers["s"], 20, q)
        with pytest.raises(ec.CudaError, match="status 41"):
            ctx.synchronize()
        dev2.free()
    ctx.synchronize()


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
def test_append_past_the_table_keeps_the_cache(ctx, dev, precision):
    """New tokens of a sequence whose pages are full: stored nowhere, the tokens before them stay and those that still
    have a place get it; status 41."""
    rng = np.random.default_rng(17)
    n, queries, page, dim, own = 6, 3, 8, 64, 16
    k, v = (values(rng, (1, 2 * n, 1, page, dim), precision) for _ in range(2))
    cos, sin = rng.uniform(-1, 1, (2, 40, dim)).astype(np.float32)
    tables = rng.permutation(2 * n).reshape(n, 2).astype(np.int32)
    lens, counts = np.array([16, 17, 17, 18, 30, 2 ** 31 - 1], np.int32), np.array([1, 1, 3, 3, 3, 3], np.int32)
    x, q = values(rng, (n * queries, 3 * dim), precision), values(rng, (n * queries, 1, dim), precision)
    kv = ec.PagedKv(dev.put("k", k, precision), dev.put("v", v, precision), 1, 2 * n, page, 1, dim, precision)
    batch = ec.PagedBatch(n, queries, dev.put("t", tables), 2, dev.put("n", lens), dev.put("c", counts))
    ctx.paged_append(kv, 0, batch, dev.put("x", x, precision), precision, 3 * dim, 1, dev.put("cos", cos), dev.put("sin", sin), 40,
                     dev.put("q", q, precision))
    with pytest.raises(ec.CudaError, match="status 41"):
        ctx.synchronize()
    got_k, got_v, got_q = dev.get("k"), dev.get("v"), dev.get("q")
    for s in range(n):
        for i in range(queries):
            place, row = int(lens[s]) - int(counts[s]) + i, s * queries + i
            if i >= counts[s] or place >= 40:
                assert np.array_equal(got_q[row], q[row])
                continue
            c, m = cos[place].astype(np.float64), sin[place].astype(np.float64)
            for got, old, at in ((got_q[row, 0], x[row, :dim], None), (None, x[row, dim:2 * dim], got_k)):
                y, size = od.rotate(old.astype(np.float64), c, m), np.abs(old) * np.abs(c) + np.abs(np.roll(old, dim // 2)) * np.abs(m)
                if at is not None:
                    if place >= own:
                        continue
                    page_at = tables[s, place // page]
                    got = at[0, page_at, 0, place % page].copy()
                    k[0, page_at, 0, place % page], v[0, page_at, 0, place % page] = got, x[row, 2 * dim:]
                limit = 3 * U * size + (H if precision == ec.BF16 else 0.0) * (np.abs(y) + 3 * U * size)
                assert (np.abs(got - y) <= limit).all(), (s, i)
    assert np.array_equal(got_k, k) and np.array_equal(got_v, v), "a token was overwritten"


# ------------------------------------------------------------------ attention
def attention_case(ctx, dev, rng, groups, per, queries, prefix, suffix, heads, kv_heads, dim, page, precision,
                   counts=None, lens=None, prefix_lens=None, layers=1, layer=0, poison=True, scale=1.0, prefix_free=False):
    """Runs one call on a cache whose unused places hold NaN; returns (got, ref, limit, untouched rows)."""
    n = groups * per
    lens = np.array(rng.integers(queries, max(queries, suffix) + 1, n) if lens is None else lens, np.int32)
    counts = np.array(rng.integers(0, queries + 1, n) if counts is None else counts, np.int32)
    prefix_lens = np.array(rng.integers(0, prefix + 1, groups) if prefix_lens is None else prefix_lens, np.int32)
    rows = [-(-int(x) // page) for x in list(prefix_lens) + list(lens)]
    every, pages = split_pages(rng, rows)
    width_p, width_s = max(1, max(rows[:groups])), max(1, max(rows[groups:]))
    prefix_tables, tables = every[:groups, :width_p].copy(), every[groups:, :width_s].copy()
    shape = (layers, pages, kv_heads, page, dim)
    clean = [values(rng, shape, precision, scale) for _ in range(2)]
    stored = [x.copy() for x in clean]
    if poison:  # what lies past the lengths, in foreign pages and layers
        used = np.zeros((pages, page), bool)
        for table, length in list(zip(prefix_tables, prefix_lens)) + list(zip(tables, lens)):
            for t in range(int(length)):
                used[table[t // page], t % page] = True
        for i, x in enumerate(stored):
            x[layer][np.broadcast_to(~used[:, None, :, None], x[layer].shape)] = (np.nan, np.inf)[i]
            for other in range(layers):
                if other != layer:
                    x[other] = np.nan
    bits = [np.where(np.isnan(x), np.uint16(0x7FC0), np.where(np.isinf(x), np.uint16(0x7F80), bf16_bits(np.nan_to_num(x, posinf=0))))
            if precision == ec.BF16 else x for x in stored]
    q = values(rng, (n * queries, heads, dim), precision, 1.5)
    before = values(rng, q.shape, precision)
    kv = ec.PagedKv(dev.put("k", bits[0]), dev.put("v", bits[1]), layers, pages, page, kv_heads, dim, precision)
    shared = {} if prefix_free else dict(groups=groups, prefix_tables=dev.put("pt", prefix_tables),
                                         max_prefix_pages=width_p, prefix_lens=dev.put("pl", prefix_lens))
    batch = ec.PagedBatch(n, queries, dev.put("t", tables), width_s, dev.put("n", lens), dev.put("c", counts), **shared)
    size = ctx.prefix_attention_workspace(kv, batch, heads)
    # scratch that holds anything
    work = dev.put("work", np.full(size, 0xFF, np.uint8))
    ctx.prefix_attention(kv, layer, batch, dev.put("q", q, precision), heads, dev.put("out", before, precision), work, size)
    ctx.synchronize()
    got = dev.get("out").astype(np.float64)
    ref = before.astype(np.float64)
    weight, spread = od.attention(clean[0], clean[1], layer, q, ref, tables, lens, counts,
                                  None if prefix_free else prefix_tables, None if prefix_free else prefix_lens)
    keys = int(lens.max() + prefix_lens.max())
    e = (dim + 4) * U * spread[:, :, None]
    limit = weight * (2 * np.expm1(2 * e) + 16 * U + 2 * (keys + 16) * U)
    if precision == ec.BF16:
        limit += H * weight
        limit += H * (np.abs(ref) + limit)
    else:
        limit += U * np.abs(ref)
    untouched = ~(np.arange(queries) < counts[:, None]).reshape(-1)
    assert np.array_equal(got[untouched], before[untouched].astype(np.float64)), "a slot without a token was written"
    limit[untouched] = 0.0
    return got, ref, limit


def holds(got, ref, limit):
    assert np.isfinite(got).all()
    over = np.abs(got - ref) - limit
    assert (over <= 0).all(), (float(np.abs(got - ref).max()), float(over.max()), np.argwhere(over > 0)[:5].tolist())


ATTENTIONS = [
    # groups, per group, queries, prefix, suffix, heads, kv heads, dim, page
    (1, 1, 1, 0, 1, 32, 8, 128, 16),      # one token, nothing before it
    (1, 5, 1, 77, 13, 32, 8, 128, 16),    # five beams
    (1, 64, 1, 300, 90, 32, 8, 128, 16),  # 256 rows behind one prefix
    (3, 4, 1, 150, 40, 8, 8, 128, 32),    # one query head per K/V head
    (2, 3, 5, 129, 33, 6, 2, 64, 8),
    (1, 2, 40, 257, 200, 7, 1, 128, 64),  # seven query heads share one
    (4, 1, 17, 33, 300, 20, 4, 64, 128),
    (2, 2, 3, 500, 20, 16, 1, 128, 128),  # sixteen share one
    (1, 3, 2, 64, 128, 48, 1, 64, 16),    # forty-eight
    (1, 37, 2, 255, 65, 24, 4, 128, 8),
    (5, 7, 1, 1, 2, 12, 6, 64, 64),
    (1, 1, 130, 0, 130, 4, 4, 128, 16),   # a prompt of its own, causal
]


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", ATTENTIONS, ids=str)
def test_attention(ctx, dev, case, precision):
    rng = np.random.default_rng(sum(case) + precision)
    holds(*attention_case(ctx, dev, rng, *case, precision, layers=2, layer=1))


LARGE = [
    # groups, per group, queries, prefix, suffix, heads, kv heads, dim, page
    (1, 200, 1, 300, 40, 32, 8, 128, 16),    # 6400 rows: four to a warp of the join
    (2, 130, 1, 700, 30, 48, 4, 64, 16),
    (1, 1, 40, 2000, 2000, 128, 1, 128, 64),  # rows of more than eight parts
    (1, 500, 1, 40, 20, 4, 2, 64, 8),        # more sequences than a CTA has threads
    (450, 2, 1, 30, 10, 4, 2, 64, 8),        # and groups
]


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", LARGE, ids=str)
def test_attention_of_large_batches(ctx, dev, case, precision):
    """Some of the sequences idle (no new token) and some empty."""
    rng = np.random.default_rng(sum(case) + precision)
    n = case[0] * case[1]
    lens, counts = rng.integers(0, case[4] + 1, n), np.full(n, case[2])
    counts[rng.random(n) < 0.2] = 0
    lens[0], counts[0] = max(case[4], case[2]), case[2]
    holds(*attention_case(ctx, dev, rng, *case, precision, lens=lens, counts=counts))


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("groups,per,queries,kind", [
    (1, 64, 32, "one long"), (3, 9, 20, "one long"), (2, 12, 33, "random"), (2, 300, 3, "random"), (5, 1, 150, "random"),
    (2, 40, 8, "last"), (3, 30, 8, "one group idle"), (2, 20, 24, "out of range"), (2, 70, 1, "random")])
def test_attention_of_mixed_batches(ctx, dev, groups, per, queries, kind, precision):
    """Sequences with one new token beside ones with many or none: the rows that share a prefix are the tokens'."""
    rng = np.random.default_rng(groups + per + queries)
    n = groups * per
    counts = {"one long": np.where(np.arange(n) % per == per // 2, queries, 1), "random": rng.integers(0, queries + 1, n),
              "last": np.where(np.arange(n) == n - 1, queries, 0), "one group idle": np.where(np.arange(n) // per == 1, 0, queries),
              "out of range": rng.integers(0, queries + 1, n)}[kind]
    lens = counts + rng.integers(0, 50, n)
    prefix = rng.integers(1, 400, groups)
    case = (groups, per, queries, 0, 0, 8, 1, 128, 16, precision)
    if kind != "out of range":
        holds(*attention_case(ctx, dev, rng, *case, counts=counts, lens=lens, prefix_lens=prefix))
        return
    counts[3], counts[per] = -2, queries + 5  # clamped to none and to all
    with pytest.raises(ec.CudaError, match="status 41"):
        attention_case(ctx, dev, rng, *case, counts=counts, lens=np.maximum(lens, 0), prefix_lens=prefix)
    counts[3], counts[per] = 0, queries
    fine = Device(ctx)
    got, want, limit = attention_case(ctx, fine, np.random.default_rng(groups + per + queries + 1), *case, counts=counts, lens=np.maximum(lens, 0),
                                      prefix_lens=prefix)
    fine.free()
    holds(got, want, limit)


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,counts,prefix", [
    ([0, 0, 0, 0], [0, 0, 0, 0], [50, 50]),      # an idle batch
    ([0, 5, 128, 1], [1, 3, 3, 1], [0, 40]),     # more new tokens than the sequence holds: rows that see nothing
    ([3, 3, 130, 129], [3, 0, 2, 3], [128, 256]),  # whole key tiles
    ([127, 128, 129, 1], [1, 1, 1, 1], [127, 129]),
], ids=["idle", "empty rows", "whole tiles", "tile edges"])
def test_attention_lengths(ctx, dev, lens, counts, prefix, precision):
    rng = np.random.default_rng(len(lens) + sum(lens))
    holds(*attention_case(ctx, dev, rng, 2, 2, 3, 0, 0, 8, 2, 128, 16, precision, counts=counts, lens=lens,
                          prefix_lens=prefix))


@pytest.mark.parametrize("seed", range(24))
def test_attention_of_random_shapes(ctx, dev, seed):
    """Any head layout, page, batch and raggedness; the largest of the 24 has some 20000 rows."""
    rng = np.random.default_rng(4000 + seed)
    kv_heads, share = int(rng.choice([1, 2, 3, 4, 8])), int(rng.choice([1, 2, 3, 4, 5, 7, 8, 16]))
    dim, page = int(rng.choice([64, 128])), int(rng.choice([8, 16, 32, 64, 128]))
    groups, per = int(rng.choice([1, 2, 3, 5])), int(np.exp(rng.uniform(0, np.log(70))))
    queries, prefix, suffix = (int(np.exp(rng.uniform(0, np.log(most)))) for most in (60, 3000, 600))
    while groups * per * queries * kv_heads * share > 20000:
        per, queries = max(1, per // 2), max(1, queries // 2)
    n, ragged = groups * per, {}
    if seed % 3 == 1:
        ragged["counts"] = np.full(n, queries)
    if seed % 3 == 2:
        ragged["counts"] = np.where(rng.random(n) < 0.3, queries, rng.integers(0, 2, n))
        ragged["lens"] = rng.integers(0, suffix + queries, n)
    holds(*attention_case(ctx, dev, rng, groups, per, queries, prefix, suffix, kv_heads * share, kv_heads, dim, page,
                          ec.BF16 if seed % 2 else ec.FP32, **ragged))


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
def test_attention_without_a_prefix(ctx, dev, precision):
    rng = np.random.default_rng(9)
    holds(*attention_case(ctx, dev, rng, 1, 6, 4, 0, 200, 8, 2, 128, 16, precision, prefix_lens=[0], prefix_free=True))


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
def test_attention_of_large_scores(ctx, dev, precision):
    """Scores up to about a hundred: one key takes nearly all the weight, the running maximum moves all the time."""
    rng = np.random.default_rng(10)
    holds(*attention_case(ctx, dev, rng, 1, 40, 1, 700, 150, 8, 2, 128, 16, precision, scale=12.0))


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("queries,per", [(1, 3), (1, 40), (9, 4)])
def test_attention_repeats_bit_for_bit_and_ignores_its_scratch(ctx, dev, queries, per, precision):
    rng = np.random.default_rng(11)
    got, ref, limit = attention_case(ctx, dev, rng, 1, per, queries, 1500, 100, 8, 2, 128, 16, precision, prefix_lens=[1500])
    holds(got, ref, limit)
    rng = np.random.default_rng(11)
    other = Device(ctx)
    again, _, _ = attention_case(ctx, other, rng, 1, per, queries, 1500, 100, 8, 2, 128, 16, precision, prefix_lens=[1500],
                                 poison=False)
    other.free()
    assert np.array_equal(got, again)


@pytest.mark.parametrize("groups,per,queries,heads,kv_heads,dim,page", [
    (1, 300, 40, 2, 2, 128, 16),   # 40 rows: two of a tile's four warps store nothing
    (1, 160, 25, 8, 2, 64, 8),     # 100 rows
    (4, 25, 33, 8, 2, 128, 32),    # 132 rows: the second tile has four
    (2, 40, 70, 6, 2, 128, 64),    # 210 rows
    (120, 5, 9, 4, 2, 128, 16)])   # many short prefixes
def test_attention_of_many_short_parts_repeats(ctx, dev, groups, per, queries, heads, kv_heads, dim, page):
    """Several parts on every CTA and tile of rows, each of one to three key tiles: a part's results leave while the
    next part's weights come in. Right once, then the same bits 200 times."""
    rng = np.random.default_rng(groups + per + queries)
    holds(*attention_case(ctx, dev, rng, groups, per, queries, 300, 300, heads, kv_heads, dim, page, ec.BF16,
                          prefix_lens=rng.integers(1, 300, groups)))
    (layers, pages), tables, prefix_tables = dev.shapes["k"][0][:2], dev.shapes["t"][0], dev.shapes["pt"][0]
    b = dev.buffers
    kv = ec.PagedKv(b["k"], b["v"], layers, pages, page, kv_heads, dim, ec.BF16)
    batch = ec.PagedBatch(groups * per, queries, b["t"], tables[1], b["n"], b["c"], groups, b["pt"], prefix_tables[1], b["pl"])
    first = dev.raw("out").copy()
    for _ in range(200):
        ctx.prefix_attention(kv, 0, batch, b["q"], heads, b["out"], b["work"], b["work"].nbytes)
        ctx.synchronize()
        assert np.array_equal(dev.raw("out"), first)


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("per", [2, 40])
def test_attention_of_bad_pages(ctx, dev, per, precision):
    """A bad page's keys count as zeros and status 41 is reported; other sequences are not touched by it."""
    rng = np.random.default_rng(12)
    heads, kv_heads, dim, page = 8, 2, 128, 16
    lens = np.full(per, 20, np.int32)
    tables, pages = split_pages(rng, [2] * per + [3])
    tables, prefix = tables[:-1, :2].copy(), tables[-1:].copy()
    k, v = (values(rng, (1, pages, kv_heads, page, dim), precision) for _ in range(2))
    q = values(rng, (per, heads, dim), precision)
    dev.put("k", k, precision), dev.put("v", v, precision), dev.put("q", q, precision)
    kv = ec.PagedKv(dev.buffers["k"], dev.buffers["v"], 1, pages, page, kv_heads, dim, precision)

    def run(tables, prefix, prefix_len):
        d = Device(ctx)
        batch = ec.PagedBatch(per, 1, d.put("t", tables), 2, d.put("n", lens), None, 1, d.put("p", prefix), 3,
                              d.put("l", np.array([prefix_len], np.int32)))
        size = ctx.prefix_attention_workspace(kv, batch, heads)
        ctx.prefix_attention(kv, 0, batch, dev.buffers["q"], heads, d.put("out", q, precision), ctx_work(d, size), size)
        try:
            ctx.synchronize()
            return d.get("out"), False
        except ec.CudaError as error:
            assert "status 41" in str(error)
            return d.get("out"), True
        finally:
            d.free()

    def ctx_work(d, size):
        return d.put("work", np.zeros(size, np.uint8))

    good, reported = run(tables, prefix, 40)
    assert not reported
    for bad in (-1, pages, 2 ** 31 - 1, -2 ** 31):
        changed = tables.copy()
        changed[0, 1] = bad
        got, reported = run(changed, prefix, 40)
        assert reported and np.isfinite(got).all()
        assert np.array_equal(got[1:], good[1:])
        k0, v0 = k.copy(), v.copy()
        k0[0, tables[0, 1]], v0[0, tables[0, 1]] = 0, 0
        ref = q.astype(np.float64)
        weight, spread = od.attention(k0, v0, 0, q, ref, tables, lens, [1] * per, prefix, [40])
        assert (np.abs(got - ref) <= weight * 0.01 + 2 * H * np.abs(ref) + 1e-6).all()
        changed = prefix.copy()
        changed[0, 2] = bad
        got, reported = run(tables, changed, 40)
        assert reported and np.isfinite(got).all()
    got, reported = run(tables, prefix, 4000)  # longer than its table: clamped
    assert reported and np.isfinite(got).all()
    got, reported = run(tables, prefix, -4)
    assert reported and np.isfinite(got).all()
    # pages that are bad but not needed are not looked at
    changed = prefix.copy()
    changed[0, 2] = -1
    assert not run(tables, changed, 32)[1]


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("per,queries", [(2, 1), (40, 1), (3, 40)])
def test_attention_of_bad_pages_and_lengths_is_what_the_header_says(ctx, dev, per, queries, precision):
    """A bad page's keys and values are zeros and count, a length outside its table is clamped: against the oracle on
    such a cache, within the roundings of the type."""
    rng = np.random.default_rng(60 + per)
    heads, kv_heads, dim, page, own, shared = 8, 2, 128, 16, 5, 3
    lens = rng.integers(queries, own * page + 1, per).astype(np.int32)
    lens[0] = own * page
    tables, pages = split_pages(rng, [own] * per + [shared])
    tables, prefix = tables[:-1].copy(), tables[-1:, :shared].copy()
    k, v = (values(rng, (1, pages, kv_heads, page, dim), precision) for _ in range(2))
    q = values(rng, (per * queries, heads, dim), precision, 1.5)
    dev.put("k", k, precision), dev.put("v", v, precision), dev.put("q", q, precision)
    kv = ec.PagedKv(dev.buffers["k"], dev.buffers["v"], 1, pages, page, kv_heads, dim, precision)

    def agrees(tables, prefix, lens, prefix_len, zeroed, lens_held, prefix_held):
        d = Device(ctx)
        batch = ec.PagedBatch(per, queries, d.put("t", tables), own, d.put("n", lens.astype(np.int32)), None, 1, d.put("p", prefix), shared,
                              d.put("l", np.array([prefix_len], np.int32)))
        size = ctx.prefix_attention_workspace(kv, batch, heads)
        ctx.prefix_attention(kv, 0, batch, dev.buffers["q"], heads, d.put("out", q, precision), d.put("w", np.zeros(size, np.uint8)), size)
        with pytest.raises(ec.CudaError, match="status 41"):
            ctx.synchronize()
        got = d.get("out").astype(np.float64)
        d.free()
        k0, v0 = k.copy(), v.copy()
        k0[0, zeroed], v0[0, zeroed] = 0, 0
        ref = q.astype(np.float64)
        weight, spread = od.attention(k0, v0, 0, q, ref, good_tables, lens_held, [queries] * per, good_prefix, [prefix_held])
        e = (dim + 4) * U * spread[:, :, None]
        limit = weight * (2 * np.expm1(2 * e) + 16 * U + 2 * (int(max(lens_held)) + prefix_held + 16) * U)
        limit = limit + H * weight + H * (np.abs(ref) + limit + H * weight) if precision == ec.BF16 else limit + U * np.abs(ref)
        holds(got, ref, limit)

    good_tables, good_prefix = tables, prefix
    for bad in (-1, pages, 2 ** 31 - 1, -2 ** 31):
        at = int(rng.integers(0, own))
        changed = tables.copy()
        changed[0, at] = bad
        agrees(changed, prefix, lens, 40, [tables[0, at]], lens, 40)
        changed = prefix.copy()
        changed[0, 2] = bad
        agrees(tables, changed, lens, 40, [prefix[0, 2]], lens, 40)
    for prefix_len, held in ((4000, shared * page), (shared * page + 1, shared * page), (-4, 0), (-2 ** 31, 0)):
        agrees(tables, prefix, lens, prefix_len, [], lens, held)
    for length in (own * page + 1, 2 ** 31 - 1):
        changed = lens.copy()
        changed[0] = length
        agrees(tables, prefix, changed, 33, [], lens, 33)
    changed = lens.copy()
    changed[-1] = -3
    emptied = lens.copy()
    emptied[-1] = 0
    agrees(tables, prefix, changed, 33, [], emptied, 33)


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("groups,per,queries", [(2, 3, 1), (2, 50, 1), (2, 4, 40), (1, 300, 2)])
def test_attention_keeps_bad_values_to_their_own_rows(ctx, dev, groups, per, queries, precision):
    """NaN and infinities in one row's query reach that row alone, those in one sequence's tokens that sequence, those
    in a prefix its group: everything else has the same bits as before."""
    rng = np.random.default_rng(groups + per + queries)
    heads, kv_heads, dim, page, n = 8, 2, 128, 16, groups * per
    lens = rng.integers(queries, 90, n).astype(np.int32)
    holds(*attention_case(ctx, dev, rng, groups, per, queries, 300, 90, heads, kv_heads, dim, page, precision, lens=lens,
                          counts=np.full(n, queries), prefix_lens=rng.integers(200, 300, groups), poison=False))
    b, (layers, pages) = dev.buffers, dev.shapes["k"][0][:2]
    own, shared = dev.shapes["t"][0][1], dev.shapes["pt"][0][1]
    kv = ec.PagedKv(b["k"], b["v"], layers, pages, page, kv_heads, dim, precision)
    batch = ec.PagedBatch(n, queries, b["t"], own, b["n"], b["c"], groups, b["pt"], shared, b["pl"])

    def run(**changed):
        kept = {name: dev.raw(name).copy() for name in changed}
        for name, array in changed.items():
            b[name].upload(array)
        ctx.prefix_attention(kv, 0, batch, b["q"], heads, b["out"], b["work"], b["work"].nbytes)
        ctx.synchronize()
        for name, array in kept.items():
            b[name].upload(array)
        return dev.raw("out").reshape(n, queries, heads, dim).copy()

    good = run()
    tables, prefix = dev.raw("t"), dev.raw("pt")
    for value in (np.nan, np.inf, -np.inf):
        bits = np.float32(value).view(np.uint32) >> 16 if precision == ec.BF16 else np.float32(value)
        slot, head = int(rng.integers(0, n * queries)), int(rng.integers(0, heads))
        q = dev.raw("q").copy()
        q.reshape(-1, heads, dim)[slot, head] = bits
        got = run(q=q)
        same = np.ones(good.shape[:3], bool)
        same.reshape(-1, heads)[slot, head] = False
        assert np.array_equal(got[same], good[same])
        for name in ("k", "v"):
            sequence = int(rng.integers(0, n))
            pool = dev.raw(name).copy()
            pool[0, tables[sequence, 0], 1, 0] = bits
            got = run(**{name: pool})
            same = np.ones(good.shape[:3], bool)
            same[sequence, :, heads // 2:] = False
            assert np.array_equal(got[same], good[same])
            group = int(rng.integers(0, groups))
            pool = dev.raw(name).copy()
            pool[0, prefix[group, 1], 0, 3] = bits
            got = run(**{name: pool})
            same = np.ones(good.shape[:3], bool)
            same[group * per:(group + 1) * per, :, :heads // 2] = False
            assert np.array_equal(got[same], good[same])
    assert np.array_equal(run(), good)


def test_attention_past_32_bit_offsets(ctx, dev):
    """Pages whose elements lie beyond 2^32 in the cache."""
    rng = np.random.default_rng(13)
    heads, kv_heads, dim, page, pages = 8, 8, 128, 128, 36000  # 4.7e9 elements each of K and V
    page_elements = kv_heads * page * dim
    kb, vb = ctx.buffer(pages * page_elements * 2), ctx.buffer(pages * page_elements * 2)
    try:
        used = np.array([35999, 33001, 32768, 7], np.int32)
        k, v = (values(rng, (1, 4, kv_heads, page, dim), ec.BF16) for _ in range(2))
        for i, p in enumerate(used):
            for buffer, x in ((kb, k), (vb, v)):
                bits = np.ascontiguousarray(bf16_bits(x[0, i]))
                ec.check(ec.lib().ernie_cuda_upload(ctx.handle, buffer.ptr + int(p) * page_elements * 2, ec.ptr(bits), bits.nbytes))
        q = values(rng, (40, heads, dim), ec.BF16)
        tables = np.repeat(used[2:3, None], 40, 0)
        kv = ec.PagedKv(kb, vb, 1, pages, page, kv_heads, dim, ec.BF16)
        lens = np.full(40, 100, np.int32)
        batch = ec.PagedBatch(40, 1, dev.put("t", tables), 1, dev.put("n", lens), None, 1, dev.put("p", used[None, :2]), 2,
                              dev.put("l", np.array([200], np.int32)))
        size = ctx.prefix_attention_workspace(kv, batch, heads)
        ctx.prefix_attention(kv, 0, batch, dev.put("q", q, ec.BF16), heads, dev.put("out", q, ec.BF16),
                             dev.put("w", np.zeros(size, np.uint8)), size)
        ctx.synchronize()
        ref = q.astype(np.float64)
        weight, _ = od.attention(k, v, 0, q, ref, np.full((40, 1), 2), lens, [1] * 40, [[0, 1]], [200])
        assert (np.abs(dev.get("out") - ref) <= H * weight * 1.1 + H * np.abs(ref) * 1.1 + 1e-4).all()
        # and stores there: one token into the last page, two copied pages by a reorder
        x = values(rng, (1, 3 * heads * dim), ec.BF16)
        one, zero = np.ones((1, dim), np.float32), np.zeros((1, dim), np.float32)
        batch = ec.PagedBatch(1, 1, dev.put("t1", used[None, :1]), 1, dev.put("n1", np.array([1], np.int32)))
        ctx.paged_append(kv, 0, batch, dev.put("x", x, ec.BF16), ec.BF16, 3 * heads * dim, heads, dev.put("one", one),
                         dev.put("zero", zero), 1, dev.put("qo", np.zeros((1, heads, dim)), ec.BF16))
        t2, n2 = np.array([[35999], [34000]], np.int32), np.array([100, 3], np.int32)
        ctx.beam_reorder(kv, 1, 2, dev.put("par", np.array([0, 0], np.int32)), dev.put("t2", t2), 1, dev.put("n2", n2),
                         dev.put("t3", t2 * 0), dev.put("n3", n2 * 0))
        ctx.synchronize()
        assert dev.raw("t3").tolist() == [[35999], [34000]] and dev.raw("n3").tolist() == [100, 100]
        for buffer, full, new in ((kb, k, x[0, heads * dim:2 * heads * dim]), (vb, v, x[0, 2 * heads * dim:])):
            got = np.empty((kv_heads, page, dim), np.uint16)
            ec.check(ec.lib().ernie_cuda_download(ctx.handle, ec.ptr(got), buffer.ptr + 34000 * page_elements * 2, got.nbytes))
            want = full[0, 0].copy()
            want[:, 0] = new.reshape(heads, dim)
            assert np.array_equal(got[:, :100], bf16_bits(want)[:, :100])
    finally:
        ctx.synchronize()
        kb.free()
        vb.free()


# ------------------------------------------------------------------ selection
def run_select(ctx, dev, logits, scores, finished, end, precision, pad=0, offset=0, alias=False):
    groups, beams, vocab = logits.shape
    wide = np.full((groups * beams, vocab + pad), np.float32(1e30))  # what lies past a row would win
    wide[:, :vocab] = logits.reshape(-1, vocab)
    if precision == ec.BF16:  # the values are exact in BF16: truncation keeps them, infinities and NaN too
        wide = (np.ascontiguousarray(wide, np.float32).view(np.uint32) >> 16).astype(np.uint16)
    size = ctx.beam_select_workspace(groups, beams, vocab)
    s, f = dev.put("s", scores.astype(np.float32)), dev.put("f", finished.astype(np.int32))
    zero = np.full((groups, beams), 77, np.int32)
    ns = s if alias else dev.put("ns", zero.astype(np.float32))
    nf = f if alias else dev.put("nf", zero)
    ctx.beam_select(dev.put("x", wide, None, offset), precision, vocab + pad, groups, beams, vocab, end, s, f,
                    dev.put("p", zero), dev.put("t", zero), ns, nf, dev.put("w", np.full(size, 0xFF, np.uint8)), size)
    ctx.synchronize()
    return dev.raw("p"), dev.raw("t"), dev.raw("s" if alias else "ns"), dev.raw("f" if alias else "nf")


def same_selection(got, logits, scores, finished, end, gap_needed=True):
    parents, tokens, totals, ended, gap = od.select(logits, scores, finished, end)
    if gap_needed:
        assert gap > 2e-5, "the inputs leave the order to roundings"
    assert np.array_equal(got[0], parents) and np.array_equal(got[1], tokens) and np.array_equal(got[3], ended)
    fine = np.isfinite(totals)
    assert np.array_equal(np.isfinite(got[2]), fine)
    limit = 101 * U + U * np.abs(totals[fine])
    assert (np.abs(got[2][fine] - totals[fine]) <= limit).all()


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("groups,beams,vocab,pad,offset", [
    (1, 1, 1, 0, 0), (1, 4, 3, 0, 0), (2, 3, 17, 1, 2), (3, 5, 1000, 0, 0), (2, 8, 5003, 5, 6), (1, 32, 40, 0, 0),
    (4, 2, 2049, 3, 0), (2, 32, 20011, 1, 2), (1, 5, 131072, 0, 0), (40, 8, 9000, 8, 0), (1, 2, 300001, 0, 4)])
def test_select(ctx, dev, groups, beams, vocab, pad, offset, precision):
    rng = np.random.default_rng(groups + beams + vocab)
    logits = values(rng, (groups, beams, vocab), precision, 3.0)
    logits[rng.random(logits.shape) < 0.05] = -np.inf
    scores = rng.standard_normal((groups, beams)).astype(np.float32) * 2 - 10
    finished = (rng.random((groups, beams)) < 0.2).astype(np.int32)
    offset = offset if precision == ec.BF16 else offset * 2
    end = int(np.argmax(logits[0, 0])) if vocab > 1 else -1  # an end token that is chosen
    got = run_select(ctx, dev, logits, scores, finished, end, precision, pad, offset)
    same_selection(got, logits, scores, finished, end)


@pytest.mark.parametrize("vocab", [31, 5000, 70000])
def test_select_of_equal_logits(ctx, dev, vocab):
    """Ties go to the lowest token, over the beams to the lowest beam; whole rows of one value."""
    beams = 6
    logits = np.zeros((2, beams, vocab), np.float32)
    logits[1, :, vocab // 2:] = 1.0
    logits[1, 3, ::7] = 1.0
    scores = np.zeros((2, beams), np.float32)
    got = run_select(ctx, dev, logits, scores, scores, -1, ec.FP32)
    same_selection(got, logits, scores, scores, -1, gap_needed=False)
    assert (got[0][0] == 0).all() and got[1][0].tolist() == list(range(beams))
    for beam in (0, 3):
        one = np.full((1, beams), -np.inf, np.float32)
        one[0, beam] = -1.0
        got = run_select(ctx, dev, logits[1:], one, scores[:1], -1, ec.FP32)
        same_selection(got, logits[1:], one, scores[:1], -1)


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
def test_select_order_of_a_sorted_vocabulary(ctx, dev, precision):
    """Logits in rising and in falling order, and the largest ones all in one thread's stretch."""
    vocab, beams = 20000, 16
    rise = values(np.random.default_rng(1), (vocab,), precision, 3.0)
    rise.sort()
    lumped = values(np.random.default_rng(2), (vocab,), precision)
    lumped[1024 * 8:1024 * 8 + 8] = np.arange(20, 28)
    lumped[np.arange(8) * 1024 + 4] = np.arange(20, 28)[::-1]
    for x in (rise, rise[::-1], lumped):
        logits = np.broadcast_to(x, (1, beams, vocab))
        scores = np.full((1, beams), -np.inf, np.float32)
        scores[0, 2] = 0.5
        got = run_select(ctx, dev, logits, scores, np.zeros((1, beams)), -1, precision)
        same_selection(got, logits, scores, np.zeros((1, beams)), -1)


def test_select_of_rows_that_offer_nothing(ctx, dev):
    """NaN, +inf, all -inf, scores that are not finite, finished beams; places left over."""
    rng = np.random.default_rng(5)
    logits = values(rng, (6, 4, 3000), ec.FP32, 3.0)
    scores = rng.standard_normal((6, 4)).astype(np.float32)
    finished = np.zeros((6, 4), np.int32)
    logits[0, 1, 2999] = np.nan
    logits[0, 2, 0] = np.inf
    logits[1] = -np.inf                      # nobody: every place is left over
    logits[2, :, 1:] = -np.inf               # one token each
    logits[3, :3] = -np.inf
    logits[3, 3, 2:] = -np.inf               # two continuations for four places
    finished[4] = 1                          # everybody has finished
    scores[4, 2] = -np.inf
    scores[5] = [np.nan, np.inf, -np.inf, -1.0]
    for alias in (False, True):
        got = run_select(ctx, dev, logits, scores, finished, 7, ec.FP32, alias=alias)
        same_selection(got, logits, scores, finished, 7)
    assert (got[0][1] == -1).all() and (got[1][1] == -1).all() and (got[3][1] == 1).all() and np.isneginf(got[2][1]).all()


@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("vocab", [700, 30011])
def test_select_of_masked_rows_and_extreme_logits(ctx, dev, vocab, precision):
    """Masks of the type's lowest value over nearly all of a row or the whole of it, and logits so large that
    neighbouring ones lie far apart: the sums of exponentials hold relative to the row's largest logit."""
    rng = np.random.default_rng(vocab)
    lowest = -3.3895313892515355e38 if precision == ec.BF16 else float(np.finfo(np.float32).min)
    beams = 4
    logits = values(rng, (10, beams, vocab), precision, 3.0)
    logits[0] = np.where(np.arange(vocab) == 333, logits[0], np.float32(lowest))  # one token left
    logits[1, :, 5:] = lowest                                                     # five left, in one lane's stretch
    logits[2] = lowest                                                            # none: all are equally good
    logits[3] = np.where(rng.random((beams, vocab)) < 0.99, np.float32(lowest), logits[3])
    for group, middle in ((4, 1e6), (5, -1e6), (6, 3e9), (7, -3e9), (8, 1e38), (9, -1e38)):
        logits[group] = middle
        logits[group, :, 11:vocab:97] = middle * (1 + 2.0 ** -5 * np.sign(middle))  # exact multiples apart
    logits = o.bf16_to_f32(bf16_bits(logits).reshape(-1)).reshape(logits.shape) if precision == ec.BF16 else logits
    scores = (-1.0 - 0.37 * np.arange(beams, dtype=np.float32))[None].repeat(10, 0)
    # one beam at a time, so that no order hangs on how different rows round
    for beam in range(beams):
        one = np.where(np.arange(beams) == beam, scores, np.float32(-np.inf))
        got = run_select(ctx, dev, logits, one, np.zeros((10, beams)), -1, precision, pad=3)
        same_selection(got, logits, one, np.zeros((10, beams)), -1)
        assert (got[0] == beam).all()


def test_select_first_step_of_identical_beams(ctx, dev):
    """All beams alike but one score: the best continuations of that beam; a bad logit elsewhere in the row wins nothing."""
    rng = np.random.default_rng(6)
    row = values(rng, (131072,), ec.FP32, 3.0)
    row[100:200] = np.finfo(np.float32).min
    logits = np.broadcast_to(row, (2, 8, 131072))
    scores = np.full((2, 8), -np.inf, np.float32)
    scores[:, 0] = 0.0
    got = run_select(ctx, dev, logits, scores, np.zeros((2, 8)), -1, ec.FP32)
    same_selection(got, logits, scores, np.zeros((2, 8)), -1)


# ------------------------------------------------------------------ reordering
@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("layers,groups,beams,page,kv_heads,dim,most", [
    (1, 1, 1, 16, 8, 128, 20), (3, 2, 2, 8, 1, 64, 30), (26, 1, 5, 16, 8, 128, 60), (2, 5, 4, 32, 3, 64, 70),
    (1, 3, 32, 8, 2, 64, 20), (2, 1, 8, 128, 4, 128, 300), (1, 300, 2, 8, 1, 64, 9)])
def test_reorder(ctx, dev, layers, groups, beams, page, kv_heads, dim, most, precision):
    rng = np.random.default_rng(layers + groups + beams)
    n, per_row = groups * beams, -(-most // page)
    for kind in ("random", "identity", "one", "none", "swap"):
        lens = rng.integers(0, most + 1, n).astype(np.int32)
        tables, pages = split_pages(rng, [per_row] * n)
        parents = {"random": rng.integers(-1, beams, (groups, beams)),
                   "identity": np.broadcast_to(np.arange(beams), (groups, beams)),
                   "one": np.full((groups, beams), beams - 1), "none": np.full((groups, beams), -1),
                   "swap": np.broadcast_to(np.arange(beams)[::-1], (groups, beams))}[kind].astype(np.int32)
        k, v = (values(rng, (layers, pages, kv_heads, page, dim), precision) for _ in range(2))
        d = Device(ctx)
        kv = ec.PagedKv(d.put("k", k, precision), d.put("v", v, precision), layers, pages, page, kv_heads, dim, precision)
        ctx.beam_reorder(kv, groups, beams, d.put("p", parents), d.put("t", tables), per_row, d.put("n", lens),
                         d.put("nt", tables * 0 - 3), d.put("nn", lens * 0 - 3))
        ctx.synchronize()
        new_tables, new_lens = od.reorder(k, v, parents, tables, lens)
        assert np.array_equal(d.raw("nt"), new_tables) and np.array_equal(d.raw("nn"), new_lens), kind
        assert np.array_equal(d.get("k"), k) and np.array_equal(d.get("v"), v), kind
        assert np.array_equal(d.raw("t"), tables) and np.array_equal(d.raw("n"), lens)
        d.free()


def test_reorder_range_reports(ctx, dev):
    """Bad parents count as none; bad pages are neither read nor written."""
    rng = np.random.default_rng(7)
    k, v = (values(rng, (1, 8, 1, 8, 64), ec.FP32) for _ in range(2))
    kv = ec.PagedKv(dev.put("k", k), dev.put("v", v), 1, 8, 8, 1, 64, ec.FP32)
    lens = np.array([9, 5, 7, 3], np.int32)
    for parents, tables in (([[0, 4, 1, -2]], [[0, 1], [2, 3], [4, 5], [6, 7]]),
                            ([[0, 0, 2, 3]], [[0, 1], [-1, 8], [4, 5], [6, 7]]),
                            ([[0, 0, 2, 3]], [[0, -9], [2, 3], [4, 5], [6, 7]])):
        parents, tables = np.array(parents, np.int32), np.array(tables, np.int32)
        d = Device(ctx)
        ctx.beam_reorder(kv, 1, 4, d.put("p", parents), d.put("t", tables), 2, d.put("n", lens), d.put("nt", tables * 0),
                         d.put("nn", lens * 0))
        with pytest.raises(ec.CudaError, match="status 41"):
            ctx.synchronize()
        if parents[0, 1] == 4:
            assert d.raw("nn").tolist() == [9, 0, 5, 0] and d.raw("nt").tolist() == [[0, 1], [4, 5], [2, 3], [6, 7]]
            assert np.array_equal(dev.get("k"), k)
        d.free()
    # the third: page 0 was copied to page 2, the bad second page was not
    k[0, 2] = k[0, 0]
    assert np.array_equal(dev.get("k"), k)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("precision", [ec.BF16, ec.FP32], ids=["bf16", "fp32"])
def test_beam_search_of_a_small_decoder(ctx, dev, precision):
    """Twelve steps of beam search for two prompts: append, attend, select, reorder on the device against a search
    that keeps every beam's tokens and recomputes its attention from them in 64 bits."""
    rng = np.random.default_rng(21)
    groups, beams, heads, kv_heads, dim, page, vocab, steps, end = 2, 4, 4, 2, 64, 8, 400, 12, 3
    n, prompt = groups * beams, [21, 13]
    width = (heads + 2 * kv_heads) * dim
    table = values(rng, (vocab, width), ec.FP32)           # a token's projection
    head = (rng.standard_normal((heads * dim, vocab)) * 0.6).astype(np.float32)
    angle = np.arange(64)[:, None] * np.concatenate([10.0 ** -np.linspace(0, 3, dim // 2)] * 2)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    prompts = [rng.integers(4, vocab, p) for p in prompt]
    shared, own = -(-max(prompt) // page), -(-(steps + 1) // page)
    order = rng.permutation(groups * shared + n * own).astype(np.int32)
    prefix_tables, tables = order[:groups * shared].reshape(groups, shared), order[groups * shared:].reshape(n, own)
    zero = np.zeros((1, len(order), kv_heads, page, dim), np.float32)
    kv = ec.PagedKv(dev.put("k", zero, precision), dev.put("v", zero, precision), 1, len(order), page, kv_heads, dim, precision)
    dev.put("cos", cos), dev.put("sin", sin), dev.put("pt", prefix_tables), dev.put("pl", np.array(prompt, np.int32))
    dev.put("t0", tables), dev.put("t1", tables * 0), dev.put("n0", np.zeros(n, np.int32)), dev.put("n1", np.zeros(n, np.int32))
    # the prompts, each appended as one sequence in its group's prefix pages
    x = np.zeros((groups, max(prompt), width), np.float32)
    for g, p in enumerate(prompts):
        x[g, :len(p)] = table[p]
    counts = np.array(prompt, np.int32)
    batch = ec.PagedBatch(groups, max(prompt), dev.buffers["pt"], shared, dev.buffers["pl"], dev.put("pc", counts))
    ctx.paged_append(kv, 0, batch, dev.put("px", x), ec.FP32, width, heads, dev.buffers["cos"], dev.buffers["sin"], 64,
                     dev.put("pq", np.zeros((groups * max(prompt), heads, dim)), precision))
    scores = np.full((groups, beams), -np.inf, np.float32)
    scores[:, 0] = 0.0
    dev.put("s", scores), dev.put("f", np.zeros((groups, beams), np.int32)), dev.put("par", np.zeros((groups, beams), np.int32))
    dev.put("tok", np.zeros((groups, beams), np.int32)), dev.put("q", np.zeros((n, heads, dim)), precision)
    dev.put("out", np.zeros((n, heads, dim)), precision), dev.put("x", np.zeros((n, width), np.float32))
    dev.put("l", np.zeros((n, vocab), np.float32))
    size = max(ctx.beam_select_workspace(groups, beams, vocab), 16)
    dev.put("sw", np.zeros(size, np.uint8))
    # the search on the host: histories of tokens after the prompt
    current = np.full((groups, beams), 5)
    history = [[[5] for _ in range(beams)] for _ in range(groups)]
    score, finished = scores.astype(np.float64), np.zeros((groups, beams), np.int64)
    round_to = (lambda a: values_of(a, precision))

    def values_of(a, precision):
        a = np.asarray(a, np.float32)
        return o.bf16_to_f32(bf16_bits(a).reshape(-1)).reshape(a.shape) if precision == ec.BF16 else a

    def attend(tokens):
        """The last token's attention output over `tokens`, in 64 bits from values the cache would hold."""
        y = table[tokens].astype(np.float64).reshape(len(tokens), -1, dim)
        turned = np.stack([od.rotate(y[t, :heads + kv_heads], cos[t].astype(np.float64), sin[t].astype(np.float64))
                           for t in range(len(tokens))])
        q, keys = round_to(turned[-1, :heads]), round_to(turned[:, heads:]).astype(np.float64)
        held = round_to(y[:, heads + kv_heads:]).astype(np.float64)
        result = np.empty((heads, dim))
        for h in range(heads):
            s = keys[:, h // 2] @ q[h].astype(np.float64) / np.sqrt(dim)
            p = np.exp(s - s.max())
            result[h] = (p / p.sum()) @ held[:, h // 2]
        return result

    a, b = ("t0", "n0"), ("t1", "n1")
    for step in range(steps):
        lens = np.full(n, step + 1, np.int32)
        dev.buffers[a[1]].upload(lens)
        dev.buffers["x"].upload(table[current.reshape(-1)])
        batch = ec.PagedBatch(n, 1, dev.buffers[a[0]], own, dev.buffers[a[1]], None, groups, dev.buffers["pt"], shared,
                              dev.buffers["pl"])
        ctx.paged_append(kv, 0, batch, dev.buffers["x"], ec.FP32, width, heads, dev.buffers["cos"], dev.buffers["sin"], 64,
                         dev.buffers["q"])
        size = ctx.prefix_attention_workspace(kv, batch, heads)
        work = ctx.buffer(size)
        ctx.prefix_attention(kv, 0, batch, dev.buffers["q"], heads, dev.buffers["out"], work, size)
        ctx.synchronize()
        work.free()
        out = dev.get("out")
        want = np.stack([attend(np.concatenate([prompts[g], history[g][i]]).astype(int)) for g in range(groups) for i in range(beams)])
        assert np.abs(out - want).max() < (0.03 if precision == ec.BF16 else 2e-5), step
        logits = (out.reshape(n, -1) @ head).astype(np.float32)
        dev.buffers["l"].upload(logits)
        ctx.beam_select(dev.buffers["l"], ec.FP32, vocab, groups, beams, vocab, end, dev.buffers["s"], dev.buffers["f"],
                        dev.buffers["par"], dev.buffers["tok"], dev.buffers["s"], dev.buffers["f"], dev.buffers["sw"],
                        dev.buffers["sw"].nbytes)
        ctx.beam_reorder(kv, groups, beams, dev.buffers["par"], dev.buffers[a[0]], own, dev.buffers[a[1]],
                         dev.buffers[b[0]], dev.buffers[b[1]])
        ctx.synchronize()
        a, b = b, a
        before = dev.raw("s").copy()
        parents, tokens, totals, ended, gap = od.select(logits.reshape(groups, beams, vocab), score.astype(np.float32), finished, end)
        assert gap > 1e-5
        assert np.array_equal(dev.raw("par"), parents) and np.array_equal(dev.raw("tok"), tokens)
        assert np.array_equal(dev.raw("f"), ended)
        history = [[history[g][parents[g, i]] + [int(tokens[g, i])] for i in range(beams)] for g in range(groups)]
        current, score, finished = tokens, before.astype(np.float64), ended
        assert dev.raw(a[1]).tolist() == [step + 1] * n
    assert sorted(dev.raw(a[0]).ravel().tolist()) == sorted(tables.ravel().tolist())


def test_two_contexts_at_once(ctx, dev):
    """Two contexts' streams run the same operators side by side, each with its own scratch."""
    other = ec.Context(0)
    d2 = Device(other)
    try:
        rng = np.random.default_rng(31)
        calls = []
        for c, d in ((ctx, dev), (other, d2)):
            k, v = (values(rng, (1, 100, 2, 16, 128), ec.BF16) for _ in range(2))
            q = values(rng, (40, 8, 128), ec.BF16)
            kv = ec.PagedKv(d.put("k", k, ec.BF16), d.put("v", v, ec.BF16), 1, 100, 16, 2, 128, ec.BF16)
            tables, prefix = rng.permutation(100)[:40].reshape(40, 1).astype(np.int32), np.arange(50)[None].astype(np.int32)
            lens = np.full(40, 9, np.int32)
            batch = ec.PagedBatch(40, 1, d.put("t", tables), 1, d.put("n", lens), None, 1, d.put("p", prefix), 50,
                                  d.put("l", np.array([777], np.int32)))
            size = c.prefix_attention_workspace(kv, batch, 8)
            d.put("q", q, ec.BF16), d.put("out", q, ec.BF16), d.put("w", np.zeros(size, np.uint8))
            ref = q.astype(np.float64)
            weight, _ = od.attention(k, v, 0, q, ref, tables, lens, [1] * 40, prefix, [777])
            calls.append((c, kv, batch, d, size, ref, weight))
        for _ in range(30):
            for c, kv, batch, d, size, _, _ in calls:
                c.prefix_attention(kv, 0, batch, d.buffers["q"], 8, d.buffers["out"], d.buffers["w"], size)
        for c, _, _, d, _, ref, weight in calls:
            c.synchronize()
            assert (np.abs(d.get("out") - ref) <= H * weight * 1.1 + H * np.abs(ref) * 1.1 + 1e-4).all()
    finally:
        other.synchronize()
        d2.free()
        other.close()


# ------------------------------------------------------------------ beside other streams, and in graphs
class Step:
    """One step of a batch of beams on torch tensors: append, attend, select, reorder."""

    def __init__(self, ctx, torch, seed, workspace=None):
        rng = np.random.default_rng(seed)
        self.ctx, self.torch = ctx, torch
        self.groups, self.beams, self.heads, self.kv_heads, self.dim, self.page, self.vocab = 2, 6, 8, 2, 128, 16, 3000
        n, own, shared = self.groups * self.beams, 3, 20
        put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
        order = rng.permutation(n * own + self.groups * shared).astype(np.int32)
        shape = (1, len(order), self.kv_heads, self.page, self.dim)
        self.k, self.v = (put(values(rng, shape, ec.FP32)).bfloat16() for _ in range(2))
        self.tables, self.prefix = put(order[:n * own].reshape(n, own)), put(order[n * own:].reshape(self.groups, shared))
        self.lens, self.prefix_lens = put(rng.integers(1, 40, n).astype(np.int32)), put(np.array([320, 211], np.int32))
        angle = np.arange(400)[:, None] * np.concatenate([10.0 ** -np.linspace(0, 3, self.dim // 2)] * 2)
        self.cos, self.sin = put(np.cos(angle).astype(np.float32)), put(np.sin(angle).astype(np.float32))
        self.width = (self.heads + 2 * self.kv_heads) * self.dim
        self.x = put(values(rng, (n, self.width), ec.FP32))
        self.q = torch.zeros(n, self.heads, self.dim, device="cuda", dtype=torch.bfloat16)
        self.out = torch.zeros_like(self.q)
        self.logits = put(values(rng, (n, self.vocab), ec.FP32, 3.0))
        self.scores = put(-rng.random((self.groups, self.beams)).astype(np.float32))
        ints = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)
        self.finished, self.parents, self.tokens = (ints(self.groups, self.beams) for _ in range(3))
        self.new_finished, self.new_scores = ints(self.groups, self.beams), torch.zeros(self.groups, self.beams, device="cuda")
        self.new_tables, self.new_lens = ints(n, own), ints(n)
        self.kv = ec.PagedKv(self.k, self.v, 1, len(order), self.page, self.kv_heads, self.dim, ec.BF16)
        self.batch = ec.PagedBatch(n, 1, self.tables, own, self.lens, None, self.groups, self.prefix, shared, self.prefix_lens)
        size = max(ctx.prefix_attention_workspace(self.kv, self.batch, self.heads), ctx.beam_select_workspace(self.groups, self.beams, self.vocab))
        self.work = torch.zeros(size, device="cuda", dtype=torch.uint8) if workspace is None else workspace

    def run(self):
        c, w = self.ctx, self.work
        c.paged_append(self.kv, 0, self.batch, self.x, ec.FP32, self.width, self.heads, self.cos, self.sin, 400, self.q)
        c.prefix_attention(self.kv, 0, self.batch, self.q, self.heads, self.out, w, w.numel())
        c.beam_select(self.logits, ec.FP32, self.vocab, self.groups, self.beams, self.vocab, 7, self.scores, self.finished,
                      self.parents, self.tokens, self.new_scores, self.new_finished, w, w.numel())
        c.beam_reorder(self.kv, self.groups, self.beams, self.parents, self.tables, self.tables.shape[1], self.lens,
                       self.new_tables, self.new_lens)

    def results(self):
        return [t.clone() for t in (self.q, self.out, self.k, self.v, self.parents, self.tokens, self.new_scores, self.new_finished,
                                    self.new_tables, self.new_lens)]


def test_steps_ordered_with_another_stream(ctx):
    """A producer and a consumer on torch's stream, each step's inputs written late, without the host waiting anywhere."""
    torch = pytest.importorskip("torch")
    library = torch.cuda.ExternalStream(ctx.stream)
    steps = [Step(ctx, torch, seed) for seed in range(6)]
    torch.cuda.synchronize()
    want = []
    for s in steps:
        kept = [t.clone() for t in (s.k, s.v)]
        torch.cuda.synchronize()
        s.run()
        ctx.synchronize()
        want.append(s.results())
        for t, old in zip((s.k, s.v), kept):
            t.copy_(old)
        s.inputs = [t.clone() for t in (s.x, s.lens, s.logits)]
        for t in (s.x, s.logits):
            t.fill_(float("nan"))
        s.lens.zero_()
        for t in (s.q, s.out, s.parents, s.tokens, s.new_scores, s.new_finished, s.new_tables, s.new_lens):
            t.zero_()
    torch.cuda.synchronize()
    mine = torch.cuda.Stream()
    got = []
    with torch.cuda.stream(mine):
        for s in steps:
            torch.cuda._sleep(3_000_000)  # the inputs come a millisecond late
            for t, new in zip((s.x, s.lens, s.logits), s.inputs):
                t.copy_(new)
            library.wait_stream(mine)
            s.run()
            mine.wait_stream(library)
            got.append(s.results())
    mine.synchronize()
    ctx.synchronize()
    for one, other in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(one, other))


def test_steps_under_the_contexts_stream(ctx):
    """torch's work on the context's own stream needs no events."""
    torch = pytest.importorskip("torch")
    s = Step(ctx, torch, 40)
    kept = [t.clone() for t in (s.k, s.v, s.x, s.logits)]
    torch.cuda.synchronize()
    s.run()
    ctx.synchronize()
    want = s.results()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(ctx.stream)):
        torch.cuda._sleep(3_000_000)
        for t, old in zip((s.k, s.v, s.x, s.logits), kept):
            t.copy_(old)
        s.out.zero_()
        s.run()
        got = s.results()
    ctx.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_steps_in_graphs_that_share_a_workspace(ctx):
    """Two captured steps with one scratch, replayed in turn on one stream with lengths, logits and projections that change
    between the replays, against the same steps called eagerly."""
    torch = pytest.importorskip("torch")
    library = torch.cuda.ExternalStream(ctx.stream)
    first = Step(ctx, torch, 50)
    steps = [first, Step(ctx, torch, 51, first.work)]
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in steps]
    for s, graph in zip(steps, graphs):
        with torch.cuda.graph(graph, stream=library):
            s.run()
    ctx.synchronize()
    rng = np.random.default_rng(52)
    for turn in range(5):
        lens = torch.from_numpy(rng.integers(1, 48, 12).astype(np.int32)).cuda()
        for s, graph in zip(steps, graphs):
            s.lens.copy_(lens)
            s.x.mul_(-0.75)
            s.logits.copy_(s.logits.roll(turn + 1, 1))
        kept = [[t.clone() for t in (s.k, s.v)] for s in steps]
        torch.cuda.synchronize()
        for s in steps:
            s.run()
        ctx.synchronize()
        want = [s.results() for s in steps]
        for s, (k, v) in zip(steps, kept):
            s.k.copy_(k), s.v.copy_(v), s.out.zero_(), s.parents.zero_(), s.new_tables.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(library):
            for graph in graphs:
                graph.replay()
        ctx.synchronize()
        for s, result in zip(steps, want):
            assert all(torch.equal(a, b) for a, b in zip(s.results(), result)), turn
        torch.cuda.synchronize()
    del graphs


@pytest.mark.parametrize("copies", [False, True], ids=["after kernels", "after copies"])
def test_a_step_forked_off_another_streams_capture(ctx, copies):
    """A graph captured on torch's stream whose middle runs on the context's, ordered both ways by events."""
    torch = pytest.importorskip("torch")
    library, mine = torch.cuda.ExternalStream(ctx.stream), torch.cuda.Stream()
    s = Step(ctx, torch, 70)
    x, logits = s.x.clone(), s.logits.clone()
    kept, late, out = [t.clone() for t in (s.k, s.v)], s.lens.clone(), torch.empty_like(s.out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=mine):
        if copies:
            s.lens.copy_(late), s.x.copy_(x), s.logits.copy_(logits)
        else:
            torch.add(late, 0, out=s.lens), torch.mul(x, 1.0, out=s.x), torch.mul(logits, 1.0, out=s.logits)
        library.wait_stream(mine)
        s.run()
        mine.wait_stream(library)
        torch.mul(s.out, 2.0, out=out)
    for turn in range(4):
        late.copy_(late % 40 + 3)
        x.mul_(-1.25)
        for t in (s.lens, s.out, s.parents):
            t.zero_()
        s.x.fill_(float("nan"))
        for t, old in zip((s.k, s.v), kept):
            t.copy_(old)
        torch.cuda.synchronize()
        with torch.cuda.stream(mine):
            graph.replay()
        torch.cuda.synchronize()
        ctx.synchronize()
        got = s.results() + [out.clone()]
        for t, old in zip((s.k, s.v), kept):
            t.copy_(old)
        torch.cuda.synchronize()
        s.run()
        ctx.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, s.results() + [s.out * 2.0])), turn
    del graph
