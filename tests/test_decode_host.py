"""Batched decoding behind shared prefixes, without a GPU: the refusals of the C entry points (arguments are checked
before the context is looked at, so a call with good arguments and no context is refused for the context alone), and
the oracle's own definitions against direct ones."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import decode as od
import ernie_cuda as ec

# addresses that no call follows: every call here is refused on the host
K, V, TABLES, LENS, COUNTS = 1 << 40, 2 << 40, 3 << 40, 4 << 40, 5 << 40
PREFIX_TABLES, PREFIX_LENS, Q, OUT, WORK = 6 << 40, 7 << 40, 8 << 40, 9 << 40, 10 << 40
QKV, COS, SIN = 11 << 40, 12 << 40, 13 << 40


class NoContext:
    handle = None


for _name in ("paged_append", "prefix_attention_workspace", "prefix_attention", "beam_select_workspace", "beam_select",
              "beam_reorder"):
    setattr(NoContext, _name, getattr(ec.Context, _name))
CTX = NoContext()


def kv(**change):
    f = dict(k=K, v=V, layers=2, pages=40, page_size=16, kv_heads=8, head_dim=128, precision=ec.BF16)
    f.update(change)
    return ec.PagedKv(**f)


def batch(**change):
    f = dict(sequences=6, queries=2, tables=TABLES, max_pages=4, lens=LENS, counts=COUNTS, groups=2,
             prefix_tables=PREFIX_TABLES, max_prefix_pages=5, prefix_lens=PREFIX_LENS)
    f.update(change)
    return ec.PagedBatch(**f)


def append(kv=None, batch_=None, **change):
    f = dict(layer=0, qkv=QKV, precision=ec.FP32, ld=48 * 128, heads=32, cos=COS, sin=SIN, rope_rows=100, q_out=Q)
    f.update(change)
    return CTX.paged_append(kv or globals()["kv"](), f["layer"], batch_ or batch(), f["qkv"], f["precision"], f["ld"],
                            f["heads"], f["cos"], f["sin"], f["rope_rows"], f["q_out"])


def attend(kv=None, batch_=None, **change):
    f = dict(layer=1, q=Q, heads=32, out=OUT, workspace=WORK, workspace_bytes=1 << 30)
    f.update(change)
    return CTX.prefix_attention(kv or globals()["kv"](), f["layer"], batch_ or batch(), f["q"], f["heads"], f["out"],
                                f["workspace"], f["workspace_bytes"])


def select(**change):
    f = dict(logits=Q, precision=ec.FP32, ld=1000, groups=3, beams=4, vocab=1000, end_token=2, scores=K, finished=V,
             parents=TABLES, tokens=LENS, new_scores=COUNTS, new_finished=OUT, workspace=WORK, workspace_bytes=1 << 30)
    f.update(change)
    return CTX.beam_select(*f.values())


def reorder(kv=None, **change):
    f = dict(groups=3, beams=4, parents=Q, tables=TABLES, max_pages=4, lens=LENS, new_tables=OUT, new_lens=COUNTS)
    f.update(change)
    return CTX.beam_reorder(kv or globals()["kv"](), *f.values())


def refused(call, words):
    with pytest.raises(ec.CudaError, match=words):
        call()


def test_good_arguments_are_refused_for_the_context_alone():
    for call in (append, attend, select, reorder):
        refused(call, "null context")
    refused(lambda: CTX.prefix_attention_workspace(kv(), batch(), 32), "null context")
    refused(lambda: CTX.beam_select_workspace(3, 4, 1000), "null context")
    refused(lambda: attend(batch_=batch(counts=None, groups=1, prefix_tables=None, max_prefix_pages=0, prefix_lens=None)),
            "null context")


@pytest.mark.parametrize("change,words", [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(precision=2), "precision"), (dict(page_size=4), "Page size"),
    (dict(page_size=24), "Page size"), (dict(page_size=256), "Page size"), (dict(page_size=0), "Page size"),
    (dict(page_size=-16), "Page size"), (dict(head_dim=96), "Head dimension"), (dict(head_dim=256), "Head dimension"),
    (dict(layers=0), "cache shape"), (dict(pages=0), "cache shape"), (dict(kv_heads=0), "cache shape"),
    (dict(kv_heads=-8), "cache shape"), (dict(pages=1 << 24), "cache shape"), (dict(pages=2 ** 31 - 1), "cache shape"),
    (dict(k=K + 8), "16-byte"), (dict(v=V + 2), "16-byte"), (dict(v=K + 4096), "overlap")])
def test_cache_refusals(change, words):
    for call in (append, attend, reorder):
        refused(lambda: call(kv(**change)), words)


@pytest.mark.parametrize("change,words", [
    (dict(tables=None), "null"), (dict(lens=None), "null"), (dict(sequences=0), "batch shape"),
    (dict(sequences=-6), "batch shape"), (dict(queries=0), "batch shape"), (dict(queries=1 << 23), "batch shape"),
    (dict(max_pages=0), "batch shape"), (dict(max_prefix_pages=-1), "batch shape"), (dict(groups=0), "groups"),
    (dict(groups=4), "groups"), (dict(groups=12), "groups"), (dict(prefix_tables=None), "prefix"),
    (dict(prefix_lens=None), "prefix"), (dict(max_prefix_pages=0), "prefix"), (dict(tables=TABLES + 2), "4-byte"),
    (dict(lens=LENS + 1), "4-byte"), (dict(counts=COUNTS + 3), "4-byte"), (dict(prefix_lens=PREFIX_LENS + 2), "4-byte"),
    (dict(max_pages=1 << 27), "2\\^31"), (dict(max_prefix_pages=1 << 30), "2\\^31")])
def test_batch_refusals(change, words):
    for call in (append, attend):
        refused(lambda: call(batch_=batch(**change)), words)


def test_layer_and_head_refusals():
    for call in (append, attend):
        for layer in (-1, 2):
            refused(lambda: call(layer=layer), "Layer")
        for heads in (0, -8, 12, 2048):
            refused(lambda: call(heads=heads), "query heads")


@pytest.mark.parametrize("change,words", [
    (dict(qkv=None), "null"), (dict(cos=None), "null"), (dict(sin=None), "null"), (dict(q_out=None), "null"),
    (dict(precision=-1), "precision"), (dict(ld=48 * 128 - 1), "row stride"), (dict(ld=1 << 31), "row stride"),
    (dict(rope_rows=0), "positions"), (dict(qkv=QKV + 2), "aligned"), (dict(cos=COS + 4), "aligned"),
    (dict(q_out=Q + 8), "aligned"), (dict(q_out=QKV + 48 * 128 * 4 * 11), "overlap")])
def test_append_refusals(change, words):
    refused(lambda: append(**change), words)


@pytest.mark.parametrize("change,words", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(workspace=None), "null"), (dict(q=Q + 2), "16-byte"),
    (dict(out=OUT + 4), "16-byte"), (dict(workspace=WORK + 8), "16-byte"), (dict(out=Q), "overlap"),
    (dict(out=Q + 12 * 32 * 128 * 2 - 16), "overlap"), (dict(workspace=OUT + 16), "overlap"),
    (dict(workspace=Q - 16), "overlap")])
def test_attention_refusals(change, words):
    refused(lambda: attend(**change), words)


@pytest.mark.parametrize("change,words", [
    (dict(beams=0), "Beam search"), (dict(beams=33), "Beam search"), (dict(groups=0), "Beam search"),
    (dict(vocab=0), "Beam search"), (dict(groups=1 << 23), "Too many"), (dict(precision=3), "precision"),
    (dict(logits=None), "null"), (dict(scores=None), "null"), (dict(finished=None), "null"), (dict(parents=None), "null"),
    (dict(tokens=None), "null"), (dict(new_scores=None), "null"), (dict(new_finished=None), "null"),
    (dict(workspace=None), "null"), (dict(ld=999), "row stride"), (dict(end_token=1000), "end token"),
    (dict(logits=Q + 2), "aligned"), (dict(tokens=LENS + 2), "aligned"), (dict(workspace=WORK + 4), "aligned")])
def test_select_refusals(change, words):
    refused(lambda: select(**change), words)


@pytest.mark.parametrize("change,words", [
    (dict(parents=None), "null"), (dict(tables=None), "null"), (dict(lens=None), "null"), (dict(new_tables=None), "null"),
    (dict(new_lens=None), "null"), (dict(beams=33), "Beam search"), (dict(groups=-1), "Beam search"),
    (dict(max_pages=0), "table width"), (dict(max_pages=1 << 28), "table width"), (dict(tables=TABLES + 1), "4-byte"),
    (dict(new_tables=TABLES), "overlap"), (dict(new_tables=TABLES + 12 * 16 - 4), "overlap"), (dict(new_lens=LENS), "overlap"),
    (dict(new_lens=OUT + 4), "overlap"), (dict(new_tables=Q), "overlap")])
def test_reorder_refusals(change, words):
    refused(lambda: reorder(**change), words)


def test_results_inside_the_cache_are_refused():
    pool = 2 * 40 * 8 * 16 * 128 * 2  # bytes of K, and of V
    for at in (K, V + 16, K + pool - 16, V + pool - 16):
        refused(lambda: append(q_out=at), "overlaps the paged cache")
        refused(lambda: attend(out=at), "overlaps the paged cache")
        refused(lambda: attend(workspace=at), "overlaps the paged cache")
        refused(lambda: reorder(new_tables=at), "overlaps the paged cache")
        refused(lambda: reorder(new_lens=at), "overlaps the paged cache")
    for at in (K + pool, V + pool):
        refused(lambda: append(q_out=at), "null context")
        refused(lambda: attend(out=at), "null context")


@pytest.mark.parametrize("change", [
    dict(tokens=TABLES + 44), dict(new_scores=TABLES), dict(new_finished=COUNTS + 8), dict(workspace=OUT),
    dict(parents=WORK + 4096), dict(new_scores=K + 4), dict(new_finished=V - 4), dict(new_scores=V), dict(tokens=K),
    dict(tokens=Q + 4 * 11999), dict(workspace=Q - 16)])
def test_select_overlaps_are_refused(change):
    refused(lambda: select(**change), "overlap")


def test_select_takes_the_new_state_in_place():
    refused(lambda: select(new_scores=K, new_finished=V), "null context")
    refused(lambda: select(tokens=Q + 4 * 12000), "null context")


def test_batches_past_the_counters_are_refused():
    for call in (attend, lambda **c: CTX.prefix_attention_workspace(kv(), c["batch_"], c.get("heads", 32))):
        refused(lambda: call(batch_=batch(sequences=1 << 20, queries=4, groups=1), heads=1024), "query rows")
        refused(lambda: call(batch_=batch(sequences=1 << 16, queries=1, max_pages=1 << 16)), "too many tokens")
        refused(lambda: call(batch_=batch(sequences=1 << 10, queries=1, groups=1 << 10, max_prefix_pages=1 << 18)),
                "too many tokens")
    refused(lambda: attend(kv(layers=65537)), "cache shape")
    refused(lambda: reorder(beams=32, max_pages=1 << 26), "table width")


def test_counts_whose_last_step_passes_32_bits_are_refused():
    """Indices step past their end by a tile of keys or a CTA's threads, which may not wrap around."""
    last = 2 ** 31 - 1
    refused(lambda: select(vocab=last, ld=last), "vocabulary of 2\\^31")
    refused(lambda: CTX.beam_select_workspace(1, 1, last - 1023), "vocabulary of 2\\^31")
    refused(lambda: CTX.beam_select_workspace(1, 1, last - 1024), "null context")
    for page, beams, pages in ((8, 8, 2 ** 28 - 1), (8, 1, 2 ** 28 - 1), (128, 1, 2 ** 24 - 1)):
        refused(lambda: reorder(kv(page_size=page, pages=4), groups=1, beams=beams, max_pages=pages, new_tables=1 << 50), "table width")
    # 2^31 - 2048 tokens
    refused(lambda: reorder(kv(page_size=128, pages=4), groups=1, beams=1, max_pages=2 ** 24 - 16, new_tables=1 << 50), "null context")
    alone = dict(prefix_tables=None, max_prefix_pages=0, prefix_lens=None, groups=1, sequences=1, queries=1)
    for call in (append, attend):
        refused(lambda: call(batch_=batch(max_pages=2 ** 27 - 1, **alone)), "2\\^31")
        refused(lambda: call(batch_=batch(max_pages=2 ** 27 - 64, **alone)), "2\\^31")
        refused(lambda: call(kv(kv_heads=1), batch(max_pages=2 ** 27 - 128, **alone)), "null context")
        refused(lambda: call(batch_=batch(max_pages=2 ** 26, max_prefix_pages=2 ** 26 - 1)), "2\\^31")
    refused(lambda: attend(batch_=batch(sequences=(1 << 21) - 1, queries=1, groups=1), heads=1024), "query rows")


def test_arrays_on_the_host_and_wide_integers_are_refused():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="device memory"):
        append(q_out=torch.zeros(4))
    with pytest.raises(ValueError, match="32-bit"):
        batch(lens=torch.zeros(6, dtype=torch.int64))
    with pytest.raises(ValueError, match="32-bit"):
        batch(tables=torch.zeros(4, 6, dtype=torch.int32).t())


class OnDevice:
    """Stands for a torch tensor in device memory: its kind, shape and strides, at an address that no call follows."""

    def __init__(self, torch, address, *shape, dtype="int32", device=0, stride=None):
        self.address, self.device_index, self.is_cuda = address, device, True
        self.meta = torch.empty(shape, dtype=getattr(torch, dtype), device="meta")
        if stride:
            self.meta = torch.empty_strided(shape, stride, dtype=getattr(torch, dtype), device="meta")

    def data_ptr(self):
        return self.address

    def get_device(self):
        return self.device_index

    def __getattr__(self, name):
        return getattr(self.meta, name)


class FirstDevice(NoContext):
    device = 0


def test_tensors_of_the_right_kind_pass_and_others_are_refused():
    """Every array of every call: another type, too few elements, gaps between them, another device."""
    torch = pytest.importorskip("torch")
    first = FirstDevice()
    n, q, h, k, d = 6, 2, 32, 8, 128
    pool = (2, 40, k, 16, d)
    good = dict(
        cache=dict(k=(K, pool, "bfloat16"), v=(V, pool, "bfloat16")),
        batch=dict(tables=(TABLES, (n, 4), "int32"), lens=(LENS, (n,), "int32"), counts=(COUNTS, (n,), "int32"),
                   prefix_tables=(PREFIX_TABLES, (2, 5), "int32"), prefix_lens=(PREFIX_LENS, (2,), "int32")),
        append=dict(qkv=(QKV, (n * q, (h + 2 * k) * d), "float32"), cos=(COS, (100, d), "float32"), sin=(SIN, (100, d), "float32"),
                    q_out=(Q, (n * q, h, d), "bfloat16")),
        attend=dict(q=(Q, (n, q, h, d), "bfloat16"), out=(OUT, (n * q, h * d), "bfloat16"), workspace=(WORK, (1 << 20,), "uint8")),
        select=dict(logits=(Q, (3, 4, 1000), "float32"), scores=(K, (3, 4), "float32"), finished=(V, (3, 4), "int32"),
                    parents=(TABLES, (3, 4), "int32"), tokens=(LENS, (12,), "int32"), new_scores=(COUNTS, (3, 4), "float32"),
                    new_finished=(OUT, (3, 4), "int32"), workspace=(WORK, (1 << 20,), "uint8")),
        reorder=dict(parents=(Q, (3, 4), "int32"), tables=(TABLES, (12, 4), "int32"), lens=(LENS, (12,), "int32"),
                     new_tables=(OUT, (12, 4), "int32"), new_lens=(COUNTS, (12,), "int32")))

    def call(where=None, name=None, change=None):
        arrays = {}
        for part, fields in good.items():
            arrays[part] = {f: OnDevice(torch, at, *shape, dtype=dtype) for f, (at, shape, dtype) in fields.items()}
        if where:
            arrays[where][name] = change(*good[where][name])
        cache, rows = kv(**arrays["cache"]), batch(**arrays["batch"])
        a, t, s, r = arrays["append"], arrays["attend"], arrays["select"], arrays["reorder"]
        return (
            lambda: first.paged_append(cache, 0, rows, a["qkv"], ec.FP32, 48 * d, h, a["cos"], a["sin"], 100, a["q_out"]),
            lambda: first.prefix_attention(cache, 1, rows, t["q"], h, t["out"], t["workspace"], 1 << 20),
            lambda: first.beam_select(s["logits"], ec.FP32, 1000, 3, 4, 1000, 2, *[s[x] for x in list(s)[1:]], 1 << 20),
            lambda: first.beam_reorder(cache, 3, 4, r["parents"], r["tables"], 4, r["lens"], r["new_tables"], r["new_lens"]))

    for one in call():
        refused(one, "null context")
    changes = dict(
        kind=lambda at, shape, dtype: OnDevice(torch, at, *shape, dtype={"int32": "bool", "float32": "bfloat16", "bfloat16": "float16",
                                                                        "uint8": "uint8"}[dtype]),
        wide=lambda at, shape, dtype: OnDevice(torch, at, *shape, dtype={"int32": "int64"}.get(dtype, "float64" if dtype != "uint8" else "uint8")),
        same_size=lambda at, shape, dtype: OnDevice(torch, at, *shape, dtype={"int32": "float32", "float32": "int32"}.get(dtype, "int16" if dtype != "uint8" else "uint8")),
        short=lambda at, shape, dtype: OnDevice(torch, at, *(shape[:-1] + (shape[-1] - 1,)), dtype=dtype),
        gaps=lambda at, shape, dtype: OnDevice(torch, at, *shape, dtype=dtype,
                                               stride=tuple(2 * x for x in torch.empty(shape, device="meta").stride())),
        spread=lambda at, shape, dtype: OnDevice(torch, at, *shape, dtype=dtype, stride=(0,) * len(shape)),
        elsewhere=lambda at, shape, dtype: OnDevice(torch, at, *shape, dtype=dtype, device=1),
        host=lambda at, shape, dtype: torch.zeros((), dtype=getattr(torch, dtype)).expand(shape))
    order = ("append", "attend", "select", "reorder")
    for where, fields in good.items():
        for name, (_, _, dtype) in fields.items():
            for change, make in changes.items():
                if dtype == "uint8" and change in ("kind", "wide", "same_size"):
                    continue
                with pytest.raises(ValueError, match=name if where in order else "arrays on different devices|the cache or the batch|" + name):
                    calls = call(where, name, make)
                    calls[order.index(where) if where in order else 0]()


def test_rows_of_wider_tensors_and_buffers():
    torch = pytest.importorskip("torch")
    first, wide = FirstDevice(), 48 * 128 + 64
    rows = lambda stride, width=48 * 128, count=12, dtype="float32": OnDevice(torch, QKV, count, width, dtype=dtype, stride=(stride, 1))
    go = lambda qkv, ld=wide: first.paged_append(kv(), 0, batch(), qkv, ec.FP32, ld, 32, COS, SIN, 100, Q)
    refused(lambda: go(rows(wide)), "null context")
    refused(lambda: go(OnDevice(torch, QKV, 6, 2, wide, dtype="float32")), "null context")
    # the sequences' slots as a dimension of their own, one slot or one row of a wider tensor
    view = lambda *shape, stride: OnDevice(torch, QKV, *shape, dtype="float32", stride=stride)
    refused(lambda: go(view(6, 2, 48 * 128, stride=(2 * wide, wide, 1))), "null context")
    refused(lambda: go(view(12, 1, 48 * 128, stride=(wide, 5, 1))), "null context")
    for bad in (view(6, 2, 48 * 128, stride=(3 * wide, wide, 1)), view(6, 2, 48 * 128, stride=(wide, 6 * wide, 1)),
                view(3, 2, 48 * 128, stride=(2 * wide, wide, 1)), view(12, 48 * 128, stride=(wide, 2)), view(12, 48 * 128, stride=(0, 1))):
        with pytest.raises(ValueError, match="qkv"):
            go(bad)
    for bad in (rows(wide + 1), rows(wide, 48 * 128 - 1), rows(wide, count=11), rows(wide, dtype="bfloat16")):
        with pytest.raises(ValueError, match="qkv"):
            go(bad)
    held = ec.Buffer.__new__(ec.Buffer)
    held.ctx, held.ptr, held.nbytes = first, Q, 12 * 32 * 128 * 2
    attended = lambda: first.prefix_attention(kv(), 1, batch(), held, 32, OUT, WORK, 1 << 20)
    refused(attended, "null context")
    held.nbytes -= 1
    with pytest.raises(ValueError, match="q: "):
        attended()


def test_the_stream_needs_a_context():
    out = ctypes.c_void_p(5)
    assert ec.lib().ernie_cuda_context_stream(None, ctypes.byref(out)) == ec.ERROR and out.value == 5


def test_null_descriptions():
    lib = ec.lib()
    n = ctypes.c_size_t(7)
    assert lib.ernie_cuda_prefix_attention_workspace(None, None, None, 32, ctypes.byref(n)) == ec.ERROR and n.value == 0
    assert lib.ernie_cuda_prefix_attention_workspace(None, kv().c, batch().c, 32, None) == ec.ERROR
    assert lib.ernie_cuda_beam_select_workspace(None, 1, 1, 1, None) == ec.ERROR
    assert lib.ernie_cuda_beam_reorder(None, None, 1, 1, None, None, 1, None, None, None) == ec.ERROR


def test_warps_of_a_tile_share_no_bytes(tmp_path):
    """Compiles the attention's layout header by itself and looks at every byte that a softmax warp touches."""
    here, exe = os.path.dirname(os.path.abspath(__file__)), str(tmp_path / "layout")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I" + os.path.join(os.path.dirname(ec.LIB_PATH), "csrc"),
                    os.path.join(here, "cpp", "test_attend_layout.cpp"), "-o", exe], check=True, capture_output=True, text=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "attention layout passed" in r.stdout, r.stderr + r.stdout


# ------------------------------------------------------------------ the oracle
def test_oracle_attention_is_dense_attention_over_the_joined_tokens():
    rng = np.random.default_rng(0)
    dim, page = 8, 8
    k, v = rng.standard_normal((2, 1, 6, 1, page, dim))
    q = rng.standard_normal((2, 2, dim))  # one sequence, two new tokens, two heads
    out = np.full(q.shape, 9.0)
    od.attention(k, v, 0, q, out, [[4, 0]], [11], [2], [[5, 2]], [13])
    keys = np.concatenate([k[0, 5, 0], k[0, 2, 0][:5], k[0, 4, 0], k[0, 0, 0][:3]])
    values = np.concatenate([v[0, 5, 0], v[0, 2, 0][:5], v[0, 4, 0], v[0, 0, 0][:3]])
    for i in range(2):
        for h in range(2):
            p = np.exp(keys[:23 + i] @ q[i, h] / np.sqrt(dim))
            assert np.allclose(out[i, h], (p / p.sum()) @ values[:23 + i], atol=1e-14)


def test_oracle_select_is_an_exhaustive_search():
    rng = np.random.default_rng(1)
    logits, scores = rng.standard_normal((2, 3, 11)), rng.standard_normal((2, 3))
    finished = np.array([[0, 1, 0], [0, 0, 0]])
    parents, tokens, totals, ended, _ = od.select(logits, scores, finished, 4)
    for g in range(2):
        every = []
        for b in range(3):
            if finished[g, b]:
                every.append((scores[g, b], b, 4))
                continue
            logp = logits[g, b] - np.log(np.exp(logits[g, b]).sum())
            every += [(scores[g, b] + logp[t], b, t) for t in range(11)]
        best = sorted(every, reverse=True)[:3]
        assert [(p, t) for p, t in zip(parents[g], tokens[g])] == [(b, t) for _, b, t in best]
        assert np.allclose(totals[g], [s for s, _, _ in best])
        assert list(ended[g]) == [int(bool(finished[g, b]) or t == 4) for _, b, t in best]


def test_oracle_reorder_keeps_every_page_and_every_history():
    rng = np.random.default_rng(2)
    for _ in range(50):
        beams, page = int(rng.integers(1, 9)), 8
        tables = rng.permutation(beams * 2 + 1)[:beams * 2].reshape(beams, 2)
        lens = rng.integers(0, 17, beams)
        k = rng.standard_normal((2, beams * 2 + 1, 1, page, 4))
        v = k + 1.0
        parents = rng.integers(-1, beams, (1, beams))
        before = [od.tokens_of(k, 1, tables[b], lens[b]) for b in range(beams)]
        new_tables, new_lens = od.reorder(k, v, parents, tables, lens)
        assert sorted(new_tables.ravel()) == sorted(tables.ravel())
        for i, p in enumerate(parents[0]):
            assert new_lens[i] == (0 if p < 0 else lens[p])
            if p >= 0:
                assert np.array_equal(od.tokens_of(k, 1, new_tables[i], new_lens[i]), before[p])
                assert np.array_equal(od.tokens_of(v, 1, new_tables[i], new_lens[i]), before[p] + 1.0)
