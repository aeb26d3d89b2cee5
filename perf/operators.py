"""Measured cases of the batched decoding operators: the paged K/V append with the position rotation, the
attention of a batch whose sequences share a long prefix, beam selection over the vocabulary, and the reordering
of the beams' cached state.

Each case has a plain form (elementary torch operations in 32 bits, 64 where a selection hangs on the last bits)
and the library's own call; `own` chooses between them. `exact` restates the definitions in 64 bits.

The library's calls enqueue on its context's stream. With `own` torch's work runs on that stream too, from the first
`prepare` on, so that inputs, calls and what uses the results are in one order; a caller who runs torch on another stream
is ordered with it by events. Either way a pass is over for torch's current stream when the calls are.

The cache of one layer is K and V [pages][kv_heads][page_size][head_dim]. A sequence's tokens lie in the pages of
its table row; the sequences of a group share the prefix in the group's own pages, which comes before their
tokens."""
import math
import os
import sys

import torch

own = False

_context = None
_stream = _context_stream = None  # the context's, for torch and as an address


def _library():
    """The library's binding and one context for the process, whose stream becomes torch's current one."""
    global _context, _stream, _context_stream
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ernie-image-ncnn-vulkan_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import ernie_cuda
    if _context is None:
        _context = ernie_cuda.Context(torch.cuda.current_device())
        _context_stream = _context.stream
        _stream = torch.cuda.ExternalStream(_context_stream)
        _stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(_stream)
    return ernie_cuda, _context


_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------ the cases
def _append(name, sequences, queries, past, heads=32, kv_heads=8, dim=128, page=16, source="fp32", cache="bf16",
            ragged=False, pad=0):
    return {"name": name, "op": "append", "sequences": sequences, "queries": queries, "past": past, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "source": source, "cache": cache, "ragged": ragged,
            "pad": pad}


def _attend(name, groups, per_group, queries, prefix, suffix, heads=32, kv_heads=8, dim=128, page=16, cache="bf16",
            ragged=False):
    return {"name": name, "op": "attend", "groups": groups, "per_group": per_group, "queries": queries,
            "prefix": prefix, "suffix": suffix, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "cache": cache, "ragged": ragged}


def _select(name, groups, beams, vocab, source="fp32", pad=0):
    return {"name": name, "op": "select", "groups": groups, "beams": beams, "vocab": vocab, "source": source,
            "pad": pad}


def _reorder(name, layers, groups, beams, suffix, kv_heads=8, dim=128, page=16, cache="bf16"):
    return {"name": name, "op": "reorder", "layers": layers, "groups": groups, "beams": beams, "suffix": suffix,
            "kv_heads": kv_heads, "dim": dim, "page": page, "cache": cache}


def listed():
    return [
        # one decode step of five beams of one prompt: the smallest call, all latency
        _append("append_step", 5, 1, 200),
        # prefill chunks of a batch, FP32 cache (the prompt enhancer's chunk of 32 rows), ragged counts
        _append("append_chunk", 24, 32, 700, cache="fp32", ragged=True),
        # a long prompt laid down at once, BF16 activations with padded rows
        _append("append_prompt", 1, 16000, 0, page=64, source="bf16", pad=64),
        # one step of five beams behind a short prompt
        _attend("attend_step", 1, 5, 1, 300, 60),
        # one step of a batch behind a long chat template
        _attend("attend_shared", 1, 64, 1, 4096, 512),
        # beams of several prompts, each group behind its own prompt, FP32 cache
        _attend("attend_groups_fp32", 12, 8, 1, 1800, 300, cache="fp32"),
        # chunks of a batch behind one template: many query rows, ragged counts
        _attend("attend_chunk", 1, 16, 32, 2000, 700, page=32, ragged=True),
        # a large serving batch behind a very long template
        _attend("attend_long", 1, 256, 1, 16384, 1024, page=64),
        # five beams over the prompt enhancer's vocabulary
        _select("select_step", 1, 5, 131072),
        # a batch of beams over the same vocabulary
        _select("select_batch", 64, 8, 131072),
        # five beams' state over the prompt enhancer's 26 layers
        _reorder("reorder_step", 26, 1, 5, 60),
        # the beams of a batch
        _reorder("reorder_batch", 26, 12, 4, 250, page=32),
    ]


_HEADS = ((32, 8), (8, 8), (16, 2), (24, 4), (20, 4), (7, 1), (32, 4), (12, 6))


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / (4e13 if "fp32" in (case.get("cache"), case.get("source")) else 8e14)


def draw(rng):
    most = max(_cost(c) for c in listed() if c["op"] != "append")
    while True:
        op = rng.choice(("append", "attend", "attend", "select", "reorder"))
        heads, kv_heads = rng.choice(_HEADS)
        dim, page, cache = rng.choice((64, 128, 128)), rng.choice((8, 16, 32, 64, 128)), rng.choice(("bf16", "bf16", "fp32"))
        if op == "append":
            c = _append("", _log(rng, 1, 256), _log(rng, 1, 512), _log(rng, 1, 2048), heads, kv_heads, dim, page,
                        rng.choice(("fp32", "bf16")), cache, rng.random() < 0.5, rng.choice((0, 0, 8, 3)))
        elif op == "attend":
            queries = rng.choice((1, 1, 1, rng.randint(2, 8), rng.randint(9, 40)))
            c = _attend("", rng.choice((1, 1, rng.randint(2, 12))), _log(rng, 1, 128), queries, _log(rng, 16, 16384),
                        _log(rng, queries, 1024), heads, kv_heads, dim, page, cache, rng.random() < 0.5)
        elif op == "select":
            c = _select("", _log(rng, 1, 64), rng.randint(1, 12), _log(rng, 500, 160000), rng.choice(("fp32", "bf16")),
                        rng.choice((0, 0, 5, 64)))
        else:
            c = _reorder("", rng.randint(1, 32), _log(rng, 1, 24), rng.randint(2, 10), _log(rng, 1, 400), kv_heads, dim,
                         page, cache)
        tokens = c.get("groups", 1) * c.get("per_group", c.get("beams", c.get("sequences", 1))) * \
            (c.get("suffix", 0) + c.get("past", 0) + c.get("queries", 0) + page)
        pool = tokens * kv_heads * dim * _BYTES[cache] * 2 * c.get("layers", 1)
        if pool < 1.6e9 and _cost(c) <= 0.8 * most:
            del c["name"]
            return c


def work(case):
    op = case["op"]
    if op == "append":
        rows = case["sequences"] * case["queries"] * (0.75 if case["ragged"] else 1.0)
        values = rows * case["dim"]
        width = case["heads"] + 2 * case["kv_heads"]
        # the projection in; the rotated queries, the keys and the values out; each position's cos and sin once
        bytes_ = values * width * (_BYTES[case["source"]] + _BYTES[case["cache"]])
        positions = min(rows, case["past"] + case["queries"]) if case["sequences"] > 1 else rows
        return {"bytes": bytes_ + positions * case["dim"] * 8,
                "flops": values * (case["heads"] + case["kv_heads"]) * 3}
    if op == "attend":
        sequences = case["groups"] * case["per_group"]
        rows = sequences * case["queries"] * (0.75 if case["ragged"] else 1.0)
        prefix = case["prefix"] * (1.0 if case["groups"] == 1 else 0.75)
        suffix = (case["suffix"] + case["queries"]) / 2
        size = _BYTES[case["cache"]]
        kv = (case["groups"] * prefix + sequences * suffix) * case["kv_heads"] * case["dim"] * 2 * size
        qo = rows * case["heads"] * case["dim"] * 2 * size
        keys = prefix + max(1.0, suffix - (case["queries"] - 1) * (0.375 if case["ragged"] else 0.5))
        return {"bytes": kv + qo, "flops": 4.0 * rows * case["heads"] * case["dim"] * keys}
    if op == "select":
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * _BYTES[case["source"]] + 24.0), "flops": 4.0 * rows * case["vocab"]}
    # reorder: about a third of the beams are copied, each token read and written in every layer
    beams = case["beams"]
    copied = case["groups"] * (beams - _survivors(beams))
    token = case["kv_heads"] * case["dim"] * _BYTES[case["cache"]] * 2 * case["layers"]
    return {"bytes": copied * 0.75 * case["suffix"] * token * 2 + case["groups"] * beams * 4.0 * 8, "flops": 0.0}


def _survivors(beams):
    """How many of a group's beams have a child in the prepared cases."""
    return beams - beams // 3 - (1 if beams > 1 and beams < 3 else 0)


# ------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(g, low, high, shape):
    """Whole numbers in [low, high]."""
    return torch.randint(low, high + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _normal(g, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype).mul_(scale)


def _pages_of(tokens, page):
    return -(-tokens // page)


def _tables(g, rows, per_row, first, pages):
    """[rows][per_row] distinct pages from a shuffled pool of `pages`, starting at entry `first` of the shuffle."""
    shuffled = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    return shuffled, shuffled[first:first + rows * per_row].reshape(rows, per_row).contiguous()


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    s.update({"append": _prepare_append, "attend": _prepare_attend, "select": _prepare_select,
              "reorder": _prepare_reorder}[case["op"]](case, g))
    if own:
        s["own"] = _handles(case, s)
    return s


def _rope_tables(positions, dim):
    frequency = 1.0 / 1000000.0 ** (torch.arange(dim // 2, device="cuda", dtype=torch.float64) / (dim // 2))
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * frequency
    angle = torch.cat([angle, angle], 1)
    return angle.cos().float(), angle.sin().float()


def _prepare_append(c, g):
    n, queries, page = c["sequences"], c["queries"], c["page"]
    lens = c["past"] + queries
    per_row = _pages_of(lens, page)
    pages = n * per_row + 3
    _, tables = _tables(g, n, per_row, 0, pages)
    counts = _ints(g, queries // 2, queries, (n,)) if c["ragged"] else torch.full((n,), queries, device="cuda", dtype=torch.int32)
    past = _ints(g, 0, c["past"], (n,)) if n > 1 else torch.full((n,), c["past"], device="cuda", dtype=torch.int32)
    width = (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
    shape = (1, pages, c["kv_heads"], page, c["dim"])
    cos, sin = _rope_tables(lens, c["dim"])
    return {"qkv": _normal(g, (n * queries, width + c["pad"]), _TYPES[c["source"]]), "cos": cos, "sin": sin,
            "tables": tables, "lens": past + counts, "counts": counts,
            "k": _normal(g, shape, _TYPES[c["cache"]]), "v": _normal(g, shape, _TYPES[c["cache"]]),
            "q": _normal(g, (n * queries, c["heads"], c["dim"]), _TYPES[c["cache"]])}


def _prepare_attend(c, g):
    groups, n, queries, page = c["groups"], c["groups"] * c["per_group"], c["queries"], c["page"]
    shared, per_row = _pages_of(c["prefix"], page), _pages_of(max(c["suffix"], queries), page)
    pages = groups * shared + n * per_row + 1
    shuffled, prefix_tables = _tables(g, groups, shared, 0, pages)
    tables = shuffled[groups * shared:groups * shared + n * per_row].reshape(n, per_row).contiguous()
    prefix_lens = _ints(g, c["prefix"] // 2, c["prefix"], (groups,)) if groups > 1 else torch.full((1,), c["prefix"], device="cuda", dtype=torch.int32)
    shape = (1, pages, c["kv_heads"], page, c["dim"])
    dtype = _TYPES[c["cache"]]
    counts = _ints(g, queries // 2, queries, (n,)) if c["ragged"] else torch.full((n,), queries, device="cuda", dtype=torch.int32)
    return {"k": _normal(g, shape, dtype), "v": _normal(g, shape, dtype), "prefix_tables": prefix_tables,
            "prefix_lens": prefix_lens, "tables": tables, "lens": _ints(g, queries, max(c["suffix"], queries), (n,)),
            "counts": counts, "q": _normal(g, (n * queries, c["heads"], c["dim"]), dtype, 1.5),
            "out": _normal(g, (n * queries, c["heads"], c["dim"]), dtype, 0.02)}


def _prepare_select(c, g):
    rows, vocab = c["groups"] * c["beams"], c["vocab"]
    logits = _normal(g, (rows, vocab + c["pad"]), torch.float32, 3.0)
    # tokens that a grammar or a stop list rules out
    logits.masked_fill_(torch.rand(logits.shape, generator=g, device="cuda") < 0.02, float("-inf"))
    scores = _normal(g, (c["groups"], c["beams"]), torch.float32, 2.0) - 20.0
    finished = (torch.rand((c["groups"], c["beams"]), generator=g, device="cuda") < 0.1).to(torch.int32)
    like = (c["groups"], c["beams"])
    return {"logits": logits.to(_TYPES[c["source"]]), "scores": scores, "finished": finished, "end": vocab // 3,
            "parents": torch.zeros(like, device="cuda", dtype=torch.int32),
            "tokens": torch.zeros(like, device="cuda", dtype=torch.int32),
            "new_scores": torch.zeros(like, device="cuda"), "new_finished": torch.zeros(like, device="cuda", dtype=torch.int32)}


def _prepare_reorder(c, g):
    groups, beams, page = c["groups"], c["beams"], c["page"]
    n, per_row = groups * beams, _pages_of(c["suffix"], page)
    pages = n * per_row + 2
    _, tables = _tables(g, n, per_row, 0, pages)
    shape = (c["layers"], pages, c["kv_heads"], page, c["dim"])
    dtype = _TYPES[c["cache"]]
    # the survivors keep one child each at least, the other places go to survivors at random, all in random order
    survivors = torch.rand((groups, beams), generator=g, device="cuda").argsort(1)[:, :_survivors(beams)]
    spare = beams - survivors.shape[1]
    again = torch.gather(survivors, 1, _ints(g, 0, survivors.shape[1] - 1, (groups, spare)).long())
    parents = torch.cat([survivors, again], 1)
    order = torch.rand((groups, beams), generator=g, device="cuda").argsort(1)
    lens = _ints(g, (c["suffix"] + 1) // 2, c["suffix"], (n,))
    return {"k": _normal(g, shape, dtype), "v": _normal(g, shape, dtype), "tables": tables, "lens": lens,
            "parents": torch.gather(parents, 1, order).to(torch.int32).contiguous(),
            "new_tables": torch.empty_like(tables), "new_lens": torch.empty_like(lens)}


def _handles(c, s):
    """What a user's program keeps: the context, the cache's and the batch's descriptions, a workspace."""
    ec, ctx = _library()
    h = {"ec": ec, "ctx": ctx}
    precision = {"bf16": ec.BF16, "fp32": ec.FP32}
    if c["op"] != "select":
        h["kv"] = ec.PagedKv(s["k"], s["v"], s["k"].shape[0], s["k"].shape[1], c["page"], c["kv_heads"], c["dim"],
                             precision[c["cache"]])
    if c["op"] == "append":
        h["batch"] = ec.PagedBatch(c["sequences"], c["queries"], s["tables"], s["tables"].shape[1], s["lens"], s["counts"])
    elif c["op"] == "attend":
        h["batch"] = ec.PagedBatch(c["groups"] * c["per_group"], c["queries"], s["tables"], s["tables"].shape[1],
                                   s["lens"], s["counts"], c["groups"], s["prefix_tables"],
                                   s["prefix_tables"].shape[1], s["prefix_lens"])
        size = ctx.prefix_attention_workspace(h["kv"], h["batch"], c["heads"])
        h["workspace"] = torch.empty(size, device="cuda", dtype=torch.uint8)
    elif c["op"] == "select":
        size = ctx.beam_select_workspace(c["groups"], c["beams"], c["vocab"])
        h["workspace"] = torch.empty(size, device="cuda", dtype=torch.uint8)
    if "source" in c:
        h["source"] = precision[c["source"]]
    return h


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        call = {"append": _own_append, "attend": _own_attend, "select": _own_select, "reorder": _own_reorder}[op]
        # (torch.cuda.current_stream() would take as long as a small call)
        if torch._C._cuda_getCurrentRawStream(_context.device) == _context_stream:
            return call(s)
        current = torch.cuda.current_stream()
        _stream.wait_stream(current)
        out = call(s)
        current.wait_stream(_stream)
        return out
    return {"append": _plain_append, "attend": _plain_attend, "select": _plain_select, "reorder": _plain_reorder}[op](s)


def _own_append(s):
    c, h = s["case"], s["own"]
    h["ctx"].paged_append(h["kv"], 0, h["batch"], s["qkv"], h["source"], s["qkv"].shape[1], c["heads"], s["cos"], s["sin"],
                          s["cos"].shape[0], s["q"])
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _own_attend(s):
    h = s["own"]
    h["ctx"].prefix_attention(h["kv"], 0, h["batch"], s["q"], s["case"]["heads"], s["out"], h["workspace"],
                              h["workspace"].numel())
    return s["out"]


def _own_select(s):
    c, h = s["case"], s["own"]
    h["ctx"].beam_select(s["logits"], h["source"], s["logits"].shape[1], c["groups"], c["beams"], c["vocab"], s["end"],
                         s["scores"], s["finished"], s["parents"], s["tokens"], s["new_scores"], s["new_finished"],
                         h["workspace"], h["workspace"].numel())
    return {"parents": s["parents"], "tokens": s["tokens"], "scores": s["new_scores"], "finished": s["new_finished"]}


def _own_reorder(s):
    c, h = s["case"], s["own"]
    h["ctx"].beam_reorder(h["kv"], c["groups"], c["beams"], s["parents"], s["tables"], s["tables"].shape[1], s["lens"],
                          s["new_tables"], s["new_lens"])
    return {"k": s["k"], "v": s["v"], "tables": s["new_tables"], "lens": s["new_lens"]}


def _new_tokens(s):
    """Of each row of the batch: whether it holds a new token, and the token's place in its sequence."""
    c = s["case"]
    i = torch.arange(c["queries"], device="cuda")
    valid = i < s["counts"][:, None]
    return valid, s["lens"][:, None] - s["counts"][:, None] + i


def _plain_append(s):
    c = s["case"]
    dim, heads, kv_heads, page = c["dim"], c["heads"], c["kv_heads"], c["page"]
    valid, place = _new_tokens(s)
    rows = valid.reshape(-1).nonzero().squeeze(1)
    place = place.reshape(-1)[rows].long()
    sequence = rows // c["queries"]
    x = s["qkv"][rows, :(heads + 2 * kv_heads) * dim].float().reshape(-1, heads + 2 * kv_heads, dim)
    qk, v = x[:, :heads + kv_heads], x[:, heads + kv_heads:]
    cos, sin = s["cos"][place][:, None], s["sin"][place][:, None]
    turned = torch.cat([-qk[..., dim // 2:], qk[..., :dim // 2]], -1)
    qk = qk * cos + turned * sin
    s["q"][rows] = qk[:, :heads].to(s["q"].dtype)
    at = s["tables"][sequence, place // page].long()
    s["k"][0, at, :, place % page] = qk[:, heads:].to(s["k"].dtype)
    s["v"][0, at, :, place % page] = v.to(s["v"].dtype)
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _gather(pool, tables, lens):
    """[rows][kv_heads][tokens][dim] in 32 bits, zero past each row's length."""
    x = pool[0][tables.long()].float()  # [rows][pages][kv_heads][page][dim]
    x = x.permute(0, 2, 1, 3, 4).reshape(tables.shape[0], x.shape[2], -1, x.shape[4])
    inside = torch.arange(x.shape[2], device="cuda") < lens[:, None]
    return torch.where(inside[:, None, :, None], x, 0.0)


def _plain_attend(s):
    c = s["case"]
    groups, per, queries, dim = c["groups"], c["per_group"], c["queries"], c["dim"]
    kv_heads, n = c["kv_heads"], c["groups"] * c["per_group"]
    share = c["heads"] // kv_heads
    scale = 1.0 / math.sqrt(dim)
    q = s["q"].float().reshape(n, queries, kv_heads, share, dim).permute(0, 2, 1, 3, 4)
    q = q.reshape(n, kv_heads, queries * share, dim)
    # the prefix: one product for all rows of a group
    pk, pv = (_gather(s[x], s["prefix_tables"], s["prefix_lens"]) for x in ("k", "v"))
    qp = q.reshape(groups, per, kv_heads, queries * share, dim).transpose(1, 2).reshape(groups, kv_heads, -1, dim)
    ps = (qp @ pk.transpose(2, 3)) * scale
    inside = torch.arange(pk.shape[2], device="cuda") < s["prefix_lens"][:, None]
    ps = torch.where(inside[:, None, None], ps, float("-inf"))
    ps = ps.reshape(groups, kv_heads, per, queries * share, -1).transpose(1, 2).reshape(n, kv_heads, queries * share, -1)
    # each sequence's own tokens, up to the row's own place
    sk, sv = (_gather(s[x], s["tables"], s["lens"]) for x in ("k", "v"))
    valid, place = _new_tokens(s)
    seen = torch.arange(sk.shape[2], device="cuda") <= place[:, :, None]  # [n][queries][tokens]
    seen = seen[:, None, :, None].expand(n, 1, queries, share, sk.shape[2]).reshape(n, 1, queries * share, -1)
    ss = torch.where(seen, (q @ sk.transpose(2, 3)) * scale, float("-inf"))
    top = torch.maximum(ps.amax(3, keepdim=True), ss.amax(3, keepdim=True))
    top = torch.where(torch.isinf(top), 0.0, top)
    ps, ss = torch.exp(ps - top), torch.exp(ss - top)
    total = ps.sum(3, keepdim=True) + ss.sum(3, keepdim=True)
    pg = ps.reshape(groups, per, kv_heads, queries * share, -1).transpose(1, 2).reshape(groups, kv_heads, per * queries * share, -1)
    o = (pg @ pv).reshape(groups, kv_heads, per, queries * share, dim).transpose(1, 2).reshape(n, kv_heads, queries * share, dim)
    o = (o + ss @ sv) / torch.where(total > 0, total, 1.0)
    o = o.reshape(n, kv_heads, queries, share, dim).permute(0, 2, 1, 3, 4).reshape(n * queries, c["heads"], dim)
    return torch.where(valid.reshape(-1, 1, 1), o.to(s["out"].dtype), s["out"])


def _plain_select(s):
    c = s["case"]
    groups, beams, vocab = c["groups"], c["beams"], c["vocab"]
    x = s["logits"][:, :vocab].double()
    # a row with a NaN or a +inf has no normaliser, and one without any token none either
    top = x.amax(1, keepdim=True)
    lse = torch.log(torch.exp(x - top).sum(1, keepdim=True)) + top
    value, token = torch.sort(x, dim=1, descending=True, stable=True)
    kept = min(beams, vocab)
    value, token = value[:, :kept], token[:, :kept]
    score = s["scores"].reshape(-1, 1).double()
    total = score + (value - lse)
    usable = torch.isfinite(lse) & torch.isfinite(score) & torch.isfinite(value)
    total = torch.where(usable, total, float("-inf"))
    # a finished beam offers itself alone, with its score as it is
    done = s["finished"].reshape(-1, 1) != 0
    first = torch.arange(kept, device="cuda")[None] == 0
    total = torch.where(done, torch.where(first & torch.isfinite(score), score, float("-inf")), total)
    token = torch.where(done, s["end"], token)
    total, place = torch.sort(total.reshape(groups, beams * kept), dim=1, descending=True, stable=True)
    total, place = total[:, :beams], place[:, :beams]
    found = total > float("-inf")
    parents = torch.where(found, place // kept, -1)
    tokens = torch.where(found, torch.gather(token.reshape(groups, -1), 1, place), -1)
    was = torch.gather(s["finished"], 1, parents.clamp(min=0))
    finished = ~found | (was != 0) | (tokens == s["end"])
    return {"parents": parents.to(torch.int32), "tokens": tokens.to(torch.int32), "scores": total.float(),
            "finished": finished.to(torch.int32)}


def _moves(parents):
    """Of each group's places: the old place whose pages the place takes, and whether its parent's tokens have to be
    copied into them. A parent's pages stay with its heir (the parent's own place where that is its child, else its
    first child); the other children take the pages of places without children, in order."""
    groups, beams = parents.shape
    place = torch.arange(beams, device=parents.device)
    child = parents[:, :, None] == place  # [group][child][parent]
    order = torch.where(place[:, None] == place[None], -1, place[:, None])
    heir = torch.where(child, order, beams).argmin(1)  # [group][parent]
    alive = child.any(1)
    is_heir = torch.gather(heir, 1, parents.clamp(min=0)) == place
    is_heir &= parents >= 0
    dead = torch.argsort(alive.to(torch.int32), dim=1, stable=True)
    nth = torch.cumsum((~is_heir).long(), 1) - 1
    takes = torch.where(is_heir, parents, torch.gather(dead, 1, nth.clamp(min=0)))
    return takes, ~is_heir & (parents >= 0)


def _plain_reorder(s):
    c = s["case"]
    groups, beams, page = c["groups"], c["beams"], c["page"]
    parents = s["parents"].long()
    takes, copied = _moves(parents)
    base = torch.arange(groups, device="cuda")[:, None] * beams
    new_tables = s["tables"][(takes + base).reshape(-1)]
    lens = torch.where(parents >= 0, s["lens"].reshape(groups, beams).gather(1, parents.clamp(min=0)), 0).reshape(-1)
    source = s["tables"][(parents.clamp(min=0) + base).reshape(-1)]
    token = torch.arange(s["tables"].shape[1] * page, device="cuda")
    row, place = (copied.reshape(-1, 1) & (token < lens[:, None])).nonzero(as_tuple=True)
    there, here = new_tables[row, place // page].long(), source[row, place // page].long()
    s["k"][:, there, :, place % page] = s["k"][:, here, :, place % page]
    s["v"][:, there, :, place % page] = s["v"][:, here, :, place % page]
    return {"k": s["k"], "v": s["v"], "tables": new_tables, "lens": lens.to(torch.int32)}


# ------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    g = _generator(seed)
    s = {"append": _prepare_append, "attend": _prepare_attend, "select": _prepare_select,
         "reorder": _prepare_reorder}[case["op"]](case, g)
    return {"append": _exact_append, "attend": _exact_attend, "select": _exact_select, "reorder": _exact_reorder}[case["op"]](case, s)


def _exact_append(c, s):
    dim, half, heads, kv_heads, queries = c["dim"], c["dim"] // 2, c["heads"], c["kv_heads"], c["queries"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    first = s["lens"] - s["counts"]
    x = s["qkv"].double()[:, :(heads + 2 * kv_heads) * dim].reshape(c["sequences"], queries, -1, dim)
    # the pair (d, d + half) is a plane turned by the angle of the token's place
    place = (first[:, None] + torch.arange(queries, device="cuda")).long()
    held = place.clamp(max=s["cos"].shape[0] - 1)
    cos, sin = s["cos"].double()[held][:, :, None], s["sin"].double()[held][:, :, None]
    low, high = x[..., :half], x[..., half:]
    turned = torch.cat([low * cos[..., :half] - high * sin[..., :half], high * cos[..., half:] + low * sin[..., half:]], -1)
    new = torch.arange(queries, device="cuda")[None] < s["counts"][:, None]
    q = q.reshape(c["sequences"], queries, heads, dim)
    q[new] = turned[:, :, :heads][new]
    page = torch.gather(s["tables"].long(), 1, (held // c["page"]))
    k[0].transpose(1, 2)[page[new], (place % c["page"])[new]] = turned[:, :, heads:heads + kv_heads][new]
    v[0].transpose(1, 2)[page[new], (place % c["page"])[new]] = x[:, :, heads + kv_heads:][new]
    return {"q": q.reshape(-1, heads, dim), "k": k, "v": v}


def _exact_attend(c, s):
    """Sequence by sequence and row by row: softmax(q k / sqrt(dim)) v over the keys that the row sees."""
    out = s["out"].double().reshape(c["groups"] * c["per_group"], c["queries"], c["heads"], c["dim"])
    q = s["q"].double().reshape(out.shape)
    share = c["heads"] // c["kv_heads"]
    if c["groups"] * c["per_group"] * c["queries"] > 6000:
        return None
    lens, counts, prefix_lens = s["lens"].tolist(), s["counts"].tolist(), s["prefix_lens"].tolist()

    def keys(pool, row, tokens):
        x = pool[0][row.long()].double().transpose(0, 1)  # [kv_heads][pages][page][dim]
        return x.reshape(c["kv_heads"], -1, c["dim"])[:, :tokens]

    for group in range(c["groups"]):
        k0, v0 = (keys(s[x], s["prefix_tables"][group], prefix_lens[group]) for x in ("k", "v"))
        for n in range(group * c["per_group"], (group + 1) * c["per_group"]):
            k1, v1 = (keys(s[x], s["tables"][n], lens[n]) for x in ("k", "v"))
            k, v = torch.cat([k0, k1], 1), torch.cat([v0, v1], 1)
            rows = q[n, :counts[n]].reshape(-1, c["kv_heads"], share, c["dim"]).permute(1, 0, 2, 3)
            score = torch.einsum("hnad,hkd->hnak", rows, k) / math.sqrt(c["dim"])
            last = prefix_lens[group] + lens[n] - counts[n] + torch.arange(counts[n], device="cuda")
            hidden = torch.arange(k.shape[1], device="cuda")[None] > last[:, None]
            p = torch.softmax(score.masked_fill(hidden[None, :, None], float("-inf")), -1)
            o = torch.einsum("hnak,hkd->nhad", p, v)
            out[n, :counts[n]] = o.reshape(counts[n], c["heads"], c["dim"])
    return out.reshape(-1, c["heads"], c["dim"])


def _exact_select(c, s):
    x = s["logits"].double()[:, :c["vocab"]].reshape(c["groups"], c["beams"], -1)
    total = torch.log_softmax(x, -1) + s["scores"].double()[..., None]
    done = s["finished"][..., None] != 0
    ends = torch.arange(c["vocab"], device="cuda") == s["end"]
    total = torch.where(done, torch.where(ends, s["scores"].double()[..., None], float("-inf")), total)
    total = total.reshape(c["groups"], -1).topk(c["beams"], 1).values
    return {"parents": None, "tokens": None, "scores": total, "finished": None}


def _exact_reorder(c, s):
    # the copied values are the cache's own: only their places change
    k, v = s["k"].double(), s["v"].double()
    beams, page = c["beams"], c["page"]
    tables, lens, parents = s["tables"].tolist(), s["lens"].tolist(), s["parents"].tolist()
    there, here, slot = [], [], []
    for group, chosen in enumerate(parents):
        base = group * beams
        heirs = {}
        for child, parent in enumerate(chosen):
            if parent >= 0 and (parent not in heirs or child == parent):
                heirs[parent] = child
        free = [p for p in range(beams) if p not in heirs]
        for child, parent in enumerate(chosen):
            if parent >= 0 and heirs[parent] == child:
                continue
            into = free.pop(0)
            for t in range(lens[base + parent] if parent >= 0 else 0):
                there.append(tables[base + into][t // page])
                here.append(tables[base + parent][t // page])
                slot.append(t % page)
    there, here, slot = (torch.tensor(x, device="cuda", dtype=torch.long) for x in (there, here, slot))
    for pool in (k, v):
        pool[:, there, :, slot] = pool[:, here, :, slot]
    return {"k": k, "v": v, "tables": None, "lens": None}
