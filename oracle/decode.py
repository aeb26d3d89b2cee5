"""Batched decoding behind shared prefixes restated in float64 numpy: the paged append with the position rotation,
the attention over a shared prefix and a sequence's own tokens, beam selection, and the reordering of the beams'
cached state. Test infrastructure only; the definitions are those of include/ernie_cuda.h.

A cache is K and V [layers][pages][kv_heads][page_size][dim]; tables [sequences][max_pages], lens and counts
[sequences]; a group's prefix lies in prefix_tables [groups][max_prefix_pages], prefix_lens [groups]."""
import numpy as np


def rotate(x, cos, sin):
    """Half-split rotation of x [..., dim] by cos, sin [dim]."""
    half = x.shape[-1] // 2
    low, high = x[..., :half], x[..., half:]
    return np.concatenate([low * cos[:half] - high * sin[:half], high * cos[half:] + low * sin[half:]], -1)


def append(k, v, layer, q, tables, lens, counts, qkv, cos, sin, prefix_lens=None):
    """Writes into float64 copies k, v of the cache and q [sequences*queries][heads][dim]; returns, beside each, the
    sum of the magnitudes of the products that made a value (the scale of its rounding)."""
    page_size, kv_heads, dim = k.shape[3], k.shape[2], k.shape[4]
    heads, sequences = q.shape[1], len(lens)
    queries, groups = q.shape[0] // sequences, 1 if prefix_lens is None else len(prefix_lens)
    scale_q, scale_k, scale_v = np.abs(q), np.abs(k), np.abs(v)
    for s in range(sequences):
        start = 0 if prefix_lens is None else int(prefix_lens[s // (sequences // groups)])
        for i in range(counts[s]):
            slot, place = s * queries + i, lens[s] - counts[s] + i
            position = start + place
            if position < 0:
                continue
            x = qkv[slot, :(heads + 2 * kv_heads) * dim].astype(np.float64).reshape(-1, dim)
            c, n = cos[position].astype(np.float64), sin[position].astype(np.float64)
            y = rotate(x[:heads + kv_heads], c, n)
            m = np.abs(x[:heads + kv_heads]) * np.abs(c) + np.abs(np.roll(x[:heads + kv_heads], dim // 2, -1)) * np.abs(n)
            q[slot], scale_q[slot] = y[:heads], m[:heads]
            if place < 0:
                continue
            page, at = tables[s][place // page_size], place % page_size
            k[layer, page, :, at], scale_k[layer, page, :, at] = y[heads:], m[heads:]
            v[layer, page, :, at] = x[heads + kv_heads:]
            scale_v[layer, page, :, at] = np.abs(x[heads + kv_heads:])
    return scale_q, scale_k, scale_v


def tokens_of(pool, layer, table, length):
    """[kv_heads][length][dim] of one table row."""
    page_size = pool.shape[3]
    pages = [pool[layer, table[j]] for j in range(-(-length // page_size))]
    if not pages:
        return np.zeros((pool.shape[2], 0, pool.shape[4]))
    return np.concatenate(pages, 1)[:, :length].astype(np.float64)


def attention(k, v, layer, q, out, tables, lens, counts, prefix_tables=None, prefix_lens=None):
    """Writes the rows that hold a token into out [sequences*queries][heads][dim]. Returns sum p|v| and, per row and
    head, the largest sum |q||k| / sqrt(dim) over its keys: the scales of the result's rounding."""
    sequences, heads, dim, kv_heads = len(lens), q.shape[1], q.shape[2], k.shape[2]
    queries, share = q.shape[0] // sequences, heads // kv_heads
    groups = 1 if prefix_lens is None else len(prefix_lens)
    weight, spread = np.zeros(out.shape), np.zeros(out.shape[:2])
    for s in range(sequences):
        g = s // (sequences // groups)
        keys, values = tokens_of(k, layer, tables[s], lens[s]), tokens_of(v, layer, tables[s], lens[s])
        start = 0
        if prefix_lens is not None:
            start = int(prefix_lens[g])
            keys = np.concatenate([tokens_of(k, layer, prefix_tables[g], start), keys], 1)
            values = np.concatenate([tokens_of(v, layer, prefix_tables[g], start), values], 1)
        for i in range(counts[s]):
            slot = s * queries + i
            seen = start + max(0, lens[s] - counts[s] + i + 1)
            for h in range(heads):
                if seen == 0:
                    out[slot, h] = 0.0
                    continue
                x, kk, vv = q[slot, h].astype(np.float64), keys[h // share][:seen], values[h // share][:seen]
                score = kk @ x / np.sqrt(dim)
                p = np.exp(score - score.max())
                p /= p.sum()
                out[slot, h] = p @ vv
                weight[slot, h] = p @ np.abs(vv)
                spread[slot, h] = (np.abs(kk) @ np.abs(x)).max() / np.sqrt(dim)
    return weight, spread


def select(logits, scores, finished, end_token):
    """logits [groups][beams][vocab]; parents, tokens, totals, finished of each group's best, and the smallest gap
    between two totals of different beams that the order hangs on."""
    groups, beams, vocab = logits.shape
    parents, tokens = np.full((groups, beams), -1), np.full((groups, beams), -1)
    totals, ended, gap = np.full((groups, beams), -np.inf), np.ones((groups, beams), np.int64), np.inf
    for g in range(groups):
        offers = []
        for b in range(beams):
            score = float(scores[g, b])
            if not np.isfinite(score):
                continue
            if finished[g, b]:
                offers.append((-score, b, 0, end_token))
                continue
            x = logits[g, b].astype(np.float64)
            top = x.max()
            if np.isnan(x).any() or not np.isfinite(top):
                continue
            log_sum = np.log(np.exp(x - top).sum())
            for rank, t in enumerate(np.lexsort((np.arange(vocab), -x))[:beams]):
                if np.isfinite(x[t]):
                    offers.append((-(score + ((x[t] - top) - log_sum)), b, rank, int(t)))
        offers.sort(key=lambda o: o[:3])
        for i, (total, b, _, t) in enumerate(offers[:beams]):
            parents[g, i], tokens[g, i], totals[g, i] = b, t, -total
            ended[g, i] = bool(finished[g, b]) or (end_token >= 0 and t == end_token)
        for one, other in zip(offers[:beams], offers[1:beams + 1]):
            if one[1] != other[1]:
                gap = min(gap, other[0] - one[0])
    return parents, tokens, totals, ended, gap


def reorder(k, v, parents, tables, lens):
    """Copies within k, v in place; the new tables and lens."""
    groups, beams = parents.shape
    page_size = k.shape[3]
    new_tables, new_lens = tables.copy(), lens.copy()
    for g in range(groups):
        heir = {}
        for child in range(beams):
            parent = int(parents[g, child])
            if parent >= 0 and (parent not in heir or child == parent):
                heir[parent] = child
        free = [p for p in range(beams) if p not in heir]
        for child in range(beams):
            parent, row = int(parents[g, child]), g * beams + child
            if parent >= 0 and heir[parent] == child:
                new_tables[row], new_lens[row] = tables[g * beams + parent], lens[g * beams + parent]
                continue
            into = tables[g * beams + free.pop(0)]
            new_tables[row], new_lens[row] = into, 0 if parent < 0 else lens[g * beams + parent]
            for t in range(new_lens[row]):
                source = tables[g * beams + parent]
                for pool in (k, v):
                    pool[:, into[t // page_size], :, t % page_size] = pool[:, source[t // page_size], :, t % page_size]
    return new_tables, new_lens
