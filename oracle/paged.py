"""Plain statements, in fp64 NumPy, of the paged-cache operators (append, attention, eviction, beam search).

The tests hold the CUDA kernels to these.  Pages are ``[num_pages, kv_heads, page_size, head_dim]``; nothing here
is fast.
"""

from __future__ import annotations

import math

import numpy as np


def slots(pages: np.ndarray, table_row: np.ndarray, n: int) -> np.ndarray:
    """The first ``n`` slots of a row, every head: [kv_heads, n, head_dim]."""
    ps = pages.shape[2]
    j = np.arange(n)
    return pages[table_row[j // ps], :, j % ps].transpose(1, 0, 2)


def append(k_pages, v_pages, table, lengths, starts, positions, q, k, v, cos=None, sin=None, pair_order=False):
    """(k_pages, v_pages, q_out) after the tokens of each row went to its slots lengths[b], ...; all fp64."""
    k_pages, v_pages = k_pages.astype(np.float64), v_pages.astype(np.float64)
    q_out = np.zeros(q.shape)
    ps, half = k_pages.shape[2], k.shape[-1] // 2

    def halves(x):
        x = x.astype(np.float64)
        return (x[..., 0::2], x[..., 1::2]) if pair_order else (x[..., :half], x[..., half:])

    for b in range(len(lengths)):
        for i, t in enumerate(range(starts[b], starts[b + 1])):
            slot, pos = lengths[b] + i, positions[b] + i
            c, s = (np.ones(half), np.zeros(half)) if cos is None else (cos[pos].astype(np.float64), sin[pos].astype(np.float64))
            for x, dst in ((q[t], q_out[t]), (k[t], k_pages[table[b, slot // ps], :, slot % ps])):
                x1, x2 = halves(x)
                dst[...] = np.concatenate([x1 * c - x2 * s, x2 * c + x1 * s], -1)
            v_pages[table[b, slot // ps], :, slot % ps] = np.concatenate(halves(v[t]), -1)
    return k_pages, v_pages, q_out


def attention(q, k_pages, v_pages, table, lengths, scale=None, exp_err=2.0**-17):
    """Per row: (out [q_heads, head_dim], probs [q_heads, n], bound [q_heads, head_dim], rel) in fp64.

    ``bound`` is how far an fp32 evaluation may be off before its last rounding, and ``rel`` a probability relative to
    itself: with u = 2^-23 (a truncating accumulator's step) a score is off by at most d = (head_dim + 2) u max_j
    scale sum|q k_j|; a probability by a factor within 1 +- (2 d + exp_err) (d in the score and d in the sum it is
    divided by; exp_err covers the exponential and, for bf16, probabilities carried in two bf16 parts: 2^-17; for
    fp32 an exponential of two units in the last place: 2^-21), and a sum of n products by n u of the sum of their
    magnitudes, in the numerator and in the denominator.
    """
    hq, hd = q.shape[1:]
    hkv = k_pages.shape[1]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    got = []
    for b, n in enumerate(lengths):
        if n == 0:
            got.append((np.zeros((hq, hd)), np.zeros((hq, 0)), np.zeros((hq, hd)), 0.0))
            continue
        k, v = (np.repeat(slots(p, table[b], n).astype(np.float64), hq // hkv, 0) for p in (k_pages, v_pages))
        qb = q[b].astype(np.float64)
        with np.errstate(invalid="ignore"):
            s = np.einsum("hd,hnd->hn", qb, k) * scale
            mag = np.einsum("hd,hnd->hn", np.abs(qb), np.where(np.isfinite(k), np.abs(k), 0)).max() * scale
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        u = 2.0**-23
        rel = 2 * (hd + 2) * u * mag + exp_err + 2 * n * u
        got.append((np.einsum("hn,hnd->hd", p, v), p, rel * np.einsum("hn,hnd->hd", p, np.abs(v)), rel))
    return got


def evict(n, next_position, weights, positions, budget, recent, sink):
    """One row and head: the slot each of the first min(n, budget) slots takes its token from."""
    if n <= budget:
        return np.arange(n)
    w = weights[:n].astype(np.float64)
    w = np.where(np.isnan(w), -np.inf, w)
    must = (positions[:n] >= next_position - recent) | (positions[:n] < sink)
    # protected first, then numbers by weight, then NaN; of equals the lower slot
    rank = np.lexsort((np.arange(n), -w, np.isnan(weights[:n]), ~must))
    keep = np.zeros(n, bool)
    keep[rank[:budget]] = True
    src = np.arange(budget)
    src[~keep[:budget]] = np.nonzero(keep[budget:])[0] + budget
    return src


def beam_select(logits, scores, k, done=None, eos=-1, pad=0):
    """(scores, parents, tokens, done) of one batch entry: logits [beams, vocab]."""
    beams, vocab = logits.shape
    cand = []
    for w in range(beams):
        if not np.isfinite(scores[w]):
            continue
        if done is not None and done[w]:
            cand.append((-float(scores[w]), w * vocab + pad))
            continue
        x = logits[w].astype(np.float64)
        x[~np.isfinite(x)] = -np.inf
        if np.isinf(x).all():
            continue
        top = x.max()
        # (the maximum first: at logits of 1e38 the sum's logarithm would be lost beside it)
        c = float(scores[w]) + ((x - top) - math.log(np.exp(x - top).sum()))
        at = np.nonzero(np.isfinite(c))[0]
        at = at[np.lexsort((at, -c[at]))][:k]
        cand += [(-c[t], w * vocab + int(t)) for t in at]
    cand = sorted(cand)[:k]
    out = [(-s, f // vocab, f % vocab, int((done is not None and bool(done[f // vocab])) or f % vocab == eos)) for s, f in cand]
    out += [(-np.inf, 0, pad, 1)] * (k - len(out))
    return tuple(np.array(c) for c in zip(*out))


def beam_reorder(pages, table, length, parents):
    """(pages, table) of one batch entry after its beams follow ``parents``; pages [blocks, num_pages, ...]."""
    pages, out, ps = pages.copy(), table.copy(), pages.shape[3]
    full, fill = length // ps, length % ps
    free = [w for w in range(len(parents)) if w not in set(parents.tolist())]
    seen = set()
    for j, p in enumerate(parents):
        out[j, :full] = table[p, :full]
        if not fill:
            continue
        if p not in seen:
            seen.add(p)
            out[j, full] = table[p, full]
        else:
            out[j, full] = table[free.pop(0), full]
            pages[:, out[j, full], :, :fill] = pages[:, table[p, full], :, :fill]
    return pages, out
