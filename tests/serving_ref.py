"""Plain NumPy forms, in 64 bits, of the operators that serve many requests over a paged cache."""
import numpy as np

from tests.decode_ref import BF16, F16, F32, HALF


def chunk(q, k_rows, v_rows, cached, n, scale, window, kind, cache, there=None):
    """q [new][heads][dim] at places cached, cached + 1, ...; k_rows, v_rows [kv][n][dim]; there [n]: which tokens are in blocks of the pool
    -> (out, lse, a bound on |error| of out and of lse).

    The bound.  A score is a sum of `dim` products in 32 bits, off by at most e = (dim + 4) 2^-24 |scale| sum |q k|, with a few roundings of the
    score itself; where 32-bit values are held as terms of a 16-bit type, the terms leave out 2^-22 of each product at most (two terms of
    fp16: 2^-22; three of bf16: 2^-24, and products of terms below 2^-23).  A weight is off by a factor of 1 + e and a few roundings, numerator and
    denominator by a rounding for each of n additions.  In 16-bit types a weight is rounded once more for its product with a value, by half a step
    of the type, or half a step of fp16's smallest numbers, 2^-25, where the largest weight is 2^5 at least; in terms by 2^-22."""
    new, heads, dim = q.shape
    kv = k_rows.shape[0]
    out, lse = np.zeros((new, heads, dim)), np.full((new, heads), -np.inf)
    tol_out, tol_lse = np.zeros((new, heads, dim)), np.zeros((new, heads))
    u = 2.0 ** -24
    place = cached + np.arange(new)
    t = np.arange(n)
    seen = (t <= place[:, None]) & (place[:, None] < n)
    if window:
        seen &= t > place[:, None] - window
    if there is not None:
        seen &= there
    for h in range(heads):
        k, v = k_rows[h // (heads // kv)], v_rows[h // (heads // kv)]
        k, v = (np.where(seen.any(0)[:, None], x, 0) for x in (k, v))
        s = q[:, h] @ k.T * scale
        size = np.where(seen, np.abs(q[:, h]) @ np.abs(k).T * abs(scale), 0)
        s = np.where(seen, s, -np.inf)
        m = s.max(1) if n else np.full(new, -np.inf)
        some = m > -np.inf
        p = np.where(some[:, None], np.exp(s - np.where(some, m, 0)[:, None]), 0)
        l = p.sum(1)
        with np.errstate(all="ignore"):
            mean = p @ np.abs(v) / np.where(some, l, 1)[:, None]
            out[:, h] = p @ v / np.where(some, l, 1)[:, None]
            lse[:, h] = np.where(some, m + np.log(l), -np.inf)
        count = seen.sum(1)
        terms = 2.0 ** -21 if kind == F32 else 0.0
        top = np.where(seen, np.abs(np.where(seen, s, 0)), 0).max(1) if n else np.zeros(new)
        e = ((dim + 8) * u + terms) * (size.max(1) if n else 0) + 8 * u * top
        vmax = np.array([np.abs(v[i]).max() if i.any() else 0 for i in seen]) if n else np.zeros(new)
        tol_out[:, h] = ((2 * e + (2 * count + 32) * u) * vmax)[:, None]
        if kind == F32:
            tol_out[:, h] += 2.0 ** -21 * mean
        else:
            tol_out[:, h] += HALF[cache] * mean
        if cache == F16:
            tol_out[:, h] += (2.0 ** -30 * count * vmax)[:, None]
        tol_lse[:, h] = e + (count + 32) * u + 4 * u * np.abs(np.where(some, lse[:, h], 0))
    return out, lse, tol_out, tol_lse


def scores(logits, tokens, top):
    """logits [rows][vocab] float64 -> (scores, ranks, entropy, top_tokens, top_scores)."""
    rows, vocab = logits.shape
    x = np.where(np.isnan(logits), -np.inf, logits)
    m = x.max(1)
    none = ~np.isfinite(m)
    with np.errstate(all="ignore"):
        y = x - np.where(none, 0, m)[:, None]
        e = np.exp(np.where(none[:, None], -np.inf, y))
        log = np.where(none, np.nan, np.log(e.sum(1)))
        entropy = log - np.where(e > 0, e * y, 0).sum(1) / np.where(none, 1, e.sum(1))
    given = (tokens >= 0) & (tokens < vocab)
    at = np.where(given, tokens, 0)
    mine = x[np.arange(rows), at][:, None]
    ranks = ((x > mine) | ((x == mine) & (np.arange(vocab) < at[:, None]))).sum(1)
    score = np.where(given, y[np.arange(rows), at] - log, -np.inf)
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return score, np.where(given, ranks, -1), entropy, order, np.take_along_axis(y, order, 1) - log[:, None]


def held(n, max_blocks, bs):
    return min(max(int(n), 0), max_blocks * bs)


def sweep(table, lengths, blocks, bs, max_blocks):
    uses, outside = np.zeros(blocks, np.int64), 0
    for row, n in zip(table, lengths):
        b = row[:-(-held(n, max_blocks, bs) // bs)].astype(np.int64)
        inside = (b >= 0) & (b < blocks)
        np.add.at(uses, b[inside], 1)
        outside += int((~inside).sum())
    free = np.flatnonzero(uses == 0)
    return uses, free, [len(free), blocks - len(free), outside]


def fork(parents, children, tokens, free, table, lengths, blocks, bs, max_blocks):
    """-> (table, lengths, counts, [(source block, target block, tokens)])."""
    table, lengths, new = table.copy(), np.array(lengths, np.int64), []
    rows, needs, refused = len(table), 0, 0
    for p, c, n in zip(parents, children, tokens):
        if not (0 <= p < rows and 0 <= c < rows) or p == c:
            refused += 1
            continue
        n = max(0, min(int(n), held(lengths[p], max_blocks, bs)))
        full, rest = divmod(n, bs)
        needs += rest > 0
        if rest and needs > len(free):
            refused += 1
            continue
        table[c, :full] = table[p, :full]
        if rest:
            source, target = int(table[p, full]), int(free[needs - 1])
            inside = 0 <= source < blocks and 0 <= target < blocks
            table[c, full] = target if inside else -1
            if inside:
                new.append((source, target, rest))
        lengths[c] = n
    return table, lengths, [min(needs, len(free)), refused], new


def compact(table, lengths, table_out, blocks, bs, max_blocks):
    """-> (table_out, counts, [(source block, target block)])."""
    uses, _, _ = sweep(table, lengths, blocks, bs, max_blocks)
    used = int((uses > 0).sum())
    source = np.flatnonzero(uses[used:] > 0)[::-1] + used
    target = np.flatnonzero(uses[:used] == 0)
    to = dict(zip(source.tolist(), target.tolist()))
    out = table_out.copy()
    for i, n in enumerate(lengths):
        for j in range(-(-held(n, max_blocks, bs) // bs)):
            out[i, j] = to.get(int(table[i, j]), int(table[i, j]))
    return out, [used, len(target)], list(to.items())
