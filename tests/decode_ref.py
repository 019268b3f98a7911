"""Plain NumPy forms, in 64 bits, of the operators of text generation, and values in 16-bit types."""
import numpy as np

F32, F16, BF16 = 0, 1, 2
# half a step of rounding to the type, relative
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def encode(x, kind):
    """float -> the bytes of `kind`, to nearest even."""
    x = np.ascontiguousarray(x, np.float32)
    if kind == F32:
        return x.copy()
    if kind == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def decode(a, kind):
    if kind == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def np_type(kind):
    return {F32: np.float32, F16: np.float16, BF16: np.uint16}[kind]


def plan(cached, added, free, table, blocks, bs, max_blocks, max_tokens):
    """Request after request, as reef_c.h says it."""
    table = table.copy()
    lengths, starts, slots = [], [0], np.full(max_tokens, -1, np.int64)
    tokens = needs = used = refused = 0
    for i, (c, a) in enumerate(zip(cached, added)):
        c, a = max(int(c), 0), max(int(a), 0)
        first, tokens = tokens, tokens + a
        have, need = -(-c // bs), -(-(c + a) // bs) - -(-c // bs)
        ok = c + a <= max_blocks * bs and tokens <= max_tokens
        if ok:
            needs += need
            ok = need == 0 or needs <= len(free)
        if ok:
            used = needs
        if ok and need:
            table[i, have:have + need] = free[needs - need:needs]
        if ok:
            for k in range(a):
                b = int(table[i, (c + k) // bs])
                slots[first + k] = b * bs + (c + k) % bs if 0 <= b < blocks else -1
        refused += not ok
        lengths.append(c + a if ok else c)
        starts.append(min(tokens, max_tokens))
    return table, lengths, starts, slots, [used, min(tokens, max_tokens), refused]


def attend(q, k_rows, v_rows, scale):
    """q [heads][dim], k_rows, v_rows [kv][tokens][dim] -> (out, lse, a bound on |error| of out and of lse in 32-bit arithmetic).

    The bound: a score is a sum of `dim` products in 32 bits, off by at most e = (dim + 4) 2^-24 scale sum |q k| (the scale and the
    subtraction of the maximum among them, with one more rounding of |s - max| each, which is at most 2 max|s|); a weight exp(s) by a
    factor of 1 + e and a few roundings, of which the argument's conversion to a power of two counts |s - max|; numerator and
    denominator by the weights' errors and by a rounding for each of n additions.  Every bound is times max|v| for out."""
    heads, dim = q.shape
    kv, n, _ = k_rows.shape
    out, lse = np.zeros((heads, dim)), np.full(heads, -np.inf)
    tol_out, tol_lse = np.zeros((heads, 1)), np.zeros(heads)
    if n == 0:
        return out, lse, tol_out, tol_lse
    u = 2.0 ** -24
    for h in range(heads):
        k, v = k_rows[h // (heads // kv)], v_rows[h // (heads // kv)]
        s = k @ q[h] * scale
        m = s.max()
        if m == -np.inf:
            continue
        p = np.exp(s - m)
        out[h], lse[h] = p @ v / p.sum(), m + np.log(p.sum())
        e = (dim + 4) * u * (np.abs(k) @ np.abs(q[h])).max() * abs(scale) + 8 * u * np.abs(s[np.isfinite(s)]).max()
        tol_out[h] = (2 * e + (2 * n + 16) * u) * np.abs(v).max()
        tol_lse[h] = e + (n + 16) * u + u * abs(lse[h]) * 2
    return out, lse, tol_out, tol_lse


def select(logits, scores, ended, beams, n, end_token):
    """logits [rows][vocab] float64 -> (best, parents, tokens), [requests][n]."""
    rows, vocab = logits.shape
    offers = np.empty((rows, vocab))
    with np.errstate(all="ignore"):
        for r in range(rows):
            m = logits[r].max()
            offers[r] = scores[r] + (logits[r] - (m + np.log(np.exp(logits[r] - m).sum())))
            if ended is not None and ended[r]:
                offers[r] = -np.inf
                if 0 <= end_token < vocab:
                    offers[r, end_token] = scores[r]
    offers = np.where(np.isfinite(offers), offers, -np.inf).reshape(rows // beams, beams * vocab)
    at = np.argsort(-offers, axis=1, kind="stable")[:, :n]
    best = np.take_along_axis(offers, at, 1)
    return best, at // vocab + np.arange(rows // beams)[:, None] * beams, at % vocab
