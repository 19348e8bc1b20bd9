"""Plain forms of the operators of speculative decoding (include/consumer_int8_drafts.h), on the CPU
in 64 bits, with what error bounds are made of."""

import numpy as np

LIMIT = 64  # rows of a sequence that are drafted at once


def ancestors(parents):
    """Of each row, itself and its ancestors, the last first."""
    chains = []
    for i, parent in enumerate(parents):
        chains.append([i] + (chains[parent] if 0 <= parent < i else []))
    return chains


def tree_seen(parents, context, window=0):
    """Bool [n, context]: which of the tokens 0 .. context-1 each row of a tree of n rows sees, row i
    being token context - n + i. A window counts positions: a row's is context - n + its depth."""
    n = len(parents)
    first = context - n
    seen = np.zeros((n, context), dtype=bool)
    for i, chain in enumerate(ancestors(parents)):
        reach = window or context + n + 1
        position = first + len(chain) - 1
        seen[i, max(0, position - reach + 1):max(0, first)] = True
        for a in chain[:reach]:
            if first + a >= 0:
                seen[i, first + a] = True
    return seen


def attention64(q, k, v, seen, scale):
    """oracle.attention.attention64 with any mask `seen` [R, C]."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    with np.errstate(all="ignore"):
        s = np.where(seen, q @ k.T * scale, -np.inf)
        off = np.where(seen, (np.abs(q) @ np.abs(k).T) * abs(scale), 0) * (k.shape[1] + 2) * 2.0**-24
        top = s.max(-1, keepdims=True, initial=-np.inf)
        top = np.where(np.isneginf(top), 0, top)
        w = np.exp(s - top)
        total = w.sum(-1, keepdims=True)
        p = np.where(seen, w / np.where(total == 0, 1, total), 0)
        lse = np.log(total[:, 0]) + top[:, 0]
    return p @ v, lse, p @ np.abs(v), off.max(-1, initial=0)


def token_probs64(logits, temperature):
    """Rows of probabilities, and how far the operator's FP32 values may be.

    Weights are exp2((l - m) c): the difference, c's division and its constant, and the product each
    round by 2^-24 of the exponent z, the exponential by 2^-23; those below 2^-126 are 0. Their sum has
    the weighted mean of these errors, and 2^-24 for each of its steps: a thread adds its values' eights
    one after the other, of 256 threads at least (2048 values a step), in chains of 5, then come waves,
    workgroups and chunks with one factor each. Two more roundings scale the weights."""
    x = np.asarray(logits, dtype=np.float64)
    rows, vocab = x.shape
    p, bound = np.zeros_like(x), np.zeros_like(x)
    for i, t in enumerate(np.broadcast_to(np.asarray(temperature, dtype=np.float64), rows)):
        row = x[i]
        if np.isnan(row).any() or not t >= 0 or (t > 0 and np.isposinf(row).any()):
            p[i] = np.nan
            continue
        if np.isneginf(row).all():
            continue
        if t == 0:
            p[i, int(np.argmax(row))] = 1
            continue
        with np.errstate(over="ignore", invalid="ignore"):
            z = np.where(np.isneginf(row), -np.inf, (row - row.max()) / t)
        w = np.exp(z)
        p[i] = w / w.sum()
        size = np.where(p[i] > 0, np.abs(np.where(np.isneginf(z), 0, z)), 0)
        steps = vocab / 2048 + 64
        one = 4 * 2.0**-24 * size + 2.0**-23
        bound[i] = p[i] * (one + (p[i] * one).sum() + (steps + 4) * 2.0**-24) + 2.0**-125
    return p, bound


def _clean(x):
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(invalid="ignore"):
        return np.where((x > 0) & np.isfinite(x), x, 0.0)


def _number(u):
    return 0.0 if np.isnan(u) else min(max(float(u), 0.0), 1 - 2.0**-24)


def verify(target, draft, tokens, parents, uniforms):
    """One sequence: (path, next token, margin). Rejection by the definition: what is left after each is
    made to sum to 1. margin: by how much of its terms the closest comparison was decided, times what
    is left where that is less than 1 (it is a difference of numbers near 1); results that round otherwise
    agree wherever it is more than their rounding."""
    n, vocab = min(len(tokens), LIMIT), np.shape(target)[1]
    if n == 0:
        return [], -1, 1.0
    if parents is None:
        parents = np.arange(-1, n - 1)
    path, row, margin = [0], 0, 1.0
    left = _clean(target[0])
    scale = 1.0
    taken = 0.0
    for i in range(1, n):
        if parents[i] != row:
            continue
        x, u = int(tokens[i]), _number(uniforms[i])
        inside = 0 <= x < vocab
        w = left[x] if inside else 0.0
        size = w
        if draft is None:
            level = u * scale
        else:
            q = _clean(draft[row])
            level = u * scale * (q[x] if inside else 0.0)
            size = w + 2 * taken * (q[x] if inside else 0.0)
        if level + size > 0 and scale > 0:  # nothing against nothing is decided exactly
            margin = min(margin, abs(level - w) / (level + size) * min(scale, 1))
        if level < w:
            path.append(i)
            row, left, scale, taken = i, _clean(target[i]), 1.0, 0.0
        elif draft is None:
            scale -= w
            left = left.copy()
            if inside:
                left[x] = 0
        else:
            taken += scale
            left = np.maximum(_clean(target[row]) - taken * q, 0)
            scale = left.sum()
    if not left.sum() > 0:
        left = _clean(target[row])
    total = left.sum()
    if not total > 0:
        return path, -1, margin
    sums, level = np.cumsum(left), _number(uniforms[0]) * total
    following = int(np.argmax(sums > level))
    if level == 0:  # the first weight above 0: by how much of its terms it is
        terms = _clean(target[row])[following]
        return path, following, min(margin, left[following] / (2 * terms - left[following]))
    # how near the level is to the sums of the token's neighbours
    near = min(sums[following] - level, level - (sums[following] - left[following]))
    return path, following, min(margin, near / total * min(total, 1))


def move(values, rows, slots, starts):
    """`values` [slots, ...] after the moves, in order."""
    values = values.copy()
    for begin, end in zip(starts[:-1], starts[1:]):
        for i in range(end - begin):
            source = int(rows[begin + i])
            if i < source < end - begin:
                a, b = int(slots[begin + source]), int(slots[begin + i])
                if 0 <= a < len(values) and 0 <= b < len(values):
                    values[b] = values[a]
    return values
