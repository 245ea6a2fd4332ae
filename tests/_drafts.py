"""Plain restatements of the operators for drafted tokens, for their tests: trees, rotary positions in float64, attention
along a tree, and the walk that says which drafts stay."""
from __future__ import annotations

import numpy as np

from bobcat_amd.backend import NO_PARENT, NO_TOKEN


def random_tree(rng, n, width=4, roots=1):
    """Parents (-1 for none) of n tokens, each after its parent."""
    parents, children = [], [0] * n
    for i in range(n):
        free = [a for a in range(i) if children[a] < width]
        if i < roots or not free:
            parents.append(-1)
            continue
        at = free[int(rng.integers(len(free)))]
        children[at] += 1
        parents.append(at)
    return parents


def as_given(trees):
    """The trees as a plan takes them."""
    return [None if t is None else [NO_PARENT if a < 0 else a for a in t] for t in trees]


def chain(n):
    return list(range(-1, n - 1))


def depths(parents):
    out = []
    for a in parents:
        out.append(0 if a < 0 else out[a] + 1)
    return out


def ancestors(parents):
    """[n, n]: the tokens that each token sees, itself among them."""
    seen = np.zeros((len(parents), len(parents)), bool)
    for i, a in enumerate(parents):
        if a >= 0:
            seen[i] = seen[a]
        seen[i, i] = True
    return seen


def tree_attention(q, k, v, past, parents):
    """q [tokens, heads, hd] over k, v [past + tokens, kv, hd], in float64: what a query does not see is left out."""
    heads, kv = q.shape[1], k.shape[1]
    out, seen = np.empty(q.shape), ancestors(parents)
    for t in range(q.shape[0]):
        at = np.concatenate([np.arange(past), past + np.flatnonzero(seen[t])])
        for h in range(heads):
            with np.errstate(invalid="ignore", over="ignore"):
                s = k[at, h * kv // heads] @ q[t, h].astype(np.float64) / np.sqrt(q.shape[2])
                p = np.exp(s - s.max())
                out[t, h] = p @ v[at, h * kv // heads] / p.sum()
    return out


def rope(x, positions, frequencies, layout, magnitude=1.0, norm=None, eps=0.0):
    """Rows x [tokens, heads, hd] turned in float64, and the size of each pair (of others their element's)."""
    x = x.astype(np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
    n = len(frequencies)
    a = np.arange(n) * (2 if layout == "pairs" else 1)
    b = a + (1 if layout == "pairs" else n)
    angle = np.asarray(positions, np.float64)[:, None, None] * np.asarray(frequencies, np.float64)
    out, size = x.copy(), np.abs(x)
    out[..., a] = magnitude * (x[..., a] * np.cos(angle) - x[..., b] * np.sin(angle))
    out[..., b] = magnitude * (x[..., a] * np.sin(angle) + x[..., b] * np.cos(angle))
    size[..., a] = size[..., b] = abs(magnitude) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return out, size


def target(logits, temperature):
    """The probabilities of a row of logits, in float64."""
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    x = np.minimum(x, np.finfo(np.float32).max)
    p = np.zeros(x.size)
    if not (x > -np.inf).any():
        return p
    if not temperature > 0:
        p[np.argmax(x)] = 1
        return p
    with np.errstate(over="ignore", under="ignore"):
        p = np.exp((x - x.max()) / np.float64(temperature))
    return p / p.sum()


def verify(parents, logits, draft, tokens, uniforms, temperature, distinct):
    """One sequence's (kept, path, next, chances), by the definition."""
    n, vocab = len(parents), logits.shape[1]
    p_of = [target(row, temperature) for row in logits]
    point = draft is None or not temperature > 0
    chances = [0.0] + [p_of[parents[i]][tokens[i]] if tokens[i] < vocab else 0.0 for i in range(1, n)]
    path = [0]
    while True:
        p, q = p_of[path[-1]], None if point else draft[path[-1]].astype(np.float64)
        left, down = 1.0, None
        for c in [i for i in range(n) if parents[i] == path[-1]]:
            x = int(tokens[c])
            if point:
                q = np.zeros(vocab)
                q[x:x + 1] = 1
            px, qx = (p[x], q[x] / left) if x < vocab else (0.0, 1.0 if point else 0.0)
            if float(uniforms[c]) * qx < px:
                down = c
                break
            p = np.maximum(p - q / left, 0)
            p = p / p.sum() if p.sum() > 0 else p
            if distinct and not point:
                left -= qx * left
        if down is None:
            break
        path.append(down)
    last = path[-1]
    p = p if p.sum() > 0 else p_of[last]
    up = np.cumsum(p)
    past = np.flatnonzero((p > 0) & (up > float(uniforms[0]) * up[-1]))
    token = NO_TOKEN if not p.sum() > 0 else int(past[0]) if past.size else int(np.flatnonzero(p)[-1])
    chances[0] = 0.0 if token == NO_TOKEN else p_of[last][token]
    return len(path), path + [NO_TOKEN] * (n - len(path)), token, chances
