"""The paged cache, attention over it and the verification of drafted tokens, in numpy and 64 bits, from their definitions.

No reference code restates these (the reference decodes one sequence from one contiguous cache and selects greedily)."""
import numpy as np


def places(starts, lengths, tokens):
    """(sequence, position) of each of the rows, (-1, -1) for one that belongs to no sequence."""
    out = [(-1, -1)] * tokens
    for b in range(len(lengths)):
        n = starts[b + 1] - starts[b]
        for i in range(n):
            out[starts[b] + i] = (b, int(lengths[b]) - n + i)
    return out


def row(pages, table, b, position):
    """[heads, dim] (or [heads] of scales) of a position."""
    page = pages.shape[2]
    return pages[table[b][position // page], :, position % page]


def gathered(pages, table, b, length):
    """[heads, length, ..]: what a sequence has in the pool."""
    return np.stack([row(pages, table, b, j) for j in range(length)], 1) if length else np.zeros((pages.shape[1], 0) + pages.shape[3:])


def attention(q, keys, values, positions, scale, window=0, steps=None):
    """One sequence: q [n, heads, dim], keys and values [kv_heads, length, dim] -> (o, sum_j p_j |v_j|, max_j (p_j t_j)
    sum_j |v_j| / t_j), all [n, heads, dim], with t the values' scales `steps` [kv_heads, length] (None: 1). A row sees
    positions max(0, p - window + 1) .. p; one that sees none gives zeros."""
    n, heads, dim = q.shape
    group = heads // keys.shape[0]
    o, size, tiny = (np.zeros((n, heads, dim)) for _ in range(3))
    steps = np.ones(values.shape[:2]) if steps is None else steps
    for i, p in enumerate(positions):
        lo = max(0, p - window + 1) if window else 0
        if p + 1 <= lo:
            continue
        for h in range(heads):
            k, v = keys[h // group, lo:p + 1], values[h // group, lo:p + 1]
            with np.errstate(all="ignore"):
                z = scale * (k @ q[i, h])
                w = np.exp(z - z.max())
                w /= w.sum()
                o[i, h], size[i, h] = w @ v, w @ np.abs(v)
                t = steps[h // group, lo:p + 1]
                tiny[i, h] = (w * t).max() * np.where(t[:, None] > 0, np.abs(v) / t[:, None], 0).sum(0)
    return o, size, tiny


def distribution(z, temperature):
    """softmax(z / temperature); below 1e-5 all on the first of the largest. None: no distribution."""
    z = z.astype(np.float64)
    if np.isnan(z).any() or (z == np.inf).any() or not np.isfinite(z.max()):
        return None
    if not temperature >= 1e-5:
        p = np.zeros(z.shape)
        p[int(np.argmax(z))] = 1
        return p
    p = np.exp((z - z.max()) / temperature)
    return p / p.sum()


def verify(target, drafted, uniform, draft=None, temperature=1.0, count=None):
    """One request: target [drafts + 1, vocab], drafted [drafts], uniform [drafts + 1], draft [drafts, vocab] or None ->
    (tokens [drafts + 1], accepted, logprobs [drafts + 1])."""
    drafts, vocab = len(drafted), target.shape[1]
    greedy = not temperature >= 1e-5
    tokens, logprobs = [-1] * (drafts + 1), [0.0] * (drafts + 1)
    count = drafts if count is None else min(max(count, 0), drafts)
    for i in range(count + 1):
        p = distribution(target[i], temperature)
        if p is None:
            return tokens, i, logprobs
        u, last, weight = float(uniform[i]), float(uniform[drafts]), p
        if i < count:
            d, keep = int(drafted[i]), False
            if greedy:
                keep = 0 <= d < vocab and p[d] == 1
            elif 0 <= d < vocab:
                if draft is None:
                    q = np.zeros(vocab)
                    q[d] = 1
                else:
                    q = distribution(draft[i], temperature)
                if q is not None:
                    keep = u * q[d] < p[d]
                    rest = np.where(q == 1, 0, p) if draft is None else np.maximum(p - q, 0)
                    weight = rest if draft is None or rest.sum() > 0 else p
            if keep:
                tokens[i], logprobs[i] = d, 0.0 if greedy else float(np.log(p[d]))
                continue
        if greedy:
            tokens[i] = int(np.argmax(p))
            return tokens, i, logprobs
        mass = np.cumsum(weight)
        if not mass[-1] > 0:
            return tokens, i, logprobs
        v = int(np.searchsorted(mass, last * mass[-1], side="right"))
        v = min(v, int(np.nonzero(weight)[0][-1]))
        tokens[i], logprobs[i] = v, float(np.log(p[v]))
        return tokens, i, logprobs
