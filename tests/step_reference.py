"""Plain restatements, in 64 bits, of the operators round the selection path (slot maps, rotary positions, attention over
slots, draft verification). NumPy on host arrays; they follow the definitions in include/kvip_b200.h."""
import math

import numpy as np

RANGE, NO_SLOT, SOURCE = 1, 4, 64


def slot_maps(lengths, counts, held, table, free, head, *, block, tokens, queries=0):
    """Returns a dict of the outputs of KvipSlotMapsArgs; `table` is copied."""
    batch, pages = table.shape
    table = table.copy()
    status, off, number = 0, 0, 0
    available = len(free) - head if head >= 0 else 0
    positions, slots = np.full(tokens, -1, np.int64), np.full(tokens, -1, np.int64)
    requests = np.full(tokens, -1, np.int32)
    starts, ends, after = np.zeros(batch + 1, np.int32), np.array(lengths, np.int32), np.array(held, np.int32)
    taken = 0
    numbered = [0] * batch
    for b in range(batch):
        n, length, own = int(counts[b]), int(lengths[b]), int(held[b])
        starts[b] = min(number, tokens)
        if n < 0 or length < 0 or own < 0 or own > pages or length + n > pages * block or (queries and n > queries):
            status |= RANGE
            n = 0
        numbered[b] = n
        need = -(-(length + n) // block) if n else 0
        fresh = max(0, need - own)
        placed = fresh == 0 or off + fresh <= available
        if not placed:
            status |= NO_SLOT
        else:
            for j in range(fresh):
                table[b, own + j] = free[head + off + j]
            after[b] = own + fresh
            ends[b] = length + n
            if fresh:
                taken = off + fresh
        for i in range(n):
            t = number + i
            if t >= tokens:
                status |= RANGE
                break
            requests[t] = b
            if placed:
                p = length + i
                positions[t] = p
                block_number = int(table[b, p // block])
                slots[t] = block_number * block + p % block if block_number >= 0 else -1
        number += n
        off += fresh
    starts[batch] = min(number, tokens)
    out = dict(positions=positions, slot_mapping=slots, requests=requests, starts=starts, ends=ends, held_after=after,
               taken=np.array([taken], np.int32), table=table, status=np.array([status], np.int32))
    if queries:
        layout = np.zeros((4, batch * queries), np.int64)
        number = 0
        for b in range(batch):
            for q in range(numbered[b]):
                layout[0, b * queries + q] = number
                layout[1, b * queries + q] = 1
                layout[2, number] = b * queries + q
                number += 1
        layout[3, :number] = 1
        out["layout"] = layout
    return out


def rotary_frequencies(width, base=10000.0, scaling=None):
    i = np.arange(width // 2, dtype=np.float64)
    f = base ** (-2 * i / width)
    if scaling is None:
        return f, 1.0
    if scaling["kind"] == "linear":
        return f / scaling["factor"], 1.0
    at = [width * math.log(scaling["original"] / (beta * 2 * math.pi)) / (2 * math.log(base))
          for beta in (scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0))]
    low, high = max(0, math.floor(at[0])), min(width - 1, math.ceil(at[1]))
    share = np.clip((i - low) / max(high - low, 1e-3), 0, 1)
    factor = scaling.get("attention_factor")
    return f * (1 - share) + f / scaling["factor"] * share, 0.1 * math.log(scaling["factor"]) + 1 if factor is None else factor


def rotary(x, positions, width, layout, base=10000.0, scaling=None):
    """x float64 [tokens, heads, dim]: the first `width` elements of every row turned. Returns (y, size), size the sum of
    the absolute values of the pair an element belongs to (0 behind `width`)."""
    f, factor = rotary_frequencies(width, base, scaling)
    angle = positions.astype(np.float64)[:, None, None] * f
    c, s = np.cos(angle) * factor, np.sin(angle) * factor
    half = width // 2
    a, b = (slice(0, half), slice(half, width)) if layout == "half" else (slice(0, width, 2), slice(1, width, 2))
    y, size = x.copy(), np.zeros_like(x)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * factor
    return y, size


def attention(query, rows, scale):
    """One token: query [heads, 576], rows [n, 576] float64. Returns (out [heads, 512], lse, weight), weight = the
    softmax-weighted sum of absolute values: what relative errors of the weights are multiplied with."""
    heads = query.shape[0]
    if len(rows) == 0:
        return np.zeros((heads, 512)), np.full(heads, -np.inf), np.zeros((heads, 512)), 0.0
    logits = query @ rows.T * scale
    top = logits.max(1, keepdims=True)
    p = np.exp(logits - top)
    total = p.sum(1, keepdims=True)
    size = (np.abs(query) @ np.abs(rows).T).max() * abs(scale)
    return p @ rows[:, :512] / total, (top + np.log(total))[:, 0], p @ np.abs(rows[:, :512]) / total, size


def verify(target, draft, tokens, parents, starts, accept, sample, depth):
    """Returns (tokens, nodes, counts, status)."""
    batch, vocabulary = len(starts) - 1, target.shape[1]
    clean = lambda x: np.where(x > 0, x.astype(np.float64), 0.0)  # noqa: E731  (NaN and negative values count as nothing)
    out_tokens, out_nodes = np.full((batch, depth + 1), -1, np.int64), np.full((batch, depth + 1), -1, np.int32)
    counts, status = np.zeros(batch, np.int32), 0
    for b in range(batch):
        first, n = int(starts[b]), int(starts[b + 1]) - int(starts[b])
        if first < 0 or n < 0 or first + n > len(target):
            status |= RANGE
            continue
        if n == 0:
            continue
        if n > 64:
            n, status = 64, status | RANGE
        usable = [False] * n
        for j in range(1, n):
            usable[j] = 0 <= tokens[first + j] < vocabulary and 0 <= parents[first + j] < j
            status |= 0 if usable[j] else RANGE
        node, length = 0, 0
        out_nodes[b, 0] = 0
        while True:
            r, z, found = clean(target[first + node]), 1.0, -1
            if length < depth:
                for child in range(node + 1, n):
                    if not usable[child] or parents[first + child] != node:
                        continue
                    t = int(tokens[first + child])
                    q = clean(draft[first + node]) if draft is not None else np.eye(1, vocabulary, t)[0]
                    if float(accept[first + child]) * q[t] * z < r[t]:
                        found = child
                        break
                    if draft is not None:
                        r = np.maximum(r - z * q, 0.0)
                    else:
                        r = r * (q == 0)
                    z = r.sum()
                    if z == 0:
                        r = clean(target[first + node])
                        break
            if found < 0:
                break
            out_tokens[b, length], node = tokens[first + found], found
            length += 1
            out_nodes[b, length] = found
        holds = np.flatnonzero(r > 0)
        last = holds[-1] if len(holds) else 0
        out_tokens[b, length] = min(np.searchsorted(np.cumsum(r), float(sample[b]) * r.sum(), side="right"), last)
        counts[b] = length + 1
    return out_tokens, out_nodes, counts, status
