"""Plain 64-bit restatements of the operators on trees of drafted tokens and on chosen
pages, from their definitions in include/qd/qd_operators.h. CPU only."""
import math

import torch

from operator_oracle import HALF_LEAST, HALF_STEP


def weighted(q, k, v, scale):
    """One query [dim] over keys and values [n, dim] of its type: the output and the error allowed at each
    element (as for the attention of one token: operator_oracle.attention)."""
    n, dim = k.shape
    kk, vv = k.double(), v.double()
    products = kk * q.double() * scale
    p = torch.softmax(products.sum(-1), 0)
    out = p @ vv
    score = (dim + 3) * 2.0 ** -24 * float(products.abs().sum(-1).max())
    weight = 2 * score + 2.0 ** -22 + 2 * (n / 4 + 64) * 2.0 ** -24
    if q.dtype != torch.float32:
        weight += HALF_STEP[q.dtype] ** 2
    bound = weight * (p @ vv.abs()) + HALF_STEP[q.dtype] * out.abs() + HALF_LEAST[q.dtype]
    if q.dtype != torch.float32:
        bound = bound + 2 * n * HALF_LEAST[q.dtype] * vv.abs().max(0).values
    return out, bound


def chain(parents, i):
    """Node i and the nodes above it, none if it is not there."""
    seen = []
    while i >= 0 and parents[i] >= -1:
        seen.append(i)
        i = parents[i]
    return seen[::-1]


def tree_attention(q, k, v, table, lengths, parents, scale):
    """q [rows, nodes, heads, dim], pages [pages, page, kv_heads, dim]."""
    rows, nodes, heads, _ = q.shape
    page, group = k.shape[1], heads // k.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for r in range(rows):
        n = int(lengths[r])
        if n == 0:
            continue
        ids = table[r, : -(-n // page)].long()
        kk, vv = (x[ids].flatten(0, 1)[:n] for x in (k, v))
        for i in range(nodes):
            seen = chain(parents[r].tolist(), i)
            if not seen:
                continue
            at = torch.tensor([*range(n - nodes), *(n - nodes + j for j in seen)])
            for h in range(heads):
                out[r, i, h], bound[r, i, h] = weighted(q[r, i, h], kk[at, h // group], vv[at, h // group], scale)
    return out, bound


def pick(x, draw, temperature):
    """The token that follows: x [vocab]."""
    x = x.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.max()
    if draw is None or not 1e30 > float(top) > -1e30:
        return int((x == top).nonzero()[0])
    upto = torch.cumsum(torch.exp((x - top) / temperature), 0)
    return int((upto <= draw * upto[-1]).sum())


def accept(logits, tokens, parents, draws, temperature=1.0):
    path, counts, following = [], [], []
    nodes = parents.shape[1]
    for r in range(parents.shape[0]):
        above, carry = parents[r].tolist(), tokens[r].tolist()
        walk, token, at = [], -1, 0 if above[0] >= -1 else None
        while at is not None:
            walk.append(at)
            token = pick(logits[r, at], None if draws is None else float(draws[r, at]), temperature)
            at = next((j for j in range(nodes) if above[j] == at and carry[j] == token), None)
        path.append(walk + [-1] * (nodes - len(walk)))
        counts.append(len(walk))
        following.append(token)
    return (torch.tensor(x, dtype=torch.int32) for x in (path, counts, following))


def bounds(k, table, lengths, recent, before):
    """k [pages, page, kv_heads, dim], before [pages, kv_heads, 2, dim]."""
    page, out = k.shape[1], before.clone()
    for r in range(len(lengths)):
        n = int(lengths[r])
        if recent == 0:
            continue
        for c in range(max(0, n - recent) // page, -(-n // page)):
            keys = k[int(table[r, c]), : min(page, n - c * page)]
            for side, fill in ((0, math.inf), (1, -math.inf)):
                x = torch.where(torch.isnan(keys), fill, keys.double())
                out[int(table[r, c]), :, side] = (x.amin(0) if side == 0 else x.amax(0)).to(k.dtype)
    return out


def choose(q, low_high, table, length, page, head, group, budget, first, last):
    """The columns that a row's KV head reads."""
    pages = -(-length // page)
    if pages <= budget:
        return list(range(pages))
    ids = table[first: pages - last].long()
    low, high = low_high[ids, head, 0].double(), low_high[ids, head, 1].double()
    below, above = (q[head * group: (head + 1) * group].double().clamp(**side).sum(0) for side in ({"max": 0}, {"min": 0}))
    score = (low * below + high * above).sum(-1)
    score = torch.where(torch.isnan(score), math.inf, score).tolist()
    best = sorted(range(len(score)), key=lambda i: (-score[i], i))[: budget - first - last]
    return [*range(first), *sorted(first + i for i in best), *range(pages - last, pages)]


def sparse_attention(q, k, v, low_high, table, lengths, scale, budget, first, last):
    rows, heads, _ = q.shape
    page, kv_heads = k.shape[1], k.shape[2]
    group = heads // kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros_like(out)
    chosen = torch.full((rows, kv_heads, budget), -1, dtype=torch.int32)
    for r in range(rows):
        n = int(lengths[r])
        if n == 0:
            continue
        for g in range(kv_heads):
            columns = choose(q[r], low_high, table[r], n, page, g, group, budget, first, last)
            chosen[r, g, : len(columns)] = torch.tensor(columns, dtype=torch.int32)
            ids = table[r, columns].long()
            m = len(columns) * page - (-n % page)
            kk, vv = (x[ids, :, g].flatten(0, 1)[:m] for x in (k, v))
            for h in range(g * group, (g + 1) * group):
                out[r, h], bound[r, h] = weighted(q[r, h], kk, vv, scale)
    return out, bound, chosen
