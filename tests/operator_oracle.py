"""Plain 64-bit restatements of the operators on device memory, from their
definitions in include/qd/qd_operators.h, and the error that each type and length
allows. CPU only."""
import math

import numpy as np
import torch

# What a rounding is off by at most, relative to the value; below the smallest normal number the step
# stays what it is there, eps times that number, and a rounding is off by at most half of it.
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
HALF_LEAST = {t: torch.finfo(t).eps * torch.finfo(t).smallest_normal / 2 for t in HALF_STEP}


def rotate(x, cos, sin, interleaved):
    """x [tokens, heads, dim] and tables [tokens, R / 2], 64 bits: the rotated x and the sum of the
    magnitudes of each element's products."""
    half = cos.shape[1]
    x = x.double().clone()
    size = x.abs()
    i = torch.arange(half)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cos.double()[:, None, :], sin.double()[:, None, :]
    a, b = x[..., first].clone(), x[..., second].clone()
    x[..., first], x[..., second] = a * c - b * s, b * c + a * s
    size[..., first], size[..., second] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return x, size


def rotate_bound(want, size, dtype):
    # Two products and a sum in FP32 (half a step each of at most `size`), one rounding to the type.
    return 3 * 2.0 ** -24 * size + HALF_STEP[dtype] * (want.abs() + 3 * 2.0 ** -24 * size) + HALF_LEAST[dtype]


def attention(q, k, v, table, lengths, scale):
    """out [rows, heads, dim] and the error allowed at each element."""
    rows, heads, dim = q.shape
    page, kv_heads = k.shape[1], k.shape[2]
    group = heads // kv_heads
    out = torch.zeros((rows, heads, dim), dtype=torch.float64)
    bound = torch.zeros_like(out)
    for r in range(rows):
        n = int(lengths[r])
        if n == 0:
            continue
        ids = table[r, : -(-n // page)].long()
        kk, vv = (x[ids].reshape(-1, kv_heads, dim)[:n].double() for x in (k, v))
        for h in range(heads):
            g = h // group
            products = kk[:, g] * q[r, h].double() * scale
            p = torch.softmax(products.sum(-1), 0)
            out[r, h] = p @ vv[:, g]
            # Scores: at most dim FP32 additions and three roundings of sum |q k| each, and
            # twice in the ratio; exponentials 2^-22 more, sums over at most n / 4 + 64
            # positions in turn, and (16 bits) what two numbers leave of a probability.
            score = (dim + 3) * 2.0 ** -24 * float(products.abs().sum(-1).max())
            weight = 2 * score + 2.0 ** -22 + 2 * (n / 4 + 64) * 2.0 ** -24
            if q.dtype != torch.float32:
                weight += HALF_STEP[q.dtype] ** 2
            bound[r, h] = weight * (p @ vv[:, g].abs()) + HALF_STEP[q.dtype] * out[r, h].abs() + HALF_LEAST[q.dtype]
            if q.dtype != torch.float32:
                # Small probabilities: the largest in the sum is 1 or more, each of n is off by the least
                # step's half, in the sum of products and in the sum that divides it.
                bound[r, h] += 2 * n * HALF_LEAST[q.dtype] * vv[:, g].abs().max(0).values
    return out, bound


class Exhausted(Exception):
    pass


def fork(table, lengths, parents, refs, append, page):
    """New (table, lengths, refs) as lists, and the (source, destination) pages copied."""
    rows, width = len(table), len(table[0]) if table else 0
    old = []
    for line in table:
        ids = []
        for p in line:
            if p < 0:
                break
            ids.append(p)
        old.append(ids)
    refs = list(refs)
    parents = list(range(rows)) if parents is None else parents
    size = [lengths[p] if p >= 0 else 0 for p in parents]
    new = [old[p][: -(-lengths[p] // page)] if p >= 0 else [] for p in parents]
    for line in old:
        for p in line:
            refs[p] -= 1
    for line in new:
        for p in line:
            refs[p] += 1
    goes_on = [append > 0 and parents[r] >= 0 and size[r] % page != 0 for r in range(rows)]
    holders = {}
    for r in range(rows):
        if goes_on[r]:
            holders.setdefault(new[r][-1], []).append(r)
    keeps = {p: h[0] for p, h in holders.items() if refs[p] == len(h)}
    free = [p for p, n in enumerate(refs) if n == 0]
    copies, at = [], 0
    for r in range(rows):
        if parents[r] < 0:
            continue
        if goes_on[r] and keeps.get(new[r][-1]) != r:
            if at == len(free):
                raise Exhausted
            copies.append((new[r][-1], free[at]))
            refs[new[r][-1]] -= 1
            refs[free[at]] += 1
            new[r][-1] = free[at]
            at += 1
        while len(new[r]) * page < size[r] + append:
            if at == len(free):
                raise Exhausted
            new[r].append(free[at])
            refs[free[at]] += 1
            at += 1
    return ([line + [-1] * (width - len(line)) for line in new],
            [size[r] + append if parents[r] >= 0 else 0 for r in range(rows)], refs, copies)


def select(logits, scores, done, eos, k):
    """Per group the sorted best k as (score, beam, token), and every continuation's score."""
    groups, beams, vocab = logits.shape
    x = logits.double().numpy().copy()
    x[np.isnan(x)] = -math.inf
    picked, every = [], []
    for g in range(groups):
        flat = np.full((beams, vocab), -math.inf)
        order = []
        for b in range(beams):
            s = float(scores[g, b])
            if not math.isfinite(s):
                continue
            if done is not None and done[g, b]:
                flat[b, eos] = s
                order.append((s, b, 0, eos))
                continue
            m = x[g, b].max()
            if m == -math.inf:
                continue
            if m == math.inf:
                d = np.where(x[g, b] == m, 0.0, -math.inf)
            else:
                d = x[g, b] - m
            flat[b] = s + (d - math.log(np.exp(d).sum()))
            best = np.argsort(-x[g, b], kind="stable")[:k]
            order += [(flat[b, t], b, rank, int(t)) for rank, t in enumerate(best) if flat[b, t] > -math.inf]
        order.sort(key=lambda e: (-e[0], e[1], e[2]))
        chosen = [(e[0], e[1], e[3]) for e in order[:k]]
        have = {(b, t) for _, b, t in chosen}
        for i in range(beams * vocab):
            if len(chosen) == k:
                break
            if (i // vocab, i % vocab) not in have:
                chosen.append((-math.inf, i // vocab, i % vocab))
        picked.append(chosen)
        every.append(flat)
    return picked, every


# Sums of exponentials: FP32 in runs of 32 terms, each exponential two steps off (its argument's
# product, its own rounding), 64 bits beyond; the score is rounded once more.
def select_bound(score):
    return 2.0 ** -24 * abs(score) + (32 + 4) * 2.0 ** -24
