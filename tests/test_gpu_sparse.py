"""Bounds of pages and attention over chosen pages against their 64-bit restatements
(drafts_oracle.py)."""
import math

import pytest
import torch

import drafts_oracle as oracle
import qd_operators as ops
from test_gpu_drafts import on_gpu, pool
from test_gpu_operators import BF16, F16, F32, NAN, close, int32, normal, say, seeded, tables_for

pytestmark = pytest.mark.gpu


def run_bounds(k, table, lengths, recent, before, errors=0):
    kc = on_gpu(k)
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = before.cuda()
    ops.page_bounds(ops.PagedCache(kc, kc, table.cuda(), int32(lengths).cuda(), error), got, recent)
    assert int(error) == errors
    return got.cpu()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kv_heads,dim,page,layout", [(2, 64, 16, "token"), (3, 128, 32, "head"), (1, 128, 64, "wide"), (2, 64, 256, "head"), (1, 128, 1024, "token")])
@pytest.mark.parametrize("recent", [0, 1, 2, 17, 100000])
def test_bounds(dtype, kv_heads, dim, page, layout, recent):
    say("bounds", dtype, kv_heads, dim, page, layout, recent)
    g = seeded(page + recent)
    lengths = [0, 1, page - 1, page, page + 1, 2 * page + 16, 3 * page]
    table, pages = tables_for(g, lengths, page, 4)
    k = pool(g, pages, page, kv_heads, dim, dtype, layout)[0]
    before = normal(g, (pages, kv_heads, 2, dim), dtype)
    assert torch.equal(run_bounds(k, table, lengths, recent, before), oracle.bounds(k, table, lengths, recent, before))


def test_bounds_of_values_that_are_not_finite():
    g = seeded(3)
    for dtype in (F32, BF16, F16):
        k = normal(g, (2, 16, 1, 64), dtype)
        k[0, 3, 0, 5], k[0, 4, 0, 6], k[0, 5, 0, 6], k[0, :, 0, 7] = NAN, math.inf, -math.inf, NAN
        k[1, 9:] = NAN  # behind the row
        got = run_bounds(k, int32([[0, 1]]), [25], 1000, torch.zeros((2, 1, 2, 64), dtype=dtype))
        assert torch.equal(got, oracle.bounds(k, int32([[0, 1]]), [25], 1000, torch.zeros((2, 1, 2, 64), dtype=dtype)))
        assert got[0, 0, :, 7].tolist() == [math.inf, -math.inf] and torch.isfinite(got[1]).all()


def test_bounds_of_bad_rows_and_shared_pages():
    g = seeded(4)
    k = normal(g, (6, 16, 2, 64), F32)
    before = torch.zeros((6, 2, 2, 64))
    table = int32([[0, 1, -1], [0, 2, -1], [3, 6, 4], [5, 5, 5], [5, 5, 5]])
    got = run_bounds(k, table, [20, 20, 48, -1, 49], 1000, before, ops.BAD_PAGE | ops.BAD_LENGTH)
    want = oracle.bounds(k, int32([[0, 1, -1], [0, 2, -1], [3, 4, -1]]), [20, 20, 32], 1000, before)
    assert torch.equal(got, want)


def page_bounds_of(k, table, lengths):
    return oracle.bounds(k, table, lengths, 1 << 30, torch.zeros((k.shape[0], k.shape[2], 2, k.shape[3]), dtype=k.dtype))


def run_sparse(q, k, v, low_high, table, lengths, budget, first, last, scale, errors=0, out=None, chosen=True):
    rows, heads, dim = q.shape
    kv_heads = k.shape[2]
    kc, vc, qc = (on_gpu(x) for x in (k, v, q))
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = ops.PagedCache(kc, vc, table.cuda(), int32(lengths).cuda(), error)
    w = ops.Workspace(ops.sparse_attention_workspace(rows, heads, kv_heads, dim, table.shape[1], budget))
    out = torch.full_like(qc, NAN) if out is None else out(qc)
    ids = torch.full((rows, kv_heads, budget), 77, dtype=torch.int32, device="cuda") if chosen else None
    ops.sparse_attention(cache, low_high.cuda(), out, qc, w, budget, first=first, last=last, chosen=ids, scale=scale)
    assert int(error) == errors
    return out.cpu(), ids.cpu() if chosen else None


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,layout", [(14, 2, 64, 16, "token"), (4, 4, 128, 32, "head"), (20, 1, 128, 16, "wide"), (3, 3, 64, 64, "token")])
@pytest.mark.parametrize("budget,first,last", [(1, 0, 1), (4, 1, 2), (9, 2, 1), (6, 3, 3), (40, 1, 1)])
def test_sparse_attention(dtype, heads, kv_heads, dim, page, layout, budget, first, last):
    say("sparse", dtype, heads, kv_heads, dim, page, layout, budget, first, last)
    g = seeded(heads + budget)
    lengths = [0, 1, page, 4 * page, 4 * page + 1, 9 * page - 1, 23 * page + 5, 31 * page]
    table, pages = tables_for(g, lengths, page, 33)
    k, v = pool(g, pages, page, kv_heads, dim, dtype, layout)
    q = normal(g, (len(lengths), heads, dim), dtype, 1.5)
    low_high = page_bounds_of(k, table, lengths)
    want, bound, ids = oracle.sparse_attention(q, k, v, low_high, table, lengths, dim ** -0.5, budget, first, last)
    out, chosen = run_sparse(q, k, v, low_high, table, lengths, budget, first, last, None)
    assert torch.equal(chosen, ids)
    close(out, want, bound, "out")


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("pages,budget", [(700, 64), (4097, 130), (5000, 4990), (9000, 7)])
def test_sparse_attention_of_many_pages(dtype, pages, budget):
    """More than one share of the scores, more keys than are kept at hand."""
    say("many pages", dtype, pages, budget)
    g, page, kv_heads, dim, first, last = seeded(pages), 16, 2, 64, 1, 2
    k, v = pool(g, 500, page, kv_heads, dim, dtype)  # (pages are listed again and again: scores tie)
    table = torch.randint(0, 500, (2, pages), generator=g, dtype=torch.int32)
    lengths = [pages * page - 3, pages * page // 2 + 1]
    q = normal(g, (2, 4, dim), dtype)
    low_high = torch.stack([k.amin(1), k.amax(1)], 2)
    ids = torch.full((2, kv_heads, budget), -1, dtype=torch.int32)
    for r in range(2):
        for h in range(kv_heads):
            columns = oracle.choose(q[r], low_high, table[r], lengths[r], page, h, 2, budget, first, last)
            ids[r, h, : len(columns)] = int32(columns)
    out, chosen = run_sparse(q, k, v, low_high, table, lengths, budget, first, last, None)
    assert torch.equal(chosen, ids)
    want, bound, _ = oracle.sparse_attention(q, k, v, low_high, table, lengths, dim ** -0.5, budget, first, last)
    close(out, want, bound, "out")


def test_equal_scores_go_to_the_lower_page():
    g, page = seeded(5), 16
    k, v = pool(g, 3, page, 1, 64, F32)
    table = int32([[0, 1, 2, 1, 2, 1, 2, 1, 2, 0, 0]])
    q = normal(g, (1, 1, 64), F32)
    low_high = torch.stack([k.amin(1), k.amax(1)], 2)
    want, bound, ids = oracle.sparse_attention(q, k, v, low_high, table, [176], 0.125, 6, 1, 1)
    out, chosen = run_sparse(q, k, v, low_high, table, [176], 6, 1, 1, 0.125)
    assert torch.equal(chosen, ids)
    close(out, want, bound, "out")
    # All equal, among them 0 and -0.
    flat = torch.zeros_like(low_high)
    flat[1] = -0.0
    _, chosen = run_sparse(q, k, v, flat, table, [176], 6, 1, 1, 0.125)
    assert chosen.flatten().tolist() == [0, 1, 2, 3, 4, 10]


def test_scores_that_are_not_finite():
    g, page = seeded(6), 16
    k, v = pool(g, 20, page, 1, 64, F32)
    table = torch.arange(20, dtype=torch.int32)[None]
    q = normal(g, (1, 2, 64), F32)
    q[:, :, 0] = 0.0
    q[:, :, 1] = 1.0
    low_high = torch.stack([k.amin(1), k.amax(1)], 2)
    low_high[7, 0, 1, 0] = math.inf   # 0 x inf: no number
    low_high[11, 0, 1, 1] = math.inf
    low_high[13, 0, 1, 1] = -math.inf
    low_high[5, 0, 0, 2] = NAN
    for budget in (4, 5, 6, 18, 19):
        _, chosen = run_sparse(q, k, v, low_high, table, [320], budget, 1, 1, 0.125)
        assert chosen.flatten().tolist() == oracle.choose(q[0], low_high, table[0], 320, page, 0, 2, budget, 1, 1), budget
    q[0, 0, 3] = NAN
    out, chosen = run_sparse(q, k, v, low_high, table, [320], 4, 1, 1, 0.125)
    assert chosen.flatten().tolist() == [0, 1, 2, 19] and torch.isnan(out[0, 0]).all() and torch.isfinite(out[0, 1]).all()


def best_pages(q, low_high, table, pages, budget, first, last):
    """What a KV head with queries q [group, dim] and bounds [pages, 2, dim] reads, from the score's definition."""
    low, high = low_high[table.long(), 0].double(), low_high[table.long(), 1].double()
    score = sum(torch.maximum(x * low, x * high).sum(-1) for x in q.double())
    score = torch.where(torch.isnan(score), math.inf, score).tolist()
    middle = sorted(range(first, pages - last), key=lambda i: (-score[i], i))[: budget - first - last]
    return [*range(first), *sorted(middle), *range(pages - last, pages)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim,group", [(64, 1), (64, 3), (128, 2)])
@pytest.mark.parametrize("signs", ["above", "below", "both"])
def test_pages_whose_bounds_are_infinite(dtype, dim, group, signs):
    """Keys that are infinite or no number in single elements: the bounds of their pages, and what queries of one sign or
    of both make of them."""
    say("infinite bounds", dtype, dim, group, signs)
    g, page, pages, kv_heads = seeded(dim + group), 16, 30, 2
    k, v = pool(g, pages, page, kv_heads, dim, dtype)
    k[3, :, :, 5] = NAN            # no number: +inf and -inf
    k[5, 2, :, 6] = math.inf
    k[7, 2, :, 6] = -math.inf
    k[9, :, :, 7] = math.inf       # all keys
    k[11, :, :, 7] = -math.inf
    k[13, 1, :, 40], k[13, 2, :, 41] = math.inf, -math.inf
    k[15, 1, :, 40], k[15, 2, :, 40] = math.inf, -math.inf
    k[17, 1, 0, 50] = math.inf     # one head's alone
    k[19, :, 1] = NAN              # a head's whole page
    k[21, 4, :, 8] = NAN           # one key's
    q = normal(g, (1, kv_heads * group, dim), dtype).abs()
    if signs == "below":
        q = -q
    elif signs == "both":
        q[:, ::2, ::2] = -q[:, ::2, ::2]
    q[:, :, 41] = 0.0
    table = torch.randperm(pages, generator=g).to(torch.int32)[None]
    low_high = run_bounds(k, table, [pages * page], 1 << 20, torch.zeros((pages, kv_heads, 2, dim), dtype=dtype))
    for budget in (3, 5, 8, 11, 14, 20, 29):
        _, chosen = run_sparse(q, k, v, low_high, table, [pages * page], budget, 1, 1, 0.125)
        for h in range(kv_heads):
            want = best_pages(q[0, h * group: (h + 1) * group], low_high[:, h], table[0], pages, budget, 1, 1)
            assert chosen[0, h].tolist() == want, (budget, h)


def test_bad_rows():
    g, page = seeded(7), 16
    lengths = [320] * 5
    table, pages = tables_for(g, lengths, page, 20)
    k, v = pool(g, pages, page, 2, 64, F32)
    q = normal(g, (5, 4, 64), F32)
    low_high = page_bounds_of(k, table, lengths)
    want, bound, ids = oracle.sparse_attention(q, k, v, low_high, table, lengths, 0.125, 6, 1, 1)
    table[1, 4] = pages
    table[2, 19] = -1
    lengths[3], lengths[4] = -5, 321
    out, chosen = run_sparse(q, k, v, low_high, table, lengths, 6, 1, 1, 0.125, errors=ops.BAD_PAGE | ops.BAD_LENGTH)
    close(out[:1], want[:1], bound[:1], "out")
    assert torch.isnan(out[1:]).all()
    assert torch.equal(chosen[0], ids[0]) and (chosen[3:] == -1).all() and (chosen[1] == 4).any(-1).all()


def test_in_place_strides_and_without_the_list():
    g, page, lengths = seeded(8), 32, [300, 40, 0]
    table, pages = tables_for(g, lengths, page, 10)
    k, v = pool(g, pages, page, 2, 64, BF16)
    q = normal(g, (3, 8, 80), BF16)[:, 1:7, :64]
    low_high = page_bounds_of(k, table, lengths)
    want, bound, _ = oracle.sparse_attention(q, k, v, low_high, table, lengths, 0.125, 5, 1, 1)
    out, _ = run_sparse(q, k, v, low_high, table, lengths, 5, 1, 1, 0.125, out=lambda x: x, chosen=False)
    close(out, want, bound, "in place")


def test_a_budget_for_all_is_paged_attention():
    g, page, lengths = seeded(9), 16, [250, 31, 0, 160]
    table, pages = tables_for(g, lengths, page, 16)
    k, v = pool(g, pages, page, 2, 128, F16)
    q = normal(g, (4, 14, 128), F16)
    out, chosen = run_sparse(q, k, v, page_bounds_of(k, table, lengths), table, lengths, 16, 0, 1, None)
    cache = ops.PagedCache(k.cuda(), v.cuda(), table.cuda(), int32(lengths).cuda())
    want = torch.empty((4, 14, 128), dtype=F16, device="cuda")
    ops.paged_attention(cache, want, q.cuda(), ops.Workspace(ops.attention_workspace(4, 14, 2, 128)))
    assert torch.equal(out, want.cpu())
    assert (chosen >= 0).sum(-1)[:, 0].tolist() == [16, 2, 0, 10]


def test_a_step_in_a_graph_and_on_another_stream():
    """Append, bounds and attention over chosen pages, captured and replayed while lengths grow."""
    say("sparse in a graph")
    g, page, rows, heads, kv_heads, dim, budget = seeded(10), 16, 2, 4, 2, 64, 5
    start, steps = [150, 70], 20
    table, pages = tables_for(g, [n + steps for n in start], page, 12)
    k, v = pool(g, pages, page, kv_heads, dim, F32)
    kc, vc = k.cuda(), v.cuda()
    lengths = int32(start).cuda()
    cache = ops.PagedCache(kc, vc, table.cuda(), lengths)
    low_high = torch.zeros((pages, kv_heads, 2, dim), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ops.page_bounds(cache, low_high, 1 << 20, stream=side.cuda_stream)
    new = torch.zeros((rows, heads + 2 * kv_heads, dim), device="cuda")
    position = lengths.clone()
    out, q_out = (torch.zeros((rows, heads, dim), device="cuda") for _ in range(2))
    chosen = torch.zeros((rows, kv_heads, budget), dtype=torch.int32, device="cuda")
    w = ops.Workspace(ops.sparse_attention_workspace(rows, heads, kv_heads, dim, 12, budget))

    def step(stream):
        q, kn, vn = new.split([heads, kv_heads, kv_heads], 1)
        position.copy_(lengths)
        lengths.add_(1)
        ops.paged_append(cache, q_out, q, kn, vn, position, stream=stream)
        ops.page_bounds(cache, low_high, 1, stream=stream)
        ops.sparse_attention(cache, low_high, out, q_out, w, budget, first=1, last=1, chosen=chosen, stream=stream)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    for i in range(steps):
        x = normal(g, tuple(new.shape), F32)
        new.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        n = [s + i + 1 for s in start]
        for r in range(rows):
            k[int(table[r, (n[r] - 1) // page]), (n[r] - 1) % page] = x[r, heads: heads + kv_heads]
            v[int(table[r, (n[r] - 1) // page]), (n[r] - 1) % page] = x[r, heads + kv_heads:]
        want_bounds = page_bounds_of(k, table, n)
        held = sorted({int(p) for r in range(rows) for p in table[r, : -(-n[r] // page)]})
        assert torch.equal(low_high.cpu()[held], want_bounds[held])
        want, bound, ids = oracle.sparse_attention(x[:, :heads], k, v, want_bounds, table, n, 0.125, budget, 1, 1)
        assert torch.equal(chosen.cpu(), ids)
        close(out, want, bound, "out")
