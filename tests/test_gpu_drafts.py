"""The operators on trees of drafted tokens against their 64-bit restatements
(drafts_oracle.py), at the sizes, trees and layouts where they can go wrong."""
import math

import pytest
import torch

import drafts_oracle as oracle
import qd_operators as ops
from test_gpu_operators import BF16, F16, F32, NAN, close, int32, normal, say, seeded, tables_for

pytestmark = pytest.mark.gpu


def tree(g, nodes, count=None):
    """Parents of a tree of `count` nodes among `nodes`."""
    count = nodes if count is None else count
    return [-1 if i == 0 else int(torch.randint(max(0, i - 4), i, (1,), generator=g)) for i in range(count)] + [-2] * (nodes - count)


def some_trees(g, rows, nodes):
    """A tree, a chain, one node, a tree with gaps that are no nodes, none."""
    all = []
    for r in range(rows):
        kind = r % 5
        if kind == 0:
            t = tree(g, nodes)
        elif kind == 1:
            t = [i - 1 for i in range(nodes)]
        elif kind == 2:
            t = tree(g, nodes, 1 + nodes // 2)
        elif kind == 3:
            t = [-1 if i < 2 else -2 if i % 3 == 0 else (i - 2 if (i - 2) % 3 or i == 2 else i - 1) for i in range(nodes)]
        else:
            t = [-2] * nodes
        all.append(t)
    return int32(all).reshape(rows, nodes)


def pool(g, pages, page, kv_heads, dim, dtype, layout="token"):
    """K and V with every unused element NaN-free; heads inside tokens, outside of them, or in wider rows."""
    if layout == "token":
        return [normal(g, (pages, page, kv_heads, dim), dtype) for _ in range(2)]
    if layout == "head":
        return [normal(g, (pages, kv_heads, page, dim), dtype).transpose(1, 2) for _ in range(2)]
    return [normal(g, (pages, page, kv_heads + 1, dim + 16), dtype)[:, :, :kv_heads, :dim] for _ in range(2)]


def on_gpu(x):
    """The same strides on the GPU."""
    y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda") if x.is_contiguous() else None
    if y is not None:
        return y.copy_(x)
    base = torch.zeros(x.untyped_storage().nbytes() // x.element_size(), dtype=x.dtype, device="cuda")
    return base.as_strided(x.shape, x.stride(), x.storage_offset()).copy_(x)


def run_tree(q, k, v, table, lengths, parents, scale, errors=None, out=None, workspace=None):
    rows, nodes, heads, dim = q.shape
    kc, vc, qc = (on_gpu(x) for x in (k, v, q))
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = ops.PagedCache(kc, vc, table.cuda(), int32(lengths).cuda(), error)
    w = workspace or ops.Workspace(ops.tree_attention_workspace(rows, nodes, heads, k.shape[2], dim))
    out = torch.full_like(qc, NAN) if out is None else out(qc)
    ops.tree_attention(cache, out, qc, parents.cuda(), w, scale=scale)
    torch.cuda.synchronize()
    if errors is None:
        assert int(error) == 0
    else:
        assert int(error) == errors
    return out


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,layout", [
    (14, 2, 64, 16, "token"), (4, 4, 128, 32, "head"), (3, 1, 128, 64, "wide"), (8, 1, 64, 1024, "head")])
@pytest.mark.parametrize("nodes", [1, 2, 9, 17, 64])
def test_tree_attention(dtype, heads, kv_heads, dim, page, layout, nodes):
    say("tree attention", dtype, heads, kv_heads, dim, page, layout, nodes)
    g = seeded(nodes * 3 + heads)
    # Lengths around the ends of steps, stages and pages; a tree alone; rows of nothing.
    lengths = [nodes, 0, nodes + 1, 31 + nodes, 64, 65, 127 + nodes, 128, 129, 200]
    lengths = [n if n >= nodes or n == 0 else n + nodes for n in lengths]
    table, pages = tables_for(g, lengths, page, max(1, -(-max(lengths) // page)))
    k, v = pool(g, pages, page, kv_heads, dim, dtype, layout)
    q = normal(g, (len(lengths), nodes, heads, dim), dtype, 1.5)
    parents = some_trees(g, len(lengths), nodes)
    want, bound = oracle.tree_attention(q, k, v, table, lengths, parents, 0.11)
    close(run_tree(q, k, v, table, lengths, parents, 0.11), want, bound, "out")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,nodes", [(2, 1, 64, 5), (7, 1, 128, 4), (16, 1, 64, 4), (4, 1, 128, 37)])
@pytest.mark.parametrize("lengths", [[2500], [900, 64, 0, 1300], [70] * 70 + [1100]])
def test_tree_attention_of_cut_rows(dtype, heads, kv_heads, dim, nodes, lengths):
    say("tree attention, cut", dtype, heads, kv_heads, dim, nodes, len(lengths))
    g = seeded(nodes + len(lengths))
    page = 32
    table, pages = tables_for(g, lengths, page, -(-max(lengths) // page) + 1)
    k, v = pool(g, pages, page, kv_heads, dim, dtype)
    q = normal(g, (len(lengths), nodes, heads, dim), dtype, 1.5)
    parents = some_trees(g, len(lengths), nodes)
    want, bound = oracle.tree_attention(q, k, v, table, lengths, parents, dim ** -0.5)
    close(run_tree(q, k, v, table, lengths, parents, None), want, bound, "out")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,nodes,page", [(2, 2, 64, 3, 16), (8, 2, 128, 4, 32), (8, 4, 64, 5, 64), (7, 1, 128, 9, 16)])
def test_tree_attention_of_many_rows(dtype, heads, kv_heads, dim, nodes, page):
    """Dealt in equal runs, cut where they end; rows that are bad spoil no others."""
    say("tree attention, many rows", dtype, heads, kv_heads, dim, nodes, page)
    g, rows = seeded(heads), 300 // kv_heads
    lengths = [int(n) for n in torch.randint(0, 500, (rows,), generator=g)]
    lengths[7], lengths[rows - 1], lengths[11] = 2900, 1700, 0
    lengths = [n if n >= nodes else 0 for n in lengths]
    table, pages = tables_for(g, lengths, page, -(-2900 // page))
    k, v = pool(g, pages, page, kv_heads, dim, dtype)
    q = normal(g, (rows, nodes, heads, dim), dtype, 1.5)
    parents = some_trees(g, rows, nodes)
    parents[7] = int32(tree(g, nodes))
    some = [0, 1, 2, 3, 4, 5, 6, 7, 8, 11, 12, 50, rows - 2, rows - 1]
    want, bound = oracle.tree_attention(q[some], k, v, table[some], [lengths[r] for r in some], parents[some], 0.1)
    close(run_tree(q, k, v, table, lengths, parents, 0.1)[some], want, bound, "out")
    table[9, 0], lengths[10], parents[13, -1] = pages, -4, nodes
    lengths[9] = max(lengths[9], nodes)
    lengths[13] = max(lengths[13], nodes)
    table[13, : -(-lengths[13] // page)] = table[7, : -(-lengths[13] // page)]
    got = run_tree(q, k, v, table, lengths, parents, 0.1, errors=ops.BAD_PAGE | ops.BAD_LENGTH | ops.BAD_PARENT)
    close(got[some], want, bound, "out beside bad rows")
    assert torch.isnan(got[[9, 10, 13]]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("scale", [-0.125, 0.0])
def test_scales_of_any_sign(dtype, scale):
    g, nodes, page, lengths = seeded(3), 9, 16, [150, 9]
    table, pages = tables_for(g, lengths, page, 10)
    k, v = pool(g, pages, page, 2, 64, dtype)
    q = normal(g, (2, nodes, 6, 64), dtype, 1.5)
    parents = some_trees(g, 2, nodes)
    want, bound = oracle.tree_attention(q, k, v, table, lengths, parents, scale)
    close(run_tree(q, k, v, table, lengths, parents, scale), want, bound, "out")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("length", [70, 1500])
@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
def test_what_is_not_seen_may_be_anything(dtype, length, bad):
    """K and V of nodes that are not seen, and behind the row; a V that is seen makes its readers not finite."""
    say("not seen", dtype, length, bad)
    g = seeded(length)
    nodes, heads, kv_heads, dim, page = 12, 4, 2, 64, 16
    table, pages = tables_for(g, [length], page, -(-length // page))
    k, v = pool(g, pages, page, kv_heads, dim, dtype)
    q = normal(g, (1, nodes, heads, dim), dtype)
    #        0
    #     1     2      5 and 6 are not there, 11 hangs below 1
    parents = int32([[-1, 0, 0, 1, 2, -2, -2, 3, 4, 4, 0, 1]])
    want, bound = oracle.tree_attention(q, k, v, table, [length], parents, 0.125)
    start = length - nodes

    def spoil(x, node, element=slice(None)):
        pos = start + node
        x[int(table[0, pos // page]), pos % page, :, element] = bad

    for x in (k, v):
        for n in (5, 6):
            spoil(x, n)
        if length % page:
            x[int(table[0, -1]), length % page:] = NAN
    spoil(k, 11)           # only node 11 itself sees it
    spoil(v, 2, 7)         # nodes 2, 4, 8, 9 do
    got = run_tree(q, k, v, table, [length], parents, 0.125).cpu()
    assert not torch.isfinite(got[0, [2, 4, 8, 9], :, 7]).any()
    clean = torch.ones(got.shape, dtype=torch.bool)
    clean[0, [2, 4, 8, 9], :, 7] = False
    clean[0, 11] = False
    got, want, bound = (torch.where(clean, x.double(), 0.0) for x in (got, want, bound))
    close(got, want, bound, "out")


def test_a_committed_value_that_is_not_finite_reaches_every_node():
    g = seeded(4)
    nodes, page = 5, 16
    table, pages = tables_for(g, [100], page, 7)
    k, v = pool(g, pages, page, 1, 64, F32)
    v[int(table[0, 1]), 3, 0, 9] = math.inf
    q = normal(g, (1, nodes, 2, 64), F32)
    got = run_tree(q, k, v, table, [100], int32([[-1, 0, 0, 1, 3]]), 0.125).cpu()
    assert not torch.isfinite(got[..., 9]).any()
    got[..., 9] = 0
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scores_of_any_size(dtype):
    """One weight holds all the rest up; the largest come last, first and far below zero."""
    say("scores of any size", dtype)
    g, nodes, page, length = seeded(6), 6, 64, 700
    for sign, where in ((1, 650), (1, 0), (-1, 0)):
        table, pages = tables_for(g, [length], page, 11)
        k, v = pool(g, pages, page, 1, 64, dtype)
        q = normal(g, (1, nodes, 3, 64), dtype)
        q[..., 0], k[..., 0] = 8.0, -4.0 if sign < 0 else 0.0
        if sign > 0:
            k[int(table[0, where // page]), where % page, 0, 0] = 24.0
        want, bound = oracle.tree_attention(q, k, v, table, [length], int32([[-1, 0, 1, 2, 0, 4]]), 0.5)
        close(run_tree(q, k, v, table, [length], int32([[-1, 0, 1, 2, 0, 4]]), 0.5), want, bound, (sign, where))


@pytest.mark.parametrize("length", [90, 2000])
def test_bad_rows_are_marked_and_no_others(length):
    g, nodes, page = seeded(5), 7, 16
    lengths = [length] * 6
    table, pages = tables_for(g, lengths, page, -(-length // page))
    k, v = pool(g, pages, page, 2, 64, F32)
    q = normal(g, (6, nodes, 4, 64), F32)
    parents = int32([[-1, 0, 1, 2, 0, 4, -2]] * 6)
    want, bound = oracle.tree_attention(q, k, v, table, lengths, parents, 0.125)
    parents[1, 3] = 3
    parents[2, 3] = 64
    parents[3, 5] = 6          # not there
    table[4, 2] = pages
    lengths[5] = nodes - 1
    got = run_tree(q, k, v, table, lengths, parents, 0.125, errors=ops.BAD_PARENT | ops.BAD_PAGE | ops.BAD_LENGTH)
    close(got[:1], want[:1], bound[:1], "out")
    assert torch.isnan(got[1:]).all()
    for bad, bits in ((-1, ops.BAD_LENGTH), (table.shape[1] * page + 1, ops.BAD_LENGTH)):
        got = run_tree(q[:1], k, v, table[:1], [bad], parents[:1], 0.125, errors=bits)
        assert torch.isnan(got).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_nothing_may_have_any_parents(dtype):
    """A row that only fills the batch: what its parents hold is not looked at."""
    g, nodes = seeded(25), 5
    lengths = [0, 40, 0, 0]
    table, pages = tables_for(g, lengths, 16, 4)
    k, v = pool(g, pages, 16, 2, 64, dtype)
    q = normal(g, (4, nodes, 4, 64), dtype)
    parents = int32([[7, -9, 4, 3, 100], tree(g, nodes), [1 << 30] * nodes, [-1, 0, 1, 2, 3]])
    want, bound = oracle.tree_attention(q[1:2], k, v, table[1:2], lengths[1:2], parents[1:2], 0.125)
    out = run_tree(q, k, v, table, lengths, parents, 0.125)
    close(out[1:2], want, bound, "out")
    assert (out[[0, 2, 3]] == 0).all()


def test_in_place_and_strides():
    g, nodes, page = seeded(8), 10, 32
    lengths = [300, 40, 0]
    table, pages = tables_for(g, lengths, page, 10)
    for dtype in (F32, BF16):
        k, v = pool(g, pages, page, 2, 64, dtype)
        wide = normal(g, (3, nodes + 1, 8, 80), dtype)
        q = wide[:, :nodes, 1:7, :64]
        parents = some_trees(g, 3, nodes)
        want, bound = oracle.tree_attention(q, k, v, table, lengths, parents, 0.125)
        close(run_tree(q, k, v, table, lengths, parents, 0.125, out=lambda x: x), want, bound, "in place")
        other = lambda x: torch.full((nodes, 6, 3, 72), NAN, dtype=dtype, device="cuda").permute(2, 0, 1, 3)[..., :64]  # noqa: E731
        close(run_tree(q, k, v, table, lengths, parents, 0.125, out=other), want, bound, "other strides")


def test_a_tree_of_one_node_is_attention_of_one_token():
    g, page, lengths = seeded(9), 16, [1, 30, 777]
    table, pages = tables_for(g, lengths, page, 49)
    k, v = pool(g, pages, page, 2, 128, F32)
    q = normal(g, (3, 1, 14, 128), F32)
    got = run_tree(q, k, v, table, lengths, int32([[-1]] * 3), None)
    cache = ops.PagedCache(k.cuda(), v.cuda(), table.cuda(), int32(lengths).cuda())
    out = torch.empty((3, 14, 128), device="cuda")
    ops.paged_attention(cache, out, q[:, 0].contiguous().cuda(), ops.Workspace(ops.attention_workspace(3, 14, 2, 128)))
    _, bound = oracle.tree_attention(q, k, v, table, lengths, int32([[-1]] * 3), 128 ** -0.5)
    assert ((got[:, 0] - out).abs().cpu() <= 2 * bound[:, 0]).all()


def test_tree_attention_of_more_rows_than_counters():
    """Rows are not cut then."""
    say("more rows than counters")
    g, rows, nodes, page = seeded(10), 33000, 2, 16
    k, v = pool(g, 40, page, 2, 64, BF16)
    table = torch.randint(0, 40, (rows, 20), generator=g, dtype=torch.int32)
    lengths = torch.randint(2, 321, (rows,), generator=g, dtype=torch.int32)
    q = normal(g, (rows, nodes, 2, 64), BF16)
    parents = int32([[-1, 0]]).expand(rows, 2).contiguous()
    got = run_tree(q, k, v, table, lengths.tolist(), parents, 0.125)
    some = torch.randperm(rows, generator=g)[:200]
    want, bound = oracle.tree_attention(q[some], k, v, table[some], lengths[some], parents[some], 0.125)
    close(got[some.cuda()], want, bound, "out")


def test_tree_attention_of_very_many_heads():
    """Rows of 24,576 items: the records of a few pieces of them would pass 32 bits."""
    say("tree attention of very many heads")
    g, kv_heads, group, nodes, dim, page, n = seeded(28), 4096, 11, 64, 128, 256, 256
    gd = torch.Generator(device="cuda").manual_seed(28)
    k, v = (torch.randn((1, page, kv_heads, dim), generator=gd, device="cuda", dtype=F16) for _ in range(2))
    q = torch.randn((1, nodes, kv_heads * group, dim), generator=gd, device="cuda", dtype=F16)
    parents, table = int32([tree(g, nodes)]), int32([[0]])
    w = ops.Workspace(ops.tree_attention_workspace(1, nodes, kv_heads * group, kv_heads, dim))
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, NAN)
    ops.tree_attention(ops.PagedCache(k, v, table.cuda(), int32([n]).cuda(), error), out, q, parents.cuda(), w, scale=0.1)
    assert int(error) == 0
    assert torch.isfinite(out).all()
    for h in (0, 1, 2047, 4095):
        heads = slice(h * group, (h + 1) * group)
        want, bound = oracle.tree_attention(q[:, :, heads].cpu(), k[:, :, h:h + 1].cpu(), v[:, :, h:h + 1].cpu(), table, [n], parents, 0.1)
        close(out[:, :, heads], want, bound, h)


def test_offsets_past_32_bits():
    say("offsets past 32 bits")
    g, page, nodes, dim = seeded(11), 16, 3, 64
    stride = (1 << 31) // 2 + 4096  # elements between pages: byte offsets past 2^32 from the fourth page on
    base_k, base_v = (torch.zeros(4 * stride + page * dim, dtype=BF16, device="cuda") for _ in range(2))
    k, v = (b.as_strided((5, page, 1, dim), (stride, dim, dim, 1)) for b in (base_k, base_v))
    small_k, small_v = (normal(g, (5, page, 1, dim), BF16) for _ in range(2))
    k.copy_(small_k)
    v.copy_(small_v)
    table, lengths = int32([[4, 0, 3]]), [40]
    q = normal(g, (1, nodes, 2, dim), BF16)
    parents = int32([[-1, 0, 0]])
    want, bound = oracle.tree_attention(q, small_k, small_v, table, lengths, parents, 0.125)
    cache = ops.PagedCache(k, v, table.cuda(), int32(lengths).cuda())
    out = torch.empty_like(q, device="cuda")
    ops.tree_attention(cache, out, q.cuda(), parents.cuda(), ops.Workspace(ops.tree_attention_workspace(1, nodes, 2, 1, dim)), scale=0.125)
    close(out, want, bound, "out")


# ---- slots ------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_append_to_slots(dtype):
    say("append to slots", dtype)
    g, heads, kv_heads, dim, page = seeded(12), 6, 2, 64, 16
    table, pages = tables_for(g, [64, 64], page, 4)
    q, k, v = (normal(g, (9, n, dim), dtype) for n in (heads, kv_heads, kv_heads))
    rows, positions, slots = [0, 0, 0, 1, 1, 1, 1, 0, 1], [20, 21, 21, 3, 4, 4, -9, 22, 5], [20, 21, 22, 30, 31, 32, 7, -8, 63 - 2]
    bias = 2
    cos, sin = (torch.from_numpy(t) for t in ops.rope_table(1e4, dim, 64))
    filled = normal(g, (2, pages, page, kv_heads, dim), dtype).cuda()
    kp, vp = filled[0].clone(), filled[1].clone()
    cache = ops.PagedCache(kp, vp, table.cuda(), int32([0, 0]).cuda())
    out = torch.full((9, heads, dim), 7.0, dtype=dtype, device="cuda")
    sides = dict(rows=int32(rows).cuda(), cos=cos.cuda(), sin=sin.cuda(), position_bias=bias)
    ops.paged_append(cache, out, q.cuda(), k.cuda(), v.cuda(), int32(positions).cuda(), slots=int32(slots).cuda(), **sides)
    # Rotated as at their positions: what appending there, without slots, gives.
    k2, v2 = filled[0].clone(), filled[1].clone()
    want_q = torch.full_like(out, 7.0)
    ops.paged_append(ops.PagedCache(k2, v2, table.cuda(), int32([0, 0]).cuda()), want_q, q.cuda(), k.cuda(), v.cuda(),
                     int32([p if s + bias >= 0 else -9 for p, s in zip(positions, slots)]).cuda(), **sides)
    assert torch.equal(out, want_q)
    want_k, want_v = filled[0].clone(), filled[1].clone()
    for t in range(9):
        if positions[t] + bias < 0 or slots[t] + bias < 0:
            continue
        one_k, one_v = filled[0].clone(), filled[1].clone()
        ops.paged_append(ops.PagedCache(one_k, one_v, table.cuda(), int32([0, 0]).cuda()), None, None, k[t:t + 1].cuda(), v[t:t + 1].cuda(),
                         int32([positions[t]]).cuda(), rows=int32([rows[t]]).cuda(), cos=cos.cuda(), sin=sin.cuda(), position_bias=bias)
        a, b = positions[t] + bias, slots[t] + bias
        want_k[int(table[rows[t], b // page]), b % page] = one_k[int(table[rows[t], a // page]), a % page]
        want_v[int(table[rows[t], b // page]), b % page] = v[t].cuda()
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)


def test_append_to_a_slot_past_the_table():
    g = seeded(13)
    table, pages = tables_for(g, [32], 16, 2)
    k = normal(g, (2, 1, 64), F32).cuda()
    kp = torch.zeros((pages, 16, 1, 64), device="cuda")
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = ops.PagedCache(kp, kp.clone(), table.cuda(), int32([0]).cuda(), error)
    ops.paged_append(cache, None, None, k, k, int32([1, 1]).cuda(), rows=int32([0, 0]).cuda(), slots=int32([32, 31]).cuda())
    assert int(error) == ops.BAD_POSITION
    assert torch.equal(kp[int(table[0, 1]), 15], k[1]) and int((kp != 0).any(-1).sum()) == 1


# ---- accept ------------------------------------------------------------------------------------


def run_accept(logits, tokens, parents, draws=None, temperature=1.0, errors=0):
    rows, nodes, vocab = logits.shape
    path = torch.full((rows, nodes), 99, dtype=torch.int32, device="cuda")
    counts, following = (torch.full((rows,), 99, dtype=torch.int32, device="cuda") for _ in range(2))
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    w = ops.Workspace(ops.tree_accept_workspace(rows, nodes, vocab))
    ops.tree_accept(on_gpu(logits), tokens.cuda(), parents.cuda(), path, counts, following, w,
                    draws=None if draws is None else draws.cuda(), temperature=temperature, errors=error)
    assert int(error) == errors
    return path.cpu(), counts.cpu(), following.cpu()


def answer(g, logits, parents, draws, temperature):
    """Tokens that are what follows their parents, three times out of four."""
    rows, nodes = parents.shape
    picks = [[oracle.pick(logits[r, i], None if draws is None else float(draws[r, i]), temperature) for i in range(nodes)] for r in range(rows)]
    tokens = torch.randint(0, logits.shape[2], (rows, nodes), generator=g).tolist()
    for r in range(rows):
        for i in range(nodes):
            p = int(parents[r, i])
            if p >= 0 and float(torch.rand(1, generator=g)) < 0.75:
                tokens[r][i] = picks[r][p]
    return int32(tokens).reshape(rows, nodes)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,nodes,vocab", [(1, 1, 1), (1, 8, 151936), (5, 16, 32003), (3, 64, 1001), (7, 3, 7), (40, 5, 4099), (2, 2, 65536)])
def test_accept_the_likeliest(dtype, rows, nodes, vocab):
    say("accept", dtype, rows, nodes, vocab)
    g = seeded(vocab + nodes)
    logits = normal(g, (rows, nodes, vocab), dtype, 2.0)  # (16-bit logits tie)
    parents = some_trees(g, rows, nodes)
    tokens = answer(g, logits, parents, None, 1.0)
    for got, want in zip(run_accept(logits, tokens, parents), oracle.accept(logits, tokens, parents, None)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,nodes,vocab,temperature", [(1, 1, 1, 1.0), (1, 8, 151936, 0.7), (5, 16, 32003, 1.3), (3, 64, 1001, 0.05), (7, 3, 7, 9.0), (40, 5, 4099, 1.0)])
def test_accept_drawn_tokens(dtype, rows, nodes, vocab, temperature):
    """Draws in the middle of a token's share of the probability: 2^-18 of the whole or more from its ends,
    where FP32 exponentials (each off by about 2^-23 of itself) move the sums by less."""
    say("accept drawn", dtype, rows, nodes, vocab, temperature)
    g = seeded(vocab + nodes)
    logits = normal(g, (rows, nodes, vocab), dtype, 3.0)
    parents = some_trees(g, rows, nodes)
    draws = torch.zeros(rows, nodes)
    for r in range(rows):
        for i in range(nodes):
            p = torch.softmax(logits[r, i].double() / temperature, 0)
            upto = torch.cumsum(p, 0)
            able = (p > 2.0 ** -16).nonzero()[:, 0]
            t = int(able[int(torch.randint(0, len(able), (1,), generator=g))])
            draws[r, i] = float(upto[t] - p[t] / 2)
    tokens = answer(g, logits, parents, draws, temperature)
    for got, want in zip(run_accept(logits, tokens, parents, draws, temperature), oracle.accept(logits, tokens, parents, draws, temperature)):
        assert torch.equal(got, want)


def test_draws_at_the_ends():
    """0 is the first token that has a probability, and so is less; just below 1 the last one, 1 and more too."""
    logits = torch.full((6, 1, 5001), -math.inf)
    logits[:, 0, [17, 4000, 4999]] = torch.tensor([0.0, 1.0, -1.0])
    draws = torch.tensor([[0.0], [1 - 2.0 ** -24], [1.0], [2.0], [-1.0], [NAN]])
    parents, tokens = int32([[-1]] * 6), int32([[0]] * 6)
    assert run_accept(logits, tokens, parents, draws)[2].tolist() == [17, 4999, 4999, 4999, 17, 17]


TEMPERATURES = [float(torch.tensor(t)) for t in (0.05, 0.1, 0.2, 0.4, 0.5, 0.7, 0.75, 0.8, 0.85, 0.9, 1.0, 1.3, 1.5, 2.0)]


def running_sums(x, temperature):
    """Of rows [n, vocab]: each token's probability, the largest 1, their running sums, and how far two of those may be
    off: p = 2^-d by (1.8 d + 4) 2^-24 of it, eight of them in FP32 by 3 x 2^-24 more."""
    x = x.cuda().double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    d = (x.amax(-1, keepdim=True) - x) / temperature / math.log(2)
    p = torch.exp2(-d)
    off = torch.where(p > 0, p * (1.8 * d + 7), 0.0).sum(-1) * 2.0 ** -24
    return p, torch.cumsum(p, -1), 2 * off


def draw_one_each(logits, draws, temperature):
    """The tokens that follow trees of one node: logits [n, vocab], draws [n]."""
    n = logits.shape[0]
    return run_accept(logits[:, None], int32([[0]] * n), int32([[-1]] * n), draws[:, None].float(), temperature)[2].cuda().long()


def check_draws(logits, draws, temperature, got):
    p, upto, off = running_sums(logits, temperature)
    n, vocab = p.shape
    assert ((got >= 0) & (got < vocab)).all(), got
    row, total = torch.arange(n, device="cuda"), upto[:, -1]
    aim = draws.cuda().double().nan_to_num(nan=0.0).clamp(0, 1) * total
    last = vocab - 1 - (p > 0).flip(-1).to(torch.uint8).argmax(-1)
    assert (p[row, got] > 0).all(), "a token without a probability"
    assert torch.equal(got[draws.cuda() >= 1], last[draws.cuda() >= 1])
    assert ((upto[row, got] > aim - off) | (got == last)).all()
    assert (upto[row, got] - p[row, got] <= aim + off).all()


def middles(g, logits, temperature):
    """A draw in the middle of a token of each row that has 2^-14 of the probability or more, and the tokens."""
    p, upto, _ = running_sums(logits, temperature)
    p, upto = (p / upto[:, -1:]).cpu(), (upto / upto[:, -1:]).cpu()
    able = [(row > 2.0 ** -14).nonzero()[:, 0] for row in p]
    token = torch.tensor([int(a[int(torch.randint(0, len(a), (1,), generator=g))]) for a in able])
    row = torch.arange(len(able))
    return (upto[row, token] - p[row, token] / 2).float(), token.cuda()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("mask", [-math.inf, "lowest", -1e30, -1e10])
def test_draws_of_masked_logits(dtype, mask):
    """Lanes, quarters and shares that hold nothing but masks, at temperatures of either sign of what rounding leaves of
    their products."""
    say("draws of masked logits", dtype, mask)
    g, vocab = seeded(21), 151936
    mask = torch.finfo(dtype).min if mask == "lowest" else mask
    keep = torch.zeros(9, vocab, dtype=torch.bool)
    keep[0, 100000] = True
    keep[1, torch.randperm(vocab, generator=g)[:40]] = True
    keep[2, vocab // 2:] = True
    keep[3, : vocab // 2] = True
    keep[4] = torch.arange(vocab) // 8 % 64 == 5
    keep[5, 40000:43000] = True
    keep[6, -1] = True
    keep[7, 0] = True
    keep[8, ::3000] = True
    x = torch.randn(keep.shape, generator=g) * 0.5
    x[:, ::1000] += 8.0
    logits = torch.where(keep, x, mask).to(dtype)
    for temperature in TEMPERATURES:
        draws, want = middles(g, logits, temperature)
        assert torch.equal(draw_one_each(logits, draws, temperature), want), temperature


@pytest.mark.parametrize("temperature,base", [(0.05, 0.0), (0.05, 30.0), (0.05, -30.0), (0.1, 30.0), (0.7, 20.0), (1.0, 40.0), (1.3, 100.0), (0.7, -300.0)])
def test_draws_at_the_ends_of_tokens(temperature, base):
    """Within what sums may be off, to either side of each token's end."""
    say("draws at the ends of tokens", temperature, base)
    g, vocab, temperature = seeded(22), 4003, float(torch.tensor(temperature))
    for _ in range(8):
        x = torch.full((vocab,), base - 200 * temperature)
        at = torch.randperm(vocab, generator=g)[:9].sort().values
        x[at] = base + 2 * temperature * torch.rand(9, generator=g)
        _, upto, off = running_sums(x[None], temperature)
        end = (upto[0, at] / upto[0, -1]).cpu()[:-1]
        by = float(off[0] / upto[0, -1])
        draws = torch.cat([end * (1 - 4 * by), end * (1 - by), end, end * (1 + by), end * (1 + 4 * by)]).float()
        logits = x.repeat(len(draws), 1)
        check_draws(logits, draws, temperature, draw_one_each(logits, draws, temperature))


def test_draws_of_one_and_almost_one():
    """Many shares: the last token that has a probability, and never one behind the vocabulary."""
    say("draws of one")
    g, vocab, rows, temperature = seeded(23), 151936, 96, float(torch.tensor(0.7))
    logits = normal(g, (rows, vocab), F32, 3.0)
    logits[::3, -1000:] = -math.inf
    logits[1::3, -40000:] = -math.inf
    draws = torch.tensor([1.0, 1 - 2.0 ** -24, 2.0, math.inf]).repeat(rows // 4)
    check_draws(logits, draws, temperature, draw_one_each(logits, draws, temperature))


def test_draws_among_tokens_far_below_the_largest():
    """What FP32 holds of the largest's size: nothing. It is a probability all the same, and masks beside it are none."""
    say("draws far below")
    vocab = 151936
    logits = torch.full((4, vocab), -math.inf)
    logits[:, 100:9000] = -120.0
    logits[:, 90000] = 0.0
    logits[:, 100000:130000] = -150.0
    draws = torch.tensor([0.0, -1.0, 1.0, 0.5])
    assert draw_one_each(logits, draws, 1.0).tolist() == [100, 100, 129999, 90000]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_draws_of_logits_of_any_size(dtype):
    """Logits of many temperatures: ties and neighbours are told apart."""
    say("draws of any size", dtype)
    g, vocab = seeded(24), 20001
    for temperature, scale, base in ((1e-6, 3.0, 0.0), (1e-3, 3.0, 50.0), (1.0, 1.0, 3e6), (1.0, 0.0, -1e10), (1.0, 0.0, 1e20), (0.7, 1e25, 0.0),
                                     (1e6, 1e5, 0.0), (1e6, 1.0, 1e20), (1.0, 1.0, -1e9)):
        temperature = float(torch.tensor(temperature))
        logits = (torch.randn((12, vocab), generator=g) * scale + base).to(dtype)
        logits[:6, ::2] = -math.inf
        logits[2, 1:] = -math.inf
        logits[3, :-1] = -math.inf
        logits[3, -1] = logits[2, 0] = base
        draws = torch.rand(12, generator=g)
        draws[0], draws[1] = 0.0, 1.0
        check_draws(logits, draws, temperature, draw_one_each(logits, draws, temperature))


@pytest.mark.parametrize("dtype,offset", [(F32, 1), (F32, 3), (BF16, 1), (F16, 3), (BF16, 7)])
@pytest.mark.parametrize("vocab", [1, 2, 7, 9, 1009, 40003])
def test_draws_of_logits_that_lie_anywhere(dtype, offset, vocab):
    """Tokens before the first 16 bytes and behind the last ones, near whole numbers and far from them."""
    say("draws of logits that lie anywhere", dtype, offset, vocab)
    g, n = seeded(26), 24
    for temperature, base in ((0.7, 0.0), (1e-5, 40.0)):
        temperature = float(torch.tensor(temperature))
        wide = (torch.randn((n, 1, vocab + offset + 2), generator=g) + base).to(dtype)
        logits = on_gpu(wide)[:, :, offset: offset + vocab]
        logits[::4, :, : vocab // 2] = -math.inf
        logits[1::4, :, vocab // 2 + 1:] = -math.inf
        draws = torch.rand(n, generator=g)
        draws[:4], draws[4:8], draws[8:12] = 0.0, 1.0, 1 - 2.0 ** -24
        path, counts, following = (torch.full(s, 99, dtype=torch.int32, device="cuda") for s in ((n, 1), (n,), (n,)))
        w = ops.Workspace(ops.tree_accept_workspace(n, 1, vocab))
        ops.tree_accept(logits, int32([[0]] * n).cuda(), int32([[-1]] * n).cuda(), path, counts, following, w,
                        draws=draws[:, None].cuda(), temperature=temperature)
        assert (counts == 1).all() and (path == 0).all()
        check_draws(logits[:, 0], draws, temperature, following.long())


def test_drawn_answers_in_a_graph():
    """Captured once; replayed over other logits, draws and trees: likely tokens, masks, logits of many temperatures, trees
    that are bad or not there in between."""
    say("drawn answers in a graph")
    g, rows, nodes, vocab, temperature = seeded(27), 6, 9, 33000, float(torch.tensor(0.8))
    logits = torch.zeros((rows, nodes, vocab), device="cuda")
    tokens, parents = (torch.zeros((rows, nodes), dtype=torch.int32, device="cuda") for _ in range(2))
    draws = torch.zeros((rows, nodes), device="cuda")
    path, counts, following = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((rows, nodes), (rows,), (rows,)))
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    w = ops.Workspace(ops.tree_accept_workspace(rows, nodes, vocab))
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        ops.tree_accept(logits, tokens, parents, path, counts, following, w, draws=draws, temperature=temperature, errors=error,
                        stream=torch.cuda.current_stream().cuda_stream)
    for step in range(8):
        x = torch.randn((rows, nodes, vocab), generator=g)
        x[:, :, ::500] += 9.0
        if step % 4 == 1:
            x[:, :, : vocab - 700] = -math.inf
        elif step % 4 == 2:
            x += 3e6
        some = some_trees(g, rows, nodes)
        middle = torch.stack([middles(g, y, temperature)[0] for y in x])
        wanted = answer(g, x, some, middle, temperature)
        logits.copy_(x), tokens.copy_(wanted), parents.copy_(some), draws.copy_(middle)
        if step % 4 == 3:
            parents[0, 3] = 7
        graph.replay()
        torch.cuda.synchronize()
        assert int(error) == (ops.BAD_PARENT if step % 4 == 3 else 0)
        error.zero_()
        first = 1 if step % 4 == 3 else 0
        want = oracle.accept(x[first:], wanted[first:], some[first:], middle[first:], temperature)
        for got, y in zip((path, counts, following), want):
            assert torch.equal(got[first:].cpu(), y), step


@pytest.mark.parametrize("sampled", [False, True])
def test_accept_of_masked_and_infinite_logits(sampled):
    vocab = 9001
    logits = torch.randn((7, 1, vocab), generator=seeded(3))
    logits[0] = -math.inf
    logits[1] = NAN
    logits[2, 0, 5000:] = NAN
    logits[2, 0, 100] = 50.0
    logits[3, 0, [70, 8000]] = math.inf
    logits[4] = -math.inf
    logits[4, 0, 8999] = -5.0
    logits[5, 0, 123] = 3e38
    logits[6] = -3e38
    logits[6, 0, 77] = -2e38
    draws = torch.full((7, 1), 0.5) if sampled else None
    got = run_accept(logits, int32([[0]] * 7), int32([[-1]] * 7), draws)
    assert got[2].tolist() == [0, 0, 100, 70, 8999, 123, 77]
    assert got[1].tolist() == [1] * 7


def test_accept_takes_the_lowest_child_and_ends_at_leaves():
    logits = torch.zeros(1, 6, 50)
    logits[0, torch.arange(6), torch.tensor([10, 11, 12, 13, 14, 15])] = 1.0
    parents = int32([[-1, 0, 0, 1, 2, 2]])
    for tokens, path, following in (([9, 10, 10, 11, 12, 12], [0, 1, 3], 13), ([9, 8, 10, 11, 12, 12], [0, 2, 4], 14), ([10] + [7] * 5, [0], 10)):
        got = run_accept(logits, int32([tokens]), parents)
        assert got[0][0].tolist() == path + [-1] * (6 - len(path)) and int(got[1]) == len(path) and int(got[2]) == following


def test_accept_of_bad_trees_and_padding():
    g = seeded(5)
    logits = normal(g, (4, 4, 300), F32)
    parents = int32([[-1, 0, 1, 2], [-2, -2, -2, -2], [-1, 2, 1, 0], [-1, -2, 1, 0]])
    tokens = int32([[0] * 4] * 4)
    path, counts, following = run_accept(logits, tokens, parents, errors=ops.BAD_PARENT)
    assert counts.tolist()[1:] == [0, 0, 0] and following.tolist()[1:] == [-1] * 3 and (path[1:] == -1).all()
    assert int(counts[0]) >= 1
    # A second root is never reached.
    path, counts, _ = run_accept(logits[:1], int32([[0, int(logits[0, 0].argmax()), 5, 5]]), int32([[-1, -1, 0, 1]]))
    assert path[0].tolist() == [0, -1, -1, -1] and int(counts) == 1


@pytest.mark.parametrize("dtype,offset", [(F32, 1), (BF16, 1), (F16, 3), (BF16, 7)])
def test_accept_of_logits_that_lie_anywhere(dtype, offset):
    g = seeded(6)
    wide = normal(g, (3, 6, 1031), dtype, 2.0)
    logits = wide[:, 1:5, offset: offset + 1009]
    parents = int32([tree(g, 4) for _ in range(3)])
    tokens = answer(g, logits, parents, None, 1.0)
    for got, want in zip(run_accept(logits, tokens, parents), oracle.accept(logits, tokens, parents, None)):
        assert torch.equal(got, want)


def test_accept_of_rows_that_share_logits():
    g = seeded(7)
    logits = normal(g, (1, 1, 5000), F32).expand(3, 4, 5000)
    parents, tokens = int32([[-1, 0, 1, 1]] * 3), int32([[0, int(logits[0, 0].argmax()), 1, 2]] * 3)
    path = torch.empty((3, 4), dtype=torch.int32, device="cuda")
    counts, following = (torch.empty((3,), dtype=torch.int32, device="cuda") for _ in range(2))
    ops.tree_accept(logits[:1, :1].contiguous().cuda().expand(3, 4, 5000), tokens.cuda(), parents.cuda(), path, counts, following,
                    ops.Workspace(ops.tree_accept_workspace(3, 4, 5000)))
    for got, want in zip((path, counts, following), oracle.accept(logits, tokens, parents, None)):
        assert torch.equal(got.cpu(), want)


# ---- commit ------------------------------------------------------------------------------------


def run_commit(memory, table, lengths, path, counts, errors=0):
    out = torch.full((len(lengths),), 99, dtype=torch.int32, device="cuda")
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.tree_commit(memory, table.cuda(), int32(lengths).cuda(), path.cuda(), counts.cuda(), out, errors=error)
    assert int(error) == errors
    return out.tolist()


def committed(x, table, lengths, path, counts, page):
    """x [planes, pages, page, ..], moved."""
    x, old = x.clone(), x
    for r, n in enumerate(lengths):
        if n:
            start = n - path.shape[1]
            for i in range(int(counts[r])):
                a, b = start + int(path[r, i]), start + i
                x[:, int(table[r, b // page]), b % page] = old[:, int(table[r, a // page]), a % page]
    return x


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nodes,page", [(1, 16), (5, 16), (16, 32), (64, 16), (64, 128)])
def test_commit(dtype, nodes, page):
    say("commit", dtype, nodes, page)
    g = seeded(nodes + page)
    lengths = [nodes, nodes + 7, 0, 100 + nodes, 64, 333]
    lengths = [n if n == 0 or n >= nodes else n + nodes for n in lengths]
    table, pages = tables_for(g, lengths, page, -(-max(lengths) // page))
    walks = [list(range(nodes)), [0], [], sorted(torch.randperm(nodes, generator=g)[: 1 + nodes // 3].tolist()), [nodes - 1],
             list(range(0, nodes, 2))]
    path = int32([w + [-1] * (nodes - len(w)) for w in walks]).reshape(6, nodes)
    counts = int32([len(w) for w in walks])
    # Planes with heads inside and outside of positions, one plane, and something else of another size.
    a = normal(g, (3, pages, page, 2, 64), dtype)
    b = normal(g, (3, pages, 2, page, 64), dtype).transpose(2, 3)
    c = normal(g, (1, pages, page, 1, 8), F32)
    tensors = [on_gpu(x) for x in (a, b, c)]
    out = run_commit(ops.TokenMemory(tensors), table, lengths, path, counts)
    assert out == [n - nodes + int(k) if n else 0 for n, k in zip(lengths, counts)]
    for x, y in zip((a, b, c), tensors):
        assert torch.equal(y.cpu(), committed(x, table, lengths, path, counts, page))


def test_commit_of_a_path_over_page_ends():
    """Every source a page behind its target, each target the source of the move before."""
    g, page, nodes = seeded(3), 16, 64
    table, pages = tables_for(g, [90], page, 6)
    x = normal(g, (24, pages, page, 1, 64), F32)
    y = x.cuda()
    path, counts = int32([[*range(16, 64)] + [-1] * 16]), int32([48])
    assert run_commit(ops.TokenMemory([y]), table, [90], path, counts) == [74]
    assert torch.equal(y.cpu(), committed(x, table, [90], path, counts, page))


def test_commit_without_planes():
    g, page, nodes = seeded(1), 16, 9
    table, pages = tables_for(g, [40, 50], page, 4)
    x = normal(g, (pages, page, 3, 128), BF16)
    y = x.cuda()
    path, counts = int32([[0, 2, 5, 8, -1, -1, -1, -1, -1], [0, 1, 7, -1, -1, -1, -1, -1, -1]]), int32([4, 3])
    assert run_commit(ops.TokenMemory([y], planes=False), table, [40, 50], path, counts) == [35, 44]
    assert torch.equal(y.cpu(), committed(x[None], table, [40, 50], path, counts, page)[0])


def test_commit_of_bad_rows_moves_nothing_of_them():
    g, page, nodes = seeded(2), 16, 6
    lengths = [30, 30, 30, 30, 30, 30, 4, 200]
    table, pages = tables_for(g, [30] * 8, page, 2)
    x = normal(g, (2, pages, page, 1, 64), F32)
    y = x.cuda()
    path = int32([[0, 2, 4, -1, -1, -1]] * 8)
    counts = int32([3, 3, 7, -1, 3, 3, 3, 3])
    path[1, 2] = 6
    path[4] = int32([0, 2, 2, 5, 5, 5])
    table[5, 1] = pages
    bits = ops.BAD_PATH | ops.BAD_PAGE | ops.BAD_LENGTH
    assert run_commit(ops.TokenMemory([y]), table, lengths, path, counts, bits) == [27, 30, 30, 30, 30, 30, 4, 200]
    assert torch.equal(y.cpu(), committed(x, table, [30] + [0] * 7, path, counts, page))


# ---- streams and graphs ------------------------------------------------------------------------


def drafting(seed, rows=3, nodes=8):
    """A step's tensors: cache, queries, tree, logits, and what comes out."""
    g, page = seeded(seed), 16
    lengths = [90, 700, 33][:rows]
    table, pages = tables_for(g, lengths, page, 44)
    k, v = pool(g, pages, page, 2, 64, F32)
    s = type("Step", (), {})()
    s.k, s.v, s.table, s.lengths = k.cuda(), v.cuda(), table.cuda(), int32(lengths).cuda()
    s.q = normal(g, (rows, nodes, 4, 64), F32).cuda()
    s.parents = int32([tree(g, nodes) for _ in range(rows)]).cuda()
    s.logits = normal(g, (rows, nodes, 4001), F32, 2.0).cuda()
    above = s.parents.long().clamp(min=0)
    s.tokens = torch.gather(s.logits.argmax(-1), 1, above).int()
    s.out, s.path, s.counts = torch.zeros_like(s.q), torch.zeros_like(s.parents), torch.zeros_like(s.lengths)
    s.next, s.lengths_out = torch.zeros_like(s.lengths), torch.zeros_like(s.lengths)
    s.cache, s.memory = ops.PagedCache(s.k, s.v, s.table, s.lengths), ops.TokenMemory([s.k, s.v], planes=False)
    return s


def drafting_workspace():
    return ops.Workspace(max(ops.tree_attention_workspace(3, 8, 4, 2, 64), ops.tree_accept_workspace(3, 8, 4001)))


def drafting_step(s, w, stream):
    ops.tree_attention(s.cache, s.out, s.q, s.parents, w, stream=stream)
    ops.tree_accept(s.logits, s.tokens, s.parents, s.path, s.counts, s.next, w, stream=stream)
    ops.tree_commit(s.memory, s.table, s.lengths, s.path, s.counts, s.lengths_out, stream=stream)


def drafting_results(s):
    return [x.clone() for x in (s.out, s.path, s.counts, s.next, s.lengths_out, s.k, s.v)]


def test_two_graphs_share_a_workspace_and_replay():
    say("two graphs")
    w = drafting_workspace()
    steps = [drafting(21), drafting(22)]
    before = [(s.k.clone(), s.v.clone()) for s in steps]
    want = []
    for s in steps:
        drafting_step(s, w, torch.cuda.current_stream().cuda_stream)
        want.append(drafting_results(s))
    side = torch.cuda.Stream()
    graphs = []
    for s in steps:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            drafting_step(s, w, torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
    for replay in range(5):
        for s, (k, v), graph, results in zip(steps, before, graphs, want):
            s.k.copy_(k)
            s.v.copy_(v)
            s.out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(drafting_results(s), results):
                assert torch.equal(a, b), replay


def test_two_streams_at_once():
    say("two streams")
    steps, streams, workspaces = [drafting(23), drafting(24)], [torch.cuda.Stream(), torch.cuda.Stream()], [drafting_workspace() for _ in range(2)]
    want = []
    for s, w in zip(steps, workspaces):
        k, v = s.k.clone(), s.v.clone()
        drafting_step(s, w, torch.cuda.current_stream().cuda_stream)
        want.append(drafting_results(s))
        s.k.copy_(k)
        s.v.copy_(v)
        s.before = (k, v)
    torch.cuda.synchronize()
    for _ in range(20):
        for s, w, stream in zip(steps, workspaces, streams):
            with torch.cuda.stream(stream):
                s.k.copy_(s.before[0])
                s.v.copy_(s.before[1])
                drafting_step(s, w, stream.cuda_stream)
    torch.cuda.synchronize()
    for s, results in zip(steps, want):
        for a, b in zip(drafting_results(s), results):
            assert torch.equal(a, b)


# ---- a whole run -------------------------------------------------------------------------------


def test_drafted_decoding_gives_the_tokens_of_plain_decoding():
    """A model of one layer decodes token by token in 64 bits; with drafts, forks for the trees' room, slots,
    tree attention, accept and commit the same tokens come out."""
    say("a whole run")
    g = seeded(31)
    vocab, dim, heads, kv_heads, page, rows, nodes, pages = 97, 64, 4, 2, 16, 3, 6, 60
    group = heads // kv_heads
    emb = torch.randn(vocab, 48, generator=g)
    wq, wk, wv = (torch.randn(48, n * dim, generator=g) / 7 for n in (heads, kv_heads, kv_heads))
    wo = torch.randn(heads * dim, vocab, generator=g) / 4
    cos, sin = (torch.from_numpy(t) for t in ops.rope_table(1e4, dim, 200))

    def turn(x, p):  # [n, heads, dim] at positions p, 64 bits
        c, s = cos[p].double()[:, None], sin[p].double()[:, None]
        a, b = x[..., : dim // 2], x[..., dim // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    def plain(tokens):  # the logits after the last of them
        x = emb[tokens].double()
        p = torch.arange(len(tokens))
        q = turn((x[-1:] @ wq.double()).view(1, heads, dim), p[-1:])[0]
        k, v = turn((x @ wk.double()).view(-1, kv_heads, dim), p), (x @ wv.double()).view(-1, kv_heads, dim)
        o = torch.cat([torch.softmax(k[:, h // group] @ q[h] * dim ** -0.5, 0) @ v[:, h // group] for h in range(heads)])
        return o @ wo.double()

    prompts = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (5, 15, 29)]
    steps, want = 25, []
    for prompt in prompts:
        tokens = list(prompt)
        for _ in range(steps):
            best = plain(tokens).topk(2).values
            assert best[0] - best[1] > 1e-4
            tokens.append(int(plain(tokens).argmax()))
        want.append(tokens)
    # The cache holds the prompts but for their last tokens.
    kp, vp = (torch.zeros((1, pages, page, kv_heads, dim), device="cuda") for _ in range(2))
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    tables = [torch.full((rows, 8), -1, dtype=torch.int32, device="cuda") for _ in range(2)]
    lengths = [torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2)]
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    keep = ops.PagePool(refs, page, [kp, vp])
    memory = ops.TokenMemory([kp, vp])
    w = ops.Workspace(max(ops.fork_workspace(rows, pages), ops.tree_attention_workspace(rows, nodes, heads, kv_heads, dim),
                          ops.tree_accept_workspace(rows, nodes, vocab)))
    dev = [t.cuda() for t in (emb, wq, wk, wv, wo, cos, sin)]

    def project(tokens, rows_of, depth, slot, cache):
        x = dev[0][tokens]
        q, k, v = (x @ dev[1]).view(-1, heads, dim), (x @ dev[2]).view(-1, kv_heads, dim), (x @ dev[3]).view(-1, kv_heads, dim)
        out = torch.empty_like(q)
        ops.paged_append(cache, out, q, k, v, depth, rows=rows_of, cos=dev[5], sin=dev[6], slots=slot)
        return out

    most = max(len(p) for p in prompts) - 1
    ops.pages_fork(keep, tables[0], lengths[0], None, most, tables[1], lengths[1], w, errors=error)
    rows_of = int32([r for r in range(rows) for _ in range(len(prompts[r]) - 1)]).cuda()
    at = int32([i for r in range(rows) for i in range(len(prompts[r]) - 1)]).cuda()
    filled = torch.tensor([t for p in prompts for t in p[:-1]]).cuda()
    project(filled, rows_of, at, None, ops.PagedCache(kp[0], vp[0], tables[1], lengths[1], error))
    lengths[1].copy_(int32([len(p) - 1 for p in prompts]))
    newest = torch.tensor([p[-1] for p in prompts])
    got = [list(p) for p in prompts]
    now, rounds = 1, 0
    while min(len(t) - len(p) for t, p in zip(got, prompts)) < steps:
        rounds += 1
        # Drafts: right for some tokens, then wrong ones.
        parents = torch.tensor([tree(g, nodes) for _ in range(rows)], dtype=torch.int32)
        tokens = torch.randint(0, vocab, (rows, nodes), generator=g)
        depth = torch.zeros((rows, nodes), dtype=torch.int32)
        for r in range(rows):
            tokens[r, 0] = newest[r]
            for i in range(1, nodes):
                p = int(parents[r, i])
                depth[r, i] = depth[r, p] + 1
                n = len(got[r]) + int(depth[r, i]) - 1
                if n < len(want[r]) and float(torch.rand(1, generator=g)) < 0.7:
                    tokens[r, i] = want[r][n]
        # Room for the trees, their keys and values, attention, the answer, and what stands of it.
        ops.pages_fork(keep, tables[now], lengths[now], None, nodes, tables[1 - now], lengths[1 - now], w, errors=error)
        old, now = lengths[now], 1 - now
        cache = ops.PagedCache(kp[0], vp[0], tables[now], lengths[now], error)
        slot = (old[:, None] + torch.arange(nodes, dtype=torch.int32, device="cuda")).flatten().int()
        where = (old[:, None] + depth.cuda()).flatten().int()
        rows_of = torch.arange(rows, dtype=torch.int32, device="cuda").repeat_interleave(nodes)
        q = project(tokens.flatten().cuda(), rows_of, where, slot, cache)
        out = torch.empty_like(q).view(rows, nodes, heads, dim)
        ops.tree_attention(cache, out, q.view(rows, nodes, heads, dim), parents.cuda(), w)
        logits = out.flatten(2) @ dev[4]
        path = torch.empty((rows, nodes), dtype=torch.int32, device="cuda")
        counts, following, after = (torch.empty((rows,), dtype=torch.int32, device="cuda") for _ in range(3))
        ops.tree_accept(logits, tokens.int().cuda(), parents.cuda(), path, counts, following, w, errors=error)
        ops.tree_commit(memory, tables[now], lengths[now], path, counts, after, errors=error)
        lengths[now] = after
        for r in range(rows):
            walk = path[r, : int(counts[r])].tolist()
            got[r] += [int(tokens[r, i]) for i in walk[1:]] + [int(following[r])]
        newest = following.cpu().long()
        assert int(error) == 0
        assert after.tolist() == [len(t) - 1 for t in got]
    assert rounds < steps  # (drafts stood)
    for tokens, right in zip(got, want):
        n = min(len(tokens), len(right))
        assert tokens[:n] == right[:n]
