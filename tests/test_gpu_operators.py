"""The operators on device memory against their 64-bit restatements
(operator_oracle.py), at the sizes, masks and layouts where they can go wrong."""
import math
import random

import pytest
import torch

import operator_oracle as oracle
import qd_operators as ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAN = float("nan")


def say(*a):
    print("[gpu-case]", *a, flush=True)


def seeded(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g) * std).to(dtype)


def int32(values):
    return torch.tensor(values, dtype=torch.int32)


def close(got, want, bound, what):
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    off = ((got - want).abs() - bound).nan_to_num(nan=-1.0)
    assert off.max() <= 0, (what, float(off.max()), float(bound.max()))


def tables_for(g, lengths, page, width, spare=2):
    """Rows with pages of their own, shuffled; -1 behind them."""
    counts = [-(-n // page) for n in lengths]
    ids = torch.randperm(sum(counts) + spare, generator=g).tolist()
    table, at = [], 0
    for n in counts:
        table.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return int32(table).reshape(len(lengths), width), len(ids)


# ---- append -------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,interleaved,page", [
    (14, 2, 64, 64, False, 16), (4, 4, 128, 128, True, 64), (6, 1, 128, 24, False, 32), (2, 2, 64, 8, True, 256),
    (3, 3, 64, 0, False, 16)])
@pytest.mark.parametrize("tokens", [1, 5, 131])
def test_append(dtype, heads, kv_heads, dim, rotary, interleaved, page, tokens):
    say("append", dtype, heads, kv_heads, dim, rotary, interleaved, page, tokens)
    g = seeded(tokens * 7 + rotary)
    rows = min(tokens, 3)
    starts = [0, 15, 40][:rows]
    row = [t % rows for t in range(tokens)]
    position = [starts[t % rows] + t // rows for t in range(tokens)]
    width = max(position) // page + 2
    table, pages = tables_for(g, [width * page] * rows, page, width)
    qkv = normal(g, (tokens, heads + 2 * kv_heads, dim), dtype)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
    cos, sin = (torch.from_numpy(t) for t in ops.rope_table(1e4, max(rotary, 2), max(position) + 1, 4.0, 64))
    bias = 3
    filled = normal(g, (2, pages, page, kv_heads, dim), dtype).cuda()
    kp, vp = filled[0].clone(), filled[1].clone()
    cache = ops.PagedCache(kp, vp, table.cuda(), int32([0] * rows).cuda())
    dq = qkv.cuda()
    q_out = torch.full((tokens, heads, dim), NAN, dtype=dtype, device="cuda")
    sides = dict(cos=cos.cuda(), sin=sin.cuda()) if rotary else {}
    ops.paged_append(cache, q_out, *dq.split([heads, kv_heads, kv_heads], 1), int32([p - bias for p in position]).cuda(),
                     rows=int32(row).cuda(), interleaved=interleaved, position_bias=bias, **sides)
    at = torch.tensor([int(table[r, p // page]) for r, p in zip(row, position)])
    inside = torch.tensor([p % page for p in position])
    want_q, want_k, bound_q, bound_k = q.double(), k.double(), torch.zeros(1), torch.zeros(1)
    if rotary:
        want_q, size = oracle.rotate(q, cos[position], sin[position], interleaved)
        bound_q = oracle.rotate_bound(want_q, size, dtype)
        want_k, size = oracle.rotate(k, cos[position], sin[position], interleaved)
        bound_k = oracle.rotate_bound(want_k, size, dtype)
    close(q_out, want_q, bound_q, "q")
    close(kp[at, inside], want_k, bound_k, "k")
    assert torch.equal(vp[at, inside].cpu(), v)
    # Nothing else was written.
    untouched = torch.ones(pages, page, dtype=torch.bool)
    untouched[at, inside] = False
    untouched = untouched.cuda()
    assert torch.equal(kp[untouched], filled[0][untouched]) and torch.equal(vp[untouched], filled[1][untouched])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_append_of_a_long_prompt(dtype):
    """Enough to be written past the caches."""
    say("append of a long prompt", dtype)
    g, heads, kv_heads, dim, page = seeded(9), 16, 4, 128, 64
    tokens = (40 << 20) // ((heads + 2 * kv_heads) * dim * (4 if dtype == F32 else 2))
    table, pages = tables_for(g, [tokens], page, -(-tokens // page))
    q, k, v = (normal(g, (tokens, n, dim), dtype) for n in (heads, kv_heads, kv_heads))
    cos, sin = (torch.from_numpy(t) for t in ops.rope_table(1e6, 64, tokens))
    kp, vp = (torch.zeros((pages, page, kv_heads, dim), dtype=dtype, device="cuda") for _ in range(2))
    cache = ops.PagedCache(kp, vp, table.cuda(), int32([0]).cuda())
    out = torch.empty((tokens, heads, dim), dtype=dtype, device="cuda")
    at = torch.arange(tokens, dtype=torch.int32, device="cuda")
    ops.paged_append(cache, out, q.cuda(), k.cuda(), v.cuda(), at, rows=torch.zeros_like(at), cos=cos.cuda(), sin=sin.cuda())
    want, size = oracle.rotate(q, cos, sin, False)
    close(out, want, oracle.rotate_bound(want, size, dtype), "q")
    want, size = oracle.rotate(k, cos, sin, False)
    where = table[0].long().cuda()
    close(kp[where].flatten(0, 1)[:tokens], want, oracle.rotate_bound(want, size, dtype), "k")
    assert torch.equal(vp[where].flatten(0, 1)[:tokens].cpu(), v)


def append_state(dtype=F32, rows=4, page=16, width=3, dim=64):
    g = seeded(5)
    table, pages = tables_for(g, [width * page] * rows, page, width)
    k, v = (torch.zeros((pages, page, 2, dim), dtype=dtype, device="cuda") for _ in range(2))
    errors = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = normal(g, (rows, 10, dim), dtype).cuda()
    return table, k, v, errors, x


def test_append_in_place_and_rows_in_order():
    say("append in place")
    table, k, v, errors, x = append_state()
    want = x.clone()
    cos, sin = (torch.from_numpy(t).cuda() for t in ops.rope_table(1e4, 64, 48))
    cache = ops.PagedCache(k, v, table.cuda(), int32([0] * 4).cuda())
    positions = int32([0, 7, 16, 47]).cuda()
    out = torch.empty((4, 6, 64), device="cuda")
    ops.paged_append(cache, out, x[:, :6], x[:, 6:8], x[:, 8:], positions, cos=cos, sin=sin)
    ops.paged_append(cache, x[:, :6], x[:, :6], x[:, 6:8], x[:, 8:], positions, cos=cos, sin=sin)
    assert torch.equal(out, x[:, :6]) and torch.equal(want[:, 6:], x[:, 6:])


def test_append_without_queries():
    say("append keys and values only")
    table, k, v, errors, x = append_state(BF16)
    cache = ops.PagedCache(k, v, table.cuda(), int32([0] * 4).cuda())
    ops.paged_append(cache, None, None, x[:, 6:8], x[:, 8:], int32([5] * 4).cuda())
    assert torch.equal(k[table[:, 0].long().cuda(), 5], x[:, 6:8]) and torch.equal(v[table[:, 0].long().cuda(), 5], x[:, 8:])
    assert int((k != 0).any(-1).sum()) == 8


def test_append_skips_padding_and_marks_what_does_not_exist():
    say("append: negative positions, rows, positions and pages that do not exist")
    table, k, v, errors, x = append_state()
    table[2, 1] = 10 ** 6
    table[3, 0] = -1
    cos, sin = (torch.from_numpy(t).cuda() for t in ops.rope_table(1e4, 64, 40))
    cache = ops.PagedCache(k, v, table.cuda(), int32([0] * 4).cuda(), errors)
    cases = [(0, -1, 0), (0, 0, 0), (-1, 3, ops.BAD_ROW), (4, 3, ops.BAD_ROW), (1, 48, ops.BAD_POSITION),
             (1, 40, ops.BAD_POSITION), (2, 16, ops.BAD_PAGE), (3, 2, ops.BAD_PAGE), (1, 2 ** 31 - 1, ops.BAD_POSITION)]
    for row, position, error in cases:
        errors.zero_(), k.zero_(), v.zero_()
        out = torch.full((1, 6, 64), 7.0, device="cuda")
        ops.paged_append(cache, out, x[:1, :6], x[:1, 6:8], x[:1, 8:], int32([position]).cuda(), rows=int32([row]).cuda(),
                         cos=cos, sin=sin)
        assert int(errors) == error, (row, position)
        if error:
            assert torch.isnan(out).all() and not k.any() and not v.any()
        elif position < 0:
            assert bool((out == 7.0).all()) and not k.any()
        else:
            assert bool(k.any())
    # A bias past 32 bits does not wrap.
    errors.zero_()
    out = torch.full((1, 6, 64), 7.0, device="cuda")
    ops.paged_append(cache, out, x[:1, :6], x[:1, 6:8], x[:1, 8:], int32([2 ** 31 - 1]).cuda(), cos=cos, sin=sin,
                     position_bias=2 ** 31 - 1)
    assert int(errors) == ops.BAD_POSITION
    ops.paged_append(cache, out[:0], x[:0, :6], x[:0, 6:8], x[:0, 8:], int32([]).cuda(), cos=cos, sin=sin)  # no tokens


# ---- attention ----------------------------------------------------------------------------


def run_attention(q, k, v, table, lengths, scale, layout="token", errors=None):
    """k and v on the host [pages, page, kv_heads, dim]; "head": heads outside of a page's tokens."""
    dk, dv = k.cuda(), v.cuda()
    if layout == "head":
        dk, dv = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (dk, dv))
    cache = ops.PagedCache(dk, dv, table.cuda(), lengths.cuda(), errors)
    out = torch.full(q.shape, NAN, dtype=q.dtype, device="cuda")
    workspace = ops.Workspace(ops.attention_workspace(q.shape[0], q.shape[1], k.shape[2], k.shape[3]))
    ops.paged_attention(cache, out, q.cuda(), workspace, scale=scale)
    again = torch.empty_like(out)
    ops.paged_attention(cache, again, q.cuda(), workspace, scale=scale)
    torch.cuda.synchronize()
    same = torch.equal(out.view(torch.int16 if q.dtype != F32 else torch.int32),
                       again.view(torch.int16 if q.dtype != F32 else torch.int32))
    assert same, "two calls differ"
    return out


def hide(k, v, table, lengths, page):
    """NaN and infinities wherever no row's length reaches."""
    seen = torch.zeros(k.shape[:2], dtype=torch.bool)
    for r, n in enumerate(lengths.tolist()):
        for p in range(-(-n // page)):
            seen[int(table[r, p]), : min(page, n - p * page)] = True
    k[~seen], v[~seen] = NAN, math.inf


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,layout", [
    (14, 2, 64, 16, "token"), (8, 2, 128, 64, "head"), (3, 3, 64, 32, "head"), (16, 1, 128, 16, "token"),
    (34, 2, 64, 128, "token"), (2, 2, 128, 256, "token")])
def test_attention_lengths(dtype, heads, kv_heads, dim, page, layout):
    say("attention", dtype, heads, kv_heads, dim, page, layout)
    g = seeded(heads + dim)
    lengths = int32(EDGES)
    table, pages = tables_for(g, EDGES, page, -(-max(EDGES) // page) + 1)
    q = normal(g, (len(EDGES), heads, dim), dtype, 1.5)
    k, v = (normal(g, (pages, page, kv_heads, dim), dtype) for _ in range(2))
    hide(k, v, table, lengths, page)
    out = run_attention(q, k, v, table, lengths, dim ** -0.5, layout)
    close(out, *oracle.attention(q, k, v, table, lengths, dim ** -0.5), "out")
    assert not out[0].any()


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page", [(F32, 7, 1, 64, 16), (BF16, 4, 2, 128, 32), (F16, 4, 1, 64, 1024)])
@pytest.mark.parametrize("lengths", [[2049], [5000, 3, 0, 2300], [1] * 70 + [4097] + [200] * 200])
def test_attention_split(dtype, heads, kv_heads, dim, page, lengths):
    say("attention split", dtype, heads, kv_heads, dim, page, len(lengths), max(lengths))
    g = seeded(len(lengths))
    table, pages = tables_for(g, lengths, page, -(-max(lengths) // page))
    q = normal(g, (len(lengths), heads, dim), dtype, 1.5)
    k, v = (normal(g, (pages, page, kv_heads, dim), dtype) for _ in range(2))
    n = int32(lengths)
    hide(k, v, table, n, page)
    out = run_attention(q, k, v, table, n, dim ** -0.5)
    close(out, *oracle.attention(q, k, v, table, n, dim ** -0.5), "out")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,lengths", [
    (14, 2, 64, 16, EDGES), (8, 2, 128, 64, EDGES + [900, 0, 0, 1500, 513, 511]), (34, 2, 64, 32, [3000, 0, 1, 520, 0, 260]),
    (4, 4, 128, 16, [1] * 300 + [2500] + [0] * 20 + [700] * 3), (7, 1, 64, 16, [20000]), (2, 2, 64, 16, [0] * 5 + [9000, 0])])
def test_attention_equal_runs(dtype, heads, kv_heads, dim, page, lengths):
    """Pools large enough for the kernel that deals equal runs of tiles: rows that begin and end
    inside a run, rows of several runs, empty ones between and at the ends."""
    say("attention runs", dtype, heads, kv_heads, dim, page, len(lengths))
    g = seeded(heads + len(lengths))
    many = (100 << 20) // (2 * page * kv_heads * dim * (4 if dtype == F32 else 2)) + 1  # pages of 100 MB
    table, used = tables_for(g, lengths, page, max(-(-many // len(lengths)), -(-max(lengths) // page)), spare=many)
    q = normal(g, (len(lengths), heads, dim), dtype, 1.5)
    k, v = (torch.zeros((used, page, kv_heads, dim), dtype=dtype) for _ in range(2))
    held = table[table >= 0].long()
    k[held], v[held] = (normal(g, (len(held), page, kv_heads, dim), dtype) for _ in range(2))
    n = int32(lengths)
    hide(k, v, table, n, page)
    out = run_attention(q, k, v, table, n, dim ** -0.5)
    close(out, *oracle.attention(q, k, v, table, n, dim ** -0.5), "out")


@pytest.mark.parametrize("dtype,dim", [(F32, 64), (F32, 128), (BF16, 64), (BF16, 128), (F16, 64), (F16, 128)])
def test_attention_of_a_pool_past_the_caches(dtype, dim):
    say("attention of a large pool", dtype, dim)
    g, page, kv_heads = seeded(dim), 64, 2
    pages = (288 << 20) // (2 * page * kv_heads * dim * (4 if dtype == F32 else 2))
    lengths = [1500, 0, 77, 640]
    table, _ = tables_for(g, lengths, page, 400)
    table = torch.where(table >= 0, table * (pages // 48), table)
    k, v = (torch.zeros((pages, page, kv_heads, dim), dtype=dtype, device="cuda") for _ in range(2))
    held = table[table >= 0].long()
    hk, hv = (normal(g, (len(held), page, kv_heads, dim), dtype) for _ in range(2))
    k[held.cuda()], v[held.cuda()] = hk.cuda(), hv.cuda()
    q = normal(g, (4, 6, dim), dtype, 1.5)
    out = torch.full(q.shape, NAN, dtype=dtype, device="cuda")
    workspace = ops.Workspace(ops.attention_workspace(4, 6, kv_heads, dim))
    ops.paged_attention(ops.PagedCache(k, v, table.cuda(), int32(lengths).cuda()), out, q.cuda(), workspace)
    small = torch.full_like(table, -1)
    small[table >= 0] = torch.arange(len(held), dtype=torch.int32)
    close(out, *oracle.attention(q, hk, hv, small, int32(lengths), dim ** -0.5), "out")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attention_scores_of_any_size(dtype):
    """A maximum that rises and falls along the row, scores near the range's ends, one key that takes all."""
    say("attention: large scores", dtype)
    g = seeded(11)
    lengths, page, dim = [900, 900, 900, 900], 16, 64
    table, pages = tables_for(g, lengths, page, 57)
    q = torch.zeros((4, 2, dim), dtype=dtype)
    q[:, :, 0] = 1.0
    k, v = torch.zeros((pages, page, 2, dim), dtype=dtype), normal(g, (pages, page, 2, dim), dtype)
    j = torch.arange(900)
    ramps = [j / 8.0, -j / 8.0, ((j * 37) % 101) - 50.0, torch.where(j == 450, 1000.0, -1000.0)]
    for r, ramp in enumerate(ramps):
        k[table[r, j // page].long(), j % page, :, 0] = ramp[:, None].to(dtype)
    n = int32(lengths)
    out = run_attention(q, k, v, table, n, 1.0)
    want, bound = oracle.attention(q, k, v, table, n, 1.0)
    close(out, want, bound, "out")
    assert torch.equal(out[3].cpu(), v[table[3, 450 // page].long(), 450 % page])


def test_attention_infinities_follow_the_formula():
    say("attention: infinite keys")
    page, dim = 16, 64
    k, v = torch.zeros((4, page, 1, dim)), torch.ones((4, page, 1, dim))
    table = int32([[0, 1, 2, 3]] * 1)
    q = torch.zeros((1, 1, dim))
    q[..., 0] = 1.0
    k[..., 0] = -math.inf
    assert torch.isnan(run_attention(q, k, v, table, int32([64]), 1.0)).all()  # no finite score: no weights
    k[3, 5, 0, 0] = 2.0
    v[3, 5] = 5.0
    assert bool((run_attention(q, k, v, table, int32([64]), 1.0) == 5.0).all())  # the only finite one
    k[0, 0, 0, 0] = math.inf
    assert torch.isnan(run_attention(q, k, v, table, int32([64]), 1.0)).all()
    k[0, 0, 0, 0] = NAN
    assert torch.isnan(run_attention(q, k, v, table, int32([64]), 1.0)).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim,length,pool_mb", [(64, 60, 0), (128, 4000, 0), (64, 4000, 100), (128, 8192, 100), (64, 30001, 100)])
def test_attention_of_one_large_score_and_many_small_ones(dtype, dim, length, pool_mb):
    """A position that takes nearly all of the weight and whose V is zero: the output is what the many
    others, of equal scores 11 to 27 below, add up to."""
    say("attention: a large score, many small ones", dtype, dim, length, pool_mb)
    gaps = [11.0, 14.0, 16.0, 17.5, 20.0, 24.0, 27.0]
    g, page, kv_heads, group = seeded(dim + length), 64, 2, 3
    spare = (pool_mb << 20) // (2 * page * kv_heads * dim * (4 if dtype == F32 else 2)) + 1
    lengths = [length] * len(gaps)
    table, pages = tables_for(g, lengths, page, max(-(-length // page), -(-spare // len(gaps))), spare=spare)
    q = torch.zeros((len(gaps), group * kv_heads, dim), dtype=dtype)
    q[:, :, 0] = 1.0
    k = torch.zeros((pages, page, kv_heads, dim), dtype=dtype)
    v = torch.zeros_like(k)
    for r, gap in enumerate(gaps):
        held = table[r, : -(-length // page)].long()
        v[held] = normal(g, (len(held), page, kv_heads, dim), dtype) + 1.0
        at = (r * 997) % length
        k[table[r, at // page].long(), at % page, :, 0] = gap
        v[table[r, at // page].long(), at % page] = 0.0
    n = int32(lengths)
    out = run_attention(q, k, v, table, n, 1.0)
    want, bound = oracle.attention(q, k, v, table, n, 1.0)
    if dtype != F32:
        # The oracle allows each weight half of the type's least step, which is all of the small ones. They
        # keep their relative precision (in its bound already) down to 2^-51 of the largest, half a step of
        # the remainder that FP16 keeps of a weight: 2^14 times the weight, and 2^12 times what is left of it,
        # in steps of 2^-24. (BF16's least step is 2^-133.)
        most = torch.stack([v[table[r, : -(-length // page)].long()].flatten(0, 1)[:length].double().abs().amax(0) for r in range(len(gaps))])
        bound -= 2 * length * oracle.HALF_LEAST[dtype] * most.repeat_interleave(group, 1)
        bound += length * 2.0 ** -51 * most.repeat_interleave(group, 1)
    close(out, want, bound, "out")


@pytest.mark.parametrize("length", [40, 3000])
def test_attention_marks_bad_rows_and_no_others(length):
    say("attention: bad lengths and pages", length)
    g, page = seeded(3), 16
    lengths = [length] * 6
    table, pages = tables_for(g, lengths, page, -(-length // page))
    q = normal(g, (6, 4, 64), F32)
    k, v = (normal(g, (pages, page, 2, 64), F32) for _ in range(2))
    n = int32(lengths)
    want, bound = oracle.attention(q, k, v, table, n, 0.125)
    for change, bit in ((lambda t, m: m.__setitem__(1, -1), ops.BAD_LENGTH),
                        (lambda t, m: m.__setitem__(1, t.shape[1] * page + 1), ops.BAD_LENGTH),
                        (lambda t, m: t.__setitem__((1, 0), pages), ops.BAD_PAGE),
                        (lambda t, m: t.__setitem__((1, t.shape[1] - 1), -7), ops.BAD_PAGE)):
        t, m = table.clone(), n.clone()
        change(t, m)
        errors = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = run_attention(q, k, v, t, m, 0.125, errors=errors)
        assert int(errors) == bit
        assert torch.isnan(out[1]).all()
        keep = [0, 2, 3, 4, 5]
        close(out[keep], want[keep], bound[keep], "others")


def test_attention_shared_pages_strides_and_in_place():
    say("attention: shared pages, strided queries, in place")
    g, page, dim = seeded(8), 32, 64
    lengths = [100, 100, 70, 97]
    table, pages = tables_for(g, lengths, page, 4)
    table[:, :2] = table[0, :2]
    n = int32(lengths)
    wide = normal(g, (4, 3, 6, dim), F16)
    q = wide[:, 1]
    k, v = (normal(g, (pages, page, 2, dim), F16) for _ in range(2))
    want, bound = oracle.attention(q, k, v, table, n, 0.2)
    dw = wide.cuda()
    cache = ops.PagedCache(k.cuda(), v.cuda(), table.cuda(), n.cuda())
    workspace = ops.Workspace(ops.attention_workspace(4, 6, 2, dim))
    across = torch.empty((6, 4, dim), dtype=F16, device="cuda").transpose(0, 1)  # heads outside of rows
    ops.paged_attention(cache, across, dw[:, 1], workspace, scale=0.2)
    close(across, want, bound, "strided")
    ops.paged_attention(cache, dw[:, 1], dw[:, 1], workspace, scale=0.2)
    assert torch.equal(dw[:, 1], across)
    assert torch.equal(dw[:, 0].cpu(), wide[:, 0]) and torch.equal(dw[:, 2].cpu(), wide[:, 2])


def test_offsets_past_32_bits():
    """Pages 3 GB apart: bytes and elements pass 32 bits."""
    say("append and attention: pages far apart")
    g, page, kv_heads, dim = seeded(4), 16, 2, 64
    apart = 3 << 29  # elements of 2 bytes
    store = torch.empty(2 * apart + page * kv_heads * dim, dtype=BF16, device="cuda")
    shape, stride = (3, page, kv_heads, dim), (apart, kv_heads * dim, dim, 1)
    kp = store.as_strided(shape, stride)
    other = torch.empty_like(store)
    vp = other.as_strided(shape, stride)
    table, lengths = int32([[2, 0, 1]]), int32([41])
    cache = ops.PagedCache(kp, vp, table.cuda(), lengths.cuda())
    k, v = (normal(g, (41, kv_heads, dim), BF16) for _ in range(2))
    ops.paged_append(cache, None, None, k.cuda(), v.cuda(), torch.arange(41, dtype=torch.int32, device="cuda"),
                     rows=int32([0] * 41).cuda())
    assert torch.equal(kp[2].cpu(), k[:16]) and torch.equal(vp[1, :9].cpu(), v[32:])
    q = normal(g, (1, 4, dim), BF16)
    out = torch.empty((1, 4, dim), dtype=BF16, device="cuda")
    ops.paged_attention(cache, out, q.cuda(), ops.Workspace(ops.attention_workspace(1, 4, 2, dim)))
    pages = torch.zeros(3, page, kv_heads, dim, dtype=BF16)
    pages[2], pages[0], pages[1, :9] = k[:16], k[16:32], k[32:]
    values = torch.zeros_like(pages)
    values[2], values[0], values[1, :9] = v[:16], v[16:32], v[32:]
    close(out, *oracle.attention(q, pages, values, table, lengths, dim ** -0.5), "out")


# ---- fork ---------------------------------------------------------------------------------


class Forked:
    """A device state and its host restatement, moved on together."""

    def __init__(self, rows, pages, width, page, planes=2, dtype=BF16, kept=()):
        g = seeded(rows + pages)
        self.page, self.rows, self.width = page, rows, width
        self.table, self.lengths, self.refs = [[-1] * width for _ in range(rows)], [0] * rows, [0] * pages
        for p in kept:  # pages that someone outside the table holds
            self.refs[p] += 1
        self.k = normal(g, (planes, pages, page, 2, 8), dtype)
        self.v = normal(g, (planes, pages, page, 2, 8), dtype)
        self.dk, self.dv = self.k.cuda(), self.v.cuda()
        self.d_refs = int32(self.refs).cuda()
        self.side = [(int32(self.table).reshape(rows, width).cuda(), int32(self.lengths).cuda()),
                     (torch.full((rows, width), 99, dtype=torch.int32, device="cuda"),
                      torch.zeros(rows, dtype=torch.int32, device="cuda"))]
        self.errors = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.pool = ops.PagePool(self.d_refs, page, [self.dk, self.dv])
        self.workspace = ops.Workspace(ops.fork_workspace(rows, pages))

    def load(self):
        self.side[0] = (int32(self.table).reshape(self.rows, self.width).cuda(), int32(self.lengths).cuda())
        self.d_refs.copy_(int32(self.refs))

    def fork(self, parents, append):
        (t, n), (t2, n2) = self.side
        d = None if parents is None else int32(parents).cuda()
        ops.pages_fork(self.pool, t, n, d, append, t2, n2, self.workspace, errors=self.errors)
        self.side.reverse()

    def step(self, parents, append):
        self.fork(parents, append)
        self.table, self.lengths, self.refs, copies = oracle.fork(self.table, self.lengths, parents, self.refs, append, self.page)
        for a, b in copies:
            self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]
        self.compare()

    def compare(self):
        t, n = self.side[0]
        assert t.cpu().tolist() == self.table
        assert n.cpu().tolist() == self.lengths
        assert self.d_refs.cpu().tolist() == self.refs
        assert torch.equal(self.dk.cpu(), self.k) and torch.equal(self.dv.cpu(), self.v)
        assert int(self.errors) == 0


@pytest.mark.parametrize("rows,pages,width,page", [(1, 9, 8, 16), (6, 90, 12, 16), (16, 300, 9, 64), (70, 9000, 70, 16)])
def test_fork_random_walk(rows, pages, width, page):
    say("fork walk", rows, pages, width, page)
    rng = random.Random(rows)
    s = Forked(rows, pages, width, page, kept=(0, 3))
    for step in range(12):
        parents = rng.choice([None, [rng.choice([-1] + list(range(rows)) * 6) for _ in range(rows)]])
        append = rng.choice([0, 1, 1, 3, page, page + 5])
        if max(s.lengths) + append > width * page or rows * (max(s.lengths) // page + 3) > pages - 2:
            parents, append = [-1] * rows, 0
        if step == 5 and rows > 1:
            # Tokens that were turned down: shorter rows, whose spare pages go.
            s.lengths = [max(0, n - page - 2) for n in s.lengths]
            s.load()
        s.step(parents, append)


def test_fork_outside_holders_force_copies():
    say("fork: a partly filled page that others hold")
    s = Forked(3, 12, 4, 16)
    s.step(None, 20)  # two pages each
    s.refs[s.table[1][1]] += 1  # kept by a cache of prefixes
    s.load()
    s.step([1, 1, 0], 1)
    s.step([2, 2, 2], 0)
    s.step([0, 1, 2], 16)


def test_fork_without_memories_and_rows():
    say("fork: counts alone")
    refs = torch.zeros(8, dtype=torch.int32, device="cuda")
    table = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    out, n_out = torch.empty_like(table), torch.empty_like(n)
    workspace = ops.Workspace(ops.fork_workspace(2, 8))
    ops.pages_fork(ops.PagePool(refs, 16, []), table, n, None, 33, out, n_out, workspace)
    assert out.tolist() == [[0, 1, 2], [3, 4, 5]] and n_out.tolist() == [33, 33] and refs.tolist() == [1] * 6 + [0] * 2
    ops.pages_fork(ops.PagePool(refs, 16, []), table[:0], n[:0], None, 1, out[:0], n_out[:0], workspace)


@pytest.mark.parametrize("what", ["exhausted", "grows", "length", "parent", "page", "short"])
def test_fork_changes_nothing_where_it_fails(what):
    say("fork fails:", what)
    s = Forked(4, 14, 4, 16)
    s.step(None, 30)
    parents, append = [0, 0, 1, 2], 1
    if what == "exhausted":
        append = 34
    elif what == "grows":
        append = 35
    elif what == "length":
        s.lengths[2] = -1
    elif what == "parent":
        parents[3] = 4
    elif what == "page":
        s.table[0][1] = 14
    else:
        s.table[0][1] = -1
    s.load()
    s.fork(parents, append)
    bit = {"exhausted": ops.EXHAUSTED, "grows": ops.BAD_LENGTH, "length": ops.BAD_LENGTH, "parent": ops.BAD_ROW,
           "page": ops.BAD_PAGE, "short": ops.BAD_PAGE}[what]
    assert int(s.errors) == bit
    s.errors.zero_()
    s.compare()


@pytest.mark.parametrize("each", [1 << 22, (1 << 22) + 1])
def test_fork_that_wants_more_pages_than_32_bits_count(each):
    """1,024 rows that want 2^22 pages each, 2^32 in all, and one more each: too many, whatever is left of
    their sum in 32 bits."""
    rows, width, pages, page = 1024, (1 << 22) + 1, 2000, 16
    say("fork of more than 2^32 pages", each)
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("two tables of 17 GB")
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    table_out = torch.zeros_like(table)
    lengths = torch.zeros(rows, dtype=torch.int32, device="cuda")
    lengths_out = torch.full_like(lengths, 7)
    refs, errors = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (pages, 1))
    refs[::3] = 1
    before = refs.clone()
    ops.pages_fork(ops.PagePool(refs, page, []), table, lengths, None, each * page, table_out, lengths_out,
                   ops.Workspace(ops.fork_workspace(rows, pages)), errors=errors)
    assert int(errors) == ops.EXHAUSTED
    assert torch.equal(refs, before) and not lengths_out.any()
    assert all(bool((part == -1).all()) for part in table_out.split(64))
    # A few rows of the same table that fit.
    errors.zero_()
    few = torch.full((rows,), -1, dtype=torch.int32)
    few[[3, 1000]] = int32([5, 5])
    ops.pages_fork(ops.PagePool(refs, page, []), table, lengths, few.cuda(), 20, table_out, lengths_out,
                   ops.Workspace(ops.fork_workspace(rows, pages)), errors=errors)
    assert int(errors) == 0 and refs.sum().item() == before.sum().item() + 4
    assert table_out[3, :3].tolist() == [1, 2, -1] and table_out[1000, :3].tolist() == [4, 5, -1]
    assert lengths_out.sum().item() == 40


# ---- select -------------------------------------------------------------------------------


def run_select(logits, scores, k, done=None, eos=None, strided=False):
    groups, beams, vocab = logits.shape
    d = logits.cuda()
    if strided:  # rows at odd addresses
        d = torch.empty((groups, beams, vocab + 3), dtype=logits.dtype, device="cuda")[:, :, 1:vocab + 1].copy_(d)
    scores_out = torch.full((groups, k), NAN, device="cuda")
    parents, tokens = (torch.full((groups, k), -5, dtype=torch.int32, device="cuda") for _ in range(2))
    sides = {}
    if done is not None:
        sides = dict(done=done.to(torch.uint8).cuda(), eos=eos,
                     done_out=torch.full((groups, k), 9, dtype=torch.uint8, device="cuda"))
    workspace = ops.Workspace(ops.select_workspace(groups, beams, k, vocab))
    for _ in range(2):  # the second call finds the counters as the first one left them
        ops.beam_select(d, scores.cuda(), scores_out, parents, tokens, workspace, **sides)
    return scores_out.cpu(), parents.cpu(), tokens.cpu(), sides["done_out"].cpu() if sides else None


def check_select(logits, scores, k, done=None, eos=None, strided=False):
    """Scores to their bound, each continuation once, and in an order that no two scores further
    apart than their errors contradict; exactly the lists where no such pair is near."""
    groups, beams, vocab = logits.shape
    got = run_select(logits, scores, k, done, eos, strided)
    picked, every = oracle.select(logits, scores, done, eos, k)
    for g in range(groups):
        names = [(int(p) - g * beams, int(t)) for p, t in zip(got[1][g], got[2][g])]
        assert len(set(names)) == k and all(0 <= b < beams and 0 <= t < vocab for b, t in names)
        for i, (b, t) in enumerate(names):
            want, true = picked[g][i][0], float(every[g][b, t])
            if math.isinf(want) or math.isinf(true):
                assert want == true == float(got[0][g, i]), (g, i)
                assert (b, t) == picked[g][i][1:], (g, i)
                continue
            room = oracle.select_bound(want)
            assert abs(float(got[0][g, i]) - true) <= room, (g, i)
            assert abs(true - want) <= 2 * room, (g, i)
            if (b, t) != picked[g][i][1:]:
                assert b != picked[g][i][1] or abs(true - want) > 0, "one beam's order goes by its logits"
            if done is not None:
                assert int(got[3][g, i]) == int(bool(done[g, b]) or t == eos)
    return got


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("groups,beams,k,vocab", [
    (1, 1, 1, 1), (1, 1, 4, 151936), (2, 16, 16, 32003), (3, 4, 8, 1000), (1, 32, 64, 2049), (5, 3, 6, 257),
    (300, 2, 2, 8193), (2, 2, 7, 4)])
def test_select(dtype, groups, beams, k, vocab):
    say("select", dtype, groups, beams, k, vocab)
    g = seeded(vocab + beams)
    logits = normal(g, (groups, beams, vocab), dtype, 3.0)
    scores = -5 * torch.rand((groups, beams), generator=g)
    check_select(logits, scores, k)
    check_select(logits, scores, k, strided=True)
    done = torch.rand((groups, beams), generator=g) < 0.4
    check_select(logits, scores, k, done, vocab // 2)


def test_select_ties_go_to_the_lower_token_and_beam():
    say("select: equal logits")
    logits = torch.zeros(1, 3, 5000)
    scores = torch.tensor([[-1.0, -0.5, -1.0]])
    got = run_select(logits, scores, 10)
    assert got[1].tolist() == [[1] * 10] and got[2].tolist() == [list(range(10))]
    logits[0, 1] = -math.inf
    logits[0, 1, 4999] = 1.0
    got = check_select(logits, scores, 4)
    assert got[1].tolist() == [[1, 0, 0, 0]] and got[2].tolist() == [[4999, 0, 1, 2]]
    logits[:] = 0.0
    logits[0, :, 7] = -0.0
    got = run_select(logits, torch.zeros(1, 3), 64)  # -0 is no lower than 0; all beams equal: the lowest
    assert got[1].tolist() == [[0] * 64] and got[2].tolist() == [list(range(64))]


def test_select_scores_of_zero_are_equal():
    say("select: finished beams of scores -0 and 0")
    got = run_select(torch.zeros(2, 3, 100), torch.tensor([[-0.0, 0.0, -0.0], [-1.0, 0.0, -0.0]]), 2,
                     torch.ones(2, 3, dtype=torch.uint8), 7)
    assert got[1].tolist() == [[0, 1], [4, 5]] and got[2].tolist() == [[7, 7], [7, 7]]
    assert got[0].tolist() == [[0.0, 0.0], [0.0, 0.0]] and got[3].tolist() == [[1, 1], [1, 1]]
    # A finished one at -0 beside one whose only token costs nothing.
    logits = torch.full((1, 2, 100), -math.inf)
    logits[0, 1, 5] = 3.0
    got = run_select(logits, torch.tensor([[-0.0, 0.0]]), 1, torch.tensor([[1, 0]], dtype=torch.uint8), 7)
    assert got[1].tolist() == [[0]] and got[2].tolist() == [[7]]


def test_select_masks():
    say("select: masks, dead and finished beams, NaN")
    g = seeded(2)
    vocab = 9000
    logits = normal(g, (4, 3, vocab), F32)
    logits[0, :, 5:] = -math.inf                      # fewer tokens than places
    logits[1, 0] = -math.inf                          # a beam without any
    logits[2] = -math.inf                             # a group without any
    logits[3, 1, 100:] = NAN
    logits[3, 2] = torch.finfo(F32).min               # the lowest finite number is a number
    scores = torch.tensor([[0.0, -math.inf, -1.0], [-1.0, -2.0, NAN], [0.0, -1.0, -2.0], [-1.0, -0.5, math.inf]])
    check_select(logits, scores, 12)
    done = torch.tensor([[0, 1, 1], [1, 0, 1], [0, 0, 1], [1, 0, 0]])
    check_select(logits, scores, 12, done, 3)
    check_select(logits[3:, 2:], torch.zeros(1, 1), 5)
    check_select(logits[:, :, :2], scores, 6, done, 1)  # as many places as continuations


@pytest.mark.parametrize("k", [1, 5, 64])
def test_select_of_one_beam(k):
    """A group of one beam: its row is the result, places left go to the lowest tokens."""
    say("select: one beam,", k)
    vocab = 9001
    logits = normal(seeded(3), (7, 1, vocab), F32)
    logits[1] = -math.inf                              # no token
    logits[2, 0, 3:] = -math.inf                       # fewer than places
    logits[3, 0, [2, 8999]] = math.inf                 # the others' share is nothing
    logits[4, 0, 1:4500] = NAN
    scores = torch.tensor([[0.0], [-1.0], [-2.0], [-3.0], [-4.0], [-math.inf], [-5.0]])
    check_select(logits, scores, k)
    check_select(logits, scores, k, torch.tensor([[0], [0], [0], [0], [0], [0], [1]]), 2)


def test_select_infinite_logits():
    say("select: infinite logits")
    logits = torch.zeros(1, 2, 3000)
    logits[0, 0, [5, 2500]] = math.inf
    got = check_select(logits, torch.zeros(1, 2), 6)
    assert got[1].tolist()[0][:2] == [0, 0] and got[2].tolist()[0][:2] == [5, 2500]
    assert abs(float(got[0][0, 0]) + math.log(2)) < 1e-6


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_select_descending_and_nearly_equal_rows(dtype):
    """Rows that put far more logits near the top than places: the longer ways of the ordering."""
    say("select: crowded tops", dtype)
    j = torch.arange(20000, dtype=torch.float64)
    crowd = (10 + ((j * 7919) % 20000) * 2.0 ** -20)
    logits = torch.stack([j * -1e-3, j * 1e-3, crowd]).to(dtype)[None]
    check_select(logits, torch.zeros(1, 3), 64)
    check_select(logits[:, 2:], torch.zeros(1, 1), 64)


# ---- calls beside each other, and the ends of the ranges --------------------------------------


def test_append_of_one_position_by_two_tokens():
    say("append: a position given twice")
    table, k, v, errors, x = append_state()
    cache = ops.PagedCache(k, v, table.cuda(), int32([0] * 4).cuda(), errors)
    ops.paged_append(cache, None, None, x[:, 6:8], x[:, 8:], int32([5, 5, 5, 6]).cuda(), rows=int32([1, 1, 1, 1]).cuda())
    for pages, new in ((k, x[:3, 6:8]), (v, x[:3, 8:])):
        got = pages[int(table[1, 0])]
        assert bool((got[5][None] == new).any(0).all()) and int((pages != 0).any(-1).sum()) == 2 * 2
    assert torch.equal(k[int(table[1, 0]), 6], x[3, 6:8]) and int(errors) == 0


def test_two_calls_at_once():
    """Two streams, a workspace each: attention, select and fork of different sizes beside each other."""
    say("two streams with a workspace each")
    g = seeded(21)
    sides = []
    for rows, most, vocab in ((9, 3000, 40000), (33, 400, 151936)):
        lengths = torch.randint(0, most, (rows,), generator=g).tolist()
        table, pages = tables_for(g, lengths, 16, -(-most // 16))
        k, v = (normal(g, (pages, 16, 2, 64), F32).cuda() for _ in range(2))
        refs = torch.bincount(table[table >= 0].long(), minlength=pages).to(torch.int32)
        refs = torch.cat([refs, torch.zeros(3 * rows, dtype=torch.int32)]).cuda()
        more = torch.zeros((refs.numel(), 16, 2, 64), device="cuda")
        sides.append(dict(
            stream=torch.cuda.Stream(), cache=ops.PagedCache(k, v, table.cuda(), int32(lengths).cuda()),
            q=normal(g, (rows, 14, 64), F32).cuda(), out=torch.empty((rows, 14, 64), device="cuda"),
            logits=normal(g, (1, 8, vocab), F32, 3.0).cuda(), scores=torch.zeros(1, 8, device="cuda"),
            best=[torch.empty((1, 8), device="cuda")] + [torch.empty((1, 8), dtype=torch.int32, device="cuda") for _ in range(2)],
            refs=refs, start=refs.clone(), pool=ops.PagePool(refs, 16, [more], planes=False),
            parents=torch.randint(0, rows, (rows,), generator=g).to(torch.int32).cuda(),
            table=torch.empty_like(table.cuda()), lengths=torch.empty(rows, dtype=torch.int32, device="cuda"),
            work=ops.Workspace(max(ops.attention_workspace(rows, 14, 2, 64), ops.select_workspace(1, 8, 8, vocab),
                                   ops.fork_workspace(rows, refs.numel())))))

    def calls(s):
        at = s["stream"].cuda_stream
        ops.paged_attention(s["cache"], s["out"], s["q"], s["work"], stream=at)
        ops.beam_select(s["logits"], s["scores"], *s["best"], s["work"], stream=at)
        with torch.cuda.stream(s["stream"]):
            s["refs"].copy_(s["start"])
        ops.pages_fork(s["pool"], s["cache"].tensors[2], s["cache"].tensors[3], s["parents"], 1, s["table"], s["lengths"],
                       s["work"], stream=at)
        with torch.cuda.stream(s["stream"]):
            return [x.clone() for x in (s["out"], *s["best"], s["table"], s["lengths"], s["refs"])]

    torch.cuda.synchronize()
    want = []
    for s in sides:
        want.append(calls(s))
        torch.cuda.synchronize()
    got = [[calls(s) for s in sides] for _ in range(20)]
    torch.cuda.synchronize()
    for turn in got:
        assert all(torch.equal(a, b) for mine, right in zip(turn, want) for a, b in zip(mine, right))


def test_two_graphs_share_a_workspace():
    """Replayed in turn on one stream, with eager calls on the same workspace between them."""
    say("two graphs, one workspace")
    g = seeded(22)
    work, graphs = ops.Workspace(max(ops.attention_workspace(40, 14, 2, 64), ops.select_workspace(2, 16, 16, 50000))), []
    for rows, most, groups in ((40, 700, 1), (3, 6000, 2)):
        lengths = torch.randint(0, most, (rows,), generator=g).tolist()
        table, pages = tables_for(g, lengths, 32, -(-most // 32))
        cache = ops.PagedCache(*(normal(g, (pages, 32, 2, 64), F32).cuda() for _ in range(2)), table.cuda(), int32(lengths).cuda())
        q, logits = normal(g, (rows, 14, 64), F32).cuda(), normal(g, (groups, 16, 50000), F32, 3.0).cuda()
        scores = torch.zeros(groups, 16, device="cuda")
        results = [torch.empty_like(q), torch.empty_like(scores)] + [torch.empty((groups, 16), dtype=torch.int32, device="cuda")
                                                                    for _ in range(2)]

        def calls(stream=0, a=(cache, results, q, logits, scores)):
            ops.paged_attention(a[0], a[1][0], a[2], work, stream=stream)
            ops.beam_select(a[3], a[4], *a[1][1:], work, stream=stream)

        calls()
        torch.cuda.synchronize()
        want = [x.clone() for x in results]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            calls(torch.cuda.current_stream().cuda_stream)
        graphs.append((graph, calls, results, want))
    for turn in range(5):
        for graph, _, results, _ in graphs:
            for x in results:
                x.fill_(-1)
            graph.replay()
        torch.cuda.synchronize()
        for _, calls, results, want in graphs:
            assert all(torch.equal(a, b) for a, b in zip(results, want)), turn
            calls()  # eager work between the replays
        torch.cuda.synchronize()


def test_attention_of_more_rows_than_counters():
    """Past 65,536 pairs of a row and a KV head no row is cut into pieces."""
    say("attention of 40,000 rows")
    g, rows, page = seeded(23), 40000, 16
    lengths = torch.randint(0, 49, (rows,), generator=g)
    table = torch.randint(0, 64, (rows, 3), generator=g).to(torch.int32)
    k, v = (normal(g, (64, page, 2, 64), F32) for _ in range(2))
    q = normal(g, (rows, 2, 64), F32, 1.5)
    cache = ops.PagedCache(k.cuda(), v.cuda(), table.cuda(), lengths.to(torch.int32).cuda())
    out = torch.empty((rows, 2, 64), device="cuda")
    ops.paged_attention(cache, out, q.cuda(), ops.Workspace(ops.attention_workspace(rows, 2, 2, 64)))
    for low in range(0, rows, 5000):
        part = slice(low, low + 5000)
        at = table[part].long()
        keys, values = (x.double()[at].reshape(-1, 48, 2, 64) for x in (k, v))
        s = (q[part].double()[:, None] * keys).sum(-1) * 64 ** -0.5
        inside = torch.arange(48)[None, :, None] < lengths[part][:, None, None]
        p = torch.softmax(s.masked_fill(~inside, -math.inf), 1).nan_to_num(0.0)
        want = (p[..., None] * values).sum(1)
        # Scores below 60 in magnitude from 64 products, 2^-24 of their sum of magnitudes (at most 64 x 8 x 4 / 8):
        # 256 x 64 x 2^-24 = 1e-3 were all roundings of one sign; a tenth of it holds with room.
        assert float((out[part].cpu().double() - want).abs().max()) < 1e-4
    assert not out[(lengths == 0).cuda()].any()


def test_attention_in_a_workspace_of_more_rows():
    """Past 65,536 pairs of a row and a KV head nothing is kept; fewer rows keep records."""
    say("attention: a workspace of more rows")
    g, page = seeded(32), 16
    workspace = ops.Workspace(ops.attention_workspace(40000, 2, 2, 64))
    for lengths in ([3000], [3000, 0, 700]):
        table, pages = tables_for(g, lengths, page, -(-3000 // page))
        q = normal(g, (len(lengths), 2, 64), F32, 1.5)
        k, v = (normal(g, (pages, page, 2, 64), F32) for _ in range(2))
        out = torch.full(q.shape, NAN, device="cuda")
        ops.paged_attention(ops.PagedCache(k.cuda(), v.cuda(), table.cuda(), int32(lengths).cuda()), out, q.cuda(), workspace)
        close(out, *oracle.attention(q, k, v, table, int32(lengths), 0.125), "out")


def test_fork_of_the_most_rows():
    say("fork of 1,024 rows")
    s = Forked(1024, 6000, 5, 16, planes=1)
    rng = random.Random(9)
    s.step(None, 20)
    for append in (1, 13, 0):
        s.step([rng.randrange(-1, 1024) for _ in range(1024)], append)


def test_fork_copies_memories_of_different_sizes():
    """Pages of one piece and of several with a rest, in planes of different numbers."""
    say("fork: memories of 512 bytes, 16,400 and 49,152")
    page, pages = 16, 12
    g = seeded(5)
    memories = [normal(g, (n, pages, page, w), F32) for n, w in ((1, 8), (3, 256 + 4), (2, 768))]
    memories[1] = memories[1].flatten(2)[:, :, :4100].contiguous()
    on = [m.cuda() for m in memories]
    table, lengths, refs = int32([[3, 5, -1], [3, 5, -1], [3, 5, -1]]).cuda(), int32([20, 20, 20]).cuda(), int32([0] * pages)
    refs[3] = refs[5] = 3
    refs = refs.cuda()
    after, more = torch.empty_like(table), torch.empty_like(lengths)
    ops.pages_fork(ops.PagePool(refs, page, on), table, lengths, None, 1, after, more, ops.Workspace(ops.fork_workspace(3, pages)))
    assert after.tolist() == [[3, 5, -1], [3, 0, -1], [3, 1, -1]] and more.tolist() == [21] * 3
    assert refs.tolist() == [1, 1, 0, 3, 0, 1, 0, 0, 0, 0, 0, 0]
    for d, m in zip(on, memories):
        m[:, 0] = m[:, 1] = m[:, 5]
        assert torch.equal(d.cpu(), m)


def test_select_in_a_workspace_of_more_rows():
    """A workspace of the largest batch serves every smaller one."""
    say("select: a workspace of more groups, beams, places and tokens")
    g, vocab = seeded(31), 30011
    workspace = ops.Workspace(ops.select_workspace(75, 8, 46, vocab))
    for groups, beams, k, tokens in ((75, 8, 46, vocab), (64, 8, 46, vocab), (1, 8, 46, vocab), (64, 8, 8, vocab),
                                     (3, 1, 45, vocab), (74, 7, 1, 28000)):
        logits, scores = normal(g, (groups, beams, tokens), F32, 3.0), torch.zeros(groups, beams)
        out = [torch.empty((groups, k), device="cuda")] + [torch.empty((groups, k), dtype=torch.int32, device="cuda") for _ in range(2)]
        ops.beam_select(logits.cuda(), scores.cuda(), *out, workspace)
        picked, _ = oracle.select(logits, scores, None, None, 1)
        for i in range(groups):
            assert abs(float(out[0][i, 0]) - picked[i][0][0]) <= oracle.select_bound(picked[i][0][0])


def test_select_of_the_largest_vocabulary():
    say("select of 2^24 tokens")
    g = seeded(24)
    check_select(normal(g, (1, 2, 1 << 24), BF16, 3.0), torch.tensor([[-1.0, -1.5]]), 64)


def test_results_are_written_as_torch_writes_them():
    """A tensor whose storage waits to be copied is copied first, and torch knows that results changed."""
    say("results: lazily copied storage, version counters")
    table, k, v, errors, x = append_state()
    cache = ops.PagedCache(k, v, table.cuda(), int32([17] * 4).cuda(), errors)
    pool = ops.PagePool(torch.zeros(40, dtype=torch.int32, device="cuda"), 16, [])
    workspace = ops.Workspace(max(ops.attention_workspace(4, 6, 2, 64), ops.fork_workspace(4, 40), ops.select_workspace(4, 6, 6, 64)))
    base = torch.full((4, 6, 64), 7.0, device="cuda")
    whole = {n: torch.full((4, 6), 7, dtype=t, device="cuda")
             for n, t in (("table", torch.int32), ("scores", F32), ("parents", torch.int32), ("tokens", torch.int32), ("done", torch.uint8))}
    lengths = torch.full((4,), 7, dtype=torch.int32, device="cuda")
    q, scores, done = x[:, :6].contiguous(), torch.zeros((4, 6), device="cuda"), torch.zeros((4, 6), dtype=torch.uint8, device="cuda")

    def calls(q_out, out, t, n, s, p, tok, d):
        ops.paged_append(cache, q_out, q, x[:, 6:8], x[:, 8:], int32([1] * 4).cuda())
        ops.paged_attention(cache, out, q, workspace)
        ops.pages_fork(pool, torch.full_like(t, -1), torch.zeros_like(n), None, 0, t, n, workspace, errors=errors)
        ops.beam_select(q, scores, s, p, tok, workspace, done, d, 3)

    originals = [base, base, whole["table"], lengths, whole["scores"], whole["parents"], whole["tokens"], whole["done"]]
    lazy = [torch._lazy_clone(t) for t in originals]
    written = lazy + [k, v, errors, pool.refs]
    versions = [t._version for t in written]
    calls(*lazy)
    assert all(bool((t == 7).all()) for t in originals)
    assert all(not bool((t == 7).all()) for t in lazy)
    assert all(t._version > n for t, n in zip(written, versions))
    # What autograd keeps is not changed behind its back.
    w = torch.ones((4, 6, 64), device="cuda", requires_grad=True)
    y = torch.zeros((4, 6, 64), device="cuda")
    loss = (w * y).sum()
    ops.paged_attention(cache, y, q, workspace)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        z = torch.empty((4, 6, 64), device="cuda")
    ops.paged_attention(cache, z, q, workspace)  # a tensor without a version counter
    assert torch.equal(z, y)


# ---- together -----------------------------------------------------------------------------


class Search:
    """Steps of a beam search on made-up queries, keys, values and logits, all on the device."""

    def __init__(self, beams=4, page=16, dim=64, heads=4, kv_heads=2, vocab=500, pages=60, width=10):
        g = seeded(75)
        self.beams, self.page, self.vocab = beams, page, vocab
        self.prompt = 21
        self.embed = normal(g, (vocab, heads + 2 * kv_heads, dim), F32).cuda()
        self.head = normal(g, (heads * dim, vocab), F32, 0.3).cuda()
        self.split = [heads, kv_heads, kv_heads]
        self.k, self.v = (torch.zeros((1, pages, page, kv_heads, dim), device="cuda") for _ in range(2))
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.tables = [torch.full((beams, width), -1, dtype=torch.int32, device="cuda") for _ in range(2)]
        self.lengths = [torch.zeros(beams, dtype=torch.int32, device="cuda") for _ in range(2)]
        self.caches = [ops.PagedCache(self.k[0], self.v[0], t, n) for t, n in zip(self.tables, self.lengths)]
        self.pool = ops.PagePool(self.refs, page, [self.k, self.v])
        self.parents = torch.arange(beams, dtype=torch.int32, device="cuda")
        self.tokens = torch.arange(beams, dtype=torch.int32, device="cuda")
        self.scores = torch.zeros(1, beams, device="cuda")
        self.new_scores = torch.zeros(1, beams, device="cuda")
        self.cos, self.sin = (torch.from_numpy(t).cuda() for t in ops.rope_table(1e4, dim, width * page))
        self.q = torch.zeros((beams, heads, dim), device="cuda")
        self.out = torch.zeros((beams, heads, dim), device="cuda")
        need = [ops.fork_workspace(beams, pages), ops.attention_workspace(beams, heads, kv_heads, dim),
                ops.select_workspace(1, beams, beams, vocab)]
        self.workspace = ops.Workspace(max(need))
        self.first = (self.tokens.clone(), self.parents.clone())
        self.reset()

    def reset(self):
        self.refs.zero_(), self.scores.zero_(), self.k.zero_(), self.v.zero_()
        self.tables[0].fill_(-1), self.lengths[0].zero_()
        self.tokens.copy_(self.first[0]), self.parents.copy_(self.first[1])

    def step(self, side, stream):
        a, b = side, 1 - side
        ops.pages_fork(self.pool, self.tables[a], self.lengths[a], self.parents, 1, self.tables[b], self.lengths[b],
                       self.workspace, stream=stream)
        x = self.embed[self.tokens.long()]
        q, k, v = x.split(self.split, 1)
        ops.paged_append(self.caches[b], self.q, q, k, v, self.lengths[b], cos=self.cos, sin=self.sin, position_bias=-1,
                         stream=stream)
        ops.paged_attention(self.caches[b], self.out, self.q, self.workspace, stream=stream)
        logits = (self.out.flatten(1) @ self.head)[None]
        ops.beam_select(logits, self.scores, self.new_scores, self.parents.view(1, -1), self.tokens.view(1, -1),
                        self.workspace, stream=stream)
        self.scores.copy_(self.new_scores)
        return logits

    def steps(self, n, stream):
        return [self.step(i % 2, stream) for i in range(n)]

    def result(self):
        return [x.clone() for x in (self.scores, self.tokens, self.parents, self.refs, self.tables[0], self.lengths[0])]


def reference_search(s, steps):
    """The same search with every beam's keys and values in a list of its own, 64 bits."""
    embed, head = s.embed.cpu().double(), s.head.cpu().double()
    cos, sin = s.cos.cpu(), s.sin.cpu()
    beams = [([], [], 0.0, int(t)) for t in s.first[0]]
    for step in range(steps):
        scored = []
        for b, (ks, vs, score, token) in enumerate(beams):
            q, k, v = embed[token].split(s.split, 0)
            q, k = (oracle.rotate(x[None], cos[step:step + 1], sin[step:step + 1], False)[0][0] for x in (q, k))
            ks, vs = ks + [k], vs + [v]
            kk, vv = torch.stack(ks), torch.stack(vs)
            out = []
            for h in range(s.split[0]):
                g = h * s.split[1] // s.split[0]
                out.append(torch.softmax(kk[:, g] @ q[h] * q.shape[1] ** -0.5, 0) @ vv[:, g])
            logp = torch.log_softmax(torch.cat(out) @ head, 0) + score
            best = torch.topk(logp, s.beams)
            scored += [(float(x), b, int(t), ks, vs) for x, t in zip(best.values, best.indices)]
        scored.sort(key=lambda e: -e[0])
        gaps = min(a[0] - b[0] for a, b in zip(scored, scored[1:s.beams + 1]))
        beams = [(list(ks), list(vs), x, t) for x, _, t, ks, vs in scored[:s.beams]]
        yield [(e[1], e[2], e[0]) for e in scored[:s.beams]], gaps


def test_a_search_of_all_four():
    say("fork, append, attention and select together")
    s = Search()
    for step, (want, gap) in enumerate(reference_search(s, 40)):
        s.step(step % 2, 0)
        # 40 steps, each rounding a score of at most 100 to FP32 (6e-6) and adding the errors of 256
        # products of logits below 10 (256 x 2^-24 x 10 = 1.6e-4 at most, a thousandth of that in the
        # mean): below 1e-3, and no two candidates are as near as 4e-3 in this search.
        assert gap > 4e-3
        assert list(zip(s.parents.tolist(), s.tokens.tolist())) == [(b, t) for b, t, _ in want], step
        assert max(abs(a - c) for a, (_, _, c) in zip(s.scores[0].tolist(), want)) < 1e-3
    held = [p for line in s.tables[0].tolist() for p in line if p >= 0]
    assert s.refs.tolist() == [held.count(p) for p in range(s.refs.numel())]


def test_a_search_on_another_stream_and_in_a_graph():
    say("the same on a stream of its own, and replayed from a graph")
    s = Search()
    s.steps(6, 0)
    want = s.result()
    stream = torch.cuda.Stream()
    s.reset()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        s.steps(6, stream.cuda_stream)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(s.result(), want))
    s.reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.steps(6, torch.cuda.current_stream().cuda_stream)
    for _ in range(4):
        s.reset()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(s.result(), want))
        s.reset()
        s.steps(6, 0)  # eager work between the replays
        torch.cuda.synchronize()


def test_tensors_that_do_not_fit_are_refused():
    say("refusals on device tensors")
    k = torch.zeros((4, 16, 2, 64), device="cuda")
    table, lengths = torch.zeros((2, 3), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    cache = ops.PagedCache(k, k.clone(), table, lengths)
    q = torch.zeros((2, 4, 64), device="cuda")
    workspace = ops.Workspace(0)
    refused = [
        lambda: ops.PagedCache(k, k[:3], table, lengths),
        lambda: ops.PagedCache(k, k.cpu(), table, lengths),
        lambda: ops.PagedCache(k, k, table.float(), lengths),
        lambda: ops.PagedCache(k, k, table, lengths[:1]),
        lambda: ops.PagedCache(k.transpose(2, 3), k.transpose(2, 3), table, lengths),
        lambda: ops.paged_attention(cache, q, q, workspace),  # too small
        lambda: ops.paged_attention(cache, q.half(), q, workspace),
        lambda: ops.paged_attention(cache, q[:1], q, workspace),
        lambda: ops.paged_append(cache, q, q, k[0, :2], k[0, :2], lengths.long()),
        lambda: ops.paged_append(cache, q, q, k[0, :3], k[0, :2], lengths),
        lambda: ops.paged_append(cache, None, q, k[0, :2], k[0, :2], lengths),
        lambda: ops.PagePool(lengths, 16, [k]),
        lambda: ops.beam_select(q, q[0, :, :1], q[0, :2], table, table, workspace),
        lambda: ops.beam_select(table, q, q, table, table, workspace),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ops.QdError):
            call()
            print("not refused:", i)
