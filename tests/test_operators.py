"""CPU checks of the operators on device memory: what they refuse before any
device work, the layout of the Python structures, the rotary tables, and that
the oracle's own fork keeps the counts."""
import ctypes as C
import math
import os
import random
import re

import numpy as np
import pytest

import operator_oracle as oracle
import qd_operators as ops
import qwen_decode as qd

_P, _I64, _U32, _I32 = C.c_void_p, C.c_int64, C.c_uint32, C.c_int32


# The calls' arguments as a ctypes program writes them.

class AppendStruct(C.Structure):
    _fields_ = [("q", _P), ("k", _P), ("v", _P), ("q_out", _P), ("q_stride", _I64), ("k_stride", _I64),
                ("v_stride", _I64), ("q_out_stride", _I64), ("positions", _P), ("rows", _P), ("position_bias", _I32),
                ("tokens", _U32), ("heads", _U32), ("rotary_dim", _U32), ("interleaved", _U32),
                ("table_positions", _U32), ("cos_table", _P), ("sin_table", _P)]


class AttentionStruct(C.Structure):
    _fields_ = [("q", _P), ("out", _P), ("q_stride", _I64), ("q_head_stride", _I64), ("out_stride", _I64),
                ("out_head_stride", _I64), ("heads", _U32), ("scale", C.c_float)]


class ForkStruct(C.Structure):
    _fields_ = [("table", _P), ("lengths", _P), ("parents", _P), ("table_out", _P), ("lengths_out", _P), ("refs", _P),
                ("table_stride", _I64), ("table_out_stride", _I64), ("errors", _P), ("memories", C.POINTER(ops.MemoryStruct)),
                ("memory_count", _U32), ("rows", _U32), ("table_width", _U32), ("pages", _U32), ("page_size", _U32),
                ("append", _U32), ("device", _I32)]


class SelectStruct(C.Structure):
    _fields_ = [("logits", _P), ("group_stride", _I64), ("beam_stride", _I64), ("scores", _P), ("done", _P),
                ("scores_out", _P), ("parents", _P), ("tokens", _P), ("done_out", _P), ("dtype", _U32), ("groups", _U32),
                ("beams", _U32), ("vocab", _U32), ("k", _U32), ("eos", _U32), ("device", _I32)]


HEADER = os.path.join(os.path.dirname(__file__), "..", "include", "qd", "qd_operators.h")
AT = 4096  # an aligned address that no refused call reads


def test_every_declared_entry_point_is_bound():
    text = open(HEADER).read()
    names = set(re.findall(r"QD_API\s+[^;(]*?\b(qd_\w+)\s*\(", text, re.S))
    assert names == set(ops._SIGNATURES)
    for n in names:
        assert hasattr(ops.lib(), n)


def test_structures_have_the_declared_fields():
    text = open(HEADER).read()
    for struct, cls in (("qd_paged_cache", ops.CacheStruct), ("qd_append_args", AppendStruct),
                        ("qd_attention_args", AttentionStruct), ("qd_page_memory", ops.MemoryStruct),
                        ("qd_fork_args", ForkStruct), ("qd_select_args", SelectStruct)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = [(m.group(1), "*" in line) for line in body.split(";") for m in [re.search(r"(\w+)\s*$", line.strip())] if m]
        assert [f for f, _ in fields] == [f for f, _ in cls._fields_], struct
        for (name, pointer), (_, kind) in zip(fields, cls._fields_):
            assert C.sizeof(kind) == 8 or not pointer, (struct, name)


def cache(**changes):
    c = dict(k=AT, v=AT, page_stride=16 * 2 * 64, token_stride=2 * 64, head_stride=64, table=AT, table_stride=8, lengths=AT,
             errors=None, rows=3, table_width=8, pages=10, page_size=16, kv_heads=2, head_dim=64, dtype=qd.DTYPE_F32, device=0)
    c.update(changes)
    return ops.CacheStruct(**c)


def append(**changes):
    a = dict(q=AT, k=AT, v=AT, q_out=AT, q_stride=14 * 64, k_stride=128, v_stride=128, q_out_stride=14 * 64, positions=AT,
             rows=None, position_bias=0, tokens=3, heads=14, rotary_dim=64, interleaved=0, table_positions=100, cos_table=AT,
             sin_table=AT)
    a.update(changes)
    return AppendStruct(**a)


def attention(**changes):
    a = dict(q=AT, out=AT, q_stride=14 * 64, q_head_stride=64, out_stride=14 * 64, out_head_stride=64, heads=14, scale=0.125)
    a.update(changes)
    return AttentionStruct(**a)


def fork(memory=None, **changes):
    m = dict(base=AT, plane_stride=1 << 20, page_stride=8192, bytes=8192, planes=2, reserved=0)
    m.update(memory or {})
    memories = (ops.MemoryStruct * 1)(ops.MemoryStruct(**m))
    a = dict(table=AT, lengths=AT, parents=None, table_out=2 * AT, lengths_out=2 * AT, refs=AT, table_stride=8,
             table_out_stride=8, errors=None, memories=memories, memory_count=1, rows=3, table_width=8, pages=10,
             page_size=16, append=1, device=0)
    a.update(changes)
    return ForkStruct(**a)


def select(**changes):
    a = dict(logits=AT, group_stride=4000, beam_stride=1000, scores=AT, done=None, scores_out=2 * AT, parents=AT, tokens=AT,
             done_out=None, dtype=qd.DTYPE_F32, groups=2, beams=4, vocab=1000, k=4, eos=0, device=0)
    a.update(changes)
    return SelectStruct(**a)


def refused(status, call, *args):
    got = getattr(ops.lib(), call)(*(C.byref(a) if isinstance(a, C.Structure) else a for a in args))
    text = ops.lib().qd_last_error().decode()
    assert got == status, (got, text)
    assert text


@pytest.mark.parametrize("status,changes", [
    (qd.INVALID_ARGUMENT, dict(dtype=3)),
    (qd.NOT_SUPPORTED, dict(page_size=8)),
    (qd.NOT_SUPPORTED, dict(page_size=24)),
    (qd.NOT_SUPPORTED, dict(page_size=2048)),
    (qd.NOT_SUPPORTED, dict(head_dim=96)),
    (qd.INVALID_ARGUMENT, dict(kv_heads=0)),
    (qd.INVALID_ARGUMENT, dict(table=None)),
    (qd.INVALID_ARGUMENT, dict(lengths=None)),
    (qd.INVALID_ARGUMENT, dict(k=None)),
    (qd.INVALID_ARGUMENT, dict(v=AT + 4)),
    (qd.INVALID_ARGUMENT, dict(table_stride=7)),
    (qd.INVALID_ARGUMENT, dict(token_stride=60)),
    (qd.INVALID_ARGUMENT, dict(token_stride=129)),
    (qd.INVALID_ARGUMENT, dict(head_stride=32)),
    (qd.INVALID_ARGUMENT, dict(page_stride=-4)),
    (qd.NOT_SUPPORTED, dict(token_stride=1 << 28)),
    (qd.NOT_SUPPORTED, dict(table_width=1 << 27, table_stride=1 << 27)),
])
def test_cache_refusals(status, changes):
    refused(status, "qd_paged_append", cache(**changes), append(), None)
    refused(status, "qd_paged_attention", cache(**changes), attention(), None, None)


@pytest.mark.parametrize("status,changes", [
    (qd.INVALID_ARGUMENT, dict(heads=13)),
    (qd.INVALID_ARGUMENT, dict(rotary_dim=12)),
    (qd.INVALID_ARGUMENT, dict(rotary_dim=72)),
    (qd.INVALID_ARGUMENT, dict(k=None)),
    (qd.INVALID_ARGUMENT, dict(q_out=None)),
    (qd.INVALID_ARGUMENT, dict(positions=None)),
    (qd.INVALID_ARGUMENT, dict(q=AT + 8)),
    (qd.INVALID_ARGUMENT, dict(cos_table=None)),
    (qd.INVALID_ARGUMENT, dict(sin_table=AT + 4)),
    (qd.INVALID_ARGUMENT, dict(q_stride=898)),
    (qd.INVALID_ARGUMENT, dict(q_out_stride=64)),
    (qd.INVALID_ARGUMENT, dict(v_stride=-128)),
    (qd.NOT_SUPPORTED, dict(tokens=1 << 30)),
    (qd.NOT_SUPPORTED, dict(q=None, q_out=None, tokens=1 << 26)),  # half of each token's wave idles: 2^32 threads
    (qd.INVALID_ARGUMENT, dict(q_out=AT, q_stride=18 * 64)),  # in place, at another stride
])
def test_append_refusals(status, changes):
    refused(status, "qd_paged_append", cache(), append(**changes), None)


@pytest.mark.parametrize("status,changes", [
    (qd.INVALID_ARGUMENT, dict(heads=0)),
    (qd.INVALID_ARGUMENT, dict(heads=15)),
    (qd.INVALID_ARGUMENT, dict(q=None)),
    (qd.INVALID_ARGUMENT, dict(out=AT + 8)),
    (qd.INVALID_ARGUMENT, dict(scale=math.nan)),
    (qd.INVALID_ARGUMENT, dict(scale=math.inf)),
    (qd.INVALID_ARGUMENT, dict(q_head_stride=66)),
    (qd.INVALID_ARGUMENT, dict(out_head_stride=0)),
    (qd.INVALID_ARGUMENT, dict(out_stride=18 * 64)),  # in place, at other strides
    (qd.INVALID_ARGUMENT, dict(out_head_stride=128)),
    (qd.INVALID_ARGUMENT, dict()),  # no workspace
])
def test_attention_refusals(status, changes):
    refused(status, "qd_paged_attention", cache(), attention(**changes), None, None)


@pytest.mark.parametrize("status,changes,memory", [
    (qd.NOT_SUPPORTED, dict(page_size=12), {}),
    (qd.NOT_SUPPORTED, dict(rows=1025), {}),
    (qd.NOT_SUPPORTED, dict(append=(1 << 30) + 1), {}),
    (qd.INVALID_ARGUMENT, dict(table=None), {}),
    (qd.INVALID_ARGUMENT, dict(refs=None), {}),
    (qd.INVALID_ARGUMENT, dict(table_out=AT), {}),
    (qd.INVALID_ARGUMENT, dict(lengths_out=AT), {}),
    (qd.INVALID_ARGUMENT, dict(table_out_stride=4), {}),
    (qd.INVALID_ARGUMENT, dict(memory_count=5), {}),
    (qd.INVALID_ARGUMENT, {}, dict(base=None)),
    (qd.INVALID_ARGUMENT, {}, dict(base=AT + 8)),
    (qd.INVALID_ARGUMENT, {}, dict(bytes=8200)),
    (qd.INVALID_ARGUMENT, {}, dict(page_stride=4096)),
    (qd.INVALID_ARGUMENT, {}, dict(plane_stride=4096)),
    (qd.INVALID_ARGUMENT, {}, dict(planes=0)),
    (qd.INVALID_ARGUMENT, {}, {}),  # no workspace
])
def test_fork_refusals(status, changes, memory):
    refused(status, "qd_pages_fork", fork(memory, **changes), None, None)


@pytest.mark.parametrize("status,changes", [
    (qd.INVALID_ARGUMENT, dict(dtype=9)),
    (qd.INVALID_ARGUMENT, dict(beams=0)),
    (qd.INVALID_ARGUMENT, dict(k=0)),
    (qd.NOT_SUPPORTED, dict(beams=33)),
    (qd.NOT_SUPPORTED, dict(k=65)),
    (qd.INVALID_ARGUMENT, dict(beams=1, vocab=3, k=4)),
    (qd.NOT_SUPPORTED, dict(vocab=(1 << 24) + 1)),
    (qd.NOT_SUPPORTED, dict(groups=20000)),
    (qd.INVALID_ARGUMENT, dict(scores=None)),
    (qd.INVALID_ARGUMENT, dict(logits=AT + 2)),
    (qd.INVALID_ARGUMENT, dict(done=AT)),
    (qd.INVALID_ARGUMENT, dict(done=AT, done_out=2 * AT, eos=1000)),
    (qd.INVALID_ARGUMENT, dict(done=AT, done_out=AT)),
    (qd.INVALID_ARGUMENT, dict(scores_out=AT)),
    (qd.INVALID_ARGUMENT, dict(beam_stride=-1)),
    (qd.INVALID_ARGUMENT, dict()),  # no workspace
])
def test_select_refusals(status, changes):
    refused(status, "qd_beam_select", select(**changes), None, None)


def test_more_workgroups_than_a_grid_has_are_refused():
    refused(qd.NOT_SUPPORTED, "qd_paged_attention", cache(rows=1 << 20, kv_heads=16, token_stride=1024, page_stride=16384),
            attention(heads=16, q_stride=1024, out_stride=1024), None, None)


def test_null_arguments_are_refused():
    refused(qd.INVALID_ARGUMENT, "qd_paged_append", None, append(), None)
    refused(qd.INVALID_ARGUMENT, "qd_paged_append", cache(), None, None)
    refused(qd.INVALID_ARGUMENT, "qd_paged_attention", cache(), None, None, None)
    refused(qd.INVALID_ARGUMENT, "qd_pages_fork", None, None, None)
    refused(qd.INVALID_ARGUMENT, "qd_beam_select", None, None, None)
    refused(qd.INVALID_ARGUMENT, "qd_workspace_create", 0, 16, None)
    assert ops.lib().qd_workspace_destroy(None) == qd.SUCCESS


def test_workspace_sizes():
    assert ops.attention_workspace(16, 14, 2, 64) > 0
    assert ops.attention_workspace(0, 14, 2, 64) >= 0
    assert ops.fork_workspace(1024, 100000) > 400000
    assert ops.select_workspace(1, 16, 16, 151936) > 0
    with pytest.raises(qd.QdError):
        ops.attention_workspace(16, 15, 2, 64)
    with pytest.raises(qd.QdError):
        ops.fork_workspace(1025, 10)
    with pytest.raises(qd.QdError):
        ops.select_workspace(1, 16, 65, 1000)


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (14, 2), (16, 1), (48, 3), (128, 8), (65536, 4096), (63000, 3000)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_never_needs_more_than_of_more_rows(heads, kv_heads, dim):
    sizes = [ops.attention_workspace(rows, heads, kv_heads, dim) for rows in [*range(40), *range(40, 1 << 17, 997), 1 << 20]]
    assert sizes == sorted(sizes)


def test_a_selection_never_needs_more_than_a_larger_one():
    rng = random.Random(7)
    for _ in range(3000):
        beams, vocab = rng.randint(1, 32), int(10 ** rng.uniform(0, 7.2))
        sizes = [rng.randint(1, 65535 // (beams + 1)), beams, rng.randint(1, min(64, beams * vocab)), vocab]
        least = [rng.randint(1, n) for n in sizes]
        fewer = [rng.choice(pair) for pair in zip(sizes, least)]
        if fewer[2] <= fewer[1] * fewer[3]:
            assert ops.select_workspace(*fewer) <= ops.select_workspace(*sizes), (fewer, sizes)
    assert ops.select_workspace(64, 8, 8, 151936) <= ops.select_workspace(75, 8, 8, 151936)


@pytest.mark.skipif(qd.device_count() > 0, reason="host-without-GPU behaviour")
def test_without_a_gpu_calls_fail_loudly():
    with pytest.raises(qd.QdError) as e:
        ops.Workspace(1024)
    assert e.value.status == qd.NOT_SUPPORTED
    refused(qd.NOT_SUPPORTED, "qd_paged_append", cache(), append(), None)


def test_numbers_that_the_structures_would_cut_are_refused():
    import torch

    k = torch.zeros(4, 16, 2, 64)
    table, lengths = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    c = ops.PagedCache(k, k, table, lengths)
    for bias in (2 ** 31, -2 ** 31 - 1, 2 ** 32):
        with pytest.raises(qd.QdError, match="position_bias"):
            ops.paged_append(c, None, None, k[0, :1], k[0, :1], lengths, position_bias=bias)
    for t in (k[:, :0], k[None][:0]):
        with pytest.raises(qd.QdError):
            ops.PagePool(torch.zeros(4, dtype=torch.int32), 16, [t], planes=t.dim() == 5)
    for dim, positions in ((-2, 4), (64, -1)):
        with pytest.raises(qd.QdError):
            ops.rope_table(1e4, dim, positions)


def test_arguments_that_are_something_else_are_refused():
    import types

    import torch

    k = torch.zeros(4, 16, 2, 64)
    table, lengths = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    c, q, new = ops.PagedCache(k, k, table, lengths), torch.zeros(1, 4, 64), k[0, :1]
    closed = types.SimpleNamespace(handle=0)
    pool = ops.PagePool(torch.zeros(4, dtype=torch.int32), 16, [k], planes=False)
    logits, best, ids = torch.zeros(1, 2, 50), torch.zeros(1, 4), torch.zeros(1, 4, dtype=torch.int32)
    for call, text in (
            (lambda: ops.paged_append(c, None, None, [1], new, lengths), "k is no tensor"),
            (lambda: ops.paged_append(c, None, None, None, new, lengths), "k is missing"),
            (lambda: ops.paged_append(c, None, None, new, new, lengths, position_bias=1.5), "position_bias"),
            (lambda: ops.paged_append(c, None, None, new, new, lengths, stream="s"), "stream"),
            (lambda: ops.paged_append(c, None, None, new, new, lengths, interleaved=q), "interleaved"),
            (lambda: ops.paged_append(c, q, q, new, new, lengths, cos=new[0, 0]), "cos and sin"),
            (lambda: ops.paged_append(c, q, q[:, :3], new, new, lengths), "q_out has shape"),
            (lambda: ops.paged_attention(c, q, q, closed), "null workspace"),
            (lambda: ops.paged_attention(c, q, q, closed, scale="x"), "scale"),
            (lambda: ops.paged_attention(c, q, q.transpose(1, 2), closed), "q has shape"),
            (lambda: ops.pages_fork(pool, table, lengths, None, -1, table.clone(), lengths.clone(), closed), "append"),
            (lambda: ops.pages_fork(pool, table, lengths, None, 1, table.clone(), lengths.clone(), closed), "null workspace"),
            (lambda: ops.pages_fork(pool, table, lengths, None, 1, table, lengths.clone(), closed), "must not be"),
            (lambda: ops.pages_fork(pool, table, lengths, lengths.long(), 1, table.clone(), lengths.clone(), closed), "parents has type"),
            (lambda: ops.beam_select(logits.double(), best, best, ids, ids, closed), "logits of type"),
            (lambda: ops.beam_select(logits, best[:, :2], best, ids, ids.clone(), closed), "must not be"),
            (lambda: ops.beam_select(logits, torch.zeros(1, 2), best, ids, ids, closed, done=ids), "go together"),
            (lambda: ops.beam_select(logits.to_sparse(), torch.zeros(1, 2), best, ids, ids, closed), None)):
        with pytest.raises(qd.QdError, match=text):
            call()


def test_cpu_tensors_are_refused():
    import torch

    k = torch.zeros(4, 16, 2, 64)
    table, lengths = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(qd.QdError):
        ops.PagedCache(k, k.bfloat16(), table, lengths)
    with pytest.raises(qd.QdError):
        ops.PagedCache(k, k, table.long(), lengths)
    c = ops.PagedCache(k, k, table, lengths)  # its device, -1, is refused by the library
    q = torch.zeros(1, 14, 64)
    with pytest.raises(qd.QdError):
        ops.paged_append(c, q, q, k[0, :1], k[0, :1], lengths)
    with pytest.raises(qd.QdError):
        ops.paged_append(c, q, q.half(), k[0, :1], k[0, :1], lengths)


def test_rope_table_plain():
    cos, sin = ops.rope_table(1e6, 64, 5000)
    p = np.arange(5000)[:, None]
    f = 1e6 ** (-np.arange(32) / 32.0)
    # The angle in 64 bits is off by 2^-53 of itself in each of two roundings; one FP32 rounding.
    assert np.abs(cos - np.cos(p * f)).max() <= 2.0 ** -25 + 5000 * 2.0 ** -50
    assert np.abs(sin - np.sin(p * f)).max() <= 2.0 ** -25 + 5000 * 2.0 ** -50


def test_rope_table_stretched():
    stretch, original = 4.0, 32768
    cos, sin = ops.rope_table(1e6, 128, 300, stretch, original)
    size = 0.1 * math.log(stretch) + 1
    for i in (0, 20, 40, 63):
        f = 1e6 ** (-i / 64.0)
        turns = original * f / (2 * math.pi)
        keep = min(1.0, max(0.0, math.log(turns) / math.log(32.0)))
        g = f * (keep + (1 - keep) / stretch)
        for p in (0, 1, 299):
            assert abs(float(cos[p, i]) - math.cos(p * g) * size) <= 2.0 ** -23
            assert abs(float(sin[p, i]) - math.sin(p * g) * size) <= 2.0 ** -23
    # The fastest rotation stays, the slowest is divided.
    assert np.allclose(sin[1, 0], math.sin(1.0) * size) and np.allclose(sin[1, 63] / size, 1e6 ** (-63 / 64.0) / 4, rtol=1e-6)


@pytest.mark.parametrize("bad", [dict(theta=0.0), dict(rotary_dim=63), dict(stretch=0.5), dict(stretch=2.0, original=0),
                                 dict(stretch=2.0, fast=1.0, slow=1.0), dict(theta=math.inf)])
def test_rope_table_refusals(bad):
    a = dict(theta=1e6, rotary_dim=64, positions=4, stretch=1.0, original=32768, fast=32.0, slow=1.0)
    a.update(bad)
    with pytest.raises(qd.QdError) as e:
        ops.rope_table(**a)
    assert e.value.status == qd.INVALID_ARGUMENT


def test_oracle_fork_keeps_the_counts():
    rng = random.Random(1)
    page, pages, width, rows = 16, 120, 12, 6
    refs = [0] * pages
    table, lengths = [[-1] * width for _ in range(rows)], [0] * rows
    for step in range(200):
        parents = [rng.choice([-1] + list(range(rows)) * 4) for _ in range(rows)]
        append = rng.choice([0, 1, 5, 16, 33])
        if max(lengths) + append > width * page:
            parents, append = [-1] * rows, 0
        table, lengths, refs, copies = oracle.fork(table, lengths, parents, refs, append, page)
        held = [p for line in table for p in line if p >= 0]
        assert refs == [held.count(p) for p in range(pages)]
        assert all(len([p for p in line if p >= 0]) == -(-n // page) for line, n in zip(table, lengths))
        # Where a row may write, it is alone.
        if append:
            assert all(n % page == 0 or refs[line[n // page]] == 1 for line, n in zip(table, lengths) if n)
