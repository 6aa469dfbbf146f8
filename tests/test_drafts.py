"""CPU checks of the operators on drafted tokens and chosen pages: what they refuse before any
device work, the layout of their structures, the sizes of their workspaces, and that the
oracle's tree and choice are what they say."""
import ctypes as C
import math
import os
import random
import re

import pytest
import torch

import drafts_oracle as oracle
import qd_operators as ops
import qwen_decode as qd
from test_operators import AT, HEADER, cache, refused

_P, _I64, _U32, _I32, _F = C.c_void_p, C.c_int64, C.c_uint32, C.c_int32, C.c_float


class TreeStruct(C.Structure):
    _fields_ = [("q", _P), ("out", _P), ("q_stride", _I64), ("q_node_stride", _I64), ("q_head_stride", _I64), ("out_stride", _I64),
                ("out_node_stride", _I64), ("out_head_stride", _I64), ("parents", _P), ("nodes", _U32), ("heads", _U32), ("scale", _F)]


class AcceptStruct(C.Structure):
    _fields_ = [("logits", _P), ("row_stride", _I64), ("node_stride", _I64), ("tokens", _P), ("parents", _P), ("draws", _P),
                ("path", _P), ("counts", _P), ("next_tokens", _P), ("errors", _P), ("temperature", _F), ("dtype", _U32), ("rows", _U32),
                ("nodes", _U32), ("vocab", _U32), ("device", _I32)]


class CommitStruct(C.Structure):
    _fields_ = [("table", _P), ("lengths", _P), ("path", _P), ("counts", _P), ("lengths_out", _P), ("table_stride", _I64),
                ("errors", _P), ("memories", C.POINTER(ops.TokenStruct)), ("memory_count", _U32), ("rows", _U32), ("nodes", _U32),
                ("table_width", _U32), ("pages", _U32), ("page_size", _U32), ("device", _I32)]


class SparseStruct(C.Structure):
    _fields_ = [("q", _P), ("out", _P), ("q_stride", _I64), ("q_head_stride", _I64), ("out_stride", _I64), ("out_head_stride", _I64),
                ("bounds", _P), ("chosen", _P), ("heads", _U32), ("budget", _U32), ("first", _U32), ("last", _U32), ("scale", _F)]


def make(cls, base, changes):
    base.update(changes)
    return cls(**base)


def tree(**changes):
    return make(TreeStruct, dict(q=AT, out=AT, q_stride=5 * 896, q_node_stride=896, q_head_stride=64, out_stride=5 * 896, out_node_stride=896,
                                 out_head_stride=64, parents=AT, nodes=5, heads=14, scale=0.125), changes)


def accept(**changes):
    return make(AcceptStruct, dict(logits=AT, row_stride=5000, node_stride=1000, tokens=AT, parents=AT, draws=None, path=2 * AT, counts=AT,
                                   next_tokens=AT, errors=None, temperature=1.0, dtype=qd.DTYPE_F32, rows=3, nodes=5, vocab=1000, device=0),
                changes)


def commit(memory=None, **changes):
    m = dict(base=AT, plane_stride=1 << 20, page_stride=8192, token_stride=512, piece_stride=256, piece_bytes=256, pieces=2, planes=2, reserved=0)
    m.update(memory or {})
    return make(CommitStruct, dict(table=AT, lengths=AT, path=AT, counts=AT, lengths_out=2 * AT, table_stride=8, errors=None,
                                   memories=(ops.TokenStruct * 1)(ops.TokenStruct(**m)), memory_count=1, rows=3, nodes=5, table_width=8, pages=10,
                                   page_size=16, device=0), changes)


def sparse(**changes):
    return make(SparseStruct, dict(q=AT, out=AT, q_stride=896, q_head_stride=64, out_stride=896, out_head_stride=64, bounds=AT, chosen=None,
                                   heads=14, budget=4, first=1, last=1, scale=0.125), changes)


def test_structures_have_the_declared_fields():
    text = open(HEADER).read()
    for struct, cls in (("qd_tree_attention_args", TreeStruct), ("qd_accept_args", AcceptStruct), ("qd_token_memory", ops.TokenStruct),
                        ("qd_commit_args", CommitStruct), ("qd_sparse_args", SparseStruct)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, re.S).group(1), flags=re.S)
        fields = [(m.group(1), "*" in line) for line in body.split(";") for m in [re.search(r"(\w+)\s*$", line.strip())] if m]
        assert [f for f, _ in fields] == [f for f, _ in cls._fields_], struct
        for (name, pointer), (_, kind) in zip(fields, cls._fields_):
            assert C.sizeof(kind) == 8 or not pointer, (struct, name)


@pytest.mark.parametrize("status,changes", [
    (qd.NOT_SUPPORTED, dict(nodes=0)), (qd.NOT_SUPPORTED, dict(nodes=65)), (qd.INVALID_ARGUMENT, dict(heads=13)),
    (qd.INVALID_ARGUMENT, dict(heads=0)), (qd.INVALID_ARGUMENT, dict(scale=math.inf)), (qd.INVALID_ARGUMENT, dict(scale=math.nan)),
    (qd.INVALID_ARGUMENT, dict(q=None)), (qd.INVALID_ARGUMENT, dict(out=None)), (qd.INVALID_ARGUMENT, dict(parents=None)),
    (qd.INVALID_ARGUMENT, dict(q=AT + 4)), (qd.INVALID_ARGUMENT, dict(out=AT + 8)), (qd.INVALID_ARGUMENT, dict(q_node_stride=-896)),
    (qd.INVALID_ARGUMENT, dict(q_node_stride=897, out=2 * AT)), (qd.INVALID_ARGUMENT, dict(out_node_stride=32, out=2 * AT)),
    (qd.INVALID_ARGUMENT, dict(out_node_stride=960)), (qd.INVALID_ARGUMENT, dict(out_stride=6 * 896)),
    (qd.INVALID_ARGUMENT, dict(out_head_stride=128)), (qd.INVALID_ARGUMENT, dict())])
def test_tree_attention_refusals(status, changes):
    refused(status, "qd_tree_attention", cache(), tree(**changes), None, None)


def test_tree_attention_of_too_much_is_refused():
    wide = cache(kv_heads=4096, rows=1 << 20, table_width=1, table_stride=1, token_stride=4096 * 64, page_stride=4096 * 64 * 16)
    refused(qd.NOT_SUPPORTED, "qd_tree_attention", wide, tree(heads=4096, q_stride=0, q=2 * AT, out_stride=64), None, None)


@pytest.mark.parametrize("status,changes", [
    (qd.INVALID_ARGUMENT, dict(dtype=3)), (qd.NOT_SUPPORTED, dict(nodes=0)), (qd.NOT_SUPPORTED, dict(nodes=65)),
    (qd.INVALID_ARGUMENT, dict(vocab=0)), (qd.NOT_SUPPORTED, dict(vocab=(1 << 24) + 1)), (qd.NOT_SUPPORTED, dict(rows=11000)),
    (qd.INVALID_ARGUMENT, dict(logits=None)), (qd.INVALID_ARGUMENT, dict(tokens=None)), (qd.INVALID_ARGUMENT, dict(parents=None)),
    (qd.INVALID_ARGUMENT, dict(path=None)), (qd.INVALID_ARGUMENT, dict(counts=None)), (qd.INVALID_ARGUMENT, dict(next_tokens=None)),
    (qd.INVALID_ARGUMENT, dict(path=AT)), (qd.INVALID_ARGUMENT, dict(logits=AT + 2)), (qd.INVALID_ARGUMENT, dict(row_stride=-1)),
    (qd.INVALID_ARGUMENT, dict(node_stride=-1)), (qd.INVALID_ARGUMENT, dict(draws=AT, temperature=0.0)),
    (qd.INVALID_ARGUMENT, dict(draws=AT, temperature=math.nan)), (qd.INVALID_ARGUMENT, dict(draws=AT, temperature=1e7)),
    (qd.INVALID_ARGUMENT, dict())])
def test_accept_refusals(status, changes):
    refused(status, "qd_tree_accept", accept(**changes), None, None)


@pytest.mark.parametrize("result", ["path", "counts", "next_tokens"])
@pytest.mark.parametrize("other,at", [("tokens", 0), ("tokens", 14), ("parents", 0), ("parents", -2), ("draws", 0), ("draws", 3), ("path", 14),
                                      ("counts", 0), ("counts", -2), ("next_tokens", 2)])
def test_accept_refuses_results_over_each_other_and_what_it_reads(result, other, at):
    names = ("tokens", "parents", "draws", "path", "counts", "next_tokens")
    changes = {name: AT + 4096 * i for i, name in enumerate(names)}
    if result == other:
        refused(qd.INVALID_ARGUMENT, "qd_tree_accept", accept(**changes), None, None)
        assert b"null workspace" in ops.lib().qd_last_error()
        return
    changes[result] = changes[other] + 4 * at
    refused(qd.INVALID_ARGUMENT, "qd_tree_accept", accept(**changes), None, None)
    assert b"overlap" in ops.lib().qd_last_error()


def test_accept_of_one_node_takes_its_tokens_in_place():
    names = ("tokens", "parents", "draws", "path", "counts")
    changes = {name: AT + 4096 * i for i, name in enumerate(names)}
    for nodes, text in ((1, b"null workspace"), (5, b"overlap")):
        refused(qd.INVALID_ARGUMENT, "qd_tree_accept", accept(nodes=nodes, next_tokens=AT, **changes), None, None)
        assert text in ops.lib().qd_last_error()


@pytest.mark.parametrize("status,memory,changes", [
    (qd.NOT_SUPPORTED, {}, dict(page_size=24)), (qd.NOT_SUPPORTED, {}, dict(nodes=0)), (qd.NOT_SUPPORTED, {}, dict(nodes=65)),
    (qd.NOT_SUPPORTED, {}, dict(rows=65536)), (qd.INVALID_ARGUMENT, {}, dict(pages=1 << 31)),
    (qd.NOT_SUPPORTED, {}, dict(table_width=1 << 27, table_stride=1 << 27)), (qd.INVALID_ARGUMENT, {}, dict(table=None)),
    (qd.INVALID_ARGUMENT, {}, dict(lengths=None)), (qd.INVALID_ARGUMENT, {}, dict(path=None)), (qd.INVALID_ARGUMENT, {}, dict(counts=None)),
    (qd.INVALID_ARGUMENT, {}, dict(lengths_out=None)), (qd.INVALID_ARGUMENT, {}, dict(lengths_out=AT)),
    (qd.INVALID_ARGUMENT, {}, dict(table_stride=7)), (qd.INVALID_ARGUMENT, {}, dict(memory_count=5)),
    (qd.INVALID_ARGUMENT, dict(base=None), {}), (qd.INVALID_ARGUMENT, dict(base=AT + 4), {}), (qd.INVALID_ARGUMENT, dict(piece_bytes=8), {}),
    (qd.INVALID_ARGUMENT, dict(piece_bytes=0), {}), (qd.INVALID_ARGUMENT, dict(pieces=0), {}), (qd.INVALID_ARGUMENT, dict(planes=0), {}),
    (qd.INVALID_ARGUMENT, dict(token_stride=128), {}), (qd.INVALID_ARGUMENT, dict(piece_stride=128), {}),
    (qd.INVALID_ARGUMENT, dict(plane_stride=-16), {}), (qd.INVALID_ARGUMENT, dict(page_stride=8), {}), (qd.INVALID_ARGUMENT, dict(page_stride=0), {}),
    (qd.INVALID_ARGUMENT, dict(plane_stride=0), {}), (qd.NOT_SUPPORTED, dict(pieces=1 << 28, planes=1), {}),
    (qd.NOT_SUPPORTED, dict(pieces=1 << 26, planes=1), dict(rows=65535))])
def test_commit_refusals(status, memory, changes):
    refused(status, "qd_tree_commit", commit(memory, **changes), None)


@pytest.mark.parametrize("other,at", [("lengths", 0), ("lengths", 2), ("counts", 0), ("counts", -2), ("path", 0), ("path", 14), ("path", -2),
                                      ("table", 0), ("table", 7), ("table", 8), ("table", 23), ("table", 12), ("table", 17)])
def test_commit_refuses_lengths_over_what_it_reads(other, at):
    """Some of a row's workgroups would read what another has written."""
    changes = {name: AT + 4096 * i for i, name in enumerate(("lengths", "counts", "path", "table"))}
    changes.update(lengths_out=changes[other] + 4 * at, table_stride=10)
    refused(qd.INVALID_ARGUMENT, "qd_tree_commit", commit(**changes), None)
    assert b"lengths_out" in ops.lib().qd_last_error()


@pytest.mark.parametrize("other,at", [("lengths", 3), ("lengths", -3), ("counts", 3), ("path", 15), ("path", -3), ("table", 30), ("table", -3),
                                      ("table", 19), ("table", 8)])
def test_commit_takes_lengths_beside_what_it_reads(other, at):
    """(In the gap behind a row of the table too, if they fit.) The device is the next thing that is looked at."""
    changes = {name: AT + 4096 * i for i, name in enumerate(("lengths", "counts", "path", "table"))}
    rows = 2 if other == "table" and at == 8 else 3
    changes.update(lengths_out=changes[other] + 4 * at, rows=rows, table_stride=10 if rows == 2 else 11, device=-1)
    refused(qd.INVALID_ARGUMENT if torch.cuda.is_available() else qd.NOT_SUPPORTED, "qd_tree_commit", commit(**changes), None)
    assert b"lengths_out" not in ops.lib().qd_last_error()


@pytest.mark.parametrize("status,changes,bounds,recent", [
    (qd.INVALID_ARGUMENT, dict(dtype=7), AT, 1), (qd.INVALID_ARGUMENT, {}, None, 1), (qd.INVALID_ARGUMENT, {}, AT + 8, 1),
    (qd.NOT_SUPPORTED, dict(rows=1 << 20, table_width=1 << 10, table_stride=1 << 10), AT, 1 << 20)])
def test_bounds_refusals(status, changes, bounds, recent):
    refused(status, "qd_page_bounds", cache(**changes), bounds, recent, None)


@pytest.mark.parametrize("status,changes", [
    (qd.INVALID_ARGUMENT, dict(budget=0)), (qd.INVALID_ARGUMENT, dict(budget=(1 << 20) + 1)), (qd.INVALID_ARGUMENT, dict(last=0)),
    (qd.INVALID_ARGUMENT, dict(first=4)), (qd.INVALID_ARGUMENT, dict(first=2, last=3)), (qd.INVALID_ARGUMENT, dict(last=1 << 31, first=1 << 31)),
    (qd.INVALID_ARGUMENT, dict(heads=13)), (qd.INVALID_ARGUMENT, dict(scale=math.nan)), (qd.INVALID_ARGUMENT, dict(q=None)),
    (qd.INVALID_ARGUMENT, dict(out=AT + 4)), (qd.INVALID_ARGUMENT, dict(bounds=None)), (qd.INVALID_ARGUMENT, dict(bounds=AT + 4)),
    (qd.INVALID_ARGUMENT, dict(q_stride=960)), (qd.INVALID_ARGUMENT, dict())])
def test_sparse_refusals(status, changes):
    refused(status, "qd_sparse_attention", cache(), sparse(**changes), None, None)


@pytest.mark.parametrize("place,text", [(AT, b"chosen"), (AT + 4 * 23, b"chosen"), (AT - 4 * 23, b"chosen"), (2 * AT + 8, b"chosen"),
                                        (AT + 4 * 24, b"null workspace"), (AT - 4 * 24, b"null workspace")])
def test_sparse_refuses_a_list_over_what_it_reads(place, text):
    """Three rows of eight columns, lists of four for two heads."""
    refused(qd.INVALID_ARGUMENT, "qd_sparse_attention", cache(lengths=2 * AT), sparse(chosen=place), None, None)
    assert text in ops.lib().qd_last_error()


def test_sparse_of_too_many_rows_is_refused():
    refused(qd.NOT_SUPPORTED, "qd_sparse_attention", cache(rows=40000), sparse(), None, None)


def test_null_arguments_are_refused():
    for call, args in (("qd_tree_attention", (cache(), None, None, None)), ("qd_tree_attention", (None, tree(), None, None)),
                       ("qd_tree_accept", (None, None, None)), ("qd_tree_commit", (None, None)), ("qd_page_bounds", (None, AT, 1, None)),
                       ("qd_sparse_attention", (cache(), None, None, None)), ("qd_sparse_attention", (None, sparse(), None, None)),
                       ("qd_paged_append_at", (cache(), None, None, None))):
        refused(qd.INVALID_ARGUMENT, call, *args)


def test_a_workspace_serves_every_smaller_call():
    rng = random.Random(5)
    for _ in range(400):
        kv_heads = rng.choice([1, 2, 3, 8, 40])
        heads, dim = kv_heads * rng.randint(1, 20), rng.choice([64, 128])
        rows, nodes = int(10 ** rng.uniform(0, 5)), rng.randint(1, 64)
        most = ops.tree_attention_workspace(rows, nodes, heads, kv_heads, dim)
        assert ops.tree_attention_workspace(rng.randint(1, rows), rng.randint(1, nodes), heads, kv_heads, dim) <= most
        rows = min(rows, 65535 // (nodes + 1))
        most = ops.tree_accept_workspace(rows, nodes, 50000)
        assert ops.tree_accept_workspace(rng.randint(1, rows), rng.randint(1, nodes), rng.randint(1, 50000)) <= most
        rows, width, budget = min(rows, 65535 // kv_heads), rng.randint(1, 5000), rng.randint(1, 300)
        most = ops.sparse_attention_workspace(rows, heads, kv_heads, dim, width, budget)
        assert ops.sparse_attention_workspace(rng.randint(1, rows), heads, kv_heads, dim, rng.randint(1, width), rng.randint(1, budget)) <= most


@pytest.mark.parametrize("rows,nodes,heads,kv_heads,dim,most", [(2, 63, 28, 4, 128, 26 << 20), (1, 8, 14, 2, 64, 13 << 20), (64, 64, 32, 8, 128, 137 << 20),
                                                                 (1, 64, 65536, 4096, 128, 4 << 30)])
def test_tree_attention_asks_for_no_more_than_its_pieces_write(rows, nodes, heads, kv_heads, dim, most):
    """Pieces of a row's items: one and `target` more in all, four times as many where rows are not few; a record has 2 more
    numbers than values. Two rows of 63 nodes of 7 heads: 16-bit, 9 nodes, 64 columns, (2 + 192) x 4 records of 64 x 130 numbers."""
    assert ops.tree_attention_workspace(rows, nodes, heads, kv_heads, dim) <= most


def test_arguments_that_are_something_else_are_refused():
    import types

    k = torch.zeros(4, 16, 2, 64)
    table, lengths = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    c, q, closed = ops.PagedCache(k, k, table, lengths), torch.zeros(1, 3, 4, 64), types.SimpleNamespace(handle=0)
    parents, logits, out = torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, 3, 50), torch.zeros(1, dtype=torch.int32)
    memory, low_high = ops.TokenMemory([k], planes=False), torch.zeros(4, 2, 2, 64)
    for call, text in (
            (lambda: ops.tree_attention(c, q, q[0], parents, closed), "q needs 4"),
            (lambda: ops.tree_attention(c, q[:, :2], q, parents, closed), "out has shape"),
            (lambda: ops.tree_attention(c, q, q, parents.long(), closed), "parents has type"),
            (lambda: ops.tree_attention(c, q, q, parents[:, :2], closed), "parents has shape"),
            (lambda: ops.tree_attention(c, q, q, parents, closed, scale="x"), "scale"),
            (lambda: ops.tree_attention(c, q, q, parents, closed), "null workspace"),
            (lambda: ops.tree_accept(logits.double(), parents, parents, parents, out, out, closed), "logits of type"),
            (lambda: ops.tree_accept(logits, parents, parents, parents, out, out, closed), "path must not be"),
            (lambda: ops.tree_accept(logits, parents, parents, parents.clone(), out, out, closed, draws=logits), "draws has shape"),
            (lambda: ops.tree_accept(logits, parents, parents, parents.clone(), out, out, closed, temperature=None), "temperature"),
            (lambda: ops.tree_commit(memory, table, lengths, parents, out, lengths), "must not be lengths"),
            (lambda: ops.tree_commit(memory, table, lengths, parents, None, out), "counts is missing"),
            (lambda: ops.tree_commit(memory, table, lengths, parents[0], out, out), "path needs 2"),
            (lambda: ops.TokenMemory([]), "without tensors"),
            (lambda: ops.TokenMemory([k, k[:, :8]], planes=False), "does not hold"),
            (lambda: ops.TokenMemory([k[..., ::2]], planes=False), "not contiguous"),
            (lambda: ops.TokenMemory([k]), "needs 5 dimensions"),
            (lambda: ops.page_bounds(c, low_high[:3], 1), "bounds has shape"),
            (lambda: ops.page_bounds(c, low_high.half(), 1), "bounds has type"),
            (lambda: ops.page_bounds(c, low_high, -1), "recent"),
            (lambda: ops.sparse_attention(c, low_high, q[:, 0], q[:, 0], closed, -1), "budget"),
            (lambda: ops.sparse_attention(c, low_high, q[:, 0], q[:, 0], closed, 2, chosen=parents), "chosen has shape"),
            (lambda: ops.sparse_attention(c, low_high, q[:, 0], q[:, 0], closed, 2), "null workspace"),
            (lambda: ops.paged_append(c, None, None, k[0, :1], k[0, :1], lengths, slots=lengths.long()), "slots has type")):
        with pytest.raises(qd.QdError, match=text):
            call()


def test_transfers_wait_for_scalar_registers_of_vector_instructions():
    """A transfer whose address is in scalar registers, which a vector instruction may have written right before:
    five wait states between them."""
    text = open(os.path.join(os.path.dirname(HEADER), "..", "..", "light-rocm-runtime_amd", "csrc", "qd_tree.hip")).read()
    found = re.findall(r's_nop (\d+)\\n\\tglobal_load_lds_dwordx4 %1, %2', text)
    assert found and all(int(n) >= 4 for n in found)


def test_oracle_chains_and_choices():
    parents = [-1, 0, 0, 1, -2, 3]
    assert [oracle.chain(parents, i) for i in range(6)] == [[0], [0, 1], [0, 2], [0, 1, 3], [], [0, 1, 3, 5]]
    # Of pages with one key each the bounds are the key, and the score its product with the queries' sum.
    k = torch.randn((30, 1, 1, 64), generator=torch.Generator().manual_seed(1))
    low_high = oracle.bounds(k, torch.arange(30)[None], [30], 30, torch.zeros((30, 1, 2, 64)))
    q = torch.randn((3, 64), generator=torch.Generator().manual_seed(2))
    score = (k[:, 0, 0].double() @ q.double().sum(0)).tolist()
    got = oracle.choose(q, low_high, torch.arange(30), 30, 1, 0, 3, 9, 2, 1)
    assert got == [0, 1, *sorted(sorted(range(2, 29), key=lambda i: -score[i])[:6]), 29]
