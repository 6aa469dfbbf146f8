"""Python mirror of the operators on device memory (include/qd/qd_operators.h).

A thin layer over libqwen_decode.so for programs that hold torch tensors on the
GPU: shapes, types, strides and devices are taken from the tensors and checked,
the work is queued on `stream` (a raw stream handle such as
torch.cuda.current_stream().cuda_stream; 0 is the null stream), and errors raise
QdError. Tensors must stay alive until the stream has run the call; a tensor of
another stream needs the caller's wait or event, as with any kernel launch.

torch brings a HIP runtime of its own, and a process can hold one: import torch, or
this module, before the first call into the engine's library.
"""
from __future__ import annotations

import ctypes as C
import sys

import numpy as np

import qwen_decode as qd
from qwen_decode import QdError  # noqa: F401  (what the calls raise)

if qd._lib is not None and "torch" not in sys.modules:
    raise ImportError("the engine's library is loaded with another HIP runtime than torch's: "
                      "import torch or qd_operators before the first call of qwen_decode")
import torch  # noqa: E402

BAD_LENGTH, BAD_PAGE, BAD_POSITION, BAD_ROW, EXHAUSTED = 1, 2, 4, 8, 16

_P, _I64, _U32, _I32 = C.c_void_p, C.c_int64, C.c_uint32, C.c_int32


class CacheStruct(C.Structure):
    _fields_ = [("k", _P), ("v", _P), ("page_stride", _I64), ("token_stride", _I64), ("head_stride", _I64),
                ("table", _P), ("table_stride", _I64), ("lengths", _P), ("errors", _P), ("rows", _U32),
                ("table_width", _U32), ("pages", _U32), ("page_size", _U32), ("kv_heads", _U32), ("head_dim", _U32),
                ("dtype", _U32), ("device", _I32)]


class AppendStruct(C.Structure):
    _fields_ = [("q", _P), ("k", _P), ("v", _P), ("q_out", _P), ("q_stride", _I64), ("k_stride", _I64),
                ("v_stride", _I64), ("q_out_stride", _I64), ("positions", _P), ("rows", _P), ("position_bias", _I32),
                ("tokens", _U32), ("heads", _U32), ("rotary_dim", _U32), ("interleaved", _U32),
                ("table_positions", _U32), ("cos_table", _P), ("sin_table", _P)]


class AttentionStruct(C.Structure):
    _fields_ = [("q", _P), ("out", _P), ("q_stride", _I64), ("q_head_stride", _I64), ("out_stride", _I64),
                ("out_head_stride", _I64), ("heads", _U32), ("scale", C.c_float)]


class MemoryStruct(C.Structure):
    _fields_ = [("base", _P), ("plane_stride", _I64), ("page_stride", _I64), ("bytes", C.c_uint64), ("planes", _U32),
                ("reserved", _U32)]


class ForkStruct(C.Structure):
    _fields_ = [("table", _P), ("lengths", _P), ("parents", _P), ("table_out", _P), ("lengths_out", _P), ("refs", _P),
                ("table_stride", _I64), ("table_out_stride", _I64), ("errors", _P), ("memories", C.POINTER(MemoryStruct)),
                ("memory_count", _U32), ("rows", _U32), ("table_width", _U32), ("pages", _U32), ("page_size", _U32),
                ("append", _U32), ("device", _I32)]


class SelectStruct(C.Structure):
    _fields_ = [("logits", _P), ("group_stride", _I64), ("beam_stride", _I64), ("scores", _P), ("done", _P),
                ("scores_out", _P), ("parents", _P), ("tokens", _P), ("done_out", _P), ("dtype", _U32), ("groups", _U32),
                ("beams", _U32), ("vocab", _U32), ("k", _U32), ("eos", _U32), ("device", _I32)]


_SIZE = C.POINTER(C.c_size_t)
_SIGNATURES = {
    "qd_workspace_create": [_I32, C.c_size_t, C.POINTER(_P)],
    "qd_workspace_destroy": [_P],
    "qd_rope_table": [C.c_double, _U32, _U32, C.c_double, _U32, C.c_double, C.c_double, C.POINTER(C.c_float),
                      C.POINTER(C.c_float)],
    "qd_paged_append": [C.POINTER(CacheStruct), C.POINTER(AppendStruct), _P],
    "qd_paged_attention": [C.POINTER(CacheStruct), C.POINTER(AttentionStruct), _P, _P],
    "qd_paged_attention_workspace": [_U32, _U32, _U32, _U32, _SIZE],
    "qd_pages_fork": [C.POINTER(ForkStruct), _P, _P],
    "qd_pages_fork_workspace": [_U32, _U32, _SIZE],
    "qd_beam_select": [C.POINTER(SelectStruct), _P, _P],
    "qd_beam_select_workspace": [_U32, _U32, _U32, _U32, _SIZE],
}

_lib = None


def lib():
    """The engine library with the operators' signatures (raises if it is not built)."""
    global _lib
    if _lib is None:
        handle = qd.lib()
        for name, args in _SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = C.c_int
            fn.argtypes = args
        _lib = handle
    return _lib


def _check(status):
    if status:
        raise QdError(status, _lib.qd_last_error().decode(errors="replace"))


# ---- what a tensor is -----------------------------------------------------------------

_TYPES = {torch.float32: qd.DTYPE_F32, torch.bfloat16: qd.DTYPE_BF16, torch.float16: qd.DTYPE_F16,
          torch.int32: "int32", torch.uint8: "uint8"}


def _dtype(t):
    """qd_dtype of a tensor, or None."""
    return _TYPES.get(t.dtype)


def _refuse(text):
    raise QdError(qd.INVALID_ARGUMENT, text)


def _dims(name, t, n):
    if t is None or t.dim() != n:
        _refuse(f"{name} needs {n} dimensions")
    return t.shape


def _expect(name, t, dtype, shape, device):
    """Address of a tensor of this type, shape and device, its last dimension contiguous."""
    if t is None or t.shape != shape:
        if t is None:
            _refuse(f"{name} is missing")
        _refuse(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    if _dtype(t) != dtype:
        _refuse(f"{name} has type {t.dtype}")
    if t.get_device() != device:
        _refuse(f"{name} is on {t.device}, not on device {device}")
    if shape and shape[-1] > 1 and t.stride(-1) != 1:
        _refuse(f"the last dimension of {name} is not contiguous")
    return t.data_ptr()


def _expect_flat(name, t, dtype, shape, device):
    if t is not None and not t.is_contiguous():
        _refuse(f"{name} is not contiguous")
    return _expect(name, t, dtype, shape, device)


def _bytes(call, *args):
    n = C.c_size_t()
    _check(getattr(lib(), call)(*args, C.byref(n)))
    return n.value


def attention_workspace(rows, heads, kv_heads, head_dim):
    return _bytes("qd_paged_attention_workspace", rows, heads, kv_heads, head_dim)


def fork_workspace(rows, pages):
    return _bytes("qd_pages_fork_workspace", rows, pages)


def select_workspace(groups, beams, k, vocab):
    return _bytes("qd_beam_select_workspace", groups, beams, k, vocab)


class Workspace:
    """Device memory for partial results, for one call at a time: work that may run at the
    same time (two streams, graphs on two streams) needs one each."""

    def __init__(self, nbytes, device=0):
        self.handle = _P()
        self.nbytes, self.device = nbytes, device
        _check(lib().qd_workspace_create(device, nbytes, C.byref(self.handle)))

    def close(self):
        if self.handle:
            handle, self.handle = self.handle, _P()
            _check(lib().qd_workspace_destroy(handle))

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PagedCache:
    """K and V pages [pages, page_size, kv_heads, head_dim] (any strides with a contiguous last
    dimension, the same for both), the rows' tables [rows, columns] and lengths [rows], int32."""

    def __init__(self, k, v, table, lengths, errors=None):
        self.tensors = (k, v, table, lengths, errors)
        _dims("k", k, 4)
        device, dtype = k.get_device(), _dtype(k)
        if dtype not in (qd.DTYPE_F32, qd.DTYPE_BF16, qd.DTYPE_F16):
            _refuse(f"pages of type {k.dtype}")
        _expect("k", k, dtype, k.shape, device)
        _expect("v", v, dtype, k.shape, device)
        if k.stride() != v.stride():
            _refuse("k and v have different strides")
        pages, page_size, kv_heads, head_dim = k.shape
        rows, width = _dims("table", table, 2)
        # The stride of a dimension of one element is not used and may be anything.
        s = [n if k.shape[i] > 1 else head_dim for i, n in enumerate(k.stride()[:3])]
        self.device, self.dtype, self.rows, self.kv_heads, self.head_dim = device, dtype, rows, kv_heads, head_dim
        self.c = CacheStruct(
            k.data_ptr(), v.data_ptr(), s[0], s[1], s[2], _expect("table", table, "int32", table.shape, device),
            table.stride(0) if rows > 1 else width, _expect_flat("lengths", lengths, "int32", (rows,), device),
            None if errors is None else _expect_flat("errors", errors, "int32", (1,), device), rows, width, pages,
            page_size, kv_heads, head_dim, dtype, device)


def _token_stride(name, t):
    """Stride from token to token of [tokens, heads, head_dim] whose heads lie together."""
    if t.shape[1] > 1 and t.stride(1) != t.shape[2]:
        _refuse(f"the heads of a token of {name} do not lie together")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]


def paged_append(cache, q_out, q, k, v, positions, rows=None, cos=None, sin=None, interleaved=False, position_bias=0,
                 stream=0):
    """Rotates new tokens' queries into q_out and writes their keys (rotated) and values into
    pages. q, q_out [tokens, heads, head_dim] (both None: keys and values only), k, v
    [tokens, kv_heads, head_dim], positions and rows [tokens] int32, cos and sin
    [positions, rotary_dim / 2] FP32 (None: no rotation)."""
    device, dtype = cache.device, cache.dtype
    tokens = _dims("k", k, 3)[0]
    shape = (tokens, cache.kv_heads, cache.head_dim)
    a = AppendStruct()
    a.k, a.v = _expect("k", k, dtype, shape, device), _expect("v", v, dtype, shape, device)
    a.k_stride, a.v_stride = _token_stride("k", k), _token_stride("v", v)
    if (q is None) != (q_out is None):
        _refuse("q and q_out go together")
    if q is not None:
        heads = _dims("q", q, 3)[1]
        shape = (tokens, heads, cache.head_dim)
        a.q, a.q_out = _expect("q", q, dtype, shape, device), _expect("q_out", q_out, dtype, shape, device)
        a.q_stride, a.q_out_stride, a.heads = _token_stride("q", q), _token_stride("q_out", q_out), heads
    a.positions = _expect_flat("positions", positions, "int32", (tokens,), device)
    if rows is not None:
        a.rows = _expect_flat("rows", rows, "int32", (tokens,), device)
    a.position_bias, a.tokens, a.interleaved = position_bias, tokens, 1 if interleaved else 0
    if (cos is None) != (sin is None):
        _refuse("cos and sin go together")
    if cos is not None:
        a.cos_table = _expect_flat("cos", cos, qd.DTYPE_F32, _dims("cos", cos, 2), device)
        a.sin_table = _expect_flat("sin", sin, qd.DTYPE_F32, cos.shape, device)
        a.table_positions, a.rotary_dim = cos.shape[0], 2 * cos.shape[1]
    _check(lib().qd_paged_append(cache.c, a, stream))


def paged_attention(cache, out, q, workspace, scale=None, stream=0):
    """Attention of one new token per cache row: q and out [rows, heads, head_dim]."""
    device, dtype = cache.device, cache.dtype
    heads = _dims("q", q, 3)[1]
    shape = (cache.rows, heads, cache.head_dim)
    a = AttentionStruct(
        _expect("q", q, dtype, shape, device), _expect("out", out, dtype, shape, device),
        q.stride(0) if cache.rows > 1 else heads * cache.head_dim, q.stride(1) if heads > 1 else cache.head_dim,
        out.stride(0) if cache.rows > 1 else heads * cache.head_dim, out.stride(1) if heads > 1 else cache.head_dim,
        heads, cache.head_dim ** -0.5 if scale is None else scale)
    _check(lib().qd_paged_attention(cache.c, a, workspace.handle, stream))


class PagePool:
    """Reference counts [pages] int32 and the tensors that hold the pages: [pages, ...] or
    [planes, pages, ...] with a page's values together."""

    def __init__(self, refs, page_size, tensors, planes=True):
        self.refs, self.page_size, self.tensors = refs, page_size, list(tensors)
        self.device, pages = refs.get_device(), _dims("refs", refs, 1)[0]
        _expect_flat("refs", refs, "int32", (pages,), self.device)
        self.memories = (MemoryStruct * max(1, len(self.tensors)))()
        for m, t in zip(self.memories, self.tensors):
            p = 1 if planes else 0
            if t.dim() <= p or t.shape[p] != pages or t.get_device() != self.device:
                _refuse(f"a tensor of shape {tuple(t.shape)} on {t.device} does not hold {pages} pages of device {self.device}")
            inner = t.select(p, 0).select(0, 0) if planes else t.select(0, 0)
            if pages and not inner.is_contiguous():
                _refuse("a page's values do not lie together")
            size = t.element_size()
            m.base, m.bytes = t.data_ptr(), inner.numel() * size
            m.planes, m.plane_stride = (t.shape[0], t.stride(0) * size) if planes else (1, 0)
            m.page_stride = t.stride(p) * size if pages > 1 else m.bytes


def pages_fork(pool, table, lengths, parents, append, table_out, lengths_out, workspace, errors=None, stream=0):
    """Row r of table_out takes over row parents[r] of table (None: its own, -1: released) with
    room for `append` more tokens; shared pages are counted and copied on write."""
    device = pool.device
    rows, width = _dims("table", table, 2)
    shape = (rows, width)
    a = ForkStruct(
        _expect("table", table, "int32", shape, device), _expect_flat("lengths", lengths, "int32", (rows,), device),
        None if parents is None else _expect_flat("parents", parents, "int32", (rows,), device),
        _expect("table_out", table_out, "int32", shape, device),
        _expect_flat("lengths_out", lengths_out, "int32", (rows,), device), pool.refs.data_ptr(),
        table.stride(0) if rows > 1 else width, table_out.stride(0) if rows > 1 else width,
        None if errors is None else _expect_flat("errors", errors, "int32", (1,), device), pool.memories,
        len(pool.tensors), rows, width, pool.refs.shape[0], pool.page_size, append, device)
    _check(lib().qd_pages_fork(a, workspace.handle, stream))


def beam_select(logits, scores, scores_out, parents, tokens, workspace, done=None, done_out=None, eos=None, stream=0):
    """The best k = scores_out.shape[1] continuations of each group: logits [groups, beams, vocab],
    scores and done [groups, beams], the results [groups, k]."""
    groups, beams, vocab = _dims("logits", logits, 3)
    device, dtype = logits.get_device(), _dtype(logits)
    if dtype not in (qd.DTYPE_F32, qd.DTYPE_BF16, qd.DTYPE_F16):
        _refuse(f"logits of type {logits.dtype}")
    k = _dims("scores_out", scores_out, 2)[1]
    if (done is None) != (done_out is None) or (done is not None and eos is None):
        _refuse("done, done_out and eos go together")
    if vocab > 1 and logits.stride(2) != 1:
        _refuse("the last dimension of logits is not contiguous")
    a = SelectStruct(
        logits.data_ptr(), logits.stride(0), logits.stride(1),
        _expect_flat("scores", scores, qd.DTYPE_F32, (groups, beams), device),
        None if done is None else _expect_flat("done", done, "uint8", (groups, beams), device),
        _expect_flat("scores_out", scores_out, qd.DTYPE_F32, (groups, k), device),
        _expect_flat("parents", parents, "int32", (groups, k), device),
        _expect_flat("tokens", tokens, "int32", (groups, k), device),
        None if done is None else _expect_flat("done_out", done_out, "uint8", (groups, k), device), dtype, groups, beams,
        vocab, k, 0 if eos is None else eos, device)
    _check(lib().qd_beam_select(a, workspace.handle, stream))


def rope_table(theta, rotary_dim, positions, stretch=1.0, original=32768, fast=32.0, slow=1.0):
    """cos and sin [positions, rotary_dim / 2] for paged_append, numpy FP32 on the host."""
    f = C.POINTER(C.c_float)
    cos, sin = (np.empty((positions, rotary_dim // 2), np.float32) for _ in range(2))
    _check(lib().qd_rope_table(theta, rotary_dim, positions, stretch, original, fast, slow, cos.ctypes.data_as(f),
                               sin.ctypes.data_as(f)))
    return cos, sin
