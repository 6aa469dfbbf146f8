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
import os
import sys

import numpy as np

import qwen_decode as qd
from qwen_decode import QdError  # noqa: F401  (what the calls raise)

if qd._lib is not None and "torch" not in sys.modules:
    raise ImportError("the engine's library is loaded with another HIP runtime than torch's: "
                      "import torch or qd_operators before the first call of qwen_decode")
import torch  # noqa: E402

try:
    import _qd_tensors  # noqa: E402  (it links to torch's libraries, which are loaded now)
except ImportError as e:
    raise ImportError(f"the operators' binding is not built: make -C {os.path.dirname(os.path.abspath(__file__))}") from e

BAD_LENGTH, BAD_PAGE, BAD_POSITION, BAD_ROW, EXHAUSTED = 1, 2, 4, 8, 16

_P, _I64, _U32, _I32 = C.c_void_p, C.c_int64, C.c_uint32, C.c_int32


class CacheStruct(C.Structure):
    _fields_ = [("k", _P), ("v", _P), ("page_stride", _I64), ("token_stride", _I64), ("head_stride", _I64),
                ("table", _P), ("table_stride", _I64), ("lengths", _P), ("errors", _P), ("rows", _U32),
                ("table_width", _U32), ("pages", _U32), ("page_size", _U32), ("kv_heads", _U32), ("head_dim", _U32),
                ("dtype", _U32), ("device", _I32)]


class MemoryStruct(C.Structure):
    _fields_ = [("base", _P), ("plane_stride", _I64), ("page_stride", _I64), ("bytes", C.c_uint64), ("planes", _U32),
                ("reserved", _U32)]


_SIZE = C.POINTER(C.c_size_t)
_SIGNATURES = {
    "qd_workspace_create": [_I32, C.c_size_t, C.POINTER(_P)],
    "qd_workspace_destroy": [_P],
    "qd_rope_table": [C.c_double, _U32, _U32, C.c_double, _U32, C.c_double, C.c_double, C.POINTER(C.c_float),
                      C.POINTER(C.c_float)],
    "qd_paged_append": [_P, _P, _P],
    "qd_paged_attention": [_P, _P, _P, _P],
    "qd_paged_attention_workspace": [_U32, _U32, _U32, _U32, _SIZE],
    "qd_pages_fork": [_P, _P, _P],
    "qd_pages_fork_workspace": [_U32, _U32, _SIZE],
    "qd_beam_select": [_P, _P, _P],
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
        _qd_tensors.bind(*(C.cast(getattr(handle, name), _P).value for name in (
            "qd_paged_append", "qd_paged_attention", "qd_pages_fork", "qd_beam_select")))
        _lib = handle
    return _lib


def _check(status):
    if status:
        raise QdError(status, _lib.qd_last_error().decode(errors="replace"))


def _answer(r):
    """Raises what a call of the binding returned: a status, or what is wrong with an argument."""
    if isinstance(r, int):
        _check(r)
    raise QdError(qd.INVALID_ARGUMENT, r)


# ---- what the calls take ----------------------------------------------------------------
# A call's tensors are checked in the binding (csrc/qd_tensors.cpp); what is made once, here.

_TYPES = {torch.float32: qd.DTYPE_F32, torch.bfloat16: qd.DTYPE_BF16, torch.float16: qd.DTYPE_F16}


def _refuse(text):
    raise QdError(qd.INVALID_ARGUMENT, text)


def _dims(name, t, n):
    if t is None or t.dim() != n:
        _refuse(f"{name} needs {n} dimensions")
    return t.shape


def _take(name, t, dtype, shape, device, together=False):
    """Address and strides of a tensor of this type, shape and device; contiguous are its last dimension
    or, `together`, all."""
    if t is None:
        _refuse(f"{name} is missing")
    if t.shape != shape:
        _refuse(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    if t.dtype is not dtype:
        _refuse(f"{name} has type {t.dtype}, not {dtype}")
    if t.get_device() != device:
        _refuse(f"{name} is on {t.device}, not on device {device}")
    s = t.stride()
    if not (t.is_contiguous() if together else s[-1] == 1 or shape[-1] <= 1):
        _refuse(f"{name} is not contiguous where it has to be (strides {s})")
    return t.data_ptr(), s


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
        self.handle = 0
        self.nbytes, self.device = nbytes, device
        handle = _P()
        _check(lib().qd_workspace_create(device, nbytes, C.byref(handle)))
        self.handle = handle.value

    def close(self):
        if self.handle:
            handle, self.handle = self.handle, 0
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
        pages, page_size, kv_heads, head_dim = _dims("k", k, 4)
        rows, width = _dims("table", table, 2)
        device, dtype = k.get_device(), k.dtype
        if dtype not in _TYPES:
            _refuse(f"pages of type {dtype}")
        k_at, s = _take("k", k, dtype, k.shape, device)
        v_at, sv = _take("v", v, dtype, k.shape, device)
        if s != sv:
            _refuse("k and v have different strides")
        # The stride of a dimension of one element is not used and may be anything.
        s = [n if k.shape[i] > 1 else head_dim for i, n in enumerate(s[:3])]
        table_at, ts = _take("table", table, torch.int32, (rows, width), device)
        self.device, self.dtype, self.rows, self.kv_heads, self.head_dim = device, dtype, rows, kv_heads, head_dim
        self.c = CacheStruct(
            k_at, v_at, s[0], s[1], s[2], table_at, ts[0] if rows > 1 else width,
            _take("lengths", lengths, torch.int32, (rows,), device, True)[0],
            None if errors is None else _take("errors", errors, torch.int32, (1,), device, True)[0], rows, width, pages,
            page_size, kv_heads, head_dim, _TYPES[dtype], device)
        self.at = C.addressof(self.c)
        lib()


def paged_append(cache, q_out, q, k, v, positions, rows=None, cos=None, sin=None, interleaved=False, position_bias=0,
                 stream=0):
    """Rotates new tokens' queries into q_out and writes their keys (rotated) and values into
    pages. q, q_out [tokens, heads, head_dim] (both None: keys and values only), k, v
    [tokens, kv_heads, head_dim], positions and rows [tokens] int32, cos and sin
    [positions, rotary_dim / 2] FP32 (None: no rotation)."""
    r = _qd_tensors.append(cache.at, q_out, q, k, v, positions, rows, cos, sin, interleaved, position_bias, stream,
                           cache.tensors)
    if r is not None:
        _answer(r)


def paged_attention(cache, out, q, workspace, scale=None, stream=0):
    """Attention of one new token per cache row: q and out [rows, heads, head_dim]; scale None:
    1 / sqrt(head_dim)."""
    r = _qd_tensors.attention(cache.at, out, q, workspace.handle, scale, stream, cache.tensors)
    if r is not None:
        _answer(r)


class PagePool:
    """Reference counts [pages] int32 and the tensors that hold the pages: [pages, ...] or
    [planes, pages, ...] with a page's values together."""

    def __init__(self, refs, page_size, tensors, planes=True):
        self.refs, self.page_size, self.tensors = refs, page_size, tuple(tensors)
        self.device, pages = refs.get_device(), _dims("refs", refs, 1)[0]
        self.pages = pages
        _take("refs", refs, torch.int32, (pages,), self.device, True)
        self.memories = (MemoryStruct * max(1, len(self.tensors)))()
        for m, t in zip(self.memories, self.tensors):
            p = 1 if planes else 0
            if t.dim() <= p or t.shape[p] != pages or t.get_device() != self.device:
                _refuse(f"a tensor of shape {tuple(t.shape)} on {t.device} does not hold {pages} pages of device {self.device}")
            if t.numel() == 0:
                _refuse(f"a tensor of shape {tuple(t.shape)} holds nothing")
            inner = t.select(p, 0).select(0, 0) if planes else t.select(0, 0)
            if not inner.is_contiguous():
                _refuse("a page's values do not lie together")
            size = t.element_size()
            m.base, m.bytes = t.data_ptr(), inner.numel() * size
            m.planes, m.plane_stride = (t.shape[0], t.stride(0) * size) if planes else (1, 0)
            m.page_stride = t.stride(p) * size if pages > 1 else m.bytes
        self.at = C.addressof(self.memories)
        lib()


def pages_fork(pool, table, lengths, parents, append, table_out, lengths_out, workspace, errors=None, stream=0):
    """Row r of table_out takes over row parents[r] of table (None: its own, -1: released) with
    room for `append` more tokens; shared pages are counted and copied on write."""
    r = _qd_tensors.fork(pool.refs, pool.page_size, pool.at, len(pool.tensors), table, lengths, parents, append, table_out,
                         lengths_out, workspace.handle, errors, stream, pool.tensors)
    if r is not None:
        _answer(r)


def beam_select(logits, scores, scores_out, parents, tokens, workspace, done=None, done_out=None, eos=None, stream=0):
    """The best k = scores_out.shape[1] continuations of each group: logits [groups, beams, vocab],
    scores and done [groups, beams], the results [groups, k]."""
    r = _qd_tensors.select(logits, scores, scores_out, parents, tokens, workspace.handle, done, done_out, eos, stream)
    if r is not None:
        _answer(r)


def rope_table(theta, rotary_dim, positions, stretch=1.0, original=32768, fast=32.0, slow=1.0):
    """cos and sin [positions, rotary_dim / 2] for paged_append, numpy FP32 on the host."""
    f = C.POINTER(C.c_float)
    if rotary_dim < 0 or positions < 0:
        _refuse("rotary_dim and positions must not be negative")
    cos, sin = (np.empty((positions, rotary_dim // 2), np.float32) for _ in range(2))
    _check(lib().qd_rope_table(theta, rotary_dim, positions, stretch, original, fast, slow, cos.ctypes.data_as(f),
                               sin.ctypes.data_as(f)))
    return cos, sin
