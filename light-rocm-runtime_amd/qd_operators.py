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
# A call takes a few microseconds on the device, so each tensor is looked at once, in few steps:
# _take and _flat return its address if it is as it has to be and say what is wrong if not.

_TYPES = {torch.float32: qd.DTYPE_F32, torch.bfloat16: qd.DTYPE_BF16, torch.float16: qd.DTYPE_F16}
_F32, _I32T, _U8T = torch.float32, torch.int32, torch.uint8


def _refuse(text):
    raise QdError(qd.INVALID_ARGUMENT, text)


def _dims(name, t, n):
    if t is None or t.dim() != n:
        _refuse(f"{name} needs {n} dimensions")
    return t.shape


def _wrong(name, t, dtype, shape, device):
    if t is None:
        _refuse(f"{name} is missing")
    if t.shape != shape:
        _refuse(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    if t.dtype is not dtype:
        _refuse(f"{name} has type {t.dtype}, not {dtype}")
    if t.get_device() != device:
        _refuse(f"{name} is on {t.device}, not on device {device}")
    _refuse(f"{name} is not contiguous where it has to be (strides {t.stride()})")


def _take(name, t, dtype, shape, device):
    """Address and strides of a tensor of this type, shape and device, its last dimension contiguous."""
    if t is not None and t.shape == shape and t.dtype is dtype and t.get_device() == device:
        s = t.stride()
        if s[-1] == 1 or shape[-1] <= 1:
            return t.data_ptr(), s
    _wrong(name, t, dtype, shape, device)


def _flat(name, t, dtype, shape, device):
    """Address of a contiguous tensor of this type, shape and device."""
    if t is not None and t.shape == shape and t.dtype is dtype and t.get_device() == device and t.is_contiguous():
        return t.data_ptr()
    _wrong(name, t, dtype, shape, device)


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
        table_at, ts = _take("table", table, _I32T, (rows, width), device)
        self.device, self.dtype, self.rows, self.kv_heads, self.head_dim = device, dtype, rows, kv_heads, head_dim
        self.c = CacheStruct(
            k_at, v_at, s[0], s[1], s[2], table_at, ts[0] if rows > 1 else width,
            _flat("lengths", lengths, _I32T, (rows,), device),
            None if errors is None else _flat("errors", errors, _I32T, (1,), device), rows, width, pages, page_size,
            kv_heads, head_dim, _TYPES[dtype], device)


def _tokens(name, t, dtype, shape, device):
    """Address and stride from token to token of [tokens, heads, head_dim] whose heads lie together."""
    if t is not None and t.shape == shape and t.dtype is dtype and t.get_device() == device:
        s = t.stride()
        if s[2] == 1 and (s[1] == shape[2] or shape[1] == 1):
            return t.data_ptr(), s[0] if shape[0] > 1 else shape[1] * shape[2]
    _wrong(name, t, dtype, shape, device)


def paged_append(cache, q_out, q, k, v, positions, rows=None, cos=None, sin=None, interleaved=False, position_bias=0,
                 stream=0):
    """Rotates new tokens' queries into q_out and writes their keys (rotated) and values into
    pages. q, q_out [tokens, heads, head_dim] (both None: keys and values only), k, v
    [tokens, kv_heads, head_dim], positions and rows [tokens] int32, cos and sin
    [positions, rotary_dim / 2] FP32 (None: no rotation)."""
    device, dtype, dim = cache.device, cache.dtype, cache.head_dim
    tokens = 0 if k is None else len(k)
    shape = (tokens, cache.kv_heads, dim)
    k_at, k_stride = _tokens("k", k, dtype, shape, device)
    v_at, v_stride = _tokens("v", v, dtype, shape, device)
    q_at = out_at = None
    q_stride = out_stride = heads = rotary = table_positions = 0
    cos_at = sin_at = None
    if q is not None and q_out is not None:
        heads = _dims("q", q, 3)[1]
        shape = (tokens, heads, dim)
        q_at, q_stride = _tokens("q", q, dtype, shape, device)
        out_at, out_stride = _tokens("q_out", q_out, dtype, shape, device)
    elif q is not None or q_out is not None:
        _refuse("q and q_out go together")
    if cos is not None and sin is not None:
        shape = _dims("cos", cos, 2)
        cos_at, sin_at = _flat("cos", cos, _F32, shape, device), _flat("sin", sin, _F32, shape, device)
        table_positions, rotary = shape[0], 2 * shape[1]
    elif cos is not None or sin is not None:
        _refuse("cos and sin go together")
    if not -2 ** 31 <= position_bias < 2 ** 31:
        _refuse(f"position_bias {position_bias} does not fit 32 bits")
    shape = (tokens,)
    status = lib().qd_paged_append(cache.c, AppendStruct(
        q_at, k_at, v_at, out_at, q_stride, k_stride, v_stride, out_stride,
        _flat("positions", positions, _I32T, shape, device),
        None if rows is None else _flat("rows", rows, _I32T, shape, device), position_bias, tokens, heads, rotary,
        1 if interleaved else 0, table_positions, cos_at, sin_at), stream)
    if status:
        _check(status)


def paged_attention(cache, out, q, workspace, scale=None, stream=0):
    """Attention of one new token per cache row: q and out [rows, heads, head_dim]."""
    device, dtype, dim, rows = cache.device, cache.dtype, cache.head_dim, cache.rows
    heads = _dims("q", q, 3)[1]
    shape = (rows, heads, dim)
    q_at, qs = _take("q", q, dtype, shape, device)
    out_at, os = _take("out", out, dtype, shape, device)
    # (The stride of a dimension of one element is not used and may be anything.)
    if rows == 1:
        qs, os = (heads * dim, qs[1]), (heads * dim, os[1])
    if heads == 1:
        qs, os = (qs[0], dim), (os[0], dim)
    status = lib().qd_paged_attention(
        cache.c, AttentionStruct(q_at, out_at, qs[0], qs[1], os[0], os[1], heads, dim ** -0.5 if scale is None else scale),
        workspace.handle, stream)
    if status:
        _check(status)


class PagePool:
    """Reference counts [pages] int32 and the tensors that hold the pages: [pages, ...] or
    [planes, pages, ...] with a page's values together."""

    def __init__(self, refs, page_size, tensors, planes=True):
        self.refs, self.page_size, self.tensors = refs, page_size, list(tensors)
        self.device, pages = refs.get_device(), _dims("refs", refs, 1)[0]
        self.pages = pages
        _flat("refs", refs, _I32T, (pages,), self.device)
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


def pages_fork(pool, table, lengths, parents, append, table_out, lengths_out, workspace, errors=None, stream=0):
    """Row r of table_out takes over row parents[r] of table (None: its own, -1: released) with
    room for `append` more tokens; shared pages are counted and copied on write."""
    device = pool.device
    rows, width = shape = _dims("table", table, 2)
    table_at, ts = _take("table", table, _I32T, shape, device)
    out_at, os = _take("table_out", table_out, _I32T, shape, device)
    flat = (rows,)
    status = lib().qd_pages_fork(ForkStruct(
        table_at, _flat("lengths", lengths, _I32T, flat, device),
        None if parents is None else _flat("parents", parents, _I32T, flat, device), out_at,
        _flat("lengths_out", lengths_out, _I32T, flat, device), pool.refs.data_ptr(), ts[0] if rows > 1 else width,
        os[0] if rows > 1 else width, None if errors is None else _flat("errors", errors, _I32T, (1,), device),
        pool.memories, len(pool.tensors), rows, width, pool.pages, pool.page_size, append, device), workspace.handle, stream)
    if status:
        _check(status)


def beam_select(logits, scores, scores_out, parents, tokens, workspace, done=None, done_out=None, eos=None, stream=0):
    """The best k = scores_out.shape[1] continuations of each group: logits [groups, beams, vocab],
    scores and done [groups, beams], the results [groups, k]."""
    groups, beams, vocab = shape = _dims("logits", logits, 3)
    device, dtype = logits.get_device(), logits.dtype
    if dtype not in _TYPES:
        _refuse(f"logits of type {dtype}")
    logits_at, s = _take("logits", logits, dtype, shape, device)
    k = _dims("scores_out", scores_out, 2)[1]
    given, chosen = (groups, beams), (groups, k)
    done_at = done_out_at = None
    if done is not None and done_out is not None and eos is not None:
        done_at, done_out_at = _flat("done", done, _U8T, given, device), _flat("done_out", done_out, _U8T, chosen, device)
    elif done is not None or done_out is not None:
        _refuse("done, done_out and eos go together")
    status = lib().qd_beam_select(SelectStruct(
        logits_at, s[0], s[1], _flat("scores", scores, _F32, given, device), done_at,
        _flat("scores_out", scores_out, _F32, chosen, device), _flat("parents", parents, _I32T, chosen, device),
        _flat("tokens", tokens, _I32T, chosen, device), done_out_at, _TYPES[dtype], groups, beams, vocab, k,
        0 if eos is None else eos, device), workspace.handle, stream)
    if status:
        _check(status)


def rope_table(theta, rotary_dim, positions, stretch=1.0, original=32768, fast=32.0, slow=1.0):
    """cos and sin [positions, rotary_dim / 2] for paged_append, numpy FP32 on the host."""
    f = C.POINTER(C.c_float)
    if rotary_dim < 0 or positions < 0:
        _refuse("rotary_dim and positions must not be negative")
    cos, sin = (np.empty((positions, rotary_dim // 2), np.float32) for _ in range(2))
    _check(lib().qd_rope_table(theta, rotary_dim, positions, stretch, original, fast, slow, cos.ctypes.data_as(f),
                               sin.ctypes.data_as(f)))
    return cos, sin
