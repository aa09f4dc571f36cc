"""Keys and values in pages: the block-table plan, rotary positions with the append, and attention over the pages.

Bindings of ptts_paged_plan, ptts_rotary_append and ptts_paged_attention (include/pocket_tts/pocket_tts_amd.h has the formulas).
Arrays live on the GPU: torch tensors, or DeviceArray for memory that a program manages by itself.  A program that passes torch
tensors calls ptts_lib.load_with_torch() before anything else loads the library (the first call here does it too).

Every call enqueues on `stream` (default: torch's current stream of the tensors' device, the default stream for DeviceArray) and
returns without waiting.  Nothing is kept between calls.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Sequence, Tuple

import numpy as np

import ptts_lib
from ptts_lib import PttsError, last_error

_SIZES = {"float32": 4, "bfloat16": 2, "float16": 2, "int32": 4, "float64": 8}
_KINDS = {"float32": 0, "bfloat16": 1, "float16": 2}


class DeviceArray:
    """A view of GPU memory that the caller owns.  strides count elements (default: contiguous)."""

    __slots__ = ("ptr", "shape", "dtype", "strides", "device")

    def __init__(self, ptr: int, shape: Sequence[int], dtype: str, strides: Optional[Sequence[int]] = None, device: int = 0):
        if dtype not in _SIZES:
            raise PttsError(f"DeviceArray: unknown type {dtype}")
        self.ptr, self.shape, self.dtype, self.device = int(ptr), tuple(int(n) for n in shape), dtype, device
        if strides is None:
            strides, n = [], 1
            for k in reversed(self.shape):
                strides.insert(0, n)
                n *= k
        self.strides = tuple(int(n) for n in strides)


_torch_names = {}


def _torch_kinds(torch):
    if not _torch_names:
        _torch_names.update({getattr(torch, n): n for n in _SIZES})
    return _torch_names


class _View:
    """What a call needs to know of an array."""

    __slots__ = ("ptr", "shape", "strides", "dtype", "device", "torch")


def _view(x, name, rank, kinds):
    v = _View()
    if isinstance(x, DeviceArray):
        v.ptr, v.shape, v.strides, v.dtype, v.device, v.torch = x.ptr, x.shape, x.strides, x.dtype, x.device, False
    else:
        cls = type(x)
        if not cls.__module__.startswith("torch"):
            raise PttsError(f"{name}: a torch tensor on the GPU or a DeviceArray is required, got {cls.__name__}")
        import torch
        if not x.is_cuda:
            raise PttsError(f"{name}: the tensor is not on the GPU")
        v.ptr, v.shape, v.strides, v.device, v.torch = x.data_ptr(), x.shape, x.stride(), x.get_device(), True
        v.dtype = _torch_kinds(torch).get(x.dtype, str(x.dtype))
    if len(v.shape) != rank:
        raise PttsError(f"{name}: {rank} axes are required, got {len(v.shape)}")
    if v.dtype not in kinds:
        raise PttsError(f"{name}: {' or '.join(kinds)} is required, got {v.dtype}")
    if rank and v.shape[-1] > 1 and v.strides[-1] != 1:
        raise PttsError(f"{name}: the last axis must be contiguous")
    strides = []
    for n, s in zip(v.shape, v.strides):
        if n > 1 and s <= 0:
            raise PttsError(f"{name}: strides must be positive (axes of one element repeated are not taken)")
        strides.append(s if n > 1 else 0)      # the stride of an axis of one element says nothing
    v.strides = strides
    return v


_INTS, _FLOATS, _DOUBLE, _FLOAT = ("int32",), ("float32", "bfloat16", "float16"), ("float64",), ("float32",)


def _shape(v, name, want):
    for got, n in zip(v.shape, want):
        if n is not None and got != n:
            raise PttsError(f"{name}: shape {tuple(v.shape)}, expected {tuple('any' if n is None else n for n in want)}")


def _same_device(views):
    first = next(v for v in views if v is not None)
    for v in views:
        if v is not None and (v.device != first.device or v.torch != first.torch):
            raise PttsError("all arrays of a call must be on one device, and all torch tensors or all DeviceArray")
    return first


def _stream(first, stream):
    if stream is not None:
        return int(getattr(stream, "cuda_stream", stream)) or None
    if first.torch:
        import torch
        return torch.cuda.current_stream(first.device).cuda_stream or None
    return None


def _lib(first):
    if first.torch:
        return ptts_lib._lib if ptts_lib.runtime == "torch" else ptts_lib.load_with_torch()
    return ptts_lib._lib or ptts_lib.load()


def _ran(rc):
    if rc < 0:
        raise PttsError(last_error())
    return rc


def _ptr(v):
    return 0 if v is None else v.ptr


_PLAN = struct.Struct("@10Pq5i0P")


def plan(cached, arriving, free_pages, block_table, page_size: int, *, slot_map, positions, cu_rows, kv_len, counts, status=None,
         stream=None) -> None:
    """Block tables and slot maps from request lengths (ptts_paged_plan).  cached, arriving, kv_len: int32 [requests]; cu_rows
    [requests + 1]; free_pages [any]; block_table [requests][width], updated in place; slot_map, positions [rows]; counts [4];
    status [1] or None."""
    v = [_view(x, n, r, _INTS) for x, n, r in ((cached, "cached", 1), (arriving, "arriving", 1), (free_pages, "free_pages", 1),
                                               (block_table, "block_table", 2), (slot_map, "slot_map", 1), (positions, "positions", 1),
                                               (cu_rows, "cu_rows", 1), (kv_len, "kv_len", 1), (counts, "counts", 1))]
    st = None if status is None else _view(status, "status", 1, _INTS)
    n, rows, width = v[0].shape[0], v[4].shape[0], v[3].shape[1]
    for x, name, want in ((v[1], "arriving", n), (v[3], "block_table", n), (v[5], "positions", rows), (v[6], "cu_rows", n + 1),
                          (v[7], "kv_len", n), (v[8], "counts", 4)):
        _shape(x, name, (want,))
    if st is not None and st.shape[0] < 1:
        raise PttsError("status: one element is required")
    first = _same_device(v + [st])
    args = _PLAN.pack(*(x.ptr for x in v), _ptr(st), v[3].strides[0], n, width, v[2].shape[0], page_size, rows)
    _ran(_lib(first).ptts_paged_plan(args, first.device, _stream(first, stream)))


def frequencies(rot_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, trained: float = 0.0, fast: float = 32.0,
                slow: float = 1.0) -> Tuple[np.ndarray, float]:
    """(float64 [rot_dim / 2] radians per position, magnitude) for rotary_append; scaling: "none", "linear" (positions divided by
    factor), "base" (stretched base) or "parts" (ptts_rotary_frequencies).  Host only."""
    names = ("none", "linear", "base", "parts")
    if scaling not in names:
        raise PttsError(f"scaling: one of {', '.join(names)}")
    out = np.empty(max(rot_dim // 2, 1), np.float64)
    mag = C.c_float()
    _ran((ptts_lib._lib or ptts_lib.load()).ptts_rotary_frequencies(rot_dim, base, names.index(scaling), factor, trained, fast, slow, out, C.byref(mag)))
    return out, float(mag.value)


_PAGES = "2P3q5i"          # PttsPages, padded to 8 bytes by what follows
_ROTARY = struct.Struct("@8P8q" + _PAGES + "0P" + "f5i0P")
_NO_PAGES = (0, 0, 0, 0, 0, 0, 0, 0, 0)


def _pages(k_pages, v_pages, kv_heads=None, dim=None):
    k, v = _view(k_pages, "k_pages", 4, _FLOATS), _view(v_pages, "v_pages", 4, _FLOATS)
    _shape(v, "v_pages", k.shape)
    _shape(k, "k_pages", (None, None, kv_heads, dim))
    if v.dtype != k.dtype or v.strides[:3] != k.strides[:3]:
        raise PttsError("v_pages: type and strides must be those of k_pages")
    pages, size, heads, dim = k.shape
    return k, v, (k.ptr, v.ptr, k.strides[0], k.strides[1], k.strides[2], _KINDS[k.dtype], pages, size, heads, dim)


def rotary_append(q, k, v, positions, freq, *, interleaved: bool = False, magnitude: float = 1.0, q_out=None, slot_map=None, k_pages=None,
                  v_pages=None, status=None, stream=None) -> None:
    """Rotates q [rows][q_heads][dim] into q_out (q itself: in place) and files k, v [rows][kv_heads][dim] into the pages
    [pages][page_size][kv_heads][dim] at slot_map [rows] (ptts_rotary_append).  positions: int32 [rows]; freq: float64 [rot_dim / 2].
    q and q_out, or k, v, slot_map and the pages, may be None."""
    qv = kv = vv = qo = sm = pk = pv = None
    if q is not None:
        qv, qo = _view(q, "q", 3, _FLOATS), _view(q if q_out is None else q_out, "q_out", 3, _FLOATS)
        _shape(qo, "q_out", qv.shape)
        if qo.dtype != qv.dtype:
            raise PttsError("q_out: must have q's type")
    if (k is None) != (v is None) or (k is None) != (slot_map is None) or (k is None) != (k_pages is None) or (k is None) != (v_pages is None):
        raise PttsError("k, v, slot_map, k_pages and v_pages come together")
    if k is not None:
        kv, vv, sm = _view(k, "k", 3, _FLOATS), _view(v, "v", 3, _FLOATS), _view(slot_map, "slot_map", 1, _INTS)
        _shape(vv, "v", kv.shape)
        if vv.dtype != kv.dtype or (qv is not None and qv.dtype != kv.dtype):
            raise PttsError("q, k and v must have one type")
        pk, pv, pages = _pages(k_pages, v_pages, kv.shape[1], kv.shape[2])
        _shape(sm, "slot_map", (kv.shape[0],))
    lead = qv if qv is not None else kv
    if lead is None:
        raise PttsError("nothing to rotate: q and k are both missing")
    rows, _, dim = lead.shape
    if kv is not None and qv is not None:
        _shape(kv, "k", (rows, None, dim))
    if kv is None:
        pages = (0, 0, 0, 0, 0, 0, 0, 0, 0, dim)
    ps, fr = _view(positions, "positions", 1, _INTS), _view(freq, "freq", 1, _DOUBLE)
    _shape(ps, "positions", (rows,))
    st = None if status is None else _view(status, "status", 1, _INTS)
    if st is not None and st.shape[0] < 1:
        raise PttsError("status: one element is required")
    first = _same_device([qv, qo, kv, vv, sm, pk, pv, ps, fr, st])
    qs = (qv.strides[0], qv.strides[1]) if qv is not None else (0, 0)
    os_ = (qo.strides[0], qo.strides[1]) if qo is not None else (0, 0)
    ks = (kv.strides[0], kv.strides[1], vv.strides[0], vv.strides[1]) if kv is not None else (0, 0, 0, 0)
    args = _ROTARY.pack(_ptr(qv), _ptr(kv), _ptr(vv), _ptr(qo), ps.ptr, _ptr(sm), fr.ptr, _ptr(st), *qs, *ks, *os_, *pages, magnitude,
                        _KINDS[lead.dtype], rows, qv.shape[1] if qv is not None else 0, 2 * fr.shape[0], 1 if interleaved else 0)
    _ran(_lib(first).ptts_rotary_append(args, first.device, _stream(first, stream)))


_ATTEND = struct.Struct("@8P7q" + _PAGES + "0P" + "f9i0P")


def _attention_args(q, k_pages, v_pages, block_table, cu_rows, kv_len, scale, window, sinks, max_rows, max_kv, out, lse, status):
    qv, ov = _view(q, "q", 3, _FLOATS), _view(out, "out", 3, _FLOATS)
    rows, heads, dim = qv.shape
    _shape(ov, "out", qv.shape)
    if ov.dtype != qv.dtype:
        raise PttsError("out: must have q's type")
    pk, pv, pages = _pages(k_pages, v_pages, None, dim)
    bt, cu, kl = _view(block_table, "block_table", 2, _INTS), _view(cu_rows, "cu_rows", 1, _INTS), _view(kv_len, "kv_len", 1, _INTS)
    n = kl.shape[0]
    _shape(bt, "block_table", (n,))
    _shape(cu, "cu_rows", (n + 1,))
    ls = None if lse is None else _view(lse, "lse", 2, _FLOAT)
    if ls is not None:
        _shape(ls, "lse", (rows, heads))
    st = None if status is None else _view(status, "status", 1, _INTS)
    if st is not None and st.shape[0] < 1:
        raise PttsError("status: one element is required")
    first = _same_device([qv, ov, pk, pv, bt, cu, kl, ls, st])

    def pack(workspace, size):
        return _ATTEND.pack(qv.ptr, ov.ptr, _ptr(ls), cu.ptr, kl.ptr, bt.ptr, _ptr(st), workspace, qv.strides[0], qv.strides[1], ov.strides[0],
                            ov.strides[1], 0 if ls is None else ls.strides[0], bt.strides[0], size, *pages,
                            dim ** -0.5 if scale is None else scale, _KINDS[qv.dtype], rows, n, heads, bt.shape[1], window, sinks, max_rows, max_kv)

    return first, pack


def attention_workspace(q, k_pages, v_pages, block_table, cu_rows, kv_len, *, scale: Optional[float] = None, window: int = 0, sinks: int = 0,
                        max_rows: int = 0, max_kv: int = 0, out=None) -> int:
    """Bytes of workspace that attention() needs for these arguments (ptts_paged_attention_workspace)."""
    first, pack = _attention_args(q, k_pages, v_pages, block_table, cu_rows, kv_len, scale, window, sinks, max_rows, max_kv, q if out is None else out, None, None)
    return _ran(_lib(first).ptts_paged_attention_workspace(pack(0, 0), first.device))


def attention(q, k_pages, v_pages, block_table, cu_rows, kv_len, *, out, lse=None, scale: Optional[float] = None, window: int = 0, sinks: int = 0,
              max_rows: int = 0, max_kv: int = 0, workspace=None, status=None, stream=None) -> None:
    """Attention of every request's new rows over its pages (ptts_paged_attention).  q, out [rows][heads][dim]; block_table int32
    [requests][width]; cu_rows [requests + 1]; kv_len [requests]; lse float32 [rows][heads] or None; scale: default dim ** -0.5.
    workspace: any array of at least attention_workspace() bytes; None: torch's allocator provides it (torch tensors only)."""
    first, pack = _attention_args(q, k_pages, v_pages, block_table, cu_rows, kv_len, scale, window, sinks, max_rows, max_kv, out, lse, status)
    L = _lib(first)
    if workspace is None:
        need = _ran(L.ptts_paged_attention_workspace(pack(0, 0), first.device))
        if need and not first.torch:
            raise PttsError(f"attention: a workspace of {need} bytes is required")
        if need:
            import torch
            s = _stream(first, stream) or 0
            with torch.cuda.stream(torch.cuda.ExternalStream(s, device=first.device)) if stream is not None else _nothing:
                workspace = torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", first.device))
            ptr = workspace.data_ptr()
        else:
            ptr = 0
    elif isinstance(workspace, DeviceArray):
        ptr, need = workspace.ptr, int(np.prod(workspace.shape)) * _SIZES[workspace.dtype]
    else:
        if not workspace.is_cuda or workspace.get_device() != first.device or not workspace.is_contiguous():
            raise PttsError("workspace: a contiguous tensor on the arrays' device is required")
        ptr, need = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _ran(L.ptts_paged_attention(pack(ptr, need), first.device, _stream(first, stream)))


class _Nothing:
    def __enter__(self):
        return None

    def __exit__(self, *_):
        return False


_nothing = _Nothing()
