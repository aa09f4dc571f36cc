"""Keys and values in pages: the block-table plan, rotary positions with the append, and attention over the pages.

Bindings of ptts_paged_plan, ptts_rotary_append and ptts_paged_attention (include/pocket_tts/pocket_tts_amd.h has the formulas);
help(ptts_paged.attention) and so on list the arguments.  Arrays live on the GPU: torch tensors, or DeviceArray for memory that a
program manages by itself.  A program that passes torch tensors calls ptts_lib.load_with_torch() before anything else loads the
library (the first call here does it too).

Every call enqueues on `stream` (a torch stream or a handle; default: torch's current stream of the tensors' device, the default
stream for DeviceArray) and returns without waiting.  Nothing is kept between calls.  Failures raise ptts_lib.PttsError.
For inference: nothing is recorded for torch's autograd, and a tensor that requires gradients is refused while torch records them.
"""
from __future__ import annotations

import ctypes as C
import os
from typing import Tuple

import numpy as np

import ptts_lib
from ptts_lib import PttsError

try:
    import _ptts_paged as _c
except ImportError as e:
    raise RuntimeError(f"{os.path.join(os.path.dirname(os.path.abspath(__file__)), '_ptts_paged.so')} cannot be loaded ({e}): "
                       f"build it with `make -C {ptts_lib.PKG}`") from e

DeviceArray = _c.DeviceArray
plan = _c.plan
rotary_append = _c.rotary_append
attention = _c.attention
attention_workspace = _c.attention_workspace


def _bind(with_torch: int) -> None:
    L = ptts_lib.load_with_torch() if with_torch else ptts_lib.load()
    names = ("ptts_paged_plan", "ptts_rotary_append", "ptts_paged_attention_workspace", "ptts_paged_attention", "pocket_tts_get_last_error")
    _c.bind(ptts_lib.runtime == "torch", *(C.cast(getattr(L, n), C.c_void_p).value for n in names))


def _allocate(device: int, size: int, stream):
    import torch
    where = torch.device("cuda", device)
    if stream is None:
        return torch.empty(size, dtype=torch.uint8, device=where)
    handle = int(getattr(stream, "cuda_stream", stream))
    with torch.cuda.stream(torch.cuda.ExternalStream(handle, device=where) if handle else torch.cuda.default_stream(where)):
        return torch.empty(size, dtype=torch.uint8, device=where)


def _records_gradients() -> bool:
    import torch
    return torch.is_grad_enabled()


_c.setup(PttsError, _bind, _allocate, _records_gradients)


def frequencies(rot_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, trained: float = 0.0, fast: float = 32.0,
                slow: float = 1.0) -> Tuple[np.ndarray, float]:
    """(float64 [rot_dim / 2] radians per position, magnitude) for rotary_append; scaling: "none", "linear" (positions divided by
    factor), "base" (stretched base) or "parts" (ptts_rotary_frequencies).  Host only: loads no
    library."""
    names = ("none", "linear", "base", "parts")
    if scaling not in names:
        raise PttsError(f"scaling: one of {', '.join(names)}")
    out = np.empty(max(rot_dim // 2, 1), np.float64)
    return out, _c._frequencies(rot_dim, base, names.index(scaling), factor, trained, fast, slow, out.ctypes.data)
