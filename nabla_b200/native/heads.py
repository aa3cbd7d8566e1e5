"""Python wrapper of the norms and rotations of heads (``csrc/norm_rotary.cu``).

Arguments are torch CUDA tensors whose shapes and types ``ops/heads.py`` has checked; scratch comes from torch's caching allocator.
``launch_count`` counts kernel launches issued from here.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import load, ptr, recorder, stream_ptr
from .serving import _rows

_lib = None
launch_count = 0
c_int, c_ll, c_f, c_vp = ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_void_p
_Strides = c_ll * 18


def _L():
    global _lib
    if _lib is None:
        lib = load("libnb_heads.so")
        lib.nb_norm_rotary.argtypes = [c_vp] * 14 + [c_int] * 10 + [c_vp, c_f, c_vp, c_int, c_vp, c_int, c_vp]
        lib.nb_norm_rotary.restype = c_int
        lib.nb_norm_rotary_scratch.argtypes = [c_int] * 6
        lib.nb_norm_rotary_scratch.restype = c_ll
        _lib = lib
    r = recorder()
    return _lib if r is None else r.library(_lib)


@functools.lru_cache(1024)
def _scratch(*sizes: int) -> int:
    """A function of the sizes alone."""
    return _L().nb_norm_rotary_scratch(*sizes)


@functools.lru_cache(256)
def _turns(base: float, rotary_dim: int):
    from ..ops.heads import turns

    return (ctypes.c_ulonglong * (rotary_dim // 2))(*turns(base, rotary_dim))


def norm_rotary(parts, dys, positions, gains, *, eps: float, base: float, rotary_dim: int, interleaved: bool, packed: bool):
    """``parts``: q, k and, where a packed projection comes back, v, each (batch, tokens, heads, dim). Without ``dys`` the results of the same
    shapes (one packed tensor (batch, tokens, heads, 3, dim) where ``packed``), with them the gradients and those of the gains
    (None where there is none)."""
    global launch_count
    parts = [_rows(t) for t in parts]
    dys = [_rows(t) for t in dys] if dys is not None else None
    gains = [g if g is None or (g.is_contiguous()) else g.contiguous() for g in gains]
    positions = positions.contiguous()
    b, t, hq, d = parts[0].shape
    x = parts[0]
    if packed:
        whole = torch.empty((b, t, hq, 3, d), dtype=x.dtype, device=x.device)
        at = whole.data_ptr()
        outs = [c_vp(at + i * d * x.element_size()) for i in range(3)]
        result = (whole,)
    else:
        result = tuple(torch.empty(p.shape, dtype=x.dtype, device=x.device) for p in parts)
        outs = [ptr(o) for o in result] + [c_vp(0)]
    v = parts[2] if len(parts) > 2 else None
    strides = _Strides(*(s for p in (*parts, *([] if v is not None else [None])) for s in (p.stride()[:3] if p is not None else (0, 0, 0))),
                       *(s for p in ((*dys, *([] if v is not None else [None])) if dys is not None else (None,) * 3)
                         for s in (p.stride()[:3] if p is not None else (0, 0, 0))))
    grads, scratch = [None, None], None
    if dys is not None and any(g is not None for g in gains):
        grads = [torch.empty((d,), dtype=x.dtype, device=x.device) if g is not None else None for g in gains]
        scratch = torch.empty(_scratch(b, t, sum(p.shape[2] for p in parts), d, rotary_dim, int(positions.dim() == 1)), dtype=torch.float32, device=x.device)
    dy = [ptr(y) for y in dys] + [c_vp(0)] * (3 - len(dys)) if dys is not None else [c_vp(0)] * 3
    rc = _L().nb_norm_rotary(ptr(parts[0]), ptr(parts[1]), ptr(v), *dy, *outs, ptr(gains[0]), ptr(gains[1]), ptr(grads[0]), ptr(grads[1]),
                             ptr(positions), int(positions.dtype == torch.int64), int(positions.dim() == 1), b, t, hq, parts[1].shape[2],
                             0 if v is None else v.shape[2], d, rotary_dim, int(interleaved), _turns(base, rotary_dim), float(eps), strides, int(packed),
                             ptr(scratch), int(x.dtype == torch.float32), stream_ptr())
    if rc != 0:
        raise RuntimeError(f"norm_rotary failed with code {rc}")
    launch_count += 1 if scratch is None else 2
    return result if dys is None else (*result, *grads)
