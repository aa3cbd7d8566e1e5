"""Python wrappers of the serving kernels (``csrc/kv_cache.cu``, ``csrc/cached_attention.cu``, ``csrc/logits.cu``).

Arguments are torch CUDA tensors whose shapes and types ``ops/serving.py`` has checked; scratch comes from torch's caching allocator.
``launch_count`` counts kernel launches issued from here.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import load, ptr, recorder, status_word, stream_ptr

_lib = None
launch_count = 0
c_int, c_ll, c_f, c_vp = ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_void_p


def _L():
    global _lib
    if _lib is None:
        lib = load("libnb_serving.so")
        sig = {
            "nb_kv_write": [c_vp] * 9 + [c_int] * 8 + [c_ll] * 6 + [c_int, c_vp],
            "nb_kv_read": [c_vp] * 9 + [c_int] * 9 + [c_vp],
            "nb_cached_attention": [c_vp] * 9 + [c_int] * 9 + [c_ll] * 3 + [c_f, c_int, c_vp, c_int, c_vp, c_vp],
            "nb_adjust_logits": [c_vp] * 9 + [c_ll, c_vp] + [c_int] * 6 + [c_vp],
        }
        for name, args in sig.items():
            fn = getattr(lib, name)
            fn.argtypes = args
            fn.restype = c_int
        lib.nb_cached_attention_scratch.argtypes = [c_int] * 8
        lib.nb_cached_attention_scratch.restype = c_ll
        _lib = lib
    r = recorder()
    return _lib if r is None else r.library(_lib)


def _ok(rc: int, what: str, launches: int = 1) -> None:
    global launch_count
    if rc != 0:
        raise RuntimeError(f"{what} failed with code {rc}")
    launch_count += launches


def _wide(*ts: torch.Tensor | None) -> int:
    """Bit i: the i-th vector of whole numbers is in 64 bits."""
    return sum(1 << i for i, t in enumerate(ts) if t is not None and t.dtype == torch.int64)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """(batch, tokens, heads, head_dim) whose rows can be read 16 bytes at a time where they are, else a copy."""
    v = 16 // t.element_size()
    ok = t.stride(3) == 1 and not t.data_ptr() & 15 and all(t.stride(i) % v == 0 for i in range(3) if t.shape[i] > 1)
    return t if ok else t.clone(memory_format=torch.contiguous_format)       # (contiguous() keeps a dense one that starts off a boundary)


def _dense(*ts: torch.Tensor) -> None:
    if any(not t.is_contiguous() or t.data_ptr() & 15 for t in ts):
        raise ValueError("the tensors of a cache have to be dense and start on 16-byte boundaries")


def kv_write(k_codes, k_scale, v_codes, v_scale, k, v, table, past, count) -> None:
    """Writes in place."""
    _dense(k_codes, k_scale, v_codes, v_scale)
    k, v = _rows(k), _rows(v)
    table, past = table.contiguous(), past.contiguous()
    count = count.contiguous() if count is not None else None
    b, t, h, d = k.shape
    _ok(_L().nb_kv_write(ptr(k_codes), ptr(k_scale), ptr(v_codes), ptr(v_scale), ptr(k), ptr(v), ptr(table), ptr(past), ptr(count),
                         _wide(table, past, count), b, t, h, d, k_codes.shape[2], k_codes.shape[0], table.shape[1], *k.stride()[:3],
                         *v.stride()[:3], int(k.dtype == torch.float32), stream_ptr()), "kv_write")


def kv_read(k_codes, k_scale, v_codes, v_scale, table, start, count, most: int, dtype: torch.dtype):
    _dense(k_codes, k_scale, v_codes, v_scale)
    table, start, count = table.contiguous(), start.contiguous(), count.contiguous()
    b, (blocks, h, n, d) = table.shape[0], k_codes.shape
    k, v = (torch.empty((b, most, h, d), dtype=dtype, device=k_codes.device) for _ in range(2))
    _ok(_L().nb_kv_read(ptr(k_codes), ptr(k_scale), ptr(v_codes), ptr(v_scale), ptr(k), ptr(v), ptr(table), ptr(start), ptr(count),
                        _wide(table, start, count), b, most, h, d, n, blocks, table.shape[1], int(dtype == torch.float32), stream_ptr()), "kv_read")
    return k, v


def cached_attention(q, k_codes, k_scale, v_codes, v_scale, table, past, count, causal: bool, scale: float):
    _dense(k_codes, k_scale, v_codes, v_scale)
    q = _rows(q)
    table, past = table.contiguous(), past.contiguous()
    count = count.contiguous() if count is not None else None
    b, t, hq, d = q.shape
    blocks, h, n, _ = k_codes.shape
    out = torch.empty((b, t, hq, d), dtype=q.dtype, device=q.device)
    fp32 = int(q.dtype == torch.float32)
    floats = _scratch(b, t, hq, h, d, n, table.shape[1], fp32)      # of parts that a second kernel joins
    part = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
    _ok(_L().nb_cached_attention(ptr(q), ptr(k_codes), ptr(k_scale), ptr(v_codes), ptr(v_scale), ptr(out), ptr(table), ptr(past), ptr(count),
                                 _wide(table, past, count), b, t, hq, h, d, n, blocks, table.shape[1], *q.stride()[:3], float(scale), int(causal),
                                 ptr(part), fp32, ptr(status_word(q.device)), stream_ptr()), "cached_attention", 2 if floats else 1)
    return out


@functools.lru_cache(1024)
def _scratch(*sizes: int) -> int:
    """A function of the sizes alone."""
    return _L().nb_cached_attention_scratch(*sizes)


def adjust_logits(logits, history, length, prompt, repetition, presence, frequency, bias, allowed):
    vocab = logits.shape[-1]
    x = logits.contiguous()
    if x.data_ptr() & 15:         # a dense view that starts off a boundary; the kernel writes vectors where it reads vectors
        x = x.clone()
    b = x.numel() // vocab
    history, length, prompt, repetition, presence, frequency, bias, allowed = (
        t.contiguous() if t is not None else None for t in (history, length, prompt, repetition, presence, frequency, bias, allowed))
    out = torch.empty_like(x)
    longest = history.shape[-1] if history is not None else 0
    if longest == 0:
        history = None
    _ok(_L().nb_adjust_logits(ptr(x), ptr(out), ptr(history), ptr(length), ptr(prompt), ptr(repetition), ptr(presence), ptr(frequency), ptr(bias),
                              0 if bias is None or bias.dim() == 1 else vocab, ptr(allowed), _wide(history, length, prompt), b, vocab, longest,
                              allowed.shape[-1] if allowed is not None else 0, int(x.dtype == torch.float32), stream_ptr()), "adjust_logits")
    return out
