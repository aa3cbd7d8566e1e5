"""Norms of queries and keys for each head and their rotation by the position, in one pass.

For the D numbers x of a head at position t:  n = x / sqrt(mean x^2 + eps),  z = n * gain,  y = R(t) z; without a gain z = x. R(t) turns the pairs
(z_i, z_(i + rotary_dim / 2)), or with ``interleaved`` the neighbours (z_2i, z_(2i + 1)), of the first ``rotary_dim`` numbers by the angle
t * base^(-2 i / rotary_dim), and leaves the others. Sums are taken in fp32, results rounded once. Angles are fractions of a turn in whole numbers of 64
bits, whose products with a position wrap at whole turns: they are off by 2^-62 for each position, so cosines and sines hold fp32's bits up to some 2^38.

``norm_rotary`` takes queries and keys as two tensors (views of a projection, fewer heads of keys than of queries), ``packed_norm_rotary``
the packed projection that ``packed_self_attention`` reads. Both have the hand-written kernels of ``csrc/norm_rotary.cu`` on CUDA, with a backward
pass of their own, and an equivalent torch expression elsewhere; derivatives beyond the first, tangents and ``vmap`` go through primitive operations.
"""
from __future__ import annotations

import decimal
import functools
import math

import numpy as np
import torch

from ..core.sharding.propagation import OpShardingRule
from ..core.tensor.api import Tensor
from ..types import DType
from .base import Operation
from .fused import _Fused

_FLOATS = (DType.bfloat16, DType.float32)
MOST_DIM = 256


def _runs_native(x: torch.Tensor) -> bool:
    from .. import native

    return x.device.type != "meta" and native.use_native(x) and x.numel() > 0


# ---------------------------------------------------------------- angles
@functools.lru_cache(256)
def turns(base: float, rotary_dim: int) -> tuple[int, ...]:
    """What each pair turns by for a position, the fraction of a turn, base^(-2 i / rotary_dim) / (2 pi) less its whole part, in whole numbers of 2^-64, rounded:
    0 <= n < 2^64. (An exponential in 64 bits is off by 2^-54 of a turn and more.)"""
    with decimal.localcontext() as c:
        c.prec = digits = 50 + max(0, -math.floor(math.log10(base)))             # in front of the point too, where base is below 1

        def atan_of_one_over(n: int) -> int:                                       # its series, in units of 10^-(digits + 10)
            term, total, k = 10 ** (digits + 10) // n, 0, 1
            while term:
                total += term // k if k % 4 == 1 else -(term // k)
                term //= n * n
                k += 2
            return total

        two_pi = decimal.Decimal(2 * (16 * atan_of_one_over(5) - 4 * atan_of_one_over(239))).scaleb(-(digits + 10))         # Machin
        log = decimal.Decimal(base).ln()
        return tuple(int((((log * (-2 * i) / rotary_dim).exp() / two_pi) % 1 * 2 ** 64).to_integral_value()) % 2 ** 64 for i in range(rotary_dim // 2))


def _signed_turns(base: float, rotary_dim: int) -> list[int]:
    return [n - 2 ** 64 if n >> 63 else n for n in turns(base, rotary_dim)]


_RADIANS = 2.0 * math.pi / 2.0 ** 64


@functools.lru_cache(64)
def _turns_on(base: float, rotary_dim: int, device: torch.device) -> torch.Tensor:
    return torch.tensor(_signed_turns(base, rotary_dim), dtype=torch.int64, device=device)


# ---------------------------------------------------------------- torch expressions
def _angles(positions, base: float, rotary_dim: int):
    """cos, sin (..., tokens, 1, rotary_dim / 2) in fp32."""
    angle = (positions.long()[..., None, None] * _turns_on(base, rotary_dim, positions.device)).double() * _RADIANS       # (the product wraps)
    return angle.cos().float(), angle.sin().float()


def _turned(y, cos, sin, rotary_dim: int, interleaved: bool):
    half = rotary_dim // 2
    a, b = (y[..., 0:rotary_dim:2], y[..., 1:rotary_dim:2]) if interleaved else (y[..., :half], y[..., half:rotary_dim])
    u, w = a * cos - b * sin, a * sin + b * cos
    return torch.cat([torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1), y[..., rotary_dim:]], -1)


def _forward(x, gain, angles, eps, rotary_dim, interleaved):
    z = x.float()
    if gain is not None:
        z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + eps) * gain.float()
    return _turned(z, *angles, rotary_dim, interleaved).to(x.dtype)


def _backward(dy, x, gain, angles, eps, rotary_dim, interleaved):
    """Gradients of the heads and of the gain (None without one)."""
    cos, sin = angles
    dz = _turned(dy.float(), cos, -sin, rotary_dim, interleaved)
    if gain is None:
        return dz.to(x.dtype), None
    z = x.float()
    r = torch.rsqrt((z * z).mean(-1, keepdim=True) + eps)
    n, dn = z * r, dz * gain.float()
    dx = r * (dn - n * (dn * n).mean(-1, keepdim=True))
    return dx.to(x.dtype), (dz * n).flatten(0, -2).sum(0).to(gain.dtype)


# ---------------------------------------------------------------- operations
class _Heads(_Fused):
    """Primals: the heads, the positions, then the gains that ``which`` names ("q", "k"). Derivatives of this operation beyond the rules that a class
    has are those of ``decomposed``."""

    n_heads = 0                  # tensors of heads in front of the positions

    def split(self, primals, which):
        gains = dict(zip(which, primals[self.n_heads + 1:]))
        return primals[:self.n_heads], primals[self.n_heads], (gains.get("q"), gains.get("k"))

    def jvp_rule(self, primals, tangents, outputs, kwargs):
        from ..transforms.jvp import jvp

        at = self.n_heads                                    # positions have no tangent
        _, t = jvp(lambda *ts: self.decomposed(*ts[:at], primals[at], *ts[at:], **kwargs),
                   tuple(primals[:at]) + tuple(primals[at + 1:]), tuple(tangents[:at]) + tuple(tangents[at + 1:]))
        return t

    def vjp_rule(self, primals, cot, outputs, kwargs):
        from ..transforms.vjp import vjp

        at = self.n_heads
        _, pull = vjp(lambda *ts: self.decomposed(*ts[:at], primals[at], *ts[at:], **kwargs), *primals[:at], *primals[at + 1:])
        grads = pull(_filled(cot, outputs))
        return (*grads[:at], None, *grads[at:])


def _filled(cot, outputs):
    """Cotangents with zeros in the place of those that are not there; one alone is not in a tuple."""
    from .creation import zeros_like

    outs = outputs if isinstance(outputs, (tuple, list)) else (outputs,)
    cot = cot if isinstance(cot, (tuple, list)) else (cot,)
    full = tuple(zeros_like(o) if c is None else c for c, o in zip(cot, outs))
    return full if isinstance(outputs, (tuple, list)) else full[0]


class NormRotaryOp(_Heads):
    """(q, k, positions, gains ...) -> (q, k), heads (batch, tokens, heads, head_dim)."""

    n_heads = 2

    def kernel(self, q, k, positions, *gains, which: str, eps: float, base: float, rotary_dim: int, interleaved: bool):
        _, _, gains = self.split((q, k, positions, *gains), which)
        if _runs_native(q):
            from ..native import heads

            return heads.norm_rotary((q, k), None, positions, gains, eps=eps, base=base, rotary_dim=rotary_dim, interleaved=interleaved, packed=False)
        if q.device.type == "meta":
            return torch.empty(q.shape, dtype=q.dtype, device="meta"), torch.empty(k.shape, dtype=k.dtype, device="meta")
        angles = _angles(positions, base, rotary_dim)
        return tuple(_forward(x, g, angles, eps, rotary_dim, interleaved) for x, g in zip((q, k), gains))

    def sharding_rule(self, input_shapes, output_shapes, **kw):
        (q, k), p = _head_rules(input_shapes[:2], input_shapes[2])
        return OpShardingRule([dict(q), dict(k), p] + [{0: ["bcast_g"]} for _ in input_shapes[3:]], [dict(q), dict(k)], summed=[set(), set()])

    def vjp_rule(self, primals, cot, outputs, kwargs):
        if cot[0] is None and cot[1] is None:
            return tuple(None for _ in primals)
        dq, dk = _filled(tuple(cot), tuple(outputs))
        got = _bwd(dq, dk, *primals, **kwargs)
        return (got[0], got[1], None, *got[2:])

    def decomposed(self, q, k, positions, *gains, which, **kw):
        _, _, gains = self.split((q, k, positions, *gains), which)
        return norm_rotary_reference(q, k, positions, *gains, **kw)


class NormRotaryBwdOp(_Heads):
    """(dq, dk, q, k, positions, gains ...) -> (dq, dk, gradients of the gains ...)."""

    n_heads = 4

    def kernel(self, dq, dk, q, k, positions, *gains, which: str, eps: float, base: float, rotary_dim: int, interleaved: bool):
        _, _, gains = self.split((dq, dk, q, k, positions, *gains), which)
        if _runs_native(q):
            from ..native import heads

            got = heads.norm_rotary((q, k), (dq.to(q.dtype), dk.to(k.dtype)), positions, gains, eps=eps, base=base, rotary_dim=rotary_dim,
                                    interleaved=interleaved, packed=False)
            return (*got[:2], *(g for g in got[2:] if g is not None))
        if q.device.type == "meta":
            return tuple(torch.empty(x.shape, dtype=x.dtype, device="meta") for x in (q, k, *(g for g in gains if g is not None)))
        angles = _angles(positions, base, rotary_dim)
        (a, ga), (b, gb) = (_backward(dy, x, g, angles, eps, rotary_dim, interleaved) for dy, x, g in zip((dq, dk), (q, k), gains))
        return (a, b, *(g for g in (ga, gb) if g is not None))

    def sharding_rule(self, input_shapes, output_shapes, *, which: str, **kw):
        (q, k), p = _head_rules(input_shapes[2:4], input_shapes[4])
        # a gain's gradient is a sum over its own heads: one head, which every device has whole beside others that are split, adds no sum over devices
        of = {"q": q, "k": k}
        return OpShardingRule([dict(q), dict(k), dict(q), dict(k), p] + [{0: ["bcast_g"]} for _ in which], [dict(q), dict(k)] + [{0: ["gn"]} for _ in which],
                              summed=[set(), set()] + [{f for fs in of[name].values() for f in fs} for name in which])

    def decomposed(self, dq, dk, q, k, positions, *gains, which, **kw):
        from ..transforms.vjp import vjp

        _, pull = vjp(lambda x, y, *g: _op.decomposed(x, y, positions, *g, which=which, **kw), q, k, *gains)
        return tuple(pull((dq, dk)))


class PackedNormRotaryOp(_Heads):
    """(qkv, positions, gains ...) -> the projection (batch, tokens, heads * 3 * head_dim) with its queries and keys normed and turned."""

    n_heads = 1

    def kernel(self, qkv, positions, *gains, head_dim: int, which: str, eps: float, base: float, rotary_dim: int, interleaved: bool):
        _, _, gains = self.split((qkv, positions, *gains), which)
        if _runs_native(qkv):
            from ..native import heads

            (y,) = heads.norm_rotary(_unpacked(qkv, head_dim), None, positions, gains, eps=eps, base=base, rotary_dim=rotary_dim, interleaved=interleaved,
                                     packed=True)
            return y.view(qkv.shape)
        if qkv.device.type == "meta":
            return torch.empty(qkv.shape, dtype=qkv.dtype, device="meta")
        angles = _angles(positions, base, rotary_dim)
        q, k, v = _unpacked(qkv, head_dim)
        y = [_forward(x, g, angles, eps, rotary_dim, interleaved) for x, g in zip((q, k), gains)]
        return torch.stack([*y, v], 3).reshape(qkv.shape)

    def sharding_rule(self, input_shapes, output_shapes, **kw):
        m, p = _rules(input_shapes[1], ("b", "s", "h"))
        return OpShardingRule([dict(m), p] + [{0: ["bcast_g"]} for _ in input_shapes[2:]], [dict(m)])

    def vjp_rule(self, primals, cot, outputs, kwargs):
        dy = cot[0] if isinstance(cot, (tuple, list)) else cot
        if dy is None:
            return tuple(None for _ in primals)
        got = _packed_bwd(dy, *primals, **kwargs)
        return (got[0], None, *got[1:]) if isinstance(got, (tuple, list)) else (got, None)

    def decomposed(self, qkv, positions, *gains, head_dim, which, **kw):
        _, _, gains = self.split((qkv, positions, *gains), which)
        return packed_norm_rotary_reference(qkv, head_dim, positions, *gains, **kw)


class PackedNormRotaryBwdOp(_Heads):
    """(dy, qkv, positions, gains ...) -> (gradient of qkv, gradients of the gains ...)."""

    n_heads = 2

    def kernel(self, dy, qkv, positions, *gains, head_dim: int, which: str, eps: float, base: float, rotary_dim: int, interleaved: bool):
        _, _, gains = self.split((dy, qkv, positions, *gains), which)
        if _runs_native(qkv):
            from ..native import heads

            got = heads.norm_rotary(_unpacked(qkv, head_dim), _unpacked(dy.to(qkv.dtype), head_dim), positions, gains, eps=eps, base=base,
                                    rotary_dim=rotary_dim, interleaved=interleaved, packed=True)
            return (got[0].view(qkv.shape), *(g for g in got[1:] if g is not None))
        if qkv.device.type == "meta":
            return tuple(torch.empty(x.shape, dtype=x.dtype, device="meta") for x in (qkv, *(g for g in gains if g is not None)))
        angles = _angles(positions, base, rotary_dim)
        (q, k, _), (dq, dk, dv) = _unpacked(qkv, head_dim), _unpacked(dy, head_dim)
        (a, ga), (b, gb) = (_backward(d, x, g, angles, eps, rotary_dim, interleaved) for d, x, g in zip((dq, dk), (q, k), gains))
        return (torch.stack([a, b, dv.to(a.dtype)], 3).reshape(qkv.shape), *(g for g in (ga, gb) if g is not None))

    def sharding_rule(self, input_shapes, output_shapes, **kw):
        m, p = _rules(input_shapes[2], ("b", "s", "h"))
        n = len(input_shapes) - 3
        return OpShardingRule([dict(m), dict(m), p] + [{0: ["bcast_g"]} for _ in range(n)], [dict(m)] + [{0: ["gn"]} for _ in range(n)])

    def decomposed(self, dy, qkv, positions, *gains, which, **kw):
        from ..transforms.vjp import vjp

        _, pull = vjp(lambda x, *g: _packed.decomposed(x, positions, *g, which=which, **kw), qkv, *gains)
        return tuple(pull(dy))


def _head_rules(shapes, positions_shape):
    """Rules of q and k, whose heads are split alike, but one head, which is not split, and of the positions."""
    m, p = _rules(positions_shape, ("b", "s", "h", "bcast_d"))
    return [m if int(s[2]) != 1 else {**m, 2: ["bcast_h"]} for s in shapes], p


def _rules(positions_shape, factors):
    m = {i: [f] for i, f in enumerate(factors)}
    return m, {0: ["s"]} if len(positions_shape) == 1 else {0: ["b"], 1: ["s"]}


def _unpacked(qkv: torch.Tensor, head_dim: int):
    b, t, w = qkv.shape
    if qkv.stride(2) != 1:
        qkv = qkv.contiguous()
    parts = qkv.view(b, t, w // (3 * head_dim), 3, head_dim)
    return tuple(parts[:, :, :, i] for i in range(3))           # (selections: a call with other views is not written down)


_op, _bwd, _packed, _packed_bwd = NormRotaryOp(), NormRotaryBwdOp(), PackedNormRotaryOp(), PackedNormRotaryBwdOp()


# ---------------------------------------------------------------- primitive operations
def _turn_reference(z: Tensor, cos: Tensor, sin: Tensor, rotary_dim: int, interleaved: bool) -> Tensor:
    from .view import concatenate, reshape, slice_tensor, squeeze, stack

    lead, d, half = tuple(int(n) for n in z.shape[:-1]), int(z.shape[-1]), rotary_dim // 2
    zero = (0,) * len(lead)

    def part(x, at, n):
        return slice_tensor(x, (*zero, at), (*lead, n))

    if interleaved:
        pairs = reshape(part(z, 0, rotary_dim), (*lead, half, 2))
        a, b = (squeeze(slice_tensor(pairs, (*zero, 0, i), (*lead, half, 1)), axis=-1) for i in range(2))
        y = reshape(stack([a * cos - b * sin, a * sin + b * cos], axis=-1), (*lead, rotary_dim))
    else:
        a, b = part(z, 0, half), part(z, half, half)
        y = concatenate([a * cos - b * sin, a * sin + b * cos], axis=-1)
    return y if rotary_dim == d else concatenate([y, part(z, rotary_dim, d - rotary_dim)], axis=-1)


def _angles_reference(positions: Tensor, base: float, rotary_dim: int):
    from .creation import constant
    from .unary import cast, cos, sin
    from .view import unsqueeze

    per = constant(np.array(_signed_turns(base, rotary_dim), dtype=np.int64), dtype=DType.int64, device=positions.device)
    radians = constant(np.array(_RADIANS), dtype=DType.float64, device=positions.device)
    angle = cast(unsqueeze(unsqueeze(cast(positions, DType.int64), axis=-1), axis=-1) * per, DType.float64) * radians
    return cast(cos(angle), DType.float32), cast(sin(angle), DType.float32)


def _heads_reference(x: Tensor, gain: Tensor | None, angles, eps: float, rotary_dim: int, interleaved: bool) -> Tensor:
    from .reduction import mean
    from .unary import cast, rsqrt

    z = cast(x, DType.float32)
    if gain is not None:
        z = z * rsqrt(mean(z * z, axis=-1, keepdims=True) + eps) * cast(gain, DType.float32)
    return cast(_turn_reference(z, *angles, rotary_dim, interleaved), x.dtype)


def norm_rotary_reference(q: Tensor, k: Tensor, positions: Tensor, q_gain: Tensor | None = None, k_gain: Tensor | None = None, *, eps: float = 1e-6,
                          base: float = 10000.0, rotary_dim: int | None = None, interleaved: bool = False) -> tuple[Tensor, Tensor]:
    """``norm_rotary`` in primitive operations."""
    rotary_dim = int(q.shape[-1]) if rotary_dim is None else int(rotary_dim)
    angles = _angles_reference(positions, base, rotary_dim)
    return tuple(_heads_reference(x, g, angles, eps, rotary_dim, interleaved) for x, g in ((q, q_gain), (k, k_gain)))


def packed_norm_rotary_reference(qkv: Tensor, head_dim: int, positions: Tensor, q_gain: Tensor | None = None, k_gain: Tensor | None = None, *,
                                 eps: float = 1e-6, base: float = 10000.0, rotary_dim: int | None = None, interleaved: bool = False) -> Tensor:
    """``packed_norm_rotary`` in primitive operations."""
    from .view import reshape, slice_tensor, squeeze, stack

    b, t, w = (int(n) for n in qkv.shape)
    h = w // (3 * head_dim)
    parts = reshape(qkv, (b, t, h, 3, head_dim))
    q, k, v = (squeeze(slice_tensor(parts, (0, 0, 0, i, 0), (b, t, h, 1, head_dim)), axis=3) for i in range(3))
    q, k = norm_rotary_reference(q, k, positions, q_gain, k_gain, eps=eps, base=base, rotary_dim=rotary_dim or head_dim, interleaved=interleaved)
    return reshape(stack([q, k, v], axis=3), (b, t, w))


# ---------------------------------------------------------------- entry points
def _need(ok: bool, text: str, error=ValueError) -> None:
    if not ok:
        raise error(text)


def _checked(x: Tensor, positions, gains, head_dim: int, eps: float, base: float, rotary_dim):
    """The gains that are there with their names, and the numbers of a call."""
    b, t = (int(n) for n in x.shape[:2])
    _need(head_dim % 16 == 0 and 16 <= head_dim <= MOST_DIM, f"head_dim {head_dim}: a multiple of 16 up to {MOST_DIM}")
    rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
    _need(rotary_dim % 16 == 0 and 16 <= rotary_dim <= head_dim, f"rotary_dim {rotary_dim}: a multiple of 16 up to head_dim")
    _need(isinstance(positions, Tensor), "positions has to be a Tensor", TypeError)
    _need(positions.dtype in (DType.int32, DType.int64), f"positions are whole numbers (int32 or int64), got {positions.dtype.name}", TypeError)
    shape = tuple(int(n) for n in positions.shape)
    _need(shape in ((t,), (b, t)), f"positions have shape ({t},) or ({b}, {t}), got {shape}")
    _need(b * t < 1 << 30, "fewer than 2^30 tokens")
    named = []
    for name, g in zip("qk", gains):
        if g is None:
            continue
        _need(isinstance(g, Tensor), f"{name}_gain has to be a Tensor", TypeError)
        _need(g.dtype is x.dtype, f"{name}_gain has to be of the heads' type, {x.dtype.name}, got {g.dtype.name}", TypeError)
        _need(tuple(int(n) for n in g.shape) == (head_dim,), f"{name}_gain has to have shape ({head_dim},), got {tuple(int(n) for n in g.shape)}")
        named.append((name, g))
    eps, base = float(eps), float(base)
    _need(eps > 0 and math.isfinite(eps), "eps has to be positive")
    _need(base > 0 and math.isfinite(base), "base has to be positive")
    devices = {t._impl.device for t in (x, positions, *(g for _, g in named))}
    _need(len(devices) == 1, f"operands on several devices: {', '.join(sorted(str(d) for d in devices))}")
    return [g for _, g in named], {"which": "".join(n for n, _ in named), "eps": eps, "base": base, "rotary_dim": rotary_dim}


def norm_rotary(q: Tensor, k: Tensor, positions: Tensor, q_gain: Tensor | None = None, k_gain: Tensor | None = None, *, eps: float = 1e-6,
                base: float = 10000.0, rotary_dim: int | None = None, interleaved: bool = False) -> tuple[Tensor, Tensor]:
    """Queries (batch, tokens, heads, head_dim) and keys (batch, tokens, kv_heads, head_dim), bf16 or fp32, views included, as attention is to see
    them: each head normed by its root mean square and multiplied by its gain (head_dim,), where one is given, then turned by its position.

    ``positions`` (tokens,) or (batch, tokens): whole numbers; an angle is off by 2^-62 for each, which fp32 begins to see at 2^38. ``rotary_dim`` (head_dim by default): how many numbers of a head are turned;
    ``interleaved``: neighbours are pairs, not halves. Gradients of queries, keys and gains."""
    from ..nn.functional.layers import use_fused

    for name, x in (("q", q), ("k", k)):
        _need(isinstance(x, Tensor), f"{name} has to be a Tensor", TypeError)
        _need(x.dtype in _FLOATS, f"{name} has to be bfloat16 or float32, got {x.dtype.name}", TypeError)
        _need(len(x.shape) == 4, f"{name} has to have shape (batch, tokens, heads, head_dim), got {tuple(int(n) for n in x.shape)}")
    sq, sk = (tuple(int(n) for n in x.shape) for x in (q, k))
    _need(sq[:2] == sk[:2] and sq[3] == sk[3] and q.dtype is k.dtype, f"q and k differ in tokens, head_dim or type: {sq} {q.dtype.name}, {sk} {k.dtype.name}")
    _need(q._impl.device == k._impl.device, "q and k are on different devices")
    gains, kw = _checked(q, positions, (q_gain, k_gain), sq[3], eps, base, rotary_dim)
    kw["interleaved"] = bool(interleaved)
    if not use_fused(q, k, positions, *gains):
        kw.pop("which")
        return norm_rotary_reference(q, k, positions, q_gain, k_gain, **kw)
    return tuple(_op(q, k, positions, *gains, **kw))


def packed_norm_rotary(qkv: Tensor, head_dim: int, positions: Tensor, q_gain: Tensor | None = None, k_gain: Tensor | None = None, *, eps: float = 1e-6,
                       base: float = 10000.0, rotary_dim: int | None = None, interleaved: bool = False) -> Tensor:
    """``norm_rotary`` on the queries and keys of a packed projection (batch, tokens, heads * 3 * head_dim) whose last axis is laid out (head, {q, k, v},
    head_dim), as ``packed_self_attention`` reads it; values come back as they are."""
    from ..nn.functional.layers import use_fused

    _need(isinstance(qkv, Tensor), "qkv has to be a Tensor", TypeError)
    _need(qkv.dtype in _FLOATS, f"qkv has to be bfloat16 or float32, got {qkv.dtype.name}", TypeError)
    shape = tuple(int(n) for n in qkv.shape)
    head_dim = int(head_dim)
    _need(len(shape) == 3 and head_dim > 0 and shape[2] % (3 * head_dim) == 0, f"qkv has to have shape (batch, tokens, heads * 3 * {head_dim}), got {shape}")
    gains, kw = _checked(qkv, positions, (q_gain, k_gain), head_dim, eps, base, rotary_dim)
    kw["interleaved"] = bool(interleaved)
    if not use_fused(qkv, positions, *gains):
        kw.pop("which")
        return packed_norm_rotary_reference(qkv, head_dim, positions, q_gain, k_gain, **kw)
    return _packed(qkv, positions, *gains, head_dim=head_dim, **kw)
