"""Operations of a decoder that answers: a key / value cache in 8 bits, attention over it, the adjustment of logits and the draw of tokens.

The cache is a dict of four tensors, ``{"k", "k_scale", "v", "v_scale"}``: codes (blocks, heads, block_size, head_dim) in int8 and one fp32
scale per block and head (blocks, heads); a code of a block stands for code * scale. Which blocks are a sequence's says a table (batch,
columns) of whole numbers: position t of sequence b lies in row ``t % block_size`` of block ``table[b, t // block_size]``. An entry that names
no block (negative, or not below the number of blocks) is a place without tokens: writes to it are dropped, reads give zeros, attention
sees no key there. Sequences may share blocks that are only read; a block that a call writes belongs to one sequence.

Each is one ``Operation`` with hand-written kernels on CUDA (``csrc/kv_cache.cu``, ``cached_attention.cu``, ``shared_prefix.cu``,
``logits.cu``, ``sample.cu``) and an equivalent torch expression on the CPU. They have no derivatives. On a mesh the heads of the cache may be split as those of the model are, where
every device then has the query heads of its own heads of the cache (attention refuses other splits).
"""
from __future__ import annotations

import math

import torch

from .. import config
from ..core.graph.tracing import note_update
from ..core.sharding.propagation import OpShardingRule
from ..core.tensor.api import Tensor
from ..types import DType
from .base import Operation

BLOCK_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
LEAST_SCALE = 2.0 ** -100            # of a block: its reciprocal and its logarithm are finite
_FLOATS = (DType.bfloat16, DType.float32)
_WHOLE = (DType.int32, DType.int64)


def _runs_native(x: torch.Tensor) -> bool:
    from .. import native

    return x.device.type != "meta" and native.use_native(x)


def _live(count: torch.Tensor | None, most: int, like: torch.Tensor) -> torch.Tensor:
    """Tokens of each sequence, from 0 to ``most``."""
    return like.new_full(like.shape, most).long() if count is None else count.long().clamp(0, most)


def _blocks_of(table: torch.Tensor, column: torch.Tensor, blocks: int):
    """(block, is there one) at columns (batch, n) of the table."""
    at = table.long().gather(1, column.clamp(0, table.shape[1] - 1))
    there = (column >= 0) & (column < table.shape[1]) & (at >= 0) & (at < blocks)
    return torch.where(there, at, 0), there


# ================================================================ writing
class KVCacheWriteOp(Operation):
    """Outputs (k codes, k scale, v codes, v scale): the arguments themselves where ``inplace``, else copies."""

    def kernel(self, k_codes, k_scale, v_codes, v_scale, k, v, table, past, count=None, *, inplace: bool = True):
        cache = (k_codes, k_scale, v_codes, v_scale)
        if not inplace:
            cache = tuple(t.clone() for t in cache)
        if k.device.type == "meta" or not k.numel():
            return cache
        if _runs_native(k):
            from ..native import serving

            serving.kv_write(*cache, k, v, table, past, count)
            return cache
        for codes, scales, new in ((cache[0], cache[1], k), (cache[2], cache[3], v)):
            self._write(codes, scales, new, table, past, count)
        return cache

    @staticmethod
    def _write(codes, scales, new, table, past, count):
        n, (b, t, h, d) = codes.shape[2], new.shape
        past = past.long().clamp(0, table.shape[1] * n)
        column = past[:, None] // n + torch.arange((t + n - 2) // n + 1, device=new.device)
        row = column[..., None] * n + torch.arange(n, device=new.device) - past[:, None, None]       # of the new tokens
        fresh = (row >= 0) & (row < _live(count, t, past)[:, None, None])
        at, there = _blocks_of(table, column, codes.shape[0])
        used = fresh.any(-1) & there
        x = new.float()[torch.arange(b, device=new.device)[:, None, None], row.clamp(0, t - 1)].transpose(2, 3)
        x = torch.where(fresh[:, :, None, :, None], x, 0.0)[used]                                     # (used, heads, block, head_dim)
        at, keep, fresh = at[used], (row < 0)[used], fresh[used]
        before = torch.where(keep.any(-1)[:, None], scales[at], 0.0)
        top = x.abs().amax((-1, -2)) * (1.0 / 127.0)
        top = torch.where(torch.isfinite(top), top.clamp(min=LEAST_SCALE), float("nan"))
        scale = torch.maximum(before, top)
        inverse = (1.0 / scale)[..., None, None]
        kept = (codes[at].float() * (before[..., None, None] * inverse)).round()
        q = torch.where(fresh[:, None, :, None], (x * inverse).round(), kept)
        q = torch.where(torch.isnan(scale)[..., None, None], torch.where(fresh[:, None, :, None], 0.0, codes[at].float()), q).clamp(-127, 127).to(torch.int8)
        codes[at] = torch.where((fresh | keep)[:, None, :, None], q, codes[at])
        scales[at] = scale

    def sharding_rule(self, input_shapes, output_shapes, **kw):
        codes, scale = {0: ["blocks"], 1: ["h"], 2: ["bcast_n"], 3: ["bcast_d"]}, {0: ["blocks"], 1: ["h"]}
        new = {0: ["bcast_b"], 1: ["bcast_t"], 2: ["h"], 3: ["bcast_d"]}
        ins = [codes, scale, codes, scale, new, new] + [{i: [f"bcast_i{i}"] for i in range(len(s))} for s in input_shapes[6:]]
        return OpShardingRule([_whole_blocks(m) for m in ins], [_whole_blocks(m) for m in (codes, scale, codes, scale)])


def _whole_blocks(m: dict) -> dict:
    """Ids of a table count the blocks of the whole cache: they are not split."""
    return {i: ["bcast_blocks"] if f == ["blocks"] else list(f) for i, f in m.items()}


# ================================================================ reading
class KVCacheReadOp(Operation):
    """Outputs (k, v), each (batch, max_tokens, heads, head_dim)."""

    def kernel(self, k_codes, k_scale, v_codes, v_scale, table, start, count, *, max_tokens: int, dtype: torch.dtype):
        b, (_, h, _, d) = table.shape[0], k_codes.shape
        if k_codes.device.type == "meta" or not b * max_tokens * h:
            return tuple(torch.empty((b, max_tokens, h, d), dtype=dtype, device=k_codes.device) for _ in range(2))
        if _runs_native(k_codes):
            from ..native import serving

            return serving.kv_read(k_codes, k_scale, v_codes, v_scale, table, start, count, max_tokens, dtype)
        return tuple(self._read(c, s, table, start, count, max_tokens, dtype) for c, s in ((k_codes, k_scale), (v_codes, v_scale)))

    @staticmethod
    def _read(codes, scales, table, start, count, most, dtype):
        n = codes.shape[2]
        i = torch.arange(most, device=table.device)
        place = start.long().clamp(0, table.shape[1] * n)[:, None] + i
        at, there = _blocks_of(table, place // n, codes.shape[0])
        x = codes[at, :, place % n].float() * scales[at][..., None]
        keep = there & (i < _live(count, most, start)[:, None])
        return torch.where(keep[..., None, None], x, 0.0).to(dtype)

    def sharding_rule(self, input_shapes, output_shapes, **kw):
        codes, scale = {0: ["bcast_blocks"], 1: ["h"], 2: ["bcast_n"], 3: ["bcast_d"]}, {0: ["bcast_blocks"], 1: ["h"]}
        out = {0: ["bcast_b"], 1: ["bcast_t"], 2: ["h"], 3: ["bcast_d"]}
        ins = [codes, scale, codes, scale] + [{i: [f"bcast_i{i}"] for i in range(len(s))} for s in input_shapes[4:]]
        return OpShardingRule([dict(m) for m in ins], [dict(out), dict(out)])


# ================================================================ attention
def _softmax_over(q, k, v, seen, scale: float):
    """softmax(scale * q k^T) v over the keys that are seen (batch, new, keys), zeros where there are none."""
    b, t, hq, d = q.shape
    h = k.shape[2]
    s = torch.einsum("bthgd,bkhd->bhgtk", q.float().reshape(b, t, h, hq // h, d), k) * scale
    s = torch.where(seen[:, None, None], s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    p = torch.where(seen[:, None, None], p, 0.0)
    total = p.sum(-1, keepdim=True)
    # what a row does not see may be anything, what it sees and is not finite (all that a block holds for a head) makes it NaN
    fine = torch.isfinite(v).all(-1)
    o = torch.einsum("bhgtk,bkhd->bthgd", p / torch.where(total == 0, 1.0, total), torch.where(fine[..., None], v, 0.0))
    reached = torch.einsum("btk,bkh->bth", seen.float(), (~fine).float()) > 0
    o = torch.where(reached[..., None, None], float("nan"), o)
    return o.reshape(b, t, hq, d).to(q.dtype)


class CachedAttentionOp(Operation):
    """softmax(scale * q k^T) v over the keys and values of a cache, (batch, new, heads, head_dim) as ``q``."""

    def kernel(self, q, k_codes, k_scale, v_codes, v_scale, table, past, count=None, *, causal: bool = True, scale: float):
        if q.device.type == "meta" or not q.numel():
            return torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if _runs_native(q):
            from ..native import serving

            return serving.cached_attention(q, k_codes, k_scale, v_codes, v_scale, table, past, count, causal, scale)
        b, t, hq, d = q.shape
        blocks, h, n, _ = k_codes.shape
        columns = torch.arange(table.shape[1], device=q.device).expand(b, -1)
        at, there = _blocks_of(table, columns, blocks)
        k, v = ((c[at].float() * s[at][..., None, None]).transpose(2, 3).reshape(b, -1, h, d) for c, s in ((k_codes, k_scale), (v_codes, v_scale)))
        there = there.repeat_interleave(n, 1)
        past = past.long().clamp(0, table.shape[1] * n)
        count = _live(count, t, past)
        i = torch.arange(t, device=q.device)
        last = past[:, None] + i if causal else (past + count - 1)[:, None].expand(b, t)
        seen = (torch.arange(k.shape[1], device=q.device) <= last[..., None]) & (i < count[:, None])[..., None] & there[:, None]
        return _softmax_over(q, k, v, seen, scale)

    def sharding_rule(self, input_shapes, output_shapes, **kw):
        codes, scale = {0: ["bcast_blocks"], 1: ["h"], 2: ["bcast_n"], 3: ["bcast_d"]}, {0: ["bcast_blocks"], 1: ["h"]}
        q = {0: ["bcast_b"], 1: ["bcast_t"], 2: ["h"], 3: ["bcast_d"]}
        ins = [q, codes, scale, codes, scale] + [{i: [f"bcast_i{i}"] for i in range(len(s))} for s in input_shapes[5:]]
        return OpShardingRule([dict(m) for m in ins], [dict(q)])

    def compute_cost(self, input_shapes, output_shapes) -> float:
        b, t, h, d = (int(n) for n in input_shapes[0])
        return 4.0 * b * t * h * d * int(input_shapes[5][1]) * int(input_shapes[1][2])


class SharedPrefixAttentionOp(Operation):
    """``CachedAttentionOp`` over sequences that all begin with the tokens of one prefix, (batch, new, heads, head_dim) as ``q``."""

    def kernel(self, q, k_codes, k_scale, v_codes, v_scale, prefix_table, prefix_length, table, past, count=None, *, causal: bool = True, scale: float):
        if q.device.type == "meta" or not q.numel():
            return torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if _runs_native(q):
            from ..native import serving

            return serving.shared_prefix_attention(q, k_codes, k_scale, v_codes, v_scale, prefix_table, prefix_length, table, past, count, causal, scale)
        b, t, hq, d = q.shape
        blocks, h, n, _ = k_codes.shape
        shared, own = prefix_table.shape[0] * n, table.shape[1] * n
        tables = torch.cat([prefix_table.long().expand(b, -1), table.long()], 1)
        at, there = _blocks_of(tables, torch.arange(tables.shape[1], device=q.device).expand(b, -1), blocks)
        k, v = ((c[at].float() * s[at][..., None, None]).transpose(2, 3).reshape(b, -1, h, d) for c, s in ((k_codes, k_scale), (v_codes, v_scale)))
        there = there.repeat_interleave(n, 1)
        past = past.long().clamp(0, own)
        count = _live(count, t, past)
        i = torch.arange(t, device=q.device)
        last = past[:, None] + i if causal else (past + count - 1)[:, None].expand(b, t)
        seen = torch.cat([(torch.arange(shared, device=q.device) < prefix_length.long()).expand(b, t, shared),
                          torch.arange(own, device=q.device) <= last[..., None]], -1)
        return _softmax_over(q, k, v, seen & (i < count[:, None])[..., None] & there[:, None], scale)

    def sharding_rule(self, input_shapes, output_shapes, **kw):
        return _attend.sharding_rule(input_shapes, output_shapes)

    def compute_cost(self, input_shapes, output_shapes) -> float:
        b, t, h, d = (int(n) for n in input_shapes[0])
        return 4.0 * b * t * h * d * (int(input_shapes[5][0]) + int(input_shapes[7][1])) * int(input_shapes[1][2])


# ================================================================ logits
class AdjustLogitsOp(Operation):
    """``which`` names the operands behind the logits, in their order."""

    def kernel(self, logits, *more, which: tuple[str, ...]):
        if logits.device.type == "meta" or not logits.numel():
            return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        given = dict(zip(which, more))
        names = ("history", "length", "prompt_length", "repetition", "presence", "frequency", "bias", "allowed")
        history, length, prompt, repetition, presence, frequency, bias, allowed = (given.get(n) for n in names)
        if _runs_native(logits):
            from ..native import serving

            return serving.adjust_logits(logits, history, length, prompt, repetition, presence, frequency, bias, allowed)
        z = logits.float()
        b, v = z.shape
        if history is not None and history.shape[1]:
            n = history.shape[1]
            i = torch.arange(n, device=z.device)
            length = _live(length, n, history[:, 0])[:, None]
            prompt = torch.minimum(prompt.long().clamp(min=0)[:, None], length) if prompt is not None else torch.zeros_like(length)
            ids = history.long()
            known = (ids >= 0) & (ids < v) & (i < length)
            ids = ids.clamp(0, v - 1)
            seen = torch.zeros_like(z).scatter_add_(1, ids, known.float()) > 0
            made = torch.zeros_like(z).scatter_add_(1, ids, (known & (i >= prompt)).float())
            if repetition is not None:
                r = repetition[:, None]
                z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
            if frequency is not None:
                z = torch.where(made > 0, z - frequency[:, None] * made, z)
            if presence is not None:
                z = torch.where(made > 0, z - presence[:, None], z)
        if bias is not None:
            z = z + bias
        if allowed is not None:
            bits = allowed[..., None] >> torch.arange(32, device=z.device, dtype=torch.int32) & 1
            z = z.masked_fill(bits.reshape(b, -1)[:, :v] == 0, float("-inf"))
        return z.to(logits.dtype)

    def sharding_rule(self, input_shapes, output_shapes, *, which, **kw):
        rows = {0: ["b"], 1: ["bcast_v"]}
        ins = [rows]
        for name, s in zip(which, input_shapes[1:]):
            ins.append({0: ["bcast_v"]} if len(s) == 1 and name == "bias" else {0: ["b"]} if len(s) == 1 else {0: ["b"], 1: [f"bcast_{name}"]})
        return OpShardingRule([dict(m) for m in ins], [dict(rows)])


# ================================================================ draw
LEAST_WEIGHT = 2.0 ** -44            # beside the likeliest token: what is less likely is not drawn
MOST_VOCAB = 1 << 20


class SampleTokensOp(Operation):
    """``which`` names the operands behind the logits and the random numbers, in their order."""

    def kernel(self, logits, uniform, *more, which: tuple[str, ...]):
        if logits.device.type == "meta" or not logits.shape[0]:
            return torch.empty(logits.shape[:1], dtype=torch.int64, device=logits.device)
        given = dict(zip(which, more))
        temperature, top_k, top_p, min_p = (given.get(n) for n in ("temperature", "top_k", "top_p", "min_p"))
        if _runs_native(logits):
            from ..native import serving

            return serving.sample_tokens(logits, uniform, temperature, top_k, top_p, min_p)
        z = torch.where(logits > float("-inf"), logits, float("-inf")).double()          # NaN too is nowhere
        b, v = z.shape
        hot = temperature > 0 if temperature is not None else torch.ones(b, dtype=torch.bool, device=z.device)
        t = torch.where(hot, temperature, 1.0).double() if temperature is not None else torch.ones(b, dtype=torch.float64, device=z.device)
        zs, order = torch.sort(z, dim=-1, descending=True, stable=True)
        top = zs[:, :1]
        w = torch.exp((zs - torch.where(torch.isinf(top), 0.0, top)) / t[:, None])
        w = torch.where(zs == top, 1.0, torch.where(torch.isinf(top) | torch.isinf(zs) | (w < LEAST_WEIGHT), 0.0, w))
        w = torch.where(zs > float("-inf"), w, 0.0)
        rank = torch.arange(v, device=z.device)
        keep = (rank == 0) | hot[:, None]
        if top_k is not None:
            keep &= (rank < top_k[:, None]) | (top_k[:, None] <= 0)
        w = torch.where(keep, w, 0.0)
        if top_p is not None:
            p = top_p.double()[:, None]
            w = torch.where((w.cumsum(-1) - w < p * w.sum(-1, keepdim=True)) | ~(p < 1) | (rank == 0), w, 0.0)
        if min_p is not None:
            m = min_p.double()[:, None]
            w = torch.where((w >= m.clamp(max=1.0)) | ~(m > 0), w, 0.0)
        weights = torch.zeros_like(w).scatter_(1, order, w)
        total = weights.cumsum(-1)
        u = uniform.double()[:, None]
        token = (total <= torch.where(u > 0, u, 0.0) * total[:, -1:]).sum(-1)
        last = torch.where(weights > 0, rank, -1).amax(-1)                                # -1: a row without a token
        return torch.minimum(token, last)

    def sharding_rule(self, input_shapes, output_shapes, **kw):
        return OpShardingRule([{0: ["b"], 1: ["bcast_v"]}] + [{0: ["b"]} for _ in input_shapes[1:]], [{0: ["b"]}])


_write, _read, _attend, _prefixed = KVCacheWriteOp(), KVCacheReadOp(), CachedAttentionOp(), SharedPrefixAttentionOp()
_adjust, _sample = AdjustLogitsOp(), SampleTokensOp()


# ---------------------------------------------------------------- checks of arguments
def _shape(t: Tensor) -> tuple[int, ...]:
    return tuple(int(n) for n in t.shape)


def _need(ok: bool, text: str, error=ValueError) -> None:
    if not ok:
        raise error(text)


def _tensor(t, name: str, dtypes, shape: tuple) -> Tensor:
    """``shape``: numbers, or None where any will do."""
    _need(isinstance(t, Tensor), f"{name} has to be a Tensor, got {type(t).__name__}", TypeError)
    _need(not t._impl.batch_dims, f"{name}: the serving operations are not mapped by vmap, they have a batch of their own")
    _need(t.dtype in dtypes, f"{name} has to be one of {', '.join(d.name for d in dtypes)}, got {t.dtype.name}", TypeError)
    got = _shape(t)
    _need(len(got) == len(shape) and all(w is None or g == w for g, w in zip(got, shape)),
          f"{name} has to have shape ({', '.join('any' if w is None else str(w) for w in shape)}), got {got}")
    return t


def _cache(cache) -> tuple[tuple[Tensor, ...], tuple[int, ...]]:
    _need(isinstance(cache, dict) and set(cache) == {"k", "k_scale", "v", "v_scale"},
          "cache has to be a dict of k, k_scale, v and v_scale, as init_kv_cache makes it", TypeError)
    _tensor(cache["k"], "cache['k']", (DType.int8,), (None,) * 4)
    blocks, heads, n, d = _shape(cache["k"])
    _need(n in BLOCK_SIZES, f"blocks of {n} tokens: they hold 16, 32, 64 or 128")
    _need(d in HEAD_DIMS, f"head_dim {d}: a cache holds heads of 64 or 128")
    _need(blocks >= 1 and heads >= 1, "a cache has at least one block and one head")
    _tensor(cache["v"], "cache['v']", (DType.int8,), (blocks, heads, n, d))
    for name in ("k_scale", "v_scale"):
        _tensor(cache[name], f"cache['{name}']", (DType.float32,), (blocks, heads))
    return (cache["k"], cache["k_scale"], cache["v"], cache["v_scale"]), (blocks, heads, n, d)


def _places(table, first, count, batch, first_name: str, n: int):
    _tensor(table, "block_table", _WHOLE, (batch, None))
    _need(_shape(table)[1] >= 1, "block_table has no columns")
    _need(_shape(table)[1] * n < 1 << 30, "a sequence has fewer than 2^30 positions")
    _tensor(first, first_name, _WHOLE, (batch,))
    if count is not None:
        _tensor(count, "count", _WHOLE, (batch,))


def _same_device(*ts: Tensor) -> None:
    devices = {t._impl.device for t in ts}
    _need(len(devices) == 1, f"operands on several devices: {', '.join(sorted(str(d) for d in devices))}")


def _need_split_groups(q: Tensor, parts: tuple[Tensor, ...], hq: int, heads: int) -> None:
    """On a mesh every device has the query heads of its own heads of the cache. One head of the cache is whole on all of them."""
    from ..core.sharding.propagation import _assign_factor_axes

    specs = [t._impl.sharding for t in (q, *parts)]
    mesh = next((s.mesh for s in specs if s is not None), None)
    if mesh is None or heads == 1:
        return
    axes = _assign_factor_axes(_attend.sharding_rule([_shape(t) for t in (q, *parts)], None), specs).get("h", [])
    n = math.prod(mesh.get_axis_size(a) for a in axes)
    _need(-(-hq // n) == hq // heads * -(-heads // n), f"{hq} query heads and {heads} heads of the cache, split over {n} devices, would part queries from their keys")


def _now(out) -> tuple[Tensor, ...]:
    """What reads or writes a cache is computed at once, so that writes and reads take place in the order of the program; in a function that is
    being compiled, its recording keeps that order."""
    if not config.get_flag("TRACING"):
        from ..core.graph.engine import GRAPH

        GRAPH.evaluate(*out)
    return tuple(out)


# ---------------------------------------------------------------- entry points
def init_kv_cache(num_blocks: int, kv_heads: int, head_dim: int, block_size: int = 64, device=None) -> dict[str, Tensor]:
    """An empty cache of ``num_blocks`` blocks of ``block_size`` tokens (16, 32, 64 or 128) for heads of 64 or 128: two bytes
    per token, head and element of the head, keys and values together."""
    from .creation import zeros

    _need(block_size in BLOCK_SIZES, f"blocks of {block_size} tokens: they hold 16, 32, 64 or 128")
    _need(head_dim in HEAD_DIMS, f"head_dim {head_dim}: a cache holds heads of 64 or 128")
    _need(num_blocks >= 1 and kv_heads >= 1, "a cache has at least one block and one head")
    cache = {}
    for name in ("k", "v"):
        cache[name] = zeros((int(num_blocks), int(kv_heads), int(block_size), int(head_dim)), dtype=DType.int8, device=device)
        cache[name + "_scale"] = zeros((int(num_blocks), int(kv_heads)), dtype=DType.float32, device=device)
    return cache


def kv_cache_write(cache: dict[str, Tensor], k: Tensor, v: Tensor, block_table: Tensor, past: Tensor, count: Tensor | None = None, *,
                   inplace: bool = True) -> dict[str, Tensor]:
    """Put the keys and values of new tokens into the cache and return it.

    ``k``, ``v``: (batch, new, heads, head_dim), bf16 or fp32, views included. ``past`` (batch,): tokens that each sequence has already; the
    new ones go to positions ``past`` ... ``past + count - 1`` (``count`` (batch,): how many of the ``new`` are there, all of them by
    default). What a sequence had at ``past`` or behind is no longer there. Positions without a block are dropped.

    A block's scale is what its largest magnitude needs, that / 127. It grows when a new token needs more, then the codes of the tokens in
    front are rounded to the new scale, and starts anew when a token is written to the block's first row. Infinities and NaN make the
    scale of their block and head NaN, and with it all that the block holds for that head.

    The cache is updated where it lies: the tensors that come back are those that were passed in. Writes, reads and attention take place in the
    order in which they are called, in compiled functions too; what other operations made of the cache's tensors has to be realized before a write
    outside of them. Under ``compile(cuda_graph=True)`` donate the cache, else the graph copies it. ``inplace=False`` works on a copy."""
    parts, (blocks, heads, n, d) = _cache(cache)
    _tensor(k, "k", _FLOATS, (None, None, heads, d))
    batch, new = _shape(k)[:2]
    _tensor(v, "v", (k.dtype,), (batch, new, heads, d))
    _places(block_table, past, count, batch, "past", n)
    more = () if count is None else (count,)
    _same_device(*parts, k, v, block_table, past, *more)
    out = _now(_write(*parts, k, v, block_table, past, *more, inplace=bool(inplace)))
    if inplace and config.get_flag("TRACING"):
        note_update((t._impl for t in parts), (t._impl for t in out))
    return dict(zip(("k", "k_scale", "v", "v_scale"), out))


def kv_cache_read(cache: dict[str, Tensor], block_table: Tensor, start: Tensor, count: Tensor, max_tokens: int, dtype=None) -> tuple[Tensor, Tensor]:
    """Keys and values of positions ``start`` ... ``start + count - 1`` of each sequence as numbers: two tensors (batch, max_tokens, heads,
    head_dim) of ``dtype`` (bf16 by default, or fp32). Rows from ``count`` on, and those of positions without a block, are zero. What is read is what the cache holds at the call."""
    parts, (blocks, heads, n, d) = _cache(cache)
    dtype = DType.bfloat16 if dtype is None else dtype
    _need(dtype in _FLOATS, "dtype has to be bfloat16 or float32", TypeError)
    _need(isinstance(block_table, Tensor) and len(block_table.shape) == 2, "block_table has to be a Tensor (batch, columns)")
    _places(block_table, start, count, _shape(block_table)[0], "start", n)
    _need(int(max_tokens) >= 0, "max_tokens is negative")
    _same_device(*parts, block_table, start, count)
    return _now(_read(*parts, block_table, start, count, max_tokens=int(max_tokens), dtype=dtype.to_torch()))


def cached_attention(q: Tensor, cache: dict[str, Tensor], block_table: Tensor, past: Tensor, count: Tensor | None = None, *, causal: bool = True,
                     scale: float | None = None) -> Tensor:
    """Attention of new tokens over all that the cache holds of their sequences, their own keys and values (written before) included.

    ``q``: (batch, new, heads, head_dim), bf16 or fp32; ``heads`` is a multiple of the cache's heads, which groups of neighbouring query
    heads share. Query i of a sequence stands at position ``past + i`` and sees positions 0 ... ``past + i``, with ``causal=False`` all of the
    ``past + count``. Queries from ``count`` on, and those that see no key, come out as zeros; a block with a NaN scale makes the queries that
    reach it NaN and no others. ``scale`` is 1 / sqrt(head_dim) by default."""
    parts, (blocks, heads, n, d) = _cache(cache)
    _tensor(q, "q", _FLOATS, (None, None, None, d))
    batch, _, hq, _ = _shape(q)
    _need(hq >= heads and hq % heads == 0, f"{hq} query heads cannot share {heads} heads of the cache evenly")
    _places(block_table, past, count, batch, "past", n)
    _need_split_groups(q, parts, hq, heads)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    _need(scale > 0 and math.isfinite(scale), "scale has to be positive")
    more = () if count is None else (count,)
    _same_device(q, *parts, block_table, past, *more)
    return _now((_attend(q, *parts, block_table, past, *more, causal=bool(causal), scale=scale),))[0]


def shared_prefix_attention(q: Tensor, cache: dict[str, Tensor], prefix_table: Tensor, prefix_length: Tensor, block_table: Tensor, past: Tensor,
                            count: Tensor | None = None, *, causal: bool = True, scale: float | None = None) -> Tensor:
    """``cached_attention`` for a batch whose sequences all begin with the same tokens, which lie in the cache once and are read once for all.

    ``prefix_table`` (columns,) names the blocks of the prefix, ``prefix_length`` (1,) says how many tokens it has: every query sees all of them, with or
    without ``causal``. ``block_table`` (batch, columns), ``past`` and ``count`` describe what each sequence has behind the prefix, as ``kv_cache_write``
    and ``cached_attention`` take them: token ``past + i`` of a sequence is the ``prefix_length + past + i``-th of the text. The prefix need not end with
    a block. Queries from ``count`` on are zeros, a prefix of no tokens leaves what ``cached_attention`` gives."""
    parts, (blocks, heads, n, d) = _cache(cache)
    _tensor(q, "q", _FLOATS, (None, None, None, d))
    batch, new, hq, _ = _shape(q)
    _need(hq >= heads and hq % heads == 0, f"{hq} query heads cannot share {heads} heads of the cache evenly")
    _need(batch * new * hq < 1 << 31, "fewer than 2^31 rows of queries")
    _tensor(prefix_table, "prefix_table", _WHOLE, (None,))
    _need(_shape(prefix_table)[0] >= 1, "prefix_table has no columns")
    _need(_shape(prefix_table)[0] * n < 1 << 30, "a prefix has fewer than 2^30 positions")
    _tensor(prefix_length, "prefix_length", _WHOLE, (1,))
    _places(block_table, past, count, batch, "past", n)
    _need_split_groups(q, parts, hq, heads)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    _need(scale > 0 and math.isfinite(scale), "scale has to be positive")
    more = () if count is None else (count,)
    _same_device(q, *parts, prefix_table, prefix_length, block_table, past, *more)
    return _now((_prefixed(q, *parts, prefix_table, prefix_length, block_table, past, *more, causal=bool(causal), scale=scale),))[0]


def adjust_logits(logits: Tensor, history: Tensor | None = None, length: Tensor | None = None, prompt_length: Tensor | None = None, *,
                  repetition: Tensor | None = None, presence: Tensor | None = None, frequency: Tensor | None = None, bias: Tensor | None = None,
                  allowed: Tensor | None = None) -> Tensor:
    """Logits (batch, vocab), bf16 or fp32, as the choice of the next token is to see them, computed in fp32 and rounded to their type at the end:

    * ``repetition`` (batch,): a token that stands in its row's history gets z / repetition where z > 0, else z * repetition;
    * ``frequency``, ``presence`` (batch,): a token that stands n > 0 times behind the prompt loses frequency * n + presence;
    * ``bias`` (vocab,) or (batch, vocab) is added;
    * ``allowed`` (batch, ceil(vocab / 32)) int32: tokens whose bit v % 32 of word v // 32 is 0 get -inf (a row of zeros hides all).

    ``history`` (batch, longest): tokens of each row, the first ``length`` of them count (all by default), the first ``prompt_length`` of
    those are the prompt (none by default); ids that are no token are passed over. The per-row numbers and the bias are fp32."""
    _tensor(logits, "logits", _FLOATS, (None, None))
    batch, vocab = _shape(logits)
    given = {}
    if history is not None:
        given["history"] = _tensor(history, "history", _WHOLE, (batch, None))
    for name, t in (("length", length), ("prompt_length", prompt_length)):
        if t is not None:
            _need(history is not None, f"{name} without a history")
            given[name] = _tensor(t, name, _WHOLE, (batch,))
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if t is not None:
            _need(history is not None, f"{name} without a history")
            given[name] = _tensor(t, name, (DType.float32,), (batch,))
    if bias is not None:
        _need(isinstance(bias, Tensor), "bias has to be a Tensor", TypeError)
        given["bias"] = _tensor(bias, "bias", (DType.float32,), (vocab,) if len(bias.shape) == 1 else (batch, vocab))
    if allowed is not None:
        given["allowed"] = _tensor(allowed, "allowed", (DType.int32,), (batch, -(-vocab // 32)))
    _same_device(logits, *given.values())
    return _adjust(logits, *given.values(), which=tuple(given))


def sample_tokens(logits: Tensor, uniform: Tensor, *, temperature: Tensor | None = None, top_k: Tensor | None = None, top_p: Tensor | None = None,
                  min_p: Tensor | None = None) -> Tensor:
    """The next token (batch,) int64 of each row of ``logits`` (batch, vocab), bf16 or fp32, drawn with the random number ``uniform`` (batch,) fp32 of [0, 1).

    Tokens are ordered by their logits, equal ones by their ids; the weight of a token is exp((z - max z) / ``temperature``), those below 2^-44 are left
    out. Of these, one filter behind the other keeps

    * ``top_k`` (whole numbers; none where it is 0 or less): the first k;
    * ``top_p`` (none from 1 on): those in front of which less than p of the weight that is left lies;
    * ``min_p`` (none at 0): those with at least this weight;

    and the first always. The token is the first one, in the order of ids, with which the sum of the weights that are left exceeds ``uniform`` of it. A
    ``temperature`` of 0 takes the first in order (the lowest id of the largest logit). A row without a token (all are -inf or NaN) gives -1.
    Each of the four is (batch,), fp32 but for ``top_k``, and may be left out. Weights are computed in 64 bits: the same row gives the same token."""
    _tensor(logits, "logits", _FLOATS, (None, None))
    batch, vocab = _shape(logits)
    _need(1 <= vocab <= MOST_VOCAB, f"a vocabulary of {vocab}: 1 to {MOST_VOCAB} tokens")
    _tensor(uniform, "uniform", (DType.float32,), (batch,))
    given = {}
    for name, t in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
        if t is not None:
            given[name] = _tensor(t, name, _WHOLE if name == "top_k" else (DType.float32,), (batch,))
    _same_device(logits, uniform, *given.values())
    return _sample(logits, uniform, *given.values(), which=tuple(given))
