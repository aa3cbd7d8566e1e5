"""Performance cases of the serving operators: attention over a key / value cache held in 8 bits, writing that cache and
reading it back, and the adjustments of logits between a decoder and its choice of a token.

The cache holds blocks of ``block`` tokens, with one scale for the keys and one for the values of each block and head; a table names the
blocks of each sequence. Sizes come from the training configurations in ``nabla_b200/models`` (16 heads of 128, vocabulary 32000, sequences
of 2048) and their smaller relatives; lengths are ragged, odd ones stand beside the round ones.

``run`` computes the operators in elementary torch operations in 32 bits where ``own`` is false, and calls ``nabla_b200`` where it is
true. A written cache is compared by what it stands for: its touched blocks are read back. ``exact`` computes the same in 64 bits, one
sequence at a time, from the definition.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TINY = 2.0 ** -100            # the least scale of a block


def _dtype(case):
    return F32 if case["dtype"] == "fp32" else BF16


def _size(case):
    return 4 if case["dtype"] == "fp32" else 2


def listed():
    return [
        # one conversation, one new token: the heads of the training configuration (latency)
        {"name": "attend_one_700", "kind": "attend", "batch": 1, "new": 1, "low": 700, "high": 700, "heads": 16, "kv_heads": 16, "head_dim": 128,
         "block": 64, "dtype": "bf16"},
        # a batch of conversations of very different lengths, four query heads for each head of the cache
        {"name": "attend_batch_4001", "kind": "attend", "batch": 32, "new": 1, "low": 200, "high": 4001, "heads": 16, "kv_heads": 4, "head_dim": 128,
         "block": 64, "dtype": "bf16"},
        # two long documents, eight query heads for each head of the cache
        {"name": "attend_long_120001", "kind": "attend", "batch": 2, "new": 1, "low": 120001, "high": 120001, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "block": 128, "dtype": "bf16"},
        # a few proposed tokens of each sequence are checked at once, in fp32, narrow heads, small blocks
        {"name": "attend_check_fp32", "kind": "attend", "batch": 8, "new": 5, "low": 500, "high": 1501, "heads": 12, "kv_heads": 4, "head_dim": 64,
         "block": 16, "dtype": "fp32"},
        # the second half of two prompts of 4096 (the largest case)
        {"name": "attend_prompt_2048", "kind": "attend", "batch": 2, "new": 2048, "low": 2048, "high": 2048, "heads": 16, "kv_heads": 4,
         "head_dim": 128, "block": 64, "dtype": "bf16"},
        # keys and values of one decoding step of a batch
        {"name": "write_step_64", "kind": "write", "batch": 64, "new": 1, "low": 16, "high": 4000, "kv_heads": 4, "head_dim": 128, "block": 64,
         "dtype": "bf16"},
        # those of a batch of prompts on the heads of the training configuration
        {"name": "write_prompt_2048", "kind": "write", "batch": 4, "new": 2048, "low": 0, "high": 100, "kv_heads": 16, "head_dim": 128, "block": 64,
         "dtype": "bf16"},
        # pieces of prompts in fp32 behind ragged pasts, narrow heads, small blocks
        {"name": "write_piece_fp32", "kind": "write", "batch": 7, "new": 333, "low": 1, "high": 900, "kv_heads": 8, "head_dim": 64, "block": 16,
         "dtype": "fp32"},
        # one short prefix read back
        {"name": "read_prefix_777", "kind": "read", "batch": 1, "low": 777, "high": 777, "kv_heads": 8, "head_dim": 64, "block": 16, "dtype": "bf16"},
        # a batch of long ones
        {"name": "read_batch_4001", "kind": "read", "batch": 16, "low": 2000, "high": 4001, "kv_heads": 4, "head_dim": 128, "block": 64,
         "dtype": "bf16"},
        # the logits of one conversation under a grammar
        {"name": "logits_one_300", "kind": "logits", "batch": 1, "vocab": 32000, "history": 300, "bias": False, "grammar": True, "dtype": "fp32"},
        # those of a large batch with long histories, an odd vocabulary and a bias
        {"name": "logits_batch_256", "kind": "logits", "batch": 256, "vocab": 32001, "history": 2001, "bias": True, "grammar": True, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "write", "write", "read", "logits"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if kind == "logits":
        batch = _log_int(rng, 1, 256)
        return {"kind": kind, "batch": batch, "vocab": rng.choice([32000, 8192, _log_int(rng, 1000, 32001)]), "history": _log_int(rng, 1, 4001),
                "bias": rng.random() < 0.5, "grammar": rng.random() < 0.7, "dtype": dtype}
    hd, block = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 64, 128])
    kv = rng.choice([1, 2, 4, 8, 16])
    if kind == "read":
        high = _log_int(rng, 30, 8001)
        return {"kind": kind, "batch": rng.randint(1, max(1, min(32, 16 * 4001 * 4 * 128 // (high * kv * hd)))), "low": max(1, high // rng.choice([1, 2, 8])),
                "high": high, "kv_heads": kv, "head_dim": hd, "block": block, "dtype": dtype}
    if kind == "write":
        new = rng.choice([1, 1, _log_int(rng, 2, 2048)])
        high = rng.choice([0, _log_int(rng, 1, 4000)])
        return {"kind": kind, "batch": _log_int(rng, 1, max(1, min(128, 4 * 2048 * 16 * 128 // (new * kv * hd)))), "new": new, "low": high // 4,
                "high": high, "kv_heads": kv, "head_dim": hd, "block": block, "dtype": dtype}
    group = rng.choice([1, 2, 3, 4, 8])
    new = rng.choice([1, 1, 1, rng.randint(2, 12), _log_int(rng, 13, 2048)])
    high = _log_int(rng, 20, 120001 if new == 1 else 4001)
    rows = 8192 * 4 // (kv * group)
    most = min(2 * 120001 * 2 * 128 // (high * kv * hd), 2 * 2048 * 16 * 3072 // (new * kv * group * (high + new)))
    # the scores of the plain form stay below 2 GB
    most = min(most, (1 << 29) // (new * kv * group * (high + new)), max(1, rows))
    return {"kind": kind, "batch": _log_int(rng, 1, max(1, min(64, most))), "new": new, "low": max(1, high // rng.choice([1, 2, 16])), "high": high,
            "heads": kv * group, "kv_heads": kv, "head_dim": hd, "block": block, "dtype": dtype}


# ---------------------------------------------------------------------------------------- inputs
class _Source:
    """Tensors of one seed, drawn on the GPU."""

    def __init__(self, seed: int):
        self.g = torch.Generator("cuda").manual_seed(int(seed))

    def normal(self, shape, std=1.0, dtype=F32):
        return (torch.randn(shape, generator=self.g, device="cuda") * std).to(dtype)

    def uniform(self, shape, low, high):
        return torch.rand(shape, generator=self.g, device="cuda") * (high - low) + low

    def between(self, shape, low, high):
        """Integers of [low, high]."""
        return torch.randint(low, high + 1, shape, generator=self.g, device="cuda", dtype=torch.int32)

    def tokens(self, shape, vocab):
        """Token ids with the skew of text: the id of rank r turns up about 1 / r as often as the first."""
        u = torch.rand(shape, generator=self.g, device="cuda", dtype=F64)
        return (torch.exp(u * math.log(vocab + 1.0)) - 1.0).to(torch.int32).clamp_(0, vocab - 1)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").to(torch.int32)


def _cache(case, s, tokens):
    """A cache with room for ``tokens`` of each sequence, all of it in use, and its table. Block 0 is no sequence's."""
    n, h, d, b = case["block"], case["kv_heads"], case["head_dim"], case["batch"]
    columns = -(-tokens // n)
    blocks = 1 + b * columns
    cache = {}
    for name in ("k", "v"):
        codes = torch.empty((blocks, h, n, d), dtype=torch.int8, device="cuda")
        codes.copy_(torch.randn(codes.shape, generator=s.g, device="cuda", dtype=BF16).mul_(36.0).round_().clamp_(-127, 127))
        cache[name] = codes
        # values of about 1, more in some blocks and heads than in others
        cache[name + "_scale"] = s.uniform((blocks, h), 0.014, 0.042)
    return cache, (s.order(blocks - 1) + 1).view(b, columns).contiguous()


def _inputs(case, seed):
    s, b = _Source(seed), case["batch"]
    if case["kind"] == "logits":
        v, t = case["vocab"], case["history"]
        length = s.between((b,), (t + 1) // 2, t)
        x = {"logits": s.normal((b, v), 3.0, _dtype(case)), "history": s.tokens((b, t), v), "length": length,
             "prompt": (length.float() * s.uniform((b,), 0.0, 0.8)).to(torch.int32), "repetition": s.uniform((b,), 1.0, 1.3),
             "presence": s.uniform((b,), 0.0, 0.6), "frequency": s.uniform((b,), 0.0, 0.4)}
        if case["bias"]:      # a few tokens are wanted, a few are not: one bias for the whole batch
            x["bias"] = torch.where(s.uniform((v,), 0.0, 1.0) < 0.01, s.normal((v,), 5.0), torch.zeros((), device="cuda"))
        if case["grammar"]:
            words = -(-v // 32)
            # a grammar lets whole stretches of the vocabulary through and little of the others
            x["allowed"] = torch.where(s.uniform((b, words), 0.0, 1.0) < 0.3, s.between((b, words), -(1 << 31), (1 << 31) - 1),
                                       torch.full((), 1, dtype=torch.int32, device="cuda"))
        return x
    past = s.between((b,), case["low"], case["high"])
    if case["kind"] == "read":
        cache, table = _cache(case, s, case["high"])
        return {"cache": cache, "table": table, "start": torch.zeros_like(past), "count": past, "most": case["high"]}
    new, h, d = case["new"], case["kv_heads"], case["head_dim"]
    cache, table = _cache(case, s, case["high"] + new)
    # a batch has slots that are idle or have fewer new tokens than others
    count = torch.where(s.uniform((b,), 0.0, 1.0) < (0.0 if b == 1 else 0.2), s.between((b,), 0, new), torch.full((), new, dtype=torch.int32, device="cuda"))
    x = {"cache": cache, "table": table, "past": past, "count": count}
    if case["kind"] == "attend":
        x["past"] = past - 1 if new == 1 else past
        return x | {"q": s.normal((b, new, case["heads"], d), 1.0, _dtype(case))}
    n = case["block"]
    # new keys and values are views of a packed projection; now and then one is far larger than those around it
    kv = s.normal((b, new, h, 2, d)) * torch.where(s.uniform((b, new, h, 2, 1), 0.0, 1.0) < 0.01, 6.0, 1.0)
    kv = kv.to(_dtype(case))
    first = past // n * n
    return x | {"k": kv[:, :, :, 0], "v": kv[:, :, :, 1], "start": first, "back": torch.where(count > 0, past - first + count, 0).to(torch.int32),
                "most": new + n - 1}


# ------------------------------------------------------------------------------------- plain forms
def _rows_of(cache, name, table):
    """(batch, columns * block, heads, head_dim) values in 32 bits of the blocks of a table."""
    at = table.long()
    x = cache[name][at].float() * cache[name + "_scale"][at][..., None, None]      # (batch, columns, heads, block, head_dim)
    b, c, h, n, d = x.shape
    return x.transpose(2, 3).reshape(b, c * n, h, d)


def _attend(x):
    q, table, past, count = x["q"].float(), x["table"], x["past"].long(), x["count"].long()
    b, t, hq, d = q.shape
    k, v = _rows_of(x["cache"], "k", table), _rows_of(x["cache"], "v", table)
    h = k.shape[2]
    q = q.view(b, t, h, hq // h, d).permute(0, 2, 3, 1, 4).reshape(b, h, -1, d)                 # rows: (head of the group, token)
    s = (q @ k.permute(0, 2, 3, 1)).mul_(d ** -0.5).view(b, h, hq // h, t, -1)
    i = torch.arange(t, device=q.device)
    seen = (torch.arange(s.shape[-1], device=q.device) <= (past[:, None] + i)[..., None]) & (i < count[:, None])[..., None]
    s = s.masked_fill_(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(b, h, -1, p.shape[-1]) @ v.transpose(1, 2)
    o = o.view(b, h, hq // h, t, d) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(b, t, hq, d).to(x["q"].dtype)


def _written(cache, name, new, table, past, count):
    """Writes the new rows into their blocks: a block's scale grows to what they need, and the rows in front of them follow it."""
    codes, scales = cache[name], cache[name + "_scale"]
    n, (b, t, h, d) = codes.shape[2], new.shape
    column = past[:, None] // n + torch.arange((t + n - 2) // n + 1, device=new.device)              # the touched columns of the table
    place = column[..., None] * n + torch.arange(n, device=new.device)                               # positions of their rows
    row = place - past[:, None, None]
    fresh = (row >= 0) & (row < count[:, None, None])
    used = fresh.any(-1) & (column < table.shape[1])
    at = torch.where(used, table.long().gather(1, column.clamp(max=table.shape[1] - 1)), 0)        # block 0 takes what is nobody's
    x = new.float()[torch.arange(b, device=new.device)[:, None, None], row.clamp(0, t - 1)]         # (batch, columns, block, heads, head_dim)
    x = torch.where(fresh[..., None, None], x, 0.0).transpose(2, 3)
    old, before = codes[at], scales[at]
    before = torch.where((column * n < past[:, None])[..., None], before, 0.0)
    scale = torch.maximum(torch.maximum(before, x.abs().amax((-1, -2)) * (1.0 / 127.0)), torch.full_like(before, TINY))
    inverse = (1.0 / scale)[..., None, None]
    kept = (old.float() * (before[..., None, None] * inverse)).round()
    now = torch.where(fresh[:, :, None, :, None], (x * inverse).round(), kept).clamp(-127, 127).to(torch.int8)
    codes[at] = now
    scales[at] = scale


def _read(cache, name, table, start, count, most, dtype):
    n = cache[name].shape[2]
    i = torch.arange(most, device=table.device)
    place = start.long()[:, None] + i
    column = (place // n).clamp(max=table.shape[1] - 1)
    at = table.long().gather(1, column)
    x = cache[name][at, :, place % n].float() * cache[name + "_scale"][at][..., None]
    return torch.where((i < count[:, None])[..., None, None], x, 0.0).to(dtype)


def _adjusted(x):
    z = x["logits"].float()
    b, v = z.shape
    i = torch.arange(x["history"].shape[1], device=z.device)
    ids, length, prompt = x["history"].long(), x["length"][:, None], x["prompt"][:, None]
    seen = torch.zeros_like(z).scatter_add_(1, ids, (i < length).float())
    made = torch.zeros_like(z).scatter_add_(1, ids, ((i >= prompt) & (i < length)).float())
    z = torch.where(seen > 0, torch.where(z > 0, z / x["repetition"][:, None], z * x["repetition"][:, None]), z)
    z = z - x["frequency"][:, None] * made - x["presence"][:, None] * (made > 0)
    if "bias" in x:
        z = z + x["bias"]
    if "allowed" in x:
        bits = x["allowed"][..., None] >> torch.arange(32, device=z.device, dtype=torch.int32) & 1
        z = z.masked_fill(bits.view(b, -1)[:, :v] == 0, float("-inf"))
    return z.to(x["logits"].dtype)


# --------------------------------------------------------------------------------- the framework's
@functools.lru_cache(None)
def _call(kind, most, names):
    """The compiled function that a program of this kind keeps."""
    import nabla_b200 as nb
    from nabla_b200.nn import functional as F

    if kind == "attend":
        return nb.compile(lambda q, cache, table, past, count: F.cached_attention(q, cache, table, past, count))
    if kind == "read":
        return nb.compile(lambda cache, table, start, count: F.kv_cache_read(cache, table, start, count, most, dtype=names))
    if kind == "write":
        def step(cache, k, v, table, past, count, start, back):
            cache = F.kv_cache_write(cache, k, v, table, past, count)
            return cache, F.kv_cache_read(cache, table, start, back, most, dtype=names)

        return nb.compile(step)
    return nb.compile(lambda logits, history, length, prompt, *more: F.adjust_logits(
        logits, history, length, prompt, **dict(zip(("repetition", "presence", "frequency", *names), more))))


ORDER = {"attend": ("q", "cache", "table", "past", "count"), "read": ("cache", "table", "start", "count"),
         "write": ("cache", "k", "v", "table", "past", "count", "start", "back"),
         "logits": ("logits", "history", "length", "prompt", "repetition", "presence", "frequency", "bias", "allowed")}


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": dict(case), "x": x}
    if own:       # the same tensors as the framework's, and the compiled function
        from nabla_b200 import DType, Tensor

        wrap = lambda v: {k: Tensor.from_torch(t) for k, t in v.items()} if isinstance(v, dict) else Tensor.from_torch(v)  # noqa: E731
        state["args"] = [wrap(x[k]) for k in ORDER[case["kind"]] if k in x]
        names = tuple(k for k in ("bias", "allowed") if k in x) if case["kind"] == "logits" else DType.from_torch(_dtype(case))
        state["call"] = _call(case["kind"], x.get("most", 0), names)
    return state


def run(state):
    x, kind = state["x"], state["case"]["kind"]
    if own:
        got = state["call"](*state["args"])
        if kind == "write":
            state["args"][0], got = got          # the program goes on with the cache that it gets back
        return [t.to_torch() for t in got] if isinstance(got, (list, tuple)) else got.to_torch()
    if kind == "attend":
        return _attend(x)
    if kind == "logits":
        return _adjusted(x)
    if kind == "write":
        past, count = x["past"].long(), x["count"].long()
        _written(x["cache"], "k", x["k"], x["table"], past, count)
        _written(x["cache"], "v", x["v"], x["table"], past, count)
    count = x["back"] if kind == "write" else x["count"]
    dtype = _dtype(state["case"])
    return [_read(x["cache"], name, x["table"], x["start"], count, x["most"], dtype) for name in ("k", "v")]


def work(case):
    b = case["batch"]
    if case["kind"] == "logits":
        v = b * case["vocab"]
        return {"bytes": 2 * _size(case) * v + (v // 8 if case["grammar"] else 0) + 4 * b * case["history"] * 3 // 4
                + (4 * case["vocab"] if case["bias"] else 0), "flops": 4 * v}
    past, h, d = (case["low"] + case["high"]) / 2, case["kv_heads"], case["head_dim"]
    scales = 2 * 4 / (case["block"] * d)         # bytes of the scales for each code
    if case["kind"] == "read":
        n = 2 * b * past * h * d
        return {"bytes": n * (1 + scales) + 2 * b * case["high"] * h * d * _size(case), "flops": n}
    live = 1.0 if b == 1 else 0.9                # of the new tokens, on average
    new = case["new"] * live
    if case["kind"] == "write":
        n, back = 2 * b * new * h * d, 2 * b * (new + case["block"] / 2) * h * d
        return {"bytes": n * _size(case) + n + back + 2 * b * (case["new"] + case["block"] - 1) * h * d * _size(case), "flops": 4 * n}
    keys = past if case["new"] == 1 else past + case["new"]
    seen = past + (0 if case["new"] == 1 else case["new"] / 2)
    return {"bytes": 2 * b * keys * h * d * (1 + scales) + b * (new + case["new"]) * case["heads"] * d * _size(case),
            "flops": 4 * b * new * case["heads"] * d * seen}


# ------------------------------------------------------------------------------------------- 64 bits
def _exact_attend(x):
    q, table, cache = x["q"].to(F64), x["table"].tolist(), x["cache"]
    b, t, hq, d = q.shape
    h, n = cache["k"].shape[1], cache["k"].shape[2]
    out = torch.zeros_like(q)
    for i, (past, count) in enumerate(zip(x["past"].tolist(), x["count"].tolist())):
        if count == 0:
            continue
        at = table[i][: -(-(past + count) // n)]
        k, v = (cache[name][at].to(F64) * cache[name + "_scale"][at].to(F64)[..., None, None] for name in ("k", "v"))
        for j in range(h):
            keys, values = (y[:, j].reshape(-1, d)[: past + count] for y in (k, v))
            s = torch.einsum("tgd,kd->gtk", q[i, :count, j * (hq // h):(j + 1) * (hq // h)], keys) / math.sqrt(d)
            ahead = torch.arange(past + count, device=q.device)[None] > torch.arange(past, past + count, device=q.device)[:, None]
            out[i, :count, j * (hq // h):(j + 1) * (hq // h)] = torch.einsum("gtk,kd->tgd", torch.softmax(s.masked_fill(ahead, -math.inf), -1), values)
    return out


def _exact_block(codes, scale, keep, fresh):
    """(rows, heads, head_dim) values of a block of which ``keep`` rows stay when ``fresh`` ones are written behind them."""
    before = scale.to(F64)[:, None] if keep else torch.zeros((scale.shape[0], 1), dtype=F64, device=scale.device)
    need = torch.maximum(torch.maximum(before, fresh.abs().amax((0, 2))[:, None] / 127.0), torch.full_like(before, TINY))
    rows = torch.cat([codes[:, :keep].transpose(0, 1).to(F64) * before, fresh])
    return torch.clamp(torch.round(rows / need), -127, 127) * need


def _exact_write(x):
    b, t, h, d = x["k"].shape
    out = []
    for name in ("k", "v"):
        codes, scales, n = x["cache"][name], x["cache"][name + "_scale"], x["cache"][name].shape[2]
        y = torch.zeros((b, x["most"], h, d), dtype=F64, device=codes.device)
        for i, (past, count, table) in enumerate(zip(x["past"].tolist(), x["count"].tolist(), x["table"].tolist())):
            done = 0
            while done < count:
                c, keep = (past + done) // n, (past + done) % n
                m = min(n - keep, count - done)
                rows = _exact_block(codes[table[c]], scales[table[c]], keep, x[name][i, done:done + m].to(F64))
                at = c * n - past // n * n
                y[i, at:at + keep + m] = rows
                done += m
        out.append(y)
    return out


def _exact_read(x):
    out = []
    for name in ("k", "v"):
        codes, scales = x["cache"][name], x["cache"][name + "_scale"]
        b, n, h, d = x["table"].shape[0], codes.shape[2], codes.shape[1], codes.shape[3]
        y = torch.zeros((b, x["most"], h, d), dtype=F64, device=codes.device)
        for i, (count, table) in enumerate(zip(x["count"].tolist(), x["table"].tolist())):
            at = table[: -(-count // n)]
            y[i, :count] = (codes[at].to(F64) * scales[at].to(F64)[..., None, None]).transpose(1, 2).reshape(-1, h, d)[:count]
        out.append(y)
    return out


def _exact_logits(x):
    z = x["logits"].to(F64)
    v = z.shape[1]
    rows = []
    for i, (length, prompt) in enumerate(zip(x["length"].tolist(), x["prompt"].tolist())):
        ids = x["history"][i].long()
        seen, made = torch.bincount(ids[:length], minlength=v) > 0, torch.bincount(ids[prompt:length], minlength=v)
        r, row = x["repetition"][i].to(F64), z[i]
        row = torch.where(seen & (row > 0), row / r, torch.where(seen, row * r, row))
        row = row - x["frequency"][i].to(F64) * made - x["presence"][i].to(F64) * (made > 0)
        if "bias" in x:
            row = row + x["bias"].to(F64)
        if "allowed" in x:
            at = torch.arange(v, device=z.device)
            row[(x["allowed"][i][at // 32] >> (at % 32).to(torch.int32)) & 1 == 0] = -math.inf
        rows.append(row)
    return torch.stack(rows)


def exact(case, seed):
    x = _inputs(case, seed)
    return {"attend": _exact_attend, "write": _exact_write, "read": _exact_read, "logits": _exact_logits}[case["kind"]](x)
