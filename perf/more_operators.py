"""Performance cases of what a decoder does around its cache when it answers many prompts behind one prefix, and of the heads that it is
trained with: the draw of tokens from filtered logits, attention over a prefix that a batch shares, and the norms of queries and keys
with the rotation by their positions.

Sizes come from the training configurations in ``nabla_b200/models`` (16 heads of 128, vocabulary 32000, sequences of 2048) and their
smaller relatives; lengths are ragged, odd ones stand beside the round ones.

``run`` computes the operators in elementary torch operations in 32 bits where ``own`` is false (weights and sums of a draw and angles of
positions in 64, for a border or a far position is lost in 32), and calls ``nabla_b200`` where it is true. ``exact`` computes the same in
64 bits from the definitions, one row, sequence or pair of coordinates at a time.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
LEAST = 2.0 ** -44            # tokens that are less likely than this beside the likeliest are not drawn
BASE, EPS = 10000.0, 1e-6     # of the rotation, of the norms


def _dtype(case):
    return F32 if case["dtype"] == "fp32" else BF16


def _size(case):
    return 4 if case["dtype"] == "fp32" else 2


def listed():
    return [
        # the next token of one conversation, all filters (latency)
        {"name": "sample_one_32000", "kind": "sample", "batch": 1, "vocab": 32000, "filters": "tkpm", "dtype": "fp32"},
        # those of a large batch, an odd vocabulary, every row with filters of its own
        {"name": "sample_batch_256", "kind": "sample", "batch": 256, "vocab": 32001, "filters": "tkpm", "dtype": "bf16"},
        # a large vocabulary, nucleus only
        {"name": "sample_wide_131072", "kind": "sample", "batch": 32, "vocab": 131072, "filters": "tp", "dtype": "fp32"},
        # many short rows, temperature only
        {"name": "sample_plain_512", "kind": "sample", "batch": 512, "vocab": 8192, "filters": "t", "dtype": "bf16"},
        # four answers to one question: the heads of the training configuration (latency)
        {"name": "prefix_few_1000", "kind": "prefix", "batch": 4, "new": 1, "prefix": 1000, "low": 1, "high": 200, "heads": 16, "kv_heads": 16,
         "head_dim": 128, "block": 64, "dtype": "bf16"},
        # a batch behind a long instruction, four query heads for each head of the cache
        {"name": "prefix_batch_8001", "kind": "prefix", "batch": 64, "new": 1, "prefix": 8001, "low": 50, "high": 1000, "heads": 16, "kv_heads": 4,
         "head_dim": 128, "block": 64, "dtype": "bf16"},
        # questions about one long document, eight query heads for each head of the cache
        {"name": "prefix_long_60001", "kind": "prefix", "batch": 16, "new": 1, "prefix": 60001, "low": 100, "high": 2000, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "block": 128, "dtype": "bf16"},
        # a few proposed tokens of each sequence are checked at once, in fp32, narrow heads, small blocks
        {"name": "prefix_check_fp32", "kind": "prefix", "batch": 8, "new": 5, "prefix": 1501, "low": 10, "high": 300, "heads": 12, "kv_heads": 4,
         "head_dim": 64, "block": 16, "dtype": "fp32"},
        # the prompts themselves, written behind the instruction
        {"name": "prefix_prompts_200", "kind": "prefix", "batch": 32, "new": 200, "prefix": 2048, "low": 0, "high": 0, "heads": 16, "kv_heads": 4,
         "head_dim": 128, "block": 64, "dtype": "bf16"},
        # queries and keys of one decoding step, far positions
        {"name": "rotate_step_64", "kind": "rotate", "batch": 64, "new": 1, "far": 120001, "heads": 16, "kv_heads": 4, "head_dim": 128,
         "rotary_dim": 128, "interleaved": False, "dtype": "bf16"},
        # a training step on the packed projection of the training configuration, forward and backward (the largest case of the three)
        {"name": "rotate_train_2048", "kind": "rotate_packed", "batch": 8, "new": 2048, "far": 0, "heads": 16, "kv_heads": 16, "head_dim": 128,
         "rotary_dim": 128, "interleaved": False, "dtype": "bf16"},
        # narrow heads in fp32 on ragged sequences, half of each head rotated, neighbours as pairs, forward and backward
        {"name": "rotate_train_fp32", "kind": "rotate_train", "batch": 3, "new": 777, "far": 4000, "heads": 12, "kv_heads": 4, "head_dim": 64,
         "rotary_dim": 32, "interleaved": True, "dtype": "fp32"},
    ]


def _log_int(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["sample", "sample", "prefix", "prefix", "prefix", "rotate", "rotate_packed", "rotate_train"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if kind == "sample":
        vocab = rng.choice([32000, 8192, _log_int(rng, 1000, 131072)])
        return {"kind": kind, "batch": _log_int(rng, 1, max(1, min(512, 256 * 32001 // vocab))), "vocab": vocab,
                "filters": rng.choice(["t", "tk", "tp", "tm", "tkp", "tkpm", "tpm"]), "dtype": dtype}
    hd, kv, group = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 3, 4, 8])
    if kind == "prefix":
        block = rng.choice([16, 32, 64, 64, 128])
        new = rng.choice([1, 1, 1, rng.randint(2, 12), _log_int(rng, 13, 400)])
        prefix, high = _log_int(rng, 30, 60001 if new == 1 else 4001), _log_int(rng, 1, 2000)
        new = max(1, min(new, 32 * 200 * 16 * 2248 // (kv * group * (prefix + high + new))))
        most = min(32 * 200 * 16 * 2248 // (kv * group * new * (prefix + high + new)), 64 * 1000 * 4 * 128 // ((high + new) * kv * hd) + 1)
        return {"kind": kind, "batch": _log_int(rng, 1, max(1, min(128, most))), "new": new, "prefix": prefix, "low": high // rng.choice([1, 2, 16]),
                "high": high, "heads": kv * group, "kv_heads": kv, "head_dim": hd, "block": block, "dtype": dtype}
    if kind == "rotate_packed":
        group = 1
    seq = 1 if kind == "rotate" and rng.random() < 0.6 else _log_int(rng, 2, 4096)
    most = 8 * 2048 * 32 * 128 * 2 // (seq * kv * (group + 1) * hd * (4 if dtype == "fp32" else 2))
    return {"kind": kind, "batch": _log_int(rng, 1, max(1, min(128, most))), "new": seq, "far": rng.choice([0, _log_int(rng, 1, 120001)]),
            "heads": kv * group, "kv_heads": kv, "head_dim": hd, "rotary_dim": rng.choice([hd, hd, hd // 2]), "interleaved": rng.random() < 0.3,
            "dtype": dtype}


# ---------------------------------------------------------------------------------------- inputs
class _Source:
    """Tensors of one seed, drawn on the GPU."""

    def __init__(self, seed: int):
        self.g = torch.Generator("cuda").manual_seed(int(seed))

    def normal(self, shape, std=1.0, mean=0.0, dtype=F32):
        return (torch.randn(shape, generator=self.g, device="cuda") * std + mean).to(dtype)

    def uniform(self, shape, low, high):
        return torch.rand(shape, generator=self.g, device="cuda") * (high - low) + low

    def between(self, shape, low, high):
        """Integers of [low, high]."""
        return torch.randint(low, high + 1, shape, generator=self.g, device="cuda", dtype=torch.int32)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").to(torch.int32)


def _sample_inputs(case, s):
    b, v = case["batch"], case["vocab"]
    x = {"logits": s.normal((b, v), 3.0, dtype=_dtype(case)), "uniform": s.uniform((b,), 0.0, 1.0)}
    # one row in ten takes the likeliest token; filters of rows differ, and some rows go without one of them
    off = s.uniform((3, b), 0.0, 1.0)
    x["temperature"] = torch.where(s.uniform((b,), 0.0, 1.0) < (0.0 if b == 1 else 0.1), 0.0, s.uniform((b,), 0.5, 1.5))
    if "k" in case["filters"]:
        x["top_k"] = torch.where(off[0] < (0.0 if b == 1 else 0.2), 0, s.between((b,), 1, 200)).to(torch.int32)
    if "p" in case["filters"]:
        x["top_p"] = torch.where(off[1] < (0.0 if b == 1 else 0.2), 1.0, s.uniform((b,), 0.5, 1.0))
    if "m" in case["filters"]:
        x["min_p"] = torch.where(off[2] < (0.0 if b == 1 else 0.5), 0.0, s.uniform((b,), 0.0, 0.1))
    return x


def _prefix_inputs(case, s):
    b, new, h, d, n = case["batch"], case["new"], case["kv_heads"], case["head_dim"], case["block"]
    shared, columns = -(-case["prefix"] // n), -(-(case["high"] + new) // n)
    blocks = 1 + shared + b * columns
    cache = {}
    for name in ("k", "v"):
        codes = torch.empty((blocks, h, n, d), dtype=torch.int8, device="cuda")
        codes.copy_(torch.randn(codes.shape, generator=s.g, device="cuda", dtype=BF16).mul_(36.0).round_().clamp_(-127, 127))
        cache[name] = codes
        # values of about 1, more in some blocks and heads than in others
        cache[name + "_scale"] = s.uniform((blocks, h), 0.014, 0.042)
    at = s.order(blocks - 1) + 1
    past = s.between((b,), case["low"], case["high"])
    # a batch has slots that are idle or have fewer new tokens than others
    count = torch.where(s.uniform((b,), 0.0, 1.0) < (0.0 if b == 1 else 0.2), s.between((b,), 0, new), torch.full((), new, dtype=torch.int32, device="cuda"))
    return {"q": s.normal((b, new, case["heads"], d), dtype=_dtype(case)), "cache": cache, "prefix_table": at[:shared].contiguous(),
            "prefix_length": torch.full((1,), case["prefix"], dtype=torch.int32, device="cuda"), "table": at[shared:].view(b, columns).contiguous(),
            "past": past, "count": count}


def _rotate_inputs(case, s):
    b, t, hq, h, d, dt = case["batch"], case["new"], case["heads"], case["kv_heads"], case["head_dim"], _dtype(case)
    x = {"q_gain": s.normal((d,), 0.1, 1.0, dt), "k_gain": s.normal((d,), 0.1, 1.0, dt)}
    if case["kind"] == "rotate_packed":
        x["qkv"] = s.normal((b, t, hq * 3 * d), 1.5, dtype=dt)
        x["cot"] = [s.normal((b, t, hq * 3 * d), dtype=dt)]
        x["positions"] = torch.arange(t, device="cuda", dtype=torch.int64) + case["far"]       # the same for all sequences
        return x
    # queries and keys are views of a projection of all heads
    qkv = s.normal((b, t, hq + 2 * h, d), 1.5, dtype=dt)
    x["q"], x["k"] = qkv[:, :, :hq], qkv[:, :, hq:hq + h]
    x["positions"] = s.between((b, 1), 0, case["far"]) + torch.arange(t, device="cuda", dtype=torch.int32)
    if case["kind"] == "rotate_train":
        x["cot"] = [s.normal((b, t, hq, d), dtype=dt), s.normal((b, t, h, d), dtype=dt)]
    return x


def _inputs(case, seed):
    return {"sample": _sample_inputs, "prefix": _prefix_inputs}.get(case["kind"], _rotate_inputs)(case, _Source(seed))


# ------------------------------------------------------------------------------------- plain forms
def _sampled(x):
    z = x["logits"].double()
    b, v = z.shape
    hot = x["temperature"] > 0
    zs, order = torch.sort(z, dim=-1, descending=True, stable=True)                  # ties: the lowest id first
    w = torch.exp((zs - zs[:, :1]) / torch.where(hot, x["temperature"], 1.0).double()[:, None])
    w = torch.where(w < LEAST, 0.0, w)
    rank = torch.arange(v, device=z.device)
    keep = (rank == 0) | hot[:, None]
    if "top_k" in x:
        keep &= (rank < x["top_k"][:, None]) | (x["top_k"][:, None] <= 0)
    w = torch.where(keep, w, 0.0)
    if "top_p" in x:
        p = x["top_p"].double()[:, None]
        keep = (w.cumsum(-1) - w < p * w.sum(-1, keepdim=True)) | (p >= 1) | (rank == 0)
        w = torch.where(keep, w, 0.0)
    if "min_p" in x:
        w = torch.where(w >= x["min_p"].double()[:, None].clamp(max=1.0), w, 0.0)
    weights = torch.zeros_like(w).scatter_(1, order, w)
    total = weights.cumsum(-1)
    token = (total <= x["uniform"].double()[:, None] * total[:, -1:]).sum(-1)
    last = torch.where(weights > 0, rank, 0).amax(-1)
    return torch.minimum(token, last)


def _rows_of(cache, name, table):
    """(columns * block, heads, head_dim) values in 32 bits of the blocks of a table, behind the axes of the table in front of its columns."""
    at = table.long()
    y = (cache[name][at].float() * cache[name + "_scale"][at][..., None, None]).transpose(-3, -2)
    return y.reshape(*table.shape[:-1], -1, *y.shape[-2:])


def _prefixed(x):
    q, past, count = x["q"].float(), x["past"].long(), x["count"].long()
    b, t, hq, d = q.shape
    kp, vp = (_rows_of(x["cache"], name, x["prefix_table"]) for name in ("k", "v"))
    k, v = (_rows_of(x["cache"], name, x["table"]) for name in ("k", "v"))
    h, shared = kp.shape[1], kp.shape[0]
    q = q.view(b, t, h, hq // h, d).permute(2, 0, 3, 1, 4)                           # (heads of the cache, batch, group, token, head_dim)
    i = torch.arange(t, device=q.device)
    live = i < count[:, None]
    s = (q.reshape(h, -1, d) @ kp.permute(1, 2, 0)).view(h, b, hq // h, t, shared)
    s = torch.cat([s, q @ k.permute(2, 0, 3, 1)[:, :, None]], -1).mul_(d ** -0.5)
    seen = (torch.arange(k.shape[1], device=q.device) <= (past[:, None] + i)[..., None])
    seen = torch.cat([(torch.arange(shared, device=q.device) < x["prefix_length"].long()).expand(b, t, shared), seen], -1) & live[..., None]
    s = s.masked_fill_(~seen[None, :, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p[..., :shared].reshape(h, -1, shared) @ vp.transpose(0, 1)).view(h, b, hq // h, t, d) + p[..., shared:] @ v.permute(2, 0, 1, 3)[:, :, None]
    o = o / torch.where(total == 0, 1.0, total)
    return o.permute(1, 3, 0, 2, 4).reshape(b, t, hq, d).to(x["q"].dtype)


def _turns(case, positions):
    """cos and sin (..., 1, rotary_dim / 2) of the angles of positions."""
    r = case["rotary_dim"]
    rate = torch.exp(torch.arange(0, r, 2, device="cuda", dtype=F64) * (-math.log(BASE) / r))
    angle = positions.double()[..., None, None] * rate
    return angle.cos().float(), angle.sin().float()


def _rotated(case, y, cos, sin):
    """Pairs of the first rotary_dim coordinates turned; with -sin, turned back."""
    r = case["rotary_dim"]
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if case["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
    u, w = a * cos - b * sin, a * sin + b * cos
    return torch.cat([torch.stack([u, w], -1).flatten(-2) if case["interleaved"] else torch.cat([u, w], -1), y[..., r:]], -1)


def _heads(case, t, gain, cos, sin):
    t = t.float()
    return _rotated(case, t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) * gain.float(), cos, sin)


def _heads_back(case, t, gain, cos, sin, cot):
    """Gradients of the heads and of the gain."""
    t, dz = t.float(), _rotated(case, cot.float(), cos, -sin)
    r = torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
    n, dn = t * r, dz * gain.float()
    return r * (dn - n * (dn * n).mean(-1, keepdim=True)), (dz * n).flatten(0, -2).sum(0)


def _rotate(case, x):
    cos, sin = _turns(case, x["positions"])
    g, dt = (x["q_gain"], x["k_gain"]), _dtype(case)
    if case["kind"] != "rotate_packed":
        out = [_heads(case, x[name], gain, cos, sin).to(dt) for name, gain in zip("qk", g)]
        if case["kind"] == "rotate":
            return out
        back = [_heads_back(case, x[name], gain, cos, sin, cot) for name, gain, cot in zip("qk", g, x["cot"])]
        return out + [back[0][0].to(dt), back[1][0].to(dt), back[0][1].to(dt), back[1][1].to(dt)]
    b, t, w = x["qkv"].shape
    d = case["head_dim"]
    qkv, cot = x["qkv"].view(b, t, -1, 3, d), x["cot"][0].view(b, t, -1, 3, d)
    y = [_heads(case, qkv[:, :, :, i], g[i], cos, sin).to(dt) for i in range(2)] + [qkv[:, :, :, 2]]
    back = [_heads_back(case, qkv[:, :, :, i], g[i], cos, sin, cot[:, :, :, i]) for i in range(2)]
    dqkv = [back[0][0].to(dt), back[1][0].to(dt), cot[:, :, :, 2]]
    return [torch.stack(y, 3).view(b, t, w), torch.stack(dqkv, 3).view(b, t, w), back[0][1].to(dt), back[1][1].to(dt)]


# --------------------------------------------------------------------------------- the framework's
@functools.lru_cache(None)
def _call(kind, d, rotary_dim, interleaved, names):
    """The compiled function that a program of this kind keeps."""
    import nabla_b200 as nb
    from nabla_b200.nn import functional as F

    if kind == "sample":
        return nb.compile(lambda logits, uniform, *more: F.sample_tokens(logits, uniform, **dict(zip(names, more))))
    if kind == "prefix":
        return nb.compile(lambda q, cache, prefix_table, prefix_length, table, past, count: F.shared_prefix_attention(
            q, cache, prefix_table, prefix_length, table, past, count))
    more = {"eps": EPS, "base": BASE, "rotary_dim": rotary_dim, "interleaved": interleaved}
    if kind == "rotate":
        return nb.compile(lambda q, k, positions, q_gain, k_gain: F.norm_rotary(q, k, positions, q_gain, k_gain, **more))

    def grads(f, primals, cot):
        y, pull = nb.vjp(f, *primals, create_graph=False)
        return y, pull(cot)

    if kind == "rotate_packed":
        return nb.compile(lambda qkv, positions, q_gain, k_gain, cot: grads(
            lambda x, g, c: F.packed_norm_rotary(x, d, positions, g, c, **more), (qkv, q_gain, k_gain), cot))
    return nb.compile(lambda q, k, positions, q_gain, k_gain, *cot: grads(
        lambda x, y, g, c: F.norm_rotary(x, y, positions, g, c, **more), (q, k, q_gain, k_gain), cot))


ORDER = {"sample": ("logits", "uniform", "temperature", "top_k", "top_p", "min_p"),
         "prefix": ("q", "cache", "prefix_table", "prefix_length", "table", "past", "count"),
         "rotate": ("q", "k", "positions", "q_gain", "k_gain"), "rotate_train": ("q", "k", "positions", "q_gain", "k_gain"),
         "rotate_packed": ("qkv", "positions", "q_gain", "k_gain")}


def _flat(t):
    return [y for x in t for y in _flat(x)] if isinstance(t, (list, tuple)) else [t.to_torch()]


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": dict(case), "x": x}
    if own:       # the same tensors as the framework's, and the compiled function
        from nabla_b200 import Tensor

        wrap = lambda v: {k: Tensor.from_torch(t) for k, t in v.items()} if isinstance(v, dict) else Tensor.from_torch(v)  # noqa: E731
        state["args"] = [wrap(x[k]) for k in ORDER[case["kind"]] if k in x] + [Tensor.from_torch(t) for t in x.get("cot", ())]
        names = tuple(k for k in ORDER["sample"][2:] if k in x) if case["kind"] == "sample" else ()
        state["call"] = _call(case["kind"], case.get("head_dim", 0), case.get("rotary_dim", 0), case.get("interleaved", False), names)
    return state


def run(state):
    x, case = state["x"], state["case"]
    if own:
        return _flat([state["call"](*state["args"])])
    if case["kind"] == "sample":
        return [_sampled(x)]
    return [_prefixed(x)] if case["kind"] == "prefix" else _rotate(case, x)


def work(case):
    b = case["batch"]
    if case["kind"] == "sample":
        n = b * case["vocab"]
        return {"bytes": _size(case) * n + 12 * b * (1 + len(case["filters"])), "flops": 4 * n}
    d, hq, h = case["head_dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "prefix":
        live = 1.0 if b == 1 else 0.9            # of the new tokens, on average
        own_keys, new = (case["low"] + case["high"]) / 2 + case["new"], case["new"] * live
        scales = 2 * 4 / (case["block"] * d)     # bytes of the scales for each code
        return {"bytes": 2 * (case["prefix"] + b * live * own_keys) * h * d * (1 + scales) + b * (new + case["new"]) * hq * d * _size(case),
                "flops": 4 * b * new * hq * d * (case["prefix"] + own_keys - case["new"] / 2)}
    n = b * case["new"] * (hq + h) * d           # numbers of queries and keys
    if case["kind"] == "rotate":
        return {"bytes": 2 * n * _size(case), "flops": 8 * n}
    if case["kind"] == "rotate_train":
        return {"bytes": 4 * n * _size(case), "flops": 24 * n}
    return {"bytes": (4 * n + 4 * n // 2) * _size(case), "flops": 24 * n}      # the packed projection holds values too


# ------------------------------------------------------------------------------------------- 64 bits
def _exact_sample(x):
    out = []
    z, u = x["logits"].to(F64).cpu(), x["uniform"].tolist()
    for i, t in enumerate(x["temperature"].tolist()):
        row = z[i]
        ids = sorted(torch.nonzero(row >= torch.topk(row, min(row.numel(), 4096)).values[-1])[:, 0].tolist(), key=lambda j: (-row[j].item(), j)) \
            if t <= 0 or ("top_k" in x and x["top_k"][i] > 0) else torch.argsort(-row, stable=True).tolist()
        if t <= 0:
            out.append(ids[0])
            continue
        if "top_k" in x and x["top_k"][i] > 0:
            ids = ids[:int(x["top_k"][i])]
        e = torch.exp((row[ids] - row[ids[0]]) / t)
        e[e < LEAST] = 0.0
        if "top_p" in x and x["top_p"][i] < 1:
            before = torch.cat([torch.zeros(1, dtype=F64), torch.cumsum(e, 0)[:-1]])
            n = max(1, int((before < x["top_p"][i].double().cpu() * e.sum()).sum()))
            ids, e = ids[:n], e[:n]
        if "min_p" in x:
            e[e < min(1.0, x["min_p"][i].item())] = 0.0
        # in the order of the ids
        at, places = torch.sort(torch.tensor(ids))
        reached = torch.cumsum(e[places], 0)
        hits = torch.nonzero((reached > u[i] * reached[-1]) & (e[places] > 0))
        out.append(int(at[hits[0, 0]]) if len(hits) else int(at[torch.nonzero(e[places] > 0)[-1, 0]]))
    return [torch.tensor(out, device="cuda")]


def _exact_prefix(x):
    q, cache = x["q"].to(F64), x["cache"]
    b, t, hq, d = q.shape
    h, n = cache["k"].shape[1], cache["k"].shape[2]
    shared = int(x["prefix_length"])

    def numbers(name, table, keys):
        at = table[: -(-keys // n)]
        return (cache[name][at].to(F64) * cache[name + "_scale"][at].to(F64)[..., None, None]).transpose(1, 2).reshape(-1, h, d)[:keys]

    first = [numbers(name, x["prefix_table"].tolist(), shared) for name in ("k", "v")]
    out = torch.zeros_like(q)
    for i, (past, count) in enumerate(zip(x["past"].tolist(), x["count"].tolist())):
        if count == 0:
            continue
        keys, values = (torch.cat([p, numbers(name, x["table"][i].tolist(), past + count)]) for p, name in zip(first, ("k", "v")))
        ahead = torch.arange(keys.shape[0], device=q.device)[None] > shared + torch.arange(past, past + count, device=q.device)[:, None]
        for j in range(h):
            heads = slice(j * (hq // h), (j + 1) * (hq // h))
            s = torch.einsum("tgd,kd->gtk", q[i, :count, heads], keys[:, j]) / math.sqrt(d)
            out[i, :count, heads] = torch.einsum("gtk,kd->tgd", torch.softmax(s.masked_fill(ahead, -math.inf), -1), values[:, j])
    return [out]


def _exact_heads(case, t, gain, positions, cots):
    """One pair of coordinates at a time, by autograd where there are cotangents: (heads, gradient of the heads, of the gain)."""
    t, gain = t.to(F64).requires_grad_(True), gain.to(F64).requires_grad_(True)
    y = t / torch.sqrt(torch.mean(t ** 2, dim=-1, keepdim=True) + EPS) * gain
    r, parts = case["rotary_dim"], list(torch.unbind(y, -1))
    for i in range(r // 2):
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
        angle = (positions.to(F64) * BASE ** (-2.0 * i / r))[..., None]
        c, s = torch.cos(angle), torch.sin(angle)
        parts[a], parts[b] = parts[a] * c - parts[b] * s, parts[b] * c + parts[a] * s
    y = torch.stack(parts, -1)
    if cots is None:
        return (y.detach(),)
    return (y.detach(), *torch.autograd.grad(y, (t, gain), cots.to(F64)))


def _exact_rotate(case, x):
    g = (x["q_gain"], x["k_gain"])
    if case["kind"] != "rotate_packed":
        cot = x.get("cot", (None, None))
        got = [_exact_heads(case, x[name], gain, x["positions"], c) for name, gain, c in zip("qk", g, cot)]
        return [part for parts in zip(*got) for part in parts]
    b, t, w = x["qkv"].shape
    qkv, cot = x["qkv"].view(b, t, -1, 3, case["head_dim"]), x["cot"][0].view(b, t, -1, 3, case["head_dim"])
    got = [_exact_heads(case, qkv[:, :, :, i], g[i], x["positions"], cot[:, :, :, i]) for i in range(2)]
    y = torch.stack([got[0][0], got[1][0], qkv[:, :, :, 2].to(F64)], 3)
    dx = torch.stack([got[0][1], got[1][1], cot[:, :, :, 2].to(F64)], 3)
    return [y.view(b, t, w), dx.view(b, t, w), got[0][2], got[1][2]]


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(x)
    return _exact_prefix(x) if case["kind"] == "prefix" else _exact_rotate(case, x)
