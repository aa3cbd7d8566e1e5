"""Answers of the decoder in ``models/transformer.py``: prompts and single tokens over a key / value cache in 8 bits, and the choice of tokens.

``decode`` runs the new tokens of a batch through the decoder: it writes their keys and values into the cache and attends over all that the
cache holds. A prompt is a call with many new tokens, or several calls with pieces of it; an answer is a call with one new token per step.
Sequences of a batch have lengths of their own (``past``, ``count``), and a block table says where their tokens lie, so a cache can be handed
out in blocks as sequences grow. Prompts that begin with the same tokens can share them: the prefix lies in the caches once and is read once for all.

    python -m nabla_b200.models.generate --batch 4 --prompt 100 --new 32

answers random prompts with random weights (nothing is downloaded) and prints the tokens of the first and the time per step.
"""
from __future__ import annotations

import argparse
import functools
import time
from typing import Any

import torch

from ..core.tensor.api import Tensor
from ..nn import functional as F
from ..ops.view import gather, reshape, slice_tensor, squeeze
from ..transforms.compile import compile as _compile
from ..types import DType
from .transformer import TransformerConfig


def init_caches(cfg: TransformerConfig, batch: int, max_tokens: int, block_size: int = 64, device=None, prefix_tokens: int = 0):
    """A cache for each layer with room for ``max_tokens`` of each sequence, and the table that gives every sequence its own blocks; with
    ``prefix_tokens`` also room for a prefix of so many that all share, and the table (columns,) of its blocks."""
    from ..ops.creation import constant

    columns, shared = -(-max_tokens // block_size), -(-prefix_tokens // block_size)
    caches = [F.init_kv_cache(batch * columns + shared, cfg.n_heads, cfg.head_dim, block_size, device=device) for _ in range(cfg.n_layers)]
    table = constant(torch.arange(batch * columns, dtype=torch.int32).view(batch, columns).numpy(), dtype=DType.int32, device=device)
    if not shared:
        return caches, table
    return caches, table, constant((torch.arange(shared, dtype=torch.int32) + batch * columns).numpy(), dtype=DType.int32, device=device)


def decode(params: dict[str, Any], tokens: Tensor, caches: list[dict[str, Tensor]], table: Tensor, past: Tensor, cfg: TransformerConfig,
           count: Tensor | None = None, positions: Tensor | None = None,
           prefix: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, list[dict[str, Tensor]]]:
    """tokens (B, S), the first ``count`` (B,) of them behind ``past`` (B,) tokens that the caches hold -> logits (B, S, vocab) and the caches.
    ``prefix``: the table (columns,) of the blocks of tokens that all sequences begin with, and their number (1,); ``past`` does not count them.
    ``positions`` (B, S) index the position embedding, or turn queries and keys: those of the whole text, ``past + i`` behind the prefix, by default,
    0 for what lies behind ``count``."""
    from ..ops.comparison import less
    from ..ops.control_flow import where
    from ..ops.creation import arange
    from ..ops.unary import cast
    from ..ops.view import unsqueeze

    B, S = (int(n) for n in tokens.shape)
    H, hd = cfg.n_heads, cfg.head_dim
    if positions is None:
        i = arange(0, S, 1, dtype=DType.int64, device=tokens.device)
        positions = unsqueeze(cast(past, DType.int64), axis=1) + i
        if prefix is not None:
            positions = positions + cast(prefix[1], DType.int64)
        if count is not None:               # there may be no such position
            positions = where(less(i, unsqueeze(cast(count, DType.int64), axis=1)), positions, positions * 0)
    x = gather(params["tok_emb"], tokens, axis=0)
    if cfg.rotary_base is None:
        x = x + gather(params["pos_emb"], positions, axis=0)
    out = []
    for p, cache in zip(params["layers"], caches):
        qkv = reshape(F.linear(F.layer_norm(x, p["ln1_g"], p["ln1_b"]), p["wqkv"], p["bqkv"]), (B, S, H, 3, hd))
        q, k, v = (squeeze(slice_tensor(qkv, (0, 0, 0, i, 0), (B, S, H, 1, hd)), axis=3) for i in range(3))
        if cfg.rotary_base is not None:
            q, k = F.norm_rotary(q, k, positions, p.get("q_gain"), p.get("k_gain"), base=cfg.rotary_base)
        cache = F.kv_cache_write(cache, k, v, table, past, count)
        a = F.cached_attention(q, cache, table, past, count) if prefix is None else F.shared_prefix_attention(q, cache, *prefix, table, past, count)
        out.append(cache)
        x = x + F.linear(reshape(a, (B, S, H * hd)), p["wo"], p["bo"])
        h = F.linear(F.layer_norm(x, p["ln2_g"], p["ln2_b"]), p["w1"], p["b1"], activation="gelu")
        x = x + F.linear(h, p["w2"], p["b2"])
    return F.linear(F.layer_norm(x, params["lnf_g"], params["lnf_b"]), params["lm_head"]), out


def move(cache: dict[str, Tensor], table: Tensor, count: Tensor, max_tokens: int, other: dict[str, Tensor], other_table: Tensor) -> dict[str, Tensor]:
    """The first ``count`` tokens of each sequence of one cache, written into another (of another block size, or with its blocks in order)."""
    zero = count * 0
    k, v = F.kv_cache_read(cache, table, zero, count, max_tokens, dtype=DType.float32)
    return F.kv_cache_write(other, k, v, other_table, zero, count)


@functools.lru_cache(8)
def _steps(layers: int, dim: int, heads: int, hidden: int, vocab: int, max_seq: int, rotary_base: float | None = None, qk_norm: bool = False):
    """Compiled once per model: the call for prompts and steps, and the choice of the next tokens, the likeliest or drawn."""
    cfg = TransformerConfig(n_layers=layers, d_model=dim, n_heads=heads, d_ff=hidden, vocab=vocab, max_seq=max_seq, rotary_base=rotary_base, qk_norm=qk_norm)

    def forward(params, tokens, caches, table, past, count, positions, *prefix):
        return decode(params, tokens, caches, table, past, cfg, count, positions, prefix or None)

    def adjusted(logits, history, length, prompt_length, repetition, presence, frequency, allowed):
        return F.adjust_logits(logits, history, length, prompt_length, repetition=repetition, presence=presence, frequency=frequency,
                               **({"allowed": allowed[0]} if allowed else {}))

    def choose(logits, history, length, prompt_length, repetition, presence, frequency, *allowed):
        from ..ops.reduction import argmax

        return argmax(adjusted(logits, history, length, prompt_length, repetition, presence, frequency, allowed), axis=-1)

    def draw(uniform, filters, logits, history, length, prompt_length, repetition, presence, frequency, *allowed):
        return F.sample_tokens(adjusted(logits, history, length, prompt_length, repetition, presence, frequency, allowed), uniform, **filters)

    return _compile(forward), _compile(choose), _compile(draw)


def generate(params: dict[str, Any], prompts: list[list[int]], cfg: TransformerConfig, max_new: int, *, block_size: int = 64, piece: int = 2048,
             repetition: float = 1.0, presence: float = 0.0, frequency: float = 0.0, allowed: Tensor | None = None, device=None,
             prefix: list[int] | None = None, temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0, seed: int = 0) -> list[list[int]]:
    """The tokens that the decoder puts behind each prompt, ``max_new`` of them: the likeliest at every step after the penalties, or with a
    ``temperature`` drawn among those that ``top_k``, ``top_p`` and ``min_p`` keep (``F.sample_tokens``), with random numbers of ``seed``. Prompts go in
    pieces of at most ``piece`` tokens. ``prefix``: tokens in front of every prompt, which are gone through once for all. ``allowed`` (batch,
    ceil(vocab / 32)) int32 hides tokens whose bit is 0; where all are hidden, token 0 follows."""
    if not prompts or any(not p for p in prompts):
        raise ValueError("every prompt has at least one token")
    if temperature < 0:
        raise ValueError("temperature is negative")
    prefix = list(prefix or [])
    P, longest = len(prefix), max(len(p) for p in prompts)
    if P + longest + max_new > cfg.max_seq:
        raise ValueError(f"{P + longest} + {max_new} tokens are more than the {cfg.max_seq} positions of the model")
    B = len(prompts)
    dev = params["tok_emb"]._impl.device.to_torch() if device is None else torch.device(device)
    put = lambda t: Tensor.from_torch(t.to(dev))  # noqa: E731
    forward, choose, draw = _steps(cfg.n_layers, cfg.d_model, cfg.n_heads, cfg.d_ff, cfg.vocab, cfg.max_seq, cfg.rotary_base, cfg.qk_norm)
    caches, table, *shared = init_caches(cfg, B, longest + max_new, block_size, device=params["tok_emb"]._impl.device, prefix_tokens=P)
    if P:
        shared = (shared[0], put(torch.tensor([P], dtype=torch.int32)))
        for at in range(0, P, piece):
            n, start = min(piece, P - at), torch.tensor([at], dtype=torch.int32)
            _, caches = forward(params, put(torch.tensor([prefix[at:at + n]])), caches, put(shared[0].to_torch()[None]), put(start),
                                put(torch.tensor([n], dtype=torch.int32)), put(torch.arange(at, at + n)[None]))
    lengths = torch.tensor([len(p) for p in prompts], dtype=torch.int32)
    history = torch.zeros((B, P + longest + max_new), dtype=torch.int32)
    history[:, :P] = torch.tensor(prefix, dtype=torch.int32)
    for i, p in enumerate(prompts):
        history[i, P:P + len(p)] = torch.tensor(p, dtype=torch.int32)
    numbers = [put(torch.full((B,), float(x))) for x in (repetition, presence, frequency)]
    last = torch.zeros((B, cfg.vocab), dtype=params["lm_head"].dtype.to_torch(), device=dev)
    for at in range(0, longest, piece):
        n = min(piece, longest - at)
        count = (lengths - at).clamp(0, n)
        past = torch.minimum(lengths, torch.tensor(at, dtype=torch.int32))
        positions = (P + past.long()[:, None] + torch.arange(n)).clamp(max=cfg.max_seq - 1)
        logits, caches = forward(params, put(history[:, P + at:P + at + n].long().contiguous()), caches, table, put(past), put(count), put(positions), *shared)
        ends = (lengths > at) & (lengths <= at + n)                       # prompts whose last token is in this piece
        rows = torch.arange(B)[ends].to(dev)
        last[rows] = logits.to_torch()[rows, (lengths[ends] - 1 - at).long().to(dev)]
    history, prompt_length, length = history.to(dev), put(lengths + P), lengths.to(dev)
    one, rows = put(torch.ones(B, dtype=torch.int32)), torch.arange(B, device=dev)
    uniform = torch.rand((max_new, B), generator=torch.Generator().manual_seed(seed)).to(dev) if temperature > 0 else None
    # filters that let all through are left out: a draw without top-k and top-p has a kernel of its own
    given = {"temperature": (float(temperature), True), "top_k": (int(top_k), top_k > 0), "top_p": (float(top_p), top_p < 1), "min_p": (float(min_p), min_p > 0)}
    filters = {k: put(torch.full((B,), x, dtype=torch.int32 if k == "top_k" else torch.float32)) for k, (x, used) in given.items() if used}
    for step in range(max_new):
        args = (Tensor.from_torch(last), Tensor.from_torch(history), Tensor.from_torch(length + P), prompt_length, *numbers, *(() if allowed is None else (allowed,)))
        if uniform is None:
            token = choose(*args).to_torch()
        else:
            token = draw(Tensor.from_torch(uniform[step]), filters, *args).to_torch().clamp(min=0)
        history[rows, P + length.long()] = token.to(torch.int32)
        if step + 1 < max_new:
            logits, caches = forward(params, Tensor.from_torch(token.long()[:, None]), caches, table, Tensor.from_torch(length), one,
                                     Tensor.from_torch(P + length.long()[:, None]), *shared)
            last = logits.to_torch()[:, 0].contiguous()
        length = length + 1
    return [history[i, P + int(n):P + int(n) + max_new].tolist() for i, n in enumerate(lengths)]


def main() -> None:
    from ..core.common.context import default_device
    from ..core.graph.engine import seed
    from ..types import CPU, Accelerator
    from .transformer import init_params

    ap = argparse.ArgumentParser(description="answer random prompts with random weights")
    for name, n in (("layers", 4), ("dim", 512), ("heads", 8), ("vocab", 8192), ("batch", 4), ("prompt", 100), ("new", 32), ("block", 64), ("prefix", 0), ("top-k", 0)):
        ap.add_argument(f"--{name}", type=int, default=n)
    for name, x in (("temperature", 0.0), ("top-p", 1.0), ("min-p", 0.0)):
        ap.add_argument(f"--{name}", type=float, default=x)
    ap.add_argument("--rotary", action="store_true", help="queries and keys normed and turned by their positions in place of a position embedding")
    a = ap.parse_args()
    gpu = torch.cuda.is_available()
    cfg = TransformerConfig(n_layers=a.layers, d_model=a.dim, n_heads=a.heads, d_ff=4 * a.dim, vocab=a.vocab,
                            dtype=DType.bfloat16 if gpu else DType.float32, max_seq=max(2048, a.prefix + a.prompt + a.new),
                            rotary_base=10000.0 if a.rotary else None, qk_norm=a.rotary)
    with default_device(Accelerator(0) if gpu else CPU()):
        seed(0)
        params = init_params(cfg)
        g = torch.Generator().manual_seed(0)
        prompts = [torch.randint(0, a.vocab, (max(1, a.prompt - i),), generator=g).tolist() for i in range(a.batch)]
        prefix = torch.randint(0, a.vocab, (a.prefix,), generator=g).tolist()
        for _ in range(2):             # the first time compiles
            t0 = time.perf_counter()
            answers = generate(params, prompts, cfg, a.new, block_size=a.block, repetition=1.1, presence=0.1, prefix=prefix, temperature=a.temperature,
                               top_k=a.top_k, top_p=a.top_p, min_p=a.min_p)
            took = time.perf_counter() - t0
    print("first answer:", answers[0])
    print(f"{took * 1e3 / a.new:.2f} ms a step, prompts included, {a.batch * a.new / took:.0f} tokens/s")


if __name__ == "__main__":
    main()
