"""The serving operations (cache in 8 bits, attention over it, adjustment of logits) against their definitions in 64 bits.

The same checks run on the CPU (torch expressions) and on a GPU (hand-written kernels). Tolerances come from the roundings that the
definitions name; each is derived where it stands.
"""
from __future__ import annotations

import math

import pytest
import torch

import nabla_b200 as nb
from nabla_b200.nn import functional as F

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TINY = 2.0 ** -100


def T(x):
    return nb.Tensor.from_torch(x)


def gen(device, seed):
    return torch.Generator(device).manual_seed(seed)


def new_cache(g, device, blocks, heads, n, d, scale=(0.014, 0.042)):
    c = {}
    for name in ("k", "v"):
        c[name] = torch.randint(-127, 128, (blocks, heads, n, d), generator=g, device=device, dtype=torch.int8)
        c[name + "_scale"] = torch.rand((blocks, heads), generator=g, device=device) * (scale[1] - scale[0]) + scale[0]
    return c


def new_table(g, device, batch, columns, blocks, dtype=torch.int32):
    """Distinct blocks in no order."""
    assert batch * columns <= blocks
    return torch.randperm(blocks, generator=g, device=device)[: batch * columns].view(batch, columns).to(dtype)


def wrap(c):
    return {k: T(v) for k, v in c.items()}


def values64(cache, name, table, n_keys):
    """(keys, there) of one sequence, places without a block as zeros."""
    blocks, h, n, d = cache[name].shape
    out = torch.zeros((len(table) * n, h, d), dtype=torch.float64, device=cache[name].device)
    there = torch.zeros(len(table) * n, dtype=torch.bool, device=out.device)
    for c, id_ in enumerate(table):
        if 0 <= id_ < blocks and c * n < n_keys:
            out[c * n:(c + 1) * n] = (cache[name][id_].double() * cache[name + "_scale"][id_].double()[:, None, None]).transpose(0, 1)
            there[c * n:(c + 1) * n] = True
    return out[:n_keys], there[:n_keys]


# ---------------------------------------------------------------- attention
def attend64(q, cache, table, past, count, causal, scale):
    b, t, hq, d = q.shape
    h, n = cache["k"].shape[1:3]
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device=q.device)
    bound = torch.zeros((b, t, hq, 1), dtype=torch.float64, device=q.device)
    for i in range(b):
        p = min(max(int(past[i]), 0), table.shape[1] * n)
        c = t if count is None else min(max(int(count[i]), 0), t)
        keys = min(p + c, table.shape[1] * n)
        if c == 0:
            continue
        k, there = values64(cache, "k", table[i].tolist(), keys)
        v, _ = values64(cache, "v", table[i].tolist(), keys)
        at = torch.arange(keys, device=q.device)
        last = p + torch.arange(c, device=q.device) if causal else torch.full((c,), p + c - 1, device=q.device)
        seen = (at[None] <= last[:, None]) & there[None]
        for x in range(hq):
            kk, vv = k[:, x // (hq // h)], v[:, x // (hq // h)]
            s = torch.where(seen, q[i, :c, x].double() @ kk.T * scale, -math.inf)
            top = s.amax(-1, keepdim=True) if keys else s.new_full((c, 1), -math.inf)
            e = torch.where(seen, torch.exp(s - torch.where(torch.isinf(top), 0.0, top)), 0.0)
            w = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
            out[i, :c, x] = w @ torch.where(seen.any(0)[:, None], vv, 0.0)
            if keys:
                # score: D products of q and k summed in fp32 (and the offset of the codes, 9 times their largest magnitude)
                ds = scale * 2.0 ** -22 * d * 9 * q[i, :c, x].double().abs().amax(-1) * torch.where(seen.any(0)[:, None], kk, 0.0).abs().max()
                bound[i, :c, x, 0] = ds * torch.where(seen.any(0)[:, None], vv, 0.0).abs().max()
    return out, bound


ATTEND = [
    # batch, new, heads, kv heads, head_dim, block, past, count, dtype, causal, table dtype
    (1, 1, 1, 1, 64, 16, [0], None, "bf16", True, "int32"),                      # a first token: one key, its own
    (1, 1, 16, 16, 128, 64, [700], None, "bf16", True, "int32"),
    (3, 1, 8, 2, 128, 16, [0, 15, 16], [1, 1, 1], "bf16", True, "int64"),
    (4, 1, 12, 4, 64, 32, [31, 32, 33, 500], [1, 0, 1, 1], "bf16", True, "int32"),
    (2, 1, 8, 1, 64, 128, [127, 1000], None, "fp32", True, "int32"),
    (2, 1, 24, 2, 128, 64, [63, 64], None, "fp32", True, "int32"),
    (1, 1, 32, 1, 128, 64, [300], None, "bf16", True, "int32"),                  # more rows than one tile of 16
    (2, 1, 4, 4, 128, 64, [3000, 1], None, "bf16", True, "int32"),
    (5, 5, 6, 2, 64, 16, [0, 7, 100, 11, 250], [5, 5, 0, 3, 1], "bf16", True, "int32"),
    (2, 7, 4, 4, 128, 32, [9, 200], [7, 2], "fp32", True, "int64"),
    (2, 5, 8, 1, 128, 64, [1, 100], None, "bf16", False, "int32"),
    (2, 33, 4, 2, 64, 16, [0, 77], [33, 20], "bf16", True, "int32"),
    (1, 130, 3, 1, 128, 64, [0], None, "bf16", True, "int32"),
    (2, 257, 4, 1, 64, 32, [0, 333], [257, 129], "bf16", True, "int32"),
    (2, 100, 8, 8, 128, 128, [1000, 5], [100, 0], "bf16", True, "int32"),
    (1, 64, 16, 2, 128, 16, [2500], None, "bf16", True, "int32"),
    (2, 70, 4, 2, 128, 64, [30, 0], [70, 64], "bf16", False, "int32"),
    (2, 40, 4, 2, 64, 64, [30, 0], [40, 39], "fp32", True, "int32"),
    (1, 300, 2, 2, 128, 64, [20], [260], "fp32", True, "int32"),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", ATTEND)
def test_attention_over_the_cache(case, device):
    b, t, hq, h, d, n, past, count, dtype, causal, whole = case
    g = gen(device, 3)
    dtype, whole = (torch.bfloat16 if dtype == "bf16" else torch.float32), getattr(torch, whole)
    columns = (max(past) + t + n - 1) // n + 2
    cache = new_cache(g, device, b * columns + 3, h, n, d)
    table = new_table(g, device, b, columns, b * columns, whole)
    past_t = torch.tensor(past, device=device, dtype=whole)
    count_t = None if count is None else torch.tensor(count, device=device, dtype=whole)
    # what lies behind a sequence's tokens is never looked at: no block, or one whose scales are NaN
    for i in range(b):
        used = -(-(past[i] + (t if count is None else count[i])) // n)
        table[i, used:] = -1
        if used + 1 < columns:
            table[i, used + 1] = b * columns + 2
    cache["k_scale"][b * columns + 2] = math.nan
    cache["v_scale"][b * columns + 2] = math.nan
    table[:, -1][table[:, -1] == -1] = 1 << 30
    q = torch.randn((b, t, hq, d), generator=g, device=device).to(dtype)
    got = F.cached_attention(T(q), wrap(cache), T(table), T(past_t), None if count_t is None else T(count_t), causal=causal).to_torch()
    want, bound = attend64(q, cache, table, past, count, causal, d ** -0.5)
    assert got.dtype == dtype and got.shape == q.shape
    check_attention(got, want, bound, cache)


def check_attention(got, want, bound, cache):
    vmax = 127 * cache["v_scale"].nan_to_num(0).max().item()
    if got.dtype == torch.bfloat16:
        # the result rounded to 8 bits, weights rounded to 11 bits on the way to the products (half a unit each, both relative)
        tol = 2.0 ** -8 * want.abs() + 2.0 ** -10 * vmax + bound
    else:
        # weights in two parts of 11 bits, exponentials in fp32 (2 units), the sum of up to some thousand products of them
        tol = 2.0 ** -18 * vmax + bound
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), f"off by {(off - tol).max().item():.3g} more than allowed ({off.max().item():.3g})"
    empty = (want == 0).all(-1)
    assert (got[empty] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new", [1, 6, 150])
def test_attention_where_blocks_are_missing_and_scales_differ_widely(device, new):
    """Blocks in the middle that are not there, a first block that is not, one sequence without any; scales from 2^-100 to 2^40."""
    g = gen(device, 5)
    b, hq, h, d, n, columns = 4, 4, 2, 128, 16, 40
    cache = new_cache(g, device, 200, h, n, d)
    cache["v_scale"][::3] = TINY
    cache["v_scale"][1::7] = 2.0 ** 40
    cache["k_scale"][::5] = TINY
    table = new_table(g, device, b, columns, 200)
    table[0, 3:5] = -1
    table[1, 0] = 200
    table[2, :] = -5
    table[3, 20] = -(1 << 31)
    past = torch.tensor([400, 37, 300, 330], device=device, dtype=torch.int32)
    q = torch.randn((b, new, hq, d), generator=g, device=device).to(torch.bfloat16)
    got = F.cached_attention(T(q), wrap(cache), T(table), T(past)).to_torch()
    want, bound = attend64(q, cache, table, past.tolist(), None, True, d ** -0.5)
    assert (got[2] == 0).all()
    check_attention(got, want, bound, cache)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("b,new,hq,h,longest", [
    (1, 12, 16, 4, 700), (2, 16, 16, 4, 5000), (9, 32, 8, 4, 1000), (4, 16, 32, 8, 1900), (4, 16, 32, 8, 2300), (16, 24, 32, 8, 300), (3, 33, 16, 4, 1500),
    (1, 9, 4, 1, 2080),
])
def test_attention_of_some_tens_of_rows(b, new, hq, h, longest, dtype):
    """Between single tokens and prompts: rows of one to several tiles, on both sides of where another form is taken."""
    g = gen("cuda", 43)
    n, d, dtype = 64, 128, torch.bfloat16 if dtype == "bf16" else torch.float32
    columns = -(-(longest + new) // n)
    cache = new_cache(g, "cuda", b * columns + 1, h, n, d)
    table = new_table(g, "cuda", b, columns, b * columns + 1)
    past = torch.randint(0, longest + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    past[-1] = 0
    past[0] = longest
    count = torch.randint(0, new + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    count[0] = new
    q = torch.randn((b, new, hq, d), generator=g, device="cuda").to(dtype)
    got = F.cached_attention(T(q), wrap(cache), T(table), T(past), T(count)).to_torch()
    want, bound = attend64(q, cache, table, past.tolist(), count.tolist(), True, d ** -0.5)
    check_attention(got, want, bound, cache)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,hq,h,columns,longest,dtype", [
    (39, 16, 4, 11, 649, "bf16"),         # more units of keys than blocks share them, fewer, and far fewer than the table has room for
    (3, 4, 1, 400, 11990, "bf16"), (3, 4, 1, 400, 300, "bf16"), (2, 8, 1, 4000, 129, "fp32"), (16, 32, 8, 40, 209, "bf16"), (5, 12, 2, 300, 9000, "fp32"),
    (200, 8, 8, 8, 200, "bf16"), (1024, 4, 2, 4, 90, "bf16"), (1025, 4, 2, 4, 90, "bf16"), (7, 32, 2, 500, 4000, "bf16"),
])
def test_ragged_batches_share_the_chip(b, hq, h, columns, longest, dtype, d):
    """Sequences of lengths from nothing to the longest, idle ones among them; scratch that holds garbage."""
    g = gen("cuda", 41)
    n, dtype = 64, torch.bfloat16 if dtype == "bf16" else torch.float32
    blocks = -(-longest // n) * b + 1
    cache = new_cache(g, "cuda", blocks, h, n, d)
    table = torch.full((b, columns), -1, device="cuda", dtype=torch.int32)
    used = -(-longest // n)
    table[:, :used] = new_table(g, "cuda", b, used, blocks)
    past = torch.randint(0, longest, (b,), generator=g, device="cuda", dtype=torch.int32)
    past[0], past[-1] = longest - 1, 0
    count = (torch.rand((b,), generator=g, device="cuda") < 0.7).to(torch.int32)
    q = torch.randn((b, 1, hq, d), generator=g, device="cuda").to(dtype)
    garbage = torch.full((64 << 20,), math.nan, device="cuda")       # what freed memory holds
    del garbage
    got = F.cached_attention(T(q), wrap(cache), T(table), T(past), T(count)).to_torch()
    want, bound = attend64(q, cache, table, past.tolist(), count.tolist(), True, d ** -0.5)
    check_attention(got, want, bound, cache)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new", [1, 150])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_with_large_and_small_queries(device, new, dtype):
    """Queries far outside the range of 16-bit floats: weights of one key, or all alike."""
    g = gen(device, 6)
    b, h, d, n = 2, 2, 64, 32
    cache = new_cache(g, device, 40, h, n, d)
    table = new_table(g, device, b, 20, 40)
    past = torch.tensor([100, 399], device=device, dtype=torch.int32)
    q = torch.randn((b, new, h, d), generator=g, device=device)
    q[0] *= 1e30
    q[1] *= 1e-30
    q = q.to(dtype)
    got = F.cached_attention(T(q), wrap(cache), T(table), T(past)).to_torch()
    want, bound = attend64(q, cache, table, past.tolist(), None, True, d ** -0.5)
    check_attention(got[1:], want[1:], bound[1:], cache)
    # the key with the largest score, exact in every arithmetic unless two are within a rounding of each other
    off = (got[0].double() - want[0]).abs() <= 2.0 ** -8 * want[0].abs() + 2.0 ** -10 * 127 * 0.042
    assert off.all(-1).float().mean() > 0.95


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new", [1, 150])
def test_what_is_not_a_number_comes_through_where_it_is_seen(device, new):
    g = gen(device, 7)
    h, d, n = 2, 128, 16
    cache = new_cache(g, device, 30, h, n, d)
    table = new_table(g, device, 1, 20, 30)
    past = torch.tensor([48], device=device, dtype=torch.int32)
    q = torch.randn((1, new, 2 * h, d), generator=g, device=device).to(torch.bfloat16)
    cache["k_scale"][int(table[0, 1]), 0] = math.nan
    cache["v_scale"][int(table[0, 1]), 1] = math.nan
    got = F.cached_attention(T(q), wrap(cache), T(table), T(past)).to_torch()
    assert torch.isnan(got).all()
    cache["k_scale"][int(table[0, 1]), 0] = 0.02
    got = F.cached_attention(T(q), wrap(cache), T(table), T(past)).to_torch()
    assert torch.isfinite(got[:, :, :2]).all() and torch.isnan(got[:, :, 2:]).all()
    cache["v_scale"][int(table[0, 1]), 1] = 0.02
    q[0, 0, 1, 5] = math.inf
    got = F.cached_attention(T(q), wrap(cache), T(table), T(past)).to_torch()
    assert torch.isnan(got[0, 0, 1]).all() and torch.isfinite(got[0, 0, 0]).all() and torch.isfinite(got[0, 1:]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new", [1, 40, 200])
def test_queries_are_read_where_they_lie(device, new):
    """Views of a packed projection, heads in front of tokens, and one that starts off a boundary."""
    g = gen(device, 8)
    b, h, d, n = 2, 4, 64, 64
    cache = wrap(new_cache(g, device, 30, 2, n, d))
    table, past = T(new_table(g, device, b, 10, 30)), T(torch.tensor([100, 70], device=device, dtype=torch.int32))
    q = torch.randn((b, new, h, d), generator=g, device=device).to(torch.bfloat16)
    want = F.cached_attention(T(q), cache, table, past).to_torch()
    packed = torch.zeros((b, new, h, 3, d), device=device, dtype=q.dtype)
    packed[:, :, :, 1] = q
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(q.numel() + 3, device=device, dtype=q.dtype)[3:].view(q.shape)
    odd.copy_(q)
    for view in (packed[:, :, :, 1], turned, odd):
        assert torch.equal(F.cached_attention(T(view), cache, table, past).to_torch(), want)


# ---------------------------------------------------------------- writing and reading
def write64(cache, k, v, table, past, count):
    """New scales, and for each code the number that was rounded; nothing where nothing is written."""
    out = {}
    for name, x in (("k", k), ("v", v)):
        blocks, h, n, d = cache[name].shape
        scales = cache[name + "_scale"].double().clone()
        exact = torch.full(cache[name].shape, math.nan, dtype=torch.float64, device=x.device)
        for i in range(x.shape[0]):
            p = min(max(int(past[i]), 0), table.shape[1] * n)
            c = x.shape[1] if count is None else min(max(int(count[i]), 0), x.shape[1])
            done = 0
            while done < c:
                col, f = divmod(p + done, n)
                m = min(n - f, c - done)
                id_ = int(table[i, col]) if col < table.shape[1] else -1
                if 0 <= id_ < blocks:
                    new = x[i, done:done + m].double()                                   # (m, h, d)
                    before = cache[name + "_scale"][id_].double() if f else torch.zeros(h, dtype=torch.float64, device=x.device)
                    scale = torch.maximum(before, (new.abs().amax((0, 2)) / 127).clamp(min=TINY))
                    exact[id_, :, :f] = cache[name][id_, :, :f].double() * (before / scale)[:, None, None]
                    exact[id_, :, f:f + m] = (new / scale[None, :, None]).transpose(0, 1)
                    scales[id_] = scale
                done += m
        out[name], out[name + "_scale"] = exact, scales
    return out


WRITE = [
    # batch, new, heads, head_dim, block, past, count, dtype, table dtype
    (1, 1, 1, 64, 16, [0], None, "bf16", "int32"),
    (3, 1, 4, 128, 64, [0, 63, 64], None, "bf16", "int32"),
    (4, 1, 2, 64, 16, [5, 15, 16, 100], [1, 0, 1, 1], "fp32", "int64"),
    (2, 16, 3, 64, 16, [0, 1], None, "bf16", "int32"),
    (3, 100, 2, 128, 32, [0, 31, 500], [100, 77, 0], "bf16", "int64"),
    (2, 129, 1, 128, 128, [0, 127], [129, 128], "fp32", "int32"),
    (2, 333, 5, 64, 64, [10, 0], None, "fp32", "int32"),
    (1, 300, 16, 128, 64, [1000], None, "bf16", "int32"),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", WRITE)
def test_writing_into_the_cache(case, device):
    b, t, h, d, n, past, count, dtype, whole = case
    g = gen(device, 11)
    dtype, whole = (torch.bfloat16 if dtype == "bf16" else torch.float32), getattr(torch, whole)
    columns = (max(past) + t) // n + 2
    cache = new_cache(g, device, b * columns + 2, h, n, d, (0.001, 0.05))
    table = new_table(g, device, b, columns, b * columns + 2, whole)
    packed = torch.randn((b, t, h, 3, d), generator=g, device=device) * torch.rand((b, t, h, 3, 1), generator=g, device=device) * 3
    packed = packed.to(dtype)
    k, v = packed[:, :, :, 1], packed[:, :, :, 2]
    past_t = torch.tensor(past, device=device, dtype=whole)
    count_t = None if count is None else T(torch.tensor(count, device=device, dtype=whole))
    before = {name: x.clone() for name, x in cache.items()}
    live = wrap(cache)
    got = F.kv_cache_write(live, T(k), T(v), T(table), T(past_t), count_t)
    want = write64(before, k, v, table, past, count)
    for name in ("k", "v"):
        assert got[name].to_torch() is cache[name] and got[name + "_scale"].to_torch() is cache[name + "_scale"]
        check_written(cache, before, want, name)
    # keys and values that start off a boundary
    odd = [torch.zeros(x.numel() + 1, device=device, dtype=dtype)[1:].view(x.shape).copy_(x) for x in (k, v)]
    third = {name: x.clone() for name, x in before.items()}
    F.kv_cache_write(wrap(third), T(odd[0]), T(odd[1]), T(table), T(past_t), count_t)
    assert all(torch.equal(third[name], cache[name]) for name in cache)
    # a copy is left alone, and comes out the same
    copy = {name: x.clone() for name, x in before.items()}
    again = F.kv_cache_write(wrap(copy), T(k), T(v), T(table), T(past_t), count_t, inplace=False)
    for name in cache:
        assert torch.equal(copy[name], before[name]) and torch.equal(again[name].to_torch()[..., :1], cache[name][..., :1])


def check_written(cache, before, want, name):
    scale, exact = want[name + "_scale"], want[name]
    written = ~exact.isnan()
    # scales: a product with 1 / 127 rounded, two roundings of 2^-24
    assert ((cache[name + "_scale"].double() - scale).abs() <= 2.0 ** -22 * scale).all()
    codes = cache[name].double()
    # a code is the nearest whole number; the quotient has three roundings of 2^-24 at most, 127 * 2^-22 from a half decides nothing
    off = (codes - exact).abs()[written]
    assert (off <= 0.5 + 127 * 2.0 ** -22).all()
    assert (codes.abs() <= 127).all()
    # rows in front of the new ones are touched only together with them, rows of other blocks never
    others = ~written.flatten(1).any(1)
    assert torch.equal(cache[name][others], before[name][others])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_codes_are_those_of_the_definition_bit_for_bit(dtype):
    """1 / scale rounded, the product rounded, the nearest whole number: quotients halfway between two are many in bf16, and kernels and torch agree."""
    g = gen("cuda", 19)
    b, t, h, d, n = 4, 300, 4, 128, 64
    cache = new_cache(g, "cuda", b * 8, h, n, d)
    table = new_table(g, "cuda", b, 8, b * 8)
    past, count = torch.tensor([0, 10, 63, 130], device="cuda", dtype=torch.int32), torch.tensor([300, 299, 0, 64], device="cuda", dtype=torch.int32)
    k, v = ((torch.randn((b, t, h, d), generator=g, device="cuda") * 3).to(dtype) for _ in range(2))
    host = F.kv_cache_write({name: T(x.cpu()) for name, x in cache.items()}, T(k.cpu()), T(v.cpu()), T(table.cpu()), T(past.cpu()), T(count.cpu()))
    F.kv_cache_write(wrap(cache), T(k), T(v), T(table), T(past), T(count))
    for name in cache:
        assert torch.equal(cache[name].cpu(), host[name].to_torch())


@pytest.mark.parametrize("device", DEVICES)
def test_writing_what_is_not_finite_or_zero_and_writing_past_the_end(device):
    h, d, n = 2, 64, 16
    cache = new_cache(gen(device, 12), device, 8, h, n, d)
    table = torch.tensor([[1, 2], [3, 9], [-1, 4]], device=device, dtype=torch.int32)
    k = torch.zeros((3, 8, h, d), device=device)
    v = torch.ones((3, 8, h, d), device=device)
    k[0, 2, 1, 3] = math.inf
    v[1, 0, 0, 0] = math.nan
    v[2] = 1e-38
    past = torch.tensor([12, 12, 28], device=device, dtype=torch.int32)
    before = {name: x.clone() for name, x in cache.items()}
    F.kv_cache_write(wrap(cache), T(k), T(v), T(table), T(past))
    ks, vs = cache["k_scale"], cache["v_scale"]
    assert ks[1, 0] == before["k_scale"][1, 0] and ks[1, 1].isnan()                # rows 12 to 15 of block 1, an infinity in head 1
    assert ks[2].tolist() == [TINY, TINY] and (cache["k"][2, :, :4] == 0).all()    # the rest starts block 2: all zero
    assert vs[3, 0].isnan() and vs[3, 1] == before["v_scale"][3, 1]
    assert vs[4, 0] == before["v_scale"][4, 0] and (cache["v"][4, :, 12:] == 0).all()      # rows 12 to 15 of block 4; the table ends there
    for i in (0, 5, 6, 7):
        assert torch.equal(cache["k"][i], before["k"][i]) and torch.equal(cache["v"][i], before["v"][i])
    assert torch.equal(cache["v"][4, :, :12], before["v"][4, :, :12])
    # a NaN stays until the block's first row is written
    one = torch.ones((3, 1, h, d), device=device)
    F.kv_cache_write(wrap(cache), T(one), T(one), T(table), T(torch.tensor([13, 13, 99], device=device, dtype=torch.int32)))
    assert ks[1, 1].isnan() and vs[3, 0].isnan()
    F.kv_cache_write(wrap(cache), T(one), T(one), T(table), T(torch.zeros(3, device=device, dtype=torch.int32)))
    assert torch.isfinite(ks[1]).all() and torch.isfinite(vs[3]).all()
    k_back, _ = F.kv_cache_read(wrap(cache), T(table), T(torch.zeros(3, device=device, dtype=torch.int32)),
                                T(torch.ones(3, device=device, dtype=torch.int32)), 1, dtype=nb.DType.float32)
    assert (k_back.to_torch()[:2] - 1).abs().max() < 1e-6 and (k_back.to_torch()[2] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("d,n,most,dtype", [(64, 16, 1, "float32"), (64, 64, 77, "bfloat16"), (128, 32, 200, "bfloat16"), (128, 128, 130, "float32")])
def test_reading_the_cache(device, d, n, most, dtype):
    g = gen(device, 13)
    b, h, columns = 4, 3, 12
    cache = new_cache(g, device, b * columns, h, n, d)
    table = new_table(g, device, b, columns, b * columns, torch.int64)
    table[1, 1] = -1
    start = torch.tensor([0, 3, n - 1, columns * n - 5], device=device)
    count = torch.tensor([most, most + 9, 0, most], device=device)
    got = F.kv_cache_read(wrap(cache), T(table), T(start), T(count), most, dtype=getattr(nb.DType, dtype))
    for name, x in zip(("k", "v"), got):
        x = x.to_torch()
        assert x.shape == (b, most, h, d) and x.dtype == getattr(torch, dtype)
        want = torch.zeros((b, most, h, d), dtype=torch.float64, device=device)
        for i in range(b):
            all_, there = values64(cache, name, table[i].tolist(), columns * n)
            rows = all_[int(start[i]):int(start[i]) + min(int(count[i]), most)]
            want[i, : rows.shape[0]] = rows
        # one rounding to the type, and one of the product in fp32
        assert ((x.double() - want).abs() <= (2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -23) * want.abs()).all()
    assert F.kv_cache_read(wrap(cache), T(table), T(start), T(count), 0)[0].to_torch().shape == (b, 0, h, d)


@pytest.mark.parametrize("device", DEVICES)
def test_a_prompt_in_pieces_and_whole(device):
    """The same tokens written at once, in pieces and one by one; attention then differs by the roundings of the codes alone."""
    g = gen(device, 14)
    b, t, h, d, n = 2, 70, 2, 64, 16
    k, v, q = (torch.randn((b, t, h, d), generator=g, device=device) for _ in range(3))
    table = T(new_table(g, device, b, 6, 12))
    scales, outs = [], []
    for pieces in ([70], [1, 15, 30, 24], [1] * 70):
        cache = F.init_kv_cache(12, h, d, n, device=T(k).device)
        done = 0
        for m in pieces:
            past = T(torch.full((b,), done, dtype=torch.int32, device=device))
            cache = F.kv_cache_write(cache, T(k[:, done:done + m]), T(v[:, done:done + m]), table, past)
            done += m
        assert int(past.to_torch()[0]) == 70 - pieces[-1]
        scales.append([cache["k_scale"].to_torch().clone(), cache["v_scale"].to_torch().clone()])
        outs.append(F.cached_attention(T(q), cache, table, T(torch.zeros(b, dtype=torch.int32, device=device))).to_torch())
    s = torch.einsum("bthd,bkhd->bhtk", q, k) / math.sqrt(d)
    s = s.masked_fill(torch.ones(t, t, dtype=torch.bool, device=device).triu(1), -math.inf)
    want = torch.einsum("bhtk,bkhd->bthd", torch.softmax(s, -1), v)
    for sc, o in zip(scales, outs):
        assert torch.equal(sc[0], scales[0][0]) and torch.equal(sc[1], scales[0][1])         # the largest magnitude, in whatever order
        # codes are off by up to a quarter of a step on average, more where they were rounded again: keys of about 1 at 127 steps to
        # their largest of about 4.5 move a score by some 0.02, and the values by 0.02 themselves
        assert (o - want).abs().max() < 0.2 and (o - want).square().mean().sqrt() < 0.02


@pytest.mark.parametrize("device", DEVICES)
def test_in_place_under_compile(device):
    """Compiled calls write into the cache they are given, call after call; what they return is that cache."""
    g = gen(device, 15)
    b, h, d, n = 2, 2, 64, 16
    table = T(new_table(g, device, b, 4, 8))
    step = nb.compile(lambda cache, k, v, q, table, past: (lambda c: (c, F.cached_attention(q, c, table, past)))(F.kv_cache_write(cache, k, v, table, past)))
    cache = F.init_kv_cache(8, h, d, n, device=table.device)
    plain = F.init_kv_cache(8, h, d, n, device=table.device)
    codes = cache["k"].to_torch()
    for i in range(20):
        k, v, q = (T(torch.randn((b, 1, h, d), generator=g, device=device).to(torch.bfloat16)) for _ in range(3))
        past = T(torch.tensor([i, i + 3], device=device, dtype=torch.int32))
        cache, got = step(cache, k, v, q, table, past)
        plain = F.kv_cache_write(plain, k, v, table, past)
        want = F.cached_attention(q, plain, table, past)
        assert cache["k"].to_torch() is codes or cache["k"].to_torch().data_ptr() == codes.data_ptr()
        assert torch.equal(got.to_torch(), want.to_torch())
        for name in cache:
            assert torch.equal(cache[name].to_torch(), plain[name].to_torch())
    assert step.stats.misses == 1
    if device == "cuda":
        assert step._taped is not None, step.tape_refused


@pytest.mark.gpu
def test_captured_steps_with_a_donated_cache():
    g = gen("cuda", 16)
    b, h, d, n = 2, 2, 128, 64
    table = T(new_table(g, "cuda", b, 4, 8))
    fn = lambda cache, k, v, q, table, past: (lambda c: (c, F.cached_attention(q, c, table, past)))(F.kv_cache_write(cache, k, v, table, past))  # noqa: E731
    step = nb.compile(fn, cuda_graph=True, donate_argnums=0)
    cache, plain = (F.init_kv_cache(8, h, d, n, device=table.device) for _ in range(2))
    for i in range(6):
        k, v, q = (T(torch.randn((b, 3, h, d), generator=g, device="cuda").to(torch.bfloat16)) for _ in range(3))
        past = T(torch.tensor([3 * i, 3 * i + 60], device="cuda", dtype=torch.int32))
        cache, got = step(cache, k, v, q, table, past)
        plain, want = fn(plain, k, v, q, table, past)
        assert torch.equal(got.to_torch(), want.to_torch())
    for name in cache:
        assert torch.equal(cache[name].to_torch(), plain[name].to_torch())


@pytest.mark.gpu
def test_on_another_stream():
    g = gen("cuda", 17)
    b, h, d, n = 3, 2, 128, 16
    cache = new_cache(g, "cuda", 60, h, n, d)
    table, past = T(new_table(g, "cuda", b, 20, 60)), T(torch.tensor([5, 100, 300], device="cuda", dtype=torch.int32))
    q = T(torch.randn((b, 2, 4, d), generator=g, device="cuda").to(torch.bfloat16))
    call = nb.compile(lambda q, c, table, past: F.cached_attention(q, c, table, past))
    want = [call(q, wrap(cache), table, past).to_torch() for _ in range(3)][-1]
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = [call(q, wrap(cache), table, past).to_torch() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(x, want) for x in got)


# ---------------------------------------------------------------- logits
def adjust64(z, history, length, prompt, repetition, presence, frequency, bias, allowed):
    z = z.double().clone()
    b, v = z.shape
    for i in range(b):
        if history is not None:
            n = history.shape[1] if length is None else min(max(int(length[i]), 0), history.shape[1])
            p = 0 if prompt is None else min(max(int(prompt[i]), 0), n)
            ids = [x for x in history[i, :n].tolist() if 0 <= x < v]
            made = [x for x in history[i, p:n].tolist() if 0 <= x < v]
            for x in set(ids):
                if repetition is not None:
                    z[i, x] = z[i, x] / repetition[i].double() if z[i, x] > 0 else z[i, x] * repetition[i].double()
            for x in set(made):
                if frequency is not None:
                    z[i, x] -= frequency[i].double() * made.count(x)
                if presence is not None:
                    z[i, x] -= presence[i].double()
        if bias is not None:
            z[i] += (bias if bias.dim() == 1 else bias[i]).double()
        if allowed is not None:
            for x in range(v):
                if not (int(allowed[i, x // 32]) >> (x % 32)) & 1:
                    z[i, x] = -math.inf
    return z


LOGITS = [
    # batch, vocab, longest, dtype, ids, with: history r p f b(1) B(b, v) a
    (1, 1, 1, "fp32", "int32", "rpfba"),
    (3, 33, 7, "bf16", "int64", "rpfba"),
    (2, 1000, 300, "fp32", "int32", "r"),
    (5, 4099, 50, "bf16", "int32", "pfBa"),
    (4, 8192, 1000, "bf16", "int64", "rpfba"),
    (3, 9001, 20, "fp32", "int64", "fB"),
    (2, 257, 0, "fp32", "int32", "rpf"),
    (2, 130, 0, "bf16", "int32", "a"),
    (2, 131, 0, "bf16", "int32", "b"),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", LOGITS)
def test_adjusting_logits(case, device):
    b, v, longest, dtype, whole, which = case
    g = gen(device, 21)
    dtype, whole = (torch.bfloat16 if dtype == "bf16" else torch.float32), getattr(torch, whole)
    z = (torch.randn((b, v), generator=g, device=device) * 3).to(dtype)
    if v > 2:
        z[0, 1], z[-1, 2] = math.inf, -math.inf
    u = lambda low, high, *shape: torch.rand(shape, generator=g, device=device) * (high - low) + low  # noqa: E731
    kw, history, length, prompt = {}, None, None, None
    if any(c in which for c in "rpf"):
        history = (u(0, 1, b, longest) ** 2 * (v + 2)).to(whole) - 1          # some are no token
        length = torch.randint(0, longest + 3, (b,), generator=g, device=device, dtype=whole)
        length[0] = longest
        prompt = torch.randint(0, longest + 1, (b,), generator=g, device=device, dtype=whole)
        for c, name, low, high in (("r", "repetition", 0.7, 1.5), ("p", "presence", -0.5, 1.0), ("f", "frequency", -0.2, 0.5)):
            if c in which:
                kw[name] = u(low, high, b)
    if "b" in which or "B" in which:
        kw["bias"] = u(-5, 5, v) if "b" in which else u(-5, 5, b, v)
    if "a" in which:
        kw["allowed"] = torch.randint(-(1 << 31), 1 << 31, (b, -(-v // 32)), generator=g, device=device, dtype=torch.int64).to(torch.int32)
        kw["allowed"][b - 1] = 0                                             # a row without any
    got = F.adjust_logits(T(z), *(None if x is None else T(x) for x in (history, length, prompt)), **{k: T(x) for k, x in kw.items()}).to_torch()
    want = adjust64(z, history, length, prompt, *(kw.get(k) for k in ("repetition", "presence", "frequency", "bias", "allowed")))
    assert got.dtype == dtype and torch.equal(got.double().isinf(), want.isinf()) and torch.equal(got[want.isinf()].double(), want[want.isinf()])
    fine = torch.isfinite(want)
    # four roundings in fp32 of numbers up to 20 + 0.5 * 1000, one to the type
    tol = 2.0 ** -21 * (want.abs() + 20 + (0.5 * longest if "f" in which else 0)) + (2.0 ** -8 * want.abs() if dtype == torch.bfloat16 else 0)
    assert ((got.double() - want).abs() <= tol)[fine].all()
    # rows that start off a boundary, and a call without any operand
    assert torch.equal(F.adjust_logits(T(z)).to_torch(), z)


# ---------------------------------------------------------------- refusals
def test_refusals():
    cache = F.init_kv_cache(4, 2, 64, 16)
    table = T(torch.zeros((2, 2), dtype=torch.int32))
    past = T(torch.zeros(2, dtype=torch.int32))
    x = lambda *s, dtype=torch.float32: T(torch.zeros(s, dtype=dtype))  # noqa: E731
    for bad in (dict(block_size=48), dict(block_size=8), dict(head_dim=80), dict(num_blocks=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            F.init_kv_cache(**{**dict(num_blocks=4, kv_heads=2, head_dim=64, block_size=16), **bad})
    q, kv = x(2, 3, 4, 64), x(2, 3, 2, 64)
    for error, call in [
        (TypeError, lambda: F.cached_attention(q, {"k": cache["k"]}, table, past)),
        (TypeError, lambda: F.cached_attention(x(2, 3, 4, 64, dtype=torch.float64), cache, table, past)),
        (TypeError, lambda: F.cached_attention(q.to_torch(), cache, table, past)),
        (ValueError, lambda: F.cached_attention(x(2, 3, 4, 128), cache, table, past)),
        (ValueError, lambda: F.cached_attention(x(2, 3, 3, 64), cache, table, past)),
        (ValueError, lambda: F.cached_attention(x(2, 3, 1, 64), cache, table, past)),
        (ValueError, lambda: F.cached_attention(x(3, 3, 4, 64), cache, table, past)),
        (ValueError, lambda: F.cached_attention(q, cache, table, T(torch.zeros(3, dtype=torch.int32)))),
        (TypeError, lambda: F.cached_attention(q, cache, table, T(torch.zeros(2)))),
        (TypeError, lambda: F.cached_attention(q, cache, T(torch.zeros((2, 2))), past)),
        (ValueError, lambda: F.cached_attention(q, cache, T(torch.zeros((2, 0), dtype=torch.int32)), past)),
        (ValueError, lambda: F.cached_attention(q, cache, table, past, scale=0.0)),
        (ValueError, lambda: F.cached_attention(q, cache, table, past, scale=math.nan)),
        (TypeError, lambda: F.cached_attention(q, dict(cache, k=x(4, 2, 16, 64)), table, past)),
        (ValueError, lambda: F.cached_attention(q, dict(cache, v_scale=x(4, 1)), table, past)),
        (ValueError, lambda: F.kv_cache_write(cache, kv, x(2, 2, 2, 64), table, past)),
        (TypeError, lambda: F.kv_cache_write(cache, kv, x(2, 3, 2, 64, dtype=torch.bfloat16), table, past)),
        (ValueError, lambda: F.kv_cache_write(cache, x(2, 3, 4, 64), x(2, 3, 4, 64), table, past)),
        (ValueError, lambda: F.kv_cache_read(cache, table, past, past, -1)),
        (TypeError, lambda: F.kv_cache_read(cache, table, past, past, 3, dtype=nb.DType.int8)),
        (ValueError, lambda: F.adjust_logits(x(2, 9), length=past)),
        (ValueError, lambda: F.adjust_logits(x(2, 9), repetition=x(2))),
        (ValueError, lambda: F.adjust_logits(x(2, 9), bias=x(8))),
        (ValueError, lambda: F.adjust_logits(x(2, 33), allowed=T(torch.zeros((2, 1), dtype=torch.int32)))),
        (TypeError, lambda: F.adjust_logits(x(2, 9, dtype=torch.int32))),
        (TypeError, lambda: F.adjust_logits(x(2, 9), T(torch.zeros((2, 3))))),
        (ValueError, lambda: nb.vmap(lambda y: F.cached_attention(y, cache, table, past))(x(5, 2, 3, 4, 64))),
    ]:
        with pytest.raises(error):
            call().to_torch() if not isinstance(call, dict) else None
    with pytest.raises(NotImplementedError):
        nb.grad(lambda y: nb.reduce_sum(nb.reshape(F.cached_attention(y, cache, table, past), (-1,))))(q)


# ---------------------------------------------------------------- together
def small_model(device, dtype):
    from nabla_b200.models import transformer as M

    cfg = M.TransformerConfig(n_layers=2, d_model=256, n_heads=4, d_ff=512, vocab=1000, max_seq=128, dtype=dtype)
    with nb.default_device(nb.Accelerator(0) if device == "cuda" else nb.CPU()):
        nb.seed(3)
        return cfg, M.init_params(cfg)


@pytest.mark.parametrize("device", DEVICES)
def test_a_decoder_over_the_cache_gives_the_logits_of_the_whole_sequence(device):
    from nabla_b200.models import generate as G
    from nabla_b200.models import transformer as M

    cfg, params = small_model(device, nb.DType.float32)
    g = gen("cpu", 31)
    tokens = torch.randint(0, cfg.vocab, (3, 60), generator=g).to(device)
    want = M.forward(params, T(tokens), cfg).to_torch()
    caches, table = G.init_caches(cfg, 3, 60, 16, device=params["tok_emb"].device)
    got, done = [], 0
    for n in (37, 1, 20, 1, 1):
        past = torch.full((3,), done, dtype=torch.int32, device=device)
        logits, caches = G.decode(params, T(tokens[:, done:done + n].contiguous()), caches, table, T(past), cfg)
        got.append(logits.to_torch())
        done += n
    got = torch.cat(got, 1)
    # keys and values in 127 steps to their block's largest (rms error of a step over sqrt(12), some 0.8 % of their rms): attention's part of the
    # residual stream is off by about that, and it is a small part of it
    assert (got - want).norm() < 0.02 * want.norm()
    # the same from a cache of another block size
    other, other_table = G.init_caches(cfg, 3, 60, 64, device=params["tok_emb"].device)
    count = T(torch.tensor([60, 59, 10], dtype=torch.int32, device=device))
    for a, b in zip(caches, other):
        G.move(a, table, count, 60, b, other_table)
    zero = T(torch.zeros(3, dtype=torch.int32, device=device))
    for a, b in zip(caches, other):
        for x, y in zip(F.kv_cache_read(a, table, zero, count, 60), F.kv_cache_read(b, other_table, zero, count, 60)):
            # half a step of either scale
            x, y = x.to_torch().float(), y.to_torch().float()
            assert (x - y).abs().max() <= 0.02 * x.abs().max()


@pytest.mark.parametrize("device", DEVICES)
def test_answers(device):
    from nabla_b200.models import generate as G

    cfg, params = small_model(device, nb.DType.float32 if device == "cpu" else nb.DType.bfloat16)
    prompts = [[5, 7, 9], [1], list(range(40))]
    plain = G.generate(params, prompts, cfg, 12, block_size=16)
    assert [len(a) for a in plain] == [12] * 3 and all(0 <= t < cfg.vocab for a in plain for t in a)
    assert G.generate(params, prompts, cfg, 12, block_size=16) == plain
    assert G.generate(params, prompts[:1], cfg, 1, block_size=16)[0] == plain[0][:1]
    # a token that has been said is never said again under a penalty that outweighs every logit
    once = G.generate(params, prompts, cfg, 12, block_size=16, presence=1e4)
    assert all(len(set(a)) == 12 for a in once)
    # and only what a grammar allows
    words = torch.zeros((3, -(-cfg.vocab // 32)), dtype=torch.int32)
    words[:, 3] = 0b1010
    allowed = G.generate(params, prompts, cfg, 12, block_size=16, allowed=T(words.to(device)))
    assert all(t in (97, 99) for a in allowed for t in a)
    with pytest.raises(ValueError):
        G.generate(params, [[1] * 120], cfg, 12)
    with pytest.raises(ValueError):
        G.generate(params, [[]], cfg, 12)


def test_heads_split_over_a_mesh():
    """Query heads and the cache's heads split over the same axis of a simulated mesh: every device does its own."""
    g = gen("cpu", 33)
    b, t, hq, h, d, n = 2, 3, 8, 4, 64, 16
    cache = wrap(new_cache(g, "cpu", 8, h, n, d))
    table, past = T(new_table(g, "cpu", b, 3, 8)), T(torch.tensor([5, 20], dtype=torch.int32))
    q, k, v = (torch.randn((b, t, x, d), generator=g) for x in (hq, h, h))
    mesh = nb.DeviceMesh("m", (2,), ("tp",))
    split = lambda x, at: T(x).shard(mesh, tuple("tp" if i == at else None for i in range(x.dim())))  # noqa: E731
    whole = F.kv_cache_write(cache, T(k), T(v), table, past, inplace=False)
    want = F.cached_attention(T(q), whole, table, past).to_torch()
    parts = {name: split(x.to_torch().clone(), 1) for name, x in cache.items()}
    parts = F.kv_cache_write(parts, split(k, 2), split(v, 2), table, past, inplace=False)
    got = F.cached_attention(split(q, 2), parts, table, past)
    assert [s.axes for s in got.sharding.dim_specs] == [[], [], ["tp"], []]
    assert torch.allclose(torch.from_numpy(got.to_numpy()), want, atol=1e-5)
    back = F.kv_cache_read(parts, table, T(torch.zeros(2, dtype=torch.int32)), T(torch.tensor([8, 23], dtype=torch.int32)), 30)
    for x, y in zip(back, F.kv_cache_read(whole, table, T(torch.zeros(2, dtype=torch.int32)), T(torch.tensor([8, 23], dtype=torch.int32)), 30)):
        assert torch.equal(torch.from_numpy(nb.cast(x, nb.DType.float32).to_numpy()), y.to_torch().float())
