"""Attention over a prefix that a batch shares, against its definition in 64 bits and against ``cached_attention`` over tables that hold the prefix.

Tolerances are those of ``cached_attention`` (``test_serving.py``, where they are derived): the result rounded to bf16, weights rounded to 11 bits on the
way to the products, or to 22 in fp32 calls. Joining two or more parts adds a few roundings of fp32 of convex combinations, 2^-22 of the largest value,
which the terms for the weights (2^-10, 2^-18 of it) hold with room to spare. A part's weight is the binary logarithm of a sum, a number as large as the
largest score s / ln 2, and is off by two units of it (2^-23) and by 2^-21; shares move by as much, values by no more than twice that. ``oracle`` adds 2^-20 of
(|s| + 8) for it.
"""
from __future__ import annotations

import math

import pytest
import torch

import nabla_b200 as nb
from nabla_b200.nn import functional as F
from test_serving import T, attend64, gen, new_cache, wrap

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def oracle(q, cache, prefix_table, prefix, table, past, count, causal, scale):
    """A sequence's blocks behind those of the prefix: keys are gathered one by one."""
    b, t, hq, d = q.shape
    blocks, h, n, _ = cache["k"].shape
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device=q.device)
    bound = torch.zeros((b, t, hq, 1), dtype=torch.float64, device=q.device)

    def keys_of(ids, keys):
        k, v, there = [], [], []
        for c, id_ in enumerate(ids):
            m = min(n, keys - c * n)
            if m <= 0:
                break
            ok = 0 <= id_ < blocks
            there.append(torch.full((m,), ok, device=q.device))
            for name, to in (("k", k), ("v", v)):
                x = cache[name][id_].double() * cache[name + "_scale"][id_].double()[:, None, None] if ok else torch.zeros((h, n, d), dtype=torch.float64, device=q.device)
                to.append(x.transpose(0, 1)[:m])
        if not k:
            return torch.zeros((0, h, d), dtype=torch.float64, device=q.device), torch.zeros((0, h, d), dtype=torch.float64, device=q.device), torch.zeros(0, dtype=torch.bool, device=q.device)
        return torch.cat(k), torch.cat(v), torch.cat(there)

    prefix = min(max(prefix, 0), len(prefix_table) * n)
    kp, vp, tp = keys_of(prefix_table.tolist(), prefix)
    for i in range(b):
        p = min(max(int(past[i]), 0), table.shape[1] * n)
        c = t if count is None else min(max(int(count[i]), 0), t)
        if c == 0:
            continue
        ko, vo, to = keys_of(table[i].tolist(), min(p + c, table.shape[1] * n))
        k, v = torch.cat([kp, ko]), torch.cat([vp, vo])
        at = torch.arange(len(ko), device=q.device)
        last = p + torch.arange(c, device=q.device) if causal else torch.full((c,), p + c - 1, device=q.device)
        seen = torch.cat([tp.expand(c, -1), (at[None] <= last[:, None]) & to[None]], 1)
        any_ = seen.any(0)[:, None]
        for x in range(hq):
            kk, vv = torch.where(any_, k[:, x // (hq // h)], 0.0), torch.where(any_, v[:, x // (hq // h)], 0.0)
            s = torch.where(seen, q[i, :c, x].double() @ kk.T * scale, -math.inf)
            top = s.amax(-1, keepdim=True) if s.shape[1] else s.new_full((c, 1), -math.inf)
            e = torch.where(seen, torch.exp(s - torch.where(torch.isinf(top), 0.0, top)), 0.0)
            out[i, :c, x] = e / e.sum(-1, keepdim=True).clamp(min=1e-300) @ vv
            if len(k):
                # score: D products of q and k summed in fp32 (and the offset of the codes); and the logarithm of a part's sum, twice
                size = q[i, :c, x].double().abs().amax(-1) * kk.abs().max() * scale
                far = torch.where(seen, s, 0.0).abs().amax(-1)
                bound[i, :c, x, 0] = (size * 2.0 ** -22 * d * 9 + 2.0 ** -20 * (far + 8)) * vv.abs().max()
    return out, bound


def check(got, want, bound, cache):
    vmax = 127 * cache["v_scale"].nan_to_num(0).max().item()
    tol = (2.0 ** -8 * want.abs() + 2.0 ** -10 * vmax if got.dtype == torch.bfloat16 else 2.0 ** -18 * vmax) + bound
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), f"off by {(off - tol).max().item():.3g} more than allowed ({off.max().item():.3g})"
    assert (got[(want == 0).all(-1)] == 0).all()


CASES = [
    # batch, new, heads, kv heads, head_dim, block, prefix, past, count, dtype, causal, table dtype
    (1, 1, 1, 1, 64, 16, 1, [0], None, "bf16", True, "int32"),
    (4, 1, 16, 16, 128, 64, 100, [0, 1, 63, 64], [1, 0, 1, 1], "bf16", True, "int32"),
    (3, 1, 8, 2, 128, 16, 33, [0, 15, 16], [1, 1, 1], "bf16", True, "int64"),
    (9, 1, 16, 4, 64, 32, 500, [31, 32, 33, 200, 0, 1, 2, 3, 4], None, "bf16", True, "int32"),          # 36 rows over the prefix
    (2, 1, 8, 1, 64, 128, 129, [127, 300], None, "fp32", True, "int32"),
    (5, 5, 6, 2, 64, 16, 77, [0, 7, 100, 11, 250], [5, 5, 0, 3, 1], "bf16", True, "int32"),
    (3, 7, 4, 4, 128, 32, 64, [9, 200, 0], [7, 2, 7], "fp32", True, "int64"),
    (2, 5, 8, 1, 128, 64, 640, [1, 100], None, "bf16", False, "int32"),
    (3, 33, 4, 2, 64, 16, 250, [0, 77, 5], [33, 20, 0], "bf16", True, "int32"),
    (2, 130, 3, 1, 128, 64, 0, [0, 3], None, "bf16", True, "int32"),                                    # no prefix
    (2, 257, 4, 1, 64, 32, 333, [0, 33], [257, 129], "bf16", True, "int32"),
    (70, 1, 8, 2, 128, 64, 1000, [i * 7 % 90 for i in range(70)], None, "bf16", True, "int32"),
    (40, 2, 4, 2, 128, 16, 300, [i * 5 % 40 for i in range(40)], None, "fp32", True, "int32"),
]


def make(case, device, seed=3):
    b, t, hq, h, d, n, prefix, past, count, dtype, causal, whole = case
    g = gen(device, seed)
    dtype, whole = (torch.bfloat16 if dtype == "bf16" else torch.float32), getattr(torch, whole)
    shared, columns = prefix // n + 2, (max(past) + t + n - 1) // n + 2
    blocks = shared + b * columns + 1
    cache = new_cache(g, device, blocks, h, n, d)
    ids = torch.randperm(blocks - 1, generator=g, device=device).to(whole)
    prefix_table, table = ids[:shared].clone(), ids[shared:shared + b * columns].view(b, columns).clone()
    # what lies behind the prefix and behind a sequence's tokens is never looked at: no block, or one whose scales are NaN
    cache["k_scale"][blocks - 1] = cache["v_scale"][blocks - 1] = math.nan
    prefix_table[-(-prefix // n):] = -1
    prefix_table[-1] = blocks - 1
    for i in range(b):
        used = -(-(past[i] + (t if count is None else count[i])) // n)
        table[i, used:] = 1 << 30
        if used + 1 < columns:
            table[i, used + 1] = blocks - 1
    q = torch.randn((b, t, hq, d), generator=g, device=device).to(dtype)
    put = lambda x: None if x is None else torch.tensor(x, device=device, dtype=whole)  # noqa: E731
    return q, cache, prefix_table, put([prefix]), table, put(past), put(count)


def call(q, cache, prefix_table, prefix, table, past, count=None, **kw):
    return F.shared_prefix_attention(T(q), wrap(cache), T(prefix_table), T(prefix), T(table), T(past), None if count is None else T(count), **kw).to_torch()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", CASES)
def test_attention_over_a_shared_prefix(case, device):
    args = make(case, device)
    q, cache, prefix_table, prefix, table, past, count = args
    got = call(*args, causal=case[10])
    want, bound = oracle(q, cache, prefix_table, int(prefix), table, past.tolist(), None if count is None else count.tolist(), case[10], q.shape[-1] ** -0.5)
    assert got.dtype == q.dtype and got.shape == q.shape
    check(got, want, bound, cache)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new,dtype", [(1, torch.bfloat16), (40, torch.bfloat16), (3, torch.float32)])
def test_as_the_whole_text(new, dtype, device):
    """A prefix of whole blocks gives what ``cached_attention`` gives over tables that begin with it."""
    g = gen(device, 11)
    b, hq, h, d, n, shared, columns = 6, 8, 2, 64, 16, 9, 8
    cache = new_cache(g, device, 80, h, n, d)
    ids = torch.randperm(80, generator=g, device=device).to(torch.int32)
    prefix_table, table = ids[:shared], ids[shared:shared + b * columns].view(b, columns)
    past = torch.randint(0, columns * n - new, (b,), generator=g, device=device, dtype=torch.int32)
    q = torch.randn((b, new, hq, d), generator=g, device=device).to(dtype)
    got = call(q, cache, prefix_table, torch.tensor([shared * n], device=device), table, past)
    whole = torch.cat([prefix_table.expand(b, -1), table], 1)
    want, bound = attend64(q, cache, whole, (past + shared * n).tolist(), None, True, d ** -0.5)
    check(got, want, bound, cache)
    other = F.cached_attention(T(q), wrap(cache), T(whole), T(past + shared * n)).to_torch()
    vmax = 127 * 0.042
    assert (got.float() - other.float()).abs().max() <= (2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -16) * vmax       # two roundings of each


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new", [1, 6, 150])
def test_missing_blocks_far_scales_and_undefined_ones(new, device):
    """Holes in the prefix and in sequences; scales from 2^-100 to 2^40; a NaN block of the prefix reaches every live row, one of a sequence its own."""
    g = gen(device, 5)
    b, hq, h, d, n, shared, columns = 4, 4, 2, 128, 16, 30, 20
    cache = new_cache(g, device, 140, h, n, d)
    cache["v_scale"][::3] = 2.0 ** -100
    cache["v_scale"][1::7] = 2.0 ** 40
    cache["k_scale"][::5] = 2.0 ** -100
    ids = torch.randperm(139, generator=g, device=device).to(torch.int32)
    prefix_table, table = ids[:shared].clone(), ids[shared:shared + b * columns].view(b, columns).clone()
    prefix_table[3:5] = -1
    prefix_table[20] = 140
    table[0, 1] = -1
    table[2, :] = -5
    prefix = torch.tensor([shared * n - 7], device=device)
    past = torch.tensor([100, 37, 120, 30], device=device, dtype=torch.int32)
    count = torch.tensor([new, new, new, 0], device=device, dtype=torch.int32)
    q = torch.randn((b, new, hq, d), generator=g, device=device).to(torch.bfloat16)
    args = [q, cache, prefix_table, prefix, table, past, count]
    want, bound = oracle(q, cache, prefix_table, int(prefix), table, past.tolist(), count.tolist(), True, d ** -0.5)
    plain = call(*args)
    check(plain, want, bound, cache)
    assert (plain[3] == 0).all()
    cache["v_scale"][139, 0] = math.nan           # of one head
    table[1, 0] = 139
    got = call(*args)
    assert got[1, :, :2].isnan().all() and torch.equal(got[1, :, 2:].isnan(), torch.zeros_like(got[1, :, 2:], dtype=torch.bool)) and torch.equal(got[0], plain[0]) \
        and torch.equal(got[2:], plain[2:])
    table[1, 0] = 5
    prefix_table[7] = 139
    got = call(*args)
    assert got[:3, :, :2].isnan().all() and torch.isfinite(got[:3, :, 2:]).all() and (got[3] == 0).all()
    # no keys at all
    empty = call(q, cache, torch.full_like(prefix_table, -1), prefix, torch.full_like(table, 999), past, count)
    assert (empty == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,new,hq,h,n,prefix,longest,dtype", [
    (64, 1, 16, 4, 64, 8001, 900, "bf16"), (16, 1, 16, 2, 128, 20001, 700, "bf16"), (4, 1, 16, 16, 64, 1000, 200, "bf16"), (200, 1, 8, 8, 64, 3000, 60, "bf16"),
    (1030, 1, 4, 2, 64, 500, 90, "bf16"), (3, 1, 4, 1, 64, 9000, 30, "bf16"), (8, 5, 12, 4, 16, 1501, 300, "fp32"), (50, 1, 8, 2, 64, 3000, 500, "fp32"),
    (12, 64, 8, 2, 64, 700, 100, "bf16"), (2, 700, 8, 2, 64, 1111, 50, "bf16"), (5, 40, 4, 2, 32, 900, 2000, "bf16"), (3, 50, 8, 1, 64, 600, 80, "fp32"),
    # both sides of where one kernel walks over the prefix and the own keys: rows of a sequence that fill tiles of 128 badly and well, few tiles in all
    (9, 70, 8, 2, 64, 1500, 300, "bf16"), (24, 33, 16, 4, 16, 777, 20, "bf16"), (1, 300, 4, 2, 32, 5000, 10, "bf16"), (2, 520, 4, 4, 64, 129, 0, "bf16"),
])
def test_ragged_batches(b, new, hq, h, n, prefix, longest, dtype, d):
    """Idle sequences and short counts; scratch that holds garbage; the same bits every time, in a graph too."""
    g = gen("cuda", 41)
    dtype = torch.bfloat16 if dtype == "bf16" else torch.float32
    shared, columns = -(-prefix // n), -(-(longest + new) // n) + 1
    cache = new_cache(g, "cuda", shared + b * columns, h, n, d)
    ids = torch.randperm(shared + b * columns, generator=g, device="cuda").to(torch.int32)
    past = torch.randint(0, longest + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    count = torch.randint(0, new + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    count[0], past[0], past[-1] = new, longest, 0
    qkv = torch.randn((b, new, hq, 2, d), generator=g, device="cuda").to(dtype)
    args = [qkv[:, :, :, 1], cache, ids[:shared], torch.tensor([prefix], device="cuda"), ids[shared:].view(b, columns), past, count]
    garbage = torch.full((64 << 20,), math.nan, device="cuda")
    del garbage
    got = call(*args)
    some = slice(0, b, max(1, b // 12))           # of many sequences, some
    want, bound = oracle(args[0][some], cache, ids[:shared], prefix, args[4][some], past[some].tolist(), count[some].tolist(), True, d ** -0.5)
    check(got[some], want, bound, cache)
    assert (got[count == 0] == 0).all()
    f = nb.compile(lambda q, c, *x: F.shared_prefix_attention(q, c, *x), cuda_graph=True)
    tensors = [T(args[0]), wrap(cache), *(T(x) for x in args[2:])]
    for _ in range(3):
        assert torch.equal(f(*tensors).to_torch(), got) and torch.equal(call(*args), got)


@pytest.mark.gpu
def test_layouts_of_queries_and_streams():
    """Queries whose batch is not the outer stride, broadcast over the batch, off boundaries; calls on two streams at once."""
    case = (6, 3, 8, 2, 64, 16, 200, [0, 5, 9, 30, 2, 1], None, "bf16", True, "int32")
    q, *rest = make(case, "cuda")
    want = call(q, *rest)
    assert torch.equal(call(q.transpose(0, 1).contiguous().transpose(0, 1), *rest), want)
    odd = torch.zeros((q.numel() + 5,), device="cuda", dtype=q.dtype)
    odd[3:3 + q.numel()] = q.flatten()
    assert torch.equal(call(odd[3:3 + q.numel()].view(q.shape), *rest), want)
    same = q[:1].expand(6, -1, -1, -1)
    assert torch.equal(call(same, *rest), call(same.contiguous(), *rest))
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            streams[i % 2].wait_stream(torch.cuda.default_stream())
            results.append(call(q, *rest))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)


@pytest.mark.parametrize("device", DEVICES)
def test_written_and_read_in_order(device):
    """A step that writes and attends, compiled: the prefix is written by one call, sequences behind it by others."""
    g = gen(device, 2)
    b, h, d, n, prefix = 3, 2, 64, 16, 21
    kv = torch.randn((2, 1, prefix, h, d), generator=g, device=device)
    new = torch.randn((3, b, 4, h, d), generator=g, device=device)
    prefix_table = torch.tensor([0, 1], device=device, dtype=torch.int32)
    table = torch.arange(2, 2 + b, device=device, dtype=torch.int32)[:, None]
    zero = torch.zeros(b, device=device, dtype=torch.int32)
    length = torch.tensor([prefix], device=device, dtype=torch.int32)

    def program(cache, k, v, q, kp, vp):
        cache = F.kv_cache_write(cache, kp, vp, T(prefix_table[None]), T(zero[:1]))
        cache = F.kv_cache_write(cache, k, v, T(table), T(zero))
        return F.shared_prefix_attention(q, cache, T(prefix_table), T(length), T(table), T(zero)), cache

    def fresh():
        c = F.init_kv_cache(5, h, d, n, device=T(zero)._impl.device)
        return {k: T(t.to_torch().to(device)) for k, t in c.items()}

    args = [T(x) for x in (new[0], new[1], new[2], kv[0], kv[1])]
    out, cache = program(fresh(), *args)
    plain = {k: t.to_torch() for k, t in cache.items()}
    want, bound = oracle(new[2], plain, prefix_table, prefix, table, [0] * b, None, True, d ** -0.5)
    check(out.to_torch(), want, bound, plain)
    step = nb.compile(program)
    for _ in range(3):
        assert torch.equal(step(fresh(), *args)[0].to_torch(), out.to_torch())


def test_over_a_mesh(mesh_2x4):
    case = (3, 2, 8, 4, 64, 16, 40, [0, 5, 9], None, "fp32", True, "int32")
    q, cache, *rest = make(case, "cpu")
    want = call(q, cache, *rest)
    heads = {"k": (None, "tp", None, None), "v": (None, "tp", None, None), "k_scale": (None, "tp"), "v_scale": (None, "tp")}
    split = {k: T(v).shard(mesh_2x4, heads[k]) for k, v in cache.items()}
    place = lambda x: T(x).shard(mesh_2x4, (None,) * x.dim())  # noqa: E731
    got = F.shared_prefix_attention(T(q).shard(mesh_2x4, (None, None, "tp", None)), split, *(place(x) for x in rest if x is not None))
    assert (torch.from_numpy(got.to_numpy()) - want).abs().max() <= 2.0 ** -20 * want.abs().max()


@pytest.mark.parametrize("hq,h,axis,fine", [(12, 3, "dp", False), (8, 2, "tp", False), (12, 6, "tp", False), (6, 3, "dp", False),
                                            (8, 4, "tp", True), (6, 3, "tp", True), (5, 5, "tp", True), (8, 1, "tp", True), (12, 6, "dp", True)])
def test_groups_of_heads_over_a_mesh(hq, h, axis, fine, mesh_2x4):
    """A split that would give a device query heads without the heads of the cache that they share is refused, with a prefix and without."""
    q, cache, prefix_table, prefix, table, past, count = make((3, 2, hq, h, 64, 16, 40, [0, 5, 9], None, "fp32", True, "int32"), "cpu")
    assert count is None
    for q_axis, c_axis in ((axis, axis), (axis, None), (None, axis)):
        split = {k: T(v).shard(mesh_2x4, (None, c_axis, None, None)[:v.dim()]) for k, v in cache.items()}
        sq = T(q).shard(mesh_2x4, (None, None, q_axis, None))
        for f, rest in ((F.shared_prefix_attention, (prefix_table, prefix, table, past)), (F.cached_attention, (table, past))):
            if not fine:
                with pytest.raises(ValueError, match="split over"):
                    f(sq, split, *(T(x) for x in rest))
                continue
            want = f(T(q), {k: T(v) for k, v in cache.items()}, *(T(x) for x in rest)).to_torch()
            got = torch.from_numpy(f(sq, split, *(T(x) for x in rest)).to_numpy())
            assert (got - want).abs().max() <= 2.0 ** -20 * want.abs().max()       # as above: the same fp32 sums head by head


def test_refusals():
    cache = F.init_kv_cache(8, 2, 64, 16)
    q = T(torch.zeros(3, 1, 4, 64))
    whole = lambda *s: T(torch.zeros(s, dtype=torch.int32))  # noqa: E731
    ok = [q, cache, whole(2), whole(1), whole(3, 2), whole(3)]
    assert F.shared_prefix_attention(*ok).shape == q.shape
    for error, at, x in [
        (TypeError, 0, torch.zeros(3, 1, 4, 64)), (ValueError, 0, T(torch.zeros(3, 1, 3, 64))), (ValueError, 0, T(torch.zeros(3, 1, 4, 128))),
        (TypeError, 0, T(torch.zeros(3, 1, 4, 64, dtype=torch.float64))), (TypeError, 1, {}), (ValueError, 2, whole(1, 2)), (TypeError, 2, T(torch.zeros(2))),
        (ValueError, 2, whole(0)), (ValueError, 3, whole(2)), (ValueError, 3, T(torch.zeros((), dtype=torch.int32))), (TypeError, 3, 5), (TypeError, 3, T(torch.zeros(1))),
        (ValueError, 4, whole(2, 2)), (ValueError, 4, whole(3, 0)), (ValueError, 5, whole(4)), (TypeError, 5, T(torch.zeros(3))),
    ]:
        with pytest.raises(error):
            F.shared_prefix_attention(*ok[:at], x, *ok[at + 1:])
    for kw in ({"count": whole(2)}, {"scale": 0.0}, {"scale": math.inf}):
        with pytest.raises(ValueError):
            F.shared_prefix_attention(*ok, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("b,hq,h,columns,dtype", [(5, 8, 2, 4, "bf16"), (40, 16, 4, 20, "bf16"), (6, 4, 2, 40, "bf16"), (64, 16, 4, 16, "fp32"), (3, 4, 4, 300, "bf16")])
def test_steps_in_a_row_see_what_was_just_written(b, hq, h, columns, dtype):
    """Tokens are written and attended to, one kernel directly behind the other, at the same addresses in every step: lengths and tables grow in place. Each
    step's result is that of the same step alone."""
    g = gen("cuda", 17)
    n, d, shared, steps = 16, 64, 40, 12
    dtype = torch.bfloat16 if dtype == "bf16" else torch.float32
    blocks = shared + b * columns
    cache0 = new_cache(g, "cuda", blocks, h, n, d)
    ids = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    prefix_table, all_table = ids[:shared].clone(), ids[shared:].view(b, columns)
    prefix = torch.tensor([shared * n - 3], device="cuda")
    start = torch.randint(0, columns * n - steps, (b,), generator=g, device="cuda", dtype=torch.int32)
    kv = torch.randn((steps, 3, b, 1, hq, d), generator=g, device="cuda").to(dtype)

    def run(wait):
        cache = {k: v.clone() for k, v in cache0.items()}
        past, table, q = start.clone(), torch.full_like(all_table, -1), torch.empty_like(kv[0, 0])
        length = torch.zeros_like(prefix)
        call = nb.compile(lambda c, k, v, q, t, p, pt, pl: (lambda c: (F.shared_prefix_attention(q, c, pt, pl, t, p), c))(F.kv_cache_write(c, k, v, t, p)))
        c, tensors, out = wrap(cache), [T(x) for x in (q, table, past, prefix_table, length)], []
        for i in range(steps):
            # everything that the call reads is written directly in front of it
            q.copy_(kv[i, 0])
            length.copy_(prefix - i)
            table.copy_(torch.where(torch.arange(columns, device="cuda") <= past[:, None] // n, all_table, -1))
            if wait:
                torch.cuda.synchronize()
            o, c = call(c, T(kv[i, 1][:, :, :h]), T(kv[i, 2][:, :, :h]), *tensors)
            if wait:
                torch.cuda.synchronize()
            out.append(o.to_torch().clone())
            past += 1
        return out

    want = run(True)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(run(False), want))


@pytest.mark.gpu
@pytest.mark.parametrize("case", [CASES[1], CASES[3], CASES[10], CASES[12]])
def test_a_compiled_call_is_written_down(case):
    from nabla_b200.transforms import tape

    if tape.module() is None:
        pytest.skip("libnb_replay.so is not built here")
    q, cache, *rest = make(case, "cuda")
    rest = [x for x in rest if x is not None]
    f = nb.compile(lambda q, c, *x: F.shared_prefix_attention(q, c, *x))
    for _ in range(4):
        f(T(q), wrap(cache), *(T(x) for x in rest))
    assert f._taped is not None and bool(f._taped[0]), f.tape_refused


_CHECKED = """
import torch
import nabla_b200 as nb
from nabla_b200 import native
from nabla_b200.nn import functional as F
T = nb.Tensor.from_torch
g = torch.Generator("cuda").manual_seed(0)
rand = lambda *s: torch.randn(s, generator=g, device="cuda")
for d, n in ((64, 16), (128, 64)):
    for b, new, hq, h, prefix, dtype in ((3, 1, 8, 2, 37, torch.bfloat16), (70, 1, 8, 2, 300, torch.bfloat16), (5, 40, 4, 2, 200, torch.bfloat16), (4, 3, 4, 4, 50, torch.float32)):
        cache = F.init_kv_cache(64 + b * 4, h, d, n, device=nb.Accelerator(0))
        shared = -(-prefix // n) + 1
        ids = torch.randperm(64 + b * 4, generator=g, device="cuda").to(torch.int32)
        table = ids[shared:shared + b * 4].view(b, 4).clone()
        past = torch.randint(0, 4 * n, (b,), generator=g, device="cuda", dtype=torch.int32)
        count = torch.randint(0, new + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        table[0, 3], table[-1, 0] = -1, 1 << 30
        for length in (prefix, 0, 1 << 40, -5):
            F.shared_prefix_attention(T(rand(b, new, hq, d).to(dtype)), cache, T(ids[:shared]), T(torch.tensor([length], device="cuda")), T(table), T(past), T(count)).to_torch()
for v, b in ((1, 2), (333, 7), (40001, 3), (40001, 300)):
    for dtype in (torch.bfloat16, torch.float32):
        z, u = rand(b, v).to(dtype), torch.rand(b, generator=g, device="cuda")
        k, p = torch.randint(-1, v + 2, (b,), generator=g, device="cuda"), torch.rand(b, generator=g, device="cuda")
        for kw in ({}, {"top_k": T(k)}, {"top_p": T(p)}, {"top_k": T(k), "top_p": T(p), "min_p": T(p * 0.1), "temperature": T(p * 2)}):
            for x in (z, z * 0, z * 1e-3):
                F.sample_tokens(T(x), T(u), **kw).to_torch()
for d, rotary, b, t in ((64, 32, 2, 5), (80, 80, 3, 1), (256, 256, 1, 700), (128, 128, 5, 999)):
    q, k, pos = rand(b, t, 5, d).bfloat16(), rand(b, t, 3, d).bfloat16(), torch.arange(t, device="cuda")
    gain = rand(d).bfloat16()
    y, pull = nb.vjp(lambda q, k, c: F.norm_rotary(q, k, T(pos), c, c, rotary_dim=rotary), T(q), T(k), T(gain), create_graph=False)
    [x.to_torch() for x in pull((T(q), T(k)))]
torch.cuda.synchronize()
native.check_status()
native.debug_check()
for name, units in (("libnb_answers.so", 3), ("libnb_heads.so", 1)):
    native.debug_selftest(name, 12, 8, 64, 16)
    print("FAILED CHECKS", name, native.debug_report()["count"] == units)
"""


@pytest.mark.gpu
def test_the_checked_build_finds_every_access_in_bounds():
    import os
    import subprocess
    import sys
    from pathlib import Path

    from nabla_b200.csrc import build

    build.build_all(debug=True)
    root = Path(__file__).resolve().parent.parent
    env = dict(os.environ, NABLA_B200_DEBUG_KERNELS="1", PYTHONPATH=str(root))
    r = subprocess.run([sys.executable, "-c", _CHECKED], capture_output=True, text=True, env=env, timeout=600, cwd=root)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    assert r.stdout.count("True") == 2
