"""Edges of the serving operations: where their loads lie, what starts off a boundary, what is hidden or comes in an unusual order.

The definitions in 64 bits are those of ``test_serving.py``.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import nabla_b200 as nb
from nabla_b200.nn import functional as F

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def T(x):
    return nb.Tensor.from_torch(x)


def gen(device, seed):
    return torch.Generator(device).manual_seed(seed)


# ---------------------------------------------------------------- where loads lie
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_loads_of_few_rows_stay_in_their_block(block):
    """A range of keys may be empty (more ranges than keys, tiles that see less than their line has): its loads lie in the block all the same."""
    from nabla_b200.native import load

    ask = load("libnb_serving.so").nb_cached_attention_last_row
    for keys in [*range(0, 300), 511, 512, 513, 1499, 1500, 4095, 120001]:
        for splits in (1, 2, 4, 8):                              # a cluster's ranges
            per = -(-keys // (32 * splits)) * 32
            for s in range(splits):
                assert ask(keys, s * per, per, block) < block, (keys, splits, s)
        for unit in (0, 1, 2, 3, 11, 937, 1 << 20):                # a line's pieces
            for pieces in (1, 3):
                assert ask(keys, unit * 128, pieces * 128, block) < block, (keys, unit, pieces)


_CHECKED = r"""
import torch
import nabla_b200 as nb
from nabla_b200 import native
from nabla_b200.nn import functional as F
assert native.DEBUG_KERNELS
T = nb.Tensor.from_torch
g = torch.Generator("cuda").manual_seed(1)
rand = lambda *s: torch.randn(s, generator=g, device="cuda")
for n in (16, 32, 64, 128):
    for d, dtype in ((64, torch.float32), (128, torch.bfloat16)):
        for new in (1, 3, 40, 200):
            # few tokens in a table with room for many, in the cache's last blocks
            b, h, used, columns = 3, 2, 512 // n, 4096 // n
            cache = F.init_kv_cache(b * used, h, d, n, device=nb.Accelerator(0))
            table = torch.full((b, columns), -1, dtype=torch.int32, device="cuda")
            table[:, :used] = torch.arange(b * used, device="cuda").flip(0).view(b, used)
            past, count = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 37, 5], [new, new - 1, min(new, 1)]))
            x = [T(rand(b, new, h, d).to(dtype)) for _ in range(2)]
            cache = F.kv_cache_write(cache, *x, T(table), T(past), T(count))
            for group in (1, 8):
                F.cached_attention(T(rand(b, new, h * group, d).to(dtype)), cache, T(table), T(past), T(count)).to_torch()
            F.kv_cache_read(cache, T(table), T(past * 0), T(past + count), 250)[0].to_torch()
torch.cuda.synchronize()
native.check_status()
native.debug_check()
native.debug_selftest("libnb_serving.so", 12, 8, 64, 16)
print("FAILED CHECKS", native.debug_report()["count"])
"""


@pytest.mark.gpu
def test_the_checked_build_finds_every_load_in_the_cache():
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
    assert "FAILED CHECKS 4" in r.stdout           # the self-test's, one for each unit of the library


# ---------------------------------------------------------------- logits that start off a boundary
def off_boundary(x, by):
    """A dense copy of x that starts ``by`` elements behind a boundary."""
    return torch.zeros(x.numel() + by, device=x.device, dtype=x.dtype)[by:].view(x.shape).copy_(x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_kernel_of_logits_is_given_rows_that_start_alike(dtype, monkeypatch):
    """It writes vectors where it reads vectors, so both addresses have to be the same distance from a boundary of 16 bytes."""
    from nabla_b200.native import load, serving

    given = []

    class Library:
        def nb_adjust_logits(self, x, out, *more):
            given.append((x.value, out.value))
            return 0

    monkeypatch.setattr(serving, "_L", Library)
    monkeypatch.setattr(serving, "stream_ptr", lambda: None)
    for by in range(9):
        for rows in (1, 3):
            serving.adjust_logits(off_boundary(torch.zeros(rows, 33, dtype=dtype), by), *[None] * 8)
    assert len(given) == 18 and all((x - out) % 16 == 0 for x, out in given)
    # and the entry refuses others
    entry = load("libnb_serving.so").nb_adjust_logits
    import ctypes

    entry.argtypes = [ctypes.c_void_p] * 9 + [ctypes.c_longlong, ctypes.c_void_p] + [ctypes.c_int] * 6 + [ctypes.c_void_p]
    for x, out in ((1 << 20 | 2, 1 << 21), (1 << 20, 1 << 21 | 8)):
        assert entry(x, out, *[None] * 7, 0, None, 0, 1, 33, 0, 0, int(dtype == torch.float32), None) == -1


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 33), (3, 4099), (5, 8192)])
def test_logits_that_start_off_a_boundary(rows, vocab, dtype, device):
    """The last token's logits of a prompt, as a view: the same as from a tensor of their own, to the last bit."""
    g = gen(device, 51)
    z = (torch.randn((rows, vocab), generator=g, device=device) * 3).to(dtype)
    history = torch.randint(0, vocab, (rows, 50), generator=g, device=device, dtype=torch.int32)
    bias = torch.randn(vocab, generator=g, device=device)
    words = torch.randint(-(1 << 31), 1 << 31, (rows, -(-vocab // 32)), generator=g, device=device).to(torch.int32)
    over = torch.full((rows,), 1.2, device=device)
    calls = (lambda x: F.adjust_logits(x), lambda x: F.adjust_logits(x, T(history), repetition=T(over), presence=T(over), bias=T(bias), allowed=T(words)),
             lambda x: F.adjust_logits(x, bias=T(off_boundary(bias, 1))))
    for call in calls:
        want = call(T(z)).to_torch()
        compiled = nb.compile(call)
        for by in (*range(1, 9), 0, 3):
            assert torch.equal(call(T(off_boundary(z, by))).to_torch(), want)
            assert torch.equal(compiled(T(off_boundary(z, by))).to_torch(), want)
    whole = torch.randn((1, 4, vocab), generator=g, device=device).to(dtype)
    last = nb.squeeze(nb.slice_tensor(T(whole), (0, 3, 0), (1, 1, vocab)), axis=1)
    assert torch.equal(F.adjust_logits(last, bias=T(bias)).to_torch(), F.adjust_logits(T(whole[:, 3].clone()), bias=T(bias)).to_torch())


# ---------------------------------------------------------------- what is hidden
def same_answers(got, want, vmax):
    """Two answers to the same question: each is off by the rounding of the result, and of weights, to the type (bf16: 8 and 11 bits; fp32: weights to 22 bits,
    exponentials and sums) at most. Scores are the same sums of the same products."""
    tol = 2.0 ** -7 * want.double().abs() + 2.0 ** -9 * vmax if got.dtype == torch.bfloat16 else torch.full_like(want, 2.0 ** -17 * vmax, dtype=torch.float64)
    return bool(((got.double() - want.double()).abs() <= tol).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("new", [3, 40, 150, 300])
def test_a_row_does_not_see_the_nan_of_a_later_token(new, which, block, dtype, device):
    """A new token that is not finite makes its block NaN: rows in front of that block come out as if it were not there, those that reach it as NaN."""
    g = gen(device, 52)
    b, hq, h, d, past = 2, 8, 2, 64, 2 * block - 2
    columns = (past + new) // block + 2
    cache = {}
    for name in ("k", "v"):
        cache[name] = torch.randint(-127, 128, (b * columns, h, block, d), generator=g, device=device, dtype=torch.int8)
        cache[name + "_scale"] = torch.rand((b * columns, h), generator=g, device=device) * 0.02 + 0.01
    table = torch.arange(b * columns, device=device, dtype=torch.int32).view(b, columns)
    first = torch.full((b,), past, device=device, dtype=torch.int32)
    q = torch.randn((b, new, hq, d), generator=g, device=device).to(dtype)
    call = lambda: F.cached_attention(T(q), {k: T(v) for k, v in cache.items()}, T(table), T(first)).to_torch()  # noqa: E731
    want = call()
    assert torch.isfinite(want).all()
    for column in sorted({2, (past + new - 1) // block}):                # the first block of new tokens alone, the last of them
        start = column * block - past                                    # the first row that sees it
        assert 0 < start < new
        kept = cache[which][column, 1].clone()                           # of the first sequence and the second head
        cache[which][column, 1] = math.nan
        got = call()
        cache[which][column, 1] = kept
        assert torch.isnan(got[0, start:, hq // 2:]).all()
        for x, y in ((got[0, :start], want[0, :start]), (got[0, :, :hq // 2], want[0, :, :hq // 2]), (got[1], want[1])):
            assert same_answers(x, y, 127 * 0.03)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new", [20, 150])
def test_a_later_token_that_is_not_finite_leaves_earlier_answers_alone(new, device):
    """The same through the cache's own writing: infinities in a key and in a value of the last new token."""
    g = gen(device, 53)
    h, d, n = 2, 128, 16
    q, k, v = (torch.randn((1, new, h, d), generator=g, device=device).to(torch.bfloat16) for _ in range(3))
    table, past = T(torch.arange(20, device=device, dtype=torch.int32)[None]), T(torch.zeros(1, device=device, dtype=torch.int32))

    def answer():
        cache = F.kv_cache_write(F.init_kv_cache(20, h, d, n, device=past.device), T(k), T(v), table, past)
        return F.cached_attention(T(q), cache, table, past).to_torch()

    want = answer()
    k[0, -1, 0, 5], v[0, -1, 1, 7] = math.inf, -math.inf
    got, start = answer(), (new - 1) // n * n
    assert torch.isnan(got[:, start:]).all() and same_answers(got[:, :start], want[:, :start], 6.0)


# ---------------------------------------------------------------- the order of reads and writes
class _Program:
    """A cache of one sequence that holds three tokens, and others to be written over them."""

    def __init__(self, device):
        g = gen(device, 54)
        self.k, self.other, self.q = (T(torch.randn((1, 3, 2, 64), generator=g, device=device)) for _ in range(3))
        self.table, self.zero = (T(torch.tensor(x, device=device, dtype=torch.int32)) for x in ([[3, 1]], [0]))
        self.three, self.five = (T(torch.tensor([x], device=device, dtype=torch.int32)) for x in (3, 5))
        self.device = self.k.device

    def cache(self):
        return F.kv_cache_write(F.init_kv_cache(4, 2, 64, 16, device=self.device), self.k, self.k, self.table, self.zero)

    def attend(self, cache):
        return F.cached_attention(self.q, cache, self.table, self.zero)

    def read(self, cache):
        return F.kv_cache_read(cache, self.table, self.zero, self.three, 3, dtype=nb.DType.float32)

    def write(self, cache, inplace=True):
        return F.kv_cache_write(cache, self.other, self.other, self.table, self.zero, inplace=inplace)

    def before(self):
        c = self.cache()
        return self.attend(c).to_torch(), self.read(c)[0].to_torch()

    def after(self):
        c = self.write(self.cache())
        return self.attend(c).to_torch(), self.read(c)[0].to_torch()


@pytest.mark.parametrize("device", DEVICES)
def test_what_was_read_before_a_write_is_what_was_there(device):
    """Answers that are looked at only after the next tokens were written."""
    p = _Program(device)
    (o, r), (o2, r2) = p.before(), p.after()
    assert not torch.equal(o, o2) and not torch.equal(r, r2)
    c = p.cache()
    early = p.attend(c), p.read(c)[0]
    copy = p.write(c, inplace=False)
    later = p.write(c)
    assert torch.equal(early[0].to_torch(), o) and torch.equal(early[1].to_torch(), r)
    assert torch.equal(p.attend(c).to_torch(), o2) and torch.equal(p.attend(later).to_torch(), o2)
    # a copy is of the cache as it was when it was asked for
    c = p.cache()
    copy = p.write(c, inplace=False)
    F.kv_cache_write(c, p.q, p.q, p.table, p.three)
    assert torch.equal(p.attend(copy).to_torch(), o2)
    five = [F.kv_cache_read(x, p.table, p.zero, p.five, 5)[0].to_torch() for x in (copy, c)]
    assert (five[0][:, 3:] == 0).all() and (five[1][:, 3:] != 0).any()
    # a compiled step in between
    c = p.cache()
    early = p.attend(c)
    nb.compile(p.write)(c)
    assert torch.equal(early.to_torch(), o) and torch.equal(p.attend(c).to_torch(), o2)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("form", ["read, write", "write, read", "the old name", "not returned", "the old name returned", "two writes", "another reader"])
def test_compiled_programs_keep_the_order_of_reads_and_writes(form, device):
    p = _Program(device)
    (o, r), (o2, r2) = p.before(), p.after()

    def program(c):
        if form == "read, write":
            early = p.attend(c), p.read(c)[0]
            return p.write(c), early
        if form == "write, read":
            early = p.attend(c), p.read(c)[0]
            c = p.write(c)
            return early, c, p.attend(c), p.read(c)[0]
        if form == "the old name":
            new = p.write(c)
            return p.attend(c), p.read(c)[0], new
        if form == "not returned":
            p.write(c)
            return p.attend(c), p.read(c)[0]
        if form == "the old name returned":
            early = p.read(c)[0]
            p.write(c)
            return c, early
        if form == "two writes":
            early = p.read(c)[0]
            p.write(c)
            middle = p.read(c)[0]
            F.kv_cache_write(c, p.k, p.k, p.table, p.zero)
            return c, middle, early, p.attend(c)
        early = c["k_scale"] * 2.0
        p.write(c)
        return c["k_scale"] * 2.0, early

    f = nb.compile(program)
    c = p.cache()
    scale, scale2 = c["k_scale"].to_torch() * 2.0, p.write(p.cache())["k_scale"].to_torch() * 2.0
    for _ in range(4):                       # recorded, replayed, and without Python
        c = p.cache()
        got = _leaves(f(c))
        codes = c["k"].to_torch()
        want = {"read, write": [None] * 4 + [o, r], "write, read": [o, r] + [None] * 4 + [o2, r2], "the old name": [o2, r2] + [None] * 4, "not returned": [o2, r2],
                "the old name returned": [None] * 4 + [r], "two writes": [None] * 4 + [r2, r, o], "another reader": [scale2, scale]}[form]
        assert len(got) == len(want) and all(w is None or torch.equal(x, w) for x, w in zip(got, want))
        assert torch.equal(codes, (p.cache() if form == "two writes" else p.write(p.cache()))["k"].to_torch())
        if None in want:                     # the cache that comes back is the one that was passed in
            assert got[want.index(None)].data_ptr() == codes.data_ptr()


def _leaves(x):
    from nabla_b200.core.common import pytree

    return [t.to_torch() for t in pytree.tree_leaves(x) if isinstance(t, nb.Tensor)]


# ---------------------------------------------------------------- waits
def test_warps_that_exchange_give_up_together():
    """A bounded wait ends by each lane's own clock. Lanes that go on to exchange values with the others have to leave as one, or the wait for those
    that left has no bound."""
    import re
    from pathlib import Path

    source = (Path(nb.__file__).parent / "csrc" / "cached_attention_tcgen05.cu").read_text()
    converting = source[source.index("if (warp < ISSUER) {"):source.index("} else if (warp == ISSUER) {")]
    assert "__shfl_sync(0xffffffffu" in converting
    assert len(re.findall(r"mbar_wait\(", converting)) == len(re.findall(r"__all_sync\(0xffffffffu, mbar_wait\(", converting)) == 2
    softmax = source[source.index("} else if (warp == ISSUER) {"):]
    softmax = softmax[softmax.index("  } else {"):]
    assert len(re.findall(r"mbar_wait\(", softmax)) == len(re.findall(r"ok = __all_sync\(0xffffffffu, ok\);", softmax)) == 2


# ---------------------------------------------------------------- sums of very many weights
@pytest.mark.gpu
@pytest.mark.parametrize("batch,new,hq", [(75, 9, 4), (1, 40, 4), (2, 1, 4)])
def test_a_million_small_weights_count(batch, new, hq):
    """One key that has 2^25.5 times the weight of each of a million others: they have 2.2 % of the sum. All values are 1, and so is the answer; a
    form that loses the others' values and not their part of the sum gives 0.978."""
    n, d, keys = 128, 64, 1 << 20
    columns = keys // n + 1
    cache = {"k": torch.zeros((columns, 1, n, d), dtype=torch.int8, device="cuda"), "v": torch.full((columns, 1, n, d), 100, dtype=torch.int8, device="cuda")}
    cache["k"][0, 0, 0, 0] = 127
    for name in ("k_scale", "v_scale"):
        cache[name] = torch.full((columns, 1), 0.01, device="cuda")
    q = torch.zeros((batch, new, hq, d), dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 13.9375                                 # times 1.27, over ln 2: 25.54
    table = torch.arange(columns, dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
    past = torch.full((batch,), keys, dtype=torch.int32, device="cuda")
    got = F.cached_attention(T(q), {k: T(v) for k, v in cache.items()}, T(table), T(past), scale=1.0).to_torch()
    # the result's rounding; a weight of 2^-25.54 against a largest of 1 loses up to half of 16-bit floats' last bit, 2^-25, taken 2^7 larger: 2^-32 for each of 2^20
    assert ((got.double() - 1).abs() <= 2.0 ** -8 + 2.0 ** -12).all(), (got.double() - 1).abs().max().item()


# ---------------------------------------------------------------- the end of a model's positions
@pytest.mark.parametrize("device", DEVICES)
def test_ragged_tokens_at_the_end_of_the_positions(device):
    """A sequence with fewer new tokens than the others whose padding lies behind the model's last position."""
    from nabla_b200.models import generate as G
    from nabla_b200.models import transformer as M

    cfg = M.TransformerConfig(n_layers=1, d_model=128, n_heads=2, d_ff=256, vocab=100, max_seq=20, dtype=nb.DType.float32)
    with nb.default_device(nb.Accelerator(0) if device == "cuda" else nb.CPU()):
        nb.seed(3)
        params = M.init_params(cfg)
    tokens = torch.randint(0, cfg.vocab, (2, 20), generator=gen("cpu", 55)).to(device)
    of = lambda *x: T(torch.tensor(x, device=device, dtype=torch.int32))  # noqa: E731

    def step(caches, table, tokens, past, count, positions=None):
        logits, caches = G.decode(params, T(tokens.contiguous()), caches, table, past, cfg, count, positions)
        return logits.to_torch(), caches

    got = []
    for given in (False, True):
        caches, table = G.init_caches(cfg, 2, 20, 16, device=params["tok_emb"].device)
        _, caches = step(caches, table, tokens[:, :18], of(0, 0), of(18, 3))
        positions = T(torch.tensor([[18, 19, 0, 0], [3, 4, 5, 6]], device=device)) if given else None
        logits, caches = step(caches, table, tokens[:, 16:20], of(18, 3), of(2, 4), positions)
        got.append(torch.cat([logits[0, :2], logits[1]]))
    assert torch.isfinite(got[0]).all() and torch.equal(got[0], got[1])


# ---------------------------------------------------------------- meshes
@pytest.mark.parametrize("compiled", [False, True])
def test_a_cache_whose_heads_are_split_is_written_where_it_lies(compiled):
    """Each device writes its own heads into its own part of the cache, and reads before a write are of what was there."""
    g = gen("cpu", 56)
    b, t, h, d, n = 2, 3, 4, 64, 16
    whole = {}
    for name in ("k", "v"):
        whole[name] = torch.randint(-127, 128, (8, h, n, d), generator=g, dtype=torch.int8)
        whole[name + "_scale"] = torch.rand((8, h), generator=g) * 0.02 + 0.01
    table, past = T(torch.randperm(8, generator=g)[:6].view(b, 3).to(torch.int32)), T(torch.tensor([5, 20], dtype=torch.int32))
    k, v = (torch.randn((b, t, h, d), generator=g) for _ in range(2))
    q = torch.randn((b, t, 2 * h, d), generator=g)
    mesh = nb.DeviceMesh("m", (2,), ("tp",))
    split = lambda x, at: T(x).shard(mesh, tuple("tp" if i == at else None for i in range(x.dim())))  # noqa: E731

    def step(cache, q, k, v):
        early = F.cached_attention(q, cache, table, past)
        cache = F.kv_cache_write(cache, k, v, table, past)
        return cache, early, F.cached_attention(q, cache, table, past)

    plain = {name: T(x.clone()) for name, x in whole.items()}
    _, early, late = step(plain, T(q), T(k), T(v))
    parts = {name: split(x.clone(), 1) for name, x in whole.items()}
    nb.realize_all(*parts.values())
    lies = {name: [x.data_ptr() for x in p._impl._buffers] for name, p in parts.items()}
    f = nb.compile(step) if compiled else step
    for again in range(2 if compiled else 1):
        got, early2, late2 = f(parts, split(q, 2), split(k, 2), split(v, 2))
        for name in parts:
            assert [x.data_ptr() for x in got[name]._impl._buffers] == lies[name]
            assert np.array_equal(parts[name].to_numpy(), plain[name].to_numpy())
        want = (early if again == 0 else late).to_torch()         # the second call finds the new tokens already there
        assert torch.allclose(torch.from_numpy(early2.to_numpy()), want, atol=1e-5)
        assert torch.allclose(torch.from_numpy(late2.to_numpy()), late.to_torch(), atol=1e-5)


# ---------------------------------------------------------------- branches and loops
@pytest.mark.parametrize("device", DEVICES)
def test_a_branch_that_writes_writes_only_when_it_is_taken(device):
    """cond and while_loop are recorded by trying their functions: what these update when they are tried is no update of the program."""
    p = _Program(device)
    (o, r), (o2, r2) = p.before(), p.after()

    def program(go, c):
        early = p.read(c)[0]
        scale = nb.cond(go, lambda c: p.write(c)["k_scale"] * 1.0, lambda c: c["k_scale"] * 1.0, c)
        return early, scale, p.read(c)[0], p.attend(c)

    f = nb.compile(program)
    for go in (False, True, False, True):
        for call in (f, program):
            c = p.cache()
            early, scale, late, answer = call(T(torch.tensor(go, device=device)), c)
            assert torch.equal(early.to_torch(), r) and torch.equal(late.to_torch(), r2 if go else r) and torch.equal(answer.to_torch(), o2 if go else o)
            assert torch.equal(scale.to_torch(), c["k_scale"].to_torch())
            assert torch.equal(c["k"].to_torch(), (p.write(p.cache()) if go else p.cache())["k"].to_torch())

    # tokens one after the other
    def loop(c, n):
        def body(i, c):
            at = nb.reshape(nb.cast(i, nb.DType.int32), (1,))
            k = F.kv_cache_read(c, p.table, p.zero, p.zero + 1, 1, dtype=nb.DType.float32)[0]
            return i + 1, F.kv_cache_write(c, k, k, p.table, at)

        i, c = nb.while_loop(lambda i, c: i < n, body, (n * 0 + 1, c))
        return c, p.read(c)[0]

    g = nb.compile(loop)
    for n in (1, 3, 2):
        for call in (g, loop):
            c = p.cache()
            got, rows = call(c, T(torch.tensor(n, device=device)))
            assert got["k"].to_torch().data_ptr() == c["k"].to_torch().data_ptr()
            rows = rows.to_torch()
            assert all(torch.equal(rows[:, i], rows[:, 0]) for i in range(n)) and (n == 3 or torch.equal(rows[:, 2], r[:, 2]))


@pytest.mark.parametrize("device", DEVICES)
def test_a_captured_cond_does_not_update_in_place(device):
    """It runs both branches and selects."""
    p = _Program(device)
    go = T(torch.tensor(False, device=device))
    f = nb.compile(lambda go, c: nb.cond(go, p.write, lambda c: c, c), cuda_graph=True)
    with pytest.raises(ValueError, match="in place"):
        f(go, p.cache())
    f = nb.compile(lambda go, c: nb.cond(go, lambda c: p.write(c, inplace=False), lambda c: c, c), cuda_graph=True)
    for go, want in ((False, p.before()[0]), (True, p.after()[0])):
        c = p.cache()
        assert torch.equal(p.attend(f(T(torch.tensor(go, device=device)), c)).to_torch(), want) and torch.equal(p.attend(c).to_torch(), p.before()[0])
