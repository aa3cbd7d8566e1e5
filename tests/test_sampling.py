"""The draw of tokens against its definition in 64 bits, on the CPU (torch expression) and on a GPU (hand-written kernels).

Tokens are whole numbers: they have to be equal. Weights are off by 2^-44 of the largest at most (their rounding to whole multiples of 2^-43), so a draw
may differ only where u times the sum, or a border of top-p or min-p, comes within about 2^-40 of a sum: the inputs here do not (``oracle`` checks it).
"""
from __future__ import annotations

import math

import pytest
import torch

import nabla_b200 as nb
from nabla_b200.nn import functional as F

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def T(x):
    return None if x is None else nb.Tensor.from_torch(x)


def oracle(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, clear=True):
    """One row and token at a time. ``clear``: borders that an error of 2^-40 would move are not allowed (but for equal weights)."""
    out = []
    for i, row in enumerate(logits.double().cpu()):
        z = torch.where(row > -math.inf, row, -math.inf)                     # NaN: nowhere
        order = sorted((v for v in range(len(z)) if z[v] > -math.inf), key=lambda v: (-z[v].item(), v))
        t = 1.0 if temperature is None else float(temperature[i])
        if not order or not t > 0:
            out.append(order[0] if order else -1)
            continue
        k = 0 if top_k is None else int(top_k[i])
        if k > 0:
            order = order[:k]
        top = z[order[0]].item()
        w = [1.0 if z[v] == top else 0.0 if math.isinf(top) else math.exp((z[v].item() - top) / t) for v in order]
        w = [x if x >= 2.0 ** -44 else 0.0 for x in w]
        p = 1.0 if top_p is None else float(top_p[i])
        if p < 1:
            want, sum_, n = p * math.fsum(w), 0.0, 0
            while n < len(w) and (n == 0 or sum_ < want):
                sum_ += w[n]
                n += 1
                assert not clear or len(set(w)) < 3 or abs(sum_ - want) > 2.0 ** -40 * want
            order, w = order[:n], w[:n]
        m = 0.0 if min_p is None else float(min_p[i])
        if m > 0:
            kept = [x >= min(m, 1.0) for x in w]
            order, w = [v for v, s in zip(order, kept) if s], [x for x, s in zip(w, kept) if s]
        left = sorted((v, x) for v, x in zip(order, w) if x > 0)
        u = max(float(uniform[i]), 0.0) if uniform[i] == uniform[i] else 0.0
        want, sum_, token = u * math.fsum(x for _, x in left), 0.0, left[-1][0]
        for v, x in left:
            sum_ += x
            if sum_ > want:
                token = v
                break
        out.append(token)
    return out


def draw(logits, uniform, **kw):
    got = F.sample_tokens(T(logits), T(uniform), **{k: T(v) for k, v in kw.items()})
    assert got.dtype is nb.DType.int64 and tuple(got.shape) == (logits.shape[0],)
    return got.to_torch().tolist()


def rows(device, seed, b, v, std, dtype):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn((b, v), generator=g) * std).to(dtype)
    kw = {"temperature": torch.rand(b, generator=g) * 1.4 + 0.1, "top_k": torch.randint(0, v + 3, (b,), generator=g, dtype=torch.int32),
          "top_p": torch.rand(b, generator=g) * 1.1, "min_p": torch.rand(b, generator=g) * 0.2}
    kw["temperature"][::5] = 0.0
    kw["top_k"][::4] = torch.randint(1, 9, kw["top_k"][::4].shape, generator=g, dtype=torch.int32)
    kw["min_p"][::3] = 0.0
    return z.to(device), torch.rand(b, generator=g).to(device), {k: x.to(device) for k, x in kw.items()}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("names", ["", "temperature", "temperature top_k", "temperature top_p", "temperature min_p", "top_k top_p", "temperature top_k top_p min_p"])
@pytest.mark.parametrize("b,v,std,dtype", [
    (1, 1, 1.0, torch.float32), (3, 2, 1.0, torch.bfloat16), (20, 37, 2.0, torch.float32), (16, 333, 3.0, torch.bfloat16), (9, 1000, 0.02, torch.float32),
    (7, 4099, 3.0, torch.bfloat16), (6, 5001, 12.0, torch.float32),
])
def test_draws(b, v, std, dtype, names, device):
    z, u, kw = rows(device, b * v, b, v, std, dtype)
    kw = {k: kw[k] for k in names.split()}
    assert draw(z, u, **kw) == oracle(z, u, **kw)


@pytest.mark.parametrize("device", DEVICES)
def test_equal_logits_are_ordered_by_id(device):
    """Rows of few different values, all alike, -0 beside 0; borders that fall inside a run of equal ones."""
    g = torch.Generator().manual_seed(3)
    z = torch.randint(0, 3, (40, 2500), generator=g).float() * 0.5
    z[0] = 1.25
    z[1, ::2], z[1, 1::2] = 0.0, -0.0
    z[2] = torch.where(torch.arange(2500) % 7 == 0, 2.0, -1000.0)
    z = z.to(device)
    u = torch.rand(40, generator=g).to(device)
    k = torch.randint(1, 2500, (40,), generator=g).to(device)
    p = (torch.randint(1, 64, (40,), generator=g) / 64.0).to(device)
    assert draw(z, u, top_k=k) == oracle(z, u, top_k=k)
    assert draw(z, u, top_p=p) == oracle(z, u, top_p=p, clear=False)
    assert draw(z, u, top_k=k, top_p=p) == oracle(z, u, top_k=k, top_p=p, clear=False)
    cold = torch.zeros(40, device=device)
    assert draw(z, u, temperature=cold) == [int(torch.nonzero(r == r.max())[0]) for r in z.cpu()]


@pytest.mark.parametrize("device", DEVICES)
def test_hidden_infinite_and_undefined_logits(device):
    """Rows where -inf hides some, all but one or all tokens; NaN; +inf; the lowest finite number as a mask."""
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    z = torch.zeros((9, 600))
    z[0] = -inf
    z[1] = -inf
    z[1, 577] = -3e38
    z[2, :] = nan
    z[3, :300] = nan
    z[4, 5::2] = -inf
    z[5, 400:] = inf
    z[6] = low
    z[6, 7], z[6, 599] = 1.0, 2.0
    z[7] = low
    z[8, 100] = 3e38
    for name, kw in [("plain", {}), ("k", {"top_k": torch.full((9,), 3)}), ("p", {"top_p": torch.full((9,), 0.75)}),
                     ("all", {"top_k": torch.full((9,), 250, dtype=torch.int32), "top_p": torch.full((9,), 0.5), "min_p": torch.full((9,), 0.01),
                              "temperature": torch.full((9,), 0.5)})]:
        kw = {k: x.to(device) for k, x in kw.items()}
        for u in (0.0, 0.3, 0.999):
            us = torch.full((9,), u, device=device)
            got = draw(z.to(device), us, **kw)
            assert got == oracle(z, us, **kw, clear=False), (name, u)
            assert got[0] == got[2] == -1 and got[1] == 577


@pytest.mark.parametrize("device", DEVICES)
def test_numbers_at_the_ends(device):
    """Random numbers 0, below 1, 1 and undefined; temperatures from next to nothing to infinity; filters outside their range."""
    g = torch.Generator().manual_seed(8)
    z = torch.randn((1, 700), generator=g).repeat(12, 1).to(device)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan, 0.5, 2.0 ** -149, 0.25, 0.75, 0.1, 0.9], device=device)
    inf = math.inf
    some = torch.rand(12, generator=g).to(device)
    assert draw(z, u) == oracle(z, u)
    for name, values in [("temperature", [1e-45, 1e-38, 1e-5, inf, 1e30, -1.0, math.nan, 0.0, 1e-2, 100.0, 5.0, 0.5]),
                         ("top_p", [0.0, -1.0, 1.0, 2.0, math.nan, 1e-30, 1 - 2.0 ** -24, 0.5, 0.1, 0.9, 0.99, 0.999]),
                         ("min_p", [0.0, -1.0, 1.0, 2.0, math.nan, 1e-30, 1e-13, 0.5, 0.1, 0.9, 1e-3, 1e-6])]:
        x = torch.tensor(values, device=device)
        assert draw(z, some, **{name: x}) == oracle(z, some, **{name: x}, clear=False), name
    k = torch.tensor([0, -5, 1, 2, 699, 700, 701, 1 << 40, -(1 << 40), 3, 350, 10], device=device)
    assert draw(z, some, top_k=k) == oracle(z, some, top_k=k)


@pytest.mark.parametrize("v,device", [(300, "cpu"), (1300, "cpu"), *(pytest.param(v, "cuda", marks=pytest.mark.gpu) for v in (300, 1300, 9001))])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_further_apart_than_the_largest_number(v, dtype, device):
    """Differences of logits past fp32's largest number, and temperatures that bring them back to a few units."""
    g = torch.Generator().manual_seed(v)
    z = ((torch.rand((6, v), generator=g) * 2 - 1) * 3.3e38).to(dtype)
    z[3, ::2] = -math.inf
    z[4] = torch.where(torch.rand(v, generator=g) < 0.5, 3e38, -3e38).to(dtype)
    t = torch.tensor([1e38, 3e38, math.inf, 2e38, 3e38, 5e37])
    u = torch.tensor([0.5, 0.03, 0.98, 0.7, 0.999, 0.6])
    k = torch.tensor([v - 40, v // 2, 7, v // 3, 0, 0])
    p = torch.tensor([0.9, 0.97, 0.999, 0.51, 0.95, 0.6])
    m = torch.tensor([0.01, 0.2, 0.5, 0.3, 0.1, 1e-4])
    z, t, u, k, p, m = (x.to(device) for x in (z, t, u, k, p, m))
    for kw in ({}, {"top_k": k}, {"top_p": p}, {"min_p": m}, {"top_k": k, "top_p": p, "min_p": m}):
        assert draw(z, u, temperature=t, **kw) == oracle(z, u, temperature=t, **kw, clear=v < 9001)       # (which is slow for long rows)


@pytest.mark.gpu
@pytest.mark.parametrize("v,dtype,std", [(131072, torch.float32, 3.0), (32001, torch.bfloat16, 3.0), (1 << 20, torch.bfloat16, 1.0), (100003, torch.float32, 0.01),
                                         (65537, torch.bfloat16, 0.0)])
def test_long_rows(v, dtype, std):
    """Flat and steep rows of large vocabularies, where borders fall into bins of thousands of tokens."""
    b = 6
    g = torch.Generator("cuda").manual_seed(v)
    z = (torch.randn((b, v), generator=g, device="cuda") * std).to(dtype)
    z[0] = z[0].float().round().to(dtype)                      # a few hundred values at most
    u = torch.rand(b, generator=g, device="cuda")
    k = torch.tensor([1000, v // 3, 7, 0, v - 1, 40], device="cuda")
    p = torch.tensor([0.5, 0.9, 0.25, 0.97, 0.5, 1.0], device="cuda")
    zs, order = torch.sort(z.double(), descending=True, stable=True)
    for kw in ({}, {"top_k": k}, {"top_p": p}, {"top_k": k, "top_p": p}):
        w = torch.exp(zs - zs[:, :1])
        rank = torch.arange(v, device="cuda")
        if "top_k" in kw:
            w = torch.where((rank < k[:, None]) | (k[:, None] <= 0), w, 0.0)
        if "top_p" in kw:
            w = torch.where((w.cumsum(-1) - w < p.double()[:, None] * w.sum(-1, keepdim=True)) | (p[:, None] >= 1), w, 0.0)
        total = torch.zeros_like(w).scatter_(1, order, w).cumsum(-1)
        want = (total <= u.double()[:, None] * total[:, -1:]).sum(-1)
        # sums of 10^6 numbers in 64 bits are off by some 2^-40: a draw that near to a border says nothing
        near = ((total / total[:, -1:] - u.double()[:, None]).abs() < 2.0 ** -38).any(-1)
        got = F.sample_tokens(T(z), T(u), **{n: T(x) for n, x in kw.items()}).to_torch()
        assert not near.any() and torch.equal(got, want)


@pytest.mark.parametrize("device", DEVICES)
def test_shares_of_draws(device):
    """Evenly spread random numbers draw each token in proportion to its weight."""
    n = 4096
    z = torch.log(torch.tensor([[1.0, 2.0, 3.0, 10.0, 0.0]], device=device)).expand(n, -1).contiguous()
    u = (torch.arange(n, device=device) + 0.5) / n
    got = torch.tensor(draw(z, u))
    share = torch.bincount(got, minlength=5) / n
    assert (share - torch.tensor([1, 2, 3, 10, 0]) / 16.0).abs().max() <= 1.0 / n and (got[1:] >= got[:-1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_and_rows_off_boundaries(dtype):
    z, u, kw = rows("cuda", 5, 12, 777, 3.0, dtype)
    wide = torch.full((12, 1000), 50.0, device="cuda", dtype=dtype)
    want = oracle(z, u, **kw)
    for off in (0, 1, 3, 200):
        wide.fill_(50.0)
        wide[:, off:off + 777] = z
        assert draw(wide[:, off:off + 777], u, **kw) == want
    flat = torch.full((12 * 777 + 9,), 50.0, device="cuda", dtype=dtype)
    for off in (1, 2, 5, 9):
        flat.fill_(50.0)
        flat[off:off + 12 * 777] = z.flatten()
        assert draw(flat[off:off + 12 * 777].view(12, 777), u, **kw) == want
    assert draw(z, u.repeat_interleave(2)[::2], **{k: x.repeat_interleave(3)[::3] for k, x in kw.items()}) == want


@pytest.mark.parametrize("device", DEVICES)
def test_compiled_and_in_streams(device):
    z, u, kw = rows(device, 6, 9, 2000, 3.0, torch.float32)
    want = draw(z, u, **kw)
    names = tuple(kw)
    f = lambda z, u, *x: F.sample_tokens(F.adjust_logits(z), u, **dict(zip(names, x)))  # noqa: E731
    args = [T(x) for x in (z, u, *kw.values())]
    step = nb.compile(f)
    for _ in range(3):
        assert step(*args).to_torch().tolist() == want
    if device == "cpu":
        return
    graph = nb.compile(f, cuda_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(3):
            other = torch.roll(z, i, 0)
            assert graph(T(other), *[T(torch.roll(x, i, 0)) for x in (u, *kw.values())]).to_torch().tolist() == want[-i:] + want[:-i] if i else want
    assert draw(z[:0], u[:0]) == []


def test_over_a_mesh(mesh_2x4):
    z, u, kw = rows("cpu", 7, 8, 300, 2.0, torch.float32)
    want = draw(z, u, **kw)
    place = lambda x: T(x).shard(mesh_2x4, ("dp",) + (None,) * (x.dim() - 1))  # noqa: E731
    got = F.sample_tokens(place(z), place(u), **{k: place(x) for k, x in kw.items()})
    assert got.to_numpy().tolist() == want
    split = T(z).shard(mesh_2x4, (None, "tp"))            # a vocabulary in parts comes together first
    assert F.sample_tokens(split, T(u).shard(mesh_2x4, (None,))).to_numpy().tolist() == draw(z, u)


def test_refusals():
    z, u = T(torch.zeros(2, 5)), T(torch.zeros(2))
    assert F.sample_tokens(z, u).to_torch().tolist() == [0, 0]
    two = torch.ones(2)
    for error, args, kw in [
        (TypeError, (torch.zeros(2, 5), u), {}), (TypeError, (z, [0.0, 0.0]), {}), (TypeError, (T(torch.zeros(2, 5, dtype=torch.float64)), u), {}),
        (ValueError, (T(torch.zeros(5)), u), {}), (ValueError, (z, T(torch.zeros(3))), {}), (TypeError, (z, T(two.double())), {}),
        (ValueError, (T(torch.zeros(2, 0)), u), {}), (ValueError, (T(torch.zeros((2, 1 << 20 | 1), dtype=torch.bfloat16)), u), {}),
        (TypeError, (z, u), {"temperature": 0.7}), (TypeError, (z, u), {"temperature": T(two.long())}), (TypeError, (z, u), {"top_k": T(two)}),
        (ValueError, (z, u), {"top_k": T(torch.ones(1, dtype=torch.int32))}), (TypeError, (z, u), {"top_p": T(two.bfloat16())}),
        (ValueError, (z, u), {"min_p": T(torch.ones(2, 1))}),
    ]:
        with pytest.raises(error):
            F.sample_tokens(*args, **kw)
    with pytest.raises(ValueError):
        nb.vmap(lambda x: F.sample_tokens(x, u))(T(torch.zeros(3, 2, 5)))


@pytest.mark.gpu
def test_a_compiled_draw_is_written_down():
    from nabla_b200.transforms import tape

    if tape.module() is None:
        pytest.skip("libnb_replay.so is not built here")
    z, u, kw = rows("cuda", 6, 9, 2000, 3.0, torch.float32)
    f = nb.compile(lambda z, u, *x: F.sample_tokens(z, u, **dict(zip(kw, x))))
    for _ in range(4):
        f(*[T(x) for x in (z, u, *kw.values())])
    assert f._taped is not None and bool(f._taped[0]), f.tape_refused
