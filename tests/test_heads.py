"""Norms and rotations of heads against their definition in 64 bits, on the CPU (torch expressions, primitive operations) and on a GPU.

Tolerances: a result is rounded once to its type (half a step, relative). In front of that, fp32: the sum of D squares (a chain of 16 and
five joins: 21 roundings, half of that behind the root), the root (2 units), two products, the cosine and sine (2 units each) and a rotation of two
products and a sum: below 2^5 units of 2^-24, so 2^-18 of the pair's length covers it with a factor of two to spare.
"""
from __future__ import annotations

import decimal
import math

import pytest
import torch

import nabla_b200 as nb
from nabla_b200.nn import functional as F
from nabla_b200.ops import heads

D = decimal.Decimal
DEVICES = ["cpu", "primitive", pytest.param("cuda", marks=pytest.mark.gpu)]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
EPS = 1e-6


def T(x):
    return nb.Tensor.from_torch(x)


@pytest.fixture
def on(request, monkeypatch):
    """The device; "cpu" runs the fused operation's torch expression, "primitive" the composition."""
    monkeypatch.setenv("NABLA_B200_FUSED", "0" if request.param == "primitive" else "1")
    return "cuda" if request.param == "cuda" else "cpu"


def turn64(y, positions, rotary, base, interleaved, back=False):
    out = y.clone()
    for i in range(rotary // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
        angle = positions.double() * base ** (-2.0 * i / rotary) * (-1 if back else 1)
        while angle.dim() < y.dim() - 1:
            angle = angle.unsqueeze(-1) if angle.dim() > 1 or y.dim() == 3 else angle[:, None]
        c, s = torch.cos(angle), torch.sin(angle)
        out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
    return out


def lengths(y, rotary, interleaved):
    """Of the pair that each number belongs to (its own magnitude where it is not turned)."""
    out = y.abs().clone()
    for i in range(rotary // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
        out[..., a] = out[..., b] = torch.hypot(y[..., a], y[..., b])
    return out


def oracle(x, gain, positions, dy, *, rotary, base=10000.0, interleaved=False):
    """(y, its scale, dx, its scale, dg, the sum of the magnitudes behind it) in 64 bits."""
    x64, dy64 = x.double(), dy.double()
    if gain is None:
        y = turn64(x64, positions, rotary, base, interleaved)
        dx = turn64(dy64, positions, rotary, base, interleaved, back=True)
        return y, lengths(x64, rotary, interleaved), dx, lengths(dy64, rotary, interleaved), None, None
    g = gain.double()
    r = 1.0 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + EPS)
    n = x64 * r
    z = n * g
    y = turn64(z, positions, rotary, base, interleaved)
    dz = turn64(dy64, positions, rotary, base, interleaved, back=True)
    dn = dz * g
    dx = r * (dn - n * (dn * n).mean(-1, keepdim=True))
    size = lengths(dy64, rotary, interleaved)
    scale = r * (size * g.abs() + n.abs() * (size * g.abs() * n.abs()).mean(-1, keepdim=True))
    dg = (dz * n).flatten(0, -2).sum(0)
    return y, lengths(z, rotary, interleaved), dx, scale, dg, (size * n.abs()).flatten(0, -2).sum(0)


def near(got, want, scale, more=2.0 ** -18):
    assert got.shape == want.shape and torch.isfinite(got).all()
    off, tol = (got.double() - want).abs(), HALF[got.dtype] * want.abs() + more * scale
    assert (off <= tol).all(), f"off by {off.max().item():.3g}, {(off / tol).max().item():.3g} times what is allowed"


CASES = [
    # batch, tokens, heads, kv heads, head_dim, rotary_dim, interleaved, dtype, gains, positions: shared?, first, type
    (1, 1, 1, 1, 64, 64, False, "bf16", "qk", True, 0, "int32"),
    (2, 1, 16, 4, 128, 128, False, "bf16", "qk", False, 120001, "int32"),
    (2, 37, 3, 1, 64, 32, True, "fp32", "qk", False, 4000, "int64"),
    (3, 5, 4, 2, 80, 80, False, "bf16", "qk", True, 7, "int64"),            # 5 of 8 lanes hold a head
    (1, 9, 2, 2, 96, 64, False, "fp32", "q", True, 1 << 33, "int64"),
    (2, 3, 5, 5, 16, 16, True, "fp32", "k", False, -50, "int32"),
    (1, 7, 2, 1, 256, 256, False, "bf16", "qk", True, 1000003, "int32"),
    (2, 33, 4, 4, 128, 64, True, "bf16", "", True, 5, "int32"),
    (1, 300, 8, 8, 128, 128, False, "fp32", "qk", True, 0, "int64"),
]


def make(case, device, seed=0):
    b, t, hq, h, d, rotary, inter, dtype, which, shared, first, whole = case
    g = torch.Generator().manual_seed(seed)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    q, k, cq, ck = (torch.randn((b, t, n, d), generator=g).mul(1.5).to(dt).to(device) for n in (hq, h, hq, h))
    q[0, 0, 0] = 0                                                         # a head of zeros
    gq, gk = ((torch.randn((d,), generator=g) * 0.2 + 1).to(dt).to(device) for _ in range(2))
    pos = torch.arange(t, dtype=getattr(torch, whole)) + first
    if not shared:
        pos = pos[None] + torch.randint(0, 50, (b, 1), generator=g).to(pos.dtype)
    return q, k, cq, ck, gq if "q" in which else None, gk if "k" in which else None, pos.to(device)


def spread(pos, x):
    return pos if pos.dim() == 2 else pos.expand(x.shape[0], -1)


@pytest.mark.parametrize("on", DEVICES, indirect=True)
@pytest.mark.parametrize("case", CASES)
def test_heads_and_their_gradients(case, on):
    q, k, cq, ck, gq, gk, pos = make(case, on)
    rotary, inter = case[5], case[6]
    wrt = [T(x) for x in (q, k, gq, gk) if x is not None]
    names = [n for n, x in zip(("q", "k", "gq", "gk"), (q, k, gq, gk)) if x is not None]

    def f(*ts):
        given = dict(zip(names, ts))
        return F.norm_rotary(given["q"], given["k"], T(pos), given.get("gq"), given.get("gk"), eps=EPS, rotary_dim=rotary, interleaved=inter)

    y, pull = nb.vjp(f, *wrt, create_graph=False)
    grads = dict(zip(names, (t.to_torch() for t in pull((T(cq), T(ck))))))
    for i, (x, gain, c, name) in enumerate(((q, gq, cq, "q"), (k, gk, ck, "k"))):
        want = oracle(x, gain, spread(pos, x), c, rotary=rotary, interleaved=inter)
        near(y[i].to_torch(), want[0], want[1])
        near(grads[name], want[2], want[3], 2.0 ** -17)                     # twice the roundings: a mean of products behind the norm
        if gain is not None:
            # a sum of all heads' terms in some order: each of its roundings is at most 2^-24 of the magnitudes so far
            near(grads["g" + name], want[4], want[5], (x.numel() // x.shape[-1] + 64) * 2.0 ** -24)


@pytest.mark.parametrize("on", DEVICES, indirect=True)
@pytest.mark.parametrize("case", [c for c in CASES if c[2] == c[3]])
def test_packed_projection(case, on):
    q, k, cq, ck, gq, gk, pos = make(case, on)
    b, t, h, d = q.shape
    rotary, inter = case[5], case[6]
    v, cv = torch.randn_like(q), torch.randn_like(q)
    pack = lambda *x: torch.stack(x, 3).reshape(b, t, 3 * h * d)  # noqa: E731
    qkv, cot = pack(q, k, v), pack(cq, ck, cv)
    wrt = [T(x) for x in (qkv, gq, gk) if x is not None]
    names = [n for n, x in zip(("x", "gq", "gk"), (qkv, gq, gk)) if x is not None]

    def f(*ts):
        given = dict(zip(names, ts))
        return F.packed_norm_rotary(given["x"], d, T(pos), given.get("gq"), given.get("gk"), eps=EPS, rotary_dim=rotary, interleaved=inter)

    y, pull = nb.vjp(f, *wrt, create_graph=False)
    grads = dict(zip(names, (g.to_torch() for g in pull(T(cot)))))
    y, dx = (u.view(b, t, h, 3, d) for u in (y.to_torch(), grads["x"]))
    assert torch.equal(y[:, :, :, 2], v) and torch.equal(dx[:, :, :, 2], cv)
    for i, (x, gain, c, name) in enumerate(((q, gq, cq, "gq"), (k, gk, ck, "gk"))):
        want = oracle(x, gain, spread(pos, x), c, rotary=rotary, interleaved=inter)
        near(y[:, :, :, i], want[0], want[1])
        near(dx[:, :, :, i], want[2], want[3], 2.0 ** -17)
        if gain is not None:
            near(grads[name], want[4], want[5], (x.numel() // d + 64) * 2.0 ** -24)


@pytest.mark.parametrize("on", DEVICES, indirect=True)
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_against_differences(interleaved, on):
    """Along one direction: the difference of two calls over their distance."""
    case = (2, 6, 4, 2, 64, 32, interleaved, "fp32", "qk", False, 100, "int32")
    q, k, cq, ck, gq, gk, pos = make(case, on)
    q[0, 0, 0] = 0.5            # (a head of zeros is bent within the step)
    xs = [q, k, gq, gk]
    g = torch.Generator().manual_seed(9)
    way = [torch.randn(x.shape, generator=g).to(on) for x in xs]

    def value(xs):
        y = F.norm_rotary(*(T(x) for x in xs[:2]), T(pos), *(T(x) for x in xs[2:]), eps=EPS, rotary_dim=32, interleaved=interleaved)
        return sum((u.to_torch().double() * c.double()).sum().item() for u, c in zip(y, (cq, ck)))

    h = 2.0 ** -7
    slope = (value([x + h * w for x, w in zip(xs, way)]) - value([x - h * w for x, w in zip(xs, way)])) / (2 * h)
    _, pull = nb.vjp(lambda a, b, c, d: F.norm_rotary(a, b, T(pos), c, d, eps=EPS, rotary_dim=32, interleaved=interleaved), *(T(x) for x in xs), create_graph=False)
    grads = [t.to_torch().double() for t in pull((T(cq), T(ck)))]
    want = sum((a * w.double()).sum().item() for a, w in zip(grads, way))
    size = sum((a * w.double()).norm().item() for a, w in zip(grads, way))
    # third derivatives of the norm times h^2 / 6 (of order one for entries of about one), and the rounding of two values over 2 h
    values = math.sqrt(cq.numel() + ck.numel()) * 1.5 * 2.0 ** -23 / (2 * h)
    assert abs(slope - want) <= 20 * h * h * size + values


def exact_turn(position, base, rotary):
    """Cosines and sines of a position's angles, which are reduced in 120 digits."""
    with decimal.localcontext() as c:
        c.prec = 120
        # pi by Machin's formula: 16 atan(1/5) - 4 atan(1/239)
        atan = lambda n: sum((-1) ** i * D(1) / (D(n) ** (2 * i + 1) * (2 * i + 1)) for i in range(180))  # noqa: E731
        whole = 2 * (16 * atan(5) - 4 * atan(239))
        rest = [(D(position) * (D(base).ln() * (-2 * i) / rotary).exp()) % whole for i in range(rotary // 2)]
        return torch.tensor([[math.cos(x), math.sin(x)] for x in rest], dtype=torch.float64)


def ones_turned(on, positions, base, d=64):
    """(cos, sin) of ``positions`` by pairs (0, 1) that are turned, and by their gradients, which are turned back: two tensors (tokens, d / 2, 2)."""
    x = torch.zeros((1, len(positions), 1, d), device=on)
    x[..., d // 2:] = 1.0
    pos = T(torch.tensor(positions, dtype=torch.int64, device=on))
    y, pull = nb.vjp(lambda q, k: F.norm_rotary(q, k, pos, base=base), T(x), T(x.clone()), create_graph=False)
    (dq, _), y = pull((T(x), T(x.clone()))), y[0].to_torch()
    y, dq = (z.double().cpu()[0, :, 0].view(-1, 2, d // 2) for z in (y, dq.to_torch()))
    return torch.stack([y[:, 1], -y[:, 0]], -1), torch.stack([dq[:, 1], dq[:, 0]], -1)


@pytest.mark.parametrize("on", DEVICES, indirect=True)
@pytest.mark.parametrize("base", [1e4, 5e5, 1e6])
def test_slow_pairs_keep_their_bits(base, on):
    """The sine of a small angle is as good, beside itself, as others beside 1: two units of 2^-24 for the sine, one for its correction by what a float
    does not hold of the angle, one to spare; and what an angle in 64 bits is off by, 2^-50 for each position."""
    positions = [1, 2, 999, -7]
    want = torch.stack([exact_turn(p, base, 64) for p in positions])
    for got in ones_turned(on, positions, base):
        tol = 2.0 ** -22 * want.abs() + 2.0 ** -50 * torch.tensor(positions).abs()[:, None, None]
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / want.abs()).max().item()


@pytest.mark.parametrize("on", DEVICES, indirect=True)
@pytest.mark.parametrize("base", [1e4, 1e6])
def test_far_positions(base, on):
    """As above; a fraction in whole numbers of 2^-64 of a turn is off by half of that at most, 2 pi 2^-65 < 2^-62 for each position."""
    positions = [(1 << 28) + 1, (1 << 33) + 7, (1 << 38) - 5, -(1 << 36) + 11, (1 << 40) + 3, -(1 << 44)]
    want = torch.stack([exact_turn(p, base, 64) for p in positions])
    for got in ones_turned(on, positions, base):
        tol = 2.0 ** -22 * want.abs() + 2.0 ** -62 * torch.tensor(positions).double().abs()[:, None, None] + 2.0 ** -50
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max().item()


@pytest.mark.parametrize("base", [1e4, 0.5, 1e-30, 3e38, 1.0])
def test_fractions_of_turns(base):
    """Against the angles of a position in 120 digits: half a unit of 2^-64 of a turn, and what a double holds of their sines."""
    n = torch.tensor([x / 2.0 ** 64 for x in heads.turns(base, 32)], dtype=torch.float64) * (2 * math.pi)
    assert len(n) == 16 and all(0 <= x < 1 << 64 for x in heads.turns(base, 32))
    want = exact_turn(1, base, 32)
    assert (n.cos() - want[:, 0]).abs().max() <= 2.0 ** -50 and (n.sin() - want[:, 1]).abs().max() <= 2.0 ** -50


@pytest.mark.gpu
@pytest.mark.parametrize("off", [1, 4, 8])
def test_views_off_boundaries_and_strides(off, monkeypatch):
    """Queries and keys as views of a projection that start anywhere; cotangents that are broadcast or transposed."""
    g = torch.Generator("cuda").manual_seed(1)
    b, t, hq, h, d = 2, 11, 4, 2, 64
    wide = torch.randn((b, t, (hq + 2 * h) * d + 2 * off), generator=g, device="cuda").to(torch.bfloat16)
    heads_ = wide[:, :, off:off + (hq + 2 * h) * d].unflatten(-1, (hq + 2 * h, d))
    q, k = heads_[:, :, :hq], heads_[:, :, hq:hq + h]
    gq, gk = (torch.randn((d,), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    pos = torch.arange(t, device="cuda")
    cq = torch.randn((t, b, hq, d), generator=g, device="cuda").to(torch.bfloat16).transpose(0, 1)
    ck = torch.randn((1, 1, 1, d), generator=g, device="cuda").to(torch.bfloat16).expand(b, t, h, d)
    y, pull = nb.vjp(lambda *x: F.norm_rotary(x[0], x[1], T(pos), *x[2:], eps=EPS), T(q), T(k), T(gq), T(gk), create_graph=False)
    grads = [x.to_torch() for x in pull((T(cq), T(ck)))]
    for i, (x, gain, c) in enumerate(((q, gq, cq), (k, gk, ck))):
        want = oracle(x, gain, spread(pos, x), c, rotary=d)
        near(y[i].to_torch(), want[0], want[1])
        near(grads[i], want[2], want[3], 2.0 ** -17)
        near(grads[2 + i], want[4], want[5], (x.numel() // d + 64) * 2.0 ** -24)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [(3, 1999), (1, 4735), (1, 4736), (8, 2048)])
def test_many_tokens(tokens):
    """On both sides of where a block takes several tokens, and of where backward blocks take several steps; the same bits every time."""
    b, t = tokens
    case = (b, t, 5, 3, 128, 128, False, "bf16", "qk", False, 77, "int64")
    q, k, cq, ck, gq, gk, pos = make(case, "cuda")
    call = nb.compile(lambda q, k, p, a, b, cq, ck: (lambda y, pull: (y, pull((cq, ck))))(
        *nb.vjp(lambda *x: F.norm_rotary(x[0], x[1], p, *x[2:], eps=EPS), q, k, a, b, create_graph=False)))
    args = [T(x) for x in (q, k, pos, gq, gk, cq, ck)]
    runs = []
    for _ in range(3):
        y, grads = call(*args)
        runs.append([x.to_torch().clone() for x in (*y, *grads)])
    for other in runs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(runs[0], other))
    for i, (x, gain, c) in enumerate(((q, gq, cq), (k, gk, ck))):
        want = oracle(x, gain, spread(pos, x), c, rotary=128)
        near(runs[0][i], want[0], want[1])
        near(runs[0][2 + i], want[2], want[3], 2.0 ** -17)
        near(runs[0][4 + i], want[4], want[5], (x.numel() // 128 + 64) * 2.0 ** -24)


@pytest.mark.parametrize("on", DEVICES, indirect=True)
def test_empty_calls(on):
    for shape in ((0, 5), (2, 0)):
        q, k = torch.zeros((*shape, 4, 64), device=on), torch.zeros((*shape, 2, 64), device=on)
        gain, pos = torch.ones(64, device=on), torch.zeros(shape, dtype=torch.int64, device=on)
        y, pull = nb.vjp(lambda a, b, g: F.norm_rotary(a, b, T(pos), g), T(q), T(k), T(gain), create_graph=False)
        grads = pull((T(q), T(k)))
        assert tuple(y[0].to_torch().shape) == q.shape and tuple(y[1].to_torch().shape) == k.shape
        assert torch.equal(grads[2].to_torch(), torch.zeros(64, device=on))


@pytest.mark.parametrize("on", DEVICES, indirect=True)
def test_transforms(on):
    """Tangents, vmap, second derivatives and a step compiled (and captured) agree with the plain call."""
    case = (2, 5, 4, 4, 32, 16, False, "fp32", "qk", True, 3, "int32")
    q, k, cq, ck, gq, gk, pos = make(case, on)
    q[0, 0, 0] = 0.25
    kw = dict(eps=EPS, rotary_dim=16)
    f = lambda *x: F.norm_rotary(x[0], x[1], T(pos), *x[2:], **kw)  # noqa: E731
    xs = [T(x) for x in (q, k, gq, gk)]
    way = [T(torch.randn_like(x)) for x in (q, k, gq, gk)]
    y, tangent = nb.jvp(f, tuple(xs), tuple(way))
    _, pull = nb.vjp(f, *xs, create_graph=False)
    grads = pull((T(cq), T(ck)))
    a = sum((t.to_torch().double() * c.double()).sum().item() for t, c in zip(tangent, (cq, ck)))
    b = sum((u.to_torch().double() * w.to_torch().double()).sum().item() for u, w in zip(grads, way))
    size = sum((u.to_torch().double() * w.to_torch().double()).abs().sum().item() for u, w in zip(grads, way))
    assert abs(a - b) <= 2.0 ** -17 * size                       # both are the same sum of products with fp32 factors
    # a batch of calls
    many = nb.vmap(lambda x, z: F.norm_rotary(x, z, T(pos), T(gq), T(gk), **kw))(T(torch.stack([q, 2 * q])), T(torch.stack([k, 3 * k])))
    one = f(T(2 * q), T(3 * k), T(gq), T(gk))
    for u, w in zip(many, one):
        assert (u.to_torch()[1] - w.to_torch()).abs().max() <= 2.0 ** -17 * w.to_torch().abs().max()

    # the gradient of a gradient, along a direction
    def slope(x):
        grad = nb.grad(lambda z: (lambda o: (o[0] * T(cq)).sum() + (o[1] * T(ck)).sum())(F.norm_rotary(z, T(k), T(pos), T(gq), T(gk), **kw)))(x)
        return (grad * way[0]).sum()

    got = nb.grad(slope)(xs[0]).to_torch().double()
    x64, g64, w64 = q.double().requires_grad_(True), gq.double(), way[0].to_torch().double()

    def torch_value(x):
        z = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * g64
        dz = turn64(cq.double(), spread(pos, q), 16, 10000.0, False, back=True)
        return (z * dz).sum()

    (first,) = torch.autograd.grad(torch_value(x64), x64, create_graph=True)
    (want,) = torch.autograd.grad((first * w64).sum(), x64)
    assert (got - want).abs().max() <= 2.0 ** -14 * want.abs().max()     # some tens of fp32 operations on numbers up to 2^3 times the result
    step = nb.compile(lambda q, k, a, b: (lambda y, pull: (y, pull((T(cq), T(ck)))))(*nb.vjp(f, q, k, a, b, create_graph=False)), cuda_graph=on == "cuda")
    for _ in range(3):
        y2, grads2 = step(*xs)
        plain_y, plain_pull = nb.vjp(f, *xs, create_graph=False)
        for u, w in zip((*y2, *grads2), (*plain_y, *plain_pull((T(cq), T(ck))))):
            assert torch.equal(u.to_torch(), w.to_torch())


@pytest.mark.parametrize("axes", [("dp", None, None), (None, "dp", None), (None, None, "tp"), ("dp", None, "tp")])
def test_split_over_a_mesh(axes, mesh_2x4, monkeypatch):
    monkeypatch.setenv("NABLA_B200_FUSED", "1")
    g = torch.Generator().manual_seed(4)
    b, t, h, d = 4, 6, 8, 32
    q, k = (torch.randn((b, t, h, d), generator=g) for _ in range(2))
    qkv = torch.randn((b, t, 3 * h * d), generator=g)
    gq, gk = torch.randn((d,), generator=g), torch.randn((d,), generator=g)
    pos = T(torch.arange(t))

    def both(q, k, qkv, gq, gk):
        y = F.norm_rotary(q, k, pos, gq, gk)
        return y[0].sum() + (y[1] * y[1] * y[1]).sum() + (F.packed_norm_rotary(qkv, d, pos, gq, gk) * 0.5).sum()

    plain = nb.grad(both, argnums=(0, 1, 2, 3, 4))(*(T(x) for x in (q, k, qkv, gq, gk)))
    split = [T(x).shard(mesh_2x4, (*axes, None)) for x in (q, k)] + [T(qkv).shard(mesh_2x4, axes)] + [T(x).shard(mesh_2x4, (None,)) for x in (gq, gk)]
    got = nb.grad(both, argnums=(0, 1, 2, 3, 4))(*split)
    for a, c in zip(got, plain):
        a, c = torch.from_numpy(a.to_numpy()).double(), c.to_torch().double()
        assert (a - c).abs().max() <= 2.0 ** -15 * c.abs().max()         # the same fp32 sums in parts


@pytest.mark.parametrize("heads_", [(8, 1), (1, 8), (8, 2), (6, 3), (1, 1)])
@pytest.mark.parametrize("axes", [("dp", None, "tp"), (None, "dp", "tp"), (None, "tp", None)])
def test_unlike_counts_of_heads_split_over_a_mesh(axes, heads_, mesh_2x4, monkeypatch):
    """One head is whole on every device and others are not: its gain's gradient is a sum over tokens, not over devices."""
    monkeypatch.setenv("NABLA_B200_FUSED", "1")
    g = torch.Generator().manual_seed(5)
    b, t, d = 2, 8, 32
    xs = [torch.randn((b, t, n, d), generator=g) for n in heads_] + [torch.randn((d,), generator=g) for _ in range(2)]
    cots = [torch.randn((b, t, n, d), generator=g) for n in heads_]
    pos = T(torch.arange(t))

    def value(q, k, gq, gk):
        y = F.norm_rotary(q, k, pos, gq, gk)
        return (y[0] * T(cots[0])).sum() + (y[1] * T(cots[1])).sum()

    plain = nb.grad(value, argnums=(0, 1, 2, 3))(*(T(x) for x in xs))
    for k_axes in (axes, (*axes[:2], None)):
        split = [T(xs[0]).shard(mesh_2x4, (*axes, None)), T(xs[1]).shard(mesh_2x4, (*k_axes, None))] + [T(x).shard(mesh_2x4, (None,)) for x in xs[2:]]
        y = F.norm_rotary(*split[:2], pos, *split[2:])
        for a, c in zip(y, F.norm_rotary(*(T(x) for x in xs[:2]), pos, *(T(x) for x in xs[2:]))):
            assert torch.equal(torch.from_numpy(a.to_numpy()), c.to_torch())         # the same operations, head by head
        for a, c in zip(nb.grad(value, argnums=(0, 1, 2, 3))(*split), plain):
            a, c = torch.from_numpy(a.to_numpy()).double(), c.to_torch().double()
            assert (a - c).abs().max() <= 2.0 ** -15 * c.abs().max()     # the same fp32 sums in parts


def test_refusals():
    q, k, pos = T(torch.zeros(2, 3, 4, 64)), T(torch.zeros(2, 3, 2, 64)), T(torch.zeros(3, dtype=torch.int32))
    gain = T(torch.ones(64))
    assert F.norm_rotary(q, k, pos, gain, gain)[1].shape == k.shape
    for error, args, kw in [
        (TypeError, (q, k, pos, T(torch.ones(64, dtype=torch.bfloat16))), {}),
        (ValueError, (q, k, pos, T(torch.ones(32))), {}),
        (TypeError, (q, k, T(torch.zeros(3))), {}),
        (ValueError, (q, k, T(torch.zeros(2, dtype=torch.int32))), {}),
        (TypeError, (q, k, [0, 1, 2]), {}),
        (TypeError, (q.to_torch(), k, pos), {}),
        (ValueError, (q, T(torch.zeros(2, 4, 2, 64)), pos), {}),
        (ValueError, (q, T(torch.zeros(2, 3, 2, 32)), pos), {}),
        (ValueError, (q, T(torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16)), pos), {}),
        (TypeError, (T(torch.zeros(2, 3, 4, 64, dtype=torch.float64)), k, pos), {}),
        (ValueError, (T(torch.zeros(2, 3, 4, 72)), T(torch.zeros(2, 3, 4, 72)), pos), {}),
        (ValueError, (T(torch.zeros(2, 3, 4, 272)), T(torch.zeros(2, 3, 4, 272)), pos), {}),
        (ValueError, (q, k, pos), {"rotary_dim": 24}), (ValueError, (q, k, pos), {"rotary_dim": 80}), (ValueError, (q, k, pos), {"rotary_dim": 0}),
        (ValueError, (q, k, pos), {"eps": 0.0}), (ValueError, (q, k, pos), {"base": -1.0}),
    ]:
        with pytest.raises(error):
            F.norm_rotary(*args, **kw)
    with pytest.raises(ValueError):
        F.packed_norm_rotary(T(torch.zeros(2, 3, 100)), 64, pos)
    with pytest.raises(ValueError):
        F.packed_norm_rotary(q, 64, pos)
    assert heads.MOST_DIM == 256


@pytest.mark.gpu
def test_compiled_calls_are_written_down():
    """Forward and backward of both forms are replayed without Python: recorded at the second call of a signature."""
    from nabla_b200.transforms import tape

    if tape.module() is None:
        pytest.skip("libnb_replay.so is not built here")
    q, k, cq, ck, gq, gk, pos = make(CASES[8], "cuda")
    b, t, h, d = q.shape
    qkv = torch.stack([q, k, q], 3).reshape(b, t, -1)
    f = nb.compile(lambda q, k, p, a, b, cq, ck: (lambda y, pull: (y, pull((cq, ck))))(*nb.vjp(lambda *x: F.norm_rotary(x[0], x[1], p, *x[2:]), q, k, a, b, create_graph=False)))
    g = nb.compile(lambda x, p, a, b, c: (lambda y, pull: (y, pull(c)))(*nb.vjp(lambda *z: F.packed_norm_rotary(z[0], d, p, *z[1:]), x, a, b, create_graph=False)))
    for call, args in ((f, (q, k, pos, gq, gk, cq, ck)), (g, (qkv, pos, gq, gk, qkv.clone()))):       # (arguments that share memory are not taken)
        for _ in range(4):
            call(*(T(x) for x in args))
        assert call._taped is not None and bool(call._taped[0]), call.tape_refused
