"""Compiled calls that were written down (``transforms/tape.py``) against the same calls run by Python. Needs a B200."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _wrap(t):
    import nabla_b200 as nb

    return nb.Tensor.from_torch(t)


def _leaves(out):
    from nabla_b200.core.common import pytree

    return [x.to_torch() if hasattr(x, "to_torch") else torch.tensor(x) for x in pytree.tree_leaves(out)]


def _taped(f):
    return f._taped is not None and bool(f._taped[0])


def _functions():
    """(function, inputs of a seed): one per family of launch functions."""
    import nabla_b200 as nb
    from nabla_b200.nn import functional as F

    def g(seed):
        return torch.Generator("cuda").manual_seed(seed)

    def r(s, *shape, dtype=BF16, std=1.0):
        return (torch.randn(shape, generator=g(s + sum(shape)), device="cuda") * std).to(dtype)

    def grads(f, primals, cot):
        y, pull = nb.vjp(f, *primals, create_graph=False)
        return (y, *pull(cot))

    def ids(s, *shape, high=50):
        return torch.randint(0, high, shape, generator=g(s), device="cuda")

    return {
        "norm": (lambda x, a, b, dy: grads(lambda *t: F.layer_norm(*t), (x, a, b), dy),
                 lambda s: [r(s, 70, 256), r(s, 256), r(s + 1, 256), r(s + 2, 70, 256)]),
        "mlp": (lambda x, w, b, v, dy: {"y": grads(lambda *t: F.linear(F.linear(t[0], t[1], t[2], activation="gelu"), t[3]), (x, w, b, v), dy), "n": [None, 3]},
                lambda s: [r(s, 100, 64), r(s, 64, 128, std=0.1), r(s, 128), r(s, 128, 64, std=0.1), r(s + 1, 100, 64)]),
        "attention": (lambda q, k, v, m, do: grads(lambda *t: F.scaled_dot_product_attention(*t, attn_mask=m), (q, k, v), do),
                      lambda s: [r(s, 2, 4, 130, 64), r(s + 1, 2, 4, 130, 64), r(s + 2, 2, 4, 130, 64), r(s, 2, 1, 1, 130, dtype=F32), r(s + 3, 2, 4, 130, 64)]),
        "decode": (lambda q, k, v: F.scaled_dot_product_attention(q, k, v, is_causal=True), lambda s: [r(s, 2, 4, 1, 128), r(s, 2, 4, 700, 128), r(s + 1, 2, 4, 700, 128)]),
        "head": (lambda x, w, t: nb.value_and_grad(lambda x, w: F.cross_entropy_loss(F.linear(x, w), t), argnums=(0, 1), create_graph=False)(x, w),
                 lambda s: [r(s, 60, 64), r(s, 64, 208, std=0.1), ids(s, 60, high=208)]),
        "embedding": (lambda t, p, i, dy: grads(lambda a, b: F.embedding(i, a) + b, (t, p), dy),
                      lambda s: [r(s, 50, 64), r(s, 9, 64), ids(s, 3, 9), r(s, 3, 9, 64)]),
        "pointwise": (lambda a, b: [nb.exp(a) * b + a, {"s": nb.reduce_sum(a * b, axis=0)}], lambda s: [r(s, 33, 40, dtype=F32), r(s + 1, 33, 40, dtype=F32)]),
    }


@pytest.mark.parametrize("name", ["norm", "mlp", "attention", "decode", "head", "embedding", "pointwise"])
@pytest.mark.parametrize("graph", [False, True])
def test_taped_calls_give_what_python_gives(name, graph, monkeypatch):
    """New inputs and new addresses on every call, results kept: bit for bit but for sums by atomics."""
    import nabla_b200 as nb

    fn, inputs = _functions()[name]
    f = nb.compile(fn, cuda_graph=graph)
    monkeypatch.setenv("NABLA_B200_TAPE", "0")
    plain = nb.compile(fn, cuda_graph=graph)
    want = [_leaves(plain(*map(_wrap, inputs(s)))) for s in range(6)]
    assert not _taped(plain)
    monkeypatch.delenv("NABLA_B200_TAPE")
    keep = []
    for s in range(6):
        args = inputs(s)
        out = f(*map(_wrap, args))
        keep.append((args, out))
        assert s < 1 or _taped(f), f.tape_refused
    for (_, out), w in zip(keep, want):
        got = _leaves(out)
        assert len(got) == len(w)
        for a, b in zip(got, w):
            assert a.shape == b.shape and a.dtype == b.dtype and a.stride() == b.stride()
            assert torch.equal(a, b) or (name == "embedding" and (a.float() - b.float()).norm() < 4e-3 * b.float().norm())
    assert f.stats.hits == 5


def test_calls_that_are_not_the_one_that_was_written_down(monkeypatch):
    """Other strides, alignments, shapes, types, structures, shared memory and switches go another way and are right."""
    import nabla_b200 as nb

    f = nb.compile(lambda d: d["a"] * d["b"][0] + nb.reduce_sum(d["a"], axis=0))
    x, y = torch.randn(32, 64, device="cuda"), torch.randn(32, 64, device="cuda")

    def check(a, b, container=list):
        out = f({"a": _wrap(a), "b": container([_wrap(b)])}).to_torch()
        assert torch.allclose(out, a * b + a.sum(0), atol=1e-4), f.tape_refused

    for _ in range(3):
        check(x, y)
    assert _taped(f)
    check(x, x)                                       # one tensor twice
    check(x.t().contiguous().t(), y)                  # columns first
    off = torch.randn(32 * 64 + 1, device="cuda")[1:].view(32, 64)
    check(off, y)                                     # on a 4-byte boundary
    check(x, y, tuple)
    check(x[:16].contiguous(), y[:16].contiguous())
    for _ in range(3):
        check(x, y)
    assert _taped(f)
    out = f({"a": _wrap(x.to(BF16)), "b": [_wrap(y.to(BF16))]}).to_torch()
    assert out.dtype == BF16
    for _ in range(2):
        check(x, y)
    monkeypatch.setenv("NABLA_B200_DISABLE_NATIVE", "1")
    check(x, y)
    monkeypatch.delenv("NABLA_B200_DISABLE_NATIVE")
    with pytest.raises(Exception):
        f({"a": _wrap(x)})
    check(x, y)


def test_arguments_that_share_memory_are_not_written_down():
    """Written down with both arguments in one place, a call could not tell them apart later."""
    import nabla_b200 as nb

    f = nb.compile(lambda a, b: a * b + a)
    x, y, z = (torch.randn(40, 8, device="cuda") for _ in range(3))
    f(_wrap(x), _wrap(x))
    f(_wrap(x), _wrap(x))
    assert not _taped(f) and "share" in f.tape_refused
    for a, b in ((x, y), (y, z), (z, z), (x, z)):
        assert torch.equal(f(_wrap(a), _wrap(b)).to_torch(), a * b + a)
    assert _taped(f)


def test_captured_tensors_and_results_that_alias():
    import nabla_b200 as nb

    w, x = torch.randn(16, 16, device="cuda"), torch.randn(4, 16, device="cuda")
    held = _wrap(w)
    f = nb.compile(lambda a: a * 2.0 + nb.reduce_sum(held * 1.0, axis=0))
    for _ in range(3):
        assert torch.allclose(f(_wrap(x)).to_torch(), x * 2 + w.sum(0), atol=1e-4)
    assert _taped(f)
    w.add_(1.0)                                       # in place: read anew on every call
    assert torch.allclose(f(_wrap(x)).to_torch(), x * 2 + w.sum(0), atol=1e-4)
    other = torch.randn(16, 16, device="cuda")
    held._impl._buffers = [other]
    assert torch.allclose(f(_wrap(x)).to_torch(), x * 2 + other.sum(0), atol=1e-4)
    g = nb.compile(lambda a: (a, nb.reshape(a, (-1,)), a + 1.0))
    for _ in range(4):
        assert [t.shape for t in _leaves(g(_wrap(x)))] == [x.shape, (x.numel(),), x.shape]
    assert not _taped(g)
    h = nb.compile(lambda a: nb.uniform((8,), device=a.device) + a)
    draws = [h(_wrap(torch.zeros(8, device="cuda"))).to_torch() for _ in range(4)]
    assert not _taped(h) and not any(torch.equal(draws[0], d) for d in draws[1:])


def test_taped_calls_on_streams_and_threads():
    import nabla_b200 as nb
    from nabla_b200.nn import functional as F

    f = nb.compile(lambda x, a, b: F.layer_norm(F.layer_norm(x, a, b), a, b))
    args = [(torch.randn(3000, 512, device="cuda") * (k + 1)).to(BF16) for k in range(8)]
    a, b = torch.ones(512, device="cuda", dtype=BF16), torch.zeros(512, device="cuda", dtype=BF16)
    want = [f(_wrap(x), _wrap(a), _wrap(b)).to_torch() for x in args]
    assert _taped(f)
    torch.cuda.synchronize()
    bad = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(30):
                x = args[(k + i) % 8].clone()
                out = f(_wrap(x), _wrap(a), _wrap(b)).to_torch()
                if not torch.equal(out, want[(k + i) % 8]):
                    bad.append((k, i))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_large_arguments_of_a_captured_function_are_not_copied():
    """Few launches on large tensors are written down and not captured; a call that does not match is captured and right, and so is
    the next that matches."""
    import nabla_b200 as nb

    f = nb.compile(lambda x, w: x @ w, cuda_graph=True)
    g = torch.Generator("cuda").manual_seed(3)
    xs = [torch.randn(4096, 4096, generator=g, device="cuda").to(BF16) for _ in range(3)]
    w = (torch.randn(4096, 2048, generator=g, device="cuda") * 0.02).to(BF16)
    want = [(x.double() @ w.double()) for x in xs]

    def check(k, x):
        out = f(_wrap(x), _wrap(w)).to_torch().double()
        assert (out - want[k]).norm() < 4e-3 * want[k].norm()

    for k, x in enumerate(xs):
        check(k, x)
    assert _taped(f) and f.stats.cuda_graphs == 0
    check(1, xs[1].t().contiguous().t())
    assert f.stats.cuda_graphs == 1
    for k, x in enumerate(xs):
        check(k, x)
    small = nb.compile(lambda x, w: x @ w, cuda_graph=True)
    for k in range(3):
        out = small(_wrap(xs[k][:64]), _wrap(w[:, :64].contiguous())).to_torch().double()
        assert torch.allclose(out, want[k][:64, :64], atol=0.1)
    assert small.stats.cuda_graphs == 1 and _taped(small)


@pytest.mark.parametrize("name", list(_functions()) if torch.cuda.is_available() else ["norm"])
@pytest.mark.parametrize("graph", [False, True])
def test_calls_in_a_row_read_their_own_inputs(name, graph):
    """Launches that are resident before the ones ahead have ended: forty calls without a synchronisation, each on other values in the same
    memory, give what calls alone give."""
    import nabla_b200 as nb

    fn, inputs = _functions()[name]
    f, plain = nb.compile(fn, cuda_graph=graph), nb.compile(fn)
    sets = [inputs(k) for k in range(4)]
    want = []
    for s in sets:
        want.append([t.clone() for t in _leaves(plain(*map(_wrap, s)))])
        torch.cuda.synchronize()
    held = [t.clone() for t in sets[0]]
    got = []
    for k in range(40):
        for h, t in zip(held, sets[k % 4]):
            h.copy_(t)
        got.append([t.clone() for t in _leaves(f(*map(_wrap, held)))])
    torch.cuda.synchronize()
    for k, outs in enumerate(got):
        for a, b in zip(outs, want[k % 4]):
            assert torch.equal(a, b), k


@pytest.mark.parametrize("graph", [False, True])
def test_a_training_run_of_calls_in_a_row(graph):
    """Two hundred steps of a small network with AdamW, parameters, moments and step count from each to the next, against the same steps
    with a synchronisation after each: equal bit for bit."""
    import nabla_b200 as nb
    from nabla_b200.nn import functional as F

    def step(params, state, x, y):
        def loss(p):
            return F.mse_loss(F.linear(F.linear(x, p["w0"], p["b0"], activation="relu"), p["w1"], p["b1"]), y)

        value, grads = nb.value_and_grad(loss, create_graph=False)(params)
        params, state = nb.nn.adamw_update(params, grads, state, lr=1e-2, weight_decay=0.01, realize=False)
        return value, params, state

    def run(f, pause):
        gen = torch.Generator("cuda").manual_seed(5)
        shapes = {"w0": (64, 256), "b0": (256,), "w1": (256, 8), "b1": (8,)}
        p = {k: _wrap((torch.randn(s, generator=gen, device="cuda") * 0.1).to(BF16)) for k, s in shapes.items()}
        st = {"m": {k: _wrap(torch.zeros(s, device="cuda")) for k, s in shapes.items()},
              "v": {k: _wrap(torch.zeros(s, device="cuda")) for k, s in shapes.items()}, "step": _wrap(torch.tensor(0.0, device="cuda"))}
        losses = []
        for k in range(200):
            x = torch.rand(100, 64, generator=gen, device="cuda").to(BF16)
            value, p, st = f(p, st, _wrap(x), _wrap(torch.sin(x[:, :8].float() * 6).to(BF16)))
            losses.append(value)
            pause()
        return [t.clone() for t in _leaves([losses, p, st])]

    got, want = run(nb.compile(step, cuda_graph=graph), lambda: None), run(nb.compile(step), torch.cuda.synchronize)
    torch.cuda.synchronize()
    assert float(want[199]) < float(want[0])
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("graph", [False, True])
def test_constants_outlive_the_calls_of_other_streams(graph):
    """Traced on one stream, called on another that is behind, and released: the memory of what was made with the plan is not handed
    out again before that stream has read it."""
    import nabla_b200 as nb
    from nabla_b200.nn import functional as F

    def fn(x, y):
        return nb.value_and_grad(lambda x: F.mse_loss(x, y), create_graph=False)(x)

    x, y = torch.randn(512, 8, device="cuda"), torch.randn(512, 8, device="cuda")
    want = 2 * (x.double() - y.double()) / x.numel()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    f = nb.compile(fn, cuda_graph=graph)
    with torch.cuda.stream(first):
        f(_wrap(x), _wrap(y))
        rec = next(iter(next(iter(f._cache.values())).values()))
        shapes = {tuple(b.shape) for o in rec.constants for b in o._buffers}
        assert shapes
        del rec
        f(_wrap(x), _wrap(y))
        assert _taped(f), f.tape_refused
    torch.cuda.synchronize()
    with torch.cuda.stream(second):
        torch.cuda._sleep(100_000_000)                # some 50 ms
        _, g = f(_wrap(x), _wrap(y))
    f.release()
    del f
    with torch.cuda.stream(first):
        held = [torch.full(s, 1e6, device="cuda") for s in shapes for _ in range(400)]
    torch.cuda.synchronize()
    assert torch.allclose(g.to_torch().double(), want, rtol=1e-4, atol=1e-9) and held


def test_a_graph_of_the_callers_outlives_the_function():
    """A compiled function in a capture of the caller's own: dropped, its constants are still the graph's."""
    import nabla_b200 as nb
    from nabla_b200.nn import functional as F

    x, y = torch.randn(512, 8, device="cuda"), torch.randn(512, 8, device="cuda")
    f = nb.compile(lambda x, y: nb.value_and_grad(lambda x: F.mse_loss(x, y), create_graph=False)(x))
    for _ in range(3):                                # traced, written down, taped
        f(_wrap(x), _wrap(y))
    assert _taped(f), f.tape_refused
    rec = next(iter(next(iter(f._cache.values())).values()))
    shapes = {tuple(b.shape) for o in rec.constants for b in o._buffers}
    assert shapes
    del rec
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _, grad = f(_wrap(x), _wrap(y))
    f.release()
    del f
    held = [torch.full(s, 1e6, device="cuda") for s in shapes for _ in range(400)]
    x.mul_(3.0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.allclose(grad.to_torch().double(), 2 * (x.double() - y.double()) / x.numel(), rtol=1e-4, atol=1e-9) and held


def test_other_threads_run_while_a_launch_waits():
    """More launches than a stream's queue holds behind a kernel of half a second: the caller waits, and Python goes on elsewhere."""
    import time

    import nabla_b200 as nb
    from nabla_b200.nn import functional as F

    f = nb.compile(lambda x, a, b: F.layer_norm(F.layer_norm(x, a, b), a, b))
    args = [_wrap(t) for t in (torch.randn(8, 512, device="cuda"), torch.ones(512, device="cuda"), torch.zeros(512, device="cuda"))]
    for _ in range(3):
        f(*args)
    assert _taped(f), f.tape_refused
    torch.cuda.synchronize()
    done, gaps = threading.Event(), [0.0]

    def tick():
        last = time.perf_counter()
        while not done.is_set():
            time.sleep(0.002)
            now = time.perf_counter()
            gaps.append(now - last)
            last = now

    other = threading.Thread(target=tick)
    other.start()
    torch.cuda._sleep(1_000_000_000)
    t0 = time.perf_counter()
    for _ in range(2500):
        f(*args)
    waited = time.perf_counter() - t0
    done.set()
    other.join()
    torch.cuda.synchronize()
    assert waited > 0.3, "the queue was never full"
    assert max(gaps) < 0.2 * waited


@pytest.mark.parametrize("graph", [False, True])
def test_calls_of_several_signatures_in_turn(graph, monkeypatch):
    """Each signature keeps its tape whatever is called in between, an odd call of its own included; none of them is run by Python again."""
    import nabla_b200 as nb
    from nabla_b200.transforms.compile import CompiledFunction

    f = nb.compile(lambda x, w: x @ w, cuda_graph=graph)
    g = torch.Generator("cuda").manual_seed(4)
    xs = [torch.randn(n, 4096, generator=g, device="cuda").to(BF16) for n in (2048, 4096)]
    w = (torch.randn(4096, 2048, generator=g, device="cuda") * 0.02).to(BF16)
    want = [x.double() @ w.double() for x in xs]

    def check(k, x):
        assert (f(_wrap(x), _wrap(w)).to_torch().double() - want[k]).norm() < 4e-3 * want[k].norm()

    for k in (0, 0, 1, 1):                            # traced and written down, one after the other
        check(k, xs[k])
    by_python = []
    for name in ("_run", "_replay_cuda_graph"):
        monkeypatch.setattr(CompiledFunction, name, lambda self, *a, _f=getattr(CompiledFunction, name), **k: by_python.append(1) or _f(self, *a, **k))
    hits = f.stats.hits
    for _ in range(4):
        for k in (0, 1):
            check(k, xs[k])
            assert _taped(f), f.tape_refused
    assert not by_python and f.stats.hits == hits + 8 and f.stats.cuda_graphs == 0
    check(1, xs[1].t().contiguous().t())              # columns first
    assert by_python
    by_python.clear()
    for k in (1, 0, 1):
        check(k, xs[k])
        assert _taped(f)
    assert not by_python


@pytest.mark.parametrize("rows,dim", [(2048, 96), (2049, 96), (8196, 96), (600, 8200)])
def test_many_small_blocks_in_a_row(rows, dim):
    """Grids that let the next launch begin by ending, and rows that begin when all ahead has ended, between others that do neither: thirty calls
    in a row on changing inputs, against the same calls with a synchronisation after each."""
    import nabla_b200 as nb
    from nabla_b200.nn import functional as F

    def fn(table, ids, a, b, t):
        x = F.layer_norm(F.embedding(ids, table), a, b)
        return (x, *nb.value_and_grad(lambda x: F.cross_entropy_loss(x, t), create_graph=False)(x), nb.softmax(x))

    g = torch.Generator("cuda").manual_seed(rows)
    table = torch.randn(500, dim, generator=g, device="cuda")
    a, b = torch.ones(dim, device="cuda"), torch.zeros(dim, device="cuda")
    sets = [(torch.randint(0, 500, (rows,), generator=g, device="cuda"), torch.randint(0, dim, (rows,), generator=g, device="cuda")) for _ in range(3)]
    f, plain = nb.compile(fn), nb.compile(fn)
    want = []
    for i, t in sets:
        want.append([x.clone() for x in _leaves(plain(*map(_wrap, (table, i, a, b, t))))])
        torch.cuda.synchronize()
    ids, tgt, got = sets[0][0].clone(), sets[0][1].clone(), []
    for k in range(30):
        ids.copy_(sets[k % 3][0])
        tgt.copy_(sets[k % 3][1])
        got.append(_leaves(f(*map(_wrap, (table, ids, a, b, tgt)))))
    torch.cuda.synchronize()
    for k, outs in enumerate(got):
        assert all(torch.equal(x, y) for x, y in zip(outs, want[k % 3])), k
    x = want[0][0].double()
    assert torch.allclose(want[0][1].double(), torch.nn.functional.cross_entropy(x, sets[0][1]), rtol=1e-5)


def test_views_of_one_tensor_as_arguments():
    """Keys and values of a packed projection lie in each other's memory: written down for views that start as far apart, others go another way."""
    import nabla_b200 as nb

    from nabla_b200.nn import functional as F

    f = nb.compile(lambda k, v, q: F.scaled_dot_product_attention(q, k, v))
    packed, other = (torch.randn(1, 2, 40, 3, 64, device="cuda").to(BF16) for _ in range(2))
    q = _wrap(torch.randn(1, 2, 40, 64, device="cuda").to(BF16))

    def check(k, v):
        assert torch.equal(f(_wrap(k), _wrap(v), q).to_torch(), F.scaled_dot_product_attention(q, _wrap(k), _wrap(v)).to_torch())

    views = lambda t, i, j: (t[:, :, :, i], t[:, :, :, j])  # noqa: E731
    for _ in range(3):
        check(*views(packed, 0, 1))
    assert _taped(f), f.tape_refused
    check(*views(other, 0, 1))
    assert _taped(f)
    for k, v in (views(packed, 0, 2), views(packed, 1, 0), (packed[:, :, :, 0], other[:, :, :, 1]), views(other, 2, 2), views(packed, 0, 1)):
        check(k, v)


def test_results_that_are_arguments_updated_in_place():
    import nabla_b200 as nb
    from nabla_b200.nn import functional as F

    f = nb.compile(lambda cache, k, table, past: F.kv_cache_write(cache, k, k, table, past))
    table, past = (_wrap(torch.zeros(s, dtype=torch.int32, device="cuda")) for s in ((1, 1), (1,)))
    caches = [F.init_kv_cache(1, 2, 64, 16, device=table.device) for _ in range(2)]
    for cache in caches * 3:
        k = torch.randn(1, 3, 2, 64, device="cuda")
        before = {n: t.to_torch() for n, t in cache.items()}
        got = f(cache, _wrap(k), table, past)
        for n in cache:
            assert got[n].to_torch() is before[n] and got[n].to_torch().data_ptr() == before[n].data_ptr()
        want = F.kv_cache_write({n: _wrap(torch.zeros_like(t)) for n, t in before.items()}, _wrap(k), _wrap(k), table, past)
        first = lambda t: t.to_torch().reshape(1, 2, -1)[..., : 3 * 64]  # noqa: E731
        assert all(torch.equal(first(got[n]), first(want[n])) for n in got)
    assert _taped(f), f.tape_refused
