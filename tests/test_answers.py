"""The decoder with rotated and normed heads: trained, split over a mesh, and answering prompts behind a prefix with drawn tokens."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import nabla_b200 as nb
from nabla_b200 import nn
from nabla_b200.models import generate as G
from nabla_b200.models import transformer as M

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def T(x):
    return nb.Tensor.from_torch(x)


def small(device, dtype, qk_norm=True, **kw):
    cfg = M.TransformerConfig(**{**dict(n_layers=2, d_model=256, n_heads=4, d_ff=512, vocab=1000, max_seq=256, dtype=dtype, rotary_base=10000.0, qk_norm=qk_norm), **kw})
    with nb.default_device(nb.Accelerator(0) if device == "cuda" else nb.CPU()):
        nb.seed(1)
        params = M.init_params(cfg)
        if qk_norm:           # gains that are no ones, and weights that make heads differ
            g = torch.Generator().manual_seed(2)
            for p in params["layers"]:
                for name in ("q_gain", "k_gain"):
                    p[name] = T((1 + 0.3 * torch.randn(cfg.head_dim, generator=g)).to(p[name].dtype.to_torch()).to(device))
        return cfg, params


@pytest.mark.parametrize("fused", ["0", "1"])
@pytest.mark.parametrize("qk_norm", [False, True])
def test_forward_and_training(qk_norm, fused, monkeypatch):
    """Logits of a plain implementation, gradients of every parameter, split over a mesh and not."""
    monkeypatch.setenv("NABLA_B200_FUSED", fused)
    cfg, params = small("cpu", nb.DType.float32, qk_norm, d_model=64, n_heads=4, d_ff=64, vocab=48, max_seq=8)
    assert "pos_emb" not in params and ("q_gain" in params["layers"][0]) == qk_norm
    assert sum(int(np.prod([int(n) for n in t.shape])) for t in nb.tree_leaves(params)) == cfg.num_params()
    rng = np.random.default_rng(0)
    tok, tgt = nb.constant(rng.integers(0, 48, (4, 8))), nb.constant(rng.integers(0, 48, (4, 8)))
    logits = M.forward(params, tok, cfg).to_numpy()
    np.testing.assert_allclose(logits, M.torch_reference_forward(params, torch.from_numpy(tok.to_numpy()), cfg).numpy(), rtol=1e-3, atol=1e-4)
    loss, grads = nb.value_and_grad(lambda p: M.loss_fn(p, tok, tgt, cfg), create_graph=False)(params)
    mesh = nb.DeviceMesh("m", (2, 2), ("dp", "tp"))
    split = M.place_params(params, mesh, "tp")
    loss2, grads2 = nb.value_and_grad(lambda p: M.loss_fn(p, tok.shard(mesh, ("dp", None)), tgt.shard(mesh, ("dp", None)), cfg), create_graph=False)(split)
    assert abs(loss.item() - loss2.item()) < 1e-5
    for a, b in zip(nb.tree_leaves(grads), nb.tree_leaves(grads2)):
        np.testing.assert_allclose(b.to_numpy(), a.to_numpy(), rtol=1e-3, atol=1e-5)
    assert all(np.abs(t.to_numpy()).max() > 0 for t in nb.tree_leaves(grads))
    sp = M.SeqParallel(mesh)
    loss3 = M.loss_fn(split, tok.shard(mesh, ("dp", None)), tgt.shard(mesh, ("dp", None)), cfg, sp)
    assert abs(loss.item() - loss3.item()) < 1e-5
    with pytest.raises(ValueError):
        M.TransformerConfig(qk_norm=True)


@pytest.mark.gpu
def test_training_step_on_the_gpu():
    """A compiled step, plain and captured, against the same step in fp32 from primitive operations."""
    cfg, params = small("cuda", nb.DType.bfloat16)
    rng = np.random.default_rng(1)
    tok, tgt = (T(torch.from_numpy(rng.integers(0, cfg.vocab, (4, 100))).cuda()) for _ in range(2))
    f = lambda p, a, b: nb.value_and_grad(lambda q: M.loss_fn(q, a, b, cfg), create_graph=False)(p)  # noqa: E731
    want_loss, want = f({**{k: nb.cast(v, nb.DType.float32) for k, v in params.items() if k != "layers"},
                         "layers": [{k: nb.cast(v, nb.DType.float32) for k, v in p.items()} for p in params["layers"]]}, tok, tgt)
    for step in (nb.compile(f), nb.compile(f, cuda_graph=True)):
        for _ in range(3):
            loss, grads = step(params, tok, tgt)
            assert abs(loss.item() - want_loss.item()) < 0.02 * want_loss.item()
            # some tens of roundings to 8 bits between a gradient and its parameter, most of them of independent numbers
            for a, b in zip(nb.tree_leaves(grads), nb.tree_leaves(want)):
                a, b = a.to_torch().float(), b.to_torch().float()
                assert (a - b).norm() <= 0.08 * b.norm() + 1e-6


@pytest.mark.parametrize("device", DEVICES)
def test_decoding_behind_a_prefix(device):
    """Pieces of sequences over the cache give the logits of the whole text, with a prefix that all share and without."""
    cfg, params = small(device, nb.DType.float32)
    g = torch.Generator().manual_seed(31)
    P, n = 41, 50
    text = torch.randint(0, cfg.vocab, (3, P + n), generator=g)
    text[:, :P] = text[0, :P]
    text = text.to(device)
    want = M.forward(params, T(text), cfg).to_torch()
    caches, table, prefix_table = G.init_caches(cfg, 3, n, 16, device=params["tok_emb"].device, prefix_tokens=P)
    zero = torch.zeros(1, dtype=torch.int32, device=device)
    logits, caches = G.decode(params, T(text[:1, :P].contiguous()), caches, T(prefix_table.to_torch()[None]), T(zero), cfg)
    got, done = [logits.to_torch().expand(3, -1, -1)], 0
    length = T(torch.tensor([P], dtype=torch.int32, device=device))
    for m in (30, 1, 18, 1):
        past = torch.full((3,), done, dtype=torch.int32, device=device)
        logits, caches = G.decode(params, T(text[:, P + done:P + done + m].contiguous()), caches, table, T(past), cfg, prefix=(prefix_table, length))
        got.append(logits.to_torch())
        done += m
    # keys and values in 127 steps to their block's largest, as without a prefix
    assert (torch.cat(got, 1) - want).norm() < 0.02 * want.norm()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rotary", [None, 10000.0])
def test_answers_behind_a_prefix(rotary, device):
    """Prompts behind a prefix of whole blocks, and the whole texts as prompts: each answer fits the logits that the plain forward pass gives for its own text.

    The two need not be the same token by token: keys and values are rounded to 127 steps, and a sum of fp32 in another order may move one by a step. Logits of
    the cache are off by 2 % of their size (``test_decoding_behind_a_prefix``). A weight exp(z / T) is then off by a factor of 1 + e / T with e the error of
    its logit, and a share of the sum by no more than the mean of |e| / T over the distribution: 2 % of the rms of the logits, over T, and no draw so far
    from the mean that four times this does not hold it."""
    cfg, params = small(device, nb.DType.float32, rotary is not None, rotary_base=rotary)
    g = torch.Generator().manual_seed(4)
    prefix = torch.randint(0, cfg.vocab, (48,), generator=g).tolist()
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (5, 1, 33)]
    whole = [prefix + p for p in prompts]
    for kw in ({}, {"temperature": 0.8, "seed": 3}, {"temperature": 0.8, "top_k": 50, "seed": 3},
               {"temperature": 1.5, "top_p": 0.9, "min_p": 0.01, "repetition": 1.2, "presence": 0.3, "piece": 20}):
        a = G.generate(params, prompts, cfg, 10, block_size=16, prefix=prefix, **kw)
        assert a == G.generate(params, prompts, cfg, 10, block_size=16, prefix=prefix, **kw)
        assert [len(x) for x in a] == [10] * 3 and all(0 <= t < cfg.vocab for x in a for t in x)
        if len(kw) > 2:
            continue
        b = G.generate(params, whole, cfg, 10, block_size=16, **kw)
        uniform = torch.rand((10, 3), generator=torch.Generator().manual_seed(kw.get("seed", 0)))
        for answers in (a, b):
            for i, answer in enumerate(answers):
                text = torch.tensor([whole[i] + answer])
                z = M.forward(params, T(text.to(device)), cfg).to_torch()[0, len(whole[i]) - 1:-1].double().cpu()
                off = 4 * 0.02 * z.pow(2).mean().sqrt().item()
                for step, token in enumerate(answer):
                    if not kw:
                        assert z[step, token] >= z[step].max() - off
                        continue
                    w = torch.exp(z[step] / kw["temperature"])
                    upto = w.cumsum(0) / w.sum()
                    before = upto[token] - w[token] / w.sum()
                    assert before - off / kw["temperature"] <= uniform[step, i] <= upto[token] + off / kw["temperature"]
    with pytest.raises(ValueError):
        G.generate(params, prompts, cfg, 10, temperature=-1.0)
    with pytest.raises(ValueError):
        G.generate(params, prompts, cfg, 10, prefix=prefix * 5)


@pytest.mark.parametrize("device", DEVICES)
def test_drawn_answers(device):
    """Random numbers decide; a grammar and filters are kept to; one token left is that token; none left is token 0."""
    cfg, params = small(device, nb.DType.float32 if device == "cpu" else nb.DType.bfloat16)
    prompts = [[5, 7, 9], [1], list(range(40))]
    hot = {"temperature": 2.0}
    a = G.generate(params, prompts, cfg, 12, block_size=16, seed=1, **hot)
    assert a != G.generate(params, prompts, cfg, 12, block_size=16, seed=2, **hot)
    likeliest = G.generate(params, prompts, cfg, 12, block_size=16)
    assert G.generate(params, prompts, cfg, 12, block_size=16, top_k=1, **hot) == likeliest
    words = torch.zeros((3, -(-cfg.vocab // 32)), dtype=torch.int32)
    words[:, 3] = 0b1010
    words[1] = 0
    words[2, 3] = 0b1000
    b = G.generate(params, prompts, cfg, 12, block_size=16, allowed=T(words.to(device)), **hot)
    assert set(b[0]) <= {97, 99} and b[1] == [0] * 12 and b[2] == [99] * 12


@pytest.mark.parametrize("device", DEVICES)
def test_a_draw_gets_the_filters_in_effect(device, monkeypatch):
    """Those that let all through are not handed on; a share of 0 leaves the likeliest, as no other filter does."""
    cfg, params = small(device, nb.DType.float32, max_seq=97)            # (compiled for itself: the calls are seen while they are)
    seen, sample = [], G.F.sample_tokens
    monkeypatch.setattr(G.F, "sample_tokens", lambda logits, uniform, **kw: (seen.append(set(kw)), sample(logits, uniform, **kw))[1])
    prompts = [[5, 7, 9], [1]]
    for kw, want in (({}, set()), ({"top_k": 0, "top_p": 1.0, "min_p": 0.0}, set()), ({"top_k": 5}, {"top_k"}), ({"top_p": 0.5}, {"top_p"}),
                     ({"min_p": 0.1}, {"min_p"}), ({"top_k": 9, "top_p": 0.0, "min_p": 0.2}, {"top_k", "top_p", "min_p"}), ({"top_k": -3, "min_p": -1.0}, set())):
        seen.clear()
        G._steps.cache_clear()
        answers = G.generate(params, prompts, cfg, 5, block_size=16, temperature=0.7, seed=2, **kw)
        assert seen and all(names == want | {"temperature"} for names in seen)
        if kw.get("top_p") == 0.0:
            assert answers == G.generate(params, prompts, cfg, 5, block_size=16)
    G._steps.cache_clear()


def misfits(cfg, params, device, texts, answers, uniform, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """How many tokens of ``answers`` the logits of ``texts`` with these answers do not bear out.

    Logits of the cache are off by 2 % of their rms (``test_decoding_behind_a_prefix``), four times that is allowed: ``off``. Where nothing is filtered the random number
    has to lie in the token's share of the sum, which an error e of logits moves by no more than the mean of |e| / T. A filter's border and the token's own logit are
    each off by ``off``; for top-p, the share in front of the token as above. Shares in the order of ids say little of a text: where nothing is filtered, the logarithms of the
    drawn tokens' shares also have to add up to what draws give, to four standard deviations, or none of them fits."""
    bad, less, variance, allowed = 0, 0.0, 0.0, 0.0
    for i, (text, answer) in enumerate(zip(texts, answers)):
        z = M.forward(params, T(torch.tensor([text + answer]).to(device)), cfg).to_torch()[0, len(text) - 1:-1].double().cpu()
        off = 4 * 0.02 * z.pow(2).mean().sqrt().item()
        for step, token in enumerate(answer):
            w = torch.softmax(z[step] / temperature, 0)
            own = z[step, token]
            if not top_k and top_p >= 1 and not min_p:
                upto = w.cumsum(0)[token]
                bad += not upto - w[token] - off / temperature <= uniform[step, i] <= upto + off / temperature
                log = torch.log_softmax(z[step] / temperature, 0)
                mean = (w * log).sum()
                less, variance, allowed = less + mean - log[token], variance + (w * (log - mean) ** 2).sum(), allowed + off / temperature
                continue
            fits = not top_k or own >= z[step].topk(top_k).values[-1] - 2 * off
            fits &= top_p >= 1 or w[z[step] > own + 2 * off].sum() < top_p + off / temperature
            fits &= not min_p or (own - z[step].max()) / temperature >= np.log(min_p) - 2 * off / temperature
            bad += not fits
    return bad if less <= 4 * variance ** 0.5 + allowed else uniform.numel()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rotary", [None, 10000.0])
def test_draws_fit_the_logits_of_their_own_texts(rotary, device):
    """Steep distributions (logits of some 3 T): drawn tokens fit the texts that they stand behind, and not those behind another prefix, nor does a draw
    that does not look at the logits."""
    cfg, params = small(device, nb.DType.float32, rotary is not None, rotary_base=rotary)
    params["lm_head"] = T(params["lm_head"].to_torch() * 8.0)
    for p in params["layers"]:                        # what attention adds outweighs the tokens themselves
        p["wo"] = T(p["wo"].to_torch() * 16.0)
    g = torch.Generator().manual_seed(14)
    prefix, other = (torch.randint(0, cfg.vocab, (41,), generator=g).tolist() for _ in range(2))
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (5, 1, 33)]
    texts, seed, n = [prefix + p for p in prompts], 6, 12
    uniform = torch.rand((n, 3), generator=torch.Generator().manual_seed(seed))
    for kw in ({}, {"top_k": 3}, {"top_p": 0.3}, {"min_p": 0.3}, {"top_k": 20, "top_p": 0.5, "min_p": 0.1}):
        kw = {"temperature": 0.8, **kw}
        fit = lambda answers: misfits(cfg, params, device, texts, answers, uniform, **kw)  # noqa: E731
        assert fit(G.generate(params, prompts, cfg, n, block_size=16, prefix=prefix, seed=seed, **kw)) == 0
        assert fit(G.generate(params, texts, cfg, n, block_size=16, seed=seed, **kw)) == 0
        assert fit(G.generate(params, prompts, cfg, n, block_size=16, prefix=other, seed=seed, **kw)) >= 3
        assert fit(G.generate(params, prompts, cfg, n, block_size=16, seed=seed, **kw)) >= 3
        assert fit([[int(u * cfg.vocab) for u in uniform[:, i]] for i in range(3)]) >= 3
