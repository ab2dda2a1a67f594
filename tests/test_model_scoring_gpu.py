"""iam_model_score against the logits of iam_model_prefill, prefix by prefix, and iam_model_set_rope against the
definition of its angles on the keys that a prefill leaves in the cache."""
import math

import numpy as np
import pytest

from test_rope_gpu import angles, config

pytestmark = pytest.mark.gpu
SMALL = dict(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, ffn_dim=512, vocab=517, max_ctx=96)


@pytest.fixture(scope="module")
def small(iam, cuda):
    m = iam.Model.random(iam.ModelConfig.make(**SMALL), seed=7)
    yield m
    m.close()


def test_score_matches_the_logits_of_every_prefix(small, iam, cuda, monkeypatch):
    """The products of the batched LM head carry 22 bits of the activations, as prefill's own logits do: log
    probabilities within 1e-3 x RMS of the logits (the prefill tests' bar)."""
    import torch
    m, vocab = small, SMALL["vocab"]
    prompt = np.random.default_rng(1).integers(0, vocab, 30).tolist()
    targets = torch.tensor(prompt[1:] + [-1], dtype=torch.int32, device="cuda")
    n, k = len(prompt), 7
    out = dict(logprob=torch.empty(n, device="cuda"), entropy=torch.empty(n, device="cuda"), rank=torch.empty(n, dtype=torch.int32, device="cuda"),
               top_logprob=torch.empty(n, k, device="cuda"), top_index=torch.empty(n, k, dtype=torch.int32, device="cuda"))
    m.reset()
    nxt = m.score(prompt, targets, **out)
    logits = torch.empty(vocab, device="cuda")
    for t in range(n):
        m.reset()
        best = m.prefill(prompt[:t + 1], 0, logits)
        x = logits.double()
        tol = 2e-3 * float(x.square().mean().sqrt())  # two logits enter a difference
        logp = torch.log_softmax(x, 0)
        if t + 1 < n:
            assert abs(float(out["logprob"][t]) - float(logp[prompt[t + 1]])) < tol
            ahead = int(out["rank"][t])
            mine = float(x[prompt[t + 1]])
            assert int((x > mine + tol).sum()) <= ahead <= int((x > mine - tol).sum())
        assert abs(float(out["entropy"][t]) + float((logp.exp() * logp).sum())) < tol * (1 + float(x.abs().max()))
        assert (out["top_logprob"][t].double() - torch.sort(logp, descending=True)[0][:k]).abs().max() < tol
        assert (logp[out["top_index"][t].long()] - out["top_logprob"][t].double()).abs().max() < tol
    assert out["logprob"][n - 1] == 0 and out["rank"][n - 1] == -1
    assert nxt == best == int(logits.argmax())


def test_score_in_two_calls_and_some_outputs(small, iam, cuda):
    import torch
    prompt = np.random.default_rng(2).integers(0, SMALL["vocab"], 24).tolist()
    targets = torch.tensor(prompt[1:] + [-1], dtype=torch.int32, device="cuda")
    whole, parts = torch.empty(24, device="cuda"), torch.empty(24, device="cuda")
    small.reset()
    small.score(prompt, targets, logprob=whole)
    small.reset()
    small.score(prompt[:10], targets[:10].contiguous(), logprob=parts[:10])
    small.score(prompt[10:], targets[10:].contiguous(), start_pos=10, logprob=parts[10:])
    assert float((whole - parts).abs().max()) < 1e-3
    ent = torch.empty(24, device="cuda")
    small.reset()
    small.score(prompt, entropy=ent)
    assert ent.isfinite().all() and (ent <= math.log(SMALL["vocab"]) + 1e-4).all()


def test_refused_scores(small, iam, cuda):
    import torch
    f = torch.empty(3, device="cuda")
    for args, kw in [(([1, 2, SMALL["vocab"]],), {}), (([1, 2, 3],), dict(logprob=f)), (([1] * 97,), {}), (([],), {}),
                     (([1, 2, 3],), dict(entropy=f[:2])), (([1, 2, 3],), dict(top_logprob=torch.empty(3, 65, device="cuda"), top_index=torch.empty(3, 65, dtype=torch.int32, device="cuda"))),
                     (([1, 2, 3],), dict(top_logprob=torch.empty(3, 2, device="cuda")))]:
        with pytest.raises(iam.IamError):
            small.score(*args, **kw)


@pytest.mark.parametrize("extra", [dict(scaling="linear", factor=4.0), dict(scaling="yarn", factor=8.0, original_ctx=2048),
                                   dict(scaling="banded", factor=8.0, original_ctx=512), dict(scaling="ntk", factor=2.0)])
def test_set_rope_turns_the_keys_by_the_scaled_angles(small, iam, cuda, extra):
    """Layer 0's keys before the rotation do not depend on it: turned back, the caches of both settings agree up to the
    fp16 rounding of each (2^-11 of a pair's length)."""
    import torch
    m, n = small, 40
    prompt = np.random.default_rng(3).integers(0, SMALL["vocab"], n).tolist()
    positions = torch.arange(n, dtype=torch.int32)

    def turned_back(cfg):
        m.reset()
        m.prefill(prompt, 0)
        k = torch.from_numpy(m.read_weight(iam.W_K_CACHE, 0).reshape(2, 96, 64)[:, :n].view(np.float16).astype(np.float64))
        cos, sin, f = angles(cfg, positions, torch)
        a, b = k[..., :32], k[..., 32:]
        return torch.cat((a * cos + b * sin, b * cos - a * sin), -1) / f, k.norm(dim=-1).max() / f

    plain, size = turned_back(config(64))
    cfg = config(64, **extra)
    try:
        m.set_rope(iam.Rope.config(**cfg))
        scaled, size2 = turned_back(cfg)
    finally:
        m.set_rope(None)
    # the default table's float angles are off by up to n 2^-24 radians, which the rounding covers
    assert float((plain - scaled).abs().max()) <= 2.0 ** -11 * float(size + size2)
    again, _ = turned_back(config(64))
    assert torch.equal(again, plain)


def test_set_rope_refusals(small, iam, cuda):
    for kw, code in ((dict(head_dim=128), iam.IAM_ERR_UNSUPPORTED), (dict(head_dim=64, rot_dim=32), iam.IAM_ERR_UNSUPPORTED),
                     (dict(head_dim=64, interleaved=True), iam.IAM_ERR_UNSUPPORTED), (dict(head_dim=64, theta=0.5), iam.IAM_ERR_ARG)):
        with pytest.raises(iam.IamError) as e:
            small.set_rope(iam.Rope.config(**kw))
        assert e.value.code == code


@pytest.mark.parametrize("chunk,n", [(7, 30), (1, 5), (16, 33), (29, 30)])
def test_score_over_several_chunks(iam, cuda, monkeypatch, chunk, n):
    """Chunks of the prompt one after another in one call, the last one shorter: every output lands at its token.  Bars as for one
    chunk, against the logits of every prefix."""
    import torch
    monkeypatch.setenv("IAM_PREFILL_CHUNK", str(chunk))
    vocab, k = SMALL["vocab"], 7
    m = iam.Model.random(iam.ModelConfig.make(**SMALL), seed=7)
    prompt = np.random.default_rng(n).integers(0, vocab, n).tolist()
    follow = prompt[1:] + [-1]
    follow[n // 2] = -1
    targets = torch.tensor(follow, dtype=torch.int32, device="cuda")
    out = dict(logprob=torch.full((n,), 99.0, device="cuda"), entropy=torch.full((n,), 99.0, device="cuda"),
               rank=torch.full((n,), 99, dtype=torch.int32, device="cuda"), top_logprob=torch.full((n, k), 99.0, device="cuda"),
               top_index=torch.full((n, k), 99, dtype=torch.int32, device="cuda"))
    nxt = m.score(prompt, targets, **out)
    logits = torch.empty(vocab, device="cuda")
    for t in range(n):
        m.reset()
        best = m.prefill(prompt[:t + 1], 0, logits)
        x = logits.double()
        tol = 2e-3 * float(x.square().mean().sqrt())
        logp = torch.log_softmax(x, 0)
        if follow[t] >= 0:
            assert abs(float(out["logprob"][t]) - float(logp[follow[t]])) < tol
            mine = float(x[follow[t]])
            assert int((x > mine + tol).sum()) <= int(out["rank"][t]) <= int((x > mine - tol).sum())
        else:
            assert out["logprob"][t] == 0 and out["rank"][t] == -1
        assert abs(float(out["entropy"][t]) + float((logp.exp() * logp).sum())) < tol * (1 + float(x.abs().max()))
        assert (out["top_logprob"][t].double() - torch.sort(logp, descending=True)[0][:k]).abs().max() < tol
        assert (logp[out["top_index"][t].long()] - out["top_logprob"][t].double()).abs().max() < tol
    assert nxt == best
    m.close()


def test_set_rope_in_decoding(small, iam, cuda):
    """The ntk scaling is another theta: single steps of the model with it against those of a model made with that theta, and
    the generation captured before the change against single steps after it.  Between the two models only the angles' last
    bits differ (as between any two summation orders: logits within 1e-3 x RMS, 5e-2 where a row on a cutoff went the other way)."""
    import torch
    m, effort, n, factor = small, 0.5, 24, 2.0
    d = SMALL["head_dim"]
    other = iam.Model.random(iam.ModelConfig.make(**SMALL, rope_theta=1e6 * factor ** (d / (d - 2))), seed=7)
    prompt = np.random.default_rng(4).integers(0, SMALL["vocab"], n).tolist()
    logits = torch.empty(SMALL["vocab"], device="cuda")
    gen, again = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")

    def steps(model):
        model.reset()
        out = []
        for pos, tok in enumerate(prompt):
            model.forward(tok, pos, effort, logits)
            out.append(logits.double().clone())
        return torch.stack(out)

    def greedy(model):
        model.reset()
        tok, out = prompt[0], []
        for pos in range(n):
            model.forward(tok, pos, effort, logits)
            tok = int(logits.argmax())
            out.append(tok)
        return out

    plain = steps(m)
    m.reset()
    m.generate(prompt[0], 0, n, effort, gen)
    try:
        m.set_rope(iam.Rope.config(d, scaling="ntk", factor=factor))
        scaled = steps(m)
        m.reset()
        m.generate(prompt[0], 0, n, effort, again)
        tokens = greedy(m)
    finally:
        m.set_rope(None)
    want = steps(other)
    rms = want.square().mean(-1).sqrt()
    err, change = (scaled - want).abs().amax(-1) / rms, (plain - want).abs().amax(-1) / rms
    print(f"ntk against theta: median {float(err.median()):.2e}, worst {float(err.max()):.2e}; without it median {float(change.median()):.2e}")
    assert float(err.max()) < 5e-2 and float(err.median()) < 1e-3 < float(change.median())
    assert again.tolist() == tokens
    assert torch.equal(steps(m), plain)
    other.close()
