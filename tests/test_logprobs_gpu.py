"""Log probabilities (iam_logprobs) against the definition in 64 bits.

Tolerance: a term's exponent y = (x - m) log2 e is off by |y| 2^-24 from one rounding, its power by 2 ulp, and
the sums of up to 10^5 positive terms are trees of short runs (at most 300 terms a run: 300 2^-24, on average
far less), so ln L is off by less than 2^-15.9; the largest differences x - m enter with one more rounding,
2^-23 |x - m|; the entropy's second sum has the same relative error on terms bounded by |x - m|."""
import math

import pytest

pytestmark = pytest.mark.gpu
TOL = 2.0 ** -15


def reference(x, targets, k, torch):
    x = x.double()
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    t = targets.long().clamp(0, x.shape[1] - 1)[:, None]
    mine = x.gather(1, t)
    index = torch.arange(x.shape[1], device=x.device)
    best, where = torch.sort(x, dim=-1, descending=True, stable=True)
    return dict(logprob=logp.gather(1, t)[:, 0], lse=torch.logsumexp(x, -1),
                entropy=-torch.where(p > 0, p * logp, 0.0).sum(-1),
                rank=((x > mine) | ((x == mine) & (index < t))).sum(-1), top_logprob=logp.gather(1, where[:, :k]), top_index=where[:, :k])


def call(iam, x, targets, k, torch, **kw):
    n = x.shape[0]
    out = {a: torch.full((n,), 99.0, device="cuda") for a in ("logprob", "lse", "entropy")}
    out["rank"] = torch.full((n,), 99, dtype=torch.int32, device="cuda")
    if k:
        out["top_logprob"], out["top_index"] = torch.full((n, k), 99.0, device="cuda"), torch.full((n, k), 99, dtype=torch.int32, device="cuda")
    iam.logprobs(x, targets, **out, **kw)
    return out


def compare(got, want, x, k, torch):
    spread = (x.double().amax(-1) - torch.where(x.isinf(), math.inf, x.double()).amin(-1)).clamp(min=0)
    for name in ("logprob", "lse", "entropy") + (("top_logprob",) if k else ()):
        g, w = got[name].double(), want[name]
        same_inf = (g == w) & w.isinf()
        tol = TOL + 2.0 ** -23 * (w.abs() + (spread if w.dim() == 1 else spread[:, None]))
        bad = ~(((g - w).abs() <= tol) | same_inf)
        assert not bad.any(), (name, g[bad][:4], w[bad][:4])
    assert torch.equal(got["rank"].long(), want["rank"])
    if k:
        assert torch.equal(got["top_index"].long(), want["top_index"])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,vocab,k", [(1, 1, 1), (3, 2, 2), (5, 7, 0), (4, 64, 64), (1, 1000, 5), (2, 4099, 20), (1, 32000, 5), (70, 32003, 20),
                                       (400, 517, 3), (3, 131071, 64), (1, 250001, 33),
                                       (2, 1000003, 20), (300, 70001, 12)])
def test_against_64_bits(iam, cuda, dtype, n, vocab, k):
    import torch
    g = torch.Generator("cuda").manual_seed(n * 31 + vocab)
    x = (torch.randn(n, vocab, generator=g, device="cuda") * 3).to(getattr(torch, dtype))
    targets = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    compare(call(iam, x, targets, k, torch), reference(x, targets, max(k, 1), torch), x, k, torch)


@pytest.mark.parametrize("shift", [0.0, 1000.0, -30000.0])
def test_far_from_zero(iam, cuda, shift):
    """An offset of all logits changes nothing but the sum's logarithm (the offsets are exact in fp32)."""
    import torch
    x = torch.randint(-4000, 4000, (9, 5003), device="cuda").float() / 256 + shift
    targets = torch.randint(0, 5003, (9,), device="cuda", dtype=torch.int32)
    compare(call(iam, x, targets, 10, torch), reference(x, targets, 10, torch), x, 10, torch)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_ties_go_to_the_lower_token(iam, cuda, dtype):
    import torch
    x = torch.randint(0, 4, (6, 20011), device="cuda").to(getattr(torch, dtype))  # thousands of equal best values
    x[1] = 2.5
    x[2] = 0.0
    x[2, ::2] = -0.0
    targets = torch.tensor([0, 7, 20010, 5, 19999, 10000], dtype=torch.int32, device="cuda")
    compare(call(iam, x, targets, 40, torch), reference(x, targets, 40, torch), x, 40, torch)


def test_masked_tokens(iam, cuda):
    """-inf leaves a token no probability; targets and alternatives among such tokens, one token left."""
    import torch
    x = torch.randn(5, 4001, device="cuda")
    x[0, 10:] = -math.inf
    x[1, :] = -math.inf
    x[1, 1234] = -7.0
    x[2, ::2] = -math.inf
    x[3] = torch.finfo(torch.float32).min
    x[4, :4000] = torch.finfo(torch.float32).min
    targets = torch.tensor([3, 1234, 0, 17, 4000], dtype=torch.int32, device="cuda")
    got, want = call(iam, x, targets, 12, torch), reference(x, targets, 12, torch)
    assert torch.equal(got["rank"].long(), want["rank"]) and torch.equal(got["top_index"].long(), want["top_index"])
    for name in ("logprob", "entropy", "top_logprob"):
        g, w = got[name].double(), want[name]
        ok = ((g - w).abs() <= TOL + 2.0 ** -22 * w.abs()) | (g == w) | ((w < -1e38) & (g <= w * (1 - 2.0 ** -22)))
        assert ok.all(), (name, g, w)


def test_rows_without_a_distribution(iam, cuda):
    import torch
    x = torch.randn(4, 3001, device="cuda")
    x[0] = -math.inf
    x[1, 5] = math.nan
    x[2, 7] = math.inf
    targets = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    got = call(iam, x, targets, 4, torch)
    for name in ("logprob", "entropy"):
        assert got[name][:3].isnan().all() and got[name][3].isfinite()
    assert got["top_logprob"][:3].isnan().all() and got["top_logprob"][3].isfinite().all()
    assert got["lse"][0] == -math.inf and got["lse"][1].isnan() and got["lse"][2].isnan()
    assert got["top_index"][0].tolist() == [0, 1, 2, 3]
    assert ((got["top_index"] >= 0) & (got["top_index"] < 3001)).all()


def test_targets_that_name_no_token(iam, cuda):
    import torch
    x = torch.randn(3, 500, device="cuda")
    got = call(iam, x, torch.tensor([-1, 500, 2 ** 31 - 1], dtype=torch.int32, device="cuda"), 0, torch)
    assert got["logprob"][0] == 0 and got["logprob"][1:].isnan().all() and got["rank"].tolist() == [-1, -1, -1]
    assert got["entropy"].isfinite().all()


@pytest.mark.parametrize("dtype,offset,pad", [("float32", 1, 3), ("bfloat16", 3, 5), ("float16", 7, 0), ("bfloat16", 1, 2)])
def test_rows_at_any_element(iam, cuda, dtype, offset, pad):
    """Rows that start and end inside a 16-byte piece, between values that must not be read into them."""
    import torch
    n, vocab = 11, 1237
    flat = torch.full((offset + n * (vocab + pad) + 16,), 60000.0, device="cuda").to(getattr(torch, dtype))
    x = torch.as_strided(flat, (n, vocab), (vocab + pad, 1), offset)
    x.copy_(torch.randn(n, vocab, device="cuda") * 2)
    targets = torch.randint(0, vocab, (n,), device="cuda", dtype=torch.int32)
    compare(call(iam, x, targets, 8, torch), reference(x, targets, 8, torch), x, 8, torch)


def test_some_outputs_only_streams_and_graph(iam, cuda):
    import torch
    x = torch.randn(6, 32000, device="cuda")
    targets = torch.randint(0, 32000, (6,), device="cuda", dtype=torch.int32)
    want = reference(x, targets, 3, torch)
    ent = torch.empty(6, device="cuda")
    iam.logprobs(x, entropy=ent)
    assert float((ent.double() - want["entropy"]).abs().max()) < TOL * 8
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = call(iam, x, targets, 3, torch)
    again = {a: torch.empty_like(b) for a, b in got.items()}
    torch.cuda.synchronize()
    iam.logprobs(x, targets, stream=s, **again)
    s.synchronize()
    assert all(torch.equal(got[a], again[a]) for a in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        iam.logprobs(x, targets, **again)
    x.copy_(torch.randn_like(x))
    graph.replay()
    torch.cuda.synchronize()
    compare(again, reference(x, targets, 3, torch), x, 3, torch)


def test_refused_calls(iam, cuda):
    import torch
    x = torch.zeros(3, 50, device="cuda")
    t = torch.zeros(3, dtype=torch.int32, device="cuda")
    f, i = torch.zeros(3, 51, device="cuda"), torch.zeros(3, 51, dtype=torch.int32, device="cuda")
    bad = [dict(logits=x.double()), dict(logits=x.cpu()), dict(logits=x.t()), dict(logits=x[0]), dict(targets=t.long()), dict(targets=t[:2]),
           dict(logprob=f[:, 0]), dict(logprob=t), dict(top_logprob=f[:, :5].contiguous()), dict(top_logprob=f, top_index=i),
           dict(targets=None, logprob=torch.zeros(3, device="cuda")), dict(logits=x[:1].expand(3, 50))]
    for change in bad:
        with pytest.raises(iam.IamError) as e:
            iam.logprobs(**dict(dict(logits=x, targets=t), **change))
        assert e.value.code == iam.IAM_ERR_ARG


def test_few_rows_on_a_busy_device(iam, cuda):
    """Rows shared by a cluster's CTAs, whose parts meet in the first one's memory: many short calls on several streams at once,
    beside products that keep most SMs busy, so that the CTAs of a cluster start at different times."""
    import torch
    g = torch.Generator("cuda").manual_seed(11)
    streams = [torch.cuda.Stream() for _ in range(4)]
    jobs = []
    for i, (n, vocab, k) in enumerate([(1, 131071, 64), (2, 32000, 5), (3, 70001, 40), (1, 8209, 20)]):
        x = torch.randn(n, vocab, generator=g, device="cuda") * 3
        targets = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
        first = call(iam, x, targets, k, torch)
        compare(first, reference(x, targets, k, torch), x, k, torch)
        jobs.append((x, targets, k, first, {name: t.clone() for name, t in first.items()}, torch.zeros((), dtype=torch.int64, device="cuda")))
    a = torch.randn(2048, 2048, device="cuda")
    busy = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(200):
        with torch.cuda.stream(busy):
            a = (a @ a).clamp(-1, 1)
        for s, (x, targets, k, first, out, off) in zip(streams, jobs):
            with torch.cuda.stream(s):
                iam.logprobs(x, targets, **out)
                for name in out:
                    off += (out[name] != first[name]).any()
                    out[name].zero_()
    torch.cuda.synchronize()
    assert all(int(job[-1]) == 0 for job in jobs)
