"""Rotary positions (iam_rope_*) against the formula in 64 bits.

Tolerance, per element of a pair (a, b) and factor f: the rotation is computed in fp32 from an angle in
(-pi, pi] rounded to fp32 (pi 2^-24), cos and sin within 2 ulp, three roundings of products and sum, and one
rounding to the type (eps/2 of the value): eps/2 |y| + f (|a| + |b|) 2^-20."""
import math

import pytest


def angles(cfg, positions, torch):
    """cos and sin [tokens][pairs] in 64 bits, written from the definition pair by pair."""
    d, theta, s, ctx = cfg["rot_dim"], cfg["theta"], cfg["factor"], cfg["original_ctx"]
    w, f = [], 1.0
    for i in range(d // 2):
        base = theta ** (-2.0 * i / d)
        if cfg["scaling"] == "ntk":
            base = (theta * s ** (d / (d - 2))) ** (-2.0 * i / d)
        if cfg["scaling"] == "linear":
            base /= s
        if cfg["scaling"] == "banded":
            lo, hi = cfg.get("low_turns") or 1.0, cfg.get("high_turns") or 4.0
            turns = ctx * base / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - lo) / (hi - lo)))
            base = base * keep + base / s * (1 - keep)
        if cfg["scaling"] == "yarn":
            lo, hi = cfg.get("low_turns") or 1.0, cfg.get("high_turns") or 32.0
            pair = lambda n: d * math.log(ctx / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
            a, b = max(math.floor(pair(hi)), 0), min(math.ceil(pair(lo)), d - 1)
            ramp = min(1.0, max(0.0, (i - a) / max(b - a, 0.001)))
            base = base / s * ramp + base * (1 - ramp)
            f = 0.1 * math.log(s) + 1.0 if s > 1 else 1.0
        w.append(base)
    f = cfg.get("attn_factor") or f
    a = positions.double()[:, None] * torch.tensor(w, dtype=torch.float64, device=positions.device)
    return a.cos(), a.sin(), f


def rotated(cfg, x, positions, torch):
    """-> (rotated x in 64 bits, the tolerance's |a| + |b| of each element)."""
    cos, sin, f = angles(cfg, positions, torch)
    r = cfg["rot_dim"]
    y, mag = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for i in range(r // 2):
        a, b = (2 * i, 2 * i + 1) if cfg["interleaved"] else (i, i + r // 2)
        u, v = x[..., a].double(), x[..., b].double()
        y[..., a] = f * (u * cos[:, None, i] - v * sin[:, None, i])
        y[..., b] = f * (v * cos[:, None, i] + u * sin[:, None, i])
        mag[..., a] = mag[..., b] = f * (u.abs() + v.abs())
    return y, mag


def config(head_dim, rot_dim=None, interleaved=False, theta=1e6, scaling="none", factor=1.0, original_ctx=0, **more):
    return dict(head_dim=head_dim, rot_dim=rot_dim or head_dim, interleaved=interleaved, theta=theta, scaling=scaling,
                factor=factor, original_ctx=original_ctx, **more)


SCALINGS = [dict(scaling="none"), dict(scaling="linear", factor=3.0), dict(scaling="ntk", factor=4.0),
            dict(scaling="yarn", factor=8.0, original_ctx=4096), dict(scaling="banded", factor=8.0, original_ctx=8192),
            dict(scaling="banded", factor=2.0, original_ctx=2048, low_turns=0.5, high_turns=16.0),
            dict(scaling="yarn", factor=4.0, original_ctx=2048, attn_factor=1.25)]


def check(cfg, got, x, positions, torch):
    want, mag = rotated(cfg, x, positions, torch)
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() + mag * 2.0 ** -20
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / tol.clamp(min=1e-30)).max()))


@pytest.mark.parametrize("cfg", SCALINGS)
def test_frequencies_match_the_definition(iam, cfg):
    torch = pytest.importorskip("torch")
    c = config(128, theta=5e5, **cfg)
    w, f = iam.Rope.frequencies(iam.Rope.config(**c))
    cos, _, want_f = angles(c, torch.tensor([1], dtype=torch.int32), torch)
    assert f == pytest.approx(want_f, rel=1e-14)
    assert [math.cos(x) for x in w] == pytest.approx(cos[0].tolist(), abs=1e-14)
    assert len(w) == 64 and all(a > b for a, b in zip(w, w[1:]))


@pytest.mark.parametrize("bad", [dict(head_dim=0), dict(rot_dim=3), dict(rot_dim=130), dict(rot_dim=0), dict(theta=1.0),
                                 dict(theta=math.nan), dict(theta=math.inf), dict(scaling="linear", factor=0.5), dict(scaling="ntk", factor=math.inf),
                                 dict(scaling="yarn", factor=2.0), dict(scaling="banded", factor=2.0, original_ctx=-1),
                                 dict(scaling="banded", factor=2.0, original_ctx=4096, low_turns=5.0),
                                 dict(scaling="banded", factor=2.0, original_ctx=4096, low_turns=-1.0),
                                 dict(attn_factor=-1.0), dict(scaling="spiral")])
def test_refused_configurations(iam, bad):
    with pytest.raises(iam.IamError) as e:
        iam.Rope.frequencies(iam.Rope.config(**dict(dict(head_dim=128), **bad)))
    assert e.value.code == iam.IAM_ERR_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot", [(1, 32, 8, 128, 128), (17, 4, 2, 64, 32), (5, 3, 1, 256, 64), (300, 8, 8, 64, 64),
                                                     (3, 5, 5, 80, 20), (2, 1, 0, 6, 2), (7, 2, 2, 33, 6)])
def test_rotation(iam, cuda, dtype, interleaved, tokens, heads, kv, dim, rot):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator("cuda").manual_seed(tokens * 7 + dim)
    for n, extra in enumerate(SCALINGS if tokens == 17 else SCALINGS[3:4]):
        cfg = config(dim, rot, interleaved, **extra)
        rope = iam.Rope(**cfg)
        qkv = torch.randn(tokens, heads + 2 * kv, dim, generator=g, device="cuda").to(dt)
        positions = torch.randint(0, 2 ** 31 - 1 if n % 2 else 40000, (tokens,), generator=g, device="cuda", dtype=torch.int32)
        positions[0] = 0
        q, k = qkv[:, :heads], qkv[:, heads:heads + kv]
        before = qkv.clone()
        q_out, k_out = torch.full(q.shape, 7.0, dtype=dt, device="cuda"), torch.full(k.shape, 7.0, dtype=dt, device="cuda")
        rope.apply(q, positions, q_out, k=k, k_out=k_out)
        assert torch.equal(qkv, before)
        check(cfg, q_out, q, positions, torch)
        check(cfg, k_out, k, positions, torch)
        rope.apply(q, positions, k=k)  # in place: the same bits, and the v heads untouched
        assert torch.equal(q, q_out) and torch.equal(k, k_out)
        assert torch.equal(qkv[:, heads + kv:], before[:, heads + kv:])
        rope.close()


@pytest.mark.gpu
@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 0), (3, 5)])
def test_rows_at_odd_offsets_and_strides(iam, cuda, offset, pad):
    import torch
    cfg = config(64, 64, False)
    rope = iam.Rope(**cfg)
    flat = torch.randn(offset + 9 * (4 * 64 + pad) + 64, device="cuda").to(torch.bfloat16)
    q = torch.as_strided(flat, (9, 4, 64), (4 * 64 + pad, 64, 1), offset)
    x = q.clone()
    positions = torch.arange(9, dtype=torch.int32, device="cuda") * 1000
    rest = flat.clone()
    rope.apply(q, positions)
    check(cfg, q, x, positions, torch)
    torch.as_strided(rest, (9, 4, 64), (4 * 64 + pad, 64, 1), offset).copy_(q)
    assert torch.equal(rest, flat)  # nothing between the rows was written


@pytest.mark.gpu
def test_scores_depend_on_distances_alone(iam, cuda):
    """What the rotation is for: q at p and k at p - 5 have one product, whatever p."""
    import torch
    rope = iam.Rope(128, theta=1e4)
    v = torch.randn(2, 1, 128, device="cuda").expand(2, 64, 128).transpose(0, 1).contiguous()
    at = torch.arange(64, dtype=torch.int32, device="cuda") * 3001
    q, k = v[:, :1].contiguous(), v[:, 1:].contiguous()
    rope.apply(q, at + 5)
    rope.apply(k, at)
    dots = (q.double() * k.double()).sum((1, 2))
    assert float((dots - dots[0]).abs().max()) < 128 * 16 * 2.0 ** -20


@pytest.mark.gpu
def test_no_tokens_other_stream_and_graph(iam, cuda):
    import torch
    cfg = config(128, 128, True, scaling="linear", factor=2.0)
    rope = iam.Rope(**cfg)
    empty = torch.empty(0, 4, 128, device="cuda")
    rope.apply(empty, torch.empty(0, dtype=torch.int32, device="cuda"))
    x = torch.randn(40, 4, 128, device="cuda", dtype=torch.float16)
    positions = torch.arange(40, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(x)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    rope.apply(x, positions, out, stream=s)
    s.synchronize()
    check(cfg, out, x, positions, torch)
    out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope.apply(x, positions, out)
    x.copy_(torch.randn_like(x))
    positions += 9
    graph.replay()
    torch.cuda.synchronize()
    check(cfg, out, x, positions, torch)


@pytest.mark.gpu
def test_refused_calls(iam, cuda):
    import torch
    rope = iam.Rope(64)
    q = torch.zeros(3, 2, 64, device="cuda")
    at = torch.zeros(3, dtype=torch.int32, device="cuda")
    for args, kw in [((q.double(), at), {}), ((q[..., :32], at), {}), ((q, at.long()), {}), ((q, at[:2]), {}), ((q, at.cpu()), {}),
                     ((q.cpu(), at), {}), ((q, at, q.half()), {}), ((q, at, q[:2]), {}), ((q.transpose(1, 2).contiguous().transpose(1, 2), at), {}),
                     ((q, at), dict(k=q[:2])), ((q, at), dict(k=q.half())), ((q, at, q[:1].expand(3, 2, 64)), {})]:
        with pytest.raises(iam.IamError) as e:
            rope.apply(*args, **kw)
        assert e.value.code == iam.IAM_ERR_ARG
    inplace = torch.as_strided(q, (2, 2, 64), (128, 64, 1))
    other = torch.as_strided(q, (2, 2, 64), (192, 64, 1))
    with pytest.raises(iam.IamError):
        rope.apply(inplace, at[:2], other)  # the same rows under other strides
