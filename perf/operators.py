"""The long-context and scoring operators, case by case: what they are measured on, their plain form in
elementary torch operations, and their definition in 64 bits.

Four operators around the model's attention and its logits:
  rope      rotary positions (half and interleaved pairs, part of the head, frequencies scaled for long contexts)
  append    new keys and values into a paged cache of 8-bit codes with one scale per page and KV head
  attend    causal attention of ragged query rows over that cache
  logprobs  log probability, rank, entropy and top alternatives of given tokens

With `own` false, run() is the plain form; with `own` true it makes the package's calls on the same state.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
TOP = {"int8": 127.0, "e4m3": 448.0}  # largest code of each cache format
HEADS = ((32, 8, 128), (4, 2, 64), (8, 8, 64), (16, 2, 128), (8, 1, 256))


def package():
    if "iam_b200" in sys.modules:
        return sys.modules["iam_b200"]
    home = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "input-adaptive-matrix-inference-optimization_b200")
    spec = importlib.util.spec_from_file_location("iam_b200", os.path.join(home, "__init__.py"), submodule_search_locations=[home])
    module = importlib.util.module_from_spec(spec)
    sys.modules["iam_b200"] = module
    spec.loader.exec_module(module)
    return module


# ------------------------------------------------------------------ cases

def listed():
    return [
        # the decode step's own rotation: one token of the 7B shape, fp32 as the bucketMul writes it
        dict(name="rope 1 token", op="rope", tokens=1, heads=32, kv=8, dim=128, rot=128, interleaved=False, theta=1e6, scaling="none",
             factor=1.0, original=0, start=4095, dtype="fp32"),
        # a prompt chunk of the 7B shape, stretched to four times its training length
        dict(name="rope prompt 2048 yarn", op="rope", tokens=2048, heads=32, kv=8, dim=128, rot=128, interleaved=False, theta=1e6,
             scaling="yarn", factor=4.0, original=8192, start=30000, dtype="bf16"),
        # interleaved pairs on the first half of the head, an odd number of tokens far out
        dict(name="rope 8191 part interleaved", op="rope", tokens=8191, heads=16, kv=16, dim=128, rot=64, interleaved=True, theta=1e4,
             scaling="banded", factor=8.0, original=8192, start=100000, dtype="fp16"),
        # one decode step of 64 requests into int8 pages
        dict(name="append 64 x 1 int8", op="append", seqs=64, new=1, longest=2048, kv=8, dim=128, page=64, fmt="int8", dtype="fp32"),
        # a ragged batch of prompts into e4m3 pages
        dict(name="append prompts e4m3", op="append", seqs=5, new=4001, longest=6001, kv=8, dim=128, page=64, fmt="e4m3", dtype="bf16"),
        # decoding after the benchmark's 8192-token context, one request, fp32 activations
        dict(name="attend 1 x 8192 fp32", op="attend", seqs=1, new=1, longest=8192, heads=32, kv=8, dim=128, page=64, fmt="int8", window=0,
             dtype="fp32"),
        # a ragged batch of requests, one token each
        dict(name="attend 48 ragged", op="attend", seqs=48, new=1, longest=8192, heads=32, kv=8, dim=128, page=64, fmt="e4m3", window=0,
             dtype="bf16"),
        # one very long document
        dict(name="attend 1 x 131071", op="attend", seqs=1, new=1, longest=131071, heads=32, kv=8, dim=128, page=128, fmt="e4m3", window=0,
             dtype="fp16"),
        # several drafted tokens of each request checked at once, sliding window
        dict(name="attend 13 x 7 drafted", op="attend", seqs=13, new=7, longest=5000, heads=16, kv=2, dim=128, page=16, fmt="int8",
             window=4096, dtype="fp16"),
        # a prompt chunk behind an 8192-token context
        dict(name="attend prompt 2048", op="attend", seqs=1, new=2048, longest=10240, heads=32, kv=8, dim=128, page=64, fmt="e4m3", window=0,
             dtype="bf16"),
        # the decode step's own logits with the five best alternatives
        dict(name="logprobs 1 x 32000", op="logprobs", rows=1, vocab=32000, top=5, dtype="fp32"),
        # a scored document's logits
        dict(name="logprobs 2048 x 32000", op="logprobs", rows=2048, vocab=32000, top=20, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope", "append", "attend", "attend", "logprobs"))
    dtype = rng.choice(("fp32", "fp16", "bf16"))
    heads, kv, dim = rng.choice(HEADS)
    if op == "rope":
        rot = rng.choice((dim, dim // 2, dim // 4))
        scaling = rng.choice(("none", "linear", "ntk", "yarn", "banded"))
        return dict(op=op, tokens=_log(rng, 1, 8192), heads=heads, kv=kv, dim=dim, rot=rot, interleaved=rng.random() < 0.5,
                    theta=rng.choice((1e4, 5e5, 1e6)), scaling=scaling, factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0)),
                    original=0 if scaling == "none" else rng.choice((2048, 4096, 8192)), start=_log(rng, 1, 200000), dtype=dtype)
    page, fmt = rng.choice((16, 32, 64, 128)), rng.choice(("int8", "e4m3"))
    if op == "append":
        new = rng.choice((1, 1, _log(rng, 2, 4096)))
        seqs = _log(rng, 1, 96 if new == 1 else min(96, max(1, 12000 // new)))
        return dict(op=op, seqs=seqs, new=new, longest=new + _log(rng, 1, 2048), kv=kv, dim=dim, page=page, fmt=fmt, dtype=dtype)
    if op == "attend":
        new = rng.choice((1, 1, rng.randint(2, 16), _log(rng, 17, 2048)))
        seqs = _log(rng, 1, 48 if new == 1 else 16 if new <= 16 else 3)
        longest = new + _log(rng, 1, 8192 if seqs > 1 or new > 16 else 131072)
        if new > 16 and seqs * new * longest > 2048 * 10240:
            longest = max(new, 2048 * 10240 // (seqs * new))
        return dict(op=op, seqs=seqs, new=new, longest=longest, heads=heads, kv=kv, dim=dim, page=page, fmt=fmt,
                    window=rng.choice((0, 0, _log(rng, 1, 8192))), dtype=dtype)
    vocab = rng.choice((32000, 32003, 32768, 4099, 131071, _log(rng, 64, 131072)))
    rows = _log(rng, 1, max(1, min(4096, 2048 * 32000 // vocab)))
    return dict(op=op, rows=rows, vocab=vocab, top=rng.choice((0, 1, 5, 20)), dtype=dtype)


# ------------------------------------------------------------------ inputs

def _lengths(case):
    """Host lists: how many new tokens each sequence has, and its length with them (the case's own, whatever the seed)."""
    g = torch.Generator().manual_seed(7919 + case["longest"])
    n, most, longest = case["seqs"], case["new"], case["longest"]
    new = torch.randint(max(1, (most + 1) // 2), most + 1, (n,), generator=g).tolist()
    new[0] = most
    span = torch.rand(n, generator=g).tolist()
    lens = [a + int(s * (longest - most)) for a, s in zip(new, span)]
    lens[-1] = max(new[-1], longest)
    return new, lens


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _quantised_pages(g, pages, kv, page, dim, fmt):
    """Codes and scales of pages of normal values with a few strong channels."""
    x = _randn(g, pages, kv, page, dim)
    x *= 1.0 + 3.0 * (torch.rand(1, kv, 1, dim, generator=g, device="cuda") < 0.03)
    scale = _scale_of(x.abs().amax((2, 3)), fmt)
    return _encode(x / scale[:, :, None, None], fmt), scale


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    op, s = case["op"], dict(case)
    if op == "rope":
        n, dt = case["tokens"], TYPES[case["dtype"]]
        # q and k heads side by side, as one projection writes them, with the v heads between two tokens
        width = (case["heads"] + 2 * case["kv"]) * case["dim"]
        qkv = _randn(g, n, width).to(dt).view(n, -1, case["dim"])
        s["q"], s["k"] = qkv[:, :case["heads"]], qkv[:, case["heads"]:case["heads"] + case["kv"]]
        s["q_out"], s["k_out"] = torch.empty(s["q"].shape, dtype=dt, device="cuda"), torch.empty(s["k"].shape, dtype=dt, device="cuda")
        s["positions"] = (torch.arange(n, device="cuda") + case["start"] + seed % 7).to(torch.int32)
        if own:
            s["rope"] = package().Rope(case["dim"], rot_dim=case["rot"], interleaved=case["interleaved"], theta=case["theta"],
                                       scaling=case["scaling"], factor=case["factor"], original_ctx=case["original"])
        return s
    if op == "logprobs":
        n, v, dt = case["rows"], case["vocab"], TYPES[case["dtype"]]
        x = _randn(g, n, v) * 2.5
        x[:: 3, : v // 10] = -math.inf  # tokens that a grammar forbids in some of the rows
        s["logits"] = x.to(dt)
        s["targets"] = torch.randint(0, v, (n,), generator=g, device="cuda").to(torch.int32)
        for name in ("logprob", "lse", "entropy"):
            s[name] = torch.empty(n, device="cuda")
        s["rank"] = torch.empty(n, dtype=torch.int32, device="cuda")
        k = case["top"]
        s["top_logprob"] = torch.empty(n, k, device="cuda") if k else None
        s["top_index"] = torch.empty(n, k, dtype=torch.int32, device="cuda") if k else None
        return s
    new, lens = _lengths(case)
    n, kv, dim, page, fmt = case["seqs"], case["kv"], case["dim"], case["page"], case["fmt"]
    need = [-(-x // page) for x in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((n, max(need)), -1, dtype=torch.int32, device="cuda")
    first = 0
    for i, c in enumerate(need):  # each sequence's pages, scattered over the pool
        table[i, :c] = order[first:first + c]
        first += c
    s["table"] = table
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["cu"] = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    # one page more than the pool: the plain form's place for what belongs to no page
    s["k_all"], s["ks_all"] = _quantised_pages(g, pages + 1, kv, page, dim, fmt)
    s["v_all"], s["vs_all"] = _quantised_pages(g, pages + 1, kv, page, dim, fmt)
    # what stands behind a sequence's last token is whatever an earlier request left: the code of NaN too
    last = torch.tensor([table[i, c - 1].item() for i, c in enumerate(need)], device="cuda")
    behind = torch.arange(page, device="cuda")[None, :] >= (s["lens"].long() - 1)[:, None] % page + 1
    for name in ("k_all", "v_all"):
        raw = s[name].view(torch.uint8)
        raw[last] = torch.where(behind[:, None, :, None], torch.tensor(0x7F, dtype=torch.uint8, device="cuda"), raw[last])
    s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"] = (s[x][:pages] for x in ("k_all", "v_all", "ks_all", "vs_all"))
    total, dt = sum(new), TYPES[case["dtype"]]
    if op == "append":
        kvx = _randn(g, total, 2 * kv, dim).to(dt)
        s["k_new"], s["v_new"] = kvx[:, :kv], kvx[:, kv:]
    else:
        s["q"] = (_randn(g, total, case["heads"], dim) * 1.5).to(dt)
        s["out"] = torch.zeros(total, case["heads"], dim, dtype=dt, device="cuda")
        s["lse"] = torch.zeros(total, case["heads"], device="cuda")
    if own:
        iam = package()
        s["kv8"] = iam.KV8(n_heads=case.get("heads", kv), n_kv_heads=kv, head_dim=dim)
        s["cache"] = iam.KV8Cache(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["table"])
    return s


# ------------------------------------------------------------------ plain forms

def _frequencies(case):
    """Radians per position of each pair (64 bits), and the factor on the rotated values."""
    d, theta, f, ctx = case["rot"], case["theta"], case["factor"], case["original"]
    i = torch.arange(d // 2, dtype=torch.float64)
    if case["scaling"] == "ntk":
        theta = theta * f ** (d / (d - 2)) if d > 2 else theta
    inv = theta ** (-2.0 * i / d)
    if case["scaling"] == "linear":
        return inv / f, 1.0
    if case["scaling"] == "banded":  # by wavelength: short ones stay, long ones are stretched, a ramp between
        turns = ctx * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return inv / f * (1 - keep) + inv * keep, 1.0
    if case["scaling"] == "yarn":  # by pair number between the pairs that turn 32 times and once within the training length
        at = lambda turns: d * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), d - 1)
        stretch = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return inv / f * stretch + inv * (1 - stretch), 0.1 * math.log(f) + 1.0 if f > 1 else 1.0
    return inv, 1.0


def _rotate(case, x, cos, sin):
    """x [tokens][heads][dim] with the first `rot` dims rotated, in the type of cos and sin."""
    x, r = x.to(cos.dtype), case["rot"]
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., r:]), -1)


def _rope(s):
    inv, factor = _frequencies(s)
    angle = s["positions"].double()[:, None, None] * inv.cuda()
    cos, sin = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    for x in ("q", "k"):
        s[x + "_out"].copy_(_rotate(s, s[x], cos, sin))
    return {"q": s["q_out"], "k": s["k_out"]}


def _scale_of(amax, fmt):
    """The smallest power of two >= 2^-126 that brings amax within the format's largest code."""
    mantissa, exponent = torch.frexp(amax.float())  # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    top_m, top_e = math.frexp(TOP[fmt])
    e = exponent - top_e + (mantissa > top_m).to(exponent.dtype)
    e = torch.where(amax > 0, e.clamp(min=-126), -126)
    return torch.ldexp(torch.ones_like(amax, dtype=torch.float32), e)


def _encode(x, fmt):
    x = torch.nan_to_num(x, nan=0.0, posinf=TOP[fmt], neginf=-TOP[fmt]).clamp(-TOP[fmt], TOP[fmt])
    return x.round().to(torch.int8) if fmt == "int8" else x.to(torch.float8_e4m3fn)


def _append_half(s, new, pages, scales):
    """`new` [tokens][kv][dim] into pages [n + 1][kv][page][dim] with scales [n + 1][kv]; the last page takes what has none."""
    page, fmt, kv = s["page"], s["fmt"], s["kv"]
    none, table, lens, cu = pages.shape[0] - 1, s["table"].long(), s["lens"].long(), s["cu"].long()
    total = new.shape[0]
    seq = torch.searchsorted(cu[1:], torch.arange(total, device="cuda"), right=True)
    start = lens - (cu[1:] - cu[:-1])
    at = start[seq] + torch.arange(total, device="cuda") - cu[seq]
    target = table[seq, at // page]
    x = new.float()
    amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    most = torch.zeros(none + 1, kv, device="cuda").scatter_reduce_(0, target[:, None].expand(-1, kv), amax, "amax")
    # the pages that hold earlier tokens of their sequence: only a sequence's first touched page can
    first = start // page
    held = start % page
    tail = torch.where(held > 0, table.gather(1, first.clamp(max=table.shape[1] - 1)[:, None])[:, 0], none)
    keep = torch.zeros(none + 1, dtype=torch.bool, device="cuda").index_fill_(0, tail, True)
    keep[none] = False
    wanted = _scale_of(most, fmt)
    now = torch.where(keep[:, None], torch.maximum(scales, wanted), wanted)
    touched = torch.zeros(none + 1, dtype=torch.bool, device="cuda").index_fill_(0, target, True)
    now = torch.where(touched[:, None], now, scales)
    old = pages[tail].float() * (scales[tail] / now[tail])[:, :, None, None]
    row = torch.arange(page, device="cuda")[None, None, :, None]
    pages[tail] = torch.where(row < held[:, None, None, None], _encode(old, fmt).view(torch.uint8), pages[tail].view(torch.uint8)).view(pages.dtype)
    scales.copy_(now)
    codes = _encode(x / now[target][:, :, None], fmt)
    pages[target, :, at % page] = codes


def _append(s):
    _append_half(s, s["k_new"], s["k_all"], s["ks_all"])
    _append_half(s, s["v_new"], s["v_all"], s["vs_all"])


def _places(s, lens, cu):
    """Of the padded query grid [seq][j]: the row of each, whether there is one, and its position."""
    n = cu[1:] - cu[:-1]
    j = torch.arange(s["new"], device="cuda")
    return (cu[:-1, None] + j).clamp(max=int(s["q"].shape[0]) - 1), j < n[:, None], (lens - n)[:, None] + j


def _attend(s):
    page, kv, dim = s["page"], s["kv"], s["dim"]
    n, g = s["seqs"], s["heads"] // s["kv"]
    lens, table = s["lens"].long(), s["table"].long().clamp(min=0)
    t = torch.arange(table.shape[1] * page, device="cuda")
    filled = (t < lens[:, None]).view(n, -1, page)[:, :, None, :, None]
    k, v = (torch.where(filled, s[x + "_pages"][table].float() * s[x + "_scale"][table][..., None, None], 0.0) for x in ("k", "v"))
    k, v = (x.transpose(1, 2).reshape(n, kv, -1, dim) for x in (k, v))
    row, there, pos = _places(s, lens, s["cu"].long())
    q = s["q"][row].float().view(n, -1, kv, g, dim).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, dim)
    seen = t <= pos[:, :, None]
    if s["window"]:
        seen &= t > pos[:, :, None] - s["window"]
    seen = seen[:, None, :, None].expand(n, kv, -1, g, -1).reshape(n, kv, q.shape[2], -1)
    score = torch.where(seen, q @ k.transpose(2, 3) * (1 / math.sqrt(dim)), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log())[..., 0]
    out = out.view(n, kv, -1, g, dim).permute(0, 2, 1, 3, 4).reshape(n, -1, s["heads"], dim).to(s["q"].dtype)
    lse = lse.view(n, kv, -1, g).permute(0, 2, 1, 3).reshape(n, -1, s["heads"])
    # the padded grid's first `total` places in row order are the ragged rows
    place = torch.argsort(torch.where(there, row, s["q"].shape[0] + 1).flatten(), stable=True)[: s["q"].shape[0]]
    s["out"].copy_(out.flatten(0, 1)[place])
    s["lse"].copy_(lse.flatten(0, 1)[place])


def _logprobs(s):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + total.log()
    target = s["targets"].long()[:, None]
    mine = x.gather(1, target)
    index = torch.arange(x.shape[1], device="cuda")
    s["logprob"].copy_((mine - top - total.log())[:, 0])
    s["lse"].copy_(lse[:, 0])
    s["entropy"].copy_((total.log() - torch.where(e > 0, (x - top) * e, 0.0).sum(-1, keepdim=True) / total)[:, 0])
    s["rank"].copy_(((x > mine) | ((x == mine) & (index < target))).sum(-1))
    if s["top"]:
        best, where = torch.sort(x, dim=-1, descending=True, stable=True)
        s["top_logprob"].copy_(best[:, : s["top"]] - top - total.log())
        s["top_index"].copy_(where[:, : s["top"]])


def run(s):
    op = s["op"]
    if op == "rope":
        if own:
            s["rope"].apply(s["q"], s["positions"], s["q_out"], k=s["k"], k_out=s["k_out"])
        else:
            _rope(s)
        return {"q": s["q_out"], "k": s["k_out"]}
    if op == "append":
        if own:
            s["kv8"].append(s["cache"], s["k_new"], s["v_new"], s["lens"], cu=s["cu"])
        else:
            _append(s)
        # the codes are exact (the scales are powers of two): they come as the cache holds them, with their scales
        return {x: s[x] for x in ("k_pages", "v_pages", "k_scale", "v_scale")}
    if op == "attend":
        if own:
            s["kv8"].attention(s["cache"], s["q"], s["lens"], s["out"], cu=s["cu"], max_q=s["new"], window=s["window"], lse=s["lse"])
        else:
            _attend(s)
        return {"out": s["out"], "lse": s["lse"]}
    if own:
        package().logprobs(s["logits"], s["targets"], s["logprob"], lse=s["lse"], entropy=s["entropy"], rank=s["rank"],
                           top_logprob=s["top_logprob"], top_index=s["top_index"])
    else:
        _logprobs(s)
    return {x: s[x] for x in ("logprob", "lse", "entropy", "rank", "top_logprob", "top_index")}


# ------------------------------------------------------------------ work

def work(case):
    op, size = case["op"], 4 if case["dtype"] == "fp32" else 2
    if op == "rope":
        values = case["tokens"] * (case["heads"] + case["kv"]) * case["dim"]
        turned = case["tokens"] * (case["heads"] + case["kv"]) * case["rot"]
        return {"bytes": 2 * values * size + 4 * case["tokens"], "flops": 3 * turned}
    if op == "logprobs":
        n, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": n * v * size + n * (20 + 8 * k), "flops": 6 * n * v}
    new, lens = _lengths(case)
    kv, dim, page = case["kv"], case["dim"], case["page"]
    if op == "append":
        touched = sum((x - 1) // page - (x - a) // page + 1 for a, x in zip(new, lens))
        return {"bytes": 2 * kv * (sum(new) * dim * (size + 1) + 8 * touched), "flops": 4 * kv * sum(new) * dim}
    seen = [(x - a + 1 + j) for a, x in zip(new, lens) for j in range(a)]
    read = sum(lens)
    if case["window"]:
        read = sum(x - max(0, x - a + 1 - case["window"]) for a, x in zip(new, lens))
        seen = [min(x, case["window"]) for x in seen]
    pages = sum(-(-x // page) for x in lens)
    rows = sum(new) * case["heads"]
    return {"bytes": 2 * kv * (read * dim + 4 * pages) + rows * (2 * dim * size + 4), "flops": 4.0 * sum(seen) * case["heads"] * dim}


# ------------------------------------------------------------------ the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        d, pairs, angle = case["rot"], case["rot"] // 2, None
        theta, f, ctx = case["theta"], case["factor"], case["original"]
        w, size = [], 1.0
        for i in range(pairs):
            base = math.exp(-2 * i / d * math.log(theta))
            if case["scaling"] == "ntk" and d > 2:
                base = math.exp(-2 * i / d * (math.log(theta) + d / (d - 2) * math.log(f)))
            if case["scaling"] == "linear":
                base /= f
            if case["scaling"] == "banded":
                wave = 2 * math.pi / base
                mix = 1.0 if wave < ctx / 4 else 0.0 if wave > ctx else (ctx / wave - 1) / 3
                base = base * (mix + (1 - mix) / f)
            if case["scaling"] == "yarn":
                lo = max(math.floor(d * math.log(ctx / (64 * math.pi)) / (2 * math.log(theta))), 0)
                hi = min(math.ceil(d * math.log(ctx / (2 * math.pi)) / (2 * math.log(theta))), d - 1)
                mix = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
                base = base * (1 - mix + mix / f)
                size = 1 + math.log(f) / 10 if f > 1 else 1.0
            w.append(base)
        angle = s["positions"].double()[:, None] * torch.tensor(w, dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.full_like(angle, size), angle)[:, None]
        back = {}
        for x in ("q", "k"):
            v = s[x].double()
            at = torch.arange(pairs, device="cuda")
            a, b = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + pairs)
            z = torch.complex(v[..., a], v[..., b]) * turn
            v[..., a], v[..., b] = z.real, z.imag
            back[x] = v
        return back
    if op == "logprobs":
        x = s["logits"].double()
        logp = torch.log_softmax(x, -1)
        p = logp.exp()
        at = s["targets"].long()
        mine = x.gather(1, at[:, None])[:, 0]
        return {"logprob": logp.gather(1, at[:, None])[:, 0], "lse": torch.logsumexp(x, -1),
                "entropy": -torch.where(p > 0, p * logp, 0.0).sum(-1), "rank": None,
                "top_logprob": (torch.topk(x, case["top"], -1)[0] - (mine - logp.gather(1, at[:, None])[:, 0])[:, None]) if case["top"] else None,
                "top_index": None}
    page, dim, kv = case["page"], case["dim"], case["kv"]
    lens, cu, table = s["lens"].tolist(), s["cu"].tolist(), s["table"].tolist()
    if op == "append":
        back = {}
        for x in ("k", "v"):
            codes, scale, new = s[x + "_pages"].double().clone(), s[x + "_scale"].double().clone(), s[x + "_new"].double()
            for i, n in enumerate(lens):
                start = n - (cu[i + 1] - cu[i])
                for c in range(start // page, (n - 1) // page + 1):
                    lo, hi, to = max(start, c * page), min(n, (c + 1) * page), table[i][c]
                    block = new[cu[i] + lo - start:cu[i] + hi - start].transpose(0, 1)
                    unit = torch.exp2(torch.ceil(torch.log2(block.abs().amax((1, 2)) / TOP[case["fmt"]])))
                    held = lo - c * page
                    if held:
                        unit = torch.maximum(unit, scale[to])
                        codes[to, :, :held] = _nearest(codes[to, :, :held] * (scale[to] / unit)[:, None, None], case["fmt"])
                    codes[to, :, held:held + hi - lo] = _nearest(block / unit[:, None, None], case["fmt"])
                    scale[to] = unit
            back[x + "_pages"], back[x + "_scale"] = codes if case["fmt"] == "e4m3" else None, scale
        return back
    g = case["heads"] // kv
    out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        rows = torch.arange(cu[i], cu[i + 1], device="cuda")
        if not len(rows):
            continue
        ids = s["table"][i, : -(-n // page)].long()
        pos = torch.arange(n - len(rows), n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        hidden = (key > pos) | ((key <= pos - case["window"]) if case["window"] else torch.zeros_like(key > pos))
        for h in range(kv):
            k = (s["k_pages"][ids, h].double() * s["k_scale"][ids, h].double()[:, None, None]).reshape(-1, dim)[:n]
            v = (s["v_pages"][ids, h].double() * s["v_scale"][ids, h].double()[:, None, None]).reshape(-1, dim)[:n]
            for j in range(h * g, (h + 1) * g):
                a = (s["q"][rows, j].double() @ k.T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
                lse[rows, j] = torch.logsumexp(a, -1)
                out[rows, j] = torch.softmax(a, -1) @ v
    return {"out": out, "lse": lse}


def _nearest(x, fmt):
    """The nearest code's value (ties to even), within the format's range."""
    step = torch.ones_like(x)
    if fmt == "e4m3":
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-TOP[fmt], TOP[fmt])
