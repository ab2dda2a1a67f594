"""Attention over the 8-bit cache where one token has nearly all of the weight and thousands of others share the rest:
small weights keep their part in the values, in each kernel and type.

One key is (64, 0, ...), the others are 0, and a query is (c, 0, ...) with the scale 2^-6: its scores are c and 0, exactly.
With w = exp(-c), the dominant token's value 0 and the others' small positive integers (one page scale, exact in every type),
    out = w sum v / (1 + w n),   lse = c + ln(1 + w n)      over the n others that a row sees.
Tolerance.  The exponent c log2 e is off by its two roundings and the difference's, 3 |c| 2^-24 of a weight (c < 26: 2^-17.7),
its power by 2^-22.  A sum over n tokens is made of runs of 16 added in fp32, n / 16 steps of at most 2^-23 of the sum each (the
matrix instructions may cut instead of rounding).  A weight rounded to fp16 is off by 2^-12 of itself in kernels that hold one term
of it, 2^-22 with two, but never by less than half a step of fp16's smallest numbers, 2^-25 over the lift that the kernel
gives its weights: n V 2^-25 / lift in all.  The sum of the weights themselves is such a sum too: in the thread that holds the
dominant token's 1 every one of its n / 16 steps rounds to a step of fp32 at 1, whatever the size of what is added, so the sum
is off by n / 16 2^-24 and its logarithm by as much (in out it is one of the two sums counted there)."""
import math

import pytest

from test_kv8_gpu import offsets

pytestmark = pytest.mark.gpu
PAGE = 64


def run(iam, torch, heads, kv, dim, seqs, lens, new, dtype, fmt, c, two_terms, lift, max_q):
    dt = getattr(torch, dtype)
    pages = -(-max(lens) // PAGE)
    g = torch.Generator().manual_seed(dim + heads)
    k = torch.zeros(pages, kv, PAGE, dim)
    k[0, :, 0, 0] = 64
    v = torch.randint(1, 8, (pages, kv, PAGE, dim), generator=g).float()
    v[0, :, 0] = 0
    code = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    one = torch.ones(pages, kv, device="cuda")
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(seqs, pages).contiguous()  # every sequence the same pages
    cache = iam.KV8Cache(k.to(code).cuda(), v.to(code).cuda(), one, one.clone(), table)
    cu = offsets([new] * seqs)
    q = torch.zeros(cu[-1], heads, dim, dtype=dt, device="cuda")
    q[:, :, 0] = c
    out, lse = torch.empty_like(q), torch.empty(cu[-1], heads, device="cuda")
    lens_dev = torch.tensor([lens[i % len(lens)] for i in range(seqs)], dtype=torch.int32, device="cuda")
    h = iam.KV8(heads, kv, dim)
    h.attention(cache, q, lens_dev, out, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_q=max_q, scale=2.0 ** -6, lse=lse)
    h.status()
    c = float(q[0, 0, 0])
    w = math.exp(-c)
    total = v.double().transpose(0, 1).reshape(kv, -1, dim).cumsum(1).cuda()  # [kv][tokens][dim]
    for i in range(seqs):
        n = lens[i % len(lens)]
        seen = torch.arange(n - new, n, device="cuda")  # the others that each row sees
        others = seen.double()[:, None]
        want = (w * total[:, seen].transpose(0, 1) / (1 + w * others[:, None])).repeat_interleave(heads // kv, 1)
        steps = n / 16 * 2.0 ** -23
        rel = 2.0 ** -17 + 2 * steps + (2.0 ** -21 if two_terms else 2.0 ** -12) + torch.finfo(dt).eps / 2
        tol = rel * want + n * 7 * 2.0 ** -25 / lift + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
        err = (out[cu[i]:cu[i + 1]].double() - want).abs()
        assert (err <= tol).all(), (i, float((err / want).max()), float((tol / want).min()))
        sums = c + torch.log1p(w * others)
        e = (lse[cu[i]:cu[i + 1]].double() - sums).abs()
        assert (e <= sums * 2.0 ** -22 + w * others * rel + 2.0 ** -20 + steps).all(), (i, float(e.max()))
    h.close()


# weights on the edges of fp16's range: 1.5 x 2^-18 less a bit, between two steps of 2^-24; 2^-21.4; below half a step
@pytest.mark.parametrize("c", [12.06, 14.82, 17.95])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim,seqs", [(16, 8, 128, 160), (8, 8, 64, 320), (8, 4, 256, 150), (4, 4, 128, 1)])
def test_small_weights_in_decoding(iam, cuda, heads, kv, dim, seqs, dtype, fmt, c):
    """Enough sequences that each is read by few warps (several thousand tokens a warp), and one that many CTAs share."""
    import torch
    run(iam, torch, heads, kv, dim, seqs, [6001, 4097], 1, dtype, fmt, c, dtype == "float32", 2.0 ** 14, 1)


@pytest.mark.parametrize("c", [12.06, 14.82, 17.95])
@pytest.mark.parametrize("heads,kv,dim,seqs,new,dtype,two_terms,lift", [
    (2, 1, 128, 3, 70, "float32", True, 2.0 ** 12), (2, 1, 256, 2, 64, "bfloat16", False, 2.0 ** 12), (2, 2, 64, 1, 300, "float16", False, 2.0 ** 7),
    (4, 1, 128, 2, 130, "bfloat16", False, 2.0 ** 7)])
def test_small_weights_in_prompts(iam, cuda, heads, kv, dim, seqs, new, dtype, two_terms, lift, c):
    import torch
    run(iam, torch, heads, kv, dim, seqs, [4000], new, dtype, "int8", c, two_terms, lift, new)
