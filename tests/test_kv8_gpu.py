"""The 8-bit paged KV cache (iam_kv8_*): the append against its definition, bit for bit, and the attention
against softmax attention in 64 bits over the cache's own values.

Tolerance of the attention, with A the largest score's sum of magnitudes (scale * sum |q_d k_d|) of a row and V
the largest |value| it sees: queries keep 22 bits (fp32) or all of theirs (fp16 and bf16 shifted into fp16), and
a score's up to 256 products are added in fp32, so scores are off by at most A (2^-22 + 2^-16) < A 2^-15.9; a
probability then has that relative error, 2 ulp of its power and its rounding to fp16 (16-bit types: 2^-11) or
to 22 bits (fp32: 2^-22); the sums of products add 2^-16 V at most; and one rounding to the type.  A row
of outputs, being a mean of values weighted by probabilities, is off by at most
    eps/2 |out| + V (2 A 2^-16 + 2^-11 or 2^-20 + 2^-16).
That bounds every element; over a whole result errors average, and its 2-norm is held to eps of the 2-norm
(fp32: 2e-5)."""
import math

import pytest

TOP = {"int8": 127.0, "e4m3": 448.0}
DTYPES = ("float32", "float16", "bfloat16")


def code_dtype(fmt, torch):
    return torch.int8 if fmt == "int8" else torch.float8_e4m3fn


def scale_of(amax, fmt):
    """The smallest power of two >= 2^-126 with amax <= top * scale, by search over the exponents (python floats)."""
    e = -126
    if amax > 0:
        e = max(-126, math.frexp(amax)[1] - 12)
        while amax > TOP[fmt] * 2.0 ** e:
            e += 1
    return 2.0 ** e


def nearest(x, fmt, torch):
    """Values to the nearest code's value, ties to even, in 64 bits; infinities to the largest, NaN to 0."""
    x = torch.nan_to_num(x.double(), nan=0.0, posinf=TOP[fmt], neginf=-TOP[fmt]).clamp(-TOP[fmt], TOP[fmt])
    step = torch.ones_like(x)
    if fmt == "e4m3":
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-TOP[fmt], TOP[fmt])


def reference_append(codes, scales, table, new, cu, lens, page, fmt, torch):
    """codes [pages][kv][page][dim] and scales [pages][kv] in 64 bits after appending new [rows][kv][dim]."""
    codes, scales = codes.double().clone(), scales.double().clone()
    for i, n in enumerate(lens):
        start = n - (cu[i + 1] - cu[i])
        first = max(start, 0)
        for c in range(first // page, (n + page - 1) // page):
            lo, hi = max(first, c * page), min(n, (c + 1) * page)
            if lo >= hi or c >= len(table[i]) or not 0 <= table[i][c] < codes.shape[0]:
                continue
            at, held = table[i][c], lo - c * page
            for h in range(codes.shape[1]):
                x = new[cu[i] + lo - start:cu[i] + hi - start, h].double()
                fin = x[x.isfinite()].abs()
                s = scale_of(float(fin.max()) if fin.numel() else 0.0, fmt)
                if held and float(scales[at, h]) > s:
                    s = float(scales[at, h])
                if held:
                    codes[at, h, :held] = nearest(codes[at, h, :held] * (scales[at, h] / s), fmt, torch)
                codes[at, h, held:held + hi - lo] = nearest(x / s, fmt, torch)
                scales[at, h] = s
    return codes, scales


def reference_attention(q, k, v, ks, vs, table, cu, lens, window, scale, torch):
    """-> out, lse in 64 bits, and the tolerance's A and V of each (row, head); rows of no sequence stay 0."""
    rows, heads, dim = q.shape
    kvh, page = k.shape[1], k.shape[2]
    out = torch.zeros(rows, heads, dim, dtype=torch.float64, device=q.device)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64, device=q.device)
    A, V = torch.zeros_like(lse), torch.zeros_like(lse)
    scale = scale or 1 / math.sqrt(dim)
    for i, n in enumerate(lens):
        if n == 0 or cu[i] == cu[i + 1]:
            continue
        ids = torch.tensor(table[i][: -(-n // page)], device=q.device)
        kk = (k[ids].double() * ks[ids].double()[..., None, None]).transpose(0, 1).reshape(kvh, -1, dim)[:, :n]
        vv = (v[ids].double() * vs[ids].double()[..., None, None]).transpose(0, 1).reshape(kvh, -1, dim)[:, :n]
        for r in range(cu[i], cu[i + 1]):
            pos = n - (cu[i + 1] - r)
            if pos < 0:
                continue
            lo = max(0, pos - window + 1) if window else 0
            for h in range(heads):
                kh, vh = kk[h // (heads // kvh), lo:pos + 1], vv[h // (heads // kvh), lo:pos + 1]
                s = kh @ q[r, h].double() * scale
                out[r, h] = torch.softmax(s, 0) @ vh
                lse[r, h] = torch.logsumexp(s, 0)
                A[r, h] = (kh.abs() @ q[r, h].double().abs()).max() * scale
                V[r, h] = vh.abs().max()
    return out, lse, A, V


def close(got_out, got_lse, want, torch):
    out, lse, A, V = want
    eps, half = torch.finfo(got_out.dtype).eps, got_out.dtype != torch.float32
    tol = eps / 2 * out.abs() + (V * (A * 2.0 ** -15 + (2.0 ** -11 if half else 2.0 ** -20) + 2.0 ** -16))[..., None]
    err = (got_out.double() - out).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-300)).max())
    norm = float(out.norm())
    if norm:
        assert float(err.norm()) <= (eps if half else 2e-5) * norm, float(err.norm()) / norm
    if got_lse is not None:
        seen = lse.isfinite()
        assert torch.equal(got_lse.isfinite(), seen) and (got_lse[~seen] == -math.inf).all()
        e = (got_lse.double() - lse).abs()[seen]
        assert (e <= (A * 2.0 ** -15 + 2.0 ** -20 + lse.abs() * 2.0 ** -23)[seen]).all()


class Batch:
    """Sequences of given lengths in pages scattered over a pool, filled with values by the definition."""

    def __init__(self, iam, torch, lens, kv, dim, page, fmt, seed=0, spare=3, big=1.0):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        width = max(max(need), 1) + 1
        self.table, at = [], 0
        for c in need:
            self.table.append(order[at:at + c])
            at += c
        rows = [t + [-1] * (width - len(t)) for t in self.table]
        shape = (self.pages, kv, page, dim)
        x = torch.randn(2, *shape, generator=g) * big
        x[0, :, :, :, ::17] *= 4
        x[:, :: 2] *= 8  # pages of different scales
        amax = x.abs().amax((3, 4))
        s = torch.tensor([scale_of(float(a), fmt) for a in amax.flatten()]).view(amax.shape)
        codes = nearest(x / s[..., None, None], fmt, torch).float().to(code_dtype(fmt, torch))
        raw = codes.view(torch.uint8)
        for i, n in enumerate(lens):  # behind the last token: e4m3's NaN
            if n % page:
                raw[:, self.table[i][n // page], :, n % page:] = 0x7F
        free = [p for p in order if p not in {y for t in self.table for y in t}]
        raw[:, free] = 0x7F
        self.lens, self.page, self.fmt = lens, page, fmt
        self.k, self.v = codes[0].cuda(), codes[1].cuda()
        self.ks, self.vs = s[0].float().cuda(), s[1].float().cuda()
        self.block_table = torch.tensor(rows, dtype=torch.int32, device="cuda")
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.cache = iam.KV8Cache(self.k, self.v, self.ks, self.vs, self.block_table)

    def attention_reference(self, q, cu, window, torch, scale=0.0):
        return reference_attention(q, self.k, self.v, self.ks, self.vs, self.table, cu, self.lens, window, scale, torch)


def offsets(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


# ------------------------------------------------------------------ append

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("page,kv,dim,lens,new", [
    (16, 2, 64, [1, 17, 40], [1, 1, 1]), (64, 8, 128, [5, 64, 65, 128, 200], [1, 1, 1, 1, 1]),
    (32, 1, 256, [70, 31, 33, 32], [70, 5, 33, 32]), (128, 2, 64, [300, 5, 0, 129, 128], [171, 5, 0, 2, 127]),
    (16, 3, 128, [100], [99]), (128, 1, 256, [256], [256])])
def test_append_is_exact(iam, cuda, dtype, fmt, page, kv, dim, lens, new):
    import torch
    dt, cu = getattr(torch, dtype), offsets(new)
    b = Batch(iam, torch, lens, kv, dim, page, fmt, seed=page + dim)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(cu[-1] + 2, 2 * kv, dim, generator=g)
    x[:, ::2] *= 40  # some pages' scales grow, some stay
    x[0, 0, 0], x[0, kv, 1], x[-3, 0, 2] = math.inf, math.nan, -math.inf
    x = x.to(dt).cuda()
    h = iam.KV8(kv, kv, dim)
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    want = [reference_append(c, s, b.table, r, cu, lens, page, fmt, torch) for c, s, r in
            ((b.k, b.ks, x[:, :kv]), (b.v, b.vs, x[:, kv:]))]
    h.append(b.cache, x[:, :kv], x[:, kv:], b.seq_lens, cu=cud)
    h.status()
    for (codes, scales), got, got_s in ((want[0], b.k, b.ks), (want[1], b.v, b.vs)):
        assert torch.equal(got_s.double(), scales)
        assert torch.equal(torch.nan_to_num(got.double(), nan=1e9), torch.nan_to_num(codes, nan=1e9))
    if all(n == 1 for n in new):  # one row per sequence without offsets: the same
        codes = b.k.view(torch.uint8).clone()
        h.append(b.cache, x[:cu[-1], :kv], x[:cu[-1], kv:], b.seq_lens)
        assert torch.equal(codes, b.k.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_values_at_the_ends_of_the_ranges(iam, cuda, fmt):
    """Zero, subnormal, largest and just-above-a-power amounts; ties; a page that only ever held zeros."""
    import torch
    top = TOP[fmt]
    rows = [0.0, 2.0 ** -149, 2.0 ** -127, 3.4028234e38, top, top * (1 + 2.0 ** -23), top * 2.0 ** -20, 1.5 * 2.0 ** 100, 2.0 ** -126 * top]
    for page in (16,):
        for later in (False, True):
            x = torch.zeros(len(rows), 1, 64)
            for i, r in enumerate(rows):
                x[i, 0] = r * torch.linspace(-1, 1, 64)
                x[i, 0, 5] = r
                x[i, 0, 6] = r / 2
            n = len(rows)
            lens = [3 if later else 1] * n
            b = Batch(iam, torch, lens, 1, 64, page, fmt, seed=1)
            if later:  # earlier tokens of all zeros: their page has the smallest scale
                for t in b.table:
                    b.k.view(torch.uint8)[t[0], 0, :2] = 0
                    b.v.view(torch.uint8)[t[0], 0, :2] = 0
                    b.ks[t[0]] = b.vs[t[0]] = 2.0 ** -126
            want = reference_append(b.k, b.ks, b.table, x, list(range(n + 1)), lens, page, fmt, torch)
            want_v = reference_append(b.v, b.vs, b.table, -x, list(range(n + 1)), lens, page, fmt, torch)
            h = iam.KV8(1, 1, 64)
            h.append(b.cache, x.cuda(), (-x).cuda(), b.seq_lens)
            h.status()
            for got, got_s, (codes, scales) in ((b.k, b.ks, want), (b.v, b.vs, want_v)):
                assert torch.equal(got_s.double(), scales)
                assert torch.equal(torch.nan_to_num(got.double(), nan=1e9), torch.nan_to_num(codes, nan=1e9))


@pytest.mark.gpu
def test_append_token_by_token_equals_the_definition_step_by_step(iam, cuda):
    """200 tokens one at a time, growing in size: each step shifts what its page holds."""
    import torch
    torch.manual_seed(3)
    x = torch.randn(200, 2, 64) * torch.exp(torch.linspace(0, 8, 200))[:, None, None]
    b = Batch(iam, torch, [200], 2, 64, 64, "int8")
    codes, scales = b.k.clone(), b.ks.clone()
    h = iam.KV8(2, 2, 64)
    for t in range(200):
        lens = torch.tensor([t + 1], dtype=torch.int32, device="cuda")
        h.append(b.cache, x[t:t + 1].cuda(), x[t:t + 1].cuda(), lens)
        codes, scales = reference_append(codes, scales, b.table, x[t:t + 1].cuda(), [0, 1], [t + 1], 64, "int8", torch)
        if t % 20 == 19 or t in (63, 64, 65):
            assert torch.equal(b.ks.double(), scales) and torch.equal(b.k.double(), codes)
    h.status()


@pytest.mark.gpu
def test_append_skips_what_has_no_place(iam, cuda):
    """Bad page numbers, a sequence longer than its table, rows before position 0: nothing else is written, the
    first two are reported, and the word is cleared."""
    import torch
    h = iam.KV8(1, 1, 64)
    x = torch.ones(3, 1, 64, device="cuda")
    for case in ("page", "long", "before", "offsets", "negative"):
        b = Batch(iam, torch, [20, 20, 20], 1, 64, 16, "int8")
        cu, lens = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda"), b.seq_lens.clone()
        if case == "page":
            b.block_table[1, 1] = b.pages
        if case == "long":
            lens[1] = 16 * b.block_table.shape[1] + 1
        if case == "before":
            lens[1] = 0
        if case == "offsets":
            cu[2] = 7
        if case == "negative":
            lens[1] = -5
        before = b.k.clone()
        h.append(b.cache, x, x, lens, cu=cu)
        if case == "before":
            h.status()
        else:
            with pytest.raises(iam.IamError) as e:
                h.status()
            assert e.value.code == iam.IAM_ERR_ARG
        h.status()
        changed = (b.k != before).any(-1).any(-1).any(-1).nonzero().flatten().tolist()
        allowed = {b.table[0][1], b.table[2][1]}
        assert set(changed) <= allowed and b.table[0][1] in changed
    torch.cuda.synchronize()


# ------------------------------------------------------------------ attention

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv,dim,page,lens,window", [
    (4, 2, 64, 16, [1], 0), (32, 8, 128, 64, [100, 1, 64, 65], 0), (8, 1, 256, 32, [33, 700], 0), (2, 2, 128, 128, [5000], 0),
    (8, 8, 64, 16, [17, 1000, 16, 15, 2], 0), (16, 2, 128, 64, [300, 90], 77), (6, 2, 64, 32, [0, 40, 0], 0), (4, 1, 128, 16, [500, 3], 1),
    (24, 2, 64, 64, [130], 0)])
def test_decode_attention(iam, cuda, dtype, fmt, heads, kv, dim, page, lens, window):
    import torch
    dt = getattr(torch, dtype)
    b = Batch(iam, torch, lens, kv, dim, page, fmt, seed=len(lens))
    q = torch.randn(len(lens), heads, dim, generator=torch.Generator().manual_seed(9)).to(dt).cuda()
    out, lse = torch.full_like(q, 3.0), torch.full((len(lens), heads), 3.0, device="cuda")
    h = iam.KV8(heads, kv, dim)
    h.attention(b.cache, q, b.seq_lens, out, window=window, lse=lse)
    h.status()
    close(out, lse, b.attention_reference(q, list(range(len(lens) + 1)), window, torch), torch)
    again = torch.zeros_like(out)
    h.attention(b.cache, q, b.seq_lens, again, window=window)
    assert torch.equal(out, again)
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv,dim,page,lens,new,window", [
    (4, 2, 64, 16, [5], [5], 0), (32, 8, 128, 64, [100, 200], [7, 3], 0), (8, 1, 256, 32, [70, 65, 10], [70, 1, 0], 0),
    (16, 2, 128, 16, [90, 33, 200], [9, 33, 64], 20), (2, 2, 64, 128, [400], [300], 0), (4, 4, 128, 64, [3, 70, 0], [5, 70, 2], 0),
    (6, 2, 64, 16, [129, 64], [65, 64], 64), (8, 1, 128, 64, [1500], [2], 0)])
def test_rows_attention(iam, cuda, dtype, fmt, heads, kv, dim, page, lens, new, window):
    import torch
    dt, cu = getattr(torch, dtype), offsets(new)
    b = Batch(iam, torch, lens, kv, dim, page, fmt, seed=7)
    spare = 2  # rows behind the last sequence stay as they are
    q = torch.randn(cu[-1] + spare, heads, dim, generator=torch.Generator().manual_seed(9)).to(dt).cuda()
    q[cu[-1]:] = math.nan
    out, lse = torch.full_like(q, 3.0), torch.full((q.shape[0], heads), 3.0, device="cuda")
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    h = iam.KV8(heads, kv, dim)
    want = b.attention_reference(q[:cu[-1]], cu, window, torch)
    for max_q in (0, max(new), 1):  # each kernel is right for any number of rows
        out.fill_(3.0)
        lse.fill_(3.0)
        h.attention(b.cache, q, b.seq_lens, out, cu=cud, max_q=max_q, window=window, lse=lse)
        h.status()
        assert (out[cu[-1]:] == 3.0).all() and (lse[cu[-1]:] == 3.0).all()
        close(out[:cu[-1]], lse[:cu[-1]], want, torch)
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("max_q", [1, 0])
@pytest.mark.parametrize("size", [1e-30, 1.0, 300.0])
def test_queries_of_any_size(iam, cuda, max_q, size):
    """fp32 and bf16 queries far outside fp16's range, and scores that leave one token all the weight."""
    import torch
    for dt in (torch.float32, torch.bfloat16):
        b = Batch(iam, torch, [90, 40], 2, 64, 16, "int8", seed=2)
        q = (torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(1)) * size).to(dt).cuda()
        q[0, 0] *= 2.0 ** 10
        out, lse = torch.zeros_like(q), torch.zeros(2, 4, device="cuda")
        cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
        h = iam.KV8(4, 2, 64)
        h.attention(b.cache, q, b.seq_lens, out, cu=cu, max_q=max_q, lse=lse)
        want = b.attention_reference(q, [0, 1, 2], 0, torch)
        tol = torch.finfo(dt).eps / 2 * want[0].abs() + (want[3] * (want[2] * 2.0 ** -15 + 2.0 ** -11))[..., None]
        assert ((out.double() - want[0]).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("max_q", [1, 0])
def test_a_row_with_nan_keeps_to_itself(iam, cuda, max_q):
    import torch
    b = Batch(iam, torch, [50, 90], 1, 64, 16, "e4m3")
    q = torch.randn(5, 2, 64, device="cuda", dtype=torch.bfloat16)
    q[1, 0, 3] = math.nan
    q[3, 1, 0] = math.inf
    cu = [0, 2, 5]
    out = torch.zeros_like(q)
    h = iam.KV8(2, 1, 64)
    h.attention(b.cache, q, b.seq_lens, out, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_q=max_q)
    clean = q.clone()
    clean[1, 0], clean[3, 1] = 0, 0
    want = b.attention_reference(clean, cu, 0, torch)
    assert out[1, 0].isnan().all()
    hurt = torch.zeros(5, 2, dtype=torch.bool, device="cuda")
    hurt[1, 0] = hurt[3, 1] = True
    tol = (want[3] * (want[2] * 2.0 ** -15 + 2.0 ** -11 + 2.0 ** -8))[..., None]
    assert ((out.double() - want[0]).abs() <= tol)[~hurt].all()


@pytest.mark.gpu
@pytest.mark.parametrize("max_q", [1, 0])
def test_pages_whose_scales_differ_widely(iam, cuda, max_q):
    """A page of zeros (the smallest scale) and pages 2^20 apart: each keeps its own precision."""
    import torch
    b = Batch(iam, torch, [96], 1, 64, 16, "int8", seed=4)
    t = b.table[0]
    b.k.view(torch.uint8)[t[0]] = 0
    b.v.view(torch.uint8)[t[0]] = 0
    b.ks[t[0]] = b.vs[t[0]] = 2.0 ** -126
    b.vs[t[1]] *= 2.0 ** -10
    b.vs[t[3]] *= 2.0 ** 10
    q = torch.randn(3, 2, 64, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(3, 2, device="cuda")
    h = iam.KV8(2, 1, 64)
    cu = [0, 3]
    h.attention(b.cache, q, b.seq_lens, out, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_q=max_q, lse=lse)
    close(out, lse, b.attention_reference(q, cu, 0, torch), torch)


@pytest.mark.gpu
def test_attention_skips_what_has_no_place(iam, cuda):
    """Bad page numbers are left out and reported; the other sequences are right."""
    import torch
    for max_q in (1, 0):
        b = Batch(iam, torch, [70, 70, 70], 1, 64, 16, "int8")
        b.block_table[1, 2] = 10 ** 6
        q = torch.randn(3, 2, 64, device="cuda")
        out = torch.zeros_like(q)
        h = iam.KV8(2, 1, 64)
        cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
        h.attention(b.cache, q, b.seq_lens, out, cu=cu, max_q=max_q)
        with pytest.raises(iam.IamError):
            h.status()
        h.status()
        want = b.attention_reference(q, [0, 1, 2, 3], 0, torch)
        keep = torch.tensor([0, 2], device="cuda")
        close(out[keep], None, tuple(w[keep] for w in want), torch)
        assert out.isfinite().all()


@pytest.mark.gpu
def test_a_long_cache_past_32_bits(iam, cuda):
    """Codes of one cache above 4 GiB, the sequence's pages at its far end."""
    import torch
    kv, dim, page = 8, 128, 128
    pages = (1 << 32) // (kv * dim * page) + 40
    k = torch.zeros(pages, kv, page, dim, dtype=torch.int8, device="cuda")
    v = torch.zeros_like(k)
    ks, vs = torch.full((pages, kv), 2.0 ** -126, device="cuda"), torch.full((pages, kv), 2.0 ** -126, device="cuda")
    table = torch.arange(pages - 1, pages - 6, -1, dtype=torch.int32, device="cuda")[None]
    cache = iam.KV8Cache(k, v, ks, vs, table)
    n = 4 * page + 7
    x = torch.randn(n, 2 * kv, dim, device="cuda", dtype=torch.float16)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    h = iam.KV8(kv, kv, dim)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    h.append(cache, x[:, :kv], x[:, kv:], lens, cu=cu)
    q = torch.randn(1, kv, dim, device="cuda")
    h.status()
    assert int((ks > 2.0 ** -126).sum()) == 5 * kv
    for max_q in (1, 0):
        out, lse = torch.zeros_like(q), torch.zeros(1, kv, device="cuda")
        h.attention(cache, q, lens, out, cu=torch.tensor([0, 1], dtype=torch.int32, device="cuda"), max_q=max_q, lse=lse)
        h.status()
        close(out, lse, reference_attention(q, k, v, ks, vs, table.tolist(), [0, 1], [n], 0, 0.0, torch), torch)


@pytest.mark.gpu
def test_strided_rows_streams_and_graphs(iam, cuda):
    """q, k, v as parts of one projection's rows at an odd offset; a call on another stream; a captured step that is
    replayed as the sequence grows."""
    import torch
    heads, kv, dim, page = 4, 2, 64, 16
    b = Batch(iam, torch, [60], kv, dim, page, "int8", seed=3, spare=4)
    h = iam.KV8(heads, kv, dim)
    width = (heads + 2 * kv) * dim
    flat = torch.randn(1 + width + 3, device="cuda")
    qkv = torch.as_strided(flat, (1, heads + 2 * kv, dim), (width, dim, 1), 1)
    out = torch.as_strided(torch.zeros(width + 5, device="cuda"), (1, heads, dim), (width, dim, 1), 3)
    lens = torch.tensor([59], dtype=torch.int32, device="cuda")

    def step():
        h.append(b.cache, qkv[:, heads:heads + kv], qkv[:, heads + kv:], lens)
        h.attention(b.cache, qkv[:, :heads], lens, out)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in (59, 60):
        lens.fill_(n)
        codes, scales = reference_append(b.k, b.ks, b.table, qkv[:, heads:heads + kv], [0, 1], [n], page, "int8", torch)
        flat.copy_(torch.randn_like(flat))
        codes, scales = reference_append(b.k, b.ks, b.table, qkv[:, heads:heads + kv], [0, 1], [n], page, "int8", torch)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b.k.double(), codes) and torch.equal(b.ks.double(), scales)
        b.lens = [n]
        close(out, None, b.attention_reference(qkv[:, :heads], [0, 1], 0, torch), torch)
    h.status()


@pytest.mark.gpu
def test_rotate_append_attend_together(iam, cuda):
    """A prompt and three single tokens as a model runs them, against fp64 attention over the cache's values."""
    import torch
    heads, kv, dim, page, n = 8, 2, 128, 32, 150
    rope, h = iam.Rope(dim, scaling="yarn", factor=4.0, original_ctx=4096), iam.KV8(heads, kv, dim)
    table = torch.randperm(8, device="cuda").to(torch.int32)[None]
    cache = iam.KV8Cache.empty(8, kv, page, dim, table, fmt="e4m3")
    for start, count in ((0, n), (n, 1), (n + 1, 1), (n + 2, 1)):
        qkv = torch.randn(count, heads + 2 * kv, dim, device="cuda", dtype=torch.bfloat16)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        positions = torch.arange(start, start + count, dtype=torch.int32, device="cuda")
        lens = torch.tensor([start + count], dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, count], dtype=torch.int32, device="cuda")
        out = torch.empty(count, heads, dim, dtype=torch.bfloat16, device="cuda")
        rope.apply(q, positions, k=k)
        h.append(cache, k, v, lens, cu=cu)
        h.attention(cache, q, lens, out, cu=cu, max_q=count)
        ck, cv, ks, vs, _ = cache.tensors
        close(out, None, reference_attention(q, ck, cv, ks, vs, table.tolist(), [0, count], [start + count], 0, 0.0, torch), torch)
    h.status()


@pytest.mark.gpu
def test_refused_calls(iam, cuda):
    import torch
    b = Batch(iam, torch, [40, 40], 2, 64, 16, "int8")
    h = iam.KV8(4, 2, 64)
    q, kx = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda")
    out = torch.zeros_like(q)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")

    def refused(f, code=iam.IAM_ERR_ARG):
        with pytest.raises(iam.IamError) as e:
            f()
        assert e.value.code == code

    good = b.cache.tensors
    odd = torch.zeros(good[0].numel() + 8, dtype=torch.int8, device="cuda")[8:].view(good[0].shape)
    for args in [(good[0].float(), *good[1:]), (good[0], good[1][:1], *good[2:]), (good[0], good[1], good[2][:1], *good[3:]),
                 (*good[:4], good[4].long()), (*good[:4], good[4][0]), (good[0].transpose(2, 3), *good[1:]), (good[0], good[1], good[2].half(), *good[3:])]:
        refused(lambda: iam.KV8Cache(*args))
    for cache in (iam.KV8Cache(odd, *good[1:]), iam.KV8Cache.empty(2, 2, 24, 64, good[4]), iam.KV8Cache.empty(2, 1, 16, 64, good[4]),
                  iam.KV8Cache.empty(2, 2, 16, 128, good[4])):
        refused(lambda: h.attention(cache, q, b.seq_lens, out))
        refused(lambda: h.append(cache, kx[:, :cache.n_kv_heads], kx[:, :cache.n_kv_heads], b.seq_lens))
    refused(lambda: h.attention(b.cache, q.double(), b.seq_lens, out))
    refused(lambda: h.attention(b.cache, q, b.seq_lens.long(), out))
    refused(lambda: h.attention(b.cache, q, b.seq_lens[:1], out))
    refused(lambda: h.attention(b.cache, q, b.seq_lens, out.half()))
    refused(lambda: h.attention(b.cache, q, b.seq_lens, out[:1].expand(2, 4, 64)))
    refused(lambda: h.attention(b.cache, q[:1], b.seq_lens, out[:1]))  # without offsets: one row per sequence
    refused(lambda: h.attention(b.cache, q, b.seq_lens, out, cu=cu[:2]))
    refused(lambda: h.attention(b.cache, q, b.seq_lens, out, cu=cu, max_q=-1))
    refused(lambda: h.attention(b.cache, q, b.seq_lens, out, window=-1))
    refused(lambda: h.attention(b.cache, q, b.seq_lens, out, scale=math.nan))
    refused(lambda: h.attention(b.cache, q, b.seq_lens, out, lse=torch.zeros(2, 2, device="cuda")))
    refused(lambda: h.append(b.cache, kx, kx.half(), b.seq_lens))
    refused(lambda: h.append(b.cache, kx[:, :1], kx[:, :1], b.seq_lens))
    refused(lambda: h.append(b.cache, kx.cpu(), kx, b.seq_lens))
    refused(lambda: iam.KV8(4, 3, 64))
    refused(lambda: iam.KV8(4, 2, 96), iam.IAM_ERR_UNSUPPORTED)


def test_refusals_that_need_no_gpu(iam):
    lib = iam.load_library()
    assert lib.iam_kv8_append(None, None, 0, 0, None, None, None, None, None) == iam.IAM_ERR_ARG
    assert lib.iam_kv8_attention(None, None, 0, 0, 0, None, None, None, 0.0, 0, None, None, None) == iam.IAM_ERR_ARG
    assert lib.iam_kv8_status(None) == iam.IAM_ERR_ARG
    assert lib.iam_kv8_destroy(None) == iam.IAM_OK and lib.iam_rope_destroy(None) == iam.IAM_OK
    assert lib.iam_rope_apply(None, 0, 1, None, 1, None, None, 0, None, None, None) == iam.IAM_ERR_ARG
    for args in [(7, 1, 8, 8), (0, -1, 8, 8), (0, 1, 0, 8), (0, 2, 8, 7)]:
        assert lib.iam_logprobs(None, *args, None, None, None, None, None, 0, None, None, None) == iam.IAM_ERR_ARG
    for k in (-1, 65, 9):
        assert lib.iam_logprobs(None, 0, 1, 8, 8, None, None, None, None, None, k, None, None, None) == iam.IAM_ERR_ARG
