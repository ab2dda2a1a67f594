"""The 8-bit cache at the ends of its arguments' ranges: windows of any size, queries overwritten by their results, the
largest tables; limits of the row counts.  Bars and reference are test_kv8_gpu.py's."""

import pytest

from test_kv8_gpu import Batch, close, nearest, offsets, reference_append

# (heads, kv, dim, new rows, type): the kernel for few rows, for some, for many
KERNELS = [(8, 2, 128, [1, 1, 1], "float16"), (4, 1, 64, [9, 30, 17], "float32"), (8, 1, 128, [60, 33, 64], "bfloat16")]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,new,dtype", KERNELS)
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30])
def test_the_largest_windows(iam, cuda, heads, kv, dim, new, dtype, window):
    """Rows before position 0 (the second sequence's) and a window of everything: as without one."""
    import torch
    cu, lens = offsets(new), [150, 0, 70]
    b = Batch(iam, torch, lens, kv, dim, 16, "int8")
    q = torch.randn(cu[-1], heads, dim, generator=torch.Generator().manual_seed(1)).to(getattr(torch, dtype)).cuda()
    out, lse = torch.empty_like(q), torch.empty(cu[-1], heads, device="cuda")
    h = iam.KV8(heads, kv, dim)
    h.attention(b.cache, q, b.seq_lens, out, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_q=max(new), window=window, lse=lse)
    h.status()
    close(out, lse, b.attention_reference(q, cu, 0, torch), torch)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,new,dtype", KERNELS)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("window,freed", [(37, True), (37, False), (100, True), (100, False)])
def test_pages_before_the_window(iam, cuda, heads, kv, dim, new, dtype, fmt, window, freed):
    """A sliding window whose earlier pages have been given back: their table entries name no page, or one that is someone
    else's by now (codes of NaN, scales of 2^100); tokens before the window in its first page are NaN."""
    import torch
    cu, lens, page = offsets(new), [150, 300, 203], 16
    b = Batch(iam, torch, lens, kv, dim, page, fmt, seed=11)
    table = b.block_table.clone()
    stale = next(p for p in range(b.pages) if all(p not in t for t in b.table))
    for x, s in ((b.k, b.ks), (b.v, b.vs)):
        x.view(torch.uint8)[stale] = 0x7F
        s[stale] = 2.0 ** 100
    q = torch.randn(cu[-1], heads, dim, generator=torch.Generator().manual_seed(6)).to(getattr(torch, dtype)).cuda()
    want = b.attention_reference(q, cu, window, torch)
    for i, (n, r) in enumerate(zip(lens, new)):
        first = max(0, n - r - window + 1)  # the first token that the sequence's first row sees
        table[i, :first // page] = -1 if freed else stale
        if first % page:
            for x in (b.k, b.v):
                x.view(torch.uint8)[b.table[i][first // page], :, :first % page] = 0x7F
    cache = iam.KV8Cache(b.k, b.v, b.ks, b.vs, table)
    out, lse = torch.empty_like(q), torch.empty(cu[-1], heads, device="cuda")
    h = iam.KV8(heads, kv, dim)
    h.attention(cache, q, b.seq_lens, out, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_q=max(new), window=window, lse=lse)
    h.status()
    close(out, lse, want, torch)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,new,dtype", KERNELS)
def test_queries_overwritten_by_their_results(iam, cuda, heads, kv, dim, new, dtype):
    """A context long enough that several CTAs share each tile of rows."""
    import torch
    cu, lens = offsets(new), [3000, 40, 900]
    b = Batch(iam, torch, lens, kv, dim, 64, "e4m3")
    q = torch.randn(cu[-1], heads, dim, generator=torch.Generator().manual_seed(2)).to(getattr(torch, dtype)).cuda()
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    h, out = iam.KV8(heads, kv, dim), torch.empty_like(q)
    h.attention(b.cache, q, b.seq_lens, out, cu=cud, max_q=max(new))
    for _ in range(3):
        x = q.clone()
        h.attention(b.cache, x, b.seq_lens, x, cu=cud, max_q=max(new))
        assert torch.equal(x, out)
    h.status()


@pytest.mark.gpu
def test_results_over_the_queries_at_other_strides_are_refused(iam, cuda):
    """Row 1's result would lie on queries that are still to be read; one row, or one head, has no such stride."""
    import torch
    b = Batch(iam, torch, [40, 40], 2, 64, 16, "int8")
    h = iam.KV8(4, 2, 64)
    flat = torch.randn(4 * 4 * 64, device="cuda")
    q = flat.view(4, 4, 64)[:2]
    for other in (torch.as_strided(flat, (2, 4, 64), (512, 64, 1)), torch.as_strided(flat, (2, 4, 64), (256, 128, 1)),
                  torch.as_strided(flat, (2, 4, 64), (64, 128, 1))):
        with pytest.raises(iam.IamError) as e:
            h.attention(b.cache, q, b.seq_lens, other)
        assert e.value.code == iam.IAM_ERR_ARG
    one = Batch(iam, torch, [40], 2, 64, 16, "int8")
    apart = torch.empty(1, 4, 64, device="cuda")
    h.attention(one.cache, q[:1], one.seq_lens, apart)
    same = torch.as_strided(flat, (1, 4, 64), (777, 64, 1))
    h.attention(one.cache, q[:1], one.seq_lens, same)
    h.status()
    assert torch.equal(same, apart)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 5, 17])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv,dim,dtype", [(4, 2, 64, "float32"), (4, 1, 128, "bfloat16"), (2, 1, 256, "float16"), (24, 1, 64, "float16"),
                                                (30, 1, 128, "float32")])
def test_lengths_around_a_group_of_tokens(iam, cuda, heads, kv, dim, dtype, fmt, window):
    """Sequences of 1 to 50 tokens with up to three rows each (the kernel for few rows and the one for some): the last token, the
    rows' own limits and the window's start at every place of a group of 16, where masks part the lanes."""
    import torch
    lens = list(range(1, 51))
    new = [1 + i % 3 for i in lens]
    cu = offsets(new)
    b = Batch(iam, torch, lens, kv, dim, 16, fmt, seed=12)
    q = torch.randn(cu[-1], heads, dim, generator=torch.Generator().manual_seed(3)).to(getattr(torch, dtype)).cuda()
    out, lse = torch.empty_like(q), torch.empty(cu[-1], heads, device="cuda")
    h = iam.KV8(heads, kv, dim)
    h.attention(b.cache, q, b.seq_lens, out, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_q=3, window=window, lse=lse)
    h.status()
    close(out, lse, b.attention_reference(q, cu, window, torch), torch)


@pytest.mark.gpu
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype,fmt,seqs,kv,dim,page,rows", [
    ("bfloat16", "int8", 120, 3, 128, 16, [1]), ("float32", "e4m3", 300, 5, 64, 32, [0, 1, 2, 7]), ("float16", "int8", 70, 5, 256, 16, [1, 30, 3]),
    ("bfloat16", "e4m3", 600, 1, 64, 16, [1, 0, 0, 17])])
def test_append_of_few_rows_to_many_sequences(iam, cuda, dtype, fmt, seqs, kv, dim, page, rows, aligned):
    """More pages and heads than blocks run at once, heads that leave a part of the last block idle, sequences without
    rows, one long one among them."""
    import torch
    g = torch.Generator().manual_seed(seqs)
    new = [rows[i % len(rows)] for i in range(seqs)]
    new[seqs // 2] = 3 * page + 5
    lens = [n + int(t) for n, t in zip(new, torch.randint(0, 2 * page, (seqs,), generator=g))]
    cu = offsets(new)
    b = Batch(iam, torch, lens, kv, dim, page, fmt, seed=3)
    x = torch.randn(cu[-1] + 2, 2 * kv, dim, generator=g)
    x[:, ::2] *= 40  # some pages' scales grow, some stay
    x = x.to(getattr(torch, dtype)).cuda()
    want = [reference_append(c, s, b.table, r, cu, lens, page, fmt, torch) for c, s, r in
            ((b.k, b.ks, x[:, :kv]), (b.v, b.vs, x[:, kv:]))]
    if not aligned:  # rows one element past a 16-byte boundary
        wide = torch.zeros(x.shape[0], 2 * kv, dim + 1, dtype=x.dtype, device="cuda")
        wide[:, :, 1:] = x
        x = wide[:, :, 1:]
    h = iam.KV8(kv, kv, dim)
    h.append(b.cache, x[:, :kv], x[:, kv:], b.seq_lens, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    h.status()
    for (codes, scales), got, got_s in ((want[0], b.k, b.ks), (want[1], b.v, b.vs)):
        assert torch.equal(got_s.double(), scales)
        assert torch.equal(torch.nan_to_num(got.double(), nan=1e9), torch.nan_to_num(codes, nan=1e9))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,fmt", [("float32", "int8"), ("bfloat16", "e4m3")])
def test_growing_scales_in_many_sequences(iam, cuda, dtype, fmt):
    """A warp a page and head: each appended token is larger than all before it, so that every page shifts what it holds
    while its scale is replaced, 40 tokens in a row for 200 sequences."""
    import torch
    seqs, kv, dim, page = 200, 2, 128, 32
    b = Batch(iam, torch, [40] * seqs, kv, dim, page, fmt, seed=6)
    codes, scales = [b.k.clone(), b.v.clone()], [b.ks.clone(), b.vs.clone()]
    h = iam.KV8(kv, kv, dim)
    g = torch.Generator().manual_seed(8)
    for t in range(40):
        x = (torch.randn(seqs, 2 * kv, dim, generator=g) * 1.6 ** t).to(getattr(torch, dtype)).cuda()
        lens = torch.full((seqs,), t + 1, dtype=torch.int32, device="cuda")
        h.append(b.cache, x[:, :kv], x[:, kv:], lens)
        if t in (7, 31, 32, 39):
            h.status()
        for i, part in enumerate((x[:, :kv], x[:, kv:])):
            # the definition for one token of each sequence, all at once (powers of two: exact)
            at = torch.tensor([r[t // page] for r in b.table], device="cuda")
            row, old = t % page, scales[i][at].double()
            amax = part.double().abs().amax(-1)
            need = torch.exp2(torch.ceil(torch.log2(amax / (127.0 if fmt == "int8" else 448.0))))
            now = torch.maximum(old, need) if row else need
            held = codes[i][at].double()
            held[:, :, :row] = nearest(held[:, :, :row] * (old / now)[..., None, None], fmt, torch)
            held[:, :, row] = nearest(part.double() / now[..., None], fmt, torch)
            codes[i][at] = held.float().to(codes[i].dtype)
            scales[i][at] = now.float()
    for got, got_s, want, want_s in ((b.k, b.ks, codes[0], scales[0]), (b.v, b.vs, codes[1], scales[1])):
        used = torch.tensor(b.table, device="cuda").flatten()
        assert torch.equal(got_s[used], want_s[used])
        last = torch.tensor([r[1] for r in b.table], device="cuda")
        first = torch.tensor([r[0] for r in b.table], device="cuda")
        assert torch.equal(got[first].float(), want[first].float())
        assert torch.equal(got[last].float()[:, :, :40 - page], want[last].float()[:, :, :40 - page])


@pytest.mark.gpu
def test_tables_and_rows_beyond_the_limits_are_refused(iam, cuda):
    import torch
    page = 128
    b = Batch(iam, torch, [40], 1, 64, page, "int8")
    h, lens = iam.KV8(1, 1, 64), b.seq_lens
    q, out = torch.zeros(1, 1, 64, device="cuda"), torch.zeros(1, 1, 64, device="cuda")
    codes = b.cache.tensors[:4]
    widest = torch.full((1, 2 ** 26 // page), -1, dtype=torch.int32, device="cuda")
    widest[:, :b.block_table.shape[1]] = b.block_table
    h.attention(iam.KV8Cache(*codes, widest), q, lens, out)
    h.status()
    too_wide = iam.KV8Cache(*codes, torch.cat((widest, widest[:, -1:]), 1))
    for call in (lambda: h.attention(too_wide, q, lens, out), lambda: h.append(too_wide, q, q, lens)):
        with pytest.raises(iam.IamError) as e:
            call()
        assert e.value.code == iam.IAM_ERR_UNSUPPORTED


def test_row_counts_beyond_the_limits_are_refused(iam):
    lib = iam.load_library()
    assert lib.iam_logprobs(None, 0, 2 ** 30 + 1, 8, 8, None, None, None, None, None, 0, None, None, None) == iam.IAM_ERR_ARG


@pytest.mark.parametrize("over", [2 ** 31, 2 ** 32, 2 ** 32 + 64, -2 ** 32])
def test_numbers_beyond_32_bits_are_refused(iam, over):
    """They would be taken modulo 2^32: a window of 2^32 as none at all.  No handle and no GPU is reached."""
    h = object.__new__(iam.KV8)
    h.h, h.device, h.n_heads, h.head_dim = None, 0, 1, 64
    h._common = lambda *a: None
    for kw in (dict(window=over), dict(max_q=over)):
        with pytest.raises(iam.IamError) as e:
            h.attention(None, None, None, None, **kw)
        assert e.value.code == iam.IAM_ERR_ARG
    for kw in (dict(head_dim=over), dict(head_dim=64, rot_dim=over), dict(head_dim=64, original_ctx=over)):
        with pytest.raises(iam.IamError) as e:
            iam.Rope.config(**kw)
        assert e.value.code == iam.IAM_ERR_ARG
