"""Attention of prompts over the 8-bit cache (more than 64 query rows of a KV head): the bars and the reference are
test_kv8_gpu.py's."""
import math

import pytest

from test_kv8_gpu import Batch, close, offsets

pytestmark = pytest.mark.gpu


def run(iam, torch, heads, kv, dim, page, fmt, lens, new, window, dtype, seed=7, scale=0.0, q=None):
    dt, cu = getattr(torch, dtype), offsets(new)
    b = Batch(iam, torch, lens, kv, dim, page, fmt, seed=seed)
    if q is None:
        q = torch.randn(cu[-1] + 3, heads, dim, generator=torch.Generator().manual_seed(9))
    q = q.to(dt).cuda()
    q[cu[-1]:] = math.nan
    out, lse = torch.full_like(q, 3.0), torch.full((q.shape[0], heads), 3.0, device="cuda")
    h = iam.KV8(heads, kv, dim)
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    h.attention(b.cache, q, b.seq_lens, out, cu=cud, max_q=max(new), window=window, lse=lse, scale=scale)
    h.status()
    assert (out[cu[-1]:] == 3.0).all() and (lse[cu[-1]:] == 3.0).all()
    want = b.attention_reference(q[:cu[-1]], cu, window, torch, scale)
    close(out[:cu[-1]], lse[:cu[-1]], want, torch)
    again = torch.zeros_like(out)
    h.attention(b.cache, q, b.seq_lens, again, cu=cud, max_q=max(new), window=window, scale=scale)
    assert torch.equal(out[:cu[-1]], again[:cu[-1]])
    h.close()


@pytest.mark.timeout(300)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv,dim,page,lens,new,window", [
    (4, 4, 64, 64, [130], [130], 0), (8, 2, 128, 64, [300], [200], 0), (4, 1, 128, 16, [257, 90, 600], [257, 80, 3], 0),
    (16, 2, 64, 32, [400, 0, 129], [130, 0, 129], 100), (2, 2, 128, 128, [1000], [520], 0), (3, 1, 64, 16, [700], [300], 128),
    (8, 8, 128, 16, [65, 66], [65, 66], 1)])
def test_prompt_attention(iam, cuda, dtype, fmt, heads, kv, dim, page, lens, new, window):
    import torch
    run(iam, torch, heads, kv, dim, page, fmt, lens, new, window, dtype)


@pytest.mark.timeout(300)
def test_prompt_rows_before_position_0(iam, cuda):
    import torch
    run(iam, torch, 4, 1, 128, 64, "e4m3", [50, 0, 300], [200, 70, 100], 0, "bfloat16")


@pytest.mark.timeout(300)
def test_prompt_with_growing_scores(iam, cuda):
    """Keys that grow along the context raise the row maximum in every tile, by more and by less than the lag."""
    import torch
    q = torch.randn(153, 2, 128, generator=torch.Generator().manual_seed(2)) * torch.linspace(0.1, 30, 153)[:, None, None]
    run(iam, torch, 2, 1, 128, 16, "int8", [900], [150], 0, "float16", q=q)
    run(iam, torch, 2, 1, 128, 16, "int8", [900], [150], 0, "bfloat16", q=q, scale=0.5)


@pytest.mark.timeout(300)
@pytest.mark.parametrize("small", [-10, -30, -126])
def test_prompt_over_pages_whose_scales_differ_widely(iam, cuda, small):
    """The largest value scale comes late; pages of zeros (scale 2^-126) and of far smaller values keep their weight."""
    import torch
    b = Batch(iam, torch, [500], 1, 64, 16, "int8", seed=4)
    for i, t in enumerate(b.table[0]):
        b.vs[t] = 2.0 ** (small if i % 3 == 0 else 5 if i > 20 else 0)
        if small == -126 and i % 3 == 0:
            b.v.view(torch.uint8)[t] = 0
    q = torch.randn(130, 2, 64, device="cuda").half()
    out, lse = torch.zeros_like(q), torch.zeros(130, 2, device="cuda")
    h = iam.KV8(2, 1, 64)
    h.attention(b.cache, q, b.seq_lens, out, cu=torch.tensor([0, 130], dtype=torch.int32, device="cuda"), lse=lse)
    h.status()
    want = b.attention_reference(q, [0, 130], 0, torch)
    ref, lse_ref, A, V = want
    tol = torch.finfo(torch.float16).eps / 2 * ref.abs() + (V * (A * 2.0 ** -15 + 2.0 ** -11))[..., None] + 2.0 ** -24
    assert ((out.double() - ref).abs() <= tol).all()
    assert float((lse.double() - lse_ref).abs().max()) < 1e-3


@pytest.mark.timeout(300)
def test_prompt_page_out_of_range(iam, cuda):
    import torch
    b = Batch(iam, torch, [200, 200], 1, 64, 16, "e4m3")
    b.block_table[1, 3] = -7
    q = torch.randn(400, 2, 64, device="cuda", dtype=torch.bfloat16)
    out = torch.zeros_like(q)
    h = iam.KV8(2, 1, 64)
    cu = [0, 200, 400]
    h.attention(b.cache, q, b.seq_lens, out, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    with pytest.raises(iam.IamError) as e:
        h.status()
    assert e.value.code == iam.IAM_ERR_ARG
    h.status()
    want = b.attention_reference(q[:200], [0, 200, 200], 0, torch)
    close(out[:200], None, want, torch)
    assert out.isfinite().all()


@pytest.mark.timeout(300)
@pytest.mark.parametrize("heads,kv,dim,page,fmt,lens,new,window", [
    (8, 2, 128, 64, "int8", [300], [200], 0), (4, 1, 128, 16, "e4m3", [700, 330], [150, 330], 0), (16, 2, 64, 32, "int8", [500, 400], [90, 160], 130),
    (32, 8, 128, 64, "e4m3", [900], [256], 0)])
def test_prompt_attention_repeats_to_the_bit(iam, cuda, heads, kv, dim, page, fmt, lens, new, window):
    """Row tiles with unequal work (masked tiles in one and not in the other), many times over: a tile's sums are read when
    all of its products are in, however far the other row tile is behind."""
    import torch
    cu = offsets(new)
    b = Batch(iam, torch, lens, kv, dim, page, fmt, seed=5)
    q = torch.randn(cu[-1], heads, dim, generator=torch.Generator().manual_seed(3)).half().cuda()
    h, out, first = iam.KV8(heads, kv, dim), torch.empty_like(q), None
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    off = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(3000):
        h.attention(b.cache, q, b.seq_lens, out, cu=cud, max_q=max(new), window=window)
        if first is None:
            first = out.clone()
            close(first, None, b.attention_reference(q, cu, window, torch), torch)
        off += (out != first).any()
    h.status()
    assert int(off) == 0


@pytest.mark.timeout(300)
@pytest.mark.parametrize("gap", [0, 8, 3])
@pytest.mark.parametrize("heads,kv,dim,new", [(3, 1, 128, [43, 61, 90, 1]), (5, 1, 64, [57, 103, 2]), (1, 1, 128, [129, 257, 300])])
def test_row_tiles_that_end_inside_a_warp(iam, cuda, heads, kv, dim, new, gap):
    """Lanes with and without a row beside each other, in every warp of a tile; results at 16-byte boundaries, off them, and in
    some rows on and in others off them (a gap of 3 elements between the heads)."""
    import torch
    cu, lens = offsets(new), [n + 70 * i for i, n in enumerate(new)]
    b = Batch(iam, torch, lens, kv, dim, 16, "int8", seed=9)
    q = torch.randn(cu[-1], heads, dim, generator=torch.Generator().manual_seed(4)).half().cuda()
    room = torch.full((cu[-1] + 1, heads, dim + gap), 5.0, dtype=torch.half, device="cuda")
    out, lse = room[:cu[-1], :, gap:], torch.empty(cu[-1], heads, device="cuda")
    h = iam.KV8(heads, kv, dim)
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    h.attention(b.cache, q, b.seq_lens, out, cu=cud, lse=lse)
    h.status()
    close(out, lse, b.attention_reference(q, cu, 0, torch), torch)
    assert (room[cu[-1]:] == 5.0).all() and (room[:, :, :gap] == 5.0).all()
    h.close()


@pytest.mark.timeout(300)
@pytest.mark.parametrize("heads,kv,dim,page,fmt,lens,new,window,dtype", [
    (4, 2, 128, 64, "e4m3", [700], [500], 0, "float32"), (2, 1, 64, 16, "int8", [900, 350], [400, 350], 200, "float32"),
    (2, 2, 256, 64, "int8", [420], [330], 0, "float32"), (2, 1, 256, 32, "e4m3", [500], [300], 0, "bfloat16"),
    (4, 1, 256, 128, "int8", [300, 200], [150, 3], 90, "float16")])
def test_long_prompts_in_fp32_and_of_large_heads(iam, cuda, heads, kv, dim, page, fmt, lens, new, window, dtype):
    """Several hundred rows in the forms that the tcgen05 kernel does not take."""
    import torch
    run(iam, torch, heads, kv, dim, page, fmt, lens, new, window, dtype)
