"""The query / key norm with rotary positions and attention over packed documents on the GPU, against their plain 64-bit statements."""
import ctypes as C
import math

import pytest
import torch

from osu_diffusion_amd import _lib, ops
from tests.operators_oracle import attention_case, check, rope_case

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def heads_of(packed, *counts, hd):
    """Views (rows, heads, hd) of the parts of a packed projection."""
    at, out = 0, []
    for n in counts:
        out.append(packed[:, at * hd:(at + n) * hd].view(packed.shape[0], n, hd))
        at += n
    return out


def normal(seed, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


# ------------------------------------------------------------------ norms and rotary positions
ROPE = [  # rows, heads, kv_heads, head_dim, rot, interleaved, extra columns between rows
    (1, 12, 12, 64, 64, False, 0), (128, 12, 12, 64, 64, True, 0), (77, 6, 2, 64, 32, False, 8), (9, 16, 16, 72, 72, False, 0),
    (33, 16, 16, 72, 72, True, 0), (50, 3, 1, 128, 128, False, 0), (50, 3, 1, 128, 96, True, 4), (17, 1, 0, 64, 64, False, 0),
    (20, 2, 1, 10, 6, False, 0), (20, 2, 1, 10, 6, True, 1), (5, 300, 7, 8, 8, False, 0), (31, 4, 4, 126, 126, False, 0), (40, 4, 2, 80, 0, False, 0),
    (1031, 2, 2, 2, 2, True, 0), (19, 5, 5, 24, 16, False, 0),
]


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("rows,heads,kv,hd,rot,inter,extra", ROPE)
def test_rope_forward_and_backward(rows, heads, kv, hd, rot, inter, extra, dtype):
    packed = normal(1, rows, (heads + 2 * kv) * hd + extra, dtype=dtype)
    q, k = heads_of(packed, heads, kv, hd=hd)
    k = k if kv else None
    pos = torch.randint(0, 1 << 20, (rows,), generator=torch.Generator().manual_seed(2), dtype=torch.int32).to(DEV)
    freqs, gain = (None, 1.0) if rot == 0 else ops.rotary_frequencies(rot, scaling="ramp", factor=4.0, original_length=256, device=DEV)
    wq, wk = normal(3, hd, dtype=F32) * 0.2 + 1, normal(4, hd, dtype=F32) * 0.2 + 1
    how = dict(interleaved=inter, gain=gain)
    q2, k2 = ops.qk_norm_rope(q, k, pos, freqs, q_weight=wq, k_weight=wk if kv else None, **how)
    check(q2, rope_case(q, wq, pos, freqs, **how)["out"], "q")
    if kv:
        check(k2, rope_case(k, wk, pos, freqs, **how)["out"], "k")
    else:
        assert k2 is None
    if dtype == HF:
        return
    dq_up, dk_up = heads_of(normal(5, rows, (heads + kv) * hd, dtype=dtype), heads, kv, hd=hd)
    dq, dk, dwq, dwk = ops.qk_norm_rope_bwd(dq_up, dk_up if kv else None, q, k, pos, freqs, q_weight=wq, k_weight=wk if kv else None, **how)
    want = rope_case(q, wq, pos, freqs, grad=dq_up, **how)
    check(dq, want["dx"], "dq")
    check(dwq, want["dw"], "dq_weight")
    if kv:
        want = rope_case(k, wk, pos, freqs, grad=dk_up, **how)
        check(dk, want["dx"], "dk")
        check(dwk, want["dw"], "dk_weight")


def test_rope_times_without_norm_in_place_and_zero_rows():
    hd, rows = 64, 37
    packed = normal(1, rows, 3 * 4 * hd)
    before = packed.clone()
    q, k, v = heads_of(packed, 4, 4, 4, hd=hd)
    times = (torch.rand(rows, generator=torch.Generator().manual_seed(2)) * 6e5).to(DEV)
    freqs, _ = ops.rotary_frequencies(hd, device=DEV)
    want = [rope_case(x, None, times, freqs, norm=False)["out"] for x in (q, k)]
    got = ops.qk_norm_rope(q, k, times, freqs, norm=False, out=(q, k))
    assert got[0] is q
    check(q, want[0], "q")
    check(k, want[1], "k")
    assert torch.equal(v, heads_of(before, 4, 4, 4, hd=hd)[2])
    zero = torch.zeros(3, 2, hd, device=DEV, dtype=BF)
    z, _ = ops.qk_norm_rope(zero, None, times[:3], freqs)
    assert torch.equal(z, zero)
    dz, _, dw, _ = ops.qk_norm_rope_bwd(torch.ones_like(zero), None, zero, None, times[:3], freqs, q_weight=torch.ones(hd, device=DEV))
    check(dz, rope_case(zero, None, times[:3], freqs, grad=torch.ones_like(zero))["dx"], "dq")
    assert not bool(dw.any())
    none = torch.empty(0, 2, hd, device=DEV, dtype=BF)
    assert ops.qk_norm_rope(none, None, times[:0], freqs)[0].shape == (0, 2, hd)
    assert not bool(ops.qk_norm_rope_bwd(none, None, none, None, times[:0], freqs, q_weight=torch.ones(hd, device=DEV))[2].any())


def test_rope_many_rows_and_large_values():
    """More rows than workgroups hold at once (weight gradients of 12000 x 3 heads), values whose squares pass bf16's and half's ranges."""
    rows, hd = 12000, 64
    q, k = normal(1, rows, 2, hd), normal(2, rows, 1, hd)
    pos = torch.arange(rows, device=DEV, dtype=torch.int32)
    freqs, _ = ops.rotary_frequencies(hd, device=DEV)
    w = torch.ones(hd, device=DEV)
    g = normal(3, rows, 2, hd)
    got = ops.qk_norm_rope_bwd(g, g[:, :1].contiguous(), q, k, pos, freqs, q_weight=w, k_weight=w)
    again = ops.qk_norm_rope_bwd(g, g[:, :1].contiguous(), q, k, pos, freqs, q_weight=w, k_weight=w)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    want = rope_case(q, w, pos, freqs, grad=g)
    check(got[0], want["dx"], "dq")
    check(got[2], want["dw"], "dq_weight")
    big = normal(4, 10, 2, hd, dtype=HF, scale=3e4).clamp(-6e4, 6e4)
    check(ops.qk_norm_rope(big, None, pos[:10], freqs)[0], rope_case(big, None, pos[:10], freqs)["out"], "q")


# ------------------------------------------------------------------ attention
MASKS = {
    "all": {}, "causal": dict(right=0), "band": dict(left=20, right=7), "self": dict(left=0, right=0), "left": dict(left=33),
    "prefix": dict(right=0, prefix=True), "prefix_band": dict(left=5, right=3, prefix=True), "cap": dict(cap=5.0), "slopes": dict(slopes=True),
    "cap_slopes_causal": dict(cap=30.0, slopes=True, right=0), "cap_large": dict(cap=80.0), "cap_band": dict(cap=2.0, left=10, right=4),
    "slopes_causal": dict(slopes=True, right=0), "slopes_prefix_causal": dict(slopes=True, right=0, prefix=True),
}
LENGTHS = [1, 0, 31, 130, 2, 64, 0, 257, 65]


def attention_inputs(dtype, heads, kv, hd, lengths, kv_lengths=None, tail=3, seed=1, packed=True):
    nq, nk = sum(lengths) + tail, sum(kv_lengths if kv_lengths is not None else lengths) + tail
    if packed and kv_lengths is None:
        return heads_of(normal(seed, nq, (heads + 2 * kv) * hd, dtype=dtype, scale=1.3), heads, kv, kv, hd=hd)
    return (normal(seed, nq, heads, hd, dtype=dtype, scale=1.3), *heads_of(normal(seed + 1, nk, 2 * kv * hd, dtype=dtype, scale=1.3), kv, kv, hd=hd))


def compare(q, k, v, lengths, kv_lengths=None, prefix=None, d_out=None, **how):
    docs = ops.Documents(lengths, device=DEV, kv_lengths=kv_lengths, prefix=prefix)
    want = attention_case(q, k, v, lengths, kv_lengths=kv_lengths, prefix=prefix, d_out=d_out, **how)
    out, lse = ops.attention(q, k, v, docs, return_lse=True, **how)
    check(out, want["out"], "out")
    check(lse, want["lse"], "lse")
    if d_out is not None:
        for name, got in zip(("dq", "dk", "dv"), ops.attention_bwd(d_out, q, k, v, out, lse, docs, **how)):
            check(got, want[name], name)
    return out, lse


def how_of(mask, heads, lengths):
    how = dict(MASKS[mask])
    prefix = [int(0.4 * n) for n in lengths] if how.pop("prefix", False) else None
    if how.pop("slopes", False):
        how["slopes"] = (2.0 ** -torch.arange(1, heads + 1).float()).to(DEV)
    return how, prefix


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("mask", list(MASKS))
def test_attention_masks_and_scores(mask, dtype):
    heads, kv, hd = 4, 2, 64
    q, k, v = attention_inputs(dtype, heads, kv, hd, LENGTHS)
    how, prefix = how_of(mask, heads, LENGTHS)
    compare(q, k, v, LENGTHS, prefix=prefix, d_out=None if dtype == HF else normal(7, *q.shape, dtype=dtype), **how)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv,hd", [(1, 1, 8), (3, 1, 40), (4, 4, 64), (5, 1, 72), (2, 2, 96), (6, 2, 104), (8, 1, 128), (2, 2, 128), (1, 1, 16)])
def test_attention_heads(heads, kv, hd, dtype):
    lengths = [70, 1, 129, 200]
    q, k, v = attention_inputs(dtype, heads, kv, hd, lengths, seed=3)
    d_out = normal(8, *q.shape, dtype=dtype)
    compare(q, k, v, lengths, d_out=d_out)
    compare(q, k, v, lengths, d_out=d_out, right=0, cap=20.0, slopes=torch.full((heads,), 0.01, device=DEV))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("queries,keys", [([1, 1, 1], [5, 900, 2000]), ([3, 0, 17], [64, 10, 1500]), ([130, 2, 5], [100, 0, 3]), ([1], [4096]), ([40, 1], [700, 1])])
def test_attention_of_few_queries_and_many_keys(queries, keys, dtype):
    """Other numbers of queries and keys, among them documents with no keys, with more queries than keys, and one query against many keys
    (split over the keys and joined)."""
    heads, kv, hd = 8, 2, 128
    q, k, v = attention_inputs(dtype, heads, kv, hd, queries, keys, tail=2, seed=11)
    d_out = None if dtype == HF else normal(12, *q.shape, dtype=dtype)
    compare(q, k, v, queries, keys, d_out=d_out)
    compare(q, k, v, queries, keys, d_out=d_out, right=0, slopes=torch.full((heads,), 0.02, device=DEV))
    compare(q, k, v, queries, keys, d_out=d_out, left=100, right=0, cap=10.0, prefix=[min(7, n) for n in keys])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 192, 193, 320])
def test_attention_lengths(length, dtype):
    q, k, v = attention_inputs(dtype, 2, 1, 64, [length, length], tail=0, seed=length)
    compare(q, k, v, [length, length], d_out=normal(9, *q.shape, dtype=dtype), right=0)


def test_attention_long_document():
    """2500 positions: several blocks per row whose maxima differ, large scores."""
    q, k, v = attention_inputs(BF, 2, 1, 64, [2500], tail=0, seed=21)
    q = (q * 3).contiguous()
    d_out = normal(22, *q.shape)
    compare(q, k, v, [2500], d_out=d_out)
    compare(q, k, v, [2500], d_out=d_out, right=0, cap=50.0)
    ramp = (torch.arange(2500, device=DEV)[:, None, None] / 100.0).to(BF)  # the row maximum grows with every block
    compare(q.abs(), (k.abs() * 0.1 + ramp).contiguous(), v.contiguous(), [2500], d_out=d_out, scale=0.05)


def test_other_documents_and_the_tail_have_no_influence():
    """NaN and infinity in other documents, behind the last one and between the columns of other tensors."""
    lengths = [70, 40, 129]
    q, k, v = (t.contiguous() for t in attention_inputs(BF, 4, 2, 72, lengths, tail=10))
    d_out = normal(5, *q.shape)
    docs = ops.Documents(lengths, device=DEV)
    how = dict(right=3, left=50)
    out, lse = ops.attention(q, k, v, docs, return_lse=True, **how)
    grads = ops.attention_bwd(d_out, q, k, v, out, lse, docs, **how)
    assert not bool(out[sum(lengths):].any()) and bool((lse[:, sum(lengths):] == -math.inf).all()) and not any(bool(g[sum(lengths):].any()) for g in grads)
    dirty = [t.clone() for t in (q, k, v, d_out)]
    for t in dirty:
        t[70:110] = math.nan
        t[sum(lengths):] = math.inf
    out2, lse2 = ops.attention(*dirty[:3], docs, return_lse=True, **how)
    grads2 = ops.attention_bwd(dirty[3], *dirty[:3], out2, lse2, docs, **how)
    keep = torch.tensor([i < 70 or i >= 110 for i in range(q.shape[0])], device=DEV)
    assert torch.equal(out2[keep], out[keep]) and torch.equal(lse2[:, keep], lse[:, keep])
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(grads2, grads))


def test_rows_behind_the_last_document_stay_as_they_are():
    lengths, rows = [33, 70], 120
    q, k, v = attention_inputs(BF, 2, 2, 64, lengths, tail=rows - sum(lengths))
    docs = ops.Documents(lengths, device=DEV)
    out = torch.full((rows, 2, 64), 7.0, device=DEV, dtype=BF)
    _, lse = ops.attention(q, k, v, docs, out=out, return_lse=True)
    assert bool((out[103:] == 7).all()) and bool((out[:103] != 7).any())
    packed = torch.full((rows, 6 * 64), 9.0, device=DEV, dtype=BF)
    ops.attention_bwd(out, q, k, v, out, lse, docs, grads=heads_of(packed, 2, 2, 2, hd=64))
    assert bool((packed[103:] == 9).all())
    for got, want in zip(heads_of(packed, 2, 2, 2, hd=64), ops.attention_bwd(out, q, k, v, out, lse, docs)):
        assert torch.equal(got[:103], want[:103])


def test_documents_without_rows():
    """No documents at all, only empty ones, queries without any key row: zeros, no gradients."""
    q, k, v = normal(1, 10, 2, 64), normal(2, 6, 1, 64), normal(3, 6, 1, 64)
    for lengths, kv in (([], []), ([0, 0], [0, 0]), ([4, 0], [0, 6])):
        docs = ops.Documents(lengths, device=DEV, kv_lengths=kv)
        out, lse = ops.attention(q, k, v, docs, return_lse=True)
        grads = ops.attention_bwd(q, q, k, v, out, lse, docs)
        assert not bool(out.any()) and bool((lse == -math.inf).all()) and not any(bool(g.any()) for g in grads)
    none = torch.empty(0, 1, 64, device=DEV, dtype=BF)
    docs = ops.Documents([10], device=DEV, kv_lengths=[0])
    out, lse = ops.attention(q, none, none, docs, return_lse=True)
    dq, dk, dv = ops.attention_bwd(q, q, none, none, out, lse, docs)
    assert not bool(out.any()) and not bool(dq.any()) and dk.shape == none.shape
    docs = ops.Documents([0], device=DEV, kv_lengths=[6])
    out, lse = ops.attention(none, k, v, docs, return_lse=True)
    dq, dk, dv = ops.attention_bwd(none, none, k, v, out, lse, docs)
    assert out.shape == none.shape and not bool(dk.any()) and not bool(dv.any())


def test_large_scores_and_every_magnitude_of_a_cap():
    """Scores of thousands without a cap; caps from a thousandth of the scores to a thousand times them (both forms of the tanh in one tile)."""
    lengths = [150, 70]
    q, k, v = (t.contiguous() for t in attention_inputs(F32, 2, 2, 64, lengths, tail=0, seed=5))
    d_out = normal(6, *q.shape, dtype=F32)
    compare(q * 300, k, v, lengths, d_out=d_out)
    for cap in (0.01, 1.0, 7.0, 59.0, 61.0, 1e4):
        compare(q * 3, k, v, lengths, d_out=d_out, cap=cap)
    q[::7] *= 30  # outliers
    for dtype in (BF, F32):
        compare(q.to(dtype), k.to(dtype), v.to(dtype), lengths, d_out=d_out.to(dtype), cap=20.0, right=0)


def test_same_bits_every_time_and_on_another_stream():
    lengths = [300, 5, 1000]
    q, k, v = attention_inputs(BF, 4, 1, 128, lengths, tail=0)
    d_out = normal(5, *q.shape)
    docs = ops.Documents(lengths, device=DEV)

    def step():
        out, lse = ops.attention(q, k, v, docs, right=0, return_lse=True)
        return (out, lse, *ops.attention_bwd(d_out, q, k, v, out, lse, docs, right=0))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    third = step()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, second, third))


def test_offsets_past_32_bits():
    """Keys and values as columns of rows 2 MiB apart: the last row starts 8 GiB behind the first."""
    rows, ld, hd = 4100, 1 << 20, 64
    store = torch.empty(rows, ld, device=DEV, dtype=BF)
    store[:, :2 * hd] = normal(1, rows, 2 * hd)
    k, v = store[:, :hd].view(rows, 1, hd), store[:, hd:2 * hd].view(rows, 1, hd)
    q = normal(2, 3, 2, hd)
    compare(q, k, v, [1, 2], [3, rows - 3], d_out=None, right=0)
    kc, vc = k.contiguous(), v.contiguous()
    q = normal(3, rows, 1, hd)
    docs = ops.Documents([rows - 100, 100], device=DEV)
    d_out = normal(4, rows, 1, hd)
    want, lse = ops.attention(q, kc, vc, docs, right=0, return_lse=True)
    got, _ = ops.attention(q, k, v, docs, right=0, return_lse=True)
    assert torch.equal(got, want)
    big = (store[:, 2 * hd:3 * hd].view(rows, 1, hd), store[:, 3 * hd:4 * hd].view(rows, 1, hd), store[:, 4 * hd:5 * hd].view(rows, 1, hd))
    for a, b in zip(ops.attention_bwd(d_out, q, k, v, got, lse, docs, right=0, grads=big), ops.attention_bwd(d_out, q, kc, vc, want, lse, docs, right=0)):
        assert torch.equal(a, b)
    freqs, _ = ops.rotary_frequencies(hd, device=DEV)
    pos = torch.arange(rows, device=DEV, dtype=torch.int32)
    assert torch.equal(ops.qk_norm_rope(k, None, pos, freqs)[0], ops.qk_norm_rope(kc, None, pos, freqs)[0])


def test_offsets_out_of_order_stay_inside_the_tensors():
    """Device offsets that are past the rows, negative or decreasing are clamped: the good documents are right, no other row of the results moves."""
    q, k, v = (t.contiguous() for t in attention_inputs(BF, 2, 2, 64, [64, 64, 64], tail=0))
    docs = ops.Documents([64, 64, 64], device=DEV)
    want = ops.attention(q, k, v, docs)
    docs.q_begin.copy_(torch.tensor([0, 64, 128, 1 << 29]))
    docs.k_begin.copy_(torch.tensor([0, 64, 128, 1 << 29]))
    assert torch.equal(ops.attention(q, k, v, docs), want)
    docs.k_begin.copy_(torch.tensor([-5, 64, 20, 192]))
    assert torch.equal(ops.attention(q, k, v, docs)[:64], want[:64])


# ------------------------------------------------------------------ refusals, gradients, graphs, the operators together
def test_refusals_on_the_gpu():
    q, k, v = attention_inputs(BF, 4, 2, 64, [10], tail=0, packed=False)
    docs = ops.Documents([10], device=DEV)
    with pytest.raises(AssertionError):
        ops.attention(q, k.float(), v.float(), docs)
    with pytest.raises(AssertionError):
        ops.attention(q, k[:, :, :56], v[:, :, :56], docs)
    with pytest.raises(AssertionError):
        ops.attention(q.transpose(0, 1), k, v, docs)
    with pytest.raises(AssertionError):
        ops.attention(q, k, v, ops.Documents([11], device=DEV))
    with pytest.raises(AssertionError):
        ops.attention(q, k, v, ops.Documents([10], device="cpu"))
    with pytest.raises(AssertionError):
        ops.attention(q, k, v, docs, left=-1)
    with pytest.raises(AssertionError):
        ops.attention(q, k, v, docs, cap=-1.0)
    with pytest.raises(AssertionError):
        ops.attention(q, k, v, docs, slopes=torch.zeros(2, device=DEV))
    with pytest.raises(AssertionError):
        ops.attention(q, k, v, docs, slopes=torch.zeros(4, device=DEV, requires_grad=True))
    with pytest.raises(AssertionError):
        ops.attention(normal(1, 10, 3, 64), k, v, docs)
    with pytest.raises(AssertionError):
        ops.attention(normal(1, 1, 4, 64).expand(10, 4, 64), k, v, docs)  # every row the same memory
    odd = torch.zeros(10 * 4 * 64 + 1, device=DEV, dtype=BF)[1:].view(10, 4, 64)  # not 16-byte aligned
    with pytest.raises(AssertionError):
        ops.attention(odd, k, v, docs)
    h = normal(1, 10, 4, 64, dtype=HF).requires_grad_()
    with pytest.raises(AssertionError):
        ops.attention(h, h, h, docs)
    freqs, _ = ops.rotary_frequencies(64, device=DEV)
    pos = torch.arange(10, device=DEV, dtype=torch.int32)
    with pytest.raises(AssertionError):
        ops.qk_norm_rope(q, k, pos.long(), freqs)
    with pytest.raises(AssertionError):
        ops.qk_norm_rope(q, k, pos[:9], freqs)
    with pytest.raises(AssertionError):
        ops.qk_norm_rope(q, k, pos, freqs.float())
    with pytest.raises(AssertionError):
        ops.qk_norm_rope(q, k, pos, ops.rotary_frequencies(66, device=DEV)[0])
    with pytest.raises(AssertionError):
        ops.qk_norm_rope(q, k, pos, freqs, q_weight=torch.ones(32, device=DEV))
    with pytest.raises(AssertionError):
        ops.qk_norm_rope(q, k[:9], pos, freqs)


def block(packed, wq, wk, pos, freqs, docs, heads, kv, hd, how):
    q, k, v = heads_of(packed, heads, kv, kv, hd=hd)
    q, k = ops.qk_norm_rope(q, k, pos, freqs, q_weight=wq, k_weight=wk)
    return ops.attention(q, k, v, docs, **how)


def test_together_with_autograd_against_differences():
    """Packed projection -> norm and rotation -> attention -> loss, fp32 tier: the gradient along a direction against the difference quotient of the
    64-bit statement (step 1e-6 in 64 bits: truncation 1e-12, cancellation 1e-10; the kernels' fp32 roundings: 1e-5 of the terms' sizes)."""
    heads, kv, hd, lengths = 4, 2, 24, [20, 1, 37]
    rows = sum(lengths)
    how = dict(right=0, cap=8.0, slopes=torch.full((heads,), 0.05, device=DEV))
    docs = ops.Documents(lengths, device=DEV)
    pos = torch.cat([torch.arange(n) for n in lengths]).float().to(DEV)
    freqs, _ = ops.rotary_frequencies(16, device=DEV)
    leaves = [normal(1, rows, (heads + 2 * kv) * hd, dtype=F32), normal(2, hd, dtype=F32) * 0.2 + 1, normal(3, hd, dtype=F32) * 0.2 + 1]
    weight = normal(4, rows, heads, hd, dtype=F32)
    ts = [t.clone().requires_grad_() for t in leaves]
    (block(*ts, pos, freqs, docs, heads, kv, hd, how) * weight).sum().backward()

    def loss(ls):
        q, k, v = heads_of(ls[0], heads, kv, kv, hd=hd)
        q, k = rope_case(q, ls[1], pos, freqs)["out"][0], rope_case(k, ls[2], pos, freqs)["out"][0]
        got = attention_case(q, k, v, lengths, **how)["out"][0]
        return float((got * weight.double().cpu()).sum())

    base = [t.double().cpu() for t in leaves]
    for i, name in enumerate(("packed", "q_weight", "k_weight")):
        for seed in (1, 2):
            d = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
            up, down = ([b + s * 1e-6 * d if j == i else b for j, b in enumerate(base)] for s in (1, -1))
            want, got = (loss(up) - loss(down)) / 2e-6, float((ts[i].grad.double().cpu() * d).sum())
            size = float((ts[i].grad.double().cpu().abs() * d.abs()).sum())
            assert abs(got - want) <= 1e-4 * size, (name, got, want, size)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_autograd_is_the_explicit_backward(dtype):
    heads, kv, hd, lengths = 4, 2, 64, [100, 29]
    rows = sum(lengths) + 4
    docs = ops.Documents(lengths, device=DEV, prefix=[10, 0])
    pos = torch.arange(rows, device=DEV, dtype=torch.int32)
    freqs, _ = ops.rotary_frequencies(hd, device=DEV)
    how = dict(right=0)
    packed = normal(1, rows, (heads + 2 * kv) * hd, dtype=dtype)
    wq, wk = torch.ones(hd, device=DEV), torch.ones(hd, device=DEV)
    d_out = normal(2, rows, heads, hd, dtype=dtype)
    ts = [t.clone().requires_grad_() for t in (packed, wq, wk)]
    out = block(*ts, pos, freqs, docs, heads, kv, hd, how)
    out.backward(d_out)
    q0, k0, v = heads_of(packed, heads, kv, kv, hd=hd)
    q, k = ops.qk_norm_rope(q0, k0, pos, freqs, q_weight=wq, k_weight=wk)
    o, lse = ops.attention(q, k, v, docs, return_lse=True, **how)
    assert torch.equal(o, out)
    dq, dk, dv = ops.attention_bwd(d_out, q, k, v, o, lse, docs, **how)
    dq, dk, dwq, dwk = ops.qk_norm_rope_bwd(dq, dk, q0, k0, pos, freqs, q_weight=wq, k_weight=wk)
    assert torch.equal(ts[0].grad, torch.cat([t.reshape(rows, -1) for t in (dq, dk, dv)], 1))
    assert torch.equal(ts[1].grad, dwq) and torch.equal(ts[2].grad, dwk)


def test_a_step_captured_into_a_graph():
    """Forward and backward of both operators, captured once and replayed on new values, with eager work between the replays; two graphs."""
    heads, kv, hd, lengths, rows = 4, 2, 64, [100, 1, 300], 401
    docs = ops.Documents(lengths, device=DEV)
    pos = torch.arange(rows, device=DEV, dtype=torch.int32)
    freqs, _ = ops.rotary_frequencies(hd, device=DEV)
    w = torch.ones(hd, device=DEV)
    packed, d_out = normal(1, rows, 8 * hd), normal(2, rows, heads, hd)

    def step():
        q0, k0, v = heads_of(packed, heads, kv, kv, hd=hd)
        q, k = ops.qk_norm_rope(q0, k0, pos, freqs, q_weight=w, k_weight=w)
        out, lse = ops.attention(q, k, v, docs, right=0, return_lse=True)
        dq, dk, dv = ops.attention_bwd(d_out, q, k, v, out, lse, docs, right=0)
        return (out, dv, *ops.qk_norm_rope_bwd(dq, dk, q0, k0, pos, freqs, q_weight=w, k_weight=w))

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got))
    for seed in (3, 4, 5):
        packed.copy_(normal(seed, rows, 8 * hd))
        want = step()
        for g, got in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, got in graphs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_leaves_are_refused_inside_a_capture():
    q = normal(1, 10, 2, 64).requires_grad_()
    docs = ops.Documents([10], device=DEV)
    eager = ops.attention(q, q, q, docs)  # an eager graph of the same leaf lives
    g = torch.cuda.CUDAGraph()
    with pytest.raises(_lib.NativeError):
        with torch.cuda.graph(g):
            ops.attention(q, q, q, docs)
    eager.sum().backward()
    assert q.grad is not None


@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_queries_of_documents_without_any_key_row(dtype):
    """A document that is long on the query side only, and tensors of keys without rows: the backward pass has nothing to split over."""
    q, none = normal(1, 2100, 2, 64, dtype=dtype), torch.empty(0, 1, 64, device=DEV, dtype=dtype)
    docs = ops.Documents([2100], device=DEV, kv_lengths=[0])
    out, lse = ops.attention(q, none, none, docs, return_lse=True)
    dq, dk, dv = ops.attention_bwd(q, q, none, none, out, lse, docs)
    assert not bool(out.any()) and bool((lse == -math.inf).all()) and not bool(dq.any()) and dk.shape == dv.shape == none.shape


def test_rope_more_rows_than_a_launch_has_threads_for():
    """2^27 + 13 rows of one small head: every turn of every workgroup, compared where a workgroup's second turn begins and at both ends."""
    rows, period = (1 << 27) + 13, 4099
    base = normal(1, period, 1, 2)
    q = base.repeat(rows // period + 1, 1, 1)[:rows]
    pos = torch.arange(rows, device=DEV, dtype=torch.int32) % period
    freqs, _ = ops.rotary_frequencies(2, device=DEV)
    out, _ = ops.qk_norm_rope(q, None, pos, freqs)
    one, _ = ops.qk_norm_rope(base, None, pos[:period].contiguous(), freqs)
    check(one, rope_case(base, None, pos[:period], freqs)["out"], "q")
    whole = rows // period * period
    assert bool((out[:whole].view(-1, period, 2).view(torch.int32) == one.view(1, period, 2).view(torch.int32)).all())
    assert torch.equal(out[whole:], one[:rows - whole])


def test_constants_that_want_a_gradient_are_refused_beside_trained_tensors():
    """slopes, positions and freqs have no gradient: asking for one raises, also where q, k and v have theirs."""
    q = normal(1, 10, 2, 64).requires_grad_()
    docs = ops.Documents([10], device=DEV)
    slopes = torch.ones(2, device=DEV, requires_grad=True)
    with pytest.raises(AssertionError):
        ops.attention(q, q, q, docs, slopes=slopes)
    freqs, _ = ops.rotary_frequencies(64, device=DEV)
    times = torch.arange(10, device=DEV).float()
    with pytest.raises(AssertionError):
        ops.qk_norm_rope(q, q, times.clone().requires_grad_(), freqs)
    with pytest.raises(AssertionError):
        ops.qk_norm_rope(q, q, times, freqs.clone().requires_grad_())
    with torch.no_grad():  # (nothing is asked for here)
        ops.attention(q, q, q, docs, slopes=slopes)


def test_gradients_that_arrive_unaligned():
    """The upstream gradient as a piece of a longer vector's, one element past 16-byte alignment."""
    q, k, v = (t.contiguous().requires_grad_() for t in attention_inputs(BF, 2, 2, 64, [20], tail=0))
    docs = ops.Documents([20], device=DEV)
    flat = normal(7, 1 + q.numel())
    d_out = flat[1:].view(q.shape)
    assert d_out.data_ptr() % 16
    got = torch.autograd.grad(ops.attention(q, k, v, docs), (q, k, v), d_out)
    want = torch.autograd.grad(ops.attention(q, k, v, docs), (q, k, v), d_out.clone())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    freqs, _ = ops.rotary_frequencies(64, device=DEV)
    pos = torch.arange(20, device=DEV, dtype=torch.int32)
    # (chunks of another width: the same formula, sums in another order; the difference is at most both results' own rounding and fp32 sums)
    for up in (d_out, d_out.clone()):
        got = torch.autograd.grad(ops.qk_norm_rope(q, None, pos, freqs)[0], q, up)[0]
        check(got, rope_case(q.detach(), None, pos, freqs, grad=up)["dx"], "dq")


def test_results_written_into_given_tensors_are_seen_by_autograd():
    """A graph that saved the old values raises in its backward; a tensor that requires grad is not written to with grad mode on."""
    docs = ops.Documents([10], device=DEV)
    q, k = normal(1, 10, 2, 64), normal(2, 10, 2, 64)
    freqs, _ = ops.rotary_frequencies(64, device=DEV)
    pos = torch.arange(10, device=DEV, dtype=torch.int32)
    with torch.no_grad():
        out, lse = ops.attention(q, k, k, docs, return_lse=True)
    writes = [lambda t: ops.qk_norm_rope(t, None, pos, freqs, out=(t, None)), lambda t: ops.attention(q, k, k, docs, out=t),
              lambda t: ops.attention_bwd(q, q, k, k, out, lse, docs, grads=(torch.empty_like(q), t, torch.empty_like(q)))]
    for write in writes:
        leaf = normal(3, 10, 2, 64).requires_grad_()
        saved = leaf * 1
        loss = saved.square().sum()
        with torch.no_grad():
            write(saved)
        with pytest.raises(RuntimeError, match="inplace operation"):
            loss.backward()
    for write in writes[1:]:
        with pytest.raises(AssertionError):
            write(normal(3, 10, 2, 64).requires_grad_())
    with torch.inference_mode():
        for write in writes:
            write(normal(3, 10, 2, 64))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("right", [None, 0])
def test_slopes_of_either_sign(right, dtype):
    """Scores that rise with the distance, fall with it, or (0) ignore it: different heads of one call."""
    lengths, heads = [150, 1, 300], 6
    q, k, v = attention_inputs(dtype, heads, 2, 64, lengths)
    d_out = normal(9, q.shape[0], heads, 64, dtype=dtype)
    slopes = torch.tensor([-0.5, -0.01, 0.0, 0.02, 0.4, 3.0], device=DEV)
    compare(q, k, v, lengths, d_out=d_out, right=right, slopes=slopes)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("how", [{}, dict(cap=50.0), dict(cap=2.0), dict(cap=90.0), dict(slopes=True), dict(cap=15.0, slopes=True)])
def test_a_row_that_sees_one_key_returns_its_value(how, dtype):
    """Its weight is 1 whatever the score: p / sum p differs from 1 by a few fp32 roundings, far less than half a step of the 16-bit type, so v comes back bit
    for bit -- from documents of one key, a mask of one key, and a long cache whose keys are split over workgroups."""
    how = dict(how)
    if how.pop("slopes", False):
        how["slopes"] = torch.tensor([0.5, 0.01], device=DEV)
    q, v = normal(1, 300, 2, 96, dtype=dtype), normal(2, 300, 2, 96, dtype=dtype)
    assert torch.equal(ops.attention(q, q, v, ops.Documents([1] * 300, device=DEV), **how), v)
    assert torch.equal(ops.attention(q, q, v, ops.Documents([300], device=DEV), left=0, right=0, **how), v)
    k, v = normal(3, 4100, 2, 96, dtype=dtype), normal(4, 4100, 2, 96, dtype=dtype)
    docs = ops.Documents([1, 1], device=DEV, kv_lengths=[4000, 100])
    assert torch.equal(ops.attention(q[:2], k, v, docs, left=0, right=0, **how), v[[3999, 4099]])
