"""Refusals of the query / key norm with rotary positions and of attention over packed documents, without a GPU: the C entries return an error
before anything is launched, the Python functions raise."""
import ctypes as C
import math

import pytest
import torch

from osu_diffusion_amd import _lib, ops

P = 4096  # a pointer that is never read


def rope(**kw):
    r = _lib.Rope(_lib.PREC_BF16, 4, 2, 64, 64, 0, 1, 0, 1e-6, 1.0, 10, 512, 512, 512, 512, 512, 512, P, P, None, None)
    for n, v in kw.items():
        setattr(r, n, v)
    return r


def docs(**kw):
    a = _lib.DocAttention(_lib.PREC_BF16, 4, 2, 64, 3, 100, 100, -1, -1, 0, 0, 0, 0.125, 0.0, 512, 512, 512, 256, 256, 256, 128, 128, P, P, None, None)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("change", [dict(heads=0), dict(kv_heads=-1), dict(head_dim=0), dict(head_dim=63), dict(head_dim=130), dict(rot_dim=66), dict(rot_dim=3),
                                    dict(rot_dim=-2), dict(eps=0.0), dict(eps=math.nan), dict(rows=-1), dict(ld_q=255), dict(ld_k=127), dict(ld_q_out=255),
                                    dict(ld_k_out=0), dict(positions=None), dict(freqs=None)])
def test_rope_refuses(change):
    L = _lib.lib()
    assert L.osud_op_qk_norm_rope(C.byref(rope(**change)), P, P, P, P, None) == _lib.ERR_ARG
    assert b"op_qk_norm_rope" in L.osud_last_error()
    assert L.osud_op_qk_norm_rope_bwd(C.byref(rope(**change)), P, P, P, P, P, P, None, None, None, 0, None) == _lib.ERR_ARG


def test_rope_refuses_pointers_precisions_and_workspaces():
    L = _lib.lib()
    ok = rope()
    for args in ((None, P, P, P), (P, None, P, P), (P, P, None, P), (P, P, P, None), (P + 1, P, P, P)):
        assert L.osud_op_qk_norm_rope(C.byref(ok), *args, None) == _lib.ERR_ARG
    assert L.osud_op_qk_norm_rope(None, P, P, P, P, None) == _lib.ERR_ARG
    assert L.osud_op_qk_norm_rope(C.byref(rope(precision=_lib.PREC_FP8)), P, P, P, P, None) == _lib.ERR_UNSUPPORTED
    f16 = rope(precision=_lib.PREC_F16)
    assert L.osud_op_qk_norm_rope_bwd(C.byref(f16), P, P, P, P, P, P, None, None, None, 0, None) == _lib.ERR_UNSUPPORTED
    n = L.osud_op_qk_norm_rope_ws(64)
    assert n > 0 and L.osud_op_qk_norm_rope_ws(0) == 0
    assert L.osud_op_qk_norm_rope_bwd(C.byref(ok), P, P, P, P, P, P, P, P, None, 0, None) == _lib.ERR_ARG
    assert L.osud_op_qk_norm_rope_bwd(C.byref(ok), P, P, P, P, P, P, P, P, P, n - 1, None) == _lib.ERR_ARG
    assert L.osud_op_qk_norm_rope_bwd(C.byref(rope(ld_dq=255)), P, P, P, P, P, P, None, None, None, 0, None) == _lib.ERR_ARG


def test_nothing_to_do_is_no_error():
    L = _lib.lib()
    assert L.osud_op_qk_norm_rope(C.byref(rope(rows=0)), None, None, None, None, None) == _lib.OK
    assert L.osud_op_doc_attention(C.byref(docs(rows_q=0)), None, P, P, None, None, None, 0, None) == _lib.OK
    assert L.osud_op_doc_attention(C.byref(docs(n_docs=0, q_begin=None, k_begin=None)), P, P, P, P, None, None, 0, None) == _lib.OK


@pytest.mark.parametrize("change", [dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(head_dim=60), dict(head_dim=136), dict(head_dim=0), dict(n_docs=-1),
                                    dict(rows_q=-1), dict(rows_k=1 << 30), dict(cap=-1.0), dict(cap=math.nan), dict(cap=math.inf), dict(cap=1e-6), dict(scale=math.nan), dict(scale=0.0), dict(scale=-1.0), dict(q_begin=None),
                                    dict(k_begin=None), dict(ld_q=248), dict(ld_q=516), dict(ld_k=120), dict(ld_v=1 << 24), dict(ld_out=255)])
def test_attention_refuses(change):
    L = _lib.lib()
    assert L.osud_op_doc_attention(C.byref(docs(**change)), P, P, P, P, P, None, 0, None) == _lib.ERR_ARG
    assert b"op_doc_attention" in L.osud_last_error()
    assert L.osud_op_doc_attention_bwd(C.byref(docs(**change)), P, P, P, P, P, P, P, P, P, P, 1 << 20, None) == _lib.ERR_ARG
    assert L.osud_op_doc_attention_ws(C.byref(docs(**change)), 1) == 0


def test_attention_refuses_pointers_precisions_and_workspaces():
    L = _lib.lib()
    ok = docs()
    for args in ((None, P, P, P), (P, None, P, P), (P, P, None, P), (P, P, P, None), (P + 8, P, P, P), (P, P + 4, P, P)):
        assert L.osud_op_doc_attention(C.byref(ok), *args, P, None, 0, None) == _lib.ERR_ARG
    assert L.osud_op_doc_attention(None, P, P, P, P, P, None, 0, None) == _lib.ERR_ARG
    assert L.osud_op_doc_attention(C.byref(docs(precision=_lib.PREC_BF16X3)), P, P, P, P, P, None, 0, None) == _lib.ERR_UNSUPPORTED
    assert L.osud_op_doc_attention_bwd(C.byref(docs(precision=_lib.PREC_F16)), P, P, P, P, P, P, P, P, P, P, 1 << 20, None) == _lib.ERR_UNSUPPORTED
    need = 2 * 4 * 100
    assert L.osud_op_doc_attention_ws(C.byref(ok), 1) >= need
    for at in range(9):
        args = [P] * 9
        args[at] = None
        assert L.osud_op_doc_attention_bwd(C.byref(ok), *args, P, need, None) == _lib.ERR_ARG, at
    assert L.osud_op_doc_attention_bwd(C.byref(ok), *[P] * 9, P, need - 1, None) == _lib.ERR_ARG
    assert L.osud_op_doc_attention_bwd(C.byref(docs(ld_dk=120)), *[P] * 9, P, need, None) == _lib.ERR_ARG


def test_python_refuses_what_is_not_on_a_gpu():
    x = torch.zeros(4, 2, 64)
    with pytest.raises(_lib.NativeError):
        ops.qk_norm_rope(x, x, None, None)
    with pytest.raises(_lib.NativeError):
        ops.attention(x, x, x, ops.Documents([4], device="cpu"))


@pytest.mark.parametrize("kw", [dict(lengths=[-1]), dict(lengths=[3], kv_lengths=[3, 4]), dict(lengths=[3], prefix=[4]), dict(lengths=[3], prefix=[1, 1]),
                                dict(lengths=[3], prefix=[-1]), dict(lengths=[1 << 30])])
def test_documents_refuse(kw):
    with pytest.raises(AssertionError):
        ops.Documents(device="cpu", **kw)


def test_documents():
    d = ops.Documents([3, 0, 5], device="cpu", kv_lengths=[4, 1, 5], prefix=[0, 1, 2])
    assert d.q_begin.tolist() == [0, 3, 3, 8] and d.k_begin.tolist() == [0, 4, 5, 10] and d.prefix.tolist() == [0, 1, 2]
    assert (d.count, d.rows, d.kv_rows, d.max_len, d.max_kv_len) == (3, 8, 10, 5, 5)
    e = ops.Documents([], device="cpu")
    assert e.count == 0 and e.rows == 0 and e.q_begin.tolist() == [0]


def test_rotary_frequencies():
    """Against the closed forms in 64 bits: values are products of at most four such operations (relative 2^-50)."""
    f, gain = ops.rotary_frequencies(64, device="cpu")
    want = torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    assert gain == 1.0 and f.dtype == torch.float64 and torch.allclose(f, want, rtol=2.0 ** -48, atol=0)
    g, gain = ops.rotary_frequencies(64, scaling="linear", factor=4, device="cpu")
    assert gain == 1.0 and torch.equal(g, f / 4)
    g, _ = ops.rotary_frequencies(64, scaling="base", factor=4, device="cpu")
    assert float(g[0]) == 1.0 and abs(float(g[-1] / f[-1]) - 0.25) < 1e-12
    g, gain = ops.rotary_frequencies(64, scaling="ramp", factor=4, original_length=512, device="cpu")
    turns = 512 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.allclose(g[turns <= 1], f[turns <= 1] / 4, rtol=1e-12, atol=0)
    mid = (turns > 1) & (turns < 32)
    assert bool(mid.any()) and bool((g[mid] < f[mid]).all()) and bool((g[mid] > f[mid] / 4).all())
    assert abs(gain - (0.1 * math.log(4) + 1)) < 1e-12
    for bad in (dict(dim=3), dict(dim=4, factor=0.5), dict(dim=4, scaling="ramp", factor=2)):
        with pytest.raises(AssertionError):
            ops.rotary_frequencies(**bad, device="cpu")
    with pytest.raises(ValueError):
        ops.rotary_frequencies(4, scaling="no", device="cpu")
