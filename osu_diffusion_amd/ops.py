"""Operators between a block's packed projection Q | K | V and its output projection, on the native kernels of libosud.so:

* ``qk_norm_rope`` -- an RMS norm of every query and key head and the rotation by position, in one pass;
* ``attention`` -- softmax attention over packed documents: no padding, no (T, T) mask tensor; band, causal and prefix masks, scores capped by
  a tanh or lowered with the distance, shared key heads, few queries against many keys.

Both have gradients: called with grad mode on they record an autograd node; ``qk_norm_rope_bwd`` and ``attention_bwd`` are the same passes for
programs that keep their own tape (or capture a step into a HIP graph).  Tensors are (rows, heads, head_dim) views with a column
stride of 1 and heads next to each other -- ``packed[:, :H * d].view(rows, H, d)`` of a projection is read where it lies.  Everything runs on
the current stream of the tensors' device; there is no fallback: a tensor that is not on a GPU raises."""
from __future__ import annotations

import ctypes as C
import math
from itertools import accumulate

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_TYPES = {torch.bfloat16: _lib.PREC_BF16, torch.float16: _lib.PREC_F16, torch.float32: _lib.PREC_F32}


# ------------------------------------------------------------------ checks that both operators share
def _heads(name, t, like=None):
    """(rows, heads, head_dim, row stride) of a tensor of heads."""
    assert isinstance(t, torch.Tensor) and t.dim() == 3, f"{name} must be a (rows, heads, head_dim) tensor"
    rows, heads, hd = t.shape
    if like is not None:
        assert t.dtype == like.dtype and t.device == like.device, f"{name} must have the type and device of the queries, got {t.dtype} on {t.device}"
    ld, step, one = t.stride()
    if ld != heads * hd or step != hd or one != 1:
        if t.numel() == 0:
            return rows, heads, hd, heads * hd
        assert (hd == 1 or one == 1) and (heads == 1 or step == hd), \
            f"{name}: the columns of a head and the heads of a row must lie next to each other, got strides {t.stride()}"
        if rows == 1:
            ld = heads * hd
    return rows, heads, hd, ld


def _precision(q):
    if q.device.type != "cuda":
        raise _lib.NativeError("osu_diffusion_amd.ops runs only on an AMD GPU through libosud.so; there is no CPU fallback")
    assert q.dtype in _TYPES, f"bfloat16, float16 or float32 tensors, got {q.dtype}"
    return _TYPES[q.dtype]


def _new(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _vector(name, t, n, dtype, device):
    assert t.dim() == 1 and t.numel() == n and t.dtype == dtype and t.device == device and t.is_contiguous(), \
        f"{name} must be a contiguous ({n},) {dtype} tensor on {device}, got {tuple(t.shape)} {t.dtype} on {t.device}"
    return t.data_ptr()


def _call(device, fn, *args):
    """fn(*args, current stream of `device`), with `device` current."""
    at = device.index
    if torch._C._cuda_getDevice() == at:  # (what torch.cuda.current_device and current_stream ask, without their objects: a call costs as much as a launch)
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(at))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(at))
    if rc:
        _lib.check(rc)


def _wants_grad(*tensors, constants=()):
    """Whether a call records a node; ``constants`` have no gradient (asked here: inside a node's forward grad mode is off)."""
    if not torch.is_grad_enabled():
        return False
    for name, t in constants:
        assert t is None or not t.requires_grad, f"{name} have no gradient"
    wants = leaf = False
    for t in tensors:
        if t is not None and t.requires_grad:
            wants, leaf = True, leaf or t.is_leaf
    if leaf and torch.cuda.is_current_stream_capturing():
        # a leaf's gradient is accumulated on the stream of its first use, whatever eager graph made that: inside a capture the engine's wait
        # for that stream ends the process
        raise _lib.NativeError("a captured graph cannot differentiate with respect to leaf tensors here: call the *_bwd functions inside the capture")
    return wants


def _written(*tensors):
    """Tensors that a kernel writes in place of new ones: autograd hears of it, so that a graph which saved their old values raises."""
    for t in tensors:
        if t is not None:
            assert not (t.requires_grad and torch.is_grad_enabled()), "a tensor that requires grad cannot be written to with grad mode on"
            if not t.is_inference():
                torch.autograd.graph.increment_version(t)


# ------------------------------------------------------------------ norms and rotary positions of queries and keys
def rotary_frequencies(dim, base=10000.0, *, scaling=None, factor=1.0, original_length=None, device="cuda"):
    """The (dim / 2,) float64 rotary frequencies base^(-2 i / dim), in radians per position, and the gain of the rotated columns.

    For contexts ``factor`` times longer than the ``original_length`` a model was trained on: ``scaling="linear"`` divides every frequency by the
    factor; ``"base"`` enlarges the base so that the lowest frequency is divided by it and the highest kept; ``"ramp"`` keeps the frequencies that
    turn at least 32 times over the original length, divides those that turn less than once, goes linearly between, and lifts the
    rotated columns by 0.1 ln(factor) + 1."""
    assert dim >= 2 and dim % 2 == 0, f"dim must be even, got {dim}"
    assert base > 0 and factor >= 1, f"base must be positive and factor at least 1, got {base} and {factor}"
    i = torch.arange(dim // 2, dtype=torch.float64)
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    f = float(base) ** (-2.0 * i / dim)
    gain = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "ramp":
        assert original_length, "scaling='ramp' needs the original length"
        keep = ((original_length * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        gain = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f"scaling must be None, 'linear', 'base' or 'ramp', got {scaling!r}")
    return f.to(device), gain


def _rope(q, k, positions, freqs, q_weight, k_weight, norm, eps, interleaved, gain):
    prec = _precision(q)
    rows, heads, hd, ld_q = _heads("q", q)
    r = _lib.Rope(prec, heads, 0, hd, 0, int(interleaved), int(norm), 0, eps, gain, rows, ld_q, 0, ld_q, 0, ld_q, 0)
    if k is not None:
        krows, r.kv_heads, khd, r.ld_k = _heads("k", k, q)
        assert (krows, khd) == (rows, hd), f"k must have the rows and the head_dim of q, got {tuple(k.shape)} and {tuple(q.shape)}"
    if freqs is not None:
        r.rot_dim = 2 * freqs.numel()
        r.freqs = _vector("freqs", freqs, freqs.numel(), torch.float64, q.device)
        assert positions is not None and positions.dtype in (torch.int32, torch.float32), "positions must be an int32 or float32 tensor"
        r.float_positions = int(positions.dtype == torch.float32)
        r.positions = _vector("positions", positions, rows, positions.dtype, q.device)
    if q_weight is not None:
        r.q_weight = _vector("q_weight", q_weight, hd, torch.float32, q.device)
    if k_weight is not None:
        r.k_weight = _vector("k_weight", k_weight, hd, torch.float32, q.device)
    assert norm or (q_weight is None and k_weight is None), "weights belong to the norm: norm=False takes none"
    return r


def _rope_results(q, k, r, out):
    if out is None:
        r.ld_q_out, r.ld_k_out = r.heads * r.head_dim, r.kv_heads * r.head_dim
        return _new(q), None if k is None else _new(k)
    q_out, k_out = out
    assert q_out.shape == q.shape and (k is None or k_out.shape == k.shape), "out must have the shapes of q and k"
    r.ld_q_out, r.ld_k_out = _heads("out[0]", q_out, q)[3], 0 if k is None else _heads("out[1]", k_out, q)[3]
    _written(q_out, None if k is None else k_out)
    return q_out, k_out


def _rope_forward(q, k, r, out):
    q_out, k_out = _rope_results(q, k, r, out)
    _call(q.device, _lib.lib().osud_op_qk_norm_rope, C.byref(r), q.data_ptr(), _ptr(k), q_out.data_ptr(), _ptr(k_out))
    return q_out, k_out


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, freqs, norm, eps, interleaved, gain):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, freqs)
        ctx.how = dict(norm=norm, eps=eps, interleaved=interleaved, gain=gain)
        q_out, k_out = _rope_forward(q, k, _rope(q, k, positions, freqs, q_weight, k_weight, norm, eps, interleaved, gain), None)
        return q_out if k is None else (q_out, k_out)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_q, d_k=None):
        q, k, q_weight, k_weight, positions, freqs = ctx.saved_tensors
        d_q = d_q.contiguous()  # (rows of any alignment: the norm and rotation take element-aligned pointers)
        d_k = None if k is None else d_k.contiguous()
        dq, dk, dqw, dkw = qk_norm_rope_bwd(d_q, d_k, q, k, positions, freqs, q_weight=q_weight, k_weight=k_weight, **ctx.how)
        return dq, dk, dqw, dkw, None, None, None, None, None, None


def qk_norm_rope(q, k, positions, freqs, *, q_weight=None, k_weight=None, norm=True, eps=1e-6, interleaved=False, gain=1.0, out=None):
    """Norm of every head of q and k (RMS over its columns, times the weight) and rotation of its first ``2 * len(freqs)`` columns by
    ``positions[row] * freqs[i]``: pairs (i, i + len(freqs)), or neighbours with ``interleaved``; ``gain`` multiplies the rotated columns.

    q (rows, heads, head_dim), k (rows, kv_heads, head_dim) or None; positions (rows,) int32 or float32 (times); freqs float64 from
    ``rotary_frequencies`` or None (norm only); weights (head_dim,) float32 or None.  Returns (q', k'), new tensors or ``out`` (a pair; may be q and k
    themselves), rounded once.  float16 has no gradients."""
    if _wants_grad(q, k, q_weight, k_weight, constants=() if freqs is None else (("positions", positions), ("freqs", freqs))):
        assert out is None, "out= cannot be combined with gradients"
        assert q.dtype != torch.float16, "the fp16 tier has no backward pass"
        got = _QkNormRope.apply(q, k, q_weight, k_weight, positions, freqs, norm, eps, interleaved, gain)
        return (got, None) if k is None else got
    return _rope_forward(q, k, _rope(q, k, positions, freqs, q_weight, k_weight, norm, eps, interleaved, gain), out)


def qk_norm_rope_bwd(d_q, d_k, q, k, positions, freqs, *, q_weight=None, k_weight=None, norm=True, eps=1e-6, interleaved=False, gain=1.0, out=None):
    """Gradients of ``qk_norm_rope`` for the gradients d_q, d_k of its results: (dq, dk, dq_weight, dk_weight); a weight that is None has none.
    q, k are the forward's inputs.  ``out``: a pair for dq, dk (may be d_q, d_k themselves)."""
    r = _rope(q, k, positions, freqs, q_weight, k_weight, norm, eps, interleaved, gain)
    assert d_q.shape == q.shape and (k is None or d_k.shape == k.shape), "d_q and d_k must have the shapes of q and k"
    r.ld_dq = _heads("d_q", d_q, q)[3]
    r.ld_dk = 0 if k is None else _heads("d_k", d_k, q)[3]
    dq, dk = _rope_results(q, k, r, out)
    hd = q.shape[2]
    dqw = None if q_weight is None else torch.empty(hd, device=q.device)
    dkw = None if k_weight is None else torch.empty(hd, device=q.device)
    L, n = _lib.lib(), 0
    ws = None
    if dqw is not None or dkw is not None:
        n = L.osud_op_qk_norm_rope_ws(hd)
        ws = torch.empty(n, device=q.device)
    _call(q.device, L.osud_op_qk_norm_rope_bwd, C.byref(r), d_q.data_ptr(), _ptr(d_k), q.data_ptr(), _ptr(k), dq.data_ptr(), _ptr(dk),
          _ptr(dqw), _ptr(dkw), _ptr(ws), n)
    return dq, dk, dqw, dkw


# ------------------------------------------------------------------ attention over packed documents
class Documents:
    """Where the documents of a packed batch lie: document d has ``lengths[d]`` query rows behind those of document d - 1, and ``kv_lengths[d]`` key
    rows (default: as many); ``prefix[d]`` keys at its start are visible to all of its queries.  Made once per batch; lengths may be 0."""

    def __init__(self, lengths, device="cuda", kv_lengths=None, prefix=None):
        lengths = [int(n) for n in lengths]
        kv = lengths if kv_lengths is None else [int(n) for n in kv_lengths]
        assert len(kv) == len(lengths), f"{len(lengths)} query lengths and {len(kv)} key lengths"
        assert all(n >= 0 for n in lengths) and all(n >= 0 for n in kv), "lengths must not be negative"
        self.count, self.rows, self.kv_rows = len(lengths), sum(lengths), sum(kv)
        assert max(self.rows, self.kv_rows) < 1 << 30, "too many rows"
        self.max_len, self.max_kv_len = max(lengths, default=0), max(kv, default=0)
        table = [0, *accumulate(lengths), 0, *accumulate(kv)]
        if prefix is not None:
            prefix = [int(n) for n in prefix]
            assert len(prefix) == len(kv) and all(0 <= n <= m for n, m in zip(prefix, kv)), "a prefix per document, not longer than its keys"
            table += prefix
        self._table = torch.tensor(table, dtype=torch.int32).to(device)  # (one copy: both offset lists and the prefixes)
        self.device = self._table.device
        self.q_begin, self.k_begin = self._table[:self.count + 1], self._table[self.count + 1:2 * self.count + 2]
        self.prefix = None if prefix is None else self._table[2 * self.count + 2:]


def _attention(q, k, v, docs, scale, cap, left, right, slopes):
    prec = _precision(q)
    rows, heads, hd, ld_q = _heads("q", q)
    krows, kv_heads, khd, ld_k = _heads("k", k, q)
    ld_v = _heads("v", v, q)[3]
    assert khd == hd and v.shape == k.shape, f"k and v must have the head_dim of q and one shape, got {tuple(k.shape)}, {tuple(v.shape)} and {tuple(q.shape)}"
    assert docs.device == q.device, f"the documents are on {docs.device}, the tensors on {q.device}"
    assert docs.rows <= rows and docs.kv_rows <= krows, f"the documents have {docs.rows} query and {docs.kv_rows} key rows, the tensors {rows} and {krows}"
    assert (left is None or left >= 0) and (right is None or right >= 0), "left and right must not be negative (None: no bound)"
    far = 1 << 30
    a = _lib.DocAttention(prec, heads, kv_heads, hd, docs.count, rows, krows, -1 if left is None else min(left, far), -1 if right is None else min(right, far),
                          docs.max_len, docs.max_kv_len, 0, 1.0 / math.sqrt(hd) if scale is None else scale, cap, ld_q, ld_k, ld_v)
    a.q_begin, a.k_begin = docs.q_begin.data_ptr(), docs.k_begin.data_ptr()
    if docs.prefix is not None:
        a.prefix = docs.prefix.data_ptr()
    if slopes is not None:
        a.slopes = _vector("slopes", slopes, heads, torch.float32, q.device)
    return a


def _attention_forward(q, k, v, docs, a, out):
    fresh = out is None
    if fresh:
        out = _new(q)
        a.ld_out = a.heads * a.head_dim
        a.clear_rest = docs.rows < q.shape[0]
    else:
        assert out.shape == q.shape, f"out must have the shape of q, got {tuple(out.shape)}"
        a.ld_out = _heads("out", out, q)[3]
        _written(out)
    lse = torch.empty(q.shape[1], q.shape[0], device=q.device)
    L = _lib.lib()
    n = L.osud_op_doc_attention_ws(C.byref(a), 0)
    ws = torch.empty(n, device=q.device) if n else None
    _call(q.device, L.osud_op_doc_attention, C.byref(a), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), _ptr(ws), n)
    if not fresh and docs.rows < q.shape[0]:
        lse[:, docs.rows:] = -math.inf
    return out, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, docs, scale, cap, left, right, slopes):
        out, lse = _attention_forward(q, k, v, docs, _attention(q, k, v, docs, scale, cap, left, right, slopes), None)
        ctx.save_for_backward(q, k, v, out, lse, slopes)
        ctx.docs, ctx.how = docs, dict(scale=scale, cap=cap, left=left, right=right)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, _):
        q, k, v, out, lse, slopes = ctx.saved_tensors
        if d_out is None:
            return (None,) * 9
        d_out = d_out.contiguous()
        if d_out.data_ptr() % 16:  # (a piece of a larger gradient: the caller cannot choose where it starts)
            d_out = d_out.clone()
        return *attention_bwd(d_out, q, k, v, out, lse, ctx.docs, slopes=slopes, **ctx.how), None, None, None, None, None, None


def attention(q, k, v, docs, *, scale=None, cap=0.0, left=None, right=None, slopes=None, return_lse=False, out=None):
    """Attention within every document of ``docs`` (a ``Documents``): softmax over the visible keys of the scores, times v.

    q (rows, heads, head_dim); k, v (kv rows, kv_heads, head_dim), query head h reads key head h // (heads // kv_heads); head_dim a multiple of 8 up
    to 128.  Query i of a document's nq stands at position nk - nq + i of its nk keys.  Scores: ``scale`` (> 0; 1 / sqrt(head_dim)) times q.k; with ``cap``
    > 0 then cap * tanh(s / cap); with ``slopes`` (heads,) float32 then minus slope * |distance|.  A key is visible within ``left`` positions before
    and ``right`` behind the query's own (None: no bound; right=0: causal), or inside the document's prefix.  A query that sees no key gets
    zeros.  Returns out (rows, heads, head_dim), zeros behind the last document (with ``out`` given, which must not overlap q, k or v, those rows stay as they are); with ``return_lse``
    also lse (heads, rows) float32, the logarithm of each row's sum of exponentials (-inf: no key), without a gradient.  slopes have no
    gradient; float16 has none at all.  What other documents and the rows behind the last one hold has no influence; inside a document k and v
    must be finite, also where a mask hides them (a hidden NaN may reach the document's other rows, as 0 * NaN)."""
    if _wants_grad(q, k, v, constants=(("slopes", slopes),)):
        assert out is None, "out= cannot be combined with gradients"
        assert q.dtype != torch.float16, "the fp16 tier has no backward pass"
        got = _Attention.apply(q, k, v, docs, scale, cap, left, right, slopes)
    else:
        got = _attention_forward(q, k, v, docs, _attention(q, k, v, docs, scale, cap, left, right, slopes), out)
    return got if return_lse else got[0]


def attention_bwd(d_out, q, k, v, out, lse, docs, *, scale=None, cap=0.0, left=None, right=None, slopes=None, grads=None):
    """Gradients (dq, dk, dv) of ``attention`` for the gradient d_out of its result; out and lse as it returned them.  Rows behind the last
    document get zeros; with ``grads`` (three tensors to write into, e.g. the parts of one packed gradient; none may overlap an input) they stay as they are."""
    a = _attention(q, k, v, docs, scale, cap, left, right, slopes)
    assert d_out.shape == q.shape and out.shape == q.shape, "d_out and out must have the shape of q"
    assert lse.shape == (q.shape[1], q.shape[0]) and lse.dtype == torch.float32 and lse.device == q.device and lse.is_contiguous(), \
        "lse must be the (heads, rows) float32 tensor that attention returned"
    a.ld_out, a.ld_d_out = _heads("out", out, q)[3], _heads("d_out", d_out, q)[3]
    fresh = grads is None
    if fresh:
        dq, dk, dv = (_new(t) for t in (q, k, v))
        a.ld_dq, a.ld_dk, a.ld_dv = a.heads * a.head_dim, a.kv_heads * a.head_dim, a.kv_heads * a.head_dim
        a.clear_rest = docs.rows < q.shape[0] or docs.kv_rows < k.shape[0]
    else:
        dq, dk, dv = grads
        assert dq.shape == q.shape and dk.shape == k.shape and dv.shape == v.shape, "grads must have the shapes of q, k and v"
        a.ld_dq, a.ld_dk, a.ld_dv = _heads("dq", dq, q)[3], _heads("dk", dk, q)[3], _heads("dv", dv, q)[3]
        _written(dq, dk, dv)
    L = _lib.lib()
    n = L.osud_op_doc_attention_ws(C.byref(a), 1)
    ws = torch.empty(max(n, 1), device=q.device)
    _call(q.device, L.osud_op_doc_attention_bwd, C.byref(a), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), d_out.data_ptr(),
          dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), n)
    return dq, dk, dv
