"""Plain 64-bit statements of the operators of `osu_diffusion_amd.ops`, with error bounds derived from the kernels' roundings.

Roundings counted (u = half a step of the element type, e = 2^-24):
* a result is rounded once: u |x|;
* the weights p and the score gradients ds are rounded to the element type before their products: u |p|, u |ds| (fp32 tier: none);
* scores are fp32 sums of exact products: relative error of p  rel = 2 (hd + 8) e max_d-sum(|q||k|) scale + (slope distance, cap: a few e of their
  size) + nk e (the sum of p), the factor 2 for the difference from the row's logarithm;
* a weight p or a score gradient ds below 2^-126, the smallest normal number of fp32 and bf16, may come out as zero (the exponential unit and the
  16-bit operands have no subnormals): 2^-126 each, so (|dp| + |delta| + 1) 2^-126 in ds.  (Seen: a key 4095 positions away at slope 0.02,
  p = e^(-86.4 + s), 2^-126 = e^-87.3; dk = 1.8e-37 lost, sums of scale |dp| |q| 2^-126 = 0.09 * 40 * 3 * 1.2e-38 over four heads = 5e-37.)
* delta = sum_d d_out out is taken from the rounded out: its error is sum_d |d_out| times the error bound of out."""
import math

import torch

E = 2.0 ** -24
TINY = 2.0 ** -126


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(x, dtype):
    """The largest error of one rounding of x: half a step relative to x, and below the smallest normal number, where steps no longer shrink, half
    the smallest subnormal one (fp16: 2^-25 = 3.0e-8; a value of 4.52e-5, under 2^-14 = 6.1e-5, moved by 2.6e-8 = 5.7e-4 of itself)."""
    f = torch.finfo(dtype)
    return (f.eps / 2 * x.abs()).clamp(min=f.tiny * f.eps / 2)


def attention_case(q, k, v, lengths, kv_lengths=None, prefix=None, scale=None, cap=0.0, left=None, right=None, slopes=None, d_out=None):
    """{name: (value, bound)} of out, lse (and dq, dk, dv with d_out): tensors of the inputs' layout, float64, on the CPU."""
    dtype = q.dtype
    u = half_step(dtype)
    up = 0.0 if dtype == torch.float32 else u  # rounding of p and ds
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    d_out = None if d_out is None else d_out.detach().double().cpu()
    slopes = None if slopes is None else slopes.double().cpu()
    h, g, hd = q.shape[1], k.shape[1], q.shape[2]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    kv_lengths = lengths if kv_lengths is None else kv_lengths
    prefix = [0] * len(lengths) if prefix is None else prefix
    z = lambda t: (torch.zeros_like(t), torch.zeros_like(t))  # noqa: E731
    out, dq, dk, dv = z(q), z(q), z(k), z(v)
    lse = (torch.full((h, q.shape[0]), -math.inf, dtype=torch.float64), torch.zeros(h, q.shape[0], dtype=torch.float64))
    a = b = 0
    for nq, nk, pre in zip(lengths, kv_lengths, prefix):
        pos, key = torch.arange(nk - nq, nk)[:, None], torch.arange(nk)[None]
        seen = torch.ones(nq, nk, dtype=torch.bool)
        if left is not None:
            seen &= key >= pos - left
        if right is not None:
            seen &= key <= pos + right
        seen |= key < pre
        for head in range(h):
            kv = head // (h // g)
            qs, ks, vs = q[a:a + nq, head], k[b:b + nk, kv], v[b:b + nk, kv]
            if nq == 0 or nk == 0:
                continue
            s = scale * qs @ ks.T
            err = scale * (hd + 8) * E * (qs.abs() @ ks.abs().T)
            t = None
            if cap:
                t = torch.tanh(s / cap)
                s = cap * t
                err = err + 4 * E * cap
            if slopes is not None:
                far = slopes[head] * (pos - key).abs()
                s = s - far
                err = err + 4 * E * far
            err = err + 4 * E * s.abs()
            s = torch.where(seen, s, -math.inf)
            norm = torch.logsumexp(s, 1, keepdim=True)
            p = torch.where(seen, torch.exp(s - torch.where(norm.isinf(), 0.0, norm)), 0.0)
            rel = 2 * torch.where(seen, err, 0.0).amax(1, keepdim=True) + (nk + 16) * E
            o = p @ vs
            mean = p @ vs.abs()
            o_err = (up + rel) * mean + rounded(o, dtype)
            if dtype == torch.float16:  # (small weights are subnormal: 2^-25 each, next to a largest one of at least 1)
                o_err = o_err + 2.0 ** -25 * seen.double() @ vs.abs()
            out[0][a:a + nq, head], out[1][a:a + nq, head] = o, o_err
            lse[0][head, a:a + nq] = norm[:, 0]
            lse[1][head, a:a + nq] = (rel + 4 * E * norm.abs())[:, 0].nan_to_num(0.0)
            if d_out is None:
                continue
            do = d_out[a:a + nq, head]
            dp = do @ vs.T
            delta = (p * dp).sum(1, keepdim=True)
            slope_of = 1.0 if t is None else 1 - t * t
            ds = p * (dp - delta) * slope_of
            d_err = (do.abs() * o_err).sum(1, keepdim=True) + (hd + 8) * E * (do.abs() * o.abs()).sum(1, keepdim=True)
            dp_err = (hd + 8) * E * (do.abs() @ vs.abs().T)
            ds_err = up * ds.abs() + p * slope_of * (d_err + dp_err) + (rel + 16 * E) * p * (dp.abs() + delta.abs())
            ds_err = ds_err + seen * TINY * (dp.abs() + delta.abs() + 1)
            if t is not None:
                ds_err = ds_err + 8 * E * p * (dp - delta).abs()
            acc = (max(nq, nk) + 8) * E  # fp32 accumulation of the last products
            dq[0][a:a + nq, head] = scale * ds @ ks
            dq[1][a:a + nq, head] = scale * (ds_err + acc * ds.abs()) @ ks.abs()
            dk[0][b:b + nk, kv] += scale * ds.T @ qs
            dk[1][b:b + nk, kv] += scale * (ds_err + acc * ds.abs()).T @ qs.abs()
            dv[0][b:b + nk, kv] += p.T @ do
            dv[1][b:b + nk, kv] += ((up + rel + acc) * p + seen * TINY).T @ do.abs()
        a, b = a + nq, b + nk
    got = {"out": out, "lse": lse}
    if d_out is not None:
        got.update({n: (x, e + rounded(x, dtype)) for n, (x, e) in (("dq", dq), ("dk", dk), ("dv", dv))})
    return got


def rope_case(x, w, positions, freqs, norm=True, eps=1e-6, interleaved=False, gain=1.0, grad=None):
    """{name: (value, bound)} of one of q, k: out, or with `grad` dx and dw.  Bounds: the result's rounding u, and about 24 + hd fp32 roundings of
    quantities no larger than the head's norm times the weight (a rotated pair, a normalised row)."""
    dtype = x.dtype
    x = x.detach().double().cpu()
    w = torch.ones(x.shape[2], dtype=torch.float64) if w is None else w.double().cpu()
    hd, n = x.shape[2], 0 if freqs is None else freqs.numel()
    first = torch.arange(0, 2 * n, 2) if interleaved else torch.arange(n)
    second = first + (1 if interleaved else n)
    x.requires_grad_(grad is not None)
    w.requires_grad_(grad is not None)
    r = (x.pow(2).mean(2, keepdim=True) + eps).rsqrt() if norm else 1.0
    z = x * r * w
    y = z.clone()
    if n:
        angle = (positions.double().cpu()[:, None] * freqs.cpu())[:, None]
        c, s = angle.cos() * gain, angle.sin() * gain
        y[..., first], y[..., second] = z[..., first] * c - z[..., second] * s, z[..., first] * s + z[..., second] * c
    slack = (24 + hd) * E * max(gain, 1.0)
    if grad is None:
        size = z.detach().abs()
        pair = size.clone()
        if n:
            pair[..., first] = pair[..., second] = size[..., first] + size[..., second]
        return {"out": (y, rounded(y, dtype) + slack * pair)}
    grad = grad.double().cpu()
    dx, dw = torch.autograd.grad(y, (x, w), grad)
    x, w, r = x.detach(), w.detach(), r.detach() if norm else 1.0
    back = grad.abs().clone()
    if n:
        back[..., first] = back[..., second] = (grad[..., first].abs() + grad[..., second].abs()) * max(gain, 1.0)
    size = r * (back * w.abs() + (x * r).abs() * (back * w.abs() * (x * r).abs()).mean(2, keepdim=True))
    rows = x.shape[0] * x.shape[1]
    return {"dx": (dx, rounded(dx, dtype) + 2 * slack * size), "dw": (dw, (slack + (rows + 64) * E) * (back * (x * r).abs()).sum((0, 1)))}


def check(got, want, what):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    same = (got == value) | (got.isnan() & value.isnan())
    bad = ~same & ~((got - value).abs() <= bound)
    if bool(bad.any()):
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at {at}: {float(got[at])} for {float(value[at])} +- {float(bound[at])}")
