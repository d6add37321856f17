"""Cases of the query / key norm with rotary positions (`osu_diffusion_amd.ops.qk_norm_rope`) and of attention over packed documents
(`osu_diffusion_amd.ops.attention`): inputs, the plain forms in elementary torch operations, the calls of the native kernels, and an
evaluation of the definitions in 64 bits.

A case is a dict of plain values.  `op` is "rope" or "attention"; `pass` is "forward", "backward" (rope: the gradients for a given
upstream gradient) or "train" (attention: forward and backward of one step)."""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ cases
def _rope(name, rows, heads, kv_heads, head_dim, rot, type_, pass_="forward", interleaved=False, positions="tokens", scaling=""):
    return {"name": name, "op": "rope", "pass": pass_, "rows": rows, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "rot": rot,
            "type": type_, "interleaved": interleaved, "positions": positions, "scaling": scaling}


def _attention(name, docs, length, spread, heads, kv_heads, head_dim, type_, pass_="forward", queries=0, left=-1, right=-1, prefix=0.0, cap=0.0,
               slopes=False, empties=0, tail=0, doc_seed=1):
    """`docs` documents of about `length` keys (times exp(+-spread)), `empties` more of none, `tail` rows behind the last one; `queries`: that
    many query rows per document at its end (0: one for every key); `prefix`: that share of a document is visible to all of it."""
    return {"name": name, "op": "attention", "pass": pass_, "docs": docs, "length": length, "spread": spread, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "type": type_, "queries": queries, "left": left, "right": right, "prefix": prefix,
            "cap": cap, "slopes": slopes, "empties": empties, "tail": tail, "doc_seed": doc_seed}


def listed():
    return [
        # one token of a guided pair, refined on its own: launch latency
        _rope("rope_one_token", 2, 12, 12, 64, 64, "f16"),
        # the training batch of the default model: 256 windows of 128 tokens
        _rope("rope_windows", 32768, 12, 12, 64, 64, "bf16"),
        # the wide model's 72-column heads, gradients, whole head rotated in neighbouring pairs
        _rope("rope_wide_backward", 32768, 16, 16, 72, 72, "bf16", "backward", interleaved=True),
        # parity arithmetic on an odd batch of one long beatmap: times in ms, half of the head rotated, shared key heads
        _rope("rope_ms_parity_backward", 5003, 6, 2, 64, 32, "f32", "backward", positions="ms", scaling="ramp"),
        # three short fragments in one call: launch latency
        _attention("attn_fragments", 3, 24, 1.0, 12, 12, 64, "f16", tail=5),
        # a training batch of ragged windows, packed without padding
        _attention("attn_windows_train", 256, 128, 0.6, 12, 12, 64, "bf16", "train", empties=2, tail=37),
        # whole beatmaps sampled with the window of the training length around every token (guided pairs of four variants)
        _attention("attn_band", 8, 4096, 0.0, 12, 12, 64, "f16", left=127, right=127),
        # long causal documents with capped scores and shared key heads
        _attention("attn_capped_causal", 2, 8191, 0.05, 12, 4, 128, "bf16", right=0, cap=30.0),
        # the newest token of each of 16 running sequences against all before it, with a distance penalty
        _attention("attn_newest_token", 16, 8000, 0.7, 16, 4, 128, "bf16", queries=1, right=0, slopes=True),
        # documents that start with a context seen by all of them, wide model's heads, capped scores
        _attention("attn_prefix_train", 6, 1900, 0.3, 16, 16, 72, "bf16", "train", right=0, prefix=0.3, cap=20.0),
        # parity arithmetic: ragged documents, band and distance penalty
        _attention("attn_parity_train", 7, 401, 0.5, 6, 3, 64, "f32", "train", left=200, right=50, slopes=True, tail=3),
        # one long causal document with a distance penalty and shared key heads: the largest
        _attention("attn_long_train", 1, 8192, 0.0, 8, 2, 128, "bf16", "train", right=0, slopes=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _price(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / (1e14 if case["type"] == "f32" else 1e15))


def draw(rng):
    most = max(_price(c) for c in listed() if c["type"] != "f32")
    while True:
        case = _draw(rng)
        del case["name"]
        if 0 < _price(case) <= (most if case["type"] != "f32" else most / 4):
            return case


def _draw(rng):
    head_dim = rng.choice([64, 64, 72, 128, 128, 8 * rng.randint(2, 16)])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
    if rng.random() < 0.35:
        pass_ = rng.choice(["forward", "backward"])
        rot = rng.choice([head_dim, head_dim, 2 * rng.randint(1, head_dim // 2)])
        return _rope("", _log(rng, 1, 40000), heads, kv_heads, head_dim, rot, rng.choice(["bf16", "bf16", "f32"] + ["f16"] * (pass_ == "forward")),
                     pass_, rng.random() < 0.5, rng.choice(["tokens", "ms", "far"]), rng.choice(["", "linear", "base", "ramp"]))
    pass_ = rng.choice(["forward", "train"])
    length = _log(rng, 1, 9000)
    mask = rng.choice(["none", "causal", "band", "prefix"])
    left, right, prefix = -1, -1, 0.0
    if mask == "band":
        left, right = _log(rng, 1, 600) - 1, rng.choice([0, _log(rng, 1, 600)])
    elif mask != "none":
        right = 0
        prefix = rng.uniform(0.02, 0.6) if mask == "prefix" else 0.0
    few = pass_ == "forward" and rng.random() < 0.3
    return _attention("", _log(rng, 1, 300 if length < 400 else 24), length, rng.choice([0.0, 0.3, 0.8]), heads, kv_heads, head_dim,
                      rng.choice(["bf16", "bf16", "bf16", "f32"] + ["f16"] * (pass_ == "forward")), pass_, rng.choice([1, 1, 3, 17]) if few else 0,
                      left, right, prefix, rng.choice([0.0, 0.0, 15.0, 50.0]), rng.random() < 0.4, rng.choice([0, 0, 1, 3]),
                      rng.choice([0, 0, 1, 50]), rng.randint(1, 10 ** 6))


def _documents(case):
    """(query rows, keys, prefix) of every document; the same for every seed of the inputs."""
    rng = random.Random(case["doc_seed"])
    lk = [max(1, int(round(case["length"] * math.exp(rng.uniform(-case["spread"], case["spread"]))))) for _ in range(case["docs"])]
    for _ in range(case["empties"]):
        lk.insert(rng.randint(0, len(lk)), 0)
    lq = [min(case["queries"], n) if case["queries"] else n for n in lk]
    return lq, lk, [int(case["prefix"] * n) for n in lk]


def _pairs(case):
    """Visible (query, key) pairs of all documents, for one head."""
    total = 0
    for lq, lk, pre in zip(*_documents(case)):
        if not lq:
            continue
        pos = torch.arange(lk - lq, lk)
        lo = (pos - case["left"]).clamp(min=0) if case["left"] >= 0 else torch.zeros_like(pos)
        hi = (pos + case["right"] + 1).clamp(max=lk) if case["right"] >= 0 else torch.full_like(pos, lk)
        total += int((torch.maximum(hi, hi.new_tensor(pre)) - lo.clamp(min=pre) + pre).where(hi > pre, hi.new_tensor(pre)).sum()) if pre \
            else int((hi - lo).sum())
    return total


def work(case):
    size = 4 if case["type"] == "f32" else 2
    h, g, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rope":
        n = case["rows"] * (h + g) * d
        if case["pass"] == "forward":
            return {"bytes": 2 * n * size + 4 * case["rows"], "flops": 10 * n}
        return {"bytes": 3 * n * size + 4 * case["rows"], "flops": 20 * n}
    lq, lk, _ = _documents(case)
    q, k = (sum(lq) + case["tail"]) * h * d * size, sum(lk) * g * d * size
    pairs = _pairs(case) * h * d
    if case["pass"] == "forward":
        return {"bytes": 2 * q + 2 * k + 4 * h * sum(lq), "flops": 4 * pairs}
    # the step's forward and backward: q, k, v, d_out in; out, lse, dq, dk, dv out (what lies between them is read again)
    return {"bytes": 4 * q + 4 * k + 4 * h * sum(lq), "flops": 14 * pairs}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 7919 + 13)
    type_ = TYPES[case["type"]]
    h, g, d = case["heads"], case["kv_heads"], case["head_dim"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(type_)

    if case["op"] == "rope":
        n, rot = case["rows"], case["rot"]
        packed = normal(n, (h + 2 * g) * d)  # the packed projection Q | K | V
        state = {"case": case, "q": packed[:, :h * d].view(n, h, d), "k": packed[:, h * d:(h + g) * d].view(n, g, d)}
        if case["positions"] == "tokens":
            state["positions"] = (torch.arange(n, device=DEV) % 128).to(torch.int32)
        elif case["positions"] == "ms":  # times of hit objects: ten minutes at most
            state["positions"] = (torch.rand(n, generator=gen, device=DEV) * 6e5).sort().values
        else:
            state["positions"] = torch.randint(0, 1 << 20, (n,), generator=gen, device=DEV, dtype=torch.int32)
        state["freqs"], state["gain"] = _frequencies(rot, case["scaling"])
        state["q_weight"] = 1 + 0.2 * torch.randn(d, generator=gen, device=DEV)
        state["k_weight"] = 1 + 0.2 * torch.randn(d, generator=gen, device=DEV)
        if case["pass"] == "backward":
            state["d_q"], state["d_k"] = normal(n, h, d), normal(n, g, d)
        return state
    lq, lk, prefix = _documents(case)
    nq, nk = sum(lq) + case["tail"], sum(lk) + (0 if case["queries"] else case["tail"])
    if case["queries"]:
        kv = normal(nk, 2 * g * d)
        state = {"q": normal(nq, h, d, scale=1.5), "k": kv[:, :g * d].view(nk, g, d), "v": kv[:, g * d:].view(nk, g, d)}
    else:
        packed = normal(nq, (h + 2 * g) * d)
        packed[:, :h * d] *= 1.5
        q, k, v = packed.split([h * d, g * d, g * d], 1)
        state = {"q": q.view(nq, h, d), "k": k.view(nk, g, d), "v": v.view(nk, g, d)}
    state.update(case=case, lq=lq, lk=lk, prefix=prefix, slopes=None)
    if case["slopes"]:
        state["slopes"] = 2.0 ** (-8.0 * torch.arange(1, h + 1, device=DEV, dtype=torch.float32) / h)
    if case["pass"] == "train":
        state["d_out"] = normal(nq, h, d)
    if own:
        from osu_diffusion_amd import ops

        state["documents"] = ops.Documents(lq, device=DEV, kv_lengths=lk if case["queries"] else None, prefix=prefix if case["prefix"] else None)
    return state


def _frequencies(rot, scaling, base=10000.0, factor=8.0, original=256.0):
    """Rotary frequencies in 64 bits and the gain of the rotated part, for contexts `factor` times the `original` length."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    if scaling == "base":
        base = base * factor ** (rot / (rot - 2)) if rot > 2 else base
    f = base ** (-2.0 * i / rot)
    gain = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "ramp":  # turns over the original length: below 1 interpolated, above 32 kept, a ramp between
        keep = ((original * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1 - keep)
        gain = 0.1 * math.log(factor) + 1.0
    return f.to(DEV), gain


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if not own:
        return _plain_rope(state) if case["op"] == "rope" else _plain_attention(state)
    from osu_diffusion_amd import ops

    if case["op"] == "rope":
        kw = dict(q_weight=state["q_weight"], k_weight=state["k_weight"], interleaved=case["interleaved"], gain=state["gain"])
        if case["pass"] == "forward":
            return ops.qk_norm_rope(state["q"], state["k"], state["positions"], state["freqs"], **kw)
        return ops.qk_norm_rope_bwd(state["d_q"], state["d_k"], state["q"], state["k"], state["positions"], state["freqs"], **kw)
    kw = dict(cap=case["cap"], left=None if case["left"] < 0 else case["left"], right=None if case["right"] < 0 else case["right"],
              slopes=state["slopes"])
    q, k, v, docs = state["q"], state["k"], state["v"], state["documents"]
    out, lse = ops.attention(q, k, v, docs, return_lse=True, **kw)
    if case["pass"] == "forward":
        return out, lse
    return (out, lse) + tuple(ops.attention_bwd(state["d_out"], q, k, v, out, lse, docs, **kw))


EPS = 1e-6


def _plain_rope(state):
    case, rot = state["case"], state["case"]["rot"]
    angle = state["positions"].double()[:, None] * state["freqs"]
    cos, sin = (t(angle).float()[:, None] * state["gain"] for t in (torch.cos, torch.sin))

    def halves(x):
        if case["interleaved"]:
            return x[..., 0:rot:2], x[..., 1:rot:2]
        return x[..., :rot // 2], x[..., rot // 2:rot]

    def joined(a, b, rest):
        both = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
        return torch.cat((both, rest), -1)

    def forward(x, w):
        x = x.float()
        z = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        a, b = halves(z)
        return joined(a * cos - b * sin, a * sin + b * cos, z[..., rot:])

    def backward(g, x, w):
        g, x = g.float(), x.float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        a, b = halves(g)
        dz = joined(a * cos + b * sin, b * cos - a * sin, g[..., rot:])
        xr = x * r
        u = dz * w
        return r * (u - xr * (u * xr).mean(-1, keepdim=True)), (dz * xr).sum((0, 1))

    type_ = state["q"].dtype
    if case["pass"] == "forward":
        return forward(state["q"], state["q_weight"]).to(type_), forward(state["k"], state["k_weight"]).to(type_)
    dq, dwq = backward(state["d_q"], state["q"], state["q_weight"])
    dk, dwk = backward(state["d_k"], state["k"], state["k_weight"])
    return dq.to(type_), dk.to(type_), dwq, dwk


def _hidden(case, lq, lk, prefix):
    """(lq, lk) truth values: pairs that the masks take out; and the distance of every pair."""
    pos = torch.arange(lk - lq, lk, device=DEV)[:, None]
    key = torch.arange(lk, device=DEV)[None]
    out = torch.zeros(lq, lk, dtype=torch.bool, device=DEV)
    if case["left"] >= 0:
        out |= key < pos - case["left"]
    if case["right"] >= 0:
        out |= key > pos + case["right"]
    return out & (key >= prefix), (pos - key).abs()


def _plain_attention(state):
    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    nq, h, d = q.shape
    g = k.shape[1]
    m, cap, scale = h // g, case["cap"], 1.0 / math.sqrt(d)
    train = case["pass"] == "train"
    out = torch.zeros(nq, h, d, device=DEV, dtype=q.dtype)
    lse = torch.full((h, nq), -math.inf, device=DEV)
    if train:
        dq, dk, dv = torch.zeros_like(out), *(torch.zeros(*k.shape, device=DEV, dtype=q.dtype) for _ in "kv")
    a = b = 0
    for lq, lk, pre in zip(state["lq"], state["lk"], state["prefix"]):
        qs, ks = slice(a, a + lq), slice(b, b + lk)
        a, b = a + lq, b + lk
        if not lq:
            continue

        def rows(x):  # the query heads that share a key head stand below each other: (g, m * lq, d)
            return x[qs].float().view(lq, g, m, d).permute(1, 2, 0, 3).reshape(g, m * lq, d)

        def back(x):
            return x.view(g, m, lq, d).permute(2, 0, 1, 3).reshape(lq, h, d).to(q.dtype)

        qd, kd, vd = rows(q), k[ks].float().transpose(0, 1).contiguous(), v[ks].float().transpose(0, 1).contiguous()
        s = torch.matmul(qd, kd.transpose(1, 2).contiguous()).mul_(scale)
        if cap:
            t = torch.tanh_(s.div_(cap))
            s = t * cap
        hidden, distance = _hidden(case, lq, lk, pre)
        s = s.view(g, m, lq, lk)
        if state["slopes"] is not None:
            s = s - state["slopes"].view(g, m, 1, 1) * distance
        s = s.masked_fill(hidden, -math.inf).view(g, m * lq, lk)
        top = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
        p = torch.exp_(s.sub_(top))
        total = p.sum(-1, keepdim=True)
        lse[:, qs] = (top + torch.log(total)).view(h, lq).masked_fill(total.view(h, lq) == 0, -math.inf)
        p = p.div_(total.clamp(min=1e-30))
        out[qs] = back(torch.matmul(p, vd))
        if train:
            do = rows(state["d_out"])
            dv[ks] = torch.matmul(p.transpose(1, 2).contiguous(), do).transpose(0, 1).to(q.dtype)
            dp = torch.matmul(do, vd.transpose(1, 2).contiguous())
            ds = p.mul_(dp.sub_((p * dp).sum(-1, keepdim=True)))
            if cap:
                ds = ds.mul_(1 - t.square_())
            ds = ds.mul_(scale)
            dq[qs] = back(torch.matmul(ds, kd))
            dk[ks] = torch.matmul(ds.transpose(1, 2).contiguous(), qd).transpose(0, 1).to(q.dtype)
    return (out, lse, dq, dk, dv) if train else (out, lse)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return _exact_rope(state) if case["op"] == "rope" else _exact_attention(state)


def _exact_rope(state):
    case = state["case"]
    rot = case["rot"]
    first = torch.arange(0, rot, 2) if case["interleaved"] else torch.arange(rot // 2)
    second = first + (1 if case["interleaved"] else rot // 2)
    turn = torch.polar(torch.full_like(state["freqs"], state["gain"]), torch.zeros_like(state["freqs"])) \
        * torch.exp(1j * (state["positions"].double()[:, None] * state["freqs"]))

    def of(x, w):
        z = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w
        y = z.clone()
        pair = torch.complex(z[..., first], z[..., second]) * turn[:, None]
        y[..., first], y[..., second] = pair.real, pair.imag
        return y

    outs, grads = [], []
    for name in "qk":
        x = state[name].double().requires_grad_(case["pass"] == "backward")
        w = state[name + "_weight"].double().requires_grad_(case["pass"] == "backward")
        y = of(x, w)
        outs.append(y.detach())
        if case["pass"] == "backward":
            grads.append(torch.autograd.grad(y, (x, w), state["d_" + name].double()))
    return tuple(outs) if not grads else (grads[0][0], grads[1][0], grads[0][1], grads[1][1])


def _exact_attention(state):
    case = state["case"]
    train = case["pass"] == "train"
    h, g, d = case["heads"], case["kv_heads"], case["head_dim"]
    q, k, v = (state[n].double() for n in "qkv")
    out = torch.zeros_like(q)
    lse = torch.full((h, q.shape[0]), -math.inf, device=DEV, dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    a = b = 0
    for lq, lk, pre in zip(state["lq"], state["lk"], state["prefix"]):
        if not lq:
            b += lk
            continue
        hidden, distance = _hidden(case, lq, lk, pre)
        group = h if lq * lk <= 1 << 20 else 1  # heads at a time
        for lo in range(0, h, group):
            heads = torch.arange(lo, min(lo + group, h), device=DEV)
            qh = q[a:a + lq, heads].transpose(0, 1).contiguous().requires_grad_(train)
            kh = k[b:b + lk, heads // (h // g)].transpose(0, 1).contiguous().requires_grad_(train)
            vh = v[b:b + lk, heads // (h // g)].transpose(0, 1).contiguous().requires_grad_(train)
            s = (qh @ kh.mT) / math.sqrt(d)
            if case["cap"]:
                s = torch.tanh(s / case["cap"]) * case["cap"]
            if state["slopes"] is not None:
                s = s - state["slopes"].double()[heads, None, None] * distance
            s = torch.where(hidden, -math.inf, s)
            norm = torch.logsumexp(s, -1)
            weights = torch.where(hidden, 0.0, torch.exp(s - torch.where(norm.isinf(), 0.0, norm)[..., None]))
            o = weights @ vh
            out[a:a + lq, heads] = o.detach().transpose(0, 1)
            lse[heads, a:a + lq] = norm.detach()
            if train:
                gq, gk, gv = torch.autograd.grad(o, (qh, kh, vh), state["d_out"][a:a + lq, heads].double().transpose(0, 1))
                dq[a:a + lq, heads] = gq.transpose(0, 1)
                dk[b:b + lk].index_add_(1, heads // (h // g), gk.transpose(0, 1))
                dv[b:b + lk].index_add_(1, heads // (h // g), gv.transpose(0, 1))
        a, b = a + lq, b + lk
    return (out, lse, dq, dk, dv) if train else (out, lse)
