"""Performance cases of the operators that carry a batch of packed documents from token ids into the decoder.

* ``attention``  ``ops.packed_attention``: causal grouped-query attention over documents that lie one behind the other in
                 one buffer of rows; a row sees its own document only (and the last ``window`` keys of it).  Forward, or
                 forward and backward
* ``embedding``  ``ops.embedding``: rows of the table looked up and scaled, and the table's whole gradient (forward and
                 backward)
* ``dropout``    ``ops.dropout``: a mask that is a function of a seed, an offset and the element's index and is never
                 stored, optionally with the residual added; forward and backward

``run`` computes a case with elementary tensor operations or, where ``own`` is set, through the framework's entry points.
Head layouts, hidden sizes and vocabularies are those of ``system_lab_b200/models/presets.py``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DTYPES = {"bf16": BF16, "fp32": F32}
DEVICE = "cuda"


def listed():
    return [
        # a few short documents through the debugging model's heads: one launch's latency
        dict(name="attention-score-short", kind="attention", heads=4, groups=4, dim=64, rows=300, tail=0, mean=60, docs=1,
             window=0, train=False),
        # evaluation on ragged documents of an odd total length, rows behind the last one unused
        dict(name="attention-score-documents", kind="attention", heads=32, groups=4, dim=128, rows=8191, tail=116,
             mean=900, docs=2, window=0, train=False),
        # a pretraining micro-batch (2 x 4096 rows) of packed documents
        dict(name="attention-train-documents", kind="attention", heads=32, groups=4, dim=128, rows=8192, tail=0, mean=700,
             docs=3, window=0, train=True),
        # fine-tuning on one document as long as the sequence
        dict(name="attention-train-whole", kind="attention", heads=64, groups=8, dim=128, rows=8192, tail=0, mean=0,
             docs=4, window=0, train=True),
        # a layer with a sliding window, narrow heads, long documents
        dict(name="attention-train-window", kind="attention", heads=64, groups=8, dim=64, rows=16384, tail=0, mean=3000,
             docs=5, window=128, train=True),
        # the debugging model's table, every type in 32 bits
        dict(name="embedding-small", kind="embedding", tokens=512, vocab=1024, hidden=256, scaled=False, dtype="fp32"),
        # a pretraining micro-batch: the gradient has far more rows than the batch has tokens
        dict(name="embedding-pretrain", kind="embedding", tokens=8192, vocab=151936, hidden=2048, scaled=True, dtype="bf16"),
        # many tokens on a smaller table: frequent tokens come thousands of times
        dict(name="embedding-frequent", kind="embedding", tokens=32749, vocab=32000, hidden=2880, scaled=True, dtype="bf16"),
        # adapters on a short prompt of an odd length
        dict(name="dropout-adapter-short", kind="dropout", rows=77, width=2880, p=0.05, residual=False, dtype="bf16"),
        # the adapters' input in fine-tuning
        dict(name="dropout-adapter", kind="dropout", rows=8192, width=8192, p=0.1, residual=False, dtype="bf16"),
        # a block's output on its way into the residual stream
        dict(name="dropout-residual", kind="dropout", rows=16384, width=2048, p=0.1, residual=True, dtype="bf16"),
        # the same in 32 bits on rows whose width is no multiple of a vector
        dict(name="dropout-residual-odd", kind="dropout", rows=4095, width=2879, p=0.25, residual=True, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "embedding", "dropout"])
    if kind == "attention":
        heads, groups, dim = rng.choice([(4, 4, 64), (32, 4, 128), (64, 8, 128), (64, 8, 64), (8, 8, 128), (6, 2, 96), (5, 1, 72)])
        window = rng.choice([0, 0, 128, rng.randint(1, 700)])
        rows = _log_int(rng, 1, 8192 if not window and heads > 32 else 12000)
        mean = rng.choice([0, _log_int(rng, 1, 4000)])
        if mean and mean < rows // 200:                # a few hundred documents at most
            mean = rows // 200
        return dict(kind=kind, heads=heads, groups=groups, dim=dim, rows=rows, tail=rng.choice([0, 0, rng.randint(0, rows // 4)]),
                    mean=mean, docs=rng.randint(0, 1 << 30), window=window, train=rng.random() < 0.6)
    if kind == "embedding":
        vocab, hidden = rng.choice([(1024, 256), (151936, 2048), (129280, 1024), (32000, 8192), (201088, 2880),
                                    (rng.randint(2, 60000), 8 * rng.randint(1, 360)), (rng.randint(2, 9000), rng.randint(1, 700))])
        tokens = _log_int(rng, 1, min(60000, 30000 * 4096 // max(hidden, 1)))
        return dict(kind=kind, tokens=tokens, vocab=vocab, hidden=hidden, scaled=rng.random() < 0.5,
                    dtype=rng.choice(["bf16", "bf16", "fp32"]))
    width = rng.choice([256, 2048, 2880, 8192, rng.randint(1, 9000)])
    return dict(kind=kind, rows=_log_int(rng, 1, min(60000, 64 * 1024 * 1024 // width)), width=width,
                p=rng.choice([0.05, 0.1, 0.5, round(rng.random() * 0.95, 3)]), residual=rng.random() < 0.5,
                dtype=rng.choice(["bf16", "bf16", "fp32"]))


def lengths(case):
    """The documents' lengths: spread widely around their mean, empty and one-row ones among them; ``mean`` 0: one document."""
    left = case["rows"] - case["tail"]
    if not case["mean"]:
        return [left]
    rng = random.Random(case["docs"])
    out = []
    while left > 0:
        n = rng.choice([0, 1]) if rng.random() < 0.05 else int(rng.lognormvariate(math.log(case["mean"]), 0.9)) + 1
        out.append(min(n, left))
        left -= out[-1]
    return out


def _spans(case):
    at, out = 0, []
    for n in lengths(case):
        out.append((at, at + n))
        at += n
    return out


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g = _generator(seed)

    def normal(*shape, dtype=BF16, std=1.0):
        return torch.empty(*shape, dtype=F32, device=DEVICE).normal_(0.0, std, generator=g).to(dtype)

    if case["kind"] == "attention":
        hq, hkv, d, rows = case["heads"], case["groups"], case["dim"], case["rows"]
        # q, k and v are columns of one packed projection, as the attention block makes them
        qkv = normal(rows, (hq + 2 * hkv) * d)
        q, k, v = (t.unflatten(-1, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], dim=-1))
        cu = [0]
        for n in lengths(case):
            cu.append(cu[-1] + n)
        state = dict(case=case, q=q, k=k, v=v, dout=normal(rows, hq, d) if case["train"] else None, spans=_spans(case),
                     cu=torch.tensor(cu, dtype=torch.int32, device=DEVICE))
        if own:
            from system_lab_b200 import ops
            state["documents"] = ops.pack_documents(state["cu"], rows)          # one plan serves every layer of a step
            if case["train"]:
                state["leaves"] = tuple(t.detach().requires_grad_(True) for t in (q, k, v))
        return state
    if case["kind"] == "embedding":
        dt, v = DTYPES[case["dtype"]], case["vocab"]
        # ids spread evenly over their logarithm: the frequent ones come often, as in text
        u = torch.rand(case["tokens"], dtype=F64, device=DEVICE, generator=g)
        tokens = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
        tokens = (tokens * 7919) % v if math.gcd(7919, v) == 1 else tokens
        weight = normal(v, case["hidden"], dtype=dt, std=0.02)
        return dict(case=case, tokens=tokens, weight=weight, dout=normal(case["tokens"], case["hidden"], dtype=dt),
                    scale=math.sqrt(case["hidden"]) if case["scaled"] else 1.0,
                    leaf=weight.detach().requires_grad_(True) if own else None)
    dt = DTYPES[case["dtype"]]
    x = normal(case["rows"], case["width"], dtype=dt)
    res = normal(case["rows"], case["width"], dtype=dt) if case["residual"] else None
    return dict(case=case, x=x, res=res, dout=normal(case["rows"], case["width"], dtype=dt), seed=1234567890123 + seed, offset=(seed % 97) << 33,
                leaf=x.detach().requires_grad_(True) if own else None)


def run(state):
    return {"attention": _attention, "embedding": _embedding, "dropout": _dropout}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ attention
def _attention(state):
    case = state["case"]
    if own:
        from system_lab_b200 import ops
        if not case["train"]:
            with torch.no_grad():
                return ops.packed_attention(state["q"], state["k"], state["v"], state["documents"], window=case["window"])
        q, k, v = state["leaves"]
        out = ops.packed_attention(q, k, v, state["documents"], window=case["window"])
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), state["dout"])
    q, k, v, dout, window = state["q"], state["k"], state["v"], state["dout"], case["window"]
    rows, hq, d = q.shape
    hkv = k.shape[1]
    g = hq // hkv
    scale = 1.0 / math.sqrt(d)
    out = torch.zeros(rows, hq, d, dtype=q.dtype, device=q.device)
    if case["train"]:
        dq = torch.zeros_like(out)
        dk = torch.zeros(hkv, rows, d, dtype=F32, device=q.device)
        dv = torch.zeros_like(dk)
    for lo, hi in state["spans"]:
        for a in range(lo, hi, 1024):                                   # query rows of one document
            b = min(a + 1024, hi)
            f = max(lo, a - window + 1) if window else lo
            qf = q[a:b].float().reshape(b - a, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * (b - a), d)
            kf = k[f:b].float().permute(1, 0, 2)
            vf = v[f:b].float().permute(1, 0, 2)
            i = torch.arange(a, b, device=q.device)[:, None]
            j = torch.arange(f, b, device=q.device)[None, :]
            hidden = j > i
            if window:
                hidden = hidden | (j <= i - window)
            s = (qf @ kf.transpose(1, 2)).mul_(scale)
            s = s.view(hkv, g, b - a, b - f).masked_fill_(hidden, -math.inf).view(hkv, g * (b - a), b - f)
            p = (s - s.amax(-1, keepdim=True)).exp_()
            p = p / p.sum(-1, keepdim=True)
            o = p @ vf
            out[a:b] = o.view(hkv, g, b - a, d).permute(2, 0, 1, 3).reshape(b - a, hq, d).to(q.dtype)
            if not case["train"]:
                continue
            do = dout[a:b].float().reshape(b - a, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * (b - a), d)
            dv[:, f:b] += p.transpose(1, 2) @ do
            ds = (do @ vf.transpose(1, 2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            dk[:, f:b] += ds.transpose(1, 2) @ qf
            dq[a:b] = (ds @ kf).view(hkv, g, b - a, d).permute(2, 0, 1, 3).reshape(b - a, hq, d).to(q.dtype)
    if not case["train"]:
        return out
    return out, dq, dk.permute(1, 0, 2).to(q.dtype).contiguous(), dv.permute(1, 0, 2).to(q.dtype).contiguous()


# ------------------------------------------------------------------ embedding
def _embedding(state):
    tokens, weight, dout, scale = state["tokens"], state["weight"], state["dout"], state["scale"]
    if own:
        from system_lab_b200 import ops
        out = ops.embedding(tokens, state["leaf"], scale=scale)
        (dw,) = torch.autograd.grad(out, state["leaf"], dout)
        return out.detach(), dw
    out = (weight[tokens].float() * scale).to(weight.dtype)
    dw = torch.zeros(weight.shape, dtype=F32, device=weight.device)
    dw.index_add_(0, tokens, dout.float())
    return out, dw.mul_(scale).to(weight.dtype)


# ------------------------------------------------------------------ dropout
_M0, _M1, _W0, _W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85


def _mul32(a: int, b):
    """High and low 32 bits of the product of a 32-bit constant and 32-bit numbers held in 64-bit integers."""
    lo = a * (b & 0xFFFF)
    hi = a * (b >> 16)
    mid = hi + (lo >> 16)
    return (mid >> 16) & 0xFFFFFFFF, ((mid & 0xFFFF) << 16) | (lo & 0xFFFF)


def _philox(n, seed, offset, device):
    """16 random bits per element: element e takes bits 16 (e % 2) .. of word (e % 8) / 2 of the block with counter
    (e / 8, offset) and key ``seed`` of Philox-4x32 with ten rounds (Salmon et al., 2011)."""
    c0 = torch.arange((n + 7) // 8, dtype=torch.int64, device=device)
    c1 = c0 >> 32
    c0 = c0 & 0xFFFFFFFF
    c2 = torch.full_like(c0, offset & 0xFFFFFFFF)
    c3 = torch.full_like(c0, (offset >> 32) & 0xFFFFFFFF)
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        h0, l0 = _mul32(_M0, c0)
        h1, l1 = _mul32(_M1, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + _W0) & 0xFFFFFFFF, (k1 + _W1) & 0xFFFFFFFF
    w = torch.stack([c0, c1, c2, c3], dim=-1)
    return torch.stack([w & 0xFFFF, w >> 16], dim=-1).reshape(-1)[:n]


def _dropout(state):
    case, x, res, dout = state["case"], state["x"], state["res"], state["dout"]
    if own:
        from system_lab_b200 import ops
        y = ops.dropout(state["leaf"], case["p"], seed=state["seed"], offset=state["offset"], residual=res)
        (dx,) = torch.autograd.grad(y, state["leaf"], dout)
        return y.detach(), dx
    t = math.floor(case["p"] * 65536 + 0.5)
    keep = (_philox(x.numel(), state["seed"], state["offset"], x.device) >= t).view(x.shape)
    scale = 65536.0 / (65536 - t)
    y = torch.where(keep, x.float() * scale, 0.0)
    if res is not None:
        y = y + res.float()
    return y.to(x.dtype), torch.where(keep, dout.float() * scale, 0.0).to(x.dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def _pairs(case):
    n = 0
    for lo, hi in _spans(case):
        length = hi - lo
        w = min(case["window"] or length, length)
        n += w * (w + 1) // 2 + (length - w) * w
    return n


def work(case):
    if case["kind"] == "attention":
        hq, hkv, d, rows = case["heads"], case["groups"], case["dim"], case["rows"]
        qo, kv = rows * hq * d * 2, rows * hkv * d * 2
        flops = 4.0 * d * hq * _pairs(case)                             # Q K^T and P V
        nbytes = 2 * qo + 2 * kv
        if case["train"]:                                               # those, and P^T dO, dO V^T, dS^T Q, dS K (S kept or made again)
            flops += 10.0 * d * hq * _pairs(case)
            nbytes += 2 * qo + 2 * kv
        return {"bytes": float(nbytes), "flops": flops}
    if case["kind"] == "embedding":
        size = 2 if case["dtype"] == "bf16" else 4
        t, v, h = case["tokens"], case["vocab"], case["hidden"]
        return {"bytes": float(8 * t + size * h * (min(t, v) + 2 * t + v)), "flops": 2.0 * t * h}
    size = 2 if case["dtype"] == "bf16" else 4
    n = case["rows"] * case["width"]
    return {"bytes": float(size * n * (5 if case["residual"] else 4)), "flops": 4.0 * n}


# ------------------------------------------------------------------ in 64 bits, from the definitions
def _exact_attention(case, state):
    """Every document by itself: softmax and products in 64 bits, gradients by differentiation of the forward pass."""
    q, k, v = state["q"], state["k"], state["v"]
    hkv, d = case["groups"], case["dim"]
    g = case["heads"] // hkv
    out = torch.zeros(q.shape, dtype=F64, device=q.device)
    grads = [torch.zeros(t.shape, dtype=F64, device=q.device) for t in (q, k, v)]
    for lo, hi in _spans(case):
        if hi == lo:
            continue
        for h in range(hkv):
            k64 = k[lo:hi, h].double().requires_grad_(case["train"])
            v64 = v[lo:hi, h].double().requires_grad_(case["train"])
            for a in range(lo, hi, 2048):
                b = min(a + 2048, hi)
                q64 = q[a:b, h * g:(h + 1) * g].double().requires_grad_(case["train"])
                f = max(0, a - lo - case["window"]) if case["window"] else 0
                away = torch.arange(a - lo, b - lo, device=q.device)[:, None] - torch.arange(f, b - lo, device=q.device)[None, :]
                seen = away >= 0
                if case["window"]:
                    seen &= away < case["window"]
                with torch.set_grad_enabled(case["train"]):
                    score = torch.einsum("igd,jd->gij", q64, k64[f:b - lo]) / math.sqrt(d)
                    prob = torch.softmax(torch.where(seen, score, -math.inf), dim=-1)
                    o = torch.einsum("gij,jd->igd", prob, v64[f:b - lo])
                out[a:b, h * g:(h + 1) * g] = o.detach()
                if case["train"]:
                    gq, gk, gv = torch.autograd.grad(o, (q64, k64, v64), state["dout"][a:b, h * g:(h + 1) * g].double())
                    grads[0][a:b, h * g:(h + 1) * g] = gq
                    grads[1][lo:hi, h] += gk
                    grads[2][lo:hi, h] += gv
                del score, prob, o
    return (out, *grads) if case["train"] else out


def _exact_embedding(state):
    tokens, dout, scale = state["tokens"], state["dout"], state["scale"]
    out = torch.nn.functional.embedding(tokens, state["weight"]).double() * scale
    ids, where = torch.unique(tokens, return_inverse=True)
    sums = torch.zeros(ids.numel(), dout.shape[1], dtype=F64, device=dout.device)
    sums.scatter_add_(0, where[:, None].expand(-1, dout.shape[1]), dout.double())
    dw = torch.zeros(state["weight"].shape, dtype=F64, device=dout.device)
    dw[ids] = sums * scale
    return out, dw


def _exact_dropout(case, state):
    x = state["x"]
    t = int(case["p"] * 65536 + 0.5)
    bits = _philox(x.numel(), state["seed"], state["offset"], x.device).reshape(x.shape)
    factor = (bits >= t).double() / (1.0 - t / 65536.0)
    y = x.double() * factor
    if state["res"] is not None:
        y += state["res"].double()
    return y, state["dout"].double() * factor


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(case, state)
    return _exact_embedding(state) if case["kind"] == "embedding" else _exact_dropout(case, state)
