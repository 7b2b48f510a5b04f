"""Packed attention on values that are no numbers, in tiles that are seen whole: what the formula gives, element by element.

The formula is a sum over what a row sees and nothing else, so the reference adds up seen pairs only (a hidden pair's zero
times an infinity is not part of it).  A result is compared by its kind (a number, NaN, either infinity) and, where it is a
number, within the bounds of test_packed_attention_gpu: an element is off by at most 2^-8 (|result| + the sum's absolute
terms), p and ds being rounded to bf16 by half a step and so being the result."""
import math

import pytest
import torch

from system_lab_b200 import ops
from system_lab_b200.ops import cuda

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 2.0 ** -8
ROWS = 400                                           # the tiles of keys 0 .. 127 and 128 .. 255 are whole for later query tiles


def make(hq, hkv, d, seed=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return [torch.randn(ROWS, n, d, device=DEV, generator=g).bfloat16() for n in (hq, hkv, hkv, hq)]


def weighted(w, x, seen):
    """sum_j w_ij x_j over the seen pairs, and the same with absolute terms."""
    terms = torch.where(seen[:, :, None], w[:, :, None] * x[None], 0.0)
    return terms.sum(1), terms.abs().sum(1)


def reference(q, k, v, dout):
    _, hq, d = q.shape
    hkv = k.shape[1]
    scale = 1 / math.sqrt(d)
    i = torch.arange(ROWS, device=DEV)
    seen = i[:, None] >= i[None, :]
    z = lambda h: torch.zeros(ROWS, h, d, dtype=torch.float64, device=DEV)
    out, dq, dk, dv, bo, bq, bk, bv = (z(h) for h in (hq, hq, hkv, hkv) * 2)
    for h in range(hq):
        u = h * hkv // hq
        qq, kk, vv, do = q[:, h].double(), k[:, u].double(), v[:, u].double(), dout[:, h].double()
        p = torch.where(seen, qq @ kk.T * scale, -math.inf).softmax(-1)
        out[:, h], bo[:, h] = weighted(p, vv, seen)
        dp, delta = do @ vv.T, (do * out[:, h]).sum(-1, keepdim=True)
        ds = p * (dp - delta) * scale
        slack = p * (dp.abs() + 2 * (do * out[:, h]).abs().sum(-1, keepdim=True)) * scale
        dq[:, h], _ = weighted(ds, kk, seen)
        bq[:, h], _ = weighted(slack, kk.abs(), seen)
        for into, x, w in ((dk, qq, ds), (bk, qq.abs(), slack), (dv, do, p), (bv, do.abs(), p)):
            into[:, u] += weighted(w.T, x, seen.T)[0]
    return (out, bo), (dq, bq), (dk, bk), (dv, bv)


def check(q, k, v, dout):
    docs = ops.pack_documents(torch.tensor([0, ROWS], dtype=torch.int32, device=DEV), ROWS)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = ops.packed_attention(*leaves, docs)
    got = (out.detach(), *torch.autograd.grad(out, leaves, dout))
    with torch.no_grad():
        scored = ops.packed_attention(q, k, v, docs)
    torch.cuda.synchronize()
    cuda.check_status(q.device)
    want = reference(q, k, v, dout)
    for name, x, (ref, bound) in zip(("out", "dq", "dk", "dv", "scored"), (*got, scored), (*want, want[0])):
        for kind in (torch.isnan, torch.isposinf, torch.isneginf):
            wrong = (kind(x) != kind(ref)).any(-1).nonzero()
            assert not len(wrong), (name, kind.__name__, wrong[:4].tolist())
        fine = torch.isfinite(ref)
        off = ((x.double() - ref).abs() - EPS * (ref.abs() + bound))[fine]
        assert not off.numel() or off.max().item() <= 1e-6, (name, off.max().item())
    return got


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (3, 3, 128)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("what", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("column", [0, 13, 14, 15, 30, 31])
def test_one_value(what, column, value, hq, hkv, d):
    """In a key of the first tile, in a query of the third: each is seen through whole tiles by (or sees whole tiles of) others."""
    t = dict(zip(("q", "k", "v", "dout"), make(hq, hkv, d)))
    t[what][column + (0 if what in "kv" else 256), 0, 3] = value
    got = check(**t)
    assert not all(x.isfinite().all() for x in got)


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (3, 3, 128)])
def test_scores_that_are_all_minus_infinity(hq, hkv, d):
    """No key is left to a row: 0 / 0.  Once the first tile's keys only, which then weigh nothing beside the others."""
    for hidden in (ROWS, 128):
        q, k, v, dout = make(hq, hkv, d)
        q[:, :, 3] = q[:, :, 3].abs() + 0.25
        k[:hidden, :, 3] = -math.inf
        got = check(q, k, v, dout)
        assert got[0][:hidden].isnan().all() and got[0][hidden:].isfinite().all()


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (3, 3, 128)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("low", [-2.0 ** 16, -math.inf])
def test_a_value_without_weight(low, value, hq, hkv, d):
    """Zero times what is no number is no number, whether the zero is an exponential's or that of a score of -inf."""
    q, k, v, dout = make(hq, hkv, d)
    q[:, :, 3] = q[:, :, 3].abs() + 0.25
    k[14, :, 3] = low
    v[14, 0, 5] = value
    check(q, k, v, dout)


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (3, 3, 128)])
def test_keys_far_below_the_maximum_weigh_nothing(hq, hkv, d):
    """The type's largest value times a probability of 2^-2000 and less is zero."""
    q, k, v, dout = make(hq, hkv, d)
    q[:, :, 3] = q[:, :, 3].abs() + 0.25
    k[10:32, :, 3] = -2.0 ** 16
    v[10:32] = torch.finfo(torch.bfloat16).max
    docs = ops.pack_documents(torch.tensor([0, ROWS], dtype=torch.int32, device=DEV), ROWS)
    out = ops.packed_attention(q, k, v, docs)
    torch.cuda.synchronize()
    cuda.check_status(out.device)
    ref, bound = reference(q, k, v, dout)[0]
    off = (out.double() - ref).abs() - EPS * (ref.abs() + bound)
    assert off[33:].max().item() <= 1e-6


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (3, 3, 128)])
@pytest.mark.parametrize("signs", [False, True])
def test_values_near_the_largest(signs, hq, hkv, d):
    """A mean of values near the type's largest is a number, though their sum is none."""
    q, k, v, dout = make(hq, hkv, d)
    large = torch.finfo(torch.bfloat16).max
    v = torch.where(v > 0, large, -large).bfloat16() if signs else torch.full_like(v, -large)
    docs = ops.pack_documents(torch.tensor([0, ROWS], dtype=torch.int32, device=DEV), ROWS)
    ref, bound = reference(q, k, v, dout)[0]
    for x in (q, q.detach().requires_grad_(True)):
        out = ops.packed_attention(x, k, v, docs).detach()
        torch.cuda.synchronize()
        cuda.check_status(out.device)
        assert out.isfinite().all()
        assert ((out.double() - ref).abs() <= EPS * (ref.abs() + bound)).all()


def test_one_row_that_takes_longer_than_a_wait_lasts():
    """dv of the first key is 2^127 in three columns, whose sum passes fp32: the row is made again, four million pairs one by one,
    some four seconds.  Nothing else is (v is small beside dout's large columns, so dP and delta stay numbers)."""
    rows, hq, d = 60000, 64, 64
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    q, k, v, dout = (torch.randn(rows, n, d, device=DEV, generator=g).bfloat16() for n in (hq, 1, 1, hq))
    v[:, :, :3] *= 2.0 ** -20
    q[-1, 0] = 8 * k[0, 0]                            # the last query sees the first key: e^60 and more, the others at most e^40
    dout[-1, 0] = 0.0
    dout[-1, 0, :3] = 2.0 ** 127
    docs = ops.pack_documents(torch.tensor([0, rows], dtype=torch.int32, device=DEV), rows)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(ops.packed_attention(*leaves, docs), leaves, dout)
    torch.cuda.synchronize()
    cuda.check_status(q.device)
    for x in grads:
        assert x.isfinite().all()
    # (p is 1 within 2^-9 there, every other term is nothing beside it)
    assert ((grads[2][0, 0, :3].double() / 2.0 ** 127 - 1).abs() <= 2 * EPS).all()
    del leaves, grads, q, k, v, dout
    torch.cuda.empty_cache()
