"""Packed-document attention kernels against a softmax in 64 bits.

Tolerances.  Operands are exact in bf16.  What is rounded is p, ds and every result, each by at most half a step, 2^-8 of
itself, and delta = sum_c do_c o_c is made from the rounded o.  So

* elements: |error| <= 2^-8 (|result| + the same sum with absolute terms); for dq and dk the terms are
  p (|dp| + 2 sum_c |do_c o_c|): ds itself, at most p (|dp| + sum_c |do_c o_c|), and what delta is off by;
* root mean squares: a rounding that is spread evenly over its step is 2^-8 / sqrt(3) of the value where its mantissa is 1 and
  half of that where it is 2, 0.41 * 2^-8 in the mean.  Roundings are independent: the result's own and that of p or ds
  together are below 0.6 * 2^-8 of the output's root mean square, 2^-8 with room.  delta's error does not shrink with
  dp - delta: it is 0.41 * 2^-8 w_i in the root mean square, w_i^2 = sum_c (do_c o_c)^2, and adds w_i scale |sum_j p_ij k_j|
  to dq_i and scale sqrt(sum_i (p_ij w_i q_i)^2) to dk_j, times that."""
import math

import pytest
import torch

from system_lab_b200 import ops
from system_lab_b200.ops import cuda, packed

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 2.0 ** -8


def cu_of(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def reference(q, k, v, cu, scale, window, dout=None):
    """Outputs, and for each the same sum with absolute terms and what delta's rounding adds."""
    t, hq, d = q.shape
    hkv = k.shape[1]
    g = hq // hkv
    z = lambda h: torch.zeros(t, h, d, dtype=torch.float64, device=q.device)
    out, dq, dk, dv = z(hq), z(hq), z(hkv), z(hkv)
    bo, bq, bk, bv = z(hq), z(hq), z(hkv), z(hkv)
    eq, ek = z(hq), z(hkv)                             # what delta's rounding adds (ek squared)
    for a, b in zip(cu[:-1], cu[1:]):
        if a == b:
            continue
        n = b - a
        i = torch.arange(n, device=q.device)
        seen = i[:, None] >= i[None, :]
        if window:
            seen &= i[:, None] - i[None, :] < window
        for h in range(hq):
            qq, kk, vv = q[a:b, h].double(), k[a:b, h // g].double(), v[a:b, h // g].double()
            p = torch.where(seen, qq @ kk.T * scale, -math.inf).softmax(-1)
            out[a:b, h] = p @ vv
            bo[a:b, h] = p @ vv.abs()
            if dout is None:
                continue
            do = dout[a:b, h].double()
            delta = (do * out[a:b, h]).sum(-1, keepdim=True)
            dp = do @ vv.T
            ds = p * (dp - delta) * scale
            slack = p * (dp.abs() + 2 * (do * out[a:b, h]).abs().sum(-1, keepdim=True)) * scale
            dv[a:b, h // g] += p.T @ do
            bv[a:b, h // g] += p.T @ do.abs()
            dq[a:b, h] = ds @ kk
            bq[a:b, h] = slack @ kk.abs()
            dk[a:b, h // g] += ds.T @ qq
            bk[a:b, h // g] += slack.T @ qq.abs()
            w = (do * out[a:b, h]).pow(2).sum(-1, keepdim=True).sqrt()
            eq[a:b, h] = w * scale * (p @ kk).abs()
            ek[a:b, h // g] += (p * w * scale).pow(2).T @ qq.pow(2)
    return (out, bo, None), (dq, bq, eq), (dk, bk, ek.sqrt()), (dv, bv, None)


def make(rows, hq, hkv, d, seed=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    qkv = torch.randn(rows, (hq + 2 * hkv) * d, device=DEV, generator=g).bfloat16()
    q, k, v = (t.unflatten(-1, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], dim=-1))
    return q, k, v, torch.randn(rows, hq, d, device=DEV, generator=g).bfloat16()


def run(q, k, v, docs, dout, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = ops.packed_attention(*leaves, docs, **kw)
    grads = torch.autograd.grad(out, leaves, dout)
    torch.cuda.synchronize()
    cuda.check_status(q.device)
    return (out.detach(), *grads)


def close(got, want, rows=slice(None)):
    for name, x, (ref, bound, extra) in zip(("out", "dq", "dk", "dv"), got, want):
        err = (x.double() - ref)[rows].abs()
        assert torch.isfinite(x[rows]).all(), name
        worst = (err - EPS * (ref.abs() + bound)[rows]).max().item()
        assert worst <= 1e-6, (name, worst, err.max().item())
        rms = ref[rows].pow(2).mean().sqrt().item()
        more = extra[rows].pow(2).mean().sqrt().item() / 2 if extra is not None else 0.0
        assert err.pow(2).mean().sqrt().item() <= EPS * (rms + more) + 1e-6, name


LAYOUTS = [(4, 4, 64), (8, 1, 128), (6, 2, 96), (3, 1, 72), (2, 2, 8), (12, 4, 128), (4, 2, 40)]
LENS = [[1], [2], [127], [128], [129], [300], [1, 0, 1, 126, 1], [64, 64, 128, 5], [7] * 40, [0, 0, 200, 0], [500, 1, 260]]


@pytest.mark.parametrize("hq,hkv,d", LAYOUTS)
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x[:5])))
def test_forward_and_gradients(hq, hkv, d, lens):
    cu = cu_of(lens)
    q, k, v, dout = make(cu[-1], hq, hkv, d)
    docs = ops.pack_documents(torch.tensor(cu, dtype=torch.int32, device=DEV), cu[-1])
    got = run(q, k, v, docs, dout)
    close(got, reference(q, k, v, cu, 1 / math.sqrt(d), 0, dout))


@pytest.mark.parametrize("window", [1, 5, 64, 127, 128, 129, 200, 10 ** 9])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (3, 3, 128)])
def test_window(hq, hkv, d, window):
    cu = cu_of([3, 400, 1, 130, 257])
    q, k, v, dout = make(cu[-1], hq, hkv, d)
    docs = ops.pack_documents(torch.tensor(cu, device=DEV), cu[-1])
    got = run(q, k, v, docs, dout, window=window, scale=0.2)
    close(got, reference(q, k, v, cu, 0.2, window, dout))


def test_large_scores_move_the_maximum():
    """Scores of up to some hundreds that grow along the row: the running maximum is brought up again and again."""
    cu = [0, 700]
    q, k, v, dout = make(700, 2, 1, 128)
    ramp = torch.linspace(0.1, 6.0, 700, device=DEV)[:, None, None]
    k = (k.float() * ramp).bfloat16()
    docs = ops.pack_documents(torch.tensor(cu, device=DEV), 700)
    got = run(q, k, v, docs, dout)
    close(got, reference(q, k, v, cu, 1 / math.sqrt(128), 0, dout))


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (3, 3, 128), (8, 1, 128)])
def test_rows_behind_the_last_document(hq, hkv, d):
    """They may hold anything and are no part of any sum; their outputs and gradients are zero."""
    cu, rows = cu_of([100, 61, 150]), 700
    q, k, v, dout = make(rows, hq, hkv, d)
    want = reference(q, k, v, cu, 1 / math.sqrt(d), 0, dout)
    for t in (q, k, v, dout):
        t[311:330] = float("nan")
        t[330:] = float("inf")
    docs = ops.pack_documents(torch.tensor(cu, device=DEV), rows)
    got = run(q, k, v, docs, dout)
    close(got, want)
    for x in got:
        assert (x[311:] == 0).all()


@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (8, 2, 128), (3, 1, 128)])
def test_blocks_with_documents_also_take_tiles_without(hq, hkv, d):
    """Far more tiles without documents than blocks: those whose tile has some meet many empty ones behind it."""
    cu = cu_of([40, 300])
    q, k, v, dout = make(40000, hq, hkv, d)
    docs = ops.pack_documents(torch.tensor(cu, dtype=torch.int32, device=DEV), len(q))
    for _ in range(3):
        got = run(q, k, v, docs, dout)
        for x in got:
            assert not x[cu[-1]:].any()
        close([x[:cu[-1]] for x in got], reference(q[:cu[-1]], k[:cu[-1]], v[:cu[-1]], cu, 1 / math.sqrt(d), 0, dout[:cu[-1]]))


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (3, 3, 128)])
def test_short_items_behind_rows_that_are_made_again(hq, hkv, d):
    """One tile of an item is stored slowly (all its rows are NaN and made again) while the next item is one step long."""
    cu = cu_of([128] * 400)
    q, k, v, _ = make(cu[-1], hq, hkv, d)
    bad = 200 * 128
    q[:bad, 0] = float("nan")
    docs = ops.pack_documents(torch.tensor(cu, dtype=torch.int32, device=DEV), len(q))
    scale = 1 / math.sqrt(d)
    qq, kk, vv = (t.unflatten(0, (400, 128)).transpose(1, 2).double() for t in (q, k, v))
    kk, vv = (t.repeat_interleave(hq // hkv, dim=1) for t in (kk, vv))
    p = (qq @ kk.mT * scale).masked_fill(~torch.ones(128, 128, dtype=torch.bool, device=DEV).tril(), -math.inf).softmax(-1)
    want, bound = ((p @ x).transpose(1, 2).flatten(0, 1) for x in (vv, vv.abs()))
    for _ in range(3):
        out = ops.packed_attention(q, k, v, docs)
        torch.cuda.synchronize()
        cuda.check_status(out.device)
        assert out[:bad, 0].isnan().all()
        close([out[:, 1:]], [(want[:, 1:], bound[:, 1:], None)])
        close([out[bad:]], [(want[bad:], bound[bad:], None)])


@pytest.mark.parametrize("lens", [[128] * 8, [900, 60, 64], [1024], [1, 1000, 0, 23], [0]])
@pytest.mark.parametrize("hq,hkv,window", [(8, 1, 0), (12, 2, 0), (16, 1, 300)])
def test_heads_of_a_group_in_as_many_parts_as_the_documents_ask_for(hq, hkv, window, lens):
    cu = cu_of(lens)
    rows = max(cu[-1], 1024)
    q, k, v, dout = make(rows, hq, hkv, 64)
    docs = ops.pack_documents(torch.tensor(cu, dtype=torch.int32, device=DEV), rows)
    assert cuda.lib().slab_packed_attn_splits(rows, hq, hkv, window) > 1
    got = run(q, k, v, docs, dout, window=window)
    if cu[-1]:
        close(got, reference(q, k, v, cu, 1 / 8, window, dout))
    for x in got:
        assert not x[cu[-1]:].any()


@pytest.mark.parametrize("rows,hq,hkv,window,least", [(2 ** 21, 64, 1, 0, 4), (2 ** 25, 8, 1, 0, 8), (2 ** 22, 128, 2, 0, 8),
                                                       (2 ** 25, 64, 1, 1024, 1)])
def test_no_item_is_longer_than_a_wait(rows, hq, hkv, window, least):
    """Steps of the longest item of dk and dv: query tiles times heads of a part, 2^18 at most."""
    parts = cuda.lib().slab_packed_attn_splits(rows, hq, hkv, window)
    assert parts >= least and (hq // hkv) % parts == 0
    tiles = min(rows, window + 127 if window else rows) // 128 + 1
    assert tiles * (hq // hkv // parts) <= 2 ** 18 + hq


def test_rows_made_again_for_longer_than_a_wait_lasts():
    """Key tiles of the long document take seconds each: every sum of dv meets an infinity in the last row."""
    lens = [6000] + [100] * 140
    cu = cu_of(lens)
    q, k, v, dout = make(cu[-1], 64, 1, 64)
    dout[5999] = math.inf
    docs = ops.pack_documents(torch.tensor(cu, dtype=torch.int32, device=DEV), len(q))
    got = run(q, k, v, docs, dout)                     # (asks for the status)
    assert got[3][:6000].isinf().all()
    rest = [x[6000:] for x in (q, k, v)]
    want = reference(*rest, [c - 6000 for c in cu[1:]], 1 / 8, 0, dout[6000:])
    close([x[6000:] for x in got], want)


@pytest.mark.parametrize("what", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("window", [0, 16])
def test_no_document_reaches_another(what, value, window):
    """A value that is no number in one row: other documents' rows are as if it were not there, rows of its own document
    that do not see it too."""
    lens, hq, hkv, d = [90, 100, 120, 40], 4, 2, 64
    cu = cu_of(lens)
    q, k, v, dout = make(cu[-1], hq, hkv, d)
    bad = cu[1] + 50
    tensors = dict(q=q, k=k, v=v, dout=dout)
    tensors[what][bad, 0, 3] = value
    docs = ops.pack_documents(torch.tensor(cu, device=DEV), cu[-1])
    got = run(q, k, v, docs, dout, window=window)
    tensors[what][bad, 0, 3] = 0.0
    want = reference(q, k, v, cu, 1 / math.sqrt(d), window, dout)
    others = torch.ones(cu[-1], dtype=torch.bool, device=DEV)
    others[cu[1]:cu[2]] = False
    close(got, want, others)
    # in the document itself: outputs and dq of rows that do not see the bad one
    clear = torch.zeros_like(others)
    clear[cu[1]:bad] = True
    if window:
        clear[bad + window:cu[2]] = True
    close(got[:2], want[:2], clear)
    assert not all(torch.isfinite(x[cu[1]:cu[2]].float()).all() for x in got)


def test_hidden_keys_at_the_types_lowest_value():
    cu = cu_of([60, 60])
    q, k, v, dout = make(120, 2, 2, 64)
    want = reference(q, k, v, cu, 0.125, 0, dout)
    low = torch.finfo(torch.bfloat16).min
    v[60:] = low
    k[60:] = low
    docs = ops.pack_documents(torch.tensor(cu, device=DEV), 120)
    got = run(q, k, v, docs, dout)
    close(got, want, slice(0, 60))


def test_strides_and_orders():
    cu = cu_of([33, 200, 95])
    t, hq, hkv, d = cu[-1], 4, 2, 64
    q, k, v, dout = make(t, hq, hkv, d)
    docs = ops.pack_documents(torch.tensor(cu, device=DEV), t)
    want = reference(q, k, v, cu, 0.125, 0, dout)
    heads_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, dout)]
    close(run(*heads_first[:3], docs, heads_first[3]), want)
    shifted = [torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(x.shape) for x in (q, k, v, dout)]      # 2 bytes off
    close(run(*shifted[:3], docs, shifted[3]), want)
    odd = [torch.cat([x, x[:, :, :3]], dim=-1)[..., :d] for x in (q, k, v, dout)]                          # odd head strides
    close(run(*odd[:3], docs, odd[3]), want)
    one = q[:, :1].expand(t, hq, d)                                                                       # stride 0
    got = run(one, k, v, docs, dout)
    close(got, reference(one, k, v, cu, 0.125, 0, dout))
    fanned = dout[:1, :1, :1].expand(t, hq, d)
    close(run(q, k, v, docs, fanned), reference(q, k, v, cu, 0.125, 0, fanned))


def test_same_bits_every_time_and_from_any_plan():
    cu = cu_of([500, 1, 260, 900])
    q, k, v, dout = make(cu[-1], 8, 2, 128)
    a = run(q, k, v, ops.pack_documents(torch.tensor(cu, device=DEV), cu[-1]), dout)
    b = run(q, k, v, ops.pack_documents(torch.tensor(cu + [cu[-1]] * 3, dtype=torch.int64, device=DEV), cu[-1]), dout)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_plan_from_tokens():
    g = torch.Generator()
    g.manual_seed(3)
    for b, s, vocab in ((1, 1, 2), (3, 700, 40), (2, 128, 3), (5, 333, 100000)):
        tok = torch.randint(0, vocab, (b, s), generator=g)
        want = ops.documents_from_tokens(tok, 0)
        got = ops.documents_from_tokens(tok.to(DEV), 0)
        assert torch.equal(got.doc_lo.cpu(), want.doc_lo) and torch.equal(got.doc_hi.cpu(), want.doc_hi)
        bounds = [0] + [i for i in range(1, b * s + 1) if i == b * s or want.doc_lo[i] == i]
        same = ops.pack_documents(torch.tensor(bounds, device=DEV), b * s)
        assert torch.equal(same.plan, got.plan)


def test_bad_offsets_are_reported_and_stay_inside():
    q, k, v, dout = make(300, 4, 2, 64)
    for cu in ([0, 200, 100, 300], [0, 100, 400], [5, 300], [-4, 300]):
        cuda.clear_status()
        docs = ops.pack_documents(torch.tensor(cu, device=DEV), 300)
        with pytest.raises(cuda.DeviceHang, match="BAD_INDEX"):
            run(q, k, v, docs, dout)
    assert docs.doc_lo.min() >= 0 and docs.doc_hi.max() <= 300


@pytest.mark.parametrize("cu", [[0, 2 ** 32 + 300], [0, -2 ** 32 + 100, 300], [2 ** 32, 300]])
def test_offsets_past_32_bits_are_reported(cu):
    cuda.clear_status()
    ops.pack_documents(torch.tensor(cu, dtype=torch.int64, device=DEV), 300)
    with pytest.raises(cuda.DeviceHang, match="BAD_INDEX"):
        torch.cuda.synchronize()
        cuda.check_status(torch.device(DEV, torch.cuda.current_device()))
    cuda.clear_status()


def test_no_documents_at_all():
    q, k, v, dout = make(500, 4, 2, 64)
    for cu in ([0], [0, 0, 0]):
        docs = ops.pack_documents(torch.tensor(cu, dtype=torch.int32, device=DEV), 500)
        for x in run(q, k, v, docs, dout):
            assert not x.any()


def test_graph_replay_with_new_documents_and_values():
    """The plan and both passes captured once: a replay takes what the buffers hold then."""
    t = 640
    q, k, v, dout = (x.contiguous() for x in make(t, 4, 2, 64))
    cu = torch.tensor([0, 300, 640, 640], dtype=torch.int32, device=DEV)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]

    def step():
        docs = ops.pack_documents(cu, t)
        out = ops.packed_attention(*leaves, docs)
        return (out, *torch.autograd.grad(out, leaves, dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for lens in ([300, 340, 0], [1, 638, 1], [200, 200, 100]):
        cu.copy_(torch.tensor(cu_of(lens)))
        with torch.no_grad():
            for i, x in enumerate((q, k, v)):
                x.copy_(torch.randn(x.shape, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        cuda.check_status(q.device)
        close([x.detach() for x in got], reference(q.detach(), k.detach(), v.detach(), cu_of(lens), 0.125, 0, dout))


def test_two_streams_at_once():
    cu = cu_of([700, 300])
    docs = ops.pack_documents(torch.tensor(cu, device=DEV), 1000)
    sets = [make(1000, 8, 2, 128, seed) for seed in range(2)]
    alone = [run(*s[:3], docs, s[3]) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                leaves = [x.detach().requires_grad_(True) for x in s[:3]]
                out = ops.packed_attention(*leaves, docs)
                got[i] = (out.detach(), *torch.autograd.grad(out, leaves, s[3]))
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_other_types_and_widths_take_the_oracle():
    cu = cu_of([40, 31])
    docs = ops.pack_documents(torch.tensor(cu, device=DEV), 71)
    for dt, d in ((torch.float32, 64), (torch.bfloat16, 20), (torch.bfloat16, 192)):
        q, k, v = (torch.randn(71, n, d, device=DEV).to(dt) for n in (4, 2, 2))
        out = ops.packed_attention(q, k, v, docs)
        (ref, bound, _), *_ = reference(q, k, v, cu, 1 / math.sqrt(d), 0)
        assert ((out.double() - ref).abs() <= EPS * (ref.abs() + bound) + 1e-6).all()


def test_one_document_is_causal_attention():
    """The framework's batched attention is the case of documents that are the batch's rows."""
    b, s = 2, 256
    q, k, v, _ = make(b * s, 4, 2, 64)
    docs = ops.documents_from_tokens(torch.ones(b, s, dtype=torch.int64, device=DEV), 0)
    got = ops.packed_attention(q, k, v, docs)
    want = ops.causal_attention(*(x.unflatten(0, (b, s)) for x in (q, k, v))).flatten(0, 1)
    assert (got.float() - want.float()).abs().max().item() <= 2 * EPS * want.float().abs().max().item()


def test_elements_past_32_bits():
    """More than 2^31 elements of q, out and their gradients; the last documents against the reference."""
    rows, hq, hkv, d = 2 ** 18 + 77, 64, 1, 128
    cu = [*range(0, rows, 100), rows]
    q, k, v, dout = make(rows, hq, hkv, d)
    docs = ops.pack_documents(torch.tensor(cu, dtype=torch.int32, device=DEV), rows)
    got = run(q, k, v, docs, dout)
    at = cu[-3]
    want = reference(*(t[at:] for t in (q, k, v)), [c - at for c in cu[-3:]], 1 / math.sqrt(d), 0, dout[at:])
    close([x[at:] for x in got], want)
    del got, q, k, v, dout
    torch.cuda.empty_cache()
