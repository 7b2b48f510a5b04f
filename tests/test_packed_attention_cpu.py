"""Packed documents on the CPU: the plan's document ranges, the oracle against a row-by-row softmax in 64 bits, refusals."""
import math

import pytest
import torch

from system_lab_b200 import ops


def rowwise(q, k, v, cu, scale, window):
    """Every row by itself, in 64 bits."""
    t, hq, d = q.shape
    g = hq // k.shape[1]
    q, k, v = (x.double() for x in (q, k, v))
    out = torch.zeros(t, hq, d, dtype=torch.float64)
    for a, b in zip(cu[:-1], cu[1:]):
        for i in range(a, b):
            f = max(a, i - window + 1) if window else a
            for h in range(hq):
                s = (k[f:i + 1, h // g] @ q[i, h]) * scale
                out[i, h] = torch.softmax(s, 0) @ v[f:i + 1, h // g]
    return out


CU = [[0, 7], [0, 1, 1, 2, 9, 9, 20], [0, 0, 16], [0]]


@pytest.mark.parametrize("cu", CU)
@pytest.mark.parametrize("tail", [0, 3])
def test_ranges_from_offsets(cu, tail):
    rows = cu[-1] + tail or 2
    p = ops.pack_documents(torch.tensor(cu, dtype=torch.int32), rows)
    lo, hi = [i + 1 for i in range(rows)], list(range(rows))
    for a, b in zip(cu[:-1], cu[1:]):
        for i in range(a, b):
            lo[i], hi[i] = a, b
    assert p.doc_lo.tolist() == lo and p.doc_hi.tolist() == hi


def test_ranges_from_tokens():
    tok = torch.tensor([[5, 0, 3, 4], [0, 1, 2, 0], [1, 1, 0, 0]])
    p = ops.documents_from_tokens(tok, 0)
    #                        5  0 | 3  4 || 0 | 1  2  0 || 1   1   0 | 0
    assert p.doc_lo.tolist() == [0, 0, 2, 2, 4, 5, 5, 5, 8, 8, 8, 11]
    assert p.doc_hi.tolist() == [2, 2, 4, 4, 5, 8, 8, 8, 11, 11, 11, 12]


@pytest.mark.parametrize("window", [0, 1, 4])
@pytest.mark.parametrize("cu,tail", [([0, 9], 0), ([0, 1, 1, 5, 14], 3)])
def test_oracle(cu, tail, window):
    torch.manual_seed(0)
    t = cu[-1] + tail
    q, k, v = torch.randn(t, 4, 8), torch.randn(t, 2, 8), torch.randn(t, 2, 8)
    v[cu[-1]:] = float("nan")                                  # rows of no document
    docs = ops.pack_documents(torch.tensor(cu), t)
    out = ops.packed_attention(q, k, v, docs, window=window)
    torch.testing.assert_close(out.double(), rowwise(q, k, v, cu, 1 / math.sqrt(8), window), rtol=1e-5, atol=1e-5)


def test_oracle_gradients_against_differences():
    torch.manual_seed(1)
    q, k, v = (torch.randn(11, n, 4, dtype=torch.float64, requires_grad=True) for n in (4, 2, 2))
    docs = ops.pack_documents(torch.tensor([0, 4, 4, 9]), 11)
    assert torch.autograd.gradcheck(lambda a, b, c: ops.packed_attention(a, b, c, docs, window=3), (q, k, v))


def test_refusals():
    t = torch.tensor
    for cu in (t([1, 4]), t([0, 5, 4]), t([0, 9])):
        with pytest.raises(ValueError):
            ops.pack_documents(cu, 8)
    for cu, rows in ((t([[0, 4]]), 8), (t([0.0, 4.0]), 8), (t([], dtype=torch.int32), 8), (t([0, 0]), 0)):
        with pytest.raises(ValueError):
            ops.pack_documents(cu, rows)
    for tok in (torch.zeros(4, dtype=torch.int64), torch.zeros(0, 4, dtype=torch.int64), torch.zeros(2, 4, dtype=torch.int32)):
        with pytest.raises(ValueError):
            ops.documents_from_tokens(tok, 0)
    docs = ops.pack_documents(t([0, 8]), 8)
    q, k = torch.randn(8, 4, 8), torch.randn(8, 2, 8)
    bad = [dict(q=torch.randn(2, 8, 4, 8)), dict(k=torch.randn(8, 3, 8), v=torch.randn(8, 3, 8)), dict(v=torch.randn(8, 2, 16)),
           dict(q=torch.randn(7, 4, 8)), dict(k=torch.randn(8, 2, 16), v=torch.randn(8, 2, 16)), dict(window=-1),
           dict(scale=0.0), dict(scale=float("nan")), dict(q=q.double()), dict(documents=ops.pack_documents(t([0, 4]), 4))]
    for kw in bad:
        args = dict(q=q, k=k, v=k, documents=docs, scale=None, window=0)
        args.update(kw)
        with pytest.raises(ValueError):
            ops.packed_attention(**args)


def test_more_rows_than_the_kernels_count_are_refused():
    with pytest.raises(ValueError, match="rows"):
        ops.pack_documents(torch.tensor([0, 4]), 2 ** 30)
    with pytest.raises(ValueError, match="rows"):
        ops.documents_from_tokens(torch.zeros(1, 1, dtype=torch.int64).expand(2 ** 15, 2 ** 15), 0)
