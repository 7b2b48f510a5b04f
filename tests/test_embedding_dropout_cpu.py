"""Embedding lookup and counter-based dropout on the CPU: oracles, the generator's published answers, refusals."""
import pytest
import torch

from system_lab_b200 import ops
from system_lab_b200.ops import reference as ref


def _words(bits):
    b = bits.view(-1, 4, 2)
    return (b[..., 0] | (b[..., 1] << 16)).tolist()


def test_philox_known_answers():
    """Philox-4x32-10 answers published with the generator (Random123's kat_vectors): counter and key zero, all ones, and
    digits of pi."""
    assert [hex(w) for w in _words(ref.philox_bits(8, 0, 0))[0]] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


def test_dropout_definition():
    x = torch.randn(7, 13)
    r = torch.randn(7, 13)
    y = ops.dropout(x, 0.3, seed=5, offset=9, residual=r)
    t = ref.dropout_threshold(0.3)
    keep = (ref.philox_bits(91, 5, 9) >= t).view(7, 13)
    torch.testing.assert_close(y, torch.where(keep, x * (65536 / (65536 - t)), 0.0) + r)
    assert torch.equal(ops.dropout(x, 0.3, 5, 9), ops.dropout(x, 0.3, torch.tensor([5]), 9))
    assert not torch.equal(ops.dropout(x, 0.3, 5, 9), ops.dropout(x, 0.3, 5, 10))
    assert not torch.equal(ops.dropout(x, 0.3, 5, 9), ops.dropout(x, 0.3, 6, 9))
    assert torch.equal(ops.dropout(x, 0.0, 5), x)
    # a prefix has the prefix of the mask, whatever the tensor's length
    assert torch.equal(ops.dropout(x.reshape(-1)[:50], 0.3, 5, 9), ops.dropout(x, 0.3, 5, 9).reshape(-1)[:50])


def test_dropout_rate_and_mean():
    """2^20 elements: the rate's standard deviation is at most 2^-11, the mean's as small for p = 1/2: five of them."""
    for p in (0.1, 0.5, 0.9):
        y = ops.dropout(torch.ones(1 << 20), p, seed=77)
        assert abs((y == 0).float().mean().item() - p) < 5 * (p * (1 - p)) ** 0.5 / 1024
        assert abs(y.double().mean().item() - 1.0) < 5 * (p / (1 - p)) ** 0.5 / 1024
    bits = ref.philox_bits(1 << 20, 77, 0)
    for e in range(8):                                     # each of a block's eight elements by itself
        share = (bits[e::8] < 6554).float().mean().item()
        assert abs(share - 0.1) < 5 * (0.09 / (1 << 17)) ** 0.5


def test_gradients_against_differences():
    x = torch.randn(3, 5, dtype=torch.float64, requires_grad=True)
    r = torch.randn(3, 5, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a, b: ops.dropout(a, 0.4, 3, residual=b), (x, r))
    w = torch.randn(6, 4, dtype=torch.float64, requires_grad=True)
    tok = torch.tensor([[1, 5, 1], [0, 1, 2]])
    assert torch.autograd.gradcheck(lambda a: ops.embedding(tok, a, scale=1.7), (w,))


def test_embedding_values():
    w = torch.randn(9, 6).bfloat16()
    tok = torch.tensor([[3, 3, 8], [0, 1, 3]], dtype=torch.int32)
    assert torch.equal(ops.embedding(tok, w), w[tok.long()])
    out = ops.embedding(tok, w, scale=2.5, dtype=torch.float32)
    assert out.dtype == torch.float32 and torch.equal(out, w[tok.long()].float() * 2.5)


def test_refusals():
    x = torch.randn(4, 8)
    for kw in (dict(p=1.0), dict(p=-0.1), dict(p=0.999999), dict(p=float("nan")), dict(seed=1.5), dict(seed=True), dict(seed=1 << 64),
               dict(seed=torch.tensor([1, 2])), dict(seed=torch.tensor([1.0])), dict(offset=-1), dict(offset=1 << 64),
               dict(residual=torch.randn(8, 4)), dict(residual=torch.randn(4, 8).double()), dict(x=torch.ones(3, dtype=torch.int64))):
        args = dict(x=x, p=0.1, seed=1)
        args.update(kw)
        with pytest.raises(ValueError):
            ops.dropout(**args)
    for tok, w in ((torch.zeros(2), torch.randn(3, 4)), (torch.zeros(2, dtype=torch.int64), torch.randn(12)),
                   (torch.zeros(2, dtype=torch.int64), torch.randn(0, 4)), (torch.zeros(2, dtype=torch.bool), torch.randn(3, 4))):
        with pytest.raises(ValueError):
            ops.embedding(tok, w)


def test_more_tokens_than_the_kernels_count_are_refused():
    with pytest.raises(ValueError, match="tokens"):
        ops.embedding(torch.zeros(1, dtype=torch.int64).expand(2 ** 30 + 1), torch.zeros(4, 8))
