"""Derivatives that the kernels of packed attention and the embedding do not have, on the kernel route with every launch left out: they are refused,
or taken by the oracle, and never lost."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from system_lab_b200 import ops
from system_lab_b200.ops import cuda


@pytest.fixture
def route(monkeypatch):
    """The kernels' route on CPU tensors; a launch fails for tensors without storage as it does on the GPU, and does nothing."""
    def launch(name, *args):
        for a in args:
            if isinstance(a, torch.Tensor):
                a.data_ptr()
        return 0
    monkeypatch.setattr(cuda, "call", launch)
    monkeypatch.setattr(cuda, "stream", lambda: 0)
    monkeypatch.setattr(cuda, "status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(ops, "use_kernels", lambda t: True)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", range(3))
def test_packed_attention_refuses_tangents(route, which, grad):
    qkv = [torch.randn(16, n, 8).bfloat16() for n in (4, 2, 2)]
    docs = ops.pack_documents(torch.tensor([0, 16]), 16)
    with torch.set_grad_enabled(grad), fw.dual_level():
        ops.packed_attention(*qkv, docs)                       # nothing carries a tangent
        qkv[which] = fw.make_dual(qkv[which], torch.ones_like(qkv[which]))
        with pytest.raises(NotImplementedError, match="forward mode"):
            ops.packed_attention(*qkv, docs)


TABLE, TOKENS = (9, 6), torch.tensor([[3, 3, 8], [0, 1, 3]])


def lookup(scale):
    return lambda w: ops.embedding(TOKENS, w, scale=scale)


@pytest.mark.parametrize("scale", [1.0, 2.5])
@pytest.mark.parametrize("grad", [True, False])
def test_embedding_tangents(route, grad, scale):
    """The lookup is linear: its tangent is the lookup of the table's."""
    w, t = torch.randn(TABLE), torch.randn(TABLE)
    with torch.set_grad_enabled(grad), fw.dual_level():
        out = fw.unpack_dual(lookup(scale)(fw.make_dual(w, t)))
        torch.testing.assert_close(out.tangent, t[TOKENS] * scale)
        torch.testing.assert_close(out.primal, w[TOKENS] * scale)
    out, tangent = torch.func.jvp(lookup(scale), (w,), (t,))
    torch.testing.assert_close(tangent, t[TOKENS] * scale)


@pytest.mark.parametrize("scale", [1.0, 2.5])
def test_embedding_transforms(route, scale):
    w, g = torch.randn(TABLE), torch.randn(*TOKENS.shape, TABLE[1])
    want = torch.zeros(TABLE).index_add_(0, TOKENS.reshape(-1), g.reshape(-1, TABLE[1]) * scale)
    torch.testing.assert_close(torch.func.vjp(lookup(scale), w)[1](g)[0], want)
    torch.testing.assert_close(torch.func.grad(lambda a: (lookup(scale)(a) * g).sum())(w), want)
    torch.testing.assert_close(torch.func.vmap(lookup(scale))(torch.stack([w, 2 * w])), torch.stack([w[TOKENS], 2 * w[TOKENS]]) * scale)


@pytest.mark.parametrize("flat", [False, True])
@pytest.mark.parametrize("scale", [1.0, 2.5])
def test_embedding_gradients_that_are_batched_or_differentiated(route, scale, flat):
    """With a flat gradient buffer too, which such a gradient must not touch."""
    w = torch.randn(TABLE).requires_grad_(True)
    if flat:
        w.main_grad, w.main_grad_written = torch.full(TABLE, 7.0), False
    g = torch.randn(2, *TOKENS.shape, TABLE[1])
    want = torch.stack([torch.zeros(TABLE).index_add_(0, TOKENS.reshape(-1), x.reshape(-1, TABLE[1]) * scale) for x in g])
    (got,) = torch.autograd.grad(lookup(scale)(w), w, g, is_grads_batched=True)
    torch.testing.assert_close(got, want)
    first = g[0].clone().requires_grad_(True)
    (got,) = torch.autograd.grad(lookup(scale)(w), w, first, create_graph=True)
    torch.testing.assert_close(got, want[0])
    again = torch.randn(TABLE)
    torch.testing.assert_close(torch.autograd.grad(got, first, again)[0], again[TOKENS] * scale)
    if flat:
        assert (w.main_grad == 7.0).all() and not w.main_grad_written


def test_embedding_gradients_of_ids_outside_the_table(route):
    w = torch.randn(TABLE).requires_grad_(True)
    tok = torch.tensor([3, -1, 9, 2 ** 40])
    g = torch.ones(4, TABLE[1])
    (got,) = torch.autograd.grad(ops.embedding(tok, w), w, g, create_graph=True)
    want = torch.zeros(TABLE)
    want[3] = 1.0
    assert torch.equal(got.detach(), want)
