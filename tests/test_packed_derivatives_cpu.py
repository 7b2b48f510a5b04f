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
