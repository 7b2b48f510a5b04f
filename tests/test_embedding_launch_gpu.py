"""The embedding gradient's launches: threads with tables of different sizes, the same bits as one after the other."""
import threading

import pytest
import torch

from system_lab_b200 import ops
from system_lab_b200.ops import cuda

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_threads_with_tables_of_different_sizes():
    """The sort's shared memory goes by the table: 60 KB for one thread, 200 KB for the other."""
    def case(v, seed):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        tok = torch.randint(0, v, (700,), device=DEV, generator=g)
        w = torch.randn(v, 8, device=DEV, generator=g).requires_grad_(True)
        return tok, w, torch.randn(700, 8, device=DEV, generator=g)

    def gradient(tok, w, dout):
        return torch.autograd.grad(ops.embedding(tok, w, scale=1.5), w, dout)[0]

    cases = [case(60000, 0), case(300000, 1)]
    want = [gradient(*c) for c in cases]
    torch.cuda.synchronize()
    wrong, together = [], threading.Barrier(2, timeout=60)

    def work(i):
        # (a stream of its own, and the kernel's entry directly: autograd's device thread would take turns)
        from system_lab_b200.ops import lookup
        tok, w, dout = cases[i]
        v, h, n = w.shape[0], w.shape[1], tok.numel()
        chunk = lookup._chunk(n)
        at = (n + 1 + (v + 31) // 32 + 3) // 4 * 4
        try:
            with torch.cuda.stream(torch.cuda.Stream()), torch.no_grad():
                scratch = torch.empty(at + (n + chunk - 1) // chunk * (2 * h + 2), dtype=torch.int32, device=DEV)
                dw = torch.empty_like(w)
                args = (tok.data_ptr(), dout.data_ptr(), 0, dw.data_ptr(), 0, scratch.data_ptr(), scratch.data_ptr() + 4 * at, n, chunk,
                        v, h, 1.5, 0, cuda.stream())
                fn = cuda.lib().slab_embedding_bwd
                together.wait()
                codes = {fn(*args) for _ in range(4000)}
                if codes != {0}:
                    wrong.append(f"table of {v} rows: codes {codes}")
                torch.cuda.current_stream().synchronize()
                if not torch.equal(dw, want[i]):
                    wrong.append(f"table of {v} rows: another gradient")
        except Exception as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_transforms_and_gradients_of_gradients(dtype):
    """The lookup is linear in the table and whole-number weights are exact: everything is equal."""
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    w, t = (torch.randint(-8, 9, (50, 24), device=DEV, generator=g).to(dtype) for _ in range(2))
    tok = torch.randint(0, 50, (3, 7), device=DEV, generator=g)
    dout = torch.randint(-2, 3, (2, 3, 7, 24), device=DEV, generator=g).to(dtype)
    look = lambda a: ops.embedding(tok, a, scale=2.0)
    out, tangent = torch.func.jvp(look, (w,), (t,))
    assert torch.equal(out, look(w)) and torch.equal(tangent, look(t))
    assert torch.equal(torch.func.vmap(look)(torch.stack([w, t])), torch.stack([look(w), look(t)]))
    leaf = w.requires_grad_(True)
    want = torch.stack([torch.autograd.grad(look(leaf), leaf, d)[0] for d in dout])
    assert torch.equal(torch.autograd.grad(look(leaf), leaf, dout, is_grads_batched=True)[0], want)
    first = dout[0].clone().requires_grad_(True)
    (got,) = torch.autograd.grad(look(leaf), leaf, first, create_graph=True)
    assert torch.equal(got, want[0])
    assert torch.equal(torch.autograd.grad(got, first, t)[0], look(t))
