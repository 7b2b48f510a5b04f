"""Embedding and dropout kernels against plain forms in 64 bits.

Tolerances: a lookup rounds the fp32 product (2^-24) and the result (half a step); the table's gradient is a sum of n terms
in fp32 with an error of at most n 2^-24 sum |terms|, times scale (2^-24), rounded once; with an old gradient added it is one
rounding more.  Dropout: fp32 product and sum (2^-24 of each), rounded once.  The mask is equal, always."""
import pytest
import torch

from system_lab_b200 import ops
from system_lab_b200.ops import cuda
from system_lab_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def check_gradient(dw, tokens, dout, scale, old=None):
    tok = tokens.reshape(-1).long()
    ok = (tok >= 0) & (tok < dw.shape[0])
    tok, d = tok[ok], dout.reshape(-1, dw.shape[1])[ok].double()
    want = torch.zeros(dw.shape, dtype=torch.float64, device=DEV)
    size, count = torch.zeros_like(want), torch.zeros(dw.shape[0], dtype=torch.float64, device=DEV)
    want.index_add_(0, tok, d)
    size.index_add_(0, tok, d.abs())
    count.index_add_(0, tok, torch.ones_like(tok, dtype=torch.float64))
    want, size = want * scale, size * abs(scale)
    tol = (count[:, None] + 3) * U * size
    if old is not None:
        want = want + old.double()
        tol = tol + U * old.double().abs()
    tol = tol + half(dw.dtype) * (want.abs() + tol) + 1e-30
    err = (dw.double() - want).abs()
    assert (err <= tol).all(), (err - tol).max().item()


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.float32, torch.bfloat16),
         (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("wd,od", TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("n,v,h", [(1, 1, 8), (1, 50000, 1), (2, 3, 7), (77, 5, 136), (300, 300, 256), (513, 1024, 100),
                                   (4100, 900, 64), (2049, 200000, 24), (20000, 33, 40), (9000, 60000, 33)])
def test_lookup_and_gradient(n, v, h, wd, od):
    g = torch.Generator(device=DEV)
    g.manual_seed(n)
    tokens = torch.randint(0, v, (n,), device=DEV, generator=g)
    w = torch.randn(v, h, device=DEV, generator=g).to(wd).requires_grad_(True)
    dout = torch.randn(n, h, device=DEV, generator=g).to(od)
    out = ops.embedding(tokens, w, scale=3.7, dtype=od)
    scale = torch.tensor(3.7, dtype=torch.float32).double()
    want = w.detach()[tokens].double() * scale.item()
    assert out.dtype == od and ((out.double() - want).abs() <= (half(od) + 2 * U) * want.abs()).all()
    (dw,) = torch.autograd.grad(out, w, dout)
    assert dw.dtype == wd
    check_gradient(dw, tokens, dout, scale.item())
    torch.cuda.synchronize()
    cuda.check_status(w.device)


@pytest.mark.parametrize("n", [5, 31, 64, 1000, 3000, 40000])
@pytest.mark.parametrize("kind", ["one", "two halves", "alternate", "ladder"])
def test_runs_over_chunk_borders(n, kind):
    """The same token everywhere, runs that end at, before and behind the chunks' borders."""
    i = torch.arange(n, device=DEV)
    tokens = {"one": i * 0 + 4, "two halves": (i >= n // 2).long() * 3, "alternate": i % 2,
              "ladder": (i.float() * 2).sqrt().long()}[kind]
    w = torch.zeros(400, 16, device=DEV, requires_grad=True)
    dout = torch.randn(n, 16, device=DEV)
    (dw,) = torch.autograd.grad(ops.embedding(tokens, w), w, dout)
    check_gradient(dw, tokens, dout, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("h", [64, 13])
def test_flat_gradient_buffer(dtype, h):
    """Written on the first micro-batch, added to on later ones; rows no token names keep what they held."""
    v = 2000
    w = torch.randn(v, h, device=DEV).to(dtype).requires_grad_(True)
    buf = torch.full((v * h + 8,), float("nan"), device=DEV, dtype=dtype)
    w.main_grad, w.main_grad_written = buf[8:].view(v, h), False
    for step in range(3):
        tokens = torch.randint(0, v, (3, 500), device=DEV)
        dout = torch.randn(3, 500, h, device=DEV).to(dtype)
        old = w.main_grad.clone() if step else None
        ops.embedding(tokens, w, scale=0.5).backward(dout)
        assert w.grad is None and w.main_grad_written
        check_gradient(w.main_grad, tokens, dout, 0.5, old)
        if step:
            untouched = torch.ones(v, dtype=torch.bool, device=DEV)
            untouched[tokens.reshape(-1)] = False
            assert torch.equal(w.main_grad[untouched], old[untouched])
    assert torch.isnan(buf[:8]).all()


def test_ids_outside_the_table():
    w = torch.randn(50, 24, device=DEV, requires_grad=True)
    tokens = torch.tensor([3, -1, 49, 50, 2 ** 40, 3, -2 ** 40], device=DEV)
    cuda.clear_status()
    out = ops.embedding(tokens, w)
    with pytest.raises(cuda.DeviceHang, match="BAD_INDEX"):
        cuda.check_status(w.device)
    bad = torch.tensor([1, 3, 4, 6], device=DEV)
    assert (out[bad] == 0).all() and torch.equal(out[[0, 2, 5]], w.detach()[[3, 49, 3]])
    dout = torch.randn(7, 24, device=DEV)
    (dw,) = torch.autograd.grad(out, w, dout)
    check_gradient(dw, tokens, dout, 1.0)


def test_shapes_strides_and_empty():
    w = torch.randn(60, 32, device=DEV).bfloat16()
    wt = torch.randn(32, 60, device=DEV).bfloat16().t().requires_grad_(True)      # a transposed table
    tokens = torch.randint(0, 60, (6, 8), device=DEV, dtype=torch.int32).t()
    out = ops.embedding(tokens, wt)
    assert torch.equal(out, wt.detach()[tokens.long()])
    dout = torch.randn(32, 6, 8, device=DEV).bfloat16().permute(2, 1, 0)
    (dw,) = torch.autograd.grad(out, wt, dout)
    check_gradient(dw, tokens, dout, 1.0)
    fanned = torch.ones(1, device=DEV).bfloat16().expand(8, 6, 32)
    (dw,) = torch.autograd.grad(ops.embedding(tokens, wt), wt, fanned)
    check_gradient(dw, tokens, fanned, 1.0)
    wr = w.clone().requires_grad_(True)
    none = ops.embedding(torch.zeros(0, 3, dtype=torch.int64, device=DEV), wr)
    assert none.shape == (0, 3, 32)
    (dw,) = torch.autograd.grad(none.sum(), wr)
    assert (dw == 0).all()
    part = torch.cat([w.reshape(-1), w.reshape(-1)])[3:3 + 60 * 32].view(60, 32)          # off a 16-byte border
    assert torch.equal(ops.embedding(tokens, part), part[tokens.long()])


def test_embedding_same_bits_every_time_and_replayed():
    w = torch.randn(3001, 128, device=DEV).bfloat16().requires_grad_(True)
    tokens = (torch.rand(9000, device=DEV) ** 4 * 3001).long()
    dout = torch.randn(9000, 128, device=DEV).bfloat16()

    def step():
        return torch.autograd.grad(ops.embedding(tokens, w, scale=2.0), w, dout)[0]

    first = step()
    for _ in range(3):
        assert torch.equal(first, step())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for top in (3001, 7, 1):
        tokens.copy_(torch.randint(0, top, (9000,), device=DEV))
        graph.replay()
        check_gradient(got, tokens, dout, 2.0)
        assert torch.equal(got, step())


# ------------------------------------------------------------------ dropout
def plain(x, p, seed, offset, residual):
    t = ref.dropout_threshold(p)
    keep = (ref.philox_bits(x.numel(), seed, offset, x.device) >= t).view(x.shape)
    y = torch.where(keep, x.double(), 0.0) / (1.0 - t / 65536.0)
    return (y + residual.double() if residual is not None else y), keep


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (2047,), (2049,), (3, 5, 17), (77, 2880), (1000, 256)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.9999])
def test_dropout(shape, p, residual, dtype):
    g = torch.Generator(device=DEV)
    g.manual_seed(len(shape))
    x = torch.randn(shape, device=DEV, generator=g).to(dtype).requires_grad_(True)
    r = torch.randn(shape, device=DEV, generator=g).to(dtype).requires_grad_(True) if residual else None
    seed, offset = -987654321987654321, (1 << 63) + 5
    y = ops.dropout(x, p, seed, offset, residual=r)
    want, keep = plain(x.detach(), p, seed, offset, r.detach() if residual else None)
    terms = x.detach().double().abs() * (65536 / (65536 - ref.dropout_threshold(p))) + (r.detach().double().abs() if residual else 0.0)
    assert ((y.double() - want).abs() <= half(dtype) * want.abs() + 3 * U * terms).all()
    if not residual:
        assert torch.equal(y != 0, keep & (x != 0))
    dout = torch.randn(shape, device=DEV, generator=g).to(dtype)
    grads = torch.autograd.grad(y, (x, r) if residual else (x,), dout)
    want, _ = plain(dout, p, seed, offset, None)
    assert ((grads[0].double() - want).abs() <= (half(dtype) + 3 * U) * want.abs()).all()
    if residual:
        assert torch.equal(grads[1], dout)


@pytest.mark.parametrize("n", [2 ** 22 - 1, 2 ** 22, 2 ** 22 + 1, 2 ** 22 + 8 * 256 + 5, 2 ** 22 + 8192 + 4099])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_of_many_elements(n, residual):
    """Around the size from which a thread takes several blocks, whole and ragged."""
    x = torch.randn(n, device=DEV).bfloat16()
    r = torch.randn(n, device=DEV).bfloat16() if residual else None
    t = ref.dropout_threshold(0.25)
    keep = ref.philox_bits(n, 3, 9, x.device) >= t
    want = torch.where(keep, x.double() * 65536 / (65536 - t), 0.0) + (r.double() if residual else 0.0)
    got = ops.dropout(x, 0.25, 3, 9, residual=r)
    # one rounding to bf16 behind a product and a sum in fp32 (two roundings of 2^-24 of the terms)
    bound = want.abs() * 2.0 ** -8 + (x.double().abs() * 1.34 + want.abs()) * 2.0 ** -23
    assert bool(((got.double() - want).abs() <= bound).all())
    assert not got[~keep].any() if not residual else torch.equal(got[~keep], r[~keep])


def test_dropped_elements_may_be_anything():
    x = torch.randn(4096, device=DEV)
    _, keep = plain(x, 0.5, 1, 0, None)
    x[~keep] = float("nan")
    assert torch.isfinite(ops.dropout(x, 0.5, 1)).all()
    r = torch.randn(4096, device=DEV)
    assert torch.equal(ops.dropout(x, 0.5, 1, residual=r)[~keep], r[~keep])


def test_dropout_strides_and_empty():
    base = torch.randn(64, 33, device=DEV)
    x = base.t()
    r = torch.randn(66, 64, device=DEV)[::2]
    y = ops.dropout(x, 0.25, 4, residual=r)
    want, _ = plain(x.contiguous(), 0.25, 4, 0, r)
    torch.testing.assert_close(y.double(), want, rtol=1e-6, atol=1e-6)
    off = torch.randn(1001, device=DEV).bfloat16()[1:]
    want, _ = plain(off, 0.25, 4, 0, None)
    assert ((ops.dropout(off, 0.25, 4).double() - want).abs() <= (half(off.dtype) + 3 * U) * want.abs()).all()
    assert ops.dropout(torch.zeros(0, 5, device=DEV), 0.5, 1).shape == (0, 5)
    xg = torch.randn(33, 64, device=DEV, requires_grad=True)
    one = torch.ones(1, device=DEV).expand(33, 64)
    (dx,) = torch.autograd.grad(ops.dropout(xg, 0.25, 4), xg, one)
    want, _ = plain(torch.ones(33, 64, device=DEV), 0.25, 4, 0, None)
    torch.testing.assert_close(dx.double(), want, rtol=1e-6, atol=0)


def test_replayed_graph_draws_with_the_seed_it_finds():
    x = torch.randn(5000, device=DEV, requires_grad=True)
    dout = torch.randn(5000, device=DEV)
    seed = torch.tensor([11], device=DEV)

    def step():
        y = ops.dropout(x, 0.3, seed, 2)
        seed.add_(0)                                        # the forward pass's value is what backward uses
        return y, torch.autograd.grad(y, x, dout)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
    for s in (11, 12, -5):
        seed.fill_(s)
        graph.replay()
        assert torch.equal(y, ops.dropout(x, 0.3, s, 2))
        assert torch.equal(dx, ops.dropout(dout, 0.3, s, 2))


def test_seed_changed_between_forward_and_backward():
    x = torch.randn(3000, device=DEV, requires_grad=True)
    seed = torch.tensor([3], device=DEV)
    y = ops.dropout(x, 0.5, seed)
    seed.fill_(4)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(x))
    assert torch.equal(dx != 0, y != 0)


def test_elements_past_32_bits():
    """A table and a dropped tensor of more than 2^31 elements: their last rows."""
    v, h = 2 ** 20 + 3, 2056
    w = torch.empty(v, h, dtype=torch.bfloat16, device=DEV)
    w[-2:] = torch.randn(2, h, device=DEV).bfloat16()
    w.requires_grad_(True)
    tokens = torch.tensor([v - 1, v - 2, v - 1], device=DEV)
    out = ops.embedding(tokens, w, 2.0)
    assert torch.equal(out, (w.detach()[tokens].float() * 2).bfloat16())
    dout = torch.randn(3, h, device=DEV).bfloat16()
    grad = torch.autograd.grad(out, w, dout)[0]
    assert torch.equal(grad[-2], (dout[1].float() * 2).bfloat16())
    assert torch.equal(grad[-1], ((dout[0].float() + dout[2].float()) * 2).bfloat16())
    assert not grad[:-2].any()
    del grad, out
    x = w.detach().flatten()
    x.fill_(1.0)
    y = ops.dropout(x, 0.25, 3)
    last = y[-2 ** 20 - 5:]
    kept = last != 0
    assert torch.equal(last[kept], torch.full_like(last[kept], 4 / 3))
    assert abs(kept.float().mean().item() - 0.75) < 6 * (0.25 * 0.75 / 2 ** 20) ** 0.5
    del x, y, w
    torch.cuda.empty_cache()
