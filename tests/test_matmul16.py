"""Batched 16-bit matrix products on the GPU never hand the library a transposed view as their right operand, in the
forward and in both directions of the backward (zoo.ops.bmm.matmul and its callers). The rule is tested on the CPU, with
the test for "16 bits on the GPU" widened to the CPU, by looking at every product that is dispatched."""
import importlib

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

bmm_module = importlib.import_module("zoo.ops.bmm")
attention_module = importlib.import_module("zoo.ops.attention")
BF, HF = torch.bfloat16, torch.float16


class Products(TorchDispatchMode):
    """Counts batched products, and those of a right operand whose rows are not contiguous."""

    def __init__(self):
        super().__init__()
        self.all, self.transposed = 0, 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func in (torch.ops.aten.bmm.default, torch.ops.aten.baddbmm.default):
            b = args[-1]
            self.all += 1
            self.transposed += b.numel() > 0 and b.dtype in (BF, HF) and not (b.stride(-1) == 1 and b.stride(-2) >= b.size(-1))
        return func(*args, **(kwargs or {}))


@pytest.fixture
def as_on_gpu(monkeypatch):
    monkeypatch.setattr(bmm_module, "_right_in_rows", lambda t: t.dtype in (BF, HF))


SHAPES = [
    ((4, 5, 7), (4, 7, 3), False, False), ((4, 5, 7), (4, 7, 3), True, True), ((2, 3, 5, 7), (2, 3, 7, 4), False, True),
    ((2, 3, 5, 7), (1, 7, 4), True, False), ((3, 1, 5, 7), (2, 7, 1), False, True), ((5, 7), (4, 7, 3), True, True),
    ((4, 5, 7), (7, 3), True, True), ((4, 1, 7), (4, 7, 1), False, True), ((0, 5, 7), (0, 7, 3), False, True),
    ((4, 5, 1), (4, 1, 3), True, True),
]


@pytest.mark.parametrize("dtype", [BF, HF, torch.float32, torch.float64])
@pytest.mark.parametrize("sa,sb,ta,tb", SHAPES)
def test_products_and_their_gradients(as_on_gpu, sa, sb, ta, tb, dtype):
    def leaf(shape, t):
        x = torch.randn(*shape[:-2], *((shape[-1], shape[-2]) if t else shape[-2:])).to(dtype)
        return x.requires_grad_(), (lambda y: y.transpose(-1, -2) if t else y)
    (a, fa), (b, fb) = leaf(sa, ta), leaf(sb, tb)
    with Products() as seen:
        c = bmm_module.matmul(fa(a), fb(b))
        do = torch.randn(c.shape).to(dtype).requires_grad_()
        da, db = torch.autograd.grad(c, (a, b), do, create_graph=True)
        dd, = torch.autograd.grad((da.double() ** 2).sum() + (db.double() ** 2).sum(), do)
    assert seen.transposed == 0
    x, y = a.detach().double().requires_grad_(), b.detach().double().requires_grad_()
    z = do.detach().double().requires_grad_()
    want = torch.matmul(fa(x), fb(y))
    wa, wb = torch.autograd.grad(want, (x, y), z, create_graph=True)
    wd, = torch.autograd.grad((wa ** 2).sum() + (wb ** 2).sum(), z)
    # one rounding per output over sums of float32 (at most 24 terms); gradients of broadcast operands are sums of up to 6
    # such, of the second order of two that were rounded themselves: four half steps of the largest
    eps = torch.finfo(dtype).eps
    for got, ref in ((c, want), (da, wa), (db, wb), (dd, wd)):
        assert got.dtype == dtype and got.shape == ref.shape
        if ref.numel():
            assert (got.double() - ref).abs().max() <= 4 * eps * ref.abs().max() * (1 if dtype != torch.float32 else 8)


def test_one_dimension_is_left_to_torch(as_on_gpu):
    a, b, v = torch.randn(3, 4, 5).to(BF), torch.randn(5, 6).to(BF), torch.randn(5).to(BF)
    assert torch.equal(bmm_module.matmul(a, v), torch.matmul(a, v))
    assert torch.equal(bmm_module.matmul(v, b), torch.matmul(v, b))
    assert torch.equal(bmm_module.matmul(a, b), torch.matmul(a, b))
    with pytest.raises(RuntimeError):
        bmm_module.matmul(a, b[:3])


@pytest.mark.parametrize("sa,sb", [((4, 5, 0), (0, 3)), ((4, 5, 0), (4, 0, 3)), ((0, 5, 7), (7, 3)), ((4, 0, 7), (7, 0))])
def test_nothing_to_sum_or_to_return(as_on_gpu, sa, sb):
    a, b = torch.ones(sa).to(BF).requires_grad_(), torch.ones(sb).to(BF).requires_grad_()
    c = bmm_module.matmul(a, b)
    assert torch.equal(c, torch.matmul(a, b)) and not c.any()
    c.sum().backward()
    assert a.grad.shape == a.shape and b.grad.shape == b.shape


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal,mask", [(True, None), (False, (2, 1, 5, 7)), (False, (1, 3, 1, 7))])
def test_plain_attention_forms_no_such_product(as_on_gpu, dtype, causal, mask):
    q, k, v = (torch.randn(2, n, 3, 16).to(dtype).transpose(1, 2).requires_grad_() for n in (5, 7, 7))
    m = None if mask is None else torch.randn(mask)
    with Products() as seen:
        o = attention_module.attention(q, k, v, mask=m, causal=causal)
        o.sum().backward()
    assert seen.all == 6 and seen.transposed == 0
    assert all(t.grad is not None and torch.isfinite(t.grad.float()).all() for t in (q, k, v))


def test_32_bits_take_no_copies(monkeypatch):
    called = []
    monkeypatch.setattr(bmm_module, "_rows", lambda t: called.append(t) or t.contiguous())
    q = torch.randn(2, 3, 5, 16)
    attention_module.attention(q, q, q, causal=True)
    assert not called


def test_loaders_and_layers_form_no_such_product(as_on_gpu):
    from zoo.pipeline.api.keras.layers import LocallyConnected1D, LocallyConnected2D
    from zoo.pipeline.api.net import tf_graph
    from zoo.pipeline.api.onnx import onnx_loader

    class Node:
        def __init__(self, **attr):
            self.attr = attr
    x, w = torch.randn(3, 5, 7).to(BF), torch.randn(3, 4, 7).to(BF)
    with Products() as seen:
        y = tf_graph._batch_matmul(None, Node(adj_x=False, adj_y=True), x, w)
        z = tf_graph._matmul(None, Node(transpose_b=True), x, w)
        u, = [onnx_loader._OPS["MatMul"]([x, w.transpose(1, 2)], {})]
        l1 = LocallyConnected1D(4, 3, input_shape=(8, 5))
        l1.build((None, 8, 5))
        l2 = LocallyConnected2D(4, 2, 2, input_shape=(3, 6, 5))
        l2.build((None, 3, 6, 5))
        a, b = torch.randn(2, 8, 5).to(BF).requires_grad_(), torch.randn(2, 3, 6, 5).to(BF).requires_grad_()
        ya, yb = l1.call(a), l2.call(b)
        (ya.float().sum() + yb.float().sum()).backward()
    assert seen.all >= 9 and seen.transposed == 0
    want = torch.matmul(x.float(), w.float().transpose(1, 2))
    for got in (y, z, u):
        assert (got.float() - want).abs().max() <= 2.0 ** -8 * want.abs().max()
    assert a.grad.shape == a.shape and b.grad.shape == b.shape
    # the locally connected layers against their definition
    win = a.detach().float().unfold(1, 3, 1).permute(0, 1, 3, 2).reshape(2, 6, -1)
    ref = (win[:, :, :, None] * l1.weight.to(BF).float()).sum(2) + l1.bias.to(BF).float()
    assert (ya.float() - ref).abs().max() <= 3 * 2.0 ** -8 * ref.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
def test_plain_attention_gradients_on_the_gpu(gpu, dtype):
    """Head widths and masks that the fused kernel does not take. Against 64 bits on the same inputs: logits, weights, the
    output and three products of the backward are rounded once each, by at most 2^-8 relative in bfloat16, and the logits
    of size up to 4 move the weights by that: (6 + 4) 2^-8 of the norms."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 3, n, 40, generator=g).to(dtype) for n in (9, 33, 33))
    mask = torch.randn(2, 1, 9, 33, generator=g)
    do = torch.randn(2, 3, 9, 40, generator=g).to(dtype)
    out = []
    for dev, dt in (("cpu", torch.float64), ("cuda", dtype)):
        x = [t.to(dev, dt).requires_grad_() for t in (q, k, v)]
        w = torch.matmul(x[0], x[1].transpose(-1, -2)) / 40 ** 0.5 + mask.to(dev, dt) if dev == "cpu" else None
        o = torch.matmul(torch.softmax(w, -1), x[2]) if dev == "cpu" else attention_module.attention(*x, mask=mask.cuda())
        out.append([o] + list(torch.autograd.grad(o, x, do.to(dev, dt))))
    for ref, got in zip(*out):
        assert ((got.double().cpu() - ref).norm() / ref.norm()).item() < 10 * torch.finfo(dtype).eps / 2
