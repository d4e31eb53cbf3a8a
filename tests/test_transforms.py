"""Dropout and the gated unit under what torch does around an operator:
recording a call and replaying it, function transforms."""

import io

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from distributed_vgg_f_amd import ops
from distributed_vgg_f_amd.models.layers import Dropout, hidden_fc, run_hidden

gpu = pytest.mark.gpu
DEV = "cuda:0"


def operands(m, k=40, n=48, bias=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    shapes = [(m, k), (k, n), (k, n)] + [(n,), (n,)] * bias
    return [(torch.randn(s, generator=gen) * 0.3).bfloat16().to(DEV)
            for s in shapes]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_traced_dropout(dtype):
    def f(x):
        return ops.dropout(x, 0.5, 3, 1)
    traced = torch.jit.trace(f, torch.randn(64, 33, device=DEV).to(dtype))
    for rows in (64, 7, 129):
        x = torch.randn(rows, 33, device=DEV).to(dtype).requires_grad_()
        dy = torch.randn(rows, 33, device=DEV).to(dtype)
        y, want = traced(x), f(x)
        assert torch.equal(y, want)
        assert torch.equal(torch.autograd.grad(y, x, dy)[0],
                           torch.autograd.grad(want, x, dy)[0])


@gpu
def test_traced_dropout_reads_the_offset_of_its_call():
    traced = torch.jit.trace(lambda x, o: ops.dropout(x, 0.5, 3, o),
                             (torch.ones(1000, device=DEV),
                              torch.zeros(1, dtype=torch.int64, device=DEV)))
    x = torch.randn(1000, device=DEV)
    for offset in (4, 5, 6):
        o = torch.full((1,), offset, device=DEV)
        assert torch.equal(traced(x, o), ops.dropout(x, 0.5, 3, offset))


@gpu
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_traced_gated_unit(bias, p):
    def f(*ts):
        return ops.gated_linear(*ts, act="gelu", p=p, seed=2, offset=5)
    traced = torch.jit.trace(f, tuple(operands(20, bias=bias)))
    for m in (20, 3, 70):
        ts = operands(m, bias=bias, seed=m)
        with torch.no_grad():
            assert torch.equal(traced(*ts), f(*ts))
        ts = [t.requires_grad_() for t in ts]
        h, want = traced(*ts), f(*ts)
        assert torch.equal(h, want)
        dh = torch.randn_like(h)
        for a, b in zip(torch.autograd.grad(h, ts, dh),
                        torch.autograd.grad(want, ts, dh)):
            assert torch.equal(a, b)


class Head(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.fc6, self.fc7 = hidden_fc(256, 96, "silu"), hidden_fc(96, 40,
                                                                   "gelu")
        self.drop6, self.drop7 = Dropout(0.5, 1), Dropout(0.5, 2)

    def forward(self, x):
        return run_hidden(self.fc7, self.drop7,
                          run_hidden(self.fc6, self.drop6, x))


@gpu
def test_traced_head():
    torch.manual_seed(0)
    head = Head().to(DEV).bfloat16().eval()
    x = [torch.randn(m, 256, device=DEV).bfloat16() for m in (4, 4, 30)]
    with torch.no_grad():
        traced = torch.jit.trace(head, x[0])
        for t in x:
            assert torch.equal(traced(t), head(t))


@gpu
def test_function_transforms_are_refused():
    x, wg, wu = operands(6, bias=False)
    with pytest.raises(RuntimeError, match="no function transforms"):
        torch.func.vmap(lambda t: ops.dropout(t, 0.5, 1, 1))(x)
    with pytest.raises(RuntimeError, match="no function transforms"):
        torch.func.vmap(lambda t: ops.gated_linear(t[None], wg, wu))(x)
    with pytest.raises(RuntimeError, match="no function transforms"):
        torch.func.vmap(lambda w: ops.gated_linear(x, w, wu))(wg[None])
    with pytest.raises(RuntimeError, match="no function transforms"):
        torch.func.grad(lambda t: ops.dropout(t, 0.5, 1, 1).sum())(x.float())


def dual_calls(dev):
    """Calls with one operand that carries a tangent, none with a gradient."""
    ext = ops.native.ext()
    x, w = torch.ones(4, 8, device=dev), torch.ones(8, 8, device=dev)
    half, b = [t.bfloat16() for t in (x, w)], torch.ones(8, device=dev)

    def gated(which):
        ts = [half[0], half[1], half[1].clone(), b.bfloat16(), b.bfloat16()]
        ts[which] = fwAD.make_dual(ts[which], torch.ones_like(ts[which]))
        return ext.gated_linear(*ts, 0, 0.0, 0, 0, None)
    return [lambda: ext.dropout(fwAD.make_dual(x, x), 0.5, 1, 1)] + \
        [lambda i=i: gated(i) for i in range(5)]


@pytest.mark.skipif(not ops.native.available(),
                    reason="needs the built extension")
@pytest.mark.parametrize("which", range(6))
def test_tangents_are_refused(which):
    # before anything asks for a GPU, so here too
    with fwAD.dual_level(), pytest.raises(NotImplementedError,
                                          match="no forward-mode"):
        dual_calls("cpu")[which]()


@gpu
@pytest.mark.parametrize("which", range(6))
def test_tangents_are_refused_on_the_gpu(which):
    with fwAD.dual_level(), pytest.raises(NotImplementedError,
                                          match="no forward-mode"):
        dual_calls(DEV)[which]()
    x, wg, wu = operands(3, bias=False)
    with fwAD.dual_level(), torch.no_grad(), \
            pytest.raises(NotImplementedError, match="no forward-mode"):
        ops.gated_linear(fwAD.make_dual(x[None], x[None]), wg, wu)


@gpu
def test_tangents_of_a_gradient_are_refused():
    x, wg, wu = [t.requires_grad_() for t in operands(3, bias=False)]
    for y in (ops.dropout(x, 0.5, 1, 1), ops.gated_linear(x, wg, wu)):
        dy = torch.ones_like(y)
        with fwAD.dual_level(), pytest.raises(NotImplementedError,
                                              match="no forward-mode"):
            torch.autograd.grad(y, x, fwAD.make_dual(dy, dy))


@gpu
def test_views_that_negate():
    z = torch.randn(40, 48, dtype=torch.complex64, device=DEV)
    for x in (z.conj().imag, torch._neg_view(z.real.contiguous()),
              torch._neg_view(z.real.bfloat16())):
        assert x.is_neg()
        real = x.clone()
        want = ops.dropout(real, 0.5, 1, 1)
        assert torch.equal(ops.dropout(x, 0.5, 1, 1), want)
        leaf = real.clone().requires_grad_()
        y = ops.dropout(leaf, 0.5, 1, 1)
        dx, = torch.autograd.grad(y, leaf, x)
        assert torch.equal(dx, want)
    ts = operands(5)
    h = ops.gated_linear(*ts)
    for which in range(5):
        neg = list(ts)
        neg[which] = torch._neg_view(-ts[which])
        assert torch.equal(ops.gated_linear(*neg), h)
    leaf = ts[0].clone().requires_grad_()
    dh = torch.randn_like(h)
    got, = torch.autograd.grad(ops.gated_linear(leaf, *ts[1:]), leaf,
                               torch._neg_view(-dh))
    want, = torch.autograd.grad(ops.gated_linear(leaf, *ts[1:]), leaf, dh)
    assert torch.equal(got, want)


def zero_calls(dev):
    ext = ops.native.ext()
    zero = torch._efficientzerotensor((8, 8), dtype=torch.bfloat16, device=dev)
    w = torch.ones(8, 8, dtype=torch.bfloat16, device=dev)
    flat = torch._efficientzerotensor((8,), dtype=torch.bfloat16, device=dev)

    def gated(x=w, g=w, u=w, b=None):
        return ext.gated_linear(x, g, u, b, None, 0, 0.0, 0, 0, None)
    return [lambda: ext.dropout(zero, 0.5, 1, 1), lambda: gated(x=zero),
            lambda: gated(g=zero), lambda: gated(u=zero),
            lambda: gated(b=flat)]


@pytest.mark.skipif(not ops.native.available(),
                    reason="needs the built extension")
@pytest.mark.parametrize("which", range(5))
def test_zeros_without_memory_are_refused(which):
    # on the CPU: the refusal comes before anything is asked of a GPU
    with pytest.raises(RuntimeError, match="zeros without memory"):
        zero_calls("cpu")[which]()


@gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_calls(backend):
    x, wg, wu = operands(6, bias=False)

    def f(t):
        return ops.dropout(ops.gated_linear(t, wg, wu) * 2, 0.5, 1, 1) + 1
    torch._dynamo.reset()
    a, b = [x.clone().requires_grad_() for _ in range(2)]
    y, want = torch.compile(f, backend=backend)(a), f(b)
    assert torch.equal(y, want)
    y.sum().backward()
    want.sum().backward()
    assert torch.equal(a.grad, b.grad)


class Wrapped(torch.Tensor):
    """A tensor type whose memory is another tensor's."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(
            cls, t.shape, dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(str(func))


def freed(t):
    t = t.clone()
    t.untyped_storage().resize_(0)
    return t


@pytest.mark.skipif(not ops.native.available(),
                    reason="needs the built extension")
@pytest.mark.parametrize("make", [Wrapped, freed])
@pytest.mark.parametrize("which", range(8))
def test_tensors_without_memory_are_refused(which, make):
    # on the CPU: the refusal comes before anything is asked of a GPU
    ext = ops.native.ext()
    w, b = torch.ones(8, 8).bfloat16(), torch.ones(8).bfloat16()
    ts = [w, w.clone(), w.clone(), b, b.clone(), torch.zeros(1).long()]
    if which < 6:
        ts[which] = make(ts[which])

    def call():
        if which == 6:
            return ext.dropout(make(w), 0.5, 1, 0)
        if which == 7:
            return ext.dropout(w, 0.5, 1, 0, make(ts[5]))
        return ext.gated_linear(*ts[:5], 0, 0.5, 0, 0, ts[5])
    with pytest.raises(RuntimeError, match="without memory"):
        call()


@gpu
def test_memory_freed_before_the_backward_pass_is_refused():
    x, wg, wu = operands(6, bias=False)
    wg.requires_grad_()
    h = ops.gated_linear(x, wg, wu)
    x.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="without memory"):
        h.backward(torch.ones_like(h))
    x = operands(6, bias=False)[0]
    wg._dvgg_gbuf = torch.empty_like(wg)
    h = ops.gated_linear(x, wg, wu)
    wg._dvgg_gbuf.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="bad gradient buffer"):
        h.backward(torch.ones_like(h))


@gpu
def test_calls_under_autocast():
    x, wg, wu = operands(6, bias=False)
    with torch.autocast("cuda", torch.float16):
        y, h = ops.dropout(x, 0.5, 1, 1), ops.gated_linear(x, wg, wu)
    assert torch.equal(y, ops.dropout(x, 0.5, 1, 1))
    assert torch.equal(h, ops.gated_linear(x, wg, wu))


@gpu
def test_traced_layer_of_an_arena_and_its_saved_form():
    from distributed_vgg_f_amd.engine.arena import ArenaOptimizer
    layer = hidden_fc(64, 40, "silu")
    ArenaOptimizer(layer, torch.device(DEV))
    x, dh = [torch.randn(9, n, device=DEV).bfloat16() for n in (64, 40)]
    traced = torch.jit.trace(layer, x)
    want = layer(x)
    want.backward(dh)
    names = [n for n, _ in layer.named_parameters()]
    grads = {n: p._dvgg_gbuf.clone() for n, p in layer.named_parameters()}
    for p in layer.parameters():
        p.grad = None
        p._dvgg_gbuf.zero_()
    h = traced(x)
    assert torch.equal(h, want)
    h.backward(dh)
    for n, p in layer.named_parameters():
        assert torch.equal(p.grad, grads[n]), n
        assert p.grad.data_ptr() == p._dvgg_gbuf.data_ptr(), n
    assert len(names) == 4

    file = io.BytesIO()
    torch.jit.save(traced, file)
    file.seek(0)
    assert torch.equal(torch.jit.load(file)(x), want)
