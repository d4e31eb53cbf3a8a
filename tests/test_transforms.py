"""Dropout and the gated unit under what torch does around an operator:
recording a call and replaying it, function transforms."""

import pytest
import torch

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
