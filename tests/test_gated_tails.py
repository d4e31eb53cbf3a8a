"""The gated unit's activations and their derivatives relative to their own
size, also where they are small: act(g) U with U = 2^k, which carries the
tails into the range of 16 bits.

Bounds. g reaches the activation exactly (one product with 1). E = 2^-24, e
half a step of the type. An exponential multiplies the errors of its argument
by the argument: for exp(-z) those are 2 E (log2 e and its product), and what
z itself is off by; each of the few operations around it adds E or 2 E. Where
exp(z) passes 2^126 its reciprocal, s, is below the smallest normal number of
32 bits and may be 0: off by 2^-126 before g, and then U, multiply it.
"""

import math

import pytest
import torch

from distributed_vgg_f_amd import ops

gpu = pytest.mark.gpu
DEV = "cuda:0"
E, FLUSH = 2.0 ** -24, 2.0 ** -126
G = torch.arange(-12 * 16, 12 * 16 + 1, dtype=torch.float64) / 16


def exact(act, g):
    """act(g), act'(g) in 64 bits, tails too: 1 + erf would cancel there."""
    if act == "gelu":
        c = torch.special.erfc(-g * math.sqrt(0.5)) / 2
        return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":               # 1 + tanh(z) = 2 sigmoid(2 z)
        c = math.sqrt(8 / math.pi)
        s = torch.sigmoid(c * (g + 0.044715 * g ** 3))
        t = torch.sigmoid(-c * (g + 0.044715 * g ** 3))
        return g * s, s + g * s * t * c * (1 + 0.134145 * g * g)
    if act == "relu":
        return g.clamp(min=0), (g > 0).double()
    s, t = torch.sigmoid(g), torch.sigmoid(-g)
    return (s, s * t) if act == "sigmoid" else (g * s, s * (1 + g * t))


def errors(act, g):
    """How far act(g) and act'(g) may be off."""
    a, s = g.abs(), torch.sigmoid(g)
    if act == "relu":
        return 0 * a, 0 * a
    if act == "gelu":
        # x: 2 E (constant, product), x^2: 5 E, its exponent 7 E g^2 / 2
        rel = (3.5 * g * g + 32) * E
        phi = torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        c = torch.special.erfc(-g * math.sqrt(0.5)) / 2
        return (rel * c + FLUSH) * a, rel * (c + a * phi) + FLUSH
    if act == "gelu_tanh":
        # z = c (g + c3 g^3): 6 E
        z = math.sqrt(8 / math.pi) * (a + 0.044715 * a ** 3)
        rel, s = (8 * z + 16) * E, torch.sigmoid(torch.copysign(z, g))
        dz = math.sqrt(8 / math.pi) * (1 + 0.134145 * g * g)
        return (rel * s + FLUSH) * a, \
            2 * rel * (s + a * s * (1 - s) * dz) + \
            (4 * E * s + FLUSH) * (1 + a * dz)
    rel = (2 * a + 8) * E
    if act == "sigmoid":
        return rel * s + FLUSH, 2 * rel * s * (1 - s) + FLUSH
    return (rel * s + FLUSH) * a, 2 * rel * (s + a * s * (1 - s)) + \
        (4 * E * s + FLUSH) * (1 + a)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu",
                                 "sigmoid"])
def test_values_and_derivatives(act, dtype):
    e = torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).smallest_normal * e
    value, slope = exact(act, G)
    off_value, off_slope = errors(act, G)
    scale = 2.0 ** torch.arange(16, dtype=torch.float64)        # U

    x = G.to(dtype).view(-1, 1)
    assert torch.equal(x.double().view(-1), G)
    one = torch.ones(1, 16, dtype=dtype)
    x, one, up = x.to(DEV), one.to(DEV), scale.to(dtype).to(DEV)
    x.requires_grad_()
    h = ops.gated_linear(x, one, 0 * one, 0 * up, up, act=act)

    want = value.view(-1, 1) * scale
    off = (h.detach().cpu().double() - want).abs()
    err = (1 + e) * (off_value.view(-1, 1) * scale + E * want.abs()) + \
        e * want.abs() + least
    bad = ~(off <= err)
    bad[want.abs() > 60000] = False                  # past fp16
    assert not bool(bad.any()), G[bad.any(1)].tolist()

    # act' of a row through the column that brings it near 2^8
    k = (8 - torch.log2(slope.abs().clamp(min=1e-30))).round().clamp(0, 15)
    dh = torch.zeros(len(G), 16, dtype=dtype)
    dh[torch.arange(len(G)), k.long()] = 1
    dx, = torch.autograd.grad(h, x, dh.to(DEV))
    want = slope * 2.0 ** k
    off = (dx.cpu().double().view(-1) - want).abs()
    err = (1 + 2 * e) * (off_slope * 2.0 ** k + 4 * E * want.abs()) + \
        (2 * e + e * e) * want.abs() + 2 * least * 2.0 ** k
    if act == "relu":
        err[G == 0] = 2.0 ** 15                     # either side of the border
    bad = ~(off <= err)
    assert not bool(bad.any()), G[bad].tolist()


@gpu
def test_infinite_gates():
    inf, nan = float("inf"), float("nan")
    b = torch.tensor([inf, -inf, nan, 1e4, -1e4], dtype=torch.bfloat16)
    x, w = torch.ones(20, 1), torch.zeros(1, 5)
    ts = [t.bfloat16().to(DEV) for t in (x, w, w, b, torch.full((5,), 2.0))]

    def run(act):
        leaf = ts[3].detach().requires_grad_()
        h = ops.gated_linear(*ts[:3], leaf, ts[4], act=act)
        db, = torch.autograd.grad(h, leaf, torch.ones_like(h))
        return h.detach()[0].cpu().float(), db.cpu().float()
    h, db = run("sigmoid")
    assert h[[0, 1, 3, 4]].tolist() == [2, 0, 2, 0]
    assert db[[0, 1, 3, 4]].tolist() == [0, 0, 0, 0]
    h, db = run("relu")
    assert h[:2].tolist() == [inf, 0] and db[[0, 1, 3, 4]].tolist() == [40, 0,
                                                                       40, 0]
    for act in ("silu", "gelu", "gelu_tanh", "relu", "sigmoid"):
        h, db = run(act)
        assert math.isnan(h[2])
        assert act == "relu" or math.isnan(db[2])
        if act not in ("sigmoid", "relu"):        # g and 0, and slopes 1 and 0
            assert h[0] == inf and h[3:].tolist() == [2 * float(b[3]), 0]
            assert db[3:].tolist() == [40, 0]
