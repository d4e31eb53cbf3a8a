"""A gated head draws its dropout in the unit's kernel. What is attached to
either layer must not notice."""

import pytest
import torch
import torch.nn as nn

from distributed_vgg_f_amd import ops
from distributed_vgg_f_amd.models.layers import (Dropout, GatedLinear, Linear,
                                                 run_hidden)


def layers(seed=4):
    torch.manual_seed(0)
    return GatedLinear(6, 8, "silu"), Dropout(0.5, seed), torch.randn(5, 6)


def calls_of_the_unit(monkeypatch):
    """p of each ops.gated_linear from here on: 0 where dropout is apart."""
    seen, real = [], ops.gated_linear

    def gated_linear(*a, **kw):
        seen.append(kw.get("p", 0.0))
        return real(*a, **kw)
    monkeypatch.setattr(ops, "gated_linear", gated_linear)
    return seen


def test_plain_layers_are_one_call(monkeypatch):
    fc, drop, x = layers()
    seen = calls_of_the_unit(monkeypatch)
    run_hidden(fc, drop, x)
    assert seen == [0.5]


def test_hooks_of_the_dropout_run():
    fc, drop, x = layers()
    got = []
    drop.register_forward_pre_hook(lambda m, a: got.append(a[0].detach()))
    drop.register_forward_hook(lambda m, a, y: got.append(y.detach()))
    y = run_hidden(fc, drop, x)
    h = fc(x)
    assert torch.equal(got[0], h.detach())
    assert torch.equal(got[1], y.detach())
    assert torch.equal(y, ops.dropout(h, 0.5, 4, 1)) and drop._calls == 1
    drop.eval()
    run_hidden(fc, drop, x)
    assert len(got) == 4


def test_a_hook_of_the_dropout_changes_its_result():
    fc, drop, x = layers()
    handle = drop.register_forward_hook(lambda m, a, y: y + 1)
    assert torch.equal(run_hidden(fc, drop, x),
                       ops.dropout(fc(x), 0.5, 4, 1) + 1)
    assert torch.equal(fc(x, drop), ops.dropout(fc(x), 0.5, 4, 2) + 1)
    handle.remove()
    assert torch.equal(run_hidden(fc, drop, x),
                       ops.dropout(fc(x), 0.5, 4, 3))


def test_gradient_hooks_of_the_dropout_run():
    fc, drop, x = layers()
    got = []
    drop.register_full_backward_hook(lambda m, gi, go: got.append(go[0]))
    drop.register_full_backward_pre_hook(lambda m, go: got.append(go[0]))
    run_hidden(fc, drop, x).sum().backward()
    assert len(got) == 2 and all(torch.equal(g, torch.ones(5, 8))
                                 for g in got)


def test_hooks_of_the_unit_see_what_it_computes():
    fc, drop, x = layers()
    got = []
    fc.register_forward_hook(lambda m, a, y: got.append((a, y.detach())))
    run_hidden(fc, drop, x)
    (args, y), = got
    assert len(args) == 1 and args[0] is x
    with torch.no_grad():
        assert torch.equal(y, ops.gated_linear(
            x, fc.weight_gate, fc.weight_up, fc.bias_gate, fc.bias_up))


def test_hooks_of_all_modules_run():
    fc, drop, x = layers()
    got = []
    handle = nn.modules.module.register_module_forward_hook(
        lambda m, a, y: got.append(type(m)))
    try:
        run_hidden(fc, drop, x)
    finally:
        handle.remove()
    assert got == [GatedLinear, Dropout]


class Doubled(Dropout):
    def forward(self, x):
        return 2 * x


@pytest.mark.parametrize("other", [nn.Identity(), nn.Dropout(0.0),
                                   Doubled(0.5)])
def test_another_layer_in_the_place_of_the_dropout(other):
    fc, _, x = layers()
    h = fc(x)
    want = 2 * h if type(other) is Doubled else h
    assert torch.equal(run_hidden(fc, other, x), want)
    assert torch.equal(fc(x, other), want)


def test_a_replaced_forward_runs():
    fc, drop, x = layers()
    drop.forward = lambda x: x - 1
    assert torch.equal(run_hidden(fc, drop, x), fc(x) - 1)
    fc.forward = lambda x: x[:, :1]
    assert torch.equal(run_hidden(fc, drop, x), x[:, :1] - 1)


def test_linear_head_as_before():
    _, drop, x = layers()
    fc = Linear(6, 8, relu=True)
    assert torch.equal(run_hidden(fc, drop, x),
                       ops.dropout(fc(x), 0.5, 4, 1))
