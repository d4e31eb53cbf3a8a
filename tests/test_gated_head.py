"""VGG heads with gated hidden layers: the unit inside a model, its optimizer
and its checkpoints."""

import pytest
import torch

from distributed_vgg_f_amd import ops
from distributed_vgg_f_amd.config import Config
from distributed_vgg_f_amd.engine import checkpoint as ckpt
from distributed_vgg_f_amd.engine.arena import ArenaOptimizer
from distributed_vgg_f_amd.engine.trainer import Trainer
from distributed_vgg_f_amd.models import build_model
from distributed_vgg_f_amd.models.layers import Dropout, GatedLinear, Linear

gpu = pytest.mark.gpu


def small(**kw):
    return Config(**{"model": "vggf", "image_size": 64, "batch_size": 2,
                     "num_classes": 16, "log_every": 0, "seed": 3, **kw})


def test_default_head_is_linear():
    m = build_model(small())
    assert type(m.fc6) is Linear and type(m.fc7) is Linear


@pytest.mark.parametrize("name", ["vggf", "vgg16"])
def test_gated_head(name):
    m = build_model(small(model=name, fc_gate="gelu"))
    assert type(m.fc6) is GatedLinear and m.fc7.act == "gelu"
    plain = build_model(small(model=name))
    count = [sum(p.numel() for p in x.parameters()) for x in (m, plain)]
    k6 = m.fc6.weight_gate.shape[0]
    assert count[0] - count[1] == (k6 + 1 + 4096 + 1) * 4096
    x = torch.randn(2, 64, 64, 3)
    m.eval()
    f = m.features(x).reshape(2, -1)
    h = ops.gated_linear(f, m.fc6.weight_gate, m.fc6.weight_up,
                         m.fc6.bias_gate, m.fc6.bias_up, act="gelu")
    h = ops.gated_linear(h, m.fc7.weight_gate, m.fc7.weight_up,
                         m.fc7.bias_gate, m.fc7.bias_up, act="gelu")
    assert torch.equal(m(x), m.fc8(h))


def test_unknown_activation_is_refused():
    with pytest.raises(ValueError, match="unknown activation"):
        build_model(small(fc_gate="tanh"))


def test_a_model_without_hidden_layers_refuses_a_gate():
    with pytest.raises(ValueError, match="no hidden fully connected"):
        build_model(small(model="resnet50", fc_gate="silu"))


def test_layer_with_its_dropout():
    torch.manual_seed(0)
    layer, drop = GatedLinear(6, 8, "silu"), Dropout(0.5, seed=4)
    x = torch.randn(5, 6)
    got = layer(x, drop)
    assert drop._calls == 1
    want = ops.dropout(layer(x), 0.5, 4, 1)
    assert torch.equal(got, want)
    drop.eval()
    assert torch.equal(layer(x, drop), layer(x)) and drop._calls == 1


def test_cpu_training_and_checkpoint(tmp_path):
    cfg = small(fc_gate="silu", dropout=0.5, checkpoint_dir=str(tmp_path))
    t = Trainer(cfg, device=torch.device("cpu"))
    before = t.arena.w32.clone()
    t.train(2)
    assert bool(torch.isfinite(t.arena.w32).all())
    for name, w in t.arena.named_master():
        if "fc6" in name and "weight" in name:
            slot = [s for s in t.arena.slots if s.name == name][0]
            old = before[slot.offset:slot.offset + slot.numel]
            assert not torch.equal(w.reshape(-1), old), name
    model = build_model(cfg)
    arena = ArenaOptimizer(model, torch.device("cpu"))
    assert ckpt.restore_latest(str(tmp_path), arena, model) == 2
    assert torch.equal(arena.w32, t.arena.w32)
    assert model.drop6._calls == t.model.drop6._calls == 2


def test_command_line_names_the_gate():
    import argparse
    p = argparse.ArgumentParser()
    Config.add_args(p)
    cfg = Config.from_args(p.parse_args(["--fc-gate", "gelu_tanh"]))
    assert cfg.fc_gate == "gelu_tanh"


@gpu
def test_gpu_model_agrees_with_cpu():
    cfg = small(fc_gate="silu", num_classes=1000)
    torch.manual_seed(cfg.seed)
    model = build_model(cfg)
    x = (torch.randn(4, 64, 64, 3) * 0.5).bfloat16()
    ref = model(x.float())
    gm = build_model(cfg)
    gm.load_state_dict(model.state_dict())
    got = gm.to("cuda:0").bfloat16()(x.to("cuda:0")).float().cpu()
    cos = torch.nn.functional.cosine_similarity(got.flatten(), ref.flatten(),
                                                dim=0)
    # 8 layers of roundings of at most 2^-8 each, in and between them
    assert float(cos.detach()) > 0.99


@gpu
def test_gpu_gradients_land_in_the_arena():
    t = Trainer(small(fc_gate="silu", dropout=0.5),
                device=torch.device("cuda", 0))
    for _ in range(2):
        assert bool(torch.isfinite(t.train_step()))
    for s in t.arena.slots:
        g = s.param.grad
        assert g.data_ptr() == s.param._dvgg_gbuf.data_ptr(), s.name
        assert bool(g.float().abs().sum() > 0), s.name


@gpu
def test_gradient_buffer_of_another_type():
    """An arena of 32-bit gradients gets the same values."""
    model = build_model(small(fc_gate="silu"))
    ArenaOptimizer(model, torch.device("cuda", 0), torch.bfloat16,
                   torch.float32)
    fc = model.fc6
    x = torch.randn(4, fc.weight_gate.shape[0], device="cuda:0",
                    dtype=torch.bfloat16)
    dh = torch.randn(4, 4096, device="cuda:0", dtype=torch.bfloat16)
    fc(x).backward(dh)
    own = [t.detach().clone().requires_grad_()
           for t in (fc.weight_gate, fc.weight_up, fc.bias_gate, fc.bias_up)]
    want = torch.autograd.grad(ops.gated_linear(x, *own, act="silu"), own, dh)
    for p, g in zip((fc.weight_gate, fc.weight_up, fc.bias_gate, fc.bias_up),
                    want):
        assert torch.equal(p._dvgg_gbuf, g.float())


@gpu
def test_gpu_step_in_a_graph():
    """That it runs: the unit's replays are compared with eager calls in
    test_gated.py (a batch of 2 leaves the numbers at the default rate,
    replayed or not)."""
    t = Trainer(small(fc_gate="gelu", use_graph=True, lr=0.001),
                device=torch.device("cuda", 0))
    assert t._graph
    for _ in range(6):
        assert bool(torch.isfinite(t.train_step().detach()))
