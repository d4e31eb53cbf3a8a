"""Dropout whose mask is drawn again instead of stored, against the generator
written out in whole numbers of 64 bits."""

import numpy as np
import pytest
import torch

from distributed_vgg_f_amd import ops
from distributed_vgg_f_amd.models.layers import Dropout

gpu = pytest.mark.gpu
DEV = "cuda:0"
U = np.uint64


def philox_words(n, seed, offset):
    """Words 0..n-1: Philox4x32-10, counter (i // 4, offset), key (seed)."""
    low, s32 = U(0xFFFFFFFF), U(32)
    c = np.arange((n + 3) // 4, dtype=np.uint64)
    v = [c & low, c >> s32, np.full_like(c, offset % 2 ** 32),
         np.full_like(c, 0x243F6A88)]
    k0, k1 = seed % 2 ** 32, 0xBB67AE85
    for _ in range(10):
        a, b = v[0] * U(0xD2511F53), v[2] * U(0xCD9E8D57)
        v = [(b >> s32) ^ v[1] ^ U(k0), b & low,
             (a >> s32) ^ v[3] ^ U(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return np.stack(v, 1).reshape(-1)[:n]


def keep_mask(shape, p, seed, offset):
    n = int(np.prod(shape))
    unit = philox_words(n, seed, offset).astype(np.float32) * \
        np.float32(2.0 ** -32)
    return torch.from_numpy(unit >= np.float32(p)).view(shape)


def expect(x, p, seed, offset):
    """Oracle in 64 bits."""
    keep = keep_mask(x.shape, p, seed, offset)
    return torch.where(keep, x.double().cpu() / (1 - p), 0.0), keep


def check(got, x, p, seed, offset):
    want, keep = expect(x, p, seed, offset)
    got = got.detach().cpu()
    assert got.dtype == x.dtype and got.shape == x.shape
    assert torch.equal(got[~keep], torch.zeros_like(got[~keep]))
    # scale rounded to 32 bits, the product rounded to 32 bits, then to the
    # type: half a step each; the subnormal range of fp16 in the last term
    eps = torch.finfo(x.dtype).eps / 2
    e32 = 2.0 ** -24
    tol = ((1 + eps) * (1 + e32) ** 2 - 1) * want.abs() + \
        torch.finfo(x.dtype).smallest_normal * eps
    assert bool(((got.double() - want).abs() <= tol).all())


# -------------------------------------------------------------------- CPU
@pytest.mark.parametrize("p", [1.5, float("nan"), float("inf")])
def test_p_refused(p):
    with pytest.raises(ValueError, match="p must not be above 1"):
        ops.dropout(torch.ones(4), p)


@pytest.mark.parametrize("p", [0.0, -0.5])
def test_p_zero_is_identity(p):
    x = torch.ones(4)
    assert ops.dropout(x, p) is x


def test_p_one_is_zero_with_zero_gradient():
    x = torch.tensor([1.0, float("inf"), float("nan")], requires_grad=True)
    y = ops.dropout(x, 1.0)
    y.sum().backward()
    assert torch.equal(y.detach(), torch.zeros(3))
    assert torch.equal(x.grad, torch.zeros(3))


def test_cpu_given_mask():
    x = torch.arange(1.0, 5.0)
    m = torch.tensor([1.0, 0.0, 0.0, 1.0])
    assert torch.equal(ops.dropout(x, 0.5, mask=m),
                       torch.tensor([2.0, 0.0, 0.0, 8.0]))


def test_oracle_is_philox():
    # the published generator's answer for an all-zero counter and key, from
    # the oracle's own round with its constants put to zero
    low, s32 = U(0xFFFFFFFF), U(32)
    v, k0, k1 = [U(0)] * 4, 0, 0
    for _ in range(10):
        a, b = v[0] * U(0xD2511F53), v[2] * U(0xCD9E8D57)
        v = [(b >> s32) ^ v[1] ^ U(k0), b & low,
             (a >> s32) ^ v[3] ^ U(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    assert [int(w) for w in v] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c,
                                   0x9b00dbd8]


# -------------------------------------------------------------------- GPU
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (7,), (8,), (9,),
                                   (257, 33), (5, 1, 13, 64), (2051, 1024)])
def test_values(shape, dtype):
    torch.manual_seed(0)
    x = (torch.randn(shape) * 3).to(dtype).to(DEV).requires_grad_()
    dy = torch.randn(shape).to(dtype).to(DEV)
    for p, seed, offset in [(0.5, 3, 0), (0.1, 2 ** 32 + 5, 2 ** 33 + 7),
                            (0.9, -1, -2)]:
        y = ops.dropout(x, p, seed, offset)
        dx, = torch.autograd.grad(y, x, dy)
        check(y, x.detach().cpu(), p, seed, offset)
        check(dx, dy.cpu(), p, seed, offset)


@gpu
def test_same_mask_as_the_stored_form():
    from distributed_vgg_f_amd.ops import native
    x = torch.randn(1003, 77).bfloat16().to(DEV)
    y, mask = native.ext().dropout_fwd(x, 0.3, 1234, 7)
    assert torch.equal(ops.dropout(x, 0.3, 1234, 7), y)


@gpu
@pytest.mark.parametrize("p", [1e-9, 2.0 ** -33, 1 - 2.0 ** -25, 0.999999])
def test_p_near_the_ends(p):
    x = torch.ones(100000, device=DEV)
    y = ops.dropout(x, p, 11, 2)
    keep = keep_mask((100000,), p, 11, 2)
    assert torch.equal(y.cpu() != 0, keep)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    torch.manual_seed(1)
    base = torch.randn(67, 130).to(dtype).to(DEV)
    for x in (base.t(), base[:, 1:], base[::2, 3:100:3],
              base.view(-1)[1:], base[:1].expand(9, 130)):
        check(ops.dropout(x, 0.25, 5, 6), x.cpu(), 0.25, 5, 6)


@gpu
def test_dropped_infinities_are_zero():
    x = torch.full((4096,), float("inf"), device=DEV)
    x[::2] = float("nan")
    y = ops.dropout(x, 0.5, 1, 1).cpu()
    keep = keep_mask((4096,), 0.5, 1, 1)
    assert torch.equal(y[~keep], torch.zeros(int((~keep).sum())))
    assert not bool(torch.isfinite(y[keep]).any())


@gpu
def test_empty_and_expanded_gradient():
    x = torch.empty(0, 7, device=DEV, requires_grad=True)
    y = ops.dropout(x, 0.5, 1, 1)
    y.sum().backward()
    assert y.shape == (0, 7) and x.grad.shape == (0, 7)
    x = torch.ones(5, 9, device=DEV, requires_grad=True)
    ops.dropout(x, 0.5, 1, 1).sum().backward()
    check(x.grad, torch.ones(5, 9), 0.5, 1, 1)


@gpu
def test_gradient_of_the_gradient():
    x = torch.randn(33, device=DEV, requires_grad=True)
    y = ops.dropout(x, 0.5, 1, 1)
    g, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    gg, = torch.autograd.grad(g.sum(), x)
    keep = keep_mask((33,), 0.5, 1, 1)
    assert torch.equal(gg.cpu(), torch.where(keep, 8.0, 0.0))


@gpu
@pytest.mark.parametrize("x,kw,match", [
    (torch.ones(4, dtype=torch.float64), {}, "bf16, fp16 or fp32"),
    (torch.ones(4, dtype=torch.int32), {}, "bf16, fp16 or fp32"),
    (torch.ones(4), {"offset": torch.zeros(1, dtype=torch.int64)},
     "one int64 on x's device"),
    (torch.ones(4), {"offset": "i32"}, "one int64 on x's device"),
    (torch.ones(4), {"offset": "two"}, "one int64 on x's device"),
])
def test_refusals(x, kw, match):
    kw = {k: {"i32": torch.zeros(1, dtype=torch.int32, device=DEV),
              "two": torch.zeros(2, dtype=torch.int64, device=DEV)}.get(v, v)
          if isinstance(v, str) else v for k, v in kw.items()}
    with pytest.raises(RuntimeError, match=match):
        ops.dropout(x.to(DEV), 0.5, **kw)


@gpu
def test_offset_on_the_device_and_replays():
    off = torch.zeros(1, dtype=torch.int64, device=DEV)
    x = torch.randn(1000, 33).bfloat16().to(DEV).requires_grad_()
    dy = torch.randn(1000, 33).bfloat16().to(DEV)
    # counted up between forward and backward: both use the forward's
    off.fill_(5)
    y = ops.dropout(x, 0.5, 9, off)
    off.fill_(6)
    dx, = torch.autograd.grad(y, x, dy)
    check(y, x.detach().cpu(), 0.5, 9, 5)
    check(dx, dy.cpu(), 0.5, 9, 5)
    del y, dx

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(ops.dropout(x, 0.5, 9, off), x, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        off.add_(1)
        y = ops.dropout(x, 0.5, 9, off)
        dx, = torch.autograd.grad(y, x, dy)
    off.fill_(100)
    for replay in range(1, 5):
        graph.replay()
        torch.cuda.synchronize()
        check(y, x.detach().cpu(), 0.5, 9, 100 + replay)
        check(dx, dy.cpu(), 0.5, 9, 100 + replay)
        eager = ops.dropout(x.detach(), 0.5, 9, 100 + replay)
        assert torch.equal(eager, y.detach())


@gpu
def test_another_stream():
    x = torch.randn(1 << 20, device=DEV, requires_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.dropout(x, 0.5, 2, 3)
        y.backward(torch.ones_like(y))
    torch.cuda.current_stream().wait_stream(side)
    check(y, x.detach().cpu(), 0.5, 2, 3)
    check(x.grad, torch.ones(1 << 20), 0.5, 2, 3)


@gpu
def test_long_tensor_draws_by_the_flat_index():
    n = 2 ** 31 + 4099                   # counters far beyond the first ones
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = ops.dropout(x, 0.5, 4, 4)
    del x
    for begin in (0, 2 ** 30 + 4, 2 ** 31 - 4096, n - 4099):
        size = min(4099, n - begin)
        low = U(0xFFFFFFFF)
        first = begin // 4
        # the oracle's counters start at 0: shift them by the block's number
        c = np.arange(first, first + (size + 3) // 4, dtype=np.uint64)
        v = [c & low, c >> U(32), np.full_like(c, 4),
             np.full_like(c, 0x243F6A88)]
        k0, k1 = 4, 0xBB67AE85
        for _ in range(10):
            a, b = v[0] * U(0xD2511F53), v[2] * U(0xCD9E8D57)
            v = [(b >> U(32)) ^ v[1] ^ U(k0), b & low,
                 (a >> U(32)) ^ v[3] ^ U(k1), a & low]
            k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
        words = np.stack(v, 1).reshape(-1)[:size]
        keep = torch.from_numpy(
            words.astype(np.float32) * np.float32(2.0 ** -32) >= 0.5)
        assert torch.equal(y[begin:begin + size].cpu() != 0, keep)


@gpu
def test_layer_draws_a_new_mask_at_each_call():
    layer = Dropout(0.5, seed=3)
    x = torch.ones(64, 64, dtype=torch.bfloat16, device=DEV)
    a, b = layer(x), layer(x)
    check(a, x.cpu(), 0.5, 3, 1)
    check(b, x.cpu(), 0.5, 3, 2)
    layer.eval()
    assert layer(x) is x


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_value_of_16_bits(dtype):
    # subnormal numbers, infinities and NaN among them, and products that
    # overflow or fall into the subnormal range
    bits = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16)
    x = bits.view(dtype).to(DEV)
    for p in (0.5, 0.3, 0.999):
        y = ops.dropout(x, p, 1, 1).cpu()
        keep = keep_mask(x.shape, p, 1, 1)
        scale = torch.tensor(1 / (1 - p), dtype=torch.float32)
        want = torch.where(keep, x.cpu().float() * scale, 0.0).to(dtype)
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(y), nan)
        assert torch.equal(y[~nan].view(torch.int16),
                           want[~nan].view(torch.int16))
