"""The gated unit against its formulas in 64 bits.

Bounds. With e = half a step of the operands' type and E = 2^-24, K products
summed in 32 bits are off by at most (K + 4) E times the sum of their
magnitudes (K additions, the product, the bias). Backward works on G and U in
32 bits, rounds dG and dU once (e) and its results once (e); each error is
carried through the formulas by the largest slope of the function that it
passes. The 32-bit activations are off by at most 2^-19
of max(1, |g|): their exponential multiplies its argument's error of E |g|.
"""

import math

import numpy as np
import pytest
import torch

from distributed_vgg_f_amd import ops

from test_dropout import keep_mask

gpu = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24
ACTS = ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]
SLOPE = {"silu": 1.1, "gelu": 1.13, "gelu_tanh": 1.13, "relu": 1.0,
         "sigmoid": 0.25}                        # max |act'|
CURVE = {"silu": 0.5, "gelu": 0.8, "gelu_tanh": 0.83, "relu": 0.0,
         "sigmoid": 0.1}                         # max |act''|


def act64(name, g):
    """act(g), act'(g) in 64 bits."""
    if name == "relu":
        return g.clamp(min=0), (g > 0).double()
    if name == "gelu":
        c = torch.special.ndtr(g)
        return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g ** 3))
        return g * (1 + t) / 2, (1 + t) / 2 + g * (1 - t * t) / 2 * c * (
            1 + 3 * 0.044715 * g * g)
    s = torch.sigmoid(g)
    if name == "sigmoid":
        return s, s * (1 - s)
    return g * s, s * (1 + g * (1 - s))


def oracle(x, wg, wu, bg, bu, dh, act, factor):
    """(h, dx, dwg, dwu, dbg, dbu) and how far the kernels may be off."""
    e = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * e
    x, wg, wu = x.double(), wg.double(), wu.double()
    K, N, M = wg.shape[0], wg.shape[1], x.shape[0]
    bg = torch.zeros(N) if bg is None else bg
    bu = torch.zeros(N) if bu is None else bu
    g, u = x @ wg + bg.double(), x @ wu + bu.double()
    a, da = act64(act, g)
    h = a * u * factor
    ag = (K + 4) * E * (x.abs() @ wg.abs() + bg.double().abs())
    au = (K + 4) * E * (x.abs() @ wu.abs() + bu.double().abs())
    fn = 2.0 ** -19 * g.abs().clamp(min=1)
    slope, curve = SLOPE[act], CURVE[act]
    eh = factor * ((slope * ag + fn) * (u.abs() + au) + a.abs() * au)
    eh = eh * (1 + e) + (e + 4 * E) * h.abs() + tiny
    v = dh.double() * factor
    du, dg = v * a, v * u * da
    edu = v.abs() * (slope * ag + fn)
    step = curve * ag + fn
    if act == "relu":                  # the border may be on the other side
        step = step + (g.abs() <= ag).double()
    edg = v.abs() * (au * (da.abs() + step) + u.abs() * step)
    edu, edg = edu + 4 * E * du.abs(), edg + 4 * E * dg.abs()
    edu2 = edu * (1 + e) + e * du.abs() + tiny       # rounded for products
    edg2 = edg * (1 + e) + e * dg.abs() + tiny
    wga, wua, xa = wg.abs().t(), wu.abs().t(), x.abs().t()
    mg, mu = dg.abs() + edg2, du.abs() + edu2
    outs = [h, dg @ wg.t() + du @ wu.t(), x.t() @ dg, x.t() @ du, dg.sum(0),
            du.sum(0)]
    errs = [eh,
            edg2 @ wga + edu2 @ wua + (2 * N + 4) * E * (mg @ wga + mu @ wua),
            xa @ edg2 + (M + 4) * E * (xa @ mg),
            xa @ edu2 + (M + 4) * E * (xa @ mu),
            edg.sum(0) + (M + 4) * E * mg.sum(0),
            edu.sum(0) + (M + 4) * E * mu.sum(0)]
    for i in range(1, 6):
        errs[i] = errs[i] * (1 + e) + e * outs[i].abs() + tiny
    return outs, errs


NAMES = ["h", "dx", "dw_gate", "dw_up", "dbias_gate", "dbias_up"]


def compare(got, outs, errs, dtype):
    for name, t, want, err in zip(NAMES, got, outs, errs):
        if t is None:
            continue
        t = t.detach().cpu()
        assert t.dtype == dtype and t.shape == want.shape, name
        off = (t.double() - want).abs()
        bad = ~(off <= err)
        assert not bool(bad.any()), \
            f"{name}: {int(bad.sum())} of {bad.numel()} beyond the bound, " \
            f"first at {bad.nonzero()[0].tolist()}"
        # all together: two roundings of at most e each, the second on top
        # of a sum of independent ones, and what 32 bits lose
        if want.numel() >= 256:
            e = torch.finfo(dtype).eps / 2
            assert float(off.square().mean().sqrt()) <= \
                2 * e * float(want.square().mean().sqrt()) + 1e-6, name


def make(M, K, N, dtype, bias, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen) * scale).to(dtype)
    s = 1.5 / math.sqrt(K)
    return (normal(M, K), normal(K, N, scale=s), normal(K, N, scale=s),
            normal(N, scale=0.3) if bias else None,
            normal(N, scale=0.3) if bias else None, normal(M, N, scale=0.5))


def run_all(ts, act, p=0.0, seed=0, offset=0):
    *leaves, dh = [None if t is None else t.detach().to(DEV) for t in ts]
    leaves = [None if t is None else t.requires_grad_() for t in leaves]
    h = ops.gated_linear(*leaves, act=act, p=p, seed=seed, offset=offset)
    have = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(h, have, dh))
    return [h] + [None if t is None else next(grads) for t in leaves]


def check_case(M, K, N, dtype, act, bias, p=0.0, seed=0):
    ts = make(M, K, N, dtype, bias, seed)
    factor = 1.0
    if p > 0:
        factor = keep_mask((M, N), p, 7, 3).double() / (1 - p)
    outs, errs = oracle(*ts, act, factor)
    got = run_all(ts, act, p, 7, 3)
    compare(got, outs, errs, dtype)
    # and without gradients: the answering form
    h = ops.gated_linear(*[None if t is None else t.to(DEV)
                           for t in ts[:5]], act=act, p=p, seed=7, offset=3)
    compare([h], outs, errs, dtype)


# -------------------------------------------------------------------- CPU
@pytest.mark.parametrize("act", ACTS)
def test_oracle_gradient_against_differences(act):
    torch.manual_seed(3)
    ts = [t.double() for t in make(3, 5, 4, torch.float32, True, 5)]
    *leaves, dh = ts
    factor = keep_mask((3, 4), 0.4, 7, 3).double() / 0.6

    def value(args):
        x, wg, wu, bg, bu = args
        return float((act64(act, x @ wg + bg)[0] * (x @ wu + bu) * factor
                      * dh).sum())
    outs, _ = oracle(*[t.float() for t in leaves], dh.float(), act, factor)
    for n, grad in enumerate(outs[1:]):
        for flat in range(0, leaves[n].numel(), 3):
            step = 1e-5
            up = [t.clone() for t in leaves]
            dn = [t.clone() for t in leaves]
            up[n].view(-1)[flat] += step
            dn[n].view(-1)[flat] -= step
            diff = (value(up) - value(dn)) / (2 * step)
            # differences: step^2 of the third derivative, and 2^-53 / step
            assert abs(diff - float(grad.reshape(-1)[flat])) < 1e-7 * 50


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias", [False, True])
def test_cpu_path(act, bias):
    ts = make(6, 9, 11, torch.float32, bias)
    *leaves, dh = ts
    leaves = [None if t is None else t.requires_grad_() for t in leaves]
    h = ops.gated_linear(*leaves, act=act)
    have = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(h, have, dh))
    got = [h] + [None if t is None else next(grads) for t in leaves]
    outs, errs = oracle(*[None if t is None else t.detach() for t in ts],
                        act, 1.0)
    compare(got, outs, errs, torch.float32)


def test_cpu_leading_dimensions_and_dropout():
    x, wg, wu, *_ = make(6, 9, 11, torch.float32, False)
    h = ops.gated_linear(x.view(2, 3, 9), wg, wu, p=0.5, seed=1, offset=2)
    full = ops.gated_linear(x, wg, wu)
    assert h.shape == (2, 3, 11)
    assert torch.equal(h, ops.dropout(full.view(2, 3, 11), 0.5, 1, 2))


@pytest.mark.parametrize("kw,match", [
    ({"act": "tanh"}, "unknown activation"), ({"p": 1.5}, "p must not"),
    ({"p": float("nan")}, "p must not")])
def test_argument_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        ops.gated_linear(torch.ones(2, 3), torch.ones(3, 4),
                         torch.ones(3, 4), **kw)


# -------------------------------------------------------------------- GPU
TYPES = [torch.bfloat16, torch.float16]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_activations(dtype, act):
    check_case(40, 72, 136, dtype, act, True)


@gpu
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65,
                               127, 128, 129, 255, 256, 257, 300])
def test_rows(M):
    check_case(M, 136, 200, torch.float16, "silu", True, p=0.25, seed=M)


@gpu
@pytest.mark.parametrize("K,N", [(1, 1), (1, 8), (8, 1), (7, 5), (8, 8),
                                 (9, 17), (63, 65), (64, 64), (65, 63),
                                 (72, 127), (128, 128), (130, 129),
                                 (264, 256), (250, 258), (520, 520)])
@pytest.mark.parametrize("M", [1, 5, 70, 260])
def test_widths(M, K, N):
    check_case(M, K, N, torch.float16, "gelu", (K + N) % 2 == 0,
               p=0.5 if N % 3 else 0.0, seed=K)


@gpu
@pytest.mark.parametrize("M,K,N", [(1, 4096, 264), (3, 4104, 128),
                                   (16, 9216, 64), (40, 4096, 192),
                                   (100, 2056, 264), (300, 2048, 72),
                                   (2100, 72, 136), (1100, 264, 1032)])
@pytest.mark.parametrize("dtype", TYPES)
def test_long_contractions(M, K, N, dtype):
    check_case(M, K, N, dtype, "silu", True, p=0.5, seed=M)


@gpu
@pytest.mark.parametrize("M,K,N", [(2, 2048, 4096), (33, 4096, 2048),
                                   (64, 2048, 4096), (129, 4096, 2048),
                                   (256, 2048, 4096), (2048, 2048, 512)])
def test_more_tiles_than_the_card_holds(M, K, N):
    """Several rounds of tiles on every CU, several tiles a CU."""
    check_case(M, K, N, torch.float16, "gelu", True, p=0.5, seed=M)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 1, 8), (1, 33, 9), (16, 31, 127),
                                   (3, 300, 129), (5, 1055, 135),
                                   (16, 64, 137), (2, 4097, 259),
                                   (1, 520, 4095), (7, 2049, 1000)])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_answers_from_rows_that_start_anywhere(M, K, N, dtype, p):
    # each operand a part of a matrix that is NaN around it
    ts = make(M, K, N, dtype, True)
    factor = keep_mask((M, N), p, 7, 3).double() / (1 - p) if p else 1.0
    outs, errs = oracle(*ts, "gelu", factor)
    parts = []
    for t in ts[:3]:
        big = torch.full((t.shape[0] + 2, t.shape[1] + 13), float("nan"),
                         dtype=dtype, device=DEV)
        part = big[1:-1, 3:-10]
        part.copy_(t)
        parts.append(part)
    h = ops.gated_linear(*parts, ts[3].to(DEV), ts[4].to(DEV), act="gelu",
                         p=p, seed=7, offset=3)
    compare([h], outs, errs, dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,act", [
    (1999, 520, 2056, "silu"),
    (2003, 1001, 4100, "gelu"),
    (2056, 4104, 1003, "gelu_tanh"),
    (4101, 1000, 2056, "sigmoid"),
    (2003, 4104, 520, "relu"),
    (4101, 136, 4104, "silu"),
    (4100, 2056, 1031, "gelu"),
    (2051, 4104, 136, "gelu_tanh"),
    (1030, 2056, 2056, "sigmoid"),
    (4099, 4104, 40, "relu"),
    (520, 1000, 1032, "silu"), (60, 2056, 4104, "gelu"),
    (1030, 8200, 90, "silu")])
def test_every_tile_whole_and_split(M, K, N, act, dtype):
    """Sizes that between them take each tile of each product, with the
    contraction in one part and in several."""
    check_case(M, K, N, dtype, act, True, 0.5)


@gpu
def test_fused_dropout_is_the_dropout_of_the_result():
    for n in (200, 199):
        ts = [None if t is None else t.to(DEV)
              for t in make(37, 64, n, torch.float16, True)]
        h = ops.gated_linear(*ts[:5])
        fused = ops.gated_linear(*ts[:5], p=0.3, seed=5, offset=9)
        apart = ops.dropout(h, 0.3, 5, 9)
        assert torch.equal(fused == 0, apart == 0)
        # apart rounds once more: half a step on top of the same value
        assert torch.allclose(fused.float(), apart.float(),
                              rtol=2 * torch.finfo(torch.float16).eps, atol=1e-6)


@gpu
def test_strides_and_alignment():
    for K, N in ((64, 136), (40, 33)):
        ts = make(50, K, N, torch.bfloat16, True)
        want = [t for t in run_all(ts, "silu")]
        x, wg, wu, bg, bu, dh = [t.to(DEV) for t in ts]
        wide = torch.zeros(50, 3 * K + 1, dtype=x.dtype, device=DEV)
        for lo, step in ((0, 1), (8, 1), (1, 1), (0, 2)):
            xv = wide[:, lo:lo + step * K:step]
            xv.copy_(x)
            wv = torch.empty(N, K, dtype=x.dtype, device=DEV).t()
            wv.copy_(wg)
            uv = torch.empty(K, N + 8, dtype=x.dtype, device=DEV)[:, :N]
            uv.copy_(wu)
            bv = torch.empty(2 * N, dtype=x.dtype, device=DEV)[::2]
            bv.copy_(bg)
            dv = torch.empty(N, 50, dtype=x.dtype, device=DEV).t()
            dv.copy_(dh)
            leaves = [t.detach().requires_grad_()
                      for t in (xv, wv, uv, bv, bu)]
            h = ops.gated_linear(*leaves)
            got = [h, *torch.autograd.grad(h, leaves, dv)]
            for name, a, b in zip(NAMES, got, want):
                assert torch.equal(a, b), name


@gpu
def test_leading_dimensions_and_expanded_gradient():
    x, wg, wu, bg, bu, _ = [t.to(DEV) for t in
                            make(24, 64, 72, torch.bfloat16, True)]
    x3 = x.view(2, 3, 4, 64).requires_grad_()
    h = ops.gated_linear(x3, wg, wu, bg, bu)
    assert h.shape == (2, 3, 4, 72)
    h.sum().backward()
    flat = x.detach().requires_grad_()
    h2 = ops.gated_linear(flat, wg, wu, bg, bu)
    g2, = torch.autograd.grad(h2, flat, torch.ones_like(h2))
    assert torch.equal(h.view(24, 72), h2)
    assert torch.equal(x3.grad.view(24, 64), g2)
    assert ops.gated_linear(x[0].detach(), wg, wu).shape == (72,)


@gpu
def test_no_rows():
    ts = make(0, 16, 24, torch.bfloat16, True)
    h, dx, *rest = run_all(ts, "silu", p=0.5)
    assert h.shape == (0, 24) and dx.shape == (0, 16)
    for g in rest:
        assert not bool(g.any())


@gpu
@pytest.mark.parametrize("which", range(5))
def test_one_gradient_alone(which):
    ts = make(70, 72, 80, torch.bfloat16, True)
    want = run_all(ts, "silu")[1:][which]
    *leaves, dh = [t.to(DEV) for t in ts]
    leaves[which].requires_grad_()
    h = ops.gated_linear(*leaves)
    got, = torch.autograd.grad(h, leaves[which], dh)
    assert torch.equal(got, want)


@gpu
def test_results_past_32_bits():
    # 2^31 results and more; only the last rows have gradients: the terms of
    # the others are zeros and add no error
    M, K, N, last = (1 << 22) + 5, 8, 520, 37
    ts = make(last, K, N, torch.bfloat16, True)
    outs, errs = oracle(*ts, "silu", 1.0)
    x, wg, wu, bg, bu, dh = [t.to(DEV) for t in ts]
    gen = torch.Generator(device=DEV).manual_seed(3)
    big = torch.randn(M, K, generator=gen, device=DEV).bfloat16()
    big[-last:] = x
    with torch.no_grad():
        plain = ops.gated_linear(big, wg, wu, bg, bu)
        h = ops.gated_linear(big, wg, wu, bg, bu, p=0.5, seed=9, offset=2)
        # doubling is exact
        assert torch.equal(h, ops.dropout(plain, 0.5, 9, 2))
    del h, plain
    leaves = [t.requires_grad_() for t in (big, wg, wu, bg, bu)]
    zero = torch.zeros(M, N, dtype=x.dtype, device=DEV)
    zero[-last:] = dh
    h = ops.gated_linear(*leaves)
    got = torch.autograd.grad(h, leaves, zero)
    assert not bool(got[0][:-last].any())
    compare([h[-last:], got[0][-last:], *got[1:]], outs, errs, x.dtype)


@gpu
def test_rows_far_apart():
    x, wg, wu, bg, bu, dh = [t.to(DEV) for t in
                             make(20, 40, 48, torch.float16, True)]
    want = run_all([x, wg, wu, bg, bu, dh], "silu")
    far = torch.empty(20, (1 << 21) + 8, dtype=x.dtype, device=DEV)
    far[:, :40] = x
    wide = torch.empty(40, (1 << 21) + 8, dtype=x.dtype, device=DEV)
    wide[:, :48] = wg
    got = run_all([far[:, :40], wide[:, :48], wu, bg, bu, dh], "silu")
    for name, a, b in zip(NAMES, got, want):
        assert torch.equal(a, b), name


@gpu
def test_one_weight_twice():
    x, w, _, b, _, dh = [t.to(DEV) for t in
                         make(33, 40, 48, torch.float16, True)]
    w, b = w.requires_grad_(), b.requires_grad_()
    h = ops.gated_linear(x, w, w, b, b)
    dw, db = torch.autograd.grad(h, (w, b), dh)
    two = [t.detach().clone().requires_grad_() for t in (w, w, b, b)]
    parts = torch.autograd.grad(ops.gated_linear(x, *two), two, dh)
    assert torch.equal(dw, parts[0] + parts[1])
    assert torch.equal(db, parts[2] + parts[3])


@gpu
def test_one_buffer_for_two_gradients_is_refused():
    x, w, _, b, _, dh = [t.to(DEV) for t in
                         make(8, 40, 48, torch.bfloat16, True)]
    w = w.requires_grad_()
    w._dvgg_gbuf = torch.zeros_like(w)
    h = ops.gated_linear(x, w, w)
    with pytest.raises(RuntimeError, match="share one gradient buffer"):
        h.backward(dh)


@gpu
def test_gradient_buffer_anywhere_in_memory():
    x, wg, wu, bg, bu, dh = [t.to(DEV) for t in
                             make(20, 40, 48, torch.bfloat16, True)]
    want = run_all([x, wg, wu, bg, bu, dh], "silu")[2:]
    leaves = [t.detach().requires_grad_() for t in (wg, wu, bg, bu)]
    room = [torch.zeros(t.numel() + 3, dtype=t.dtype, device=DEV)
            for t in leaves]
    for t, r in zip(leaves, room):
        t._dvgg_gbuf = r[3:].view(t.shape)
    ops.gated_linear(x, *leaves).backward(dh)
    for name, t, w in zip(NAMES[2:], leaves, want):
        assert torch.equal(t._dvgg_gbuf, w), name
        assert torch.equal(t.grad, w), name


@gpu
def test_broadcast_input_and_inference_mode():
    x, wg, wu, bg, bu, dh = [t.to(DEV) for t in
                             make(1, 40, 48, torch.float16, True)]
    row = x.detach().requires_grad_()
    h = ops.gated_linear(row.expand(30, 40), wg, wu, bg, bu)
    g, = torch.autograd.grad(h, row, dh.expand(30, 48))
    full = x.expand(30, 40).contiguous().requires_grad_()
    h2 = ops.gated_linear(full, wg, wu, bg, bu)
    g2, = torch.autograd.grad(h2, full, dh.expand(30, 48).contiguous())
    assert torch.equal(h, h2)
    assert torch.equal(g, g2.sum(0, keepdim=True))
    with torch.inference_mode():
        assert torch.equal(ops.gated_linear(full, wg, wu, bg, bu), h2)


@gpu
def test_changed_input_is_noticed():
    x, wg, wu, *_ = [None if t is None else t.to(DEV)
                     for t in make(20, 40, 48, torch.float16, False)]
    wg.requires_grad_()
    h = ops.gated_linear(x, wg, wu)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        h.sum().backward()


@gpu
def test_two_streams_at_once():
    sets = [make(70, 2056, 136, torch.bfloat16, True, seed=s)
            for s in range(2)]
    want = [run_all(ts, "silu", 0.5, 7, 3) for ts in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = run_all(sets[i], "silu", 0.5, 7, 3)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for name, p, q in zip(NAMES, a, b):
            assert torch.equal(p, q), name


@gpu
def test_rows_of_infinities_stay_apart():
    x, wg, wu, *_ = [None if t is None else t.to(DEV)
                     for t in make(40, 64, 72, torch.bfloat16, False)]
    clean = ops.gated_linear(x, wg, wu)
    bad = x.clone()
    bad[7] = float("inf")
    bad[9, 3] = float("nan")
    h = ops.gated_linear(bad, wg, wu)
    rows = [i for i in range(40) if i not in (7, 9)]
    assert torch.equal(h[rows], clean[rows])
    assert bool(torch.isnan(h[9]).all())


@gpu
@pytest.mark.parametrize("act", ACTS)
def test_far_arguments(act):
    # g from -60000 to 60000 through one weight; the result and the
    # derivative stay finite where the function does
    g = torch.tensor([-6e4, -200.0, -90.0, -20.0, -5.0, 0.0, 5.0, 20.0, 90.0,
                      200.0, 6e4])
    x = g.to(torch.bfloat16).view(-1, 1)
    one = torch.ones(1, 1, dtype=torch.bfloat16)
    zero, unit = torch.zeros(1), torch.ones(1)
    ts = (x, one, 0 * one, zero.bfloat16(), unit.bfloat16(),
          torch.ones(11, 1, dtype=torch.bfloat16))
    outs, errs = oracle(*ts, act, 1.0)
    compare(run_all(ts, act), outs, errs, torch.bfloat16)


@gpu
def test_dropped_rows_pass_nothing_on():
    ts = list(make(64, 32, 40, torch.float16, True))
    keep = keep_mask((64, 40), 0.5, 7, 3)
    dh = ts[5].clone()
    dh[~keep] = float("nan")             # masked places may hold anything
    clean = run_all(ts, "silu", 0.5, 7, 3)
    ts[5] = dh
    for name, a, b in zip(NAMES, run_all(ts, "silu", 0.5, 7, 3), clean):
        assert torch.equal(a, b), name


@gpu
def test_same_result_every_time():
    ts = make(100, 2056, 264, torch.bfloat16, True)
    first = run_all(ts, "gelu", 0.1)
    for _ in range(3):
        for name, a, b in zip(NAMES, run_all(ts, "gelu", 0.1), first):
            assert torch.equal(a, b), name


@gpu
def test_differentiates_once():
    x, wg, wu, *_ = [None if t is None else t.to(DEV).requires_grad_()
                     for t in make(4, 8, 8, torch.bfloat16, False)[:3]]
    with pytest.raises(RuntimeError, match="differentiates once"):
        torch.autograd.grad(ops.gated_linear(x, wg, wu).sum(), x,
                            create_graph=True)


def _args(**kw):
    a = {"x": torch.ones(4, 8, dtype=torch.bfloat16, device=DEV),
         "w_gate": torch.ones(8, 16, dtype=torch.bfloat16, device=DEV),
         "w_up": torch.ones(8, 16, dtype=torch.bfloat16, device=DEV)}
    a.update({k: f(a) for k, f in kw.items()})
    return a


@gpu
@pytest.mark.parametrize("kw,match", [
    ({"x": lambda a: a["x"].float()}, "bf16 or fp16"),
    ({"x": lambda a: a["x"].double()}, "bf16 or fp16"),
    ({"w_gate": lambda a: a["w_gate"].half()}, "w_gate is"),
    ({"w_up": lambda a: a["w_up"].half()}, "w_up is"),
    ({"w_up": lambda a: a["w_up"].cpu()}, "w_up is on"),
    ({"w_up": lambda a: a["w_up"][:, :8]}, "w_up has shape"),
    ({"w_gate": lambda a: a["w_gate"][:4]}, "w_gate has shape"),
    ({"w_gate": lambda a: a["w_gate"][0]}, "must be a matrix"),
    ({"bias_up": lambda a: a["w_up"][0, :8]}, "bias_up has shape"),
    ({"bias_gate": lambda a: a["w_up"]}, "bias_gate has shape"),
    ({"bias_gate": lambda a: a["w_up"][0].float()}, "bias_gate is"),
    ({"offset": lambda a: torch.zeros(1, dtype=torch.int64)},
     "one int64 on x's device"),
    ({"x": lambda a: a["x"][:, :0], "w_gate": lambda a: a["w_gate"][:0],
      "w_up": lambda a: a["w_up"][:0]}, "must not be 0"),
])
def test_refusals(kw, match):
    with pytest.raises((RuntimeError, ValueError), match=match):
        ops.gated_linear(**_args(**kw))


@gpu
def test_replayed_graph_and_another_stream():
    ts = make(70, 2056, 136, torch.bfloat16, True)
    *leaves, dh = [t.to(DEV) for t in ts]
    leaves = [t.requires_grad_() for t in leaves]
    off = torch.zeros(1, dtype=torch.int64, device=DEV)

    def both():
        h = ops.gated_linear(*leaves, act="silu", p=0.5, seed=7, offset=off)
        return [h, *torch.autograd.grad(h, leaves, dh)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        off.fill_(3)
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    factor = keep_mask((70, 136), 0.5, 7, 3).double() / 0.5
    outs, errs = oracle(*ts, "silu", factor)
    compare(got, outs, errs, torch.bfloat16)
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        off.add_(1)
        got = both()
    for replay in range(4):
        other = make(70, 2056, 136, torch.bfloat16, True, seed=50 + replay)
        with torch.no_grad():
            for t, v in zip(leaves + [dh], other):
                t.copy_(v)
        off.fill_(replay)
        graph.replay()
        torch.cuda.synchronize()
        # the same program, eager, on another buffer of offsets
        want = run_all(other, "silu", 0.5, 7, replay + 1)
        for name, a, b in zip(NAMES, got, want):
            assert torch.equal(a, b), (name, replay)


@gpu
@pytest.mark.parametrize("K,N", [(2056, 136), (2055, 133)])
def test_two_graphs_in_turn(K, N):
    # answers of few and of more rows, each split and joined, in two graphs
    # whose replays alternate
    sets = [[t.to(DEV) for t in make(M, K, N, torch.float16, True)[:5]]
            for M in (4, 40)]
    graphs, got = [], []
    for ts in sets:
        ops.gated_linear(*ts, act="gelu")
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(ops.gated_linear(*ts, act="gelu"))
    for replay in range(4):
        for i, ts in enumerate(sets):
            ts[0].copy_(make(ts[0].shape[0], K, N, torch.float16, True,
                             seed=replay)[0])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for h, ts in zip(got, sets):
            assert torch.equal(h, ops.gated_linear(*ts, act="gelu")), replay


@gpu
def test_offset_counted_up_before_backward():
    ts = make(20, 64, 72, torch.bfloat16, True)
    *leaves, dh = [t.to(DEV) for t in ts]
    leaves = [t.requires_grad_() for t in leaves]
    off = torch.full((1,), 3, dtype=torch.int64, device=DEV)
    h = ops.gated_linear(*leaves, p=0.5, seed=7, offset=off)
    off.add_(5)
    got = [h, *torch.autograd.grad(h, leaves, dh)]
    for name, a, b in zip(NAMES, got, run_all(ts, "silu", 0.5, 7, 3)):
        assert torch.equal(a, b), name


@gpu
def test_two_in_a_row_with_dropout_between():
    """Unit, dropout, next layer: as a head runs them."""
    torch.manual_seed(0)
    x, wg, wu, bg, bu, _ = make(48, 96, 104, torch.bfloat16, True)
    w2 = (torch.randn(104, 40) * 0.1).bfloat16()
    dy = torch.randn(48, 40).bfloat16()
    leaves = [t.to(DEV).requires_grad_() for t in (x, wg, wu, bg, bu)]
    h = ops.gated_linear(*leaves, act="gelu")
    y = ops.linear(ops.dropout(h, 0.5, 7, 3), w2.to(DEV))
    got = torch.autograd.grad(y, leaves, dy.to(DEV))
    dh = (dy.double() @ w2.double().t())
    factor = keep_mask((48, 104), 0.5, 7, 3).double() / 0.5
    # what reaches the unit is dh after three roundings: linear's, dropout's
    # and the type's own; they pass through linearly
    outs, errs = oracle(x, wg, wu, bg, bu, dh.bfloat16(), "gelu", factor)
    e = torch.finfo(torch.bfloat16).eps / 2
    v, g, u = dh.abs() * factor, x.double() @ wg.double() + bg.double(), \
        x.double() @ wu.double() + bu.double()
    a, da = act64("gelu", g)
    mg, mu = v * (u * da).abs() * 4 * e, v * a.abs() * 4 * e
    xa = x.double().abs().t()
    more = [mg @ wg.double().abs().t() + mu @ wu.double().abs().t(),
            xa @ mg, xa @ mu, mg.sum(0), mu.sum(0)]
    for name, t, want, err, m in zip(NAMES[1:], got, outs[1:], errs[1:],
                                     more):
        off = (t.cpu().double() - want).abs()
        assert bool((off <= err + m).all()), name
