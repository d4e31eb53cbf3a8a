"""Every tile that the gated unit's products take, whole and split, against the
formulas in 64 bits. The sizes are held to what make_plan chooses, so that a
change of its model cannot leave a kernel untested."""

import math
import random

import pytest
import torch

from distributed_vgg_f_amd import ops
from distributed_vgg_f_amd.ops import native

from test_gated import (ACTS, NAMES, check_case, compare, make, oracle,
                        run_all)

gpu = pytest.mark.gpu

# rows, K, N: between them all of what random sizes take
SIZES = [(17, 72, 65), (144, 146, 64), (17, 8360, 276), (4141, 394, 207),
         (2082, 3035, 65), (5442, 71, 1303), (659, 13512, 65),
         (641, 422, 7842), (3619, 3332, 267), (135, 10894, 3032),
         (560, 3969, 1667), (2271, 8344, 131), (6809, 2762, 133)]
# those of one weight gradient alone
ONE = [(18, 71, 65), (647, 67, 74), (132, 66, 65), (520, 64, 66),
       (65, 21978, 266), (6931, 134, 5752), (74, 24854, 144),
       (1817, 8212, 131), (17, 24824, 143), (148, 8321, 133),
       (6182, 679, 131), (516, 20090, 550), (2712, 16538, 139)]


def kernels(M, K, N):
    """(product, tile, in parts) of the three products of a training pass."""
    return {kernel(0, M, N, K), kernel(1, M, K, N), kernel(2, K, N, M)}


def kernel(what, rows, cols, k_len):
    *tile, splits = native.ext().gated_plan(what, rows, cols, k_len)
    return what, *tile, splits > 1


@pytest.mark.skipif(not native.available(),
                    reason="needs the built extension")
def test_the_sizes_take_every_tile():
    rng = random.Random(3)

    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    reached = set()
    for _ in range(60000):
        reached |= kernels(size(17, 8192), size(1, 25088), size(1, 8192))
    # the largest products of any model here, and those of long batches
    for M in (17, 64, 256, 1024, 8192, 65536, 1 << 20):
        for K, N in ((9216, 4096), (25088, 4096), (4096, 4096), (64, 64)):
            reached |= kernels(M, K, N)
    taken = set().union(*(kernels(*s) for s in SIZES))
    assert reached - taken == set()


@pytest.mark.skipif(not native.available(),
                    reason="needs the built extension")
def test_the_sizes_take_every_tile_of_one_gradient():
    rng = random.Random(4)

    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    reached = {kernel(3, size(1, 25088), size(1, 8192), size(1, 8192))
               for _ in range(60000)}
    for M in (17, 64, 256, 1024, 8192, 65536, 1 << 20):
        for K, N in ((9216, 4096), (25088, 4096), (4096, 4096), (64, 64)):
            reached.add(kernel(3, K, N, M))
    assert reached - {kernel(3, K, N, M) for M, K, N in ONE} == set()


@pytest.mark.skipif(not native.available(),
                    reason="needs the built extension")
@pytest.mark.parametrize("args", [(4, 1, 1, 1), (-1, 1, 1, 1), (0, 0, 1, 1),
                                  (1, 1, -5, 1), (2, 1, 1, 0)])
def test_no_plan_for_no_product(args):
    with pytest.raises(RuntimeError, match="no such product"):
        native.ext().gated_plan(*args)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("which", range(len(SIZES)))
def test_values(which, dtype):
    check_case(*SIZES[which], dtype, ACTS[which % 5], which % 3 > 0, 0.5)


@gpu
@pytest.mark.parametrize("size", SIZES)
def test_the_same_every_time(size):
    ts = make(*size, torch.bfloat16, True)
    first = run_all(ts, "silu", 0.1)
    for _ in range(2):
        for name, a, b in zip(NAMES, run_all(ts, "silu", 0.1), first):
            assert torch.equal(a, b), name


def one_alone(ts, which):
    """The gradient of one weight, the other frozen, and the memory that its
    pass took besides, in bytes."""
    x, wg, wu, bg, bu, dh = ts
    leaf = (wg, wu)[which].requires_grad_()
    h = ops.gated_linear(x, wg, wu, bg, bu)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grad, = torch.autograd.grad(h, leaf, dh)
    leaf.requires_grad_(False)
    return grad, torch.cuda.max_memory_allocated() - before


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", ONE)
def test_one_weight_gradient_alone(size, dtype):
    ts = [t.to("cuda:0") for t in make(*size, dtype, True)]
    outs, errs = oracle(*ts, "silu", 1.0)
    for which in range(2):
        grad, _ = one_alone(ts, which)
        none = [None] * (2 + which)
        compare([*none, grad], [o.cpu() for o in outs],
                [e.cpu() for e in errs], dtype)


@gpu
@pytest.mark.parametrize("which", range(2))
def test_a_frozen_weight_takes_no_room(which):
    ts = [t.to("cuda:0") for t in make(32, 4096, 4096, torch.bfloat16, True)]
    one_alone(ts, which)
    # the gradient, and dG and dU of 32 rows: not the other's gradient too
    assert one_alone(ts, which)[1] < 1.25 * 4096 * 4096 * 2
