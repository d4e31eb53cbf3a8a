"""Every tile that the gated unit's products take, whole and split, against the
formulas in 64 bits. The sizes are held to what make_plan chooses, so that a
change of its model cannot leave a kernel untested."""

import math
import random

import pytest
import torch

from distributed_vgg_f_amd.ops import native

from test_gated import ACTS, NAMES, check_case, make, run_all

gpu = pytest.mark.gpu

# rows, K, N: between them all of what random sizes take
SIZES = [(17, 72, 65), (144, 146, 64), (17, 8360, 276), (4141, 394, 207),
         (2082, 3035, 65), (5442, 71, 1303), (659, 13512, 65),
         (641, 422, 7842), (3619, 3332, 267), (135, 10894, 3032),
         (560, 3969, 1667), (2271, 8344, 131), (6809, 2762, 133)]


def kernels(M, K, N):
    """(product, tile, in parts) of the three products of a training pass."""
    def one(what, rows, cols, k_len):
        *tile, splits = native.ext().gated_plan(what, rows, cols, k_len)
        return what, *tile, splits > 1
    return {one(0, M, N, K), one(1, M, K, N), one(2, K, N, M)}


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
@pytest.mark.parametrize("args", [(3, 1, 1, 1), (-1, 1, 1, 1), (0, 0, 1, 1),
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
