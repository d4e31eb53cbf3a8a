"""Functional op layer: dispatches CPU -> cpu_ref (torch fp32, differentiable)
and CUDA -> hand-written HIP kernels via custom autograd Functions.

This is the single seam between the model zoo and the two execution paths.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import cpu_ref
from . import native  # noqa: F401  (re-export for engine / tests)


ACTIVATIONS = tuple(cpu_ref.ACTIVATIONS)      # of gated_linear
_ACT_ID = {name: i for i, name in enumerate(ACTIVATIONS)}


def conv2d(x, w, bias=None, stride: int = 1, pad: int = 0, relu: bool = False):
    if x.is_cuda:
        from .autograd import ConvFunction
        return ConvFunction.apply(x, w, bias, stride, pad, relu)
    return cpu_ref.conv2d(x, w, bias, stride, pad, relu)


def linear(x, w, bias=None, relu: bool = False):
    if x.is_cuda:
        from .autograd import LinearFunction
        return LinearFunction.apply(x, w, bias, relu)
    return cpu_ref.linear(x, w, bias, relu)


def gated_linear(x, w_gate, w_up, bias_gate=None, bias_up=None,
                 act: str = "silu", p: float = 0.0, seed: int = 0,
                 offset: Union[int, torch.Tensor] = 0):
    """dropout(act(x @ w_gate + bias_gate) * (x @ w_up + bias_up), p)

    x [..., K], both weights [K, N], biases [N] or None; the result is
    [..., N]. act: silu, gelu (erf), gelu_tanh, relu or sigmoid. p, seed and
    offset are those of `dropout`, which draws the same mask from them; p = 0
    leaves it out.

    GPU: bf16 or fp16, one type and one device for all operands, K and N from
    1 to 2^21, any strides; sums in 32 bits. Operands whose rows do not start
    on 16 bytes are copied to rows that do, once a call (not for answers of up
    to 16 rows). Differentiates once, backward; no tangents and no function
    transforms. A traced call replays the operator.
    """
    if act not in _ACT_ID:
        raise ValueError(f"gated_linear: unknown activation {act!r}; have "
                         f"{list(ACTIVATIONS)}")
    if not p <= 1.0:
        raise ValueError(f"gated_linear: p must not be above 1, got {p}")
    if not x.is_cuda or p == 1.0:
        h = cpu_ref.gated_linear(x, w_gate, w_up, bias_gate, bias_up, act) \
            if not x.is_cuda else \
            gated_linear(x, w_gate, w_up, bias_gate, bias_up, act)
        return dropout(h, p, seed, offset)
    if x.dim() < 1:
        raise ValueError("gated_linear: x must have a last dimension")
    flat = x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]),
                                            x.shape[-1])
    on_device = isinstance(offset, torch.Tensor)
    h = native.ext().gated_linear(
        flat, w_gate, w_up, bias_gate, bias_up, _ACT_ID[act], max(p, 0.0),
        seed, 0 if on_device else offset, offset if on_device else None)
    return h if x.dim() == 2 else h.view(*x.shape[:-1], h.shape[-1])


def lrn(x, size: int = 5, alpha: float = 1e-4, beta: float = 0.75, k: float = 2.0):
    if x.is_cuda:
        from .autograd import LRNFunction
        return LRNFunction.apply(x, size, alpha, beta, k)
    return cpu_ref.lrn(x, size, alpha, beta, k)


def maxpool(x, kernel: int = 3, stride: int = 2, pad: Tuple[int, int] = (0, 0)):
    if x.is_cuda:
        from .autograd import MaxPoolFunction
        return MaxPoolFunction.apply(x, kernel, stride, pad[0], pad[1])
    return cpu_ref.maxpool(x, kernel, stride, pad)


def dropout(x, p: float, seed: int = 0, offset: Union[int, torch.Tensor] = 0,
            mask: Optional[torch.Tensor] = None):
    """y = keep * x / (1 - p), p <= 1; p <= 0 returns x itself, p = 1 zeros.

    GPU: bf16, fp16 or fp32 of any shape and strides. The mask is a function
    of (element index, p, seed, offset), drawn again in the backward pass and
    never stored; a dropped element is 0 whatever x holds there. seed and
    offset count modulo 2^32. offset may be one int64 on x's device: a
    captured graph then draws a new mask at each replay if the caller counts
    it up. Differentiates backward, any number of times; no tangents and no
    function transforms; a traced call replays the operator, with the seed and
    the offset of the recording (an offset on the device is read anew). CPU:
    the mask is torch's own, or the one that is given (`mask` is
    not read on the GPU).
    """
    if p <= 0.0:
        return x
    if not p <= 1.0:
        raise ValueError(f"dropout: p must not be above 1, got {p}")
    if p == 1.0:
        return x.masked_fill(torch.ones((), dtype=torch.bool,
                                        device=x.device), 0.0)
    if x.is_cuda:
        if isinstance(offset, torch.Tensor):
            return native.ext().dropout(x, p, seed, 0, offset)
        return native.ext().dropout(x, p, seed, offset)
    if mask is None:
        gen = torch.Generator().manual_seed(int(seed + offset))
        mask = (torch.rand(x.shape, generator=gen) >= p).to(x.dtype)
    return cpu_ref.dropout(x, p, mask)


def softmax_xent(logits, labels):
    """Returns per-row loss [M] (fp32)."""
    if logits.is_cuda:
        from .autograd import SoftmaxXentFunction
        return SoftmaxXentFunction.apply(logits, labels)
    # CPU: differentiable composition
    import torch.nn.functional as F
    return F.cross_entropy(logits.float(), labels, reduction="none")


def batchnorm(x, gamma, beta, eps: float = 1e-5, relu: bool = False,
              run_mean=None, run_var=None, momentum: float = 0.9, res=None):
    if x.is_cuda:
        if res is not None:
            from .autograd import BNAddReluFunction
            return BNAddReluFunction.apply(x, gamma, beta, res, eps,
                                           run_mean, run_var, momentum)
        from .autograd import BatchNormFunction
        return BatchNormFunction.apply(x, gamma, beta, eps, relu,
                                       run_mean, run_var, momentum)
    y = cpu_ref.batchnorm(x, gamma, beta, eps, relu and res is None)
    if res is not None:
        y = cpu_ref.add_relu(y, res)
    if run_mean is not None:
        with torch.no_grad():
            m = x.float().mean(dim=(0, 1, 2))
            v = x.float().var(dim=(0, 1, 2), unbiased=False)
            run_mean.mul_(momentum).add_(m, alpha=1 - momentum)
            run_var.mul_(momentum).add_(v, alpha=1 - momentum)
    return y


def add_relu(a, b):
    if a.is_cuda:
        from .autograd import AddReluFunction
        return AddReluFunction.apply(a, b)
    return cpu_ref.add_relu(a, b)


def sgd_momentum_step(w32, w_model, g, m32, lr, momentum, weight_decay=0.0,
                      grad_scale=1.0):
    """Fused flat-arena SGD+momentum (K14). On GPU one kernel updates the fp32
    master, momentum, and rewrites the model-dtype param arena; on CPU w_model
    IS w32 and the torch composition applies."""
    if w32.is_cuda:
        native.ext().sgd_step(w32, w_model, g, m32, float(lr), float(momentum),
                              float(weight_decay), float(grad_scale))
    else:
        cpu_ref.sgd_momentum(w32, g, m32, lr, momentum, weight_decay, grad_scale)
        if w_model.data_ptr() != w32.data_ptr():
            w_model.copy_(w32)
