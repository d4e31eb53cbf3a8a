"""Custom autograd Functions wrapping the HIP kernels (GPU path only).

Each Function mirrors one K# row of SURVEY.md section 2.4 (those of dropout
and of the gated unit are in csrc/fn.cpp). The CPU path never
reaches these — layers dispatch CPU tensors to ops.cpu_ref compositions and
let torch autograd differentiate those. Here, forward/backward both call
hand-written CDNA4 kernels via ops.native.ext().

Fusion contract with the kernels:
  * conv/linear forward fuses bias add + ReLU into the GEMM epilogue (K10/K11
    fwd); backward first applies the ReLU mask to dy (one elementwise kernel)
    then runs dgrad/wgrad.
  * wgrad kernels accumulate in fp32 and emit the gradient dtype of the
    grad arena (bf16 by default).
  * softmax_xent computes dlogits in forward (K13 is one fused kernel); the
    backward just scales it by the incoming dloss scalar.
"""

from __future__ import annotations

import torch

from . import native


def _ext():
    return native.ext()



def _fresh(t):
    """Return a fresh view (new TensorImpl, use_count 1) of an
    arena-homed gradient. AccumulateGrad only STORES an incoming grad
    whose TensorImpl is not referenced elsewhere; the tensors our
    kernels write (and ctx holds) fail that check, so torch silently
    CLONED every param grad — one DtoD blit per param per step (146 on
    ResNet-50). The alias passes the use-count check and .grad becomes
    the arena view itself (verified by tests/test_gpu_engine
    direct-grad assertion)."""
    return t.view_as(t) if t is not None else None


class ConvFunction(torch.autograd.Function):
    """K1/K2/K3 + fused bias/ReLU. x [N,H,W,C] bf16, w [kh,kw,Ci,Co] bf16."""

    @staticmethod
    def forward(ctx, x, w, bias, stride: int, pad: int, relu: bool):
        cw = getattr(w, "_dvgg_wcache", False)  # arena-homed: persistent wT
        y = _ext().conv2d_fwd(x, w, bias, stride, pad, relu, cw)
        ctx.save_for_backward(x, w, y if relu else torch.empty(0, device=x.device))
        ctx.stride, ctx.pad, ctx.relu = stride, pad, relu
        ctx.has_bias = bias is not None
        ctx.cw = cw
        # direct-grad: arena views attached by ArenaOptimizer (engine/arena.py)
        ctx.gw = getattr(w, "_dvgg_gbuf", None)
        ctx.gb = getattr(bias, "_dvgg_gbuf", None) if bias is not None else None
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, y = ctx.saved_tensors
        need_dx = ctx.needs_input_grad[0]
        need_db = ctx.has_bias and ctx.needs_input_grad[2]
        # fused path: one pass over dy produces the ReLU-masked dy, the
        # wgrad transpose and the bias grad, then the dgrad/wgrad GEMMs run
        # on the shared intermediates (csrc conv2d_bwd: K10/K11 fused into
        # the K2/K3 preamble). dw/db land directly in the grad arena when
        # the params carry _dvgg_gbuf views (skips AccumulateGrad adds).
        dx, dw, db = _ext().conv2d_bwd(dy.contiguous(), y, x, w, ctx.stride,
                                       ctx.pad, ctx.relu, need_dx, need_db,
                                       ctx.gw, ctx.gb, ctx.cw)
        return (dx if need_dx else None, _fresh(dw),
                _fresh(db) if need_db else None, None, None, None)


class LinearFunction(torch.autograd.Function):
    """K8/K9 + fused bias/ReLU. x [M,K], w [K,N]."""

    @staticmethod
    def forward(ctx, x, w, bias, relu: bool):
        y = _ext().linear_fwd(x, w, bias, relu,
                              getattr(w, "_dvgg_wcache", False))
        ctx.save_for_backward(x, w, y if relu else torch.empty(0, device=x.device))
        ctx.relu = relu
        ctx.has_bias = bias is not None
        ctx.gw = getattr(w, "_dvgg_gbuf", None)
        ctx.gb = getattr(bias, "_dvgg_gbuf", None) if bias is not None else None
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, y = ctx.saved_tensors
        dy = dy.contiguous()
        if ctx.relu:
            dy = _ext().relu_bwd(dy, y)
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = _ext().linear_dgrad(dy, w)      # dy @ w^T
        if ctx.needs_input_grad[1]:
            dw = _ext().linear_wgrad(x, dy, ctx.gw)  # x^T @ dy, into arena
        if ctx.has_bias and ctx.needs_input_grad[2]:
            db = _ext().bias_grad(dy, ctx.gb)
        return dx, _fresh(dw), _fresh(db), None


class LRNFunction(torch.autograd.Function):
    """K4/K5. Fwd saves only x: backward recomputes the window scale s
    (cheap FMAs over the x it reloads anyway) and sb/snb via the same
    fast_log2/fast_exp2 polynomials — 2-stream fwd, 3-stream bwd instead
    of storing+reloading sb/snb (csrc/lrnpool.hip)."""

    @staticmethod
    def forward(ctx, x, size: int, alpha: float, beta: float, k: float):
        y = _ext().lrn_fwd(x, size, alpha, beta, k)
        ctx.save_for_backward(x)
        ctx.params = (size, alpha, beta, k)
        return y

    @staticmethod
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        size, alpha, beta, k = ctx.params
        dx = _ext().lrn_bwd(dy.contiguous(), x, size, alpha, beta, k)
        return dx, None, None, None, None


class MaxPoolFunction(torch.autograd.Function):
    """K6/K7: 3x3 s2 maxpool with saved u8 argmax; bwd is a gather over dx."""

    @staticmethod
    def forward(ctx, x, kernel: int, stride: int, pad_l: int, pad_r: int):
        y, idx = _ext().maxpool_fwd(x, kernel, stride, pad_l, pad_r)
        ctx.save_for_backward(idx)
        ctx.geom = (x.shape[1], x.shape[2], kernel, stride, pad_l, pad_r)
        return y

    @staticmethod
    def backward(ctx, dy):
        (idx,) = ctx.saved_tensors
        H, W, kernel, stride, pad_l, pad_r = ctx.geom
        dx = _ext().maxpool_bwd(dy.contiguous(), idx, H, W, kernel, stride,
                                pad_l, pad_r)
        return dx, None, None, None, None


class SoftmaxXentFunction(torch.autograd.Function):
    """K13: one fused kernel computes per-row loss AND dlogits in forward."""

    @staticmethod
    def forward(ctx, logits, labels):
        loss, dlogits = _ext().softmax_xent_fwd(logits, labels)
        ctx.save_for_backward(dlogits)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        (dlogits,) = ctx.saved_tensors
        # dloss is [M]; benchmark path uses loss.sum() (scale folded into SGD
        # grad_scale), so dloss is a vector of ones — still handle general case.
        return (dlogits * dloss.unsqueeze(1)).to(dlogits.dtype), None


class BatchNormFunction(torch.autograd.Function):
    """K17 (ResNet-50): training-mode BN over N,H,W with optional fused ReLU."""

    @staticmethod
    def forward(ctx, x, gamma, beta, eps: float, relu: bool,
                run_mean=None, run_var=None, momentum: float = 0.9):
        y, mean, rstd = _ext().bn_fwd(x, gamma, beta, eps, relu,
                                      run_mean, run_var, momentum)
        ctx.save_for_backward(x, gamma, mean, rstd,
                              y if relu else torch.empty(0, device=x.device))
        ctx.relu = relu
        ctx.gg = getattr(gamma, "_dvgg_gbuf", None)
        ctx.gb = getattr(beta, "_dvgg_gbuf", None)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, gamma, mean, rstd, y = ctx.saved_tensors
        # ReLU mask fused into the BN backward kernels (no separate pass)
        dx, dgamma, dbeta = _ext().bn_bwd(dy.contiguous(), x, gamma, mean,
                                          rstd, y, ctx.relu, ctx.gg, ctx.gb)
        return dx, _fresh(dgamma), _fresh(dbeta), None, None, None, None, None


class BNAddReluFunction(torch.autograd.Function):
    """K17+K18 fused: z = relu(bn(x) + res) in one apply pass (the
    separate add_relu kernel read+wrote the whole block output)."""

    @staticmethod
    def forward(ctx, x, gamma, beta, res, eps: float,
                run_mean=None, run_var=None, momentum: float = 0.9):
        z, mean, rstd = _ext().bn_fwd(x, gamma, beta, eps, True,
                                      run_mean, run_var, momentum, res)
        ctx.save_for_backward(x, gamma, mean, rstd, z)
        ctx.gg = getattr(gamma, "_dvgg_gbuf", None)
        ctx.gb = getattr(beta, "_dvgg_gbuf", None)
        return z

    @staticmethod
    def backward(ctx, dz):
        x, gamma, mean, rstd, z = ctx.saved_tensors
        # da feeds BOTH the bn input grad chain and the residual branch
        da = _ext().relu_bwd(dz.contiguous(), z)
        dx, dgamma, dbeta = _ext().bn_bwd(da, x, gamma, mean, rstd,
                                          torch.empty(0, device=x.device),
                                          False, ctx.gg, ctx.gb)
        return dx, _fresh(dgamma), _fresh(dbeta), da, None, None, None, None


class AddReluFunction(torch.autograd.Function):
    """K18 (ResNet-50): y = relu(a + b)."""

    @staticmethod
    def forward(ctx, a, b):
        y = _ext().add_relu_fwd(a, b)
        ctx.save_for_backward(y)
        return y

    @staticmethod
    def backward(ctx, dy):
        (y,) = ctx.saved_tensors
        da = _ext().relu_bwd(dy.contiguous(), y)
        return da, da
