"""The contrastive loss over the feature bank, on HIP kernels: the logits (`linear`), the log probabilities of the slots' own bank
rows with entropy and best alternatives (`log_probs`), and both joined without the [slots, bank rows] matrix (`bank_log_probs`).

The reference computes this loss in torch from FeatureBankNeMo's similarity and MaskCreater's weights (nemo/models/nemo.py:138-209):
softmax over the bank's rows of similarity / T - weight, cross entropy at the slot's own row.  All functions are differentiable (once),
run on the current stream of their tensors' device, never synchronise, and raise before any launch on arguments they do not take.
"""
from collections import namedtuple

import torch
from torch.autograd.function import once_differentiable

from . import ops


def _device_tensors(what, dtypes, **tensors):
    """All tensors on one GPU and of one of `dtypes` (None entries are skipped)."""
    first = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not torch.is_tensor(t):
            raise TypeError(f"{what}: {name} must be a tensor")
        if not t.is_cuda:
            raise RuntimeError(f"{what}: {name} is a CPU tensor; nemo_amd kernels need device tensors, there is no CPU path")
        if t.dtype not in dtypes:
            raise TypeError(f"{what}: {name} is {t.dtype}, takes {', '.join(str(d) for d in dtypes)}")
        if first is None:
            first = (name, t)
        elif t.device != first[1].device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, {first[0]} on {first[1].device}")
        elif t.dtype != first[1].dtype:
            raise TypeError(f"{what}: {name} is {t.dtype}, {first[0]} {first[1].dtype}")


def _number(what, name, value):
    value = float(value)
    if value != value or value in (float("inf"), -float("inf")):
        raise ValueError(f"{what}: {name} must be finite, got {value}")
    return value


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, alpha, beta):
        need_pre = activation != "none" and any(ctx.needs_input_grad[:3])
        y, pre = ops.linear(x, weight, bias, residual, activation, alpha, beta, want_pre=need_pre)
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, weight if ctx.needs_input_grad[0] else None, pre)
        ctx.sizes = (x.shape[0], weight.shape[0], x.shape[1])
        ctx.args = (activation, alpha, beta)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        x, weight, pre = ctx.saved_tensors
        activation, alpha, beta = ctx.args
        M, N, K = ctx.sizes
        want = list(ctx.needs_input_grad[:4])
        pass_through = want[3] and beta == 1.0          # the residual's gradient is grad_y itself
        if pass_through:
            want[3] = False
        grads = [None] * 4
        if any(want):
            grads = list(ops.linear_backward(grad_y, (M, K) if x is None else x, (N, K) if weight is None else weight, pre, activation,
                                             alpha, beta, want))
        if pass_through:
            grads[3] = grad_y
        return (*grads, None, None, None)


def linear(x, weight, bias=None, residual=None, activation="none", alpha=1.0, beta=1.0):
    """act(alpha x weight^T + bias) + beta residual in one product kernel.

    x [..., K], weight [N, K], bias [N], residual [..., N] of one type (float32, bfloat16 or float16) -> [..., N] of that type.
    activation: "none", "relu", "gelu" (the exact one, with erf) or "silu".  Products are summed in 32 bits (float32: on the f32 matrix
    cores, so infinities and NaN come out as in any f32 product) and the result is rounded once.  x, weight, bias and residual are
    differentiable.  Rows of x, weight and residual may be strided; alignment matters for speed only."""
    _device_tensors("linear", tuple(ops.DTYPES), x=x, weight=weight, bias=bias, residual=residual)
    if activation not in ops.ACTIVATIONS:
        raise ValueError(f"linear: activation {activation!r} (takes {', '.join(ops.ACTIVATIONS)})")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x must be [..., K] and weight [N, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    N, K = weight.shape
    lead = x.shape[:-1]
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"linear: bias must be [{N}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != lead + (N,):
        raise ValueError(f"linear: residual must be {tuple(lead) + (N,)}, got {tuple(residual.shape)}")
    alpha, beta = _number("linear", "alpha", alpha), _number("linear", "beta", beta)
    M = 1
    for n in lead:
        M *= n
    y = _Linear.apply(x.reshape(M, K), weight, bias, None if residual is None else residual.reshape(M, N), activation, alpha, beta)
    return y.reshape(lead + (N,))
