"""The contrastive loss over the feature bank, on HIP kernels: the logits (`linear`), the log probabilities of the slots' own bank
rows with entropy and best alternatives (`log_probs`), and both joined without the [slots, bank rows] matrix (`bank_log_probs`).

The reference computes this loss in torch from FeatureBankNeMo's similarity and MaskCreater's weights (nemo/models/nemo.py:138-209):
softmax over the bank's rows of similarity / T - weight, cross entropy at the slot's own row.  All functions are differentiable (once, by a
backward pass; tensors with forward-mode tangents are refused), run on the current stream of their tensors' device, and raise before any launch on
arguments they do not take.  They never synchronise on device tensors; targets on the host are checked there and copied, which waits for the
stream and is refused while it is captured.
They may be captured into a graph, with their backward pass too; as with torch's own operators no eager autograd graph of the same leaves may
be alive then (the leaves' gradients would be gathered on the stream of that graph, outside the capture): drop its results first.
"""
from collections import namedtuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops


def _device_tensors(what, dtypes, names, *tensors):
    """All tensors on one GPU and of one of `dtypes`; bias and residual may be None."""
    first = tensors[0]
    for name, t in zip(names, tensors):
        if t is None and name in ("bias", "residual"):
            continue
        if not torch.is_tensor(t):
            raise TypeError(f"{what}: {name} must be a tensor")
        if not t.is_cuda:
            raise RuntimeError(f"{what}: {name} is a CPU tensor; nemo_amd kernels need device tensors, there is no CPU path")
        if t.dtype not in dtypes:
            raise TypeError(f"{what}: {name} is {t.dtype}, takes {', '.join(str(d) for d in dtypes)}")
        if t is not first and t.device != first.device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, {names[0]} on {first.device}")
        if t.dtype != first.dtype:
            raise TypeError(f"{what}: {name} is {t.dtype}, {names[0]} {first.dtype}")


def _no_tangents(what, *tensors):
    if getattr(forward_ad, "_current_level", 0) >= 0:                  # within forward_ad.dual_level()
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what}: no tangent for forward-mode derivatives (backward passes only)")


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _once(gradients):
    """`gradients` as a backward pass that is not differentiable itself; what that takes is only paid where a graph of it is asked for."""
    guarded = once_differentiable(gradients)

    def backward(ctx, *grads):
        _no_tangents("backward pass", *grads)
        return guarded(ctx, *grads) if torch.is_grad_enabled() else gradients(ctx, *grads)
    return backward


def _number(what, name, value):
    if torch.is_tensor(value):
        raise TypeError(f"{what}: {name} must be a number, not a tensor (it is read on the host and has no gradient)")
    value = float(value)
    if not abs(value) <= 3.4028234663852886e38:
        raise ValueError(f"{what}: {name} must be finite in 32 bits, got {value}")
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
    @_once
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
    differentiable.  Rows of x, weight and residual may be strided; alignment matters for speed only.  Rows of x and weight take
    up to 4 MiB, and so do rows of the result where x or weight gets a gradient."""
    _device_tensors("linear", ops.DTYPES, ("x", "weight", "bias", "residual"), x, weight, bias, residual)
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
    if x.dim() != 2:
        x, residual = x.reshape(M, K), None if residual is None else residual.reshape(M, N)
    _no_tangents("linear", x, weight, bias, residual)
    if _wants_grad(x, weight, bias, residual):
        if M and K and N * x.element_size() > 1 << 22 and _wants_grad(x, weight):       # what the backward pass takes
            raise ValueError(f"linear: rows of {N} results, more than 4 MiB, with gradients of x or weight")
        y = _Linear.apply(x, weight, bias, residual, activation, alpha, beta)
    else:
        y, _ = ops.linear(x, weight, bias, residual, activation, alpha, beta)
    return y if len(lead) == 1 else y.reshape(lead + (N,))


LogProbs = namedtuple("LogProbs", "logp entropy lse top_logp top_index")


def _probs_arguments(what, rows, cols, device, targets, weights, scale, top):
    """Checks what log_probs and bank_log_probs share -> (targets as i64, scale, top)."""
    if not torch.is_tensor(targets) or targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: targets must be an int64 or int32 tensor")
    if tuple(targets.shape) != (rows,):
        raise ValueError(f"{what}: targets must be [{rows}], got {tuple(targets.shape)}")
    if targets.device != device:
        if targets.is_cuda:
            raise RuntimeError(f"{what}: targets are on {targets.device}, the rows on {device}")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what}: targets are on the host, a capture takes none (the copy waits for the stream): copy them to the device before")
        if targets.numel() and (int(targets.min()) < -1 or int(targets.max()) >= cols):      # on the host: nothing to wait for
            raise ValueError(f"{what}: targets must lie in -1 .. {cols - 1}")
    if weights is not None:
        _device_tensors(what, (torch.float32,), ("weights",), weights)
        if weights.device != device:
            raise RuntimeError(f"{what}: weights are on {weights.device}, the rows on {device}")
        if tuple(weights.shape) not in ((cols,), (rows, cols)):
            raise ValueError(f"{what}: weights must be [{cols}] or [{rows}, {cols}], got {tuple(weights.shape)}")
        if weights.requires_grad:
            raise ValueError(f"{what}: weights are constants, they get no gradient: pass weights.detach()")
    if isinstance(top, bool) or int(top) != top or not 0 <= top <= 16:
        raise ValueError(f"{what}: top must be a whole number in 0 .. 16, got {top}")
    if targets.dtype != torch.int64 or targets.device != device:
        targets = targets.to(device=device, dtype=torch.int64)
    return targets, _number(what, "scale", scale), int(top)


def _results(out):
    return out.logp, out.entropy, out.lse, out.top_logp, out.top_index


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, weights, scale, top):
        out = ops.log_probs(logits, targets, weights, scale, top)
        ctx.save_for_backward(logits, targets, weights, out.stats)
        ctx.scale = scale
        if top:
            ctx.mark_non_differentiable(out.top_logp, out.top_index)
        ctx.set_materialize_grads(False)
        return _results(out)

    @staticmethod
    @_once
    def backward(ctx, g_logp, g_entropy, g_lse, *_):
        logits, targets, weights, stats = ctx.saved_tensors
        if g_logp is None and g_entropy is None and g_lse is None:
            return None, None, None, None, None
        return ops.log_probs_backward(logits, targets, weights, stats, g_logp, g_entropy, g_lse, ctx.scale), None, None, None, None


def log_probs(logits, targets, weights=None, scale=1.0, top=0):
    """Log probabilities of one place of every row of logits [S, V] under softmax(z), z = scale logits - weights.

    -> LogProbs(logp [S] of the targets, entropy [S], lse [S] = log sum exp z, top_logp [S, top], top_index [S, top]), statistics in
    float32 whatever the logits' type (float32, bfloat16, float16); top_logp and top_index (int64) are the `top` most probable places in
    descending order, the lowest place first among equal ones (None, None for top = 0; they carry no gradient).

    targets [S] int64 or int32: the place, or -1 for a row without a target (logp 0, no gradient through it).  Other values outside the row
    are refused where the tensor is on the host and give NaN in that row (values and gradient) where it is on the device, which is not read
    back.  Targets on the host cost a blocking copy.  weights float32, [V] for all rows or [S, V]: subtracted constants; +inf leaves the place
    out, whatever the logit there is (NaN too).  A row with nothing left: lse and logp -inf, entropy 0, top_index -1, gradient 0.  A row with a
    NaN or +inf left: NaN, top_index -1.  Fewer places left than `top`: -inf and -1 in their stead."""
    _device_tensors("log_probs", ops.DTYPES, ("logits",), logits)
    if logits.dim() != 2:
        raise ValueError(f"log_probs: logits must be [S, V], got {tuple(logits.shape)}")
    S, V = logits.shape
    targets, scale, top = _probs_arguments("log_probs", S, V, logits.device, targets, weights, scale, top)
    _no_tangents("log_probs", logits, weights)
    if _wants_grad(logits):
        return LogProbs(*_LogProbs.apply(logits, targets, weights, scale, top))
    return LogProbs(*_results(ops.log_probs(logits, targets, weights, scale, top, want_stats=False)))


class _BankLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, features, bank, targets, weights, scale, top):
        out = ops.bank_log_probs(features, bank, targets, weights, scale, top)
        ctx.save_for_backward(features, bank, targets, weights, out.stats)
        ctx.scale, ctx.top = scale, top
        if top:
            ctx.mark_non_differentiable(out.top_logp, out.top_index)
        ctx.set_materialize_grads(False)
        return _results(out)

    @staticmethod
    @_once
    def backward(ctx, g_logp, g_entropy, g_lse, *_):
        features, bank, targets, weights, stats = ctx.saved_tensors
        if g_logp is None and g_entropy is None and g_lse is None:
            return (None,) * 6
        grads = ops.bank_log_probs_backward(features, bank, targets, weights, stats, g_logp, g_entropy, g_lse, ctx.scale, ctx.top,
                                            ctx.needs_input_grad[:2])
        return (*grads, None, None, None, None)


def bank_log_probs(features, bank, targets, weights=None, scale=1.0, top=0):
    """log_probs(linear(features, bank), ...) without the [S, V] matrix: features [S, C] and bank [V, C], both float32 or both bfloat16, C up
    to 256, S and V below 2^24.  Scores are z = scale <feature, bank row> - weights, summed in 32 bits; arguments, results and rules are
    those of log_probs.  float32 rows are multiplied as three bfloat16 pieces (24 bits together): products are as exact as float32's, but
    an infinity in a row makes its scores NaN, whatever its sign.  Without weights and `top` scores beyond 2.3e38 count as infinities.
    Differentiable with respect to features and bank; the gradient computes the scores again instead of keeping them; it may be split in
    another way than the values, and two calls give the same bits."""
    _device_tensors("bank_log_probs", (torch.float32, torch.bfloat16), ("features", "bank"), features, bank)
    if features.dim() != 2 or bank.dim() != 2 or features.shape[1] != bank.shape[1]:
        raise ValueError(f"bank_log_probs: features must be [S, C] and bank [V, C], got {tuple(features.shape)} and {tuple(bank.shape)}")
    if not 1 <= features.shape[1] <= 256:
        raise ValueError(f"bank_log_probs: {features.shape[1]} channels (takes 1 to 256: use linear and log_probs)")
    S, V = features.shape[0], bank.shape[0]
    targets, scale, top = _probs_arguments("bank_log_probs", S, V, features.device, targets, weights, scale, top)
    _no_tangents("bank_log_probs", features, bank, weights)
    if _wants_grad(features, bank):
        return LogProbs(*_BankLogProbs.apply(features, bank, targets, weights, scale, top))
    return LogProbs(*_results(ops.bank_log_probs(features, bank, targets, weights, scale, top, want_stats=False)))
