"""Autograd wrapper (pysiglib/torch_api/torch_api.py:76-117): forward saves (path, signature),
backward un-multiplies the saved signature instead of storing per-step states."""
import torch

from .sig import sig as _sig_forward
from .sig import sig_backprop as _sig_backprop


class Sig(torch.autograd.Function):
    @staticmethod
    def forward(ctx, path, degree, time_aug, lead_lag, end_time, horner, scalar_term, n_jobs):
        out = _sig_forward(path, degree, time_aug=time_aug, lead_lag=lead_lag, end_time=end_time, horner=horner,
                           scalar_term=scalar_term, n_jobs=n_jobs)
        ctx.save_for_backward(path, out)
        ctx.args = (degree, time_aug, lead_lag, end_time, n_jobs)
        return out

    @staticmethod
    def backward(ctx, grad_output):
        path, out = ctx.saved_tensors
        degree, time_aug, lead_lag, end_time, n_jobs = ctx.args
        grad = _sig_backprop(path, out, grad_output, degree, time_aug=time_aug, lead_lag=lead_lag,
                             end_time=end_time, n_jobs=n_jobs)
        return grad, None, None, None, None, None, None, None


def sig(path, degree, *, time_aug=False, lead_lag=False, end_time=1., horner=True, scalar_term=False, n_jobs=1):
    """Differentiable ``sig``."""
    return Sig.apply(path, degree, time_aug, lead_lag, end_time, horner, scalar_term, n_jobs)


signature = sig


class SigCombine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, sig1, sig2, dimension, degree, time_aug, lead_lag):
        from .ops import sig_combine as _combine
        out = _combine(sig1, sig2, dimension, degree, time_aug=time_aug, lead_lag=lead_lag)
        ctx.save_for_backward(sig1, sig2)
        ctx.args = (dimension, degree, time_aug, lead_lag)
        return out

    @staticmethod
    def backward(ctx, grad_output):
        from .ops import sig_combine_backprop as _combine_backprop
        sig1, sig2 = ctx.saved_tensors
        dimension, degree, time_aug, lead_lag = ctx.args
        d1, d2 = _combine_backprop(grad_output, sig1, sig2, dimension, degree, time_aug=time_aug, lead_lag=lead_lag)
        return d1, d2, None, None, None, None


def sig_combine(sig1, sig2, dimension, degree, *, time_aug=False, lead_lag=False, n_jobs=1):
    """Differentiable ``sig_combine``."""
    return SigCombine.apply(sig1, sig2, dimension, degree, time_aug, lead_lag)


class TransformPath(torch.autograd.Function):
    @staticmethod
    def forward(ctx, path, time_aug, lead_lag, end_time):
        from .ops import transform_path as _transform
        ctx.args = (time_aug, lead_lag, end_time)
        return _transform(path, time_aug=time_aug, lead_lag=lead_lag, end_time=end_time)

    @staticmethod
    def backward(ctx, grad_output):
        from .ops import transform_path_backprop as _transform_backprop
        time_aug, lead_lag, end_time = ctx.args
        return _transform_backprop(grad_output, time_aug=time_aug, lead_lag=lead_lag, end_time=end_time), None, None, None


def transform_path(path, *, time_aug=False, lead_lag=False, end_time=1., n_jobs=1):
    """Differentiable ``transform_path``."""
    if (not time_aug) and (not lead_lag):
        return path
    return TransformPath.apply(path, time_aug, lead_lag, end_time)


class SigJoin(torch.autograd.Function):
    @staticmethod
    def forward(ctx, sig, displacement, dimension, degree, prepend):
        from .ops import sig_join as _join
        ctx.save_for_backward(sig, displacement)
        ctx.args = (dimension, degree, prepend)
        return _join(sig, displacement, dimension, degree, prepend=prepend)

    @staticmethod
    def backward(ctx, grad_output):
        from .ops import sig_join_backprop as _join_backprop
        sig, displacement = ctx.saved_tensors
        dimension, degree, prepend = ctx.args
        d_sig, d_disp = _join_backprop(grad_output, sig, displacement, dimension, degree, prepend=prepend)
        return d_sig, d_disp, None, None, None


def sig_join(sig, displacement, dimension, degree, *, prepend=False, n_jobs=1):
    """Differentiable ``sig_join``."""
    return SigJoin.apply(sig, displacement, dimension, degree, bool(prepend))


class SigCoef(torch.autograd.Function):
    @staticmethod
    def forward(ctx, path, words, time_aug, lead_lag, end_time):
        from .coef import sig_coef as _coef
        coefs = _coef(path, words, time_aug=time_aug, lead_lag=lead_lag, end_time=end_time, prefixes=True)
        ctx.save_for_backward(coefs, path)
        ctx.args = (words, time_aug, lead_lag, end_time)
        return coefs

    @staticmethod
    def backward(ctx, grad_output):
        from .coef import sig_coef_backprop as _coef_backprop
        coefs, path = ctx.saved_tensors
        words, time_aug, lead_lag, end_time = ctx.args
        grad = _coef_backprop(path, words, coefs, grad_output, time_aug=time_aug, lead_lag=lead_lag, end_time=end_time)
        return grad, None, None, None, None


def sig_coef(path, words, *, time_aug=False, lead_lag=False, end_time=1., prefixes=False, n_jobs=1):
    """Differentiable ``sig_coef``: computes the prefixes layout and, without ``prefixes``, keeps each word's last
    entry (pysiglib/torch_api/torch_api.py:156-202)."""
    coefs = SigCoef.apply(path, words, time_aug, lead_lag, end_time)
    if prefixes:
        return coefs
    word_list = [words] if isinstance(words, tuple) else words
    ends, pos = [], 0
    for w in word_list:
        pos += max(len(w), 1)
        ends.append(pos - 1)
    return coefs[..., ends].contiguous()


class SigToLogSig(torch.autograd.Function):
    @staticmethod
    def forward(ctx, sig_, dimension, degree, time_aug, lead_lag, method):
        from .log_sig import sig_to_log_sig as _to_log
        ctx.save_for_backward(sig_)
        ctx.args = (dimension, degree, time_aug, lead_lag, method)
        return _to_log(sig_, dimension, degree, time_aug=time_aug, lead_lag=lead_lag, method=method)

    @staticmethod
    def backward(ctx, grad_output):
        from .log_sig import sig_to_log_sig_backprop as _to_log_backprop
        (sig_,) = ctx.saved_tensors
        dimension, degree, time_aug, lead_lag, method = ctx.args
        grad = _to_log_backprop(sig_, grad_output, dimension, degree, time_aug=time_aug, lead_lag=lead_lag, method=method)
        return grad, None, None, None, None, None


def sig_to_log_sig(sig_, dimension, degree, *, time_aug=False, lead_lag=False, method=1, n_jobs=1):
    """Differentiable ``sig_to_log_sig``."""
    return SigToLogSig.apply(sig_, dimension, degree, time_aug, lead_lag, method)


def log_sig(path, degree, *, time_aug=False, lead_lag=False, end_time=1., method=1, scalar_term=False, n_jobs=1):
    """Differentiable ``log_sig``: the differentiable signature followed by the differentiable ``sig_to_log_sig``."""
    sig_ = sig(path, degree, time_aug=time_aug, lead_lag=lead_lag, end_time=end_time, scalar_term=scalar_term)
    return sig_to_log_sig(sig_, path.shape[-1], degree, time_aug=time_aug, lead_lag=lead_lag, method=method)


class _Gradients(torch.autograd.Function):
    @staticmethod
    def forward(ctx, anchor, *grads):
        return grads

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("the gradients of pysiglib_amd's sequence layers are not differentiable")


def _once(*grads):
    """Gradients for a backward function to return.  Where a graph of them is asked for, they refuse to be differentiated
    instead of being constants in it."""
    if not torch.is_grad_enabled():
        return grads
    at = [i for i, g in enumerate(grads) if g is not None]
    out = list(grads)
    for i, g in zip(at, _Gradients.apply(torch.empty(0, requires_grad=True), *(grads[i] for i in at))):
        out[i] = g
    return tuple(out)


class LinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, log_decay, initial_state, offsets):
        from .sequence import linear_recurrence as _recurrence
        h, final = _recurrence(x, log_decay, initial_state=initial_state, offsets=offsets)
        ctx.save_for_backward(h, log_decay, initial_state, offsets)
        ctx.set_materialize_grads(False)
        return h, final

    @staticmethod
    def backward(ctx, grad_h, grad_final):
        from .sequence import linear_recurrence_backprop as _recurrence_backprop
        h, log_decay, initial_state, offsets = ctx.saved_tensors
        grad_h = torch.zeros_like(h) if grad_h is None else grad_h
        dx, dg, d0 = _recurrence_backprop(h, log_decay, grad_h, grad_final=grad_final, initial_state=initial_state,
                                          offsets=offsets)
        return _once(dx, dg, d0 if initial_state is not None else None, None)


def linear_recurrence(x, log_decay, *, initial_state=None, offsets=None):
    """Differentiable ``linear_recurrence``."""
    return LinearRecurrence.apply(x, log_decay, initial_state, offsets)


class NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        from .sequence import norm_rotary as _norm_rotary
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.args = (eps, interleaved)
        return _norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, eps=eps, interleaved=interleaved)

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        from .sequence import norm_rotary_backprop as _norm_rotary_backprop
        eps, interleaved = ctx.args
        grads = _norm_rotary_backprop(grad_q, grad_k, *ctx.saved_tensors, eps=eps, interleaved=interleaved)
        return _once(*grads, None, None, None, None, None)


def norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, *, eps=1e-6, interleaved=False):
    """Differentiable ``norm_rotary`` (with respect to queries, keys and both weights)."""
    return NormRotary.apply(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)


class Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_offsets, k_offsets, causal, scale):
        from .sequence import attention as _attention
        out, lse = _attention(q, k, v, q_offsets, k_offsets, causal=causal, scale=scale)
        ctx.save_for_backward(q, k, v, out, lse, q_offsets, k_offsets)
        ctx.args = (causal, scale)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        from .sequence import attention_backprop as _attention_backprop
        q, k, v, out, lse, q_offsets, k_offsets = ctx.saved_tensors
        causal, scale = ctx.args
        grads = _attention_backprop(grad_out, q, k, v, out, lse, q_offsets, k_offsets, causal=causal, scale=scale)
        return _once(*grads, None, None, None, None)


def attention(q, k, v, q_offsets, k_offsets, *, causal=True, scale=None):
    """Differentiable ``attention`` of whole sequences; the output alone, without the sums' logarithms."""
    return Attention.apply(q, k, v, q_offsets, k_offsets, causal, scale)


class NormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        from .sequence import norm_residual as _norm_residual
        out, total = _norm_residual(x, residual, weight, eps=eps)
        ctx.save_for_backward(total, weight)
        ctx.eps, ctx.alone, ctx.dtype = eps, residual is None, x.dtype
        ctx.set_materialize_grads(False)
        return (out, None) if ctx.alone else (out, total)

    @staticmethod
    def backward(ctx, grad_out, grad_total):
        from .sequence import norm_residual_backprop as _norm_residual_backprop
        total, weight = ctx.saved_tensors
        if grad_out is None:
            if grad_total is None:
                return None, None, None, None
            grad_out = torch.zeros(total.shape, dtype=ctx.dtype, device=total.device)
        dx, dr, dw = _norm_residual_backprop(grad_out, total, weight, grad_total=grad_total, eps=ctx.eps)
        return _once(dx, None if ctx.alone else dr, dw, None)


def norm_residual(x, residual, weight, *, eps=1e-6):
    """Differentiable ``norm_residual``; without a residual ``total`` is ``x`` itself."""
    out, total = NormResidual.apply(x, residual, weight, eps)
    return out, x if residual is None else total


class CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial_state, offsets, silu):
        from .sequence import causal_conv as _causal_conv
        y, final = _causal_conv(x, weight, bias, initial_state=initial_state, offsets=offsets, silu=silu)
        ctx.save_for_backward(x, weight, bias, initial_state, offsets)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    def backward(ctx, grad_y, grad_final):
        from .sequence import causal_conv_backprop as _causal_conv_backprop
        x, weight, bias, initial_state, offsets = ctx.saved_tensors
        grad_y = torch.zeros_like(x) if grad_y is None else grad_y
        dx, dw, db, d0 = _causal_conv_backprop(grad_y, x, weight, bias, grad_final=grad_final, initial_state=initial_state, offsets=offsets,
                                               silu=ctx.silu)
        return _once(dx, dw, db, d0 if initial_state is not None else None, None, None)


def causal_conv(x, weight, bias=None, *, initial_state=None, offsets=None, silu=True):
    """Differentiable ``causal_conv``."""
    return CausalConv.apply(x, weight, bias, initial_state, offsets, silu)


class SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, a, b, c, d, z, delta_bias, initial_state, softplus, offsets):
        from .sequence import selective_scan as _selective_scan
        y, final = _selective_scan(x, delta, a, b, c, d=d, z=z, delta_bias=delta_bias, softplus=softplus, initial_state=initial_state, offsets=offsets)
        ctx.save_for_backward(x, delta, a, b, c, d, z, delta_bias, initial_state, offsets)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    def backward(ctx, grad_y, grad_final):
        from .sequence import selective_scan_backprop as _selective_scan_backprop
        x, delta, a, b, c, d, z, delta_bias, initial_state, offsets = ctx.saved_tensors
        grad_y = torch.zeros_like(x) if grad_y is None else grad_y
        grads = _selective_scan_backprop(grad_y, x, delta, a, b, c, d=d, z=z, delta_bias=delta_bias, softplus=ctx.softplus, grad_final=grad_final,
                                         initial_state=initial_state, offsets=offsets)
        return _once(*grads[:8], grads[8] if initial_state is not None else None, None, None)


def selective_scan(x, delta, a, b, c, *, d=None, z=None, delta_bias=None, softplus=True, initial_state=None, offsets=None):
    """Differentiable ``selective_scan``."""
    return SelectiveScan.apply(x, delta, a, b, c, d, z, delta_bias, initial_state, softplus, offsets)
