"""Layers of a sequence model over path features: the gated linear recurrence, norms of queries and keys with the rotation by
position, and causal attention over packed sequences; the norm of the residual stream, the short causal convolution and the selective scan
of a state space block; each with its gradients and its form for single tokens.

They take the place after the signature: windows of a path give signatures, these are the tokens.  No counterpart in the
reference.  Tensors are float32, bfloat16 or float16 on one GPU; sums, states and norms are 32-bit throughout.  The work is
enqueued on the current stream of the tensors' device and not waited for; scratch comes from torch's allocator.  Tensors
may have gaps between their rows (parts of one projection, say); only the last axis has to be contiguous, others are copied.

Sequences of different lengths are packed behind each other, with ``offsets`` (int32, on the GPU): sequence ``i`` has the rows
``offsets[i]`` to ``offsets[i + 1]``; the offsets ascend, usually from 0 to the number of rows.  They are not read on the host.
Where there are rows before the first or behind the last of them, outputs and gradients hold no values there; offsets that leave
the tensors are cut to them.
"""
import math

import torch

from ._loader import (CUSIG_ATTENTION, CUSIG_ATTENTION_BACKPROP, CUSIG_ATTENTION_BACKPROP_WORKSPACE,
                      CUSIG_ATTENTION_WORKSPACE, CUSIG_CAUSAL_CONV, CUSIG_CAUSAL_CONV_BACKPROP, CUSIG_CAUSAL_CONV_BACKPROP_WORKSPACE,
                      CUSIG_CAUSAL_CONV_STEP, CUSIG_LINEAR_RECURRENCE, CUSIG_LINEAR_RECURRENCE_BACKPROP, CUSIG_LINEAR_RECURRENCE_STEP,
                      CUSIG_LINEAR_RECURRENCE_WORKSPACE, CUSIG_NORM_ROTARY, CUSIG_NORM_ROTARY_BACKPROP,
                      CUSIG_NORM_ROTARY_BACKPROP_WORKSPACE, CUSIG_NORM_RESIDUAL, CUSIG_NORM_RESIDUAL_BACKPROP,
                      CUSIG_NORM_RESIDUAL_BACKPROP_WORKSPACE, CUSIG_SELECTIVE_SCAN, CUSIG_SELECTIVE_SCAN_BACKPROP,
                      CUSIG_SELECTIVE_SCAN_BACKPROP_WORKSPACE, CUSIG_SELECTIVE_SCAN_STEP, CUSIG_SELECTIVE_SCAN_WORKSPACE, SEQUENCE_DTYPES)
from .data_handlers import on_device
from .error_codes import err_msg
from .param_checks import check_type

_CODES = {getattr(torch, name): code for name, code in SEQUENCE_DTYPES.items()}
_stream_of = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _tensor(value, name, rank=None, like=None):
    """Checks that ``value`` is a GPU tensor of a supported type (of the type and device of ``like``)."""
    if not isinstance(value, torch.Tensor):
        raise TypeError(name + " must be a torch tensor, got " + type(value).__name__ + " instead")
    if like is None:
        if value.dtype not in _CODES:
            raise TypeError(name + ".dtype must be float32, bfloat16 or float16, got " + str(value.dtype) + " instead")
        if not value.is_cuda:
            raise RuntimeError(name + " must be on the GPU: pysiglib_amd has no CPU implementation")
    else:
        if value.dtype != like.dtype:
            raise TypeError(name + ".dtype must be " + str(like.dtype) + ", got " + str(value.dtype) + " instead")
        if value.device != like.device:
            raise ValueError(name + " must be on " + str(like.device) + ", got " + str(value.device))
    if rank is not None and value.dim() != rank:
        raise ValueError(name + " must have rank " + str(rank) + ", got rank " + str(value.dim()) + ".")
    return value


def _other(value, name, dtype, shape, device):
    """A contiguous tensor of a given type, shape and device."""
    if not isinstance(value, torch.Tensor):
        raise TypeError(name + " must be a torch tensor, got " + type(value).__name__ + " instead")
    if value.dtype != dtype:
        raise TypeError(name + ".dtype must be " + str(dtype) + ", got " + str(value.dtype) + " instead")
    if value.shape != shape:
        raise ValueError(name + " must have shape " + str(tuple(shape)) + ", got " + str(tuple(value.shape)))
    if value.device != device:
        raise ValueError(name + " must be on " + str(device) + ", got " + str(value.device))
    return value if value.is_contiguous() else value.contiguous()


def _offsets(value, name, device):
    if not isinstance(value, torch.Tensor):
        raise TypeError(name + " must be a torch tensor, got " + type(value).__name__ + " instead")
    if value.dtype != torch.int32:
        raise TypeError(name + ".dtype must be torch.int32, got " + str(value.dtype) + " instead")
    if value.dim() != 1 or value.shape[0] < 1:
        raise ValueError(name + " must have rank 1 and at least one entry")
    if value.device != device:
        raise ValueError(name + " must be on " + str(device) + ", got " + str(value.device))
    return value if value.is_contiguous() else value.contiguous()


def _call(fn, name, device, *args):
    index = device.index
    if index == _current_device():
        code = fn(*args, _stream_of(index))
    else:
        with on_device(device):
            code = fn(*args, _stream_of(index))
    if code:
        raise Exception("Error in pysiglib." + name + ": " + err_msg(code))


def _rows(x):
    """A tensor of rank 2 or more as rows a fixed distance apart: (tensor that holds them, distance)."""
    shape = x.shape
    if x.is_contiguous():
        return x, shape[-1]
    if (x.stride(-1) == 1 or shape[-1] <= 1) and x.stride(-2) <= 1 << 20:       # the scan's offsets inside a chunk are 32-bit
        step = x.stride(-2)
        want = step
        for axis in range(x.dim() - 2, -1, -1):
            if shape[axis] != 1 and x.stride(axis) != want:
                break
            want = want * shape[axis] if shape[axis] != 1 else want
        else:
            return x, step
    return x.contiguous(), shape[-1]


def _sequences(x, offsets, name):
    """(number of sequences, length or 0, rows, leading shape of the states, offsets' address)."""
    shape = x.shape
    if offsets is None:
        length = shape[-2]
        lead = shape[:-2]
        n = math.prod(lead)
        return n, length, n * length, lead, 0
    if len(shape) != 2:
        raise ValueError(name + " must have rank 2 where offsets are given, got rank " + str(len(shape)) + ".")
    n = offsets.shape[0] - 1
    return n, 0, shape[0], (n,), offsets.data_ptr()


def _workspace(size, device):
    return torch.empty(size, dtype=torch.uint8, device=device)


def linear_recurrence(x, log_decay, *, initial_state=None, offsets=None):
    """``h_t = exp(log_decay_t) * h_{t-1} + x_t`` for each channel, over sequences of any length.

    ``x``, ``log_decay``: ``(..., length, channels)``, or with ``offsets`` ``(rows, channels)``, the sequences packed.
    ``log_decay`` is meant to be at most 0; where its exponential is zero in 32 bits (``-inf``, and below about -87) it forgets the
    state, also one that is not finite.  ``initial_state``: float32 ``(..., channels)``, with
    ``offsets`` ``(sequences, channels)``; zero where it is not given.

    Returns ``(h, final_state)``: ``h`` like ``x``, the states behind the last steps like ``initial_state``.
    """
    _tensor(x, "x")
    if x.dim() < 2:
        raise ValueError("x must have at least rank 2, got rank " + str(x.dim()) + ".")
    _tensor(log_decay, "log_decay", like=x)
    if log_decay.shape != x.shape:
        raise ValueError("x and log_decay must have the same shape")
    device, channels = x.device, x.shape[-1]
    if offsets is not None:
        offsets = _offsets(offsets, "offsets", device)
    n, length, rows, lead, at = _sequences(x, offsets, "x")
    state = (*lead, channels)
    if initial_state is not None:
        initial_state = _other(initial_state, "initial_state", torch.float32, state, device)
    h = torch.empty(x.shape, dtype=x.dtype, device=device)
    final = torch.empty(state, dtype=torch.float32, device=device)
    x, x_step = _rows(x)
    log_decay, decay_step = _rows(log_decay)
    code = _CODES[x.dtype]
    size = CUSIG_LINEAR_RECURRENCE_WORKSPACE(code, rows, n, channels)
    space = _workspace(size, device) if size else None
    _call(CUSIG_LINEAR_RECURRENCE, "linear_recurrence", device, code, x.data_ptr(), log_decay.data_ptr(),
          0 if initial_state is None else initial_state.data_ptr(), h.data_ptr(), final.data_ptr(), at, n, length, rows, channels,
          x_step, decay_step, space.data_ptr() if size else 0, size)
    return h, final


def linear_recurrence_backprop(h, log_decay, grad_h, *, grad_final=None, initial_state=None, offsets=None):
    """Gradients of ``linear_recurrence`` from its output ``h`` and the gradients of its outputs (``grad_final`` float32 like
    the final state, zero where it is not given).  Returns ``(grad_x, grad_log_decay, grad_initial_state)``, the last in
    float32.

    ``grad_log_decay`` is a product with the state before the step, which is taken from ``h`` as it was rounded: in 16-bit types
    its error is about 1.4 times that of a result rounded once, and where ``h`` passed float16's range it is not finite."""
    _tensor(h, "h")
    if h.dim() < 2:
        raise ValueError("h must have at least rank 2, got rank " + str(h.dim()) + ".")
    _tensor(log_decay, "log_decay", like=h)
    _tensor(grad_h, "grad_h", like=h)
    if log_decay.shape != h.shape or grad_h.shape != h.shape:
        raise ValueError("h, log_decay and grad_h must have the same shape")
    device, channels = h.device, h.shape[-1]
    if offsets is not None:
        offsets = _offsets(offsets, "offsets", device)
    n, length, rows, lead, at = _sequences(h, offsets, "h")
    state = (*lead, channels)
    if initial_state is not None:
        initial_state = _other(initial_state, "initial_state", torch.float32, state, device)
    if grad_final is not None:
        grad_final = _other(grad_final, "grad_final", torch.float32, state, device)
    dx = torch.empty(h.shape, dtype=h.dtype, device=device)
    dg = torch.empty(h.shape, dtype=h.dtype, device=device)
    d0 = torch.empty(state, dtype=torch.float32, device=device)
    h = h if h.is_contiguous() else h.contiguous()
    log_decay, decay_step = _rows(log_decay)
    grad_h, grad_step = _rows(grad_h)
    code = _CODES[h.dtype]
    size = CUSIG_LINEAR_RECURRENCE_WORKSPACE(code, rows, n, channels)
    space = _workspace(size, device) if size else None
    _call(CUSIG_LINEAR_RECURRENCE_BACKPROP, "linear_recurrence_backprop", device, code, h.data_ptr(), log_decay.data_ptr(),
          grad_h.data_ptr(), 0 if grad_final is None else grad_final.data_ptr(),
          0 if initial_state is None else initial_state.data_ptr(), dx.data_ptr(), dg.data_ptr(), d0.data_ptr(), at, n, length,
          rows, channels, decay_step, grad_step, space.data_ptr() if size else 0, size)
    return dx, dg, d0


def linear_recurrence_step(x, log_decay, state):
    """One step of ``linear_recurrence`` for single tokens: ``x``, ``log_decay`` ``(..., channels)``; ``state`` float32 of the same
    shape, contiguous, is replaced by ``exp(log_decay) * state + x``.  Returns the new state rounded to the type of ``x``."""
    _tensor(x, "x")
    _tensor(log_decay, "log_decay", like=x)
    shape, device = x.shape, x.device
    if log_decay.shape != shape or len(shape) < 1:
        raise ValueError("x and log_decay must have the same shape, of rank 1 at least")
    if _other(state, "state", torch.float32, shape, device) is not state:
        raise ValueError("state must be contiguous: it is written")
    h = torch.empty(shape, dtype=x.dtype, device=device)
    if len(shape) == 1:
        x, log_decay = x[None], log_decay[None]
    x, x_step = _rows(x)
    log_decay, decay_step = _rows(log_decay)
    channels = shape[-1]
    _call(CUSIG_LINEAR_RECURRENCE_STEP, "linear_recurrence_step", device, _CODES[x.dtype], x.data_ptr(), log_decay.data_ptr(),
          state.data_ptr(), h.data_ptr(), h.numel() // channels if channels else 0, channels, x_step, decay_step)
    torch.autograd.graph.increment_version(state)       # written through its address: operations that kept it find out
    return h


def rotary_tables(length, rotary_dim, *, base=10000., scale=1., device="cuda"):
    """Tables for ``norm_rotary``: ``(cos, sin)``, float32 ``(length, rotary_dim / 2)``, of the angles
    ``position / scale * base ** (-2 i / rotary_dim)``; ``scale`` above 1 stretches positions for longer contexts."""
    check_type(length, "length", int)
    check_type(rotary_dim, "rotary_dim", int)
    if rotary_dim < 0 or rotary_dim % 2 or length < 0:
        raise ValueError("length must not be negative, and rotary_dim an even number that is not negative")
    half = rotary_dim // 2
    at = torch.arange(length, dtype=torch.float64, device=device) / scale
    angle = at[:, None] * base ** (-torch.arange(half, dtype=torch.float64, device=device) / max(half, 1))
    return angle.cos().float(), angle.sin().float()


_APART = 1 << 23        # tokens of the attention are nearer than that: its kernels' offsets inside a tile are 32-bit


def _heads(x, name, like, rows=None, dim=None, apart=None):
    """(tokens, heads, dim) whose last axis is contiguous, and the distances of its tokens and heads; tokens that are ``apart``
    or further are copied."""
    _tensor(x, name, 3, like)
    if (rows is not None and x.shape[0] != rows) or (dim is not None and x.shape[2] != dim):
        raise ValueError(name + " must have shape (" + str(rows) + ", heads, " + str(dim) + "), got " + str(tuple(x.shape)))
    if x.shape[0] <= 1:         # no next token: what the stride says has no meaning
        x = x if x.stride(2) == 1 or x.shape[2] <= 1 else x.contiguous()
        return x, x.shape[1] * x.shape[2], x.stride(1)
    if (x.stride(2) != 1 and x.shape[2] > 1) or (apart is not None and x.stride(0) >= apart):
        x = x.contiguous()
    return x, x.stride(0), x.stride(1)


def _rotary_args(q, k, q_weight, k_weight, cos, sin, positions, interleaved):
    check_type(interleaved, "interleaved", bool)
    q, q_token, q_head = _heads(q, "q", None)
    tokens, heads, dim = q.shape
    k, k_token, k_head = _heads(k, "k", q, tokens, dim)
    device = q.device
    q_weight = _other(q_weight, "q_weight", torch.float32, (dim,), device)
    k_weight = _other(k_weight, "k_weight", torch.float32, (dim,), device)
    _tensor(cos, "cos", 2, q_weight)
    cos, sin = _other(cos, "cos", torch.float32, cos.shape, device), _other(sin, "sin", torch.float32, cos.shape, device)
    positions = _other(positions, "positions", torch.int32, (tokens,), device)
    rotary = 2 * cos.shape[1]
    if dim % 2 or dim > 256 or dim < 2:
        raise ValueError("q and k must have 2 to 256 channels to a head, an even number, got " + str(dim))
    if rotary > dim:
        raise ValueError("cos and sin turn " + str(rotary) + " channels, a head has " + str(dim))
    return (q, k, q_weight, k_weight, cos, sin, positions,
            (tokens, heads, k.shape[1], dim, rotary, cos.shape[0], q_token, q_head, k_token, k_head))


def norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, *, eps=1e-6, interleaved=False):
    """Root-mean-square norm of every head of ``q`` and ``k`` with a weight for each channel, then the rotation of the first
    channels by the token's position, in one pass.

    ``q`` ``(tokens, heads, dim)``, ``k`` ``(tokens, key heads, dim)``, parts of one projection or not; ``q_weight``, ``k_weight``
    float32 ``(dim,)``; ``cos``, ``sin`` float32 ``(positions, rotary_dim / 2)``, see ``rotary_tables``; ``positions`` int32
    ``(tokens,)``.  The pairs that turn are channels ``i`` and ``i + rotary_dim / 2``, with ``interleaved`` ``2 i`` and
    ``2 i + 1``; channels behind ``rotary_dim`` are only normed.  A position outside the tables gives NaN.

    Returns ``(q, k)``, normed and turned, contiguous.
    """
    q, k, q_weight, k_weight, cos, sin, positions, sizes = _rotary_args(q, k, q_weight, k_weight, cos, sin, positions, interleaved)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=q.device)
    _call(CUSIG_NORM_ROTARY, "norm_rotary", q.device, _CODES[q.dtype], q.data_ptr(), k.data_ptr(), q_weight.data_ptr(),
          k_weight.data_ptr(), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), *sizes,
          eps, interleaved)
    return q_out, k_out


def norm_rotary_backprop(grad_q, grad_k, q, k, q_weight, k_weight, cos, sin, positions, *, eps=1e-6, interleaved=False):
    """Gradients of ``norm_rotary`` from the gradients of its outputs and its inputs.  Returns
    ``(grad_q, grad_k, grad_q_weight, grad_k_weight)``; the weights' are summed over tokens and heads in a fixed order."""
    q, k, q_weight, k_weight, cos, sin, positions, sizes = _rotary_args(q, k, q_weight, k_weight, cos, sin, positions, interleaved)
    grad_q, gq_token, gq_head = _heads(grad_q, "grad_q", q)
    grad_k, gk_token, gk_head = _heads(grad_k, "grad_k", q)
    if grad_q.shape != q.shape or grad_k.shape != k.shape:
        raise ValueError("grad_q and grad_k must have the shapes of q and k")
    device, dim = q.device, q.shape[2]
    dq = torch.empty(q.shape, dtype=q.dtype, device=device)
    dk = torch.empty(k.shape, dtype=q.dtype, device=device)
    dw = torch.empty((2, dim), dtype=torch.float32, device=device)
    size = CUSIG_NORM_ROTARY_BACKPROP_WORKSPACE(dim)
    space = _workspace(size, device)
    _call(CUSIG_NORM_ROTARY_BACKPROP, "norm_rotary_backprop", device, _CODES[q.dtype], grad_q.data_ptr(), grad_k.data_ptr(),
          q.data_ptr(), k.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(), cos.data_ptr(), sin.data_ptr(),
          positions.data_ptr(), dq.data_ptr(), dk.data_ptr(), dw.data_ptr(), dw.data_ptr() + 4 * dim, *sizes, gq_token, gq_head,
          gk_token, gk_head, eps, interleaved, space.data_ptr(), size)
    return dq, dk, dw[0], dw[1]


def _attention_args(q, k, v, q_offsets, k_offsets, causal, scale):
    check_type(causal, "causal", bool)
    q, q_token, q_head = _heads(q, "q", None, apart=_APART)
    if q.dtype == torch.float32:
        raise TypeError("q.dtype must be bfloat16 or float16, got torch.float32 instead")
    dim, device = q.shape[2], q.device
    k, k_token, k_head = _heads(k, "k", q, None, dim, _APART)
    v, v_token, v_head = _heads(v, "v", q, k.shape[0], dim, _APART)
    heads, kv_heads = q.shape[1], k.shape[1]
    if v.shape[1] != kv_heads:
        raise ValueError("k and v must have the same heads")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError("the heads of q must be a multiple of those of k, got " + str(heads) + " and " + str(kv_heads))
    if dim < 8 or dim > 128 or dim % 8:
        raise ValueError("q, k and v must have 8 to 128 channels to a head, a multiple of 8, got " + str(dim))
    q_offsets, k_offsets = _offsets(q_offsets, "q_offsets", device), _offsets(k_offsets, "k_offsets", device)
    if q_offsets.shape != k_offsets.shape:
        raise ValueError("q_offsets and k_offsets must have the same length")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("scale must be positive and finite, got " + str(scale))
    return (q, k, v, q_offsets, k_offsets, (q.shape[0], k.shape[0], q_offsets.shape[0] - 1, heads, kv_heads, dim),
            (q_token, q_head, k_token, k_head, v_token, v_head, scale, causal))


def attention(q, k, v, q_offsets, k_offsets, *, k_lengths=None, causal=True, scale=None):
    """Softmax attention over packed sequences: query ``j`` of a sequence with ``n`` queries and ``m`` keys sees, with ``causal``,
    the keys up to ``j + m - n`` (both count from the sequences' ends), otherwise all of them.  A query that sees no key gets 0.

    ``q`` ``(rows, heads, dim)``, ``k`` and ``v`` ``(key rows, key heads, dim)``, bfloat16 or float16; ``heads`` is a multiple of the
    key heads, which neighbouring heads share; ``dim`` a multiple of 8 up to 128.  ``q_offsets``, ``k_offsets``: where sequences
    begin, see above.  ``k_lengths`` (int32, a number for each sequence): only that many keys from ``k_offsets[i]`` on are in
    use, as in a cache with room for more: with one query to each sequence this is the form for single tokens.  ``scale`` of
    the scores: ``dim ** -0.5`` where it is not given.

    Returns ``(out, lse)``: ``out`` like ``q``, and the logarithm of the sum of exponentials of each query's scores, float32
    ``(rows, heads)``.
    """
    q, k, v, q_offsets, k_offsets, sizes, rest = _attention_args(q, k, v, q_offsets, k_offsets, causal, scale)
    device = q.device
    if k_lengths is not None:
        k_lengths = _other(k_lengths, "k_lengths", torch.int32, (sizes[2],), device)
    out = torch.empty(q.shape, dtype=q.dtype, device=device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=device)
    size = CUSIG_ATTENTION_WORKSPACE(*sizes)
    space = _workspace(size, device) if size else None
    _call(CUSIG_ATTENTION, "attention", device, _CODES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), q_offsets.data_ptr(),
          k_offsets.data_ptr(), 0 if k_lengths is None else k_lengths.data_ptr(), out.data_ptr(), lse.data_ptr(), *sizes, *rest,
          space.data_ptr() if size else 0, size)
    return out, lse


def attention_backprop(grad_out, q, k, v, out, lse, q_offsets, k_offsets, *, causal=True, scale=None):
    """Gradients of ``attention`` (whole sequences, without ``k_lengths``) from the gradient of ``out``, the inputs and both
    outputs.  Returns ``(grad_q, grad_k, grad_v)``; the same inputs give the same bits."""
    q, k, v, q_offsets, k_offsets, sizes, rest = _attention_args(q, k, v, q_offsets, k_offsets, causal, scale)
    device, dtype = q.device, q.dtype
    grad_out, g_token, g_head = _heads(grad_out, "grad_out", q, q.shape[0], q.shape[2], _APART)
    if grad_out.shape != q.shape:
        raise ValueError("grad_out must have the shape of q")
    out = _other(out, "out", dtype, q.shape, device)
    lse = _other(lse, "lse", torch.float32, q.shape[:2], device)
    dq, dk, dv = (torch.empty(t.shape, dtype=dtype, device=device) for t in (q, k, v))
    size = CUSIG_ATTENTION_BACKPROP_WORKSPACE(*sizes[:4], sizes[5])
    space = _workspace(size, device)
    _call(CUSIG_ATTENTION_BACKPROP, "attention_backprop", device, _CODES[dtype], grad_out.data_ptr(), q.data_ptr(), k.data_ptr(),
          v.data_ptr(), out.data_ptr(), lse.data_ptr(), q_offsets.data_ptr(), k_offsets.data_ptr(), dq.data_ptr(), dk.data_ptr(),
          dv.data_ptr(), *sizes, *rest[:6], g_token, g_head, *rest[6:], space.data_ptr(), size)
    return dq, dk, dv


def _norm_args(x, residual, weight):
    """(x, its rows' distance, residual or None, its rows' distance, the sum's type, weight, rows, channels)."""
    _tensor(x, "x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 16384:
        raise ValueError("x must have rows of 1 to 16384 channels")
    channels, device = x.shape[-1], x.device
    weight = _other(weight, "weight", torch.float32, (channels,), device)
    step = 0
    if residual is not None:
        if not isinstance(residual, torch.Tensor):
            raise TypeError("residual must be a torch tensor, got " + type(residual).__name__ + " instead")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError("residual.dtype must be " + str(x.dtype) + " or torch.float32, got " + str(residual.dtype) + " instead")
        if residual.shape != x.shape:
            raise ValueError("x and residual must have the same shape")
        if residual.device != device:
            raise ValueError("residual must be on " + str(device) + ", got " + str(residual.device))
        residual, step = _rows(residual if residual.dim() > 1 else residual[None])
    rows = x.numel() // channels
    x, x_step = _rows(x if x.dim() > 1 else x[None])
    return x, x_step, residual, step, x.dtype if residual is None else residual.dtype, weight, rows, channels


def norm_residual(x, residual, weight, *, eps=1e-6):
    """``total = x + residual`` and its root-mean-square norm with a weight for each channel, in one pass.

    ``x`` ``(..., channels)``, up to 16384 of them; ``residual`` of the same shape, in the type of ``x`` or float32, or None: ``total`` is then
    ``x`` itself; ``weight`` float32 ``(channels,)``.  The norm is of ``total`` as it is stored, in the residual's type.

    Returns ``(out, total)``: ``out`` in the type of ``x``, contiguous.
    """
    shape, like = x.shape if isinstance(x, torch.Tensor) else None, x
    x, x_step, residual, step, kind, weight, rows, channels = _norm_args(x, residual, weight)
    out = torch.empty(shape, dtype=x.dtype, device=x.device)
    total = like if residual is None else torch.empty(shape, dtype=kind, device=x.device)
    _call(CUSIG_NORM_RESIDUAL, "norm_residual", x.device, _CODES[x.dtype], _CODES[kind], x.data_ptr(),
          0 if residual is None else residual.data_ptr(), weight.data_ptr(), out.data_ptr(), 0 if residual is None else total.data_ptr(),
          0, rows, channels, x_step, step, eps)
    return out, total


def norm_residual_float8(x, residual, weight, *, eps=1e-6):
    """``norm_residual`` with its output in 8 bits: ``out`` is ``float8_e4m3fn`` and stands for ``out * scales``, ``scales`` float32
    ``(..., 1)`` the largest value of each row divided by 448 (1 where that is zero, or the row holds NaN).  A row that holds an infinity has that scale:
    its finite values are then zero and its infinities NaN, the quotients by it.  Returns ``(out, scales, total)``."""
    shape, like = x.shape if isinstance(x, torch.Tensor) else None, x
    x, x_step, residual, step, kind, weight, rows, channels = _norm_args(x, residual, weight)
    out = torch.empty(shape, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty((*shape[:-1], 1), dtype=torch.float32, device=x.device)
    total = like if residual is None else torch.empty(shape, dtype=kind, device=x.device)
    if rows:
        _call(CUSIG_NORM_RESIDUAL, "norm_residual_float8", x.device, _CODES[x.dtype], _CODES[kind], x.data_ptr(),
              0 if residual is None else residual.data_ptr(), weight.data_ptr(), out.data_ptr(), 0 if residual is None else total.data_ptr(),
              scales.data_ptr(), rows, channels, x_step, step, eps)
    return out, scales, total


def norm_residual_backprop(grad_out, total, weight, *, grad_total=None, eps=1e-6):
    """Gradients of ``norm_residual`` from the gradients of its outputs (``grad_total`` like ``total``, zero where it is not given) and
    ``total``.  Returns ``(grad_x, grad_residual, grad_weight)``: the first in the type of ``grad_out``, which is that of ``x``, the second in that of
    ``total`` (where the types are the same, both are one tensor); the weight's is summed over the rows in a fixed order."""
    _tensor(grad_out, "grad_out")
    shape, dtype = grad_out.shape, grad_out.dtype
    if not isinstance(total, torch.Tensor):
        raise TypeError("total must be a torch tensor, got " + type(total).__name__ + " instead")
    total_step = _norm_args(grad_out, total, weight)
    grad_out, grad_step, total, step, kind, weight, rows, channels = total_step
    after = 0
    if grad_total is not None:
        _tensor(grad_total, "grad_total", like=total)
        if grad_total.shape != shape:
            raise ValueError("grad_total must have the shape of total")
        grad_total, after = _rows(grad_total if grad_total.dim() > 1 else grad_total[None])
    device = grad_out.device
    dx = torch.empty(shape, dtype=dtype, device=device)
    dr = dx if kind == dtype else torch.empty(shape, dtype=kind, device=device)
    dw = torch.empty(channels, dtype=torch.float32, device=device)
    size = CUSIG_NORM_RESIDUAL_BACKPROP_WORKSPACE(channels)
    space = _workspace(size, device)
    _call(CUSIG_NORM_RESIDUAL_BACKPROP, "norm_residual_backprop", device, _CODES[dtype], _CODES[kind], grad_out.data_ptr(),
          0 if grad_total is None else grad_total.data_ptr(), total.data_ptr(), weight.data_ptr(), dx.data_ptr(), dr.data_ptr(), dw.data_ptr(),
          rows, channels, grad_step, after, step, eps, space.data_ptr(), size)
    return dx, dr, dw


def _conv_args(x, weight, bias, silu, offsets):
    check_type(silu, "silu", bool)
    _tensor(x, "x")
    if x.dim() < 2:
        raise ValueError("x must have at least rank 2, got rank " + str(x.dim()) + ".")
    device, channels = x.device, x.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight must have shape (" + str(channels) + ", width)")
    width = weight.shape[1]
    if not 1 <= width <= 8:
        raise ValueError("weight must have 1 to 8 taps for each channel, got " + str(width))
    weight = _other(weight, "weight", torch.float32, (channels, width), device)
    if bias is not None:
        bias = _other(bias, "bias", torch.float32, (channels,), device)
    if offsets is not None:
        offsets = _offsets(offsets, "offsets", device)
    return weight, bias, offsets, width, _sequences(x, offsets, "x")


def causal_conv(x, weight, bias=None, *, initial_state=None, offsets=None, silu=True):
    """Short causal convolution of each channel, ``y_t = f(bias + sum_k weight[:, k] * x_{t - width + 1 + k})`` with ``f(v) = v * sigmoid(v)``
    (``silu``) or ``f(v) = v``.

    ``x``: ``(..., length, channels)``, or with ``offsets`` ``(rows, channels)``, the sequences packed.  ``weight`` float32 ``(channels,
    width)``, 1 to 8 taps, the last for the row itself; ``bias`` float32 ``(channels,)``.  ``initial_state``: the ``width - 1`` rows before
    each sequence, in the type of ``x``, ``(..., width - 1, channels)``, with ``offsets`` ``(sequences, width - 1, channels)``; zero where it is not
    given.

    Returns ``(y, final_state)``: ``y`` like ``x``, and the last ``width - 1`` rows of each sequence like ``initial_state``.
    """
    weight, bias, offsets, width, (n, length, rows, lead, at) = _conv_args(x, weight, bias, silu, offsets)
    device, dtype, channels = x.device, x.dtype, x.shape[-1]
    state = (*lead, width - 1, channels)
    if initial_state is not None:
        initial_state = _other(initial_state, "initial_state", dtype, state, device)
    y = torch.empty(x.shape, dtype=dtype, device=device)
    final = torch.empty(state, dtype=dtype, device=device)
    x, x_step = _rows(x)
    _call(CUSIG_CAUSAL_CONV, "causal_conv", device, _CODES[dtype], x.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
          0 if initial_state is None else initial_state.data_ptr(), y.data_ptr(), final.data_ptr(), at, n, length, rows, channels, width,
          x_step, silu)
    return y, final


def causal_conv_backprop(grad_y, x, weight, bias=None, *, grad_final=None, initial_state=None, offsets=None, silu=True):
    """Gradients of ``causal_conv`` from the gradients of its outputs (``grad_final`` like the final state, zero where it is not given) and its
    inputs.  Returns ``(grad_x, grad_weight, grad_bias, grad_initial_state)``, the third None where there is no bias; the weights' are
    summed over the rows in a fixed order."""
    weight, bias, offsets, width, (n, length, rows, lead, at) = _conv_args(x, weight, bias, silu, offsets)
    _tensor(grad_y, "grad_y", like=x)
    if grad_y.shape != x.shape:
        raise ValueError("grad_y and x must have the same shape")
    device, dtype, channels = x.device, x.dtype, x.shape[-1]
    state = (*lead, width - 1, channels)
    if initial_state is not None:
        initial_state = _other(initial_state, "initial_state", dtype, state, device)
    if grad_final is not None:
        grad_final = _other(grad_final, "grad_final", dtype, state, device)
    dx = torch.empty(x.shape, dtype=dtype, device=device)
    dw = torch.empty((channels, width), dtype=torch.float32, device=device)
    db = None if bias is None else torch.empty(channels, dtype=torch.float32, device=device)
    d0 = torch.empty(state, dtype=dtype, device=device)
    x, x_step = _rows(x)
    grad_y, grad_step = _rows(grad_y)
    size = CUSIG_CAUSAL_CONV_BACKPROP_WORKSPACE(rows, channels, width)
    space = _workspace(size, device) if size else None
    _call(CUSIG_CAUSAL_CONV_BACKPROP, "causal_conv_backprop", device, _CODES[dtype], grad_y.data_ptr(), x.data_ptr(), weight.data_ptr(),
          0 if bias is None else bias.data_ptr(), 0 if initial_state is None else initial_state.data_ptr(),
          0 if grad_final is None else grad_final.data_ptr(), dx.data_ptr(), dw.data_ptr(), 0 if bias is None else db.data_ptr(), d0.data_ptr(),
          at, n, length, rows, channels, width, grad_step, x_step, silu, space.data_ptr() if size else 0, size)
    return dx, dw, db, d0


def causal_conv_step(x, state, weight, bias=None, *, silu=True):
    """One row of ``causal_conv`` for single tokens: ``x`` ``(..., channels)``; ``state`` ``(..., width - 1, channels)``, the rows before it, of
    the same type, contiguous, is replaced by the rows before the next.  Returns ``y`` like ``x``."""
    _tensor(x, "x")
    shape, device, dtype = x.shape, x.device, x.dtype
    if len(shape) < 1:
        raise ValueError("x must have at least rank 1, got rank 0.")
    weight, bias, _, width, _ = _conv_args(x if len(shape) > 1 else x[None], weight, bias, silu, None)
    if _other(state, "state", dtype, (*shape[:-1], width - 1, shape[-1]), device) is not state:
        raise ValueError("state must be contiguous: it is written")
    y = torch.empty(shape, dtype=dtype, device=device)
    x, x_step = _rows(x if len(shape) > 1 else x[None])
    channels = shape[-1]
    _call(CUSIG_CAUSAL_CONV_STEP, "causal_conv_step", device, _CODES[dtype], x.data_ptr(), state.data_ptr(), weight.data_ptr(),
          0 if bias is None else bias.data_ptr(), y.data_ptr(), y.numel() // channels if channels else 0, channels, width, x_step, silu)
    torch.autograd.graph.increment_version(state)
    return y


def _shared(value, name, like, groups, states):
    """``b`` or ``c``, ``(..., groups, states)``: (tensor, distance of its rows, of its groups)."""
    _tensor(value, name, like=like)
    shape = (*like.shape[:-1], groups, states)
    if value.shape != shape:
        raise ValueError(name + " must have shape " + str(shape) + ", got " + str(tuple(value.shape)))
    if value.stride(-1) != 1 and states > 1:
        value = value.contiguous()
    if len(shape) == 3:
        return value, value.stride(0) if shape[0] > 1 else groups * states, value.stride(1)
    # rows a fixed distance apart
    want = None
    for axis in range(value.dim() - 3, -1, -1):
        if value.shape[axis] == 1:
            continue
        if want is not None and value.stride(axis) != want:
            value = value.contiguous()
            return value, groups * states, states
        want = value.stride(axis) * value.shape[axis]
    step = next((value.stride(axis) for axis in range(value.dim() - 3, -1, -1) if value.shape[axis] != 1), groups * states)
    return value, step, value.stride(-2)


def _scan_args(x, delta, a, b, c, d, z, delta_bias, softplus):
    """Checked inputs, and (states, groups) and the strides that the entry points take."""
    check_type(softplus, "softplus", bool)
    _tensor(x, "x")
    _tensor(delta, "delta", like=x)
    if delta.shape != x.shape:
        raise ValueError("x and delta must have the same shape")
    device, channels = x.device, x.shape[-1]
    if not isinstance(a, torch.Tensor) or a.dim() != 2 or not 1 <= a.shape[1] <= 64:
        raise ValueError("a must have shape (" + str(channels) + ", states), with 1 to 64 states")
    states = a.shape[1]
    a = _other(a, "a", torch.float32, (channels, states), device)
    if not isinstance(b, torch.Tensor) or b.dim() != x.dim() + 1:
        raise ValueError("b must have shape (..., groups, states)")
    groups = b.shape[-2]
    if groups < 1 or channels % groups:
        raise ValueError("the channels must be a multiple of the groups, got " + str(channels) + " and " + str(groups))
    b, b_step, b_group = _shared(b, "b", x, groups, states)
    c, c_step, c_group = _shared(c, "c", x, groups, states)
    if d is not None:
        d = _other(d, "d", torch.float32, (channels,), device)
    if delta_bias is not None:
        delta_bias = _other(delta_bias, "delta_bias", torch.float32, (channels,), device)
    x, x_step = _rows(x)
    delta, delta_step = _rows(delta)
    z_step = 0
    if z is not None:
        _tensor(z, "z", like=x)
        if z.shape != delta.shape:
            raise ValueError("x and z must have the same shape")
        z, z_step = _rows(z)
    tensors = (x, delta, a, b, c, d, z, delta_bias)
    return tensors, states, groups, (x_step, delta_step, z_step, b_step, b_group, c_step, c_group)


def _addresses(tensors):
    return tuple(0 if t is None else t.data_ptr() for t in tensors)


def selective_scan(x, delta, a, b, c, *, d=None, z=None, delta_bias=None, softplus=True, initial_state=None, offsets=None):
    """Scan of a selective state space model: for each channel and state ``h_t = exp(dt_t * a) * h_{t-1} + dt_t * b_t * x_t``, and
    ``y_t = (sum over states of c_t * h_t + d * x_t) * z_t * sigmoid(z_t)``, with ``dt = softplus(delta + delta_bias)``, or without ``softplus``
    ``delta + delta_bias``.

    ``x``, ``delta``, ``z`` (the gate, or None): ``(..., length, channels)``, or with ``offsets`` ``(rows, channels)``, the sequences packed.
    ``a`` float32 ``(channels, states)``, meant to be negative (decays of many steps are formed at once: where they grow past float32's
    range, so do the results), 1 to 64 states; ``b``, ``c``: ``(..., length, groups, states)`` or
    ``(rows, groups, states)``, each group's for ``channels / groups`` neighbouring channels; ``d``, ``delta_bias``: float32 ``(channels,)`` or None.
    ``initial_state``: float32 ``(..., channels, states)``, with ``offsets`` ``(sequences, channels, states)``; zero where it is not given.

    Numbers of states are rounded up to 4, 8, 16, 32 or 64, and each group's channels to 256, 128, 64, 32 or 16 of them, in time: many small groups cost
    most.  States that are not finite stay so; long sequences are cut, and whether such a state is infinite or NaN behind a cut may differ from a walk
    step by step.

    Returns ``(y, final_state)``: ``y`` like ``x``, the states behind the last steps like ``initial_state``.
    """
    _tensor(x, "x")
    if x.dim() < 2:
        raise ValueError("x must have at least rank 2, got rank " + str(x.dim()) + ".")
    shape, device = x.shape, x.device
    tensors, states, groups, strides = _scan_args(x, delta, a, b, c, d, z, delta_bias, softplus)
    if offsets is not None:
        offsets = _offsets(offsets, "offsets", device)
    n, length, rows, lead, at = _sequences(x, offsets, "x")
    channels = shape[-1]
    state = (*lead, channels, states)
    if initial_state is not None:
        initial_state = _other(initial_state, "initial_state", torch.float32, state, device)
    y = torch.empty(shape, dtype=x.dtype, device=device)
    final = torch.empty(state, dtype=torch.float32, device=device)
    size = CUSIG_SELECTIVE_SCAN_WORKSPACE(offsets is not None, n, length, rows, channels, states, groups)
    space = _workspace(size, device) if size else None
    _call(CUSIG_SELECTIVE_SCAN, "selective_scan", device, _CODES[x.dtype], *_addresses(tensors),
          0 if initial_state is None else initial_state.data_ptr(), y.data_ptr(), final.data_ptr(), at, n, length, rows, channels, states, groups,
          *strides, softplus, space.data_ptr() if size else 0, size)
    return y, final


def selective_scan_backprop(grad_y, x, delta, a, b, c, *, d=None, z=None, delta_bias=None, softplus=True, grad_final=None, initial_state=None,
                            offsets=None):
    """Gradients of ``selective_scan`` from the gradients of its outputs (``grad_final`` float32 like the final state, zero where it is not
    given) and its inputs; the states are formed again.  Returns ``(grad_x, grad_delta, grad_a, grad_b, grad_c, grad_d, grad_z,
    grad_delta_bias, grad_initial_state)``, None for what was not given; those of float32 inputs and of the initial state are float32.  The
    same inputs give the same bits.

    Its scratch holds the states before every eighth row (every fourth with up to 4 states), half a byte (a byte) for each row, channel and state, these
    rounded up as in ``selective_scan``, and each row's sums over 1024 or 4096 pairs of channel and state, 8 bytes for each state: 5.4 GB for 32768 rows of
    4096 channels of 64 states."""
    _tensor(x, "x")
    if x.dim() < 2:
        raise ValueError("x must have at least rank 2, got rank " + str(x.dim()) + ".")
    shape, device, dtype = x.shape, x.device, x.dtype
    _tensor(grad_y, "grad_y", like=x)
    if grad_y.shape != shape:
        raise ValueError("grad_y and x must have the same shape")
    tensors, states, groups, strides = _scan_args(x, delta, a, b, c, d, z, delta_bias, softplus)
    if offsets is not None:
        offsets = _offsets(offsets, "offsets", device)
    n, length, rows, lead, at = _sequences(x, offsets, "x")
    channels = shape[-1]
    state = (*lead, channels, states)
    if initial_state is not None:
        initial_state = _other(initial_state, "initial_state", torch.float32, state, device)
    if grad_final is not None:
        grad_final = _other(grad_final, "grad_final", torch.float32, state, device)
    grad_y, grad_step = _rows(grad_y)
    make = lambda shape, kind=torch.float32: torch.empty(shape, dtype=kind, device=device)          # noqa: E731
    grads = (make(shape, dtype), make(shape, dtype), make((channels, states)), make((*shape[:-1], groups, states), dtype),
             make((*shape[:-1], groups, states), dtype), None if d is None else make(channels), None if z is None else make(shape, dtype),
             None if delta_bias is None else make(channels), make(state))
    size = CUSIG_SELECTIVE_SCAN_BACKPROP_WORKSPACE(offsets is not None, n, length, rows, channels, states, groups)
    space = _workspace(size, device) if size else None
    _call(CUSIG_SELECTIVE_SCAN_BACKPROP, "selective_scan_backprop", device, _CODES[dtype], grad_y.data_ptr(), *_addresses(tensors),
          0 if grad_final is None else grad_final.data_ptr(), 0 if initial_state is None else initial_state.data_ptr(), *_addresses(grads),
          at, n, length, rows, channels, states, groups, grad_step, *strides, softplus, space.data_ptr() if size else 0, size)
    return grads


def selective_scan_step(x, delta, a, b, c, state, *, d=None, z=None, delta_bias=None, softplus=True):
    """One step of ``selective_scan`` for single tokens: ``x``, ``delta``, ``z`` ``(..., channels)``, ``b``, ``c`` ``(..., groups, states)``; ``state``
    float32 ``(..., channels, states)``, contiguous, is replaced by the state behind the step.  Returns ``y`` like ``x``."""
    _tensor(x, "x")
    shape, device = x.shape, x.device
    if len(shape) < 1:
        raise ValueError("x must have at least rank 1, got rank 0.")
    if len(shape) == 1:
        if not all(isinstance(t, torch.Tensor) for t in (delta, b, c)):
            raise TypeError("delta, b and c must be torch tensors")
        x, delta, b, c, z = x[None], delta[None], b[None], c[None], z if z is None else z[None]
    tensors, states, groups, strides = _scan_args(x, delta, a, b, c, d, z, delta_bias, softplus)
    if _other(state, "state", torch.float32, (*shape, states), device) is not state:
        raise ValueError("state must be contiguous: it is written")
    y = torch.empty(shape, dtype=x.dtype, device=device)
    channels = shape[-1]
    _call(CUSIG_SELECTIVE_SCAN_STEP, "selective_scan_step", device, _CODES[x.dtype], *_addresses(tensors), state.data_ptr(), y.data_ptr(),
          y.numel() // channels if channels else 0, channels, states, groups, *strides, softplus)
    torch.autograd.graph.increment_version(state)
    return y
