"""Layers of a sequence model over path features: the gated linear recurrence, norms of queries and keys with the rotation by
position, and causal attention over packed sequences, each with its gradients and its form for single tokens.

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
                      CUSIG_ATTENTION_WORKSPACE, CUSIG_LINEAR_RECURRENCE, CUSIG_LINEAR_RECURRENCE_BACKPROP, CUSIG_LINEAR_RECURRENCE_STEP,
                      CUSIG_LINEAR_RECURRENCE_WORKSPACE, CUSIG_NORM_ROTARY, CUSIG_NORM_ROTARY_BACKPROP,
                      CUSIG_NORM_ROTARY_BACKPROP_WORKSPACE, SEQUENCE_DTYPES)
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
