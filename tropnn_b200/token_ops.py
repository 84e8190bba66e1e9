"""Operators of a token model around the routed layers, over the sm_100a C ABI.

* ``gated_recurrence_b200`` / ``gated_recurrence_step_b200``: the sequence mixer, for whole
  sequences (differentiable) and for one decoded token.
* ``distill_loss_b200`` / ``distill_loss_grad_b200``: the loss of a student's logits against a
  teacher's top logits, through autograd or with the gradient in the same launch.
* ``sample_tokens_b200``: temperature, top-k, top-p and min-p sampling from given uniform numbers.

The reference has no counterpart of these. They keep the conventions of the other operators:
CUDA tensors only (``ValueError`` otherwise, there is no CPU path), ``TypeError`` for a dtype,
kernels on ``torch.cuda.current_stream()``, buffers from PyTorch's caching allocator, no host
synchronisation, deterministic results.
"""

from __future__ import annotations

import math
from typing import Any

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as nat
from .ops import _launch, _require_cuda

__all__ = [
    "distill_loss_b200",
    "distill_loss_grad_b200",
    "gated_recurrence_b200",
    "gated_recurrence_step_b200",
    "sample_tokens_b200",
]

MAX_TEACHER_TOP = 1024
_REDUCTIONS = ("mean", "sum", "none")


def _call(device: torch.device, name: str, fn: Any, *args: Any) -> None:
    """Launches on the device's current stream, whichever device is current."""
    if device.index == torch.cuda.current_device():
        _launch(name, fn, *args, nat.stream_handle(device))
    else:
        with torch.cuda.device(device):
            _launch(name, fn, *args, nat.stream_handle(device))


def _same_device(device: torch.device, t: Tensor, name: str) -> None:
    if t.device != device:
        _require_cuda(t, name)
        raise ValueError(f"{name} is on {t.device}, expected {device}")


def _no_tangent(name: str, *tensors: Any) -> None:
    """Refuses forward-mode derivatives, which a call past autograd would give as 0."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # no dual tensors about (unpacking takes 0.3 us each)
        return
    for t in tensors:
        if isinstance(t, Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has no forward-mode derivative")


def _unit_last(t: Tensor) -> Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


# ---------------------------------------------------------------------------
# gated linear recurrence
# ---------------------------------------------------------------------------


def _recurrence_workspace(lib: Any, gate: Tensor, shape: tuple[int, int, int]) -> tuple[Tensor | None, int]:
    size = lib.tropnn_b200_recurrence_workspace_size(*shape, nat.float_code(gate.dtype))
    return (torch.empty(size, device=gate.device, dtype=torch.uint8), size) if size else (None, 0)


def _recurrence_forward(
    gate: Tensor, value: Tensor, h0: Tensor | None, reset: Tensor | None, keep: bool
) -> tuple[Tensor, Tensor, Tensor | None]:
    """``(h, h_last, saved)``; ``saved`` are the states that the backward starts from."""
    batch, steps, dim = shape = tuple(gate.shape)
    dev = gate.device
    lib = nat.load()
    h = gate.new_empty(shape)
    h_last = torch.empty((batch, dim), device=dev, dtype=torch.float32)
    saved, saved_bytes = None, 0
    if keep:
        saved_bytes = lib.tropnn_b200_recurrence_saved_size(batch, steps, dim)
        saved = h_last.new_empty(saved_bytes // 4)
    ws, ws_bytes = _recurrence_workspace(lib, gate, shape)
    _call(
        dev, "recurrence_forward", lib.tropnn_b200_recurrence_forward, gate.data_ptr(), gate.stride(0), gate.stride(1),
        value.data_ptr(), value.stride(0), value.stride(1), nat.float_code(gate.dtype), nat.ptr(h0), nat.ptr(reset),
        batch, steps, dim, h.data_ptr(), h_last.data_ptr(), nat.ptr(saved), saved_bytes, nat.ptr(ws), ws_bytes,
    )
    return h, h_last, saved


class _GatedRecurrenceFunction(torch.autograd.Function):
    @staticmethod
    def forward(  # type: ignore[override]
        ctx: Any, gate: Tensor, value: Tensor, h0: Tensor | None, reset: Tensor | None
    ) -> tuple[Tensor, Tensor]:
        h, h_last, saved = _recurrence_forward(gate, value, h0, reset, True)
        ctx.save_for_backward(gate, value, reset, saved)
        ctx.set_materialize_grads(False)
        return h, h_last

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad_h: Tensor | None, grad_last: Tensor | None) -> tuple[Any, ...]:
        if grad_h is None and grad_last is None:
            return None, None, None, None
        gate, value, reset, saved = ctx.saved_tensors
        batch, steps, dim = shape = tuple(gate.shape)
        # Hooks may bring a saved tensor back with other strides.
        gate_batch, gate_step, unit = gate.stride()
        value_batch, value_step, value_unit = value.stride()
        if unit != 1 or value_unit != 1:
            gate, value = gate.contiguous(), value.contiguous()
            gate_batch, gate_step = value_batch, value_step = steps * dim, dim
        saved = saved.contiguous()
        reset = None if reset is None else reset.contiguous()
        lib = nat.load()
        grad_h = None if grad_h is None else grad_h.contiguous()
        grad_last = None if grad_last is None else grad_last.contiguous()
        grad_gate = gate.new_empty(shape)
        grad_value = torch.empty_like(grad_gate)
        grad_h0 = saved.new_empty((batch, dim)) if ctx.needs_input_grad[2] else None
        ws, ws_bytes = _recurrence_workspace(lib, gate, shape)
        _call(
            gate.device, "recurrence_backward", lib.tropnn_b200_recurrence_backward, gate.data_ptr(), gate_batch,
            gate_step, value.data_ptr(), value_batch, value_step, nat.float_code(gate.dtype), nat.ptr(reset), batch,
            steps, dim, saved.data_ptr(), saved.numel() * 4, nat.ptr(grad_h), nat.ptr(grad_last),
            grad_gate.data_ptr(), grad_value.data_ptr(), nat.ptr(grad_h0), nat.ptr(ws), ws_bytes,
        )
        return grad_gate, grad_value, grad_h0, None


def _check_gate_value(gate: Tensor, value: Tensor, ndim: int) -> None:
    _require_cuda(gate, "gate")
    _same_device(gate.device, value, "value")
    if gate.ndim != ndim or value.shape != gate.shape:
        want = "[batch, steps, dim]" if ndim == 3 else "[batch, dim]"
        raise ValueError(f"gate and value must both have shape {want}, got {tuple(gate.shape)} and {tuple(value.shape)}")
    nat.float_code(gate.dtype)
    if value.dtype != gate.dtype:
        raise TypeError(f"gate and value must have one dtype, got {gate.dtype} and {value.dtype}")


def _check_reset(reset: Tensor, shape: tuple[int, ...], device: torch.device) -> Tensor:
    _same_device(device, reset, "reset")
    if reset.dtype not in (torch.bool, torch.uint8):
        raise TypeError(f"reset must be bool or uint8, got {reset.dtype}")
    if reset.shape != shape:
        raise ValueError(f"reset must have shape {shape}, got {tuple(reset.shape)}")
    return reset.contiguous()


def gated_recurrence_b200(
    gate: Tensor, value: Tensor, h0: Tensor | None = None, *, reset: Tensor | None = None
) -> tuple[Tensor, Tensor]:
    """Gated linear recurrence over whole sequences, per channel:

        h_t = keep_t * a_t * h_{t-1} + (1 - a_t) * value_t,   a = sigmoid(gate)

    ``gate`` and ``value`` are ``[batch, steps, dim]`` in one of f32/f16/bf16, any batch and step
    strides (the two halves of one projection's output are read in place). ``h0`` ``[batch, dim]``
    is the state before the first token (zeros by default), ``reset`` ``[batch, steps]`` marks the
    tokens that start a document: nothing of the state before them is kept. Returns ``(h, h_last)``:
    ``h`` in the inputs' dtype and the last state in f32, which continues a sequence as ``h0`` of
    the next call or as the state of ``gated_recurrence_step_b200``. The state is f32 throughout. One
    that is not finite stays so until a reset, but an infinity may become a NaN on the way (0 times it,
    where the gates of a stretch multiply to less than f32 holds).
    Differentiable in gate, value and h0 (once, in reverse mode); the backward scans the states again
    from every eighth, saved in f32, instead of reading ``h``.
    """
    _check_gate_value(gate, value, 3)
    _no_tangent("gated_recurrence_b200", gate, value, h0)
    if h0 is not None:
        _same_device(gate.device, h0, "h0")
        if h0.shape != (gate.shape[0], gate.shape[2]):
            raise ValueError(f"h0 must have shape {(gate.shape[0], gate.shape[2])}, got {tuple(h0.shape)}")
        nat.float_code(h0.dtype)
        h0 = h0.to(torch.float32).contiguous()
    if reset is not None:
        reset = _check_reset(reset, tuple(gate.shape[:2]), gate.device)
    gate, value = _unit_last(gate), _unit_last(value)
    if torch.is_grad_enabled() and (
        gate.requires_grad or value.requires_grad or (h0 is not None and h0.requires_grad)
    ):
        return _GatedRecurrenceFunction.apply(gate, value, h0, reset)
    return _recurrence_forward(gate, value, h0, reset, False)[:2]


def gated_recurrence_step_b200(gate: Tensor, value: Tensor, state: Tensor, *, reset: Tensor | None = None) -> Tensor:
    """One token of ``gated_recurrence_b200`` for every row: ``gate`` and ``value`` ``[batch, dim]``,
    ``state`` f32 ``[batch, dim]``, updated in place; ``reset`` ``[batch]`` clears a row's state
    first. Returns the new state rounded to the inputs' dtype. Not differentiable."""
    _check_gate_value(gate, value, 2)
    _no_tangent("gated_recurrence_step_b200", gate, value, state)
    shape = gate.shape
    dev = gate.device
    _same_device(dev, state, "state")
    if state.shape != shape:
        raise ValueError(f"state must have shape {tuple(shape)}, got {tuple(state.shape)}")
    if state.dtype != torch.float32:
        raise TypeError(f"state must be float32, got {state.dtype}")
    batch, dim = shape
    state_row, unit = state.stride()
    if (dim > 1 and unit != 1) or (batch > 1 and state_row < dim):
        raise ValueError("state must have unit stride over dim and rows of its own")
    if torch.is_grad_enabled() and (gate.requires_grad or value.requires_grad or state.requires_grad):
        raise ValueError("gated_recurrence_step_b200 is not differentiable: call it under torch.no_grad()")
    if reset is not None:
        reset = _check_reset(reset, (batch,), dev)
    gate, value = _unit_last(gate), _unit_last(value)
    h = gate.new_empty(shape)
    _call(
        dev, "recurrence_step", nat.load().tropnn_b200_recurrence_step, gate.data_ptr(), gate.stride(0),
        value.data_ptr(), value.stride(0), nat.float_code(gate.dtype), None if reset is None else reset.data_ptr(),
        batch, dim, state.data_ptr(), state_row, h.data_ptr(),
    )
    torch.autograd.graph.increment_version(state)  # autograd is told, as of torch's in-place operations
    return h


# ---------------------------------------------------------------------------
# logits as rows
# ---------------------------------------------------------------------------


def _logit_rows(logits: Tensor) -> tuple[Tensor, int, int, int, int]:
    """``(logits, rows, inner, outer_stride, inner_stride)``: row n of ``logits[..., vocab]`` starts
    at element ``(n // inner) * outer_stride + (n % inner) * inner_stride``. A slice such as
    ``logits[:, :-1]`` of a batch of sequences is read in place; other layouts are copied."""
    stride = logits.stride()
    if stride[-1] != 1 and logits.shape[-1] > 1:
        logits = logits.detach().contiguous()
        stride = logits.stride()
    shape = logits.shape
    if len(shape) == 2:
        return logits, shape[0], 1, stride[0], 0
    if len(shape) == 3:
        return logits, shape[0] * shape[1], max(1, shape[1]), stride[0], stride[1]
    return logits.detach().contiguous(), math.prod(shape[:-1]), 1, shape[-1], 0


# ---------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------


def _distill_check(
    logits: Tensor, teacher: Tensor, indices: Tensor, labels: Tensor | None, temperature: float, label_weight: float,
    ignore_index: int,
) -> tuple[Tensor, Tensor, Tensor | None, tuple[int, float, float]]:
    """The teacher's entries and the labels as the kernels take them, and the settings."""
    _require_cuda(logits, "logits")
    dev = logits.device
    _same_device(dev, teacher, "teacher_logits")
    _same_device(dev, indices, "teacher_indices")
    nat.float_code(logits.dtype)
    nat.float_code(teacher.dtype)
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must have shape [..., vocab] with vocab >= 1, got {tuple(logits.shape)}")
    lead = logits.shape[:-1]
    if teacher.ndim != logits.ndim or teacher.shape[:-1] != lead or indices.shape != teacher.shape:
        raise ValueError(
            f"teacher_logits and teacher_indices must both have shape {(*lead, 'top')}, got {tuple(teacher.shape)} "
            f"and {tuple(indices.shape)}"
        )
    if teacher.shape[-1] > MAX_TEACHER_TOP:
        raise ValueError(f"at most {MAX_TEACHER_TOP} teacher entries a row, got {teacher.shape[-1]}")
    if indices.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"teacher_indices must be int64 or int32, got {indices.dtype}")
    if labels is not None:
        _same_device(dev, labels, "labels")
        if labels.shape != lead:
            raise ValueError(f"labels must have shape {tuple(lead)}, got {tuple(labels.shape)}")
        if labels.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"labels must be int64 or int32, got {labels.dtype}")
        if labels.dtype != torch.int64 or not labels.is_contiguous():
            labels = labels.to(torch.int64).contiguous()
    temperature, label_weight = float(temperature), float(label_weight)
    if not (0.0 < temperature < math.inf):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    if not (0.0 <= label_weight <= 1.0):
        raise ValueError(f"label_weight must be in [0, 1], got {label_weight}")
    if label_weight < 1.0 and not (2.0**-60 <= temperature <= 2.0**60):
        raise ValueError(f"temperature must be in [2**-60, 2**60] for a teacher, got {temperature}")
    if label_weight > 0.0 and labels is None:
        raise ValueError("label_weight > 0 needs labels")
    if teacher.requires_grad or not teacher.is_contiguous():
        teacher = teacher.detach().contiguous()
    return teacher, indices.contiguous(), labels, (int(ignore_index), temperature, label_weight)


def _distill_args(
    logits: Tensor, teacher: Tensor, indices: Tensor, labels: Tensor | None, settings: tuple[int, float, float]
) -> tuple[Tensor, int, tuple[Any, ...]]:
    """``(logits as read, rows, the C entry points' common arguments)``."""
    read, rows, inner, outer_stride, inner_stride = _logit_rows(logits)
    return read, rows, (
        read.data_ptr(), nat.float_code(read.dtype), rows, inner, outer_stride, inner_stride, read.shape[-1],
        teacher.data_ptr(), nat.float_code(teacher.dtype), indices.data_ptr(),
        nat.I64 if indices.dtype == torch.int64 else nat.I32, teacher.shape[-1], nat.ptr(labels), *settings,
    )


def _distill_loss(
    logits: Tensor, teacher: Tensor, indices: Tensor, labels: Tensor | None, settings: tuple[int, float, float],
    reduction: str,
) -> tuple[Tensor, Tensor, Tensor | None]:
    """``(loss, stats, count)``: the statistics that the gradient needs, and the divisor of a mean or
    sum."""
    lib = nat.load()
    dev = logits.device
    read, rows, args = _distill_args(logits, teacher, indices, labels, settings)
    losses = torch.empty(logits.shape[:-1], device=dev, dtype=torch.float32)
    stats = losses.new_empty((rows, 4))
    _call(dev, "distill_loss", lib.tropnn_b200_distill_loss, *args, losses.data_ptr(), stats.data_ptr())
    if reduction == "none":
        return losses, stats, None
    loss, count = losses.new_empty(()), losses.new_empty(())
    _call(dev, "distill_reduce", lib.tropnn_b200_distill_reduce, losses.data_ptr(), stats.data_ptr(), rows,
          int(reduction == "mean"), loss.data_ptr(), count.data_ptr())
    return loss, stats, count


class _DistillLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(  # type: ignore[override]
        ctx: Any, logits: Tensor, teacher: Tensor, indices: Tensor, labels: Tensor | None,
        settings: tuple[int, float, float], reduction: str,
    ) -> Tensor:
        loss, stats, count = _distill_loss(logits, teacher, indices, labels, settings, reduction)
        ctx.save_for_backward(logits, stats, count, teacher, indices, labels)
        ctx.settings = settings
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad_loss: Tensor) -> tuple[Any, ...]:
        logits, stats, count, teacher, indices, labels = ctx.saved_tensors
        # Hooks may bring a saved tensor back with other strides.
        stats, teacher, indices = stats.contiguous(), teacher.contiguous(), indices.contiguous()
        labels = None if labels is None else labels.contiguous()
        read, _, args = _distill_args(logits, teacher, indices, labels, ctx.settings)
        grad = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
        scale = grad_loss.contiguous()
        _call(logits.device, "distill_grad", nat.load().tropnn_b200_distill_grad, *args, stats.data_ptr(),
              scale.data_ptr(), int(count is None), nat.ptr(count), grad.data_ptr())
        return grad, None, None, None, None, None


def distill_loss_b200(
    logits: Tensor,
    teacher_logits: Tensor,
    teacher_indices: Tensor,
    labels: Tensor | None = None,
    *,
    temperature: float = 1.0,
    label_weight: float = 0.0,
    ignore_index: int = -100,
    reduction: str = "mean",
) -> Tensor:
    """Loss of a student's ``logits`` ``[..., vocab]`` against a teacher's top logits.

    ``teacher_logits`` and ``teacher_indices`` ``[..., top]`` (top <= 1024) are the teacher's
    largest logits and their tokens; an index outside ``[0, vocab)`` (such as -1) or a logit of
    -inf is padding. With ``q = softmax(teacher_logits / T)`` over a row's entries, ``p =
    softmax(logits / T)`` and ``w = label_weight``::

        loss = (1 - w) * T**2 * KL(q || p) + w * cross_entropy(logits, label)

    A row without entries has no teacher term; a label that is ``ignore_index`` or outside ``[0,
    vocab)`` gives no label term; a row with neither has loss 0 and gradient 0 and does not count in
    the "mean" (which is 0 where no row counts). ``reduction`` is "mean", "sum" or "none" (a loss a
    row). ``temperature`` is in ``[2**-60, 2**60]``, whose squares f32 holds (any positive number where
    ``label_weight`` is 1). Everything is computed in f32 and the loss is f32; logits of f32/f16/bf16,
    sliced rows and steps in place. Differentiable (once, in reverse mode) in the logits; the teacher gets no gradient.
    The backward reads the logits again: ``distill_loss_grad_b200`` does both in one pass.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {_REDUCTIONS}, got {reduction!r}")
    teacher, indices, labels, settings = _distill_check(
        logits, teacher_logits, teacher_indices, labels, temperature, label_weight, ignore_index)
    _no_tangent("distill_loss_b200", logits, teacher_logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _DistillLossFunction.apply(logits, teacher, indices, labels, settings, reduction)
    return _distill_loss(logits, teacher, indices, labels, settings, reduction)[0]


def distill_loss_grad_b200(
    logits: Tensor,
    teacher_logits: Tensor,
    teacher_indices: Tensor,
    labels: Tensor | None = None,
    *,
    temperature: float = 1.0,
    label_weight: float = 0.0,
    ignore_index: int = -100,
    row_scale: Tensor | float | None = None,
) -> tuple[Tensor, Tensor]:
    """The losses of ``distill_loss_b200`` a row (f32 ``[...]``) and the gradient of ``sum(row_scale
    * losses)`` in the logits (their dtype, contiguous), in one launch. ``row_scale`` is a number, a
    one-element f32 tensor, or f32 ``[...]``: the upstream gradient with the divisor of a mean and
    a loss scale in it, so that a gradient in f16 is scaled before it is rounded. For training
    loops that call the head's backward themselves, such as a head in chunks of rows."""
    teacher, indices, labels, settings = _distill_check(
        logits, teacher_logits, teacher_indices, labels, temperature, label_weight, ignore_index)
    _no_tangent("distill_loss_grad_b200", logits, teacher_logits, row_scale)
    dev, lead = logits.device, logits.shape[:-1]
    scale: Tensor | None = None
    if isinstance(row_scale, Tensor):
        _same_device(dev, row_scale, "row_scale")
        if row_scale.dtype != torch.float32:
            raise TypeError(f"row_scale must be float32, got {row_scale.dtype}")
        if row_scale.numel() != 1 and row_scale.shape != lead:
            raise ValueError(f"row_scale must have one element or shape {tuple(lead)}, got {tuple(row_scale.shape)}")
        scale = row_scale.detach().contiguous()
    elif row_scale is not None:
        scale = torch.full((1,), float(row_scale), device=dev, dtype=torch.float32)
    per_row = scale is not None and scale.shape == lead
    read, _, args = _distill_args(logits, teacher, indices, labels, settings)
    losses = torch.empty(lead, device=dev, dtype=torch.float32)
    grad = logits.new_empty(logits.shape)
    _call(dev, "distill_loss_grad", nat.load().tropnn_b200_distill_loss_grad, *args, nat.ptr(scale), int(per_row),
          losses.data_ptr(), grad.data_ptr())
    return losses, grad


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------


def _setting(
    value: Tensor | float, name: str, lead: torch.Size, device: torch.device, lo: float, hi: float
) -> tuple[Tensor | None, float]:
    """A sampling setting as (one a row, or None; the value where it is one for all)."""
    if isinstance(value, Tensor):
        _same_device(device, value, name)
        if value.dtype != torch.float32:
            raise TypeError(f"{name} must be a number or float32, got {value.dtype}")
        if value.shape != lead:
            raise ValueError(f"{name} must be a number or have shape {tuple(lead)}, got {tuple(value.shape)}")
        return value.contiguous(), 0.0
    number = float(value)
    if not (lo <= number <= hi):
        raise ValueError(f"{name} must be in [{lo:g}, {hi:g}], got {number}")
    return None, number


def sample_tokens_b200(
    logits: Tensor,
    uniforms: Tensor,
    *,
    temperature: Tensor | float = 1.0,
    top_k: Tensor | int = 0,
    top_p: Tensor | float = 1.0,
    min_p: Tensor | float = 0.0,
) -> Tensor:
    """One token (int64 ``[...]``) a row of ``logits`` ``[..., vocab]`` from ``uniforms`` (f32
    ``[...]``, in [0, 1)).

    Tokens rank by (logit descending, index ascending). Kept are the ``top_k`` first (0: all); of
    those the ones with less than ``top_p`` of their probability before them; of those the ones with
    at least ``min_p`` of the likeliest one's probability; the likeliest one always. The token is
    where ``uniforms`` falls in the kept probabilities, in index order. ``temperature`` 0 takes the
    likeliest. Each setting is a number or a tensor of one a row (f32, ``top_k`` int32/int64), whose
    values are not checked: temperatures <= 0 are greedy and top_k <= 0 keeps all. A row with a NaN, or
    with nothing above -inf, gives -1.

    Probabilities are whole numbers (2^31 for the likeliest token) and add up exactly, so a row's
    token depends on its logits and settings alone: not on the batch, the strides or the run.
    """
    _require_cuda(logits, "logits")
    nat.float_code(logits.dtype)
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must have shape [..., vocab] with vocab >= 1, got {tuple(logits.shape)}")
    lead, dev, vocab = logits.shape[:-1], logits.device, logits.shape[-1]
    _same_device(dev, uniforms, "uniforms")
    if uniforms.dtype != torch.float32:
        raise TypeError(f"uniforms must be float32, got {uniforms.dtype}")
    if uniforms.shape != lead:
        raise ValueError(f"uniforms must have shape {tuple(lead)}, got {tuple(uniforms.shape)}")
    t, t_value = _setting(temperature, "temperature", lead, dev, 0.0, 3.4e38)
    p, p_value = _setting(top_p, "top_p", lead, dev, 0.0, 1.0)
    floor, floor_value = _setting(min_p, "min_p", lead, dev, 0.0, 1.0)
    k, k_value, k_code = None, 0, nat.I64
    if isinstance(top_k, Tensor):
        _same_device(dev, top_k, "top_k")
        if top_k.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"top_k must be a number or int32/int64, got {top_k.dtype}")
        if top_k.shape != lead:
            raise ValueError(f"top_k must be a number or have shape {tuple(lead)}, got {tuple(top_k.shape)}")
        k, k_code = top_k.contiguous(), nat.I64 if top_k.dtype == torch.int64 else nat.I32
    else:
        k_value = int(top_k)
        if k_value < 0:
            raise ValueError(f"top_k must be >= 0, got {k_value}")
        k_value = min(k_value, vocab)
    logits, rows, inner, outer_stride, inner_stride = _logit_rows(logits)
    uniforms = uniforms.contiguous()
    tokens = torch.empty(lead, device=dev, dtype=torch.int64)
    _call(
        dev, "sample_tokens", nat.load().tropnn_b200_sample_tokens, logits.data_ptr(), nat.float_code(logits.dtype),
        rows, inner, outer_stride, inner_stride, vocab, uniforms.data_ptr(), nat.ptr(t), t_value, nat.ptr(k), k_code,
        k_value, nat.ptr(p), p_value, nat.ptr(floor), floor_value, tokens.data_ptr(),
    )
    return tokens
