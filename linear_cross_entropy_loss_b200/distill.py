"""Distillation of a vocabulary head from a teacher's top logits, fused with the head's matrix product.

    z    = logit_scale * (x @ At)
    q_ik = softmax over the row's K listed teacher logits / T       (or exp(t_ik / T - teacher_lse_i))
    loss = T^2 / n * sum_i sum_k q_ik (log q_ik - log_softmax(z_i / T)[idx_ik])

over the n rows whose list has any weight. The pass is the one of the cross-entropy loss -- row chunks, one slab of
exponentials, both gradients during ``forward`` -- with K soft targets per row in the place of the label: nothing of
size N x V exists beyond one chunk, and the teacher's distribution is never spread over the vocabulary. The reference
project has no counterpart.
"""
from __future__ import annotations

import os
from typing import Optional

import torch

from . import _native
from .ops import (
    _DTYPE_CODE,
    LinearCrossEntropyLoss,
    _aligned_rows_like,
    _autocast_target,
    _device_guard,
    _scaled_grads,
    _tma_ready,
    get_backend,
    scaled_op,
    slab_mode_policy,
)


def _run_pass(x, At, t, idx, lse, temperature, logit_scale, N_chunk_size, want_dx, want_dW):
    """(loss, dx, dW); x (N, H) and At (H, V) as the kernels read them (:func:`_operands`)."""
    backend = get_backend()
    N, H = x.shape
    V = At.shape[1]
    dev = x.device
    want_grad = want_dx or want_dW
    N_group = -(-min(N, int(N_chunk_size)) // 128) * 128
    capturing = dev.type == "cuda" and torch.cuda.is_current_stream_capturing()
    policy_key = (dev.index, x.dtype, H, V, N_group, 1, "distill")
    if capturing and x.dtype != torch.float16 and os.environ.get("LCE_SLAB_MODE", "auto") == "auto":
        # the policy polls an event, which a capture does not allow: the mode that never recomputes for small chunks,
        # the default one otherwise
        small = N_group * V < slab_mode_policy.small_slab_elems
        slab_mode = _native.SLAB_PER_TILE if small else _native.SLAB_DEFAULT
    else:
        slab_mode = slab_mode_policy.choose(policy_key, x.dtype)
    prob = _native.Problem(
        n_rows_total=N, chunk_rows=N_group, hidden=H, vocab_local=V, vocab_offset=0, ignore_index=-100, world=1,
        dtype=_DTYPE_CODE[x.dtype], monitoring=0, want_grad=1 if want_grad else 0, logit_scale=float(logit_scale),
        z_regularization=0.0, slab_mode=slab_mode,
    )
    k = t.shape[1]
    workspace = torch.empty(backend.distill_workspace_bytes(prob, k), dtype=torch.uint8, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    dx = torch.empty((N, H), dtype=x.dtype, device=dev) if want_dx else None
    dW = dW_res = None
    if want_dW:
        # rows on 32-byte boundaries (16 elements of the 16-bit types): the contraction then writes whole sectors. On
        # 16-byte ones it goes element by element: 556 against 86 us for 1000 x 1000 x 50257 in fp16.
        dW = _aligned_rows_like((H, V), At.dtype, dev, 16)
        if N > N_group and At.dtype != torch.float32:
            dW_res = _aligned_rows_like((H, V), At.dtype, dev, 16)  # the rounding residual of the sum over the chunks
    teacher = _native.Teacher(
        logits=t.data_ptr(), indices=idx.data_ptr(), lse=None if lse is None else lse.data_ptr(),
        logits_ld=t.stride(0), indices_ld=idx.stride(0), k=k, logits_dtype=_DTYPE_CODE[t.dtype],
        indices_bits=64 if idx.dtype == torch.int64 else 32, temperature=float(temperature),
    )
    backend.distill_pass(prob, teacher, x, At, workspace, dx, dW, dW_res, loss)
    if (getattr(backend, "requires_cuda", True) and not capturing and slab_mode == _native.SLAB_DEFAULT
            and os.environ.get("LCE_SLAB_MODE", "auto") == "auto"):
        slab_mode_policy.record(policy_key, backend, workspace)
    return loss, dx, dW


def _operands(x, At):
    """x and At with rows on 16-byte boundaries and a hidden size that is a multiple of 8 (copies where they are not)."""
    H, V = At.shape
    H8 = -(-H // 8) * 8
    if H8 != H:  # zero columns of x and zero rows of the weight leave the logits as they are
        x_pad = x.new_zeros((x.shape[0], H8))
        x_pad[:, :H] = x
        A_pad = _aligned_rows_like((H8, V), At.dtype, At.device)
        A_pad[:H] = At
        A_pad[H:] = 0
        return x_pad, A_pad
    return _aligned(x), _aligned(At)


def _aligned(m):
    """m, or a copy of it whose rows start on 16-byte boundaries."""
    if _tma_ready(m) and m.stride(0) >= m.shape[1]:  # (an expanded row has stride 0)
        return m
    copy = _aligned_rows_like(m.shape, m.dtype, m.device)
    if m.stride(1) == 1:
        get_backend().align_rows(m, copy)
    else:
        copy.copy_(m)
    return copy


class LinearDistillationImplementation(torch.autograd.Function):
    """Computes the loss and both gradients in ``forward``; ``backward`` multiplies them by ``grad_output``."""

    @staticmethod
    def forward(ctx, x_in, At_in, t, idx, lse, temperature, logit_scale, N_chunk_size):
        with _device_guard(x_in):
            H = x_in.shape[-1]
            x, At = _operands(x_in if x_in.dim() == 2 else x_in.reshape(-1, H), At_in)
            loss, dx, dW = _run_pass(x, At, t, idx, lse, temperature, logit_scale, N_chunk_size,
                                     ctx.needs_input_grad[0], ctx.needs_input_grad[1])
            if x.shape[1] != H:  # the padding is dropped again
                dx = None if dx is None else dx[:, :H]
                dW = None if dW is None else dW[:H]
            ctx.lce_grads = (dx, dW) if dx is not None or dW is not None else None
            ctx.lce_x_shape = x_in.shape
            ctx.lce_x_dtype = x_in.dtype
            return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        if ctx.lce_grads is None:
            raise RuntimeError("backward called twice, or forward ran without any input requiring grad")
        dx, dW = ctx.lce_grads
        with _device_guard(grad_output):
            if dx is None or dW is None:
                dx, dW = _scaled_grads(ctx, grad_output)
            else:
                ctx.lce_grads = None
                factor = grad_output
                if factor.dtype != torch.float32 or factor.device != dx.device:
                    factor = factor.to(device=dx.device, dtype=torch.float32)
                get_backend().grad_scale_pair(dx, dW, factor)
                dx = dx.view(ctx.lce_x_shape) if dx.is_contiguous() else dx.reshape(ctx.lce_x_shape)
        return dx, dW, None, None, None, None, None, None


def linear_distillation(
    x: torch.Tensor,
    teacher_logits: torch.Tensor,
    teacher_indices: torch.Tensor,
    At: torch.Tensor,
    teacher_lse: Optional[torch.Tensor] = None,
    temperature: float = 1.0,
    logit_scale: float = 1.0,
    N_chunk_size: int = 4096,
) -> torch.Tensor:
    """The distillation loss of the head ``x @ At`` against a teacher's top logits (a scalar, float32).

    x: (..., H); At: (H, V), the transposed weight of :class:`LinearCrossEntropyLoss`; float16, bfloat16 or float32
    (multiplied as TF32), any sizes. teacher_logits: (..., K) in any of these types; teacher_indices: (..., K) int64 or
    int32; 1 <= K <= 1024. Both as :func:`top_logits` returns them; any order will do.

    The teacher's distribution is softmax(teacher_logits / temperature) over the K listed tokens, or, with
    teacher_lse: (...) = logsumexp(all teacher logits / temperature), exp(teacher_logits / temperature - teacher_lse):
    then the mass that the list leaves out has no target, and with Q = sum(q) < 1 the gradient of a row's logits is
    Q softmax - q. teacher_lse has to be at least the log-sum-exp of the listed logits.

    An entry with an index outside [0, V) is not there, whatever its logit (lists of different lengths are padded with
    -1); one with logit -inf has no weight; rows without any weight do not count (if none counts, the loss is NaN, like
    that of the cross-entropy). NaN or +inf in an entry that is there make the loss NaN. An index that is listed twice
    counts twice.

    Gradients for x and At only (those that are wanted are computed during the forward pass; no second derivatives; a step
    may be captured into a graph under torch's own rule, that no autograd graph of the same leaves from outside is alive);
    under CUDA autocast x and At are cast as :func:`set_autocast_policy` says.
    """
    assert x.dim() >= 1 and At.dim() == 2 and At.shape[0] == x.shape[-1], "x and the weight disagree on the hidden size"
    rows = x.shape[:-1]
    assert teacher_logits.shape[:-1] == rows, "teacher_logits must have one list per row of x"
    assert teacher_indices.shape == teacher_logits.shape, "teacher_indices must have the shape of teacher_logits"
    k = teacher_logits.shape[-1]
    assert 1 <= k <= _native.TEACHER_MAX, f"between 1 and {_native.TEACHER_MAX} entries per row"
    assert teacher_logits.dtype in _DTYPE_CODE, f"unsupported dtype {teacher_logits.dtype} of teacher_logits"
    assert teacher_indices.dtype in (torch.int64, torch.int32), "teacher_indices must be int64 or int32"
    assert 2**-126 <= temperature < float("inf"), "temperature must be positive"
    assert logit_scale > 0
    for scale in (logit_scale / temperature, logit_scale * temperature):  # of the logits, of the gradients
        assert 2**-126 <= scale < 2**128, "logit_scale and temperature scale the logits or their gradients out of range"
    assert int(N_chunk_size) >= 1
    assert x.numel() > 0 and At.shape[1] >= 1, "x must have at least one row"
    if teacher_lse is not None:
        assert teacher_lse.shape == rows, "teacher_lse must have one entry per row of x"
        assert teacher_lse.is_floating_point(), "teacher_lse must be floating point"
        teacher_lse = teacher_lse.detach().to(torch.float32).reshape(-1).contiguous()
        assert teacher_lse.device == x.device, "all tensors must be on one device"
    dev = x.device
    assert At.device == dev and teacher_logits.device == dev and teacher_indices.device == dev, \
        "all tensors must be on one device"
    target = _autocast_target(x)
    if target is not None:
        x, At = x.to(target), At.to(target)
    assert x.dtype == At.dtype, "x and the weight must have the same dtype"
    assert x.dtype in _DTYPE_CODE, f"unsupported dtype {x.dtype}"
    if getattr(get_backend(), "requires_cuda", True) and not x.is_cuda:
        raise RuntimeError("linear_cross_entropy_loss_b200 runs on CUDA tensors only; there is no CPU fallback")

    def lists(t):
        t = t.detach()
        if t.dim() != 2:
            t = t.reshape(-1, k)
        return t if t.stride(1) == 1 or k == 1 else t.contiguous()

    if not torch.is_grad_enabled():
        x, At = x.detach(), At.detach()
    if torch.compiler.is_compiling():
        want_grad = torch.is_grad_enabled() and (x.requires_grad or At.requires_grad)
        lse = None if teacher_lse is None else teacher_lse.reshape(rows)
        return distillation_op(x, At, teacher_logits.detach(), teacher_indices, lse, float(temperature),
                               float(logit_scale), int(N_chunk_size), want_grad)[0]
    return LinearDistillationImplementation.apply(
        x, At, lists(teacher_logits), lists(teacher_indices), teacher_lse, temperature, logit_scale, N_chunk_size)


# While a compiler traces, the pass is one opaque operator with its gradients among the outputs, as for the loss.
@torch.library.custom_op("lce_b200::distillation", mutates_args=())
def distillation_op(x: torch.Tensor, At: torch.Tensor, t: torch.Tensor, idx: torch.Tensor, lse: Optional[torch.Tensor],
                    temperature: float, logit_scale: float, N_chunk_size: int,
                    want_grad: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(loss, dx, dAt); the gradients are empty without want_grad."""
    xd, Ad = x.detach(), At.detach()
    if not want_grad:
        loss = linear_distillation(xd, t, idx, Ad, lse, temperature, logit_scale, N_chunk_size)
        return loss, x.new_empty(0), x.new_empty(0)
    with torch.enable_grad():
        xd, Ad = xd.requires_grad_(), Ad.requires_grad_()
        loss = linear_distillation(xd, t, idx, Ad, lse, temperature, logit_scale, N_chunk_size)
    dx, dA = loss.grad_fn.lce_grads
    return loss.detach(), dx.reshape(x.shape).contiguous(), dA.contiguous()


@distillation_op.register_fake
def _distillation_fake(x, At, t, idx, lse, temperature, logit_scale, N_chunk_size, want_grad):
    loss = x.new_empty((), dtype=torch.float32)
    if not want_grad:
        return loss, x.new_empty(0), x.new_empty(0)
    return loss, x.new_empty(x.shape), At.new_empty(At.shape)


def _distillation_setup(ctx, inputs, output):
    ctx.lce_want_grad = inputs[-1]
    ctx.save_for_backward(output[1], output[2])


def _distillation_backward(ctx, grad_loss, grad_dx, grad_dA):
    if not ctx.lce_want_grad:
        raise RuntimeError("the distillation loss was traced without gradients")
    dx, dA = ctx.saved_tensors
    return scaled_op(dx, grad_loss), scaled_op(dA, grad_loss), None, None, None, None, None, None, None


distillation_op.register_autograd(_distillation_backward, setup_context=_distillation_setup)


class LinearDistillationLoss(LinearCrossEntropyLoss):
    """The head of :class:`LinearCrossEntropyLoss` (same constructor, weight and ``state_dict``) with
    ``forward(x, teacher_logits, teacher_indices, teacher_lse=None)`` = :func:`linear_distillation`.

    Assign ``distill.weight = head.weight`` to train one weight with both losses. ``ignore_index``, ``z_regularization``
    and ``monitoring`` have no meaning here.
    """

    def __init__(self, in_features: int, out_features: int, device=None, dtype=None, temperature: float = 1.0,
                 logit_scale: float = 1.0, N_chunk_size: int = 4096, init_method=None):
        assert temperature > 0
        super().__init__(in_features, out_features, device=device, dtype=dtype, logit_scale=logit_scale,
                         N_chunk_size=N_chunk_size, init_method=init_method)
        self.temperature = temperature

    def forward(self, x, teacher_logits, teacher_indices, teacher_lse=None):
        return linear_distillation(x, teacher_logits, teacher_indices, self.weight, teacher_lse, self.temperature,
                                   self.logit_scale, self.N_chunk_size)
