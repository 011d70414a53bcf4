"""What a vocabulary head answers with: the largest logits of a row, and tokens drawn from it.

``top_logits`` lists the k largest logits of each row with the row's log-sum-exp -- the form in which a teacher's
distribution is kept for :func:`linear_distillation`. ``sample_logits`` draws one token per row from given random
numbers. Both read the logits once, in ``liblce_b200.so``, on the current stream of the logits' device; like the loss
they have no CPU fallback. ``linear_logits``, ``linear_top_logits`` and ``linear_sample`` start from the head's input and
weight instead and take their logits from the contraction of the loss. The reference project has no counterpart of any of
them.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from . import _native
from .ops import _DTYPE_CODE, _device_guard, get_backend


class TopLogits(NamedTuple):
    values: torch.Tensor   # (..., k) in the type of the logits, descending
    indices: torch.Tensor  # (..., k) int64
    lse: torch.Tensor      # (...) float32: logsumexp(logits / temperature) over the whole row


class Sampled(NamedTuple):
    tokens: torch.Tensor    # (...) int64
    logprobs: torch.Tensor  # (...) float32: of the token, in the distribution that was drawn from


def _rows_of(logits: torch.Tensor) -> torch.Tensor:
    """(rows, V) with unit inner stride; leading dimensions merged (a copy only where the strides do not allow it)."""
    assert logits.dim() >= 1 and logits.shape[-1] >= 1, "logits must have at least one column"
    assert logits.dtype in _DTYPE_CODE, f"unsupported dtype {logits.dtype}"
    rows = logits.detach()
    if rows.dim() != 2:
        rows = rows.reshape(-1, logits.shape[-1])
    return rows if rows.stride(1) == 1 or rows.shape[1] == 1 else rows.contiguous()


def _require_cuda(backend, *tensors) -> None:
    if getattr(backend, "requires_cuda", True) and not all(t.is_cuda for t in tensors):
        raise RuntimeError("linear_cross_entropy_loss_b200 runs on CUDA tensors only; there is no CPU fallback")


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The k largest logits of each row, descending, equal ones by ascending index, and the row's log-sum-exp.

    logits: (..., V) in float16, bfloat16 or float32; rows may start anywhere and lie any distance apart.
    1 <= k <= min(V, 1024). NaN counts as larger than everything, as in ``torch.topk``; ``lse`` is NaN then.
    ``temperature`` only enters ``lse`` = logsumexp(logits / temperature). Not differentiable.
    """
    k = int(k)
    rows = _rows_of(logits)
    assert 1 <= k <= rows.shape[1], "k must lie between 1 and the number of columns"
    assert k <= _native.TOP_MAX, f"k must be at most {_native.TOP_MAX}"
    assert 2**-126 <= temperature < float("inf"), "temperature must be positive"
    if torch.compiler.is_compiling():
        return TopLogits(*top_logits_op(logits.detach(), k, float(temperature)))
    backend = get_backend()
    _require_cuda(backend, rows)
    lead = logits.shape[:-1]
    n, dev = rows.shape[0], rows.device
    values = torch.empty((n, k), dtype=rows.dtype, device=dev)
    indices = torch.empty((n, k), dtype=torch.int64, device=dev)
    lse = torch.empty(n, dtype=torch.float32, device=dev)
    with _device_guard(rows):
        backend.top_logits(rows, k, float(temperature), values, indices, lse)
    if len(lead) != 1:
        values, indices, lse = values.view(*lead, k), indices.view(*lead, k), lse.view(lead)
    return TopLogits(values, indices, lse)


def _head_operands(x: torch.Tensor, At: torch.Tensor):
    """x as (rows, H) and At, as the kernels read them (while a compiler traces: as linear_logits_op takes them)."""
    from .distill import _operands
    from .ops import _autocast_target

    assert x.dim() >= 1 and At.dim() == 2 and At.shape[0] == x.shape[-1], "x and the weight disagree on the hidden size"
    assert At.shape[0] >= 1 and At.shape[1] >= 1
    assert x.device == At.device, "all tensors must be on one device"
    x, At = x.detach(), At.detach()
    target = _autocast_target(x)
    if target is not None:
        x, At = x.to(target), At.to(target)
    assert x.dtype == At.dtype, "x and the weight must have the same dtype"
    assert x.dtype in _DTYPE_CODE, f"unsupported dtype {x.dtype}"
    x = x.reshape(-1, x.shape[-1])
    if torch.compiler.is_compiling():
        return x, At
    _require_cuda(get_backend(), x)
    if x.shape[0] == 0:
        return x, At
    with _device_guard(x):
        return _operands(x, At)


def _logit_rows(x, At, scale: float) -> torch.Tensor:
    """(rows, V) float32 logits, rows on 16-byte boundaries. NaN throughout if a wait inside the contraction ran out: the
    status word is looked at on the device."""
    if torch.compiler.is_compiling():
        return linear_logits_op(x, At, float(scale))
    V = At.shape[1]
    out = torch.empty((x.shape[0], -(-V // 4) * 4), dtype=torch.float32, device=x.device)
    if x.shape[0] > 0:
        status = torch.zeros(1, dtype=torch.int32, device=x.device)
        with _device_guard(x):
            get_backend().linear_logits(x, At, float(scale), out, status)
    return out if out.shape[1] == V else out[:, :V]


def linear_logits(x: torch.Tensor, At: torch.Tensor, logit_scale: float = 1.0) -> torch.Tensor:
    """``logit_scale * (x @ At)`` in float32, (..., V), from the tensor-core contraction of the loss (products accumulated
    in fp32; float32 inputs are multiplied as TF32). Not differentiable: the losses never need the logits themselves."""
    assert logit_scale > 0
    rows, A = _head_operands(x, At)
    return _logit_rows(rows, A, logit_scale).reshape(*x.shape[:-1], At.shape[1])


def linear_top_logits(x: torch.Tensor, At: torch.Tensor, k: int, temperature: float = 1.0, logit_scale: float = 1.0,
                      N_chunk_size: int = 4096) -> TopLogits:
    """:func:`top_logits` of ``logit_scale * (x @ At)``, N_chunk_size rows of logits at a time: a teacher's head."""
    assert logit_scale > 0 and int(N_chunk_size) >= 1
    rows, A = _head_operands(x, At)
    lead, k = x.shape[:-1], int(k)
    # (a batch without rows is one chunk without rows; split() of one cannot be traced)
    chunks = rows.split(int(N_chunk_size)) if rows.shape[0] > 0 else (rows,)
    parts = [top_logits(_logit_rows(c, A, logit_scale), k, temperature) for c in chunks]
    values, indices, lse = parts[0] if len(parts) == 1 else (torch.cat(t) for t in zip(*parts))
    return TopLogits(values.view(*lead, k), indices.view(*lead, k), lse.view(lead))


def linear_sample(x: torch.Tensor, At: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                  logit_scale: float = 1.0, N_chunk_size: int = 4096) -> Sampled:
    """:func:`sample_logits` of ``logit_scale * (x @ At)``, N_chunk_size rows of logits at a time: a head that answers."""
    assert logit_scale > 0 and int(N_chunk_size) >= 1
    rows, A = _head_operands(x, At)
    lead, n = x.shape[:-1], rows.shape[0]
    assert u.shape == lead, "u must have one entry per row of x"
    u = u.reshape(-1)

    def per_row(v, name):
        if not isinstance(v, torch.Tensor):
            return v
        assert v.numel() in (1, n), f"{name} must be a number or have one entry per row"
        return v.reshape(-1).expand(n)

    settings = [per_row(v, name) for v, name in ((temperature, "temperature"), (top_k, "top_k"), (top_p, "top_p"),
                                                 (min_p, "min_p"))]
    parts = []
    for r in range(0, max(n, 1), int(N_chunk_size)):
        here = slice(r, r + int(N_chunk_size))
        parts.append(sample_logits(_logit_rows(rows[here], A, logit_scale), u[here],
                                   *(v[here] if isinstance(v, torch.Tensor) else v for v in settings)))
    tokens, logprobs = parts[0] if len(parts) == 1 else (torch.cat(t) for t in zip(*parts))
    return Sampled(tokens.view(lead), logprobs.view(lead))


def _setting(value, name: str, dtype, n: int, device):
    """(value for all rows, None) or (None, one value per row on the device)."""
    if not isinstance(value, torch.Tensor):
        return value, None
    assert value.numel() in (1, n), f"{name} must be a number or have one entry per row"
    assert value.device == device, f"{name} must be on the device of the logits"
    if dtype == torch.int32 and value.dtype != torch.int32:
        assert not value.is_floating_point() and not value.is_complex(), f"{name} must hold whole numbers"
        value = value.to(torch.int64).clamp(0, 2**31 - 1)
    if value.dtype == dtype and value.dim() == 1 and value.shape[0] == n and value.is_contiguous():
        return None, value
    return None, value.detach().reshape(-1).to(dtype).expand(n).contiguous()


def sample_logits(
    logits: torch.Tensor,
    u: torch.Tensor,
    temperature: Union[float, torch.Tensor] = 1.0,
    top_k: Union[int, torch.Tensor] = 0,
    top_p: Union[float, torch.Tensor] = 1.0,
    min_p: Union[float, torch.Tensor] = 0.0,
) -> Sampled:
    """One token of each row, drawn with the random number that is given for it.

    logits: (..., V) in float16, bfloat16 or float32. u: (...) float32 or float64 in [0, 1).
    With w_j = exp((l_j - max l) / temperature) and the order (logit descending, index ascending): the first ``top_k`` of
    the order stay (0: all); of those the shortest prefix whose mass reaches ``top_p`` of their mass; of those
    w_j >= ``min_p``. The token is the first one in INDEX order at which the kept weights, added up, exceed u times their
    sum; ``logprobs`` is log(w / sum). temperature 0 gives the largest logit (the lowest index among equals).

    Each setting is a number, which is checked, or a tensor with one entry per row (taken as float32; ``top_k`` as int32),
    which is not: out-of-range entries are taken as the nearest value that means something. -inf and NaN logits are never
    drawn; +inf logits share all the mass. A row without any logit to draw gives token -1 and logprob -inf.

    Weights and sums are kept in 64-bit integers (steps of 2^-44 of the largest weight for up to 2^18 columns), so the
    answer for a row depends on its inputs alone; weights below half a step are none.
    """
    if torch.compiler.is_compiling():
        given = [v.detach() if isinstance(v, torch.Tensor) else None for v in (temperature, top_k, top_p, min_p)]
        numbers = [default if isinstance(v, torch.Tensor) else v
                   for v, default in ((temperature, 1.0), (top_k, 0), (top_p, 1.0), (min_p, 0.0))]
        return Sampled(*sample_logits_op(logits.detach(), u.detach(), *given, float(numbers[0]), int(numbers[1]),
                                         float(numbers[2]), float(numbers[3])))
    rows = _rows_of(logits)
    n, dev = rows.shape[0], rows.device
    assert u.numel() == n, "u must have one entry per row of the logits"
    assert u.dtype in (torch.float32, torch.float64), "u must be float32 or float64"
    assert u.device == dev, "u must be on the device of the logits"
    s = _native.Sampling(u_dtype=_native.DTYPE_F32 if u.dtype == torch.float32 else _native.SAMPLING_U_F64)
    if u.dim() != 1 or not u.is_contiguous():
        u = u.detach().reshape(-1).contiguous()
    s.u = u.data_ptr()
    s.temperature_all = s.top_p_all = 1.0  # numbers that the library takes, where a tensor (or no row) stands for them
    alive = []  # what the pointers in `s` refer to, until the kernel has been enqueued
    for name, dtype, value, valid, rule in (
        ("temperature", torch.float32, temperature, lambda v: v >= 0, "temperature must not be negative"),
        ("top_k", torch.int32, top_k, lambda v: v >= 0, "top_k must not be negative"),
        ("top_p", torch.float32, top_p, lambda v: 0 < v <= 1, "top_p must lie in (0, 1]"),
        ("min_p", torch.float32, min_p, lambda v: 0 <= v <= 1, "min_p must lie in [0, 1]"),
    ):
        number, tensor = _setting(value, name, dtype, n, dev)
        if tensor is None:
            number = min(int(number), 2**62) if name == "top_k" else float(number)
            assert valid(number), rule
            setattr(s, f"{name}_all", number)
        else:
            alive.append(tensor)
            setattr(s, name, tensor.data_ptr())
    backend = get_backend()
    _require_cuda(backend, rows, u)
    tokens = torch.empty(n, dtype=torch.int64, device=dev)
    logprobs = torch.empty(n, dtype=torch.float32, device=dev)
    with _device_guard(rows):
        backend.sample_logits(rows, s, tokens, logprobs)
    lead = logits.shape[:-1]
    return Sampled(tokens, logprobs) if len(lead) == 1 else Sampled(tokens.view(lead), logprobs.view(lead))


# ------------------------------------------------------------------------------------------------
# torch.library registration, as for the loss: while a compiler traces, each call is one opaque operator.
# ------------------------------------------------------------------------------------------------
@torch.library.custom_op("lce_b200::top_logits", mutates_args=())
def top_logits_op(logits: torch.Tensor, k: int, temperature: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return tuple(top_logits(logits, k, temperature))


@top_logits_op.register_fake
def _top_logits_fake(logits, k, temperature):
    lead = logits.shape[:-1]
    return (logits.new_empty((*lead, k)), logits.new_empty((*lead, k), dtype=torch.int64),
            logits.new_empty(lead, dtype=torch.float32))


@torch.library.custom_op("lce_b200::linear_logits", mutates_args=())
def linear_logits_op(x: torch.Tensor, At: torch.Tensor, logit_scale: float) -> torch.Tensor:
    """x: (rows, H)."""
    return linear_logits(x, At, logit_scale).contiguous()


@linear_logits_op.register_fake
def _linear_logits_fake(x, At, logit_scale):
    return x.new_empty((x.shape[0], At.shape[1]), dtype=torch.float32)


@torch.library.custom_op("lce_b200::sample_logits", mutates_args=())
def sample_logits_op(logits: torch.Tensor, u: torch.Tensor, temperatures: Optional[torch.Tensor],
                     top_ks: Optional[torch.Tensor], top_ps: Optional[torch.Tensor], min_ps: Optional[torch.Tensor],
                     temperature: float, top_k: int, top_p: float, min_p: float) -> tuple[torch.Tensor, torch.Tensor]:
    """Each setting as a tensor, or, where that is None, as a number."""
    return tuple(sample_logits(logits, u, temperature if temperatures is None else temperatures,
                               top_k if top_ks is None else top_ks, top_p if top_ps is None else top_ps,
                               min_p if min_ps is None else min_ps))


@sample_logits_op.register_fake
def _sample_logits_fake(logits, u, temperatures, top_ks, top_ps, min_ps, temperature, top_k, top_p, min_p):
    lead = logits.shape[:-1]
    return logits.new_empty(lead, dtype=torch.int64), logits.new_empty(lead, dtype=torch.float32)
