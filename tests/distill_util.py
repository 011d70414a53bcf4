"""linear_distillation in 64 bits on the CPU, straight from its definition, with bounds for what rounding may do."""
import math

import torch


def teacher_weights(t, idx, V, T, lse=None):
    """(q (N, K), plogp (N)): zero where an entry is not there."""
    there = (idx >= 0) & (idx < V)
    l = torch.where(there, t.double() / T, torch.full(t.shape, -math.inf, dtype=torch.float64))
    # (the largest logit is taken off before the sum: next to the lowest number of a type a logarithm is lost)
    base = l.amax(1) if lse is None else lse.double()
    base = torch.where(base == -math.inf, torch.zeros_like(base), base)
    q = torch.where(there, torch.exp(l - base[:, None]), torch.zeros_like(l))
    if lse is None:
        q = q / q.sum(1, keepdim=True).clamp(min=1e-300)
    return q, torch.special.xlogy(q, q).sum(1)


def reference(x, At, t, idx, T=1.0, scale=1.0, lse=None):
    """dict: loss, dx, dW and dz (the gradient of n * loss / (scale T) with respect to the logits), p, q, log-sum-exp."""
    x, At = x.double().reshape(-1, x.shape[-1]), At.double()
    K = t.shape[-1]
    t, idx = t.reshape(-1, K), idx.reshape(-1, K).long()
    lse = None if lse is None else lse.reshape(-1)
    V = At.shape[1]
    z = scale / T * (x @ At)
    q, plogp = teacher_weights(t, idx, V, T, lse)
    mass = q.sum(1)
    n = int((mass > 0).sum())
    row_lse = torch.logsumexp(z, 1)
    p = torch.exp(z - row_lse[:, None])
    dense = torch.zeros_like(z).scatter_add_(1, idx.clamp(0, V - 1), q)
    loss = T * T / n * (plogp - (dense * z).sum(1) + mass * row_lse).sum() if n else torch.tensor(math.nan)
    dz = mass[:, None] * p - dense
    c = scale * T / n if n else math.nan
    return dict(loss=float(loss), dx=c * dz @ At.T, dW=c * x.T @ dz, dz=dz, p=p, mass=mass, c=c, z=z, lse=row_lse, x=x,
                At=At, q_z=(dense * z.abs()).sum(1))


HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def loss_bound(ref, T, n):
    """fp32 arithmetic on the row terms: the exponentials and their sum to 2^-20, logits and log-sum-exp to 2^-21 of their size."""
    size = (ref["mass"] * ref["lse"].abs() + ref["q_z"]).sum().item() / max(n, 1)
    return T * T * (2.0 ** -18 + 2.0 ** -20 * size) + 2.0 ** -23 * abs(ref["loss"])


def gradient_bounds(ref, dtype):
    """Largest element-wise errors (dx, dW) of a 16-bit pass. dZ is rounded to the type at most twice (per-tile slabs), or once
    and the rows of x once more (one base per row); the sums are rounded once; logits in fp32 move dZ by 2^-19 of the softmax.
    fp16 keeps exp(z - tile max) and 2^14 dZ with a smallest step of 2^-24."""
    h = HALF_STEP[dtype]
    dz, x, At, c = ref["dz"].abs(), ref["x"].abs(), ref["At"].abs(), ref["c"]
    err = 2.02 * h * dz + 2.0 ** -17 * ref["p"] * ref["mass"][:, None]
    tiny = 2.0 ** -126
    if dtype == torch.float16:
        err = err + (2.0 ** -24 * ref["p"].amax(1, keepdim=True) + 2.0 ** -39) * (ref["mass"] > 0)[:, None]
        tiny = 2.0 ** -25
    dx = 1.02 * c * err @ At.T + 1.01 * h * ref["dx"].abs() + tiny
    # the sum over the chunks is carried as value + residual, good to h^2
    dW = 1.02 * c * x.T @ err + (1.01 * h + 8 * h * h) * ref["dW"].abs() + tiny
    dW = dW + 8 * h * h * c * x.T @ dz
    return dx, dW
