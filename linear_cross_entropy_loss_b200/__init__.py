"""B200-native fused linear + cross-entropy loss.

Same public names as ``linear_cross_entropy`` (the reference package, __init__.py:1):
``LinearCrossEntropyLoss``, ``linear_cross_entropy``, ``fwd_configs``, ``bwd_configs``. Beside them, on the same heads:
``LinearDistillationLoss``, ``linear_distillation``, ``top_logits`` and ``sample_logits``.
"""
from .ops import (  # noqa: F401
    LinearCrossEntropyLoss,
    LinearXentImplementation,
    bwd_configs,
    fwd_configs,
    linear_cross_entropy,
    set_autocast_policy,
)

from .distill import LinearDistillationLoss, linear_distillation  # noqa: F401
from .head import Sampled, TopLogits, sample_logits, top_logits  # noqa: F401

__all__ = ["LinearCrossEntropyLoss", "linear_cross_entropy", "fwd_configs", "bwd_configs", "set_autocast_policy",
           "LinearDistillationLoss", "linear_distillation", "top_logits", "TopLogits", "sample_logits", "Sampled"]
