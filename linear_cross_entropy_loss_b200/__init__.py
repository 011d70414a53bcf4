"""B200-native fused linear + cross-entropy loss.

Same public names as ``linear_cross_entropy`` (the reference package, __init__.py:1):
``LinearCrossEntropyLoss``, ``linear_cross_entropy``, ``fwd_configs``, ``bwd_configs``. Beside them, on the same heads:
``LinearDistillationLoss``, ``linear_distillation``, ``top_logits`` and ``sample_logits``, the last two also from
the head's input (``linear_top_logits``, ``linear_sample``, ``linear_logits``).
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
from .head import (  # noqa: F401
    Sampled,
    TopLogits,
    linear_logits,
    linear_sample,
    linear_top_logits,
    sample_logits,
    top_logits,
)

__all__ = ["LinearCrossEntropyLoss", "linear_cross_entropy", "fwd_configs", "bwd_configs", "set_autocast_policy",
           "LinearDistillationLoss", "linear_distillation", "top_logits", "TopLogits", "sample_logits", "Sampled",
           "linear_logits", "linear_top_logits", "linear_sample"]
