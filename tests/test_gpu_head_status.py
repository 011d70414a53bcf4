"""A wait that ran out inside the contraction of a head: what is made from its logits says so."""
import math

import pytest
import torch

from linear_cross_entropy_loss_b200 import LinearCrossEntropyLoss, linear_logits, ops

pytestmark = pytest.mark.gpu


class WaitRanOut(ops.NativeBackend):
    """The library, with the status word as such a contraction leaves it."""

    def linear_logits(self, x, At, scale, out, status):
        status.fill_(1)
        super().linear_logits(x, At, scale, out, status)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,V,chunk", [(1, 1001, 4096), (3, 1, 4096), (300, 2048, 128), (130, 5003, 4096)])
def test_answers_of_a_head_whose_contraction_gave_up(dtype, N, V, chunk):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(N, 64, generator=g).to(dtype).cuda()
    u = torch.rand(N, generator=g).cuda()
    head = LinearCrossEntropyLoss(64, V, device="cuda", dtype=dtype, N_chunk_size=chunk)
    try:
        ops.set_backend(WaitRanOut())
        logits, top, drawn = head.logits(x), head.top_logits(x, 1), head.sample(x, u, top_p=0.9)
        short = head.sample(x, u, top_k=1)
    finally:
        ops.set_backend(None)
    assert logits.shape == (N, V) and logits.isnan().all()
    assert top.values.isnan().all() and top.lse.isnan().all()
    for got in (drawn, short):
        assert (got.tokens == -1).all() and (got.logprobs == -math.inf).all()
    assert linear_logits(x, head.weight).isfinite().all()  # the next call is a call of its own


def test_nothing_beside_the_logits_is_written():
    x = torch.randn(5, 64, device="cuda", dtype=torch.bfloat16)
    At = torch.randn(64, 1000, device="cuda", dtype=torch.bfloat16)
    for given in (0, 1):
        wide = torch.full((7, 1040), 3.0, device="cuda")
        status = torch.full((1,), given, dtype=torch.int32, device="cuda")
        ops.get_backend().linear_logits(x, At, 1.0, wide[1:6, 20:1020], status)
        assert wide[1:6, 20:1020].isnan().all() if given else wide[1:6, 20:1020].isfinite().all()
        wide[1:6, 20:1020] = 3.0
        assert (wide == 3.0).all() and status.item() == given
