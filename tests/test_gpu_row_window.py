"""Gradients of rows whose logits lie far above the base that the slab of their exponentials was made with.

With one base per row the exponentials go up to exp(72) and more, and the row's factor, exp(base - log-sum-exp) times
whatever else scales the row, far below what the operands of the gradient products can hold by itself. Row maxima on
both sides of the border of the re-run, and far apart between the shards of a vocabulary.
"""
import pytest
import torch

from distill_util import gradient_bounds, loss_bound, reference
from gpu_util import TOL, check_against_oracle, cosine, rel_err
from linear_cross_entropy_loss_b200 import _native, ops
from oracle import oracle
from test_gpu_distill import problem, run

pytestmark = pytest.mark.gpu


@pytest.fixture
def one_base_per_row(monkeypatch):
    monkeypatch.setenv("LCE_SLAB_MODE", "row")


def lift(x, At, height, row=0, first=0):
    """Adds `height` to the logits of all columns from `first` on (an integer or half: exact in every type)."""
    x[:, row] = height
    At[row] = 0
    At[row, first:] = 1


def check_distillation(x, At, t, idx, **kw):
    """The bounds of gradient_bounds hold with room for these heights: the products' sums are rounded to 2^-23 of 73 a
    few times, which moves the softmax by 4.4e-5 of itself at most, and the bounds count 2.02 half steps of bf16 where two
    are made (7.8e-5 more) and 2^-17."""
    ref = reference(x, At, t, idx, lse=kw.get("lse"))
    n = int((ref["mass"] > 0).sum())
    loss, dx, dW = run(x, At, t, idx, **kw)
    dx, dW = dx.double().cpu(), dW.double().cpu()
    if x.dtype == torch.float32:  # TF32 products, as in the other tests of the distillation
        assert abs(loss - ref["loss"]) <= 2e-3 * abs(ref["loss"]) + 1e-4
        for a, b in ((dx, ref["dx"]), (dW, ref["dW"])):
            assert (a - b).norm() <= 6e-3 * b.norm(), ((a - b).norm() / b.norm()).item()
        return
    assert abs(loss - ref["loss"]) <= loss_bound(ref, 1.0, n)
    bx, bw = gradient_bounds(ref, x.dtype)
    assert ((dx - ref["dx"]).abs() <= bx).all(), ((dx - ref["dx"]).abs() / bx).max().item()
    assert ((dW - ref["dW"]).abs() <= bw).all(), ((dW - ref["dW"]).abs() / bw).max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("height", [0, 55, 60, 62, 64, 65, 66, 68, 69, 70, 71, 72, 75])
def test_distillation_near_the_top_of_the_window(one_base_per_row, dtype, height):
    x, At, t, idx = problem(128, 64, 1024, 4, dtype, seed=height)
    lift(x, At, height)
    check_distillation(x, At, t, idx)


@pytest.mark.parametrize("height,log_mass", [(60, -11.5), (70, -4.6), (64, -30.0), (0, -70.0), (40, -60.0), (70, -60.0)])
def test_distillation_of_lists_with_little_mass(one_base_per_row, height, log_mass):
    """The teacher's log-sum-exp says that the lists hold a share of exp(log_mass)."""
    x, At, t, idx = problem(128, 64, 1024, 4, torch.bfloat16, seed=3)
    lift(x, At, height)
    check_distillation(x, At, t, idx, lse=(torch.logsumexp(t.double(), 1) - log_mass).float())


def test_distillation_rows_of_all_kinds_in_one_chunk(one_base_per_row):
    x, At, t, idx = problem(300, 64, 1024, 4, torch.bfloat16, seed=4)
    lift(x, At, 0)
    x[:, 0] = torch.tensor([0.0, 30.0, 64.0, 70.0])[torch.arange(300) % 4].to(x.dtype)
    lse = (torch.logsumexp(t.double(), 1) + torch.tensor([0.0, 2.0, 12.0, 50.0, 80.0])[torch.arange(300) % 5].double()).float()
    check_distillation(x, At, t, idx, lse=lse)
    idx[::7] = -1
    check_distillation(x, At, t, idx, lse=lse, N_chunk_size=128)


@pytest.mark.parametrize("height", [100, 122, 126, 128, 130])
def test_distillation_above_the_columns_that_were_probed(one_base_per_row, height):
    """From 64 tiles of columns on, the base is 58 above the largest of the first two tiles."""
    x, At, t, idx = problem(128, 64, 16700, 4, torch.bfloat16, seed=5)
    lift(x, At, height, first=600)
    ref = reference(x, At, t, idx)
    loss, dx, dW = run(x, At, t, idx)
    # the sums' roundings grow with the height: 2^-23 of 131 a few times, 8e-5 of the softmax, against half a step of 3.9e-3
    for got, want in zip((dx, dW), gradient_bounds(ref, x.dtype)):
        exact = ref["dx"] if got is dx else ref["dW"]
        assert ((got.double().cpu() - exact).abs() <= 1.03 * want).all()
    assert abs(loss - ref["loss"]) <= loss_bound(ref, 1.0, 128)


# ---------------------------------------------------------------------------------------------------- cross-entropy
def labelled(N, H, V, dtype, seed):
    x, At, _, idx = problem(N, H, V, 1, dtype, seed=seed)
    return x, idx[:, 0], At


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("height", [0, 60, 62, 65, 68, 69, 70, 71, 72, 75])
def test_cross_entropy_near_the_top_of_the_window(dtype, height):
    x, y, At = labelled(128, 64, 1024, dtype, height)
    lift(x, At, height)
    check_against_oracle(x, y, At, dtype, monitoring=False)


@pytest.mark.parametrize("height", [100, 126, 128, 130])
def test_cross_entropy_above_the_columns_that_were_probed(height):
    x, y, At = labelled(128, 64, 16700, torch.bfloat16, 6)
    lift(x, At, height, first=600)
    check_against_oracle(x, y, At, torch.bfloat16, monitoring=False)


def test_cross_entropy_rows_of_all_kinds_in_one_chunk():
    x, y, At = labelled(300, 64, 1024, torch.bfloat16, 7)
    lift(x, At, 0)
    x[:, 0] = torch.tensor([0.0, 30.0, 64.0, 70.0, 71.0])[torch.arange(300) % 5].to(x.dtype)
    y[::6] = -100
    check_against_oracle(x, y, At, torch.bfloat16, zreg=1e-3, chunk=128, monitoring=False)


@pytest.mark.parametrize("heights", [(70, 0), (68, 74), (66, 80), (60, 70), (71, 84), (50, 200), (0, 0)])
def test_shards_whose_logits_lie_apart(heights):
    """Two shards, one after the other on this GPU: a row's factor follows the log-sum-exp of both, which may lie as far
    above a shard's own logits as it likes."""
    dtype, N, H, V = torch.bfloat16, 256, 64, 2048
    x, y, W = labelled(N, H, V, dtype, 8)
    x[:, 0], x[:, 1] = heights
    W[:2] = 0
    W[0, :V // 2], W[1, V // 2:] = 1, 1
    be, xd, yd = ops.get_backend(), x.cuda(), y.cuda()
    slabs = [w.contiguous().cuda() for w in W.split(V // 2, dim=1)]
    probs = [_native.Problem(n_rows_total=N, chunk_rows=N, hidden=H, vocab_local=V // 2, vocab_offset=g * V // 2,
                             ignore_index=-1, world=2, dtype=_native.DTYPE_BF16, monitoring=0, want_grad=1,
                             logit_scale=1.0, z_regularization=0.0, slab_mode=_native.SLAB_DEFAULT) for g in range(2)]
    ws = [torch.empty(be.workspace_bytes(p), dtype=torch.uint8, device="cuda") for p in probs]
    parts = torch.empty(2, 6 * N, dtype=torch.float32, device="cuda")
    dx = [torch.zeros(N, H, dtype=torch.float32, device="cuda") for _ in range(2)]
    dW = [torch.empty(H, V // 2, dtype=dtype, device="cuda") for _ in range(2)]
    for g in range(2):
        be.begin(probs[g], yd, ws[g])
        be.forward_chunk(probs[g], xd, slabs[g], yd, 0, N, ws[g], parts[g])
    for g in range(2):
        be.combine_chunk(probs[g], parts, yd, 0, N, ws[g])
        be.dz_chunk(probs[g], xd, yd, 0, N, ws[g])
        be.dx_chunk(probs[g], slabs[g], 0, N, ws[g], dx[g])
        be.dw_chunk(probs[g], xd, 0, N, ws[g], dW[g], None, True, True)
    torch.cuda.synchronize()
    ref = oracle.forward_backward(x, y, W, -1, 0.0, 1.0)
    got = (dx[0].double() + dx[1].double()).cpu().numpy(), torch.cat(dW, dim=1).double().cpu().numpy()
    for a, b in zip(got, (ref.dx, ref.dW)):
        assert cosine(a, b) >= TOL[dtype]["cos"] and rel_err(a, b) <= TOL[dtype]["rel"] + 2e-3, (cosine(a, b), rel_err(a, b))
