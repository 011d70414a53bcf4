"""linear_distillation against its definition in 64 bits."""
import math
import os

import pytest
import torch

from distill_util import gradient_bounds, loss_bound, reference
from linear_cross_entropy_loss_b200 import (LinearCrossEntropyLoss, LinearDistillationLoss, linear_cross_entropy,
                                            linear_distillation, linear_logits, sample_logits, top_logits)

pytestmark = pytest.mark.gpu


def problem(N, H, V, K, dtype, seed=0, pads=False, t_dtype=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, H, generator=g).to(dtype)
    At = (torch.randn(H, V, generator=g).clamp(-2, 2) * H ** -0.5).to(dtype)
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)])
    t = (2.5 * torch.randn(N, K, generator=g) + 5).to(t_dtype or dtype)
    if pads:
        length = torch.randint(0, K + 1, (N, 1), generator=g)
        length[0] = K
        pad = torch.arange(K) >= length
        idx = idx.masked_fill(pad, -1)
        t = t.masked_fill(pad, math.nan)  # what stands in a place that is not there does not matter
    return x, At, t, idx


def run(x, At, t, idx, **kw):
    xd, Ad = x.cuda().requires_grad_(), At.cuda().requires_grad_()
    lse = kw.pop("lse", None)
    loss = linear_distillation(xd, t.cuda(), idx.cuda(), Ad, teacher_lse=None if lse is None else lse.cuda(), **kw)
    dx, dW = torch.autograd.grad(loss, (xd, Ad))
    return loss.item(), dx, dW


def check(x, At, t, idx, T=1.0, scale=1.0, lse=None, chunk=4096, modes=("auto", "row", "tile")):
    ref = reference(x, At, t, idx, T, scale, lse)
    n = int((ref["mass"] > 0).sum())
    dtype = x.dtype
    old = os.environ.get("LCE_SLAB_MODE")
    try:
        for mode in modes if dtype != torch.float16 else modes[:1]:
            os.environ["LCE_SLAB_MODE"] = mode
            loss, dx, dW = run(x, At, t, idx, temperature=T, logit_scale=scale, lse=lse, N_chunk_size=chunk)
            assert dx.dtype == dtype and dx.shape == x.shape and dW.dtype == dtype and dW.shape == At.shape
            dx, dW = dx.double().cpu().reshape(ref["dx"].shape), dW.double().cpu()
            if dtype == torch.float32:  # operands of the products are TF32: 2^-10 of each, which moves the logits too
                assert abs(loss - ref["loss"]) <= 2e-3 * abs(ref["loss"]) + 1e-4
                for a, b in ((dx, ref["dx"]), (dW, ref["dW"])):
                    assert (a - b).norm() <= 6e-3 * b.norm(), (mode, ((a - b).norm() / b.norm()).item())
                continue
            assert abs(loss - ref["loss"]) <= loss_bound(ref, T, n), (mode, loss, ref["loss"])
            bx, bw = gradient_bounds(ref, dtype)
            assert ((dx - ref["dx"]).abs() <= bx).all(), (mode, ((dx - ref["dx"]).abs() / bx).max().item())
            assert ((dW - ref["dW"]).abs() <= bw).all(), (mode, ((dW - ref["dW"]).abs() / bw).max().item())
    finally:
        os.environ.pop("LCE_SLAB_MODE", None)
        if old is not None:
            os.environ["LCE_SLAB_MODE"] = old
    return ref


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,H,V,K,chunk", [
    (1, 64, 300, 1, 4096), (2, 8, 256, 4, 4096), (16, 256, 4096, 8, 4096), (128, 64, 257, 64, 4096), (130, 128, 1000, 33, 128),
    (300, 256, 2048, 16, 256), (257, 72, 5003, 100, 128), (64, 64, 1025, 1000, 4096), (33, 40, 1024, 1024, 4096),
    (700, 136, 999, 7, 512), (256, 512, 20000, 50, 4096),
])
def test_against_the_definition(dtype, N, H, V, K, chunk):
    check(*problem(N, H, V, K, dtype, seed=N + V), chunk=chunk)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,scale", [(2.0, 1.0), (0.5, 1.0), (1.0, 3.0), (4.0, 0.25)])
def test_temperature_and_scale(dtype, T, scale):
    check(*problem(200, 128, 3000, 20, dtype, seed=5), T=T, scale=scale, chunk=128)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_given_log_sum_exp(dtype):
    x, At, t, idx = problem(140, 96, 1500, 12, dtype, seed=6)
    lse = torch.logsumexp(t.double() / 1.5, 1).float() + torch.rand(140, generator=torch.Generator().manual_seed(1))
    check(x, At, t, idx, T=1.5, lse=lse)
    x, At, t, idx = problem(140, 96, 1500, 12, dtype, seed=7, pads=True)
    lse = torch.logsumexp(torch.where(idx >= 0, t.double(), torch.tensor(-math.inf, dtype=torch.float64)), 1).float()
    lse = torch.where(torch.isfinite(lse), lse + 0.25, torch.full_like(lse, math.nan))  # rows without entries
    ref = check(x, At, t, idx, lse=torch.nan_to_num(lse))
    assert 0 < (ref["mass"] > 0).sum() < 140


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_padded_lists_and_rows_without_any(dtype):
    x, At, t, idx = problem(300, 64, 2000, 24, dtype, seed=8, pads=True)
    idx[17:60] = -1
    idx[100, 5] = 2000       # outside on the other side
    idx[101, 3] = 2 ** 40
    check(x, At, t, idx, chunk=128)


def test_entries_without_weight():
    x, At, t, idx = problem(64, 64, 700, 9, torch.bfloat16, seed=9)
    t[:, 4] = -math.inf
    t[3] = -math.inf         # nothing left of this row
    t[5, :8] = -math.inf     # one entry left
    t[6] = torch.finfo(torch.bfloat16).min
    check(x, At, t, idx)


@pytest.mark.parametrize("dtype,T", [(torch.bfloat16, 0.5), (torch.float32, 0.25), (torch.float32, 0.9), (torch.float16, 0.5)])
def test_lists_at_the_ends_of_a_type_at_low_temperatures(dtype, T):
    """Finite logits have weight whatever they are: divided by the temperature they may be more than a float holds, their
    distances from the largest one are what counts."""
    x, At, t, idx = problem(64, 64, 700, 9, torch.bfloat16, seed=30, t_dtype=dtype)
    lowest, largest = torch.finfo(dtype).min, torch.finfo(dtype).max
    t[6], t[7] = lowest, largest         # nine equal ones
    t[8], t[8, 3] = lowest, 1.0          # one far above the others
    t[9], t[9, 3:5] = lowest, largest
    t[10, 2:] = -math.inf
    t[10, :2] = lowest
    check(x, At, t, idx, T=T)


def test_an_index_listed_twice_counts_twice():
    x, At, t, idx = problem(70, 64, 700, 10, torch.bfloat16, seed=10)
    idx[:, 3] = idx[:, 0]
    idx[:, 9] = idx[:, 0]
    idx[5] = 699
    idx[6] = 0
    check(x, At, t, idx)


def test_lists_on_tile_borders():
    x, At, t, idx = problem(40, 64, 1024, 8, torch.bfloat16, seed=11)
    idx[:] = torch.tensor([0, 255, 256, 511, 512, 767, 768, 1023])
    check(x, At, t, idx)
    idx[:] = torch.tensor([256, 257, 258, 259, 260, 300, 400, 511])
    check(x, At, t, idx)


def test_types_and_layouts_of_the_lists():
    x, At, t, idx = problem(48, 64, 900, 12, torch.bfloat16, seed=12, t_dtype=torch.float32)
    want = run(x, At, t, idx)
    check(x, At, t, idx)
    wide_t, wide_i = torch.zeros(48, 30), torch.zeros(48, 30, dtype=torch.int32)
    wide_t[:, 5:17], wide_i[:, 5:17] = t, idx
    xd, Ad = x.cuda(), At.cuda()
    got = linear_distillation(xd, wide_t.cuda()[:, 5:17], wide_i.cuda()[:, 5:17], Ad)
    assert got.item() == want[0]
    got = linear_distillation(xd, t.cuda().t().contiguous().t(), idx.cuda().t().contiguous().t(), Ad)
    assert got.item() == want[0]
    got = linear_distillation(xd.view(6, 8, 64), t.cuda().view(6, 8, 12), idx.cuda().view(6, 8, 12), Ad)
    assert got.item() == want[0]
    for order in (torch.randperm(12), torch.arange(11, -1, -1)):
        got = linear_distillation(xd, t[:, order].cuda(), idx[:, order].cuda(), Ad)
        assert abs(got.item() - want[0]) <= 1e-6 * abs(want[0])
    half = t.half()
    check(x, At, half, idx)


@pytest.mark.parametrize("N,H,V,K,T,chunk", [(513, 8, 9000, 17, 0.5, 128), (513, 200, 9000, 1, 0.5, 1),
                                             (300, 64, 9000, 300, 0.5, 256), (700, 70, 9001, 64, 1.0, 128)])
def test_small_gradients_summed_over_chunks(N, H, V, K, T, chunk):
    """dW below fp16's normal numbers: every chunk adds to it, only the last may round to a step of 2^-24."""
    check(*problem(N, H, V, K, torch.float16, seed=N + K), T=T, chunk=chunk)


@pytest.mark.parametrize("H,V", [(60, 777), (250, 1001), (64, 1003), (13, 256)])
def test_sizes_that_need_copies(H, V):
    check(*problem(150, H, V, 11, torch.bfloat16, seed=H), chunk=128)


def test_strided_operands():
    x, At, t, idx = problem(96, 64, 1024, 8, torch.bfloat16, seed=13)
    wide_x, wide_A = torch.zeros(96, 96, dtype=torch.bfloat16), torch.zeros(64, 1100, dtype=torch.bfloat16)
    wide_x[:, 16:80], wide_A[:, 24:1048] = x, At
    want = run(x, At, t, idx)
    xd, Ad = wide_x.cuda()[:, 16:80].requires_grad_(), wide_A.cuda()[:, 24:1048].requires_grad_()
    loss = linear_distillation(xd, t.cuda(), idx.cuda(), Ad)
    dx, dW = torch.autograd.grad(loss, (xd, Ad))
    assert loss.item() == want[0] and torch.equal(dx, want[1]) and torch.equal(dW, want[2])


def test_no_row_counts():
    x, At, t, idx = problem(20, 64, 300, 5, torch.bfloat16)
    idx[:] = -1
    assert math.isnan(linear_distillation(x.cuda(), t.cuda(), idx.cuda(), At.cuda()).item())


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_nan_and_inf_of_a_listed_logit_reach_the_loss(bad):
    x, At, t, idx = problem(20, 64, 300, 5, torch.bfloat16)
    t[7, 2] = bad
    assert math.isnan(linear_distillation(x.cuda(), t.cuda(), idx.cuda(), At.cuda()).item())


def test_rows_that_do_not_count_do_not_matter():
    """Rows behind the last one of a sequence: whatever x holds there, with an empty list its gradient is zero."""
    x, At, t, idx = problem(90, 64, 512, 6, torch.bfloat16, seed=14)
    idx[70:] = -1
    want = run(x[:70], At, t[:70], idx[:70])
    loss, dx, dW = run(x, At, t, idx)
    assert abs(loss - want[0]) <= 1e-6 * abs(want[0])
    assert (dx[70:] == 0).all()
    assert torch.allclose(dW.float(), want[2].float(), rtol=2 ** -7, atol=1e-6)


def test_one_listed_token_is_the_cross_entropy():
    N, H, V = 320, 128, 4096
    x, At, t, idx = problem(N, H, V, 1, torch.bfloat16, seed=15)
    y = idx[:, 0].clone()
    y[::7] = -100
    idx[::7] = -1
    loss, dx, dW = run(x, At, t, idx)
    xd, Ad = x.cuda().requires_grad_(), At.cuda().requires_grad_()
    ce = linear_cross_entropy(xd, y.cuda(), Ad)[0]
    gx, gA = torch.autograd.grad(ce, (xd, Ad))
    assert abs(loss - ce.item()) <= 1e-6 * abs(loss)
    assert (dx.float() - gx.float()).norm() <= 4e-3 * gx.float().norm()
    assert (dW.float() - gA.float()).norm() <= 4e-3 * gA.float().norm()


def test_gradient_against_differences_of_the_loss():
    """Central differences along random directions whose steps the type holds exactly (x and At on a grid of 2^-5)."""
    g = torch.Generator().manual_seed(16)
    N, H, V, K, T = 48, 64, 512, 6, 1.5
    x = (torch.randn(N, H, generator=g) * 8).round() / 8
    At = (torch.randn(H, V, generator=g) * 16).round().clamp(-24, 24) / 128
    _, _, t, idx = problem(N, H, V, K, torch.bfloat16, seed=17)
    x, At = x.to(torch.bfloat16), At.to(torch.bfloat16)
    _, dx, dW = run(x, At, t, idx, temperature=T)

    def loss_at(x, At):
        return linear_distillation(x.cuda(), t.cuda(), idx.cuda(), At.cuda(), temperature=T).item()

    for which, grad, step in (("x", dx, 2.0 ** -5), ("At", dW, 2.0 ** -9)):
        v = torch.sign(grad.float().cpu())  # the steepest direction of steps of one size
        base = x if which == "x" else At
        up, down = (base.float() + step * v).to(torch.bfloat16), (base.float() - step * v).to(torch.bfloat16)
        moved = (up.double() - down.double())
        want = (moved * grad.double().cpu()).sum().item()
        got = (loss_at(up, At) - loss_at(down, At)) if which == "x" else (loss_at(x, up) - loss_at(x, down))
        assert abs(got - want) <= 0.03 * abs(want), (which, got, want)


def test_only_what_is_asked_for():
    x, At, t, idx = problem(200, 64, 1000, 8, torch.bfloat16, seed=18)
    loss, dx, dW = run(x, At, t, idx)
    td, id_ = t.cuda(), idx.cuda()
    xd, Ad = x.cuda().requires_grad_(), At.cuda()
    out = linear_distillation(xd, td, id_, Ad)
    assert torch.equal(torch.autograd.grad(out, xd)[0], dx)
    xd, Ad = x.cuda(), At.cuda().requires_grad_()
    out = linear_distillation(xd, td, id_, Ad)
    assert torch.equal(torch.autograd.grad(out, Ad)[0], dW)
    with torch.no_grad():
        assert not linear_distillation(xd, td, id_, Ad).requires_grad
    assert abs(linear_distillation(x.cuda(), td, id_, At.cuda()).item() - loss) <= 1e-6 * abs(loss)


def test_factor_of_backward_and_second_call():
    x, At, t, idx = problem(100, 64, 600, 5, torch.bfloat16, seed=19)
    _, dx, dW = run(x, At, t, idx)
    xd, Ad = x.cuda().requires_grad_(), At.cuda().requires_grad_()
    loss = linear_distillation(xd, t.cuda(), idx.cuda(), Ad)
    (4 * loss).backward()
    assert torch.equal(xd.grad, 4 * dx) and torch.equal(Ad.grad, 4 * dW)
    loss = linear_distillation(xd, t.cuda(), idx.cuda(), Ad)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="backward called twice"):
        loss.backward()


def test_module_and_autocast():
    torch.manual_seed(0)
    head = LinearDistillationLoss(64, 900, temperature=2.0, logit_scale=0.5, N_chunk_size=128, device="cuda")
    assert list(head.state_dict()) == ["weight"] and head.weight.shape == (64, 900)
    x, _, t, idx = problem(150, 64, 900, 9, torch.bfloat16, seed=20)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        xd = x.float().cuda().requires_grad_()
        loss = head(xd, t.float().cuda(), idx.cuda())
    loss.backward()
    ref = reference(x.half(), head.weight.detach().cpu().half(), t, idx, 2.0, 0.5)  # the policy "reference" casts to fp16
    assert abs(loss.item() - ref["loss"]) <= 1e-5 * abs(ref["loss"])
    assert xd.grad.dtype == torch.float32 and head.weight.grad.dtype == torch.float32
    assert (xd.grad.double().cpu() - ref["dx"]).norm() <= 3e-3 * ref["dx"].norm()
    assert (head.weight.grad.double().cpu() - ref["dW"]).norm() <= 3e-3 * ref["dW"].norm()


def test_recomputed_row_groups_keep_their_lists():
    """Logits far outside the window of the first pass: the groups that are run again list their logits again."""
    x, At, t, idx = problem(600, 64, 1024, 8, torch.bfloat16, seed=21)
    x[300:340] *= 16
    check(x, At, t, idx, scale=4.0, chunk=512, modes=("row",))


def test_same_result_on_another_stream_and_twice():
    x, At, t, idx = problem(500, 128, 3000, 16, torch.bfloat16, seed=22, pads=True)
    want = run(x, At, t, idx, N_chunk_size=256)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, At, t, idx, N_chunk_size=256)
    torch.cuda.synchronize()
    assert got[0] == want[0] and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_captured_step(dtype):
    x, At, t, idx = (v.cuda() for v in problem(300, 64, 2000, 8, dtype, seed=23))
    x.requires_grad_()
    At.requires_grad_()

    def step():
        loss = linear_distillation(x, t, idx, At, N_chunk_size=128)
        return (loss.detach(), *torch.autograd.grad(loss, (x, At)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        x.copy_(problem(300, 64, 2000, 8, dtype, seed=24)[0].cuda())
    graph.replay()
    torch.cuda.synchronize()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_student_samples_teacher_lists_student_learns():
    """The operators as an on-policy distillation step runs them."""
    torch.manual_seed(0)
    H, V, B = 128, 5000, 64
    teacher = LinearCrossEntropyLoss(H, V, device="cuda", dtype=torch.bfloat16)
    student = LinearDistillationLoss(H, V, device="cuda", dtype=torch.bfloat16, temperature=1.5)
    states = torch.randn(B, H, device="cuda", dtype=torch.bfloat16)
    tokens = sample_logits(states @ student.weight, torch.rand(B, device="cuda"), top_k=50, top_p=0.95).tokens
    assert ((tokens >= 0) & (tokens < V)).all()
    values, indices, lse = top_logits((states @ teacher.weight)[:, :], 32, temperature=1.5)
    h = states.clone().requires_grad_()
    loss = student(h, values, indices, lse)
    loss.backward()
    ref = reference(states.cpu(), student.weight.detach().cpu(), values.cpu(), indices.cpu(), 1.5, 1.0, lse.cpu())
    assert abs(loss.item() - ref["loss"]) <= loss_bound(ref, 1.5, B)
    bx, bw = gradient_bounds(ref, torch.bfloat16)
    assert ((h.grad.double().cpu() - ref["dx"]).abs() <= bx).all()
    assert ((student.weight.grad.double().cpu() - ref["dW"]).abs() <= bw).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols,ld,offset", [(1, 1, 1, 0), (3, 7, 7, 1), (5, 50257, 50257, 0), (64, 1003, 1010, 3), (9, 64, 64, 5)])
def test_rows_are_moved_to_boundaries(dtype, rows, cols, ld, offset):
    from linear_cross_entropy_loss_b200.distill import _aligned

    g = torch.Generator().manual_seed(cols)
    flat = torch.randn(rows * ld + offset, generator=g).to(dtype).cuda()
    src = flat[offset:].view(rows, ld)[:, :cols]
    got = _aligned(src)
    assert torch.equal(got, src) and got.data_ptr() % 16 == 0
    assert rows == 1 or got.stride(0) * got.element_size() % 16 == 0


def test_traced_by_torch_compile_without_a_graph_break():
    x, At, t, idx = problem(100, 64, 700, 6, torch.bfloat16, seed=25)
    want = run(x, At, t, idx, temperature=1.5)
    xd, Ad, td, id_ = x.cuda().requires_grad_(), At.cuda().requires_grad_(), t.cuda(), idx.cuda()
    step = torch.compile(lambda a, b: 2.0 * linear_distillation(a, td, id_, b, temperature=1.5), fullgraph=True, backend="aot_eager")
    loss = step(xd, Ad)
    loss.backward()
    assert loss.item() == 2 * want[0]
    assert torch.equal(xd.grad, 2 * want[1]) and torch.equal(Ad.grad, 2 * want[2])


@pytest.mark.parametrize("factor", [65536.0, 0.3])
def test_traced_fp16_gradients_are_scaled_like_eager_ones(factor):
    """A GradScaler's factor is not a number of fp16, the gradients that it scales are."""
    x, At, t, idx = problem(100, 64, 700, 6, torch.float16, seed=31)
    td, id_ = t.cuda(), idx.cuda()

    def grads(call):
        xd, Ad = x.cuda().requires_grad_(), At.cuda().requires_grad_()
        return torch.autograd.grad(factor * call(xd, Ad), (xd, Ad))

    call = lambda a, b: linear_distillation(a, td, id_, b)  # noqa: E731
    for got, want in zip(grads(torch.compile(call, fullgraph=True, backend="aot_eager")), grads(call)):
        assert want.isfinite().all() and torch.equal(got, want)


def test_a_head_traced_by_torch_compile_without_a_graph_break():
    head = LinearCrossEntropyLoss(64, 1001, device="cuda", dtype=torch.bfloat16, N_chunk_size=50)
    h, u = torch.randn(4, 30, 64, device="cuda", dtype=torch.bfloat16), torch.rand(4, 30, device="cuda")
    call = lambda h, u: (head.logits(h), *head.top_logits(h, 5), *head.sample(h, u, top_p=0.9))  # noqa: E731
    got = torch.compile(call, fullgraph=True, backend="aot_eager")(h, u)
    want = call(h, u)
    assert all(a.shape == b.shape and a.dtype == b.dtype for a, b in zip(got, want))
    # rows of the traced logits lie 1001 elements apart, not 1004, so their exponentials are added up in another order: at
    # most 64 one after the other, in both
    lse = got[3], want[3]
    assert ((lse[0] - lse[1]).abs() <= 2 * (64 + lse[0].abs()) * 2.0**-24).all()
    assert all(torch.equal(a, b) for i, (a, b) in enumerate(zip(got, want)) if i != 3)


def test_traced_operators_are_what_their_shapes_promise():
    """Sizes and strides of the outputs, at a vocabulary whose rows are padded inside."""
    x, At, t, idx = (v.cuda() for v in problem(40, 60, 701, 6, torch.bfloat16, seed=26))
    ops, utils = torch.ops.lce_b200, ("test_schema", "test_faketensor")
    lse, u = torch.logsumexp(t.float(), 1), torch.rand(40, device="cuda")
    ks = torch.full((40,), 9, device="cuda")
    torch.library.opcheck(ops.distillation.default, (x, At, t, idx, lse, 2.0, 1.0, 128, True), test_utils=utils)
    torch.library.opcheck(ops.distillation.default, (x, At, t, idx, None, 2.0, 1.0, 4096, False), test_utils=utils)
    torch.library.opcheck(ops.linear_logits.default, (x, At, 1.0), test_utils=utils)
    logits = linear_logits(x, At).view(4, 10, 701)
    torch.library.opcheck(ops.top_logits.default, (logits, 5, 1.0), test_utils=utils)
    torch.library.opcheck(ops.sample_logits.default, (logits, u.view(4, 10), None, ks, None, None, 1.0, 0, 0.9, 0.0),
                          test_utils=utils)


def test_broadcast_inputs_and_lists():
    """One row of x and one list for all rows: the gradient is the sum, the loss that of one row."""
    x, At, t, idx = problem(1, 64, 700, 6, torch.float32, seed=27)
    one = run(x, At, t, idx)
    xd, Ad = x.cuda().requires_grad_(), At.cuda().requires_grad_()
    loss = linear_distillation(xd.expand(40, 64), t.cuda().expand(40, 6), idx.cuda().expand(40, 6), Ad)
    loss.backward()
    assert abs(loss.item() - one[0]) <= 1e-6 * abs(one[0])
    for got, want in ((xd.grad, one[1]), (Ad.grad, one[2])):  # each within the 6e-3 of check() from the formula
        assert (got - want).norm() <= 1.2e-2 * want.norm()


def test_given_log_sum_exp_of_rows_without_a_list():
    """What a teacher's log-sum-exp is where its list is empty does not matter, and -inf lists with -inf neither."""
    x, At, t, idx = problem(50, 64, 700, 6, torch.bfloat16, seed=28)
    lse = torch.logsumexp(t.double(), 1).float() + 0.3
    idx[3], idx[4] = -1, 700
    t[5] = -math.inf
    want = run(x, At, t, idx, lse=lse)
    lse[3], lse[4], lse[5] = math.nan, math.inf, -math.inf
    got = run(x, At, t, idx, lse=lse)
    assert math.isfinite(got[0]) and got[0] == want[0] and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


def test_lists_further_apart_than_31_bits():
    x, At, t, idx = problem(2, 64, 700, 6, torch.bfloat16, seed=29)
    far = torch.zeros(2**31 + 100, dtype=torch.bfloat16, device="cuda").as_strided((2, 6), (2**31 + 5, 1), 3)
    far.copy_(t)
    want, got = run(x, At, far.cpu(), idx), None
    xd, Ad = x.cuda().requires_grad_(), At.cuda().requires_grad_()
    got = linear_distillation(xd, far, idx.cuda(), Ad)
    got.backward()
    assert got.item() == want[0] and torch.equal(xd.grad, want[1]) and torch.equal(Ad.grad, want[2])


def test_second_derivatives_are_refused():
    x, At, t, idx = problem(16, 64, 300, 4, torch.bfloat16)
    xd = x.cuda().requires_grad_()
    loss = linear_distillation(xd, t.cuda(), idx.cuda(), At.cuda())
    (g,) = torch.autograd.grad(loss, xd, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


# ---------------------------------------------------------------------------------------------------- the head itself
def grid_head(N, H, V, dtype, seed):
    """x and At on grids on which every sum of products is exact in fp32 in any order: multiples of 2^-3 below 4 and of
    2^-7 below 1/2 give multiples of 2^-10 below 2 H < 2^13."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(N, H, generator=g) * 8).round().clamp(-31, 31) / 8
    At = (torch.randn(H, V, generator=g) * 16).round().clamp(-63, 63) / 128
    return x.to(dtype), At.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,H,V", [(1, 64, 256), (3, 60, 1001), (130, 128, 5003), (300, 256, 2048)])
def test_logits_of_a_head(dtype, N, H, V):
    x, At = grid_head(N, H, V, dtype, N)
    got = linear_logits(x.cuda(), At.cuda(), 0.5)
    assert got.dtype == torch.float32 and got.shape == (N, V)
    assert torch.equal(got.double().cpu(), 0.5 * (x.double() @ At.double()))


@pytest.mark.parametrize("N,chunk", [(1, 4096), (50, 4096), (300, 128)])
def test_head_lists_and_draws_like_its_logits(N, chunk):
    x, At = grid_head(N, 64, 3001, torch.bfloat16, 7)
    x, At = x.cuda(), At.cuda()
    head = LinearCrossEntropyLoss(64, 3001, device="cuda", dtype=torch.bfloat16, logit_scale=0.5, N_chunk_size=chunk)
    with torch.no_grad():
        head.weight.copy_(At)
    logits = head.logits(x)
    assert torch.equal(logits, (0.5 * (x.double() @ At.double())).float())
    got, want = head.top_logits(x, 20, temperature=1.5), top_logits(logits, 20, temperature=1.5)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not got.values.requires_grad
    u = torch.rand(N, generator=torch.Generator().manual_seed(1)).cuda()
    T = (0.5 + torch.rand(N, generator=torch.Generator().manual_seed(2))).cuda()
    for kw in (dict(temperature=T, top_k=30, top_p=0.9), dict(top_p=0.8), dict(temperature=T[:1])):
        got, want = head.sample(x, u, **kw), sample_logits(logits, u, **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = head.sample(x.view(1, N, 64), u.view(1, N), top_k=5)
    assert got.tokens.shape == (1, N) and got.logprobs.shape == (1, N)
    assert head.top_logits(x[:0], 3).values.shape == (0, 3) and head.sample(x[:0], u[:0]).tokens.shape == (0,)


def test_a_distillation_step_with_two_heads():
    """The student draws, the teacher lists, the student learns: one step through the modules, against the definition."""
    torch.manual_seed(1)
    H, V, B = 64, 2000, 96
    teacher = LinearCrossEntropyLoss(H, V, device="cuda", dtype=torch.bfloat16)
    student = LinearDistillationLoss(H, V, device="cuda", dtype=torch.bfloat16, temperature=1.5, N_chunk_size=128)
    x = torch.randn(B, H, device="cuda", dtype=torch.bfloat16).requires_grad_()
    tokens, logprobs = student.sample(x, torch.rand(B, device="cuda"), top_p=0.95)
    assert ((tokens >= 0) & (tokens < V)).all() and (logprobs <= 0).all()
    lists = teacher.top_logits(x, 16, temperature=1.5)
    loss = student(x, lists.values, lists.indices, lists.lse)
    loss.backward()
    ref = reference(x.detach().cpu(), student.weight.detach().cpu(), lists.values.cpu(), lists.indices.cpu(), 1.5, 1.0, lists.lse.cpu())
    assert abs(loss.item() - ref["loss"]) <= loss_bound(ref, 1.5, B)
    bx, bw = gradient_bounds(ref, torch.bfloat16)
    assert ((x.grad.double().cpu() - ref["dx"]).abs() <= bx).all()
    assert ((student.weight.grad.double().cpu() - ref["dW"]).abs() <= bw).all()
