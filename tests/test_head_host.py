"""The operators of a head without a GPU, on a stand-in for the library: batches without rows, and traced calls."""
import pytest
import torch

from linear_cross_entropy_loss_b200 import (linear_distillation, linear_sample, linear_top_logits, ops, sample_logits,
                                            top_logits)


class Stub:
    """Answers of the right shape for every call (and, of the logits and lists, the right ones)."""

    requires_cuda = False

    def linear_logits(self, x, At, scale, out, status):
        out[:, :At.shape[1]] = scale * (x.float() @ At.float())

    def top_logits(self, logits, k, temperature, values, indices, lse):
        v, i = torch.topk(logits, k, dim=1)
        values.copy_(v), indices.copy_(i), lse.copy_(torch.logsumexp(logits.float() / temperature, 1))

    def sample_logits(self, logits, sampling, tokens, logprobs):
        self.sampling = sampling
        tokens.copy_(logits.argmax(1)), logprobs.zero_()

    def distill_workspace_bytes(self, prob, k):
        return 8

    def distill_pass(self, prob, teacher, x, At, workspace, dx, dW, dW_res, loss):
        loss.fill_(1.0)
        for d in (dx, dW):
            if d is not None:
                d.fill_(0.5)

    def align_rows(self, src, dst):
        dst.copy_(src)

    def grad_scale_pair(self, a, b, factor):
        for m in (a, b):
            m.copy_(m.float() * factor)

    def grad_scale_cast(self, src, dst, factor):
        dst.copy_(src.float() * factor)


@pytest.fixture
def stub():
    backend = Stub()
    ops.set_backend(backend)
    yield backend
    ops.set_backend(None)


def traced(call):
    return torch.compile(call, fullgraph=True, backend="aot_eager")


# ---------------------------------------------------------------------------------------------------- no rows
SETTINGS = [dict(temperature=0.7), dict(top_k=4), dict(top_p=0.9), dict(min_p=0.1)]


@pytest.mark.parametrize("kw", SETTINGS, ids=lambda kw: next(iter(kw)))
@pytest.mark.parametrize("entries", [0, 1])
@pytest.mark.parametrize("lead", [(0,), (0, 3), (2, 0)])
def test_an_empty_batch_with_settings_per_row(stub, kw, entries, lead):
    ((name, value),) = kw.items()
    per_row = torch.full((entries,), value)
    got = sample_logits(torch.zeros(*lead, 8), torch.zeros(lead), **{name: per_row})
    assert got.tokens.shape == lead and got.tokens.dtype == torch.int64 and got.logprobs.shape == lead
    head = linear_sample(torch.zeros(*lead, 16), torch.zeros(16, 8), torch.zeros(lead), **{name: per_row})
    assert head.tokens.shape == lead and head.logprobs.shape == lead


@pytest.mark.parametrize("kw", [dict(temperature=-1.0), dict(top_k=-1), dict(top_p=0.0), dict(min_p=2.0)])
def test_an_empty_batch_is_refused_what_a_full_one_is(stub, kw):
    for n in (0, 3):
        with pytest.raises(AssertionError):
            sample_logits(torch.zeros(n, 8), torch.zeros(n), **kw)


def test_the_library_takes_an_empty_batch_as_the_python_layer_hands_it_over(stub):
    """Pointers of empty tensors are null: the numbers that then count have to be ones that the C entry accepts."""
    import ctypes

    from linear_cross_entropy_loss_b200 import _native

    none = torch.zeros(0)
    sample_logits(torch.zeros(0, 8), none, temperature=none, top_k=none.int(), top_p=none, min_p=none)
    assert _native.load().lce_sample_logits(_native.DTYPE_F32, None, 8, 0, 8, ctypes.byref(stub.sampling), None, None, None) == 0


# ---------------------------------------------------------------------------------------------------- traced calls
@pytest.mark.parametrize("lead", [(), (6,), (2, 3), (2, 1, 3)])
@pytest.mark.parametrize("given", [False, True])
def test_traced_distillation_takes_the_shapes_of_an_eager_one(stub, lead, given):
    x, At = torch.randn(*lead, 8, requires_grad=True), torch.randn(8, 16, requires_grad=True)
    t, idx = torch.randn(*lead, 4), torch.randint(0, 16, (*lead, 4))
    lse = torch.logsumexp(t, -1) if given else None
    want = linear_distillation(x, t, idx, At, lse)
    loss = traced(lambda x, At: linear_distillation(x, t, idx, At, lse))(x, At)
    assert loss.shape == want.shape == () and loss.item() == want.item()
    loss.backward()
    assert x.grad.shape == x.shape and At.grad.shape == At.shape


def test_traced_lists_and_draws_of_logits_that_require_a_gradient(stub):
    """They are not differentiable, and do not stand in the way of what is."""
    x, u = torch.randn(6, 9, requires_grad=True), torch.rand(6)

    def call(x):
        top, drawn = top_logits(2 * x, 3), sample_logits(2 * x, u, top_p=0.9)
        return (x * x).sum() + top.values.sum() + top.lse.sum() + drawn.logprobs.sum(), top, drawn

    for run in (call, traced(call)):
        x.grad = None
        loss, top, drawn = run(x)
        assert not any(v.requires_grad for v in (*top, *drawn))
        loss.backward()
        assert torch.equal(x.grad, 2 * x.detach())


def test_traced_head_without_rows(stub):
    At = torch.randn(8, 16)
    call = lambda x, u: (*linear_top_logits(x, At, 3), *linear_sample(x, At, u))  # noqa: E731
    for lead in ((0,), (0, 2), (2, 0)):
        want = call(torch.zeros(*lead, 8), torch.zeros(lead))
        got = traced(call)(torch.zeros(*lead, 8), torch.zeros(lead))
        assert [v.shape for v in got] == [v.shape for v in want]


@pytest.mark.parametrize("factor", [65536.0, 0.3, 1.0, 2.0 ** -10])
def test_traced_gradients_are_scaled_like_eager_ones(stub, factor):
    """The factor of backward is a float: a loss scale that fp16 does not hold, and one that it rounds."""
    x, At = torch.randn(6, 8).half().requires_grad_(), torch.randn(8, 16).half().requires_grad_()
    t, idx = torch.randn(6, 4), torch.randint(0, 16, (6, 4))

    def grads(call):
        x.grad = At.grad = None
        (call(x, At) * factor).backward()
        return x.grad, At.grad

    call = lambda x, At: linear_distillation(x, t, idx, At)  # noqa: E731
    for got, want in zip(grads(traced(call)), grads(call)):
        assert got.dtype == torch.float16 and torch.equal(got, want)
