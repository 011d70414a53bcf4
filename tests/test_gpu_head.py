"""top_logits and sample_logits against their definitions in 64 bits. Indices and tokens have to be equal."""
import numpy as np
import pytest
import torch

from head_util import sample_reference, top_reference
from linear_cross_entropy_loss_b200 import sample_logits, top_logits

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
INF, NAN = float("inf"), float("nan")


def normal(n, V, dtype, seed=0, std=3.0):
    g = torch.Generator().manual_seed(seed)
    return (std * torch.randn(n, V, generator=g)).to(dtype)


# Row sums run over V terms of relative error (|d| + 3) 2^-23 each (the exponential and its argument; the terms weigh
# exp(d), so |d| counts 1/e at most), added in fewer than 64 + log2 steps of 2^-24; the logarithm turns the relative error of
# the sum into an absolute one, and max / T + log(sum) and 1 / T are rounded once each.
def lse_tolerance(lse, largest, T):
    return 2.0 ** -17 + 2.0 ** -22 * (abs(lse) + abs(largest / T))


def check_top(logits, k, T=1.0):
    got = top_logits(logits, k, temperature=T)
    flat = logits.reshape(-1, logits.shape[-1])
    host = flat.double().cpu().numpy()
    indices, lse = top_reference(host, k, T)
    assert got.values.shape == (*logits.shape[:-1], k) and got.values.dtype == logits.dtype
    assert got.indices.shape == (*logits.shape[:-1], k) and got.indices.dtype == torch.int64
    assert got.lse.shape == logits.shape[:-1] and got.lse.dtype == torch.float32
    assert np.array_equal(got.indices.reshape(-1, k).cpu().numpy(), indices)
    values = got.values.reshape(-1, k).double().cpu().numpy()
    want = np.take_along_axis(host, indices, 1)
    assert np.array_equal(values, want, equal_nan=True)
    for r, (a, b) in enumerate(zip(got.lse.reshape(-1).double().cpu().numpy(), lse)):
        if np.isfinite(b):
            assert abs(a - b) <= lse_tolerance(b, host[r].max(), T), (r, a, b)
        else:
            assert a == b or (np.isnan(a) and np.isnan(b)), (r, a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(1, 1), (2, 1), (2, 2), (7, 3), (31, 31), (33, 8), (256, 64), (1000, 1000), (1025, 1024),
                                 (4099, 100), (8192, 1), (20000, 513), (50257, 64), (131072, 50), (262147, 128)])
def test_top_logits(dtype, V, k):
    check_top(normal(5, V, dtype, seed=V + k).cuda(), k)


@pytest.mark.parametrize("n", [1, 2, 3, 64, 149, 700])
def test_top_logits_row_counts(n):
    check_top(normal(n, 3001, torch.bfloat16, seed=n).cuda(), 20, T=0.7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 5000, 70001])
def test_top_logits_orders(dtype, V):
    up = torch.linspace(-8, 8, V).to(dtype)
    few = torch.randint(0, 3, (V,), generator=torch.Generator().manual_seed(V)).to(dtype)
    zeros = torch.zeros(V, dtype=dtype)
    zeros[1::2] = -0.0
    last = torch.zeros(V, dtype=dtype)
    last[-1] = 1.0
    lowest = torch.full((V,), torch.finfo(dtype).min, dtype=dtype)
    lowest[V // 2] = 0.5
    rows = torch.stack([up, up.flip(0), few, zeros, last, lowest, torch.full((V,), 2.0, dtype=dtype)])
    check_top(rows.cuda(), 33)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 9001])
def test_top_logits_infinities_and_nan(dtype, V):
    rows = normal(7, V, dtype, seed=3)
    rows[0] = -INF
    rows[1, :] = -INF
    rows[1, [3, V - 1]] = torch.tensor([1.0, 2.0], dtype=dtype)
    rows[2, [0, V - 2]] = INF
    rows[3, [5, 6, V - 1]] = NAN
    rows[4, 7] = NAN
    rows[4, 8] = INF
    rows[4, 9] = -INF
    rows[5] = NAN
    rows[6] = INF
    check_top(rows.cuda(), 20)


def test_top_logits_layouts():
    base = normal(24, 1200, torch.bfloat16).cuda()
    check_top(base[:, 1:-2], 17)                       # rows off the 16-byte grid
    check_top(base[::3, 5:1000], 17)
    check_top(base.view(2, 3, 4, 1200), 9)
    check_top(base.t().contiguous().t(), 9)             # inner stride 24
    check_top(base[:1].expand(6, 1200), 9)              # one row, six times
    check_top(base[3], 9)
    empty = top_logits(base[:0], 4)
    assert empty.values.shape == (0, 4) and empty.indices.shape == (0, 4) and empty.lse.shape == (0,)
    f32 = normal(9, 1501, torch.float32).cuda()
    check_top(f32[:, 3:], 100)
    check_top(f32[:, :1], 1)


# ---------------------------------------------------------------------------------------------------- sampling
# The logarithm is taken in 64 bits of weights that are rounded to 2^-45 of the largest one, then rounded to float32.
def check_sample(logits, u, T=1.0, top_k=0, top_p=1.0, min_p=0.0):
    got = sample_logits(logits, u, temperature=T, top_k=top_k, top_p=top_p, min_p=min_p)
    assert got.tokens.shape == logits.shape[:-1] and got.tokens.dtype == torch.int64
    assert got.logprobs.shape == logits.shape[:-1] and got.logprobs.dtype == torch.float32
    host = logits.reshape(-1, logits.shape[-1]).double().cpu().numpy()
    uu = u.reshape(-1).double().cpu().numpy()

    def of(v, r):
        return float(v.reshape(-1)[r if v.numel() > 1 else 0]) if isinstance(v, torch.Tensor) else v

    want = [sample_reference(host[r], uu[r], of(T, r), int(of(top_k, r)), of(top_p, r), of(min_p, r)) for r in range(len(host))]
    assert got.tokens.reshape(-1).tolist() == [w[0] for w in want]
    lp = got.logprobs.reshape(-1).double().cpu().numpy()
    for a, (_, b) in zip(lp, want):
        assert a == b or abs(a - b) <= 2.0 ** -24 * abs(b) + 1e-8, (a, b)
    return got


def uniform(n, seed=0, dtype=torch.float32):
    return torch.rand(n, generator=torch.Generator().manual_seed(1000 + seed), dtype=dtype).cuda()


SETTINGS = [dict(), dict(T=0.6), dict(T=2.5), dict(top_k=1), dict(top_k=5), dict(top_k=50, T=0.8), dict(top_p=0.9),
            dict(top_p=0.3, T=1.5), dict(min_p=0.05), dict(min_p=1.0), dict(top_k=40, top_p=0.8), dict(top_k=300, top_p=0.95, min_p=0.01),
            dict(top_k=3000, top_p=0.7), dict(top_p=0.999, min_p=0.002), dict(T=0.0), dict(top_k=10**6), dict(top_p=1e-6),
            dict(T=1e-6), dict(T=1e4, top_p=0.5)]


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype,V", [(torch.float32, 5000), (torch.bfloat16, 32768), (torch.float16, 50257)])
def test_sample_logits(dtype, V, settings):
    check_sample(normal(7, V, dtype, seed=V).cuda(), uniform(7, V), **settings)


@pytest.mark.parametrize("V", [1, 2, 3, 31, 32, 33, 257, 1023, 8193, 131072, 300001])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=20, top_p=0.9), dict(top_p=0.9)], ids=str)
def test_sample_logits_vocabularies(V, settings):
    check_sample(normal(3, V, torch.bfloat16, seed=V).cuda(), uniform(3, V), **settings)
    check_sample(normal(2, V, torch.float32, seed=V).cuda(), uniform(2, V + 1), **settings)


@pytest.mark.parametrize("n", [1, 2, 5, 63, 150, 600])
def test_sample_logits_row_counts(n):
    check_sample(normal(n, 2000, torch.bfloat16, seed=n).cuda(), uniform(n, n), top_k=50, top_p=0.9)
    check_sample(normal(n, 2000, torch.float16, seed=n).cuda(), uniform(n, n), top_p=0.9)


def test_sample_logits_settings_per_row():
    n, V = 96, 6000
    g = torch.Generator().manual_seed(5)
    logits = normal(n, V, torch.bfloat16, seed=9)
    logits[::4, ::2] = -INF
    T = torch.where(torch.rand(n, generator=g) < 0.2, torch.zeros(n), 0.3 + torch.rand(n, generator=g)).cuda()
    top_k = torch.randint(-1, 2500, (n,), generator=g).cuda()
    top_k[::5] = 0
    top_p = torch.rand(n, generator=g).cuda()
    top_p[::3] = 1.0
    min_p = (0.2 * torch.rand(n, generator=g)).cuda()
    min_p[1::3] = 0.0
    u = uniform(n)
    check_sample(logits.cuda(), u, T, top_k, top_p, min_p)
    check_sample(logits.cuda(), u, T, top_k.to(torch.int32), 0.9, min_p)
    check_sample(logits.cuda(), u, T[:1], top_k, top_p, 0.0)
    check_sample(logits.cuda().view(8, 12, V), u.view(8, 12), T, top_k, top_p, min_p)


def test_sample_logits_takes_settings_out_of_range_as_the_nearest():
    logits, u = normal(6, 300, torch.float32).cuda(), uniform(6)
    same = sample_logits(logits, u)
    off = sample_logits(logits, u, top_p=torch.tensor([1.5, NAN, 2.0, 1.0, INF, 1.1]).cuda(),
                        min_p=torch.tensor([-1.0, NAN, 0.0, -INF, -0.5, 0.0]).cuda(),
                        top_k=torch.tensor([-5, 0, -1, 300, 10**9, 301]).cuda())
    assert torch.equal(same.tokens, off.tokens)
    first = logits.argmax(1)
    assert torch.equal(sample_logits(logits, u, temperature=torch.tensor([0.0, -1.0, NAN, 0.0, -INF, 0.0]).cuda()).tokens, first)
    assert torch.equal(sample_logits(logits, u, top_p=torch.zeros(6).cuda() - 1).tokens, first)
    assert torch.equal(sample_logits(logits, u, min_p=torch.full((6,), 3.0).cuda()).tokens, first)
    lo = sample_logits(logits, torch.zeros(6).cuda()).tokens
    hi = sample_logits(logits, torch.full((6,), 1 - 2.0 ** -24).cuda()).tokens
    assert torch.equal(sample_logits(logits, torch.tensor([-1.0, NAN, -INF, 0.0, -0.0, -3.0]).cuda()).tokens, lo)
    assert torch.equal(sample_logits(logits, torch.tensor([1.0, 2.0, INF, 1.0, 7.0, 1.0]).cuda()).tokens, hi)


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_logits_ties(dtype):
    """Equal logits everywhere: counts and masses end inside a run of equal values."""
    V = 40000
    flat = torch.zeros(5, V, dtype=dtype)
    flat[1, 1::2] = -0.0
    flat[2] = torch.randint(0, 3, (V,), generator=torch.Generator().manual_seed(1)).to(dtype)
    flat[3] = torch.finfo(dtype).min
    flat[3, 100:30000] = 1.0
    flat[4] = -7.5
    flat = flat.cuda()
    for settings in [dict(), dict(top_k=100), dict(top_k=12345), dict(top_p=0.37), dict(top_k=2000, top_p=0.5),
                     dict(top_k=20000, top_p=0.5), dict(top_p=0.9, min_p=0.5, T=1e3)]:
        check_sample(flat, uniform(5), **settings)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("settings", [dict(), dict(top_k=7), dict(top_p=0.8), dict(min_p=0.3), dict(T=0.0), dict(top_k=2000, top_p=0.6)], ids=str)
def test_sample_logits_masks_infinities_and_nan(dtype, settings):
    V = 3000
    rows = normal(8, V, dtype, seed=4)
    rows[0] = -INF
    rows[1] = NAN
    rows[2] = -INF
    rows[2, V - 1] = -3.0
    rows[3, [4, 77, 2999]] = INF
    rows[4, ::3] = NAN
    rows[5, 10:] = torch.finfo(dtype).min
    rows[6, :2999] = -INF
    rows[6, 5] = NAN
    rows[7] = torch.finfo(dtype).min
    check_sample(rows.cuda(), uniform(8), **settings)


def test_sample_logits_borders():
    """u on the borders between tokens of equal weight: the token above the border is drawn."""
    logits = torch.zeros(9, 8).cuda()
    u = torch.tensor([0, 1 / 8, 2 / 8, 3 / 8, 4 / 8, 5 / 8, 6 / 8, 7 / 8, 1 - 2.0 ** -53], dtype=torch.float64).cuda()
    assert sample_logits(logits, u).tokens.tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 7]
    # one token outweighs the rest by more than the weights resolve
    logits = torch.full((1, 64), -60.0).cuda()
    logits[0, 20] = 0.0
    for v in (0.0, 0.5, 1 - 2.0 ** -24):
        assert sample_logits(logits, torch.tensor([v]).cuda()).tokens.item() == 20


def test_sample_logits_layouts():
    base = normal(24, 1200, torch.bfloat16).cuda()
    for settings in (dict(top_k=30, top_p=0.9), dict(top_p=0.9)):
        check_sample(base[:, 1:-2], uniform(24), **settings)
        check_sample(base[::3, 5:1000], uniform(8), **settings)
        check_sample(base.t().contiguous().t(), uniform(24), **settings)
        check_sample(base[:1].expand(6, 1200), uniform(12)[::2], **settings)
        check_sample(base[2], uniform(1).view(()), **settings)
        check_sample(base.view(4, 6, 1200), uniform(24, dtype=torch.float64).view(4, 6), **settings)
    none = sample_logits(base[:0], uniform(24)[:0])
    assert none.tokens.shape == (0,) and none.logprobs.shape == (0,)


def test_sample_logits_draws_the_distribution():
    """Tokens of a grid of random numbers: their shares are the probabilities, to one grid step each."""
    n = 4096
    row = normal(1, 200, torch.float32, std=1.0)
    p = torch.softmax(row[0].double(), 0)
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).cuda()
    tokens = sample_logits(row.expand(n, 200).cuda(), u).tokens.cpu()
    counts = torch.bincount(tokens, minlength=200).double()
    assert (counts - n * p).abs().max() <= 1.0


@pytest.mark.parametrize("what", ["top", "sample", "nucleus"])
def test_other_streams_and_captured_graphs(what):
    logits, u = normal(40, 5001, torch.bfloat16).cuda(), uniform(40)
    call = {"top": lambda: top_logits(logits, 30), "sample": lambda: sample_logits(logits, u, top_k=30, top_p=0.9),
            "nucleus": lambda: sample_logits(logits, u, top_p=0.9)}[what]
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    old = logits.clone()
    logits.copy_(normal(40, 5001, torch.bfloat16, seed=8).cuda())
    graph.replay()
    torch.cuda.synchronize()
    new = call()
    assert all(torch.equal(a, b) for a, b in zip(got, new))
    logits.copy_(old)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_side_by_side_on_two_streams():
    a, b = normal(64, 20000, torch.float32, seed=1).cuda(), normal(64, 20000, torch.float32, seed=2).cuda()
    u = uniform(64)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append((*top_logits(x, 100), *sample_logits(x, u, top_p=0.9), *sample_logits(x, u, top_k=50)))
    torch.cuda.synchronize()
    for runs in got:
        for run in runs[1:]:
            assert all(torch.equal(p, q) for p, q in zip(run, runs[0]))


@pytest.mark.parametrize("dtype,V", [(torch.float32, 500003), (torch.bfloat16, 1000003), (torch.float16, 3000001)])
def test_rows_longer_than_shared_memory(dtype, V):
    logits = normal(2, V, dtype, seed=V).cuda()
    logits[1, ::2] = -INF
    check_top(logits, 50)
    check_top(logits, 1024, T=3.0)
    for settings in (dict(), dict(top_p=0.9), dict(min_p=0.01), dict(top_k=5000, top_p=0.9), dict(top_k=40)):
        check_sample(logits, uniform(2, V), **settings)
    equal = torch.full((1, V), 0.5, dtype=dtype).cuda()
    check_sample(equal, uniform(1, V), top_p=0.3)
    check_sample(equal, uniform(1, V), top_k=1500)
    check_top(equal, 300)


@pytest.mark.parametrize("T", [1e38, 3e37, 1e30, float("inf")])
def test_sample_logits_spans_that_a_float_does_not_hold(T):
    rows = normal(4, 2000, torch.float32, seed=6)
    rows[:, ::3] = torch.finfo(torch.float32).max
    rows[:, 1::3] = torch.finfo(torch.float32).min
    for settings in (dict(), dict(top_p=0.5), dict(top_p=0.95), dict(top_k=1500), dict(min_p=0.2)):
        check_sample(rows.cuda(), uniform(4), T=T, **settings)


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_logits_many_values_in_one_bin(dtype):
    """A temperature so high that a whole row of different logits falls into the first bins."""
    logits = normal(3, 40000, dtype, seed=2).cuda()
    for settings in (dict(top_p=0.5), dict(top_k=20000), dict(top_k=30000, top_p=0.7)):
        check_sample(logits, uniform(3), T=300.0, **settings)


def test_rows_in_rising_order_split_over_blocks():
    """All of the largest logits lie in the last part of a row: its list runs full."""
    up = torch.linspace(-20, 20, 131072).repeat(2, 1)
    up[1] = up[1].flip(0)
    for k in (1, 64, 512, 1024):
        check_top(up.cuda(), k)
        check_top(up.to(torch.bfloat16).cuda(), k)
    check_sample(up.cuda(), uniform(2), top_k=100, top_p=0.9)


@pytest.mark.parametrize("what", ["top", "sample"])
def test_traced_by_torch_compile_without_a_graph_break(what):
    logits, u = normal(6, 500, torch.bfloat16).cuda(), uniform(6)
    T = torch.full((6,), 0.8).cuda()
    if what == "top":
        call = lambda x, v: tuple(top_logits(x + 0, 9, temperature=1.5))  # noqa: E731
    else:
        call = lambda x, v: tuple(sample_logits(x + 0, v, temperature=T, top_k=20, top_p=0.9))  # noqa: E731
    got = torch.compile(call, fullgraph=True, backend="aot_eager")(logits, u)
    assert all(torch.equal(a, b) for a, b in zip(got, call(logits, u)))


def test_rows_further_apart_than_31_bits():
    flat = torch.full((2**31 + 9000,), -INF, dtype=torch.float16, device="cuda")
    rows = flat.as_strided((2, 5003), (2**31 + 5, 1), 3)
    rows.copy_(normal(2, 5003, torch.float16, seed=8))
    check_top(rows, 33)
    for settings in (dict(), dict(top_k=30), dict(top_p=0.8)):
        check_sample(rows, uniform(2), **settings)


@pytest.mark.parametrize("T", [2.0**-126, 2.0**-123, 1e-30, 1e-12, 1e-9, 3e-8, 1e-6, 1e-3, 1e30])
def test_log_sum_exp_at_any_temperature(T):
    """Up to quotients that a float does not hold."""
    rows = normal(3, 3000, torch.float32, seed=3).abs() + 1
    rows[1] = -rows[1]
    rows[2, 5] = 0.0
    got = top_logits(rows.cuda(), 4, temperature=T).lse.cpu()
    T = float(torch.tensor(T, dtype=torch.float32))
    want = torch.logsumexp(rows.double() / T, 1)
    # the rounding of 1 / T and of the result, of the sum's 3000 terms (at most 64 of them one after the other)
    bound = want.abs() * 2.0**-23 + 68 * 2.0**-24
    big = want.abs() > torch.finfo(torch.float32).max
    assert torch.equal(got[big], want[big].float())
    assert ((got.double() - want).abs()[~big] <= bound[~big]).all(), (got, want)


def test_few_with_weight_before_a_second_cut_in_a_cluster():
    """top_k keeps all that have weight, and top_p follows at once: the blocks of a row share the same arrays for both."""
    logits = torch.full((40, 131072), -1e4)
    logits[:, ::1000] = normal(40, 132, torch.float32, seed=4)
    for _ in range(20):
        check_sample(logits.cuda(), uniform(40), top_k=2000, top_p=0.6)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int64, torch.bool])
def test_top_k_per_row_in_any_whole_type(dtype):
    logits, u = normal(5, 700, torch.float32, seed=5).cuda(), uniform(5)
    ks = torch.tensor([0, 1, 1, 0, 1]).to(dtype).cuda()
    want = sample_logits(logits, u, top_k=ks.to(torch.int32))
    got = sample_logits(logits, u, top_k=ks)
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.logprobs, want.logprobs)


def test_two_threads():
    import threading

    jobs = [(normal(64, 20000 + 64 * i, torch.bfloat16, seed=i).cuda(), uniform(64, i)) for i in range(4)]
    want = [(top_logits(x, 20), sample_logits(x, u, top_p=0.9)) for x, u in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                x, u = jobs[i]
                got = (top_logits(x, 20), sample_logits(x, u, top_p=0.9))
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for g, w in zip(got, want[i]) for a, b in zip(g, w)):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []


@pytest.mark.parametrize("k_list", [1, 40, 200])
def test_what_follows_both_kernels_waits_for_both(k_list):
    """Settings per row: two kernels side by side. All rows, or none, or half of them have a short list; what reads the
    answers next in the stream has to find all of them."""
    n, V = 30, 70001
    logits = normal(n, V, torch.bfloat16, seed=k_list).cuda()
    for share in (0, 1, 2):
        ks = torch.full((n,), k_list)
        if share != 0:
            ks[::share] = 5000
        ks = ks.cuda()
        want = [sample_logits(logits, uniform(n, i), top_k=ks, top_p=0.9) for i in range(8)]
        torch.cuda.synchronize()
        tokens, logprobs = torch.zeros(8, n, dtype=torch.int64, device="cuda"), torch.zeros(8, n, device="cuda")
        us = [uniform(n, i) for i in range(8)]
        static, graph = us[0].clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = sample_logits(logits, static, top_k=ks, top_p=0.9)
            copy = got.tokens.clone(), got.logprobs.clone()
        for i in range(8):
            got = sample_logits(logits, us[i], top_k=ks, top_p=0.9)
            tokens[i], logprobs[i] = got.tokens, got.logprobs
            del got
            torch.full((n,), -7, device="cuda")  # may take the place of the answers
        for i in range(8):
            assert torch.equal(tokens[i], want[i].tokens) and torch.equal(logprobs[i], want[i].logprobs)
            static.copy_(us[i])
            graph.replay()
            assert torch.equal(copy[0], want[i].tokens) and torch.equal(copy[1], want[i].logprobs)
