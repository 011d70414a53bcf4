"""Calls from several host threads at once: what goes wrong in one of them ends the test."""
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest
import torch

from distill_util import loss_bound, reference
from linear_cross_entropy_loss_b200 import linear_distillation, sample_logits, top_logits
from test_gpu_distill import problem
from test_gpu_head import normal, uniform

pytestmark = pytest.mark.gpu
THREADS, ROUNDS = 4, 20


def in_threads(work):
    with ThreadPoolExecutor(THREADS) as pool:
        rounds = [f.result(timeout=120) for f in [pool.submit(work, i) for i in range(THREADS)]]
    assert rounds == [ROUNDS] * THREADS


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_lists_and_draws_of_four_threads(dtype):
    jobs = [(normal(64, 20000 + 64 * i, dtype, seed=i).cuda(), uniform(64, i)) for i in range(THREADS)]

    def answers(i):
        x, u = jobs[i]
        return *top_logits(x, 20), *sample_logits(x, u, top_p=0.9), *sample_logits(x, u, top_k=30)

    want = [answers(i) for i in range(THREADS)]
    torch.cuda.synchronize()

    def work(i):
        done = 0
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(ROUNDS):
                got = answers(i)
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want[i])), i
                done += 1
        return done

    in_threads(work)


def test_distillation_steps_of_four_threads():
    jobs = [problem(200, 64, 2000 + 8 * i, 8, torch.bfloat16, seed=i) for i in range(THREADS)]
    refs = [reference(*job) for job in jobs]
    torch.cuda.synchronize()

    def work(i):
        done = 0
        x, At, t, idx = (v.cuda() for v in jobs[i])
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            x.requires_grad_()
            first = None
            for _ in range(ROUNDS):
                loss = linear_distillation(x, t, idx, At, N_chunk_size=128)
                (dx,) = torch.autograd.grad(loss, x)
                torch.cuda.current_stream().synchronize()
                assert abs(loss.item() - refs[i]["loss"]) <= loss_bound(refs[i], 1.0, 200)
                first = dx if first is None else first
                assert torch.equal(dx, first), i
                done += 1
        return done

    in_threads(work)


FIRST_CALLS = """
import threading
from concurrent.futures import ThreadPoolExecutor

import torch
from linear_cross_entropy_loss_b200 import linear_logits, sample_logits, top_logits

n = 6
x = [torch.randn(20, 30000, device="cuda").to(t) for t in (torch.float32, torch.bfloat16, torch.float16) for _ in range(2)]
u = torch.rand(20, device="cuda")
torch.cuda.synchronize()
start = threading.Barrier(n)

def work(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait(60)
        got = (*top_logits(x[i], 5), *sample_logits(x[i], u, top_p=0.9), *sample_logits(x[i], u, top_k=9),
               linear_logits(x[i][:, :64], x[i].t()[:64]))
        torch.cuda.current_stream().synchronize()
    return got

with ThreadPoolExecutor(n) as pool:
    first = [f.result(timeout=120) for f in [pool.submit(work, i) for i in range(n)]]
for i in range(n):
    start = threading.Barrier(1)
    again = work(i)
    assert all(torch.equal(a, b) for a, b in zip(first[i], again)), i
print("done", len(first))
"""


def test_first_calls_of_a_process_in_six_threads():
    """Nothing has been called before: loading the library and the setup of each kernel is raced too."""
    root = Path(__file__).resolve().parent.parent
    out = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.split() == ["done", "6"], out.stdout + out.stderr
