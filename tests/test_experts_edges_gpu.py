"""Routed experts where they are easiest to get wrong: sums that cancel, dropped pairs, derivatives of derivatives,
captured first calls, extreme scores, and the kernel forms that only larger or rarer shapes take.

Tolerances as in test_experts_gpu.py: u = 2^-24 / 2^-11 / 2^-8 for one rounding to float32 / float16 / bfloat16, and
2 n 2^-24 of the sum of the magnitudes for a float32 sum of n products.
"""
import os
import subprocess
import sys
import textwrap
import threading

import pytest
import torch

from conftest import ROOT
from test_experts_gpu import HALF, INF, TINY, TYPES, U, near, plan, ref_groups, ref_matmul, ref_route, ref_route_grad, rng

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status(cuda_device):
    """No kernel gave up on a barrier in any of these tests."""
    yield
    from mlx_kmeans_b200 import expert_status
    expert_status()


# ---------------------------------------------------------------- calls from other threads

def _in_new_threads(n, f):
    """f(i) in n new threads at once; their results, or the first exception."""
    start, out = threading.Barrier(n), [None] * n

    def work(i):
        try:
            start.wait()
            out[i] = f(i)
        except BaseException as e:                            # noqa: BLE001  (handed to the test)
            out[i] = e

    threads = [threading.Thread(target=work, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for r in out:
        if isinstance(r, BaseException):
            raise r
    return out


@pytest.mark.parametrize("call", ["forward", "dx", "dw"])
def test_first_cuda_work_of_a_thread(call):
    """A thread that has done nothing on the GPU yet has no context of the driver's: the products work all the same."""
    from mlx_kmeans_b200 import expert_matmul, expert_matmul_grad
    T, k, E, N, D = 700, 2, 4, 128, 64
    g = rng(0)
    groups = plan(T, k, E, 0)
    x, w = torch.randn(T, D, generator=g).half().cuda(), torch.randn(E, N, D, generator=g).half().cuda()
    dy = torch.randn(T * k, N, generator=g).half().cuda()
    xg = x[groups.rows.long().clamp(min=0)].contiguous()
    run = {"forward": lambda: expert_matmul(xg, w, groups, gather=False),
           "dx": lambda: expert_matmul_grad(dy, xg, w, groups, gather=False)[0],
           "dw": lambda: expert_matmul_grad(dy, xg, w, groups, gather=False)[1]}[call]
    want = run()
    torch.cuda.synchronize()
    got, = _in_new_threads(1, lambda i: run())
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_first_backward_of_the_autograd_thread():
    """The gradients as the first CUDA work of a process's backward thread."""
    code = """
        import torch
        from mlx_kmeans_b200 import expert_matmul, expert_matmul_grad, group_rows
        torch.manual_seed(0)
        x, w = torch.randn(40, 64, device="cuda").half(), torch.randn(4, 48, 64, device="cuda").half()
        groups = group_rows((torch.arange(40, device="cuda") % 4).int(), 4)
        dy = torch.randn(40, 48, device="cuda").half()
        want = expert_matmul_grad(dy, x, w, groups, gather=False)
        x.requires_grad_(True), w.requires_grad_(True)
        expert_matmul(x, w, groups, gather=False).backward(dy)
        assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])
        print("backward")
    """
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "backward" in r.stdout, r.stderr
