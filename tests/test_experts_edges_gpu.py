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


# ---------------------------------------------------------------- the gradient of gathered rows

def by_row(groups, v):
    """float64 values by position summed over each row's pairs."""
    slot = groups.slot.cpu().long()
    slot = slot if slot.ndim == 2 else slot[:, None]
    return torch.where((slot >= 0)[:, :, None], v[slot.clamp(min=0)], 0.0).sum(1)


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("shape", [(1, 4, 8, 40, 64), (5, 2, 4, 129, 264), (48, 4, 12, 200, 336), (64, 2, 5, 33, 35),
                                   (333, 3, 5, 77, 51), (700, 3, 7, 384, 192), (1100, 2, 3, 136, 1002), (300, 8, 16, 64, 4),
                                   (900, 2, 2, 130, 577)])
def test_dx_of_a_row_is_rounded_once(shape, dt):
    """A row's positions are summed in float32, and only the sum is rounded: no term's own rounding enters."""
    from mlx_kmeans_b200 import expert_matmul_grad
    T, k, E, N, D = shape
    g = rng(T + D)
    groups = plan(T, k, E, T)
    x = torch.randn(T, D, generator=g).to(dt).cuda()
    w = (torch.randn(E, N, D, generator=g) / N ** 0.5).to(dt).cuda()
    dy = torch.randn(T * k, N, generator=g).to(dt).cuda()
    dx, _ = expert_matmul_grad(dy, x, w, groups)
    _, (rx, xm), _ = ref_matmul(x, w, groups, True, dy)
    assert dx.dtype == dt
    near(dx, by_row(groups, rx), by_row(groups, xm), N + k)


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("T,D", [(1, 16), (5, 33), (700, 264), (200, 2)])
def test_dx_terms_past_the_types_range_cancel(T, D, dt):
    """Two positions of a row with gradients of +70000 and -70000, which float16 does not hold: their sum is 0."""
    from mlx_kmeans_b200 import expert_matmul, expert_matmul_grad, group_rows
    groups = group_rows(torch.tensor([[0, 1]], dtype=torch.int32).repeat(T, 1).cuda(), 2)
    w = torch.full((2, 8, D), 100.0)
    w[1] = -100.0
    w, x = w.to(dt).cuda(), torch.zeros(T, D, dtype=dt, device="cuda", requires_grad=True)
    dy = torch.full((2 * T, 8), 87.5, dtype=dt, device="cuda")            # 8 * 87.5 * 100 = 70000
    assert torch.equal(expert_matmul_grad(dy, x.detach(), w, groups)[0], torch.zeros_like(x))
    expert_matmul(x, w, groups).backward(dy)
    assert torch.equal(x.grad, torch.zeros_like(x))


def test_dx_of_labels_and_of_single_choices():
    """One choice a row: the position's gradient itself, 0 where the row has none."""
    from mlx_kmeans_b200 import expert_matmul_grad, group_rows
    for lab in (torch.randint(-1, 5, (300,), generator=rng(1), dtype=torch.int32),
                torch.randint(-1, 5, (300, 1), generator=rng(2), dtype=torch.int32)):
        groups = group_rows(lab.cuda(), 5)
        g = rng(3)
        x, w = torch.randn(300, 72, generator=g).half().cuda(), torch.randn(5, 40, 72, generator=g).half().cuda()
        dy = torch.randn(300, 40, generator=g).half().cuda()
        dx, _ = expert_matmul_grad(dy, x, w, groups)
        _, (rx, xm), _ = ref_matmul(x, w, groups, True, dy)
        near(dx, by_row(groups, rx), by_row(groups, xm), 40)
        assert int(dx[lab.reshape(-1).cuda() < 0].abs().max()) == 0


# ---------------------------------------------------------------- pairs dropped after the grouping

@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("T,k,H", [(1, 1, 1), (1, 8, 64), (3, 2, 33), (130, 8, 515), (40, 3, 2048), (2500, 4, 24)])
def test_combine_grad_of_positions_without_a_pair(T, k, H, weighted, dt):
    """Slots set to -1 after the grouping (experts over their capacity): their positions' rows of dy are zeros, and
    dW, which sums positions by the offsets, gets nothing from them."""
    from mlx_kmeans_b200 import combine_rows_grad, expert_matmul_grad
    E = max(4, k)
    groups = plan(T, k, E, T + H, drop=0.1)
    g = rng(H)
    groups.slot[(torch.rand(T, k, generator=g) < 0.3).cuda()] = -1
    if T > 2:
        groups.slot[1] = -1
    y, dout = torch.randn(T * k, H, generator=g).to(dt).cuda(), torch.randn(T, H, generator=g).to(dt).cuda()
    w = torch.rand(T, k, generator=g).cuda() if weighted else None
    stale = torch.full_like(y, float("nan"))
    del stale                                                 # the allocator's next block of this size
    dy, dw = combine_rows_grad(dout, y, groups, w)
    slot = groups.slot.cpu().long()
    wv = (w.double().cpu() if weighted else torch.ones(T, k, dtype=torch.float64))[:, :, None]
    ref = torch.zeros(T * k, H, dtype=torch.float64)
    ref[slot[slot >= 0]] = (wv * dout.double().cpu()[:, None, :]).expand(T, k, H)[slot >= 0]
    near(dy, ref, ref.abs(), 1)
    assert torch.all(dy.cpu()[ref.abs().sum(1) == 0] == 0)
    if weighted:
        assert torch.all(dw[groups.slot < 0] == 0)
    if dt in HALF and H > 1:
        x, m = torch.randn(T, 16, generator=g).to(dt).cuda(), torch.zeros(E, H, 16, dtype=dt, device="cuda")
        _, _, (rw, wm) = ref_matmul(x, m, groups, True, dy)
        near(expert_matmul_grad(dy, x, m, groups)[1], rw, wm, T * k)


def test_combine_grad_where_rows_and_slots_disagree():
    """dy follows the slots alone: a position whose row entry was changed keeps its gradient."""
    from mlx_kmeans_b200 import RowGroups, combine_rows_grad, group_rows
    ids = torch.tensor([[0, 1], [1, 2], [0, 2]], dtype=torch.int32).cuda()
    groups = group_rows(ids, 3)
    y, dout = torch.ones(6, 8).cuda(), torch.arange(1.0, 4.0)[:, None].expand(3, 8).contiguous().cuda()
    want, _ = combine_rows_grad(dout, y, groups)
    odd = RowGroups(groups.offsets, torch.full_like(groups.rows, 99), groups.slot)
    assert torch.equal(combine_rows_grad(dout, y, odd)[0], want) and bool((want != 0).all())


# ---------------------------------------------------------------- derivatives of the derivatives

def _differentiable_calls():
    """name -> (function of its float inputs, those inputs)."""
    from mlx_kmeans_b200 import combine_rows, expert_matmul, group_rows, route
    g = rng(12)
    ids = torch.stack([torch.randperm(4, generator=g)[:2] for _ in range(6)]).to(torch.int32).cuda()
    groups = group_rows(ids, 4)
    l, y, c = torch.randn(6, 4, generator=g).cuda(), torch.randn(12, 8, generator=g).cuda(), torch.rand(6, 2, generator=g).cuda()
    x, w = torch.randn(6, 16, generator=g).half().cuda(), torch.randn(4, 8, 16, generator=g).half().cuda()
    return {"route": (lambda l: route(l, 2, renormalize=False)[1], [l]),
            "expert_matmul": (lambda x, w: expert_matmul(x, w, groups), [x, w]),
            "combine_rows": (lambda y, c: combine_rows(y, groups, c), [y, c])}


@pytest.mark.parametrize("name", ["route", "expert_matmul", "combine_rows"])
def test_second_derivatives_are_refused(name):
    """The gradients have no derivative of their own: a loss made from them raises, beside other terms too, whether or
    not the gradient that came in had one, and whichever input's derivative is asked for."""
    f, args = _differentiable_calls()[name]
    for loss in (lambda v: v.float().sum(), lambda v: v.float().square().sum()):
        for i in range(len(args)):
            ins = [a.clone().requires_grad_(True) for a in args]
            grads = torch.autograd.grad(loss(f(*ins)), ins, create_graph=True)
            penalty = grads[i].float().square().sum() + sum(a.float().square().sum() for a in ins)
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad(penalty, ins)
            ins = [a.clone().requires_grad_(True) for a in args]
            grads = torch.autograd.grad(loss(f(*ins)), ins, create_graph=True)
            with pytest.raises(RuntimeError, match="second derivative"):
                (grads[i].float().square().sum() + sum(a.float().square().sum() for a in ins)).backward()


@pytest.mark.parametrize("name", ["route", "expert_matmul", "combine_rows"])
def test_first_derivatives_with_a_graph_kept(name):
    """create_graph alone changes no gradient, and one that is not differentiated again raises nothing."""
    f, args = _differentiable_calls()[name]
    ins = [a.clone().requires_grad_(True) for a in args]
    plain = torch.autograd.grad(f(*ins).float().square().sum(), ins)
    kept = torch.autograd.grad(f(*ins).float().square().sum(), ins, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, kept))
    only = args[0].clone().requires_grad_(True)               # one input alone
    kept, = torch.autograd.grad(f(only, *args[1:]).float().square().sum(), [only], create_graph=True)
    assert torch.equal(kept, plain[0])


@pytest.mark.parametrize("requires", [False, True])
@pytest.mark.parametrize("name", ["route", "expert_matmul", "combine_rows"])
def test_forward_mode_is_refused(name, requires):
    """A tangent is not dropped: the functions have no forward-mode derivative and say so."""
    import torch.autograd.forward_ad as fw
    f, args = _differentiable_calls()[name]
    for i in range(len(args)):
        with fw.dual_level():
            ins = [a.clone().requires_grad_(requires) for a in args]
            ins[i] = fw.make_dual(ins[i], torch.ones_like(ins[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(*ins)
        assert torch.isfinite(f(*args).float()).all()         # without a tangent as before


def test_forward_mode_of_the_gradients_is_refused():
    import torch.autograd.forward_ad as fw
    from mlx_kmeans_b200 import combine_rows_grad, expert_matmul_grad, group_rows, route_grad
    ids = torch.tensor([[0, 1], [1, 2]], dtype=torch.int32).cuda()
    groups = group_rows(ids, 3)
    half = lambda *s: torch.ones(*s, dtype=torch.float16, device="cuda")  # noqa: E731
    full = lambda *s: torch.ones(*s, device="cuda")                      # noqa: E731
    calls = [(lambda a, b: route_grad(a, b, ids), [full(2, 2), full(2, 3)]),
             (lambda a, b, c: expert_matmul_grad(a, b, c, groups), [half(4, 8), half(2, 16), half(3, 8, 16)]),
             (lambda a, b, c: combine_rows_grad(a, b, groups, c), [full(2, 8), full(4, 8), full(2, 2)])]
    for f, args in calls:
        for i in range(len(args)):
            with fw.dual_level():
                ins = list(args)
                ins[i] = fw.make_dual(ins[i], torch.ones_like(ins[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(*ins)


# ---------------------------------------------------------------- the error word

def test_first_call_of_a_process_can_be_captured():
    """A process whose first expert_matmul is inside a graph capture: the graph replays, and no fault is reported."""
    code = """
        import torch
        from mlx_kmeans_b200 import expert_matmul, expert_status, group_rows
        torch.manual_seed(0)
        x, w = torch.randn(40, 64, device="cuda").half(), torch.randn(4, 48, 64, device="cuda").half()
        groups = group_rows((torch.arange(80, device="cuda").reshape(40, 2) % 4).int(), 4)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = expert_matmul(x, w, groups)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, expert_matmul(x, w, groups))
        expert_status()
        print("captured")
    """
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr


def test_a_kernel_that_gave_up_is_raised_by_the_next_call():
    """The word that a kernel sets when it gives up, set here from the host: forward and both gradients raise once."""
    from mlx_kmeans_b200 import _experts, expert_matmul, expert_matmul_grad, expert_status, group_rows
    groups = group_rows(torch.tensor([[0, 1], [1, 2]], dtype=torch.int32).cuda(), 3)
    x, w = torch.ones(2, 16).half().cuda(), torch.ones(3, 8, 16).half().cuda()
    dy = torch.ones(4, 8).half().cuda()
    y = expert_matmul(x, w, groups)
    torch.cuda.synchronize()
    word = _experts.error_word(x.device.index)
    assert word.dtype == torch.int32 and word.tolist() == [0]
    for f in (lambda: expert_matmul(x, w, groups), lambda: expert_matmul_grad(dy, x, w, groups), lambda: expert_status(),
              lambda: expert_matmul(x.clone().requires_grad_(True), w, groups)):
        word[0] = 1
        with pytest.raises(RuntimeError, match="gave up"):
            f()
        assert word.tolist() == [0]
        assert torch.equal(expert_matmul(x, w, groups), y)


# ---------------------------------------------------------------- extreme scores

@pytest.mark.parametrize("E", [2, 64, 200])
def test_route_grad_of_very_small_sigmoids(E):
    """Renormalised sigmoids around exp(-87): (g - dot) / S alone leaves float32's range, the gradient does not."""
    from mlx_kmeans_b200 import route, route_grad
    T = 40
    l = torch.full((T, E), -95.0)
    l[:, 0], l[:, 1] = -87.0 - torch.rand(T, generator=rng(1)), -86.5 - torch.rand(T, generator=rng(2))
    g = torch.randn(T, 2, generator=rng(3)) * 10
    ids, _ = route(l.cuda(), 2, score="sigmoid")
    assert int(ids.max()) == 1
    dl = route_grad(g.cuda(), l.cuda(), ids, score="sigmoid")
    ref, mag = ref_route_grad(l, ids.cpu(), g, "sigmoid", True, 1.0)
    # each sigmoid: 4 ulp (exponential, sum, quotient) and half a step of the subnormals, 2^-149 of at least exp(-88);
    # it enters three times, and four products and quotients round
    assert torch.all((dl.double().cpu() - ref).abs() <= (3 * (4 + 2) + 4) * 2.0 ** -23 * mag)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("E", [8, 64, 200, 600])
def test_route_grad_of_masked_rows_is_zero_whatever_they_hold(E, renorm, score, dt):
    from mlx_kmeans_b200 import route, route_grad
    T, k = 32, 2
    l = torch.randn(T, E, generator=rng(E))
    mask = torch.arange(T) % 2 == 0
    for i, v in enumerate((INF, float("nan"), -INF, torch.finfo(dt).max)):
        l[2 * i + 1, i] = v
        l[2 * i + 9, :] = v
    l, clean = l.to(dt).cuda(), torch.where(mask[:, None], l, 0.0).to(dt).cuda()
    ids, w = route(l, k, score=score, renormalize=renorm, mask=mask.cuda())
    g = torch.randn(T, k, generator=rng(1)).cuda()
    dl = route_grad(g, l, ids, score=score, renormalize=renorm)
    assert torch.all(w[~mask.cuda()] == 0) and torch.all(dl[~mask.cuda()] == 0)
    ids2, w2 = route(clean, k, score=score, renormalize=renorm, mask=mask.cuda())
    assert torch.equal(ids, ids2) and torch.equal(w, w2)
    assert torch.equal(dl[mask.cuda()], route_grad(g, clean, ids2, score=score, renormalize=renorm)[mask.cuda()])


@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("E", [8, 33, 200])
def test_softmax_of_float32_logits_far_apart(E, renorm):
    """Whole-number logits down to 85 below the largest, so that l - m is exact: what is left are the exponential's own
    2 ulp, the sum's and the quotient's rounding."""
    from mlx_kmeans_b200 import route, route_grad
    T, k = 500, 8
    l = -torch.randint(1, 86, (T, E), generator=rng(E)).float()
    l[:, 3] = 0.0
    ids, w = route(l.cuda(), k, renormalize=renorm)
    rid, rw = ref_route(l, k, "softmax", None, 1, 1, renorm, 1.0, None)
    assert (ids.cpu().numpy() == rid).all()
    # 2 ulp in the choice's exponential, 2 in the sum's terms, E additions, one quotient
    tol = (2 + 2 + E / 2 + 1) * 2.0 ** -23
    assert float(((w.cpu().double().numpy() - rw) / rw).__abs__().max()) <= tol
    g = torch.zeros(T, k)
    g[:, 0] = 1.0                                             # only the largest: the others' gradients are -p_i p_0
    dl = route_grad(g.cuda(), l.cuda(), ids, renormalize=renorm).double().cpu()
    ref, _ = ref_route_grad(l, ids.cpu(), g, "softmax", renorm, 1.0)
    small = (ref != 0) & (l < 0)
    assert float(((dl - ref) / ref)[small].abs().max()) <= 2 * tol + 2.0 ** -22


# ---------------------------------------------------------------- the library's own labels

def test_group_rows_of_fitted_labels():
    """KMeans.labels_ is a NumPy array on the host; as an int32 CUDA tensor it groups, and nothing else does."""
    import numpy as np
    from mlx_kmeans_b200 import KMeans, expert_matmul, group_rows
    X = torch.randn(3000, 8, generator=rng(5)).numpy()
    km = KMeans(n_clusters=6, random_state=0, n_init=1).fit(X)
    labels = torch.as_tensor(km.labels_).to("cuda", torch.int32)
    groups = group_rows(labels, 6)
    for a, b in zip(groups, ref_groups(np.asarray(km.labels_), 6)):
        assert np.array_equal(a.cpu().numpy(), b)
    y = expert_matmul(torch.from_numpy(X).half().cuda(), torch.ones(6, 8, 8).half().cuda(), groups)
    assert y.shape == (3000, 8)
    for bad in (km.labels_, torch.as_tensor(km.labels_), labels.long()):
        with pytest.raises(ValueError):
            group_rows(bad, 6)


# ---------------------------------------------------------------- forms that only larger or rarer shapes take

def _products(T, k, E, N, D, dt, ids=None, grads=False):
    """expert_matmul of gathered rows (and its gradients) against float64."""
    from mlx_kmeans_b200 import expert_matmul, expert_matmul_grad, group_rows
    g = rng(T + N + D)
    groups = plan(T, k, E, T) if ids is None else group_rows(ids.cuda(), E)
    x = torch.randn(T, D, generator=g).to(dt).cuda()
    w = (torch.randn(E, N, D, generator=g) / D ** 0.5).to(dt).cuda()
    dy = torch.randn(T * k, N, generator=g).to(dt).cuda() if grads else None
    (ry, ym), (rx, xm), (rw, wm) = ref_matmul(x, w, groups, True, dy)
    near(expert_matmul(x, w, groups), ry, ym, D)
    if grads:
        dx, dw = expert_matmul_grad(dy, x, w, groups)
        near(dx, by_row(groups, rx), by_row(groups, xm), N + k)
        near(dw, rw, wm, max(1, int((groups.offsets[1:] - groups.offsets[:-1]).max())))
    return x, w, groups


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("T,k,E,N,D", [(48, 4, 32, 1000, 1336), (40, 2, 8, 1000, 1336), (40, 2, 8, 1003, 1337),
                                       (45, 2, 8, 600, 2048)])
def test_products_that_gather_in_the_kernel(T, k, E, N, D, dt):
    """4 to 12 rows an expert of large matrices: x's rows are read by their indices; a row outside x reads zeros."""
    from mlx_kmeans_b200 import RowGroups, expert_matmul
    ids = torch.stack([torch.randperm(E, generator=rng(T + t))[:k] for t in range(T)]).to(torch.int32)
    ids[T // 2] = -1                                          # (pairs left out: the products' tiles end inside a group)
    x, w, groups = _products(T, k, E, N, D, dt, ids)
    y = expert_matmul(x, w, groups)
    taken = int(groups.offsets[-1])
    assert taken == (T - 1) * k and int(y[taken:].abs().max()) == 0
    rows = groups.rows.clone()
    out = torch.tensor([0, taken // 2, taken - 1])
    rows[out.cuda()] = torch.tensor([T, -7, 2 ** 31 - 1], dtype=torch.int32).cuda()
    y2 = expert_matmul(x, w, RowGroups(groups.offsets, rows, groups.slot))
    keep = torch.ones(T * k, dtype=torch.bool)
    keep[out] = False
    assert int(y2[out.cuda()].abs().max()) == 0 and torch.equal(y2[keep.cuda()], y[keep.cuda()])


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("T,k,E,N,D", [(1, 8, 12, 2048, 2048), (1, 2, 4, 256, 1024), (1, 2, 4, 130, 2184),
                                       (3, 2, 8, 72, 4104), (2, 2, 4, 65, 1337), (2, 2, 4, 40, 2565)])
def test_products_of_few_rows_with_the_depth_shared(T, k, E, N, D, dt):
    """Four warps share the depth (from 1024 on, or rows of any alignment), one to three rounds each."""
    _products(T, k, E, N, D, dt)


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("T,k,E,N,D", [(3, 2, 8, 100, 520), (3, 2, 8, 100, 776), (5, 3, 8, 33, 1000), (1, 8, 8, 1000, 1544)])
def test_products_of_few_rows_in_three_rounds_of_depth(T, k, E, N, D, dt):
    """One warp over the whole depth, past its two rounds in flight."""
    _products(T, k, E, N, D, dt)


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("D", [776, 1032, 1337])
def test_products_of_few_rows_all_on_one_expert(D, dt):
    """More rows on one expert than a pass takes (16), beside experts with none."""
    ids = torch.full((37, 1), 11, dtype=torch.int32)
    ids[5], ids[30] = 2, -1
    _products(37, 1, 12, 90, D, dt, ids)


@pytest.mark.parametrize("T,k,E,N,D", [(2000, 2, 200, 40, 24), (4300, 2, 500, 24, 40), (10300, 2, 500, 136, 72),
                                       (900, 2, 4096, 8, 16), (3000, 1, 390, 130, 33)])
def test_products_of_many_experts(T, k, E, N, D):
    """More experts than threads in the products' scan of tiles, and more than dW sorts by their rows."""
    _products(T, k, E, N, D, torch.float16, grads=True)


def _route_reference(l, k, score, bias, renorm, dw):
    """ids, float64 weights and gradients of whole rows (every logit finite)."""
    key = l.float() if score == "softmax" else 1.0 / (1.0 + torch.exp(-l.float()))
    key = key if bias is None else key + bias
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    l, dw = l.double(), dw.double()
    up = torch.zeros_like(l).scatter_(1, ids, dw)
    if score == "softmax":
        over = torch.full_like(l, -INF).scatter(1, ids, l.gather(1, ids)) if renorm else l
        p = torch.softmax(over, 1)
        return ids, p.gather(1, ids), p * (up - (up * p).sum(1, keepdim=True)), p * (up.abs() + (up * p).abs().sum(1, keepdim=True))
    s = torch.sigmoid(l)
    got = torch.zeros_like(l).scatter_(1, ids, 1.0)
    slope = s * torch.sigmoid(-l) * got
    if not renorm:
        return ids, s.gather(1, ids), up * slope, (up * slope).abs()
    total = (s * got).sum(1, keepdim=True)
    mean = (up * s).sum(1, keepdim=True) / total
    return (ids, (s / total).gather(1, ids), (up - mean) / total * slope,
            (up.abs() + (up * s).abs().sum(1, keepdim=True) / total) / total * slope)


def _check_route(l, k, score, bias, renorm):
    from mlx_kmeans_b200 import route, route_grad
    T, E = l.shape
    dw = torch.randn(T, k, generator=rng(7)).cuda()
    ids, w = route(l, k, score=score, bias=bias, renormalize=renorm)
    dl = route_grad(dw, l, ids, score=score, renormalize=renorm)
    rid, rw, rdl, mag = _route_reference(l, k, score, bias, renorm, dw)
    assert torch.equal(ids.long(), rid)
    spread = float(l.float().max() - l.float().min())
    eps = (spread + 16 + E ** 0.5) * 2.0 ** -23               # as eps_of in test_experts_gpu.py
    assert torch.all((w.double() - rw).abs() <= eps * rw + 1e-37)
    tol = U[l.dtype] * rdl.abs() + 4 * (eps + k * 2.0 ** -23) * mag + TINY[l.dtype]
    assert torch.all((dl.double() - rdl).abs() <= tol)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("T,E,k,biased", [(16384, 129, 16, False), (16385, 200, 8, True), (16391, 256, 3, False), (16384, 250, 9, True)])
def test_route_of_many_rows_of_many_experts(T, E, k, biased, renorm, score, dt):
    """129 to 256 experts and 16384 rows on: sixteen lanes a row with sixteen experts each."""
    g = rng(T + E)
    l = (torch.randn(T, E, generator=g) * 2).to(dt).cuda()
    _check_route(l, k, score, (torch.randn(E, generator=g) * 0.3).cuda() if biased else None, renorm)


@pytest.mark.parametrize("T,E,k", [(70, 8, 2), (70, 32, 8), (70, 64, 4), (70, 64, 8), (70, 128, 8), (70, 128, 16), (70, 33, 20),
                                   (16390, 200, 8), (70, 256, 20), (70, 500, 9), (70, 1000, 32)])
@pytest.mark.parametrize("dt", TYPES)
def test_route_keys_that_differ_in_their_last_bits(T, E, k, dt):
    """Keys whose upper bits agree (the choice's fast path cuts the lower ones off for the index): float32 logits or
    biased 16-bit ones next to each other, in some of the rows."""
    g = rng(E + k)
    step = torch.stack([torch.randperm(E, generator=g) for _ in range(70)]).repeat((T + 69) // 70, 1)[:T].float()
    close = (torch.rand(T, 1, generator=g) < 0.5).float()
    if dt == torch.float32:
        l = (1.0 + step * 2.0 ** -23) * close + torch.randn(T, E, generator=g) * (1 - close)
        _check_route(l.cuda(), k, "softmax", None, True)
        _check_route((-l).cuda(), k, "softmax", None, True)
    else:
        l = torch.where(close > 0, torch.ones(T, E), torch.randn(T, E, generator=g)).to(dt)
        bias = step[0] * 2.0 ** -23 + 0.5
        _check_route(l.cuda(), k, "softmax", bias.cuda(), True)
        _check_route((-l).cuda(), k, "softmax", (-bias).cuda(), True)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("T,k,H", [(3, 2, 33), (130, 8, 512)])
def test_combine_grad_of_whole_plans_through_the_c_entry(T, k, H, dt):
    """kmc_combine_grad, told where the pairs end, gives what kmc_combine_grad_slots finds out."""
    from mlx_kmeans_b200 import _lib, combine_rows_grad
    L, g = _lib.load(), rng(T)
    groups = plan(T, k, max(4, k), T, drop=0.2)
    y, dout = torch.randn(T * k, H, generator=g).to(dt).cuda(), torch.randn(T, H, generator=g).to(dt).cuda()
    w = torch.rand(T, k, generator=g).cuda()
    want_dy, want_dw = combine_rows_grad(dout, y, groups, w)
    dy, dw = torch.full_like(y, float("nan")), torch.full_like(w, float("nan"))
    kind = {torch.float32: _lib.KMC_F32, torch.bfloat16: _lib.KMC_BF16, torch.float16: _lib.KMC_F16}[dt]
    _lib.check(L.kmc_combine_grad(dout.data_ptr(), y.data_ptr(), kind, T, k, H, groups.slot.data_ptr(), w.data_ptr(),
                                  groups.offsets[-1:].data_ptr(), dy.data_ptr(), dw.data_ptr(),
                                  torch.cuda.current_stream().cuda_stream), "kmc_combine_grad")
    assert torch.equal(dy, want_dy) and torch.equal(dw, want_dw)
