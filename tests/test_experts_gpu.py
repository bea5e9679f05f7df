"""Routed experts on the GPU (route, group_rows, expert_matmul, combine_rows and their gradients) against plain
float64 implementations of the formulas, at the sizes, masks and strides where they can go wrong.

Tolerances come from the arithmetic: u = 2^-24 / 2^-11 / 2^-8 is the unit roundoff of a float32 / float16 / bfloat16
result (one rounding), a float32 sum of n products adds at most 2 n 2^-24 of the sum of their magnitudes (2: a tensor
core may cut instead of round), and a float32 exponential of a difference l - m is off by (|l - m| + 8) 2^-23 at most.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}   # below: no relative bound
INF = float("inf")
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _status(cuda_device):
    """No kernel gave up on a barrier in any of these tests."""
    yield
    from mlx_kmeans_b200 import expert_status
    expert_status()


def rng(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------- routing

def ref_route(logits, k, score, bias, groups, top_groups, renorm, scale, mask):
    """ids and float64 weights; keys in float32 as defined (torch's float32 exp on the GPU for the sigmoid)."""
    l = logits.float()
    key = l if score == "softmax" else 1.0 / (1.0 + torch.exp(-l))
    if bias is not None:
        key = key + bias
    key, l = key.cpu().numpy(), l.cpu().numpy().astype(np.float64)
    T, E = l.shape
    ids = np.full((T, k), -1, np.int32)
    w = np.zeros((T, k))
    for t in range(T):
        ok = (l[t] > -INF) & (key[t] > -INF)
        if mask is not None and not mask[t]:
            ok[:] = False
        if groups > 1:
            gs = E // groups
            scores = []
            for g in range(groups):
                best = sorted((key[t, i] for i in range(g * gs, (g + 1) * gs) if ok[i]), reverse=True)[:2]
                scores.append(np.float32(sum(best[1:], best[0])) if best else -INF)
            order = sorted((g for g in range(groups) if scores[g] > -INF), key=lambda g: (-scores[g], g))[:top_groups]
            ok &= np.isin(np.arange(E) // gs, order)
        pick = sorted(np.nonzero(ok)[0], key=lambda i: (-key[t, i], i))[:k]
        ids[t, :len(pick)] = pick
        if not pick:
            continue
        if score == "softmax":
            over = l[t][pick] if renorm else l[t][l[t] > -INF]
            m = over.max()
            w[t, :len(pick)] = np.exp(l[t][pick] - m) / np.exp(over - m).sum()
        else:
            s = 1.0 / (1.0 + np.exp(-l[t][pick]))
            w[t, :len(pick)] = s / s.sum() if renorm else s
    return ids, scale * w


def eps_of(logits, E):
    l = logits.float().cpu().double()
    l = l[torch.isfinite(l)]
    spread = float(l.max() - l.min()) if l.numel() else 0.0
    return (spread + 16 + E ** 0.5) * 2.0 ** -23


ROUTES = [
    # T, E, k, dtype, score, bias, groups, top_groups, renorm
    (1, 1, 1, torch.float32, "softmax", False, 1, 1, True),
    (1, 64, 4, torch.bfloat16, "softmax", False, 1, 1, True),
    (3, 5, 5, torch.float16, "softmax", False, 1, 1, False),
    (37, 31, 3, torch.float32, "sigmoid", True, 1, 1, True),
    (37, 33, 8, torch.bfloat16, "softmax", True, 1, 1, False),
    (19, 60, 4, torch.float16, "sigmoid", False, 1, 1, False),
    (23, 96, 6, torch.float32, "softmax", False, 4, 2, True),
    (23, 96, 7, torch.bfloat16, "sigmoid", True, 3, 2, True),
    (41, 256, 8, torch.float32, "sigmoid", True, 8, 4, True),
    (41, 256, 8, torch.bfloat16, "softmax", True, 8, 3, False),
    (9, 160, 8, torch.float16, "softmax", False, 32, 5, True),
    (9, 64, 32, torch.float32, "softmax", False, 32, 16, False),
    (11, 257, 9, torch.bfloat16, "sigmoid", False, 1, 1, True),
    (5, 1000, 16, torch.float32, "softmax", False, 8, 3, True),
    (5, 1024, 32, torch.bfloat16, "sigmoid", True, 16, 2, True),
    (1030, 128, 8, torch.bfloat16, "softmax", False, 1, 1, True),
]


def route_inputs(case, seed=0, hard=True):
    T, E, k, dt, score, bias, *_ = case
    g = rng(seed)
    l = torch.randn(T, E, generator=g) * 2
    if hard and E > 4:
        l[:, 1] = l[:, 0]                                     # ties in every row
        l[T // 2, E // 2:] = -INF                             # a row with half its experts masked
        l[T // 3, 0] = float("nan")                           # not available
        l[-1] = -INF                                          # a row with none
        l[0, E - 1] = torch.finfo(dt).min                     # masked by the type's lowest value
    l = l.to(dt).cuda()
    b = (torch.randn(E, generator=g) * 0.3).cuda() if bias else None
    return l, b


@pytest.mark.parametrize("case", ROUTES)
@pytest.mark.parametrize("masked", [False, True])
def test_route(case, masked):
    from mlx_kmeans_b200 import route
    T, E, k, dt, score, _, groups, top, renorm = case
    l, b = route_inputs(case)
    mask = None
    if masked:
        mask = torch.rand(T, generator=rng(5)) < 0.7
    ids, w = route(l, k, score=score, bias=b, groups=groups, top_groups=top, renormalize=renorm, scale=2.5,
                   mask=mask.cuda() if masked else None)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32 and ids.shape == w.shape == (T, k)
    rid, rw = ref_route(l, k, score, b, groups, top, renorm, 2.5, mask)
    assert np.array_equal(ids.cpu().numpy(), rid)
    assert np.all(np.abs(w.cpu().double().numpy() - rw) <= eps_of(l, E) * rw + 1e-37)


def ref_route_grad(l, ids, g, score, renorm, scale):
    l = l.double().cpu()
    T, E = l.shape
    out, mag = torch.zeros(T, E, dtype=torch.float64), torch.zeros(T, E, dtype=torch.float64)
    for t in range(T):
        js = [j for j in range(ids.shape[1]) if ids[t, j] >= 0]
        if not js:
            continue
        pick = [int(ids[t, j]) for j in js]
        up = scale * g[t, js].double()
        live = torch.nan_to_num(l[t], nan=-INF)
        if score == "softmax":
            p = torch.zeros(E, dtype=torch.float64)
            if renorm:
                p[pick] = torch.softmax(live[pick], 0)
            else:
                p = torch.softmax(live, 0)
            s = torch.zeros(E, dtype=torch.float64)
            s[pick] = up
            out[t] = p * (s - (s * p).sum())
            mag[t] = p * (s.abs() + (s * p).abs().sum())
        else:
            sg = torch.sigmoid(live[pick])
            slope = sg * torch.sigmoid(-live[pick])
            if renorm:
                S = sg.sum()
                out[t, pick] = (up - (up * sg).sum() / S) / S * slope
                mag[t, pick] = (up.abs() + (up * sg).abs().sum() / S) / S * slope
            else:
                out[t, pick] = up * slope
                mag[t, pick] = (up * slope).abs()
    return out, mag


@pytest.mark.parametrize("case", ROUTES)
def test_route_grad(case):
    from mlx_kmeans_b200 import route, route_grad
    T, E, k, dt, score, _, groups, top, renorm = case
    l, b = route_inputs(case, 1)
    ids, _ = route(l, k, score=score, bias=b, groups=groups, top_groups=top, renormalize=renorm, scale=2.5)
    g = torch.randn(T, k, generator=rng(2))
    dl = route_grad(g.cuda(), l, ids, score=score, renormalize=renorm, scale=2.5)
    assert dl.dtype == dt and dl.shape == l.shape
    ref, mag = ref_route_grad(l, ids.cpu(), g, score, renorm, 2.5)
    tol = U[dt] * ref.abs() + 4 * (eps_of(l, E) + k * 2.0 ** -23) * mag + TINY[dt]
    assert torch.all((dl.double().cpu() - ref).abs() <= tol)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("E,k", [(8, 2), (32, 8), (64, 8), (128, 16), (128, 20), (300, 4)])
def test_route_rows_without_a_choice_beside_others(E, k, score, renorm):
    """Rows that share a warp with masked rows, in every order: the weights and gradients of the rows alone."""
    from mlx_kmeans_b200 import route, route_grad
    T = 64
    l = torch.randn(T, E, generator=rng(E), dtype=torch.float32).cuda()
    mask = torch.rand(T, generator=rng(k)) < 0.5
    g = torch.randn(T, k, generator=rng(1)).cuda()
    ids, w = route(l, k, score=score, renormalize=renorm, mask=mask.cuda())
    dl = route_grad(g, l, ids, score=score, renormalize=renorm)
    alone_ids, alone_w = route(l[mask.cuda()], k, score=score, renormalize=renorm)
    alone_dl = route_grad(g[mask.cuda()], l[mask.cuda()], alone_ids, score=score, renormalize=renorm)
    assert torch.equal(ids[mask.cuda()], alone_ids) and torch.equal(w[mask.cuda()], alone_w)
    assert torch.equal(dl[mask.cuda()], alone_dl)
    off = ~mask.cuda()
    assert int(ids[off].max()) == -1 and float(w[off].abs().max()) == 0.0 and float(dl[off].abs().max()) == 0.0


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [8, 64, 128, 256, 1000])
def test_route_lone_renormalised_choice(E, score):
    """One choice renormalised has the weight `scale` whatever its logit, and a gradient of exactly 0."""
    from mlx_kmeans_b200 import route, route_grad
    l = (torch.randn(300, E, generator=rng(E)) * 3).cuda()
    ids, w = route(l, 1, score=score, scale=2.5)
    assert torch.all(w == 2.5)
    dl = route_grad(torch.randn(300, 1, generator=rng(1)).cuda(), l, ids, score=score, scale=2.5)
    assert torch.all(dl == 0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_grad_against_differences(score, renorm):
    """The central difference of L = sum g w along a direction, the choice kept by logits 0.25 apart."""
    from mlx_kmeans_b200 import route
    T, E, k, h = 4, 24, 3, 2.0 ** -7
    gen = rng(3)
    l = torch.stack([torch.randperm(E, generator=gen) for _ in range(T)]).float().cuda() * 0.25 - 3
    g, v = torch.randn(T, k, generator=gen).cuda(), torch.randn(T, E, generator=gen).cuda().clamp(-1, 1)
    x = l.clone().requires_grad_(True)
    _, w = route(x, k, score=score, renormalize=renorm)
    (w * g).sum().backward()
    loss = lambda z: float((route(z, k, score=score, renormalize=renorm)[1].double() * g.double()).sum())  # noqa: E731
    diff = (loss(l + h * v) - loss(l - h * v)) / (2 * h)
    size = float(g.abs().sum())
    # third derivatives of the weights along v stay below 6; each weight is off by at most 32 2^-23
    assert abs(diff - float((x.grad.double() * v.double()).sum())) <= size * (h * h + 32 * 2.0 ** -23 / h)
    assert float(x.grad.abs().max()) > 1e-3


def test_route_rows_apart_and_unaligned():
    from mlx_kmeans_b200 import route, route_grad
    base = torch.randn(50, 131, generator=rng(7)).cuda()
    for dt in TYPES:
        wide = base.to(dt)
        for view in (wide[:, 3:67], wide[::2, 1:65], wide.t()[:64, :50].t(), wide[:1, 5:69].expand(6, 64)):
            dense = view.contiguous()
            a, b = route(view, 4), route(dense, 4)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
            g = torch.ones_like(a[1])
            g[:, 0] = 3
            assert torch.equal(route_grad(g, view, a[0]), route_grad(g, dense, b[0]))


def test_route_infinite_and_lowest_logits():
    from mlx_kmeans_b200 import route
    low = torch.finfo(torch.float32).min
    l = torch.tensor([[low, low, low, -INF], [-INF, -INF, -INF, low], [-INF] * 4, [float("nan")] * 4,
                      [1.0, float("nan"), -INF, 2.0]]).cuda()
    ids, w = route(l, 2)
    assert ids.tolist() == [[0, 1], [3, -1], [-1, -1], [-1, -1], [3, 0]]
    assert w[:4].tolist() == [[0.5, 0.5], [1.0, 0.0], [0.0, 0.0], [0.0, 0.0]]
    ids, w = route(l, 2, score="sigmoid")
    assert ids.tolist() == [[0, 1], [3, -1], [-1, -1], [-1, -1], [3, 0]]
    assert w[:4].tolist() == [[0.0, 0.0], [0.0, 0.0], [0.0, 0.0], [0.0, 0.0]]      # every chosen score is 0
    bias = torch.tensor([0.0, -INF, 0.0, float("nan")]).cuda()                     # experts taken out by the bias
    ids, _ = route(torch.zeros(2, 4).cuda(), 3, bias=bias)
    assert ids.tolist() == [[0, 2, -1], [0, 2, -1]]
    ids, w = route(torch.tensor([[-0.0, 0.0, -0.0]]).cuda(), 3)                    # equal keys: index order
    assert ids.tolist() == [[0, 1, 2]]


# ---------------------------------------------------------------- grouping

def ref_groups(ids, E):
    ids = np.asarray(ids)
    flat = ids.reshape(-1)
    k = ids.shape[1] if ids.ndim == 2 else 1
    off, rows, slot = [0], [], np.full(flat.shape, -1, np.int32)
    for e in range(E):
        for p in np.nonzero(flat == e)[0]:
            slot[p] = len(rows)
            rows.append(p // k)
        off.append(len(rows))
    return np.array(off, np.int32), np.array(rows + [-1] * (flat.size - len(rows)), np.int32), slot.reshape(ids.shape)


@pytest.mark.parametrize("T,k,E", [(0, 2, 4), (1, 1, 1), (1, 8, 64), (24, 8, 128), (33, 3, 7), (1000, 2, 60),
                                   (1025, 8, 1000), (4097, 2, 16), (9001, 1, 4096), (20011, 3, 5), (5000, 8, 1100)])
def test_group_rows(T, k, E):
    from mlx_kmeans_b200 import group_rows
    ids = torch.randint(-2, E + 2, (T, k), generator=rng(T + k), dtype=torch.int32)
    if E > 3:
        ids[ids == 2] = 1                                     # an expert with no pair
    got = group_rows(ids.cuda(), E)
    want = ref_groups(ids.numpy(), E)
    for a, b in zip(got, want):
        assert a.dtype == torch.int32 and np.array_equal(a.cpu().numpy(), b)


def test_group_rows_of_labels_and_extremes():
    from mlx_kmeans_b200 import group_rows
    lab = torch.randint(0, 37, (70_003,), generator=rng(1), dtype=torch.int32)
    got = group_rows(lab.cuda(), 37)
    order = np.argsort(lab.numpy(), kind="stable")
    assert np.array_equal(got.rows.cpu().numpy(), order)
    assert np.array_equal(got.slot.cpu().numpy()[order], np.arange(lab.numel()))
    one = group_rows(torch.full((30_000, 1), 3, dtype=torch.int32).cuda(), 4)          # every pair on one expert
    assert one.offsets.tolist() == [0, 0, 0, 0, 30_000] and torch.equal(one.rows, torch.arange(30_000, dtype=torch.int32).cuda())
    none = group_rows(torch.full((20_000, 1), -1, dtype=torch.int32).cuda(), 4)
    assert none.offsets.tolist() == [0] * 5 and int(none.rows.max()) == -1 and int(none.slot.max()) == -1
    big = torch.randint(0, 256, (300_000, 4), generator=rng(2), dtype=torch.int32)
    got = group_rows(big.cuda(), 256)
    order = np.argsort(big.numpy().reshape(-1), kind="stable")
    assert np.array_equal(got.rows.cpu().numpy(), order // 4)


# ---------------------------------------------------------------- products per expert

def plan(T, k, E, seed, drop=0.1, empty=()):
    """Random choices with some pairs left out and some experts empty; the last rows all on one expert."""
    from mlx_kmeans_b200 import group_rows
    g = rng(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32) if T else torch.zeros(0, k, dtype=torch.int32)
    ids[torch.rand(T, k, generator=g) < drop] = -1
    for e in empty:
        ids[ids == e] = -1
    return group_rows(ids.cuda(), E)


def ref_matmul(x, w, groups, gather, dy=None):
    """Products and their gradients, and the same of the magnitudes, in float64."""
    off, rows = groups.offsets.cpu().tolist(), groups.rows.cpu().long()
    xs, ws = x.double().cpu(), w.double().cpu()
    P, (E, N, D) = rows.numel(), w.shape
    y, ym = torch.zeros(P, N, dtype=torch.float64), torch.zeros(P, N, dtype=torch.float64)
    dxp, dxm = torch.zeros(P, D, dtype=torch.float64), torch.zeros(P, D, dtype=torch.float64)
    dw, dwm = torch.zeros(E, N, D, dtype=torch.float64), torch.zeros(E, N, D, dtype=torch.float64)
    for e in range(E):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        xe = xs[rows[a:b]] if gather else xs[a:b]
        y[a:b], ym[a:b] = xe @ ws[e].T, xe.abs() @ ws[e].abs().T
        if dy is not None:
            de = dy[a:b].double().cpu()
            dxp[a:b], dxm[a:b] = de @ ws[e], de.abs() @ ws[e].abs()
            dw[e], dwm[e] = de.T @ xe, de.abs().T @ xe.abs()
    return (y, ym), (dxp, dxm), (dw, dwm)


def near(got, ref, mag, n, extra=0.0):
    dt = got.dtype
    tol = U[dt] * ref.abs() + 2 * n * 2.0 ** -24 * mag + TINY[dt] + extra
    assert torch.all((got.double().cpu() - ref).abs() <= tol)


SHAPES = [
    # T, k, E, N, D: one token, sizes below, at and past the tiles, odd ones, many and few rows an expert
    (1, 1, 1, 1, 1), (1, 8, 64, 64, 64), (1, 4, 16, 256, 512), (3, 2, 8, 40, 72), (5, 2, 4, 129, 264),
    (16, 4, 8, 100, 136), (48, 4, 12, 200, 336), (64, 2, 5, 33, 35), (130, 1, 2, 128, 128), (257, 2, 3, 130, 66),
    (300, 1, 1, 256, 64), (515, 2, 4, 65, 515), (700, 3, 7, 384, 192), (1100, 2, 3, 136, 1000), (2100, 1, 2, 72, 48),
]


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_expert_matmul(shape, gather, dt):
    from mlx_kmeans_b200 import expert_matmul, expert_matmul_grad
    T, k, E, N, D = shape
    g = rng(T + N)
    groups = plan(T, k, E, T, empty=(1,) if E > 2 else ())
    x = torch.randn(T if gather else T * k, D, generator=g).to(dt).cuda()
    w = (torch.randn(E, N, D, generator=g) / D ** 0.5).to(dt).cuda()
    dy = torch.randn(T * k, N, generator=g).to(dt).cuda()
    taken = int(groups.offsets[-1])
    if not gather:
        x[taken:] = float("nan")                              # positions no pair took are not read
    dy[taken:] = float("nan")
    y = expert_matmul(x, w, groups, gather=gather)
    dx, dw = expert_matmul_grad(dy, x, w, groups, gather=gather)
    (ry, ym), (rx, xm), (rw, wm) = ref_matmul(x, w, groups, gather, dy)
    near(y, ry, ym, D)
    near(dw, rw, wm, max(1, int((groups.offsets[1:] - groups.offsets[:-1]).max())))
    if not gather:
        near(dx, rx, xm, N)
        return
    slot = groups.slot.cpu().long()
    got = (slot >= 0)[:, :, None]
    pick = lambda v: torch.where(got, v[slot.clamp(min=0)], 0.0)  # noqa: E731
    # each position's gradient is rounded to the type before the float32 sum over a row's choices
    near(dx, pick(rx).sum(1), pick(xm).sum(1), N + k, extra=pick(U[dt] * rx.abs() + TINY[dt]).sum(1))


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("shape", [(1, 4, 8, 48, 40), (40, 2, 6, 96, 80), (700, 2, 3, 264, 96), (333, 3, 5, 77, 51)])
def test_expert_matmul_whole_numbers_exactly(shape, dt):
    """Products of -1, 0, 1: every sum is a whole number below 2^8, so any wrong index shows; and the gradients are
    the exact differences of L = <dy, y> (L is linear in x and in w)."""
    from mlx_kmeans_b200 import combine_rows, expert_matmul, expert_matmul_grad
    T, k, E, N, D = shape
    g = rng(N)
    groups = plan(T, k, E, N)
    ints = lambda *s: torch.randint(-1, 2, s, generator=g).to(dt).cuda()  # noqa: E731
    x, w, dy = ints(T, D), ints(E, N, D), ints(T * k, N)
    dy[torch.rand(T * k, generator=g) > 60.0 / T] = 0           # |dw| and |dx| below 2^8 too
    y = expert_matmul(x, w, groups)
    dx, dw = expert_matmul_grad(dy, x, w, groups)
    (ry, _), (rx, _), (rw, _) = ref_matmul(x, w, groups, True, dy)
    assert torch.equal(y.double().cpu(), ry) and torch.equal(dw.double().cpu(), rw)
    loss = lambda xx, ww: float((expert_matmul(xx, ww, groups).double() * dy.double()).sum())  # noqa: E731
    row, e = T // 2, int((groups.offsets[1:] > groups.offsets[:-1]).nonzero()[0])
    x2 = x.clone()
    x2[row] += 1
    assert loss(x2, w) - loss(x, w) == float(dx[row].double().sum())
    w2 = w.clone()
    w2[e, N // 2] += 1
    assert loss(x, w2) - loss(x, w) == float(dw[e, N // 2].double().sum())
    assert torch.equal(combine_rows(y, groups).double().cpu(),
                       torch.where((groups.slot.cpu() >= 0)[:, :, None], ry[groups.slot.cpu().long().clamp(min=0)], 0.0).sum(1))


@pytest.mark.parametrize("shape", [(6, 2, 4, 64, 64), (400, 1, 3, 128, 64), (400, 1, 3, 50, 33)])
def test_expert_matmul_keeps_non_finite_rows_apart(shape):
    """NaN and infinity in a row, in an expert's matrix or in a gradient touch only the results made from them."""
    from mlx_kmeans_b200 import expert_matmul, expert_matmul_grad, group_rows
    T, k, E, N, D = shape
    ids = (torch.arange(T * k).reshape(T, k) % E).to(torch.int32)
    groups = group_rows(ids.cuda(), E)
    g = rng(0)
    mk = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    x, w, dy = mk(T, D), mk(E, N, D), mk(T * k, N)
    y = expert_matmul(x, w, groups)
    dx, dw = expert_matmul_grad(dy, x, w, groups)
    bad = x.clone()
    bad[3, 1], bad[0, 0] = INF, float("nan")
    hit = torch.zeros(T * k, dtype=torch.bool)
    hit[groups.slot[[0, 3]].cpu().long().reshape(-1)] = True
    yb = expert_matmul(bad, w, groups).cpu()
    assert torch.equal(yb[~hit], y.cpu()[~hit]) and not torch.isfinite(yb[hit]).any()
    dwb = expert_matmul_grad(dy, bad, w, groups)[1].cpu()
    hit_e = sorted({int(e) for e in ids[[0, 3]].reshape(-1)})
    keep = [e for e in range(E) if e not in hit_e]
    assert torch.equal(dwb[keep], dw.cpu()[keep])
    wbad = w.clone()
    wbad[E - 1] = float("nan")
    mine = torch.zeros(T * k, dtype=torch.bool)
    mine[int(groups.offsets[E - 1]):int(groups.offsets[E])] = True
    yb = expert_matmul(x, wbad, groups).cpu()
    assert torch.equal(yb[~mine], y.cpu()[~mine]) and torch.isnan(yb[mine]).all()
    dyb = dy.clone()
    dyb[int(groups.offsets[1])] = float("nan")                  # the first position of expert 1
    dwb = expert_matmul_grad(dyb, x, w, groups)[1].cpu()
    assert torch.equal(dwb[[e for e in range(E) if e != 1]], dw.cpu()[[e for e in range(E) if e != 1]])
    assert torch.isnan(dwb[1]).all()


def test_expert_matmul_strides_and_alignment():
    from mlx_kmeans_b200 import RowGroups, expert_matmul, expert_matmul_grad
    T, k, E, N, D = 150, 2, 4, 72, 64
    g = rng(4)
    groups = plan(T, k, E, 4)
    wide = torch.randn(2 * T, D + 24, generator=g).to(torch.bfloat16).cuda()
    w = torch.randn(E, N, D, generator=g).to(torch.bfloat16).cuda()
    dy = torch.randn(T * k, N, generator=g).to(torch.bfloat16).cuda()
    odd = torch.empty(T * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, D)      # 2-byte aligned only
    odd.copy_(wide[:T, :D])
    oddw = torch.empty(E * N * D + 3, dtype=torch.bfloat16, device="cuda")[3:].view(E, N, D)
    oddw.copy_(w)
    odddy = torch.empty(T * k * N + 5, dtype=torch.bfloat16, device="cuda")[5:].view(T * k, N)
    odddy.copy_(dy)
    for view in (wide[:T, :D], wide[::2, 8:8 + D], wide[:T, 3:3 + D], wide[:T, :D].t().contiguous().t(), odd,
                 wide[:1, :D].expand(T, D)):
        dense = view.contiguous()
        y = expert_matmul(dense, w, groups)
        dx, dw = expert_matmul_grad(dy, dense, w, groups)
        for ww, dd in ((w, dy), (oddw, odddy), (w.transpose(1, 2).contiguous().transpose(1, 2), dy)):
            assert torch.equal(expert_matmul(view, ww, groups), y)
            dx2, dw2 = expert_matmul_grad(dd, view, ww, groups)
            assert torch.equal(dx2, dx) and torch.equal(dw2, dw)
    # positions whose row lies outside x read zeros
    rows = groups.rows.clone()
    rows[:3] = torch.tensor([T, -7, 2 ** 31 - 1], dtype=torch.int32)
    y = expert_matmul(wide[:T, :D], w, RowGroups(groups.offsets, rows, groups.slot))
    assert int(y[:3].abs().max()) == 0 and int(y[3].abs().max()) != 0


def test_expert_matmul_many_experts_and_none():
    from mlx_kmeans_b200 import expert_matmul, expert_matmul_grad, group_rows
    E, N, D = 4096, 8, 16
    ids = torch.randint(0, E, (900, 2), generator=rng(9), dtype=torch.int32).cuda()
    groups = group_rows(ids, E)
    w = torch.randn(E, N, D, generator=rng(1)).half().cuda()
    x = torch.randn(900, D, generator=rng(2)).half().cuda()
    (ry, ym), _, _ = ref_matmul(x, w, groups, True)
    near(expert_matmul(x, w, groups), ry, ym, D)
    empty = group_rows(torch.zeros(0, 2, dtype=torch.int32).cuda(), 3)
    x0, w3 = x[:0], w[:3]
    assert expert_matmul(x0, w3, empty).shape == (0, N)
    dx, dw = expert_matmul_grad(torch.zeros(0, N).half().cuda(), x0, w3, empty)
    assert dx.shape == (0, D) and int(dw.abs().max()) == 0
    none = group_rows(torch.full((50, 2), -1, dtype=torch.int32).cuda(), 3)
    assert int(expert_matmul(x[:50], w3, none).abs().max()) == 0
    dx, dw = expert_matmul_grad(torch.full((100, N), float("nan")).half().cuda(), x[:50], w3, none)
    assert int(dx.abs().max()) == 0 and int(dw.abs().max()) == 0


def test_expert_matmul_offsets_past_32_bits():
    """y of 2^31 elements and more: positions whose byte and element offsets pass 32 bits."""
    from mlx_kmeans_b200 import expert_matmul, group_rows
    T, k, N, D = 300_000, 8, 1024, 8
    ids = torch.arange(8, dtype=torch.int32).repeat(T, 1).cuda()
    groups = group_rows(ids, 8)
    x = torch.randn(T, D, generator=rng(3)).to(torch.bfloat16).cuda()
    w = torch.randn(8, N, D, generator=rng(4)).to(torch.bfloat16).cuda()
    y = expert_matmul(x, w, groups)
    assert y.numel() > 2 ** 31
    for p in (0, T * k // 2 + 17, T * k - 1):
        e, t = p // T, p % T
        ref = w[e].double() @ x[t].double()
        assert torch.all((y[p].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-5)


# ---------------------------------------------------------------- combination

@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("T,k,H", [(1, 1, 1), (1, 8, 64), (3, 2, 33), (48, 4, 200), (130, 8, 515), (77, 32, 24), (40, 3, 2048)])
@pytest.mark.parametrize("weighted", [True, False])
def test_combine_rows(T, k, H, dt, weighted):
    from mlx_kmeans_b200 import combine_rows, combine_rows_grad
    E = max(4, k)
    groups = plan(T, k, E, T + H, drop=0.2)
    if T > 2:
        groups.slot[1] = -1                                   # a row with no pair (its positions then have none)
    g = rng(H)
    y = torch.randn(T * k, H, generator=g).to(dt).cuda()
    dout = torch.randn(T, H, generator=g).to(dt).cuda()
    w = torch.rand(T, k, generator=g).cuda() if weighted else None
    out = combine_rows(y, groups, w)
    dy, dw = combine_rows_grad(dout, y, groups, w)
    slot = groups.slot.cpu().long()
    got = (slot >= 0)[:, :, None]
    wv = (w.double().cpu() if weighted else torch.ones(T, k, dtype=torch.float64))[:, :, None]
    yg = torch.where(got, y.double().cpu()[slot.clamp(min=0)], 0.0)
    near(out, (yg * wv).sum(1), (yg * wv).abs().sum(1), k + 1)
    do = dout.double().cpu()[:, None, :]
    ref = torch.zeros(T * k, H, dtype=torch.float64)
    ref[slot[slot >= 0]] = (wv * do).expand(T, k, H)[slot >= 0]
    has = torch.zeros(T * k, dtype=torch.bool)
    has[slot[slot >= 0]] = True
    has[int(groups.offsets[-1]):] = True                      # these are written too: zeros
    near(dy.cpu()[has], ref[has], ref[has].abs(), 1)
    if weighted:
        near(dw, (yg * do).sum(2), (yg * do).abs().sum(2), H)
    else:
        assert dw is None


def test_combine_rows_against_differences():
    """out is linear in y and in the weights: whole numbers give exact differences."""
    from mlx_kmeans_b200 import combine_rows, combine_rows_grad
    T, k, H = 20, 3, 40
    groups = plan(T, k, 6, 1)
    g = rng(6)
    y, dout = (torch.randint(-4, 5, s, generator=g).float().cuda() for s in ((T * k, H), (T, H)))
    w = torch.randint(1, 5, (T, k), generator=g).float().cuda()
    dy, dw = combine_rows_grad(dout, y, groups, w)
    loss = lambda yy, ww: float((combine_rows(yy, groups, ww).double() * dout.double()).sum())  # noqa: E731
    y2, w2 = y.clone(), w.clone()
    y2[5] += 1
    w2[7, 1] += 1
    assert loss(y2, w) - loss(y, w) == float(dy[5].double().sum())
    assert loss(y, w2) - loss(y, w) == float(dw[7, 1])


def test_combine_rows_ignores_what_no_pair_reads():
    from mlx_kmeans_b200 import combine_rows, group_rows
    ids = torch.tensor([[0, 1], [-1, 2], [-1, -1]], dtype=torch.int32).cuda()
    groups = group_rows(ids, 3)
    y = torch.ones(6, 8).cuda()
    y[3:] = float("nan")                                      # positions past offsets[-1]
    out = combine_rows(y, groups, torch.tensor([[0.5, 0.25], [float("nan"), 2.0], [INF, 1.0]]).cuda())
    assert out[:, 0].tolist() == [0.75, 2.0, 0.0]


# ---------------------------------------------------------------- together

def test_autograd_is_the_plain_gradients():
    from mlx_kmeans_b200 import (combine_rows, combine_rows_grad, expert_matmul, expert_matmul_grad, group_rows, route,
                                 route_grad)
    T, k, E, N, D = 90, 2, 6, 56, 64
    g = rng(8)
    l = torch.randn(T, E, generator=g).cuda().requires_grad_(True)
    x = torch.randn(T, D, generator=g).to(torch.bfloat16).cuda().requires_grad_(True)
    w = torch.randn(E, N, D, generator=g).to(torch.bfloat16).cuda().requires_grad_(True)
    dout = torch.randn(T, N, generator=g).to(torch.bfloat16).cuda()
    ids, weights = route(l, k, score="sigmoid", bias=torch.zeros(E).cuda())
    groups = group_rows(ids, E)
    y = expert_matmul(x, w, groups)
    out = combine_rows(y, groups, weights)
    out.backward(dout)
    dy, dweights = combine_rows_grad(dout, y.detach(), groups, weights.detach())
    dx, dw = expert_matmul_grad(dy, x.detach(), w.detach(), groups)
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)
    assert torch.equal(l.grad, route_grad(dweights, l.detach(), ids, score="sigmoid"))


def test_on_another_stream_and_in_a_graph():
    """Work goes to the current stream, repeats bit for bit, and a graph of the four steps replays on new inputs."""
    from mlx_kmeans_b200 import combine_rows, expert_matmul, group_rows, route
    T, k, E, N, D = 300, 4, 16, 128, 256
    g = rng(10)
    w = torch.randn(E, N, D, generator=g).to(torch.bfloat16).cuda()
    data = [(torch.randn(T, E, generator=g).cuda(), torch.randn(T, D, generator=g).to(torch.bfloat16).cuda()) for _ in range(2)]

    def step(l, x):
        ids, weights = route(l, k)
        groups = group_rows(ids, E)
        return combine_rows(expert_matmul(x, w, groups), groups, weights)

    want = [step(*d) for d in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [step(*d) for d in data]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))
    l, x = (t.clone() for t in data[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(l, x)
    for (dl, dx), ref in zip(data[::-1], want[::-1]):
        l.copy_(dl)
        x.copy_(dx)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
