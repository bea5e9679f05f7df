"""Routed experts: the argument checks of the C entry points and of the Python functions (no GPU: every call below is
refused before any CUDA call)."""
import pytest
import torch

P = 4096          # a nonzero stand-in for device pointers, never dereferenced


def lib():
    from mlx_kmeans_b200 import _lib
    return _lib, _lib.load()


def test_route_arguments():
    _l, L = lib()

    def call(dtype=1, rows=4, experts=8, stride=8, choices=2, groups=1, top=1, flags=0, logits=P, ids=P):
        return L.kmc_route(logits, dtype, rows, experts, stride, None, None, choices, groups, top, 1.0, flags, ids, P, None)

    bad, no = _l.KMC_ERR_INVALID, _l.KMC_ERR_UNSUPPORTED
    assert call(dtype=3) == bad and b"dtype" in L.kmc_last_error()
    assert call(rows=-1) == bad and call(experts=0) == bad and call(choices=0) == bad and call(choices=9) == bad
    assert call(stride=7) == bad and call(flags=4) == bad
    assert call(groups=3) == bad and b"groups" in L.kmc_last_error()
    assert call(groups=0) == bad and call(groups=4, top=5) == bad and call(groups=4, top=0) == bad
    assert call(experts=128, stride=128, groups=64) == bad
    assert call(experts=1025, stride=1025) == no and call(experts=64, stride=64, choices=33) == no
    assert call(rows=2 ** 31, choices=1) == no and b"pairs" in L.kmc_last_error()
    assert call(logits=None) == bad and b"null" in L.kmc_last_error()
    assert call(ids=None) == bad
    assert call(rows=0, logits=None, ids=None) == _l.KMC_OK
    assert L.kmc_route_grad(P, P, 0, 4, 8, 8, None, 2, 1.0, 0, P, None) == bad
    assert L.kmc_route_grad(P, P, 0, 4, 8, 8, P, 9, 1.0, 0, P, None) == bad


def test_group_arguments():
    _l, L = lib()
    bad, no = _l.KMC_ERR_INVALID, _l.KMC_ERR_UNSUPPORTED

    def call(rows=10, choices=2, experts=4, ids=P, offsets=P, ws=None, nb=0):
        return L.kmc_group_rows(ids, rows, choices, experts, offsets, P, P, ws, nb, None)

    assert call(rows=-1) == bad and call(choices=0) == bad and call(experts=0) == bad
    assert call(experts=4097) == no and call(rows=2 ** 31) == no
    assert call(ids=None) == bad and call(offsets=None) == bad
    assert L.kmc_group_bytes(100, 64) == 0
    need = L.kmc_group_bytes(1 << 20, 256)
    assert need > 0 and call(rows=1 << 19, experts=256, ws=P, nb=need - 1) == bad and b"workspace" in L.kmc_last_error()
    assert call(rows=1 << 19, experts=256) == bad


def test_expert_arguments():
    _l, L = lib()
    bad, no = _l.KMC_ERR_INVALID, _l.KMC_ERR_UNSUPPORTED

    def fwd(x=P, x_rows=4, ldx=16, rows=P, w=P, off=P, pairs=8, E=4, n=8, d=16, dtype=1, y=P, err=P):
        return L.kmc_expert_matmul(x, x_rows, ldx, rows, w, off, pairs, E, n, d, dtype, y, None, 0, err, None)

    assert fwd(dtype=0) == bad and fwd(ldx=15) == bad and fwd(n=0) == bad and fwd(d=0) == bad and fwd(E=0) == bad
    assert fwd(pairs=-1) == bad and fwd(E=4097) == no and fwd(n=(1 << 20) + 1) == no and fwd(pairs=2 ** 31) == no
    assert fwd(pairs=2 ** 31 - 1024) == no and b"positions" in L.kmc_last_error()
    assert fwd(w=None) == bad and fwd(off=None) == bad and fwd(err=None) == bad and fwd(y=None) == bad and fwd(x=None) == bad
    assert fwd(rows=None) == bad and b"grouped" in L.kmc_last_error()
    assert L.kmc_expert_matmul_dx(P, None, P, 8, 4, 8, 16, 1, P, None, 0, P, None) == bad
    assert L.kmc_expert_matmul_dx(P, P, P, 8, 4, 8, 16, 0, P, None, 0, P, None) == bad
    assert L.kmc_expert_matmul_dw(P, P, 4, 16, P, P, 8, 4, 8, 16, 1, None, None, 0, P, None) == bad
    assert L.kmc_expert_matmul_dw(P, P, 4, 15, P, P, 8, 4, 8, 16, 1, P, None, 0, P, None) == bad


def test_combine_arguments():
    _l, L = lib()
    bad, no = _l.KMC_ERR_INVALID, _l.KMC_ERR_UNSUPPORTED
    assert L.kmc_combine(P, 3, 4, 2, 8, P, None, P, None) == bad
    assert L.kmc_combine(P, 0, 4, 0, 8, P, None, P, None) == bad
    assert L.kmc_combine(P, 0, 4, 2, 0, P, None, P, None) == bad
    assert L.kmc_combine(P, 0, 4, 2, (1 << 20) + 1, P, None, P, None) == no
    assert L.kmc_combine(None, 0, 4, 2, 8, P, None, P, None) == bad
    assert L.kmc_combine_grad(P, P, 0, 4, 2, 8, P, None, None, P, None, None) == bad
    assert L.kmc_combine_grad(P, None, 0, 4, 2, 8, P, P, P, P, P, None) == bad


def test_python_functions_want_cuda_tensors():
    from mlx_kmeans_b200 import (RowGroups, combine_rows, combine_rows_grad, expert_matmul, expert_matmul_grad,
                                 group_rows, route, route_grad)
    t = torch.zeros(4, 8)
    ids = torch.zeros(4, 2, dtype=torch.int32)
    g = RowGroups(torch.zeros(9, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), ids)
    for f in (lambda: route(t, 2), lambda: route_grad(t[:, :2], t, ids), lambda: group_rows(ids, 8),
              lambda: expert_matmul(t, torch.zeros(8, 4, 8), g), lambda: combine_rows(t, g),
              lambda: expert_matmul_grad(t, t, torch.zeros(8, 4, 8), g), lambda: combine_rows_grad(t, t, g),
              lambda: route([[1.0]], 1)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            f()


@pytest.mark.gpu
def test_python_refusals(cuda_device):
    from mlx_kmeans_b200 import RowGroups, combine_rows, combine_rows_grad, expert_matmul, expert_matmul_grad, group_rows, route, route_grad
    l = torch.zeros(6, 8, device="cuda")
    ids, w = route(l, 2)
    g = group_rows(ids, 8)
    half = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    x, m, y = half(6, 16), half(8, 4, 16), half(12, 4)
    bad = [
        lambda: route(l.double(), 2), lambda: route(l[0], 2), lambda: route(l, 9), lambda: route(l, 0),
        lambda: route(l, 2, score="tanh"), lambda: route(l, 2, bias=torch.zeros(7, device="cuda")),
        lambda: route(l, 2, bias=half(8)), lambda: route(l, 2, mask=torch.ones(5, dtype=torch.bool, device="cuda")),
        lambda: route(l, 2, mask=torch.ones(6, device="cuda")), lambda: route(l, 2, groups=3),
        lambda: route(l, 2, groups=4, top_groups=5), lambda: route(torch.zeros(2, 1025, device="cuda"), 2),
        lambda: route_grad(w, l, ids[:, :1]), lambda: route_grad(w[:5], l, ids[:5]),
        lambda: group_rows(ids.long(), 8), lambda: group_rows(ids, 0), lambda: group_rows(ids, 4097),
        lambda: group_rows(ids.reshape(1, 6, 2), 8),
        lambda: expert_matmul(x.float(), m.float(), g), lambda: expert_matmul(x.half(), m, g),
        lambda: expert_matmul(x[:5], m, g), lambda: expert_matmul(x, m[:7], g), lambda: expert_matmul(x[:, :15], m, g),
        lambda: expert_matmul(x, m, g, gather=False), lambda: expert_matmul_grad(y[:11], x, m, g),
        lambda: expert_matmul(x, m, RowGroups(g.offsets, g.rows[:11], g.slot)),
        lambda: combine_rows(y[:11], g, w), lambda: combine_rows(y, g, w[:, :1]), lambda: combine_rows(y, g, w.double()),
        lambda: combine_rows(y.double(), g, w), lambda: combine_rows_grad(x, y, g, w),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
