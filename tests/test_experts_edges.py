"""Routed experts: argument checks of the C entry points and Python functions beyond test_experts.py (no GPU: every call
below is refused before any CUDA call)."""
from test_experts import P, lib


def test_dx_rows_arguments():
    _l, L = lib()
    bad, no = _l.KMC_ERR_INVALID, _l.KMC_ERR_UNSUPPORTED

    def call(dy=P, w=P, off=P, slot=P, rows=4, choices=2, E=4, n=8, d=16, dtype=1, dx=P, ws=P, nb=1 << 20, err=P):
        return L.kmc_expert_matmul_dx_rows(dy, w, off, slot, rows, choices, E, n, d, dtype, dx, ws, nb, err, None)

    assert call(rows=-1) == bad and call(choices=0) == bad and call(E=0) == bad and call(n=0) == bad and call(d=0) == bad
    assert call(dtype=0) == bad and call(dtype=3) == bad
    assert call(rows=2 ** 30, choices=2) == no and call(E=4097) == no and call(d=(1 << 20) + 1) == no
    for missing in ("dy", "w", "off", "slot", "dx", "err"):
        assert call(**{missing: None}) == bad and b"null" in L.kmc_last_error()
    need = L.kmc_expert_dx_rows_bytes(P, P, 4, 2, 4, 8, 16)
    assert need == 4 * 2 * 16 * 4 and call(nb=need - 1) == bad and b"workspace" in L.kmc_last_error()
    assert call(ws=None) == bad
    assert L.kmc_expert_dx_rows_bytes(P, P, 4, 1, 4, 8, 16) == 256                  # 16-bit: nothing is summed
    assert L.kmc_expert_dx_rows_bytes(P, P, 4, 2, 4, 8, 15) == 512 + 4 * 8 * 16 * 2  # and W's rows padded
    assert call(rows=0, dy=None, slot=None, dx=None, ws=None, nb=0) == _l.KMC_OK


def test_combine_grad_slots_arguments():
    _l, L = lib()
    bad, no = _l.KMC_ERR_INVALID, _l.KMC_ERR_UNSUPPORTED

    def call(dout=P, y=P, dtype=0, rows=4, choices=2, width=8, slot=P, dy=P, dw=P, ws=P, nb=32):
        return L.kmc_combine_grad_slots(dout, y, dtype, rows, choices, width, slot, None, dy, dw, ws, nb, None)

    assert call(dtype=3) == bad and call(rows=-1) == bad and call(choices=0) == bad and call(width=0) == bad
    assert call(rows=2 ** 31, choices=1) == no and call(width=(1 << 20) + 1) == no
    for missing in ("dout", "y", "slot", "dy"):
        assert call(**{missing: None}) == bad and b"null" in L.kmc_last_error()
    assert L.kmc_combine_bytes(4, 2) == 32 and L.kmc_combine_bytes(0, 2) == 0 and L.kmc_combine_bytes(2 ** 31, 1) == 0
    assert call(nb=31) == bad and b"workspace" in L.kmc_last_error() and call(ws=None) == bad
    assert call(rows=0, dout=None, y=None, slot=None, dy=None, ws=None, nb=0) == _l.KMC_OK


def test_arguments_of_other_types():
    """What is no tensor, and no plan, is a ValueError like any other bad argument."""
    import pytest
    import torch

    from mlx_kmeans_b200 import RowGroups, combine_rows, combine_rows_grad, expert_matmul, expert_matmul_grad, route
    t, w = torch.zeros(4, 8), torch.zeros(8, 4, 8)
    ids = torch.zeros(4, 2, dtype=torch.int32)
    g = RowGroups(torch.zeros(9, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), ids)
    plans = (None, g[:2], ids, RowGroups(None, g.rows, g.slot), "offsets")
    calls = [lambda: route(t, 2, bias=[0.0] * 8), lambda: route(t, 2, mask=[True] * 4), lambda: route(t, 2, bias=0.0),
             lambda: combine_rows(t, g, [1.0]), lambda: combine_rows_grad(t, t, g, 1.0)]
    for p in plans:
        calls += [lambda p=p: expert_matmul(t, w, p), lambda p=p: expert_matmul_grad(t, t, w, p),
                  lambda p=p: combine_rows(t, p), lambda p=p: combine_rows_grad(t, t, p),
                  lambda p=p: expert_matmul(t.clone().requires_grad_(True), w, p)]
    for f in calls:
        with pytest.raises(ValueError, match="CUDA tensor|RowGroups"):
            f()


def test_workspaces_off_their_alignment():
    """A workspace that does not start where the header says is refused: its vectors would be read off their boundary."""
    _l, L = lib()
    bad, big = _l.KMC_ERR_INVALID, 1 << 20
    x = P + 2                                                  # rows off 16 bytes: copied to the workspace
    for at in (P + 4, P + 16, P + 128):
        for rc in (L.kmc_expert_matmul(x, 400, 16, None, P, P, 400, 4, 8, 16, 1, P, at, big, P, None),
                   L.kmc_expert_matmul_dx(x, P, P, 400, 4, 8, 16, 1, P, at, big, P, None),
                   L.kmc_expert_matmul_dw(x, P, 400, 16, None, P, 400, 4, 8, 16, 1, P, at, big, P, None),
                   L.kmc_expert_matmul_dx_rows(P, P, P, P, 4, 2, 4, 8, 16, 1, P, at, big, P, None)):
            assert rc == bad and b"256" in L.kmc_last_error()
    assert L.kmc_group_rows(P, 1 << 19, 2, 256, P, P, P, P + 2, big, None) == bad and b"4-byte" in L.kmc_last_error()
    assert L.kmc_combine_grad_slots(P, P, 0, 4, 2, 8, P, None, P, P, P + 2, 32, None) == bad and b"4-byte" in L.kmc_last_error()
