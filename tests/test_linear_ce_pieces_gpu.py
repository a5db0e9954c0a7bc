"""The loss where its work is cut: the backward's vocabulary in pieces, a packed matrix in pieces, rows of tiles in groups.

How many pieces a case has is read off the workspace that it asks for, so that a change of the limits cannot make one of them unnoticed.
Tolerances: those of the whole cases."""
import ctypes as C

import pytest
import torch

import mixlab_b200
from mixlab_b200 import _lib, ops
from oracle import step_ends
from test_linear_ce_gpu import check_gradients, make, slack

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def workspace_bytes(n, V, D, io, bwd):
    lib = mixlab_b200.lib()
    d = _lib.LinearCeDesc(n, V, D, 8, _lib.MXB_BF16 if io == BF16 else _lib.MXB_F32)
    return (lib.mxb_linear_ce_bwd_workspace_bytes if bwd else lib.mxb_linear_ce_fwd_workspace_bytes)(C.byref(d))


def up(v, to):
    return -(-v // to) * to


# columns of one tile and of several, whole pieces of rows and ragged ones, tiles that are cut and that are not
@pytest.mark.parametrize("n,V,D,io,pieces", [(8192, 60001, 40, BF16, 2), (8000, 90001, 23, BF16, 3), (8192, 50000, 136, BF16, 2), (8192, 60003, 449, BF16, 2),
                                             (30000, 15000, 520, BF16, 2), (4097, 60000, 24, F32, 2), (4097, 30000, 136, F32, 2)])
def test_gradients(n, V, D, io, pieces):
    # (were a piece as wide as the vocabulary's share of fewer pieces, g alone would take more than the whole workspace)
    column = up(n, 256) * 2 * (1 if io == BF16 else 3)
    assert workspace_bytes(n, V, D, io, True) < V / (pieces - 1) * column, "fewer pieces"
    x, w, t, g = make(n, V, D, io)
    lse = ops.linear_cross_entropy(x, w, t)[1]
    a = torch.rand(n, generator=g).cuda()
    got = ops.linear_cross_entropy_backward(x, w, t, lse, a)
    check_gradients(x, w, t, lse, a, None, got, io)
    again = ops.linear_cross_entropy_backward(x, w, t, lse, a)
    assert torch.equal(got["dx"], again["dx"]) and torch.equal(got["dweight"], again["dweight"])


def check_loss(x, w, t, io):
    loss, lse = ops.linear_cross_entropy(x, w, t)
    want_loss, want_lse = step_ends.linear_cross_entropy(x.double(), w.double(), t)
    z, rest = slack(x, w, io)
    off = (lse.double() - want_lse).abs() - (z + rest + 2 * U * want_lse.abs())
    assert torch.isfinite(lse).all() and (off <= 0).all(), off.max()
    off = (loss.double() - want_loss).abs() - (2 * z + rest + 3 * U * (want_lse.abs() + want_loss.abs()))
    assert torch.isfinite(loss).all() and (off <= 0).all(), off.max()


@pytest.mark.parametrize("n,V,D,io", [(33, 140001, 1001, BF16), (40, 50001, 1032, F32), (1100, 90001, 519, F32)])
def test_loss_of_a_packed_matrix_in_pieces(n, V, D, io):
    """Without the packed matrix, whose pieces take at most so much, there is room for less than its rows."""
    row = up(D, 8) * 2 * (1 if io == BF16 else 3)
    assert workspace_bytes(n, V, D, io, False) < V * row, "one piece"
    x, w, t, _ = make(n, V, D, io)
    check_loss(x, w, t, io)


@pytest.mark.parametrize("n,V,D,io", [(3000, 700, 7000, BF16), (4200, 300, 2100, F32)])
def test_rows_of_tiles_in_groups(n, V, D, io):
    """Eight rows of tiles, 2048 tokens, of such wide rows stand together: the others follow in a group of fewer."""
    x, w, t, g = make(n, V, D, io, masked=False)
    check_loss(x, w, t, io)
    lse, a = ops.linear_cross_entropy(x, w, t)[1], torch.rand(n, generator=g).cuda()
    check_gradients(x, w, t, lse, a, None, ops.linear_cross_entropy_backward(x, w, t, lse, a), io)
