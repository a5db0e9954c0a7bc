"""The workspaces of the ends of a training step: any base on 16 bytes, nothing written outside."""
import ctypes as C

import pytest
import torch

import mixlab_b200
from mixlab_b200 import _lib, ops

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
BASES = [0, 16, 48, 144, 240]  # from a multiple of 512 on


def p(t):
    return C.c_void_p(t.data_ptr())


def in_place(need, base, call):
    """call(workspace, bytes) on a workspace of exactly the bytes asked for, with other memory on either side."""
    flat = torch.full((need + 1024,), 0x5A, dtype=torch.uint8, device="cuda")
    assert flat.data_ptr() % 512 == 0
    lo = 512 + base
    assert call(p(flat[lo:]), need, C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    assert (flat[:lo] == 0x5A).all() and (flat[lo + need:] == 0x5A).all()


def rnd(g, *shape):
    return torch.randn(*shape, generator=g)


@pytest.mark.parametrize("n,V,D", [(700, 37, 24), (5000, 300, 16), (66000, 40, 8), (700, 37, 23)])
@pytest.mark.parametrize("base", BASES)
def test_embedding_gradient(base, n, V, D):
    lib, g = mixlab_b200.lib(), torch.Generator().manual_seed(n)
    tok, d_out = torch.randint(-1, V, (n,), generator=g).cuda(), rnd(g, n, D).cuda()
    want, dw = ops.embedding_backward(tok, d_out, V), torch.empty(V, D, device="cuda")
    d = _lib.EmbeddingDesc(n, V, D, 8, _lib.MXB_F32, _lib.MXB_F32, 1.0)
    in_place(lib.mxb_embedding_bwd_workspace_bytes(C.byref(d)), base,
             lambda ws, size, st: lib.mxb_embedding_bwd(C.byref(d), p(tok), p(d_out), p(dw), 0, ws, size, st))
    assert torch.equal(dw, want)


@pytest.mark.parametrize("n,D", [(300, 64), (4001, 40), (37, 4104), (300, 63)])
@pytest.mark.parametrize("base", BASES)
def test_layer_norm_gradients(base, n, D):
    lib, g = mixlab_b200.lib(), torch.Generator().manual_seed(n)
    x, w, dn = rnd(g, n, D).cuda(), rnd(g, D).cuda(), rnd(g, n, D).cuda()
    want = ops.layer_norm_backward(x, w, dn)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    d = _lib.LayerNormDesc(n, D, _lib.MXB_F32, _lib.MXB_F32, 1e-5)
    in_place(lib.mxb_layer_norm_bwd_workspace_bytes(C.byref(d)), base,
             lambda ws, size, st: lib.mxb_layer_norm_bwd(C.byref(d), p(x), p(w), None, p(dn), p(dx), p(dw), p(db), ws, size, st))
    assert torch.equal(dx, want["dx"]) and torch.equal(dw, want["dweight"]) and torch.equal(db, want["dbias"])


@pytest.mark.parametrize("io,n,V,D", [(BF16, 300, 600, 24), (BF16, 1100, 600, 23), (F32, 300, 600, 24)])
@pytest.mark.parametrize("base", BASES)
def test_loss(base, io, n, V, D):
    lib, g = mixlab_b200.lib(), torch.Generator().manual_seed(n)
    x, w, t, a = rnd(g, n, D).to(io).cuda(), rnd(g, V, D).to(io).cuda(), torch.randint(-1, V, (n,), generator=g).cuda(), torch.rand(n, generator=g).cuda()
    want_loss, want_lse = ops.linear_cross_entropy(x, w, t)
    want = ops.linear_cross_entropy_backward(x, w, t, want_lse, a)
    loss, lse, dx, dw = torch.empty_like(a), torch.empty_like(a), torch.empty_like(x), torch.empty_like(w)
    d = _lib.LinearCeDesc(n, V, D, 8, _lib.MXB_BF16 if io == BF16 else _lib.MXB_F32)
    in_place(lib.mxb_linear_ce_fwd_workspace_bytes(C.byref(d)), base,
             lambda ws, size, st: lib.mxb_linear_ce_fwd(C.byref(d), p(x), p(w), p(t), p(loss), p(lse), ws, size, st))
    in_place(lib.mxb_linear_ce_bwd_workspace_bytes(C.byref(d)), base,
             lambda ws, size, st: lib.mxb_linear_ce_bwd(C.byref(d), p(x), p(w), p(t), p(lse), p(a), None, p(dx), p(dw), ws, size, st))
    assert torch.equal(loss, want_loss) and torch.equal(lse, want_lse) and torch.equal(dx, want["dx"]) and torch.equal(dw, want["dweight"])
