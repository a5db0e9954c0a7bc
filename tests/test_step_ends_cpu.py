"""What the operators at the ends of a training step refuse before a device is touched."""
import ctypes as C

import pytest
import torch

import mixlab_b200
from mixlab_b200 import _lib, ops

FAKE, ODD = C.c_void_p(4096), C.c_void_p(4100)


def test_embedding_refusals():
    lib = mixlab_b200.lib()
    desc = lambda **kw: _lib.EmbeddingDesc(*dict(dict(tokens=8, V=16, D=8, token_bytes=4, io=1, out=1, scale=1.0), **kw).values())  # noqa: E731
    fwd = lambda d, tok=FAKE, w=FAKE: lib.mxb_embedding_fwd(C.byref(d), tok, w, FAKE, None)  # noqa: E731
    bwd = lambda d, ws, n, dw=FAKE, tok=FAKE: lib.mxb_embedding_bwd(C.byref(d), tok, FAKE, dw, 0, ws, n, None)  # noqa: E731
    for kw in (dict(tokens=-1), dict(V=0), dict(D=0), dict(token_bytes=2), dict(io=0), dict(out=3)):
        assert fwd(desc(**kw)) == -1 and bwd(desc(**kw), FAKE, 1 << 40) == -1, kw
        assert lib.mxb_embedding_bwd_workspace_bytes(C.byref(desc(**kw))) == 0
    assert fwd(desc(), None) == -1 and fwd(desc(), w=None) == -1 and fwd(desc(tokens=0), None, None) == 0
    assert lib.mxb_embedding_fwd(None, FAKE, FAKE, FAKE, None) == -1
    n = lib.mxb_embedding_bwd_workspace_bytes(C.byref(desc()))
    assert n > 0 and bwd(desc(), None, 0) == -3 and bwd(desc(), FAKE, n - 1) == -3 and bwd(desc(), ODD, n) == -5
    assert bwd(desc(), FAKE, n, dw=None) == -1 and bwd(desc(), FAKE, n, tok=None) == -1
    assert bwd(desc(tokens=1 << 31), FAKE, 1 << 60) == -2


def test_layer_norm_refusals():
    lib = mixlab_b200.lib()
    desc = lambda rows=4, D=64, io=2, res=2, eps=1e-5: _lib.LayerNormDesc(rows, D, io, res, eps)  # noqa: E731
    fwd = lambda d, x=FAKE, resid=None, out=None: lib.mxb_layer_norm_fwd(C.byref(d), resid, x, FAKE, None, out, FAKE, None)  # noqa: E731
    assert fwd(desc(D=16385)) == -2 and fwd(desc(D=0)) == -1 and fwd(desc(io=1, res=2)) == -1 and fwd(desc(eps=-1.0)) == -1
    assert fwd(desc(eps=float("nan"))) == -1 and fwd(desc(), None) == -1 and fwd(desc(rows=0), None) == 0 and fwd(desc(), resid=FAKE) == -1
    bwd = lambda d, ws, n, dx=FAKE: lib.mxb_layer_norm_bwd(C.byref(d), FAKE, FAKE, None, FAKE, dx, FAKE, FAKE, ws, n, None)  # noqa: E731
    n = lib.mxb_layer_norm_bwd_workspace_bytes(C.byref(desc()))
    assert n > 0 and bwd(desc(), None, 0) == -3 and bwd(desc(), FAKE, n - 1) == -3 and bwd(desc(), ODD, n) == -5 and bwd(desc(), FAKE, n, None) == -1


def test_linear_cross_entropy_refusals():
    lib = mixlab_b200.lib()
    desc = lambda **kw: _lib.LinearCeDesc(*dict(dict(rows=8, V=16, D=8, target_bytes=4, io=2), **kw).values())  # noqa: E731
    fwd = lambda d, ws, n, w=FAKE, x=FAKE: lib.mxb_linear_ce_fwd(C.byref(d), x, w, FAKE, FAKE, FAKE, ws, n, None)  # noqa: E731
    bwd = lambda d, ws, n, w=FAKE, dw=FAKE: lib.mxb_linear_ce_bwd(C.byref(d), FAKE, w, FAKE, FAKE, FAKE, None, FAKE, dw, ws, n, None)  # noqa: E731
    for kw, want in [(dict(rows=-1), -1), (dict(V=0), -1), (dict(D=0), -1), (dict(target_bytes=1), -1), (dict(io=3), -1), (dict(rows=1 << 40), -2),
                     (dict(rows=1 << 29, V=1 << 29), -2), (dict(V=(1 << 30) + 8), -2), (dict(D=1 << 30), -2)]:
        assert fwd(desc(**kw), FAKE, 1 << 60) == want and bwd(desc(**kw), FAKE, 1 << 60) == want, kw
        assert lib.mxb_linear_ce_fwd_workspace_bytes(C.byref(desc(**kw))) == 0 == lib.mxb_linear_ce_bwd_workspace_bytes(C.byref(desc(**kw)))
    for call, n in ((fwd, lib.mxb_linear_ce_fwd_workspace_bytes(C.byref(desc()))), (bwd, lib.mxb_linear_ce_bwd_workspace_bytes(C.byref(desc())))):
        assert n > 0 and call(desc(), None, 0) == -3 and call(desc(), FAKE, n - 1) == -3 and call(desc(), ODD, n) == -5
        assert call(desc(), FAKE, n, w=C.c_void_p(4098)) == -5 and call(desc(), FAKE, n, w=None) == -1
    assert lib.mxb_linear_ce_bwd_workspace_bytes(C.byref(desc(rows=0))) > 0  # (nothing is divided by the rows)
    assert fwd(desc(rows=0), None, 0, x=None) == 0 and bwd(desc(), FAKE, 1 << 40, dw=None) == -1


def test_the_backward_keeps_a_piece_of_the_vocabulary():
    """Its workspace is far below the logits' size, whatever the vocabulary."""
    lib = mixlab_b200.lib()
    for V in (50001, 400001):
        d = _lib.LinearCeDesc(32768, V, 1024, 8, _lib.MXB_BF16)
        assert lib.mxb_linear_ce_bwd_workspace_bytes(C.byref(d)) < (1 << 30)
    d = _lib.LinearCeDesc(1 << 21, 50001, 64, 8, _lib.MXB_BF16)  # (so many tokens that a piece is one tile)
    assert lib.mxb_linear_ce_bwd_workspace_bytes(C.byref(d)) < (3 << 30)


def test_cpu_tensors_are_refused():
    t, tok = torch.zeros(4, 64), torch.zeros(4).long()
    for call in (lambda: ops.embedding(tok, t), lambda: ops.embedding_backward(tok, t, 9), lambda: ops.layer_norm(t, torch.ones(64)),
                 lambda: ops.layer_norm_backward(t, torch.ones(64), t), lambda: ops.linear_cross_entropy(t, torch.zeros(9, 64), tok),
                 lambda: ops.linear_cross_entropy_backward(t, torch.zeros(9, 64), tok, torch.zeros(4), torch.zeros(4))):
        with pytest.raises(ValueError, match="CUDA tensors only"):
            call()


F32, BF16 = "float32", "bfloat16"
_OPERANDS = {  # operator: its tensor operands (shape, dtype), the other arguments; the first settles what the others are held to
    "embedding": (dict(weight=((11, 24), BF16), tokens=((2, 6), "int64")), {}),
    "embedding_backward": (dict(d_out=((2, 6, 24), BF16), tokens=((2, 6), "int32"), dweight=((11, 24), F32)), dict(V=11)),
    "layer_norm": (dict(x=((2, 6, 24), BF16), weight=((24,), F32), bias=((24,), F32), resid=((2, 6, 24), F32)), {}),
    "layer_norm_backward": (dict(x=((2, 6, 24), F32), weight=((24,), F32), dn=((2, 6, 24), BF16), d_resid=((2, 6, 24), F32)), {}),
    "linear_cross_entropy": (dict(x=((2, 6, 24), BF16), weight=((11, 24), BF16), targets=((2, 6), "int64")), {}),
    "linear_cross_entropy_backward": (dict(x=((2, 6, 24), BF16), weight=((11, 24), BF16), targets=((2, 6), "int32"), lse=((2, 6), F32),
                                           d_loss=((2, 6), F32), d_lse=((2, 6), F32)), {}),
}


@pytest.mark.parametrize("op", _OPERANDS)
def test_every_operand_is_checked(op):
    from torch._subclasses.fake_tensor import FakeTensorMode
    specs, rest = _OPERANDS[op]
    first = next(iter(specs))

    def refused(name, error, make):
        args = {n: torch.empty(shape, dtype=getattr(torch, dt), device="cuda:0") for n, (shape, dt) in specs.items()}
        args[name] = make(*specs[name])
        with pytest.raises(error) as e:
            getattr(ops, op)(**args, **rest)
        return str(e.value)

    with FakeTensorMode():
        for name, (shape, dt) in specs.items():
            own = getattr(torch, dt)
            refused(name, ValueError, lambda s, _: torch.empty(s, dtype=own, device="cpu"))
            refused(name, TypeError, lambda s, _: torch.empty(s, dtype=torch.float16, device="cuda:0"))
            msg = refused(name, ValueError, lambda s, _: torch.empty(*s[:-1], 2 * s[-1], dtype=own, device="cuda:0")[..., ::2])
            assert "contiguous" in msg, (name, msg)
            if name != first and (op, name) != ("embedding", "tokens") and (op[:6], name) != ("linear", "weight"):
                refused(name, ValueError, lambda s, _: torch.empty(s[0] + 1, *s[1:], dtype=own, device="cuda:0"))
            if name != first:
                assert "cuda:1" in refused(name, ValueError, lambda s, _: torch.empty(s, dtype=own, device="cuda:1"))


def test_types_that_do_not_go_together():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, dt=torch.float32: torch.empty(*s, dtype=dt, device="cuda:0")  # noqa: E731
        half, w = torch.bfloat16, e(8)
        for call in (lambda: ops.layer_norm(e(4, 8, dt=half), w, dtype=torch.float32), lambda: ops.layer_norm(e(4, 8), w, resid=e(4, 8, dt=half)),
                     lambda: ops.layer_norm(e(4, 8), w, resid=e(4, 8), dtype=half), lambda: ops.layer_norm(e(4, 8), w, dtype=torch.float16),
                     lambda: ops.layer_norm_backward(e(4, 8, dt=half), w, e(4, 8)), lambda: ops.embedding(e(4, dt=torch.long), e(9, 8), dtype=torch.int8),
                     lambda: ops.embedding(e(4, dt=torch.long), e(9, 8), dtype="float32"),
                     lambda: ops.embedding_backward(e(4, dt=torch.long), e(4, 8), 9, dtype=half, dweight=e(9, 8))):
            with pytest.raises(TypeError):
                call()
        with pytest.raises(ValueError):
            ops.embedding_backward(e(4, dt=torch.long), e(4, 8), 0)
        with pytest.raises(ValueError, match="beyond 32 bits"):
            ops.embedding_backward(e(4, dt=torch.long), e(4, 8), 1 << 32)
