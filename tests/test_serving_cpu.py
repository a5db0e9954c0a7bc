"""What the serving operators refuse before a device is touched, and their oracle's own consistency."""
import ctypes as C

import pytest
import torch

import mixlab_b200
from mixlab_b200 import _lib, ops
from oracle import mamba3, mamba3_block, serving

FAKE = C.c_void_p(4096)
ODD = C.c_void_p(4100)


def _serve(**kw):
    d = dict(rows=8, S=2, slots=4, D=64, N=16, G=1, nheads=1, io_dtype=_lib.MXB_BF16, flags=0)
    d.update(kw)
    return _lib.Mamba3ServeDesc(*d.values())


def _prefill(d, state=None, cu=FAKE, x=FAKE, ws=None, n=0):
    s = _lib.Mamba3StatePointers(*([4096] * 4)) if state is None else state
    return mixlab_b200.lib().mxb_mamba3_prefill(C.byref(d), x, *([FAKE] * 6), cu, None, None, C.byref(s), FAKE, ws, n, None)


def test_scan_refusals():
    for kw, want in [(dict(S=-1), -1), (dict(rows=-1), -1), (dict(io_dtype=3), -1), (dict(nheads=-1), -1), (dict(N=15), -2), (dict(N=258), -2),
                     (dict(G=3), -2), (dict(nheads=5), -2), (dict(G=4, nheads=2), -2), (dict(D=1 << 17), -2)]:
        assert _prefill(_serve(**kw)) == want, kw
        assert mixlab_b200.lib().mxb_mamba3_prefill_workspace_bytes(C.byref(_serve(**kw))) == 0
    assert _prefill(_serve(), x=None) == -1 and _prefill(_serve(), cu=None) == -1
    assert _prefill(_serve(), state=_lib.Mamba3StatePointers(4096, 4096, 4096, None)) == -1
    assert _prefill(_serve(), state=_lib.Mamba3StatePointers(4100, 4096, 4096, 4096)) == -5
    assert _prefill(_serve(rows=0)) == 0 and _prefill(_serve(S=0)) == 0  # nothing to do
    long = _serve(rows=100000)  # one head: the time axis is cut, which needs a workspace
    n = mixlab_b200.lib().mxb_mamba3_prefill_workspace_bytes(C.byref(long))
    assert n > 0 and _prefill(long) == -3 and _prefill(long, ws=FAKE, n=n - 1) == -3 and _prefill(long, ws=ODD, n=n) == -5
    s = _lib.Mamba3StatePointers(*([4096] * 4))
    step = lambda d, x=FAKE: mixlab_b200.lib().mxb_mamba3_decode_step(C.byref(d), C.byref(s), x, *([FAKE] * 6), None, FAKE, None)  # noqa: E731
    assert step(_serve(N=3)) == -2 and step(_serve(), None) == -1 and step(_serve(S=0)) == 0


def test_convolution_and_norm_refusals():
    lib = mixlab_b200.lib()
    conv = lambda K=4, act=0, io=2, rows=8: _lib.ShortConvDesc(rows, 2, 4, 64, K, io, act, K, 1)  # noqa: E731
    run = lambda d, x=FAKE, cu=FAKE: lib.mxb_short_conv_prefill(C.byref(d), x, FAKE, None, cu, None, None, FAKE, FAKE, None)  # noqa: E731
    assert run(conv(5)) == -2 and run(conv(0)) == -1 and run(conv(act=2)) == -1 and run(conv(io=0)) == -1
    assert run(conv(), x=None) == -1 and run(conv(), cu=None) == -1 and run(conv(rows=0)) == 0
    norm = lambda D=64, io=2, res=2, eps=1e-5, rows=4: _lib.ResidualNormDesc(rows, D, io, res, eps)  # noqa: E731
    fwd = lambda d, y=FAKE: lib.mxb_residual_norm_fwd(C.byref(d), FAKE, y, FAKE, None, None, None, FAKE, FAKE, None)  # noqa: E731
    assert fwd(norm(16385)) == -2 and fwd(norm(0)) == -1 and fwd(norm(io=1, res=2)) == -1 and fwd(norm(eps=-1.0)) == -1
    assert fwd(norm(eps=float("nan"))) == -1 and fwd(norm(), None) == -1 and fwd(norm(rows=0)) == 0
    bwd = lambda d, ws, n: lib.mxb_residual_norm_bwd(C.byref(d), *([FAKE] * 8), *([FAKE] * 6), ws, n, None)  # noqa: E731
    n = lib.mxb_residual_norm_workspace_bytes(C.byref(norm()))
    assert n > 0 and bwd(norm(), None, 0) == -3 and bwd(norm(), FAKE, n - 1) == -3 and bwd(norm(), ODD, n) == -5


def test_cpu_tensors_are_refused():
    t = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        ops.residual_norm(t, t, torch.ones(64))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        ops.short_conv_step(torch.zeros(4, 3, 64), t, torch.zeros(64, 4))
    s = ops.mamba3_state(4, 64, 16, 1, nheads=1, dtype=torch.float32, device="cpu")
    b, per = torch.zeros(4, 1, 16), torch.zeros(4, 1)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        ops.mamba3_decode_step(s, t, per, per, per, torch.zeros(1), b, b, nheads=1)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        ops.mamba3_prefill(t, per, per, per, torch.zeros(1), b, b, torch.zeros(2).int(), s, nheads=1)


@pytest.mark.parametrize("nheads", [0, 2])
def test_oracle_is_the_scan(nheads):
    """A sequence from nothing is the scan's; cut anywhere it is the same."""
    D, N, G, T = 8, 6, 2, 11
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    per = (T, nheads or D)
    x, dt, lam, theta = r(T, D), r(*per), r(*per), r(*(per if nheads else per + (N // 2,)))
    a_log, b, c = r(*((nheads,) if nheads else (D, N))), r(T, G, N), r(T, G, N)
    wide = (lambda t: t.repeat_interleave(D // nheads, -1)) if nheads else (lambda t: t)
    y_want, h_want = mamba3.scan_forward(x[None], wide(dt)[None], wide(lam)[None], wide(theta)[None, ..., None].expand(1, T, D, N // 2) if nheads else theta[None],
                                         wide(a_log)[:, None].expand(D, N) if nheads else a_log, b[None], c[None], return_state=True)
    for cut in (0, 1, 5):
        state, ys = serving.fresh_mamba3_state(D, N, G, nheads), []
        for q in (slice(0, cut), slice(cut, T)):
            y, state = serving.mamba3_rows(state, x[q], dt[q], lam[q], theta[q], a_log, b[q], c[q], nheads)
            ys.append(y)
        assert torch.allclose(torch.cat(ys), y_want[0], rtol=1e-12, atol=1e-12) and torch.allclose(state[0], h_want[0], rtol=1e-12, atol=1e-12)
    w, pool = r(D, 3), torch.zeros(1, 2, D, dtype=torch.float64)
    parts = [serving.short_conv(pool, x[q], w, None, [len(x[q])], [0], [i > 0], False) for i, q in enumerate((slice(0, 1), slice(1, T)))]
    assert torch.allclose(torch.cat(parts), mamba3_block.depthwise_conv(x[None], w)[0])


@pytest.mark.parametrize("nheads,D,N", [(32, 2048, 128), (0, 448, 16), (2, 256, 64)])
def test_scratch_of_many_sequences(nheads, D, N):
    """What a cut needs goes by the sequences that can be longer than a segment, not by all: many short ones beside a long one
    take no state's room each.  (Step by step: nothing; in chunks their scores and scalars, a chunk's 2 KB a head and 20 KB; heads
    of several slabs 8 bytes each.)"""
    need = lambda S, flags: mixlab_b200.lib().mxb_mamba3_prefill_workspace_bytes(  # noqa: E731
        C.byref(_serve(rows=32768, S=S, slots=S, D=D, N=N, nheads=nheads, flags=flags)))
    walk = _lib.MXB_MAMBA3_RECURRENT_KERNELS
    small, large = 512, 4096  # (more than the segments that there can be)
    assert need(small, walk) > D * N * 4  # a cut it is
    assert need(large, walk) - need(small, walk) <= 8 * nheads * (large - small) * (nheads > 0 and D // nheads > 64) + 256
    assert need(large, 0) - need(small, 0) <= (2048 * nheads + 20480 + 8 * nheads) * (large - small) + 1024


def test_sizes_near_32_bits_are_refused():
    most = (1 << 31) - 1
    conv = lambda rows=8, S=2, D=64: _lib.ShortConvDesc(rows, S, 4, D, 4, 2, 0, 4, 1)  # noqa: E731
    lib = mixlab_b200.lib()
    assert _prefill(_serve(rows=most)) == -2 and mixlab_b200.lib().mxb_mamba3_prefill_workspace_bytes(C.byref(_serve(rows=most))) == 0
    for d in (conv(rows=most), conv(S=most), conv(D=most)):
        assert lib.mxb_short_conv_prefill(C.byref(d), FAKE, FAKE, None, FAKE, None, None, FAKE, FAKE, None) == -2
        assert lib.mxb_short_conv_step(C.byref(d), FAKE, FAKE, FAKE, None, None, FAKE, None) == -2
