"""The residual stage against the float64 oracle: forward, every gradient, its refusals.

Tolerances: float32 results carry a few roundings of 2^-24 and one 2^-24 more for every doubling of the sums' length (pairs, by
lanes): 1e-6 covers 16; column sums over up to 3000 rows one after the other in a CTA, at most rows / CTAs x 2^-24 more: 1e-5.
bf16 results are rounded once: 2^-8."""
import ctypes as C

import pytest
import torch

from mixlab_b200 import _lib, ops
from oracle import serving
from util import assert_close

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TOL = {F32: 1e-6, BF16: 2.0 ** -8}


def inputs(rows, D, io, res, post, gate, scale, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(resid=(2 * r(rows, D)).to(res), y=r(rows, D).to(io), norm=1 + 0.1 * r(D), post_norm=1 + 0.1 * r(D) if post else None,
                z=r(rows, D).to(io) if gate else None, scale=0.5 + 0.1 * r(D) if scale else None, d=r(rows, D).to(res), dn=r(rows, D).to(io))


def on(a, f):
    return {k: None if v is None else f(v) for k, v in a.items()}


def call(a, eps=1e-5):
    return ops.residual_norm(a["resid"], a["y"], a["norm"], post_norm=a["post_norm"], z=a["z"], scale=a["scale"], eps=eps)


def back(a, d=True, eps=1e-5):
    return ops.residual_norm_backward(a["resid"], a["y"], a["norm"], a["d"] if d else None, a["dn"], post_norm=a["post_norm"], z=a["z"],
                                      scale=a["scale"], eps=eps)


def oracle_grads(a, d=True, eps=1e-5):
    """resid is the forward's result here: d reaches it directly and through its norm."""
    a = on(a, lambda t: t.double().requires_grad_())
    stream, n = serving.residual_norm(a["resid"], torch.zeros_like(a["resid"]), a["norm"], eps=eps)
    dr, dnorm = torch.autograd.grad((n * a["dn"]).sum(), (a["resid"], a["norm"]))
    dr = dr + a["d"] if d else dr
    out = serving.residual_norm(torch.zeros_like(a["resid"]), a["y"], a["norm"], a["post_norm"], a["z"], a["scale"], eps)[0]
    names = [k for k in ("y", "z", "post_norm", "scale") if a[k] is not None]
    g = dict(zip(names, torch.autograd.grad((out * dr.detach()).sum(), [a[k] for k in names])))
    return dict(d_resid=dr.detach(), dy=g["y"], dz=g.get("z"), dnorm=dnorm, dpost_norm=g.get("post_norm"), dscale=g.get("scale"))


OPTIONS = [(False, False, False), (True, False, False), (False, True, True), (True, True, True), (True, False, True)]
SIZES = [(1, 1), (3, 7), (5, 64), (1, 449), (700, 40), (33, 1000), (9, 2048), (300, 2600), (400, 4096), (2, 5000), (3, 8200), (2, 16384)]


@pytest.mark.parametrize("io,res", [(F32, F32), (BF16, F32), (BF16, BF16)], ids=["f32", "bf16 on f32", "bf16"])
@pytest.mark.parametrize("rows,D", SIZES)
def test_forward_and_gradients(rows, D, io, res):
    for n, (post, gate, scale) in enumerate(OPTIONS):
        a = inputs(rows, D, io, res, post, gate, scale, n)
        dev = on(a, lambda t: t.cuda())
        r, nn = call(dev)
        f = on(a, lambda t: t.double())
        r_want, n_want = serving.residual_norm(f["resid"], f["y"], f["norm"], f["post_norm"], f["z"], f["scale"])
        assert_close(r.cpu(), r_want, TOL[res], "resid")
        assert_close(nn.cpu(), n_want, TOL[io], "n")
        for d in (True, False):
            got, want = back(dev, d), oracle_grads(a, d)
            if D == 1:
                # Of one column the norm is a sign: k (t - r k^2 t r) = k t (1 - k^2 r^2), k^2 r^2 = 1 - eps k^2, cancels down to
                # eps k^3 t, below the half steps of its two terms (three roundings of k^2 r^2 of 2^-24, and rsqrt's two): 8 x 2^-24
                # of k t = dn norm / |r| is what is left to demand, and likewise of whatever is made of it.
                size = (f["dn"] * f["norm"] / f["resid"].abs()).abs()
                assert ((got["d_resid"].cpu().double() - want["d_resid"]).abs() <= 8 * 2.0 ** -24 * size + TOL[res] * want["d_resid"].abs()).all()
                continue
            for k, w in want.items():
                if w is None:
                    assert got[k] is None
                else:
                    assert_close(got[k].cpu(), w, TOL[io] if k in ("dy", "dz") else TOL[res] if k == "d_resid" else 1e-5, k)


def test_gradients_against_differences():
    """The formulas themselves: differences of the oracle in float64 along random directions.  A difference over 2e-5 is off by
    the third derivative times 4e-10 / 6 and by rounding, 1e-16 x the loss (about 100) / 2e-5: 1e-7 is far above both."""
    a = inputs(4, 24, F32, F32, True, True, True, 5)
    f = on(a, lambda t: t.double())
    g = torch.Generator().manual_seed(6)

    def loss(**change):
        b = dict(f, **change)
        r, n = serving.residual_norm(b["resid"], b["y"], b["norm"], b["post_norm"], b["z"], b["scale"])
        return (r * f["d"]).sum() + (n * f["dn"]).sum()

    out = serving.residual_norm(f["resid"], f["y"], f["norm"], f["post_norm"], f["z"], f["scale"])[0]
    got = back(on(dict(a, resid=out.float()), lambda t: t.cuda()))
    for name, grad in (("resid", "d_resid"), ("y", "dy"), ("z", "dz"), ("norm", "dnorm"), ("post_norm", "dpost_norm"), ("scale", "dscale")):
        v = torch.randn(f[name].shape, generator=g, dtype=torch.float64)
        diff = (loss(**{name: f[name] + 1e-5 * v}) - loss(**{name: f[name] - 1e-5 * v})) / 2e-5
        along = (got[grad].double().cpu() * v).sum()
        size = (got[grad].double().cpu().norm() * v.norm()).item()
        assert abs(along.item() - diff.item()) <= 1e-5 * size, name  # (float32 gradients: 16 roundings of 2^-24, and the input's own)


def test_many_rows_odd_views_and_none():
    a = on(inputs(3000, 24, BF16, F32, True, True, True, 7), lambda t: t.cuda())
    want = oracle_grads(on(a, lambda t: t.cpu()))
    first = back(a)
    for k, w in want.items():
        assert_close(first[k].cpu(), w, 2.0 ** -8 if k in ("dy", "dz") else 1e-5 if k[:2] == "dn" or k in ("dpost_norm", "dscale") else 1e-6, k)
    again = back(a)
    assert all(torch.equal(first[k], again[k]) for k in first)  # column sums have a fixed order

    def odd(t):
        raw = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        raw[1:] = t.flatten()
        return raw[1:].view(t.shape)

    shifted = on(a, odd)
    for t, u in zip(call(shifted), call(a)):
        assert_close(t, u.double(), 2.0 ** -8 if t.dtype == BF16 else 1e-6)
    for k, t in back(shifted).items():
        assert_close(t, first[k].double(), 2.0 ** -8 if t.dtype == BF16 else 1e-6, k)
    none = on(inputs(0, 24, BF16, F32, True, True, True), lambda t: t.cuda())
    r, n = call(none)
    g = back(none)
    assert r.shape == n.shape == (0, 24) and not g["dnorm"].any() and not g["dscale"].any() and not g["dpost_norm"].any()


def test_gradients_in_a_graph_and_on_a_stream():
    a = on(inputs(65, 512, BF16, BF16, True, False, True, 8), lambda t: t.cuda())
    want = {k: t.clone() for k, t in back(a).items() if t is not None}
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = back(a)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(got[k], t) for k, t in want.items())


@pytest.mark.parametrize("io,res", [(F32, F32), (BF16, F32), (BF16, BF16)], ids=["f32", "bf16 on f32", "bf16"])
@pytest.mark.parametrize("rows,D", [(700, 2048), (1300, 1000), (660, 1999), (330, 5000), (310, 8200), (300, 16384)])
def test_several_rows_a_thread(rows, D, io, res):
    """More rows than the GPU holds at once: a CTA walks over two or three, with the next one under way, and adds up their columns."""
    a = inputs(rows, D, io, res, True, True, True, 9)
    dev, f = on(a, lambda t: t.cuda()), on(a, lambda t: t.double())
    r, n = call(dev)
    r_want, n_want = serving.residual_norm(f["resid"], f["y"], f["norm"], f["post_norm"], f["z"], f["scale"])
    assert_close(r.cpu(), r_want, TOL[res], "resid")
    assert_close(n.cpu(), n_want, TOL[io], "n")
    got, want = back(dev), oracle_grads(a)
    for k, w in want.items():
        assert_close(got[k].cpu(), w, TOL[io] if k in ("dy", "dz") else TOL[res] if k == "d_resid" else 1e-5, k)


@pytest.mark.parametrize("rows,D", [(700, 2048), (5, 64), (9, 449), (300, 4096)])
@pytest.mark.parametrize("io,res", [(F32, F32), (BF16, F32), (BF16, BF16)], ids=["f32", "bf16 on f32", "bf16"])
def test_stream_in_place(rows, D, io, res):
    """resid_out on resid, d_resid on d_resid_out: the bits of separate arrays."""
    a = on(inputs(rows, D, io, res, True, True, True, 10), lambda t: t.cuda())
    lib, p = _lib.lib(), lambda t: C.c_void_p(t.data_ptr())
    code = lambda t: _lib.MXB_F32 if t == F32 else _lib.MXB_BF16  # noqa: E731
    d = _lib.ResidualNormDesc(rows, D, code(io), code(res), 1e-5)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    want_r, want_n = call(a)
    r, n = a["resid"].clone(), torch.empty_like(a["y"])
    assert lib.mxb_residual_norm_fwd(C.byref(d), p(r), p(a["y"]), p(a["norm"]), p(a["post_norm"]), p(a["z"]), p(a["scale"]), p(r), p(n), stream) == 0
    assert torch.equal(r, want_r) and torch.equal(n, want_n)
    want = back(a)
    g = {k: torch.empty_like(v) for k, v in want.items()}
    g["d_resid"] = a["d"].clone()
    ws = torch.empty(lib.mxb_residual_norm_workspace_bytes(C.byref(d)), dtype=torch.uint8, device="cuda")
    assert lib.mxb_residual_norm_bwd(C.byref(d), p(a["resid"]), p(a["y"]), p(a["norm"]), p(a["post_norm"]), p(a["z"]), p(a["scale"]), p(g["d_resid"]),
                                     p(a["dn"]), p(g["d_resid"]), p(g["dy"]), p(g["dz"]), p(g["dnorm"]), p(g["dpost_norm"]), p(g["dscale"]), p(ws),
                                     ws.numel(), stream) == 0
    assert all(torch.equal(g[k], want[k]) for k in want)


def test_refusals():
    a = on(inputs(4, 24, BF16, BF16, True, True, True), lambda t: t.cuda())
    for bad in (dict(y=a["y"][:3]), dict(norm=a["norm"].bfloat16()), dict(norm=a["norm"][:5]), dict(z=a["z"].float()), dict(scale=a["scale"][:1]),
                dict(resid=a["resid"].double()), dict(y=a["y"].float()), dict(resid=a["resid"].t().contiguous().t())):
        with pytest.raises((ValueError, TypeError)):
            call(dict(a, **bad))
    with pytest.raises(_lib.MxbError):
        call(a, eps=-1.0)
    big = on(inputs(1, 16392, F32, F32, False, False, False), lambda t: t.cuda())
    with pytest.raises(_lib.MxbError):
        call(big)
