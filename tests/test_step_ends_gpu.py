"""The token rows and the layer norm, with their gradients, against float64.

Tolerances are counted before the first run: a rounding to a type is off by half of its eps relative to the value (u = 2^-24 in
float32), and a chain of n float32 operations on terms whose absolute values add up to S by n u S."""
import ctypes as C

import pytest
import torch

import mixlab_b200
from mixlab_b200 import _lib, ops
from oracle import step_ends

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def half(t):
    return torch.finfo(t).eps / 2


def near(got, want, slack, what):
    """|got - want| at most its type's rounding of want and slack, element by element.  what: the type, a name."""
    got, slack = got.double().cpu(), torch.as_tensor(slack, dtype=torch.float64)
    off = (got - want).abs() - (half(what[0]) * want.abs() + slack * 1.01)
    assert torch.isfinite(got).all() and (off <= 0).all(), (what, off.max().item(), int((off > 0).sum()))


def rnd(g, *shape):
    return torch.randn(*shape, generator=g)


# ------------------------------------------------------------------ the token rows
def words(g, n, V, skew):
    """Tokens, a few of them often; padding on either side of the range."""
    u = torch.rand(n, generator=g, dtype=torch.float64)
    tok = ((V + 1.0) ** u - 1).long().clamp(0, V - 1) if skew else (u * V).long().clamp(0, V - 1)
    if n > 4:
        tok[1], tok[n // 2] = -1, V
    return tok


ROWS = [(1, 1, 8), (5, 3, 1), (1, 70000, 16), (37, 5, 449), (300, 1, 64), (257, 1025, 24), (2047, 257, 448), (2048, 9001, 24), (2049, 2, 40), (4096, 300, 16), (4097, 300, 16), (65536, 33, 8), (65537, 4000, 8), (4100, 50001, 72),
        (6000, 40, 2050), (70001, 700, 32), (131, 131, 2056)]


@pytest.mark.parametrize("io,out", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("n,V,D", ROWS)
def test_rows_and_their_gradient(n, V, D, io, out):
    g = torch.Generator().manual_seed(n + V)
    tok = words(g, n, V, D % 16 == 0)
    w, d = rnd(g, V, D).to(io), rnd(g, n, D).to(io)
    scale = D ** 0.5
    s32 = torch.tensor(scale, dtype=F32).item()  # the call rounds it
    tokens = tok.cuda() if n % 2 else tok.int().cuda()
    y = ops.embedding(tokens, w.cuda(), scale=scale, dtype=out)
    assert y.dtype == out and y.shape == (n, D)
    want = step_ends.embedding(tok, w.double(), s32)
    near(y, want, U * want.abs(), (out, "rows"))
    dw = ops.embedding_backward(tokens, d.cuda(), V, scale=scale, dtype=out)
    assert dw.dtype == out and dw.shape == (V, D)
    want, size, terms = step_ends.embedding_backward(tok, d.double(), V, s32)
    near(dw, want, (terms[:, None] + 2) * U * size, (out, "gradient"))
    # added to what is there: one more operation
    old = rnd(g, V, D).to(out)
    into = old.cuda()
    assert ops.embedding_backward(tokens, d.cuda(), V, scale=scale, dweight=into) is not None
    near(into, old.double() + want, (terms[:, None] + 3) * U * (size + old.double().abs()), (out, "sum"))
    again = old.cuda()
    ops.embedding_backward(tokens, d.cuda(), V, scale=scale, dweight=again)
    assert torch.equal(into, again)  # a fixed order


def test_rows_of_shaped_tokens_defaults_and_empty_calls():
    g = torch.Generator().manual_seed(1)
    w = rnd(g, 11, 24).to(BF16).cuda()
    tok = torch.randint(0, 11, (3, 5), generator=g)
    y = ops.embedding(tok.cuda(), w)
    assert y.dtype == BF16 and y.shape == (3, 5, 24) and torch.equal(y, w[tok.cuda()])
    dw = ops.embedding_backward(tok.cuda(), y, 11)
    assert dw.dtype == BF16 and dw.shape == (11, 24)
    none = torch.empty(0, dtype=torch.long, device="cuda")
    assert ops.embedding(none, w).shape == (0, 24)
    assert (ops.embedding_backward(none, torch.empty(0, 24, device="cuda"), 11) == 0).all()
    kept = torch.ones(11, 24, device="cuda")
    assert (ops.embedding_backward(none, torch.empty(0, 24, device="cuda"), 11, dweight=kept) == 1).all()
    pad = torch.full((700,), -7, dtype=torch.int32, device="cuda")
    assert (ops.embedding(pad, w) == 0).all()
    assert (ops.embedding_backward(pad, torch.full((700, 24), float("nan"), device="cuda"), 11) == 0).all()


def test_padding_may_hold_anything():
    """Rows of padding are not read into the sums, tokens of 64 bits beyond 32 are padding."""
    d = torch.full((600, 16), float("inf"), device="cuda")
    d[::3] = 1.0
    tok = torch.full((600,), (1 << 32) + 1, dtype=torch.long, device="cuda")
    tok[::3] = 1
    dw = ops.embedding_backward(tok, d, 3)
    assert (dw[1] == 200).all() and (dw[0] == 0).all() and (dw[2] == 0).all()
    assert (ops.embedding(tok, torch.ones(3, 16, device="cuda"))[:, 0] == (tok == 1)).all()


@pytest.mark.parametrize("D", [24, 20])
def test_rows_at_any_element(D):
    """Bases off 16 bytes, through the C ABI."""
    lib, g = mixlab_b200.lib(), torch.Generator().manual_seed(3)
    n, V = 700, 37
    tok, flat = torch.randint(0, V, (n,), generator=g), rnd(g, V * D + 1).cuda()
    w, out = flat[1:].view(V, D), torch.full((n * D + 1,), 9.0, device="cuda")
    d = _lib.EmbeddingDesc(n, V, D, 8, _lib.MXB_F32, _lib.MXB_F32, 1.0)
    p, st = lambda t: C.c_void_p(t.data_ptr()), C.c_void_p(torch.cuda.current_stream().cuda_stream)  # noqa: E731
    t = tok.cuda()
    assert lib.mxb_embedding_fwd(C.byref(d), p(t), p(w), p(out[1:]), st) == 0
    assert out[0] == 9 and torch.equal(out[1:].view(n, D), w[t])
    ws, dw = torch.empty(lib.mxb_embedding_bwd_workspace_bytes(C.byref(d)), dtype=torch.uint8, device="cuda"), torch.full((V * D + 2,), 9.0, device="cuda")
    assert lib.mxb_embedding_bwd(C.byref(d), p(t), p(out[1:]), p(dw[1:]), 0, p(ws), ws.numel(), st) == 0
    assert dw[0] == 9 and dw[-1] == 9
    want, size, terms = step_ends.embedding_backward(tok, out[1:].view(n, D).double().cpu(), V)
    near(dw[1:-1].view(V, D), want, (terms[:, None] + 2) * U * size, (F32, "gradient"))


# ------------------------------------------------------------------ the layer norm
# Longest chains: a column sum of a row runs over 8 columns of up to 4 pieces, 5 shuffles and 32 warps: 70 additions.
CHAIN = 70
NORMS = [(1, 1), (1, 2048), (3, 7), (5, 64), (129, 449), (37, 1000), (700, 24), (4001, 40), (9, 4096), (11, 5000), (2, 8200), (3, 16384), (2, 12289)]


def norm_slack(h, w, b, eps):
    """What float32 leaves open in n: the mean is off by CHAIN u mean|h|, which enters u and (squared, below) k; k by CHAIN + 4."""
    m = h.mean(-1, keepdim=True)
    k = torch.rsqrt((h - m).square().mean(-1, keepdim=True) + eps)
    shift = (CHAIN + 1) * U * h.abs().mean(-1, keepdim=True) * k + 2 * U * (h.abs() + m.abs()) * k
    unit = ((h - m) * k).abs()
    # a shifted mean changes the squares' mean by its own square: the relative change of k is at most (shift + CHAIN u)
    return (shift + unit * (shift.square() + (CHAIN + 6) * U)) * w.abs() + 2 * U * (unit * w.abs() + (0 if b is None else b.abs()))


@pytest.mark.parametrize("io,res", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows,D", NORMS)
def test_layer_norm(rows, D, io, res):
    g = torch.Generator().manual_seed(rows + D)
    x, stream = rnd(g, rows, D).to(io), (0.5 + 2 * rnd(g, rows, D)).to(res)
    w, b = 1 + 0.1 * rnd(g, D), 0.1 * rnd(g, D)
    cuda = lambda *ts: [t.cuda() for t in ts]  # noqa: E731
    xc, sc, wc, bc = cuda(x, stream, w, b)
    f = lambda t: t.double()  # noqa: E731
    for bias in (b, None):
        h, n = step_ends.layer_norm(f(x), f(w), None if bias is None else f(bias), f(stream))
        slack = norm_slack(h, f(w), None if bias is None else f(bias), 1e-5) + U * 4 * (f(x).abs() + f(stream).abs()) * f(w).abs() * torch.rsqrt(h.var(-1, unbiased=False, keepdim=True) + 1e-5)
        got_h, got = ops.layer_norm(xc, wc, None if bias is None else bc, resid=sc)
        assert got_h.dtype == res and got.dtype == io
        near(got_h, h, U * h.abs(), (res, "stream"))
        near(got, n, slack, (io, "norm"))
    # without a stream: one tensor in the stream's type, the result in io
    n = step_ends.layer_norm(f(stream), f(w), f(b))[1]
    got = ops.layer_norm(sc, wc, bc, dtype=io)
    assert got.dtype == io
    near(got, n, norm_slack(f(stream), f(w), f(b), 1e-5), (io, "plain norm"))


def grad_slack(x, w, dn, eps):
    m = x.mean(-1, keepdim=True)
    k = torch.rsqrt((x - m).square().mean(-1, keepdim=True) + eps)
    shift = (CHAIN + 1) * U * x.abs().mean(-1, keepdim=True) * k + 2 * U * (x.abs() + m.abs()) * k  # of u
    u, t = (x - m) * k, dn * w
    tu = (t * u).abs().mean(-1, keepdim=True)
    far = (CHAIN + 8) * U
    inner = far * (t.abs() + t.abs().mean(-1, keepdim=True) + 2 * u.abs() * tu) + shift * tu + u.abs() * (t.abs() * shift).mean(-1, keepdim=True)
    du = shift + u.abs() * (shift.square() + far)
    return k * inner * (1 + far), du


@pytest.mark.parametrize("io,res", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows,D", NORMS)
def test_layer_norm_gradients(rows, D, io, res):
    g = torch.Generator().manual_seed(rows * D)
    x, dn, d = (0.5 + 2 * rnd(g, rows, D)).to(res), rnd(g, rows, D).to(io), rnd(g, rows, D).to(res)
    w = 1 + 0.1 * rnd(g, D)
    f = lambda t: t.double()  # noqa: E731
    slack, du = grad_slack(f(x), f(w), f(dn), 1e-5)
    u = step_ends.layer_norm(f(x), torch.ones(D).double())[1]
    for other in (d, None):
        want = step_ends.layer_norm_backward(f(x), f(w), f(dn), None if other is None else f(other))
        got = ops.layer_norm_backward(x.cuda(), w.cuda(), dn.cuda(), d_resid=None if other is None else other.cuda())
        assert got["dx"].dtype == res and got["dweight"].dtype == got["dbias"].dtype == F32
        near(got["dx"], want["dx"], slack + 2 * U * (want["dx"].abs() + (0 if other is None else f(other).abs())), (res, "dx"))
        adds = (rows + 70) * U  # a column's sum: the rows, the slices
        near(got["dweight"], want["dweight"], ((f(dn).abs() * (du + 2 * U * u.abs())).sum(0) + adds * (f(dn) * u).abs().sum(0)), (F32, "dweight"))
        near(got["dbias"], want["dbias"], adds * f(dn).abs().sum(0), (F32, "dbias"))


def test_layer_norm_gradient_is_the_slope():
    """The formulas against differences, in float64 on the CPU."""
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, b, dn = r(3, 5), r(5), r(5), r(3, 5)
    got = step_ends.layer_norm_backward(x, w, dn)
    for name, t in (("dx", x), ("dweight", w), ("dbias", b)):
        for i in range(t.numel()):
            e = torch.zeros_like(t)
            e.view(-1)[i] = 1e-5
            at = lambda s: step_ends.layer_norm(*(v + s * e if v is t else v for v in (x, w, b)))[1]  # noqa: E731
            slope = ((at(1) - at(-1)) * dn).sum() / 2e-5
            assert abs(slope - got[name].reshape(-1)[i]) < 1e-8, (name, i)


def test_layer_norm_of_a_constant_row_and_far_means():
    x = torch.full((4, 96), 3.0, device="cuda")
    w, b = torch.ones(96, device="cuda"), torch.full((96,), 0.25, device="cuda")
    assert (ops.layer_norm(x, w, b) == 0.25).all()
    g = torch.Generator().manual_seed(2)
    far = 1000 + rnd(g, 7, 512)
    want = step_ends.layer_norm(far.double(), torch.ones(512).double())[1]
    near(ops.layer_norm(far.cuda(), torch.ones(512, device="cuda")), want, norm_slack(far.double(), torch.ones(512).double(), None, 1e-5), (F32, "far mean"))


def test_layer_norm_of_no_rows():
    w = torch.ones(16, device="cuda")
    none = torch.empty(0, 16, device="cuda")
    assert ops.layer_norm(none, w).shape == (0, 16)
    g = ops.layer_norm_backward(none, w, none)
    assert g["dx"].shape == (0, 16) and (g["dweight"] == 0).all() and (g["dbias"] == 0).all()


@pytest.mark.parametrize("D", [24, 21])
def test_layer_norm_at_any_element_and_in_place(D):
    lib, g = mixlab_b200.lib(), torch.Generator().manual_seed(4)
    rows = 3000
    flat = rnd(g, rows * D + 1).cuda()
    x, w = flat[1:].view(rows, D), (1 + 0.1 * rnd(g, D)).cuda()
    n = torch.full((rows * D + 2,), 9.0, device="cuda")
    d = _lib.LayerNormDesc(rows, D, _lib.MXB_F32, _lib.MXB_F32, 1e-5)
    p, st = lambda t: C.c_void_p(t.data_ptr()), C.c_void_p(torch.cuda.current_stream().cuda_stream)  # noqa: E731
    assert lib.mxb_layer_norm_fwd(C.byref(d), None, p(x), p(w), None, None, p(n[1:]), st) == 0
    # (single elements a thread add up in another order than whole pieces: the same bounds, not the same bits)
    want = step_ends.layer_norm(x.double().cpu(), w.double().cpu())[1]
    near(n[1:-1].view(rows, D), want, norm_slack(x.double().cpu(), w.double().cpu(), None, 1e-5), (F32, "norm"))
    assert n[0] == 9 and n[-1] == 9
    # the stream and its gradient in place
    r, y = rnd(g, rows, D).cuda(), rnd(g, rows, D).cuda()
    want_h, want_n = ops.layer_norm(y, w, resid=r)
    got = torch.empty_like(y)
    assert lib.mxb_layer_norm_fwd(C.byref(d), p(r), p(y), p(w), None, p(r), p(got), st) == 0
    assert torch.equal(r, want_h) and torch.equal(got, want_n)
    dr = rnd(g, rows, D).cuda()
    want = ops.layer_norm_backward(r, w, y, d_resid=dr)
    ws, dw, db = torch.empty(lib.mxb_layer_norm_bwd_workspace_bytes(C.byref(d)), dtype=torch.uint8, device="cuda"), torch.empty_like(w), torch.empty_like(w)
    assert lib.mxb_layer_norm_bwd(C.byref(d), p(r), p(w), p(dr), p(y), p(dr), p(dw), p(db), p(ws), ws.numel(), st) == 0
    assert torch.equal(dr, want["dx"]) and torch.equal(dw, want["dweight"]) and torch.equal(db, want["dbias"])


@pytest.mark.parametrize("D", [24, 40])
def test_bf16_rows_on_sixteen_bytes(D):
    """Views that begin in the middle of a matrix: whole pieces of bf16 on 16 bytes, float32 beside them on 32 or not."""
    g = torch.Generator().manual_seed(8)
    n, V = 300, 50
    w, tok = rnd(g, V + 1, D).to(BF16), torch.randint(0, V, (n,), generator=g)
    part = w.cuda()[1:]
    for out in (BF16, F32):
        y = ops.embedding(tok.cuda(), part, dtype=out)
        assert torch.equal(y.cpu(), w[1:][tok].to(out))
    d = rnd(g, n + 1, D).to(BF16)
    want, size, terms = step_ends.embedding_backward(tok, d[1:].double(), V)
    near(ops.embedding_backward(tok.cuda(), d.cuda()[1:], V, dtype=F32), want, (terms[:, None] + 2) * U * size, (F32, "gradient"))
    stream = rnd(g, n + 1, D)
    for x in (d, stream):
        x64 = x[1:].double()
        got = ops.layer_norm(x.cuda()[1:], torch.ones(D + 4, device="cuda")[4:], dtype=BF16)
        near(got, step_ends.layer_norm(x64, torch.ones(D).double())[1], norm_slack(x64, torch.ones(D).double(), None, 1e-5), (BF16, "norm"))
