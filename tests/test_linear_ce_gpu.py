"""The output head's loss and its gradients against float64.

Tolerances are counted before the first run.  u = 2^-24.  A sum on the tensor cores is off by at most 2 u of the terms' absolute
values for every step of 16 terms (the accumulator may be cut rather than rounded); float32 operands come in three parts, which
leaves 4 u of the terms, and their sums are handed over every 2048 terms.  g is rounded to bf16: at most 2^-8 of it, each
independently of the others, so that a sum's error has at most the deviation 2^-8 sqrt(sum of squares)."""
import ctypes as C

import pytest
import torch

import mixlab_b200
from mixlab_b200 import _lib, ops
from oracle import step_ends

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def make(n, V, D, io, seed=0, masked=True, tokens=torch.int64):
    g = torch.Generator().manual_seed(seed + n + V + D)
    w = 2 / D ** 0.5 * torch.randn(V, D, generator=g)
    t = ((V + 1.0) ** torch.rand(n, generator=g, dtype=torch.float64) - 1).long().clamp(0, V - 1)
    x = (torch.randn(n, D, generator=g) + w[t]).to(io)
    if masked and n > 3:
        t[2::5] = -1
        t[3::7] = V
        t[n - 1] = -100
        x[t < 0] = float("nan")
        x[t == V] = float("inf")
    return x.cuda(), w.to(io).cuda(), t.to(tokens).cuda(), g


def steps(terms, io):
    """Relative to the terms' absolute values: what a sum of so many is off by."""
    # (bf16 too is handed over, every 65536 terms)
    return (2 * (min(terms, 65536) / 16 + 2) + terms / 65536 if io == BF16 else 2 * (min(terms, 2048) / 16 + 2) + 4 + terms / 2048) * U


def slack(x, w, io):
    """Of a logit; of lse beyond the logits'."""
    ok = torch.isfinite(x).all(-1)
    size = torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    for rows in ok.nonzero()[:, 0].split(2048):
        size[rows] = (x[rows].double().abs() @ w.double().abs().T).amax(1)
    z = steps(x.shape[1], io) * size
    V = w.shape[0]
    # exponents are rounded at up to 3 places, 2 u of the largest; 128 + V / 2048 + 8 terms one after the other, exponentials good to 4 u
    return z, (6 * 1.5 * size + 128 + V / 2048 + 16) * U


SIZES = [(1, 1, 1), (1, 100, 16), (3, 7, 8), (5, 257, 24), (64, 1000, 64), (255, 511, 72), (256, 512, 128), (257, 513, 136), (130, 128, 449),
         (300, 5003, 448), (1025, 300, 40), (1024, 129, 31), (700, 2000, 1000), (33, 33000, 264), (513, 1025, 2050), (6000, 70, 24), (5, 300, 70000)]


@pytest.mark.parametrize("io", [BF16, F32])
@pytest.mark.parametrize("n,V,D", SIZES)
def test_loss(n, V, D, io):
    x, w, t, _ = make(n, V, D, io, tokens=torch.int32 if n % 2 else torch.int64)
    loss, lse = ops.linear_cross_entropy(x, w, t)
    want_loss, want_lse = step_ends.linear_cross_entropy(x.double(), w.double(), t)
    z, rest = slack(x, w, io)
    assert loss.dtype == lse.dtype == F32 and loss.shape == lse.shape == (n,)
    off = (lse.double() - want_lse).abs() - (z + rest + 2 * U * want_lse.abs())
    assert torch.isfinite(lse).all() and (off <= 0).all(), off.max()
    off = (loss.double() - want_loss).abs() - (2 * z + rest + 3 * U * (want_lse.abs() + want_loss.abs()))
    assert torch.isfinite(loss).all() and (off <= 0).all(), off.max()
    dead = (t < 0) | (t >= V)
    assert (loss[dead] == 0).all() and (lse[dead] == 0).all()


def check_gradients(x, w, t, lse, a, c, got, io):
    xd, wd = torch.nan_to_num(x.double(), 0.0, 0.0, 0.0), w.double()
    want = step_ends.linear_cross_entropy_backward(xd, wd, t, lse.double(), a.double(), None if c is None else c.double())
    ok = (t >= 0) & (t < w.shape[0]) & ((a != 0) | (torch.zeros_like(a) if c is None else c).ne(0))
    assert got["dx"].dtype == got["dweight"].dtype == io and (got["dx"][~ok] == 0).all()
    rows = xd[ok]
    z, _ = slack(x[ok], w, io)
    both = (a + (0 if c is None else c)).double()[ok]
    p = both.abs()[:, None] * torch.exp(rows @ wd.T - lse.double()[ok][:, None])
    size = (rows.abs() @ wd.abs().T).amax(1, keepdim=True)
    sure = p * (z[:, None] + (8 + 6 * 1.5 * (size + lse.double()[ok].abs()[:, None])) * U)  # g's own error
    g = p.clone()
    at = t[ok].long()[:, None]
    g.scatter_(1, at, (both[:, None] * torch.exp(rows @ wd.T - lse.double()[ok][:, None])).gather(1, at) - a.double()[ok][:, None])
    g = g.abs()
    sure = sure + 2 * U * g
    half = 2.0 ** -8 if io == BF16 else 4 * U
    for name, e, other, terms in (("dx", sure, wd, w.shape[0]), ("dweight", sure.T, rows, int(ok.sum()))):
        gg = g if name == "dx" else g.T
        always = e @ other.abs() + steps(terms, io) * (gg @ other.abs())
        have, need = got[name].double(), want[name]
        if name == "dx":
            have, need = have[ok], need[ok]
        last = (2.0 ** -8 if io == BF16 else U) * need.abs()
        off = (have - need).abs()
        assert torch.isfinite(have).all(), name
        assert (off <= always + half * (gg @ other.abs()) + last + 1e-37).all(), (name, "element", (off - always - last).max())
        by_chance = half * torch.sqrt(gg.square() @ other.square())
        bound = by_chance.norm() + always.norm() + last.norm() + 1e-37
        assert off.norm() <= bound, (name, "norm", (off.norm() / bound).item())


@pytest.mark.parametrize("io", [BF16, F32])
@pytest.mark.parametrize("n,V,D", SIZES)
def test_gradients(n, V, D, io):
    x, w, t, g = make(n, V, D, io, tokens=torch.int32 if V % 2 else torch.int64)
    lse = ops.linear_cross_entropy(x, w, t)[1]
    a, c = torch.rand(n, generator=g).cuda(), 0.3 * torch.randn(n, generator=g).cuda()
    a[::4] = 0.0
    got = ops.linear_cross_entropy_backward(x, w, t, lse, a)
    check_gradients(x, w, t, lse, a, None, got, io)
    again = ops.linear_cross_entropy_backward(x, w, t, lse, a)
    assert torch.equal(got["dx"], again["dx"]) and torch.equal(got["dweight"], again["dweight"])  # a fixed order
    c[::8] = 0.0
    check_gradients(x, w, t, lse, a, c, ops.linear_cross_entropy_backward(x, w, t, lse, a, d_lse=c), io)


@pytest.mark.parametrize("n,V,D,io", [(8192, 40001, 40, BF16), (4097, 40000, 24, F32)])
def test_gradients_in_pieces_of_the_vocabulary(n, V, D, io):
    x, w, t, g = make(n, V, D, io)
    lse = ops.linear_cross_entropy(x, w, t)[1]
    a = torch.rand(n, generator=g).cuda()
    check_gradients(x, w, t, lse, a, None, ops.linear_cross_entropy_backward(x, w, t, lse, a), io)


@pytest.mark.parametrize("io", [BF16, F32])
def test_no_token_counts(io):
    x = torch.full((300, 72), float("nan"), dtype=io, device="cuda")
    w = torch.randn(500, 72, device="cuda").to(io)
    t = torch.full((300,), -1, device="cuda")
    loss, lse = ops.linear_cross_entropy(x, w, t)
    assert (loss == 0).all() and (lse == 0).all()
    g = ops.linear_cross_entropy_backward(x, w, t, lse, torch.ones(300, device="cuda"))
    assert (g["dx"] == 0).all() and (g["dweight"] == 0).all()
    g = ops.linear_cross_entropy_backward(x, w, t.zero_(), lse, torch.zeros(300, device="cuda"))
    assert (g["dx"] == 0).all() and (g["dweight"] == 0).all()
    loss, lse = ops.linear_cross_entropy(x[:0], w, t[:0])
    assert loss.shape == lse.shape == (0,)
    g = ops.linear_cross_entropy_backward(x[:0], w, t[:0], lse, loss)
    assert g["dx"].shape == (0, 72) and (g["dweight"] == 0).all()


def test_large_logits():
    """Logits far from zero, on either side, and infinite ones."""
    w = torch.randn(700, 64, device="cuda")
    x = torch.randn(40, 64, device="cuda")
    t = torch.randint(0, 700, (40,), device="cuda")
    for shift in (-300.0, 3000.0):
        ws = torch.cat([w, torch.full((700, 8), 1.0, device="cuda")], 1)
        xs = torch.cat([x, torch.full((40, 8), shift / 8, device="cuda")], 1)
        loss, lse = ops.linear_cross_entropy(xs, ws, t)
        want, want_lse = step_ends.linear_cross_entropy(xs.double(), ws.double(), t)
        z, rest = slack(xs, ws, F32)
        assert ((loss.double() - want).abs() <= 2 * z + rest + 3 * U * want_lse.abs()).all()
        g = ops.linear_cross_entropy_backward(xs, ws, t, lse, torch.ones(40, device="cuda"))
        check_gradients(xs, ws, t, lse, torch.ones(40, device="cuda"), None, g, F32)
    b = w.to(BF16)
    b[13] = 0
    b[13, 5] = float("-inf")
    xb = x.abs().to(BF16)
    loss, lse = ops.linear_cross_entropy(xb, b, t.clamp(14))
    rest_of = torch.cat([b[:13], b[14:]])
    assert torch.allclose(lse, torch.logsumexp(xb.float() @ rest_of.float().T, 1), atol=1e-3) and torch.isfinite(loss).all()


@pytest.mark.parametrize("io,D", [(BF16, 24), (BF16, 23), (F32, 24), (F32, 7)])
def test_at_any_element(io, D):
    """Bases off 16 bytes give the same bits; the words on either side of the results stay."""
    n, V = 300, 600
    x, w, t, g = make(n, V, D, io)
    a = torch.rand(n, generator=g).cuda()
    loss, lse = ops.linear_cross_entropy(x, w, t)
    want = ops.linear_cross_entropy_backward(x, w, t, lse, a)

    def shifted(v):
        flat = torch.full((v.numel() + 2,), 9, dtype=v.dtype, device="cuda")
        flat[1:-1] = v.flatten()
        return flat[1:-1].view(v.shape), flat

    sx, sa, slse, st_ = (shifted(v)[0] for v in (x, a, lse, t.int()))
    sw = w if io == BF16 and D % 8 == 0 else shifted(w)[0]
    got, got_lse = ops.linear_cross_entropy(sx, sw, st_)
    assert torch.equal(got, loss) and torch.equal(got_lse, lse)
    lib, code = mixlab_b200.lib(), _lib.MXB_BF16 if io == BF16 else _lib.MXB_F32
    d = _lib.LinearCeDesc(n, V, D, 4, code)
    (dx, fx), (dw, fw) = shifted(torch.zeros_like(x)), shifted(torch.zeros_like(w))
    p, st = lambda v: C.c_void_p(v.data_ptr()), C.c_void_p(torch.cuda.current_stream().cuda_stream)  # noqa: E731
    ws = torch.full((lib.mxb_linear_ce_bwd_workspace_bytes(C.byref(d)),), 255, dtype=torch.uint8, device="cuda")
    assert lib.mxb_linear_ce_bwd(C.byref(d), p(sx), p(sw), p(st_), p(slse), p(sa), None, p(dx), p(dw), p(ws), ws.numel(), st) == 0
    assert torch.equal(dx, want["dx"]) and torch.equal(dw, want["dweight"])
    assert fx[0] == 9 and fx[-1] == 9 and fw[0] == 9 and fw[-1] == 9
    out = C.c_int32(-1)
    assert lib.mxb_gdn_device_status(p(ws), C.byref(out)) == 0 and out.value == 0


def test_gradient_is_the_slope():
    """The formulas against differences, in float64 on the CPU."""
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, a, c, t = r(4, 3), r(6, 3), r(4), r(4), torch.tensor([5, -1, 0, 2])
    lse = step_ends.linear_cross_entropy(x, w, t)[1]
    got = step_ends.linear_cross_entropy_backward(x, w, t, lse, a, c)
    for name, v in (("dx", x), ("dweight", w)):
        for i in range(v.numel()):
            e = torch.zeros_like(v)
            e.view(-1)[i] = 1e-5

            def at(s):
                loss, lse_ = step_ends.linear_cross_entropy(*(u + s * e if u is v else u for u in (x, w)), t)
                return (loss * a + lse_ * c).sum()
            assert abs((at(1) - at(-1)) / 2e-5 - got[name].view(-1)[i]) < 1e-8, (name, i)


def test_shaped_tokens():
    x, w, t, g = make(60, 90, 32, BF16)
    loss, lse = ops.linear_cross_entropy(x, w, t)
    l3, s3 = ops.linear_cross_entropy(x.view(3, 4, 5, 32), w, t.view(3, 4, 5))
    assert l3.shape == (3, 4, 5) and torch.equal(l3.flatten(), loss) and torch.equal(s3.flatten(), lse)
    a = torch.rand(60, generator=g).cuda()
    flat = ops.linear_cross_entropy_backward(x, w, t, lse, a)
    got = ops.linear_cross_entropy_backward(x.view(3, 4, 5, 32), w, t.view(3, 4, 5), s3, a.view(3, 4, 5))
    assert got["dx"].shape == (3, 4, 5, 32) and torch.equal(got["dx"].view(60, 32), flat["dx"]) and torch.equal(got["dweight"], flat["dweight"])
