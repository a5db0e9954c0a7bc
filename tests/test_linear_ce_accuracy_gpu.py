"""What the output head's loss and its gradients are off by, sum by sum, against float64.

Tolerances are counted before the first run.  u = 2^-24; a bf16 is off by half of its eps, 2^-8, relative to the value."""
import pytest
import torch

from mixlab_b200 import ops
from oracle import step_ends

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U, HALF = 2.0 ** -24, 2.0 ** -8


@pytest.mark.parametrize("weight", [1 / 28672, 0.3, -5.2])
def test_equal_weights_have_no_part_in_the_rounding(weight):
    """Gradients of a mean: what is left of got - want along want, element for element independent errors add up to little there, a
    weight that is rounded does in full (0.0020, 0.0026 and 0.0018 for these weights)."""
    n, V, D = 512, 8000, 64
    g = torch.Generator().manual_seed(11)
    w = torch.randn(V, D, generator=g).to(BF16).cuda()
    x = (0.02 * torch.randn(n, D, generator=g)).to(BF16).cuda()
    t = torch.randint(0, V, (n,), generator=g)
    t[0] = -1  # (the first row has no part)
    d = torch.full((n,), weight)
    d[1::9] = 0.0
    lse = ops.linear_cross_entropy(x, w, t.cuda())[1]
    got = ops.linear_cross_entropy_backward(x, w, t.cuda(), lse, d.cuda())
    t, d = t.cuda(), torch.where(t.cuda() >= 0, d.cuda(), 0.0).double()
    xd, wd = x.double(), w.double()
    want = step_ends.linear_cross_entropy_backward(xd, wd, t, lse.double(), d)
    live = d != 0
    p = live[:, None] * torch.exp(xd @ wd.T - lse.double()[:, None])
    most = p.max().item()
    grad = p * d.abs()[:, None]
    grad[live.nonzero()[:, 0], t[live]] += d[live].abs()
    for name, e, other in (("dx", grad, wd), ("dweight", grad.T, xd)):
        need = want[name]
        size = need.norm()
        along = ((got[name].double() - need) * need).sum().abs() / size ** 2
        last = 4 * HALF * need.square().norm() / size ** 2  # by chance, four deviations
        hits = 1.5 * most  # 1 - p to the nearest bf16, 1 among them
        others = 4 * HALF * most * abs(weight) * other.norm() / size  # by chance: |W need^T| <= |W| |need|
        sums = 2 * U * (e.shape[1] / 16 + 2) * (e @ other.abs()).norm() / size  # accumulators that are cut
        assert along <= last + hits + others + sums + 8 * U, (name, along.item(), last.item(), hits, others.item(), sums.item())
        assert last + hits + others + sums < 1e-3, name  # (far below what a rounded weight leaves)


@pytest.mark.parametrize("n", [40, 1100])
@pytest.mark.parametrize("D", [64, 63])
def test_infinite_logits(n, D):
    """lse of a logit of +infinity is +infinity, wherever its tile stands and however large the others are; one of -infinity has no part."""
    g = torch.Generator().manual_seed(n)
    V = 900
    x = torch.randn(n, D, generator=g)
    x[:, 0], x[:, 1] = 1.0, 1.0
    x[1::2, 0] = -1.0
    for word in (3, 130, 256, 511, 899):
        for other in (5, 200, 700):
            for large in (1.0, 250.0):
                w = 0.1 * torch.randn(V, D, generator=g)
                w[:, 0] = 0.0
                w[word, 0], w[other, 1] = float("inf"), large
                xb, wb = x.to(BF16).cuda(), w.to(BF16).cuda()
                t = torch.full((n,), other, device="cuda")
                loss, lse = ops.linear_cross_entropy(xb, wb, t)
                assert (lse[::2] == float("inf")).all() and (loss[::2] == float("inf")).all(), (word, other, large)
                rest = torch.cat([wb[:word], wb[word + 1:]]).double()
                want, want_lse = step_ends.linear_cross_entropy(xb.double(), rest, t - int(word < other))
                size = (xb.double().abs() @ rest.abs().T).amax(1)[1::2]
                slack = (12 * size + 16 * size + 128 + V / 2048 + 16) * U  # the logits' sums (64 terms), exponents, the sum of exponentials
                assert ((lse[1::2].double() - want_lse[1::2]).abs() <= slack).all(), (word, other, large)
                assert ((loss[1::2].double() - want[1::2]).abs() <= 2 * slack).all(), (word, other, large)


# Terms after which an accumulator on the tensor cores, which is cut with every step of 16 terms, is handed over to a float32 sum; a step of float32
# operands is six products of their parts.  Terms of one sign make what is cut add up: a share of it would be seen.
LOGIT = {F32: (128, 6), BF16: (1024, 1)}
GRADIENT_LOGIT = {F32: (128, 6), BF16: (2048, 1)}


def cut(terms, segment, products, io):
    """Relative to a sum of terms of one sign: the accumulator, the hand-overs, parts of float32 operands."""
    return (2 * (products * min(terms, segment) / 16 + 2) + -(-terms // segment) + (4 if io == F32 else 0)) * U


@pytest.mark.parametrize("io,D", [(BF16, 4096), (BF16, 16384), (F32, 2048), (F32, 8192)])
def test_a_logit(io, D):
    """One word: lse is the logit."""
    g = torch.Generator().manual_seed(D)
    n, size = 1100, 100.0
    x = torch.randn(n, D, generator=g).abs().to(io).cuda()
    w = (size * 1.5708 / D * torch.randn(1, D, generator=g).abs()).to(io).cuda()
    lse = ops.linear_cross_entropy(x, w, torch.zeros(n, dtype=torch.long, device="cuda"))[1]
    want = (x.double() @ w.double().T)[:, 0]
    # the exponent's two roundings, lse's own, the exponential and the logarithm
    off = (lse.double() - want).abs() / ((cut(D, *LOGIT[io], io) + 3 * U) * want + 8 * U)
    assert (off <= 1).all(), off.max()


def test_a_gradients_logits():
    """bf16: what a long logit is off by is in all elements of a token's g alike, the roundings of g and of the results by chance."""
    g = torch.Generator().manual_seed(7)
    n, V, D, size = 64, 256, 65536, 20.0
    x = torch.randn(n, D, generator=g).abs().to(BF16).cuda()
    w = (size * 1.5708 / D * torch.randn(V, D, generator=g).abs()).to(BF16).cuda()
    t = torch.zeros(n, dtype=torch.long, device="cuda")
    xd, wd = x.double(), w.double()
    z = xd @ wd.T
    lse = torch.logsumexp(z, 1)
    zero, one = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    got = ops.linear_cross_entropy_backward(x, w, t, lse.float(), zero, d_lse=one)
    p = torch.exp(z - lse.float().double()[:, None])
    most = z.max().item()
    for name, e, other in (("dx", p, wd), ("dweight", p.T, xd)):
        need = e @ other
        along = ((got[name].double() - need) * need).sum().abs() / need.norm() ** 2
        logits = cut(D, *GRADIENT_LOGIT[BF16], BF16) * most + 4 * most * U
        g_by_chance = 4 * HALF * (e * (need @ other.T)).norm() / need.norm() ** 2
        last = 4 * HALF * need.square().norm() / need.norm() ** 2
        bound = logits + g_by_chance + last + 2 * (e.shape[1] / 16 + 2) * U + 8 * U
        assert along <= bound, (name, along.item(), bound.item())


def test_float32_sums_of_gradients():
    """What long sums are off by along the result, in which roundings of single elements add up to little.  So many rows that no
    pair of CTAs sums less than 2048 terms."""
    g = torch.Generator().manual_seed(8)
    n, V, D = 74 * 256, 2048, 40
    x, w = 0.002 * torch.randn(n, D, generator=g).abs().cuda(), torch.randn(V, D, generator=g).abs().cuda()
    t = torch.zeros(n, dtype=torch.long, device="cuda")
    xd, wd = x.double(), w.double()
    z = xd @ wd.T
    lse = torch.logsumexp(z, 1)
    got = ops.linear_cross_entropy_backward(x, w, t, lse.float(), torch.zeros(n, device="cuda"), d_lse=torch.ones(n, device="cuda"))
    p = torch.exp(z - lse.float().double()[:, None])
    # g's own: the logit, log2 e as a float32 in the exponent, the exponential, the product
    own = cut(D, *GRADIENT_LOGIT[F32], F32) * z.max().item() + (0.5 * lse.max().item() + 6) * U
    for name, e, other in (("dx", p, wd), ("dweight", p.T, xd)):
        need = e @ other
        along = ((got[name].double() - need) * need).sum().abs() / need.norm() ** 2
        bound = own + cut(e.shape[1], 128, 6, F32) + 4 * U + U
        assert along <= bound, (name, along.item() / U, bound / U)
