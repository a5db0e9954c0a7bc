"""Operators at the two ends of a language model's training step, as measurable cases.

  embed        rows of the token matrix, scaled: the residual stream's first value
  embed_grad   the token matrix's gradient: the rows of the stream's gradient summed by token
  norm         the layer norm over the residual stream, with the addition to the stream in front of it or without
  norm_grad    its gradients: of the stream, of the weight and of the bias
  loss         the output head and its loss: softmax cross entropy of x W^T for every token, with the logarithm of the sum
  loss_grad    its gradients: of x and of the head's matrix

``listed()`` names a dozen, ``draw()`` gives others of the same ranges.  ``run()`` computes a case with elementary torch
operations, or, where ``own`` is true, with the framework's entry points; ``exact()`` from the definition in 64 bits.
"""
import math

import torch

own = False

BF16, F32 = "bf16", "f32"
DT = {BF16: torch.bfloat16, F32: torch.float32}
SIZE = {BF16: 2, F32: 4}


def listed():
    return [
        # the next token of a serving batch of 256 sequences: latency
        dict(name="embed_step", kind="embed", io=BF16, out=BF16, N=256, V=32768, D=2048, scale=1.0, padded=0),
        # the training configuration's tokens (8 x 4096, rows of 2048) into a float32 residual stream
        dict(name="embed_train", kind="embed", io=BF16, out=F32, N=8 * 4096, V=65536, D=2048, scale=math.sqrt(2048.0), padded=0),
        # the reference's larger training run's width with a vocabulary of bytes, an odd number of tokens, some of them padding
        dict(name="embed_grad_bytes", kind="embed_grad", io=F32, out=F32, N=2047, V=257, D=448, scale=1.0, padded=100),
        # the training configuration's tokens, few words often and many seldom, into the float32 buckets of the gradient exchange
        dict(name="embed_grad_train", kind="embed_grad", io=BF16, out=F32, N=8 * 4096, V=65536, D=2048, scale=math.sqrt(2048.0), padded=0),
        # one token of a float32 stream: latency
        dict(name="norm_one", kind="norm", io=BF16, res=F32, N=1, D=2048, add=True),
        # the training configuration's tokens, the stream updated on the way
        dict(name="norm_train", kind="norm", io=BF16, res=BF16, N=8 * 4096, D=2048, add=True),
        # an odd number of odd rows
        dict(name="norm_grad_odd", kind="norm_grad", io=F32, res=F32, N=4001, D=449, add=True),
        # the training configuration's tokens
        dict(name="norm_grad_train", kind="norm_grad", io=BF16, res=BF16, N=8 * 4096, D=2048, add=True),
        # the probability of one text of 512 tokens: the head's matrix is read for few rows
        dict(name="loss_score", kind="loss", io=BF16, N=512, V=32768, D=1024, masked=0),
        # a training step's tokens, an eighth of them behind the ends of texts
        dict(name="loss_train", kind="loss", io=BF16, N=8 * 4096, V=65536, D=1024, masked=4096),
        # the reference's larger training run's width, float32 throughout, a ragged vocabulary
        dict(name="loss_grad_f32", kind="loss_grad", io=F32, N=2048, V=5003, D=448, masked=77),
        # a training step's gradients, a ragged vocabulary
        dict(name="loss_grad_train", kind="loss_grad", io=BF16, N=8 * 4096, V=50001, D=1024, masked=4096),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(("embed", "embed_grad", "norm", "norm_grad", "loss", "loss", "loss_grad", "loss_grad"))
    io = rng.choice((BF16, BF16, F32))
    width = rng.choice((rng.randint(16, 700), 8 * _log_int(rng, 4, 256), 64 * rng.randint(1, 32)))
    c = dict(kind=kind, io=io, D=width)
    if kind in ("embed", "embed_grad"):
        c.update(out=rng.choice((io, F32)), V=_log_int(rng, 50, 65536), N=_log_int(rng, 1, 32768), scale=rng.choice((1.0, math.sqrt(width))))
        c["padded"] = rng.choice((0, c["N"] // 7))
    elif kind in ("norm", "norm_grad"):
        c.update(res=rng.choice((io, F32)), add=rng.random() < 0.5, N=_log_int(rng, 1, 32768 if io == BF16 else 16384))
    else:
        most = 32768 * 50001 * 1024 // (1 if io == BF16 else 64)
        c["V"] = _log_int(rng, 100, min(131072, 65536 * 2048 // width))
        c["N"] = _log_int(rng, 1, min(32768, max(1, most // (c["V"] * width))))
        c["masked"] = rng.choice((0, c["N"] // 8, c["N"] // 2))
    return c


# ------------------------------------------------------------------ inputs
class _Draw:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda")

    def words(self, n, V):
        """Tokens as texts have them: word k about 1 / k as often as the first."""
        u = torch.rand(n, generator=self.g, device="cuda", dtype=torch.float64)
        return (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp_(0, V - 1)

    def some(self, n, k):
        """k of n places."""
        return torch.randperm(n, generator=self.g, device="cuda")[:k]


def prepare(case, seed):
    r, c, io = _Draw(seed), case, DT[case["io"]]
    s, N, D = dict(case), case["N"], case["D"]
    if c["kind"] in ("embed", "embed_grad"):
        s["tokens"] = r.words(N, c["V"])
        s["tokens"][r.some(N, c["padded"])] = -1
        if c["kind"] == "embed":
            s["weight"] = (0.02 * r.normal(c["V"], D)).to(io)
        else:
            s["d_out"] = r.normal(N, D).to(io)
    elif c["kind"] in ("norm", "norm_grad"):
        # a stream whose mean is not zero
        s.update(weight=1.0 + 0.1 * r.normal(D), bias=0.1 * r.normal(D), eps=1e-5)
        stream = (0.5 + 2.0 * r.normal(N, D)).to(DT[c["res"]])
        if c["kind"] == "norm":
            s.update(resid=stream if c["add"] else None, x=r.normal(N, D).to(io) if c["add"] else stream)
        else:
            s.update(x=stream, dn=r.normal(N, D).to(io), d_resid=r.normal(N, D).to(DT[c["res"]]) if c["add"] else None)
    else:
        # rows of a final norm that lean towards their target's row, as a trained model's do
        V, targets = c["V"], r.words(N, c["V"])
        weight = (2.0 / math.sqrt(D)) * r.normal(V, D)
        x = (r.normal(N, D) + 1.5 * weight[targets]).to(io)
        weight, dead = weight.to(io), r.some(N, c["masked"])
        targets[dead] = -1
        s.update(x=x, weight=weight, targets=targets)
        if c["kind"] == "loss_grad":
            # gradients of the mean over the tokens that count; lse is what the forward pass returned
            s.update(lse=_plain_loss(s)["lse"], d_loss=torch.full((N,), 1.0 / max(1, N - c["masked"]), device="cuda"))
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return _own(s) if own else _PLAIN[s["kind"]](s)


def _own(s):
    from mixlab_b200 import ops
    kind = s["kind"]
    if kind == "embed":
        return ops.embedding(s["tokens"], s["weight"], scale=s["scale"], dtype=DT[s["out"]])
    if kind == "embed_grad":
        return ops.embedding_backward(s["tokens"], s["d_out"], s["V"], scale=s["scale"], dtype=DT[s["out"]])
    if kind == "norm":
        out = ops.layer_norm(s["x"], s["weight"], s["bias"], resid=s["resid"], eps=s["eps"], dtype=None if s["add"] else DT[s["io"]])
        return dict(resid=out[0], n=out[1]) if s["add"] else dict(n=out)
    if kind == "norm_grad":
        return ops.layer_norm_backward(s["x"], s["weight"], s["dn"], d_resid=s["d_resid"], eps=s["eps"])
    if kind == "loss":
        loss, lse = ops.linear_cross_entropy(s["x"], s["weight"], s["targets"])
        return dict(loss=loss, lse=lse)
    return ops.linear_cross_entropy_backward(s["x"], s["weight"], s["targets"], s["lse"], s["d_loss"])


# ------------------------------------------------------------------ plain forms
def _plain_embed(s):
    tok = s["tokens"]
    y = s["weight"][tok.clamp(min=0)].float() * s["scale"]
    return torch.where((tok >= 0)[:, None], y, 0.0).to(DT[s["out"]])


def _plain_embed_grad(s):
    tok = s["tokens"]
    # (a row of its own for the padding)
    d = torch.zeros(s["V"] + 1, s["D"], device="cuda")
    d.index_add_(0, torch.where(tok >= 0, tok, s["V"]), s["d_out"].float() * s["scale"])
    return d[:s["V"]].to(DT[s["out"]])


def _moments(h, eps):
    m = h.mean(-1, keepdim=True)
    u = h - m
    k = torch.rsqrt(u.square().mean(-1, keepdim=True) + eps)
    return u * k, k


def _plain_norm(s):
    h = s["x"].float()
    if s["add"]:
        h = s["resid"].float() + h
    n = (_moments(h, s["eps"])[0] * s["weight"] + s["bias"]).to(DT[s["io"]])
    return dict(resid=h.to(DT[s["res"]]), n=n) if s["add"] else dict(n=n)


def _plain_norm_grad(s):
    u, k = _moments(s["x"].float(), s["eps"])
    dn = s["dn"].float()
    t = dn * s["weight"]
    dx = k * (t - t.mean(-1, keepdim=True) - u * (t * u).mean(-1, keepdim=True))
    if s["add"]:
        dx = dx + s["d_resid"].float()
    return dict(dx=dx.to(DT[s["res"]]), dweight=(dn * u).sum(0), dbias=dn.sum(0))


_PIECE = 8192  # rows of the vocabulary at a time


def _plain_loss(s):
    x, weight, tok = s["x"].float(), s["weight"], s["targets"]
    top = torch.full((s["N"],), -math.inf, device="cuda")
    total, hit = torch.zeros_like(top), torch.zeros_like(top)
    for v in range(0, s["V"], _PIECE):
        z = x @ weight[v:v + _PIECE].float().T
        new = torch.maximum(top, z.amax(1))
        total = total * torch.exp(top - new) + torch.exp(z - new[:, None]).sum(1)
        top = new
        here = (tok >= v) & (tok < v + z.shape[1])
        hit = torch.where(here, z.gather(1, (tok - v).clamp(0, z.shape[1] - 1)[:, None])[:, 0], hit)
    lse = top + torch.log(total)
    return dict(loss=torch.where(tok >= 0, lse - hit, 0.0), lse=torch.where(tok >= 0, lse, 0.0))


def _plain_loss_grad(s):
    x, weight, tok = s["x"].float(), s["weight"], s["targets"]
    d = torch.where(tok >= 0, s["d_loss"], 0.0)[:, None]
    dx, dweight = torch.zeros_like(x), torch.empty_like(weight)
    rows = torch.arange(s["N"], device="cuda")
    for v in range(0, s["V"], _PIECE):
        w = weight[v:v + _PIECE].float()
        g = torch.exp(x @ w.T - s["lse"][:, None])
        here = (tok >= v) & (tok < v + w.shape[0])
        at = (tok - v).clamp(0, w.shape[0] - 1)
        g[rows, at] -= here.float()
        g = torch.where(tok[:, None] >= 0, g * d, 0.0)
        dx += g @ w
        dweight[v:v + _PIECE] = (g.T @ x).to(dweight.dtype)
    return dict(dx=dx.to(s["x"].dtype), dweight=dweight)


_PLAIN = {"embed": _plain_embed, "embed_grad": _plain_embed_grad, "norm": _plain_norm, "norm_grad": _plain_norm_grad, "loss": _plain_loss,
          "loss_grad": _plain_loss_grad}


# ------------------------------------------------------------------ work
def work(case):
    c, io, N, D = case, SIZE[case["io"]], case["N"], case["D"]
    if c["kind"] == "embed":  # (no more rows of the matrix than there are)
        n = N - c["padded"]
        return dict(bytes=min(n, c["V"]) * D * io + N * (D * SIZE[c["out"]] + 8), flops=n * D)
    if c["kind"] == "embed_grad":
        n = N - c["padded"]
        return dict(bytes=n * D * io + N * 8 + c["V"] * D * SIZE[c["out"]], flops=2 * n * D)
    if c["kind"] == "norm":
        res = SIZE[c["res"]]
        return dict(bytes=N * D * (2 * res + 2 * io if c["add"] else res + io) + 8 * D, flops=N * D * 8)
    if c["kind"] == "norm_grad":
        res = SIZE[c["res"]]
        return dict(bytes=N * D * (res * (3 if c["add"] else 2) + io) + 12 * D, flops=N * D * 16)
    n = N - c["masked"]  # what a token without a target would cost is not needed
    if c["kind"] == "loss":
        return dict(bytes=(n + c["V"]) * D * io + N * 16, flops=2 * n * c["V"] * D)
    return dict(bytes=(n + N + 2 * c["V"]) * D * io + N * 16, flops=6 * n * c["V"] * D)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))


def _exact_embed(s):
    y = torch.zeros(s["N"], s["D"], dtype=torch.float64, device="cuda")
    real = (s["tokens"] >= 0).nonzero()[:, 0]
    y[real] = s["weight"].double().index_select(0, s["tokens"][real]).mul_(s["scale"])
    return y


def _exact_embed_grad(s):
    real = (s["tokens"] >= 0).nonzero()[:, 0]
    out = torch.zeros(s["V"], s["D"], dtype=torch.float64, device="cuda")
    out.scatter_add_(0, s["tokens"][real][:, None].expand(-1, s["D"]), s["d_out"].double()[real])
    return out.mul_(s["scale"])


def _norm64(h, weight, bias, eps):
    var, mean = torch.var_mean(h, dim=-1, unbiased=False, keepdim=True)
    return (h - mean) / torch.sqrt(var + eps) * weight + bias


def _exact_norm(s):
    h = s["x"].double() + (s["resid"].double() if s["add"] else 0.0)
    n = _norm64(h, s["weight"].double(), s["bias"].double(), s["eps"])
    return dict(resid=h, n=n) if s["add"] else dict(n=n)


def _exact_norm_grad(s):
    h, w, b = (s[k].double().requires_grad_() for k in ("x", "weight", "bias"))
    dx, dw, db = torch.autograd.grad(_norm64(h, w, b, s["eps"]), (h, w, b), s["dn"].double())
    if s["add"]:
        dx = dx + s["d_resid"].double()
    return dict(dx=dx, dweight=dw, dbias=db)


def _live(s):
    return (s["targets"] >= 0).nonzero()[:, 0]


def _exact_loss(s):
    weight = s["weight"].double()
    loss = torch.zeros(s["N"], dtype=torch.float64, device="cuda")
    lse = torch.zeros_like(loss)
    for rows in _live(s).split(4096):
        z = s["x"][rows].double() @ weight.T
        lse[rows] = torch.logsumexp(z, 1)
        loss[rows] = lse[rows] - z.gather(1, s["targets"][rows][:, None])[:, 0]
    return dict(loss=loss, lse=lse)


def _exact_loss_grad(s):
    weight = s["weight"].double()
    dx, dweight = torch.zeros(s["N"], s["D"], dtype=torch.float64, device="cuda"), torch.zeros_like(weight)
    for rows in _live(s).split(2048):
        x = s["x"][rows].double()
        g = (x @ weight.T).sub_(s["lse"][rows].double()[:, None]).exp_()
        g[torch.arange(rows.numel(), device="cuda"), s["targets"][rows]] -= 1.0
        g *= s["d_loss"][rows].double()[:, None]
        dx[rows] = g @ weight
        dweight.addmm_(g.T, x)
    return dict(dx=dx, dweight=dweight)


_EXACT = {"embed": _exact_embed, "embed_grad": _exact_embed_grad, "norm": _exact_norm, "norm_grad": _exact_norm_grad, "loss": _exact_loss,
          "loss_grad": _exact_loss_grad}
