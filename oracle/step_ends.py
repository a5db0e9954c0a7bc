"""The ends of a training step in float64: the token rows, the layer norm, the output head's loss, each with its gradients from the
formulas.  Everything is computed in the type that the arguments have."""
import torch


def _real(tokens, V):
    return (tokens >= 0) & (tokens < V)


def embedding(tokens, weight, scale=1.0):
    out = weight.new_zeros(*tokens.shape, weight.shape[1])
    ok = _real(tokens, weight.shape[0])
    out[ok] = scale * weight[tokens[ok].long()]
    return out


def embedding_backward(tokens, d_out, V, scale=1.0):
    """The gradient, and the sums of absolute values and the numbers of terms behind its elements."""
    ok = _real(tokens, V)
    at, rows = tokens[ok].long(), d_out[ok]
    dw, size = d_out.new_zeros(V, d_out.shape[-1]), d_out.new_zeros(V, d_out.shape[-1])
    dw.index_add_(0, at, rows)
    size.index_add_(0, at, rows.abs())
    return scale * dw, abs(scale) * size, torch.bincount(at, minlength=V)


def layer_norm(x, weight, bias=None, resid=None, eps=1e-5):
    h = x if resid is None else resid + x
    u = h - h.mean(-1, keepdim=True)
    n = u * torch.rsqrt(u.square().mean(-1, keepdim=True) + eps) * weight
    return h, n if bias is None else n + bias


def layer_norm_backward(x, weight, dn, d_resid=None, eps=1e-5):
    u = x - x.mean(-1, keepdim=True)
    k = torch.rsqrt(u.square().mean(-1, keepdim=True) + eps)
    u, t = u * k, dn * weight
    dx = k * (t - t.mean(-1, keepdim=True) - u * (t * u).mean(-1, keepdim=True))
    rows = tuple(range(x.dim() - 1))
    return dict(dx=dx if d_resid is None else d_resid + dx, dweight=(dn * u).sum(rows), dbias=dn.sum(rows))


def linear_cross_entropy(x, weight, targets):
    """loss and lse; a target outside 0 .. V-1 gives zeros, whatever its x holds."""
    ok = _real(targets, weight.shape[0])
    loss, lse = x.new_zeros(targets.shape), x.new_zeros(targets.shape)
    z = x[ok] @ weight.T
    lse[ok] = torch.logsumexp(z, -1)
    loss[ok] = lse[ok] - z.gather(-1, targets[ok].long()[:, None])[:, 0]
    return loss, lse


def linear_cross_entropy_backward(x, weight, targets, lse, d_loss, d_lse=None):
    """Tokens whose target is outside 0 .. V-1, or whose gradients are zero, have no part, whatever their x holds."""
    ok = _real(targets, weight.shape[0]) & ((d_loss != 0) | (torch.zeros_like(d_loss) if d_lse is None else d_lse).ne(0))
    rows, a = x[ok], d_loss[ok][:, None]
    both = a if d_lse is None else a + d_lse[ok][:, None]
    g = both * torch.exp(rows @ weight.T - lse[ok][:, None])
    g.scatter_add_(1, targets[ok].long()[:, None], -a)
    dx = torch.zeros_like(x)
    dx[ok] = g @ weight
    return dict(dx=dx, dweight=g.T @ rows)
