"""CPU restatement of the serving operators and of the residual stage - TEST INFRASTRUCTURE ONLY.

Sequences one after the other, step by step, in the type of the inputs (float64 in the tests).  The scan is the recurrence of
``oracle/mamba3.py`` (gpu/cuda_kernels/mamba3_selective_scan_fwd_v2_emit.cu:65-115) with a state that goes in and comes out; the
convolution that of gpu/ir.cpp:1397-1425 and arch/blocks_gated_deltanet.go:345-368 behind the inputs of the past.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .mamba3 import rotate_pairs


def mamba3_rows(state, x, dt, lam, theta, a_log, b, c, nheads):
    """The rows of one sequence on state = (h [D,N], phase, x_prev [D], b_prev [nheads or G, N]).  Returns y and the new state."""
    h, phase, x_prev, b_prev = (t.clone() for t in state)
    rows, D = x.shape
    G, N = b.shape[1:]
    H = nheads or D
    P = D // H
    phi = torch.atan2(phase[..., 1], phase[..., 0])                       # [nheads] or [D, N/2]
    wide = (lambda t: t.repeat_interleave(P, 0)) if nheads else (lambda t: t)
    angles = (lambda p: p.repeat_interleave(P)[:, None].expand(D, N // 2)) if nheads else (lambda p: p)
    A = -torch.exp(a_log)
    A = A.repeat_interleave(P)[:, None].expand(D, N) if nheads else A
    prev = rotate_pairs(b_prev.repeat_interleave(D // b_prev.shape[0], 0), angles(phi))
    y = torch.empty_like(x)
    for t in range(rows):
        d, l = F.softplus(dt[t]), torch.sigmoid(lam[t])
        phi = phi + (d if nheads else d[:, None]) * theta[t]
        d, l = wide(d)[:, None], wide(l)[:, None]
        br = rotate_pairs(b[t].repeat_interleave(D // G, 0), angles(phi))
        cr = rotate_pairs(c[t].repeat_interleave(D // G, 0), angles(phi))
        h = torch.exp(d * A) * (h + (1 - l) * d * prev * x_prev[:, None]) + l * d * br * x[t][:, None]
        y[t] = (h * cr).sum(-1)
        prev, x_prev = br, x[t]
    if rows:
        phase = torch.stack((torch.cos(phi), torch.sin(phi)), -1)
        x_prev, b_prev = x[-1].clone(), b[-1].repeat_interleave(b_prev.shape[0] // G, 0)
    return y, (h, phase, x_prev, b_prev)


def fresh_mamba3_state(D, N, G, nheads, dtype=torch.float64):
    phase = torch.zeros(*((nheads,) if nheads else (D, N // 2)), 2, dtype=dtype)
    phase[..., 0] = 1
    return torch.zeros(D, N, dtype=dtype), phase, torch.zeros(D, dtype=dtype), torch.zeros(nheads or G, N, dtype=dtype)


def mamba3_prefill(pool, x, dt, lam, theta, a_log, b, c, lens, slots, go_on, nheads):
    """Packed prompts on a pool of states (four tensors, changed in place).  Rows of no sequence come back as NaN."""
    D, (G, N) = x.shape[1], b.shape[1:]
    y, at = torch.full_like(x, float("nan")), 0
    for i, n in enumerate(lens):
        r = slice(at, at + n)
        at += n
        if n == 0:
            continue
        keeps = 0 <= slots[i] < pool[0].shape[0]
        state = tuple(t[slots[i]] for t in pool) if go_on[i] and keeps else fresh_mamba3_state(D, N, G, nheads, x.dtype)
        y[r], new = mamba3_rows(state, x[r], dt[r], lam[r], theta[r], a_log, b[r], c[r], nheads)
        if keeps:
            for t, v in zip(pool, new):
                t[slots[i]] = v
    return y


def short_conv(pool, x, w, bias, lens, slots, go_on, silu):
    """Packed prompts on a pool of the last K-1 inputs (changed in place).  Rows of no sequence come back as NaN."""
    K, y, at = w.shape[1], torch.full_like(x, float("nan")), 0
    for i, n in enumerate(lens):
        if n == 0:
            continue
        keeps = 0 <= slots[i] < pool.shape[0]
        line = torch.cat([pool[slots[i]] if go_on[i] and keeps else x.new_zeros(K - 1, x.shape[1]), x[at:at + n]])
        o = sum(line[K - 1 - k:K - 1 - k + n] * w[:, k] for k in range(K))
        o = o if bias is None else o + bias
        y[at:at + n] = F.silu(o) if silu else o
        if keeps:
            pool[slots[i]] = line[n:]
        at += n
    return y


def residual_norm(resid, y, norm, post_norm=None, z=None, scale=None, eps=1e-5):
    def unit(t):
        return t * torch.rsqrt((t * t).mean(-1, keepdim=True) + eps)

    a = y if post_norm is None else unit(y) * post_norm
    a = a if z is None else a * F.silu(z)
    out = resid + (a if scale is None else scale * a)
    return out, unit(out) * norm
