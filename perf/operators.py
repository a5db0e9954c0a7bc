"""Operators of serving and of the residual stream around the framework's layers, as measurable cases.

  prefill   the Mamba-3 selective scan of packed prompts of different lengths on a pool of recurrent states: prompts that
            start from nothing and prompts that go on from their state, in both parameter layouts
  step      the same recurrence for one token of every sequence, the state updated in place
  conv      the short causal convolution that stands in front of both scans, on a pool of the last inputs: packed prompts, or
            one token of every sequence
  norm      the norms before and after a block, fused with its gate, the residual scale and the addition to the residual
            stream: forward, or every gradient

``listed()`` names a dozen, ``draw()`` gives others of the same ranges.  ``run()`` computes a case with elementary torch
operations, or, where ``own`` is true, with the framework's entry points; ``exact()`` from the definition in 64 bits.
"""
import math
import random

import torch

own = False

BF16, F32 = "bf16", "f32"
DT = {BF16: torch.bfloat16, F32: torch.float32}


def listed():
    return [
        # one user's short question: one prompt of 37 tokens for a small layer, where launches and latency count
        dict(name="prefill_one_short", kind="prefill", io=BF16, S=1, T=37, slots=1, D=512, N=128, G=1, nheads=8, go_on=False, split=1),
        # a serving batch: sixteen prompts of uneven lengths, half of them later parts of longer prompts; the layer is the
        # Mamba-3 training configuration's (32 heads of 64 channels, 128 states)
        dict(name="prefill_batch", kind="prefill", io=BF16, S=16, T=32768, slots=24, D=2048, N=128, G=1, nheads=32, go_on=True, split=2),
        # one long document for a narrow layer: few heads, so that the time axis has to be split
        dict(name="prefill_long", kind="prefill", io=BF16, S=1, T=16381, slots=1, D=512, N=128, G=1, nheads=8, go_on=False, split=3),
        # prompts of the reference's larger training run's layer: float32, parameters of every channel and state
        dict(name="prefill_channels_f32", kind="prefill", io=F32, S=7, T=4003, slots=8, D=448, N=16, G=4, nheads=0, go_on=True, split=4),
        # one user's next token: 1 MB of state, the smallest call there is
        dict(name="step_one", kind="step", io=BF16, S=1, slots=1, D=2048, N=128, G=1, nheads=32),
        # the next token of a full batch, in a pool with other sequences
        dict(name="step_256", kind="step", io=BF16, S=256, slots=300, D=2048, N=128, G=1, nheads=32),
        # the next token of a batch for a layer with parameters of every channel, float32
        dict(name="step_channels_f32", kind="step", io=F32, S=61, slots=64, D=448, N=16, G=4, nheads=0),
        # the convolution of the serving batch's prompts
        dict(name="conv_batch", kind="conv", io=BF16, S=16, T=32768, slots=24, D=2048, K=4, silu=False, go_on=True, split=2),
        # the convolution of the next token of a full batch, as a gated_deltanet layer has it (an odd width, SiLU behind it)
        dict(name="conv_step", kind="conv", io=F32, S=256, T=0, slots=300, D=449, K=4, silu=True, go_on=True, split=0),
        # the residual stream between two layers for one token: only latency
        dict(name="norm_one", kind="norm", io=BF16, rows=1, D=2048, res=F32, grad=False, post=True, gate=False, scale=True),
        # a prefill's rows with everything on
        dict(name="norm_prefill", kind="norm", io=BF16, rows=8191, D=2048, res=F32, grad=False, post=True, gate=True, scale=True),
        # the training configuration's tokens, gradients of everything
        dict(name="norm_train", kind="norm", io=BF16, rows=8 * 4096, D=2048, res=BF16, grad=True, post=True, gate=True, scale=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("prefill", "prefill", "prefill", "step", "step", "conv", "conv", "norm", "norm"))
    if kind in ("prefill", "step"):
        if rng.random() < 0.7:  # heads that share their parameters
            nheads = rng.choice((1, 2, 4, 8, 16, 32))
            c = dict(kind=kind, io=rng.choice((BF16, BF16, BF16, F32)), D=nheads * rng.choice((16, 32, 64, 64, 64, 128)),
                     N=rng.choice((16, 32, 64, 128, 128)), nheads=nheads)
            c["G"] = rng.choice([g for g in (1, 1, 2, 4) if nheads % g == 0])
            most = 32768 * 2048 // c["D"] if c["io"] == BF16 else 8192 * 512 // c["D"]
        else:                   # parameters of every channel
            c = dict(kind=kind, io=rng.choice((BF16, F32)), D=4 * rng.randint(8, 112), N=rng.choice((8, 16, 16, 32)), nheads=0,
                     G=rng.choice((1, 2, 4)))
            most = 4096 * 448 * 16 // (c["D"] * c["N"])
        if kind == "step":
            c["S"] = _log_int(rng, 1, 256)
        else:
            c["T"] = _log_int(rng, 1, min(most, 32768))
            c.update(S=min(_log_int(rng, 1, 64), c["T"]), go_on=rng.random() < 0.5, split=rng.randint(1, 1 << 20))
        c["slots"] = c["S"] + rng.randint(0, 16)
    elif kind == "conv":
        c = dict(kind=kind, io=rng.choice((BF16, BF16, F32)), D=rng.choice((rng.randint(16, 512), 8 * rng.randint(8, 256))),
                 K=rng.choice((2, 3, 4, 4, 4)), silu=rng.random() < 0.5, go_on=True, split=0, T=0, S=_log_int(rng, 1, 256))
        if rng.random() < 0.7:
            c["T"] = _log_int(rng, 1, 32768 * 2048 // max(c["D"], 2048))
            c.update(S=min(c["S"], c["T"]), go_on=rng.random() < 0.5, split=rng.randint(1, 1 << 20))
        c["slots"] = c["S"] + rng.randint(0, 16)
    else:
        io = rng.choice((BF16, BF16, F32))
        c = dict(kind=kind, io=io, D=rng.choice((rng.randint(16, 1024), 8 * rng.randint(16, 512))), res=rng.choice((io, F32)),
                 grad=rng.random() < 0.5, post=rng.random() < 0.6, gate=rng.random() < 0.5, scale=rng.random() < 0.6)
        c["rows"] = _log_int(rng, 1, (8 if io == BF16 else 4) * 4096 * 2048 // max(c["D"], 2048))
    return c


def _lengths(case):
    """T rows cut into S sequences at places drawn from the case's own number; a sequence may be empty."""
    if case["S"] == 1:
        return [case["T"]]
    r = random.Random(case["split"])
    cuts = sorted(r.randint(0, case["T"]) for _ in range(case["S"] - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [case["T"]])]


# ------------------------------------------------------------------ inputs
class _Draw:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda")

    def uniform(self, lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(*shape, generator=self.g, device="cuda")


def _slots(r, case):
    return torch.randperm(case["slots"], generator=r.g, device="cuda")[:case["S"]].int()


def _packed(s, case):
    """Lengths, their running sum on the GPU and which prompts go on from their state."""
    s["lens"] = torch.tensor(_lengths(case))
    s["cu_seqlens"] = torch.cat([torch.zeros(1, dtype=torch.long), s["lens"].cumsum(0)]).int().cuda()
    s["go_on"] = (torch.arange(case["S"], device="cuda") % 2 == 0) & case["go_on"]


def prepare(case, seed):
    r, c, io = _Draw(seed), case, DT[case["io"]]
    s = dict(case)
    if c["kind"] in ("prefill", "step"):
        # what the scan meets: dt before its softplus around -2, decay rates between 1 and 16, angles over the whole circle
        D, N, G, nh, rows, n = c["D"], c["N"], c["G"], c["nheads"], c["T"] if c["kind"] == "prefill" else c["S"], c["slots"]
        per = (rows, nh or D)
        s.update(x=r.normal(rows, D).to(io), b=r.normal(rows, G, N).to(io), c=r.normal(rows, G, N).to(io), dt=-2.0 + 0.5 * r.normal(*per),
                 lam=r.normal(*per), theta=r.uniform(-math.pi, math.pi, *(per if nh else per + (N // 2,))),
                 a_log=r.uniform(0.0, math.log(16.0), *((nh,) if nh else (D, N))))
        angle = r.uniform(-math.pi, math.pi, *((n, nh) if nh else (n, D, N // 2)))
        s["state"] = (0.5 * r.normal(n, D, N), torch.stack((angle.cos(), angle.sin()), -1), r.normal(n, D).to(io),
                      r.normal(n, nh or G, N).to(io))
        if nh:  # (every head of a group keeps the group's last row)
            s["state"][3].copy_(s["state"][3].view(n, G, nh // G, N)[:, :, :1].expand(-1, -1, nh // G, -1).reshape(n, nh, N))
        s["slots"] = _slots(r, c)
        if c["kind"] == "prefill":
            _packed(s, c)
    elif c["kind"] == "conv":
        rows = c["T"] or c["S"]
        s.update(x=r.normal(rows, c["D"]).to(io), w=r.normal(c["D"], c["K"]) / math.sqrt(c["K"]), bias=0.1 * r.normal(c["D"]),
                 state=r.normal(c["slots"], c["K"] - 1, c["D"]).to(io), slots=_slots(r, c))
        if c["T"]:
            _packed(s, c)
    else:
        rows, D = c["rows"], c["D"]
        s.update(resid=(2.0 * r.normal(rows, D)).to(DT[c["res"]]), y=r.normal(rows, D).to(io), norm=1.0 + 0.1 * r.normal(D),
                 post_norm=1.0 + 0.1 * r.normal(D) if c["post"] else None, z=r.normal(rows, D).to(io) if c["gate"] else None,
                 scale=0.5 + 0.1 * r.normal(D) if c["scale"] else None, eps=1e-5)
        if c["grad"]:
            s.update(d_resid=r.normal(rows, D).to(DT[c["res"]]), dn=r.normal(rows, D).to(io))
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return _own(s) if own else _PLAIN[s["kind"]](s)


def _own(s):
    from mixlab_b200 import ops
    if s["kind"] in ("prefill", "step"):
        state = ops.Mamba3State(*s["state"])
        if s["kind"] == "prefill":
            y = ops.mamba3_prefill(s["x"], s["dt"], s["lam"], s["theta"], s["a_log"], s["b"], s["c"], s["cu_seqlens"], state,
                                   slots=s["slots"], go_on=s["go_on"], nheads=s["nheads"])
        else:
            y = ops.mamba3_decode_step(state, s["x"], s["dt"], s["lam"], s["theta"], s["a_log"], s["b"], s["c"], slots=s["slots"],
                                       nheads=s["nheads"])
        return dict(y=y, **state._asdict())
    if s["kind"] == "conv":
        act = "silu" if s["silu"] else None
        if s["T"]:
            y = ops.short_conv_prefill(s["x"], s["w"], s["cu_seqlens"], s["state"], slots=s["slots"], go_on=s["go_on"], bias=s["bias"],
                                       activation=act)
        else:
            y = ops.short_conv_step(s["state"], s["x"], s["w"], slots=s["slots"], bias=s["bias"], activation=act)
        return dict(y=y, state=s["state"])
    kw = dict(post_norm=s["post_norm"], z=s["z"], scale=s["scale"], eps=s["eps"])
    if not s["grad"]:
        resid, n = ops.residual_norm(s["resid"], s["y"], s["norm"], **kw)
        return dict(resid=resid, n=n)
    return ops.residual_norm_backward(s["resid"], s["y"], s["norm"], s["d_resid"], s["dn"], **kw)


# ------------------------------------------------------------------ plain forms
def _rotate(v, phi):
    """Pairs (even, odd) of the last axis turned back by phi."""
    v = v.unflatten(-1, (-1, 2))
    c, s = phi.cos().float(), phi.sin().float()
    return torch.stack((c * v[..., 0] + s * v[..., 1], c * v[..., 1] - s * v[..., 0]), -1).flatten(-2)


def _table(lens, Q):
    """The chunks of Q rows of every sequence: their rows [C, Q], which of them there are, the sequence of each chunk, the
    chunk's number in it, and for each sequence its first row and the chunk behind its last."""
    start, chunks = lens.cumsum(0) - lens, (lens + Q - 1) // Q
    seq = torch.repeat_interleave(torch.arange(len(lens)), chunks)
    nth = torch.arange(len(seq)) - (chunks.cumsum(0) - chunks)[seq]
    rows = start[seq][:, None] + nth[:, None] * Q + torch.arange(Q)
    there = rows < (start + lens)[seq][:, None]
    return [t.cuda() for t in (torch.where(there, rows, rows[:, :1]), there, seq, nth, start, chunks.cumsum(0))]


def _prefill(s):
    """In chunks: products within a chunk, the state that every chunk adds, and what has reached each chunk of all chunks in
    front of it in its sequence.  A step's outer product counts g = lam dt for its own step and e = g + (1 - lam) dt of the
    step behind it for all later ones.  Angles and running sums of the decay in 64 bits."""
    D, N, G, nh = s["D"], s["N"], s["G"], s["nheads"]
    H, heads = nh or D, nh > 0
    h, phase, x_prev, b_prev = s["state"]
    lens, slots = s["lens"], s["slots"].long()
    Q = 64 if heads else 16
    rows, there, seq, nth, start, behind = _table(lens, Q)
    dt = torch.logaddexp(s["dt"].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    lam = torch.sigmoid(s["lam"].double())
    theta = s["theta"].double() if not heads else s["theta"].double()[..., None]
    T = dt.shape[0]
    length = lens.cuda()
    of = torch.repeat_interleave(torch.arange(len(lens)), lens).cuda()
    last = (start + length - 1)[of] == torch.arange(T, device="cuda")

    def running(v):  # sums within each sequence, this step's among them
        t = torch.cat([torch.zeros_like(v[:1]), v.cumsum(0)])
        return t[1:] - t[start[of]]

    start_angle = torch.atan2(phase[slots][..., 1].double(), phase[slots][..., 0].double())
    start_angle = torch.where(s["go_on"].view(-1, *(1,) * (start_angle.dim() - 1)), start_angle, 0.0)
    start_angle = start_angle[..., None] if heads else start_angle
    phi = running(dt[..., None] * theta) + start_angle[of]                # [T, H, 1 or N/2]
    tau = running(dt)                                                     # [T, H]
    look = (1.0 - lam) * dt
    g = lam * dt
    e = g + torch.where(last[:, None], 0.0, torch.cat([look[1:], look[:1]]))
    rep = H // G
    br = _rotate(s["b"].float().repeat_interleave(rep, 1), phi)           # [T, H, N]
    cr = _rotate(s["c"].float().repeat_interleave(rep, 1), phi)
    A = -torch.exp(s["a_log"].double())
    A = A[:, None].expand(H, N) if heads else A                           # [H, N]
    x = s["x"].float().unflatten(-1, (H, -1))                             # [T, H, P]
    P = x.shape[-1]
    # what a prompt starts from: its state, and the step in front of its first
    h0 = h[slots].unflatten(1, (H, P))
    bp = b_prev[slots].float().repeat_interleave(H // b_prev.shape[1], 1)
    bp = _rotate(bp, start_angle)
    first = start.clamp(max=T - 1)
    h0 = h0 + look[first].float()[..., None, None] * x_prev[slots].float().unflatten(-1, (H, P))[..., None] * bp[:, :, None]
    h0 = torch.where(s["go_on"][:, None, None, None], h0, 0.0)            # [S, H, P, N]

    m = there[..., None]
    e_c, g_c = torch.where(m, e[rows], 0.0), torch.where(m, g[rows], 0.0)  # [C, Q, H]
    end = torch.where(there, rows, 0).amax(1)
    tau_c, tau_end = tau[rows], tau[end]                                  # [C, Q, H], [C, H]
    tau_in = torch.where((nth == 0)[:, None], 0.0, torch.cat([tau_end[:1], tau_end[:-1]]))
    x_c, b_c, c_c = x[rows], br[rows], cr[rows]
    causal = torch.ones(Q, Q, dtype=torch.bool, device="cuda").tril()
    before = torch.ones(Q, Q, dtype=torch.bool, device="cuda").tril(-1)
    diff = (tau_c[:, :, None] - tau_c[:, None]).clamp(min=0.0)            # [C, i, j, H]
    weight = torch.where(before[..., None], e_c[:, None], g_c[:, None]) * causal[..., None]
    between = (seq[:, None] == seq) & (nth[:, None] > nth)                # [c, c'] the second in front of the first
    if heads:
        a = A[:, 0]
        w = (torch.exp(a * diff) * weight).float()
        y = torch.einsum("cijh,cijh,cjhp->cihp", torch.einsum("cihn,cjhn->cijh", c_c, b_c), w, x_c)
        to_end = (torch.exp(a * (tau_end[:, None] - tau_c)) * e_c).float()
        adds = torch.einsum("cjhp,cjhn->chpn", x_c * to_end[..., None], b_c)
        over = torch.where(between[..., None], torch.exp(a * (tau_in[:, None] - tau_end).clamp(min=0.0)), 0.0).float()
        h_in = torch.einsum("cdh,dhpn->chpn", over, adds) + torch.exp(a * tau_in).float()[..., None, None] * h0[seq]
        y = y + torch.exp(a * (tau_c - tau_in[:, None])).float()[..., None] * torch.einsum("cihn,chpn->cihp", c_c, h_in)
        h_out = torch.exp(a * (tau_end - tau_in)).float()[..., None, None] * h_in + adds
    else:
        f = A.float()
        u = x_c * b_c                                                     # [C, Q, H, N]
        w = torch.exp(f * diff.float()[..., None]) * weight.float()[..., None]
        states = torch.einsum("cijhn,cjhn->cihn", w, u)
        to_end = torch.exp(f * (tau_end[:, None] - tau_c).float()[..., None]) * e_c.float()[..., None]
        adds = (to_end * u).sum(1)
        over = torch.exp(f * (tau_in[:, None] - tau_end).clamp(min=0.0).float()[..., None]) * between[..., None, None]
        h_in = torch.einsum("cdhn,dhn->chn", over, adds) + torch.exp(f * tau_in.float()[..., None]) * h0[seq][:, :, 0]
        states = states + torch.exp(f * (tau_c - tau_in[:, None]).float()[..., None]) * h_in[:, None]
        y = (states * c_c).sum(-1)[..., None]
        h_out = (torch.exp(f * (tau_end - tau_in).float()[..., None]) * h_in + adds)[:, :, None]
    out = s["x"].new_empty(T, D)
    out[rows[there]] = y[there].flatten(1).to(out.dtype)
    some = (length > 0).nonzero()[:, 0]
    at, final = slots[some], (start + length - 1)[some]
    h[at] = h_out[behind[some] - 1].flatten(1, 2)
    turn = phi[final]
    phase[at] = (torch.stack((turn.cos(), turn.sin()), -1).squeeze(2) if heads else torch.stack((turn.cos(), turn.sin()), -1)).float()
    x_prev[at] = s["x"][final]
    b_prev[at] = s["b"][final].repeat_interleave(b_prev.shape[1] // G, 1)
    return dict(y=out, h=h, phase=phase, x_prev=x_prev, b_prev=b_prev)


def _step(s):
    D, N, G, nh = s["D"], s["N"], s["G"], s["nheads"]
    H = nh or D
    h, phase, x_prev, b_prev = s["state"]
    at = s["slots"].long()
    dt = torch.logaddexp(s["dt"], torch.zeros((), device="cuda"))
    lam = torch.sigmoid(s["lam"])
    old = torch.atan2(phase[at][..., 1].double(), phase[at][..., 0].double())
    new = old + (dt if nh else dt[..., None]).double() * s["theta"].double()
    spread = (lambda t: t[..., None]) if nh else (lambda t: t)
    bp = _rotate(b_prev[at].float().repeat_interleave(H // b_prev.shape[1], 1), spread(old))
    br = _rotate(s["b"].float().repeat_interleave(H // G, 1), spread(new))
    cr = _rotate(s["c"].float().repeat_interleave(H // G, 1), spread(new))
    A = -torch.exp(s["a_log"])
    alpha = torch.exp(dt[..., None] * (A[:, None] if nh else A))          # [S, H, 1 or N]
    x, xp = s["x"].float().unflatten(-1, (H, -1)), x_prev[at].float().unflatten(-1, (H, -1))
    v = h[at].unflatten(1, (H, -1))
    v = alpha[:, :, None] * (v + ((1.0 - lam) * dt)[..., None, None] * xp[..., None] * bp[:, :, None])
    v = v + (lam * dt)[..., None, None] * x[..., None] * br[:, :, None]
    y = (v * cr[:, :, None]).sum(-1).flatten(1).to(s["x"].dtype)
    h[at] = v.flatten(1, 2)
    phase[at] = torch.stack((new.cos(), new.sin()), -1).float()
    x_prev[at] = s["x"]
    b_prev[at] = s["b"].repeat_interleave(b_prev.shape[1] // G, 1)
    return dict(y=y, h=h, phase=phase, x_prev=x_prev, b_prev=b_prev)


def _conv(s):
    """Every output row gathers its K inputs from the rows of its sequence and of its state."""
    x, w, state, slots, K = s["x"], s["w"], s["state"], s["slots"].long(), s["K"]
    if s["T"]:
        lens, go_on = s["lens"].cuda(), s["go_on"]
        of = torch.repeat_interleave(torch.arange(s["S"]), s["lens"]).cuda()
    else:
        lens, go_on = torch.ones(s["S"], dtype=torch.long, device="cuda"), torch.ones(s["S"], dtype=torch.bool, device="cuda")
        of = torch.arange(s["S"], device="cuda")
    start, S = lens.cumsum(0) - lens, s["S"]
    old = torch.where(go_on[:, None, None], state[slots], torch.zeros((), dtype=state.dtype, device="cuda")).flatten(0, 1)
    rows = torch.cat([old, x])                                            # the state's rows of all sequences, then the inputs

    def place(seq, pos):  # the row of a sequence's input at pos, which is in its state where it is below 0
        return torch.where(pos < 0, seq * (K - 1) + K - 1 + pos, S * (K - 1) + start[seq] + pos)

    pos = torch.arange(x.shape[0], device="cuda") - start[of]
    taps = rows[place(of[:, None], pos[:, None] - torch.arange(K, device="cuda"))].float()  # [T, K, D]
    y = (taps * w.t()).sum(1) + s["bias"]
    if s["silu"]:
        y = y * torch.sigmoid(y)
    kept = rows[place(torch.arange(S, device="cuda")[:, None], lens[:, None] + torch.arange(1 - K, 0, device="cuda"))]
    state[slots] = torch.where((lens > 0)[:, None, None], kept, state[slots])
    return dict(y=y.to(x.dtype), state=state)


def _norm(s):
    r, y, eps = s["resid"].float(), s["y"].float(), s["eps"]
    rn = torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) if s["post"] else 1.0
    pn = s["post_norm"] if s["post"] else 1.0
    z = s["z"].float() if s["gate"] else None
    gate = z * torch.sigmoid(z) if s["gate"] else 1.0
    scale = s["scale"] if s["scale"] is not None else 1.0
    a = y * rn * pn * gate
    if not s["grad"]:
        out = r + scale * a
        n = out * torch.rsqrt((out * out).mean(-1, keepdim=True) + eps) * s["norm"]
        return dict(resid=out.to(s["resid"].dtype), n=n.to(s["y"].dtype))
    # here resid is what the forward returned
    k = torch.rsqrt((r * r).mean(-1, keepdim=True) + eps)
    dn = s["dn"].float()
    t = dn * s["norm"]
    d = s["d_resid"].float() + k * (t - r * (k * k * (t * r).mean(-1, keepdim=True)))
    da = d * scale
    t = da * pn * gate
    dy = rn * (t - y * (rn * rn * (t * y).mean(-1, keepdim=True))) if s["post"] else t
    dz = None
    if s["gate"]:
        sg = torch.sigmoid(z)
        dz = (da * y * rn * pn * (sg * (1.0 + z * (1.0 - sg)))).to(s["z"].dtype)
    return dict(d_resid=d.to(s["resid"].dtype), dy=dy.to(s["y"].dtype), dz=dz, dnorm=(dn * r * k).sum(0),
                dpost_norm=(da * y * rn * gate).sum(0) if s["post"] else None, dscale=(d * a).sum(0) if s["scale"] is not None else None)


_PLAIN = {"prefill": _prefill, "step": _step, "conv": _conv, "norm": _norm}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, io = case, 2 if case["io"] == BF16 else 4
    if c["kind"] in ("prefill", "step"):
        D, N, G, nh = c["D"], c["N"], c["G"], c["nheads"]
        H = nh or D
        rows = c["T"] if c["kind"] == "prefill" else c["S"]
        per_row = io * (2 * D + 2 * G * N) + 4 * (2 * H + (nh or D * N // 2))
        per_state = 4 * D * N + 8 * (nh or D * N // 2) + io * (D + (nh or G) * N)
        state_moves = 2 * c["S"] if c["kind"] == "step" else sum(n > 0 for n in _lengths(c)) * 2 - sum(n > 0 and not (c["go_on"] and i % 2 == 0)
                                                                                                       for i, n in enumerate(_lengths(c)))
        # the recurrence itself: decay, two outer products, read-out; rotations of b and c per head or channel
        return dict(bytes=rows * per_row + state_moves * per_state + 4 * (nh or D * N), flops=rows * (8 * D * N + 6 * H * N))
    if c["kind"] == "conv":
        D, K, rows = c["D"], c["K"], c["T"] or c["S"]
        return dict(bytes=2 * io * rows * D + 4 * D * (K + 1) + 2 * io * c["S"] * (K - 1) * D, flops=rows * D * (2 * K + 4 * c["silu"]))
    n, res = c["rows"] * c["D"], 2 if c["res"] == BF16 else 4
    if not c["grad"]:
        return dict(bytes=n * (2 * res + io * (2 + c["gate"])) + 12 * c["D"], flops=n * 16)
    return dict(bytes=n * (3 * res + io * (3 + 2 * c["gate"])) + 24 * c["D"], flops=n * 40)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))


def _walk(s, lens):
    """The recurrence step by step, all sequences side by side.  A head, or a channel with a head of its own."""
    D, N, G, nh = s["D"], s["N"], s["G"], s["nheads"]
    H = nh or D
    P, K = D // H, N // 2
    f = lambda t: t.double()  # noqa: E731
    h, phase, x_prev, b_prev = (f(t) for t in s["state"])
    slots = s["slots"].long()
    A = -torch.exp(f(s["a_log"])).view(H, 1, -1)
    dt_all, lam_all = torch.nn.functional.softplus(f(s["dt"])), torch.sigmoid(f(s["lam"]))
    theta_all = f(s["theta"]).view(-1, H, nh and 1 or K)
    x_all, b_all, c_all = f(s["x"]).view(-1, H, P), f(s["b"]), f(s["c"])
    start = torch.cat([torch.zeros(1, dtype=torch.long), torch.tensor(lens).cumsum(0)[:-1]]).cuda()
    length = torch.tensor(lens).cuda()
    goes = s["go_on"].double() if "go_on" in s else torch.ones(len(lens), dtype=torch.float64, device="cuda")
    ph = torch.atan2(phase[slots][..., 1], phase[slots][..., 0]).view(len(lens), H, -1) * goes.view(-1, 1, 1)
    v = h[slots].view(-1, H, P, K, 2) * goes.view(-1, 1, 1, 1, 1)
    back = b_prev[slots].repeat_interleave(H // b_prev.shape[1], 1).view(-1, H, K, 2)
    xb = x_prev[slots].view(-1, H, P) * goes.view(-1, 1, 1)

    def turned(t, ang):
        co, si = torch.cos(ang), torch.sin(ang)
        return torch.stack((co * t[..., 0] + si * t[..., 1], -si * t[..., 0] + co * t[..., 1]), -1)

    y = torch.zeros(x_all.shape, dtype=torch.float64, device="cuda")
    prev = turned(back, ph)[:, :, None] * xb[..., None, None]             # the outer product of the step before
    order = sorted(range(len(lens)), key=lambda i: -lens[i])              # those that still run stand in front
    idx = torch.tensor(order).cuda()
    ph, v, prev, start, length, slots = ph[idx], v[idx], prev[idx], start[idx], length[idx], slots[idx]
    live = sorted(lens, reverse=True)
    n = len(live)
    for t in range(live[0] if live else 0):
        while n and live[n - 1] <= t:
            n -= 1
        row = start[:n] + t
        dt, lam = dt_all[row], lam_all[row]
        ph[:n] += dt[..., None] * theta_all[row]
        br = turned(b_all[row].view(n, G, 1, K, 2).expand(n, G, H // G, K, 2).reshape(n, H, K, 2), ph[:n])
        cr = turned(c_all[row].view(n, G, 1, K, 2).expand(n, G, H // G, K, 2).reshape(n, H, K, 2), ph[:n])
        alpha = torch.exp(dt[..., None, None] * A).view(n, H, 1, -1, 2 if not nh else 1)
        now = br[:, :, None] * x_all[row][..., None, None]
        v[:n] = alpha * (v[:n] + ((1 - lam) * dt)[..., None, None, None] * prev[:n]) + (lam * dt)[..., None, None, None] * now
        prev[:n] = now
        y[row] = (v[:n] * cr[:, :, None]).sum((-1, -2))
    some = length > 0
    at, final = slots[some], (start + length - 1)[some]
    h[at] = v[some].reshape(-1, D, N)
    ph = ph[some]
    phase[at] = torch.stack((ph.cos(), ph.sin()), -1).view(-1, *phase.shape[1:])
    x_prev[at] = x_all[final].reshape(-1, D)
    b_prev[at] = b_all[final].repeat_interleave(b_prev.shape[1] // G, 1)
    return dict(y=y.view(-1, D), h=h, phase=phase, x_prev=x_prev, b_prev=b_prev)


def _exact_conv(s):
    x, w, state, bias = s["x"].double(), s["w"].double(), s["state"].double(), s["bias"].double()
    K, lens = s["K"], s["lens"].tolist() if s["T"] else [1] * s["S"]
    goes = s["go_on"].tolist() if s["T"] else [True] * s["S"]
    y, at = torch.empty_like(x), 0
    for i, n in enumerate(lens):
        slot = int(s["slots"][i])
        line = torch.cat([state[slot] if goes[i] else torch.zeros_like(state[slot]), x[at:at + n]])
        y[at:at + n] = sum(line[K - 1 - k:K - 1 - k + n] * w[:, k] for k in range(K)) + bias
        if n:
            state[slot] = line[n:]
        at += n
    return dict(y=y / (1 + torch.exp(-y)) if s["silu"] else y, state=state)


def _exact_norm(s):
    leaf = {n: s[n].double().requires_grad_() for n in ("y", "norm", "post_norm", "z", "scale") if s[n] is not None}
    unit = lambda t: t / torch.sqrt(t.square().sum(-1, keepdim=True) / t.shape[-1] + s["eps"])  # noqa: E731
    a = leaf["y"]
    if s["post"]:
        a = unit(a) * leaf["post_norm"]
    if s["gate"]:
        a = a * leaf["z"] / (1 + torch.exp(-leaf["z"]))
    if "scale" in leaf:
        a = a * leaf["scale"]
    r = s["resid"].double()
    if not s["grad"]:
        out = r + a
        return dict(resid=out.detach(), n=(unit(out) * leaf["norm"]).detach())
    r.requires_grad_()
    (d_norm, d) = torch.autograd.grad((unit(r) * leaf["norm"] * s["dn"].double()).sum(), (leaf["norm"], r))
    d = d + s["d_resid"].double()
    names = [n for n in leaf if n != "norm"]
    g = dict(zip(names, torch.autograd.grad((a * d).sum(), [leaf[n] for n in names])))
    return dict(d_resid=d, dy=g["y"], dz=g.get("z"), dnorm=d_norm, dpost_norm=g.get("post_norm"), dscale=g.get("scale"))


_EXACT = {"prefill": lambda s: _walk(s, s["lens"].tolist()), "step": lambda s: _walk(s, [1] * s["S"]), "conv": _exact_conv, "norm": _exact_norm}
