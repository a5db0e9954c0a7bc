"""Packed prompts and single tokens on pools of states (Mamba-3 scan, short convolution) against the float64 oracle.

Tolerances, relative in the 2-norm and in the largest element.  float32 results: every step rounds a few times by at most
2^-24, what it adds decays, and an angle that sums up n steps is off by at most n times half a step of dt theta, which is below
1 here: 400 steps x 2^-24 = 2.4e-5, so 5e-5 for prompts and 2e-6 for a single token (a dozen roundings of 6e-8).  bf16 results:
the rounding of y itself and, on the tensor-core kernels, one each of the weights and of the state that y is read from, each at
most half a step, 2^-8: together at most 3 x 2^-8 = 1.2e-2.  States are float32 whatever the inputs' type and keep the float32
bound; x_prev and b_prev are copies."""
import ctypes as C
import math

import pytest
import torch

from mixlab_b200 import _lib, ops
from oracle import mamba3_block, serving
from util import assert_close

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TOL = {F32: 5e-5, BF16: 1.2e-2}
WALK, SERIAL = _lib.MXB_MAMBA3_RECURRENT_KERNELS, _lib.MXB_MAMBA3_SERIAL_WALK


def scan_inputs(rows, D, N, G, nheads, io, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    u = lambda *s: torch.rand(*s, generator=g)  # noqa: E731
    per = (rows, nheads or D)
    return dict(x=r(rows, D).to(io), dt=-2.0 + 0.5 * r(*per), lam=r(*per),
                theta=(2 * u(*(per if nheads else per + (N // 2,))) - 1) * math.pi,
                a_log=math.log(16.0) * u(*((nheads,) if nheads else (D, N))), b=r(rows, G, N).to(io), c=r(rows, G, N).to(io))


def pool_inputs(slots, D, N, G, nheads, io, seed):
    g = torch.Generator().manual_seed(seed)
    angle = (2 * torch.rand(*((slots, nheads) if nheads else (slots, D, N // 2)), generator=g) - 1) * math.pi
    b_prev = torch.randn(slots, G, N, generator=g).to(io)
    if nheads:
        b_prev = b_prev.repeat_interleave(nheads // G, 1)
    return (0.5 * torch.randn(slots, D, N, generator=g), torch.stack((angle.cos(), angle.sin()), -1),
            torch.randn(slots, D, generator=g).to(io), b_prev)


def cu_of(lens):
    return torch.tensor([0] + lens).cumsum(0).int().cuda()


def double(ts):
    return tuple(t.double() for t in ts)


def gpu_state(pool):
    return ops.Mamba3State(*(t.cuda().contiguous() for t in pool))


def args_of(a, rows=slice(None)):
    return [a[k] if k == "a_log" else a[k][rows] for k in ("x", "dt", "lam", "theta", "a_log", "b", "c")]


def check_state(state, want, io, tol, used):
    """The rows of `used` slots near the oracle's pool."""
    for name, t, w in zip(state._fields, state, want):
        assert_close(t[used].cpu(), w[used].to(t.dtype) if name in ("x_prev", "b_prev") else w[used], 0.0 if name in ("x_prev", "b_prev") else tol, name)


# (D, N, G, nheads)
SHAPES = [(128, 128, 1, 2), (256, 128, 2, 4), (64, 64, 1, 1), (96, 16, 1, 3), (80, 38, 2, 2), (24, 2, 1, 1), (256, 256, 1, 2), (160, 128, 1, 1),
          (512, 96, 1, 8), (48, 16, 4, 0), (40, 16, 1, 0), (9, 6, 3, 0), (20, 80, 2, 0), (8, 256, 1, 0), (128, 2, 1, 0), (36, 64, 1, 0),
          (24, 4, 1, 0), (32, 8, 2, 0), (12, 8, 3, 0), (6, 32, 2, 0), (5, 128, 1, 0)]
LENS = {"one token": [1], "one": [37], "ragged": [64, 0, 1, 130, 65, 0, 63, 2], "longer": [3, 333, 64], "empty ends": [0, 5, 0]}


@pytest.mark.parametrize("lens", LENS.values(), ids=LENS.keys())
@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_prefill(shape, io, lens):
    D, N, G, nheads = shape
    rows, S = sum(lens), len(lens)
    a = scan_inputs(rows, D, N, G, nheads, io, 1)
    pool = pool_inputs(S + 2, D, N, G, nheads, io, 2)
    slots = [(3 * i + 1) % (S + 2) for i in range(S)] if (S + 2) % 3 else list(range(S))[::-1]
    go_on = [i % 2 == 0 for i in range(S)]
    for i in range(S):  # what a sequence that starts anew finds in its row does not matter
        if not go_on[i] and lens[i]:
            for t in pool:
                t[slots[i]] = float("nan")
    want = list(double(pool))
    y_want = serving.mamba3_prefill(want, *double(args_of(a)), lens, slots, go_on, nheads)
    for flags in (0, WALK, WALK | SERIAL):
        state = gpu_state(pool)
        y = ops.mamba3_prefill(*(t.cuda() for t in args_of(a)), cu_of(lens), state, slots=torch.tensor(slots).int().cuda(),
                               go_on=torch.tensor(go_on).cuda(), nheads=nheads, flags=flags)
        assert_close(y.cpu(), y_want, TOL[io], f"y flags {flags}")
        for s in range(S + 2):
            if s in slots and lens[slots.index(s)]:
                check_state(state, want, io, TOL[F32], [s])
            else:  # rows of no sequence, and of sequences without tokens
                for t, w in zip(state, pool):
                    assert torch.equal(t[s].cpu(), w[s])


@pytest.mark.parametrize("shape", [(64, 128, 1, 1), (128, 128, 1, 2), (64, 32, 1, 1), (24, 16, 1, 0)], ids=str)
@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
def test_long_sequences_are_cut(shape, io):
    """Few heads and many steps: the time axis is split, with short prompts beside the long ones."""
    D, N, G, nheads = shape
    lens = [5, 700, 64, 1, 391, 128]
    a = scan_inputs(sum(lens), D, N, G, nheads, io, 3)
    pool = pool_inputs(6, D, N, G, nheads, io, 4)
    go_on = [True, True, False, True, False, True]
    want = list(double(pool))
    y_want = serving.mamba3_prefill(want, *double(args_of(a)), lens, list(range(6)), go_on, nheads)
    d = _lib.Mamba3ServeDesc(sum(lens), 6, 6, D, N, G, nheads, _lib.MXB_F32 if io == F32 else _lib.MXB_BF16, WALK)
    assert _lib.lib().mxb_mamba3_prefill_workspace_bytes(d) > 0  # what a cut needs
    for flags in (0, WALK):
        state = gpu_state(pool)
        y = ops.mamba3_prefill(*(t.cuda() for t in args_of(a)), cu_of(lens), state, go_on=torch.tensor(go_on).cuda(), nheads=nheads, flags=flags)
        assert_close(y.cpu(), y_want, TOL[io], f"y flags {flags}")
        # (700 steps: the bound of the angles grows with them)
        check_state(state, want, io, 2 * TOL[F32], list(range(6)))


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_decode_step(shape, io):
    D, N, G, nheads = shape
    slots = [4, -1, 0, 7, 2, 6]  # -1 and 7: padding
    a = scan_inputs(6, D, N, G, nheads, io, 5)
    pool = pool_inputs(7, D, N, G, nheads, io, 6)
    want = list(double(pool))
    y_want = torch.cat([serving.mamba3_prefill(want, *double(args_of(a, slice(i, i + 1))), [1], [s], [True], nheads) for i, s in enumerate(slots)])
    state = gpu_state(pool)
    out = torch.full((6, D), 7.0, dtype=io).cuda()
    got = ops.mamba3_decode_step(state, *(t.cuda() for t in args_of(a)), slots=torch.tensor(slots).int().cuda(), nheads=nheads, out=out)
    assert got.data_ptr() == out.data_ptr()
    kept, padding = [0, 2, 4, 5], [1, 3]
    assert_close(out[kept].cpu(), y_want[kept], 2e-6 if io == F32 else TOL[BF16], "y")
    assert bool((out[padding] == 7.0).all())
    check_state(state, want, io, 2e-6, [0, 2, 4, 6])
    for t, w in zip(state, pool):
        assert torch.equal(t[[1, 3, 5]].cpu(), w[[1, 3, 5]])


@pytest.mark.parametrize("nheads,io", [(0, F32), (2, F32), (2, BF16)])
def test_prompts_in_parts_then_tokens(nheads, io):
    """A prompt whole, in two parts, and token by token: the same outputs and states."""
    D, N, G = 128, 64, 1
    a = scan_inputs(150, D, N, G, nheads, io, 7)
    dev = [t.cuda() for t in args_of(a)]
    part = lambda lo, hi: [t if i == 4 else t[lo:hi].contiguous() for i, t in enumerate(dev)]  # noqa: E731
    states = [ops.mamba3_state(3, D, N, G, nheads=nheads, dtype=io) for _ in range(3)]
    at, yes = torch.tensor([1]).int().cuda(), torch.tensor([True]).cuda()
    ys = [ops.mamba3_prefill(*dev, cu_of([150]), states[0], slots=at, nheads=nheads)]
    ys.append(torch.cat([ops.mamba3_prefill(*part(lo, hi), cu_of([hi - lo]), states[1], slots=at, go_on=yes, nheads=nheads) for lo, hi in ((0, 101), (101, 150))]))
    steps = [ops.mamba3_prefill(*part(0, 101), cu_of([101]), states[2], slots=at, nheads=nheads)]
    steps += [ops.mamba3_decode_step(states[2], *part(t, t + 1), slots=at, nheads=nheads) for t in range(101, 150)]
    ys.append(torch.cat(steps))
    for y, s in zip(ys[1:], states[1:]):
        assert_close(y, ys[0].double(), TOL[io])
        for t, w in zip(s, states[0]):
            assert_close(t, w.double(), TOL[F32])


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
def test_rows_of_no_sequence_stay(io):
    """Rows behind the last sequence are not written, and what stands there (or in another sequence) reaches nobody."""
    D, N, G, nheads, lens = 128, 128, 1, 2, [70, 33]
    a = scan_inputs(150, D, N, G, nheads, io, 8)
    whole = ops.mamba3_prefill(*(t.cuda() for t in args_of(a, slice(0, 103))), cu_of(lens), ops.mamba3_state(2, D, N, G, nheads=nheads, dtype=io), nheads=nheads)
    for t in args_of(a):
        if t.shape[0] == 150:
            t[103:] = float("nan")
            t[:70] = float("nan")
    out = torch.full((150, D), 3.0, dtype=io).cuda()
    state = ops.mamba3_state(2, D, N, G, nheads=nheads, dtype=io)
    ops.mamba3_prefill(*(t.cuda() for t in args_of(a)), cu_of(lens), state, nheads=nheads, out=out)
    assert bool((out[103:] == 3.0).all()) and torch.equal(out[70:103], whole[70:103])
    assert bool(torch.isnan(out[:70].float()).all()) and bool(torch.isfinite(state.h[1]).all())


@pytest.mark.parametrize("shape", [(128, 128, 1, 2), (24, 16, 1, 0)], ids=str)
def test_angle_that_is_not_finite(shape):
    """From the step with an infinite theta on, everything that the angle turns is NaN, across segments too; nothing before."""
    D, N, G, nheads = shape
    a = scan_inputs(700, D, N, G, nheads, F32, 9)
    a["theta"][200] = float("inf")
    for flags in (WALK, WALK | SERIAL):
        state = ops.mamba3_state(1, D, N, G, nheads=nheads, dtype=F32)
        y = ops.mamba3_prefill(*(t.cuda() for t in args_of(a)), cu_of([700]), state, nheads=nheads, flags=flags)
        assert bool(torch.isfinite(y[:200]).all()) and bool(torch.isnan(y[200:]).all())
        assert bool(torch.isnan(state.phase).all()) and bool(torch.isnan(state.h).all())


@pytest.mark.parametrize("shape", [(128, 128, 1, 2), (64, 64, 1, 1), (24, 16, 1, 0)], ids=str)
@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("name", ["x", "dt", "lam", "theta", "b", "c"])
def test_what_is_not_finite_reaches_no_earlier_row(name, io, shape):
    """A step with an infinity or a NaN leaves the rows in front of it, and the other sequences, what they were."""
    D, N, G, nheads = shape
    lens, first = [50, 167, 50], 50
    a = scan_inputs(267, D, N, G, nheads, io, 19)
    for flags in (0, WALK):
        ys = []
        for value, step in ((None, 0), (float("inf"), 9), (float("nan"), 100), (-float("inf"), 127), (float("nan"), 166)):
            b = {k: v.clone() for k, v in a.items()}
            if value is not None:
                b[name][first + step].view(-1)[0] = value
            state = ops.mamba3_state(3, D, N, G, nheads=nheads, dtype=io)
            ys.append(ops.mamba3_prefill(*(t.cuda() for t in args_of(b)), cu_of(lens), state, nheads=nheads, flags=flags))
            if value is None:
                continue
            assert_close(ys[-1][:first + step].cpu(), ys[0][:first + step].cpu().double(), TOL[io], f"in front of step {step}")
            assert torch.equal(ys[-1][217:], ys[0][217:])
            reached = value != value or name in "xbc"  # (dt, lam of -inf weigh 0)
            assert not reached or not bool(torch.isfinite(ys[-1][first + step].float()).all())
            if name == "x":
                assert bool(torch.isfinite(ys[-1][:, 1:].float()).all())  # the other channels


def test_pool_beyond_32_bit_offsets():
    """Rows of a pool of 2.2 billion elements, the first and the last: 64-bit offsets."""
    D, N, G, nheads, slots = 2048, 128, 1, 32, 8300
    a = scan_inputs(4, D, N, G, nheads, BF16, 10)
    dev = [t.cuda() for t in args_of(a)]
    small, big = ops.mamba3_state(2, D, N, G, nheads=nheads), ops.mamba3_state(slots, D, N, G, nheads=nheads)
    for state, at in ((small, [0, 1]), (big, [0, slots - 1])):
        at = torch.tensor(at).int().cuda()
        ops.mamba3_prefill(*dev, cu_of([1, 3]), state, slots=at, nheads=nheads)
        y = ops.mamba3_decode_step(state, *(t if i == 4 else t[:2].contiguous() for i, t in enumerate(dev)), slots=at, nheads=nheads)
        if state is small:
            want = y
    assert torch.equal(y, want)
    for t, w in zip(big, small):
        assert torch.equal(t[[0, slots - 1]], w)


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [1, 40, 449, 1024])
@pytest.mark.parametrize("K", [1, 2, 3, 4])
def test_short_conv(K, D, io):
    """Tolerance: K products and sums in float32, an exponential and a division, a dozen roundings of 2^-24; bf16 rounds once."""
    g = torch.Generator().manual_seed(11)
    lens = [1, 0, 2, 9, 3, 0, 130, 8, 4]
    S, rows = len(lens), sum(lens)
    x, pool = torch.randn(rows, D, generator=g).to(io), torch.randn(S + 1, K - 1, D, generator=g).to(io)
    w, bias = torch.randn(D, K, generator=g), torch.randn(D, generator=g)
    slots, go_on = [8, 1, 2, -1, 4, 0, 6, 9, 3], [i % 3 != 1 for i in range(S)]
    slots[7] = 10  # beyond the pool
    for i, s in enumerate(slots):
        if not go_on[i] and 0 <= s <= S and lens[i]:
            pool[s] = float("nan")
    tol = 2e-6 if io == F32 else 2.0 ** -8
    for silu, b, turned in ((False, None, False), (True, bias, True)):
        want = pool.double()
        y_want = serving.short_conv(want, x.double(), w.double(), None if b is None else b.double(), lens, slots, go_on, silu)
        wd = w.t().contiguous().cuda().t() if turned else w.cuda()
        state = pool.cuda()
        out = torch.full((rows + 3, D), 5.0, dtype=io).cuda()
        xp = torch.cat([x, torch.full((3, D), float("nan"), dtype=io)]).cuda()
        ops.short_conv_prefill(xp, wd, cu_of(lens), state, slots=torch.tensor(slots).int().cuda(), go_on=torch.tensor(go_on).cuda(),
                               bias=None if b is None else b.cuda(), activation="silu" if silu else None, out=out)
        assert_close(out[:rows].cpu(), y_want, tol, "y")
        assert bool((out[rows:] == 5.0).all())
        assert torch.equal(torch.nan_to_num(state.cpu().double(), 99.0), torch.nan_to_num(want, 99.0))
        # one token of every sequence
        at, want1 = [5, 0, -1, 3], torch.nan_to_num(pool).double()
        state = torch.nan_to_num(pool).cuda()
        y_want = torch.cat([serving.short_conv(want1, x[i:i + 1].double(), w.double(), None if b is None else b.double(), [1], [s], [True], silu) for i, s in enumerate(at)])
        out = torch.full((4, D), 5.0, dtype=io).cuda()
        ops.short_conv_step(state, x[:4].cuda(), wd, slots=torch.tensor(at).int().cuda(), bias=None if b is None else b.cuda(),
                            activation="silu" if silu else None, out=out)
        assert_close(out[[0, 1, 3]].cpu(), y_want[[0, 1, 3]], tol, "y of a step")
        assert bool((out[2] == 5.0).all()) and torch.equal(state.cpu().double(), want1)


def test_short_conv_keeps_sequences_apart():
    """A tap that is not there, and a neighbour's rows, do not matter even where they are infinite; views that start at odd
    elements give what whole tensors give."""
    x = torch.randn(40, 64).cuda()
    x[:17] = float("inf")
    w = torch.randn(64, 3).cuda()
    y = ops.short_conv_prefill(x, w, cu_of([17, 23]), torch.zeros(2, 2, 64).cuda())
    want = ops.short_conv_prefill(x[17:].contiguous(), w, cu_of([23]), torch.zeros(1, 2, 64).cuda())
    assert torch.equal(y[17:], want)
    # an infinite input ahead of the taps of later rows leaves them alone
    x = torch.randn(12, 64).cuda()
    x[3] = float("inf")
    y = ops.short_conv_prefill(x, w, cu_of([12]), torch.zeros(1, 2, 64).cuda())
    assert bool(torch.isfinite(y[[0, 1, 2, 6, 7, 8, 9, 10, 11]]).all())
    raw = torch.randn(12 * 64 + 1).cuda()
    odd = raw[1:].view(12, 64)
    assert torch.equal(ops.short_conv_prefill(odd, w, cu_of([12]), torch.zeros(1, 2, 64).cuda()),
                       ops.short_conv_prefill(odd.clone(), w, cu_of([12]), torch.zeros(1, 2, 64).cuda()))


def test_unaligned_operands_give_the_same():
    D, N, G, nheads = 128, 128, 1, 2
    a = scan_inputs(100, D, N, G, nheads, BF16, 12)
    dev = [t.cuda() for t in args_of(a)]

    def odd(t):
        raw = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        raw[1:] = t.flatten()
        return raw[1:].view(t.shape)

    want = [ops.mamba3_state(1, D, N, G, nheads=nheads), ops.mamba3_state(1, D, N, G, nheads=nheads)]
    ys = [ops.mamba3_prefill(*args, cu_of([100]), s, nheads=nheads) for args, s in zip((dev, [odd(t) for t in dev]), want)]
    assert_close(ys[1], ys[0].double(), TOL[BF16])
    for t, w in zip(want[1], want[0]):
        assert_close(t, w.double(), TOL[F32])
    with pytest.raises(_lib.MxbError):  # the state itself has to be aligned
        s = want[0]
        ops.mamba3_decode_step(ops.Mamba3State(odd(s.h), *s[1:]), *(t if i == 4 else t[:1].contiguous() for i, t in enumerate(dev)), nheads=nheads)


@pytest.mark.parametrize("shape", [(128, 128, 1, 2), (128, 40, 2, 2), (64, 64, 1, 1), (24, 16, 1, 0), (36, 64, 1, 0)], ids=str)
@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
def test_pool_rows_may_start_at_any_element(io, shape):
    """x_prev and b_prev as views that start at an odd element, beside operands on 16 bytes, of prompts that go on from them:
    short ones, one that is cut, and single tokens.  The same kernels on the same values give the same bits; bf16 prompts that
    would run in chunks go step by step then."""
    D, N, G, nheads = shape
    lens = [40, 1, 900, 130]
    a = [t.cuda() for t in args_of(scan_inputs(sum(lens), D, N, G, nheads, io, 27))]
    pool = gpu_state(pool_inputs(4, D, N, G, nheads, io, 28))

    def odd(t):
        raw = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        raw[1:] = t.flatten()
        return raw[1:].view(t.shape)

    results = []
    for move in (torch.clone, odd):
        for flags in (0, WALK):
            state = ops.Mamba3State(pool.h.clone(), pool.phase.clone(), move(pool.x_prev), move(pool.b_prev))
            y = ops.mamba3_prefill(*a, cu_of(lens), state, go_on=torch.ones(4, dtype=torch.bool, device="cuda"), nheads=nheads, flags=flags)
            y1 = ops.mamba3_decode_step(state, *(t if i == 4 else t[:4].contiguous() for i, t in enumerate(a)), nheads=nheads)
            results.append([y, y1, *state])
    for flags, got, want in zip((0, WALK), results[2:], results[:2]):
        if flags or io == F32 or not nheads:
            assert all(torch.equal(t, u) for t, u in zip(got, want))
            continue
        for t, u in zip(got[:2], want):
            assert_close(t, u.double(), TOL[BF16])
        for t, u in zip(got[2:4], want[2:]):  # (900 steps: the bound of the angles grows with them)
            assert_close(t, u.double(), 3 * TOL[F32])
        assert torch.equal(got[4], want[4]) and torch.equal(got[5], want[5])


def test_a_layer_serves_prompts_then_tokens():
    """The operators as a layer uses them: prompts through norm, projections, convolution, scan and gate, then five tokens
    each; the same rows in one go by the oracle in float64."""
    E, D, N, G, nheads, K, io = 96, 128, 64, 1, 2, 4, F32
    g = torch.Generator().manual_seed(13)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    W = dict(x=r(E, D) / E ** 0.5, z=r(E, D) / E ** 0.5, b=r(E, G * N) / E ** 0.5, c=r(E, G * N) / E ** 0.5, dt=r(E, nheads) / E ** 0.5,
             lam=r(E, nheads) / E ** 0.5, theta=r(E, nheads) / E ** 0.5, o=r(D, E) / D ** 0.5, conv=r(D, K) / 2, a_log=torch.rand(nheads, generator=g),
             norm=1 + 0.1 * r(E), post=1 + 0.1 * r(D), b_scale=1 + 0.1 * r(N), c_scale=1 + 0.1 * r(N), b_bias=0.1 * r(G * N), c_bias=0.1 * r(G * N),
             scale=0.5 + 0.1 * r(E), out_norm=1 + 0.1 * r(E))
    lens, tokens = [40, 7, 0, 66], 5
    have = [i for i, n in enumerate(lens) if n]
    seqs = [r(n + tokens, E) for n in lens]
    d64 = {k: v.double() for k, v in W.items()}

    want = []
    for i in have:  # the oracle, each sequence whole
        h = seqs[i].double()
        n = serving.residual_norm(torch.zeros_like(h), h, d64["norm"])[1]
        x = serving.short_conv(torch.zeros(1, K - 1, D, dtype=torch.float64), n @ d64["x"], d64["conv"], None, [len(h)], [0], [False], True)
        b, c = mamba3_block.bc_norm((n @ d64["b"])[None], (n @ d64["c"])[None], d64["b_scale"], d64["c_scale"], d64["b_bias"], d64["c_bias"], G, N)
        y, _ = serving.mamba3_rows(serving.fresh_mamba3_state(D, N, G, nheads), x, n @ d64["dt"] - 2, n @ d64["lam"], n @ d64["theta"], d64["a_log"], b[0], c[0], nheads)
        o = mamba3_block.post(y, n @ d64["z"], d64["post"]) @ d64["o"]
        want.append(serving.residual_norm(h, o, d64["out_norm"], scale=d64["scale"]))

    P = {k: v.cuda() for k, v in W.items()}
    state, conv = ops.mamba3_state(4, D, N, G, nheads=nheads, dtype=io), torch.zeros(4, K - 1, D).cuda()

    def layer(h, convolve, scan):
        n = ops.residual_norm(torch.zeros_like(h), h, P["norm"])[1]
        x = convolve(n @ P["x"])
        b, c = ops.mamba3_block_bc((n @ P["b"])[None], (n @ P["c"])[None], P["b_scale"], P["c_scale"], P["b_bias"], P["c_bias"], G, N)
        y = scan(x, n @ P["dt"] - 2, n @ P["lam"], n @ P["theta"], P["a_log"], b[0], c[0])
        o = ops.mamba3_block_post(y[None], (n @ P["z"])[None], P["post"])[0] @ P["o"]
        return ops.residual_norm(h, o, P["out_norm"], scale=P["scale"])

    cu = cu_of(lens)
    prompt = layer(torch.cat([s[:n] for s, n in zip(seqs, lens)]).cuda(), lambda x: ops.short_conv_prefill(x, P["conv"], cu, conv, activation="silu"),
                   lambda *a: ops.mamba3_prefill(*a, cu, state, nheads=nheads))
    at = torch.tensor(have).int().cuda()
    rows = [torch.stack([seqs[i][lens[i] + t] for i in have]).cuda() for t in range(tokens)]
    steps = [layer(h, lambda x: ops.short_conv_step(conv, x, P["conv"], slots=at, activation="silu"),
                   lambda *a: ops.mamba3_decode_step(state, *a, slots=at, nheads=nheads)) for h in rows]
    for which in (0, 1):
        at_row = 0
        for k, i in enumerate(have):
            got = torch.cat([prompt[which][at_row:at_row + lens[i]]] + [s[which][k:k + 1] for s in steps])
            assert_close(got.cpu(), want[k][which], 1e-4)  # (the framework's bound for float32 chains: six stages one behind the other)
            at_row += lens[i]


def test_streams_graphs_and_repeats():
    """On another stream, captured and replayed, and twice: the same bits."""
    D, N, G, nheads = 128, 128, 1, 2
    lens = [300, 11]
    a = [t.cuda() for t in args_of(scan_inputs(311, D, N, G, nheads, BF16, 14))]
    one = [t if i == 4 else t[:2].contiguous() for i, t in enumerate(a)]
    w, cu = torch.randn(D, 4).cuda(), cu_of(lens)

    def work(state, conv):
        x = ops.short_conv_prefill(a[0], w, cu, conv, activation="silu")
        y = ops.mamba3_prefill(x, *a[1:], cu, state, nheads=nheads)
        x1 = ops.short_conv_step(conv, one[0], w, activation="silu")
        return [y, ops.mamba3_decode_step(state, x1, *one[1:], nheads=nheads), *state, conv]

    def fresh():
        return ops.mamba3_state(2, D, N, G, nheads=nheads), torch.zeros(2, 3, D, dtype=BF16).cuda()

    want = [t.clone() for t in work(*fresh())]
    assert all(torch.equal(t, u) for t, u in zip(work(*fresh()), want))
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        got = work(*fresh())
    stream.synchronize()
    assert all(torch.equal(t, u) for t, u in zip(got, want))
    state, conv = fresh()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        got = work(state, conv)
    for _ in range(2):  # (prompts start from nothing: a second replay gives the same)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, u) for t, u in zip(got, want))


@pytest.mark.parametrize("io,nheads,D,N", [(BF16, 8, 512, 128), (F32, 8, 512, 128), (F32, 0, 64, 16)])
def test_two_calls_at_once(io, nheads, D, N):
    """Two streams on rows of their own of one pool: the same as one call behind the other."""
    a, b = ([t.cuda() for t in args_of(scan_inputs(900, D, N, 1, nheads, io, s))] for s in (23, 24))
    cu, rows = cu_of([400, 0, 500]), [torch.tensor(r).int().cuda() for r in ([0, 1, 2], [3, 4, 5])]
    want, state = (ops.mamba3_state(6, D, N, 1, nheads=nheads, dtype=io) for _ in range(2))
    ys = [ops.mamba3_prefill(*v, cu, want, slots=r, nheads=nheads) for v, r in zip((a, b), rows)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for v, r, s in zip((a, b), rows, streams):
            with torch.cuda.stream(s):
                got.append(ops.mamba3_prefill(*v, cu, state, slots=r, nheads=nheads))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, ys)) and all(torch.equal(p, q) for p, q in zip(state, want))


@pytest.mark.parametrize("io,nheads,D,N", [(BF16, 1, 8, 8), (F32, 1, 8, 8), (F32, 0, 8, 4)])
def test_thousands_of_sequences(io, nheads, D, N):
    """One token of each of 5000 sequences, as prompts and as tokens; sequences without tokens only, and no sequence at all."""
    S = 5000
    a = [t.cuda() for t in args_of(scan_inputs(S, D, N, 1, nheads, io, 25))]
    states = [ops.mamba3_state(S, D, N, 1, nheads=nheads, dtype=io) for _ in range(2)]
    y = ops.mamba3_prefill(*a, cu_of([1] * S), states[0], nheads=nheads)
    assert_close(y, ops.mamba3_decode_step(states[1], *a, nheads=nheads).double(), TOL[io])
    for t, w in zip(*states):
        assert_close(t, w.double(), TOL[F32])
    for lens in ([0, 0, 0], []):
        out = torch.full((S, D), 5.0, dtype=io).cuda()
        ops.mamba3_prefill(*a, cu_of(lens), states[0], nheads=nheads, out=out)
        assert bool((out == 5.0).all())


@pytest.mark.parametrize("io,nheads,D,N", [(BF16, 4, 256, 64), (F32, 4, 256, 64), (F32, 0, 32, 16)])
def test_long_prompts_beside_many_short_ones(io, nheads, D, N):
    """More sequences than a warp looks at together, two of them cut: the same as the walk that cuts none."""
    lens = [1] * 70 + [700] + [0] * 5 + [33] * 40 + [3000] + [2] * 9
    a = [t.cuda() for t in args_of(scan_inputs(sum(lens), D, N, 1, nheads, io, 26))]
    states = [ops.mamba3_state(len(lens), D, N, 1, nheads=nheads, dtype=io) for _ in range(2)]
    ys = [ops.mamba3_prefill(*a, cu_of(lens), s, nheads=nheads, flags=f) for s, f in zip(states, (0, WALK | SERIAL))]
    assert_close(ys[0], ys[1].double(), TOL[io])
    for t, w in zip(*states):  # (3000 steps: the bound of the angles grows with them)
        assert_close(t, w.double(), 8 * TOL[F32])


def test_refusals():
    D, N, G, nheads = 64, 16, 1, 1
    a = [t.cuda() for t in args_of(scan_inputs(8, D, N, G, nheads, BF16, 15))]
    s = ops.mamba3_state(2, D, N, G, nheads=nheads)
    cu = cu_of([3, 5])
    ok = dict(nheads=nheads)
    ops.mamba3_prefill(*a, cu, s, **ok)
    for bad, err in [((a[:7] + [cu.long(), s], ok), TypeError), ((a[:7] + [cu, s[:3]], ok), ValueError), ((a[:7] + [cu_of([1, 1, 1]), s], ok), ValueError),
                     ((a[:7] + [cu, s], dict(nheads=0)), (ValueError, TypeError)), (([a[0].float()] + a[1:7] + [cu, s], ok), TypeError),
                     ((a[:7] + [cu, s], dict(ok, go_on=torch.zeros(2).cuda())), TypeError), ((a[:7] + [cu, s], dict(ok, slots=torch.zeros(3).int().cuda())), ValueError),
                     ((a[:7] + [cu, s], dict(ok, out=a[0][:4])), ValueError), ((a[:7] + [cu, s._replace(h=s.h[:1])], ok), ValueError),
                     ((a[:7] + [cu.cpu(), s], ok), ValueError), (([a[0].t().contiguous().t()] + a[1:7] + [cu, s], ok), ValueError)]:
        with pytest.raises(err):
            ops.mamba3_prefill(*bad[0], **bad[1])
    with pytest.raises(ValueError):
        ops.mamba3_decode_step(s, *a, nheads=nheads)  # eight sequences, two rows of state
    conv = torch.zeros(2, 3, D, dtype=BF16).cuda()
    for kw in (dict(activation="relu"), dict(bias=torch.zeros(3).cuda())):
        with pytest.raises(ValueError):
            ops.short_conv_prefill(a[0], torch.zeros(D, 4).cuda(), cu, conv, **kw)
    with pytest.raises(_lib.MxbError):
        ops.short_conv_step(torch.zeros(8, 4, D, dtype=BF16).cuda(), a[0], torch.zeros(D, 5).cuda())


@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(128, 64, 2, 2), (64, 16, 1, 0)], ids=str)
def test_results_on_top_of_operands(shape, io):
    """A prompt's result anywhere on an operand or the state is refused, a token's too, but for x as a whole: that gives what a
    result of its own gives."""
    D, N, G, nheads = shape
    a = [t.cuda() for t in args_of(scan_inputs(40, D, N, G, nheads, io, 29))]
    cu, w = cu_of([40]), torch.randn(D, 3).cuda()
    new = lambda: ops.mamba3_state(40, D, N, G, nheads=nheads, dtype=io)  # noqa: E731
    conv = lambda: torch.ones(40, 2, D, dtype=io).cuda()  # noqa: E731
    s, k = new(), conv()
    raw = torch.randn(41 * D + 1, generator=torch.Generator().manual_seed(30)).to(io).cuda()
    x, apart = raw[:40 * D].view(40, D), torch.empty(40, D, dtype=io, device="cuda")
    tops = [raw[o:o + 40 * D].view(40, D) for o in (1, D)] + [t.flatten()[:40 * D].view(40, D) for t in (s.x_prev,)]
    if io == F32:
        tops += [s.h.flatten()[:40 * D].view(40, D)]
    for out in tops + [x]:
        with pytest.raises(ValueError, match="out: overlaps"):
            ops.mamba3_prefill(x, *a[1:], cu, s, nheads=nheads, out=out)
        if out is x:
            break
        with pytest.raises(ValueError, match="out: overlaps"):
            ops.mamba3_decode_step(s, x, *a[1:], nheads=nheads, out=out)
    for out in tops[:2] + [k[:20].view(40, D), x]:
        with pytest.raises(ValueError, match="out: overlaps"):
            ops.short_conv_prefill(x, w, cu, k, out=out)
        if out is x:
            break
        with pytest.raises(ValueError, match="out: overlaps"):
            ops.short_conv_step(k, x, w, out=out)
    ops.mamba3_prefill(raw[D + 1:].view(40, D), *a[1:], cu, s, nheads=nheads, out=apart)  # (beside each other)
    want = ops.mamba3_decode_step(new(), x, *a[1:], nheads=nheads), ops.short_conv_step(conv(), x, w)
    y = x.clone()
    assert torch.equal(ops.mamba3_decode_step(new(), y, *a[1:], nheads=nheads, out=y), want[0])
    y = x.clone()
    assert torch.equal(ops.short_conv_step(conv(), y, w, out=y), want[1])


@pytest.mark.parametrize("lens,chunks", [([16], False), ([17], True), ([1] * 64, False), ([4] * 64, False), ([5] * 64, True), ([1] * 63 + [512], True),
                                         ([64] * 16, True)], ids=["16", "17", "64 of 1", "64 of 4", "64 of 5", "63 of 1 and one of 512", "16 of 64"])
def test_short_prompts_go_step_by_step(lens, chunks):
    """bf16 prompts of few rows each go step by step, where only y is rounded (half a step of bf16, and the float32 bound beside it);
    the others in chunks."""
    D, N, G, nheads, S = 128, 64, 1, 2, len(lens)
    a = scan_inputs(sum(lens), D, N, G, nheads, BF16, 31)
    pool = pool_inputs(S, D, N, G, nheads, BF16, 32)
    want = list(double(pool))
    y_want = serving.mamba3_prefill(want, *double(args_of(a)), lens, list(range(S)), [True] * S, nheads)
    state, lib = gpu_state(pool), _lib.lib()
    args = [t.cuda() for t in args_of(a)], cu_of(lens), torch.ones(S, dtype=torch.bool, device="cuda")
    lib.mxb_trace_enable(1)
    y = ops.mamba3_prefill(*args[0], args[1], state, go_on=args[2], nheads=nheads)
    torch.cuda.synchronize()
    buf = C.create_string_buffer(4096)
    lib.mxb_trace_summary(buf, len(buf))
    lib.mxb_trace_enable(0)
    assert (b"m3p_chunks_kernel" in buf.value) == chunks and (b"m3k_heads_kernel" in buf.value) != chunks, buf.value
    if not chunks:
        assert bool(((y.cpu().double() - y_want).abs() <= 2.0 ** -8 * y_want.abs() + TOL[F32] * y_want.abs().max()).all())
    assert_close(y.cpu(), y_want, TOL[BF16])
    check_state(state, want, BF16, 2 * TOL[F32], list(range(S)))


@pytest.mark.parametrize("D", [64, 128, 320], ids=lambda D: f"head of {D}")
def test_angle_of_a_long_prompt(D):
    """The phase behind 16384 bf16 steps that all turn the same way, by 8 radians each, whole and in two parts, for heads of one,
    two and five slabs.  Each step is rounded to half of 2^-32 turns, 16384 x 2^-33 x 2 pi = 1.2e-5 in all; the phase goes through at
    most 148 segments' products of unit vectors, off by at most four roundings of 2^-24 each: 3.6e-5."""
    T, N = 16384, 16
    a = scan_inputs(T, D, N, 1, 1, BF16, 33)
    a["dt"].fill_(2.5)
    a["theta"].fill_(3.1)
    angle = (T * torch.nn.functional.softplus(a["dt"][0].double()) * a["theta"][0].double()).item()
    want = torch.tensor([math.cos(angle), math.sin(angle)], dtype=torch.float64)
    dev = [t.cuda() for t in args_of(a)]
    for cuts in ((0, T), (0, 7001, T)):
        state = ops.mamba3_state(1, D, N, 1, nheads=1)
        for lo, hi in zip(cuts, cuts[1:]):
            ops.mamba3_prefill(*(t if i == 4 else t[lo:hi].contiguous() for i, t in enumerate(dev)), cu_of([hi - lo]), state, nheads=1,
                               go_on=torch.tensor([lo > 0]).cuda())
        assert (state.phase.cpu().double() - want).abs().max() <= 1.2e-5 + 3.6e-5


@pytest.mark.parametrize("shape", [(128, 64, 1, 1), (160, 128, 1, 1), (320, 32, 2, 2), (130, 6, 1, 1)], ids=str)
@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
def test_wide_heads_of_cut_sequences(shape, io):
    """Heads of more than 64 channels (several CTAs a head) whose sequences are cut in segments, beside others; a padding entry."""
    D, N, G, nheads = shape
    lens, slots = [5, 700, 0, 391, 64, 200], [3, 0, 2, 1, 5, -1]
    a = scan_inputs(sum(lens), D, N, G, nheads, io, 34)
    pool = pool_inputs(6, D, N, G, nheads, io, 35)
    go_on = [True, True, True, False, True, True]
    want = list(double(pool))
    y_want = serving.mamba3_prefill(want, *double(args_of(a)), lens, slots, go_on, nheads)
    for flags in (0, WALK, WALK | SERIAL):
        state = gpu_state(pool)
        y = ops.mamba3_prefill(*(t.cuda() for t in args_of(a)), cu_of(lens), state, slots=torch.tensor(slots).int().cuda(),
                               go_on=torch.tensor(go_on).cuda(), nheads=nheads, flags=flags)
        assert_close(y.cpu(), y_want, TOL[io], f"y flags {flags}")
        check_state(state, want, io, 2 * TOL[F32], [0, 1, 3, 5])  # (700 steps: the bound of the angles grows with them)
        for t, w in zip(state, pool):
            assert torch.equal(t[[2, 4]].cpu(), w[[2, 4]])


@pytest.mark.parametrize("raw", [200.0, 3e5])
@pytest.mark.parametrize("io", [F32, BF16], ids=["f32", "bf16"])
def test_steps_that_forget_everything(io, raw):
    """Steps with a decay of thousands and millions of powers of two, among slow ones: what follows them is as exact as elsewhere."""
    D, N, G, nheads, lens = 128, 64, 1, 2, [150, 70]
    a = scan_inputs(sum(lens), D, N, G, nheads, io, 36)
    a["dt"] -= 4.0
    a["a_log"].fill_(math.log(16.0))
    steps = [20, 100, 150 + 33]
    a["dt"][steps] = raw
    want = list(double(pool_inputs(2, D, N, G, nheads, io, 37)))
    pool = [t.float() for t in want]
    y_want = serving.mamba3_prefill(want, *double(args_of(a)), lens, [0, 1], [True, True], nheads)
    for flags in (0, WALK):
        state = gpu_state([t.to(w.dtype) for t, w in zip(pool, (torch.zeros((), dtype=F32), torch.zeros((), dtype=F32), a["x"], a["x"]))])
        y = ops.mamba3_prefill(*(t.cuda() for t in args_of(a)), cu_of(lens), state, go_on=torch.ones(2, dtype=torch.bool, device="cuda"), nheads=nheads, flags=flags)
        for lo, hi in zip([0] + steps, steps + [sum(lens)]):
            assert_close(y[lo:hi].cpu(), y_want[lo:hi], TOL[io], f"rows {lo} to {hi}, flags {flags}")
        check_state(state, want, io, TOL[F32], [0, 1])


def test_sizes_beyond_32_bits_are_refused():
    """2^32 + 8 rows or columns are not taken for 8."""
    big = torch.empty((1 << 32) + 8, 1, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="beyond 32 bits"):
        ops.short_conv_prefill(big, torch.ones(1, 1).cuda(), cu_of([8]), torch.empty(1, 0, 1, dtype=BF16, device="cuda"))
    with pytest.raises(ValueError, match="beyond 32 bits"):
        ops.residual_norm(big.t(), big.t(), torch.empty((1 << 32) + 8, device="cuda"))


@pytest.mark.parametrize("nheads,D,N", [(2, 128, 64), (0, 48, 16)])
def test_a_served_layer_is_the_trained_one(nheads, D, N):
    """A Mamba-3 layer by the stages of training over [1, T] and by those of serving, prompt and tokens: float32, the bound of
    prompts on either side."""
    E, G, K, T, cut = 40, 1, 4, 90, 83
    g = torch.Generator().manual_seed(38)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    H = nheads or D
    n, w, post, next_norm, scale = r(T, E), r(D, K) / 2, 1 + 0.1 * r(D), 1 + 0.1 * r(E), 0.5 + 0.1 * r(E)
    W = {k: r(E, c) / E ** 0.5 for k, c in dict(x=D, z=D, b=N, c=N, dt=H, lam=H, theta=H if nheads else D * N // 2).items()}
    W_o, h, a_log = r(D, E) / D ** 0.5, r(T, E), torch.rand(*((nheads,) if nheads else (D, N)), generator=g).cuda()
    p = {k: n @ v for k, v in W.items()}
    p["dt"], p["theta"] = p["dt"] - 2, p["theta"] if nheads else p["theta"].view(T, D, N // 2)
    b, c = ops.mamba3_block_bc(p["b"][None], p["c"][None], 1 + 0.1 * r(N), 1 + 0.1 * r(N), 0.1 * r(N), 0.1 * r(N), G, N)
    b, c = b.view(1, T, G, N), c.view(1, T, G, N)

    def behind(y, rows):
        o = ops.mamba3_block_post(y[None], p["z"][rows][None].contiguous(), post)[0] @ W_o
        return torch.stack(ops.residual_norm(h[rows], o, next_norm, scale=scale))

    x = ops.mamba3_block_conv(p["x"][None], w)
    y = ops.mamba3_selective_scan(x, p["dt"][None], p["lam"][None], p["theta"][None], a_log, b, c, nheads=nheads)
    want = behind(y[0], slice(0, T))
    state, conv, rows = ops.mamba3_state(1, D, N, G, nheads=nheads, dtype=F32), torch.zeros(1, K - 1, D).cuda(), slice(0, cut)
    part = lambda q: [t[q].contiguous() for t in (p["dt"], p["lam"], p["theta"])] + [a_log, b[0, q].contiguous(), c[0, q].contiguous()]  # noqa: E731
    got = [behind(ops.mamba3_prefill(ops.short_conv_prefill(p["x"][rows], w, cu_of([cut]), conv), *part(rows), cu_of([cut]), state, nheads=nheads), rows)]
    for t in range(cut, T):
        q = slice(t, t + 1)
        got.append(behind(ops.mamba3_decode_step(state, ops.short_conv_step(conv, p["x"][q], w), *part(q), nheads=nheads), q))
    assert_close(torch.cat(got, 1), want.double(), 2 * TOL[F32])
