"""The ends of a training step as they are used: around a scan of the framework, with a matrix that embedding and head share, in
graphs, on several streams and from several threads."""
import threading

import pytest
import torch

from mixlab_b200 import ops
from oracle import gdn, step_ends
from util import assert_close

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
B, T, H, DK, V = 2, 70, 2, 16, 61
D = H * DK


def weights(g, io):
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(token=(0.5 * r(V, D)).to(io), w0=1 + 0.1 * r(D), b0=0.1 * r(D), w1=1 + 0.1 * r(D), b1=0.1 * r(D))


def batch(g):
    tokens = torch.randint(0, V, (B, T), generator=g)
    tokens[1, T - 9:] = -1  # a text that ends early
    targets = torch.full_like(tokens, -1)
    targets[:, :-1] = tokens[:, 1:]
    gates = torch.rand(B, T, H, generator=g), 0.8 + 0.2 * torch.rand(B, T, H, generator=g)
    return tokens, targets, gates


def step(w, tokens, targets, gates, io, flags=0):
    """Loss per token, gradients as numerators (a sum over the tokens that count) and how many count."""
    beta, gate = gates
    stream = ops.embedding(tokens, w["token"], scale=D ** 0.5, dtype=F32)
    n = ops.layer_norm(stream, w["w0"], w["b0"], dtype=io)
    heads = n.view(B, T, H, DK)
    y = ops.gated_delta_scan(heads, heads, heads, beta, gate, 64)
    out, n1 = ops.layer_norm(y.view(B, T, D), w["w1"], w["b1"], resid=stream)
    loss, lse = ops.linear_cross_entropy(n1, w["token"], targets)
    ones = torch.ones_like(loss)
    head = ops.linear_cross_entropy_backward(n1, w["token"], targets, lse, ones)
    g1 = ops.layer_norm_backward(out, w["w1"], head["dx"])
    dy = g1["dx"].to(io).view(B, T, H, DK)
    gs = ops.gated_delta_scan_backward(heads, heads, heads, beta, gate, dy, 64)
    dn = (gs["dq"].float() + gs["dk"].float() + gs["dv"].float()).to(io).view(B, T, D)
    g0 = ops.layer_norm_backward(stream, w["w0"], dn, d_resid=g1["dx"])
    token = ops.embedding_backward(tokens, g0["dx"], V, scale=D ** 0.5, dweight=head["dweight"])
    return loss, dict(token=token, w0=g0["dweight"], b0=g0["dbias"], w1=g1["dweight"], b1=g1["dbias"]), (targets >= 0).sum()


def oracle_step(w, tokens, targets, gates):
    w = {k: v.double().requires_grad_() for k, v in w.items()}
    beta, gate = (t.double() for t in gates)
    ok = tokens >= 0
    stream = torch.where(ok[..., None], D ** 0.5 * w["token"][tokens.clamp(min=0)], 0.0)
    n = step_ends.layer_norm(stream, w["w0"], w["b0"])[1]
    heads = n.view(B, T, H, DK)
    y = gdn.scan_chunked(heads, heads, heads, beta, gate, 64)[0]
    n1 = step_ends.layer_norm(y.reshape(B, T, D), w["w1"], w["b1"], stream)[1]
    z = n1 @ w["token"].T
    loss = torch.where(targets >= 0, torch.logsumexp(z, -1) - z.gather(-1, targets.clamp(min=0)[..., None])[..., 0], 0.0)
    names = list(w)
    return loss.detach(), dict(zip(names, torch.autograd.grad(loss.sum(), [w[k] for k in names])))


def test_a_training_step():
    """float32 from the tokens to every gradient, at the scan's own bound."""
    g = torch.Generator().manual_seed(3)
    w = weights(g, F32)
    tokens, targets, gates = batch(g)
    want_loss, want = oracle_step(w, tokens, targets, gates)
    cuda = lambda t: t.cuda()  # noqa: E731
    loss, got, count = step({k: cuda(v) for k, v in w.items()}, cuda(tokens), cuda(targets), tuple(map(cuda, gates)), F32)
    assert_close(loss, want_loss, 1e-4, "loss")
    assert count.item() == int((targets >= 0).sum())
    for k in want:
        assert_close(got[k], want[k], 1e-4, k)


def test_a_training_step_in_bf16_link_by_link(monkeypatch):
    """Each call of the step against the oracle on what it was given.  (From end to end bf16 has no bound here: the keys' squared norms
    are about 16, so that a step of the scan multiplies a rounding by up to 15.)  A result of bf16 is off by its rounding, 2^-8 of the
    largest at most, and for the head's gradients by the rounding of g, as much again; float32 results of sums by a few 2^-24 a term."""
    calls = []
    for name in ("embedding", "layer_norm", "layer_norm_backward", "linear_cross_entropy", "linear_cross_entropy_backward", "embedding_backward"):
        def spy(*args, name=name, fn=getattr(ops, name), **kw):
            copy = lambda v: v.clone() if torch.is_tensor(v) else {k: u.clone() for k, u in v.items()} if isinstance(v, dict) else v  # noqa: E731
            kept = {k: copy(v) for k, v in kw.items()}  # (dweight is changed in place)
            out = fn(*args, **kw)
            calls.append((name, args, kept, copy(out)))
            return out
        monkeypatch.setattr(ops, name, spy)
    g = torch.Generator().manual_seed(3)
    w = {k: v.cuda() for k, v in weights(g, BF16).items()}
    tokens, targets, gates = batch(g)
    step(w, tokens.cuda(), targets.cuda(), tuple(t.cuda() for t in gates), BF16)
    assert len(calls) == 8
    f = lambda t: t.double().cpu() if torch.is_tensor(t) and t.is_floating_point() else t.cpu() if torch.is_tensor(t) else t  # noqa: E731
    tol = {BF16: 2.0 ** -7, F32: 2e-5}
    for name, args, kw, out in calls:
        a, k = [f(t) for t in args], {n: f(t) for n, t in kw.items() if n not in ("dtype",)}
        if name == "embedding":
            want, out = {"rows": step_ends.embedding(*a, **k)}, {"rows": out}
        elif name == "embedding_backward":
            old = k.pop("dweight")
            want, out = {"token": old + step_ends.embedding_backward(*a, **k)[0]}, {"token": out}
        elif name == "layer_norm":
            h, n = step_ends.layer_norm(*a, **k)
            want, out = ({"stream": h, "n": n}, dict(zip(("stream", "n"), out))) if isinstance(out, tuple) else ({"n": n}, {"n": out})
        elif name == "linear_cross_entropy":
            want, out = dict(zip(("loss", "lse"), step_ends.linear_cross_entropy(*a))), dict(zip(("loss", "lse"), out))
        else:
            want = getattr(step_ends, name)(*a, **k)
        for key, need in want.items():
            assert_close(out[key], need, tol[out[key].dtype], f"{name}: {key}")


def test_graphs_of_two_steps_and_calls_between():
    """Two captured steps, replayed by turns with other batches than they were captured with, calls on the same stream between: the
    bits of the same calls outside a graph."""
    g = torch.Generator().manual_seed(4)
    w = {k: v.cuda() for k, v in weights(g, BF16).items()}
    batches = [batch(g) for _ in range(4)]
    put = lambda dst, b: [d.copy_(s) for d, s in zip((dst[0], dst[1], *dst[2]), (b[0], b[1], *b[2]))]  # noqa: E731
    dev = lambda b: (b[0].cuda(), b[1].cuda(), tuple(t.cuda() for t in b[2]))  # noqa: E731
    want = []
    for b in batches:
        loss, grads, _ = step(w, *dev(b), BF16)
        want.append([loss.clone()] + [v.clone() for v in grads.values()])
    graphs = []
    for _ in range(2):
        ins = dev(batches[0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(w, *ins, BF16)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss, grads, _ = step(w, *ins, BF16)
        graphs.append((graph, ins, [loss] + list(grads.values())))
    for i in range(8):
        graph, ins, outs = graphs[i % 2]
        put(ins, batches[i % 4])
        graph.replay()
        big = torch.randn(3000, D, device="cuda").to(BF16)
        ops.linear_cross_entropy_backward(big, w["token"], torch.zeros(3000, dtype=torch.long, device="cuda"), torch.zeros(3000, device="cuda"),
                                          torch.ones(3000, device="cuda"))
        torch.cuda.synchronize()
        for x, y in zip(outs, want[i % 4]):
            assert torch.equal(x, y), i
    assert ops.device_status() == 0


def cases():
    g = torch.Generator().manual_seed(6)
    out = []
    for n, V_, D_, io in ((700, 900, 64, BF16), (3000, 5000, 136, BF16), (300, 700, 40, F32)):
        x, w = torch.randn(n, D_, generator=g).to(io).cuda(), torch.randn(V_, D_, generator=g).to(io).cuda()
        t = torch.randint(-1, V_, (n,), generator=g).cuda()
        d = torch.rand(n, generator=g).cuda()

        def run(x=x, w=w, t=t, d=d, V_=V_):
            loss, lse = ops.linear_cross_entropy(x, w, t)
            grads = ops.linear_cross_entropy_backward(x, w, t, lse, d)
            norm = ops.layer_norm_backward(grads["dx"], torch.ones(x.shape[1], device="cuda"), x)
            return [loss, lse, grads["dx"], ops.embedding_backward(t, x, V_, dweight=grads["dweight"]), norm["dx"], norm["dweight"], norm["dbias"]]

        out.append(run)
    return out


def test_streams_and_threads():
    runs = cases()
    want = [[t.clone() for t in r()] for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(15):  # one thread, several streams at once
        got = []
        for st, r in zip(streams, runs):
            with torch.cuda.stream(st):
                got.append(r())
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))
    failures = []

    def work(i, own):
        try:
            with torch.cuda.stream(torch.cuda.Stream() if own else torch.cuda.default_stream()):
                for _ in range(25):
                    got = runs[i]()
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
        except BaseException as e:
            failures.append(e)

    for own in (True, False):
        threads = [threading.Thread(target=work, args=(i, own)) for i in range(len(runs))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not failures, failures


def test_tensors_of_another_stream():
    """Operands made on one stream, the call on another that waits for it."""
    run = cases()[0]
    want = [t.clone() for t in run()]
    made, used = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(made):
            torch.cuda._sleep(1000000)
        used.wait_stream(made)
        with torch.cuda.stream(used):
            got = run()
        used.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
