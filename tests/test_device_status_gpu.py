"""The device's error word behind calls that keep none: what an earlier call reported stays, and nothing else looks like an error."""
import pytest
import torch

from mixlab_b200 import _lib, ops
from test_step_ends_use_gpu import batch, step, weights

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def r(*s):
    return torch.randn(*s, device="cuda")


def n(t):
    return torch.ones(t, device="cuda")


def mamba3(T, D, N, heads, io):
    H = heads or D
    pos = lambda *s: torch.rand(*s, device="cuda")  # noqa: E731
    theta, a_log = (0.1 * r(*T, H), -pos(H)) if heads else (0.1 * r(*T, H, N // 2), -pos(H, N))
    return r(*T, D).to(io), pos(*T, H), pos(*T, H), theta, a_log, r(*T, 1, N).to(io), r(*T, 1, N).to(io)


def gdn_pre():
    B, T, H, Dk, Dv = 2, 40, 2, 32, 32
    q, k, v = r(B, T, H * Dk), r(B, T, H * Dk), r(B, T, H * Dv)
    ops.gdn_block_pre_backward(q, k, v, r(4, H * Dk), r(4, H * Dk), r(4, H * Dv), r(B, T, H), r(B, T, H), r(H), r(H), H, Dk, Dv,
                               r(B, T, H, Dk), r(B, T, H, Dk), r(B, T, H, Dv), r(B, T, H), r(B, T, H))


def prefill():
    a = mamba3((300,), 64, 16, 0, F32)
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    ops.mamba3_prefill(*a, cu, ops.mamba3_state(2, 64, 16, 1, dtype=F32), flags=0)


def scan():
    a = mamba3((1, 300), 64, 16, 0, F32)
    ops.mamba3_selective_scan(*a)
    ops.mamba3_selective_scan_backward(*a, r(1, 300, 64))


def scan_heads():
    a = mamba3((1, 90), 64, 16, 2, F32)
    ops.mamba3_selective_scan_backward(*a, r(1, 90, 64), nheads=2)


CALLS = {
    "embedding": lambda: ops.embedding_backward(torch.randint(0, 50, (9000,), device="cuda"), r(9000, 16), 50),
    "embedding of few": lambda: ops.embedding_backward(torch.randint(0, 50, (200,), device="cuda"), r(200, 16), 50),
    "layer_norm": lambda: ops.layer_norm_backward(r(300, 64), n(64), r(300, 64)),
    "residual_norm": lambda: ops.residual_norm_backward(r(300, 64), r(300, 64), n(64), None, r(300, 64)),
    "gdn_block_pre": gdn_pre,
    "gdn_block_post": lambda: ops.gdn_block_post_backward(r(2, 40, 2, 32), r(2, 40, 64), n(32), r(2, 40, 64)),
    "mamba3_block_conv": lambda: ops.mamba3_block_conv_backward(r(2, 40, 64), r(64, 4), r(2, 40, 64)),
    "mamba3_block_bc": lambda: ops.mamba3_block_bc_backward(r(2, 40, 32), r(2, 40, 32), n(32), n(32), r(2, 40, 1, 32), r(2, 40, 1, 32), 1, 32),
    "mamba3_block_post": lambda: ops.mamba3_block_post_backward(r(2, 40, 64), r(2, 40, 64), n(64), r(2, 40, 64)),
    "mamba3_prefill": prefill,
    "mamba3_scan": scan,
    "mamba3_scan of heads": scan_heads,
}


def plant(word):
    ops.workspace(256, torch.device("cuda", torch.cuda.current_device()))[:4].view(torch.int32).fill_(word)


@pytest.mark.parametrize("name", CALLS)
def test_calls_that_keep_no_word_leave_it(name):
    """From a buffer of the smallest size, which the call outgrows, and from one that is large enough."""
    with torch.cuda.stream(torch.cuda.Stream()):
        for word in (11, 3):
            plant(word)
            CALLS[name]()
            assert ops.device_status() == word
        loss, lse = ops.linear_cross_entropy(r(20, 16), r(30, 16), torch.zeros(20, dtype=torch.long, device="cuda"))
        assert ops.device_status() == 0  # (a call that keeps one)


def test_a_stream_without_calls():
    """The memory that its buffer gets held something else."""
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.full((1 << 20,), -1, dtype=torch.int32, device="cuda")
        torch.full((64,), -1, dtype=torch.int32, device="cuda")
        assert ops.device_status() == 0


@pytest.mark.parametrize("io", [F32, BF16])
def test_after_a_whole_training_step(io):
    g = torch.Generator().manual_seed(3)
    w = {k: v.cuda() for k, v in weights(g, io).items()}
    tokens, targets, gates = batch(g)
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(2):
            step(w, tokens.cuda(), targets.cuda(), tuple(t.cuda() for t in gates), io)
            assert ops.device_status() == 0


def test_a_saved_forward_is_found_behind_its_larger_buffer():
    """The status block that goes along does not disturb what a forward leaves for its backward."""
    a = mamba3((1, 300), 64, 16, 0, F32)
    dy = r(1, 300, 64)
    want = ops.mamba3_selective_scan_backward(*a, dy, flags=_lib.MXB_MAMBA3_WINDOW_PARALLEL)
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.synchronize()
        plant(0)
        ops.mamba3_selective_scan(*a, flags=_lib.MXB_MAMBA3_WINDOW_PARALLEL, save_for_backward=True)
        got = ops.mamba3_selective_scan_backward(*a, dy, flags=_lib.MXB_MAMBA3_WINDOW_PARALLEL, use_saved=True)
        torch.cuda.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in want)
