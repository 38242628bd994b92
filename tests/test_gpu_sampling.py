"""The choice of the next token from logits that a mask has changed (GPU): a draw never takes a
token of no weight, and a row without any token left is reported."""

import ctypes as C

import numpy as np
import pytest
import torch

from orchard_b200 import _lib
from orchard_b200._lib import F32, call

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    assert torch.cuda.is_available()
    call("orch_init", 0, None)
    flags()
    yield
    torch.cuda.synchronize()


def flags():
    torch.cuda.synchronize()
    f = C.c_uint32(0)
    call("orch_device_check", C.byref(f), None)
    return int(f.value)


def S():
    return torch.cuda.current_stream().cuda_stream


def D(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def sample(logits, T, u):
    M, V = logits.shape
    tok = torch.full((M,), -7, dtype=torch.int32, device="cuda")
    call("orch_sample_rows", logits, M, V, T, D(np.asarray(u, np.float32)), tok, S())
    return tok.cpu().numpy()


def masked(x, allowed):
    """x [M, V] through orch_logits_process with one mask per row."""
    M, V = x.shape
    words = (V + 31) // 32
    m = np.zeros((M, words), np.uint32)
    for r, ids in enumerate(allowed):
        for v in ids:
            m[r, v // 32] |= np.uint32(1 << (v % 32))
    d = D(x)
    call("orch_logits_process", d, d, F32, M, V, V, 0, None, 0, None, None, None, None, None, None, 0, D(m.view(np.int32)), words,
         M, D(np.arange(M, dtype=np.int32)), S())
    return d


def test_a_draw_at_the_end_of_a_running_sum_takes_a_token_of_positive_weight():
    """Token 0 has weight 1; tokens 32..47 have e^-17 = 4.1e-8 each, less than half a unit in the
    last place of 1: added one by one to a running sum of 1 they leave it at 1, while their own
    sum (16 of them, 5.6 units) does not vanish. A target between the two is passed by no prefix
    of the walk over 32..63, of which 48..63 are forbidden: the last allowed one has to be taken."""
    V = 32 * 1024
    x = np.full((3, V), -1.0, np.float32)
    x[:, 0] = 17.0
    x[:, 32:48] = 0.0
    lg = masked(x, [[0, *range(32, 48)]] * 3)
    u = [1 - 2.0 ** -22, 1 - 3 * 2.0 ** -23, 0.5]
    assert sample(lg, 1.0, u).tolist() == [47, 47, 0]


@pytest.mark.parametrize("T", [0.3, 1.0, 2.5])
def test_draws_under_a_mask_are_allowed_tokens(T):
    """Uniforms over all of [0, 1), its ends among them, on masks that leave few tokens, a third of
    them, or a run."""
    g = np.random.default_rng([20261206, 31, int(10 * T)])
    V, M = 4000, 300
    x = (3 * g.standard_normal((M, V), dtype=np.float32)).astype(np.float32)
    allowed = [[int(v) for v in (g.choice(V, 2, replace=False) if m % 3 == 0 else np.arange(m % 7, V, 3) if m % 3 == 1
                                 else np.arange(m, m + 5))] for m in range(M)]
    u = g.random(M).astype(np.float32)
    u[::5], u[1::5] = 0.0, np.float32(1 - 2.0 ** -24)
    got = sample(masked(x, allowed), T, u)
    assert all(got[m] in allowed[m] for m in range(M))
    assert flags() == 0


def test_a_row_without_any_token_is_reported():
    """All -inf: token 0 and device check bit 32, greedy and drawn; other rows are not affected."""
    V = 1000
    x = np.tile(np.linspace(-1, 1, V, dtype=np.float32), (4, 1))
    lg = masked(x, [[5, 9], [], [V - 1], []])
    tok = torch.full((4,), -7, dtype=torch.int32, device="cuda")
    call("orch_argmax_rows", lg, 4, V, tok, S())
    assert flags() == 32 and tok.tolist() == [9, 0, V - 1, 0]
    assert sample(lg, 0.7, [0.0, 0.5, 0.9, 0.1]).tolist() == [5, 0, V - 1, 0]
    assert flags() == 32
    lg = masked(x, [[5, 9], [7], [V - 1], [0]])
    call("orch_argmax_rows", lg, 4, V, tok, S())
    sample(lg, 0.7, [0.0, 0.5, 0.9, 0.1])
    assert flags() == 0
    lg[1] = float("nan")  # a NaN is a value as before
    call("orch_argmax_rows", lg, 4, V, tok, S())
    assert flags() == 0 and tok[1] == 0
