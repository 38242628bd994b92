"""The projections that put a token's key at an entry apart from its position (GPU): bit-equal to
the forms without, at the other place."""

import ctypes as C

import numpy as np
import pytest
import torch

from oracle import ops
from orchard_b200 import quantizer
from orchard_b200._lib import call
from test_gpu_tiled import S, device, pack_dev  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu


def flags():
    torch.cuda.synchronize()
    f = C.c_uint32(0)
    call("orch_device_check", C.byref(f), None)
    return int(f.value)


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("lora", [False, True])
@pytest.mark.parametrize("slotted", [False, True])
@pytest.mark.parametrize("M", [1, 3, 8, 9, 17, 33, 64, 65, 130, 300])
def test_keys_at_an_entry_apart_from_the_position(M, lora, slotted, rms):
    if rms and lora:
        pytest.skip("the fused form takes no LoRA terms")
    H, nh, seq, r, max_pos = 256, 4, 40, 16, 700
    hd = H // nh
    g = np.random.default_rng([20261206, M, lora, slotted])
    w = (g.standard_normal((3 * H, H), dtype=np.float32) * 0.05).astype(np.float16).astype(np.float32)
    tq = pack_dev(*quantizer.quantize_q4_0(w))
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    x16 = d(g.standard_normal((M, H), dtype=np.float32).astype(np.float16))
    x32, gamma = d(g.standard_normal((M, H), dtype=np.float32)), d(1 + 0.1 * g.standard_normal(H, dtype=np.float32))
    cos, sin = (d(t) for t in ops.precompute_freqs_cis(hd, max_pos))
    lt, lb = d(g.standard_normal((M, 3, r), dtype=np.float32)), d(0.1 * g.standard_normal((3, r, H), dtype=np.float32))
    tail = (lt, lb, r) if lora else (None, None, 0)
    pos, index = g.integers(0, max_pos, M).astype(np.int32), g.integers(0, seq, M).astype(np.int32)
    slots = g.permutation(M + 2)[:M].astype(np.int32)
    n = M + 2

    def run(form, seq, *where):
        q = torch.zeros((M, H), dtype=torch.float16, device="cuda")
        kc = torch.zeros((n, nh, seq, hd), dtype=torch.float16, device="cuda")
        vc, xn = torch.zeros_like(kc), torch.zeros_like(q)
        out = (cos, sin, max_pos, q, kc, vc, seq, n)
        where = (*where, d(slots) if slotted else None)
        if rms:
            call("orch_q4t_rms_qkv_rope" + form, tq, x32, gamma, 1e-5, xn, M, H, H, nh, *where, *out, S())
        else:
            call("orch_q4t_qkv_rope" + form, tq, x16, M, H, H, nh, *where, *out, *tail, S())
        return q, kc, vc

    q0, k0, v0 = run("", max_pos, d(pos))
    assert flags() == 0
    q1, k1, v1 = run("_at", seq, d(pos), d(index))
    assert flags() == 0 and torch.equal(q0, q1)
    for m in range(M):
        t = int(slots[m]) if slotted else m
        assert torch.equal(k1[t, :, index[m]], k0[t, :, pos[m]]) and torch.equal(v1[t, :, index[m]], v0[t, :, pos[m]])
        k1[t, :, index[m]] = 0
        v1[t, :, index[m]] = 0
    assert not k1.any() and not v1.any() and bool(q0.any())
    bad = index.copy()
    bad[M // 2] = seq  # past the slot: neither key nor value, reported
    _, k2, v2 = run("_at", seq, d(pos), d(bad))
    assert flags() == 1
    t = int(slots[M // 2]) if slotted else M // 2
    assert not k2[t].any() and not v2[t].any() and (M == 1 or bool(k2.any()))
