"""Buffers that are not aligned for their elements, and sizes past what the kernels count with, are
refused before any device work (an unaligned access would fault)."""

import pytest

from orchard_b200 import _lib
from test_serving_args import P, attention, evict, logits, pytestmark  # noqa: F401 (no GPU may see the pointers)

WS = dict(ws=P, wb=1 << 30)


@pytest.mark.parametrize("by", [1, 2, 3])
@pytest.mark.parametrize("name", ["lens", "slots", "mass"])
def test_attention_refuses_unaligned_buffers(name, by):
    assert attention(**WS, **{name: P + by}) == 1 and b"aligned" in _lib.lib().orch_last_error()


@pytest.mark.parametrize("by", [1, 2, 3])
@pytest.mark.parametrize("name", ["mass", "pos", "lens", "slots", "mo", "po", "lo"])
def test_evict_refuses_unaligned_buffers(name, by):
    apart = dict(mo=2 * P, po=3 * P)  # separate outputs
    assert evict(**{**apart, name: P + by}) == 1 and b"aligned" in _lib.lib().orch_last_error()


@pytest.mark.parametrize("kw", [dict(x=P + 2), dict(out=P + 1), dict(x=P + 2, out=P + 2), dict(x=P + 1, dt=1), dict(out=P + 3, dt=1),
                                dict(hist=P + 2, hl=4, hn=P, pen=P), dict(hist=P, hl=4, hn=P + 1, pen=P), dict(hist=P, hl=4, hn=P, pen=P + 3),
                                dict(hist=P, hl=4, hn=P, pen=P, gs=P + 2), dict(bi=P + 2, bv=P, bo=P, nb=1), dict(bi=P, bv=P + 2, bo=P, nb=1),
                                dict(bi=P, bv=P, bo=P + 2, nb=1), dict(masks=P + 2, mr=P, mw=1, nm=1), dict(masks=P, mr=P + 2, mw=1, nm=1)])
def test_logits_refuse_unaligned_buffers(kw):
    assert logits(**kw) == 1 and b"aligned" in _lib.lib().orch_last_error()


def test_projections_refuse_an_unaligned_index():
    L = _lib.lib()
    assert L.orch_q4t_qkv_rope_at(P, P, 1, 256, 256, 4, P, P + 2, None, P, P, 8, P, P, P, 8, 1, None, None, 0, None) == 1
    assert b"index" in L.orch_last_error()
    assert L.orch_q4t_rms_qkv_rope_at(P, P, P, 1e-5, P, 1, 256, 256, 4, P, P + 1, None, P, P, 8, P, P, P, 8, 1, None) == 1
    assert b"index" in L.orch_last_error()


@pytest.mark.parametrize("size", [2 ** 31 - 1, 2 ** 31 - 65535])
def test_logits_refuse_lists_past_what_a_loop_counts(size):
    """A list's index is a 32-bit number that goes on by up to 2,048 past its end."""
    assert logits(hist=P, hl=size, hn=P, pen=P) == 1 and b"history" in _lib.lib().orch_last_error()
    assert logits(bi=P, bv=P, bo=P, nb=size) == 1 and b"bias" in _lib.lib().orch_last_error()
