"""orch_cache_evict with outputs that overlap its inputs otherwise than in place: CTAs of one row would
read lengths or masses that others have already written, so they are refused."""

import pytest

from orchard_b200 import _lib
from test_serving_args import P, evict, pytestmark  # noqa: F401 (no GPU may see the pointers)

# 3 rows, 4 slots of 2 heads x 8 entries: lens 12 B, masses 256 B
SHAPE = dict(M=3, nkv=2, cap=8, ns=4, lens=P, slots=P + 1024, mass=P + 2048, pos=P + 4096, lo=P + 512, mo=P + 8192, po=P + 16384)


@pytest.mark.parametrize("kw", [dict(lo=P + 4), dict(lo=P + 8), dict(lens=P + 516), dict(lo=P + 1024), dict(lo=P + 1032), dict(lo=P + 1016),
                                dict(mo=P + 2048 + 4), dict(mo=P + 2048 + 252), dict(mo=P + 2048 - 252), dict(po=P + 4096 + 64),
                                dict(mo=P + 4096), dict(po=P + 2048 + 128), dict(mo=P + 16384 + 128), dict(lo=P + 2048), dict(lo=P + 4096 + 252),
                                dict(lo=P + 8192 + 8), dict(lo=P + 16384 - 8)])
def test_overlapping_outputs_are_refused(kw):
    assert evict(**{**SHAPE, **kw}) == 1 and b"overlap" in _lib.lib().orch_last_error()


@pytest.mark.parametrize("kw", [dict(), dict(lo=P + 12), dict(mo=P + 2048 + 256), dict(po=P + 4096 - 256), dict(lo=P + 1012), dict(lo=P + 1036),
                                dict(slots=None), dict(mo=P + 2048, po=P + 4096)])
def test_neighbours_and_in_place_pass_the_checks(kw):
    """Without a device the call fails after them, for want of one."""
    assert evict(**{**SHAPE, **kw}) != 1
