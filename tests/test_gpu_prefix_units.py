"""Units of orch_attention_prefix that overlap, are rejected or find no room (GPU): rows of valid
units keep their results, or are left unwritten and reported. Error bounds as in
test_gpu_serving.py (another number of units cuts the keys into other ranges, so sums differ in
their last bits from a call without the rejected units)."""

import numpy as np
import pytest
import torch

from oracle import serving
from test_gpu_serving import D, attention, case, device, flags  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu


def go(host, units, bound, mass=None):
    """The output for `units`: NaN wherever it is made of workspace that nothing was written to, 7
    wherever it was not written itself."""
    q, kp, vp, _, kc, vc, lens, slots = host
    pad = np.zeros((kp.shape[0], kp.shape[1], max(0, bound - kp.shape[2]), kp.shape[3]), np.float16)
    return attention(D(q), D(np.concatenate([kp, pad], 2)), D(np.concatenate([vp, pad], 2)),
                     D(np.asarray(units, np.int32).reshape(-1, 4)), D(kc), D(vc), D(lens), D(slots), mass,
                     max_prefix=max(bound, kp.shape[2]) if kp.shape[2] > 1 else 0).cpu()


def expected(host, units):
    """Values, and what each may be off by, for the rows as if `units` were all: outputs, masses."""
    q, kp, vp, _, kc, vc, lens, slots = host
    zero = np.zeros((kc.shape[0], kc.shape[1], kc.shape[2]))
    want, absv, mass, big = serving.attention_prefix(q, kp, vp, units, kc, vc, lens, slots, zero)
    return want, 2.0 ** -11 * (np.abs(want) + absv) + 2.0 ** -19 * big * absv + 2.0 ** -24, mass, (2 * 2.0 ** -19 * big + 2.0 ** -19) * mass


def close(a, want, bound):
    return bool(np.all(np.abs(np.asarray(a, np.float64) - want) <= bound))  # False for a NaN


# rows, units that are taken, units listed before and between them that are not
EMPTY = (0, 0, 0, 0)
SHAPES = [(33, [(0, 33, 0, 300)], [EMPTY], 1), (33, [(0, 33, 0, 300)], [EMPTY] * 31, 1), (128, [(0, 128, 0, 300)], [(5, 0, 0, 1)] * 3, 1),
          (97, [(0, 33, 0, 300), (33, 64, 0, 299)], [(0, -1, 0, 5), (90, 129, 0, 5), EMPTY, (96, 2, 0, 3)], 3)]


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("bound", [0, 40000])
@pytest.mark.parametrize("hd,nh,nkv", [(64, 4, 4), (128, 8, 2), (32, 4, 4)])
@pytest.mark.parametrize("rows,good,bad,every", SHAPES)
def test_rejected_units_take_nothing_from_others(rows, good, bad, every, hd, nh, nkv, bound, track):
    """Records that stand for no rows, or whose rows lie outside the batch, listed among units whose
    query rows end just past a tile, on both kinds of tiles."""
    lens = [(7 * i) % 20 for i in range(rows)]
    host = case(rows, hd, nh, nkv, good, lens, 20, pcap=305)
    mass = torch.zeros((rows, nkv, 20), device="cuda") if track else None
    units = [u for i, g in enumerate(good) for u in (*bad[i::len(good)], g)]
    # rows named by a rejected unit are left out
    out = [m for m in range(rows) if not any(u[0] <= m < u[0] + u[1] for u in bad)]
    named = [m for m in range(rows) if m not in out]
    want, limit, wmass, mlimit = expected(host, good)
    got = go(host, units, bound, mass)
    assert flags() == 2
    assert close(got[out], want[out], limit[out]) and bool((got[named] == 7).all())
    if track:
        at, none = host[7][out], host[7][named]
        mass = mass.cpu().numpy()
        assert close(mass[at], wmass[at], mlimit[at]) and not mass[none].any()


@pytest.mark.parametrize("bound", [0, 40000])
@pytest.mark.parametrize("rows,units,hd,nh,nkv", [(128, [(0, 64, 0, 300)] * 4 + [(64, 64, 0, 300)], 64, 4, 4),
                                                  (200, [(0, 128, 0, 300)] * 2 + [(128, 72, 0, 300)], 64, 4, 4),
                                                  (200, [(0, 128, 0, 300)] * 9 + [(128, 72, 0, 300)], 128, 16, 4),
                                                  (100, [(0, 99, 0, 300)] * 99 + [(99, 1, 0, 77)], 128, 2, 2)])
def test_units_that_overlap(rows, units, hd, nh, nkv, bound):
    """Rows in two units are not written. A row of the unit after them has its result, or is left
    unwritten and reported where the overlapping units used up the call's tiles; no row is made of
    what the workspace held."""
    lens = [(7 * i) % 20 for i in range(rows)]
    last = units[-1]
    host = case(rows, hd, nh, nkv, [last], lens, 20, pcap=305)
    mass = torch.zeros((rows, nkv, 20), device="cuda")
    want, limit, wmass, mlimit = expected(host, [last])
    got = go(host, units, bound, mass)
    assert flags() == 2
    mass = mass.cpu().numpy()
    for m in range(rows):
        t = host[7][m]
        if bool((got[m] == 7).all()):
            assert not mass[t].any(), m
        else:
            assert m >= last[0] and close(got[m], want[m], limit[m]) and close(mass[t], wmass[t], mlimit[t]), m


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("rows,cap", [(3, 10), (3, 700), (70, 30)])
def test_units_without_room_for_a_prefix(rows, cap, track):
    """max_prefix 0: units of length 0 are as none; a longer one is out of range, its rows are left
    unwritten and reported."""
    lens = [(7 * i) % cap for i in range(rows)]
    host = case(rows, 64, 4, 2, [], lens, cap, pcap=1)
    want, limit, wmass, mlimit = expected(host, [])
    for units, left in (([(0, 2, 0, 0), (2, 1, 0, 0)], None), ([(0, 1, 0, 0), (1, 1, 0, 5)], 1)):
        mass = torch.zeros((rows, 2, cap), device="cuda") if track else None
        got = go(host, units, 0, mass)
        assert flags() == (0 if left is None else 2)
        keep = [r for r in range(rows) if r != left]
        assert close(got[keep], want[keep], limit[keep]) and (left is None or bool((got[left] == 7).all()))
        if track:
            at, mass = host[7][keep], mass.cpu().numpy()
            assert close(mass[at], wmass[at], mlimit[at]) and (left is None or not mass[host[7][left]].any())
