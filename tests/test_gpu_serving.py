"""Serving operators through the C ABI against 64-bit NumPy (GPU): attention over shared
prefixes with tracked weights, eviction from the cache, logits processing.

Error bounds, from the formats (u = 2^-11, half a unit in the last place of fp16):
* attention: each weight is rounded to fp16 once (u sum p|v|), the output once (u |out|); the
  scores' fp32 error moves the weights by another 2^-20 of the largest sum of |q k|.
* tracked weights: fp32; twice the scores' error, and a few 2^-22 from the exponentials.
* eviction: whole numbers and copies, equal.
* logits: three or four fp32 operations (2^-22 of the values' magnitudes), or one fp16 rounding.
"""

import ctypes as C

import numpy as np
import pytest
import torch

from oracle import serving
from orchard_b200 import _lib
from orchard_b200._lib import F16, F32, call

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


def rng(*key):
    return np.random.default_rng([20261206, *key])


def D(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ------------------------------------------------------------------ attention over a prefix
def attention(q, kp, vp, units, kc, vc, lens, slots, mass=None, max_prefix=None, max_own=None, out=None):
    """Device tensors in, output (and mass, in place) out."""
    M, nh, hd = q.shape
    nkv, cap = kc.shape[1], kc.shape[2]
    nu = 0 if units is None else units.shape[0]
    max_prefix = (kp.shape[2] if nu else 0) if max_prefix is None else max_prefix
    max_own = cap if max_own is None else max_own
    n = _lib.lib().orch_attention_prefix_workspace_bytes(M, nh, nkv, hd, nu, max_prefix, max_own, int(mass is not None))
    ws = torch.full((n // 4 + 4,), float("nan"), device="cuda")
    out = torch.full((M, nh, hd), 7.0, dtype=torch.float16, device="cuda") if out is None else out
    call("orch_attention_prefix", q, kp, vp, units, nu, max_prefix, kp.shape[2] if nu else 0, kp.shape[0] if nu else 0,
         kc, vc, lens, slots, max_own, cap, kc.shape[0], mass, out, M, nh, nkv, hd, ws, n, S())
    return out


def case(seed, hd, nh, nkv, units, lens, cap, nslots=None, prefixes=1, pcap=1, poison=True, qs=1.0):
    """Host arrays; entries past the lengths (and prefix entries no unit reads) hold NaN and
    infinities, as memory that nothing wrote may."""
    g = rng(1, seed, hd, nh)
    M = len(lens)
    nslots = nslots or M
    half = lambda *s: g.standard_normal(s, dtype=np.float32).astype(np.float16)  # noqa: E731
    q, kp, vp = half(M, nh, hd) * np.float16(qs), half(prefixes, nkv, pcap, hd), half(prefixes, nkv, pcap, hd)
    kc, vc = half(nslots, nkv, cap, hd), half(nslots, nkv, cap, hd)
    slots = g.permutation(nslots)[:M].astype(np.int32)
    if poison:
        for p in range(prefixes):
            n = max([u[3] for u in units if u[2] == p], default=0)
            kp[p, :, n:], vp[p, :, n:] = np.inf, np.nan
        full = {int(s): int(n) for s, n in zip(slots, lens)}
        for s in range(nslots):
            kc[s, :, full.get(s, 0):], vc[s, :, full.get(s, 0):] = np.nan, -np.inf
    return q, kp, vp, np.asarray(units, np.int32).reshape(-1, 4), kc, vc, np.asarray(lens, np.int32), slots


def check_attention(host, mass=None, got=None):
    q, kp, vp, units, kc, vc, lens, slots = host
    dm = None if mass is None else D(mass)
    if got is None:
        got = attention(D(q), D(kp), D(vp), D(units) if len(units) else None, D(kc), D(vc), D(lens), D(slots), dm)
    want, absv, wmass, big = serving.attention_prefix(q, kp, vp, units, kc, vc, lens, slots, mass)
    o = got.double().cpu().numpy()
    bound = 2.0 ** -11 * (np.abs(want) + absv) + 2.0 ** -19 * big * absv + 2.0 ** -24
    assert np.all(np.abs(o - want) <= bound), float((np.abs(o - want) / bound).max())
    if mass is not None:
        m = dm.double().cpu().numpy()
        rel = 2 * 2.0 ** -19 * big + 2.0 ** -19
        w = np.abs(wmass) + 1e-30
        assert np.all(np.abs(m - wmass) <= rel * w), float((np.abs(m - wmass) / w).max() / rel)
    assert flags() == 0
    return got


@pytest.mark.parametrize("hd,nh,nkv", [(32, 2, 2), (64, 6, 2), (128, 8, 1), (128, 4, 4), (64, 20, 1), (32, 40, 1), (128, 70, 1)])
@pytest.mark.parametrize("plen,lens", [(0, [1, 5, 64]), (1, [0, 1, 2]), (63, [0, 63, 200]), (64, [64, 65, 1]),
                                       (129, [0, 0, 0]), (700, [3, 130, 517])])
def test_prefix_attention(hd, nh, nkv, plen, lens):
    units = [(0, 3, 0, plen)] if plen else []
    check_attention(case(plen, hd, nh, nkv, units, lens, 520, nslots=5, pcap=max(plen, 1) + 3))


@pytest.mark.parametrize("rows", [1, 2, 9, 16, 17, 33, 64, 65, 128])
@pytest.mark.parametrize("nh,nkv", [(2, 2), (4, 1)])
def test_prefix_rows_per_unit(rows, nh, nkv):
    lens = [(7 * i) % 40 for i in range(rows)]
    check_attention(case(rows, 128, nh, nkv, [(0, rows, 0, 333)], lens, 40, pcap=340))


@pytest.mark.parametrize("bound", [0, 40000])
@pytest.mark.parametrize("hd,nh,nkv,rows,plen", [(128, 2, 2, 33, 1), (128, 2, 2, 64, 129), (64, 6, 2, 50, 63), (64, 20, 1, 3, 700),
                                                 (128, 70, 1, 3, 128), (128, 4, 1, 65, 333), (64, 4, 1, 128, 1000)])
def test_prefix_tiles_by_the_bound(hd, nh, nkv, rows, plen, bound):
    """Both kinds of prefix tiles at the same lengths: a bound far above them asks for the tcgen05
    tiles (blocks of 128 x 128 are counted by the bounds), whose last blocks then end anywhere."""
    host = case(rows + plen, hd, nh, nkv, [(0, rows, 0, plen)], [(7 * i) % 40 for i in range(rows)], 40, pcap=plen + 5)
    q, kp, vp, units, kc, vc, lens, slots = host
    pad = np.zeros((1, nkv, max(0, bound - plen - 5), hd), np.float16)
    t = [D(x) for x in (q, np.concatenate([kp, pad], 2), np.concatenate([vp, pad], 2), units, kc, vc, lens, slots)]
    check_attention(host, got=attention(*t, max_prefix=max(plen, bound)))


@pytest.mark.parametrize("rows,nh,nkv,hd,plen", [(128, 32, 32, 128, 1777), (96, 32, 8, 64, 2500), (40, 160, 160, 64, 1300)])
def test_prefix_of_many_blocks_per_range(rows, nh, nkv, hd, plen):
    """Enough row tiles that one CTA goes through a long range; scores that grow along the keys,
    so that the running scale has to move again and again."""
    q, kp, vp, units, kc, vc, lens, slots = case(rows, hd, nh, nkv, [(0, rows, 0, plen)], [(3 * i) % 7 for i in range(rows)], 8, pcap=plen)
    for k in (kp, kc):
        k[...] = 0.25 * k + np.float16(0.5) * np.sign(q[0, 0, :]) * (np.arange(k.shape[2]) % 640 / 64)[:, None].astype(np.float16)
    t = [D(x) for x in (q, kp, vp, units, kc, vc, lens, slots)]
    out = attention(*t).double()
    M, G = rows, nh // nkv
    k, v = t[1][0, :, :plen].double(), t[2][0, :, :plen].double()
    for m in range(0, M, 13):
        n, s = int(lens[m]), int(slots[m])
        kk, vv = torch.cat([k, t[4][s, :, :n].double()], 1), torch.cat([v, t[5][s, :, :n].double()], 1)
        qq = t[0][m].double().view(nkv, G, hd)
        p = torch.softmax(torch.einsum("kgd,kjd->kgj", qq, kk) / hd ** 0.5, -1)
        want, absv = torch.einsum("kgj,kjd->kgd", p, vv), torch.einsum("kgj,kjd->kgd", p, vv.abs())
        big = float(torch.einsum("kgd,kjd->kgj", qq.abs(), kk.abs()).max() / hd ** 0.5)
        err = (out[m].view(nkv, G, hd) - want).abs()
        assert (err <= 2.0 ** -11 * (want.abs() + absv) + 2.0 ** -19 * big * absv + 2.0 ** -24).all()
    assert flags() == 0


def test_several_units_and_rows_in_none():
    """Three units of different sizes and lengths (one of length 0, two with one prefix), rows
    before, between and after them without any, rows with nothing at all."""
    lens = [4, 0, 3, 9, 0, 17, 1, 0, 80, 2, 5, 0]
    units = [(1, 3, 1, 150), (4, 1, 0, 0), (6, 4, 1, 77)]
    got = check_attention(case(5, 64, 8, 4, units, lens, 80, nslots=15, prefixes=2, pcap=151))
    assert not got[4].any() and not got[11].any()  # an empty unit, no unit: zeros


def test_large_scores_and_one_dominant_key():
    """Scores of several hundred: the running maximum moves a long way, small weights vanish."""
    host = case(11, 128, 4, 4, [(0, 4, 0, 500)], [300, 1, 77, 0], 300, pcap=500, qs=16.0)
    check_attention(host)


def test_infinite_and_nan_keys_inside_the_lengths():
    """What is attended to propagates as softmax does: a NaN key makes its rows NaN, a key of
    score -inf gets no weight; other rows and heads are untouched."""
    q, kp, vp, units, kc, vc, lens, slots = case(12, 64, 2, 2, [(0, 3, 0, 70)], [5, 6, 7], 8, pcap=70, poison=False)
    q[:, :, 0] = np.abs(q[:, :, 0]) + np.float16(0.5)
    kc[slots[0], 0, 2, 0] = np.nan
    kc[slots[1], 1, 3, 0] = -np.inf
    out = attention(D(q), D(kp), D(vp), D(units), D(kc), D(vc), D(lens), D(slots)).cpu().numpy()
    assert np.isnan(out[0, 0]).all() and np.isfinite(out[0, 1]).all() and np.isfinite(out[1:]).all()
    kc[slots[0], 0, 2, 0] = 1.0
    k2, v2, l2 = kc.copy(), vc.copy(), lens.copy()
    t = slots[1]  # the -inf key of (row 1, head 1) dropped by hand
    k2[t, 1, 3:5], v2[t, 1, 3:5] = kc[t, 1, 4:6], vc[t, 1, 4:6]
    l2[1] -= 1
    want, absv, _, big = serving.attention_prefix(q, kp, vp, units, k2, v2, l2, slots)
    bound = 2.0 ** -11 * (np.abs(want) + absv) + 2.0 ** -19 * big * absv + 2.0 ** -24
    assert np.all(np.abs(out[1, 1] - want[1, 1]) <= bound[1, 1])


@pytest.mark.parametrize("hd,nh,nkv,plen,lens", [(128, 4, 4, 0, [577]), (64, 60, 3, 100, [66]), (32, 5, 5, 77, [0]),
                                                 (128, 32, 32, 0, [190]), (64, 70, 1, 10, [40]), (128, 6, 2, 130, [1]), (64, 8, 2, 100, [1, 2, 63, 64, 65, 0]),
                                                 (32, 6, 1, 30, [1500, 3]), (128, 40, 2, 0, [1, 1030])])
def test_tracked_weights(hd, nh, nkv, plen, lens):
    M = len(lens)
    units = [(0, M, 0, plen)] if plen else []
    cap = max(1500 if M > 1 else 0, max(lens), 1)
    host = case(20 + M, hd, nh, nkv, units, lens, cap, nslots=M + 1, pcap=max(plen, 1))
    mass = rng(2, M).random((M + 1, nkv, cap), dtype=np.float32)
    check_attention(host, mass)


def test_tracked_rows_that_share_a_slot_add_in_row_order():
    """The last tokens of a prompt as rows of one call: each row sees one entry more, and the
    sums repeat bit for bit."""
    lens, T = [40, 41, 42, 7, 43], 2
    q, kp, vp, units, kc, vc, _, _ = case(30, 64, 4, 2, [], lens, 50, nslots=3, poison=False)
    slots = np.array([T, T, T, 0, T], np.int32)
    mass = rng(3).random((3, 2, 50), dtype=np.float32)
    host = (q, kp, vp, units, kc, vc, np.asarray(lens, np.int32), slots)
    check_attention(host, mass)
    runs = []
    for _ in range(3):
        dm = D(mass)
        attention(D(q), D(kp), D(vp), None, D(kc), D(vc), D(host[6]), D(slots), dm)
        runs.append(dm.cpu())
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_prefix_attention_repeats_and_serves_a_captured_graph():
    """Bit-equal repeats; a graph captured with bounds above the lengths serves other lengths."""
    q, kp, vp, units, kc, vc, lens, slots = case(40, 128, 8, 2, [(0, 6, 0, 900)], [1, 2, 30, 64, 200, 256], 256, pcap=900,
                                                poison=False)
    t = [D(x) for x in (q, kp, vp, units, kc, vc, lens, slots)]
    a = attention(*t)
    assert torch.equal(a, attention(*t))
    out = torch.zeros_like(a)
    n = _lib.lib().orch_attention_prefix_workspace_bytes(6, 8, 2, 128, 1, 900, 256, 0)
    ws = torch.zeros(n // 4 + 4, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call("orch_attention_prefix", t[0], t[1], t[2], t[3], 1, 900, 900, 1, t[4], t[5], t[6], t[7], 256, 256, 6, None,
             out, 6, 8, 2, 128, ws, n, S())
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, out)
    units[0, 3], lens[:] = 65, [256, 0, 1, 9, 63, 17]
    t[3].copy_(D(units))
    t[6].copy_(D(lens))
    g.replay()
    torch.cuda.synchronize()
    check_attention((q, kp, vp, units, kc, vc, lens, slots), got=out)


@pytest.mark.parametrize("rows,nh,nkv", [(64, 32, 32), (70, 44, 11), (20, 4, 4)])
def test_captured_calls_in_a_row(rows, nh, nkv):
    """Large units (the prefix in a kernel of its own beside the own entries') and small ones: several calls that share a workspace, captured back to back and replayed with other lengths,
    weights added up in call order."""
    lens = [(11 * i) % 60 for i in range(rows)]
    q, kp, vp, units, kc, vc, lens, slots = case(70, 128, nh, nkv, [(0, rows, 0, 900)], lens, 64, pcap=900, poison=False)
    t = [D(x) for x in (q, kp, vp, units, kc, vc, lens, slots)]
    mass = torch.zeros((rows, nkv, 64), device="cuda")
    outs = [torch.zeros((rows, nh, 128), dtype=torch.float16, device="cuda") for _ in range(4)]
    n = _lib.lib().orch_attention_prefix_workspace_bytes(rows, nh, nkv, 128, 1, 900, 64, 1)
    ws = torch.zeros(n // 4 + 4, device="cuda")
    q2 = t[0].flip(0).contiguous()

    def calls():
        for i, o in enumerate(outs):
            call("orch_attention_prefix", q2 if i % 2 else t[0], t[1], t[2], t[3], 1, 900, 900, 1, t[4], t[5], t[6], t[7], 64,
                 64, rows, mass, o, rows, nh, nkv, 128, ws, n, S())

    calls()
    torch.cuda.synchronize()
    mass.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        calls()
    for step in range(2):
        if step:
            units[0, 3], lens = 513, np.asarray([(7 * i + 3) % 65 for i in range(rows)], np.int32)
            t[3].copy_(D(units))
            t[6].copy_(D(lens))
        mass.zero_()
        g.replay()
        torch.cuda.synchronize()
        check_attention((q, kp, vp, units, kc, vc, lens, slots), got=outs[0])
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
        # each call adds the same weights again, and starts the newest entry anew
        zero = np.zeros((rows, nkv, 64), np.float64)
        _, _, w1, big = serving.attention_prefix(q, kp, vp, units, kc, vc, lens, slots, zero)
        o2, absv, w2, big2 = serving.attention_prefix(q[::-1], kp, vp, units, kc, vc, lens, slots, zero)
        bound = 2.0 ** -11 * (np.abs(o2) + absv) + 2.0 ** -19 * big2 * absv + 2.0 ** -24
        assert np.all(np.abs(outs[1].double().cpu().numpy() - o2) <= bound)
        want = 2 * (w1 + w2)
        for m in range(rows):
            if lens[m]:
                want[slots[m], :, lens[m] - 1] = w2[slots[m], :, lens[m] - 1]
        rel = 2 * 2.0 ** -19 * max(big, big2) + 2.0 ** -19
        assert np.all(np.abs(mass.double().cpu().numpy() - want) <= rel * np.abs(want) + 1e-30)


@pytest.mark.parametrize("track,cap", [(True, 10), (False, 10), (False, 700)])
def test_prefix_attention_skips_bad_rows_and_units(track, cap):
    q, kp, vp, units, kc, vc, lens, slots = case(50, 64, 4, 2, [(0, 2, 0, 30), (2, 2, 0, 30), (4, 2, 0, 30)], [3, 4, 5, 6, 7, 8],
                                                cap, nslots=6, pcap=30, poison=False)
    mass = torch.zeros((6, 2, cap), device="cuda")

    def go(u=units, n=lens, s=slots):
        mass.zero_()
        return attention(D(q), D(kp), D(vp), D(u), D(kc), D(vc), D(n), D(s), mass if track else None).cpu()

    good = go()
    assert flags() == 0

    for bad in (-1, cap + 1, 2 ** 31 - 1):
        n = lens.copy()
        n[1] = bad
        o = go(n=n)
        assert flags() == 2 and (o[1] == 7).all() and torch.equal(o[[0, 2, 3, 4, 5]], good[[0, 2, 3, 4, 5]])
        assert not mass[slots[1]].any() and bool(mass[slots[0]].any()) == track
    for bad in (-1, 6, 2 ** 31 - 1):
        s = slots.copy()
        s[4] = bad
        o = go(s=s)
        assert flags() == 8 and (o[4] == 7).all() and torch.equal(o[[0, 1, 2, 3, 5]], good[[0, 1, 2, 3, 5]])
    for u1, bit in (((2, 2, 1, 30), 8), ((2, 2, -1, 30), 8), ((2, 2, 0, 31), 2), ((2, 2, 0, -1), 2), ((2, 129, 0, 30), 2)):
        u = units.copy()
        u[1] = u1
        o = go(u=u)
        assert flags() == bit and (o[2:4] == 7).all() and torch.equal(o[:2], good[:2])
        assert u1[1] == 129 or torch.equal(o[4:], good[4:])
    u = units.copy()
    u[2] = (4, 3, 0, 30)  # one row more than there are
    o = go(u=u)
    assert flags() == 2 and (o[4:] == 7).all() and torch.equal(o[:4], good[:4])
    u = units.copy()
    u[1] = (1, 3, 0, 30)  # row 1 in two units
    o = go(u=u)
    assert flags() == 2 and (o[1] == 7).all() and (o[0] != 7).any()


def test_prefix_attention_beyond_32_bit_offsets():
    """A cache of more than 2^31 elements and a prefix region of more than 2^31: the last slot
    and the last prefix are the ones in use."""
    nkv, hd, cap, nslots = 8, 128, 32768, 66
    assert nslots * nkv * cap * hd > 2 ** 31
    kc = torch.empty((nslots, nkv, cap, hd), dtype=torch.float16, device="cuda")
    vc = torch.empty_like(kc)
    kp, vp = torch.empty_like(kc), torch.empty_like(kc)
    g = torch.Generator(device="cuda").manual_seed(5)
    for t in (kc, vc, kp, vp):
        t[-1].normal_(generator=g)
    q = torch.randn((2, nkv, hd), generator=g, device="cuda", dtype=torch.float16)
    lens, slots = torch.tensor([cap, 0], dtype=torch.int32, device="cuda"), torch.tensor([nslots - 1, 3], dtype=torch.int32, device="cuda")
    units = torch.tensor([[0, 2, nslots - 1, cap]], dtype=torch.int32, device="cuda")
    out = attention(q, kp, vp, units, kc, vc, lens, slots).double()
    for m in range(2):
        k = torch.cat([kp[-1], kc[-1]] if m == 0 else [kp[-1]], dim=1).double()
        v = torch.cat([vp[-1], vc[-1]] if m == 0 else [vp[-1]], dim=1).double()
        p = torch.softmax(torch.einsum("hd,hjd->hj", q[m].double(), k) / hd ** 0.5, -1)
        want, absv = torch.einsum("hj,hjd->hd", p, v), torch.einsum("hj,hjd->hd", p, v.abs())
        assert ((out[m] - want).abs() <= 2.0 ** -11 * (want.abs() + absv) + 2.0 ** -15 * absv + 2.0 ** -24).all()
    assert flags() == 0


def test_serving_operators_on_another_stream():
    host = case(60, 64, 4, 2, [(0, 3, 0, 100)], [9, 60, 0], 64, pcap=100)
    t = [D(x) for x in host]
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        out = attention(*t)
    st.synchronize()
    check_attention(host, got=out)


# ------------------------------------------------------------------------------ eviction
def evict_state(seed, M, nkv, hd, cap, lens, nslots=None, ties=True):
    g = rng(4, seed, M, cap)
    nslots = nslots or M
    mass = np.exp(2 * g.standard_normal((nslots, nkv, cap), dtype=np.float32)).astype(np.float32)
    if ties:
        mass[g.random(mass.shape) < 0.3] = 0.0
        mass[g.random(mass.shape) < 0.1] = 1.0
    pos = np.stack([np.stack([g.permutation(3 * cap)[:cap] for _ in range(nkv)]) for _ in range(nslots)]).astype(np.int32)
    k = g.standard_normal((nslots, nkv, cap, hd), dtype=np.float32).astype(np.float16)
    v = g.standard_normal((nslots, nkv, cap, hd), dtype=np.float32).astype(np.float16)
    slots = g.permutation(nslots)[:M].astype(np.int32)
    return k, v, mass, pos, np.asarray(lens, np.int32), slots


def evict(k, v, mass, pos, lens, slots, budget, recent, apart):
    """Runs the operator on copies; returns host arrays."""
    dk, dv, dm, dp, dl, ds = (D(x) for x in (k, v, mass, pos, lens, slots))
    mo = torch.full_like(dm, -5.0) if apart else dm
    po = torch.full_like(dp, -5) if apart else dp
    lo = torch.full_like(dl, -5)
    nslots, nkv, cap, hd = k.shape
    call("orch_cache_evict", dk, dv, dm, dp, dl, ds, mo, po, lo, len(lens), nkv, hd, cap, nslots, budget, recent, S())
    return [x.cpu().numpy() for x in (dk, dv, mo, po, lo)]


def check_evict(state, budget, recent, apart):
    k, v, mass, pos, lens, slots = state
    gk, gv, gm, gp, gl = evict(*state, budget, recent, apart)
    wk, wv = k.copy(), v.copy()
    wm, wp = (np.full_like(mass, -5.0), np.full_like(pos, -5)) if apart else (mass.copy(), pos.copy())
    for m, t in enumerate(slots):
        for h in range(k.shape[1]):
            src = serving.cache_evict(mass[t, h], pos[t, h], int(lens[m]), budget, recent)
            n = len(src)
            wk[t, h, :n], wv[t, h, :n] = k[t, h, src], v[t, h, src]
            wm[t, h, :n], wp[t, h, :n] = mass[t, h, src], pos[t, h, src]
    np.testing.assert_array_equal(gl, np.minimum(lens, budget))
    np.testing.assert_array_equal(gp, wp)
    np.testing.assert_array_equal(gm, wm)
    np.testing.assert_array_equal(gk.view(np.uint16), wk.view(np.uint16))
    np.testing.assert_array_equal(gv.view(np.uint16), wv.view(np.uint16))
    assert flags() == 0


@pytest.mark.parametrize("apart", [True, False])
@pytest.mark.parametrize("budget,recent", [(0, 0), (1, 0), (1, 5), (31, 8), (64, 64), (100, 0), (100, 300), (300, 40), (700, 1)])
def test_evict(budget, recent, apart):
    lens = [0, 1, 2, 31, 32, 33, 64, 65, 100, 101, 299, 300, 301, 640]
    check_evict(evict_state(1, len(lens), 2, 64, 640, lens, nslots=16), budget, recent, apart)


@pytest.mark.parametrize("hd", [8, 32, 80, 128, 256])
def test_evict_head_dims(hd):
    check_evict(evict_state(2, 3, 3, hd, 97, [97, 50, 96]), 40, 7, False)


@pytest.mark.parametrize("cap,budget,recent", [(5000, 4999, 100), (9001, 100, 0), (9001, 7777, 3000), (48000, 20000, 5000)])
def test_evict_long(cap, budget, recent):
    """More moves than one list holds; 48,000 entries are past what shared memory stages."""
    check_evict(evict_state(3, 2, 1, 32, cap, [cap, cap - 1]), budget, recent, False)
    check_evict(evict_state(3, 2, 1, 32, cap, [cap, cap - 1]), budget, recent, True)


def test_evict_equal_masses_keep_the_lowest_indices():
    k, v, mass, pos, lens, slots = evict_state(4, 2, 2, 32, 3000, [3000, 2999])
    mass[:] = 0.25
    check_evict((k, v, mass, pos, lens, slots), 1500, 0, False)
    check_evict((k, v, mass, pos, lens, slots), 1500, 700, True)
    pos[:] = 7  # equal positions: all protected, or none
    check_evict((k, v, mass, pos, lens, slots), 1500, 1, False)
    check_evict((k, v, mass, pos, lens, slots), 1500, 0, False)


def test_evict_special_masses():
    k, v, mass, pos, lens, slots = evict_state(5, 2, 2, 32, 500, [500, 333])
    g = rng(9)
    for val in (np.nan, np.inf, -np.inf, -0.0, 0.0, -1.0, 1e-42, -1e-42, np.float32(3.4e38)):
        mass[g.random(mass.shape) < 0.1] = val
    pos[0, 0, :3] = (2 ** 31 - 1, -2 ** 31, 2 ** 31 - 5)
    for budget, recent in ((20, 5), (250, 30), (320, 2 ** 31 - 1), (320, 2 ** 32 - 1), (470, 0)):
        check_evict((k, v, mass, pos, lens, slots), budget, recent, False)


def test_evict_skips_bad_rows():
    state = evict_state(6, 4, 2, 32, 64, [64, 64, 64, 64], nslots=5)
    k, v, mass, pos, lens, slots = state
    for at, bad, bit in ((0, -1, 2), (1, 65, 2), (2, -1, 8), (3, 5, 8), (3, int(slots[1]), 8)):
        n, s = lens.copy(), slots.copy()
        (n if bit == 2 else s)[at] = bad
        gk, gv, gm, gp, gl = evict(k, v, mass, pos, n, s, 20, 4, False)
        assert flags() == bit and gl[at] == -5
        t = slots[at]
        np.testing.assert_array_equal(gk[t].view(np.uint16), k[t].view(np.uint16))
        np.testing.assert_array_equal(gm[t], mass[t])
        ok = [i for i in range(4) if i != at]
        assert (gl[ok] == 20).all()
        for m in ok:
            src = serving.cache_evict(mass[slots[m], 1], pos[slots[m], 1], 64, 20, 4)
            np.testing.assert_array_equal(gp[slots[m], 1, :20], pos[slots[m], 1, src])


def test_evict_beyond_32_bit_offsets():
    nkv, hd, cap, nslots = 8, 128, 32768, 66
    k = torch.empty((nslots, nkv, cap, hd), dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    g = torch.Generator(device="cuda").manual_seed(6)
    for t in (k, v):
        t[-1].normal_(generator=g)
    mass = torch.rand((nslots, nkv, cap), generator=g, device="cuda")
    pos = torch.arange(cap, dtype=torch.int32, device="cuda").expand(nslots, nkv, cap).contiguous()
    k0, v0, m0, p0 = (t[-1].cpu().numpy() for t in (k, v, mass, pos))
    lens, slots = torch.tensor([cap], dtype=torch.int32, device="cuda"), torch.tensor([nslots - 1], dtype=torch.int32, device="cuda")
    lo = torch.zeros_like(lens)
    call("orch_cache_evict", k, v, mass, pos, lens, slots, mass, pos, lo, 1, nkv, hd, cap, nslots, 30000, 100, S())
    torch.cuda.synchronize()
    assert int(lo[0]) == 30000 and flags() == 0
    for h in range(nkv):
        src = serving.cache_evict(m0[h], p0[h], cap, 30000, 100)
        np.testing.assert_array_equal(pos[-1, h, :30000].cpu().numpy(), p0[h, src])
        np.testing.assert_array_equal(k[-1, h, :30000].cpu().numpy(), k0[h, src])
        np.testing.assert_array_equal(v[-1, h, :30000].cpu().numpy(), v0[h, src])


# ------------------------------------------------------------------------------ logits
def bits(allowed, words):
    m = np.zeros(words, np.uint32)
    for v in allowed:
        if v // 32 < words:
            m[v // 32] |= np.uint32(1 << (v % 32))
    return m


def run_logits(x, base=0, ld=None, hist=None, hist_len=None, gen=None, pen=None, bias=None, masks=None, mask_rows=None,
               inplace=False, shift=(0, 0)):
    """x: host [M, V]; bias: per row lists of (id, value); shift: elements that in and out begin
    past an aligned place."""
    M, V = x.shape
    ld = ld or V
    buf = np.full((M, ld), 3.0, x.dtype)
    buf[:, :V] = x
    room = torch.full((M * ld + 64,), 5.0, dtype=D(buf).dtype, device="cuda")
    room2 = torch.full_like(room, 5.0)
    din = room[shift[0]:shift[0] + M * ld].view(M, ld)
    din.copy_(D(buf))
    dout = din if inplace else room2[shift[1]:shift[1] + M * ld].view(M, ld).fill_(9.0)
    ids = vals = off = None
    nb = 0
    if bias is not None:
        off = D(np.cumsum([0] + [len(b) for b in bias]).astype(np.int32))
        nb = sum(len(b) for b in bias)
        ids = D(np.array([v for b in bias for v, _ in b] + [0], np.int32))
        vals = D(np.array([w for b in bias for _, w in b] + [0.0], np.float32))
    call("orch_logits_process", din, dout, F16 if x.dtype == np.float16 else F32, M, V, ld, base,
         None if hist is None else D(hist), 0 if hist is None else hist.shape[1], None if hist_len is None else D(hist_len),
         None if gen is None else D(gen), None if pen is None else D(pen), ids, vals, off, nb,
         None if masks is None else D(masks.view(np.int32)), 0 if masks is None else masks.shape[1],
         0 if masks is None else masks.shape[0], None if mask_rows is None else D(mask_rows), S())
    out = dout.cpu().numpy()
    for r, k in ((room, shift[0]), (room2, shift[0] if inplace else shift[1])):  # nothing around them is touched
        assert (r[:k] == 5).all() and (r[k + M * ld:] == 5).all()
    assert (out[:, V:] == (3.0 if inplace else 9.0)).all()  # columns between rows are not touched
    return out[:, :V]


@pytest.mark.parametrize("dt", [np.float32, np.float16])
@pytest.mark.parametrize("V,M,base,pad", [(1, 2, 0, 0), (31, 3, 0, 1), (64, 1, 40, 0), (1000, 5, 17, 3), (32000, 2, 0, 0),
                                          (9001, 4, 12345, 2), (2047, 6, 0, 0), (2049, 3, 32, 1)])
def test_logits(V, M, base, pad, dt):
    g = rng(7, V, M)
    x = (3 * g.standard_normal((M, V), dtype=np.float32)).astype(dt)
    H = 70
    hist = g.integers(base - 5, base + max(V + 5, 20), (M, H)).astype(np.int32)
    hist[:, ::7] = -1
    hist[:, 1::5] = base + V // 2
    hist_len = np.array([(17 * i + 70) % 71 for i in range(M)], np.int32)
    gen = np.array([(11 * i) % 60 for i in range(M)], np.int32)
    pen = np.stack([1 + g.random(M), g.random(M), g.random(M)], 1).astype(np.float32)
    bias = [[(int(v), float(w)) for v, w in zip(g.integers(base - 3, base + V + 3, 6 * (i % 3)), 5 * g.standard_normal(6 * (i % 3)))]
            for i in range(M)]
    bias[0] = [(base, 1.5), (base, -2.5), (base + V - 1, -np.inf), (base, 0.75)]
    words = (base + V + 31) // 32
    allow = [set(int(v) for v in g.integers(base, base + V, V // 3 + 1)), set(), set(range(base + V))]
    masks = np.stack([bits(a, words) for a in allow])
    mask_rows = np.array([(-1, 0, 2, 1)[i % 4] for i in range(M)], np.int32)
    for inplace, shift in ((False, (0, 0)), (True, (0, 0)), (False, (1, 1)), (True, (3, 3)), (False, (7, 7)), (False, (2, 5))):
        got = run_logits(x, base, V + pad, hist, hist_len, gen, pen, bias, masks, mask_rows, inplace, shift)
        for m in range(M):
            want = serving.logits_process(x[m], base, hist[m, :hist_len[m]], int(gen[m]), pen[m],
                                          [(v, np.float32(w)) for v, w in bias[m]],
                                          None if mask_rows[m] < 0 else allow[mask_rows[m]])
            fin = np.isfinite(want)
            np.testing.assert_array_equal(got[m][~fin], want[~fin].astype(dt))
            u = 2.0 ** -11 if dt == np.float16 else 0.0
            bound = u * np.abs(want[fin]) + 2.0 ** -22 * (np.abs(want[fin]) + 2 * np.abs(x[m][fin]) + 100) + (2.0 ** -25 if u else 0)
            assert np.all(np.abs(got[m][fin] - want[fin]) <= bound)
    assert flags() == 0


def test_logits_parts_alone():
    """Each control without the others; none at all copies the logits bit for bit."""
    x = rng(8).standard_normal((2, 300), dtype=np.float32)
    np.testing.assert_array_equal(run_logits(x), x)
    hist, n = np.array([[5, 5, 9], [1, 2, 3]], np.int32), np.array([3, 0], np.int32)
    got = run_logits(x, hist=hist, hist_len=n, pen=np.array([[2, 0, 0], [2, 1, 1]], np.float32))
    want = x.copy()
    for v in (5, 9):
        want[0, v] = want[0, v] / 2 if want[0, v] > 0 else want[0, v] * 2
    np.testing.assert_array_equal(got, want)
    got = run_logits(x, bias=[[(299, 2.0)], []])
    assert got[0, 299] == np.float32(x[0, 299] + np.float32(2)) and np.array_equal(got[1], x[1])
    got = run_logits(x, masks=bits({7}, 2)[None], mask_rows=np.array([0, -1], np.int32))  # two words only
    assert got[0, 7] == x[0, 7] and np.isneginf(np.delete(got[0], 7)).all() and np.array_equal(got[1], x[1])


def test_logits_infinities():
    """-inf stays -inf under every penalty, a mask ends any value (NaN included), a bias of -inf
    bans an id."""
    x = np.zeros((1, 64), np.float32)
    x[0, :4] = (np.inf, -np.inf, np.nan, 1.0)
    hist = np.array([[0, 1, 2, 3]], np.int32)
    got = run_logits(x, hist=hist, hist_len=np.array([4], np.int32), pen=np.array([[1.5, 0.5, 0.5]], np.float32))
    assert got[0, 0] == np.inf and got[0, 1] == -np.inf and np.isnan(got[0, 2])
    got = run_logits(x, masks=bits({5}, 2)[None], mask_rows=np.zeros(1, np.int32), bias=[[(5, -np.inf)]])
    assert np.isneginf(got).all()


def test_logits_skips_bad_rows():
    x = rng(10).standard_normal((3, 100), dtype=np.float32)
    hist, pen = np.zeros((3, 8), np.int32), np.full((3, 3), 1.25, np.float32)
    for n in ([8, 9, 8], [8, -1, 8], [8, 2 ** 31 - 1, 8]):
        got = run_logits(x, hist=hist, hist_len=np.array(n, np.int32), pen=pen)
        assert flags() == 16 and (got[1] == 9).all() and (got[[0, 2]] != 9).all()
    got = run_logits(x, masks=np.full((2, 4), 2 ** 32 - 1, np.uint32), mask_rows=np.array([0, 2, -7], np.int32))
    assert flags() == 16 and (got[1] == 9).all() and np.array_equal(got[[0, 2]], x[[0, 2]])
    for off in ([0, 2, 1, 3], [0, -1, 2, 3], [0, 1, 4, 4]):  # row 1's range is bad in each; others may be
        dout = torch.full((3, 100), 9.0, device="cuda")
        call("orch_logits_process", D(x), dout, F32, 3, 100, 100, 0, None, 0, None, None, None, D(np.zeros(3, np.int32)),
             D(np.zeros(3, np.float32)), D(np.array(off, np.int32)), 3, None, 0, 0, None, S())
        assert (dout[1] == 9).all() and flags() == 16


@pytest.mark.parametrize("H,nb", [(40001, 3), (9, 70000)])
def test_logits_long_lists(H, nb):
    """Histories past 32,767 ids and bias lists past 65,534 entries: counts and list positions
    that no longer fit half a table word."""
    V = 70
    g = rng(11, H)
    x = g.standard_normal((2, V), dtype=np.float32)
    hist = g.integers(0, V, (2, H)).astype(np.int32)
    hist[0, 5:] = 7
    n, gen = np.array([H, H - 2], np.int32), np.array([0, 3], np.int32)
    pen = np.array([[1.25, 0.5, 2.0 ** -10]] * 2, np.float32)
    bias = [[(int(v), float(np.float32(w))) for v, w in zip(g.integers(0, V, nb), g.standard_normal(nb))], [(3, 1.0)]]
    got = run_logits(x, hist=hist, hist_len=n, gen=gen, pen=pen, bias=bias)
    for m in range(2):
        want = x[m].astype(np.float64)
        ids, c = np.unique(hist[m, gen[m]:n[m]], return_counts=True)
        seen = np.unique(hist[m, :n[m]])
        want[seen] = np.where(want[seen] > 0, want[seen] / 1.25, want[seen] * 1.25)
        want[ids] -= c * 2.0 ** -10 + 0.5
        for v, b in dict(bias[m]).items():
            want[v] += b
        assert np.all(np.abs(got[m] - want) <= 2.0 ** -22 * (np.abs(want) + np.abs(x[m]) + 100))
    assert flags() == 0


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("hd,nh,nkv,rows,plen,cap", [(128, 32, 32, 12, 0, 70), (64, 64, 8, 45, 90, 256), (32, 48, 16, 21, 200, 17),
                                                     (128, 48, 3, 101, 33, 130), (64, 7, 7, 50, 900, 256)])
def test_many_rows_with_short_entries(hd, nh, nkv, rows, plen, cap, track):
    """Enough rows and K/V heads that single warps take the own entries (up to 256 of them), with
    and without a prefix beside them, empty and rejected rows among them."""
    lens = [(i * 37) % (cap + 1) for i in range(rows)]
    host = case(rows + hd, hd, nh, nkv, [(0, rows - 1, 0, plen)] if plen else [], lens, cap, nslots=rows + 2, pcap=max(plen, 1))
    mass = rng(4, rows).random((rows + 2, nkv, cap), dtype=np.float32) if track else None
    got = check_attention(host, mass)
    q, kp, vp, units, kc, vc, n, slots = host
    n, slots = n.copy(), slots.copy()
    n[3], slots[5] = cap + 1, -1
    dm = D(mass) if track else None
    out = attention(D(q), D(kp), D(vp), D(units) if len(units) else None, D(kc), D(vc), D(n), D(slots), dm)
    assert flags() == 2 | 8 and (out[[3, 5]] == 7).all()
    ok = [i for i in range(rows) if i not in (3, 5)]
    assert torch.equal(out[ok], got[ok])
