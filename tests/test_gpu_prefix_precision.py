"""Attention weights keep their fp32 value through the product with V (GPU), whatever the number of
rows and heads in the call and on every kind of tile.

Bound: the output is rounded to fp16 once (2^-11 of it). A weight in two fp16 terms is off by 2^-22 of
itself, the exponential by 2^-22, and the fp32 scores by 2^-20 of the largest sum of |q k| at most
(head_dim products of 24 bits, added in groups of 16): together below 2^-19 (largest + 1) of
sum p |v|. Queries are small, so that this is far below the 2^-12 that a weight rounded to fp16
once may be off."""

import numpy as np
import pytest
import torch

from oracle import serving
from test_gpu_serving import D, attention, case, device, flags  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,hd,nh,nkv,plen,bound,lens,cap", [
    (12, 128, 8, 8, 0, 0, 17, 64),       # own entries by single warps
    (12, 64, 16, 8, 0, 0, 23, 700),      # own entries by tiles, joined
    (70, 32, 2, 2, 19, 0, 3, 8),         # a prefix on mma.sync tiles
    (2, 128, 64, 64, 40, 0, 9, 20),
    (64, 128, 2, 2, 16, 40000, 0, 8),    # tcgen05 tiles of 128 rows
    (64, 64, 3, 3, 130, 40000, 0, 8),
    (128, 64, 8, 2, 21, 40000, 2, 8),    # of 256 rows
    (100, 128, 4, 1, 257, 40000, 0, 8)])
def test_weights_are_not_rounded_to_fp16(rows, hd, nh, nkv, plen, bound, lens, cap):
    units = [(0, rows, 0, plen)] if plen else []
    q, kp, vp, units, kc, vc, lens, slots = case(rows + plen, hd, nh, nkv, units, [lens] * rows, cap, pcap=max(plen, 1), qs=0.125)
    pad = np.zeros((1, nkv, max(0, bound - plen), hd), np.float16)
    got = attention(D(q), D(np.concatenate([kp, pad], 2)), D(np.concatenate([vp, pad], 2)), D(units) if plen else None, D(kc), D(vc),
                    D(lens), D(slots), max_prefix=max(plen, bound)).double().cpu().numpy()
    want, absv, _, big = serving.attention_prefix(q, kp, vp, units, kc, vc, lens, slots)
    limit = 2.0 ** -11 * np.abs(want) + 2.0 ** -19 * (big + 1) * absv + 2.0 ** -25
    assert np.all(np.abs(got - want) <= limit), float((np.abs(got - want) / limit).max())
    assert flags() == 0
