"""How orch_attention_prefix cuts a call, seen through the size of its workspace (no device needed):
one record of head_dim + 2 floats per (row, head) and key range."""

import pytest

from orchard_b200 import _lib


def ranges(M, nh, nkv, hd, units, prefix, own):
    n = _lib.lib().orch_attention_prefix_workspace_bytes(M, nh, nkv, hd, units, prefix, own, 0)
    return n / 4 / (M * nh * (hd + 2))


@pytest.mark.parametrize("rows,per,G,nkv", [(128, 4, 4, 8), (128, 8, 1, 32), (64, 8, 1, 32), (512, 4, 1, 32)])
def test_many_small_units_are_cut_by_a_unit_s_rows(rows, per, G, nkv):
    """Units of up to 16 query rows take tiles of 16, as many CTAs as fill the SMs a few times: cut into
    the same ranges however many of them there are (by the rows of the whole batch they would take
    tiles of 128 or 256 rows, nearly all of them empty, one CTA per SM)."""
    one = ranges(per, nkv * G, nkv, 64, 1, 1024, 16)
    many = ranges(rows, nkv * G, nkv, 64, rows // per, 1024, 16)
    assert one == int(one) and many == int(many) and many >= 2
    # two rounds of three CTAs per SM (148), in ranges of 256 keys at least, and one of own entries
    want = min(-(-6 * 148 // (nkv * (rows // per))), 4)
    assert many == want + 1, (many, want)
