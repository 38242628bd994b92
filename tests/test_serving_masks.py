"""Host side of the serving path: grammar masks of a step, before any device work."""

import numpy as np
import pytest

from orchard_b200 import serving


def controls(rows, vocab, **kw):
    return serving.RowControls(serving.LogitsControls(allowed=lambda s, a: None, **kw), rows, vocab, 8, "cpu")


def test_masks_for_fewer_rows_than_the_batch_are_refused():
    """A later step's masks for some rows would leave the others under an earlier step's."""
    rc = controls(3, 70)
    rc.set_masks(np.full((3, 3), 0xFFFFFFFF, np.uint32))
    assert rc.mask_rows.tolist() == [0, 1, 2]
    for shape in ((1, 3), (2, 3), (4, 3), (3, 2), (3,), (0, 3)):
        with pytest.raises(ValueError, match="words"):
            rc.set_masks(np.ones(shape, np.uint32))
    rc.set_masks(None)
    assert rc.mask_rows.tolist() == [-1, -1, -1]


def test_a_mask_that_allows_nothing_is_refused():
    """Per row that still answers; bits past the vocabulary do not count."""
    rc = controls(3, 70)
    m = np.zeros((3, 3), np.uint32)
    m[0, 0], m[2, 2] = 1, 1 << 5  # ids 0 and 69
    m[1, 2] = 1 << 6  # id 70: not in the vocabulary
    with pytest.raises(ValueError, match="row 1"):
        rc.set_masks(m)
    rc.set_masks(m, np.array([True, False, True]))  # row 1 has ended: its mask does not matter
    assert rc.mask_rows.tolist() == [0, -1, 2]
    m[1, 2] = 1 << 31 | 1
    rc.set_masks(m)
    assert rc.mask_rows.tolist() == [0, 1, 2]
    for vocab in (1, 31, 32, 33, 64):
        rc = controls(1, vocab)
        w = (vocab + 31) // 32
        rc.set_masks(serving_bit(vocab - 1, w))
        if vocab % 32:
            with pytest.raises(ValueError, match="row 0"):
                rc.set_masks(serving_bit(vocab, w))


def serving_bit(v, words):
    m = np.zeros((1, words), np.uint32)
    m[0, v // 32] = np.uint32(1 << (v % 32))
    return m
