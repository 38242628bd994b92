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
