"""BatchServer's controls where they end a row's choices, change size or meet a draw (GPU), and its
tokens at batches of many heads."""

import numpy as np
import pytest

from conftest import rel_err
from oracle import model as om
from orchard_b200 import serving
from orchard_b200.loader import from_tensors
from orchard_b200.model import EOS_ID, Llama
from test_gpu_serving_model import hf_tensors, small  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu

WORDS = (300 + 31) // 32


def mask(rows):
    m = np.zeros((len(rows), WORDS), np.uint32)
    for r, ids in enumerate(rows):
        for v in ids:
            m[r, v // 32] |= np.uint32(1 << (v % 32))
    return m


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_every_token_is_one_that_the_mask_allows(small, temperature):  # noqa: F811
    _, llm = small
    g = np.random.default_rng(3)
    prompts = [g.integers(3, 300, n).tolist() for n in (5, 12, 3, 20)]
    sets = [[[int(v) for v in g.choice(np.arange(3, 300), 1 + (s + b) % 40, replace=False)] for b in range(4)] for s in range(30)]
    np.random.seed(11)
    out = serving.BatchServer(llm).generate(prompts, max_tokens=30, temperature=temperature, ignore_eos=True,
                                            controls=serving.LogitsControls(1.2, 0.1, 0.1, allowed=lambda s, a: mask(sets[s])))
    assert all(out[b][s] in sets[s][b] for b in range(4) for s in range(30))


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_a_mask_that_allows_nothing_is_refused(small, temperature):  # noqa: F811
    """For a row that still answers; ids past the vocabulary do not count. What the mask of a row
    that has ended says does not matter."""
    _, llm = small
    srv = serving.BatchServer(llm)
    prompts = [[5, 6, 7], [8, 9], [10]]

    def beyond(step, answers):
        m = mask([range(3, 300)] * 3)
        if step == 2:
            m[1] = 0
            m[1, WORDS - 1] = 1 << 20  # id 308
        return m

    with pytest.raises(ValueError, match="row 1"):
        srv.generate(prompts, max_tokens=5, temperature=temperature, ignore_eos=True,
                     controls=serving.LogitsControls(allowed=beyond))

    def ends(step, answers):
        if step == 1:
            return mask([range(3, 300), [EOS_ID], range(3, 300)])
        return mask([range(3, 300), [] if step > 1 else range(3, 300), range(3, 300)])

    out = srv.generate(prompts, max_tokens=6, temperature=temperature, controls=serving.LogitsControls(allowed=ends))
    assert len(out[1]) == 2 and out[1][1] == EOS_ID and len(out[0]) == 6 and len(out[2]) == 6


def test_biases_that_leave_nothing_are_reported(small):  # noqa: F811
    _, llm = small
    with pytest.raises(RuntimeError, match="32"):
        serving.BatchServer(llm).generate([[5, 6, 7], [8]], max_tokens=2, ignore_eos=True,
                                          controls=serving.LogitsControls(bias={v: float("-inf") for v in range(300)}))
