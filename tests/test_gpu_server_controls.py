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


@pytest.mark.parametrize("hidden,heads,rows", [(512, 16, 6), (1024, 8, 12)])
def test_batches_of_many_heads_give_the_engine_s_own_tokens(hidden, heads, rows):
    """Rows x heads above 64, with and without the prompts' common beginning held apart: the tokens
    of generate_batch_ids, as far as its logits tell two tokens apart (1e-3 of the largest; both
    sides round fp16 activations in another order)."""
    cfg = dict(hidden_size=hidden, num_attention_heads=heads, intermediate_size=512, num_hidden_layers=2, vocab_size=300,
               rms_norm_eps=1e-5, max_position_embeddings=512)
    _, raw = om.random_model(cfg, seed=6)
    llm = Llama(checkpoint=from_tensors(cfg, hf_tensors(raw, 2)), max_batch=rows, max_seq=160)
    g = np.random.default_rng(hidden)
    head = g.integers(3, 300, 40).tolist()
    tails = [g.integers(3, 300, 3 + 5 * i).tolist() for i in range(rows)]
    whole = [head + t for t in tails]
    steps = 10
    want = llm.generate_batch_ids(whole, max_tokens=steps, temperature=0, ignore_eos=True)
    for srv, prompts in ((serving.BatchServer(llm), whole), (serving.BatchServer(llm, prefix=head), tails)):
        got = srv.generate(prompts, max_tokens=steps, ignore_eos=True)
        for n in range(1, steps + 1):  # a row is compared up to its first difference
            if all(got[b][:n] == want[b][:n] for b in range(rows)):
                continue
            llm.generate_batch_ids(whole, max_tokens=n, temperature=0, ignore_eos=True)
            lg = llm.engine.logits[:rows].cpu().numpy()
            for b in range(rows):
                if got[b][:n] != want[b][:n] and got[b][:n - 1] == want[b][:n - 1]:
                    assert lg[b, want[b][n - 1]] - lg[b, got[b][n - 1]] <= 1e-3 * np.abs(lg[b]).max(), (b, n)
        llm.generate_batch_ids(whole, max_tokens=1, temperature=0, ignore_eos=True)
        first = llm.engine.logits[:rows].cpu().numpy().copy()
        srv.generate(prompts, max_tokens=1, ignore_eos=True)
        assert rel_err(llm.engine.logits[:rows].cpu().numpy(), first) <= 2e-3
