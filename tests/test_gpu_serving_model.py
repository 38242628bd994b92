"""BatchServer end to end (GPU): the shared prefix, the bounded cache and the logits controls in
the engine's decode step, against the reference's tokens and against an oracle that keeps a
bounded cache per head and changes the logits by their definitions. Logits tolerance as for
the engine: max|gpu - ref| / max|ref| <= 1e-2."""

import numpy as np
import pytest
import torch

from conftest import rel_err
from oracle import model as om
from oracle import ops, serving as osrv
from orchard_b200 import serving
from orchard_b200.loader import from_tensors
from orchard_b200.model import Llama

pytestmark = pytest.mark.gpu


def hf_tensors(raw, nl):
    names = {"wq": "self_attn.q_proj", "wk": "self_attn.k_proj", "wv": "self_attn.v_proj", "wo": "self_attn.o_proj",
             "w1": "mlp.gate_proj", "w3": "mlp.up_proj", "w2": "mlp.down_proj"}
    t = {"model.embed_tokens.weight": raw["embed"], "model.norm.weight": raw["norm"], "lm_head.weight": raw["lm_head"]}
    for li in range(nl):
        p, L = f"model.layers.{li}.", raw["layers"][li]
        for k, v in names.items():
            t[p + v + ".weight"] = L["fp16"][k]
        t[p + "input_layernorm.weight"], t[p + "post_attention_layernorm.weight"] = L["attn_norm"], L["ffn_norm"]
    return t


CFG = dict(hidden_size=256, num_attention_heads=2, intermediate_size=512, num_hidden_layers=2, vocab_size=300,
           rms_norm_eps=1e-5, max_position_embeddings=512)


@pytest.fixture(scope="module")
def small():
    oracle_model, raw = om.random_model(CFG, seed=5)
    oracle_model.cache_dequant = True
    llm = Llama(checkpoint=from_tensors(CFG, hf_tensors(raw, 2)), max_batch=5, max_seq=160)
    return oracle_model, llm


@pytest.mark.parametrize("graphs", [True, False])
def test_server_without_options_is_generate_batch_ids(golden_model, graphs):
    g = golden_model
    llm = Llama.from_tensors(g["config"], g["ckpt"], max_batch=4, use_graphs=graphs)
    srv = serving.BatchServer(llm)
    assert srv.generate(g["prompts"], max_tokens=g["max_tokens"]) == g["tokens"]
    np.random.seed(g["sample_seed"])
    assert srv.generate(g["prompts"], max_tokens=g["sample_tokens"], temperature=g["sample_t"]) == g["tokens_sampled"]


@pytest.mark.parametrize("cut", [1, 70, 200])
def test_shared_prefix_gives_the_tokens_of_whole_prompts(small, cut):
    """Prompts with a common beginning: what the engine generates from the whole prompts, and the
    oracle's logits at the last step."""
    ref, llm = small
    g = np.random.default_rng(cut)
    head = g.integers(3, 300, cut).tolist()
    tails = [g.integers(3, 300, n).tolist() for n in (1, 9, 30, 17)]
    n = 12
    srv = serving.BatchServer(llm, prefix=head, chunk=23)
    got = srv.generate(tails, max_tokens=n, ignore_eos=True)
    logits = llm.engine.logits[:4].cpu().numpy()
    want = ref.generate([head + t for t in tails], n, 0.0, ignore_eos=True)
    assert got == want
    ref.reset()
    for b, t in enumerate(tails):
        seq = head + t + [t[-1]] + want[b][:-1]
        for i, tok in enumerate(seq[:-1]):
            ref.forward_tokens([tok], [i], [b], logits=False)
        lg = ref.forward_tokens([seq[-1]], [len(seq) - 1], [b])
        assert rel_err(logits[b], lg[0]) <= 1e-2


class BoundedOracle(om.OracleModel):
    """The oracle with a cache that drops entries by weight, per head, and a prefix that stays."""

    def setup(self, plen):
        self.reset()
        self.plen, self.track = plen, False
        self.mass = [dict() for _ in self.layers]
        self.pos = [dict() for _ in self.layers]

    def layer_forward(self, li, x, cos, sin, seq_ids):
        before = {b: self.k_cache[li].get(b, np.zeros((self.heads, 0, 1))).shape[1] for b in seq_ids}
        self._li, self._seq, self._i = li, seq_ids, 0
        keep = ops.attention_one
        ops.attention_one = self.attend
        try:
            out = super().layer_forward(li, x, cos, sin, seq_ids)
        finally:
            ops.attention_one = keep
        assert all(self.k_cache[li][b].shape[1] == n + 1 for b, n in before.items())
        return out

    def attend(self, q, kc, vc):
        b = self._seq[self._i]
        self._i += 1
        s = np.einsum("hd,hld->hl", q.astype(np.float64), kc.astype(np.float64)) / np.sqrt(q.shape[-1])
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        own = kc.shape[1] - self.plen
        if own > 0:
            m = self.mass[self._li].get(b, np.zeros((self.heads, 0)))
            e = self.pos[self._li].get(b, np.zeros((self.heads, 0), np.int64))
            self.mass[self._li][b] = np.concatenate([m, np.zeros((self.heads, 1))], 1)
            self.pos[self._li][b] = np.concatenate([e, np.full((self.heads, 1), self.now[b])], 1)
            if self.track:
                self.mass[self._li][b] += p[:, self.plen:]
        return np.einsum("hl,hld->hd", p, vc.astype(np.float64)).astype(np.float32)

    def feed(self, tok, pos, b, track):
        self.now, self.track = {b: pos}, track
        return self.forward_tokens([tok], [pos], [b])

    def evict(self, b, budget, recent):
        for li in range(len(self.layers)):
            m, e, k, v = self.mass[li][b], self.pos[li][b], self.k_cache[li][b], self.v_cache[li][b]
            n = min(m.shape[1], budget)
            out = [[], [], [], []]
            for h in range(self.heads):
                src = osrv.cache_evict(m[h].astype(np.float32), e[h], m.shape[1], budget, recent)
                for o, a in zip(out, (m[h, src], e[h, src],
                                      np.concatenate([k[h, :self.plen], k[h, self.plen:][src]]),
                                      np.concatenate([v[h, :self.plen], v[h, self.plen:][src]]))):
                    o.append(a)
            self.mass[li][b], self.pos[li][b], self.k_cache[li][b], self.v_cache[li][b] = (np.stack(o) for o in out)
            assert self.mass[li][b].shape[1] == n


@pytest.mark.parametrize("graphs", [True, False])
def test_prefix_budget_and_controls_together(small, graphs):
    """One decode path with all three operators against the bounded oracle, step by step: the
    cache's positions per head, each step's controlled logits and the tokens."""
    ref, llm = small
    g = np.random.default_rng(77)
    head = g.integers(3, 300, 40).tolist()
    tails = [g.integers(3, 300, n).tolist() for n in (60, 25, 41)]
    budget, recent, every, window, steps = 32, 8, 4, 5, 14
    pen = (1.3, 0.4, 0.2)
    bias = {7: 2.0, 250: -1.5}
    words = (300 + 31) // 32
    seen_logits = []

    def allowed(step, answers):
        if step:
            seen_logits.append(llm.engine.logits[:3].cpu().numpy().copy())
        if step % 2:
            return None
        m = np.zeros((3, words), np.uint32)
        for v in range(step, 300, 3):
            m[:, v // 32] |= np.uint32(1 << (v % 32))
        return m

    llm.use_graphs = graphs
    srv = serving.BatchServer(llm, prefix=head, budget=budget, recent=recent, every=every, window=window, chunk=50)
    got = srv.generate(tails, max_tokens=steps, ignore_eos=True,
                       controls=serving.LogitsControls(*pen, bias=bias, allowed=allowed))
    seen_logits.append(llm.engine.logits[:3].cpu().numpy().copy())
    llm.use_graphs = True

    o = BoundedOracle(CFG, ref.layers, ref.embed, ref.norm, ref.lm_head)
    o.cache_dequant = True
    o.setup(len(head))
    own = []
    for b, t in enumerate(tails):
        o.now = {b: 0}
        for i, tok in enumerate(head):
            o.forward_tokens([tok], [i], [b], logits=False)
        for i, tok in enumerate(t):
            o.feed(tok, len(head) + i, b, i >= len(t) - window)
        o.evict(b, budget, recent)
        own.append(min(len(t), budget))
    answers = [[] for _ in tails]
    for s in range(steps):
        for b, t in enumerate(tails):
            tok = t[-1] if s == 0 else answers[b][-1]
            lg = o.feed(tok, len(head) + len(t) + s, b, True)[0]
            ok = None if s % 2 else set(range(s, 300, 3))
            lg = osrv.logits_process(lg, 0, head + t + answers[b], len(head) + len(t), pen, bias.items(), ok)
            fin = np.isfinite(lg)
            mine = seen_logits[s][b]
            assert np.array_equal(np.isfinite(mine), fin), (s, b)
            assert rel_err(mine[fin], lg[fin]) <= 1e-2, (s, b)
            assert got[b][s] == int(np.argmax(mine))
            answers[b].append(got[b][s])
            own[b] += 1
        if max(own) >= budget + every:
            for b in range(3):
                o.evict(b, budget, recent)
                own[b] = min(own[b], budget)
    pos = srv.positions.cpu().numpy()
    for li in range(2):
        for b in range(3):
            for h in range(2):
                assert sorted(pos[li, b, h, :own[b]]) == sorted(o.pos[li][b][h].tolist())


def test_server_refusals(small):
    _, llm = small
    with pytest.raises(ValueError, match="cache"):
        serving.BatchServer(llm, budget=150, every=16)
    with pytest.raises(ValueError, match="positive"):
        serving.BatchServer(llm, budget=10, every=0)
    srv = serving.BatchServer(llm)
    with pytest.raises(ValueError, match="prompts"):
        srv.generate([], max_tokens=1)
    with pytest.raises(ValueError, match="prompts"):
        srv.generate([[1], []], max_tokens=1)
    with pytest.raises(ValueError, match="cache"):
        srv.generate([[1] * 100], max_tokens=100)
    with pytest.raises(ValueError, match="vocabulary"):
        srv.generate([[1]], max_tokens=1, controls=serving.LogitsControls(bias={300: 1.0}))
    with pytest.raises(ValueError, match="positive"):
        srv.generate([[1]], max_tokens=1, controls=serving.LogitsControls(repetition=0.0))
    with pytest.raises(ValueError, match="words"):
        srv.generate([[1]], max_tokens=1, controls=serving.LogitsControls(allowed=lambda s, a: np.zeros((1, 3), np.uint32)))
    with pytest.raises(ValueError, match="empty"):
        serving.SharedPrefix(llm, [])
