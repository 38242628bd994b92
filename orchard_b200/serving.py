"""Serving a batch with a shared prefix, a bounded cache and controlled logits.

The reference answers a batch by attending per sequence over a host cache that keeps every
position, and samples from the logits as they are (orchard/model.py:254-381). ``BatchServer``
drives the same fused engine with the three operators that a server of many requests needs
beside it:

* ``orch_attention_prefix``: what all prompts begin with (instructions, a document) is run and
  held once; every row attends to it together with its own entries;
* ``orch_cache_evict``: a row's own entries are bounded; those that attention weighted least go,
  the newest stay;
* ``orch_logits_process``: repetition, presence and frequency penalties, biases and grammar masks.

Without options ``BatchServer.generate`` returns what ``Llama.generate_batch_ids`` returns.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import Callable, Dict, List, Optional, Sequence

import numpy as np
import torch

from . import _lib
from ._lib import F16, F32, call, ptr
from .model import EOS_ID, Llama, RowBuffers, _stream, prefill_units

UNIT_ROWS = 128  # rows of a unit of orch_attention_prefix at most


@dataclass
class LogitsControls:
    """How the next token is chosen, for every row of a batch.

    ``repetition`` divides positive logits of tokens seen before (in prefix, prompt or answer)
    and multiplies negative ones; ``presence`` and ``frequency`` are subtracted once and per
    occurrence for tokens of the answer. ``bias`` maps token ids to additions. ``allowed(step,
    answers)`` returns the step's grammar masks, uint32 ``[rows, ceil(vocab / 32)]`` (bit v & 31
    of word v >> 5 set: token v allowed), or None for no restriction; it is given the answers so
    far, so with it every step waits for the one before. A mask has to leave every row that still
    answers a token; those of rows that have ended are not looked at."""

    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    bias: Dict[int, float] = field(default_factory=dict)
    allowed: Optional[Callable[[int, List[List[int]]], Optional[np.ndarray]]] = None


def prefix_units(rows: int, prefix: int, length: int) -> np.ndarray:
    """Records (row0, rows, prefix, length) of orch_attention_prefix for ``rows`` consecutive
    rows that share one prefix."""
    return np.asarray([(r, min(UNIT_ROWS, rows - r), prefix, length) for r in range(0, rows, UNIT_ROWS)],
                      np.int32).reshape(-1, 4)


class SharedPrefix:
    """Keys and values of a token sequence that several prompts begin with, all layers, fp16
    ``[layers, 1, heads, length, head_dim]``, computed once by the engine's prefill."""

    def __init__(self, llm: Llama, tokens: Sequence[int], chunk: int = 4096):
        eng, c = llm.engine, llm.engine.cfg
        self.tokens = [int(t) for t in tokens]
        self.length = n = len(self.tokens)
        if n == 0:
            raise ValueError("empty prefix")
        if n > eng.max_pos:
            raise ValueError(f"prefix of {n} tokens exceeds the RoPE table ({eng.max_pos})")
        shape = (c.num_hidden_layers, 1, c.num_attention_heads, n, c.head_dim)
        self.k = torch.zeros(shape, dtype=torch.float16, device=eng.device)
        self.v = torch.zeros_like(self.k)
        rows = min(chunk, n)
        b = RowBuffers(rows, c, n, eng.device, logits=False)
        for r0 in range(0, n, rows):
            m = min(rows, n - r0)
            b.tok_in[:m].copy_(torch.as_tensor(np.asarray(self.tokens[r0:r0 + m], np.int32)))
            pos = torch.arange(r0, r0 + m, dtype=torch.int32, device=eng.device)
            serve = ServeRows(m, pos, pos, pos + 1, torch.zeros(m, dtype=torch.int32, device=eng.device),
                              (self.k, self.v), max_own=r0 + m, causal=True)
            eng.run_layers(m, b, serve=serve)


class ServeRows:
    """The rows of one engine call whose caches are not laid out one position after another:
    where their keys go (entry ``index`` of slot ``slots``), what they attend to (``lens`` own
    entries, the prefix) and, with ``mass``, where the weights of the entries are added up."""

    def __init__(self, rows: int, pos, index, lens, slots, caches, max_own: int,
                 prefix: Optional[SharedPrefix] = None, mass=None, causal: bool = False):
        self.pos, self.index, self.lens, self.slots = pos, index, lens, slots
        self.kc, self.vc = caches  # [layers, slots, heads, entries, head_dim]
        self.max_own, self.prefix, self.mass = max_own, prefix, mass
        _, self.num_slots, self.heads, self.cap, self.hd = self.kc.shape
        self.units, self.num_units, self.plen = None, 0, 0
        # rows of prompts that hold every position, one entry after another, and share nothing: the
        # prefill kernel reads a sequence's keys once per 64 rows (head_dim 128)
        self.prefill = None
        if causal and prefix is None and mass is None and self.hd == 128:
            self.prefill = torch.as_tensor(prefill_units(index.cpu().numpy(), slots.cpu().numpy())).to(self.kc.device)
        if prefix is not None:
            self.units = torch.as_tensor(prefix_units(rows, 0, prefix.length)).to(self.kc.device)
            self.num_units, self.plen = self.units.shape[0], prefix.length
        n = _lib.lib().orch_attention_prefix_workspace_bytes(rows, self.heads, self.heads, self.hd, self.num_units,
                                                             self.plen, max_own, int(mass is not None))
        self.ws = torch.empty(max(n, 16), dtype=torch.uint8, device=self.kc.device)

    def append(self, eng, li: int, M: int, b: RowBuffers):
        """RMSNorm, Q/K/V projection (+ LoRA), rotation for ``pos``, K and V into ``index``."""
        L, c, s = eng.layers[li], eng.cfg, _stream()
        H, nh = c.hidden_size, c.num_attention_heads
        tail = (ptr(eng.cos), ptr(eng.sin), eng.max_pos, ptr(b.q), ptr(self.kc[li]), ptr(self.vc[li]), self.cap,
                self.num_slots)
        rows = (ptr(self.pos), ptr(self.index), ptr(self.slots))
        if "qkv" not in L.lora:
            call("orch_q4t_rms_qkv_rope_at", ptr(L.tqkv), ptr(b.x), ptr(L.attn_norm), c.rms_norm_eps, ptr(b.xn), M, H, H,
                 nh, *rows, *tail, s)
            return
        call("orch_rmsnorm_ex", ptr(b.x), F32, ptr(L.attn_norm), F32, ptr(b.xn), F16, c.rms_norm_eps, H, M, s)
        lt, lb, lr = eng._lora(L, "qkv", b.xn, M, s, b)
        call("orch_q4t_qkv_rope_at", ptr(L.tqkv), ptr(b.xn), M, H, H, nh, *rows, *tail, lt, lb, lr, s)

    def attend(self, eng, li: int, M: int, b: RowBuffers):
        p = self.prefix
        if self.prefill is not None:
            call("orch_attention_prefill", ptr(b.q), ptr(self.kc[li]), ptr(self.vc[li]), ptr(self.prefill),
                 self.prefill.shape[0], ptr(b.attn), M, self.heads, self.hd, self.cap, self.num_slots, _stream())
            return
        call("orch_attention_prefix", ptr(b.q), None if p is None else ptr(p.k[li]), None if p is None else ptr(p.v[li]),
             ptr(self.units), self.num_units, self.plen, self.plen, 1 if p is not None else 0, ptr(self.kc[li]),
             ptr(self.vc[li]), ptr(self.lens), ptr(self.slots), self.max_own, self.cap, self.num_slots,
             None if self.mass is None else ptr(self.mass[li]), ptr(b.attn), M, self.heads, self.heads, self.hd,
             ptr(self.ws), self.ws.numel(), _stream())


class RowControls:
    """Device state of LogitsControls for up to ``rows`` rows: token history, penalties, biases
    and the step's masks. ``apply`` runs orch_logits_process on a batch of logits in place."""

    def __init__(self, controls: LogitsControls, rows: int, vocab: int, history: int, device):
        c = controls
        ids = np.asarray(list(c.bias.keys()), np.int32)
        if len(ids) and (ids.min() < 0 or ids.max() >= vocab):
            raise ValueError("bias for a token id outside the vocabulary")
        if c.repetition <= 0:
            raise ValueError("the repetition penalty must be positive")
        i32 = dict(dtype=torch.int32, device=device)
        self.history = torch.zeros((rows, history), **i32)
        self.hist_len, self.gen_start = torch.zeros(rows, **i32), torch.zeros(rows, **i32)
        self.penalties = torch.tensor([[c.repetition, c.presence, c.frequency]] * rows, dtype=torch.float32, device=device)
        self.penal = (c.repetition, c.presence, c.frequency) != (1.0, 0.0, 0.0)
        self.num_bias = rows * len(ids)
        self.bias_ids = torch.as_tensor(np.tile(ids, rows)).to(device)
        self.bias_vals = torch.as_tensor(np.tile(np.asarray(list(c.bias.values()), np.float32), rows)).to(device)
        self.bias_off = torch.arange(0, rows + 1, **i32) * len(ids)
        self.vocab, self.words = vocab, (vocab + 31) // 32
        self.masks = torch.zeros((rows, self.words), **i32) if c.allowed is not None else None
        self.mask_rows = torch.full((rows,), -1, **i32)

    def set_masks(self, masks: Optional[np.ndarray], active: Optional[np.ndarray] = None):
        """The next step's masks, one per row (None: every token allowed); ``active`` (None: all)
        says which rows still answer."""
        if masks is None:
            self.mask_rows.fill_(-1)
            return
        m = np.ascontiguousarray(masks, np.uint32)
        if m.shape != tuple(self.masks.shape):  # fewer rows would leave the others an earlier step's masks
            raise ValueError(f"grammar masks must be [{self.masks.shape[0]} rows, {self.words} words]")
        active = np.ones(len(m), bool) if active is None else np.asarray(active, bool)
        left = m.any(axis=1)
        if self.vocab % 32:  # bits past the vocabulary do not count
            left = m[:, :-1].any(axis=1) | (m[:, -1] & np.uint32((1 << self.vocab % 32) - 1) != 0)
        if (active & ~left).any():
            raise ValueError(f"the grammar mask of row {int(np.argmax(active & ~left))} allows no token")
        self.masks.copy_(torch.from_numpy(m.view(np.int32)))
        self.mask_rows.copy_(torch.from_numpy(np.where(active, np.arange(len(m)), -1).astype(np.int32)))

    def apply(self, logits: torch.Tensor, M: int, V: int):
        pen = self.penal
        call("orch_logits_process", ptr(logits), ptr(logits), F32, M, V, logits.stride(0), 0,
             ptr(self.history) if pen else None, self.history.shape[1] if pen else 0, ptr(self.hist_len) if pen else None,
             ptr(self.gen_start) if pen else None, ptr(self.penalties) if pen else None,
             ptr(self.bias_ids) if self.num_bias else None, ptr(self.bias_vals) if self.num_bias else None,
             ptr(self.bias_off) if self.num_bias else None, self.num_bias,
             None if self.masks is None else ptr(self.masks), self.words, 0 if self.masks is None else self.masks.shape[0],
             None if self.masks is None else ptr(self.mask_rows), _stream())


class BatchServer:
    """Answers batches of prompts on a ``Llama`` (tiled weights, one GPU).

    ``prefix``: tokens that every prompt begins with (prompts are then what follows them).
    ``budget`` > 0 bounds each row's own entries: once a row holds ``budget + every`` of them, all
    rows are cut to ``budget``, of which the ``recent`` newest are protected. The weights that
    decide are those of the last ``window`` prompt tokens and of every decoded token. Without a
    budget a row's entries are limited by the engine's ``max_seq``."""

    def __init__(self, llm: Llama, prefix: Optional[Sequence[int]] = None, budget: int = 0, recent: Optional[int] = None,
                 every: int = 16, window: int = 16, chunk: int = 512):
        eng = llm.engine
        if eng.split is not None or not eng.tiled:
            raise ValueError("BatchServer runs on one GPU with tiled weights")
        if budget < 0 or every < 1 or window < 1:
            raise ValueError("budget must not be negative; every and window must be positive")
        if budget and budget + every > eng.max_seq:
            raise ValueError(f"budget + every ({budget + every}) exceeds the cache ({eng.max_seq} entries per row)")
        self.llm, self.eng = llm, eng
        self.budget, self.every, self.window, self.chunk = budget, every, window, chunk
        self.recent = budget // 4 if recent is None else recent
        self.prefix = SharedPrefix(llm, prefix) if prefix is not None and len(prefix) else None
        self.plen = self.prefix.length if self.prefix else 0
        self.mass = self.positions = None
        if budget:
            shape = eng.k_cache.shape[:4]
            self.mass = torch.zeros(shape, dtype=torch.float32, device=eng.device)
            self.positions = torch.zeros(shape, dtype=torch.int32, device=eng.device)
            nl, B = eng.cfg.num_hidden_layers, eng.max_batch
            # every layer's slots are slots of one cache here, so an eviction is one launch
            self.all_lens = torch.zeros(nl * B, dtype=torch.int32, device=eng.device)
            self.all_lens_out = torch.zeros_like(self.all_lens)

    # -- prompts ------------------------------------------------------------------------
    def _prefill(self, prompts: Sequence[Sequence[int]]):
        """Every prompt token through the layers, ``chunk`` rows at a time in token order; the last
        ``window`` tokens of each prompt in rows of their own whose weights are tracked."""
        eng = self.eng
        keep = [max(0, len(p) - self.window) if self.budget else len(p) for p in prompts]
        parts = [([(s, i) for s, p in enumerate(prompts) for i in range(keep[s])], None),
                 ([(s, i) for s, p in enumerate(prompts) for i in range(keep[s], len(p))], self.mass)]
        if self.budget:
            self.mass.zero_()
            span = torch.arange(self.plen, self.plen + eng.max_seq, dtype=torch.int32, device=eng.device)
            self.positions.copy_(span.expand_as(self.positions))
        for rows, mass in parts:
            for r0 in range(0, len(rows), self.chunk):
                part = np.asarray(rows[r0:r0 + self.chunk], np.int32)
                m = len(part)
                if eng.pre is None or eng.pre.rows < min(self.chunk, len(rows)):
                    eng.pre = RowBuffers(min(self.chunk, len(rows)), eng.cfg, eng.max_seq, eng.device, logits=False)
                b = eng.pre
                d = lambda a: torch.as_tensor(np.ascontiguousarray(a, np.int32)).to(eng.device)  # noqa: E731
                index = d(part[:, 1])
                b.tok_in[:m].copy_(d([prompts[s][i] for s, i in part]))
                serve = ServeRows(m, index + self.plen, index, index + 1, d(part[:, 0]), (eng.k_cache, eng.v_cache),
                                  max_own=int(part[:, 1].max()) + 1, prefix=self.prefix, mass=mass, causal=True)
                eng.run_layers(m, b, serve=serve)

    # -- eviction -----------------------------------------------------------------------
    def _evict(self, lens: np.ndarray) -> np.ndarray:
        """Cuts rows 0 .. len(lens) - 1 of every layer to the budget; returns the new lengths."""
        eng, B, c = self.eng, len(lens), self.eng.cfg
        nl, slots = c.num_hidden_layers, eng.num_slots
        where = (torch.arange(nl, dtype=torch.int32, device=eng.device)[:, None] * slots
                 + torch.arange(B, dtype=torch.int32, device=eng.device)[None, :]).reshape(-1).contiguous()
        n = torch.as_tensor(lens.astype(np.int32)).to(eng.device).repeat(nl)
        self.all_lens[:nl * B].copy_(n)
        call("orch_cache_evict", ptr(eng.k_cache), ptr(eng.v_cache), ptr(self.mass), ptr(self.positions), ptr(self.all_lens),
             ptr(where), ptr(self.mass), ptr(self.positions), ptr(self.all_lens_out), nl * B, c.num_attention_heads,
             c.head_dim, eng.max_seq, nl * slots, self.budget, self.recent, _stream())
        return np.minimum(lens, self.budget)

    # -- answers ------------------------------------------------------------------------
    def generate(self, prompt_ids: Sequence[Sequence[int]], max_tokens: int = 50, temperature: float = 0.0,
                 controls: Optional[LogitsControls] = None, ignore_eos: bool = False) -> List[List[int]]:
        """Token ids in, token ids out, with the token flow and the draws of
        ``Llama.generate_batch_ids``. The decode step (with its masks' place and the history's
        update) is one CUDA graph per call; evictions run between steps."""
        eng, dev = self.eng, self.eng.device
        B = len(prompt_ids)
        lens = np.array([len(p) for p in prompt_ids], np.int64)
        if B == 0 or B > eng.max_batch or lens.min() < 1:
            raise ValueError(f"between 1 and {eng.max_batch} prompts of at least one token each")
        if self.plen + int(lens.max()) + max_tokens > eng.max_pos:
            raise ValueError("prefix + prompt + max_tokens exceed the RoPE table")
        held = int(lens.max()) + (max_tokens if not self.budget else 0)
        if held > eng.max_seq:
            raise ValueError(f"{held} entries per row exceed the cache ({eng.max_seq})")
        self._prefill(prompt_ids)
        own = lens.copy()  # entries of each row
        if self.budget:
            own = self._evict(own)

        i32 = dict(dtype=torch.int32, device=dev)
        pos, index, n_own = torch.zeros(B, **i32), torch.zeros(B, **i32), torch.zeros(B, **i32)
        slots = torch.arange(B, **i32)
        cap = min(eng.max_seq, self.budget + self.every) if self.budget else held
        serve = ServeRows(B, pos, index, n_own, slots, (eng.k_cache, eng.v_cache), max_own=cap, prefix=self.prefix,
                          mass=self.mass)
        rc = None
        if controls is not None:
            rc = RowControls(controls, B, eng.cfg.vocab_size, self.plen + int(lens.max()) + max_tokens, dev)
            head = self.prefix.tokens if self.prefix else []
            for b, p in enumerate(prompt_ids):
                rc.history[b, :self.plen + len(p)].copy_(torch.as_tensor(np.asarray(head + list(p), np.int32)))
            rc.gen_start.copy_(torch.as_tensor((self.plen + lens).astype(np.int32)))

        def step():
            if self.budget:  # the new entry's position, in every layer and head
                self.positions[:, slots.long(), :, index.long()] = pos[:, None, None]
            eng.run_layers(B, eng.dec, serve=serve)
            if rc is not None:
                # the token fed in is the last of the history (the last prompt token at first)
                rc.history.scatter_(1, (pos - 1).long()[:, None], eng.dec.tok_in[:B, None])
                rc.hist_len.copy_(pos)
            eng.run_head(B, temperature, rc)

        eng.dec.tok_in[:B].copy_(torch.as_tensor(np.array([p[-1] for p in prompt_ids], np.int32)))
        graph = None
        gen: List[List[int]] = [[] for _ in range(B)]
        active = np.ones(B, bool)
        for s in range(max_tokens):
            state = np.stack([self.plen + lens + s, own, own + 1]).astype(np.int32)
            up = torch.as_tensor(state).pin_memory().to(dev, non_blocking=True)
            pos.copy_(up[0])
            index.copy_(up[1])
            n_own.copy_(up[2])
            if controls is not None and controls.allowed is not None:
                rc.set_masks(controls.allowed(s, gen), active)
            if temperature > 0:  # one uniform per active row, in row order
                u = np.full(B, 0.5, np.float32)
                u[active] = np.random.random_sample(int(active.sum()))
                eng.dec.uniforms[:B].copy_(torch.as_tensor(u))
            if self.llm.use_graphs and s > 0:  # the first step runs eagerly and sets kernel attributes
                if graph is None:
                    torch.cuda.synchronize(dev)
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        step()
                graph.replay()
            else:
                step()
            own = own + 1
            if self.budget and int(own.max()) >= self.budget + self.every:
                own = self._evict(own)
            eng.dec.tok_in[:B].copy_(eng.dec.tok_out[:B])
            nxt = eng.dec.tok_out[:B].cpu().numpy()
            for b in np.nonzero(active)[0]:
                gen[b].append(int(nxt[b]))
                if not ignore_eos and nxt[b] == EOS_ID:
                    active[b] = False
            if not active.any():
                break
        torch.cuda.synchronize(dev)
        flags = _lib.C.c_uint32(0)
        call("orch_device_check", _lib.C.byref(flags), _stream())
        if flags.value:
            raise RuntimeError(("the controls left a row no token (device check bit 32)" if flags.value == 32 else
                                f"a kernel rejected its input (device check bits {flags.value})"))
        return gen
