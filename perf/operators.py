"""Cases and plain forms of the serving operators around one decode step.

* ``prefix``: attention of a batch of rows whose sequences share a long prefix that is held
  once, beside each row's own cache entries; optionally the weight that every own entry
  received is added to a running mass (``orch_attention_prefix``).
* ``evict``: cache entries dropped by accumulated mass, the newest protected, survivors moved
  into the holes (``orch_cache_evict``).
* ``logits``: repetition, presence and frequency penalties over the token history, sparse
  biases and a grammar bit mask on a batch of logits rows (``orch_logits_process``).

``own`` chooses between the plain form (elementary torch operations in 32 bits) and the
library's entry points.
"""

import math

import torch

own = False

NEG = float("-inf")


# ---------------------------------------------------------------------------------- cases
def listed():
    return [
        # the tiny checkpoint's layer: two sequences behind a short system prompt, launch cost only
        dict(name="prefix_tiny", op="prefix", groups=1, rows=2, heads=2, kv_heads=2, hd=32, prefix=24, own_lo=1,
             own_hi=8, cap=64, track=False),
        # one user's question sampled sixteen times over a 1,000-token instruction
        dict(name="prefix_b16", op="prefix", groups=1, rows=16, heads=32, kv_heads=32, hd=128, prefix=1000, own_lo=1,
             own_hi=128, cap=640, track=False),
        # the benchmark's batch of 64 behind a long document, own parts up to the benchmark's 640 positions
        dict(name="prefix_b64", op="prefix", groups=1, rows=64, heads=32, kv_heads=32, hd=128, prefix=4096, own_lo=1,
             own_hi=577, cap=640, track=False),
        # two tenants with a long document each, grouped key/value heads
        dict(name="prefix_gqa_b128", op="prefix", groups=2, rows=64, heads=32, kv_heads=8, hd=128, prefix=16384,
             own_lo=0, own_hi=512, cap=640, track=False),
        # one sequence at the benchmark's mean position, its entries' weights tracked
        dict(name="tracked_b1", op="prefix", groups=1, rows=1, heads=32, kv_heads=32, hd=128, prefix=0, own_lo=577,
             own_hi=577, cap=640, track=True),
        # a ragged batch behind a system prompt, weights tracked for a bounded cache
        dict(name="tracked_b32", op="prefix", groups=1, rows=32, heads=32, kv_heads=8, hd=128, prefix=512, own_lo=1,
             own_hi=2048, cap=2048, track=True),
        # a bounded cache in its steady state: every step one entry has to go
        dict(name="evict_step_b8", op="evict", rows=8, kv_heads=32, hd=128, budget=512, recent=128, len_lo=513,
             len_hi=513, cap=640),
        # a ragged batch after prompts of different lengths: some rows fit, others lose a third
        dict(name="evict_b32", op="evict", rows=32, kv_heads=8, hd=128, budget=1024, recent=256, len_lo=1, len_hi=1537,
             cap=2048),
        # long prompts cut to a quarter in one go
        dict(name="evict_long_b4", op="evict", rows=4, kv_heads=32, hd=128, budget=4096, recent=1024, len_lo=12001,
             len_hi=16384, cap=16384),
        # one sequence, the checkpoint's vocabulary, penalties only
        dict(name="logits_b1", op="logits", rows=1, vocab=32000, hist=577, bias=0, masks=0, f16=False),
        # the benchmark's batch with penalties, biases and a grammar for half the rows
        dict(name="logits_b64", op="logits", rows=64, vocab=32000, hist=640, bias=300, masks=8, f16=False),
        # a wide vocabulary with long histories
        dict(name="logits_wide_b128", op="logits", rows=128, vocab=131072, hist=4095, bias=64, masks=16, f16=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("prefix", "prefix", "tracked", "evict", "logits"))
    if op in ("prefix", "tracked"):
        hd = rng.choice((32, 64, 128, 128))
        kv = rng.choice((1, 2, 4, 8, 8, 32))
        heads = kv * (1 if kv == 32 else rng.choice((1, 2, 4, 7, 8)) if kv < 8 else rng.choice((1, 2, 4)))
        groups, rows = rng.choice((1, 1, 2, 3)), _log(rng, 1, 64)
        if op == "prefix":
            prefix, hi = _log(rng, 16, 16384), _log(rng, 1, 640)
        else:
            groups, prefix, hi = 1, rng.choice((0, 0, _log(rng, 16, 2048))), _log(rng, 2, 4096)
            rows = min(rows, 32)
        while groups * rows * kv * hi > 32 * 8 * 2048:
            hi = max(1, hi // 2)
        while groups * prefix * max(kv * 128, rows * heads) > 2 * 16384 * 64 * 32:
            prefix = max(16, prefix // 2)
        lo = rng.choice((1, max(1, hi // 2), hi)) if prefix == 0 or rng.random() < 0.5 else 0
        return dict(op="prefix", groups=groups, rows=rows, heads=heads, kv_heads=kv, hd=hd, prefix=prefix, own_lo=lo,
                    own_hi=hi, cap=hi + rng.randrange(0, 64), track=op == "tracked")
    if op == "evict":
        hi = _log(rng, 2, 16384)
        budget = max(1, int(hi * rng.uniform(0.2, 1.0)))
        kv = rng.choice((1, 2, 8, 32))
        rows = max(1, min(_log(rng, 1, 64), 4 * 32 * 16384 // (kv * hi)))
        return dict(op="evict", rows=rows, kv_heads=kv, hd=rng.choice((32, 64, 128)), budget=budget,
                    recent=int(budget * rng.uniform(0.0, 0.5)), len_lo=rng.choice((1, max(1, hi // 2), hi)), len_hi=hi,
                    cap=hi + rng.randrange(0, 64))
    return dict(op="logits", rows=_log(rng, 1, 128), vocab=_log(rng, 1000, 131072), hist=_log(rng, 1, 4095),
                bias=rng.choice((0, 1, 64, 300)), masks=rng.choice((0, 1, 16)), f16=rng.random() < 0.3)


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, in an order that is not sorted."""
    k = next(s for s in (7, 5, 3, 11, 1) if n % s or s == 1)
    return [lo + ((hi - lo) * ((i * k) % n)) // max(1, n - 1) for i in range(n)]


# ------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape, dtype=torch.float16):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    return dict(prefix=_prepare_prefix, evict=_prepare_evict, logits=_prepare_logits)[case["op"]](case, g)


def _prepare_prefix(c, g):
    M, kv, hd, cap = c["groups"] * c["rows"], c["kv_heads"], c["hd"], c["cap"]
    P = max(1, c["prefix"])
    lens = _spread(M, c["own_lo"], c["own_hi"])
    # group i has the whole prefix less a few tokens; its rows are cut into units of at most 64
    plen = [c["prefix"] - (c["prefix"] // 37) * i for i in range(c["groups"])]
    units = [(i * c["rows"] + r, min(64, c["rows"] - r), i, plen[i])
             for i in range(c["groups"]) for r in range(0, c["rows"], 64)] if c["prefix"] else []
    return dict(
        c=c, q=_randn(g, M, c["heads"], hd) * 1.5, kp=_randn(g, c["groups"], kv, P, hd),
        vp=_randn(g, c["groups"], kv, P, hd), kc=_randn(g, M, kv, cap, hd), vc=_randn(g, M, kv, cap, hd),
        lens=_i32(lens), slots=torch.randperm(M, generator=g, device="cuda").to(torch.int32), units=_i32(units),
        num_units=len(units), plen=_i32(plen), out=torch.empty((M, c["heads"], hd), dtype=torch.float16, device="cuda"),
        mass=torch.rand((M, kv, cap), generator=g, device="cuda") if c["track"] else None)


def _prepare_evict(c, g):
    M, kv, hd, cap, n = c["rows"], c["kv_heads"], c["hd"], c["cap"], c["budget"]
    lens = _i32(_spread(M, c["len_lo"], c["len_hi"]))
    # entries past the budget were appended since the last eviction and are the newest; the
    # ones before lie in the order that earlier evictions left them in
    e = torch.arange(cap, device="cuda")
    key = torch.where(e < n, torch.rand((M, kv, cap), generator=g, device="cuda"), 2.0)
    positions = torch.argsort(torch.argsort(key, dim=-1, stable=True), dim=-1).to(torch.int32)
    # a few entries hold most of the weight; some have none at all, so that there are ties
    mass = torch.exp(2.0 * _randn(g, M, kv, cap, dtype=torch.float32))
    mass = torch.where(torch.rand((M, kv, cap), generator=g, device="cuda") < 0.1, 0.0, mass)
    return dict(c=c, kc=_randn(g, M, kv, cap, hd), vc=_randn(g, M, kv, cap, hd), mass=mass, positions=positions,
                lens=lens, slots=torch.randperm(M, generator=g, device="cuda").to(torch.int32),
                mass_out=torch.zeros_like(mass), positions_out=torch.zeros_like(positions),
                lens_out=torch.zeros_like(lens))


def _prepare_logits(c, g):
    M, V, H = c["rows"], c["vocab"], c["hist"]
    lens = _i32(_spread(M, max(1, H // 2), H))
    # tokens repeat as text does: a few frequent ids, a long tail
    u = torch.rand((M, H), generator=g, device="cuda")
    history = (V * u ** 4).to(torch.int32).clamp_(max=V - 1)
    nb, words = c["bias"], (V + 31) // 32
    ids = torch.argsort(torch.rand((M, min(V, 4096)), generator=g, device="cuda"), dim=-1)[:, :nb] * (V // min(V, 4096))
    masks = torch.randint(-2 ** 31, 2 ** 31, (c["masks"], words), generator=g, device="cuda").to(torch.int32)
    if c["masks"] > 1:  # one grammar state allows almost nothing
        masks[1] = 0
        masks[1, words // 2] = 5
    rows = torch.arange(M, device="cuda")
    dt = torch.float16 if c["f16"] else torch.float32
    pen = torch.stack([1.0 + 0.3 * torch.rand(M, generator=g, device="cuda"),
                       0.5 * torch.rand(M, generator=g, device="cuda"),
                       0.2 * torch.rand(M, generator=g, device="cuda")], dim=1).contiguous()
    return dict(c=c, logits=(3.0 * _randn(g, M, V, dtype=torch.float32)).to(dt), out=torch.empty((M, V), dtype=dt, device="cuda"),
                history=history, hist_len=lens, gen_start=lens // 2, penalties=pen,
                bias_ids=ids.reshape(-1).to(torch.int32).contiguous(),
                bias_vals=4.0 * _randn(g, M * nb, dtype=torch.float32), bias_off=(rows.new_ones(M + 1).cumsum(0) - 1).mul(nb).to(torch.int32),
                masks=masks, mask_rows=torch.where(rows % 2 == 0, rows // 2 % max(1, c["masks"]), -1).to(torch.int32)
                if c["masks"] else None)


# ---------------------------------------------------------------------------------- plain forms
def run(s):
    op = s["c"]["op"]
    if own:
        return dict(prefix=_own_prefix, evict=_own_evict, logits=_own_logits)[op](s)
    return dict(prefix=_plain_prefix, evict=_plain_evict, logits=_plain_logits)[op](s)


def _plain_prefix(s):
    c = s["c"]
    groups, rows, heads, kv, hd, P = c["groups"], c["rows"], c["heads"], c["kv_heads"], c["hd"], c["prefix"]
    M, G, L = groups * rows, heads // kv, c["own_hi"]
    slots, lens = s["slots"].long(), s["lens"].long()
    q = s["q"].float() / math.sqrt(hd)
    scores = []
    if P:
        # the rows of a group against its prefix: [group, kv head, rows x G, hd] . [.., hd, P]
        qg = q.view(groups, rows, kv, G, hd).permute(0, 2, 1, 3, 4).reshape(groups, kv, rows * G, hd)
        sp = torch.matmul(qg, s["kp"][:, :, :P].float().transpose(-1, -2))
        sp = torch.where(torch.arange(P, device="cuda") < s["plen"].long()[:, None, None, None], sp, NEG)
        scores.append(sp.view(groups, kv, rows, G, P).permute(0, 2, 1, 3, 4).reshape(M, kv, G, P))
    k = s["kc"][slots, :, :L].float()
    so = torch.matmul(q.view(M, kv, G, hd), k.transpose(-1, -2))
    live = torch.arange(L, device="cuda") < lens[:, None, None, None]
    scores.append(torch.where(live, so, NEG))
    x = torch.cat(scores, dim=-1)
    e = torch.exp(x - x.amax(dim=-1, keepdim=True))
    p = e / e.sum(dim=-1, keepdim=True)
    po = p[..., P:]
    out = torch.matmul(po, s["vc"][slots, :, :L].float())
    if P:
        pg = p[..., :P].view(groups, rows, kv, G, P).permute(0, 2, 1, 3, 4).reshape(groups, kv, rows * G, P)
        og = torch.matmul(pg, s["vp"][:, :, :P].float())
        out = out + og.view(groups, kv, rows, G, hd).permute(0, 2, 1, 3, 4).reshape(M, kv, G, hd)
    s["out"].copy_(out.reshape(M, heads, hd))
    if not c["track"]:
        return {"out": s["out"]}
    w = po.sum(dim=2)  # over the query heads of a key/value head
    at = torch.arange(L, device="cuda")[None, None, :]
    n = lens[:, None, None]
    old = s["mass"][slots, :, :L]
    s["mass"][slots, :, :L] = torch.where(at < n - 1, old + w, torch.where(at == n - 1, w, old))
    return {"out": s["out"], "mass": s["mass"]}


def _plain_evict(s):
    c = s["c"]
    cap, budget, recent, hd = c["cap"], c["budget"], c["recent"], c["hd"]
    slots, lens = s["slots"].long(), s["lens"].long()
    mass, pos = s["mass"][slots], s["positions"][slots].long()
    at = torch.arange(cap, device="cuda")[None, None, :]
    valid = at < lens[:, None, None]
    n = lens.clamp(max=budget)
    newest = torch.where(valid, pos, -1).amax(dim=-1, keepdim=True)
    first = torch.where(valid, (pos > newest - recent).long(), -1)  # protected, others, nothing
    by_mass = torch.argsort(mass, dim=-1, descending=True, stable=True)
    order = torch.gather(by_mass, -1, torch.argsort(torch.gather(first, -1, by_mass), dim=-1, descending=True, stable=True))
    rank = torch.argsort(order, dim=-1)
    keep = rank < n[:, None, None]
    hole, tail = ~keep & (at < n[:, None, None]), keep & (at >= n[:, None, None])
    tails = torch.argsort(torch.where(tail, at, cap + at), dim=-1)  # the kept entries past n, in order
    src = torch.where(hole, torch.gather(tails, -1, (hole.long().cumsum(-1) - 1).clamp(min=0)), at)[..., :budget]
    live = (at < n[:, None, None])[..., :budget]
    at_rows = src[..., None].expand(-1, -1, -1, hd)
    k, v = s["kc"][slots], s["vc"][slots]
    b = min(budget, cap)
    s["kc"][slots, :, :b] = torch.where(live[..., None], torch.gather(k, 2, at_rows), k[:, :, :b])
    s["vc"][slots, :, :b] = torch.where(live[..., None], torch.gather(v, 2, at_rows), v[:, :, :b])
    s["mass_out"][slots, :, :b] = torch.where(live, torch.gather(mass, -1, src), s["mass_out"][slots, :, :b])
    s["positions_out"][slots, :, :b] = torch.where(live, torch.gather(pos, -1, src).to(torch.int32), s["positions_out"][slots, :, :b])
    s["lens_out"].copy_(n)
    return {"k": s["kc"], "v": s["vc"], "mass": s["mass_out"], "positions": s["positions_out"], "lens": s["lens_out"]}


def _plain_logits(s):
    c = s["c"]
    M, V, H, nb = c["rows"], c["vocab"], c["hist"], c["bias"]
    x = s["logits"].float()
    ids = s["history"].long()
    at = torch.arange(H, device="cuda")[None, :]
    live = (at < s["hist_len"][:, None]).float()
    made = live * (at >= s["gen_start"][:, None]).float()
    zeros = torch.zeros((M, V), dtype=torch.float32, device="cuda")
    seen = zeros.scatter_add(1, ids, live) > 0
    count = zeros.scatter_add(1, ids, made)
    rep, pres, freq = s["penalties"][:, 0:1], s["penalties"][:, 1:2], s["penalties"][:, 2:3]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (count * freq + (count > 0).float() * pres)
    if nb:
        x = x + zeros.scatter(1, s["bias_ids"].long().view(M, nb), s["bias_vals"].view(M, nb))
    if c["masks"]:
        rows = s["mask_rows"].long()
        bits = (s["masks"][rows.clamp(min=0)][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        allowed = (bits.reshape(M, -1)[:, :V] != 0) | (rows < 0)[:, None]
        x = torch.where(allowed, x, NEG)
    s["out"].copy_(x)
    return {"out": s["out"]}


# -------------------------------------------------------------------------- the library's calls
def _own_prefix(s):
    from orchard_b200 import _lib
    c, M = s["c"], s["q"].shape[0]
    heads, kv, hd = c["heads"], c["kv_heads"], c["hd"]
    if "ws" not in s:  # kept by the program, as the engine keeps its attention workspace
        n = _lib.lib().orch_attention_prefix_workspace_bytes(M, heads, kv, hd, s["num_units"], c["prefix"], c["own_hi"],
                                                             int(c["track"]))
        s["ws"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    _lib.call("orch_attention_prefix", s["q"], s["kp"], s["vp"], s["units"], s["num_units"], c["prefix"], s["kp"].shape[2],
              s["kp"].shape[0], s["kc"], s["vc"], s["lens"], s["slots"], c["own_hi"], c["cap"], s["kc"].shape[0],
              s["mass"], s["out"], M, heads, kv, hd, s["ws"], s["ws"].numel(), torch.cuda.current_stream().cuda_stream)
    return {"out": s["out"], "mass": s["mass"]} if c["track"] else {"out": s["out"]}


def _own_evict(s):
    from orchard_b200 import _lib
    c = s["c"]
    _lib.call("orch_cache_evict", s["kc"], s["vc"], s["mass"], s["positions"], s["lens"], s["slots"], s["mass_out"],
              s["positions_out"], s["lens_out"], c["rows"], c["kv_heads"], c["hd"], c["cap"], s["kc"].shape[0],
              c["budget"], c["recent"], torch.cuda.current_stream().cuda_stream)
    return {"k": s["kc"], "v": s["vc"], "mass": s["mass_out"], "positions": s["positions_out"], "lens": s["lens_out"]}


def _own_logits(s):
    from orchard_b200 import _lib
    c = s["c"]
    V, nb, nm = c["vocab"], c["bias"], c["masks"]
    _lib.call("orch_logits_process", s["logits"], s["out"], _lib.F16 if c["f16"] else _lib.F32, c["rows"], V, V, 0,
              s["history"], c["hist"], s["hist_len"], s["gen_start"], s["penalties"],
              s["bias_ids"] if nb else None, s["bias_vals"] if nb else None, s["bias_off"] if nb else None, c["rows"] * nb,
              s["masks"] if nm else None, (V + 31) // 32, nm, s["mask_rows"], torch.cuda.current_stream().cuda_stream)
    return {"out": s["out"]}


# ------------------------------------------------------------------------------------- floors
def work(case):
    c = case
    if c["op"] == "prefix":
        M, kv, hd = c["groups"] * c["rows"], c["kv_heads"], c["hd"]
        lens = _spread(M, c["own_lo"], c["own_hi"])
        plen = [c["prefix"] - (c["prefix"] // 37) * i for i in range(c["groups"])]
        entries = sum(plen) + sum(lens)
        pairs = c["rows"] * sum(plen) + sum(lens)
        return {"bytes": 4 * hd * kv * entries + 4 * M * c["heads"] * hd + (8 * kv * sum(lens) if c["track"] else 0),
                "flops": 4 * hd * c["heads"] * pairs}
    if c["op"] == "evict":
        kv, hd, n, r = c["kv_heads"], c["hd"], c["budget"], c["recent"]
        total = 0.0
        for L in _spread(c["rows"], c["len_lo"], c["len_hi"]):
            kept = min(L, n)
            total += 8 * L + 8 * kept
            if L > n:  # the protected entries past the budget have to move, and the others' share that stays
                guard = min(r, L - n)
                moved = guard + (L - n - guard) * (n - min(r, n)) / max(1, L - r)
                total += 8 * hd * moved
        return {"bytes": kv * total, "flops": 0}
    size = 2 if c["f16"] else 4
    hist = sum(_spread(c["rows"], max(1, c["hist"] // 2), c["hist"]))
    return {"bytes": 2 * size * c["rows"] * c["vocab"] + 4 * hist + 8 * c["bias"] * c["rows"] + c["masks"] * c["vocab"] // 8,
            "flops": 0}


# ---------------------------------------------------------------------------- from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    return dict(prefix=_exact_prefix, evict=_exact_evict, logits=_exact_logits)[case["op"]](s)


def _exact_prefix(s):
    c = s["c"]
    heads, kv, hd = c["heads"], c["kv_heads"], c["hd"]
    G, lens, slots, plen = heads // kv, s["lens"].tolist(), s["slots"].tolist(), s["plen"].tolist()
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    mass = s["mass"].double() if c["track"] else None
    for m in range(len(lens)):
        n, t, i = lens[m], slots[m], m // c["rows"]
        k = torch.cat([s["kp"][i, :, :plen[i]], s["kc"][t, :, :n]], dim=1).double() if c["prefix"] else s["kc"][t, :, :n].double()
        v = torch.cat([s["vp"][i, :, :plen[i]], s["vc"][t, :, :n]], dim=1).double() if c["prefix"] else s["vc"][t, :, :n].double()
        p = torch.softmax(torch.einsum("kgd,kjd->kgj", s["q"][m].double().view(kv, G, hd), k) * hd ** -0.5, dim=-1)
        out[m] = torch.einsum("kgj,kjd->kgd", p, v).reshape(heads, hd)
        if c["track"] and n:
            w = p.sum(dim=1)[:, p.shape[2] - n:]
            mass[t, :, :n - 1] += w[:, :-1]
            mass[t, :, n - 1] = w[:, -1]
    return {"out": out, "mass": mass} if c["track"] else {"out": out}


def _exact_evict(s):
    """One (row, head) pair at a time, sorted on the host."""
    import numpy as np
    c = s["c"]
    if c["rows"] * c["kv_heads"] * c["len_hi"] > 3_000_000:
        return None
    lens, slots = s["lens"].tolist(), s["slots"].tolist()
    mass, pos = s["mass"].double().cpu().numpy(), s["positions"].cpu().numpy()
    mo, po = np.zeros_like(mass), np.zeros_like(pos)
    k, v = s["kc"].double(), s["vc"].double()
    for m, (L, t) in enumerate(zip(lens, slots)):
        n = min(L, c["budget"])
        for h in range(c["kv_heads"]):
            a, p = mass[t, h, :L], pos[t, h, :L]
            guard = p > p.max() - c["recent"]
            kept = np.zeros(L, bool)
            kept[np.lexsort((np.arange(L), -a, ~guard))[:n]] = True
            src = np.arange(n)
            src[~kept[:n]] = np.flatnonzero(kept[n:]) + n
            mo[t, h, :n], po[t, h, :n] = a[src], p[src]
            move = torch.from_numpy(src).to("cuda")
            k[t, h, :n], v[t, h, :n] = k[t, h, move], v[t, h, move]
    return {"k": k, "v": v, "mass": torch.from_numpy(mo), "positions": torch.from_numpy(po),
            "lens": s["lens"].clamp(max=c["budget"])}


def _exact_logits(s):
    import numpy as np
    c = s["c"]
    x = s["logits"].double().cpu().numpy()
    hist, lens, start = s["history"].cpu().numpy(), s["hist_len"].tolist(), s["gen_start"].tolist()
    pen = s["penalties"].double().cpu().numpy()
    ids, vals = s["bias_ids"].cpu().numpy(), s["bias_vals"].double().cpu().numpy()
    if c["masks"]:
        allow = np.unpackbits(s["masks"].cpu().numpy().astype("<i4").view(np.uint8), axis=1, bitorder="little")[:, :c["vocab"]]
        which = s["mask_rows"].tolist()
    for m in range(c["rows"]):
        row = x[m]
        seen = np.unique(hist[m, :lens[m]])
        row[seen] = np.where(row[seen] > 0, row[seen] / pen[m, 0], row[seen] * pen[m, 0])
        made, times = np.unique(hist[m, start[m]:lens[m]], return_counts=True)
        row[made] -= pen[m, 2] * times + pen[m, 1]
        row[ids[m * c["bias"]:(m + 1) * c["bias"]]] += vals[m * c["bias"]:(m + 1) * c["bias"]]
        if c["masks"] and which[m] >= 0:
            row[allow[which[m]] == 0] = -np.inf
    return {"out": torch.from_numpy(x)}
