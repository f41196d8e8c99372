"""The operators of a speculative, bounded-cache decode over the int8 KV cache, as cases that can be timed:

* ``tree``: attention of a tree of drafted tokens over a cache (``kernels.attend_tree``);
* ``mass``: an attention job that also adds up the weight each slot received (``kernels.attend_mass``);
* ``select``: which slots a bounded cache keeps, by that weight (``kernels.kv_select``);
* ``move``: cache slots moved together, an accepted path or the kept slots (``kernels.kv_move``).

Attention here is the library's: the query of each head in 8 bits (amax / 127
steps, float32 arithmetic), scores and softmax in float, the weights times the
V scales in 16 bits below the row's largest.  Both quantisations belong to the
operators' definition, so the plain forms and the 64-bit ones make them too.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda"


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one drafted token of one sequence in a sliding-window layer: launch- and latency-bound
        {"name": "tree_one_token", "kind": "tree", "seqs": 1, "nodes": 1, "ctx": 117, "window": 512, "ring": True,
         "nh": 8, "kvh": 1, "hd": 256},
        # small trees over short ragged contexts, two kv heads
        {"name": "tree_small_gqa", "kind": "tree", "seqs": 3, "nodes": 7, "ctx": 1203, "window": 0, "ring": False,
         "nh": 8, "kvh": 2, "hd": 128},
        # a sliding-window layer's part of verifying four trees, ring caches that have wrapped
        {"name": "tree_sliding", "kind": "tree", "seqs": 4, "nodes": 26, "ctx": 20001, "window": 512, "ring": True,
         "nh": 8, "kvh": 1, "hd": 256},
        # batched verification over long contexts, a full-attention layer
        {"name": "tree_full_batch", "kind": "tree", "seqs": 8, "nodes": 16, "ctx": 8192, "window": 0, "ring": False,
         "nh": 8, "kvh": 1, "hd": 512},
        # the widest tree over one very long context
        {"name": "tree_full_long", "kind": "tree", "seqs": 1, "nodes": 64, "ctx": 24001, "window": 0, "ring": False,
         "nh": 8, "kvh": 1, "hd": 512},
        # one decode row that keeps its slots' weights, a short context
        {"name": "mass_decode_short", "kind": "mass", "seqs": 1, "rows": 1, "ctx": 301, "nh": 8, "kvh": 1, "hd": 256},
        # batched decode over long contexts, a full-attention layer
        {"name": "mass_decode_full", "kind": "mass", "seqs": 8, "rows": 1, "ctx": 8192, "nh": 8, "kvh": 1, "hd": 512},
        # the last rows of a long prompt, whose weights choose what the cache keeps
        {"name": "mass_prompt_tail", "kind": "mass", "seqs": 1, "rows": 64, "ctx": 16000, "nh": 8, "kvh": 2, "hd": 256},
        # a cache that has grown some slots past its budget
        {"name": "select_short", "kind": "select", "seqs": 1, "ctx": 1100, "budget": 512, "sink": 4, "recent": 64},
        # long prompts cut to a budget, a whole batch
        {"name": "select_batch", "kind": "select", "seqs": 16, "ctx": 32000, "budget": 4096, "sink": 4,
         "recent": 256},
        # the accepted paths of a verified batch: a few slots of many caches, wrapped rings
        {"name": "move_paths", "kind": "move", "seqs": 16, "ctx": 543, "ring": True, "window": 0, "count": 26,
         "row": 512, "mass": False},
        # caches cut to the slots that were selected, their weights with them
        {"name": "move_evicted", "kind": "move", "seqs": 8, "ctx": 8192, "ring": False, "window": 0, "count": 2048,
         "row": 512, "mass": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kvh, hd = rng.choice([(1, 256), (1, 512), (2, 256), (4, 128), (1, 64), (2, 192), (1, 320)])
    return {"nh": kvh * rng.choice([1, 2, 4, 8, 8, 12, 16]) if kvh < 4 else 8, "kvh": kvh, "hd": hd}


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "mass", "mass", "select", "move"])
    if kind == "tree":
        window = rng.choice([0, 0, rng.randint(48, 1024)])
        c = {"kind": kind, "seqs": rng.randint(1, 8), "nodes": _log(rng, 1, 64), "ctx": _log(rng, 1, 9000),
             "window": window, "ring": window > 0, **_heads(rng)}
        while c["seqs"] > 1 and c["seqs"] * c["nodes"] * c["ctx"] * c["nh"] > 8 << 20:
            c["seqs"] //= 2
        return c
    if kind == "mass":
        rows = rng.choice([1, 1, 1, _log(rng, 2, 64)])
        return {"kind": kind, "seqs": rng.randint(1, 8) if rows == 1 else 1, "rows": rows,
                "ctx": max(rows, _log(rng, 8, 9000)), **_heads(rng)}
    if kind == "select":
        n = _log(rng, 16, 32000)
        budget = _log(rng, 8, n)
        sink = rng.randint(0, min(8, budget // 2))
        return {"kind": kind, "seqs": rng.randint(1, 16), "ctx": n, "budget": budget, "sink": sink,
                "recent": rng.randint(0, (budget - sink) // 2)}
    ring = rng.random() < 0.5
    ctx = _log(rng, 64, 1200 if ring else 8192)
    return {"kind": "move", "seqs": rng.randint(1, 16 if ring else 8), "ctx": ctx, "ring": ring, "window": 0,
            "count": _log(rng, 1, min(64, ctx // 2)) if ring else _log(rng, 1, ctx // 2 + 1),
            "row": 64 * rng.randint(1, 16), "mass": not ring}


# ------------------------------------------------------------------ inputs
class _Gen:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed & 0x7FFFFFFF)
        self.r = np.random.RandomState(seed & 0x7FFFFFFF)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device=DEV)

    def uniform(self, lo, hi, *shape):
        return torch.rand(*shape, generator=self.g, device=DEV) * (hi - lo) + lo


def _cache(g, seqs, slots, row):
    """Filled int8 caches of `seqs` sequences: K [seq][slot][row], V
    [seq][slot / 4][row][4], a scale per slot.  Rows of unit normals have their
    largest entry near 3.5, so steps of about 3.5 / 127."""
    q = lambda *s: (g.normal(*s) * 36).round_().clamp_(-127, 127).to(torch.int8)  # noqa: E731
    quads = (slots + 3) // 4
    return {"kc": q(seqs, slots, row), "vt": q(seqs, quads, row, 4), "ks": g.uniform(0.02, 0.04, seqs, slots),
            "vs": g.uniform(0.02, 0.04, seqs, slots)}


def _lens(g, ctx, seqs):
    """Ragged lengths, the longest of ctx."""
    return [ctx] + [max(1, int(ctx * f)) for f in g.r.uniform(0.75, 1.0, seqs - 1)]


def _trees(g, seqs, nodes):
    """Masks of random drafted trees: a node's parent is one of the few before
    it, so that paths are some nodes long and siblings frequent."""
    m = np.zeros((seqs, nodes), np.uint64)
    for s in range(seqs):
        for i in range(nodes):
            parent = i - 1 - int(g.r.geometric(0.4) - 1)
            m[s, i] = (m[s, parent] if parent >= 0 else np.uint64(0)) | np.uint64(1 << i)
    return torch.from_numpy(m.view(np.int64)).to(DEV)


def _path(g, nodes, count):
    """Ascending choices out of `nodes`, `count` of them."""
    return np.sort(g.r.choice(nodes, count, replace=False)).astype(np.int32)


# ----------------------------------------------------------------- prepare
def prepare(case, seed):
    c, g = case, _Gen(seed)
    st = {"case": c}
    s = c["seqs"]
    if c["kind"] == "select":
        # a few slots with most of the weight, many with nearly none
        st["mass"] = torch.exp(3.0 * g.normal(s, c["ctx"]))
        st["lens"] = _lens(g, c["ctx"], s)
        st["n"] = torch.tensor(st["lens"], device=DEV)
        st["keep"] = torch.empty(s, c["budget"], dtype=torch.int32, device=DEV)
        st["seqs"] = [(st["keep"][i], st["mass"][i], n) for i, n in enumerate(st["lens"])]
        return st
    if c["kind"] == "move":
        slots = c["ctx"]
        st["cache"] = _cache(g, s, slots, c["row"])
        if c["mass"]:
            st["cache"]["mass"] = torch.exp(3.0 * g.normal(s, slots))
        # rings: the accepted nodes of a tree drafted at a position past the wrap; else the kept slots of a full cache
        st["pos"] = [5 * slots + int(p) for p in g.r.randint(0, slots, s)] if c["ring"] else [0] * s
        span = min(64, slots) if c["ring"] else slots
        idx = np.full((s, c["count"]), -1, np.int32)
        for i in range(s):
            n = min(c["count"], span) if i == 0 else g.r.randint(1, min(c["count"], span) + 1)
            idx[i, :n] = _path(g, span, n)
        st["index"], st["first"] = torch.from_numpy(idx).to(DEV), torch.tensor(st["pos"], device=DEV)
        ca = st["cache"]
        st["moves"] = [{
            "src": (ca["kc"][i], ca["ks"][i], ca["vt"][i], ca["vs"][i], ca["mass"][i] if c["mass"] else None),
            "cap": slots, "ring": slots if c["ring"] else 0, "pos": st["pos"][i], "index": st["index"][i]}
            for i in range(s)]
        return st
    rows = c["nodes"] if c["kind"] == "tree" else c["rows"]
    nh, kvh, hd = c["nh"], c["kvh"], c["hd"]
    lens = _lens(g, c["ctx"], s)
    ring = c["kind"] == "tree" and c["ring"]
    slots = -(-(c["window"] + rows) // 8) * 8 if ring else c["ctx"] + (rows if c["kind"] == "tree" else 0)
    st["cache"] = ca = _cache(g, s, slots, kvh * hd)
    # rms-normalised heads: scores of a few units, as after the query norm
    st["q"] = g.normal(s, rows, nh, hd) * (3.0 / math.sqrt(hd))
    st["out"] = torch.empty(s, rows, nh, hd, device=DEV)
    if c["kind"] == "tree":
        st["pos"], st["mask"] = lens, _trees(g, s, rows)
    else:
        st["pos"] = [max(n - rows, 0) for n in lens]
        # what the rows before these have given each slot, a few rows' worth in all
        st["mass"] = torch.exp(1.5 * g.normal(s, slots)) * (nh / c["ctx"])
    st["first"] = torch.tensor(st["pos"], device=DEV)
    per = [(ca["kc"][i], ca["ks"][i], ca["vt"][i], ca["vs"][i], slots, slots if ring else 0, st["pos"][i])
           for i in range(s)]
    if c["kind"] == "tree":
        st["seqs"] = [p + (st["mask"][i],) for i, p in enumerate(per)]
    else:
        st["seqs"] = [p + (rows, st["mass"][i]) for i, p in enumerate(per)]
    if own:
        from fastgemma_amd import kernels as K
        nb = K.attend_scratch_bytes(s * rows, nh, kvh, hd, slots)
        st["scratch"] = torch.empty(nb + 256, dtype=torch.uint8, device=DEV)
    return st


# ------------------------------------------------------------- plain forms
def _quant_q(q):
    """The 8-bit query: float32 steps, ties to even."""
    amax = q.abs().amax(-1, keepdim=True)
    inv = torch.where(amax > 0, torch.full_like(amax, 127.0) / amax, torch.zeros_like(amax))  # one rounding
    return torch.clamp(torch.round(q * inv), -127, 127), amax / 127.0


def _attention(q, ca, live, kvh):
    """q [s, rows, nh, hd] over caches of `slots` slots, live [s, rows, slots]:
    the outputs, and the softmax weights [s, kvh, rows * grp, slots]."""
    s, rows, nh, hd = q.shape
    grp, slots = nh // kvh, ca["ks"].shape[1]
    q8, qs = _quant_q(q)
    by_kv = lambda x: x.view(s, rows, kvh, grp, -1).transpose(1, 2).reshape(s, kvh, rows * grp, -1)  # noqa: E731
    k = ca["kc"].view(s, slots, kvh, hd).permute(0, 2, 3, 1).float().contiguous()
    w = torch.matmul(by_kv(q8), k)
    w = w * by_kv(qs) * ca["ks"].view(s, 1, 1, slots)
    seen = live.view(s, 1, rows, 1, slots).expand(s, kvh, rows, grp, slots).reshape(s, kvh, rows * grp, slots)
    w = torch.where(seen, w, torch.full_like(w, -math.inf))
    top = w.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(w - top), torch.zeros_like(w))  # a row that sees nothing: zeros
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    w = p * ca["vs"].view(s, 1, 1, slots)
    top = w.amax(-1, keepdim=True)
    iw = torch.floor(w * torch.where(top > 0, 65535.0 / top, torch.zeros_like(top)) + 0.5)
    v = ca["vt"].permute(0, 1, 3, 2).reshape(s, -1, kvh, hd)[:, :slots].permute(0, 2, 1, 3).float().contiguous()
    out = torch.matmul(iw, v) * (top / 65535.0)
    return out.view(s, kvh, rows, grp, hd).transpose(1, 2).reshape(s, rows, nh, hd), p


def _tree_live(first, mask, slots, ring, window):
    """Which slots each node sees: the committed positions below first and its
    visible nodes at first, first + 1, ..., of all those the last `window`."""
    s, n = mask.shape
    at = torch.arange(slots, device=DEV)
    last = (first + n - 1).view(s, 1)
    p = last - torch.remainder(last - at, ring) if ring else at.expand(s, slots)  # position in each slot
    bit = (mask.view(s, n, 1) >> torch.arange(n, device=DEV)) & 1
    start = first.view(s, 1) + bit.sum(-1) - window if window else torch.zeros(s, n, dtype=torch.int64, device=DEV)
    rank = first.view(s, 1, 1) + torch.cumsum(bit, -1) - bit  # a visible node's place in the node's sequence
    node = (p - first.view(s, 1)).clamp(0, n - 1).view(s, 1, slots).expand(s, n, slots)
    drafted = (torch.gather(bit, 2, node) == 1) & (torch.gather(rank, 2, node) >= start.view(s, n, 1))
    pr, fr = p.view(s, 1, slots), first.view(s, 1, 1)
    committed = (pr >= 0) & (pr < fr) & (pr >= start.view(s, n, 1))
    return committed | ((pr >= fr) & (pr < fr + n) & drafted)


def _row_live(first, rows, slots):
    at = torch.arange(slots, device=DEV)
    return at.view(1, 1, slots) <= first.view(-1, 1, 1) + torch.arange(rows, device=DEV).view(1, rows, 1)


def _add_mass(mass, p, first, rows):
    """mass of the slots that were there before the rows, plus what the rows
    gave each slot; slots behind the last row keep what they hold."""
    got = p.sum((1, 2))
    at, f = torch.arange(mass.shape[1], device=DEV), first.view(-1, 1)
    return torch.where(at < f, mass + got, torch.where(at < f + rows, got, mass))


def _select(mass, n, budget, sink, recent):
    """The sink first and recent last of n slots and the heaviest others, in
    order; ties and NaN (as minus infinity) by the lower index."""
    at, n = torch.arange(mass.shape[1], device=DEV), n.view(-1, 1)
    v = torch.where(torch.isnan(mass), torch.full_like(mass, -math.inf), mass)
    rank = torch.where((at < sink) | (at >= n - recent), 2, 1) * (at < n)
    order = torch.argsort(v, dim=1, descending=True, stable=True)
    order = torch.gather(order, 1, torch.argsort(torch.gather(rank, 1, order), dim=1, descending=True, stable=True))
    keep = order[:, :budget]
    big = mass.shape[1]
    keep = torch.sort(torch.where(keep < n, keep, big), 1)[0]
    keep = torch.where(keep < big, keep, -1).to(torch.int32)
    return torch.nn.functional.pad(keep, (0, budget - keep.shape[1]), value=-1)


def _move(ca, index, first, ring):
    """Slot first + index[j] to slot first + j of every cache, in place; a
    negative index moves nothing."""
    s, count = index.shape
    i = torch.arange(s, device=DEV).view(s, 1).expand(s, count)
    f, at = first.view(s, 1), torch.arange(count, device=DEV)
    to = f + at
    frm = torch.where(index >= 0, f + index, to)
    if ring:
        to, frm = torch.remainder(to, ring), torch.remainder(frm, ring)
    for name in [k for k in ("kc", "ks", "vs", "mass") if k in ca]:
        ca[name][i, to] = ca[name][i, frm]
    ca["vt"][i, to // 4, :, to % 4] = ca["vt"][i, frm // 4, :, frm % 4]


# --------------------------------------------------------------------- run
# Lengths and positions change from one decode step to the next, and the library's
# descriptors hold them: a user's program makes those for each call, and so does run.
def run(st):
    c = st["case"]
    if c["kind"] == "select":
        if own:
            from fastgemma_amd import kernels as K
            K.kv_select(st["seqs"], c["budget"], c["sink"], c["recent"])
        else:
            st["keep"] = _select(st["mass"], st["n"], c["budget"], c["sink"], c["recent"])
        return {"keep": st["keep"]}
    ca = st["cache"]
    if c["kind"] == "move":
        if own:
            from fastgemma_amd import kernels as K
            K.kv_move(st["moves"], c["row"])
        else:
            _move(ca, st["index"], st["first"], c["ctx"] if c["ring"] else 0)
        # moved bytes are whole numbers that have to be equal
        return dict(ca)
    nh, kvh, hd = c["nh"], c["kvh"], c["hd"]
    slots = ca["ks"].shape[1]
    if c["kind"] == "tree":
        if own:
            from fastgemma_amd import kernels as K
            K.attend_tree(st["out"], st["q"], st["seqs"], nh, kvh, hd, c["window"], st["scratch"])
        else:
            live = _tree_live(st["first"], st["mask"], slots, slots if c["ring"] else 0, c["window"])
            st["out"] = _attention(st["q"], ca, live, kvh)[0]
        return {"out": st["out"]}
    if own:
        from fastgemma_amd import kernels as K
        K.attend_mass(st["out"], st["q"], st["seqs"], nh, kvh, hd, decay=1.0, scratch=st["scratch"])
    else:
        st["out"], p = _attention(st["q"], ca, _row_live(st["first"], c["rows"], slots), kvh)
        st["mass"] = _add_mass(st["mass"], p, st["first"], c["rows"])
    return {"out": st["out"], "mass": st["mass"]}


# -------------------------------------------------------------------- work
def _some(c, first, most):
    """The mean of the ragged lengths: the first, and others of 0.75 to 1 times it."""
    return (first + (c["seqs"] - 1) * 0.875 * first) / c["seqs"] if most else first


def work(case):
    c = case
    s = c["seqs"]
    if c["kind"] == "select":
        return {"bytes": s * (4 * _some(c, c["ctx"], True) + 4 * c["budget"]), "flops": 0}
    if c["kind"] == "move":
        # half the sequences' shortened lists, each moved slot read and written once
        n = c["count"] * (1 + 0.5 * (s - 1))
        return {"bytes": n * (4 * c["row"] + 16 + (8 if c["mass"] else 0) + 4), "flops": 0}
    rows = c["nodes"] if c["kind"] == "tree" else c["rows"]
    nh, kvh, hd = c["nh"], c["kvh"], c["hd"]
    n = _some(c, c["ctx"], True)
    if c.get("window"):
        n = min(n, c["window"])
    by = s * ((n + rows) * (2 * kvh * hd + 8) + 8 * rows * nh * hd)
    if c["kind"] == "tree":
        return {"bytes": by + 8 * s * rows, "flops": s * rows * nh * 4.0 * (n + min(rows, 8) / 2) * hd}
    return {"bytes": by + 8 * s * n, "flops": s * rows * nh * 4.0 * n * hd}


# ------------------------------------------------------------------- exact
def _x_attention(q, kf, ks, vf, vs, sees, kvh):
    """One sequence in float64: q [rows, nh, hd], kf / vf [slots, kvh * hd],
    sees [rows, slots]; the outputs and each slot's weight."""
    rows, nh, hd = q.shape
    grp = nh // kvh
    out = torch.zeros(rows, nh, hd, dtype=torch.float64, device=DEV)
    got = torch.zeros(ks.shape[0], dtype=torch.float64, device=DEV)
    # the query's 8 bits are float32 arithmetic by definition: the quotient and
    # the product each rounded to float32
    amax = q.abs().amax(-1, keepdim=True)
    step = (127.0 / amax.double()).float().double()
    q8 = torch.round((q.double() * step).float().double()).clamp(-127, 127)
    q8 = torch.where(amax > 0, q8, torch.zeros_like(q8))
    scale = amax.double() / 127
    for h in range(nh):
        g = h // grp
        x = q8[:, h] @ kf[:, g * hd:(g + 1) * hd].t() * scale[:, h] * ks
        x = x.masked_fill(~sees, -math.inf)
        p = torch.softmax(x, 1).nan_to_num(0.0)
        got += p.sum(0)
        w = p * vs
        unit = w.amax(1, keepdim=True) / 65535
        iw = torch.where(unit > 0, torch.floor(w / unit + 0.5), torch.zeros_like(w))
        out[:, h] = iw @ vf[:, g * hd:(g + 1) * hd] * unit
    return out, got


def _x_tree_sees(pos, mask, slots, ring, window):
    """By each node's own list of positions, first to last."""
    n = len(mask)
    sees = np.zeros((n, slots), bool)
    for i, m in enumerate(mask):
        line = np.concatenate([np.arange(max(0, pos - (window or pos)), pos),
                               [pos + j for j in range(n) if (int(m) >> j) & 1]]).astype(np.int64)
        if window:
            line = line[-window:]
        sees[i, line % ring if ring else line] = True
    return torch.from_numpy(sees).to(DEV)


def exact(case, seed):
    c = case
    if c["kind"] == "select":
        return None  # whole numbers
    st = prepare(dict(c), seed)
    ca = st["cache"]
    if c["kind"] == "move":
        index, ring = st["index"].cpu().numpy(), c["ctx"] if c["ring"] else 0
        out = {"kc": None, "vt": None}
        for name in [k for k in ("ks", "vs", "mass") if k in ca]:
            x = ca[name].double().cpu().numpy()
            for i, p in enumerate(st["pos"]):
                take = index[i][index[i] >= 0].astype(np.int64) + p
                put = p + np.arange(len(take))
                x[i, put % ring if ring else put] = x[i, take % ring if ring else take]
            out[name] = torch.from_numpy(x)
        return out
    slots, rows = ca["ks"].shape[1], st["q"].shape[1]
    outs, mass = [], []
    for i, p in enumerate(st["pos"]):
        kf = ca["kc"][i].double()
        vf = ca["vt"][i].transpose(1, 2).reshape(-1, kf.shape[1])[:slots].double()
        if c["kind"] == "tree":
            sees = _x_tree_sees(p, st["mask"][i].cpu().numpy(), slots, slots if c["ring"] else 0, c["window"])
        else:
            sees = torch.from_numpy(np.tri(rows, slots, p, bool)).to(DEV)
        o, got = _x_attention(st["q"][i], kf, ca["ks"][i].double(), vf, ca["vs"][i].double(), sees, c["kvh"])
        outs.append(o)
        if c["kind"] == "mass":
            had = st["mass"][i].double()
            had[p:p + rows] = 0
            mass.append(had + got)
    return {"out": torch.stack(outs)} if c["kind"] == "tree" else {"out": torch.stack(outs), "mass": torch.stack(mass)}
