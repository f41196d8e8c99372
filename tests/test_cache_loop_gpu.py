"""GPU tests of the drafted-tree and bounded-cache calls as a decode loop makes them
one step after the other: descriptors of a position, and weights of slots that a
committed tree brings into use."""
from __future__ import annotations

import numpy as np
import pytest

from fastgemma_amd import kernels as K
from tests import cache_util as U
from tests import hip_util as H
from tests.test_bounded_cache_gpu import by_oracle, dev_cache, queries, words

pytestmark = pytest.mark.gpu


def bytes_of(x):
    return H.host(x).view(np.uint32)


def test_descriptors_hold_the_position_they_were_made_for():
    """Kept descriptors go on at their own position; those of the next step are
    made from its position, or by the call."""
    nh, kvh, hd, cap, n = 8, 1, 64, 120, 5
    rng = np.random.default_rng(40)
    c = U.Cache(rng, cap, hd)
    t = H.torch()
    dc, q, m = dev_cache(c), H.dev(queries(rng, n, nh, hd)), words(K.tree_mask([-1, 0, 0, 1, 2]))
    def attend(seqs):
        out = t.zeros((n, nh, hd), device="cuda")
        K.attend_tree(out, q, seqs, nh, kvh, hd)
        return bytes_of(out)
    at = lambda pos: [(*dc, cap, 0, pos, m)]  # noqa: E731
    kept = K.tree_seqs(at(60))
    first, moved = attend(kept), attend(at(63))
    assert np.array_equal(attend(at(60)), first) and not np.array_equal(moved, first)
    assert np.array_equal(attend(kept), first)
    assert np.array_equal(attend(K.tree_seqs(at(63))), moved)


def test_draft_commit_weigh_and_cut():
    """Steps of a loop that drafts into a cache of bounded size: verify a tree, commit
    its path, give the new slots a mass of 0, weigh by the next row, and cut once
    the cache is full; against the same steps on the host."""
    nh, kvh, hd, cap, budget, sink, recent = 8, 2, 64, 96, 64, 2, 8
    row, pos, n = kvh * hd, 70, 9
    rng = np.random.default_rng(41)
    t = H.torch()
    c = U.Cache(rng, cap, row)
    dc, mass = dev_cache(c), t.full((cap,), float("nan"), device="cuda")
    mass[:pos] = H.dev(rng.uniform(0, 2, pos).astype(np.float32))
    cuts = 0
    for step in range(6):
        masks = K.tree_mask(U.random_tree(rng, n)).view(np.uint64)
        new = U.Cache(rng, n + 1, row)  # the nodes, and the row after them
        def store(at, lo, hi):
            c.k[at:at + hi - lo], c.v[at:at + hi - lo] = new.k[lo:hi], new.v[lo:hi]
            c.ks[at:at + hi - lo], c.vs[at:at + hi - lo] = new.ks[lo:hi], new.vs[lo:hi]
            for x, y in zip(dc, (c.k, c.ks, c.vt, c.vs)):
                x.copy_(H.dev(y))
        store(pos, 0, n)
        q = queries(rng, n + 1, nh, hd)
        out = t.zeros((n, nh, hd), device="cuda")
        K.attend_tree(out, H.dev(q[:n]), [(*dc, cap, 0, pos, words(masks))], nh, kvh, hd)
        deepest = max(range(n), key=lambda i: bin(int(masks[i])).count("1"))
        path = [j for j in range(n) if int(masks[deepest]) >> j & 1]
        want, plain = by_oracle(q[deepest], c, U.line(pos, masks[deepest], n, 0), nh, kvh)
        assert not plain or np.array_equal(H.host(out)[deepest].view(np.uint32), want.view(np.uint32))
        index = np.full(n, -1, np.int32)
        index[:len(path)] = path
        K.kv_move([{"src": (*dc, None), "cap": cap, "pos": pos, "index": H.dev(index)}], row)
        slots = {"k": c.k, "v": c.v, "ks": c.ks, "vs": c.vs}
        U.move(slots, slots, path, 0, pos, 0, pos, cap - pos)
        mass[pos:pos + len(path)] = 0
        pos += len(path)
        store(pos, n, n + 1)
        had = H.host(mass).astype(np.float64)
        one = t.zeros((1, nh, hd), device="cuda")
        K.attend_mass(one, H.dev(q[n:]), [(*dc, cap, 0, pos, 1, mass)], nh, kvh, hd, decay=0.75)
        pos += 1
        w = U.attend64(q[n], c, np.arange(pos), nh, kvh)[1].sum(0)
        had[pos - 1] = 0
        got = H.host(mass)
        s = 9 * 127 * np.abs(q[n]).sum(-1).max() * c.ks.max()  # bounds 9 times any score
        off = (w * (s + 4 + pos / 16 + 24) + (nh + 20) * (w + had[:pos])) * U.EPS + 1e-37
        assert np.all(np.abs(got[:pos] - (0.75 * had[:pos] + w)) <= off), step
        if pos + n + 1 <= cap:
            continue
        keep = t.empty(budget, dtype=t.int32, device="cuda")
        K.kv_select([(keep, mass, pos)], budget, sink, recent)
        kept = H.host(keep)
        assert np.array_equal(kept, U.select(got, pos, budget, sink, recent))
        K.kv_move([{"src": (*dc, mass), "cap": cap, "pos": 0, "index": keep}], row)
        U.move(slots, slots, kept, 0, 0, 0, 0, cap)
        assert np.array_equal(H.host(mass)[:budget], got[kept])
        pos, cuts = budget, cuts + 1
    assert cuts > 0
