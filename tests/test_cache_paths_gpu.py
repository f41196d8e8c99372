"""GPU tests of the kernels that longer and wider calls of attend, attend_tree and
attend_mass take: every softmax instance past 8192 slots, row tiles of several kv
heads and of head_dims that are no multiple of 128, sums past 32 bits within one
chunk of slots.  Each case names the kernel that it is there for and asserts that
the call launches it."""
from __future__ import annotations

import numpy as np
import pytest

from fastgemma_amd import kernels as K
from tests import cache_util as U
from tests import hip_util as H
from tests.launch_util import launches
from tests.test_attn_gpu import check_job
from tests.test_bounded_cache_gpu import by_oracle, dev_cache, queries, words

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,kernel", [
    (8999, "attn_softmax_kernel<5, 512, 0, 1>"), (10201, "attn_softmax_kernel<5, 512, 0, 1>"),
    (10303, "attn_softmax_kernel<6, 512, 0, 0>"), (12277, "attn_softmax_kernel<6, 512, 0, 0>"),
    (12301, "attn_softmax_kernel<4, 1024, 0, 1>"), (16007, "attn_softmax_kernel<4, 1024, 0, 1>"),
    (16500, "attn_softmax_kernel<5, 1024, 0, 1>"), (20303, "attn_softmax_kernel<5, 1024, 0, 1>"),
])
def test_attend_softmax_instances(n, kernel):
    print(f"attend {n} {kernel}", flush=True)
    check_job([(n, 0, n - 33, 33)], 8, 1, 64, 0, some=2)
    t = H.torch()
    c = [H.dev(np.zeros(s, d)) for s, d in ((n * 64, np.int8), (n, np.float32), ((n + 3) // 4 * 4 * 64, np.int8), (n, np.float32))]
    q, out = t.zeros(33 * 512, device="cuda"), t.zeros(33 * 512, device="cuda")
    sc = t.empty(K.attend_scratch_bytes(33, 8, 1, 64, n) + 256, dtype=t.uint8, device="cuda")
    run = lambda: K.attend(out, q, [(*c, n, 0, n - 33, 33)], 8, 1, 64, 0, sc)  # noqa: E731
    run()
    assert kernel in launches(run)


# name: nh, kvh, hd, window, [(cap, ring, pos, nodes)], what is launched
TREES = {
    "five_groups": (8, 1, 64, 0, [(9100, 0, 9001, 61)], "attn_softmax_kernel<5, 512, 1, 1>"),
    "five_groups_window": (8, 1, 64, 8833, [(9300, 9290, 30011, 64)], "attn_softmax_kernel<5, 512, 1, 1>"),
    "six_groups": (8, 1, 64, 0, [(11100, 0, 11003, 64)], "attn_softmax_kernel<6, 512, 1, 0>"),
    "four_wide_ring": (8, 1, 64, 14999, [(15071, 15071, 40007, 64)], "attn_softmax_kernel<4, 1024, 1, 1>"),
    "four_wide_empty_rows": (8, 2, 64, 0, [(12500, 0, 12431, 33), (9, 0, 0, 5)], "attn_softmax_kernel<4, 1024, 1, 1>"),
    "five_wide": (8, 1, 64, 0, [(20400, 0, 20301, 64)], "attn_softmax_kernel<5, 1024, 1, 1>"),
    "five_wide_window": (12, 1, 64, 17001, [(17100, 17077, 90001, 50)], "attn_softmax_kernel<5, 1024, 1, 1>"),
    "tiles_hd192_two_kv": (8, 2, 192, 0, [(2400, 0, 2305, 64)], "attn_pv_tile_kernel<1, 2, 1>"),
    "tiles_hd320": (8, 1, 320, 0, [(1600, 0, 1501, 64), (900, 0, 811, 9)], "attn_pv_tile_kernel<1, 2, 1>"),
    "tiles_hd448": (4, 1, 448, 0, [(2200, 0, 2101, 64)], "attn_pv_tile_kernel<1, 2, 1>"),
    "tiles_hd512": (8, 1, 512, 0, [(1600, 0, 1503, 50)], "attn_pv_tile_kernel<1, 2, 1>"),
    "tiles_hd512_two_kv": (6, 2, 512, 1300, [(1400, 1370, 5003, 64)], "attn_pv_tile_kernel<1, 2, 1>"),
    "tiles_four_kv": (8, 4, 128, 0, [(2300, 0, 2201, 64)], "attn_pv_tile_kernel<1, 2, 1>"),
    "tiles_three_heads": (9, 3, 64, 0, [(2500, 0, 2399, 64)], "attn_pv_tile_kernel<1, 2, 1>"),
    "tiles_sixteen_heads": (16, 1, 128, 0, [(4100, 0, 4001, 64)], "attn_pv_tile_kernel<1, 2, 1>"),
}


@pytest.mark.parametrize("name", TREES)
def test_tree_paths(name):
    """The oracle's bytes for the first, last and some other rows of each sequence."""
    nh, kvh, hd, window, shapes, kernel = TREES[name]
    print(f"tree {name}", flush=True)
    rng = np.random.default_rng(sum(map(ord, name)))
    caches = [U.Cache(rng, cap, kvh * hd) for cap, *_ in shapes]
    masks = [K.tree_mask(U.random_tree(rng, n)).view(np.uint64) for *_, n in shapes]
    if "empty" in name:
        masks[1][2:4] = 0  # rows that see nothing beside long ones
    q = queries(rng, sum(map(len, masks)), nh, hd)
    t = H.torch()
    out, dq = t.full(q.shape, 7.0, device="cuda"), H.dev(q)
    d = K.tree_seqs([(*dev_cache(c), c.cap, ring, pos, words(m)) for c, m, (_, ring, pos, _) in zip(caches, masks, shapes)],
                    window)
    sc = t.empty(K.attend_scratch_bytes(len(q), nh, kvh, hd, d.span) + 256, dtype=t.uint8, device="cuda")
    run = lambda: K.attend_tree(out, dq, d, nh, kvh, hd, window, sc)  # noqa: E731
    run()
    got, r = H.host(out), 0
    for c, m, (_, ring, pos, n) in zip(caches, masks, shapes):
        for i in range(n):
            if i in (0, 1, n // 3, n // 2, n - 2, n - 1) or pos == 0:
                p = U.line(pos, m[i], n, window)
                want, plain = by_oracle(q[r + i], c, p % ring if ring else p, nh, kvh)
                if plain:
                    assert np.array_equal(got[r + i].view(np.uint32), want.view(np.uint32)), (name, i)
                else:  # an exponential of the tail that the oracle's libm rounds the other way
                    assert np.max(np.abs(got[r + i] - want)) <= 1e-6 * max(np.max(np.abs(want)), 1e-30), (name, i)
        r += n
    assert kernel in launches(run), launches(run)


# name: nh, kvh, hd, sequences of one cache, pos, nodes, the P.V kernel
SUMS = {
    "tiles": (8, 1, 128, 1, 20000, 60, "attn_pv_tile_kernel<1, 2, 1>"),
    "tiles_one_chunk": (16, 1, 512, 16, 1100, 64, "attn_pv_tile_kernel<1, 2, 1>"),
    "rows": (8, 1, 128, 1, 8000, 3, "attn_pv_kernel<0, 1, 1>"),
    "rows_sixteen_heads": (16, 1, 128, 1, 8000, 3, "attn_pv_kernel<1, 1, 1>"),
    "rows_one_chunk": (16, 2, 512, 16, 1100, 1, "attn_pv_kernel<0, 2, 1>"),
    "rows_sixteen_one_chunk": (32, 2, 512, 16, 1100, 1, "attn_pv_kernel<1, 2, 1>"),
}


@pytest.mark.parametrize("value", [127, -127])
@pytest.mark.parametrize("name", SUMS)
def test_sums_past_32_bits_in_a_chunk(name, value):
    """Equal weights of 65535 on values of one size: a chunk of more than 258 slots
    passes 2^31 by itself, in the partial sums between kernels or (one chunk) in
    the sum that is stored."""
    nh, kvh, hd, nseq, pos, n, kernel = SUMS[name]
    print(f"sums {name} {value}", flush=True)
    c = U.Cache(np.random.default_rng(6), pos + n, kvh * hd, fill=value)
    c.vs[:] = 0.0078125
    t = H.torch()
    dc, m = dev_cache(c), words(K.tree_mask(range(-1, n - 1)))
    q, out = t.zeros((nseq * n, nh, hd), device="cuda"), t.zeros((nseq * n, nh, hd), device="cuda")
    d = K.tree_seqs([(*dc, c.cap, 0, pos, m)] * nseq)
    sc = t.empty(K.attend_scratch_bytes(nseq * n, nh, kvh, hd, d.span) + 256, dtype=t.uint8, device="cuda")
    run = lambda: K.attend_tree(out, q, d, nh, kvh, hd, scratch=sc)  # noqa: E731
    run()
    got, want = H.host(out), value * 0.0078125
    # weights (1 / count) * vs: three roundings before 65535 of them, then the sum's and the product's
    assert np.all(np.abs(got - want) <= abs(want) * (0.5 / 65535 + 8 * U.EPS))
    found = launches(run)
    assert kernel in found, found
    chunks = found[kernel][2]
    assert pos // chunks > 258 and ("one_chunk" in name) == (chunks == 1), chunks


def weights64(q, c, pos, window, nh, kvh):
    """Softmax weights of rows at pos, pos + 1, ... in float64: [rows, nh, end].  The
    8-bit query is float32 arithmetic by definition."""
    rows, _, hd = q.shape
    end, grp = pos + rows, nh // kvh
    amax = np.abs(q).max(-1, keepdims=True)
    step = np.where(amax > 0, np.float32(127) / np.where(amax > 0, amax, 1), 0).astype(np.float32)
    q8 = np.clip(np.rint((q * step).astype(np.float32)), -127, 127).astype(np.float64)
    at, last = np.arange(end), pos + np.arange(rows)[:, None]
    seen = (at <= last) & ((at > last - window) if window else True)
    w = np.zeros((rows, nh, end))
    for h in range(nh):
        g = h // grp
        s = q8[:, h] @ c.k[:end, g * hd:(g + 1) * hd].astype(np.float64).T * (amax[:, h].astype(np.float64) / 127.0) \
            * c.ks[:end].astype(np.float64)
        s = np.where(seen, s, -np.inf)
        e = np.exp(s - s.max(1, keepdims=True))
        w[:, h] = e / e.sum(1, keepdims=True)
    return w


def weights_off(q, c, w, nh):
    """How far float32 sums of the weights may be off, as a multiple of 2^-24: a
    score's four roundings and its distance to the maximum bound by nine times the
    largest score, the exponential by four, the sum of n exponentials by n / 16 + 24,
    the adding up by one for each (row, head) and 20."""
    s = 9 * 127 * np.abs(q).sum(-1).max() * c.ks.max()
    return (w.sum((0, 1)) * (s + 4 + w.shape[2] / 16 + 24 + len(q) * nh + 20)) * U.EPS + 1e-37


# name: nh, kvh, hd, window, (cap, pos, rows), what is launched
MASSES = {
    "five_groups": (8, 1, 64, 0, (9050, 8970, 33), "attn_softmax_kernel<5, 512, 2, 1>"),
    "six_groups": (8, 1, 64, 0, (11100, 11007, 40), "attn_softmax_kernel<6, 512, 2, 0>"),
    "four_wide": (8, 1, 64, 0, (15050, 15009, 37), "attn_softmax_kernel<4, 1024, 2, 1>"),
    "four_wide_window": (8, 1, 64, 14001, (16100, 16011, 40), "attn_softmax_kernel<4, 1024, 2, 1>"),
    "five_wide": (8, 1, 64, 0, (20400, 20301, 33), "attn_softmax_kernel<5, 1024, 2, 1>"),
    "six_wide": (8, 1, 64, 0, (24100, 24001, 33), "attn_softmax_kernel<6, 1024, 2, 0>"),
    "tiles_two_kv": (8, 2, 128, 0, (2500, 2405, 64), "attn_mass_kernel<1024, 1>"),
    "tiles_three_heads": (9, 3, 64, 2200, (2600, 2501, 64), "attn_mass_kernel<1024, 1>"),
    "tiles_sixteen_heads": (16, 1, 128, 0, (4100, 4001, 50), "attn_mass_kernel<1024, 1>"),
    "tiles_hd320": (8, 1, 320, 0, (1800, 1701, 40), "attn_mass_kernel<1024, 1>"),
    "rows_hd512": (8, 1, 512, 0, (1300, 1201, 3), "attn_mass_kernel<128, 1>"),
    "single_launch": (8, 2, 64, 0, (700, 611, 40), "attn_mass_kernel<128, 0>"),
}


@pytest.mark.parametrize("name", MASSES)
def test_mass_paths(name):
    """attend's bytes, and the weights against 64 bits."""
    nh, kvh, hd, window, (cap, pos, rows), kernel = MASSES[name]
    print(f"mass {name}", flush=True)
    rng = np.random.default_rng(sum(map(ord, name)))
    c, q = U.Cache(rng, cap, kvh * hd), queries(rng, rows, nh, hd)
    had = rng.uniform(0, 3, cap).astype(np.float32)
    had[pos:] = np.nan
    t = H.torch()
    dc, dq, m = dev_cache(c), H.dev(q), H.dev(had)
    out, plain = t.full(q.shape, 7.0, device="cuda"), t.full(q.shape, 9.0, device="cuda")
    d = K.mass_seqs([(*dc, cap, 0, pos, rows, m)], window)
    sc = t.empty(K.attend_scratch_bytes(rows, nh, kvh, hd, d.span) + 256, dtype=t.uint8, device="cuda")
    run = lambda: K.attend_mass(out, dq, d, nh, kvh, hd, window, 0.5, sc)  # noqa: E731
    run()
    got = H.host(m).copy()
    K.attend(plain, dq, [(*dc, cap, 0, pos, rows)], nh, kvh, hd, window)
    assert np.array_equal(H.host(out).view(np.uint32), H.host(plain).view(np.uint32))
    end = pos + rows
    w = weights64(q, c, pos, window, nh, kvh)
    first = np.where(np.arange(end) < pos, 0.5 * had[:end].astype(np.float64), 0)
    off = weights_off(q, c, w, nh) + 20 * first * U.EPS
    assert np.all(np.abs(got[:end] - w.sum((0, 1)) - first) <= off)
    assert np.array_equal(got[end:].view(np.uint32), had[end:].view(np.uint32))
    assert kernel in launches(run), launches(run)


# the other sequence of the batch: what it makes of the call
BESIDE = {"long_rows": (3000, 2900, 2), "tiles": (5200, 5100, 64), "short": (90, 70, 3)}


@pytest.mark.parametrize("beside", BESIDE)
@pytest.mark.parametrize("pos,rows", [(400, 1), (900, 20), (2301, 40)])
def test_alone_and_in_a_batch(pos, rows, beside):
    """out's bytes do not depend on what a sequence is batched with; its weights are the
    same for the same call, and else differ by their rounding alone."""
    nh, kvh, hd = 8, 1, 64
    rng = np.random.default_rng(pos)
    cap2, pos2, rows2 = BESIDE[beside]
    a, b = U.Cache(rng, pos + rows, hd), U.Cache(rng, cap2, hd)
    q = queries(rng, rows + rows2, nh, hd)
    t = H.torch()
    da, db, dq = dev_cache(a), dev_cache(b), H.dev(q)
    ma, mb = (words(K.tree_mask(U.random_tree(rng, n))) for n in (rows, rows2))
    one, two = t.zeros((rows, nh, hd), device="cuda"), t.zeros((rows + rows2, nh, hd), device="cuda")
    K.attend_tree(one, dq[:rows], [(*da, a.cap, 0, pos, ma)], nh, kvh, hd)
    K.attend_tree(two, dq, [(*da, a.cap, 0, pos, ma), (*db, cap2, 0, pos2, mb)], nh, kvh, hd)
    assert np.array_equal(H.host(one).view(np.uint32), H.host(two)[:rows].view(np.uint32))
    alone = t.zeros(a.cap, device="cuda")
    K.attend_mass(one, dq[:rows], [(*da, a.cap, 0, pos, rows, alone)], nh, kvh, hd)
    batch = []
    for _ in range(2):
        m, m2 = t.zeros(a.cap, device="cuda"), t.zeros(cap2, device="cuda")
        K.attend_mass(two, dq, [(*da, a.cap, 0, pos, rows, m), (*db, cap2, 0, pos2, rows2, m2)], nh, kvh, hd)
        batch.append(H.host(m))
    assert np.array_equal(H.host(one).view(np.uint32), H.host(two)[:rows].view(np.uint32))
    assert np.array_equal(batch[0].view(np.uint32), batch[1].view(np.uint32))
    w = weights64(q[:rows], a, pos, 0, nh, kvh)
    off = weights_off(q[:rows], a, w, nh)
    for got in (H.host(alone), batch[0]):
        assert np.all(np.abs(got - w.sum((0, 1))) <= off)
