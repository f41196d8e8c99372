"""Attention over caches past the 32-bit offsets that its reads have: served where
the slots in use lie below 4 GiB, refused where they do not."""
from __future__ import annotations

import numpy as np
import pytest

import fastgemma_amd as F
from fastgemma_amd import kernels as K
from tests import hip_util as H

pytestmark = pytest.mark.gpu  # these calls look for the device before anything else
P = 1 << 40  # an address that is checked, never read


@pytest.mark.parametrize("ring,pos,rows", [(0, (1 << 24) - 3, 3), (0, 1 << 24, 1), (1 << 24, 70, 1), ((1 << 24) + 64, 1 << 25, 2)])
def test_slots_past_four_gib_are_refused(ring, pos, rows):
    """2^24 slots of 256 bytes in use: 4 GiB.  (Without scratch no call is launched, whatever it holds.)"""
    L = F.lib()
    arr = (F.AttnSeq * 1)(F.AttnSeq(P, P, P, P, (1 << 24) + 64, ring, pos, rows))
    assert L.fgm_hip_attend_dev(P, P, arr, 1, 8, 1, 256, 64, None, 0, None) == 1
    assert b"4 GiB" in L.fgm_hip_last_error(), L.fgm_hip_last_error()
    arr[0].rows = 0  # nothing to read
    assert L.fgm_hip_attend_dev(P, P, arr, 1, 8, 1, 256, 64, None, 0, None) == 0


def test_heads_past_four_gib_are_refused():
    L = F.lib()
    end = 1 << 24
    assert L.fgm_hip_attend_heads_dev(P, P, P, P, P, P, 8, 1, 256, end - 9, end, 0, 8, 0, end, None, 0, None) == 1
    assert b"4 GiB" in L.fgm_hip_last_error(), L.fgm_hip_last_error()


@pytest.mark.parametrize("pos,rows,window", [(300, 2, 0), (5000, 40, 0), (2000, 1, 1500)])
def test_slots_in_use_of_a_cache_past_four_gib(pos, rows, window):
    """A cache of 4 GiB and some gives the bytes of one that ends at the last row:
    the single launch, row tiles, single rows."""
    t = H.torch()
    nh, kvh, hd, cap = 8, 1, 256, (1 << 24) + 5
    print(f"attn cache of {cap} slots, {rows} rows at {pos}", flush=True)
    rng = np.random.default_rng(pos)
    end = pos + rows
    small = (end + 3) // 4 * 4
    kc, vt = t.empty(cap * hd, dtype=t.int8, device="cuda"), t.empty((cap + 3) // 4 * 4 * hd, dtype=t.int8, device="cuda")
    ks, vs = t.empty(cap, device="cuda"), t.empty(cap, device="cuda")
    for x in (kc, vt):
        x[:small * hd] = H.dev(rng.integers(-127, 128, small * hd).astype(np.int8))
    for x in (ks, vs):
        x[:small] = H.dev(rng.uniform(0.005, 0.02, small).astype(np.float32))
    q = H.dev((rng.standard_normal(rows * nh * hd) / 8).astype(np.float32))
    got, want = t.full_like(q, 7.0), t.full_like(q, 9.0)
    K.attend(got, q, [(kc, ks, vt, vs, cap, 0, pos, rows)], nh, kvh, hd, window)
    K.attend(want, q, [(kc, ks, vt, vs, small, 0, pos, rows)], nh, kvh, hd, window)
    assert np.array_equal(H.host(got).view(np.uint32), H.host(want).view(np.uint32))
    assert np.abs(H.host(want)).max() > 0
