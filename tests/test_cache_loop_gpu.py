"""GPU tests of the drafted-tree and bounded-cache calls as a decode loop makes them
one step after the other: descriptors hold a position."""
from __future__ import annotations

import numpy as np
import pytest

from fastgemma_amd import kernels as K
from tests import cache_util as U
from tests import hip_util as H
from tests.test_bounded_cache_gpu import dev_cache, queries, words

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
