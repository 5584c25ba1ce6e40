"""The serving operators at their edges, as far as no GPU is needed."""
import random

import torch

from mlir_edsl import _native, serving

INVALID = 1


def test_expire_limits():
    L = _native.lib()
    assert L.b200_debug_w4_expire(-1) == INVALID
    assert "negative" in L.b200_last_error().decode()
    assert L.b200_debug_w4_expire(0) == 0


def test_overlap_of_rows():
    """Against the sets of bytes, over rows of one buffer and several pitches."""
    overlap = serving._calls.overlap_of
    rng = random.Random(1)
    buf = torch.zeros(200, dtype=torch.uint8)
    found = [0, 0]
    for _ in range(4000):
        views, taken = [], []
        for _ in range(2):
            ld, m = rng.choice([5, 8, 8, 8, 13]), rng.randint(0, 5)
            n, start = rng.randint(0, ld), rng.randint(0, 60)
            views.append(buf.as_strided((m, n), (ld, 1), start))
            taken.append({start + i * (ld if m > 1 else n) + k for i in range(m) for k in range(n)})
        want = bool(taken[0] & taken[1])
        found[want] += 1
        assert overlap(*views) == want, (views[0].shape, views[0].stride(), views[1].shape)
    assert min(found) > 500
    cols = torch.zeros(6, 32)
    assert not overlap(cols[:, :16], cols[:, 16:]) and not overlap(cols[:3], cols[3:])
    assert not overlap(cols[:, 4:8], cols[:, 8:32]) and overlap(cols[:, 4:9], cols[:, 8:32])
    assert overlap(cols[:, 30:], cols.view(3, 64)[:, 62:])
    assert not overlap(cols[:, 30:], cols.view(3, 64)[:, :30])
