"""Beams whose scores are nearly equal while the errors of their rows' sums are not."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from vinfer_b200 import SAMPLER, BackendContext

pytestmark = pytest.mark.gpu
NEG = float("-inf")


@pytest.fixture(scope="module")
def backend():
    return SAMPLER.resolve("b200", BackendContext(torch.device("cuda", 0), torch.bfloat16))


def constant_tail_row(V, raised, seed):
    """256 tokens raised above a constant tail, one in each thread's first vector (or anywhere): a
    rounding of one addition is the same in each."""
    x = np.zeros(V, np.float32)
    at = np.arange(256) * 4
    if seed is not None:
        at = np.random.default_rng(seed).permutation(V)[:256]
    x[at] = raised
    return x


# Heights over 248,320 float32 tokens whose scores came out 3.4e-6 to 3.7e-6 too high, and too low, when a
# thread added its rounds in float32.
GRID = np.linspace(4, 18, 2048).astype(np.float32)
HIGH, LOW = GRID[[1584, 1010, 1140, 1469]], GRID[[1782, 1902, 1313, 1647]]


@pytest.mark.parametrize("case", range(6))
def test_near_ties_of_rows_whose_sums_round_apart(backend, case):
    """32 requests of two live beams, rows of 248,320 float32 in one part each. The exact scores (sums in
    double) are 2e-6 to 8e-6 apart, either way; their order decides which beam's tokens are listed."""
    R, W, V, n = 32, 16, 248320, 32
    g = np.random.default_rng(case)
    dev = backend.device
    x = torch.zeros(R * W, V, device=dev)
    scores = np.full((R, W), NEG, np.float32)
    want = []
    for r in range(R):
        hard = r % 2 == 0
        up = (HIGH[g.integers(4)], LOW[g.integers(4)]) if hard else g.uniform(6, 16, 2)
        gap = g.uniform(2e-6, 5e-6) if hard else g.choice([-1, 1]) * g.uniform(2e-6, 8e-6)
        if r % 4 == 2:
            up, gap = up[::-1], -gap
        rows = [constant_tail_row(V, np.float32(u), None if hard else 1000 * case + r) for u in up]
        lse = []
        for w, row in enumerate(rows):
            x[r * W + w] = torch.from_numpy(row).to(dev)
            a = np.sort(row.astype(np.float64))
            lse.append(a[-1] + np.log(np.exp(a - a[-1]).sum()))
        best = [float(row.max()) - s for row, s in zip(rows, lse)]
        scores[r, 0] = -1.0
        scores[r, 1] = np.float32(-1.0 + best[0] - best[1] + gap)
        d = (float(scores[r, 1]) + best[1]) - (-1.0 + best[0])
        assert abs(d) > 1e-6
        want.append(int(d > 0))
    got = backend.beam_select(x, torch.from_numpy(scores).to(dev), n)
    first = got.beams[:, 0].tolist()
    assert first == want, [r for r in range(R) if first[r] != want[r]]
    backend.check()
