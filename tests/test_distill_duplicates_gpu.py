"""An id that a list holds more than once: what the loss and the gradient make of it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_distill_gpu import make, tolerances
from vinfer_b200 import SAMPLER, BackendContext

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("N,V,k", [(4, 3001, 8), (100, 90001, 40)])
def test_an_id_listed_more_than_once(N, V, k, tail):
    """Its masses add up: the gradient is that of the list with one entry for them, and so is the loss but
    for the teacher's own terms, p ln p of each entry in place of one of the sum."""
    backend = SAMPLER.resolve("b200", BackendContext(torch.device("cuda", 0), torch.float32))
    x, ids, lp, w = make(N, V, k, torch.float32)
    ids[:, 3] = ids[:, 0]
    ids[:, 5] = ids[:, 0]
    ids[:, 7] = ids[:, 2]
    p = lp.double().exp()
    one, one_p = ids.clone(), p.clone()
    for to, others in ((0, (3, 5)), (2, (7,))):
        for o in others:
            one_p[:, to] += p[:, o]
            one[:, o] = -1
            one_p[:, o] = 0
    one_lp = one_p.log().float()  # entries without id are not read
    norm = torch.ones(N, 1) if tail else p.sum(1, keepdim=True)

    def own(q):  # the teacher's terms
        q = q / norm
        return torch.where(q > 0, q * q.log(), 0.0).sum(1)

    apart = (own(p) - own(one_p)) * w
    assert (apart < -0.01).any()
    d = [t.to(backend.device) for t in (x, ids, lp, w)]
    l2, g2 = backend.distill_step(*d, tail=tail)
    l1, g1 = backend.distill_step(d[0], one.to(backend.device), one_lp.to(backend.device), d[3],
                                  tail=tail)
    # each side's own tolerance, and the merged log-probability's rounding (2^-24 of up to 16, by a mass
    # of one at most)
    x64 = x.double().numpy()
    grad = g1.double().cpu().numpy()
    tl, tg = tolerances(x64, 1.0, l1.double().cpu().numpy(), grad, x.dtype, w.double().numpy())
    assert np.all(np.abs((l2 - l1).double().cpu().numpy() - apart.numpy())
                  <= 2 * tl + w.numpy() * (2.0**-19 + 2.0**-22))
    assert np.all(np.abs(g2.double().cpu().numpy() - grad) <= 2 * tg + w.numpy()[:, None] * 2.0**-19)
    backend.check()
