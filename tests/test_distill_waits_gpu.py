"""The limit of the one-pass step's waits: a call whose waits run out says so, wherever it happened, and
the next call is right."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from tests.test_distill_clusters_gpu import make
from vinfer_b200 import SAMPLER, BackendContext, _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    return SAMPLER.resolve("b200", BackendContext(torch.device("cuda", 0), torch.float32))


def step_within(backend, x, ids, lp, w, wait_ns):
    a = backend._distill_args(x, ids, lp, w, 1.0, True)
    loss, grad = torch.zeros(a.rows, device=x.device), torch.zeros_like(x)
    nbytes = backend.lib.vinfer_distill_workspace_bytes(a.rows, a.vocab, a.dtype, a.k)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    backend._call(lambda s: backend.lib.vinfer_distill_step_within(
        C.byref(a), loss.data_ptr(), grad.data_ptr(), a.vocab, ws.data_ptr(), nbytes, wait_ns, s),
        "vinfer_distill_step_within")
    bits = int(backend.status[0])
    backend.status.zero_()
    return loss, grad, bits


@pytest.mark.parametrize("N,V,dtype", [(300, 120007, torch.bfloat16), (300, 120007, torch.float32),
                                       (96, 248320, torch.float32), (160, 248320, torch.float32)],
                         ids=["1", "2", "4", "4 long"])
def test_waits_that_run_out_are_reported(backend, N, V, dtype):
    x, ids, lp, w = make(backend.device, N, V, 9, dtype, V)
    want_l, want_g = backend.distill_step(x, ids, lp, w, tail=True)
    backend.check()
    # one look a wait: the first wait for HBM does not last
    _, _, bits = step_within(backend, x, ids, lp, w, 0)
    assert bits == _lib.ST_INTERNAL
    ran_out = 0
    for wait_ns in [100, 200, 300, 500, 700, 1000, 1300, 1700, 2200, 3000, 4000, 6000, 9000, 14000,
                    20000, 60000] * 4:
        l, g, bits = step_within(backend, x, ids, lp, w, wait_ns)
        assert bits in (0, _lib.ST_INTERNAL)
        ran_out += bits != 0
        if not bits:  # what is not reported is right
            assert torch.equal(l, want_l) and torch.equal(g, want_g), wait_ns
    assert ran_out
    for wait_ns in (-1, 10**12):  # the usual limit, and no more than that
        l, g, bits = step_within(backend, x, ids, lp, w, wait_ns)
        assert bits == 0 and torch.equal(l, want_l) and torch.equal(g, want_g)
