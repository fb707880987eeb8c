"""Tensors that interleave in one buffer: every operator writes its own elements and no others."""

from __future__ import annotations

import pytest
import torch

from tests.test_distill_gpu import compare, make
from vinfer_b200 import SAMPLER, BackendContext
from vinfer_b200.sampling import DecodeStates

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    return SAMPLER.resolve("b200", BackendContext(torch.device("cuda", 0), torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("N,V,gap", [(5, 999, 0), (5, 1001, 3), (130, 90001, 0), (110, 131072, 8)])
def test_a_gradient_beside_its_logits(backend, N, V, gap, dtype):
    x, ids, lp, w = make(N, V, 9, dtype)
    w[1] = 0.0
    buf = torch.full((N, 2 * V + 2 * gap), -77.0, dtype=dtype, device=backend.device)
    buf[:, :V] = x
    grad = buf[:, V + gap:2 * V + gap]
    loss, got = backend.distill_step(buf[:, :V], *(t.to(backend.device) for t in (ids, lp, w)),
                                     tail=True, out=grad)
    assert got is grad and torch.equal(buf[:, :V].cpu(), x)
    assert (buf[:, V:V + gap] == -77).all() and (buf[:, 2 * V + gap:] == -77).all()
    s = slice(0, 24)
    compare(x[s], ids[s], lp[s], w[s], 1.0, True, loss[s], grad[s])
    backend.check()


def test_states_and_outputs_in_one_buffer(backend):
    g = torch.Generator(backend.device).manual_seed(2)
    buf = torch.randn(6, 3, 5, 7, generator=g, device=backend.device)
    before = buf.clone()
    parents = torch.tensor([5, 0, 1, 2, 3, 3], dtype=torch.int32, device=backend.device)
    backend.reorder_states(DecodeStates([buf[:, 0]], out=[buf[:, 2]]), parents)
    assert torch.equal(buf[:, :2], before[:, :2])
    assert torch.equal(buf[:, 2], before[parents.long(), 0])
    # two states that share bytes of a slot, in place
    parents = torch.tensor([0, 0, 2, 2, 2, 0], dtype=torch.int32, device=backend.device)
    before = buf.clone()
    backend.reorder_states(DecodeStates([buf[:, 1], buf[:, 1, 2:], buf[:, 1]]), parents)
    assert torch.equal(buf[:, 1], before[parents.long(), 1])
    assert torch.equal(buf[:, 0], before[:, 0]) and torch.equal(buf[:, 2], before[:, 2])
    backend.check()
