"""Logits of large magnitude, by themselves or over a low temperature: the exponents' reference is then
a large number, and what rounding it leaves is not small."""

from __future__ import annotations

import pytest
import torch

from tests.beam_reference import beam_step
from tests.test_beam_gpu import check
from tests.test_distill_gpu import compare, run_all
from vinfer_b200 import SAMPLER, BackendContext

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    return SAMPLER.resolve("b200", BackendContext(torch.device("cuda", 0), torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [1000, 40001])
def test_beams_of_large_logits(backend, V, dtype):
    """Rows far from zero: the exponents' reference is rounded by up to 64 and more there. The last
    rows are masks of one finite value throughout, and with one token left."""
    g = torch.Generator().manual_seed(V)
    rows = [torch.randn(V, generator=g) * 2 + off
            for off in (2e4, -3e5, 1e6, -5e6, 3e7, -2e8, 4e9, 1e30)]
    rows += [torch.full((V,), v) for v in (-1e4, -65504.0, -1e9, -1e30)]
    few = torch.full((4, V), -1e9)
    few[0, 17] = 3.0
    few[1, V - 1] = -7.0
    few[2, :5] = torch.arange(5.0)
    few[3, V // 2] = 1e8
    x = torch.cat([torch.stack(rows), few]).to(dtype)
    scores, eos = -torch.rand(4, 4, generator=g) - 3, torch.tensor([V - 1], dtype=torch.int32)
    got = backend.beam_select(x.to(backend.device), scores.to(backend.device), 12,
                              eos=eos.to(backend.device))
    # scores do not change when a row is shifted, and a double at 1e30 has steps of 1e14
    xd = x.double().numpy()
    check(got, beam_step(xd - xd.max(1, keepdims=True), scores.double().numpy(), 12, [V - 1]))
    backend.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("N,V", [(12, 3001), (120, 90001)])
def test_distillation_of_large_logits(backend, N, V, tail, dtype):
    """The same, in the loss and both forms of the gradient; by magnitude and by a low temperature."""
    g = torch.Generator().manual_seed(N)
    k = 5
    ids = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(N)]).int()
    lp = torch.log_softmax(torch.randn(N, k, generator=g), 1) - 0.5
    w = torch.ones(N)
    off = torch.tensor([2e4, -3e5, 1e6, -5e6, 3e7, -2e8, 4e9, -1e9])[torch.arange(N) % 8]
    x = torch.randn(N, V, generator=g) * 2 + off[:, None]
    x[3::8] = -1e9                                     # one finite value throughout
    x = x.to(dtype)
    _, _, loss, grad, steps = run_all(backend, x, ids, lp, w, 1.0, tail)
    sel = slice(0, 24)
    compare(x[sel], ids[sel], lp[sel], w[sel], 1.0, tail, loss[sel], grad[sel])
    for l, gr in steps:
        compare(x[sel], ids[sel], lp[sel], w[sel], 1.0, tail, l[sel], gr[sel])
    T = 2.0**-12                                       # z = x / T is exact
    x = ((torch.randn(N, V, generator=g) * 8).round() / 8 * T * 2 + 64.0).to(dtype)
    if dtype == torch.float32:
        _, _, loss, grad, steps = run_all(backend, x, ids, lp, w, T, tail)
        for l, gr in [(loss, grad), *steps]:
            compare(x[sel], ids[sel], lp[sel], w[sel], T, tail, l[sel], gr[sel])


@pytest.mark.parametrize("N,V", [(400, 501), (300, 40001)])
def test_large_losses_are_rounded_once(backend, N, V):
    """Listed tokens under a finite mask: losses of thousands, whose rounding is all that shows."""
    g = torch.Generator().manual_seed(N)
    k = 4
    x = torch.randn(N, V, generator=g)
    x[:, 100:] = -30000.0
    ids = torch.stack([torch.randperm(V - 100, generator=g)[:k] + 100 for _ in range(N)]).int()
    lp = torch.log_softmax(torch.randn(N, k, generator=g), 1) - 0.5
    w = torch.rand(N, generator=g) * 1e-3 + 1e-3  # a mean's weights
    _, _, loss, _, steps = run_all(backend, x, ids, lp, w, 1.0, True)
    for l in [loss] + [l for l, _ in steps]:
        compare(x, ids, lp, w, 1.0, True, l)
