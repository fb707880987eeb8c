"""The one-pass distillation step over clusters that take many rows each: the rows' buffers are used
again and again, and nothing may depend on which CTA of which cluster is ahead."""

from __future__ import annotations

import pytest
import torch

from vinfer_b200 import SAMPLER, BackendContext

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    return SAMPLER.resolve("b200", BackendContext(torch.device("cuda", 0), torch.float32))


def make(dev, N, V, k, dtype, seed):
    """Students, lists of the teacher's top k (of different lengths) and weights, a tenth of them 0."""
    g = torch.Generator(dev).manual_seed(seed)
    x = torch.randn(N, V, generator=g, device=dev) * 2
    x[:, :16] += torch.rand(N, 16, generator=g, device=dev) * 12
    top, ids = (x + 0.5 * torch.randn(N, V, generator=g, device=dev)).topk(k, dim=1)
    lp = torch.log_softmax(top, 1) - 0.1
    gone = torch.arange(k, device=dev) >= torch.randint(1, k + 1, (N, 1), generator=g, device=dev)
    ids = torch.where(gone, -1, ids).to(torch.int32)
    w = torch.rand(N, generator=g, device=dev) + 0.5
    w[::10] = 0.0
    return x.to(dtype), ids, lp, w


# at most 148 clusters of two or 74 of four fit the SMs at once: seven rows each at least
@pytest.mark.parametrize("N,V,k,dtype", [
    (560, 248320, 128, torch.float32), (530, 248319, 7, torch.float32),
    (1060, 120007, 20, torch.float32), (1040, 262144, 33, torch.bfloat16)],
    ids=["4 f32", "4 f32 ragged", "2 f32 ragged", "2 bf16"])
def test_clusters_that_take_many_rows(backend, N, V, k, dtype):
    """Three steps one behind the other, 20 times, on tensors that are held: the same bits; and every
    element against the three kernels of the two-call form."""
    dev = backend.device
    x, ids, lp, w = make(dev, N, V, k, dtype, V)
    a = dict(temperature=1.5, tail=True)
    loss, saved = backend.distill_loss(x, ids, lp, w, **a, for_grad=True)
    apart = backend.distill_grad(x, ids, lp, w, saved, **a)
    first_l, first_g = backend.distill_step(x, ids, lp, w, **a)
    for i in range(20):
        three = [backend.distill_step(x, ids, lp, w, **a) for _ in range(3)]
        for l, g in three:
            if not (torch.equal(l, first_l) and torch.equal(g, first_g)):
                at = (g != first_g).nonzero()
                raise AssertionError((i, (l != first_l).nonzero()[:8].tolist(), len(at),
                                      at[:8].tolist(), g[g != first_g][:8].tolist(),
                                      first_g[g != first_g][:8].tolist()))
        del three
    # Each form's q is off by its exponents (2^-20, 2^-19 for the scale's rounding), ex2 (2^-22) and at
    # most 64 additions in a chain (2^-24 each), relative; a gradient has it in each of two parts and is
    # rounded once. The two forms together: twice that, a rounding step of the type apart.
    rel = 2.0**-20 + 2.0**-19 + 2.0**-22 + 64 * 2.0**-24
    assert torch.all((loss - first_l).abs() <= 2 * (w * rel + loss.abs() * 2.0**-24))
    for r in range(0, N, 64):
        q = torch.softmax(x[r:r + 64].double() / 1.5, 1) * (w[r:r + 64, None] / 1.5)
        f, t = first_g[r:r + 64].double(), apart[r:r + 64].double()
        tol = 4 * rel * q + f.abs() * (torch.finfo(dtype).eps + 8 * rel) + 2.0**-125
        assert torch.all((f - t).abs() <= tol), (r, ((f - t).abs() - tol).max())
    backend.check()


@pytest.mark.parametrize("N,V,dtype,pad", [(530, 248320, torch.float32, 0), (1040, 120007, torch.float32, 3),
                                           (1040, 262144, torch.bfloat16, 8),
                                           (1200, 151936, torch.bfloat16, 0)],
                         ids=["4 f32", "2 f32 ragged", "2 bf16", "1 bf16"])
def test_the_gradient_in_the_logits_place(backend, N, V, dtype, pad):
    """The same bits as out of place, whatever is written while other chunks of the row are read again."""
    x, ids, lp, w = make(backend.device, N, V, 20, dtype, V + 1)
    wide = torch.full((N, V + pad), -77.0, dtype=dtype, device=x.device)
    wide[:, :V] = x  # of the same strides: a row's sum is added in an order that its alignment gives
    want_l, want_g = backend.distill_step(wide[:, :V], ids, lp, w, temperature=2.0)
    for _ in range(8):
        wide[:, :V] = x
        loss, grad = backend.distill_step(wide[:, :V], ids, lp, w, temperature=2.0, out=wide[:, :V])
        assert torch.equal(loss, want_l) and torch.equal(grad, want_g)
        assert (wide[:, V:] == -77).all()
    backend.check()
