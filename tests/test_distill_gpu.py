"""Distillation from top log-probabilities against the 64-bit formulas and against differences."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.beam_reference import distill
from vinfer_b200 import SAMPLER, BackendContext, _lib
from vinfer_b200.distill import distillation_loss
from vinfer_b200.sampling import RowParams

pytestmark = pytest.mark.gpu
NEG = float("-inf")
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def backend():
    return SAMPLER.resolve("b200", BackendContext(torch.device("cuda", 0), torch.bfloat16))


def make(N, V, k, dtype, temperature=1.0, seed=0, noise=0.5):
    g = torch.Generator().manual_seed(seed + N * 13 + V + k)
    x = torch.randn(N, V, generator=g) * 2.5
    at = torch.randint(V, (N, 4), generator=g)
    x.scatter_add_(1, at, torch.rand(N, 4, generator=g) * 6)
    t = (x + noise * torch.randn(N, V, generator=g)) / temperature
    lp, ids = torch.log_softmax(t, 1).topk(min(k, V), dim=1)
    if k > V:  # lists longer than the vocabulary: empty entries
        lp = torch.cat([lp, torch.full((N, k - V), NEG)], 1)
        ids = torch.cat([ids, torch.full((N, k - V), -1)], 1)
    return x.to(dtype), ids.int(), lp, torch.rand(N, generator=g) + 0.5


def tolerances(x, temperature, loss, grad, dtype, weights):
    """Loss: the streamed sum is off by the rounding of its exponents (2^-20, below 32 where they
    count), of the scale (2^-24 of (max - x) / T: below 32 where it counts, 2^-19), by ex2 (2^-22)
    and by at most 64 additions in a chain (2^-24 each); all relative, so absolute in its
    logarithm, times the row's weight (the target's mass is one), then one rounding.
    Gradient: the same relative error on q in each of its two parts, then one rounding to the
    logits' type, or half its smallest step."""
    rel = 2.0**-20 + 2.0**-19 + 2.0**-22 + 64 * 2.0**-24
    tl = np.abs(weights) * rel + np.abs(loss) * 2.0**-24
    eps = torch.finfo(dtype).eps / 2
    z = x / temperature
    q = np.exp(z - z.max(1, keepdims=True))
    q = q / q.sum(1, keepdims=True)
    scale = np.abs(weights)[:, None] / temperature
    tg = scale * q * 2 * rel + np.abs(grad) * (eps + 4 * rel) + 2.0**-126
    return tl, tg


def compare(x, ids, lp, w, temperature, tail, loss, grad=None):
    xd = x.double().cpu().numpy()
    want_l, want_g = distill(xd, ids.cpu().numpy(), lp.double().cpu().numpy(),
                             w.double().cpu().numpy(), temperature, tail)
    tl, tg = tolerances(xd, temperature, want_l, want_g, x.dtype, w.double().cpu().numpy())
    got = loss.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        d = np.where(got == want_l, 0.0, np.abs(got - want_l))  # an infinite loss is met exactly
        tl = np.where(np.isfinite(want_l), tl, 0.0)
    assert np.all(d <= tl), (d.max(), np.argmax(d - tl))
    if grad is not None:
        assert grad.dtype == x.dtype
        d = np.abs(grad.double().cpu().numpy() - want_g)
        assert np.all(d <= tg), (d.max(), np.argwhere(d > tg)[:4].tolist())


def run_all(backend, x, ids, lp, w, temperature, tail, status=0):
    """Loss alone, loss and gradient through autograd, and the step, out of place and in place."""
    dev = backend.device
    d = [t.to(dev) for t in (ids, lp, w)]
    xd = x.to(dev)
    if x.stride(0) != x.shape[1] and x.shape[0] > 1:
        wide = torch.zeros(x.shape[0], x.stride(0), dtype=x.dtype, device=dev)
        wide[:, :x.shape[1]] = xd
        xd = wide[:, :x.shape[1]]
    kw = dict(temperature=temperature, tail=tail)
    only = distillation_loss(backend, xd, *d, **kw)
    leaf = xd.detach().requires_grad_(True)
    loss = distillation_loss(backend, leaf, *d, **kw)
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    l2, g2 = backend.distill_step(xd, *d, **kw)
    l3, g3 = backend.distill_step(xd, *d, **kw, out=torch.empty(x.shape, dtype=x.dtype, device=dev))
    inplace = xd.clone() if xd.is_contiguous() else xd
    keep = xd.clone()
    l4, g4 = backend.distill_step(inplace, *d, **kw, out=inplace)
    assert g4 is inplace
    bits = int(backend.status[0])
    backend.status.zero_()
    assert bits == status
    return keep, only, loss.detach(), grad, [(l2, g2), (l3, g3), (l4, g4)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("N,V,k,T,pad", [
    (1, 1, 1, 1.0, 0), (1, 2, 1, 1.0, 0), (3, 7, 3, 2.0, 1), (5, 9, 12, 1.0, 0), (33, 4097, 7, 1.5, 0),
    (2, 151936, 20, 1.0, 0), (6, 40001, 128, 4.0, 3), (300, 1000, 16, 1.0, 8),
    (1, 262144, 32, 0.5, 0), (2100, 257, 5, 1.0, 0)])
def test_matches_the_formulas(backend, N, V, k, T, pad, tail, dtype):
    x, ids, lp, w = make(N, V, k, dtype, T)
    if pad:
        wide = torch.zeros(N, V + pad, dtype=dtype)
        wide[:, :V] = x
        x = wide[:, :V]
    if N > 4:
        w[N // 2] = 0.0
    kept, only, loss, grad, steps = run_all(backend, x, ids, lp, w, T, tail)
    assert torch.equal(only, loss)
    compare(x, ids, lp, w, T, tail, loss, grad)
    for l, g in steps:
        compare(x, ids, lp, w, T, tail, l, g)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("N,V,k,pad", [(301, 32776, 9, 0), (310, 33001, 128, 0), (297, 50003, 33, 5),
                                       (299, 120007, 20, 1), (610, 65536, 4, 0), (100, 262144, 6, 0),
                                       (97, 248319, 128, 0)])
def test_many_long_rows(backend, N, V, k, pad, dtype):
    """Rows taken whole by one CTA: more than the CTAs, ragged, masked, with bad lists among them."""
    x, ids, lp, w = make(N, V, k, dtype, 1.5)
    if pad:
        wide = torch.zeros(N, V + pad, dtype=dtype)
        wide[:, :V] = x
        x = wide[:, :V]
    w[3::7] = 0.0
    w[-1] = 0.0
    ids[5, 1:] = -1
    ids[6, 1] = ids[6, 0]
    ids[7] = torch.arange(k)            # neighbours in few vectors
    ids[8, 0], ids[8, 1], ids[8, 2] = 0, V - 1, V - 2
    x[9, 100:V - 5] = NEG
    bad = [11, 13]
    ids[11, 0] = V
    x[13, 77] = float("nan")
    good = [r for r in range(N) if r not in bad]
    for tail in (False, True):
        _, _, loss, grad, steps = run_all(backend, x, ids, lp, w, 1.5, tail,
                                          _lib.ST_BAD_LIST | _lib.ST_NONFINITE)
        rows = good if tail else good[:40]
        for l, g in [(loss, grad), *steps]:
            assert torch.isnan(l[bad]).all() and torch.isnan(g[bad]).all()
            compare(x[rows], ids[rows], lp[rows], w[rows], 1.5, tail, l[rows], g[rows])


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("tail", [False, True])
def test_lists_where_it_can_go_wrong(backend, tail, dtype):
    V, k, N = 5003, 8, 9
    x, ids, lp, w = make(N, V, k, dtype)
    ids[0] = -1                        # no entry at all
    ids[1, 3:] = -1                    # a short list
    ids[1, 0] = -5                     # with a hole
    lp[2, 4:] = NEG                    # listed with mass 0
    ids[3] = ids[3, 0]                 # the same id eight times
    lp[3] = np.log(0.1)
    ids[4, 1] = ids[4, 0]              # twice
    lp[5] = NEG                        # nothing but mass 0
    ids[6, 0], ids[6, 1] = 0, V - 1    # the row's ends
    ids[7, :] = torch.arange(16, 24)   # one vector full of them
    lp[8, 0], lp[8, 1:] = 0.0, NEG     # one-hot: cross entropy
    _, _, loss, grad, steps = run_all(backend, x, ids, lp, w, 1.0, tail)
    compare(x, ids, lp, w, 1.0, tail, loss, grad)
    for l, g in steps:
        compare(x, ids, lp, w, 1.0, tail, l, g)
    if not tail:
        assert float(loss[0]) == 0 and not grad[0].any()
        assert float(loss[5]) == 0 and not grad[5].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_masked_and_confident_students(backend, dtype):
    V, k = 3001, 6
    x, ids, lp, w = make(6, V, k, dtype)
    x[0, 200:1500] = NEG                                   # masked vocabulary
    ids[0] = torch.arange(2000, 2000 + k)
    x[1] = torch.finfo(dtype).min                          # a mask of the lowest value
    x[1, :k] = torch.arange(k).to(dtype)
    ids[1] = torch.arange(k)
    x[2, ids[2, 0].long()] = 90.0                           # all mass on one listed token
    x[3] = 0.0                                             # flat
    x[4] = NEG                                             # only the list is left: q_t = 0
    x[4, ids[4].long()] = 1.0
    lp[4] = torch.log_softmax(torch.arange(k).float(), 0)
    x[5, 17] = 60.0                                        # all mass outside the list
    ids[5] = torch.arange(100, 100 + k)
    for tail in (False, True):
        if tail:  # rows 1 and 4 leave no mass outside; a full list has no tail to match
            lp[1] = torch.log_softmax(lp[1], 0) - 1e-3
            sel = [0, 2, 3, 5]
        else:
            sel = list(range(6))
        a = [t[sel].contiguous() for t in (x, ids, lp, w)]
        _, _, loss, grad, steps = run_all(backend, *a, 1.0, tail)
        compare(*a, 1.0, tail, loss, grad)
        for l, g in steps:
            compare(*a, 1.0, tail, l, g)


def test_impossible_targets_are_infinite(backend):
    """Mass on a token the student cannot give: the loss is +inf, as the formula says."""
    dev = backend.device
    x = torch.zeros(2, 50, device=dev)
    x[0, 3] = NEG
    x[1, 5:] = NEG
    ids = torch.tensor([[3], [2]], dtype=torch.int32, device=dev)
    lp = torch.full((2, 1), -0.5, device=dev)
    loss, grad = backend.distill_step(x, ids, lp, tail=True)
    assert loss[0] == float("inf") and abs(float(grad[0, 3]) + np.exp(-0.5)) < 1e-6
    loss, _ = backend.distill_step(x[1:, :], ids[1:], lp[1:], tail=False)
    assert abs(float(loss[0]) - np.log(5.0)) < 1e-6
    backend.check()


def test_bad_rows_are_nan_and_spare_the_others(backend):
    x, ids, lp, w = make(8, 700, 4, torch.float32)
    good = [0, 7]
    ids[1, 2] = 700
    lp[2, 0] = float("nan")
    lp[3, 1] = float("inf")
    x[4, 699] = float("nan")
    x[5, int(ids[5, 0])] = float("inf")
    x[6] = NEG
    for tail in (False, True):
        _, _, loss, grad, steps = run_all(backend, x, ids, lp, w, 1.0, tail,
                                          _lib.ST_BAD_LIST | _lib.ST_NONFINITE)
        for l, g in [(loss, grad), *steps]:
            assert torch.isnan(l[1:7]).all() and torch.isnan(g[1:7]).all()
            compare(x[good], ids[good], lp[good], w[good], 1.0, tail, l[good], g[good])


def test_a_row_of_weight_zero_is_not_read(backend):
    x, ids, lp, w = make(3, 999, 4, torch.bfloat16)
    x[1] = float("nan")
    ids[1] = 5000
    w[1] = 0.0
    _, _, loss, grad, steps = run_all(backend, x, ids, lp, w, 1.0, True)
    for l, g in [(loss, grad), *steps]:
        assert float(l[1]) == 0 and not g[1].any() and torch.isfinite(g).all()


@pytest.mark.parametrize("tail", [False, True])
def test_gradient_against_differences(backend, tail):
    """Central differences of the 64-bit loss at steps of 1e-4: off by h^2 / 6 of the third
    derivative (below 1, the loss is a log-sum) and by 2^-52 * loss / h: under 1e-8. The float32
    gradient adds its own tolerance."""
    V, k, h = 23, 5, 1e-4
    x, ids, lp, w = make(2, V, k, torch.float32, 1.5)
    _, _, loss, grad, _ = run_all(backend, x, ids, lp, w, 1.5, tail)
    a = [t.double().numpy() for t in (lp, w)]
    for r in range(2):
        for i in range(V):
            up, dn = x.double().numpy(), x.double().numpy()
            up[r, i] += h
            dn[r, i] -= h
            lu, _ = distill(up, ids.numpy(), *a, 1.5, tail)
            ld, _ = distill(dn, ids.numpy(), *a, 1.5, tail)
            want = (lu[r] - ld[r]) / (2 * h)
            assert abs(float(grad[r, i]) - want) < 1e-8 + 8e-6 * (abs(want) + 1)


def test_upstream_gradients(backend):
    """A mean (an expanded gradient), unequal rows, a scaled sum; float32 leaves behind bf16."""
    dev = backend.device
    x, ids, lp, w = make(12, 777, 6, torch.bfloat16)
    d = [t.to(dev) for t in (ids, lp, w)]
    up = torch.randn(12, generator=torch.Generator().manual_seed(1))
    for f, weights in ((lambda l: l.mean(), w / 12), (lambda l: (l * up.to(dev)).sum(), w * up),
                       (lambda l: 3 * l.sum(), w * 3)):
        leaf = x.to(dev).requires_grad_(True)
        f(distillation_loss(backend, leaf, *d)).backward()
        _, want = distill(x.double().numpy(), ids.numpy(), lp.double().numpy(),
                          weights.double().numpy(), 1.0, False)
        _, tg = tolerances(x.double().numpy(), 1.0, np.zeros(12), want, torch.bfloat16,
                           weights.double().numpy())
        # the weight is rounded once more on the way (float32): 2^-23 of the gradient
        assert np.all(np.abs(leaf.grad.double().cpu().numpy() - want) <= tg + np.abs(want) * 2.0**-23)


@pytest.mark.parametrize("N,V,dtype", [(40, 30001, torch.bfloat16), (99, 120007, torch.bfloat16),
                                       (98, 120007, torch.float32)], ids=str)
def test_captured_and_side_streams(backend, N, V, dtype):
    dev = backend.device
    x, ids, lp, w = make(N, V, 9, dtype)
    w[::5] = 0.0
    d = [t.to(dev) for t in (x, ids, lp, w)]
    eager_l, eager_g = backend.distill_step(*d, tail=True)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    graphs, outs = [], []
    for s in (s1, s2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            outs.append(backend.distill_step(*d, tail=True))
        graphs.append(gr)
    for _ in range(10):
        for gr, s in zip(graphs, (s1, s2)):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for l, g in outs:
        assert torch.equal(l, eager_l) and torch.equal(g, eager_g)


def test_a_captured_backward_pass(backend):
    """Loss and gradient through autograd inside a captured graph, replayed on new inputs."""
    dev = backend.device
    x, ids, lp, w = make(64, 9001, 9, torch.bfloat16)
    d = [t.to(dev) for t in (ids, lp, w)]
    leaf = x.to(dev).requires_grad_(True)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream())
    gr = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(gr, stream=s):
        loss = distillation_loss(backend, leaf, *d, tail=True)
        (grad,) = torch.autograd.grad(loss.mean(), leaf)
    for seed in (0, 1):
        y, ids2, lp2, w2 = make(64, 9001, 9, torch.bfloat16, seed=seed)
        with torch.no_grad():
            for to, t in zip((leaf, *d), (y, ids2, lp2, w2)):
                to.copy_(t)
        gr.replay()
        torch.cuda.synchronize()
        compare(y, ids2, lp2, w2, 1.0, True, loss.detach())
        _, want = backend.distill_step(leaf.detach(), d[0], d[1], d[2] / 64, tail=True)
        # two roundings of the same value, the weight's to float32 between them: one bf16 step
        assert torch.allclose(grad.float(), want.float(), rtol=2.0**-7, atol=1e-9)


def test_extreme_temperatures(backend):
    """At the ends of the range all mass is on the largest logit, or every token's is the same."""
    dev = backend.device
    x = torch.tensor([[3.0, 1.0, 2.0, -7.0]], device=dev)
    ids = torch.tensor([[0, 2]], dtype=torch.int32, device=dev)
    lp = torch.tensor([[-0.1, -5.0]], device=dev)
    loss, grad = backend.distill_step(x, ids[:, :1].contiguous(), torch.zeros(1, 1, device=dev),
                                      temperature=1e-37)
    assert float(loss[0]) == 0 and torch.isfinite(grad).all()
    loss, grad = backend.distill_step(x, ids, lp, temperature=1e37)
    p = np.exp([-0.1, -5.0]) / np.exp([-0.1, -5.0]).sum()
    assert abs(float(loss[0]) - (p * np.log(p)).sum() - np.log(4)) < 1e-6
    backend.check()


def test_an_output_given_is_seen_to_change(backend):
    dev = backend.device
    x, ids, lp, w = make(4, 300, 3, torch.float32)
    h = x.to(dev).requires_grad_(True)
    logits = h * 1.0
    y = logits.exp()                  # saves its output
    z = (logits ** 2).sum()           # saves logits
    backend.distill_step(logits.detach(), ids.to(dev), lp.to(dev), out=logits.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    y.sum().backward()


def test_no_rows(backend):
    dev = backend.device
    e = [torch.empty(0, 3, dtype=torch.int32, device=dev), torch.empty(0, 3, device=dev)]
    x = torch.empty(0, 50, device=dev, requires_grad=True)
    distillation_loss(backend, x, *e).sum().backward()
    assert x.grad.shape == (0, 50)
    loss, grad = backend.distill_step(x.detach(), *e)
    assert loss.shape == (0,) and grad.shape == (0, 50)


def test_the_teachers_lists_come_from_the_sampler(backend):
    """top_logprobs after a sampling call is the teacher: its ids and prices go in as they are."""
    dev = backend.device
    g = torch.Generator().manual_seed(6)
    t = (torch.randn(16, 5000, generator=g) * 3).to(torch.bfloat16)
    x = (t.float() + torch.randn(16, 5000, generator=g)).to(torch.bfloat16)
    params = RowParams.from_arrays(dev, temperature=np.full(16, 2.0), top_p=np.full(16, 0.9))
    u = torch.rand(16, generator=g).to(dev)
    backend.sample_batch(t.to(dev), params, u)
    ids, lp = backend.top_logprobs(t.to(dev), params, u, None, 20)
    w = torch.ones(16)
    for tail in (False, True):
        _, _, loss, grad, _ = run_all(backend, x, ids, lp, w, 2.0, tail)
        compare(x, ids, lp, w, 2.0, tail, loss, grad)


def test_a_loss_without_gradient_records_nothing(backend):
    x, ids, lp, w = (t.to(backend.device) for t in make(4, 300, 3, torch.float32))
    leaf = x.clone().requires_grad_(True)
    recorded = distillation_loss(backend, leaf, ids, lp, w)
    with torch.no_grad():
        alone = distillation_loss(backend, leaf, ids, lp, w)
    assert recorded.requires_grad and not alone.requires_grad
    assert not distillation_loss(backend, x, ids, lp, w).requires_grad
    assert torch.equal(recorded.detach(), alone)
    with torch.autograd.forward_ad.dual_level():  # a tangent is refused, not dropped
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError)):
            distillation_loss(backend, dual, ids, lp, w)
    backend.check()
