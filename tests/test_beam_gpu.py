"""beam_select against the 64-bit form: ids, beams and slots exactly, scores to their rounding."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.beam_reference import beam_step
from vinfer_b200 import SAMPLER, BackendContext, _lib
from vinfer_b200.sampling import BeamStep

pytestmark = pytest.mark.gpu
NEG = float("-inf")


@pytest.fixture(scope="module")
def backend():
    return SAMPLER.resolve("b200", BackendContext(torch.device("cuda", 0), torch.bfloat16))


def tolerance(want: np.ndarray) -> np.ndarray:
    """A score is one rounding of b + (x - lse) taken in double: 2^-24 of it. The streamed sum is
    off by the rounding of its exponents' arguments (below 32 in magnitude where they count: 2^-20
    ln 2), by ex2 (2^-22) and by at most 64 additions in a chain (2^-24 each)."""
    return np.abs(want) * 2.0**-24 + 2.0**-20 + 2.0**-22 + 64 * 2.0**-24


def check(got: BeamStep, want: dict, tag=""):
    for k in ("beams", "tokens", "parents", "next_tokens"):
        g = getattr(got, k).cpu().numpy()
        assert np.array_equal(g, want[k]), (tag, k, np.argwhere(g != want[k])[:5].tolist())
    for k in ("scores", "next_scores"):
        g, w = getattr(got, k).cpu().numpy().astype(np.float64), want[k]
        fin = np.isfinite(w)
        assert np.array_equal(np.isfinite(g), fin), (tag, k)
        assert np.all(np.abs(g[fin] - w[fin]) <= tolerance(w[fin])), (tag, k)


def run(backend, x, scores, n, eos, tag="", status=0):
    dev = backend.device
    e = torch.tensor(eos, dtype=torch.int32, device=dev) if eos else None
    got = backend.beam_select(x.to(dev), scores.to(dev), n, eos=e)
    want = beam_step(x.double().numpy(), scores.double().numpy(), n, eos)
    bits = int(backend.status[0])
    backend.status.zero_()
    check(got, want, tag)
    assert bits == status, (tag, bits)
    return got


def logits(g, rows, V, dtype, spread=2.5):
    x = torch.randn(rows, V, generator=g) * spread
    at = torch.randint(V, (rows, 6), generator=g)
    return x.scatter_add_(1, at, torch.rand(rows, 6, generator=g) * 8).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("R,W,V,n,E,pad", [
    (1, 1, 1, 1, 0, 0), (1, 1, 7, 3, 1, 0), (2, 3, 2, 9, 0, 1), (3, 4, 96, 8, 1, 0),
    (2, 5, 1000, 15, 2, 3), (7, 3, 4097, 9, 1, 0), (1, 4, 151936, 8, 1, 0), (2, 32, 2049, 128, 1, 1),
    (5, 16, 40000, 32, 1, 8), (300, 4, 1000, 8, 1, 0), (1, 2, 248320, 100, 0, 5), (1500, 1, 97, 2, 1, 0),
    (1, 1, 262144, 128, 0, 0)])
def test_matches_the_plain_form(backend, R, W, V, n, E, pad, dtype):
    g = torch.Generator().manual_seed(R * 7919 + W * 31 + V + n)
    x = logits(g, R * W, V, dtype)
    if pad:
        wide = torch.full((R * W, V + pad), 77.0, dtype=dtype)
        wide[:, :V] = x
        x = wide[:, :V]
    scores = -4 * torch.rand(R, W, generator=g) - 5
    eos = torch.randperm(V, generator=g)[:E].tolist()
    if eos:  # stop ids among the best of some beams
        for r in range(0, R * W, 3):
            x[r, eos[0]] = x[r].max()
    run(backend, x, scores, n, eos)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [33, 4099, 70001])
def test_hard_rows(backend, V, dtype):
    """Flat, sorted, clustered and mostly masked rows; equal beams; dead beams; first step."""
    g = torch.Generator().manual_seed(V)
    W, n = 4, 20
    rows = []
    rows.append(torch.zeros(W, V))                                    # flat: order by beam, token
    rows.append(torch.arange(V).float().repeat(W, 1) / V * 20)        # ascending: every part's end
    rows.append(-torch.arange(V).float().repeat(W, 1) / V * 20)
    clustered = torch.randn(W, V, generator=g)
    clustered[:, V // 2:V // 2 + min(V // 4, 700)] += 12               # many large neighbours
    rows.append(clustered)
    masked = torch.full((W, V), NEG)                                  # two or no tokens left
    for w in range(W):
        masked[w, torch.randperm(V, generator=g)[:w % 3 + 1]] = float(w)
    rows.append(masked)
    same = torch.randn(1, V, generator=g).repeat(W, 1)                # equal beams: ties by beam
    rows.append(same)
    lowest = torch.full((W, V), torch.finfo(dtype).min)               # a mask of the lowest value
    lowest[:, :3] = torch.randn(W, 3, generator=g)
    rows.append(lowest)
    few = torch.randint(0, 3, (W, V), generator=g).float()            # three values: long ties
    rows.append(few)
    rows.append(torch.randn(W, V, generator=g))
    rows.append(torch.randn(W, V, generator=g))
    x = torch.cat(rows).to(dtype)
    R = len(rows)
    scores = -torch.rand(R, W, generator=g) - 3
    scores[0] = -2.0
    scores[5] = -2.5
    scores[8, 1:] = NEG                                               # the first step
    scores[9] = NEG                                                   # a request that is done
    run(backend, x, scores, n, [V - 1])
    run(backend, x, scores, 1, [])
    run(backend, x, scores, 128, [0, V // 2])


def test_bad_rows_are_reported_and_spare_the_others(backend):
    g = torch.Generator().manual_seed(2)
    W, V = 3, 5000
    x = logits(g, 4 * W, V, torch.float32)
    scores = -torch.rand(4, W, generator=g)
    x[1, 17] = float("nan")
    run(backend, x, scores, 6, [], "nan", _lib.ST_NONFINITE)
    x[1, 17] = float("inf")
    run(backend, x, scores, 6, [], "inf", _lib.ST_NONFINITE)
    x[1] = NEG
    run(backend, x, scores, 6, [], "masked", _lib.ST_NONFINITE)
    scores[0, 1] = NEG  # dead: not read, not reported
    run(backend, x, scores, 6, [], "dead", 0)
    scores[2, 2] = float("nan")
    scores[3, 0] = float("inf")
    run(backend, x, scores, 6, [], "scores", _lib.ST_BAD_SCORE)


@pytest.mark.parametrize("gap", [0, 1, 3])
def test_beams_closer_than_the_rounding_of_their_sums(backend, gap):
    """The same values in another order: the exact sums are equal, so beams a few float steps apart
    in score order by that step alone, and by beam where there is none."""
    g = torch.Generator().manual_seed(5)
    W, V, n = 4, 151936, 16
    base = logits(g, 1, V, torch.float32, 3.0)[0]
    x = torch.stack([base[torch.randperm(V, generator=g)] for _ in range(W)])
    s = np.full((1, W), np.float32(-9.5))
    for _ in range(gap):
        s[0, 2] = np.nextafter(s[0, 2], np.float32(0))
        s[0, 1] = np.nextafter(s[0, 1], np.float32(-99))
    got = run_exact_sums(backend, x, torch.from_numpy(s), n)
    first = got.beams.cpu().numpy()[0, :4].tolist()
    assert first == ([0, 1, 2, 3] if gap == 0 else [2, 0, 3, 1])


def run_exact_sums(backend, x, scores, n):
    """As run(), with the rows' sums taken in order of value, so that equal sums are equal."""
    got = backend.beam_select(x.to(backend.device), scores.to(backend.device), n)
    xs = x.double().numpy()
    order = np.sort(xs, axis=1)
    lse = np.log(np.exp(order - order[:, -1:]).sum(axis=1)) + order[:, -1]
    assert np.all(lse == lse[0])
    total = scores.double().numpy().reshape(-1, 1) + (xs - lse[:, None])
    V = xs.shape[1]
    flat = np.argsort(-total.reshape(-1), kind="stable")[:n]
    assert got.beams.cpu().numpy()[0].tolist() == (flat // V).tolist()
    assert got.tokens.cpu().numpy()[0].tolist() == (flat % V).tolist()
    return got


def test_scores_may_be_updated_in_place_and_outputs_reused(backend):
    g = torch.Generator().manual_seed(9)
    dev, R, W, V, n = backend.device, 6, 4, 999, 8
    scores = -torch.rand(R, W, generator=g)
    x = logits(g, R * W, V, torch.bfloat16)
    want = beam_step(x.double().numpy(), scores.double().numpy(), n, [])
    out = BeamStep.empty(R, W, n, dev)
    live = scores.to(dev)
    out.next_scores = live
    got = backend.beam_select(x.to(dev), live, n, out=out)
    assert got is out
    check(got, want)


def test_graphs_and_streams(backend):
    """Two captured steps and an eager one on three streams at once: nothing is shared."""
    dev = backend.device
    g = torch.Generator().manual_seed(12)
    cases, outs, graphs = [], [], []
    for i in range(3):
        R, W, V, n = 5 + i, 4, 20001 + i, 8
        x, s = logits(g, R * W, V, torch.bfloat16), -torch.rand(R, W, generator=g)
        cases.append((x.to(dev), s.to(dev), n, beam_step(x.double().numpy(), s.double().numpy(), n,
                                                         [])))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(3)]
    for i in range(2):
        x, s, n, _ = cases[i]
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=streams[i]):
            outs.append(backend.beam_select(x, s, n))
        graphs.append(gr)
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            x, s, n, want = cases[2]
            eager = backend.beam_select(x, s, n)
    torch.cuda.synchronize()
    for i in range(2):
        check(outs[i], cases[i][3], f"graph {i}")
    check(eager, cases[2][3], "eager")


def test_the_same_inputs_give_the_same_bits(backend):
    g = torch.Generator().manual_seed(21)
    dev = backend.device
    x, s = logits(g, 32, 50001, torch.bfloat16).to(dev), -torch.rand(8, 4, generator=g).to(dev)
    a = backend.beam_select(x, s, 8)
    for _ in range(5):
        b = backend.beam_select(x, s, 8)
        assert torch.equal(a.scores, b.scores) and torch.equal(a.tokens, b.tokens)


def test_no_requests(backend):
    dev = backend.device
    got = backend.beam_select(torch.empty(0, 50, device=dev), torch.empty(0, 4, device=dev), 8)
    assert got.scores.shape == (0, 8) and got.parents.shape == (0, 4)
