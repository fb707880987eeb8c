"""The operators together: a batched beam search over a small language model whose state lives in
slots, against an exhaustive plain search on the host; then distillation on what it decoded."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.beam_reference import distill, log_sums
from vinfer_b200 import SAMPLER, BackendContext, SlotHistogram
from vinfer_b200.beam import BeamSearch
from vinfer_b200.distill import distillation_loss
from vinfer_b200.sampling import DecodeStates, RowParams

pytestmark = pytest.mark.gpu
NEG = float("-inf")


@pytest.fixture(scope="module")
def backend():
    return SAMPLER.resolve("b200", BackendContext(torch.device("cuda", 0), torch.bfloat16))


class Model:
    """Logits from the last token and a running sum over the whole sequence, which is the slot's state
    (and, once more, a cache of the tokens): a beam with another's state would get other logits."""

    def __init__(self, V, H, seed):
        g = torch.Generator().manual_seed(seed)
        self.emb = torch.randint(-3, 4, (V, H), generator=g).float()
        self.head = torch.randint(-2, 3, (H, V), generator=g).float() / 4
        self.bias = torch.randn(V, generator=g)
        self.V, self.H = V, H

    def step(self, state, tokens):
        state = state * 0.5 + self.emb.to(state.device)[tokens]
        return state, (state @ self.head.to(state.device) + self.bias.to(state.device))


def host_search(model, start, W, T, eos, penalty):
    """One request, plainly, in float32 logits and 64-bit sums."""
    s0, x0 = model.step(torch.zeros(1, model.H), torch.tensor([start]))
    beams = [(0.0, [], s0, x0)]
    done = []
    for _ in range(T):
        cand = []
        for b, (sc, seq, st, x) in enumerate(beams):
            xd = x.double().numpy()
            lp = xd[0] - log_sums(xd)[0]
            cand += [(np.float32(sc).astype(np.float64) + lp[t], b, t) for t in range(model.V)]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        nxt = []
        for i, (sc, b, t) in enumerate(cand):
            if t in eos:
                if i < W:
                    done.append((sc / (len(beams[b][1]) + 1) ** penalty, beams[b][1] + [t]))
                continue
            if len(nxt) < W:
                nxt.append((sc, b, t))
        beams = [(float(np.float32(sc)), beams[b][1] + [t],
                  *model.step(beams[b][2], torch.tensor([t]))) for sc, b, t in nxt]
    done += [(sc / len(seq) ** penalty, seq) for sc, seq, _, _ in beams]
    return sorted(done, key=lambda d: -d[0])[:W]


@pytest.mark.parametrize("W,eos,penalty", [(1, [3], 1.0), (4, [3, 17], 1.0), (5, [], 0.0),
                                           (8, [0], 0.7)])
def test_search_matches_the_host(backend, W, eos, penalty):
    dev = backend.device
    R, V, H, T = 6, 211, 16, 9
    model = Model(V, H, seed=W)
    slots = R * W
    starts = torch.arange(R).repeat_interleave(W) + 20
    state = torch.zeros(slots, H, device=dev)
    cache = torch.full((slots, 2, T + 1, 3), -1.0, device=dev)
    counts = SlotHistogram.from_token_lists([[int(t)] for t in starts], 32, dev)
    state[:], logits = model.step(state, starts.to(dev))
    cache[:, :, 0] = starts.to(dev)[:, None, None].float()
    search = BeamSearch(backend, R, W, T, eos=eos, length_penalty=penalty,
                        states=[DecodeStates([state]), DecodeStates([cache], length_dim=2),
                                counts.states()])
    for i in range(T):
        lengths = torch.full((slots,), i + 1, dtype=torch.int32, device=dev)
        tokens = search.step(logits, lengths)
        backend.append_tokens(counts, torch.where(search.scores.reshape(-1) > NEG, tokens, -1))
        cache[:, :, i + 1] = tokens[:, None, None].float()
        state[:], logits = model.step(state, tokens.long())
    # every slot's states are its own sequence's
    seqs = search.tokens.cpu()
    alive = (search.scores.reshape(-1) > NEG).cpu()
    for s in range(slots):
        if alive[s]:
            want = torch.cat([starts[s:s + 1], seqs[s].long()]).float()
            assert torch.equal(cache[s, 1, :, 2].cpu(), want)
            ids, n = torch.cat([starts[s:s + 1], seqs[s].long()]).unique(return_counts=True)
            assert counts.to_counts()[s] == dict(zip(ids.tolist(), n.tolist()))
    got = search.finish()
    for r in range(R):
        want = host_search(model, 20 + r, W, T, set(eos), penalty)
        assert [t for _, t in got[r]] == [t for _, t in want], r
        # each step rounds the score once (2^-24 of it) and adds a log-sum off by less than 4e-6
        tol = T * (2.0**-24 * 60 + 4e-6)
        assert all(abs(a - b) < tol for (a, _), (b, _) in zip(got[r], want))


def test_decode_then_distil(backend):
    """A teacher decodes with beams; its top lists at each step train a student in one pass."""
    dev = backend.device
    R, W, V, T, k = 3, 4, 5000, 4, 20
    g = torch.Generator().manual_seed(8)
    search = BeamSearch(backend, R, W, T, eos=[1])
    params = RowParams.from_arrays(dev, temperature=np.ones(R * W))
    u = torch.rand(R * W, generator=g).to(dev)
    rows, lists = [], []
    for _ in range(T):
        t = (torch.randn(R * W, V, generator=g) * 3).to(torch.bfloat16).to(dev)
        backend.sample_batch(t, params, u)
        ids, lp = backend.top_logprobs(t, params, u, None, k)
        alive = (search.scores.reshape(-1) > NEG).float()
        search.step(t)
        rows.append(t)
        lists.append((ids, lp, alive))
    student = torch.cat([(t.float() + torch.randn(R * W, V, generator=g).to(dev)).to(torch.bfloat16)
                         for t in rows]).requires_grad_(True)
    ids, lp, w = (torch.cat(x).contiguous() for x in zip(*lists))
    loss = distillation_loss(backend, student, ids, lp, w, tail=True)
    loss.sum().backward()
    backend.check()
    want, grad = distill(student.detach().double().cpu().numpy(), ids.cpu().numpy(),
                         lp.double().cpu().numpy(), w.double().cpu().numpy(), 1.0, True)
    assert np.allclose(loss.detach().cpu().numpy(), want, rtol=1e-6, atol=1e-5)
    # bf16 gradients: half a step (2^-9 relative to twice the value), and 1e-5 of their parts
    got = student.grad.double().cpu().numpy()
    assert np.all(np.abs(got - grad) <= np.abs(grad) * 2.0**-8 + 1e-5)
    assert all(len(h) for h in search.finish())


def test_settled_and_refusals(backend):
    search = BeamSearch(backend, 2, 2, 3, eos=[0])
    x = torch.zeros(4, 10, device=backend.device)
    x[:, 0] = 30.0                       # ends at once, nothing else has any mass
    search.step(x)
    assert not search.settled().any()    # one hypothesis of two
    search.step(x)
    assert search.settled().all()
    assert [t for _, t in search.finish()[0]][0] == [0]
    with pytest.raises(ValueError, match="width"):
        BeamSearch(backend, 1, 33, 4)
    with pytest.raises(ValueError, match="stop ids"):
        BeamSearch(backend, 1, 32, 4, eos=[1, 2, 3, 4])
    with pytest.raises(ValueError, match="slots"):
        BeamSearch(backend, 2, 2, 3, states=[DecodeStates([torch.zeros(3, 2)])])
    s = BeamSearch(backend, 1, 2, 1)
    s.step(torch.zeros(2, 5, device=backend.device))
    with pytest.raises(ValueError, match="has taken"):
        s.step(torch.zeros(2, 5, device=backend.device))
