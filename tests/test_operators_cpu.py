"""Beam search, state copies and distillation on the host: more refusals, and host logic."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from vinfer_b200 import _lib
from vinfer_b200.beam import BeamSearch
from vinfer_b200.build import build
from vinfer_b200.kernels.sampler.b200 import B200Sampler
from vinfer_b200.sampling import BeamStep, DecodeStates


@pytest.fixture(scope="module")
def backend():
    """The backend's checks, on CPU tensors: nothing here gets past them."""
    build()
    b = object.__new__(B200Sampler)
    b.device = torch.device("cpu")
    b.lib = _lib.load()
    b.status = torch.zeros(1, dtype=torch.int32)
    b._call = None
    return b


def test_the_step_with_a_limit_refuses_as_the_step_does(backend):
    d = _lib.DistillArgs()
    f = backend.lib.vinfer_distill_step_within
    assert f(C.byref(d), 16, 16, 10, 16, 1 << 30, 0, None) == _lib.E_ARG
    d.logits = d.ids = d.logprobs = 16
    d.dtype, d.k, d.rows, d.vocab, d.ld, d.temperature = 0, 4, 2, 10, 10, 1.0
    assert f(C.byref(d), 16, 16, 9, 16, 1 << 30, 0, None) == _lib.E_ARG
    assert f(C.byref(d), 16, 16, 10, 16, 8, 0, None) == _lib.E_LIMIT


# ---- the search ----------------------------------------------------------------------------------
class Untouched:
    """Stands for a search's state: all that a refused step must leave as it was."""

    def __init__(self, search):
        self.search = search
        self.before = {k: v.clone() if torch.is_tensor(v) else v for k, v in vars(search).items()
                       if torch.is_tensor(v) or isinstance(v, int)}

    def check(self):
        for k, v in self.before.items():
            now = getattr(self.search, k)
            assert torch.equal(now, v) if torch.is_tensor(v) else now == v, k


@pytest.mark.parametrize("lengths", [
    torch.zeros(4, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), [1, 1, 1, 1],
    torch.zeros(8, dtype=torch.int32)[::2], torch.zeros(4, dtype=torch.int32, device="meta")],
    ids=["int64", "three slots", "a list", "strided", "elsewhere"])
def test_a_step_with_wrong_lengths_changes_nothing(backend, lengths):
    launched = []

    class Recorder(B200Sampler):
        def beam_select(self, *a, **k):
            launched.append("beam_select")
            raise AssertionError("launched")

    b = object.__new__(Recorder)
    vars(b).update(vars(backend))
    search = BeamSearch(b, 2, 2, 3, states=[DecodeStates([torch.zeros(4, 3, 5)], length_dim=1)])
    kept = Untouched(search)
    with pytest.raises((ValueError, TypeError)):
        search.step(torch.zeros(4, 10), lengths)
    assert not launched
    kept.check()


def test_a_search_refuses_what_its_steps_would(backend):
    """Found when the search is made, not by the first step after it has replaced the scores."""
    with pytest.raises(ValueError, match="states are on meta"):
        BeamSearch(backend, 2, 2, 3, states=[DecodeStates([torch.zeros(4, 3, device="meta")])])
    with pytest.raises(ValueError, match="stop ids"):
        BeamSearch(backend, 1, 1, 3, eos=range(17))
    BeamSearch(backend, 1, 1, 3, eos=range(16))


@pytest.mark.parametrize("w,stops", [(32, 4), (16, 8), (1, 16)])
def test_the_default_number_of_candidates_finds_all_beams_or_is_refused(backend, w, stops):
    """n = W * (1 + stop ids) always holds W that do not end; 128 of them where that is more would not."""
    call = dict(logits=torch.zeros(w, 300), scores=torch.zeros(1, w),
                eos=torch.zeros(stops, dtype=torch.int32))
    if w * (1 + stops) > _lib.BEAM_MAX_N:
        with pytest.raises(ValueError, match="n must be given"):
            backend.beam_select(**call)
    with pytest.raises(TypeError):  # past the checks: there is no launch here
        backend.beam_select(**call, n=100)


@pytest.mark.parametrize("penalty", [-2.0, -1.0, 0.0, 0.6, 1.0])
def test_settled_means_that_no_beam_enters_any_more(backend, penalty):
    """Against finish(), now or after any further steps of a beam (its score only falls)."""
    R, W, T, steps = 400, 2, 9, 2
    g = torch.Generator().manual_seed(3)

    def search(live, at):
        s = BeamSearch(backend, R, W, T, length_penalty=penalty)
        s.steps = at
        s.scores.copy_(live)
        s.done_scores.copy_(done)
        s.done_lengths.fill_(1)
        return s

    done = (-8 * torch.rand(R, W, generator=g)).sort(descending=True).values
    live = -6 * torch.rand(R, W, generator=g)
    if penalty == -1.0:
        done[0], live[0] = torch.tensor([-1.0, -7.0]), torch.tensor([-3.0, -9.0])  # -3 counts -6 now
    done[1], live[1] = torch.tensor([-0.1, -0.2]), torch.tensor([-5.0, -6.0])  # at any penalty here
    settled = search(live, steps).settled()
    assert settled.any() and not settled.all()
    for at in range(steps, T + 1):
        got = search(live, at).finish()
        for r in range(R):
            if settled[r]:
                assert [v for v, _ in got[r]] == done[r].tolist(), (r, at)
    assert settled[1] and not (penalty == -1.0 and settled[0])


# ---- tensors that share memory -------------------------------------------------------------------
def test_states_in_place_must_not_share_memory_across_slots():
    """A slot read through one tensor and written through another: which comes first is not said."""
    buf = torch.zeros(6, 8)
    with pytest.raises(ValueError, match="state 1 overlaps state 0"):
        DecodeStates([buf[:5], buf[1:]])                       # shifted by a slot
    sq = torch.zeros(4, 4)
    with pytest.raises(ValueError, match="state 1 overlaps state 0"):
        DecodeStates([sq, sq.t()])                             # the slots of one are positions of the other
    flat = torch.zeros(64)
    with pytest.raises(ValueError, match="state 2 overlaps state 0"):
        DecodeStates([flat[:32].view(4, 8), torch.zeros(4, 3), flat[28:60].view(4, 8)])
    with pytest.raises(ValueError, match="state 1 overlaps state 0"):
        DecodeStates([flat[:32].view(4, 8), flat[:16].view(4, 4)])  # other strides
    # no shared element, or the same bytes of the same slot
    kv = torch.zeros(4, 2, 3, 5)
    DecodeStates([kv[:, 0], kv[:, 1]])
    layers = torch.zeros(3, 2, 4, 5)
    DecodeStates([layers[:, 0], layers[:, 1]], slot_dim=1)
    packed = torch.zeros(4, 20)
    DecodeStates([packed[:, :7], packed[:, 7:12].view(4, 5, 1), packed[:, 12:]])
    DecodeStates([packed, packed[:, 3:9], packed])
    last = torch.zeros(5, 2, 8)
    DecodeStates([last[:, 0], last[:, 1]], slot_dim=1)


def test_outputs_must_not_share_memory():
    t, u = torch.zeros(4, 8), torch.zeros(4, 8)
    buf = torch.zeros(5, 8)
    with pytest.raises(ValueError, match="output 1 overlaps output 0"):
        DecodeStates([t, u], out=[buf[:4], buf[1:]])
    with pytest.raises(ValueError, match="output 0 overlaps a state"):
        DecodeStates([buf[:4]], out=[buf[1:]])
    # side by side in one buffer, states and outputs too
    both = torch.zeros(4, 3, 8)
    DecodeStates([both[:, 0]], out=[both[:, 2]])
    DecodeStates([t, u], out=[both[:, 0], both[:, 1]])


def test_reordering_refuses_what_it_would_write(backend):
    """Parents and lengths that lie in the states are read while the states change."""
    counts = torch.zeros(4, 3, dtype=torch.int32)
    flat = counts.view(-1)
    with pytest.raises(ValueError, match="parents must not lie in the states"):
        backend.reorder_states(DecodeStates([torch.zeros(4, 2), counts]), flat[2:6])
    st = DecodeStates([counts.view(4, 3, 1)], length_dim=1)
    with pytest.raises(ValueError, match="lengths must not lie in the states"):
        backend.reorder_states(st, torch.zeros(4, dtype=torch.int32), flat[8:])
    out = torch.zeros(4, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="parents must not lie in the states"):
        backend.reorder_states(DecodeStates([counts], out=[out]), out.view(-1)[:4])


def test_a_gradient_may_lie_between_the_logits(backend):
    ids, lp = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    buf = torch.zeros(3, 20)
    for out in (buf[:, 9:19], buf[:, 5:15]):
        with pytest.raises(ValueError, match="not overlap"):
            backend.distill_step(buf[:, :10], ids, lp, out=out)
    with pytest.raises(TypeError):  # past the checks: there is no launch here
        backend.distill_step(buf[:, :10], ids, lp, out=buf[:, 10:])


def test_beam_outputs_are_six_tensors(backend):
    """An output given twice would hold whichever was written last."""
    scores = torch.zeros(2, 4)
    for a, b in (("scores", "next_scores"), ("beams", "tokens"), ("parents", "next_tokens"),
                 ("tokens", "parents")):
        out = BeamStep.empty(2, 4, 4, "cpu")
        setattr(out, a, getattr(out, b))
        with pytest.raises(ValueError, match="given twice"):
            backend.beam_select(torch.zeros(8, 10), scores, 4, out=out)
    out = BeamStep.empty(2, 4, 4, "cpu")
    out.next_scores = scores  # as documented
    with pytest.raises(TypeError):  # past the checks: there is no launch here
        backend.beam_select(torch.zeros(8, 10), scores, 4, out=out)
