"""Beam search, state reordering and distillation on the host: refusals before any launch, the
layout of decode states, the C structs."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from vinfer_b200 import _lib
from vinfer_b200.beam import BeamSearch
from vinfer_b200.build import build
from vinfer_b200.kernels.sampler.b200 import B200Sampler
from vinfer_b200.sampling import BeamStep, DecodeStates, SlotHistogram


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


def test_struct_layouts_match_the_header():
    assert C.sizeof(_lib.BeamArgs) == 8 + 8 + 3 * 8 + 2 * 8 + 8 + 7 * 8
    assert C.sizeof(_lib.State) == 2 * 8 + 4 * 8 + 8 + 3 * 4 * 8
    assert C.sizeof(_lib.DistillArgs) == 8 + 8 + 3 * 8 + 3 * 8 + 8 + 8


def test_workspace_sizes():
    lib = _lib.load()
    f = lib.vinfer_beam_workspace_bytes
    assert 0 < f(64, 4, 151936, _lib.DTYPE_BF16, 8) < 1 << 20
    for bad in ((0, 4, 100, 1, 8), (1, 0, 100, 1, 8), (1, 33, 100, 1, 8), (1, 4, 0, 1, 8),
                (1, 4, _lib.MAX_VOCAB + 1, 1, 8), (1, 4, 100, 7, 8), (1, 4, 100, 1, 129),
                (_lib.MAX_BATCH, 2, 100, 1, 8)):
        assert f(*bad) == 0
    d = lib.vinfer_distill_workspace_bytes
    assert 0 < d(4096, 151936, _lib.DTYPE_BF16, 32) < 1 << 20
    assert d(0, 10, 0, 1) == d(1, 10, 0, 129) == d(1, 10, 5, 1) == d(_lib.DISTILL_MAX_ROWS + 1, 10, 0, 1) == 0


def test_c_entries_refuse_bad_arguments():
    lib = _lib.load()
    assert lib.vinfer_beam_select(None, None, 0, None) == _lib.E_ARG
    a = _lib.BeamArgs()
    for f in ("logits", "scores", "out_scores", "out_beams", "out_tokens"):
        setattr(a, f, 16)
    a.dtype, a.beams, a.requests, a.vocab, a.ld, a.n = _lib.DTYPE_BF16, 4, 2, 100, 100, 8
    big = 1 << 30
    assert lib.vinfer_beam_select(C.byref(a), None, big, None) == _lib.E_ARG      # no workspace
    assert lib.vinfer_beam_select(C.byref(a), 16, 8, None) == _lib.E_LIMIT         # too small
    assert lib.vinfer_beam_select(C.byref(a), 24, big, None) == _lib.E_ARG         # misaligned
    a.parents = 16                                                                # one of three
    assert lib.vinfer_beam_select(C.byref(a), 16, big, None) == _lib.E_ARG
    a.parents, a.n_eos = None, 1                                                  # no stop ids
    assert lib.vinfer_beam_select(C.byref(a), 16, big, None) == _lib.E_ARG
    a.n_eos, a.beams = 0, 33
    assert lib.vinfer_beam_select(C.byref(a), 16, big, None) == _lib.E_LIMIT
    a.beams, a.ld = 4, 99
    assert lib.vinfer_beam_select(C.byref(a), 16, big, None) == _lib.E_ARG
    a.ld, a.logits = 100, 17
    assert lib.vinfer_beam_select(C.byref(a), 16, big, None) == _lib.E_ARG

    s = (_lib.State * 1)()
    assert lib.vinfer_reorder_states(None, 1, 16, 4, None, None, None) == _lib.E_ARG
    assert lib.vinfer_reorder_states(s, 1, 16, 4, None, None, None) == _lib.E_ARG  # null tensors
    s[0].src = s[0].dst = 16
    s[0].run_bytes, s[0].len_outer = 64, -1
    assert lib.vinfer_reorder_states(s, 1, 16, _lib.STATE_MAX_SLOTS + 1, None, None, None) == _lib.E_LIMIT
    s[0].len_unit_bytes = 24                                                      # no divisor
    assert lib.vinfer_reorder_states(s, 1, 16, 4, 16, None, None) == _lib.E_ARG
    s[0].len_unit_bytes = 16                                                      # no lengths
    assert lib.vinfer_reorder_states(s, 1, 16, 4, None, None, None) == _lib.E_ARG
    s[0].len_unit_bytes, s[0].src_slot_stride, s[0].dst_slot_stride = 0, 64, 128   # one tensor, two layouts
    assert lib.vinfer_reorder_states(s, 1, 16, 4, None, None, None) == _lib.E_ARG
    s[0].dst_slot_stride, s[0].n_outer = 64, 1
    s[0].outer_size[0], s[0].src_outer_stride[0], s[0].dst_outer_stride[0] = 2, 256, 512
    assert lib.vinfer_reorder_states(s, 1, 16, 4, None, None, None) == _lib.E_ARG

    d = _lib.DistillArgs()
    assert lib.vinfer_distill_loss(C.byref(d), 16, None, None, 16, big, None) == _lib.E_ARG
    d.logits = d.ids = d.logprobs = 16
    d.dtype, d.k, d.rows, d.vocab, d.ld, d.temperature = 0, 4, 2, 10, 10, 1.0
    assert lib.vinfer_distill_loss(C.byref(d), 16, 16, None, 16, big, None) == _lib.E_ARG
    assert lib.vinfer_distill_loss(C.byref(d), 16, None, None, 16, 8, None) == _lib.E_LIMIT
    assert lib.vinfer_distill_step(C.byref(d), 16, 16, 9, 16, big, None) == _lib.E_ARG
    assert lib.vinfer_distill_grad(C.byref(d), 16, None, None, 0, 16, 10, None) == _lib.E_ARG
    assert lib.vinfer_distill_grad(C.byref(d), 16, 16, 16, -1, 16, 10, None) == _lib.E_ARG
    for t in (0.0, -1.0, 1e-40, 1e38, float("inf"), float("nan")):
        d.temperature = t
        assert lib.vinfer_distill_loss(C.byref(d), 16, None, None, 16, big, None) == _lib.E_ARG
    d.temperature, d.k = 1.0, 129
    assert lib.vinfer_distill_loss(C.byref(d), 16, None, None, 16, big, None) == _lib.E_LIMIT


@pytest.mark.parametrize("what,err", [
    (dict(logits=torch.zeros(8, 10, dtype=torch.float16)), "not supported"),
    (dict(logits=torch.zeros(8, 20)[:, ::2]), "unit column stride"),
    (dict(logits=torch.zeros(10).expand(8, 10)), "must not overlap"),
    (dict(logits=torch.zeros(7, 10)), "for 7 rows"),
    (dict(logits=torch.zeros(8, 0)), "vocabulary"),
    (dict(scores=torch.zeros(2, 4, dtype=torch.float64)), "scores must be"),
    (dict(scores=torch.zeros(4, 2).t()), "scores must be"),
    (dict(logits=torch.zeros(66, 10), scores=torch.zeros(2, 33)), "beams are supported"),
    (dict(n=0), "n must be"), (dict(n=129), "n must be"),
    (dict(eos=torch.zeros(1, dtype=torch.int64)), "eos must be"),
    (dict(eos=torch.zeros(17, dtype=torch.int32)), "stop ids"),
    (dict(out=BeamStep.empty(2, 4, 7, "cpu")), "out.scores"),
])
def test_beam_select_refuses(backend, what, err):
    call = dict(logits=torch.zeros(8, 10), scores=torch.zeros(2, 4), n=8, eos=None, out=None)
    call.update(what)
    with pytest.raises(ValueError, match=err):
        backend.beam_select(**call)


def _lists(n=3, k=2):
    return torch.zeros(n, k, dtype=torch.int32), torch.zeros(n, k)


@pytest.mark.parametrize("what,err", [
    (dict(logits=torch.zeros(3, 10, dtype=torch.float16)), "not supported"),
    (dict(logits=torch.zeros(10).expand(3, 10)), "must not overlap"),
    (dict(ids=torch.zeros(3, 2, dtype=torch.int64)), "ids must be"),
    (dict(ids=torch.zeros(3, 0, dtype=torch.int32)), "k in"),
    (dict(ids=torch.zeros(3, 129, dtype=torch.int32)), "k in"),
    (dict(logprobs=torch.zeros(3, 2, dtype=torch.bfloat16)), "logprobs must be"),
    (dict(logprobs=torch.zeros(2, 2)), "logprobs must be"),
    (dict(weights=torch.zeros(3, 1)), "weights must be"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=1e-40), "temperature"),
])
def test_distill_refuses(backend, what, err):
    ids, lp = _lists()
    call = dict(logits=torch.zeros(3, 10), ids=ids, logprobs=lp)
    call.update(what)
    with pytest.raises(ValueError, match=err):
        backend.distill_loss(**call)
    with pytest.raises(ValueError, match=err):
        backend.distill_step(**call)


def test_distill_step_refuses_outputs(backend):
    ids, lp = _lists()
    buf = torch.zeros(7, 10)
    with pytest.raises(ValueError, match="not overlap"):
        backend.distill_step(buf[:3], ids, lp, out=buf[1:4])
    with pytest.raises(ValueError, match="out must have"):
        backend.distill_step(buf[:3], ids, lp, out=torch.zeros(3, 9))
    with pytest.raises(ValueError, match="out must have"):
        backend.distill_step(buf[:3], ids, lp, out=torch.zeros(10).expand(3, 10))


# ---- decode states -------------------------------------------------------------------------------
def copy_by_description(states: DecodeStates, parents, lengths=None):
    """The copies the description names, byte by byte on the host (tensors live in CPU memory):
    every address is checked against its tensor."""
    base = [(t.data_ptr(), t.data_ptr() + _span(t)) for t in states.tensors if t.numel()]
    obase = [(t.data_ptr(), t.data_ptr() + _span(t)) for t in states.out if t.numel()]
    for i in range(states.count):
        d = states.array[i]
        moves = []
        for s in range(states.slots):
            p = int(parents[s])
            if d.src == d.dst and p == s:
                continue
            n_len = None if lengths is None else int(lengths[s])
            for idx in np.ndindex(*[d.outer_size[k] for k in range(d.n_outer)]):
                if d.len_outer >= 0 and idx[d.len_outer] >= n_len:
                    continue
                nbytes = d.run_bytes
                if d.len_unit_bytes:
                    nbytes = min(nbytes, max(0, n_len) * d.len_unit_bytes)
                if not nbytes:
                    continue
                so = d.src + p * d.src_slot_stride + sum(
                    idx[k] * d.src_outer_stride[k] for k in range(d.n_outer))
                do = d.dst + s * d.dst_slot_stride + sum(
                    idx[k] * d.dst_outer_stride[k] for k in range(d.n_outer))
                assert any(a <= so and so + nbytes <= b for a, b in base)
                assert any(a <= do and do + nbytes <= b for a, b in obase)
                moves.append((do, C.string_at(so, nbytes)))
        for to, data in moves:
            C.memmove(to, data, len(data))


def _span(t):
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def make_states(S):
    g = torch.Generator().manual_seed(4)
    base = torch.randn(5, S, 3, 12, 7, generator=g)
    return {
        "plain": (torch.randn(S, 9, generator=g), 0, None),
        "cache": (torch.randn(S, 3, 11, 8, generator=g), 0, 2),
        "cache, positions first": (torch.randn(S, 11, 3, 8, generator=g), 0, 1),
        "layers outside": (base, 1, 3),
        "sliced": (base[:, :, :, 2:9], 1, 3),
        "length outside": (torch.randn(6, S, 2, 5, generator=g), 1, 0),
        "transposed": (torch.randn(S, 7, 4, generator=g).transpose(1, 2), 0, 1),
        "bf16 odd": (torch.randn(S, 5, 3, generator=g).bfloat16(), 0, 1),
        "one position": (torch.randn(S, 4, 1, 6, generator=g), 0, 2),
        "bytes": (torch.randint(255, (S, 13), generator=g, dtype=torch.uint8), 0, 1),
        "slots last": (torch.randn(4, 5, S, generator=g), 2, 1),
    }


def want_reordered(t, sd, ld, parents, lengths):
    x = t.movedim(sd, 0)
    new = x[torch.as_tensor(parents).long()].clone()
    if lengths is not None:
        shape = [1] * x.dim()
        d = (ld if ld < sd else ld - 1) + 1
        shape[d] = x.shape[d]
        pos = torch.arange(x.shape[d]).reshape(shape)
        live = pos < torch.as_tensor(lengths).reshape([-1] + [1] * (x.dim() - 1))
        new = torch.where(live, new, x)
    return new.movedim(0, sd)


@pytest.mark.parametrize("name", list(make_states(6)))
@pytest.mark.parametrize("with_lengths", [False, True])
def test_descriptions_copy_what_an_index_does(name, with_lengths):
    S = 6
    t, sd, ld = make_states(S)[name]
    if with_lengths and ld is None:
        return
    parents = [0, 0, 2, 2, 4, 0]
    lengths = [0, 3, 1, 99, 2, 5] if with_lengths else None
    want = want_reordered(t, sd, ld, parents, lengths)
    copy_by_description(DecodeStates([t], sd, ld if with_lengths else None), parents, lengths)
    assert torch.equal(t, want)
    # into another tensor, of other strides, from any parent
    t, sd, ld = make_states(S)[name]
    out = torch.zeros(t.shape[::-1], dtype=t.dtype).permute(*reversed(range(t.dim())))
    parents = [5, 0, 1, 2, 3, 3]
    want = want_reordered(t, sd, None, parents, None)
    copy_by_description(DecodeStates([t], sd, out=[out]), parents)
    assert torch.equal(out, want)


def test_decode_states_refuse():
    t = torch.zeros(4, 3, 5)
    with pytest.raises(ValueError, match="no states"):
        DecodeStates([])
    with pytest.raises(ValueError, match="slots"):
        DecodeStates([t, torch.zeros(5, 3)])
    with pytest.raises(ValueError, match="1 to 8192 slots"):
        DecodeStates([torch.zeros(8193, 1)])
    with pytest.raises(ValueError, match="slot_dim"):
        DecodeStates([t], slot_dim=3)
    with pytest.raises(ValueError, match="length_dim must not be"):
        DecodeStates([t], length_dim=0)
    with pytest.raises(ValueError, match="overlaps itself"):
        DecodeStates([torch.zeros(5).expand(4, 5)])
    with pytest.raises(ValueError, match="overlaps a state"):
        DecodeStates([t], out=[t])
    u = torch.zeros(4, 3, 5)
    with pytest.raises(ValueError, match="overlaps a state"):
        DecodeStates([t, u], out=[u, t])
    kv = torch.zeros(4, 2, 3, 5)  # outputs side by side in one buffer are fine
    DecodeStates([t, u], out=[kv[:, 0], kv[:, 1]])
    with pytest.raises(ValueError, match="shape and type"):
        DecodeStates([t], out=[torch.zeros(4, 3, 4)])
    with pytest.raises(ValueError, match="too scattered"):
        DecodeStates([torch.zeros(4, 4, 4, 4, 4, 4, 4)[:, ::2, ::2, ::2, ::2, ::2, ::2]])
    assert DecodeStates([torch.zeros(4, 0)]).count == 0


def test_outputs_are_given_once():
    t, u, out = torch.zeros(4, 3), torch.ones(4, 3), torch.zeros(4, 3)
    with pytest.raises(ValueError, match="given twice"):
        DecodeStates([t, u], out=[out, out])
    e = torch.zeros(4, 0)
    assert DecodeStates([e, e], out=[torch.zeros(4, 0)] * 2).count == 0


def test_search_refuses_states(backend):
    t = torch.zeros(4, 3, 5)
    with pytest.raises(ValueError, match="in place"):
        BeamSearch(backend, 2, 2, 3, states=[DecodeStates([t], out=[torch.zeros(4, 3, 5)])])
    search = BeamSearch(backend, 2, 2, 3, states=[DecodeStates([t], length_dim=1)])
    with pytest.raises(ValueError, match="need lengths"):
        search.step(torch.zeros(4, 10))
    assert search.steps == 0 and search.scores[:, 0].eq(0).all()


def test_reorder_refuses(backend):
    st = DecodeStates([torch.zeros(4, 3, 5)])
    ok = torch.zeros(4, dtype=torch.int32)
    for bad in (ok[:3], ok.long(), torch.zeros(8, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="parents"):
            backend.reorder_states(st, bad)
    with pytest.raises(ValueError, match="go together"):
        backend.reorder_states(st, ok, ok)
    with pytest.raises(ValueError, match="go together"):
        backend.reorder_states(DecodeStates([torch.zeros(4, 3, 5)], length_dim=1), ok)


def test_histograms_are_states():
    slots = SlotHistogram.from_token_lists([[1, 2, 2], [5], [7, 8, 9]], 4, "cpu")
    copy_by_description(slots.states(), [0, 0, 2])
    assert slots.to_counts() == [{1: 1, 2: 2}, {1: 1, 2: 2}, {7: 1, 8: 1, 9: 1}]
