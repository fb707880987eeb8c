"""reorder_states on the device against indexing: copies are exact, and nothing else changes."""

from __future__ import annotations

import pytest
import torch

from tests.test_beam_cpu import make_states, want_reordered
from vinfer_b200 import SAMPLER, BackendContext, SlotHistogram, _lib
from vinfer_b200.sampling import DecodeStates

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    return SAMPLER.resolve("b200", BackendContext(torch.device("cuda", 0), torch.bfloat16))


def on_device(t, dev):
    """The tensor on the device with its strides (slices keep their surroundings)."""
    span = (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) if t.numel() else 0
    flat = torch.as_strided(t, (span,), (1,), t.storage_offset()).to(dev)
    return torch.as_strided(flat, t.shape, t.stride())


def layout(R, W, g):
    """Parents as a beam step leaves them: survivors in place, the others copies of survivors."""
    parents = torch.arange(R * W).reshape(R, W)
    for r in range(R):
        order = torch.randperm(W, generator=g)
        keep = int(torch.randint(1, W + 1, (1,), generator=g))
        for i in range(keep, W):
            parents[r, order[i]] = r * W + order[int(torch.randint(keep, (1,), generator=g))]
    return parents.reshape(-1).int()


@pytest.mark.parametrize("name", list(make_states(6)))
@pytest.mark.parametrize("with_lengths", [False, True])
def test_layouts(backend, name, with_lengths):
    dev, S = backend.device, 6
    t, sd, ld = make_states(S)[name]
    if with_lengths and ld is None:
        return
    parents = torch.tensor([0, 0, 2, 2, 4, 0], dtype=torch.int32)
    lengths = torch.tensor([0, 3, 1, 99, -2, 5], dtype=torch.int32) if with_lengths else None
    want = want_reordered(t, sd, ld, parents, lengths)
    d = on_device(t, dev)
    st = DecodeStates([d], sd, ld if with_lengths else None)
    backend.reorder_states(st, parents.to(dev), None if lengths is None else lengths.to(dev))
    assert torch.equal(d.cpu(), want)
    # into another tensor, from any parent
    d = on_device(make_states(S)[name][0], dev)
    src = d.clone()
    out = torch.zeros(d.shape[::-1], dtype=d.dtype, device=dev).permute(*reversed(range(d.dim())))
    parents = torch.tensor([5, 0, 1, 2, 3, 3], dtype=torch.int32)
    want = want_reordered(src.cpu(), sd, None, parents, None)
    backend.reorder_states(DecodeStates([d], sd, out=[out]), parents.to(dev))
    assert torch.equal(out.cpu(), want) and torch.equal(d, src)
    backend.check()


@pytest.mark.parametrize("R,W,shape,dtype,ld", [
    (1, 2, (1,), torch.int32, None), (64, 4, (2048,), torch.int32, None),
    (16, 4, (8, 300, 64), torch.bfloat16, 2), (3, 16, (5, 33, 80), torch.float32, 2),
    (7, 5, (97, 3), torch.bfloat16, None), (2, 32, (4097,), torch.uint8, 1),
    (1024, 8, (3,), torch.float32, None), (5, 3, (1, 70001), torch.bfloat16, 2)])
def test_in_place(backend, R, W, shape, dtype, ld):
    dev = backend.device
    g = torch.Generator().manual_seed(R * 100 + W)
    t = (torch.randint(255, (R * W, *shape), generator=g, dtype=torch.uint8) if dtype == torch.uint8
         else (torch.randn(R * W, *shape, generator=g) * 100).to(dtype))
    parents = layout(R, W, g)
    lengths = None
    if ld is not None:
        lengths = torch.randint(t.shape[ld] + 1, (R,), generator=g).repeat_interleave(W).int()
    want = want_reordered(t, 0, ld, parents, lengths)
    d = t.to(dev)
    st = DecodeStates([d], length_dim=ld)
    for _ in range(2):  # the same layout again changes nothing
        backend.reorder_states(st, parents.to(dev), None if lengths is None else lengths.to(dev))
        assert torch.equal(d.cpu(), want)
    backend.check()


def test_many_tensors_one_call(backend):
    dev = backend.device
    g = torch.Generator().manual_seed(3)
    parents = layout(5, 4, g)
    ts = [torch.randn(20, 3 + i % 7, 2 + i % 3, generator=g).to(dev) for i in range(150)]
    want = [t[parents.long().to(dev)].clone() for t in ts]
    ts.append(torch.empty(20, 0, device=dev))
    backend.reorder_states(DecodeStates(ts), parents.to(dev))
    for t, w in zip(ts, want):
        assert torch.equal(t, w)


def test_bad_parents_leave_their_slots(backend):
    dev = backend.device
    t = torch.arange(6.0, device=dev).reshape(6, 1).repeat(1, 40)
    st = DecodeStates([t])
    # 1 takes a slot that moves itself; 3 and 5 are out of range
    parents = torch.tensor([2, 0, 2, -1, 2, 6], dtype=torch.int32, device=dev)
    backend.reorder_states(st, parents)
    assert t[:, 0].cpu().tolist() == [2.0, 1.0, 2.0, 3.0, 2.0, 5.0]
    assert int(backend.status[0]) == _lib.ST_BAD_PARENT
    backend.status.zero_()
    out = torch.full_like(t, -7.0)
    backend.reorder_states(DecodeStates([t], out=[out]), parents)
    assert out[:, 39].cpu().tolist() == [2.0, 2.0, 2.0, -7.0, 2.0, -7.0]
    with pytest.raises(RuntimeError, match="parent"):
        backend.check()


def test_offsets_past_32_bits(backend):
    dev = backend.device
    t = torch.zeros(3, 5, (1 << 30) // 4, dtype=torch.int32, device=dev)  # 5 GiB a slot
    t[2, 4, -3:] = 9
    t[2, 0, 0] = 8
    lengths = torch.tensor([t.shape[2]] * 3, dtype=torch.int32, device=dev)
    backend.reorder_states(DecodeStates([t], length_dim=2),
                           torch.tensor([2, 1, 2], dtype=torch.int32, device=dev), lengths)
    assert t[0, 4, -4:].tolist() == [0, 9, 9, 9] and int(t[0, 0, 0]) == 8
    assert int(t[1].sum()) == 0 and int(t[0].sum(dtype=torch.int64)) == 35


def test_captured(backend):
    dev = backend.device
    t = torch.randn(8, 1000, device=dev)
    st = DecodeStates([t])
    parents = torch.arange(8, dtype=torch.int32, device=dev)
    s = torch.cuda.Stream(dev)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=s):
        backend.reorder_states(st, parents)
    for p in ([0, 0, 2, 2, 4, 4, 6, 6], [0, 1, 2, 3, 0, 5, 6, 1]):
        want = t[torch.tensor(p, device=dev)].clone()
        parents.copy_(torch.tensor(p, dtype=torch.int32))
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(t, want)


def test_histograms_follow_the_beams(backend):
    dev = backend.device
    slots = SlotHistogram.from_token_lists([[1, 2, 2], [5], [7, 8, 9], []], 40, dev)
    backend.reorder_states(slots.states(), torch.tensor([0, 0, 2, 2], dtype=torch.int32,
                                                        device=dev))
    backend.append_tokens(slots, torch.tensor([1, 4, -1, 7], dtype=torch.int32, device=dev))
    assert slots.to_counts() == [{1: 2, 2: 2}, {1: 1, 2: 2, 4: 1}, {7: 1, 8: 1, 9: 1},
                                 {7: 2, 8: 1, 9: 1}]
