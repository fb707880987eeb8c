"""Calls from several host threads at once, whose kernels need different amounts of shared memory."""

from __future__ import annotations

import ctypes as C
import threading
import time

import pytest
import torch

from vinfer_b200 import SAMPLER, BackendContext, _lib
from vinfer_b200.sampling import BeamStep, DecodeStates

pytestmark = pytest.mark.gpu


def together(calls, seconds=3.0):
    """Runs each call over and over in a thread and stream of its own; their exceptions and counts."""
    errors, counts = [], [0] * len(calls)
    end = time.monotonic() + seconds

    def body(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                while time.monotonic() < end and not errors:
                    calls[i]()
                    counts[i] += 1
                    if counts[i] % 64 == 0:
                        torch.cuda.current_stream().synchronize()
                torch.cuda.current_stream().synchronize()
        except Exception as exc:  # noqa: BLE001
            errors.append(exc)

    threads = [threading.Thread(target=body, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return errors, counts


def beam_call(b, x, w, n):
    """One beam step of w beams through the C entry, its arguments made ahead; and its output."""
    rows, v, ld = b._rows(x[:w])
    out = BeamStep.empty(1, w, n, b.device)
    scores = torch.zeros(1, w, device=b.device)
    a = _lib.BeamArgs(
        logits=x.data_ptr(), dtype=_lib.DTYPE_F32, beams=w, requests=1, vocab=v, ld=ld,
        scores=scores.data_ptr(), n=n, out_scores=out.scores.data_ptr(),
        out_beams=out.beams.data_ptr(), out_tokens=out.tokens.data_ptr(),
        status=b.status.data_ptr())
    nbytes = b.lib.vinfer_beam_workspace_bytes(1, w, v, a.dtype, n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=b.device)
    hold = (scores, ws)

    def call():
        b._call(b.lib.vinfer_beam_select, "vinfer_beam_select", C.byref(a), hold[1].data_ptr(), nbytes)

    return call, out


def test_steps_and_copies_of_different_sizes():
    dev = torch.device("cuda", 0)
    b = [SAMPLER.resolve("b200", BackendContext(dev, torch.float32)) for _ in range(4)]
    x = torch.randn(32, 2000, device=dev)
    wide, wide_out = beam_call(b[0], x, 32, 128)      # 128 KiB in the picking kernel
    narrow, narrow_out = beam_call(b[1], x, 16, 100)  # 50 KiB
    many, few = (DecodeStates([torch.zeros(n, 1, device=dev)]) for n in (8192, 6000))
    stay = torch.arange(8192, dtype=torch.int32, device=dev)
    stay_few = stay[:6000]
    want = [b[0].beam_select(x, torch.zeros(1, 32, device=dev), 128),
            b[0].beam_select(x[:16], torch.zeros(1, 16, device=dev), 100)]
    torch.cuda.synchronize()
    for calls in ([wide, narrow], [lambda: b[2].reorder_states(many, stay),
                                   lambda: b[3].reorder_states(few, stay_few)]):
        errors, counts = together(calls)
        assert not errors, (errors, counts)
        assert min(counts) > 100
    for g, w in zip([wide_out, narrow_out], want):
        assert torch.equal(g.tokens, w.tokens) and torch.equal(g.scores, w.scores)
