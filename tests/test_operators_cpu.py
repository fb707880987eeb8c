"""Beam search, state copies and distillation on the host: more refusals, and host logic."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from vinfer_b200 import _lib
from vinfer_b200.build import build
from vinfer_b200.kernels.sampler.b200 import B200Sampler


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
