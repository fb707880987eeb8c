"""Beam search over a batch of requests, on the device.

The reference decodes one sequence a request (``src/vinfer/runtime/generate.py:105-146``); here R
requests of W beams decode together, request r's beams in slots ``r * W .. r * W + W - 1`` of the
runtime's decode states. One step is ``B200Sampler.beam_select`` (the best continuations over beams
and vocabulary, the beams that go on laid into their slots), ``reorder_states`` for everything that
belongs to a slot (the sequences here, the model's caches, token counts), and a few operations on
``[R, W]`` tensors that keep the finished hypotheses. Nothing leaves the device until ``finish``::

    search = BeamSearch(backend, requests, width, max_tokens, eos=stop_ids, states=[caches])
    logits = model(prompt tokens of every slot)
    for _ in range(max_tokens):
        tokens = search.step(logits, lengths)     # int32 [R * W], 0 where a beam is dead
        logits = model(tokens)
    sequences = search.finish()

A hypothesis that ends at a stop id is scored by its log-probability divided by its number of tokens
(the stop id among them) to the power ``length_penalty``; a request keeps its W best.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from vinfer_b200 import _lib
from vinfer_b200.kernels.sampler.b200 import B200Sampler
from vinfer_b200.sampling import BeamStep, DecodeStates


class BeamSearch:
    """``states`` are the decode states (``DecodeStates`` of R * W slots, in place) that follow the
    beams; those with a length dimension take the ``lengths`` given to ``step``."""

    def __init__(self, backend: B200Sampler, requests: int, width: int, max_tokens: int, *,
                 eos: Sequence[int] = (), length_penalty: float = 1.0,
                 states: Sequence[DecodeStates] = ()) -> None:
        if requests < 1 or max_tokens < 1:
            raise ValueError("at least one request and one token are needed")
        if not 1 <= width <= _lib.BEAM_MAX_WIDTH:
            raise ValueError(f"width must be in [1, {_lib.BEAM_MAX_WIDTH}], got {width}")
        eos = sorted(set(eos))
        if len(eos) > _lib.BEAM_MAX_EOS:
            raise ValueError(f"at most {_lib.BEAM_MAX_EOS} stop ids are supported, got {len(eos)}")
        if width * (1 + len(eos)) > _lib.BEAM_MAX_N:
            raise ValueError(f"width * (1 + stop ids) must be at most {_lib.BEAM_MAX_N}")
        for s in states:
            if s.slots != requests * width:
                raise ValueError(f"states have {s.slots} slots for {requests} * {width} beams")
            if not s.in_place:
                raise ValueError("the states that follow the beams are copied in place, without out")
            if s.device != backend.device:
                raise ValueError(f"states are on {s.device}, backend on {backend.device}")
        self.backend, self.requests, self.width = backend, requests, width
        self.max_tokens, self.length_penalty, self.states = max_tokens, length_penalty, list(states)
        dev = backend.device
        self.eos = torch.tensor(eos, dtype=torch.int32, device=dev) if eos else None
        self.n = width * (1 + len(eos))
        self.scores = torch.full((requests, width), float("-inf"), device=dev)
        self.scores[:, 0] = 0.0  # the beams of a request begin alike: one is enough
        self.steps = 0
        self.out = BeamStep.empty(requests, width, self.n, dev)
        self.out.next_scores = self.scores
        slots = requests * width
        self.tokens = torch.zeros(slots, max_tokens, dtype=torch.int32, device=dev)
        self._sequences = DecodeStates([self.tokens], length_dim=1)
        self._held = torch.zeros(slots, dtype=torch.int32, device=dev)
        # the finished hypotheses, best first
        self.done_scores = torch.full((requests, width), float("-inf"), device=dev)
        self.done_tokens = torch.zeros(requests, width, max_tokens, dtype=torch.int32, device=dev)
        self.done_lengths = torch.zeros(requests, width, dtype=torch.int64, device=dev)

    def _keep(self, scores: torch.Tensor, slots: torch.Tensor, last: torch.Tensor | None,
              length: int) -> None:
        """Enters hypotheses ``[R, m]`` (the sequence of ``slots``, then ``last``) where ``scores``
        are above -inf, and keeps the W best of each request."""
        seq = self.tokens[slots.clamp(min=0).long()]
        if last is not None:
            seq[:, :, length - 1] = last
        scores = scores / length ** self.length_penalty
        every = torch.cat([self.done_scores, scores], 1)
        best, at = every.sort(dim=1, descending=True, stable=True)
        at = at[:, :self.width]
        self.done_scores = best[:, :self.width].contiguous()
        lengths = torch.cat([self.done_lengths, torch.full_like(slots, length).long()], 1)
        self.done_lengths = lengths.gather(1, at)
        seqs = torch.cat([self.done_tokens, seq], 1)
        self.done_tokens = seqs.gather(1, at[:, :, None].expand(-1, -1, self.max_tokens))

    def step(self, logits: torch.Tensor, lengths: torch.Tensor | None = None) -> torch.Tensor:
        """Takes the next token of every beam from ``logits`` ``[R * W, vocab]`` and moves the states
        with the beams. Returns each slot's token (int32 ``[R * W]``, 0 for a dead beam).
        ``lengths`` (int32 ``[R * W]``): the positions of the states that hold data."""
        if self.steps >= self.max_tokens:
            raise ValueError(f"the search has taken its {self.max_tokens} tokens")
        if any(s.has_lengths for s in self.states):  # before anything of the search changes
            if lengths is None:
                raise ValueError("states with a length_dim need lengths")
            self.backend._slot_values("lengths", lengths, self.requests * self.width)
        b = self.backend.beam_select(logits, self.scores, self.n, eos=self.eos, out=self.out)
        self.steps += 1
        if self.eos is not None:
            # a candidate that ends counts where it is among the W best
            ends = (b.tokens[:, :, None] == self.eos).any(2)
            ends[:, self.width:] = False
            base = torch.arange(self.requests, device=logits.device)[:, None] * self.width
            self._keep(torch.where(ends, b.scores, float("-inf")), base + b.beams, b.tokens,
                       self.steps)
        self.backend.reorder_states(self._sequences, b.parents, self._held)
        for s in self.states:
            self.backend.reorder_states(s, b.parents, lengths if s.has_lengths else None)
        tokens = b.next_tokens.reshape(-1).clamp(min=0)
        self.tokens[:, self.steps - 1] = tokens
        self._held += 1
        return tokens

    def settled(self) -> torch.Tensor:
        """Whether each request's worst kept hypothesis is better than its best beam could become
        (bool ``[R]`` on the device): every further token lowers a beam's log-probability, and
        its length counts for it with a positive penalty, against it with a negative one."""
        last = self.max_tokens if self.length_penalty > 0 else max(1, self.steps)
        bound = self.scores.amax(1) / last ** self.length_penalty
        return self.done_scores[:, -1] >= bound

    def finish(self) -> list[list[tuple[float, list[int]]]]:
        """Each request's hypotheses as (score, tokens), best first; beams that have not ended count
        as they stand. Synchronises."""
        if self.steps:
            base = torch.arange(self.requests * self.width, device=self.tokens.device)
            self._keep(self.scores, base.reshape(self.requests, self.width), None, self.steps)
            self.scores.fill_(float("-inf"))
        self.backend.check()
        scores, tokens = self.done_scores.tolist(), self.done_tokens.tolist()
        lengths = self.done_lengths.tolist()
        return [[(s, t[:n]) for s, t, n in zip(*row) if s > float("-inf")]
                for row in zip(scores, tokens, lengths)]
