"""The ``b200`` sampler backend: the fused sm_100a kernel behind the C ABI.

Registered with ``devices={"cuda"}``, ``dtypes={bfloat16, float32}`` and a ``supports``
check for compute capability 10.0 and a loadable library, so resolving it anywhere else fails
with the reason (``src/vinfer/kernels/registry.py:84-88``), never by falling back.
"""

from __future__ import annotations

import ctypes as C

import torch

from vinfer_b200 import _lib
from vinfer_b200.kernels.sampler.base import SAMPLER
from vinfer_b200.registry import BackendContext
from vinfer_b200.sampling import (
    BeamStep,
    DecodeStates,
    RowParams,
    SamplingParams,
    SlotHistogram,
    TokenHistogram,
    _overlap,
    position_uniform,
)

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def _supports(ctx: BackendContext) -> str | None:
    if not torch.cuda.is_available():
        return "needs a CUDA device (none is available)"
    cc = torch.cuda.get_device_capability(ctx.device)
    if cc != (10, 0):
        return f"needs compute capability 10.0 (B200, sm_100a); device has {cc[0]}.{cc[1]}"
    try:
        _lib.load()
    except (RuntimeError, OSError) as exc:
        return str(exc)
    return None


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


@SAMPLER.register("b200", devices={"cuda"}, dtypes={torch.bfloat16, torch.float32},
                  supports=_supports)
class B200Sampler:
    """Fused single-pass sampler. One instance per device; calls on one instance are
    stream-ordered on the current stream and must not overlap (they share a workspace)."""

    def __init__(self, ctx: BackendContext) -> None:
        self.ctx = ctx
        self.device = torch.device(ctx.device)
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.lib = _lib.load()
        self._workspaces: dict[tuple[int, int, int], torch.Tensor] = {}
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)

    # ---- workspace ---------------------------------------------------------------------------
    def workspace(self, batch: int, vocab: int, dtype: int) -> torch.Tensor:
        key = (batch, vocab, dtype)
        ws = self._workspaces.get(key)
        if ws is None:
            nbytes = self.lib.vinfer_sampler_workspace_bytes(batch, vocab, dtype)
            if nbytes == 0:
                raise ValueError(f"unsupported shape: batch {batch}, vocab {vocab}")
            ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            _lib.check(self.lib.vinfer_sampler_workspace_init(ws.data_ptr(), nbytes,
                                                              self._stream()), "workspace init")
            self._workspaces[key] = ws
        return ws

    def _stream(self) -> int:
        return torch._C._cuda_getCurrentRawStream(self.device.index)

    # ---- argument packing ----------------------------------------------------------------------
    def args(self, logits: torch.Tensor, params: RowParams, uniforms: torch.Tensor | None,
             history: TokenHistogram | None, out: torch.Tensor, probs_out: torch.Tensor | None,
             exact: bool = False, vocab_offset: int = 0,
             vocab_total: int | None = None) -> _lib.SampleArgs:
        if logits.dim() != 2 or logits.stride(1) != 1:
            raise ValueError("logits must be [batch, vocab] with unit column stride")
        if logits.dtype not in _DTYPES:
            raise ValueError(f"logits dtype {logits.dtype} is not supported (float32, bfloat16)")
        if logits.device != self.device:
            raise ValueError(f"logits are on {logits.device}, backend on {self.device}")
        B, V = logits.shape
        for name in ("temperature", "top_k", "top_p", "min_p", "repetition_penalty",
                     "presence_penalty", "frequency_penalty"):
            t = getattr(params, name)
            want = torch.int32 if name == "top_k" else torch.float32
            if t.shape != (B,) or t.dtype != want or not t.is_contiguous() or t.device != self.device:
                raise ValueError(f"params.{name} must be a contiguous {want} [{B}] on {self.device}")
        if uniforms is not None and (uniforms.shape != (B,) or uniforms.dtype != torch.float32
                                     or uniforms.device != self.device):
            raise ValueError(f"uniforms must be float32 [{B}] on {self.device}")
        if out.shape != (B,) or out.dtype != torch.int32 or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous int32 [{B}]")
        if probs_out is not None and (probs_out.shape != (B, V) or probs_out.dtype != torch.float32
                                      or not probs_out.is_contiguous()):
            raise ValueError(f"probs_out must be a contiguous float32 [{B}, {V}]")
        a = _lib.SampleArgs()
        a.logits = logits.data_ptr()
        a.dtype = _DTYPES[logits.dtype]
        a.flags = _lib.FLAG_EXACT_ALL if exact else 0
        a.batch, a.vocab, a.ld = B, V, logits.stride(0)
        a.vocab_offset = vocab_offset
        a.vocab_total = V if vocab_total is None else vocab_total
        a.temperature = _ptr(params.temperature)
        a.top_k = _ptr(params.top_k)
        a.top_p = _ptr(params.top_p)
        a.min_p = _ptr(params.min_p)
        a.repetition_penalty = _ptr(params.repetition_penalty)
        a.presence_penalty = _ptr(params.presence_penalty)
        a.frequency_penalty = _ptr(params.frequency_penalty)
        if history is not None:
            if history.row_ptr.shape != (B + 1,):
                raise ValueError(f"history.row_ptr must be int64 [{B + 1}]")
            a.hist_row_ptr = _ptr(history.row_ptr)
            a.hist_ids = _ptr(history.ids)
            a.hist_counts = _ptr(history.counts)
        a.uniforms = _ptr(uniforms)
        a.out_ids = out.data_ptr()
        a.out_probs = _ptr(probs_out)
        a.status = self.status.data_ptr()
        return a

    # ---- SamplerBackend ------------------------------------------------------------------------
    def sample_batch(self, logits: torch.Tensor, params: RowParams, uniforms: torch.Tensor,
                     history: TokenHistogram | None = None, out: torch.Tensor | None = None,
                     probs_out: torch.Tensor | None = None, exact: bool = False,
                     logprobs_out: torch.Tensor | None = None) -> torch.Tensor:
        """Sample one id per row into ``out``. ``logprobs_out`` (float32 [B], optional)
        receives each sampled token's log-probability under the row's final distribution
        (0 for greedy rows, NaN for rows without a result)."""
        B, V = logits.shape
        if out is None:
            out = torch.empty(B, dtype=torch.int32, device=self.device)
        if logprobs_out is not None and (logprobs_out.shape != (B,) or
                                         logprobs_out.dtype != torch.float32 or
                                         logprobs_out.device != self.device or
                                         not logprobs_out.is_contiguous()):
            raise ValueError(f"logprobs_out must be a contiguous float32 [{B}] on {self.device}")
        a = self.args(logits, params, uniforms, history, out, probs_out, exact)
        ws = self.workspace(B, V, a.dtype)
        _lib.check(self.lib.vinfer_sample(C.byref(a), ws.data_ptr(), ws.numel(), self._stream()),
                   "vinfer_sample")
        if logprobs_out is not None:
            _lib.check(self.lib.vinfer_sample_logprobs(C.byref(a), logprobs_out.data_ptr(),
                                                       ws.data_ptr(), ws.numel(),
                                                       self._stream()), "vinfer_sample_logprobs")
        return out

    def top_logprobs(self, logits: torch.Tensor, params: RowParams, uniforms: torch.Tensor,
                     history: TokenHistogram | None, n: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The ``n`` most likely tokens of each row's final distribution and their
        log-probabilities (``[B, n]`` int32 ids, float32 log-probabilities; -inf outside the
        kept set, id -1 for an empty slot). Call right after ``sample_batch`` on the same
        inputs: it prices tokens with the row results that call left."""
        B, V = logits.shape
        if not 1 <= n <= _lib.TOP_LOGPROBS_MAX or n >= V:
            raise ValueError(f"n must be in [1, {_lib.TOP_LOGPROBS_MAX}] and below the vocabulary")
        ids = torch.empty(B, n, dtype=torch.int32, device=self.device)
        lp = torch.empty(B, n, dtype=torch.float32, device=self.device)
        scratch = torch.empty(B, dtype=torch.int32, device=self.device)
        a = self.args(logits, params, uniforms, history, scratch, None)
        ws = self.workspace(B, V, a.dtype)
        _lib.check(self.lib.vinfer_sample_top_logprobs(C.byref(a), n, ids.data_ptr(),
                                                       lp.data_ptr(), ws.data_ptr(), ws.numel(),
                                                       self._stream()),
                   "vinfer_sample_top_logprobs")
        return ids, lp

    # ---- batched decode with slotted histories ------------------------------------------------
    def append_tokens(self, slots: SlotHistogram, tokens: torch.Tensor) -> None:
        """Count ``tokens[s]`` once more in slot ``s`` (id order kept; a negative id is no
        token). Stream-ordered on the current stream; a full slot sets a status bit."""
        if tokens.shape != (slots.slots,) or tokens.dtype != torch.int32 or \
                tokens.device != self.device or not tokens.is_contiguous():
            raise ValueError(f"tokens must be a contiguous int32 [{slots.slots}] on {self.device}")
        _lib.check(self.lib.vinfer_hist_append(tokens.data_ptr(), slots.slots,
                                               slots.ids.data_ptr(), slots.counts.data_ptr(),
                                               slots.lens.data_ptr(), slots.cap,
                                               self.status.data_ptr(), self._stream()),
                   "vinfer_hist_append")

    def reset_slots(self, slots: SlotHistogram, which: torch.Tensor) -> None:
        """Empty the listed slots (int32 slot numbers on the device): a request leaving."""
        if which.dtype != torch.int32 or which.device != self.device or which.dim() != 1:
            raise ValueError(f"which must be int32 [n] on {self.device}")
        if which.numel() == 0:
            return
        _lib.check(self.lib.vinfer_hist_reset(which.contiguous().data_ptr(), which.numel(),
                                              slots.slots, slots.ids.data_ptr(),
                                              slots.counts.data_ptr(), slots.lens.data_ptr(),
                                              slots.cap, self._stream()), "vinfer_hist_reset")

    def decode_step(self, logits: torch.Tensor, params: RowParams, uniforms: torch.Tensor,
                    slots: SlotHistogram, out: torch.Tensor | None = None) -> torch.Tensor:
        """One decode step of every slot: sample with the slots' histories (penalties) and count
        the sampled ids into them, in one call (``vinfer_sample_decode``: the finishing kernel
        updates each row's slot once the row is decided). Nothing leaves the device; the ids
        are in ``out``."""
        B, V = logits.shape
        if slots.slots != B:
            raise ValueError(f"{slots.slots} slots for {B} rows")
        if out is None:
            out = torch.empty(B, dtype=torch.int32, device=self.device)
        a = self.args(logits, params, uniforms, slots.history, out, None)
        ws = self.workspace(B, V, a.dtype)
        _lib.check(self.lib.vinfer_sample_decode(C.byref(a), slots.lens.data_ptr(), slots.cap,
                                                 ws.data_ptr(), ws.numel(), self._stream()),
                   "vinfer_sample_decode")
        return out

    # ---- beam search ---------------------------------------------------------------------------
    def _call(self, fn, what: str, *args) -> None:
        """``fn(*args, current stream)`` with the backend's device current."""
        if torch.cuda.current_device() == self.device.index:
            _lib.check(fn(*args, self._stream()), what)
        else:
            with torch.cuda.device(self.device):
                _lib.check(fn(*args, self._stream()), what)

    def _rows(self, logits: torch.Tensor) -> tuple[int, int, int]:
        """(rows, vocabulary, row stride) of checked logits."""
        if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
            raise ValueError("logits must be [rows, vocab] with unit column stride")
        if logits.dtype not in _DTYPES:
            raise ValueError(f"logits dtype {logits.dtype} is not supported (float32, bfloat16)")
        if logits.device != self.device:
            raise ValueError(f"logits are on {logits.device}, backend on {self.device}")
        n, v = logits.shape
        if not 1 <= v <= _lib.MAX_VOCAB:
            raise ValueError(f"the vocabulary must have 1 to {_lib.MAX_VOCAB} tokens, got {v}")
        ld = logits.stride(0) if n > 1 else v
        if ld < v:
            raise ValueError("rows of logits must not overlap")
        return n, v, ld

    def _vector(self, name: str, t: torch.Tensor, dtype: torch.dtype, *shape: int) -> int:
        if t.dtype != dtype or t.shape != shape or not t.is_contiguous() or t.device != self.device:
            raise ValueError(f"{name} must be a contiguous {dtype} {list(shape)} on {self.device}")
        return t.data_ptr()

    def beam_select(self, logits: torch.Tensor, scores: torch.Tensor, n: int | None = None,
                    eos: torch.Tensor | None = None, out: BeamStep | None = None) -> BeamStep:
        """One step of beam search for R requests of W beams: ``logits`` ``[R * W, vocab]``,
        ``scores`` ``[R, W]`` (float32, accumulated log-probabilities; -inf: a dead beam, whose
        row is not read). Lists each request's ``n`` best continuations over beams and
        vocabulary (descending score; ties by beam, then token) and lays the W best that do not
        end in one of ``eos`` (int32 stop ids on the device) into its slots: the best child of a
        beam stays in the beam's slot, so ``reorder_states`` only copies the others. ``n``
        defaults to ``W * (1 + len(eos))``, which always finds W; where that exceeds 128 it has to
        be given, and with fewer a slot may go without a beam although one was left.
        ``out.next_scores`` may be ``scores``. Nothing leaves the device."""
        rows, v, ld = self._rows(logits)
        if scores.dim() != 2 or scores.shape[0] * scores.shape[1] != rows:
            raise ValueError(f"scores must be [requests, beams] for {rows} rows of logits")
        r, w = scores.shape
        if not 1 <= w <= _lib.BEAM_MAX_WIDTH:
            raise ValueError(f"1 to {_lib.BEAM_MAX_WIDTH} beams are supported, got {w}")
        if rows > _lib.MAX_BATCH:
            raise ValueError(f"at most {_lib.MAX_BATCH} rows are supported, got {rows}")
        stops = 0 if eos is None else eos.numel()
        if stops > _lib.BEAM_MAX_EOS:
            raise ValueError(f"at most {_lib.BEAM_MAX_EOS} stop ids are supported, got {stops}")
        if n is None:
            n = w * (1 + stops)
            if n > _lib.BEAM_MAX_N:
                raise ValueError(f"n must be given for {w} beams and {stops} stop ids: the {n} that "
                                 f"always find {w} beams are more than {_lib.BEAM_MAX_N}")
        if not 1 <= n <= _lib.BEAM_MAX_N:
            raise ValueError(f"n must be in [1, {_lib.BEAM_MAX_N}], got {n}")
        a = _lib.BeamArgs()
        a.scores = self._vector("scores", scores, torch.float32, r, w)
        if out is None:
            out = BeamStep.empty(r, w, n, self.device)
        else:
            at = {self._vector(f"out.{name}", getattr(out, name), dt, r, m)
                  for name, dt, m in (("scores", torch.float32, n), ("beams", torch.int32, n),
                                      ("tokens", torch.int32, n), ("next_scores", torch.float32, w),
                                      ("parents", torch.int32, w), ("next_tokens", torch.int32, w))}
            if len(at) < 6 and r:
                raise ValueError("an output is given twice")
        if stops:
            a.eos = self._vector("eos", eos, torch.int32, stops)
        if r == 0:
            return out
        a.logits, a.dtype, a.beams = logits.data_ptr(), _DTYPES[logits.dtype], w
        a.requests, a.vocab, a.ld, a.n_eos, a.n = r, v, ld, stops, n
        a.out_scores, a.out_beams = out.scores.data_ptr(), out.beams.data_ptr()
        a.out_tokens, a.next_scores = out.tokens.data_ptr(), out.next_scores.data_ptr()
        a.parents, a.next_tokens = out.parents.data_ptr(), out.next_tokens.data_ptr()
        a.status = self.status.data_ptr()
        nbytes = self.lib.vinfer_beam_workspace_bytes(r, w, v, a.dtype, n)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self._call(self.lib.vinfer_beam_select, "vinfer_beam_select", C.byref(a), ws.data_ptr(),
                   nbytes)
        return out

    def _slot_values(self, name: str, t: torch.Tensor, slots: int) -> None:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if t.dtype != torch.int32 or t.numel() != slots or not t.is_contiguous() or \
                t.device != self.device:
            raise ValueError(f"{name} must be a contiguous int32 of {slots} slots on {self.device}")

    def reorder_states(self, states: DecodeStates, parents: torch.Tensor,
                       lengths: torch.Tensor | None = None) -> None:
        """Slot ``s`` of every state takes the contents of slot ``parents[s]`` (int32, one for each
        slot, any shape: ``BeamStep.parents``). In place a moved slot's parent must keep its own
        state, as ``beam_select`` lays beams out; into ``out`` tensors any parent will do. With
        a ``length_dim``, only the first ``lengths[s]`` (int32) positions are copied. A parent
        out of range, or one that moves itself, leaves the slot alone and sets a status bit.
        Neither tensor may lie in the states that are written."""
        if states.device != self.device:
            raise ValueError(f"states are on {states.device}, backend on {self.device}")
        self._slot_values("parents", parents, states.slots)
        if lengths is not None:
            self._slot_values("lengths", lengths, states.slots)
        if (lengths is not None) != states.has_lengths:
            raise ValueError("lengths and a length_dim of the states go together")
        if states.count == 0:
            return
        at, held, nbytes = parents.data_ptr(), _ptr(lengths), 4 * states.slots
        if states.writes_to(at, at + nbytes):
            raise ValueError("parents must not lie in the states that are written")
        if held is not None and states.writes_to(held, held + nbytes):
            raise ValueError("lengths must not lie in the states that are written")
        self._call(self.lib.vinfer_reorder_states, "vinfer_reorder_states", states.array,
                   states.count, at, states.slots, held, self.status.data_ptr())

    # ---- distillation ---------------------------------------------------------------------------
    def _distill_args(self, logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor,
                      weights: torch.Tensor | None, temperature: float,
                      tail: bool) -> _lib.DistillArgs:
        n, v, ld = self._rows(logits)
        if n > _lib.DISTILL_MAX_ROWS:
            raise ValueError(f"at most {_lib.DISTILL_MAX_ROWS} rows are supported, got {n}")
        k = ids.shape[1] if ids.dim() == 2 else 0
        if not 1 <= k <= _lib.DISTILL_MAX_K:
            raise ValueError(f"ids must be [rows, k] with k in [1, {_lib.DISTILL_MAX_K}]")
        if not 1e-37 <= temperature <= 1e37:
            raise ValueError(f"temperature must be in [1e-37, 1e37], got {temperature}")
        a = _lib.DistillArgs()
        a.ids = self._vector("ids", ids, torch.int32, n, k)
        a.logprobs = self._vector("logprobs", logprobs, torch.float32, n, k)
        if weights is not None:
            a.weights = self._vector("weights", weights, torch.float32, n)
        a.logits, a.dtype, a.k = logits.data_ptr(), _DTYPES[logits.dtype], k
        a.rows, a.vocab, a.ld = n, v, ld
        a.temperature, a.tail = temperature, bool(tail)
        a.status = self.status.data_ptr()
        return a

    def _grad_like(self, logits: torch.Tensor, ld: int) -> torch.Tensor:
        """The gradient's tensor, with the logits' row stride where that is a padded one, so that
        rows of both are aligned alike."""
        n, v = logits.shape
        if v < ld <= 2 * v:
            return torch.empty(n, ld, dtype=logits.dtype, device=self.device)[:, :v]
        return torch.empty(n, v, dtype=logits.dtype, device=self.device)

    def distill_loss(self, logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor,
                     weights: torch.Tensor | None = None, *, temperature: float = 1.0,
                     tail: bool = False, for_grad: bool = False
                     ) -> tuple[torch.Tensor, torch.Tensor | None]:
        """The rows' distillation losses (float32 ``[rows]``), and with ``for_grad`` what
        ``distill_grad`` needs of them (float32 ``[rows * (2 + k)]``).
        ``vinfer_b200.distill.distillation_loss`` is the differentiable form."""
        a = self._distill_args(logits, ids, logprobs, weights, temperature, tail)
        n, k = a.rows, a.k
        loss = torch.empty(n, dtype=torch.float32, device=self.device)
        saved = stats = lists = None
        if for_grad:
            saved = torch.empty(n * (2 + k), dtype=torch.float32, device=self.device)
            stats = saved.data_ptr()
            lists = stats + 8 * n
        if n:
            nbytes = self.lib.vinfer_distill_workspace_bytes(n, a.vocab, a.dtype, k)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            self._call(self.lib.vinfer_distill_loss, "vinfer_distill_loss", C.byref(a),
                       loss.data_ptr(), stats, lists, ws.data_ptr(), nbytes)
        return loss, saved

    def distill_grad(self, logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor,
                     weights: torch.Tensor | None, saved: torch.Tensor,
                     grad_out: torch.Tensor | None = None, *, temperature: float = 1.0,
                     tail: bool = False) -> torch.Tensor:
        """The gradient of ``sum(grad_out * loss)`` with respect to the logits, of their type
        (``grad_out``: float32 ``[rows]`` of any stride, None for ones), from what
        ``distill_loss`` saved for the same arguments."""
        a = self._distill_args(logits, ids, logprobs, weights, temperature, tail)
        stats = self._vector("saved", saved, torch.float32, a.rows * (2 + a.k))
        gp, step = None, 0
        if grad_out is not None:
            if grad_out.shape != (a.rows,) or grad_out.dtype != torch.float32 or \
                    grad_out.device != self.device:
                raise ValueError(f"grad_out must be float32 [{a.rows}] on {self.device}")
            gp, step = grad_out.data_ptr(), grad_out.stride(0)
        grad = self._grad_like(logits, a.ld)
        if a.rows:
            self._call(self.lib.vinfer_distill_grad, "vinfer_distill_grad", C.byref(a), stats,
                       stats + 8 * a.rows, gp, step, grad.data_ptr(),
                       grad.stride(0) if a.rows > 1 else a.vocab)
        return grad

    def distill_step(self, logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor,
                     weights: torch.Tensor | None = None, *, temperature: float = 1.0,
                     tail: bool = False, out: torch.Tensor | None = None
                     ) -> tuple[torch.Tensor, torch.Tensor]:
        """The rows' losses and the gradient of their sum with respect to the logits in one call,
        for a training step whose row weights are known ahead (``logits.backward(grad)``
        carries on). ``out`` receives the gradient; it may be ``logits`` itself, whose memory
        the step then reuses. Nothing is recorded for autograd."""
        a = self._distill_args(logits, ids, logprobs, weights, temperature, tail)
        given = out is not None
        if not given:
            out = self._grad_like(logits, a.ld)
        elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != self.device or \
                (out.stride(1) != 1 and a.vocab > 1) or (a.rows > 1 and out.stride(0) < a.vocab):
            raise ValueError("out must have the logits' shape and type, with unit column stride")
        loss = torch.empty(a.rows, dtype=torch.float32, device=self.device)
        if a.rows:
            if given and (out.data_ptr() != logits.data_ptr()
                          or (a.rows > 1 and out.stride(0) != a.ld)) and _overlap(logits, out):
                raise ValueError("out must be the logits themselves or not overlap them")
            nbytes = self.lib.vinfer_distill_workspace_bytes(a.rows, a.vocab, a.dtype, a.k)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            self._call(self.lib.vinfer_distill_step, "vinfer_distill_step", C.byref(a),
                       loss.data_ptr(), out.data_ptr(),
                       out.stride(0) if a.rows > 1 else a.vocab, ws.data_ptr(), nbytes)
        if given:  # whoever saved it for a backward pass learns that it changed
            torch.autograd.graph.increment_version(out)
        return loss, out

    def sample(self, logits: torch.Tensor, params: SamplingParams, seed: int,
               position: int) -> int:
        row = logits.reshape(1, -1)
        if row.dtype not in _DTYPES:
            row = row.float()
        rp = RowParams.pack([params], self.device)
        u = torch.tensor([position_uniform(seed, position)], dtype=torch.float32,
                         device=self.device)
        ids = self.sample_batch(row, rp, u)
        tok = int(ids[0])
        self.check()
        return tok

    def check(self) -> None:
        """Raise ``RuntimeError`` if a device-side problem was reported (synchronises)."""
        bits = int(self.status[0])
        if bits:
            self.status.zero_()
            raise RuntimeError(f"sampler: {_lib.status_message(bits)}")
