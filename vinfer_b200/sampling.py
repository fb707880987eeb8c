"""Sampling parameters, per-position seeds and the host-side packing of a batch.

``SamplingParams`` keeps every field, default and validation message of vinfer's
(``src/vinfer/runtime/sampler.py:18-41``) and adds the four the B200 sampler implements beyond
the reference: ``min_p`` and the repetition / presence / frequency penalties, all defaulting
to "off". ``position_seed`` is the reference's (``sampler.py:44-47``); the draw's uniform for
a position is derived from it with SplitMix64, so ``sample(logits, params, seed, position)``
is reproducible from ``(seed, position)`` alone, as in the reference.
"""

from __future__ import annotations

import bisect
import hashlib
from collections.abc import Sequence
from dataclasses import dataclass

import numpy as np
import torch

from vinfer_b200 import _lib


@dataclass(frozen=True)
class SamplingParams:
    max_tokens: int = 16
    temperature: float = 1.0  # 0 = greedy
    top_k: int = 0  # 0 = off
    top_p: float = 1.0  # 1 = off
    seed: int | None = None  # None: the runtime picks one per request
    stop: tuple[str, ...] = ()
    stop_token_ids: tuple[int, ...] = ()
    ignore_eos: bool = False
    # extensions (no counterpart in the reference)
    min_p: float = 0.0  # 0 = off
    repetition_penalty: float = 1.0  # 1 = off
    presence_penalty: float = 0.0  # 0 = off
    frequency_penalty: float = 0.0  # 0 = off

    def __post_init__(self) -> None:
        if self.temperature < 0:
            raise ValueError(f"temperature must be >= 0, got {self.temperature}")
        if not 0 < self.top_p <= 1:
            raise ValueError(f"top_p must be in (0, 1], got {self.top_p}")
        if self.top_k < 0:
            raise ValueError(f"top_k must be >= 0, got {self.top_k}")
        if self.max_tokens < 1:
            raise ValueError(f"max_tokens must be >= 1, got {self.max_tokens}")
        if not 0 <= self.min_p <= 1:
            raise ValueError(f"min_p must be in [0, 1], got {self.min_p}")
        if not self.repetition_penalty > 0:
            raise ValueError(f"repetition_penalty must be > 0, got {self.repetition_penalty}")

    @property
    def greedy(self) -> bool:
        return self.temperature == 0

    @property
    def penalized(self) -> bool:
        return (self.repetition_penalty != 1 or self.presence_penalty != 0
                or self.frequency_penalty != 0)


def position_seed(seed: int, position: int) -> int:
    """A 63-bit seed derived from ``(seed, position)`` (stable across runs and platforms)."""
    digest = hashlib.blake2b(f"{seed}:{position}".encode(), digest_size=8).digest()
    return int.from_bytes(digest, "little") & ((1 << 63) - 1)


_MASK64 = (1 << 64) - 1


def _splitmix64(state: int) -> int:
    """SplitMix64 (Steele, Lea & Flood, OOPSLA 2014), one output."""
    z = (state + 0x9E3779B97F4A7C15) & _MASK64
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _MASK64
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _MASK64
    return z ^ (z >> 31)


def position_uniform(seed: int, position: int) -> float:
    """The draw's uniform in ``[0, 1)`` for ``(seed, position)``: 24 bits, exact in float32."""
    return (_splitmix64(position_seed(seed, position)) >> 40) * (1.0 / (1 << 24))


@dataclass
class RowParams:
    """Per-row parameters as device arrays (struct of arrays), the layout the kernel reads."""

    temperature: torch.Tensor  # float32 [B]
    top_k: torch.Tensor  # int32 [B]
    top_p: torch.Tensor  # float32 [B]
    min_p: torch.Tensor  # float32 [B]
    repetition_penalty: torch.Tensor  # float32 [B]
    presence_penalty: torch.Tensor  # float32 [B]
    frequency_penalty: torch.Tensor  # float32 [B]

    @property
    def batch(self) -> int:
        return self.temperature.shape[0]

    @classmethod
    def pack(cls, params: Sequence[SamplingParams], device: torch.device | str) -> RowParams:
        f = np.array([[p.temperature, p.top_p, p.min_p, p.repetition_penalty,
                       p.presence_penalty, p.frequency_penalty] for p in params],
                     dtype=np.float32).reshape(len(params), 6)
        k = np.array([p.top_k for p in params], dtype=np.int32)
        ft = torch.from_numpy(f).to(device)
        return cls(ft[:, 0].contiguous(), torch.from_numpy(k).to(device), ft[:, 1].contiguous(),
                   ft[:, 2].contiguous(), ft[:, 3].contiguous(), ft[:, 4].contiguous(),
                   ft[:, 5].contiguous())

    @classmethod
    def from_arrays(cls, device: torch.device | str, **arrays: np.ndarray) -> RowParams:
        def f32(name: str, default: float, n: int) -> torch.Tensor:
            a = arrays.get(name)
            a = np.full(n, default, np.float32) if a is None else np.asarray(a, np.float32)
            return torch.from_numpy(np.ascontiguousarray(a)).to(device)

        n = len(arrays["temperature"])
        k = arrays.get("top_k")
        k = np.zeros(n, np.int32) if k is None else np.asarray(k, np.int32)
        return cls(f32("temperature", 1.0, n), torch.from_numpy(np.ascontiguousarray(k)).to(device),
                   f32("top_p", 1.0, n), f32("min_p", 0.0, n), f32("repetition_penalty", 1.0, n),
                   f32("presence_penalty", 0.0, n), f32("frequency_penalty", 0.0, n))


@dataclass
class TokenHistogram:
    """Per-row token counts in CSR form: ids strictly ascending within a row."""

    row_ptr: torch.Tensor  # int64 [B + 1]
    ids: torch.Tensor  # int32 [nnz]
    counts: torch.Tensor  # int32 [nnz]

    @classmethod
    def from_token_lists(cls, rows: Sequence[Sequence[int]],
                         device: torch.device | str) -> TokenHistogram:
        ptr = [0]
        ids: list[np.ndarray] = []
        cnts: list[np.ndarray] = []
        for toks in rows:
            u, c = np.unique(np.asarray(toks, dtype=np.int64), return_counts=True)
            ids.append(u.astype(np.int32))
            cnts.append(c.astype(np.int32))
            ptr.append(ptr[-1] + len(u))
        cat = (lambda xs: np.concatenate(xs) if xs else np.zeros(0, np.int32))
        return cls.from_csr(np.array(ptr, np.int64), cat(ids), cat(cnts), device)

    @classmethod
    def from_csr(cls, row_ptr: np.ndarray, ids: np.ndarray, counts: np.ndarray,
                 device: torch.device | str) -> TokenHistogram:
        row_ptr = np.asarray(row_ptr, np.int64)
        ids = np.asarray(ids, np.int32)
        for r in range(len(row_ptr) - 1):
            seg = ids[row_ptr[r]:row_ptr[r + 1]]
            if len(seg) > 1 and not np.all(seg[1:] > seg[:-1]):
                raise ValueError(f"histogram ids of row {r} must be strictly ascending")
        t = (lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(device))
        # a zero-length tensor still needs a valid device pointer for the C ABI
        if len(ids) == 0:
            ids, counts = np.zeros(1, np.int32), np.zeros(1, np.int32)
        return cls(t(row_ptr), t(ids), t(np.asarray(counts, np.int32)))


HIST_PAD_ID = 0x7FFFFFFF  # VINFER_HIST_PAD_ID


@dataclass
class SlotHistogram:
    """Per-slot token counts kept on the device across decode steps (``vinfer_hist_*``).

    Slot ``s`` owns entries ``[s * cap, (s + 1) * cap)`` of ``ids`` / ``counts``: its first
    ``lens[s]`` entries are its tokens (ids strictly ascending, counts > 0), the others padding
    (count 0, ids ascending above every vocabulary id). ``history`` is therefore a CSR
    ``TokenHistogram`` the sampler reads as it is, and the backend's ``append_tokens`` updates
    it in place from the ids a step sampled, without leaving the device. The slots play the
    role of vinfer's per-request state slots (``src/vinfer/state/pool.py:70-82``).
    """

    cap: int
    ids: torch.Tensor  # int32 [slots * cap]
    counts: torch.Tensor  # int32 [slots * cap]
    lens: torch.Tensor  # int32 [slots]
    row_ptr: torch.Tensor  # int64 [slots + 1], s * cap

    @property
    def slots(self) -> int:
        return self.lens.shape[0]

    @property
    def history(self) -> TokenHistogram:
        return TokenHistogram(self.row_ptr, self.ids, self.counts)

    @staticmethod
    def host_layout(rows: Sequence[Sequence[int]], cap: int
                    ) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
        """(ids, counts, lens) of the slotted layout for the given token lists, on the host."""
        if cap < 1:
            raise ValueError("cap must be at least 1")
        n = len(rows)
        pos = np.arange(cap, dtype=np.int64)
        pad = (HIST_PAD_ID - (cap - 1 - pos)).astype(np.int32)
        ids = np.tile(pad, n)
        counts = np.zeros(n * cap, np.int32)
        lens = np.zeros(n, np.int32)
        for s, toks in enumerate(rows):
            u, c = np.unique(np.asarray(toks, dtype=np.int64), return_counts=True)
            if len(u) > cap:
                raise ValueError(f"slot {s} has {len(u)} distinct tokens, more than cap {cap}")
            if len(u) and (u[0] < 0 or u[-1] >= HIST_PAD_ID - cap):
                raise ValueError(f"slot {s} has a token id outside the vocabulary range")
            ids[s * cap:s * cap + len(u)] = u
            counts[s * cap:s * cap + len(u)] = c
            lens[s] = len(u)
        return ids, counts, lens

    @classmethod
    def from_token_lists(cls, rows: Sequence[Sequence[int]], cap: int,
                         device: torch.device | str) -> SlotHistogram:
        ids, counts, lens = cls.host_layout(rows, cap)
        t = (lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(device))
        row_ptr = np.arange(len(rows) + 1, dtype=np.int64) * cap
        return cls(cap, t(ids), t(counts), t(lens), t(row_ptr))

    @classmethod
    def from_csr(cls, row_ptr: np.ndarray, ids: np.ndarray, counts: np.ndarray, cap: int,
                 device: torch.device | str) -> SlotHistogram:
        """Slots holding the rows of a CSR history (ids ascending within a row)."""
        row_ptr = np.asarray(row_ptr, np.int64)
        n = len(row_ptr) - 1
        lens = np.diff(row_ptr).astype(np.int32)
        if n and lens.max() > cap:
            raise ValueError(f"a row has {lens.max()} entries, more than cap {cap}")
        pos = np.arange(cap, dtype=np.int64)
        sid = np.tile((HIST_PAD_ID - (cap - 1 - pos)).astype(np.int32), n)
        sc = np.zeros(n * cap, np.int32)
        for r in range(n):
            a, b = row_ptr[r], row_ptr[r + 1]
            sid[r * cap:r * cap + (b - a)] = ids[a:b]
            sc[r * cap:r * cap + (b - a)] = counts[a:b]
        t = (lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(device))
        return cls(cap, t(sid), t(sc), t(lens), t(np.arange(n + 1, dtype=np.int64) * cap))

    def states(self) -> DecodeStates:
        """The slots' counts as decode states, for ``reorder_states``."""
        s, c = self.slots, self.cap
        return DecodeStates([self.ids.view(s, c), self.counts.view(s, c), self.lens.view(s, 1)])

    def to_counts(self) -> list[dict[int, int]]:
        """Each slot's {token: count}, read back to the host (synchronises)."""
        ids, counts, lens = (x.cpu().numpy() for x in (self.ids, self.counts, self.lens))
        out = []
        for s in range(self.slots):
            a = s * self.cap
            out.append({int(i): int(c) for i, c in zip(ids[a:a + lens[s]], counts[a:a + lens[s]])})
        return out


@dataclass
class BeamStep:
    """What one ``beam_select`` leaves on the device, for R requests of W beams."""

    scores: torch.Tensor  # float32 [R, n]: the best continuations' scores, descending; -inf: none
    beams: torch.Tensor  # int32 [R, n]: the beam each continues; -1: none
    tokens: torch.Tensor  # int32 [R, n]; -1: none
    next_scores: torch.Tensor  # float32 [R, W]: the score each slot goes on with; -inf: dead
    parents: torch.Tensor  # int32 [R, W]: the slot (r * W + beam) whose state each slot takes
    next_tokens: torch.Tensor  # int32 [R, W]: the token each slot appends; -1: none

    @classmethod
    def empty(cls, requests: int, width: int, n: int, device: torch.device | str) -> BeamStep:
        f = (lambda m: torch.empty(requests, m, dtype=torch.float32, device=device))
        i = (lambda m: torch.empty(requests, m, dtype=torch.int32, device=device))
        return cls(f(n), i(n), i(n), f(width), i(width), i(width))


class DecodeStates:
    """Tensors that hold one decode state for each slot, described once for ``reorder_states``.

    ``tensors`` share ``slot_dim``, the dimension that counts the slots (key/value caches
    ``[slots, heads, length, dim]``, recurrent states, token counts, in any strided layout
    without overlap). ``length_dim``, if given, is the dimension along which a call's ``lengths``
    say how many positions of a slot hold data. ``out`` are the tensors that receive the copies
    (same shapes and types, any strides; they share no element with each other or a state);
    without it slots are copied in place, and tensors may share bytes of the same slot alone. The
    tensors are
    held and their addresses used by every call: they are not to be resized meanwhile. They
    play the role of vinfer's per-request state slots (``src/vinfer/state/pool.py:70-131``).
    """

    def __init__(self, tensors: Sequence[torch.Tensor], slot_dim: int = 0,
                 length_dim: int | None = None,
                 out: Sequence[torch.Tensor] | None = None) -> None:
        self.tensors = list(tensors)
        self.out = self.tensors if out is None else list(out)
        if not self.tensors:
            raise ValueError("no states")
        if len(self.out) != len(self.tensors):
            raise ValueError(f"{len(self.out)} outputs for {len(self.tensors)} states")
        self.device = self.tensors[0].device
        self.has_lengths = length_dim is not None
        self.slots = self._dim(self.tensors[0], slot_dim, "slot_dim")[1]
        if not 1 <= self.slots <= _lib.STATE_MAX_SLOTS:
            raise ValueError(f"states must have 1 to {_lib.STATE_MAX_SLOTS} slots, got {self.slots}")
        found = []
        for i, (t, u) in enumerate(zip(self.tensors, self.out)):
            if t.device != self.device or u.device != self.device:
                raise ValueError(f"state {i} is not on {self.device}")
            if t.shape != u.shape or t.dtype != u.dtype:
                raise ValueError(f"output {i} must have the shape and type of its state")
            sd, n = self._dim(t, slot_dim, "slot_dim")
            if n != self.slots:
                raise ValueError(f"state {i} has {n} slots, the first {self.slots}")
            ld = None if length_dim is None else self._dim(t, length_dim, "length_dim")[0]
            if ld == sd:
                raise ValueError("length_dim must not be slot_dim")
            if out is not None and any(_overlap(v, u) for v in self.tensors):
                raise ValueError(f"output {i} overlaps a state")
            if out is not None and t.numel() and any(u.data_ptr() == v.data_ptr()
                                                     for v in self.out[:i] if v.numel()):
                raise ValueError(f"output {i} is given twice")
            if t.numel():
                found.append(_describe(i, t, u, sd, ld))
        for i, j in _close_pairs(self.out):
            if out is not None and _overlap(self.out[i], self.out[j]):
                raise ValueError(f"output {j} overlaps output {i}")
            if out is None and _overlap_across(self.out[i], self.out[j], slot_dim):
                raise ValueError(f"state {j} overlaps state {i}")
        # where slots are written: (first byte, behind the last), ascending, without overlap
        self.written: list[list[int]] = []
        for a, b in sorted((u.data_ptr(), u.data_ptr() + _extent(u)) for u in self.out if u.numel()):
            if self.written and a <= self.written[-1][1]:
                self.written[-1][1] = max(b, self.written[-1][1])
            else:
                self.written.append([a, b])
        self.count = len(found)
        self.in_place = all(d.src == d.dst for d in found)
        self.array = (_lib.State * max(1, self.count))(*found)

    def writes_to(self, a: int, b: int) -> bool:
        """Whether slots are written within the bytes [a, b)."""
        if not self.written or b <= self.written[0][0] or a >= self.written[-1][1]:
            return False
        i = bisect.bisect_left(self.written, [b])  # the spans that begin below b
        return i > 0 and self.written[i - 1][1] > a

    @staticmethod
    def _dim(t: torch.Tensor, dim: int, name: str) -> tuple[int, int]:
        if not -t.dim() <= dim < t.dim():
            raise ValueError(f"{name} {dim} is out of range for a state of {t.dim()} dimensions")
        return dim % t.dim(), t.shape[dim]


def _extent(t: torch.Tensor) -> int:
    """Bytes from a tensor's first element to behind its last."""
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _overlap(t: torch.Tensor, u: torch.Tensor) -> bool:
    """Whether two tensors share a byte (True also where finding out would take thousands of steps)."""
    if not t.numel() or not u.numel():
        return False
    a, b = t.data_ptr(), u.data_ptr()
    if a >= b + _extent(u) or b >= a + _extent(t):
        return False
    return _meet(b - a, *_nested(t), *_nested(u))


def _overlap_across(t: torch.Tensor, u: torch.Tensor, slot_dim: int) -> bool:
    """Whether a slot of one tensor shares a byte with another slot of the other. (The same slot's bytes
    are copied from the same place by both.)"""
    if not _overlap(t, u):
        return False
    step = t.stride(slot_dim) * t.element_size()
    if t.shape[slot_dim] > 1 and step != u.stride(slot_dim) * u.element_size():
        return True
    d = u.data_ptr() - t.data_ptr()
    a, b = _nested(t.select(slot_dim, 0)), _nested(u.select(slot_dim, 0))
    return any(_meet(d + k * step, *a, *b) or _meet(d - k * step, *a, *b)
               for k in range(1, t.shape[slot_dim]))


def _close_pairs(tensors: Sequence[torch.Tensor]) -> list[tuple[int, int]]:
    """The pairs (i < j) of tensors whose extents overlap."""
    spans = sorted((t.data_ptr(), t.data_ptr() + _extent(t), i) for i, t in enumerate(tensors)
                   if t.numel())
    pairs, open_ = [], []
    for a, b, j in spans:
        open_ = [(end, i) for end, i in open_ if end > a]
        pairs += [(min(i, j), max(i, j)) for _, i in open_]
        open_.append((b, j))
    return sorted(pairs)


def _nested(t: torch.Tensor) -> tuple[list[tuple[int, int]], int]:
    """A tensor's dimensions (size, stride in bytes), outermost first, over its contiguous run of
    bytes."""
    run, dims = t.element_size(), []
    for s, n in sorted((s * t.element_size(), n) for n, s in zip(t.shape, t.stride()) if n > 1 and s):
        if not dims and s == run:
            run *= n
        elif dims and s == dims[-1][0] * dims[-1][1]:
            dims[-1] = (dims[-1][0] * n, dims[-1][1])
        else:
            dims.append((n, s))
    return dims[::-1], run


def _meet(d: int, a: list[tuple[int, int]], ra: int, b: list[tuple[int, int]], rb: int) -> bool:
    """Whether two tensors, the second's first byte d behind the first's, share a byte. Where strides
    nest, no more than a few places of the outermost dimension can, each decided by what is inside."""
    ea = ra + sum((n - 1) * s for n, s in a)
    eb = rb + sum((n - 1) * s for n, s in b)
    if d >= ea or -d >= eb:
        return False
    if not a and not b:
        return True
    if a and b and a[0][1] == b[0][1]:  # only the difference of the two places matters
        (n, s), m = a[0], b[0][0]
        ia, ib = ea - (n - 1) * s, eb - (m - 1) * s
        lo, hi = max(-(n - 1), -((ib - 1 + d) // s)), min(m - 1, (ia - 1 - d) // s)
        inside = (a[1:], ra, b[1:], rb)
    elif a and (not b or a[0][1] > b[0][1]):
        n, s = a[0]
        ia = ea - (n - 1) * s
        lo, hi = max(-(n - 1), -((d + eb - 1) // s)), min(0, (ia - 1 - d) // s)
        inside = (a[1:], ra, b, rb)
    else:
        m, s = b[0]
        ib = eb - (m - 1) * s
        lo, hi = max(0, -((ib - 1 + d) // s)), min(m - 1, (ea - 1 - d) // s)
        inside = (a, ra, b[1:], rb)
    if hi - lo >= 4096:
        return True
    return any(_meet(d + k * s, *inside) for k in range(lo, hi + 1))


def _describe(i: int, t: torch.Tensor, u: torch.Tensor, slot_dim: int,
              length_dim: int | None) -> _lib.State:
    """A state as contiguous runs under outer dimensions (``VinferState``)."""
    es = t.element_size()
    for x in (t, u):  # dimensions nest: each stride steps over all that is inside it
        inside = es
        for n, s in sorted(((n, s * es) for n, s in zip(x.shape, x.stride()) if n > 1),
                           key=lambda d: d[1]):
            if s < inside:
                raise ValueError(f"state {i} overlaps itself (shape {tuple(x.shape)}, strides "
                                 f"{tuple(x.stride())})")
            inside += (n - 1) * s
    dims = [(t.stride(d) * es, u.stride(d) * es, t.shape[d], d == length_dim)
            for d in range(t.dim()) if d != slot_dim and (t.shape[d] > 1 or d == length_dim)]
    dims.sort(key=lambda d: d[0] if d[2] > 1 else 0)  # innermost first
    run, unit = es, 0
    while dims and not unit and (dims[0][2] == 1 or dims[0][0] == dims[0][1] == run):
        _, _, n, is_len = dims.pop(0)
        if is_len:
            unit = run
        run *= n
    outer: list[list] = []  # innermost first
    for a, b, n, is_len in dims:
        if outer and not is_len and not outer[-1][3] and a == outer[-1][0] * outer[-1][2] \
                and b == outer[-1][1] * outer[-1][2]:
            outer[-1][2] *= n
        else:
            outer.append([a, b, n, is_len])
    if len(outer) > _lib.STATE_MAX_OUTER:
        raise ValueError(f"state {i} is too scattered (shape {tuple(t.shape)}, strides "
                         f"{tuple(t.stride())})")
    outer.reverse()
    d = _lib.State()
    d.src, d.dst = t.data_ptr(), u.data_ptr()
    d.src_slot_stride, d.dst_slot_stride = t.stride(slot_dim) * es, u.stride(slot_dim) * es
    d.run_bytes, d.len_unit_bytes = run, unit
    d.len_outer, d.n_outer = -1, len(outer)
    for k, (a, b, n, is_len) in enumerate(outer):
        d.outer_size[k], d.src_outer_stride[k], d.dst_outer_stride[k] = n, a, b
        if is_len:
            d.len_outer = k
    return d
