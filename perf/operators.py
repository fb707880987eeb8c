"""The operators beside the sampler that are timed: their cases, inputs, plain forms and definitions.

* ``beam``: one step of beam search. For each request with ``width`` beams (rows of logits and
  the beams' accumulated log-probabilities): the ``n`` best continuations over beams and
  vocabulary, and the beams that go on, laid into the request's slots.
* ``reorder``: every decode state (histories, recurrent states, key/value caches) follows the
  beams: slot ``s`` takes the state of slot ``parents[s]``.
* ``distill``: distillation from a teacher's top log-probabilities: the loss of each row
  (``form`` "loss"), loss and gradient through autograd ("train"), and both in one call with the
  rows' weights known ahead ("step").

``run`` computes the plain forms with elementary torch operations where ``own`` is false, and
makes the framework's calls where it is true.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
NEG = float("-inf")
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
ID_BITS = 18  # token ids of every case fit 18 bits


# ---- cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # one chat request decoded with four beams: latency counts
        dict(name="beam one request", op="beam", requests=1, width=4, vocab=151936, n=8, eos=1,
             dtype="bf16", pad=0, first=False),
        # a full decode batch of 256 rows
        dict(name="beam batch", op="beam", requests=64, width=4, vocab=151936, n=8, eos=1,
             dtype="bf16", pad=0, first=False),
        # the first step of small odd requests: one live beam each, padded rows, two stop ids
        dict(name="beam first odd", op="beam", requests=37, width=5, vocab=40001, n=15, eos=2,
             dtype="f32", pad=3, first=True),
        # wide beams over the larger vocabulary in float32
        dict(name="beam wide", op="beam", requests=32, width=16, vocab=248320, n=32, eos=1,
             dtype="f32", pad=0, first=False),
        # the decode slots' token counts: three small arrays
        dict(name="reorder counts", op="reorder", kind="counts", requests=16, width=4, moved=2,
             layers=1, heads=1, length=2048, dim=1, dtype="bf16"),
        # recurrent layers: a float32 matrix state and a short convolution state for each layer
        dict(name="reorder recurrent", op="reorder", kind="recurrent", requests=8, width=4,
             moved=2, layers=6, heads=32, length=128, dim=128, dtype="bf16"),
        # key/value caches of a decode batch with ragged lengths
        dict(name="reorder cache", op="reorder", kind="cache", requests=16, width=4, moved=2,
             layers=8, heads=8, length=1024, dim=128, dtype="bf16"),
        # a small odd vocabulary, losses only (validation)
        dict(name="distill loss odd", op="distill", form="loss", rows=33, vocab=4097, k=7,
             dtype="f32", tail=True, temperature=1.5, masked=2),
        # validation of a batch over the whole vocabulary
        dict(name="distill loss", op="distill", form="loss", rows=1024, vocab=151936, k=20,
             dtype="bf16", tail=False, temperature=1.0, masked=0),
        # fine-tuning of a student on recorded top-20 lists
        dict(name="distill train", op="distill", form="train", rows=256, vocab=151936, k=20,
             dtype="bf16", tail=False, temperature=1.0, masked=16),
        # a full training step with the prompt's rows masked and the tail's mass matched
        dict(name="distill step", op="distill", form="step", rows=4096, vocab=151936, k=32,
             dtype="bf16", tail=True, temperature=2.0, masked=512),
        # float32 logits over the larger vocabulary, long lists
        dict(name="distill step f32", op="distill", form="step", rows=512, vocab=248320, k=128,
             dtype="f32", tail=True, temperature=1.0, masked=0),
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["beam", "reorder", "distill"])
    if op == "beam":
        width = rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 32])
        vocab = _log(rng, 1000, 248320)
        eos = rng.randint(0, 2)
        dtype = rng.choice(["bf16", "f32"])
        most = max(1, min(512 * 248320 * 4 // (width * vocab * (2 if dtype == "bf16" else 4)),
                          1024 // width))
        return dict(op=op, requests=_log(rng, 1, most), width=width, vocab=vocab,
                    n=rng.randint(width, min(128, width * (1 + eos) + 4)), eos=eos, dtype=dtype,
                    pad=rng.choice([0, 0, 1, 8]), first=rng.random() < 0.25)
    if op == "reorder":
        kind = rng.choice(["counts", "recurrent", "cache"])
        width = rng.randint(2, 16)
        case = dict(op=op, kind=kind, requests=_log(rng, 1, 256 // width), width=width,
                    moved=rng.randint(1, width - 1), layers=1, heads=1, length=1, dim=1,
                    dtype=rng.choice(["bf16", "f32"]))
        if kind == "counts":
            case["length"] = _log(rng, 16, 4096)
        elif kind == "recurrent":
            case.update(layers=rng.randint(1, 6), heads=_log(rng, 1, 32),
                        length=rng.choice([64, 96, 128]), dim=rng.choice([64, 100, 128]))
        else:
            case.update(layers=rng.randint(1, 4), heads=rng.choice([1, 2, 4, 8]),
                        length=_log(rng, 16, 512), dim=rng.choice([64, 80, 128, 256]))
        slots = case["requests"] * width
        while slots * case["layers"] * case["heads"] * case["length"] * case["dim"] > 1 << 27:
            case["heads"], case["layers"] = max(1, case["heads"] // 2), max(1, case["layers"] // 2)
            if case["heads"] == 1 and case["layers"] == 1:
                break
        return case
    vocab = _log(rng, 500, 248320)
    rows = _log(rng, 1, max(1, min(4096, 400_000_000 // vocab)))
    return dict(op=op, form=rng.choice(["loss", "train", "step"]), rows=rows, vocab=vocab,
                k=_log(rng, 1, 128), dtype=rng.choice(["bf16", "f32"]),
                tail=rng.random() < 0.5, temperature=rng.choice([1.0, 1.5, 2.0, 4.0]),
                masked=rng.randint(0, rows // 4))


# ---- work ----------------------------------------------------------------------------------------
def _size(dtype):
    return 2 if dtype == "bf16" else 4


def work(case):
    c = case
    if c["op"] == "beam":
        live = c["requests"] * (1 if c["first"] else c["width"])
        elements = live * c["vocab"]
        small = c["requests"] * (c["width"] * 16 + c["n"] * 12)
        # a comparison, a subtraction, an exponential and a sum for each element
        return {"bytes": elements * _size(c["dtype"]) + small, "flops": 4 * elements}
    if c["op"] == "reorder":
        sources = min(c["moved"], c["width"] - c["moved"])
        rows = c["requests"] * (sources + c["moved"])  # rows read and rows written
        if c["kind"] == "counts":
            row = c["length"] * 8 + 4
        elif c["kind"] == "recurrent":
            row = c["layers"] * (c["heads"] * c["length"] * c["dim"] * 4
                                 + c["heads"] * c["dim"] * 3 * _size(c["dtype"]))
        else:
            mean = sum(_lengths(c)) / c["requests"]
            row = 2 * c["layers"] * c["heads"] * mean * c["dim"] * _size(c["dtype"])
        return {"bytes": rows * row + 4 * c["requests"] * c["width"], "flops": 0}
    rows = c["rows"] - c["masked"]
    read = rows * c["vocab"] * _size(c["dtype"]) + c["rows"] * (8 * c["k"] + 8)
    if c["form"] == "loss":
        return {"bytes": read, "flops": 4 * rows * c["vocab"]}
    write = c["rows"] * c["vocab"] * _size(c["dtype"])
    return {"bytes": read + write, "flops": 7 * rows * c["vocab"]}


def _lengths(c):
    """Cache lengths of the requests, spread evenly up to the longest."""
    r = c["requests"]
    return [max(1, c["length"] * (i + 1) // r) for i in range(r)]


# ---- inputs --------------------------------------------------------------------------------------
def _backend(dtype):
    from vinfer_b200 import SAMPLER, BackendContext

    return SAMPLER.resolve("b200", BackendContext(torch.device(DEV, 0), dtype))


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    s = {"beam": _prepare_beam, "reorder": _prepare_reorder,
         "distill": _prepare_distill}[case["op"]](case, g)
    s["case"] = dict(case)
    if own:
        s["backend"] = _backend(DTYPES[case["dtype"]])
        if case["op"] == "reorder":  # the states are described once, as their program holds them
            from vinfer_b200.sampling import DecodeStates

            s["handle"] = DecodeStates(s["states"], length_dim=s["length_dim"])
    return s


def _logits(g, rows, vocab, dtype):
    """Normal logits with a spread of their own for each row and sixteen raised tokens."""
    sigma = torch.rand(rows, 1, generator=g, device=DEV) * 2 + 1
    x = torch.randn(rows, vocab, generator=g, device=DEV) * sigma
    at = torch.randint(vocab, (rows, 16), generator=g, device=DEV)
    up = torch.rand(rows, 16, generator=g, device=DEV) * 7 + 5
    return x.scatter_add_(1, at, up).to(dtype)


def _prepare_beam(c, g):
    rows = c["requests"] * c["width"]
    x = _logits(g, rows, c["vocab"], DTYPES[c["dtype"]])
    eos = torch.randperm(c["vocab"], generator=g, device=DEV)[:c["eos"]].to(torch.int32)
    if c["eos"]:  # about a third of the beams are ready to end
        ends = torch.rand(rows, generator=g, device=DEV) < 0.35
        x[:, eos[0]] = torch.where(ends, x.amax(1), x[:, eos[0]])
    if c["pad"]:
        wide = torch.zeros(rows, c["vocab"] + c["pad"], dtype=x.dtype, device=DEV)
        wide[:, :c["vocab"]] = x
        x = wide[:, :c["vocab"]]
    scores = -4 * torch.rand(c["requests"], c["width"], generator=g, device=DEV) - 6
    if c["first"]:
        scores[:, 0] = 0.0
        scores[:, 1:] = NEG
    return {"logits": x, "scores": scores, "eos": eos}


def _prepare_reorder(c, g):
    r, w = c["requests"], c["width"]
    keep = w - c["moved"]
    # in each request `keep` beams stay; the others take over a survivor's state, in turn
    order = torch.rand(r, w, generator=g, device=DEV).argsort(1)
    parents = torch.arange(w, device=DEV).repeat(r, 1)
    source = order[:, :keep][:, torch.arange(c["moved"], device=DEV) % keep]
    parents.scatter_(1, order[:, keep:], source)
    parents = (parents + torch.arange(r, device=DEV)[:, None] * w).reshape(-1).to(torch.int32)
    slots, dt = r * w, DTYPES[c["dtype"]]
    lengths = None
    if c["kind"] == "counts":
        states = [torch.randint(1 << 17, (slots, c["length"]), generator=g, device=DEV,
                                dtype=torch.int32),
                  torch.randint(9, (slots, c["length"]), generator=g, device=DEV,
                                dtype=torch.int32),
                  torch.randint(c["length"] + 1, (slots, 1), generator=g, device=DEV,
                                dtype=torch.int32)]
    elif c["kind"] == "recurrent":
        states = [torch.randn(slots, c["heads"], c["length"], c["dim"], generator=g, device=DEV)
                  for _ in range(c["layers"])]
        states += [torch.randn(slots, c["heads"] * c["dim"], 3, generator=g, device=DEV).to(dt)
                   for _ in range(c["layers"])]
    else:
        states = [torch.randn(slots, c["heads"], c["length"], c["dim"], generator=g,
                              device=DEV).to(dt) for _ in range(2 * c["layers"])]
        mixed = torch.randperm(r, generator=g, device=DEV)
        lengths = torch.tensor(_lengths(c), device=DEV)[mixed].repeat_interleave(w).to(torch.int32)
    return {"states": states, "parents": parents, "lengths": lengths,
            "length_dim": None if lengths is None else 2}


def _prepare_distill(c, g):
    n, k = c["rows"], c["k"]
    x = _logits(g, n, c["vocab"], torch.float32)
    t = x + 0.5 * torch.randn(n, c["vocab"], generator=g, device=DEV)
    t.div_(c["temperature"])
    top, ids = t.topk(k, dim=1)
    lp = top - torch.logsumexp(t, 1, keepdim=True)
    del t
    # lists of different lengths: a teacher cut by top-p records fewer tokens
    held = torch.randint((k + 1) // 2, k + 1, (n, 1), generator=g, device=DEV)
    gone = torch.arange(k, device=DEV) >= held
    ids = torch.where(gone, -1, ids).to(torch.int32)
    lp = torch.where(gone, NEG, lp)
    weights = torch.full((n,), 1.0 / (n - c["masked"]), device=DEV)
    weights[torch.randperm(n, generator=g, device=DEV)[:c["masked"]]] = 0.0
    return {"logits": x.to(DTYPES[c["dtype"]]), "ids": ids, "logprobs": lp, "weights": weights}


# ---- one pass ------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    return {"beam": _run_beam, "reorder": _run_reorder, "distill": _run_distill}[c["op"]](state, c)


def _run_beam(s, c):
    if own:
        b = s["backend"].beam_select(s["logits"], s["scores"], c["n"], eos=s["eos"])
        return {"scores": b.scores, "beams": b.beams, "tokens": b.tokens,
                "next_scores": b.next_scores, "parents": b.parents, "next_tokens": b.next_tokens}
    return _plain_beam(s["logits"], s["scores"], c["n"], s["eos"])


def _run_reorder(s, c):
    if own:
        s["backend"].reorder_states(s["handle"], s["parents"], s["lengths"])
        return s["states"]
    parents, lengths = s["parents"].long(), s["lengths"]
    if lengths is None:
        return [t.copy_(t[parents]) for t in s["states"]]
    live = (torch.arange(c["length"], device=DEV) < lengths[:, None])[:, None, :, None]
    return [t.copy_(torch.where(live, t[parents], t)) for t in s["states"]]


def _run_distill(s, c):
    if own:
        from vinfer_b200.distill import distillation_loss

        if c["form"] == "step":
            loss, grad = s["backend"].distill_step(s["logits"], s["ids"], s["logprobs"],
                                                   s["weights"], temperature=c["temperature"],
                                                   tail=c["tail"])
            return {"loss": loss, "grad": grad}
        x = s["logits"].detach().requires_grad_(c["form"] == "train")
        loss = distillation_loss(s["backend"], x, s["ids"], s["logprobs"], s["weights"],
                                 temperature=c["temperature"], tail=c["tail"])
        if c["form"] == "loss":
            return {"loss": loss}
        (grad,) = torch.autograd.grad(loss.sum(), x)
        return {"loss": loss.detach(), "grad": grad}
    return _plain_distill(s["logits"], s["ids"], s["logprobs"], s["weights"], c["temperature"],
                          c["tail"], c["form"] != "loss")


# ---- plain forms ---------------------------------------------------------------------------------
def _plain_beam(logits, scores, n, eos):
    """Scores in 64 bits: where two beams' continuations are close, 32 would order them by
    their rounding."""
    r, w = scores.shape
    v = logits.shape[1]
    k = min(n, v)
    x = logits.float()
    m = x.amax(1, keepdim=True)
    lse = m.double() + torch.exp((x - m).double()).sum(1, keepdim=True).log()
    # each row's k best tokens, equal logits by ascending id: unique 64-bit keys
    bits = x.view(torch.int32) if x.is_contiguous() else x.contiguous().view(torch.int32)
    bits = bits.long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) << ID_BITS
    key += (1 << ID_BITS) - 1 - torch.arange(v, device=x.device)
    ids = (1 << ID_BITS) - 1 - (key.topk(k, dim=1).values & ((1 << ID_BITS) - 1))
    total = scores.double().reshape(-1, 1) + (x.gather(1, ids).double() - lse)
    # over the beams of a request, ties by beam, then token: the rows are in that order
    tok, order = ids.sort(1)
    total = total.gather(1, order).reshape(r, w * k)
    best, at = total.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    if best.shape[1] < n:
        best = torch.cat([best, best.new_full((r, n - best.shape[1]), NEG)], 1)
        at = torch.cat([at, at.new_zeros(r, n - at.shape[1])], 1)
    none = best == NEG
    beams = torch.where(none, -1, at // k)
    tokens = torch.where(none, -1, tok.reshape(r, w * k).gather(1, at))
    # the first w candidates that do not end a sequence go on
    ends = (tokens[:, :, None] == eos.long()).any(2) if eos.numel() else torch.zeros_like(none)
    on = ~none & ~ends
    rank = on.cumsum(1) - 1
    on &= rank < w
    # the best child of a beam stays in its slot, the others fill the free slots in turn
    slot = torch.arange(w, device=x.device)
    mine = on[:, :, None] & (beams[:, :, None] == slot)  # [r, n, w]
    kept = mine.any(1)
    head = on & (mine & (mine.cumsum(1) == 1)).any(2)
    extra = on & ~head
    nth = extra.cumsum(1) - 1
    free = (kept.int() * w + slot).argsort(1)  # the free slots first, ascending
    to = torch.where(head, beams, free.gather(1, nth.clamp(0, w - 1)))
    to = torch.where(on, to, w)  # a place behind the slots for candidates that go nowhere
    base = torch.arange(r, device=x.device)[:, None] * w
    parents = (base + slot).new_empty(r, w + 1)
    parents[:, :w] = base + slot
    parents.scatter_(1, to, base + beams.clamp(min=0))
    next_scores = best.new_full((r, w + 1), NEG).scatter_(1, to, best)
    next_tokens = tokens.new_full((r, w + 1), -1).scatter_(1, to, tokens)
    return {"scores": best.float(), "beams": beams.int(), "tokens": tokens.int(),
            "next_scores": next_scores[:, :w].float(),
            "parents": parents[:, :w].int(), "next_tokens": next_tokens[:, :w].int()}


def _plain_distill(logits, ids, lp, weights, temperature, tail, with_grad):
    """The rows of the vocabulary in 32 bits; the terms of the list and the sums in 64: where
    nearly all mass is in the tail, its share is one less a small sum."""
    z = logits.float() / temperature
    held = ids >= 0
    at = torch.where(held, ids, ids[:, :1]).long()  # every row lists a token first
    p = torch.where(held, lp.double().exp(), 0.0)
    if not tail:
        p = p / p.sum(1, keepdim=True)
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    logq = (z.gather(1, at) - m).double() - total.log()
    term = torch.where(p > 0, p * (p.log() - logq), 0.0)
    loss = term.sum(1)
    scale = torch.ones_like(total)
    if tail:
        rest = e.scatter(1, at, 0.0).sum(1, keepdim=True, dtype=torch.float64)
        mass = (1 - p.sum(1, keepdim=True)).clamp(min=0)
        part = rest / total
        loss = loss + torch.where(mass > 0, mass * (mass.log() - part.log()), 0.0)[:, 0]
        scale = 1 - mass / part
    loss = torch.where(weights != 0, loss * weights, 0.0).float()
    if not with_grad:
        return {"loss": loss}
    w = (weights / temperature)[:, None]
    grad = e * ((scale / total) * w).float()
    grad.scatter_(1, at, (logq.exp() * w).float())
    grad.scatter_add_(1, at, (-p * w).float())
    return {"loss": loss, "grad": grad.to(logits.dtype)}


# ---- definitions in 64 bits ----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "reorder":
        return None  # copies: there is nothing to round
    if c["op"] == "beam":
        return _exact_beam(s, c)
    return _exact_distill(s, c)


def _exact_beam(s, c):
    best, nxt = [], []
    stops = set(s["eos"].tolist())
    for i in range(c["requests"]):
        x = s["logits"][i * c["width"]:(i + 1) * c["width"]].double()
        total = (torch.log_softmax(x, 1) + s["scores"][i].double()[:, None]).reshape(-1)
        v, at = total.sort(descending=True, stable=True)
        v, at = v[:c["n"]].tolist(), at[:c["n"]].tolist()
        best.append(v + [NEG] * (c["n"] - len(v)))
        # the continuing candidates: first child in place, the others into the free slots
        on = [(a, q // c["vocab"]) for a, q in zip(v, at)
              if a > NEG and q % c["vocab"] not in stops][:c["width"]]
        slots = [NEG] * c["width"]
        used, late = set(), []
        for a, b in on:
            if b in used:
                late.append(a)
            else:
                used.add(b)
                slots[b] = a
        for b, a in zip([b for b in range(c["width"]) if b not in used], late):
            slots[b] = a
        nxt.append(slots)
    as64 = lambda v: torch.tensor(v, dtype=torch.float64, device=DEV)  # noqa: E731
    return {"scores": as64(best), "beams": None, "tokens": None, "next_scores": as64(nxt),
            "parents": None, "next_tokens": None}


def _exact_distill(s, c):
    losses, grads = [], []
    step = max(1, (1 << 26) // c["vocab"])
    for a in range(0, c["rows"], step):
        x = s["logits"][a:a + step].double().requires_grad_(True)
        ids, lp = s["ids"][a:a + step].long(), s["logprobs"][a:a + step].double()
        logq = torch.log_softmax(x / c["temperature"], 1)
        target = torch.zeros_like(logq).scatter_add_(1, ids.clamp(min=0),
                                                     torch.where(ids >= 0, lp.exp(), 0.0))
        listed_ = torch.zeros_like(logq, dtype=torch.int32).scatter_add_(
            1, ids.clamp(min=0), (ids >= 0).int()) > 0
        if not c["tail"]:
            target = target / target.sum(1, keepdim=True)
        loss = torch.special.entr(target).neg().sum(1) - (target * logq).sum(1)
        if c["tail"]:
            mass = (1 - target.sum(1)).clamp(min=0)
            rest = torch.logsumexp(logq.masked_fill(listed_, NEG), 1)
            loss = loss - torch.special.entr(mass) - mass * rest
        loss = loss * s["weights"][a:a + step].double()
        losses.append(loss.detach())
        if c["form"] != "loss":
            (grad,) = torch.autograd.grad(loss.sum(), x)
            grads.append(grad)
    out = {"loss": torch.cat(losses)}
    if grads:
        out["grad"] = torch.cat(grads)
    return out
