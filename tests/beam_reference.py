"""Plain 64-bit forms of the operators beside the sampler, on the host."""

from __future__ import annotations

import numpy as np


def log_sums(x: np.ndarray) -> np.ndarray:
    """ln sum exp of each row (float64); -inf for a row of -inf, NaN where a NaN or +inf is."""
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(axis=1)
        m = np.where(np.isfinite(m), m, 0.0)
        return m + np.log(np.exp(x - m[:, None]).sum(axis=1))


def beam_step(x: np.ndarray, scores: np.ndarray, n: int, eos: list[int]) -> dict:
    """One beam step: ``x`` float64 [R * W, V], ``scores`` [R, W]."""
    R, W = scores.shape
    lse = log_sums(x)
    out = {"scores": np.full((R, n), -np.inf), "beams": np.full((R, n), -1),
           "tokens": np.full((R, n), -1), "next_scores": np.full((R, W), -np.inf),
           "parents": np.arange(R * W).reshape(R, W).copy(), "next_tokens": np.full((R, W), -1)}
    for r in range(R):
        s, b, t = [], [], []
        for w in range(W):
            row = r * W + w
            if not np.isfinite(scores[r, w]) or not np.isfinite(lse[row]):
                continue
            ids = np.argsort(-x[row], kind="stable")[:n]  # descending, ties by id
            ids = ids[x[row, ids] > -np.inf]
            s += list(float(scores[r, w]) + (x[row, ids] - lse[row]))
            b += [w] * len(ids)
            t += list(ids)
        order = np.lexsort((t, b, -np.array(s)))[:n] if s else []
        for i, j in enumerate(order):
            out["scores"][r, i], out["beams"][r, i], out["tokens"][r, i] = s[j], b[j], t[j]
        on = [j for j in order if t[j] not in eos][:W]
        slot, late = {}, []
        for j in on:
            if b[j] in slot:
                late.append(j)
            else:
                slot[b[j]] = j
        for w, j in zip([w for w in range(W) if w not in slot], late):
            slot[w] = j
        for w, j in slot.items():
            out["next_scores"][r, w], out["next_tokens"][r, w] = s[j], t[j]
            out["parents"][r, w] = r * W + b[j]
    return out


def distill(x: np.ndarray, ids: np.ndarray, lp: np.ndarray, weights: np.ndarray,
            temperature: float, tail: bool) -> tuple[np.ndarray, np.ndarray]:
    """Losses [N] and the gradient of their sum [N, V], from the formulas, row by row."""
    N, V = x.shape
    loss, grad = np.zeros(N), np.zeros((N, V))
    for r in range(N):
        if weights[r] == 0:
            continue
        held = ids[r] >= 0
        p = np.where(held, np.exp(lp[r]), 0.0)
        if not tail:
            if p.sum() == 0:
                continue
            p = p / p.sum()
        z = x[r] / temperature
        logq = z - log_sums(z[None])[0]
        target = np.zeros(V)
        np.add.at(target, ids[r][held], p[held])
        inside = np.zeros(V, bool)
        inside[ids[r][held]] = True
        with np.errstate(divide="ignore", invalid="ignore"):
            lnp = lp[r] - (0.0 if tail else np.log(np.exp(lp[r][held]).sum()))
            terms = p * (lnp - logq[np.where(held, ids[r], 0)])
        total = terms[p > 0].sum()
        q = np.exp(logq)
        mass = p.sum()
        g = q.copy()
        if tail and not inside.all():
            pt = max(0.0, 1.0 - mass)
            rest = log_sums(logq[~inside][None])[0]
            with np.errstate(divide="ignore", over="ignore"):
                if pt > 0:
                    total += pt * (np.log(pt) - rest)
                M = mass + pt
                if rest > -np.inf:
                    g[~inside] = np.exp(logq[~inside] - rest) * (M * np.exp(rest) - pt)
        else:
            M = mass
            g[~inside] *= M
        g[inside] = M * q[inside] - target[inside]
        loss[r] = weights[r] * total
        grad[r] = weights[r] * g / temperature
    return loss, grad
