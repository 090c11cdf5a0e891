"""Exact statement of the verification of drafted tokens, in Python integers.  Test infrastructure only.

Row distributions are those of the sampling oracle (oracle/ka_oracle.c: scaled values, top-k with ties, top-p on integer
masses, ties by ascending index); acceptance and the draw are evaluated on rationals.
"""
from __future__ import annotations

import math
from fractions import Fraction

import torch

from oracle import exact


def row_masses(row: torch.Tensor, temperature: float = 1.0, top_k=None, top_p=None) -> list:
    """Integer mass of every entry of one row (0: filtered out)."""
    y = exact.scale(row.reshape(1, -1), temperature).reshape(-1)
    y = torch.where(torch.isnan(y), torch.full_like(y, -math.inf), y)
    top = y.max().item()
    values = y.tolist()
    cache = {v: exact.weight(0.0 if v == top else float(torch.tensor(v) - torch.tensor(top))) for v in set(values)}
    w = [cache[v] for v in values]
    n = len(w)
    keep = list(range(n))
    if top_k and 0 < top_k < n:
        kth = sorted(values, reverse=True)[top_k - 1]
        keep = [i for i in keep if values[i] >= kth]
    if top_p is not None and top_p < 1.0:
        keep.sort(key=lambda i: (-values[i], i))
        theta = exact.floor_scale(float(torch.tensor(top_p, dtype=torch.float32)), sum(w[i] for i in keep))
        before, kept = 0, []
        for i in keep:
            if before > theta:
                break
            kept.append(i)
            before += w[i]
        keep = kept
    out = [0] * n
    for i in keep:
        out[i] = w[i]
    return out


def _uniform(u: float) -> Fraction:
    u = float(torch.tensor(u, dtype=torch.float32))
    if not u >= 0.0:
        return Fraction(0)
    return Fraction(min(u, 1.0 - 2.0 ** -24))


def _value(v, b, default):
    if v is None:
        return default
    return v[b].item() if isinstance(v, torch.Tensor) else v


def verify(target, draft_ids, uniforms, draft_logits=None, draft_lens=None, temperature=1.0, top_k=None, top_p=None):
    """(ids [B, K + 1], accepted [B], log-probability of every emitted token under the unfiltered target row, float64)."""
    target = target.detach().cpu()
    batch, positions, vocab = target.shape
    k = positions - 1
    out = torch.full((batch, k + 1), -1, dtype=torch.int64)
    accepted = torch.zeros(batch, dtype=torch.int64)
    logp = torch.zeros(batch, k + 1, dtype=torch.float64)
    for b in range(batch):
        t, kk, pp = _value(temperature, b, 1.0), _value(top_k, b, 0), _value(top_p, b, 1.0)
        t = float(torch.tensor(t, dtype=torch.float32))
        t = t if t > 0.0 else 1.0
        kk = kk if kk > 0 else 0
        pp = pp if 0.0 < pp <= 1.0 else 1.0
        length = k if draft_lens is None else max(0, min(k, int(draft_lens[b])))
        n = 0
        while True:
            wp = row_masses(target[b, n], t, kk, pp)
            if n == length:
                left = wp
                break
            d = int(draft_ids[b, n])
            if draft_logits is None:
                wq = [0] * vocab
                if 0 <= d < vocab:
                    wq[d] = 1
                zq = 1
            else:
                wq = row_masses(draft_logits[b, n].detach().cpu(), t, kk, pp)
                zq = sum(wq)
            zp = sum(wp)
            p_d = Fraction(wp[d], zp) if 0 <= d < vocab else Fraction(0)
            q_d = Fraction(wq[d], zq) if 0 <= d < vocab else Fraction(1 if draft_logits is None else 0)
            if _uniform(float(uniforms[b, n])) * q_d < p_d:
                out[b, n] = d
                n += 1
                continue
            if draft_logits is None:
                left = [0 if i == d else m for i, m in enumerate(wp)]
            else:
                left = [max(a * zq - c * zp, 0) for a, c in zip(wp, wq)]
            if not any(left):  # P = Q and a draft that Q cannot have drawn
                left = wp
            break
        tau = math.floor(_uniform(float(uniforms[b, k])) * sum(left))
        upto = 0
        for i, m in enumerate(left):
            upto += m
            if upto > tau:
                out[b, n] = i
                break
        accepted[b] = n
        rows = target[b, :n + 1].double()
        rows = torch.where(torch.isnan(rows), torch.full_like(rows, math.nan), rows)
        logp[b, :n + 1] = rows.gather(1, out[b, :n + 1].clamp(min=0).unsqueeze(1)).squeeze(1) - torch.logsumexp(rows, 1)
    return out, accepted, logp
