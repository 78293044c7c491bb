"""CPU oracle of the distillation loss in float64, row by row from its definition, with padding, repeated entries, the rest
bucket and infinite logits as distill.py documents them."""
import math

import torch


def row(z, idx, t, tau, lse=None):
    """(loss, d loss / d z) of one row: z [V] float64, idx and t lists of the teacher's entries."""
    V = z.numel()
    zero = torch.zeros(V, dtype=torch.float64)
    ent = [(int(j), float(v)) for j, v in zip(idx, t) if 0 <= int(j) < V and float(v) != -math.inf]
    if not ent:
        return 0.0, zero
    a = (z - z.max()) / tau if z.max() > -math.inf else z  # the largest first: the lowest finite values swallow a logarithm
    tt = torch.tensor([v for _, v in ent], dtype=torch.float64) / tau
    logp = tt - (torch.logsumexp(tt, 0) if lse is None else float(lse))
    p = logp.exp()
    S = sorted({j for j, _ in ent})
    rest = max(0.0, 1.0 - p.sum().item()) if lse is not None else 0.0
    dead = bool((a == -math.inf).all())
    logq = torch.full_like(a, -math.inf) if dead else a - torch.logsumexp(a, 0)
    loss = sum(pi * (lp - logq[j].item()) for (j, _), lp, pi in zip(ent, logp.tolist(), p.tolist()) if pi > 0)
    mask = torch.zeros(V, dtype=torch.bool)
    mask[S] = True
    log_rest = torch.logsumexp(logq.masked_fill(mask, -math.inf), 0).item()
    if log_rest == -math.inf and rest < 2.0 ** -16:
        rest = 0.0
    if rest > 0:
        loss += rest * (math.log(rest) - log_rest)
    if dead:
        return loss * tau * tau, zero
    q = logq.exp()
    total = p.sum().item() + rest if lse is not None else 1.0
    g = q * total
    if rest > 0:
        g = g - torch.where(q > 0, rest * (logq - log_rest).exp(), torch.zeros_like(q))
    g[mask] = q[mask] * total
    for (j, _), pi in zip(ent, p.tolist()):
        g[j] -= pi
    return loss * tau * tau, g * tau


def rows(z, idx, t, weight=None, tau=1.0, lse=None):
    """(loss [T], weight · gradient [T, V]) in float64."""
    T = z.shape[0]
    losses, grads = [], []
    for i in range(T):
        loss, g = row(z[i].double(), idx[i].tolist(), t[i].double().tolist(), tau, None if lse is None else lse[i].item())
        w = 1.0 if weight is None else weight[i].item()
        losses.append(loss)
        grads.append(g * w if w else torch.zeros_like(g))
    return torch.tensor(losses, dtype=torch.float64), torch.stack(grads) if grads else z.double()
