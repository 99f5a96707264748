"""Oracle of the operators over class scores, in 64 bits on the CPU, row by row from their definitions."""
import math

import torch


def order(x):
    """Classes of one row by (score descending, class ascending), NaN first."""
    n = x.numel()
    nan = torch.isnan(x)
    return torch.tensor(sorted(range(n), key=lambda j: (0 if nan[j] else 1, 0.0 if nan[j] else -float(x[j]), j)))


def lse(z):
    z = z[z > -math.inf]
    return -math.inf if z.numel() == 0 else float(z.max() + torch.log(torch.exp(z - z.max()).sum()))


def top_logits(x, k, T):
    x = x.double()
    vals, idx, rest = [], [], []
    for row in x:
        o = torch.argsort(row, descending=True, stable=True) if not torch.isnan(row).any() else order(row)
        vals.append(row[o[:k]])
        idx.append(o[:k])
        rest.append(lse(row[o[k:]] / T))
    return torch.stack(vals), torch.stack(idx), torch.tensor(rest, dtype=torch.float64)


def teacher(row_val, row_idx, rho, T):
    """[(class, p)], p_rest of one row's teacher; None without entries."""
    e = [(int(i), float(v) / T) for i, v in zip(row_idx, row_val) if i >= 0 and float(v) > -math.inf]
    if not e:
        return None
    r = -math.inf if rho is None else float(rho)
    a = lse(torch.tensor([t for _, t in e] + [r], dtype=torch.float64))
    listed = [int(i) for i in row_idx if i >= 0]
    return [(i, math.exp(t - a)) for i, t in e], math.exp(r - a), sorted(set(listed))


def distill_row(x, val, idx, rho, label, T, w):
    """(loss, gradient) of one row."""
    n = x.numel()
    x = x.double()
    g = torch.zeros(n, dtype=torch.float64)
    bad = any(int(i) >= n for i in idx) or (w > 0 and label is not None and label >= n)
    bad |= any(int(i) >= 0 and not float(v) < math.inf for i, v in zip(idx, val))
    tea = teacher(val, idx, rho, T) if w < 1 and not bad else None
    if tea is not None and rho is not None and not float(rho) < math.inf:
        bad = True
    hard = w > 0 and label is not None and label >= 0
    if bad:
        return math.nan, g * math.nan
    if tea is None and not hard:
        return 0.0, g
    if torch.isnan(x).any() or (x == math.inf).any():
        return math.nan, g * math.nan
    if x.max() == -math.inf:
        return 0.0, g
    x = x - x.max()                    # a softmax does not see it, and sums next to scores of 1e38 would
    loss = 0.0
    if tea is not None:
        entries, pr, listed = tea
        z = x / T
        S = lse(z)
        q = torch.exp(z - S)
        other = torch.ones(n, dtype=torch.bool)
        other[listed] = False
        kl = 0.0
        for i, p in entries:
            if p > 0:
                kl += p * (math.log(p) - float(z[i]) + S) if float(z[i]) > -math.inf else math.inf
        if pr > 0:
            So = lse(z[other])
            kl += pr * (math.log(pr) - So + S) if So > -math.inf else math.inf
            if So > -math.inf:
                q[other] -= pr * torch.exp(z[other] - So)
        g += (1 - w) * T * q
        for i, p in entries:
            g[i] -= (1 - w) * T * p
        loss += (1 - w) * T * T * kl
    if hard:
        S1 = lse(x)
        g += w * torch.exp(x - S1)
        g[label] -= w
        loss += w * (S1 - float(x[label])) if float(x[label]) > -math.inf else math.inf
    return loss, g


def distill(x, val, idx, rest, labels, T, w):
    """Row losses and the rows' gradients (of the sum of the losses)."""
    out = [distill_row(x[r], val[r], idx[r], None if rest is None else rest[r], None if labels is None else int(labels[r]), T, w)
           for r in range(x.shape[0])]
    return torch.tensor([o[0] for o in out], dtype=torch.float64), torch.stack([o[1] for o in out])


def sample_row(x, u, T, k, p, q):
    """(label, log-probability) of one row; the parameters are 32-bit numbers."""
    x = x.double()
    n = x.numel()
    if torch.isnan(x).any() or not (0 <= T < math.inf and k >= 0 and 0 < p <= 1 and 0 <= q <= 1 and 0 <= u < 1):
        return -1, math.nan
    if x.max() == -math.inf:
        return -1, -math.inf
    o = torch.argsort(x, descending=True, stable=True)
    if T == 0:
        return int(o[0]), 0.0
    w = torch.where(x == x.max(), 1.0, torch.exp((x - x.max()) / T))
    if k:
        o = o[:k]
    if p < 1:
        reach = w[o].cumsum(0)
        o = o[:int((reach - w[o] < p * reach[-1]).sum())]
    keep = [int(j) for i, j in enumerate(o) if i == 0 or float(w[j]) >= q]
    keep.sort()
    reach = w[keep].cumsum(0)
    j = min(int((reach <= u * reach[-1]).sum()), len(keep) - 1)
    while j > 0 and float(w[keep[j]]) == 0:
        j -= 1
    return keep[j], math.log(float(w[keep[j]]) / float(reach[-1]))


def sample(x, u, T, k, p, q):
    r = x.shape[0]
    f = lambda v, i: float(v[i]) if torch.is_tensor(v) else float(torch.tensor(float(v), dtype=torch.float32))   # noqa: E731
    out = [sample_row(x[i], float(u[i]), f(T, i), int(k[i]) if torch.is_tensor(k) else int(k), f(p, i), f(q, i)) for i in range(r)]
    return torch.tensor([o[0] for o in out]), torch.tensor([o[1] for o in out], dtype=torch.float64)
