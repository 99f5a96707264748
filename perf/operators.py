"""Workloads of the operators that learn from and answer with class scores: a teacher's top logits, the distillation loss
with its gradient, and labels sampled from scores.

`run` computes them in elementary torch operations, or, with `own`, through stgcn_rt.functional and stgcn_rt.ops.
Class counts: 60 (NTU RGB+D) and 400 (Kinetics-skeleton) are the framework's own; the larger ones stand for open
vocabularies of labels."""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # top-5 scores of one evaluation batch of NTU clips: the smallest call, latency counts
        {"name": "top_ntu", "op": "top", "rows": 64, "classes": 60, "type": "f32", "k": 5, "t": 1.0, "masked": 0, "sigma": 2.0},
        # a teacher over a wide label set, scores kept for later training: one pass over half a gigabyte
        {"name": "top_wide", "op": "top", "rows": 4096, "classes": 65536, "type": "bf16", "k": 64, "t": 2.0, "masked": 0, "sigma": 2.0},
        # few clips, an odd class count: not enough rows to fill the chip with one workgroup each
        {"name": "top_few", "op": "top", "rows": 4, "classes": 131071, "type": "f32", "k": 128, "t": 1.0, "masked": 1000, "sigma": 2.5},
        # the training step of the NTU recipe: 64 clips, hard and soft term, through autograd
        {"name": "distil_ntu", "op": "distil", "rows": 64, "classes": 60, "type": "f32", "k": 5, "t": 4.0, "rest": True, "label_weight": 0.5,
         "autograd": True, "pad": 0.0, "masked": 0, "sigma": 2.0},
        # Kinetics classes, many clips (or scores per frame), a quarter of them without a teacher
        {"name": "distil_kinetics", "op": "distil", "rows": 16384, "classes": 400, "type": "f32", "k": 16, "t": 2.0, "rest": True,
         "label_weight": 0.3, "autograd": False, "pad": 0.25, "masked": 0, "sigma": 2.0},
        # the largest: loss and gradient in one call over half a billion scores
        {"name": "distil_wide", "op": "distil", "rows": 8192, "classes": 65536, "type": "bf16", "k": 64, "t": 2.0, "rest": True,
         "label_weight": 0.0, "autograd": False, "pad": 0.0, "masked": 0, "sigma": 2.0},
        # an odd class count through autograd, renormalised teacher, classes masked out
        {"name": "distil_odd", "op": "distil", "rows": 1000, "classes": 50001, "type": "f32", "k": 100, "t": 1.0, "rest": False,
         "label_weight": 0.5, "autograd": True, "pad": 0.1, "masked": 501, "sigma": 2.5},
        # few rows of a very wide head
        {"name": "distil_few", "op": "distil", "rows": 8, "classes": 131072, "type": "bf16", "k": 128, "t": 3.0, "rest": True,
         "label_weight": 0.2, "autograd": True, "pad": 0.0, "masked": 0, "sigma": 2.0},
        # pseudo-labels of one batch of Kinetics clips, the same cuts for every row
        {"name": "sample_kinetics", "op": "sample", "rows": 64, "classes": 400, "type": "f32", "t": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0,
         "mixed": False, "masked": 0, "sigma": 2.0},
        # one answer over a wide label set: latency counts
        {"name": "sample_one", "op": "sample", "rows": 1, "classes": 131072, "type": "bf16", "t": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0,
         "mixed": False, "masked": 0, "sigma": 2.5},
        # many requests, each with cuts of its own: greedy, uncut, top-k, top-p, min-p, all of them
        {"name": "sample_wide", "op": "sample", "rows": 512, "classes": 65536, "type": "bf16", "t": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0,
         "mixed": True, "masked": 0, "sigma": 2.5},
        # an odd class count, top-p alone on rows whose mass is spread over thousands of classes
        {"name": "sample_odd", "op": "sample", "rows": 200, "classes": 40961, "type": "f32", "t": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0,
         "mixed": False, "masked": 400, "sigma": 2.0},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["top", "distil", "distil", "sample"])
    n = _spread(rng, 20, 131072)
    if rng.random() < 0.3:
        n = max(20, n // 64 * 64)
    most = {"top": 4096 * 65536, "distil": 8192 * 65536, "sample": 512 * 65536}[op]
    rows = _spread(rng, 1, max(1, min(16384 if op != "sample" else 2048, most // n)))
    c = {"op": op, "rows": rows, "classes": n, "type": rng.choice(["f32", "bf16"]), "masked": rng.choice([0, 0, n // 100]),
         "sigma": round(rng.uniform(1.0, 4.0), 2)}
    if op == "top":
        c |= {"k": _spread(rng, 1, min(256, n // 2)), "t": rng.choice([1.0, 2.0, 3.5])}
    elif op == "distil":
        c |= {"k": _spread(rng, 1, min(256, n // 2)), "t": rng.choice([1.0, 2.0, 4.0, 0.7]), "rest": rng.random() < 0.6,
              "label_weight": rng.choice([0.0, 0.3, 0.5]), "autograd": rng.random() < 0.5, "pad": rng.choice([0.0, 0.0, 0.25])}
        if c["type"] == "f32" and rows * n > 4096 * 65536:
            c["type"] = "bf16"
    else:
        kind = rng.choice(["uncut", "top_k", "top_p", "min_p", "all", "mixed"])
        c |= {"t": rng.choice([1.0, 0.7, 1.5]), "top_k": _spread(rng, 2, n) if kind in ("top_k", "all") else 0,
              "top_p": round(rng.uniform(0.3, 0.99), 3) if kind in ("top_p", "all") else 1.0,
              "min_p": round(10 ** rng.uniform(-3, -0.7), 4) if kind in ("min_p", "all") else 0.0, "mixed": kind == "mixed"}
    return c


def _scores(case, seed, g):
    """Scores as a trained head gives them: a broad bulk and a few classes that stand out."""
    r, n = case["rows"], case["classes"]
    x = torch.randn((r, n), generator=g, device=DEV).mul_(case["sigma"])
    few = torch.randint(0, n, (r, max(1, min(8, n // 8))), generator=g, device=DEV)
    x.scatter_add_(1, few, 6.0 * torch.rand(few.shape, generator=g, device=DEV))
    if case["masked"]:
        x[:, n - case["masked"]:] = -math.inf             # classes that the data set does not use
    return x


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["type"]]
    x = _scores(case, seed, g)
    s = {"case": case}
    r, n = case["rows"], case["classes"]
    if case["op"] == "top":
        s["x"] = x.to(dt)
    elif case["op"] == "distil":
        t, k = case["t"], case["k"]
        # the student's scores: the teacher's, halfway there, with noise of its own
        step = max(1, (1 << 26) // n)
        xs = torch.empty((r, n), dtype=dt, device=DEV)
        val = torch.empty((r, k), device=DEV)
        idx = torch.empty((r, k), dtype=torch.int64, device=DEV)
        rest = torch.empty((r,), device=DEV)
        for a in range(0, r, step):
            b = min(r, a + step)
            xs[a:b] = (0.6 * x[a:b] + 0.7 * torch.randn((b - a, n), generator=g, device=DEV)).to(dt)
            val[a:b], idx[a:b] = torch.topk(x[a:b], k, dim=1)
            rest[a:b] = torch.logsumexp((x[a:b] / t).scatter(1, idx[a:b], -math.inf), 1)
        if case["pad"]:
            none = torch.rand((r,), generator=g, device=DEV) < case["pad"]
            idx[none] = -1                                # rows of a padded batch: no teacher
            val[none] = math.nan
        s["x"] = xs.requires_grad_(case["autograd"])
        s["val"], s["idx"], s["rest"] = val, idx, rest if case["rest"] else None
        s["labels"] = torch.randint(0, n - case["masked"], (r,), generator=g, device=DEV) if case["label_weight"] else None
    else:
        s["x"] = x.to(dt)
        s["u"] = torch.rand((r,), generator=g, device=DEV)
        if case["mixed"]:
            i = torch.arange(r, device=DEV) % 6
            s["t"] = torch.where(i == 0, 0.0, 0.7 + 0.2 * (i % 3)).float()
            s["top_k"] = torch.where((i == 2) | (i == 5), 50, 0).to(torch.int32)
            s["top_p"] = torch.where((i == 3) | (i == 5), 0.9, 1.0).float()
            s["min_p"] = torch.where((i == 4) | (i == 5), 0.05, 0.0).float()
        else:
            s["t"], s["top_k"], s["top_p"], s["min_p"] = case["t"], case["top_k"], case["top_p"], case["min_p"]
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        if _package not in sys.path:
            sys.path.insert(0, _package)
        return {"top": _own_top, "distil": _own_distil, "sample": _own_sample}[op](s)
    with torch.no_grad():
        return {"top": _plain_top, "distil": _plain_distil, "sample": _plain_sample}[op](s)


_package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "st-gcn_amd")


def _own_top(s):
    from stgcn_rt import functional as F
    return list(F.top_logits(s["x"], s["case"]["k"], temperature=s["case"]["t"]))


def _own_distil(s):
    c = s["case"]
    more = dict(rest=s["rest"], labels=s["labels"], temperature=c["t"], label_weight=c["label_weight"])
    if c["autograd"]:
        from stgcn_rt import functional as F
        loss = F.distillation(s["x"], s["val"], s["idx"], **more)
        return [loss.detach(), torch.autograd.grad(loss, s["x"])[0]]
    from stgcn_rt import ops as P
    return list(P.distillation(s["x"], s["val"], s["idx"], **more))


def _own_sample(s):
    from stgcn_rt import functional as F
    return list(F.sample_labels(s["x"], s["u"], temperature=s["t"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"]))


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _plain_top(s):
    c = s["case"]
    k = c["k"]
    v, i = torch.sort(s["x"].float(), dim=1, descending=True, stable=True)
    z = v[:, k:] / c["t"]
    m = z[:, :1]
    m = torch.where(torch.isinf(m), 0.0, m)
    rest = m[:, 0] + torch.log(torch.exp(z - m).sum(1))
    return [v[:, :k].contiguous(), i[:, :k].contiguous(), rest]


def _plain_distil(s):
    c, x, idx, val = s["case"], s["x"].float(), s["idx"], s["val"]
    t, w = c["t"], c["label_weight"]
    r, n = x.shape
    there = idx >= 0
    any_ = there.any(1, keepdim=True)
    at = idx.clamp(min=0)
    z = x / t
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    is_listed = torch.zeros((r, n), dtype=torch.bool, device=x.device).scatter_(1, at, there)
    sl = torch.where(is_listed, e, 0.0).sum(1, keepdim=True)
    sr = torch.where(is_listed, 0.0, e).sum(1, keepdim=True)
    ss = sl + sr
    # the teacher's distribution over its listed classes and the rest
    tz = torch.where(there, val / t, -math.inf)
    rho = s["rest"][:, None] if s["rest"] is not None else torch.full((r, 1), -math.inf, device=x.device)
    a = torch.maximum(torch.where(any_, tz.max(1, keepdim=True).values, 0.0), rho)
    a = a + torch.log(torch.exp(tz - a).sum(1, keepdim=True) + torch.exp(rho - a))
    lp = tz - a
    p = torch.where(any_, torch.exp(lp), 0.0)
    pr = torch.where(any_, torch.exp(rho - a), 0.0)
    lq = z.gather(1, at) - m - torch.log(ss)
    kl = torch.where(p > 0, p * (lp - lq), 0.0).sum(1, keepdim=True)
    kl = kl + torch.where(pr > 0, pr * (rho - a - torch.log(sr) + torch.log(ss)), 0.0)
    loss = (1 - w) * t * t * kl
    g = torch.where(is_listed, e / ss, e / ss - e * torch.where(pr > 0, pr / sr, 0.0))
    g.scatter_add_(1, at, -p)
    g = (1 - w) * t * torch.where(any_, g, 0.0)
    if w:
        y = s["labels"][:, None]
        m1 = x.max(1, keepdim=True).values
        e1 = torch.exp(x - m1)
        s1 = e1.sum(1, keepdim=True)
        loss = loss + w * (torch.log(s1) + m1 - x.gather(1, y))
        g = g + w * (e1 / s1)
        g.scatter_add_(1, y, torch.full_like(m1, -w))
    return [loss.sum() / r, (g / r).to(s["x"].dtype)]


def _column(v, like, dtype):
    return v.to(dtype)[:, None] if torch.is_tensor(v) else torch.full((like.shape[0], 1), v, dtype=dtype, device=like.device)


def _plain_sample(s):
    """In 64 bits: an answer next to a border between two classes has to be the same whoever adds up."""
    x = s["x"].double()
    r, n = x.shape
    # the cuts as the call takes them: 32-bit numbers
    t, p, q = (_column(s[k], x, torch.float32).double() for k in ("t", "top_p", "min_p"))
    k = _column(s["top_k"], x, torch.int64)
    k = torch.where(t == 0, 1, torch.where(k == 0, n, k))
    v, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((v - v[:, :1]) / torch.where(t == 0, 1.0, t))
    keep = torch.arange(n, device=x.device)[None] < k
    wk = torch.where(keep, w, 0.0)
    before = wk.cumsum(1) - wk
    keep &= (before < p * wk.sum(1, keepdim=True)) | (p >= 1)
    keep &= w >= q
    keep[:, 0] = True
    wk = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    total = wk.sum(1, keepdim=True)
    at = (wk.cumsum(1) <= s["u"].double()[:, None] * total).sum(1, keepdim=True).clamp(max=n - 1)
    return [at[:, 0], torch.log(wk.gather(1, at) / total)[:, 0].float()]


# ---- what the calls cannot do without -------------------------------------------------------------------------------

def work(case):
    r, n = case["rows"], case["classes"]
    e = 4 if case["type"] == "f32" else 2
    if case["op"] == "top":
        return {"bytes": r * n * e + r * (12 * case["k"] + 4), "flops": 4 * r * n}
    if case["op"] == "distil":
        more = r * 12 * case["k"] + (4 * r if case["rest"] else 0) + (8 * r if case["label_weight"] else 0) + 4
        return {"bytes": 2 * r * n * e + more, "flops": (12 if case["label_weight"] else 8) * r * n}
    return {"bytes": r * n * e + 16 * r + (16 * r if case["mixed"] else 0), "flops": 4 * r * n}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    def top(s):
        c = s["case"]
        x = s["x"].detach().double()
        values = torch.topk(x, c["k"], dim=1)
        rest = torch.logsumexp((x / c["t"]).scatter_(1, values.indices, -math.inf), 1)
        return [values.values, None, rest]

    def distil(s):
        """The loss from log-probabilities in 64 bits, its gradient by differentiation, some rows at a time."""
        c = s["case"]
        t, w = c["t"], c["label_weight"]
        r, n = s["x"].shape
        step = max(1, (1 << 27) // n)
        loss, grads = 0.0, []
        for a in range(0, r, step):
            b = min(r, a + step)
            x = s["x"][a:b].detach().double().requires_grad_(True)
            idx, val = s["idx"][a:b], s["val"][a:b].double()
            none = idx[:, 0] < 0
            at = idx.clamp(min=0)
            lq_all = torch.log_softmax(x / t, 1)
            teacher = torch.where(none[:, None], 0.0, val / t)
            if s["rest"] is not None:
                lp = torch.log_softmax(torch.cat([teacher, s["rest"][a:b, None].double()], 1), 1)
                others = torch.logsumexp(lq_all.scatter(1, at, -math.inf), 1, keepdim=True)
                lq = torch.cat([lq_all.gather(1, at), others], 1)
            else:
                lp, lq = torch.log_softmax(teacher, 1), lq_all.gather(1, at)
            kl = (lp.exp() * (lp - lq)).sum(1)
            total = (1 - w) * t * t * torch.where(none, 0.0, kl).sum() / r
            if w:
                total = total - w * torch.log_softmax(x, 1).gather(1, s["labels"][a:b, None]).sum() / r
            total.backward()
            loss = loss + total.detach()
            grads.append(x.grad if s["x"].numel() <= 1 << 28 else x.grad.float())     # bf16 results: 32 bits tell enough
            del x, lq_all, total
        return [loss, torch.cat(grads)]

    def sample(s):
        """The probability of the class that the definition gives, found row by row from the sorted classes' masses."""
        x = s["x"].detach().double().cpu()
        r, n = x.shape
        pick = lambda v, i: float(v[i]) if torch.is_tensor(v) else float(torch.tensor(float(v), dtype=torch.float32))  # noqa: E731
        par = {k: (s[k].cpu() if torch.is_tensor(s[k]) else s[k]) for k in ("t", "top_k", "top_p", "min_p")}
        u = s["u"].cpu()
        labels, logp = [], []
        for i in range(r):
            t, k, p, q = pick(par["t"], i), int(pick(par["top_k"], i)), pick(par["top_p"], i), pick(par["min_p"], i)
            order = torch.sort(x[i], descending=True, stable=True).indices
            if t == 0:
                labels.append(int(order[0]))
                logp.append(0.0)
                continue
            if k:
                order = order[:k]
            mass = torch.exp((x[i][order] - x[i][order[0]]) / t)
            if p < 1:
                reach = mass.cumsum(0)
                order = order[:int((reach < p * reach[-1]).sum()) + 1]
            mass = mass[:len(order)]
            order = order[(mass >= q) | (torch.arange(len(order)) == 0)].sort().values
            mass = torch.exp((x[i][order] - x[i][order].max()) / t)
            reach = mass.cumsum(0)
            j = min(int((reach <= float(u[i]) * reach[-1]).sum()), len(order) - 1)
            labels.append(int(order[j]))
            logp.append(float(torch.log(mass[j] / reach[-1])))
        return [torch.tensor(labels), torch.tensor(logp, dtype=torch.float64)]

    s = prepare(case, seed)
    return {"top": top, "distil": distil, "sample": sample}[case["op"]](s)
