"""Operators over class scores (top_logits, distillation, sample_labels) against their 64-bit definitions.

Tolerances.  S, a sum of exponentials, is made of v_exp_f32 values (one unit in the last place, 2^-23) at arguments
y = (x - max) c whose subtraction, product and c are rounded to 24 bits (each 2^-24 |y|, so 3 * 2^-24 |y| ln 2 in the
value; |y| <= 127 where the value is not flushed to zero), added up in 32 bits by threads of at most `chain` terms each
(chain * 2^-24) and joined in 64 bits.  EPS_S(case) = 2^-23 + (2.1 D + chain) 2^-24 bounds the relative error of S, D the
largest |y|.  The gradients are products of e, of factors of 1/S and of the incoming gradient (each rounded once:
8 * 2^-24 covers them) minus p, rounded once more to the type of the scores: eps / 2 of the value."""
import ctypes
import itertools
import math

import pytest
import torch

from oracle import scores_oracle as O

DEV = "cuda:0"
U = 2.0 ** -24
CHAIN = 600        # terms one thread adds up in 32 bits, at most, over the class counts tested here


@pytest.fixture(scope="module")
def rt():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a GPU")
    from stgcn_rt import functional as F, ops as P
    return F, P


def half_step(dt):
    return torch.finfo(dt).eps / 2


def scores(rows, n, dt, seed, sigma=2.0, masked=0, offset=0, gap=0, quant=0.0):
    """Scores [rows, n] on the GPU: `offset` elements into their memory, rows `gap` elements apart."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, n, generator=g) * sigma
    if quant:
        x = torch.round(x / quant) * quant
    if masked:
        x[:, torch.randperm(n, generator=g)[:masked]] = -math.inf
    buf = torch.full((offset + rows * (n + gap) + 8,), 77.0, dtype=dt)
    v = torch.as_strided(buf, (rows, n), (n + gap, 1), offset)
    v.copy_(x.to(dt))
    return torch.as_strided(buf.to(DEV), (rows, n), (n + gap, 1), offset)


def eps_sum(x, T):
    """EPS_S of the docstring for rows x at temperature T (a number)."""
    f = x.double().cpu()
    f = torch.where(torch.isfinite(f), f, f[torch.isfinite(f)].max() if torch.isfinite(f).any() else 0.0)
    d = min(127.0, float((f.max(1).values - f.min(1).values).max()) * 1.4427 / min(T, 1.0))
    return 2.0 ** -23 + (2.1 * d + CHAIN) * U


# ---- top_logits --------------------------------------------------------------------------------------------------

TOP = [(1, 1, 1), (3, 2, 2), (5, 7, 3), (64, 60, 5), (33, 61, 61), (9, 400, 16), (4, 401, 256), (3, 1027, 100), (2, 8191, 128),
       (2, 8200, 1), (3, 20011, 256), (1, 70001, 64), (1, 131075, 200), (600, 5000, 20), (520, 9001, 256)]


def check_top(F, x, k, T):
    got = F.top_logits(x, k, T)
    xc = x.float().cpu()
    v, i, rest = O.top_logits(xc, k, T)
    assert got.values.dtype == torch.float32 and got.indices.dtype == torch.int64 and got.rest.dtype == torch.float32
    assert torch.equal(got.indices.cpu(), i)
    assert torch.equal(torch.nan_to_num(got.values.cpu().double(), nan=5.0), torch.nan_to_num(v, nan=5.0))
    g = got.rest.cpu().double()
    fin = torch.isfinite(rest)
    assert torch.equal(g[~fin], rest[~fin])
    # log of S (EPS_S), the maximum over T in 64 bits, one rounding to 32
    tol = eps_sum(x, T) + U * rest[fin].abs() + 1e-30
    assert bool(((g[fin] - rest[fin]).abs() <= tol).all()), (g, rest)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,n,k", TOP)
def test_top_logits(rt, rows, n, k, dt):
    for j, (off, gap, masked, quant) in enumerate([(0, 0, 0, 0.0), (1, 3, n // 5, 0.0), (5, 0, 0, 0.5)]):
        print("top", rows, n, k, dt, off, gap, masked, quant, flush=True)
        check_top(rt[0], scores(rows, n, dt, 10 * n + j, masked=masked, offset=off, gap=gap, quant=quant), k, [1.0, 2.0, 0.5][j])


def special_rows(n, dt):
    """Rows that a mask leaves nothing of, equal rows, sorted rows, the type's extremes, infinities, both zeros."""
    low, high = torch.finfo(dt).min, torch.finfo(dt).max
    g = torch.Generator().manual_seed(n)
    base = torch.randn(n, generator=g)
    rows = [torch.full((n,), -math.inf), torch.zeros(n), torch.full((n,), low), torch.full((n,), high),
            torch.linspace(-9, 9, n), torch.linspace(9, -9, n),
            torch.where(torch.arange(n) % 7 == 3, base, torch.tensor(float(low))),
            torch.where(torch.arange(n) == n // 2, 1.0, -math.inf),
            torch.where(torch.arange(n) % 2 == 0, 0.0, -0.0) * (torch.arange(n) % 5 > 1),
            torch.where(torch.arange(n) < 16, base + 30, base),
            torch.where(torch.arange(n) % 1024 < 8, base.abs() + 40, torch.zeros(n))]
    return torch.stack(rows).to(dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,k", [(60, 7), (400, 130), (9001, 256), (40000, 33)])
def test_top_logits_special_rows(rt, n, k, dt):
    check_top(rt[0], special_rows(n, dt).to(DEV), k, 1.0)


@pytest.mark.gpu
def test_top_logits_infinity_and_nan(rt):
    x = scores(6, 500, torch.float32, 3)
    x[1, 77] = math.inf
    x[2, 400] = math.nan
    x[2, 13] = math.nan
    x[3, :] = math.nan
    x[4, 5] = math.inf
    x[4, 2] = math.nan
    got = rt[0].top_logits(x, 4)
    v, i, _ = O.top_logits(x.cpu(), 4, 1.0)
    assert torch.equal(got.indices.cpu(), i)
    assert torch.equal(torch.nan_to_num(got.values.cpu().double(), nan=5.0), torch.nan_to_num(v, nan=5.0))
    assert torch.isnan(got.rest.cpu()[3])


# ---- distillation ------------------------------------------------------------------------------------------------

def teacher_lists(x, k, T, seed, pad=0.0, dup=False):
    """A teacher near x's scores: values, indices, rest on the GPU; some rows and entries absent."""
    g = torch.Generator().manual_seed(seed)
    xs = x.float().cpu()
    t = xs * 0.7 + torch.randn(xs.shape, generator=g)
    v, i, rest = O.top_logits(t, k, T)
    v = v.float()
    if dup and k > 2:
        i[:, k - 1] = i[:, 0]                       # the same class twice
    if pad:
        gone = torch.rand(i.shape[0], generator=g) < pad
        i[gone] = -1
        some = torch.rand(i.shape, generator=g) < 0.1
        i[some] = -5
        v[i < 0] = math.nan
    return v.to(DEV), i.to(DEV), rest.float().to(DEV)


def check_distill(rt, x, val, idx, rest, labels, T, w, rows_grad=None):
    """Row losses, mean, sum and their gradients, and the pair of ops.distillation, against the definition."""
    F, P = rt
    xc = x.detach().float().cpu()
    L_, G_ = O.distill(xc, val.cpu(), idx.cpu(), None if rest is None else rest.cpu(), None if labels is None else labels.cpu(), T, w)
    rows, n = xc.shape
    es = eps_sum(xc, T)
    D = (es - 2.0 ** -23) / U
    e1 = es + (8 + D) * U
    # sizes of the parts that a gradient is made of: q, p and the rest's factor, which can cancel each other
    Qs, Ls = [], []
    for r in range(rows):
        q = torch.zeros(n, dtype=torch.float64)
        size = 0.0
        row = xc[r].double()
        tea = O.teacher(val[r].cpu(), idx[r].cpu(), None if rest is None else float(rest[r]), T) if w < 1 else None
        live = bool(torch.isfinite(L_[r])) and row.max() > -math.inf
        if live:
            row = row - row.max()
        if tea is not None and live:
            z = row / T
            S = O.lse(z)
            qz = torch.exp(z - S)
            other = torch.ones(n, dtype=torch.bool)
            other[tea[2]] = False
            q += (1 - w) * T * qz
            if tea[1] > 0 and O.lse(z[other]) > -math.inf:
                q[other] += (1 - w) * T * qz[other] * tea[1] * math.exp(S - O.lse(z[other]))
            for i, p in tea[0]:
                q[i] += (1 - w) * T * p
            # log S and log S_r enter with weight 1 and p_r; z_k with the rounding of c; log p in 64 bits from 32-bit inputs
            size += (1 - w) * T * T * 2 + (1 - w) * T * T * sum(p * abs(float(z[i]) - float(z.max())) for i, p in tea[0]) * U / es
        if w > 0 and labels is not None and int(labels[r]) >= 0 and live:
            q += w * torch.exp(row - O.lse(row))
            q[int(labels[r])] += w
            size += w + w * abs(float(row[int(labels[r])]) - float(row.max())) * U / es
        Qs.append(q)
        Ls.append(size)
    Q, Lt = torch.stack(Qs), torch.tensor(Ls, dtype=torch.float64) * es
    hs = half_step(x.dtype)
    flush = 2.0 ** -126 * max(1.0, T)                       # results below the normal range may be flushed to zero

    def close(got, want, tol, what):
        got, want = got.detach().cpu().double(), want.double()
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan), what
        inf = torch.isinf(want)
        assert torch.equal(got[inf], want[inf]), what
        ok = ~(nan | inf)
        bad = (got - want).abs()[ok] > torch.broadcast_to(tol, want.shape)[ok]
        assert not bool(bad.any()), (what, got[ok][bad][:5], want[ok][bad][:5], torch.broadcast_to(tol, want.shape)[ok][bad][:5])

    tol_rows = Lt + U * torch.nan_to_num(L_.abs(), posinf=0.0) + 1e-12
    more = dict(rest=rest, labels=labels, temperature=T, label_weight=w)
    leaf = x.detach().requires_grad_(True)
    loss = F.distillation(leaf, val, idx, reduction="none", **more)
    close(loss, L_, tol_rows, "rows")
    gr = torch.linspace(-1.5, 2.0, rows, dtype=torch.float32)
    (dx,) = torch.autograd.grad(loss, leaf, gr.to(DEV))
    assert dx.dtype == x.dtype and dx.shape == x.shape
    G = G_ * gr.double()[:, None]
    close(dx, G, Q * e1 * gr.double().abs()[:, None] + hs * torch.nan_to_num(G.abs()) + flush, "rows' gradient")
    for red, f in (("mean", 1.0 / rows), ("sum", 1.0)):
        loss = F.distillation(leaf, val, idx, reduction=red, **more)
        close(loss, L_.sum() * f, (tol_rows.sum() * f + U * abs(float(torch.nan_to_num(L_.sum(), posinf=0.0))) * f), red)
        (dx,) = torch.autograd.grad(loss * 3.0, leaf)
        G = G_ * (3.0 * f)
        close(dx, G, (Q * e1 * 3 * f) + hs * torch.nan_to_num(G.abs()) + flush, red + " gradient")
        pair = P.distillation(x, val, idx, reduction=red, **more)
        assert torch.equal(torch.nan_to_num(pair[0], nan=9.0), torch.nan_to_num(loss.detach(), nan=9.0))
        G = G_ * f
        close(pair[1], G, (Q * e1 * f) + hs * torch.nan_to_num(G.abs()) + flush, red + " pair")


DIST = [(1, 1, 1), (17, 100, 64), (35, 511, 33), (18, 1023, 65),  (6, 256, 30), (5, 512, 40), (3, 1024, 9), (2, 16384, 33), (2, 32768, 20), (1, 65536, 64), (3, 2, 1), (5, 7, 7), (64, 60, 5), (7, 61, 20), (9, 400, 16), (3, 401, 256), (4, 1027, 100), (2, 4099, 64),
        (2, 8191, 128), (3, 16390, 9), (2, 33000, 256), (1, 65537, 30), (2, 131075, 64), (1, 131072, 256), (1, 140001, 50)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,n,k", DIST)
def test_distillation(rt, rows, n, k, dt):
    g = torch.Generator().manual_seed(n)
    for j, (T, w, with_rest, off, gap, pad, masked) in enumerate([
            (1.0, 0.0, True, 0, 0, 0.0, 0), (2.0, 0.0, False, 1, 0, 0.3, 0), (4.0, 0.5, True, 3, 5, 0.3, n // 7),
            (1.0, 0.3, False, 0, 1, 0.0, 0), (0.7, 0.6, True, 0, 8, 0.0, 0), (2.0, 1.0, True, 0, 0, 0.0, 0)]):
        if masked and n - masked < k:
            masked = 0
        print("distill", rows, n, k, dt, T, w, with_rest, off, gap, pad, masked, flush=True)
        x = scores(rows, n, dt, 7 * n + j, offset=off, gap=gap, masked=masked)
        val, idx, rest = teacher_lists(x, k, T, j, pad=pad, dup=j % 2 == 1)
        labels = torch.randint(0, n, (rows,), generator=g)
        labels[torch.isinf(x.float().cpu().gather(1, labels[:, None]))[:, 0]] = -1
        if rows > 2:
            labels[1] = -100
        check_distill(rt, x, val, idx, rest if with_rest else None, labels.to(DEV), T, w)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,dt", [(520, 8211, torch.float32), (513, 20003, torch.bfloat16), (515, 401, torch.float32)])
def test_distillation_many_rows(rt, rows, n, dt):
    """Enough rows that each gets fewer waves."""
    x = scores(rows, n, dt, n, offset=1, gap=2)
    val, idx, rest = teacher_lists(x, 20, 2.0, n, pad=0.1)
    lab = torch.randint(-1, n, (rows,), generator=torch.Generator().manual_seed(rows)).to(DEV)
    check_distill(rt, x, val, idx, rest, lab, 2.0, 0.25)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [60, 1500, 40000])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_distillation_rows_without_anything(rt, n, dt):
    """Padding (no entry, no label) over garbage, rows of -inf, masks of the type's lowest value, +inf and NaN scores,
    classes out of range, teacher scores that are no numbers: each row by itself."""
    x = scores(12, n, dt, n)
    val, idx, rest = teacher_lists(x, 6, 2.0, 1)
    labels = torch.arange(12)
    idx[0] = -1; labels[0] = -1; x[0] = math.nan; val[0] = math.inf; rest[0] = math.nan       # padding over garbage
    idx[1] = -1; val[1] = math.nan                                                            # a label alone
    x[2] = -math.inf                                                                          # no class at all
    x[3, :] = torch.finfo(dt).min                                                             # equal, at the type's lowest value
    x[4, n // 3:] = torch.finfo(dt).min
    idx[4] = torch.arange(6, device=DEV)
    labels[4] = 3
    idx[5, 2] = n                                                                             # out of range: this row is NaN
    labels[6] = n
    val[7, 1] = math.nan
    x[8, n - 1] = math.nan
    x[9, n - 2] = math.inf
    rest[10] = -math.inf
    val[11, 3:] = -math.inf                                                                   # entries that weigh nothing
    check_distill(rt, x, val, idx, rest, labels.to(DEV), 2.0, 0.4)
    check_distill(rt, x, val, idx, None, None, 1.0, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_distillation_concentrated_teacher_and_student(rt, dt):
    """Both carry nearly all mass in the list: the others' sum has to be their own, not a difference."""
    n, k = 5000, 8
    x = scores(3, n, dt, 5, sigma=0.5)
    x[:, 100:108] += 17.0
    val, idx, rest = teacher_lists(x, k, 1.0, 2)
    check_distill(rt, x, val, idx, rest, None, 1.0, 0.0)
    check_distill(rt, x, val, idx, torch.full_like(rest, -60.0), None, 1.0, 0.0)


@pytest.mark.gpu
def test_distillation_gradient_against_differences(rt):
    """Central differences of the 64-bit loss at a few classes, listed and not."""
    T, w, n = 2.0, 0.3, 300
    x = scores(4, n, torch.float32, 9)
    val, idx, rest = teacher_lists(x, 10, T, 3)
    labels = torch.tensor([3, 290, 7, 11])
    _, dx = rt[1].distillation(x, val, idx, rest=rest, labels=labels.to(DEV), temperature=T, label_weight=w, reduction="sum")
    h = 1e-4
    for r in range(4):
        for j in [int(idx[r, 0]), int(idx[r, 9]), int(labels[r]), 0, 150, 299]:
            f = []
            for s in (h, -h):
                xx = x[r].cpu().double()
                xx[j] += s
                f.append(O.distill_row(xx, val[r].cpu(), idx[r].cpu(), float(rest[r]), int(labels[r]), T, w)[0])
            # the difference's own error: h^2 / 6 times a third derivative below T^-1..1, and 2^-52 |loss| / h
            assert abs(float(dx[r, j]) - (f[0] - f[1]) / (2 * h)) < h * h + 1e-10 + 4e-6, (r, j)


# ---- sample_labels -----------------------------------------------------------------------------------------------

def check_sample(F, x, u, T=1.0, k=0, p=1.0, q=0.0):
    got = F.sample_labels(x, u, temperature=T, top_k=k, top_p=p, min_p=q)
    cpu = lambda v: v.cpu() if torch.is_tensor(v) else v                                       # noqa: E731
    lab, lp = O.sample(x.float().cpu(), u.cpu(), cpu(T), cpu(k), cpu(p), cpu(q))
    assert got[0].dtype == torch.int64 and got[1].dtype == torch.float32
    assert torch.equal(got[0].cpu(), lab), (got[0].cpu()[got[0].cpu() != lab], lab[got[0].cpu() != lab], (got[0].cpu() != lab).nonzero()[:, 0])
    g = got[1].cpu().double()
    assert torch.equal(torch.isnan(g), torch.isnan(lp)) and torch.equal(g[torch.isinf(lp)], lp[torch.isinf(lp)])
    ok = torch.isfinite(lp)
    # 64-bit weights and sums (1e-11 over a row), one rounding to 32 bits
    assert bool(((g[ok] - lp[ok]).abs() <= U * lp[ok].abs() + 1e-10).all()), (g[ok], lp[ok])


def uniforms(rows, seed):
    u = torch.rand(rows, generator=torch.Generator().manual_seed(seed))
    u[0] = 0.0
    u[rows - 1] = 1 - 2.0 ** -24 if rows > 1 else u[0]
    return u.to(DEV)


SAMP = [(1, 1), (4, 2), (7, 61), (64, 400), (9, 1027), (5, 8191), (4, 20011), (3, 65537), (2, 131075)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,n", SAMP)
def test_sample_labels(rt, rows, n, dt):
    for j, (T, k, p, q, masked, off, gap, sigma, quant) in enumerate([
            (1.0, 0, 1.0, 0.0, 0, 0, 0, 2.0, 0.0), (0.7, 50, 1.0, 0.0, 0, 1, 0, 2.5, 0.0), (1.0, 0, 0.9, 0.0, n // 9, 0, 3, 2.0, 0.0),
            (1.3, 0, 1.0, 0.05, 0, 3, 1, 2.0, 0.0), (1.0, 200, 0.8, 0.01, 0, 0, 0, 3.0, 0.5), (0.0, 0, 1.0, 0.0, 0, 0, 0, 1.0, 1.0),
            (4.0, 0, 0.6, 0.0, 0, 0, 0, 0.3, 0.0), (1.0, max(1, n // 2), 0.95, 0.0, 0, 0, 0, 1.0, 0.25), (1.0, n + 5, 0.5, 1.0, 0, 0, 0, 1.0, 0.0)]):
        print("sample", rows, n, dt, T, k, p, q, masked, off, gap, sigma, quant, flush=True)
        x = scores(rows, n, dt, 3 * n + j, sigma=sigma, masked=min(masked, n - 1), offset=off, gap=gap, quant=quant)
        check_sample(rt[0], x, uniforms(rows, n + j), T, k, p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [61, 2000, 30001])
def test_sample_labels_special_rows(rt, n, dt):
    x = special_rows(n, dt)
    x = torch.cat([x, x[-3:]]).to(DEV)
    x[-1, 3] = math.nan
    x[-2, 5] = math.inf
    x[-2, 8] = math.inf
    u = uniforms(x.shape[0], n)
    for T, k, p, q in [(1.0, 0, 1.0, 0.0), (1.0, 9, 1.0, 0.0), (0.5, 0, 0.7, 0.0), (2.0, 0, 1.0, 0.3), (1.0, 30, 0.5, 0.1), (0.0, 0, 1.0, 0.0), (1e-3, 0, 0.9, 0.0),
                       (1e6, 0, 0.25, 0.0)]:
        print("special", n, dt, T, k, p, q, flush=True)
        check_sample(rt[0], x, u, T, k, p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [600, 9001, 40003])
def test_sample_labels_crowded_rows(rt, n, dt):
    """Thousands of scores in a small part of the row's range, around one value, two, or all over a bin: the borders take
    several rounds."""
    g = torch.Generator().manual_seed(n)
    noise = torch.randn(n, generator=g)
    rows = [noise * 1e-3, noise * 1e-3 - 7, 2 + noise * 1e-6, torch.where(torch.arange(n) % 3 == 0, 4 + noise * 1e-4, -4 + noise * 1e-4),
            torch.where(torch.arange(n) % 2 == 0, noise * 1e-3, -math.inf), noise.abs() * -1e-30]
    x = torch.stack(rows)
    x[0, 5], x[1, n - 1], x[3, 0] = 25.0, 1.0, 4.5
    x = x.to(dt).to(DEV)
    for j, (k, p, q) in enumerate([(0, 0.9, 0.0), (0, 0.3, 0.0), (n // 3, 1.0, 0.0), (n // 2, 0.5, 0.0), (0, 0.99, 0.2), (n - 7, 0.97, 1e-3), (n // 4, 1.0, 0.999)]):
        check_sample(rt[0], x, uniforms(len(rows), 7 * n + j), k=k, p=p, q=q)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,dt", [(270, 9001, torch.float32), (260, 16500, torch.bfloat16), (300, 3001, torch.float32)])
def test_sample_labels_many_rows(rt, rows, n, dt):
    """Enough rows that each gets fewer waves, every row with cuts of its own."""
    x = scores(rows, n, dt, n, sigma=2.5, masked=n // 9, offset=3, gap=5)
    g = torch.Generator().manual_seed(rows)
    pick = lambda *v: torch.tensor(v, dtype=torch.float32)[torch.randint(0, len(v), (rows,), generator=g)].to(DEV)         # noqa: E731
    check_sample(rt[0], x, uniforms(rows, rows), T=pick(0.0, 0.5, 1.0, 1.7), k=pick(0, 1, 40, 300, 4000).int(), p=pick(0.2, 0.9, 0.999, 1.0),
                 q=pick(0.0, 0.0, 0.01, 1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [400, 9001])
def test_sample_labels_parameters_per_row(rt, n, dt):
    """Every combination of cuts in one batch, and parameters out of range, each row by itself."""
    combos = list(itertools.product([0.0, 0.8, 1.5], [0, 1, 5, n], [1.0, 0.6], [0.0, 0.2]))
    bad = [(-1.0, 0, 1.0, 0.0), (math.nan, 0, 1.0, 0.0), (math.inf, 0, 1.0, 0.0), (1.0, -2, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.5, 0.0),
           (1.0, 0, math.nan, 0.0), (1.0, 0, 1.0, -0.1), (1.0, 0, 1.0, 2.0), (1.0, 0, 1.0, math.nan)]
    every = combos + bad
    T, k, p, q = (torch.tensor([c[i] for c in every], dtype=torch.int32 if i == 1 else torch.float32, device=DEV) for i in range(4))
    x = scores(len(every), n, dt, n, quant=0.25)
    u = uniforms(len(every), 4)
    check_sample(rt[0], x, u, T, k, p, q)
    u[3], u[7], u[9] = 1.0, -0.5, math.nan
    check_sample(rt[0], x, u, T, k, p, q)


@pytest.mark.gpu
def test_sample_labels_follow_the_distribution(rt):
    """Many draws of one row: counts within five standard deviations of the kept classes' shares."""
    n, draws = 40, 20000
    row = scores(1, n, torch.float32, 8, sigma=1.5)
    lab, _ = rt[0].sample_labels(row.expand(draws, n), torch.rand(draws, generator=torch.Generator().manual_seed(1)).to(DEV), top_p=0.8)
    w = torch.softmax(row[0].cpu().double(), 0)
    o = torch.argsort(w, descending=True)
    keep = o[:int((w[o].cumsum(0) - w[o] < 0.8).sum())]
    share = torch.zeros(n, dtype=torch.float64)
    share[keep] = w[keep] / w[keep].sum()
    got = torch.bincount(lab.cpu(), minlength=n).double() / draws
    assert bool(((got - share).abs() <= 5 * torch.sqrt(share * (1 - share) / draws)).all())


# ---- together, streams, graphs, sizes ----------------------------------------------------------------------------

@pytest.mark.gpu
def test_teach_and_learn_together(rt):
    """A teacher's scores kept by top_logits, the student's loss on them: with every class listed it is the whole KL."""
    F, _ = rt
    t, s = scores(16, 60, torch.float32, 1), scores(16, 60, torch.float32, 2)
    for k in (60, 10):
        top = F.top_logits(t, k, temperature=3.0)
        leaf = s.detach().requires_grad_(True)
        loss = F.distillation(leaf, top.values, top.indices, rest=top.rest, temperature=3.0)
        (dx,) = torch.autograd.grad(loss, leaf)
        if k == 60:
            a = t.cpu().double()
            b = s.cpu().double().requires_grad_(True)
            ref = 9.0 * torch.nn.functional.kl_div(torch.log_softmax(b / 3, 1), torch.softmax(a / 3, 1), reduction="batchmean")
            ref.backward()
            # es = EPS_S: log S (twice) and c on the loss; on the gradient e1 of its parts q and p, T / rows at most
            es = eps_sum(s, 3.0)
            assert abs(float(loss.detach()) - float(ref.detach())) < 9.0 * 4 * es
            assert float((dx.cpu().double() - b.grad).abs().max()) < 3.0 / 16 * 4 * es


@pytest.mark.gpu
def test_calls_on_another_stream_and_at_once(rt):
    """Two streams at once, many calls: each answers as alone."""
    F, P = rt
    xs = [scores(40, 5003, torch.bfloat16, i) for i in (1, 2)]
    tl = [F.top_logits(x, 20) for x in xs]
    us = [uniforms(40, i) for i in (1, 2)]
    alone = [(P.distillation(x, t.values, t.indices, rest=t.rest), F.sample_labels(x, u, top_p=0.9)) for x, t, u in zip(xs, tl, us)]
    torch.cuda.synchronize()
    ss = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(6):
        for i in range(2):
            with torch.cuda.stream(ss[i]):
                t = F.top_logits(xs[i], 20)
                outs[i].append((t, P.distillation(xs[i], t.values, t.indices, rest=t.rest), F.sample_labels(xs[i], us[i], top_p=0.9)))
    torch.cuda.synchronize()
    for i in range(2):
        for t, d, s in outs[i]:
            assert torch.equal(t.indices, tl[i].indices) and torch.equal(t.rest, tl[i].rest)
            assert torch.equal(d[0], alone[i][0][0]) and torch.equal(d[1], alone[i][0][1])
            assert torch.equal(s[0], alone[i][1][0]) and torch.equal(s[1], alone[i][1][1])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,dt", [(16, 60, torch.float32), (6, 30001, torch.bfloat16)])
def test_captured_and_replayed(rt, rows, n, dt):
    """top_logits, the loss with its backward and sampling in two graphs, replayed in turn with eager work in between."""
    F, _ = rt
    static = [scores(rows, n, dt, i) for i in (1, 2)]
    teach = [scores(rows, n, dt, i + 5) for i in (1, 2)]
    u = uniforms(rows, 1)

    def step(x, t):
        top = F.top_logits(t, 7, 2.0)
        leaf = x.detach().requires_grad_(True)
        loss = F.distillation(leaf, *top, temperature=2.0)
        (dx,) = torch.autograd.grad(loss, leaf)
        return [loss.detach(), dx, *F.sample_labels(x, u, top_k=20, top_p=0.9), *top]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, t in zip(static, teach):
            step(x, t)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x, t in zip(static, teach):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x, t))
        graphs.append(g)
    for rep in range(4):
        for i in (0, 1):
            new = scores(rows, n, dt, 100 + 10 * rep + i)
            static[i].copy_(new)
            graphs[i].replay()
            want = step(new, teach[i])
            torch.cuda.synchronize()
            for a, b in zip(outs[i], want):
                assert torch.equal(a, b), (rep, i)


@pytest.mark.gpu
def test_the_same_bits_every_time(rt):
    F, P = rt
    x = scores(300, 4099, torch.bfloat16, 1)
    top = F.top_logits(scores(300, 4099, torch.bfloat16, 2), 50)
    first = P.distillation(x, *top)
    for _ in range(3):
        again = P.distillation(x, *top)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.gpu
def test_offsets_beyond_32_bits(rt):
    """2.2e9 scores: the last rows' elements lie behind 2^31 elements and 2^32 bytes."""
    F, P = rt
    rows, n = 33000, 65536
    x = torch.zeros((rows, n), dtype=torch.bfloat16, device=DEV)
    tail = scores(3, n, torch.bfloat16, 1)
    x[-3:] = tail
    got = F.top_logits(x, 5)
    want = F.top_logits(tail, 5)
    assert torch.equal(got.indices[-3:], want.indices) and torch.equal(got.rest[-3:], want.rest)
    assert torch.equal(got.indices[0].cpu(), torch.arange(5))
    u = torch.full((rows,), 0.37, device=DEV)
    a, b = F.sample_labels(x, u, top_p=0.9), F.sample_labels(tail, u[:3], top_p=0.9)
    assert torch.equal(a[0][-3:], b[0]) and torch.equal(a[1][-3:], b[1])
    loss, dx = P.distillation(x, *got, reduction="sum")
    loss3, dx3 = P.distillation(tail, *want, reduction="sum")
    assert torch.equal(dx[-3:], dx3)
    assert float(dx[:100].float().abs().max()) < 1e-6


@pytest.mark.gpu
def test_inputs_stay_and_nothing_is_written_beside(rt):
    F, P = rt
    for dt, n in itertools.product((torch.float32, torch.bfloat16), (61, 9001)):
        x = scores(5, n, dt, n, offset=3, gap=5)
        whole = torch.as_strided(x, (3 + 5 * (n + 5) + 8,), (1,), 0)
        before = whole.clone()
        top = F.top_logits(x, 4)
        P.distillation(x, *top)
        F.sample_labels(x, uniforms(5, 1), top_p=0.9)
        assert torch.equal(whole, before)


@pytest.mark.gpu
def test_no_rows(rt):
    F, P = rt
    for dt in (torch.float32, torch.bfloat16):
        x = torch.empty((0, 60), dtype=dt, device=DEV, requires_grad=True)
        top = F.top_logits(x, 5)
        assert top.values.shape == (0, 5) and top.rest.shape == (0,)
        loss = F.distillation(x, *top, reduction="sum")
        assert float(loss.detach()) == 0 and torch.autograd.grad(loss, x)[0].shape == (0, 60)
        assert F.distillation(x, *top, reduction="none").shape == (0,)
        with pytest.raises(ValueError, match="no rows"):
            F.distillation(x, *top)
        assert F.sample_labels(x, torch.empty(0, device=DEV))[0].shape == (0,)


@pytest.mark.gpu
def test_other_layouts_are_copied(rt):
    """Classes that are not contiguous: the same answers as of a contiguous copy."""
    F, _ = rt
    x = scores(60, 33, torch.float32, 3).t()
    assert x.stride(1) != 1
    top, ref = F.top_logits(x, 6), F.top_logits(x.contiguous(), 6)
    assert torch.equal(top.indices, ref.indices) and torch.equal(top.rest, ref.rest)
    a, b = x.detach().requires_grad_(True), x.contiguous().requires_grad_(True)
    la, lb = F.distillation(a, *top), F.distillation(b, *top)
    assert torch.equal(la, lb) and torch.equal(torch.autograd.grad(la, a)[0], torch.autograd.grad(lb, b)[0])
    one = scores(1, 33, torch.float32, 4).expand(7, 33)
    assert torch.equal(F.top_logits(one, 3).indices, F.top_logits(one.contiguous(), 3).indices)


# ---- refusals (CPU) ----------------------------------------------------------------------------------------------

def test_refusals():
    from stgcn_rt import functional as F, ops as P
    x = torch.zeros(4, 10)
    v, i, rest, lab = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4), torch.zeros(4, dtype=torch.int64)
    u = torch.zeros(4)
    V, R, TE = ValueError, RuntimeError, TypeError
    for exc, match, f in [
            (V, "rows, classes", lambda: F.top_logits(x[0], 3)),
            (TE, "float32 or bfloat16", lambda: F.top_logits(x.double(), 3)),
            (TE, "float32 or bfloat16", lambda: F.top_logits(x.half(), 3)),
            (V, "got k = 0", lambda: F.top_logits(x, 0)),
            (V, "got k = 11", lambda: F.top_logits(x, 11)),
            (V, "got k = 257", lambda: F.top_logits(torch.zeros(1, 400), 257)),
            (V, "classes", lambda: F.top_logits(torch.zeros(1, 0), 1)),
            (V, "classes", lambda: F.top_logits(torch.zeros(1, (1 << 20) + 1), 1)),
            (V, "2.24 rows", lambda: F.top_logits(x[:1].expand(1 << 24, 10), 3)),
            (V, "2.24 rows", lambda: F.sample_labels(x[:1].expand(1 << 24, 10), u[:1].expand(1 << 24))),
            (V, "temperature", lambda: F.top_logits(x, 3, temperature=0.0)),
            (V, "temperature", lambda: F.top_logits(x, 3, temperature=math.nan)),
            (R, "no CPU fallback", lambda: F.top_logits(x, 3)),
            (V, "values wants", lambda: F.distillation(x, v[:3], i)),
            (V, "values wants", lambda: F.distillation(x, v.double(), i)),
            (V, "values wants", lambda: F.distillation(x, torch.zeros(4, 257), torch.zeros(4, 257, dtype=torch.int64))),
            (V, "values wants", lambda: F.distillation(x, torch.zeros(4, 0), torch.zeros(4, 0, dtype=torch.int64))),
            (V, "indices wants", lambda: F.distillation(x, v, i.int())),
            (V, "indices wants", lambda: F.distillation(x, v, i[:, :2])),
            (V, "rest wants", lambda: F.distillation(x, v, i, rest=rest[:2])),
            (V, "labels wants", lambda: F.distillation(x, v, i, labels=lab.int(), label_weight=0.5)),
            (V, "wants labels", lambda: F.distillation(x, v, i, label_weight=0.5)),
            (V, "label_weight", lambda: F.distillation(x, v, i, labels=lab, label_weight=1.5)),
            (V, "label_weight", lambda: F.distillation(x, v, i, labels=lab, label_weight=math.nan)),
            (V, "temperature", lambda: F.distillation(x, v, i, temperature=-1.0)),
            (V, "reduction", lambda: F.distillation(x, v, i, reduction="batchmean")),
            (V, "no rows", lambda: F.distillation(x[:0], v[:0], i[:0])),
            (V, "one number", lambda: P.distillation(x, v, i, reduction="none")),
            (R, "no CPU fallback", lambda: F.distillation(x, v, i)),
            (V, "u wants", lambda: F.sample_labels(x, u[:3])),
            (V, "u wants", lambda: F.sample_labels(x, u.double())),
            (V, "temperature wants", lambda: F.sample_labels(x, u, temperature=-0.5)),
            (V, "temperature wants", lambda: F.sample_labels(x, u, temperature=torch.ones(3))),
            (V, "top_k wants", lambda: F.sample_labels(x, u, top_k=-1)),
            (V, "top_k wants", lambda: F.sample_labels(x, u, top_k=2.5)),
            (V, "top_k wants", lambda: F.sample_labels(x, u, top_k=torch.ones(4))),
            (V, "top_p wants", lambda: F.sample_labels(x, u, top_p=0.0)),
            (V, "top_p wants", lambda: F.sample_labels(x, u, top_p=1.1)),
            (V, "min_p wants", lambda: F.sample_labels(x, u, min_p=1.1)),
            (V, "min_p wants", lambda: F.sample_labels(x, u, min_p=math.nan)),
            (R, "no CPU fallback", lambda: F.sample_labels(x, u))]:
        with pytest.raises(exc, match=match):
            f()


def test_c_entry_points_refuse():
    """Status 1 before anything is launched: null pointers, sizes out of range, unknown types."""
    from stgcn_rt import lib as L
    l = L.load()
    p = 4096                                                   # never dereferenced by the host
    top = lambda dt=0, x=p, st=10, r=4, n=10, k=3, T=1.0: l.stgcn_top_logits(dt, x, st, r, n, k, T, p, p, p, None, 0, None)   # noqa: E731
    for kw in (dict(dt=7), dict(x=None), dict(st=9), dict(r=0), dict(n=0), dict(n=1 << 21, st=1 << 21), dict(k=0), dict(k=11), dict(T=0.0), dict(T=math.nan)):
        assert top(**kw) == 1, kw
    assert top(r=1 << 24) == 1 and top(r=1 << 30) == 1
    assert top(n=100000, st=100000) == 3                       # few rows want a workspace
    need = ctypes.c_size_t(7)
    assert l.stgcn_top_logits_workspace(4, 100000, 3, ctypes.addressof(need)) == 0 and need.value > 0
    assert l.stgcn_top_logits_workspace(4000, 100000, 3, ctypes.addressof(need)) == 0 and need.value == 0
    assert l.stgcn_top_logits_workspace(4, 100000, 300, ctypes.addressof(need)) == 1 and l.stgcn_top_logits_workspace(4, 10, 3, None) == 1
    fwd = lambda dt=0, x=p, st=10, v=p, i=p, lab=None, r=4, n=10, k=3, T=1.0, w=0.0, red=1, rows=p: l.stgcn_distill_fwd(      # noqa: E731
        dt, x, st, v, i, None, lab, r, n, k, T, w, red, p, rows, p, p, None)
    for kw in (dict(dt=2), dict(x=None), dict(st=9), dict(v=None), dict(i=None), dict(r=-1), dict(n=0), dict(k=257), dict(T=-1.0), dict(w=0.5), dict(w=1.5, lab=p),
               dict(red=3), dict(red=2, rows=None)):
        assert fwd(**kw) == 1, kw
    bwd = lambda dt=0, x=p, dx=p, stats=p, w=0.0, lab=None: l.stgcn_distill_bwd(dt, x, 10, p, lab, stats, p, None, 0, 1.0, 4, 10, 3, 1.0, w, dx, None)  # noqa: E731
    for kw in (dict(dt=3), dict(x=None), dict(dx=None), dict(stats=None), dict(w=0.5), dict(w=math.nan)):
        assert bwd(**kw) == 1, kw
    smp = lambda dt=0, x=p, st=10, u=p, out=p, r=4, n=10: l.stgcn_sample_labels(dt, x, st, u, None, 1.0, None, 0, None, 1.0, None, 0.0, out, p, r, n, None)  # noqa: E731
    for kw in (dict(dt=9), dict(x=None), dict(st=9), dict(u=None), dict(out=None), dict(r=0), dict(n=0), dict(n=1 << 21, st=1 << 21)):
        assert smp(**kw) == 1, kw


def test_plain_forms_agree_with_the_definitions():
    """The oracle itself: whole-list distillation is torch's KL divergence, its gradient torch's."""
    g = torch.Generator().manual_seed(0)
    t, s = torch.randn(3, 20, generator=g, dtype=torch.float64), torch.randn(3, 20, generator=g, dtype=torch.float64)
    v, i, rest = O.top_logits(t, 20, 2.0)
    assert bool((rest == -math.inf).all())
    lab = torch.tensor([1, 5, 19])
    loss, grad = O.distill(s, v, i, rest, lab, 2.0, 0.25)
    b = s.clone().requires_grad_(True)
    ref = 0.75 * 4 * torch.nn.functional.kl_div(torch.log_softmax(b / 2, 1), torch.softmax(t / 2, 1), reduction="none").sum(1) \
        + 0.25 * torch.nn.functional.cross_entropy(b, lab, reduction="none")
    ref.sum().backward()
    assert torch.allclose(loss, ref.detach(), rtol=1e-12, atol=1e-12) and torch.allclose(grad, b.grad, rtol=1e-12, atol=1e-12)
    v, i, rest = O.top_logits(t, 4, 2.0)
    loss, grad = O.distill(s, v, i, rest, None, 2.0, 0.0)
    b = s.clone().requires_grad_(True)
    lp, lq = torch.log_softmax(t / 2, 1), torch.log_softmax(b / 2, 1)
    m = torch.zeros(3, 20, dtype=torch.bool).scatter_(1, i, True)
    fold = lambda a: torch.cat([a.gather(1, i), a.masked_fill(m, -math.inf).logsumexp(1, keepdim=True)], 1)      # noqa: E731
    ref = 4 * (fold(lp).exp() * (fold(lp) - fold(lq))).sum()
    ref.backward()
    assert torch.allclose(loss.sum(), ref.detach(), rtol=1e-12) and torch.allclose(grad, b.grad, rtol=1e-11, atol=1e-13)
