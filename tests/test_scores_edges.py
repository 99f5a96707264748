"""Operators over class scores where their formulas, maps and sums reach an end: wide gaps between scores, NaN in every
place, rows longer than one segment of the bit map, long sums, infinite incoming gradients.  Tolerances as in
tests/test_scores.py, derived at each check."""
import os
import subprocess

import pytest
import torch

from oracle import scores_oracle as O
from tests.test_scores import DEV, U, check_sample, eps_sum, half_step, rt, scores, teacher_lists  # noqa: F401  (rt: a fixture)

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "st-gcn_amd", "csrc")


# ---- bit map of the listed classes (CPU) ---------------------------------------------------------------------------

MAP = """
#include "%s/listed_map.h"
#include <cstdio>
int main() {
    long bad = 0;
    for (int n = 1; n <= 1 << 20; ++n) {
        const int some = segment_words(n), last = n < SEG ? n - 1 : SEG - 1;     // words cleared; last class of a segment from its base on
        if (some > SEG_WORDS) ++bad;                                            // cleared beyond the map
        if ((BIT0 + last) / 32 >= some) ++bad;                                  // looked at, not cleared
    }
    printf("%%ld %%d", bad, (int)(SEG_WORDS * 4 >= (BIT0 + SEG + 7) / 8));       // the bytes of every vector of a segment are the map's
}
"""


def test_the_bit_map_of_a_segment_holds_what_is_cleared_and_read(tmp_path):
    src, exe = tmp_path / "map.cpp", tmp_path / "map"
    src.write_text(MAP % CSRC)
    subprocess.check_call(["g++", "-std=c++17", "-O1", str(src), "-o", str(exe)])
    assert subprocess.check_output([str(exe)], text=True) == "0 1"


# ---- build (CPU) ---------------------------------------------------------------------------------------------------

def test_a_change_of_flags_builds_every_object_again():
    """Old objects, made with packed float32 instructions, must not be linked into a library whose flags leave them out.  (A dry run.)"""
    sources = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))
    plan = subprocess.check_output(["make", "-C", CSRC, "-n", "-W", "Makefile"], text=True)
    built = [line.split(" -c ")[1].split()[0] for line in plan.splitlines() if " -c " in line]
    assert sorted(built) == sources
    assert all("-packed-fp32-ops" in line for line in plan.splitlines() if " -c " in line)


# ---- refusals (CPU) ------------------------------------------------------------------------------------------------

def test_temperatures_without_a_32_bit_inverse_are_refused():
    """log2(e) / T beyond float32 would make NaN of 0 * inf: both ends, through the operators and the C entries."""
    from stgcn_rt import functional as F, lib as L
    from stgcn_rt.ddp import Trainer
    import net.st_gcn as m
    x, v, i = torch.zeros(4, 10), torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    l, p = L.load(), 4096                                      # p: never dereferenced by the host
    net = [m.Model(3, 7, dict(layout="ntu-rgb+d", strategy="spatial"), True) for _ in range(2)]
    for T in (1e-30, 1e-39, 1e-45, 5e-324, 1e30, 1e300):
        for f in (lambda: F.top_logits(x, 3, temperature=T), lambda: F.distillation(x, v, i, temperature=T), lambda: Trainer(net[0], teacher=net[1], temperature=T)):
            with pytest.raises(ValueError, match="temperature"):
                f()
        assert l.stgcn_top_logits(0, p, 10, 4, 10, 3, T, p, p, p, None, 0, None) == 1
        assert l.stgcn_distill_fwd(0, p, 10, p, p, None, None, 4, 10, 3, T, 0.0, 1, p, p, p, p, None) == 1
        assert l.stgcn_distill_step(0, p, 10, p, p, None, None, 4, 10, 3, T, 0.0, 1, p, p, p, p, p, None) == 1
        assert l.stgcn_distill_bwd(0, p, 10, p, None, p, p, None, 0, 1.0, 4, 10, 3, T, 0.0, p, None) == 1
    for T in (1.1e-30, 0.9e30):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            F.top_logits(x, 3, temperature=T)


# ---- distillation over selected rows -------------------------------------------------------------------------------

def row_parts(x, val, idx, rho, label, T, w, es):
    """(sizes of a gradient's parts [n], tolerance of the loss) of one live row x (float64).  The loss: log S and log S_r enter
    with weight 1 and p_r (es each); the listed classes' z, and log S_r's own maximum, with the rounding of c (2^-24)."""
    x = x - x.max()
    q, size = torch.zeros_like(x), 0.0
    tea = O.teacher(val, idx, rho, T) if w < 1 else None
    if tea is not None:
        z = x / T
        S = O.lse(z)
        other = torch.ones(x.numel(), dtype=torch.bool)
        other[tea[2]] = False
        So = O.lse(z[other])
        qz = torch.exp(z - S)
        q += (1 - w) * T * qz
        if tea[1] > 0 and So > -float("inf"):
            q[other] += (1 - w) * T * tea[1] * torch.exp(z[other] - So)
            size += (1 - w) * T * T * tea[1] * (abs(float(z[other].max())) * U + es)
        for i, p in tea[0]:
            q[i] += (1 - w) * T * p
            size += (1 - w) * T * T * p * abs(float(z[i])) * U
        size += (1 - w) * T * T * es
    if w > 0 and label is not None and label >= 0:
        q += w * torch.exp(x - O.lse(x))
        q[label] += w
        size += w * (es + abs(float(x[label])) * U)
    return q, size


def close(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.double()
    nan, inf = torch.isnan(want), torch.isinf(want)
    assert torch.equal(torch.isnan(got), nan), (what, got, want)
    assert torch.equal(got[inf], want[inf]), (what, got, want)
    ok = ~(nan | inf)
    bad = ((got - want).abs() > torch.broadcast_to(tol, want.shape)) & ok
    assert not bool(bad.any()), (what, got[bad][:5], want[bad][:5], torch.broadcast_to(tol, want.shape)[bad][:5])


def check_rows(rt, x, val, idx, rest, labels, T, w, sel=None):
    """Losses and gradients of the rows `sel` (all): the loss with its backward, and the pair."""
    F, P = rt
    rows, n = x.shape
    sel = list(range(rows)) if sel is None else sel
    more = dict(rest=rest, labels=labels, temperature=T, label_weight=w)
    leaf = x.detach().requires_grad_(True)
    loss = F.distillation(leaf, val, idx, reduction="none", **more)
    (dx,) = torch.autograd.grad(loss, leaf, torch.full((rows,), -1.25, device=DEV))
    _, pair = P.distillation(x, val, idx, reduction="sum", **more)
    got, dx, pair = loss[sel].detach().cpu(), dx[sel].cpu(), pair[sel].cpu()
    xs, val, idx = x[sel].detach().float().cpu(), val[sel].cpu(), idx[sel].cpu()
    rest, labels = (None if t is None else t[sel].cpu() for t in (rest, labels))
    L, G = O.distill(xs, val, idx, rest, labels, T, w)
    es = eps_sum(xs, T)
    e1 = es + (8 + (es - 2.0 ** -23) / U) * U
    hs, flush = half_step(x.dtype), 2.0 ** -125 * max(1.0, T)         # e, and its product with a factor below 2 T, may be flushed
    for r in range(len(sel)):
        q, size = torch.zeros(n, dtype=torch.float64), 0.0
        if bool(torch.isfinite(L[r])) and float(xs[r].max()) > -float("inf"):
            q, size = row_parts(xs[r].double(), val[r], idx[r], None if rest is None else float(rest[r]), None if labels is None else int(labels[r]), T, w, es)
        what = (x.dtype, rows, n, T, w, "row", sel[r])
        close(got[r], L[r], torch.tensor(size + U * (abs(float(L[r])) if bool(torch.isfinite(L[r])) else 0.0) + 1e-12), what + ("loss",))
        for g, f in ((dx, -1.25), (pair, 1.0)):
            close(g[r], G[r] * f, q * e1 * abs(f) + hs * torch.nan_to_num(G[r] * f).abs() + flush, what + ("gradient", f))


DTS = pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


@pytest.mark.gpu
@DTS
@pytest.mark.parametrize("rows,n", [(513, 140001), (1, 270000), (3, 131072)])
def test_distillation_over_several_segments(rt, rows, n, dt):
    """Classes on both sides of every border of the bit map, with the same class in the list twice."""
    x = scores(rows, n, dt, n, offset=3, gap=2)
    val, idx, rest = teacher_lists(x[:3], 12, 2.0, 1)
    most = torch.tensor([131060, 131071, n - 1, min(n - 1, 131072), min(n - 1, 131080), min(n - 2, 262143), 0, 5], device=DEV)
    idx[:, 4:] = most
    val, idx, rest = (torch.cat([t] * (rows // t.shape[0] + 1))[:rows].contiguous() for t in (val, idx, rest))
    labels = torch.arange(rows, device=DEV) * 251 % n
    labels[0] = 131071
    sel = sorted({0, rows // 2, rows - 1})
    for T, w in ((2.0, 0.3), (1.0, 0.0)):
        print("segments", rows, n, dt, T, w, flush=True)
        check_rows(rt, x, val, idx, rest, labels, T, w, sel)


@pytest.mark.gpu
@DTS
@pytest.mark.parametrize("rows,n,k", [(3, 20, 2), (4, 400, 5), (2, 1500, 70), (2, 5000, 8), (1, 140001, 4), (514, 9001, 8)])
def test_distillation_gap_between_listed_and_others(rt, rows, n, k, dt):
    """A student far surer of the listed classes than of the others, and the other way: each side's sum is its own, however
    far the other's maximum lies above it."""
    for j, (gap, T, w) in enumerate([(90.0, 1.0, 0.0), (200.0, 0.7, 0.3), (1e4, 1.0, 0.0), (1e4, 4.0, 0.5), (95.0, 1.0, 0.4), (61.0, 0.7, 0.0), (350.0, 4.0, 0.0),
                                     (-90.0, 1.0, 0.0), (-1e4, 2.0, 0.3)]):
        print("gap", rows, n, k, dt, gap, T, w, flush=True)
        x = scores(rows, n, dt, n + j, sigma=1.0, offset=1)
        val, idx, _ = teacher_lists(x, k, T, j)
        x.scatter_add_(1, idx, torch.full(idx.shape, gap, dtype=dt, device=DEV))
        # the teacher's rest: 0.3 of its mass
        rest = torch.logsumexp(val / T, 1) - 0.85
        labels = torch.arange(rows, device=DEV) * 7 % n
        labels[0] = idx[0, 0]
        check_rows(rt, x, val, idx, rest, labels, T, w, sorted({0, 1 % rows, rows - 1}))


@pytest.mark.gpu
def test_distillation_gap_gradient_against_differences(rt):
    """Central differences of the 64-bit loss where e^z of the others would vanish next to the listed ones'."""
    x = scores(2, 40, torch.float32, 3, sigma=0.7)
    val, idx, _ = teacher_lists(x, 3, 1.0, 1)
    x.scatter_add_(1, idx, torch.full(idx.shape, 120.0, device=DEV))
    rest = torch.logsumexp(val, 1) - 0.5
    _, dx = rt[1].distillation(x, val, idx, rest=rest, reduction="sum")
    h = 1e-4
    for r in range(2):
        for j in range(40):
            f = []
            for s in (h, -h):
                xx = x[r].cpu().double()
                xx[j] += s
                f.append(O.distill_row(xx, val[r].cpu(), idx[r].cpu(), float(rest[r]), None, 1.0, 0.0)[0])
            # the difference's own error: h^2 / 6 times a third derivative below 1, and 2^-52 |loss| / h (loss < 100); the gradient's: parts of 1
            # at most, es = 2^-23 + (2.1 * 127 + 40) 2^-24 and its 8 roundings
            assert abs(float(dx[r, j]) - (f[0] - f[1]) / (2 * h)) < h * h + 100 * 2.0 ** -52 / h + 2 * (2.1 * 127 + 50) * U, (r, j)


@pytest.mark.gpu
@DTS
@pytest.mark.parametrize("rows,n,k", [(5, 61, 1), (5, 400, 5), (5, 512, 200), (5, 5000, 16), (5, 20011, 100), (5, 70001, 256), (515, 5000, 33)])
def test_top_logits_many_nan(rt, rows, n, k, dt):
    """NaN come first, by class, however many there are; one that is not listed makes the rest NaN."""
    x = scores(rows, n, dt, n + k)
    g = torch.Generator().manual_seed(k)
    x[0] = float("nan")
    x[1, torch.randperm(n, generator=g)[:n // 2].to(DEV)] = float("nan")
    x[2, torch.randperm(n, generator=g)[:k].to(DEV)] = float("nan")
    x[3, n // 2:] = float("nan")
    x[4, torch.randperm(n, generator=g)[:k + 1].to(DEV)] = float("nan")
    x[rows - 1, ::3] = -x[rows - 1, ::3].abs() * float("nan")
    got = rt[0].top_logits(x, k, 2.0)
    sel = [0, 1, 2, 3, 4, rows - 1]
    xc = x[sel].float().cpu()
    v, i, rest = O.top_logits(xc, k, 2.0)                    # its rest passes NaN over
    left = torch.ones_like(xc, dtype=torch.bool).scatter_(1, i, False)
    rest[(torch.isnan(xc) & left).any(1)] = float("nan")
    assert torch.equal(got.indices[sel].cpu(), i)
    assert torch.equal(torch.nan_to_num(got.values[sel].cpu().double(), nan=5.0), torch.nan_to_num(v, nan=5.0))
    g = got.rest[sel].cpu().double()
    assert torch.equal(torch.isnan(g), torch.isnan(rest))
    ok = torch.isfinite(rest)
    # log of S (EPS_S), the maximum over T in 64 bits, one rounding to 32
    assert bool(((g[ok] - rest[ok]).abs() <= eps_sum(x[2:3], 2.0) + 2.0 ** -23 + U * rest[ok].abs()).all()), (g, rest)


@pytest.mark.gpu
@DTS
@pytest.mark.parametrize("n", [60, 401, 5000, 140001])
@pytest.mark.parametrize("k", [1, 4])
def test_distillation_nan_on_every_listed_class(rt, n, k, dt):
    """A NaN score makes its row NaN wherever it stands: on all listed classes, on some, twice in the list, next to -inf."""
    for T, w in ((1.0, 0.0), (2.0, 0.5), (1.0, 1.0), (2.0, 1.0)):
        for others in (0.0, -float("inf")):
            print("nan", n, k, dt, T, w, others, flush=True)
            x = scores(5, n, dt, n)
            val, idx, rest = teacher_lists(x, k, T, 1)
            if others:
                x[:4].fill_(others)
            x[0].scatter_(0, idx[0], float("nan"))
            x[1, idx[1, k - 1]] = float("nan")
            idx[2] = int(idx[2, 0])
            x[2, idx[2, 0]] = float("nan")
            x[3].scatter_(0, idx[3], -float("inf"))
            x[3, idx[3, 0]] = float("nan")
            labels = torch.arange(5, device=DEV)
            labels[0] = idx[0, 0]
            check_rows(rt, x, val, idx, rest, labels, T, w)


@pytest.mark.gpu
@DTS
@pytest.mark.parametrize("rows,n", [(6, 60), (5, 401), (3, 400001)])
def test_distillation_padding_takes_no_gradient(rt, rows, n, dt):
    """Rows without entries and label keep a gradient of zero whatever comes in: infinite, NaN."""
    F, _ = rt
    x = scores(rows, n, dt, 1)
    val, idx, rest = teacher_lists(x, 4, 2.0, 1)
    labels = torch.arange(rows, device=DEV)
    idx[1:] = -1
    labels[2:] = -1
    for red, up in [("none", float("inf")), ("none", float("nan")), ("mean", float("inf")), ("sum", float("nan")), ("mean", 3.0)]:
        leaf = x.detach().requires_grad_(True)
        loss = F.distillation(leaf, val, idx, rest=rest, labels=labels, temperature=2.0, label_weight=0.5, reduction=red)
        (dx,) = torch.autograd.grad(loss, leaf, torch.full_like(loss, up))
        assert dx.dtype == dt and bool((dx[2:] == 0).all()), (red, up)
        # what has an entry or a label takes it
        assert bool(torch.isfinite(dx[:2]).all()) == (up == 3.0) and bool((dx[:2] != 0).any(1).all())
    # a second backward of one loss, with another gradient, leaves the first one's result as it is
    leaf = x.detach().requires_grad_(True)
    loss = F.distillation(leaf, val, idx, rest=rest, labels=labels, temperature=2.0, label_weight=0.5)
    first, second = (torch.autograd.grad(loss * f, leaf, retain_graph=True)[0] for f in (2.0, 4.0))
    assert first.data_ptr() != second.data_ptr() and torch.equal(first * 2, second)


@pytest.mark.gpu
@DTS
def test_long_rows_add_up(rt, dt):
    """The most classes, in rows that few threads share: every thread sees one, then thousands of e^{(x - max) / T} that lie a
    little above a half, which a sum of 32 bits between 1024 and 2048 would lose the little of at each step (2^-14 of 2^-13
    steps: a thousand units of the sum's last place).  Bound: the chain of tests/test_scores.py."""
    F, P = rt
    import math
    rows, n, k = 512, 1 << 20, 2
    low = -0.69140625                                               # a bf16 number
    T = low / math.log(0.5 + 0.98 * 2.0 ** -14)
    row = torch.full((n,), low)
    row[:1 << 14] = 0.0                                             # every thread's first vectors
    row[torch.tensor([77777, 999999])] = 3.0
    x = row.to(dt).to(DEV).expand(rows, n).contiguous()
    some = row[None].double()
    check = [0, rows - 1]
    top = F.top_logits(x, k, T)
    v, i, rest = O.top_logits(some, k, T)
    assert torch.equal(top.indices[check].cpu(), i.expand(2, k))
    es = eps_sum(some, T)
    assert bool(((top.rest[check].cpu().double() - rest).abs() <= es + U * abs(float(rest))).all()), (top.rest[check], rest, es)
    up = torch.linspace(-9, 9, n).to(dt)                            # every batch is earlier in the order than those before it
    got = F.top_logits(up.to(DEV).expand(rows, n).contiguous(), 64, 2.0)
    v, i, rest = O.top_logits(up[None].double(), 64, 2.0)
    assert torch.equal(got.indices[check].cpu(), i.expand(2, 64)) and torch.equal(got.values[check].cpu().double(), v.expand(2, 64))
    assert bool(((got.rest[check].cpu().double() - rest).abs() <= eps_sum(up[None], 2.0) + U * abs(float(rest))).all()), (got.rest[check], rest)
    val = torch.tensor([[1.0, 0.5]], device=DEV).expand(rows, k).contiguous()
    tr = torch.full((rows,), 0.7, device=DEV)
    check_rows(rt, x, val, top.indices, tr, None, T, 0.0, check)
    check_rows(rt, x, val, top.indices, tr, torch.full((rows,), 5, device=DEV), T, 0.5, [1])


@pytest.mark.gpu
@DTS
def test_the_ends_of_the_temperatures(rt, dt):
    """As good as a maximum, and as good as equal shares: finite numbers, no NaN."""
    F, P = rt
    x = scores(6, 700, dt, 5)
    for T in (1.1e-30, 1e-20, 0.9e30):
        print("ends", dt, T, flush=True)
        top = F.top_logits(x, 3, T)
        v, i, rest = O.top_logits(x.float().cpu(), 3, T)
        assert torch.equal(top.indices.cpu(), i)
        # log of S: at most log 700, one rounding; beyond float32's range its infinity
        want = rest.float().double()
        assert bool((torch.isinf(want) == torch.isinf(top.rest.cpu())).all())
        ok = torch.isfinite(want)
        assert bool(((top.rest.cpu().double() - want).abs()[ok] <= 2 * U * want.abs()[ok] + eps_sum(x, 1.0)).all())
        for more in (None, top.rest):
            if more is None or bool(torch.isfinite(more).all()):
                loss, dx = P.distillation(x, top.values, top.indices, rest=more, temperature=T)
                assert not bool(torch.isnan(dx).any()) and not bool(torch.isnan(loss))


@pytest.mark.gpu
@DTS
def test_distillation_small_temperatures(rt, dt):
    """The teacher's t / T are thousands to 1e20 then; differences of scores are what counts of them."""
    F, P = rt
    x = scores(6, 700, dt, 5)
    for T, w in ((1e-3, 0.3), (1e-6, 0.0)):                     # small ones, where 64 bits still tell
        print("small", dt, T, flush=True)
        val, idx, rest = teacher_lists(x, 5, T, 3)
        for more in (None, rest, torch.logsumexp(val / T, 1) + 0.5):
            check_rows(rt, x, val, idx, more, torch.arange(6, device=DEV), T, w)
    top = F.top_logits(x, 3, 1e-20)
    loss, dx = P.distillation(x, top.values, top.indices, temperature=1e-20)
    assert not bool(torch.isnan(dx).any()) and not bool(torch.isnan(loss))


@pytest.mark.gpu
@pytest.mark.parametrize("n,dt", [(1 << 20, torch.float32), ((1 << 20) - 1, torch.bfloat16)])
def test_the_most_classes(rt, n, dt):
    """Few rows, which are split or have sixteen waves, and many, of which some are looked at."""
    F, _ = rt
    cuts = [(1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.0, 300000, 1.0, 0.0), (1.0, 40, 0.8, 0.0), (2.0, 0, 0.5, 0.02), (1.5, n - 5, 0.999, 0.0)]
    for j, (rows, sel) in enumerate(((2, [1]), (260, [131]))):
        x = scores(2, n, dt, n + rows, sigma=2.5, offset=1)
        if rows > 2:
            x = torch.cat([x, x[:1].expand(rows - 3, n), -x[:1]])
        got = F.top_logits(x, 200, 2.0)
        xc = x[sel].float().cpu()
        v, i, rest = O.top_logits(xc, 200, 2.0)
        assert torch.equal(got.indices[sel].cpu(), i) and torch.equal(got.values[sel].cpu().double(), v)
        assert bool(((got.rest[sel].cpu().double() - rest).abs() <= eps_sum(xc, 2.0) + U * rest.abs()).all())
        val, idx, tr = teacher_lists(x[sel], 20, 2.0, 1)
        val, idx, tr = (torch.zeros((rows,) + t.shape[1:], dtype=t.dtype, device=DEV).index_copy(0, torch.tensor(sel, device=DEV), t) for t in (val, idx, tr))
        check_rows(rt, x, val, idx, tr, torch.full((rows,), n - 1, device=DEV), 2.0, 0.3, sel)
        u = torch.full((rows,), 0.61, device=DEV)
        for T, k, p, q in cuts[j::2]:
            print("most", n, dt, rows, T, k, p, q, flush=True)
            lab, lp = F.sample_labels(x, u, T, k, p, q)
            want, wp = O.sample(xc, u[sel].cpu(), T, k, p, q)
            assert torch.equal(lab[sel].cpu(), want)
            # 64-bit weights and sums (1e-11 over a row), one rounding to 32 bits
            assert bool(((lp[sel].cpu().double() - wp).abs() <= U * wp.abs() + 1e-10).all())


@pytest.mark.gpu
@DTS
@pytest.mark.parametrize("rows,n,k", [(4, 61, 3), (4, 400, 60), (4, 9001, 16), (4, 70001, 200), (515, 5000, 20)])
def test_top_logits_many_infinities(rt, rows, n, k, dt):
    """More +inf than are listed, and with NaN and -inf among them: listed by class, the rest +inf, or NaN."""
    x = scores(rows, n, dt, n + k)
    inf = float("inf")
    x[0], x[1, ::2], x[1, 1::2] = inf, inf, -inf
    x[2, n // 3:] = inf
    x[3, ::3] = inf
    x[3, 1], x[3, n - 1] = float("nan"), float("nan")
    got = rt[0].top_logits(x, k)
    xc = x[:4].float().cpu()
    v, i, _ = O.top_logits(xc, k, 1.0)
    left = torch.ones_like(xc, dtype=torch.bool).scatter_(1, i, False)
    assert torch.equal(got.indices[:4].cpu(), i)
    assert torch.equal(torch.nan_to_num(got.values[:4].cpu().double(), nan=5.0, posinf=6.0), torch.nan_to_num(v, nan=5.0, posinf=6.0))
    want = [float("nan") if bool((torch.isnan(a) & b).any()) else inf if bool(((a == inf) & b).any()) else None for a, b in zip(xc, left)]
    assert want[:3] == [inf] * 3
    for g, w in zip(got.rest[:4].tolist(), want):
        assert g == w or (w != w and g != g) or w is None, (g, w)


@pytest.mark.gpu
@DTS
@pytest.mark.parametrize("rows,n", [(7, 25), (5, 400), (4, 600), (4, 9001), (270, 9001), (3, 70001)])
def test_sample_labels_at_zero(rt, rows, n, dt):
    """u = 0: the first kept class, by class number, however little it weighs next to the row's largest."""
    for j, (T, k, p, q) in enumerate([(1.0, 0, 1.0, 0.0), (1.0, n // 2 + 1, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 20, 0.999, 0.0), (2.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 1e-12),
                                      (1.0, n - 3, 1.0, 1e-30)][::3 if rows > 200 else 1]):
        print("zero", rows, n, dt, T, k, p, q, flush=True)
        x = scores(rows, n, dt, n + j, sigma=15.0, offset=j)
        check_sample(rt[0], x, torch.zeros(rows, device=DEV), T, k, p, q)


@pytest.mark.gpu
@DTS
@pytest.mark.parametrize("rows,n,down", [(2, 1 << 20, 26.0), (2, 140001, 16.0), (300, 20011, 22.0), (2, 5000, 25.0)])
def test_sample_labels_among_many_small_ones(rt, rows, n, down, dt):
    """One class with nearly all of the mass and a flat tail of all others, in which the border of top-p lies and u falls: each of
    them decides, and each weighs next to nothing beside the first."""
    g = torch.Generator().manual_seed(n)
    x = torch.randn(rows, n, generator=g) * 0.3 - down
    x[1:] = x[1:].round()                                       # equal ones too
    x[:, n - 1] = 0.0                                           # the last class: the tail comes first
    x = x.to(dt).to(DEV)
    w = torch.exp(x[:2].double()).sum(1) - 1.0                  # the tail's mass
    sel = [0, 1]
    xc = x[sel].float().cpu()
    for share, at in ((0.5, 0.4), (0.9, 0.77)):
        # p: the first class and `share` of the tail; u: `at` of that
        p = ((1.0 + share * w) / (1.0 + w)).float()
        u = (at * share * w).float()
        full = lambda t: t.repeat((rows + 1) // 2)[:rows].contiguous()                      # noqa: E731
        print("small", rows, n, down, dt, share, p.tolist(), u.tolist(), flush=True)
        lab, lp = rt[0].sample_labels(x, full(u), top_p=full(p))
        want, wp = O.sample(xc, u.cpu(), 1.0, 0, p.cpu(), 0.0)
        assert torch.equal(lab[sel].cpu(), want), (lab[sel], want)
        assert bool(((lp[sel].cpu().double() - wp).abs() <= U * wp.abs() + 1e-10).all()), (lp[sel], wp)
