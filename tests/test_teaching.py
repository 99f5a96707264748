"""A model that learns from another one's top scores: ddp.Trainer(teacher=...), evaluate.teacher_targets and
evaluate.pseudo_labels, launch by launch and from captured graphs."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from oracle import scores_oracle as S
from oracle import stgcn_oracle as O

DEV = "cuda:0"
U = 2.0 ** -24


@pytest.fixture(scope="module")
def st():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a GPU")
    import net.st_gcn as m
    return m


def model(st, tag, dtype=torch.float32, dropout=0.0):
    m = st.Model(3, 60, dict(layout="ntu-rgb+d", strategy="spatial"), True, dropout=dropout, compute_dtype=dtype).to(DEV)
    m.load_state_dict(O.det_state(3, 60, O.build_graph("ntu-rgb+d", "spatial")["A"], True, dtype=torch.float32), strict=True)
    g = torch.Generator().manual_seed(tag)
    with torch.no_grad():
        for p in m.parameters():
            p.add_((0.05 * torch.randn(p.shape, generator=g)).to(DEV) * p.abs().mean())
    return m.train()


def trainer(st, dtype=torch.float32, dropout=0.0, teacher=True, **kw):
    from stgcn_rt.ddp import Trainer
    torch.manual_seed(99)
    more = dict(teacher=model(st, 2, dtype)) if teacher else {}
    return Trainer(model(st, 1, dtype, dropout), lr=0.01, momentum=0.9, weight_decay=1e-4, nesterov=True, **more, **kw)


def clips(n, tag):
    return O.det_input(n, 3, 24, 25, 2, tag=tag).float().to(DEV)


LABELS = [4, -1, 33, 58]


@pytest.mark.gpu
@pytest.mark.parametrize("k,w", [(16, 0.5), (60, 0.0), (200, 1.0)])
def test_taught_step(st, k, w):
    """Loss and gradients of one step: the loss is the definition's of the two models' scores, the gradients are the
    model's backward of the operator's."""
    from stgcn_rt import functional as F
    tr = trainer(st, teacher_k=k, temperature=2.0, label_weight=w)
    x, lab = clips(4, 41), torch.tensor(LABELS, device=DEV)
    before = {n: v.clone() for n, v in tr.model.state_dict().items()}
    loss = tr.step(x, lab)
    got = tr.flat.grad.clone()
    assert not tr.teacher.training and all(p.grad is None for p in tr.teacher.parameters())
    tr.model.load_state_dict(before)
    out = tr.model(x)
    with torch.no_grad():
        teach = tr.teacher(x)
    v, i, rest = S.top_logits(teach.cpu(), min(k, 60), 2.0)
    rows, _ = S.distill(out.detach().cpu(), v.float(), i, rest.float(), lab.cpu(), 2.0, w)
    # 60 terms a sum and |y| <= 127 (tests/test_scores.py): es = 2^-23 + (2.1 * 127 + 60) 2^-24, in log S and log S_r of each
    # row (T^2 (1 - w) of them, w of the label's), and the rounding of c at |z| <= 127 T ln 2, of rest and of the mean
    es = 2.0 ** -23 + (2.1 * 127 + 60) * U
    tol = (4 * (1 - w) * 2 + w) * es + (4 * (1 - w) + w) * 127 * 2 * U + U * float(rows.abs().sum())
    assert abs(float(loss) - float(rows.mean())) < tol, (float(loss), float(rows.mean()))
    top = F.top_logits(teach, min(k, 60), 2.0)
    taught = F.distillation(out, *top, labels=lab, temperature=2.0, label_weight=w)
    (dout,) = torch.autograd.grad(taught, out, retain_graph=True)
    for p in tr.flat.params:
        p.grad = None
    out.backward(dout)
    want = torch.cat([p.grad.reshape(-1) for p in tr.flat.params])
    assert torch.equal(got, want) and bool(torch.isfinite(got).all()) and float(got.abs().max()) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_taught_steps_captured_and_replayed(st, dtype):
    """Seven steps on changing batches, with dropout: launch by launch, one graph, two graphs, and with the teacher's top
    logits handed over.  Every loss and every parameter ends the same, bit for bit."""
    from stgcn_rt import evaluate as E
    xs = [clips(4, 50 + i) for i in range(7)]
    labs = [torch.tensor([(v + 5 * i) % 60 if v >= 0 else -1 for v in LABELS], device=DEV) for i in range(7)]
    runs = []
    for kw, given in ((dict(), False), (dict(graph=True), False), (dict(graph=True, split=True), False), (dict(graph=True), True)):
        tr = trainer(st, dtype, 0.5, teacher=not given, teacher_k=10, temperature=3.0, label_weight=0.3, **kw)
        target = [None] * 7
        if given:
            whole = E.teacher_targets(model(st, 2, dtype), [(x, None) for x in xs], torch.device(DEV), k=10, temperature=3.0)
            assert whole.values.shape == (28, 10) and whole.values.device.type == "cpu"
            target = [tuple(t[4 * i:4 * i + 4].to(DEV) for t in whole) for i in range(7)]
        losses = []
        for x, lab, t in zip(xs, labs, target):
            print(kw, given, len(losses), flush=True)
            losses.append(float(tr.step(x, lab, target=t).detach()))
        assert tr.graph_segments() == (0 if not kw else 2 if "split" in kw else 1)
        runs.append((losses, tr.flat.flat.clone()))
    for losses, params in runs[1:]:
        assert losses == runs[0][0] and torch.equal(params, runs[0][1])


@pytest.mark.gpu
def test_a_graph_keeps_to_its_loss(st):
    """One trainer, steps with and without a target and at another temperature: each is captured by itself, and agrees
    with the eager step on the same state."""
    from stgcn_rt import evaluate as E
    x, lab = clips(4, 60), torch.tensor([4, 9, 33, 58], device=DEV)
    top = tuple(t.to(DEV) for t in E.teacher_targets(model(st, 2), [(x, lab)], torch.device(DEV), k=5))
    tr = trainer(st, teacher=False, graph=True)
    tr.opt.lr, tr.opt.weight_decay = 0.0, 0.0                        # the parameters stay
    seen = []
    for _ in range(5):
        for t, temp in ((None, 2.0), (top, 2.0), (top, 4.0), ((top[0], top[1], None), 2.0)):
            tr.temperature = temp
            print(len(seen), flush=True)
            seen.append(float(tr.step(x, lab, target=t).detach()))
    assert len(tr._graphs) == 4
    for j in range(4):
        assert len(set(seen[j::4])) == 1, seen
    assert len(set(seen[:4])) == 4


@pytest.mark.gpu
def test_pseudo_labels(st):
    from stgcn_rt import evaluate as E
    m = model(st, 3)
    x = clips(6, 70)
    dev = torch.device(DEV)
    batches = [(x[:4], torch.zeros(4)), (x[4:], torch.zeros(2))]
    res = E.evaluate(m, batches, dev, evaluation=False)["result"]
    best = E.pseudo_labels(m, batches, dev, temperature=0.0)
    assert (best["label"] == res.argmax(1)).all() and (best["logp"] == 0).all()
    got = E.pseudo_labels(m, batches, dev, temperature=1.5, top_k=20, top_p=0.9, generator=torch.Generator().manual_seed(5))
    u = torch.rand(6, generator=torch.Generator().manual_seed(5))
    lab, lp = S.sample(torch.from_numpy(res), u, 1.5, 20, 0.9, 0.0)
    assert torch.equal(torch.from_numpy(got["label"]), lab)
    # 64-bit weights and sums, one rounding to 32 bits
    assert bool(((torch.from_numpy(got["logp"]).double() - lp).abs() <= U * lp.abs() + 1e-10).all())


def test_refusals():
    from stgcn_rt.ddp import Trainer
    import net.st_gcn as st
    g = dict(layout="ntu-rgb+d", strategy="spatial")
    a, b = st.Model(3, 60, g, True), st.Model(3, 60, g, True)
    for kw in (dict(teacher=a), dict(teacher=torch.nn.Sequential(a)), dict(teacher=b, teacher_k=0), dict(teacher=b, teacher_k=257),
               dict(teacher=b, temperature=0.0), dict(teacher=b, label_weight=1.5), dict(label_weight=float("nan"))):
        with pytest.raises(ValueError, match="teacher"):
            Trainer(a, **kw)
    tr = Trainer(a)
    with pytest.raises(ValueError, match="target"):
        tr.step(torch.zeros(1), torch.zeros(1), target=(torch.zeros(1, 1), torch.zeros(1, 1)))


def _teacher_worker(rank, port, out):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=2)
    import net.st_gcn as st
    from stgcn_rt.ddp import Trainer
    torch.manual_seed(10 + rank)
    g = dict(layout="ntu-rgb+d", strategy="spatial")
    tr = Trainer(st.Model(3, 7, g, True), teacher=st.Model(3, 7, g, True))
    tr.broadcast_from_rank0()
    torch.save([t.clone() for m in (tr.model, tr.teacher) for t in list(m.parameters()) + list(m.buffers())], "%s%d" % (out, rank))
    dist.destroy_process_group()


def test_every_rank_learns_from_the_same_teacher(tmp_path):
    """Two gloo ranks with different seeds: model and teacher are rank 0's afterwards."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_teacher_worker, args=(port, str(tmp_path / "t")), nprocs=2, join=True)
    a, b = (torch.load(str(tmp_path / "t") + str(r), weights_only=True) for r in (0, 1))
    assert len(a) == len(b) > 100 and all(torch.equal(x, y) for x, y in zip(a, b))
