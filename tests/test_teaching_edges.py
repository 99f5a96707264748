"""Learning from a teacher over a long run: temperatures and label weights that change, targets that do not fit."""
import pytest
import torch

from tests.test_teaching import DEV, LABELS, clips, model, st, trainer  # noqa: F401  (st: a fixture)


def cpu_trainer(**kw):
    import net.st_gcn as m
    from stgcn_rt.ddp import Trainer
    return Trainer(m.Model(3, 7, dict(layout="ntu-rgb+d", strategy="spatial"), True), **kw)


def test_graphs_of_passed_temperatures_are_dropped():
    """A stand-in for the capture: of one shape the graphs used last stay, other shapes and steps without a target keep theirs."""
    tr = cpu_trainer(graph=True)
    made = []
    tr._capture = lambda d, l, t: made.append((tr.temperature, tr.label_weight)) or ((object(),) + (d, l, t, None))
    x, lab = torch.zeros(2, 3, 4, 25, 1), torch.zeros(2, dtype=torch.int64)
    top = (torch.zeros(2, 5), torch.zeros(2, 5, dtype=torch.int64), torch.zeros(2))
    plain, other = tr._graph_for(x, lab, None), tr._graph_for(x[:1], lab[:1], tuple(t[:1] for t in top))
    kept = tr.GRAPHS_KEPT
    for i in range(20):
        tr.temperature, tr.label_weight = 4.0 - 0.1 * (i // 2), 0.5 + 0.01 * (i % 2)
        first = tr._graph_for(x, lab, top)
        assert tr._graph_for(x, lab, top) is first
        assert len(tr._graphs) <= kept + 2
    assert len(made) == 22 and len(tr._graphs) == kept + 2
    tr.temperature, tr.label_weight = made[-kept]                    # the oldest that is there: used again, it outlives the next ones
    first = tr._graph_for(x, lab, top)
    for i in range(kept - 1):
        tr.temperature = 1.0 - 0.1 * i
        tr._graph_for(x, lab, top)
    tr.temperature, tr.label_weight = made[22 - kept]
    assert tr._graph_for(x, lab, top) is first and len(made) == 22 + kept - 1
    tr.temperature, tr.label_weight = 2.0, 0.5
    assert tr._graph_for(x, lab, None) is plain and tr._graph_for(x[:1], lab[:1], tuple(t[:1] for t in top)) is other


def test_a_value_is_captured_from_its_second_step_on():
    tr = cpu_trainer(graph=True)
    top = (torch.zeros(2, 5),)
    assert tr._settled(None) and tr._settled(None)
    assert not tr._settled(top) and tr._settled(top)
    for i in range(50):                                              # annealed at every step: never
        tr.temperature = 4.0 - 0.05 * i if i else 5.0
        assert not tr._settled(top)
    assert len(tr._met) <= 2 * tr.GRAPHS_KEPT
    tr.temperature = 2.0
    assert not tr._settled(top) and tr._settled(top)


def test_targets_that_do_not_fit_are_refused():
    """Before anything runs, with a graph and without: a replay would cast, broadcast or move what it copies."""
    x, lab = torch.zeros(2, 3, 4, 25, 1), torch.zeros(2, dtype=torch.int64)
    v, i, r = torch.zeros(2, 5), torch.zeros(2, 5, dtype=torch.int64), torch.zeros(2)
    for graph in (False, True):
        tr = cpu_trainer(graph=graph)
        tr._eager_steps = tr._taught_steps = 5
        tr._capture = lambda *a: pytest.fail("captured")
        for target, match in [((v.double(), i, r), "values"), ((v[:1], i, r), "values"), ((v, i.int(), r), "indices"), ((v, i[:, :4], r), "indices"),
                              ((v, i, r.double()), "rest"), ((v, i, r[:1]), "rest"), ((v, None, r), "a target"), ((None, i, r), "a target"), ((v[0], i, r), "a target"),
                              ((v.tolist(), i, r), "a target"), ((v, i), "a target")]:
            for f in (lambda: tr.step(x, lab, target=target), lambda: tr.prepare_graph(x, lab, target=target)):
                with pytest.raises(ValueError, match=match):
                    f()
        for label in (lab.int(), lab.float(), lab[:1]):
            with pytest.raises(ValueError, match="labels"):
                tr.step(x, label, target=(v, i, r))
        with pytest.raises(ValueError, match="wants labels"):
            tr.step(x, None, target=(v, i, r))
        with pytest.raises(RuntimeError, match="target values lives on"):
            tr.step(x, lab, target=(v.to("meta"), i, r))


def test_values_set_between_steps_are_checked():
    """As in the constructor, before a step runs or is captured (a capture that fails would switch graphs off)."""
    x, lab = torch.zeros(2, 3, 4, 25, 1), torch.zeros(2, dtype=torch.int64)
    top = (torch.zeros(2, 5), torch.zeros(2, 5, dtype=torch.int64), torch.zeros(2))
    for name, value in (("temperature", 0.0), ("temperature", float("nan")), ("temperature", -1.0), ("label_weight", 1.5), ("label_weight", float("nan"))):
        tr = cpu_trainer(graph=True)
        tr._eager_steps = tr._taught_steps = 5
        tr._capture = lambda *a: pytest.fail("captured")
        setattr(tr, name, value)
        for f in (lambda: tr.step(x, lab, target=top), lambda: tr.prepare_graph(x, lab, target=top)):
            with pytest.raises(ValueError, match="a teacher wants"):
                f()


@pytest.mark.gpu
def test_annealed_temperature_keeps_its_memory(st):
    """Ten temperatures, four steps each: as launch by launch bit for bit, and the memory of the graphs that passed is free again."""
    x, lab = clips(4, 80), torch.tensor(LABELS, device=DEV)
    ends, held = [], []
    for graph in (False, True):
        tr = trainer(st, graph=graph, teacher_k=10)
        losses = []
        for i in range(10):
            tr.temperature, tr.label_weight = 4.0 - 0.25 * i, 0.1 * i
            for _ in range(4):
                print(graph, i, len(losses), flush=True)
                losses.append(float(tr.step(x, lab).detach()))
            assert len(tr._graphs) == (min(i + 1, tr.GRAPHS_KEPT) if graph else 0)
            if graph:
                torch.cuda.synchronize()
                torch.cuda.empty_cache()                             # a dropped graph's pool is given back here, or when memory runs short
                held.append(torch.cuda.memory_reserved())
        ends.append((losses, tr.flat.flat.clone()))
    assert ends[0][0] == ends[1][0] and torch.equal(ends[0][1], ends[1][1])
    grows = held[1] - held[0]                                        # what one graph holds
    assert grows > 1 << 20 and held[9] <= held[4] + grows // 2, held


@pytest.mark.gpu
def test_steps_without_labels(st):
    """label_weight 0 and no labels: launch by launch and captured, bit for bit as with labels that do not count."""
    x, ends = clips(4, 81), []
    for graph, lab in ((False, torch.tensor(LABELS, device=DEV)), (False, None), (True, None)):
        tr = trainer(st, graph=graph, label_weight=0.0)
        losses = [float(tr.step(x, lab).detach()) for _ in range(6)]
        assert tr.graph_ready() == graph
        ends.append((losses, tr.flat.flat.clone()))
    for losses, params in ends[1:]:
        assert losses == ends[0][0] and torch.equal(params, ends[0][1])
