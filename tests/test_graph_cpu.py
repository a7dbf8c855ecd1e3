"""The host side of a captured training step, without a GPU: stubs stand in for the graph and for the trainer's kernels."""
import contextlib
from types import SimpleNamespace

import pytest
import torch


class _Optimizer:
    steps = 0

    def _flat_ok(self):
        return True

    def next_hyper(self):
        self.steps += 1
        return [0.0] * 7


@pytest.fixture
def graphed(monkeypatch):
    """(captured GraphedTrainStep, its trainer, step()) for a teacher that is a plain module or what ``make`` returns."""
    from vitm_amd import GraphedTrainStep, training
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: SimpleNamespace(replay=lambda: None))
    monkeypatch.setattr(torch.cuda, "graph", lambda g: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda dev: None)

    def make(teacher, loss=None, top=None):
        tr = SimpleNamespace(params=object(), reducer=SimpleNamespace(active=False), optimizer=_Optimizer(), scheduler=None,
                             distillation=loss or training.DistillationLoss(), teacher=teacher, teacher_top_k=4,
                             step=lambda *a: torch.zeros(()),
                             device_step=lambda x, y, hyper, top=None: (torch.zeros(()), torch.zeros(())))
        g = GraphedTrainStep(tr, warmup=1)
        x, y = torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64)
        step = lambda: g.step(x, y, top)
        for _ in range(3):
            step()
        assert tr.optimizer.steps == 2
        return g, tr, step
    return make


def _teacher():
    m = torch.nn.Sequential(torch.nn.Linear(3, 5), torch.nn.BatchNorm1d(5))
    return m.eval()


def _assign(m):
    m.load_state_dict({k: v.clone() for k, v in m.state_dict().items()}, assign=True)


def _data(m):
    m[0].weight.data = m[0].weight.data.clone()


def _parameter(m):
    m[0].weight = torch.nn.Parameter(m[0].weight.detach().clone())


def _buffer(m):
    m[1].running_mean = torch.ones(5)


def _in_place(m):
    with torch.no_grad():
        m[0].bias.add_(1.0)


@pytest.mark.parametrize("change", [_assign, _data, _parameter, _buffer, _in_place, lambda m: m.bfloat16(), lambda m: m.double()])
def test_captured_step_refuses_a_teacher_that_changed(graphed, change):
    m = _teacher()
    _, tr, step = graphed(m)
    change(m)
    with pytest.raises(RuntimeError, match="teacher's weights"):
        step()
    assert tr.optimizer.steps == 2                # refused before the step counters move


def test_captured_step_refuses_another_teacher_and_other_settings(graphed):
    from vitm_amd import training
    m = _teacher()
    for change in (lambda tr: setattr(tr, "teacher", _teacher()), lambda tr: setattr(tr, "teacher", lambda x: x),
                   lambda tr: setattr(tr, "teacher_top_k", 3)):
        _, tr, step = graphed(m)
        change(tr)
        with pytest.raises(RuntimeError, match="teacher"):
            step()
        assert tr.optimizer.steps == 2
    for change in (lambda tr: setattr(tr.distillation, "temperature", 3.0), lambda tr: setattr(tr.distillation, "tail", True),
                   lambda tr: setattr(tr, "distillation", training.DistillationLoss(reduction="sum"))):
        for top in (None, (torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int64))):
            _, tr, step = graphed(m, training.DistillationLoss(), top)
            change(tr)
            with pytest.raises(RuntimeError, match="settings of the distillation loss"):
                step()
            assert tr.optimizer.steps == 2


def test_captured_step_without_its_teacher_ignores_the_teacher(graphed):
    m = _teacher()
    _, tr, step = graphed(m, top=(torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int64)))
    m.bfloat16()
    tr.teacher = None
    step()
    assert tr.optimizer.steps == 3


def test_captured_step_keeps_what_its_kernels_read(graphed):
    """The teacher's tensors, and packed weights and fp32 vectors that were looked up while the step was captured, stay alive."""
    import weakref
    from vitm_amd import _ops
    m = _teacher()

    class Pack:
        pass

    owner, made = torch.nn.Module(), []

    def build():
        made.append(weakref.ref(p := Pack()))
        return p

    half = torch.nn.Parameter(torch.ones(4, dtype=torch.bfloat16))
    from vitm_amd import GraphedTrainStep
    g, tr, step = graphed(m)
    capture = GraphedTrainStep._capture
    tr.device_step = lambda x, y, hyper: (_ops.cached_pack(owner, "w", (m[0].weight,), build).__class__ and torch.zeros(()),
                                               _ops.f32vec(half))
    capture(g, torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64), None)
    vec = weakref.ref(half._vitm_f32[1])
    g.norm = None
    storage = m[0].weight.untyped_storage().data_ptr()
    del half
    m.bfloat16()
    _ops.cached_pack(owner, "w", (m[0].weight,), build)
    assert made[0]() is not None and vec() is not None
    assert any(t.untyped_storage().data_ptr() == storage for t in g.held if isinstance(t, torch.Tensor))
    del g, step
    tr.device_step = None
    assert made[0]() is None


def test_captured_step_takes_both_parts_of_teacher_top(graphed):
    """A tuple of another length would leave the captured indices as they were."""
    top = (torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int64))
    g, tr, _ = graphed(None, top=top)
    for bad in ((torch.ones(2, 4),), (*top, torch.ones(2, 4))):
        with pytest.raises(RuntimeError, match="log probabilities, indices"):
            g.step(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64), bad)
    assert tr.optimizer.steps == 2


def test_a_capture_that_failed_is_not_replayed(graphed):
    from vitm_amd import GraphedTrainStep
    _, tr, _ = graphed(None, top=(torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int64)))
    good, fails = tr.device_step, []

    def device_step(*a):
        if not fails:
            fails.append(1)
            raise ValueError("refused")
        return good(*a)

    tr.device_step = device_step
    g = GraphedTrainStep(tr, warmup=1)
    args = (torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64), (torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int64)))
    g.step(*args)
    with pytest.raises(ValueError, match="refused"):
        g.step(*args)
    assert g.graph is None and tr.optimizer.steps == 2
    g.step(*args)
    assert g.graph is not None and tr.optimizer.steps == 3


def test_captured_step_of_a_trainer_without_distillation(graphed, monkeypatch):
    """A trainer of the caller's own, or a subclass, whose steps take images and labels only."""
    from vitm_amd import GraphedTrainStep
    tr = SimpleNamespace(params=object(), reducer=SimpleNamespace(active=False), optimizer=_Optimizer(), scheduler=None,
                         step=lambda images, labels: torch.zeros(()), device_step=lambda images, labels, hyper: (torch.zeros(()), torch.zeros(())))
    g = GraphedTrainStep(tr, warmup=1)
    for _ in range(3):
        g.step(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))
    assert tr.optimizer.steps == 2
