"""HIP-graph replay of a forward.

A forward of this package is a fixed sequence of kernel launches for a fixed input shape (the reference's
modules have no data-dependent control flow, vitm/models/models.py:208-211,352-361,408-416), so it can be
captured once into a HIP graph and replayed with one host call.  That matters where the launches themselves are
the cost: the small configurations (CIFAR ViT-tiny: ~90 launches of a few microseconds each per forward) and
host-bound multi-GPU driving.  The kernels are the same ones, on the same buffers: a replay is bit-identical to
the eager call.
"""
from __future__ import annotations

import torch

from . import _ops


class GraphedForward:
    """``g = GraphedForward(module, example_input)`` then ``y = g(x)`` for any ``x`` of that shape and dtype.

    The returned tensor is the graph's static output buffer: it is overwritten by the next call (clone it to
    keep it).  Weights are read from the module's packed copies as they were at capture time (the graph
    keeps that memory, whatever becomes of the module); re-capture after changing them.
    """

    def __init__(self, module: torch.nn.Module, example: torch.Tensor, warmup: int = 2):
        if not example.is_cuda:
            raise RuntimeError("GraphedForward needs a CUDA example input")
        self.module = module
        self.static_in = example.detach().clone()
        with torch.no_grad():
            side = torch.cuda.Stream(device=example.device)
            side.wait_stream(torch.cuda.current_stream(example.device))
            with torch.cuda.stream(side):
                for _ in range(max(1, warmup)):   # packs the weights, opts the kernels into their LDS sizes
                    module(self.static_in)
            torch.cuda.current_stream(example.device).wait_stream(side)
            torch.cuda.synchronize(example.device)
            self.graph, self.held = torch.cuda.CUDAGraph(), []
            with _ops.holding(self.held), torch.cuda.graph(self.graph):
                self.static_out = module(self.static_in)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape != self.static_in.shape or x.dtype != self.static_in.dtype:
            raise RuntimeError(f"captured for {tuple(self.static_in.shape)} {self.static_in.dtype}, "
                               f"got {tuple(x.shape)} {x.dtype}")
        if x.data_ptr() != self.static_in.data_ptr():
            self.static_in.copy_(x, non_blocking=True)
        self.graph.replay()
        return self.static_out


class GraphedTrainStep:
    """``Trainer.step`` replayed from a HIP graph: ``g = GraphedTrainStep(trainer)`` then ``loss = g.step(images, labels)``.

    A training step of this package is a fixed sequence of ~900 kernel launches for a fixed batch shape; at the
    reference's own batch sizes (32 .. 64 CIFAR images, vitm/config/config.yaml) the launches, not the kernels, are the
    step time.  The first ``warmup`` calls run ``trainer.step`` eagerly (real steps: they also opt the kernels into their
    LDS sizes); the next call captures the kernels of a step and from then on every call is: write the seven AdamW scalars
    for the current learning rate and step count to the device, copy the batch into the static input buffers, one graph
    launch, ``scheduler.step()``.  The kernels and their order are those of the eager step.  Needs the flat AdamW of this
    package, a single process (no gradient all-reduce) and batches of one shape; the returned loss is a copy.

    A teacher of the trainer's is captured with the step, its weights as they are then.  A module whose parameters were
    written in place, moved, cast or replaced since is refused (hand ``step`` the ``teacher_top`` of such a teacher), and so
    are another teacher and other settings of the distillation loss.  An in-place write through ``p.data`` leaves no trace
    that could be looked at and goes unseen; a teacher that is no module has to stay what it was.
    """

    def __init__(self, trainer, warmup: int = 2):
        if trainer.params is None or trainer.reducer.active:
            raise RuntimeError("GraphedTrainStep needs vitm_amd.training.AdamW in flat mode and a single process")
        self.trainer, self.warmup, self.calls = trainer, max(1, int(warmup)), 0
        self.graph = None

    def _distilled_from(self):
        """(settings of the loss, what the captured teacher's weights were made from): the latter is what packed weights are
        kept by; buffers are read where they are, so only their place counts."""
        tr = self.trainer
        if getattr(tr, "distillation", None) is None:
            return None, None
        t = tr.teacher
        if self.top is not None:
            weights = None
        elif not isinstance(t, torch.nn.Module):
            weights = t
        else:
            weights = (t, [(p.data_ptr(), p._version, p.dtype, p.device) for p in t.parameters()],
                       [(b.data_ptr(), b.dtype, b.device) for b in t.buffers()])
        return tr.distillation._cfg(), (tr.teacher_top_k if self.top is None else None, weights)

    def _capture(self, images, labels, teacher_top):
        tr = self.trainer
        dev = images.device
        self.x, self.y = images.detach().clone(), labels.detach().clone()
        self.top = None if teacher_top is None else tuple(t.detach().clone() for t in teacher_top)
        self.distilled_from = self._distilled_from()
        # what the graph's kernels read has to outlive whatever becomes of the teacher
        self.held = []
        teacher = getattr(tr, "teacher", None)
        if self.top is None and isinstance(teacher, torch.nn.Module):
            self.held += [t.detach() for t in (*teacher.parameters(), *teacher.buffers())]
        self.hyper = torch.zeros(8, dtype=torch.float32, device=dev)
        torch.cuda.synchronize(dev)
        graph = torch.cuda.CUDAGraph()
        with _ops.holding(self.held), torch.cuda.graph(graph):
            self.loss, self.norm = tr.device_step(self.x, self.y, self.hyper, *(() if self.top is None else (self.top,)))
        self.graph = graph

    def step(self, images: torch.Tensor, labels: torch.Tensor, teacher_top=None) -> torch.Tensor:
        tr = self.trainer
        self.calls += 1
        if self.calls <= self.warmup:
            return tr.step(images, labels, *(() if teacher_top is None else (teacher_top,)))
        if self.graph is None:
            self._capture(images, labels, teacher_top)
        if images.shape != self.x.shape or images.dtype != self.x.dtype or labels.shape != self.y.shape:
            raise RuntimeError(f"captured for images {tuple(self.x.shape)} {self.x.dtype}, got {tuple(images.shape)} {images.dtype}")
        if (teacher_top is None) != (self.top is None):
            raise RuntimeError("captured with teacher_top, got none" if teacher_top is None else "captured without teacher_top")
        if len(teacher_top or ()) != len(self.top or ()):
            raise RuntimeError(f"teacher_top is (log probabilities, indices), got {len(teacher_top)} entries")
        for mine, t in zip(self.top or (), teacher_top or ()):
            if t.shape != mine.shape or t.dtype != mine.dtype:
                raise RuntimeError(f"captured for teacher_top {tuple(mine.shape)} {mine.dtype}, got {tuple(t.shape)} {t.dtype}")
        settings, teacher = self._distilled_from()
        if settings != self.distilled_from[0]:
            raise RuntimeError("the settings of the distillation loss changed after the step was captured: capture anew")
        if teacher != self.distilled_from[1]:
            raise RuntimeError("the teacher, or the teacher's weights, changed after the step was captured: capture anew, or a step "
                               "that is given teacher_top")
        if not tr.optimizer._flat_ok():
            raise RuntimeError("the parameters or gradients left the flat buffers the graph was captured on")
        vals = tr.optimizer.next_hyper()
        # a pageable source: the copy is staged at once, so the next call may overwrite nothing that is still to be read
        self.hyper[:7].copy_(torch.tensor(vals, dtype=torch.float32))
        self.x.copy_(images, non_blocking=True)
        self.y.copy_(labels.to(self.y.dtype), non_blocking=True)
        for mine, t in zip(self.top or (), teacher_top or ()):
            mine.copy_(t, non_blocking=True)
        self.graph.replay()
        tr.last_grad_norm = self.norm
        if tr.scheduler is not None:
            tr.scheduler.step()
        return self.loss.clone()

