"""Log probabilities out of class scores (logits): of given classes, with the entropy and the best alternatives.

No counterpart in the reference, whose classifier ends at the logits (vitm/models/classifier.py:39).  One pass over the
scores in a HIP kernel (``vitm_log_probs``), differentiable with respect to them (``vitm_log_probs_bwd``)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib, _ops
from . import _score_ops as S


class LogProbs(NamedTuple):
    """Result of ``log_probs``; what was not asked for is None.  fp32, indices int64."""
    logprobs: Optional[torch.Tensor]
    lse: torch.Tensor
    entropy: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]
    top_indices: Optional[torch.Tensor]


def check_scores(logits: torch.Tensor, temperature: float, what: str, most: float = _lib.SCORES_MAX_TEMPERATURE) -> None:
    """The checks every operator on class scores shares."""
    if logits.dim() < 1:
        raise ValueError(f"{what}: logits need a class dimension")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{what}: unsupported logits dtype {logits.dtype} (bf16 or fp32)")
    if not 1 <= logits.shape[-1] <= _lib.SCORES_MAX_CLASSES:
        raise ValueError(f"{what}: {logits.shape[-1]} classes, supported are 1 to {_lib.SCORES_MAX_CLASSES}")
    if logits.numel() > _lib.SCORES_MAX_ROWS * logits.shape[-1]:
        raise ValueError(f"{what}: {logits.numel() // logits.shape[-1]} rows, supported are at most {_lib.SCORES_MAX_ROWS}")
    check_temperature(temperature, what, most)
    refuse_tangents(what, logits)


def refuse_tangents(what: str, *inputs: torch.Tensor) -> None:
    """A dual tensor's values alone would pass for a derivative of 0."""
    for t in inputs:
        if forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative")


def check_temperature(temperature: float, what: str, most: float = _lib.SCORES_MAX_TEMPERATURE) -> None:
    if not 1e-6 <= temperature <= most:
        raise ValueError(f"{what}: temperature {temperature}, supported are 1e-6 to {most:g}")


def check_indices(t: torch.Tensor, logits: torch.Tensor, what: str) -> None:
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what} must be int64 or int32, got {t.dtype}")
    if t.device != logits.device:
        raise RuntimeError(f"{what} are on {t.device}, the logits on {logits.device}")


def as_indices(t: torch.Tensor) -> torch.Tensor:
    """Contiguous int64, as the kernels read indices."""
    return t.contiguous() if t.dtype == torch.int64 else t.to(torch.int64).contiguous()


class _NoSecondDerivative(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, dz, *sources):
        ctx.what = what
        return dz.view_as(dz)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.what} has no second derivative")


def first_derivative(what: str, dz: torch.Tensor, *sources: Optional[torch.Tensor]) -> torch.Tensor:
    """``dz``, a gradient made from ``sources``: under ``create_graph=True`` one that raises when it is differentiated itself,
    instead of passing for a constant."""
    return _NoSecondDerivative.apply(what, dz, *sources) if torch.is_grad_enabled() else dz


class _LogProbsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, n_targets, top_k, entropy, temperature, ignore_index):
        with _ops.on_device_of(logits):
            rows = S.rows_of(logits)
            lp, lse, ent, top_lp, top_idx, stats = S.log_probs(rows, logits.shape[:-1], targets, n_targets, top_k, entropy, temperature,
                                                               ignore_index, want_stats=True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, targets, top_idx, stats, ent)
        ctx.plain = (n_targets, top_k, temperature, ignore_index)
        if top_idx is not None:
            ctx.mark_non_differentiable(top_idx)
        return lp, lse, ent, top_lp, top_idx

    @staticmethod
    def backward(ctx, g_lp, g_lse, g_ent, g_top, _):
        logits, targets, top_idx, stats, ent = ctx.saved_tensors
        n_targets, top_k, temperature, ignore_index = ctx.plain
        gs = [None if g is None else g.contiguous() for g in (g_lp if n_targets else None, g_lse, g_ent, g_top)]
        with _ops.on_device_of(logits):
            dz = S.log_probs_bwd(S.rows_of(logits), logits.shape, targets, n_targets, ignore_index, top_idx, top_k, temperature,
                                 stats, ent, *gs)
        return first_derivative("log_probs", dz, logits, *gs), None, None, None, None, None, None


def log_probs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *, top_k: int = 0, entropy: bool = False,
              temperature: float = 1.0, ignore_index: int = -100) -> LogProbs:
    """Log probabilities of ``softmax(logits / temperature)`` over the last dimension.

    ``logits``: (..., V), bf16 or fp32.  ``targets``: classes whose log probabilities are wanted, of shape (...) or
    (..., G); an entry equal to ``ignore_index`` gives 0, any other index outside [0, V) gives NaN.  ``top_k``: how many of
    the largest log probabilities come back with their classes, in order, equal ones by the lower class first.
    ``lse`` is always returned, ``entropy`` (in nats) on request.

    -inf marks a masked class.  A row with nothing else has log probabilities and lse -inf and entropy 0; a row with NaN or
    +inf gives NaN (top classes -1).  Differentiable with respect to ``logits`` through every floating-point output; the
    gradient has the logits' dtype.  Rows may be strided (no copy as long as the classes of a row lie side by side)."""
    what = "log_probs"
    temperature, top_k = float(temperature), int(top_k)
    check_scores(logits, temperature, what)
    most = _lib.SCORES_MAX_TOP
    V, lead = logits.shape[-1], logits.shape[:-1]
    if not 0 <= top_k <= min(V, most):
        raise ValueError(f"{what}: top_k {top_k}, supported are 0 to {most} and at most the {V} classes")
    n_targets = 0
    if targets is not None:
        check_indices(targets, logits, f"{what}: targets")
        if targets.shape == lead:
            n_targets = 1
        elif targets.shape[:-1] == lead and targets.dim() == len(lead) + 1:
            n_targets = targets.shape[-1]
            if n_targets > most:
                raise ValueError(f"{what}: {n_targets} targets a row, supported are at most {most}")
        else:
            raise ValueError(f"{what}: targets of shape {tuple(targets.shape)} for logits of shape {tuple(logits.shape)}")
    _ops.require_cuda(logits, what)
    if logits.numel() == 0:                   # no rows: empty results, part of the graph as others are
        none = logits.float().sum(-1)
        return LogProbs(None if targets is None else none.reshape(targets.shape), none, none + 0 if entropy else None,
                        none.reshape((*lead, top_k)) if top_k else None,
                        torch.empty((*lead, top_k), dtype=torch.int64, device=logits.device) if top_k else None)
    if targets is not None:
        targets = as_indices(targets)
    if logits.requires_grad and torch.is_grad_enabled():
        return LogProbs(*_LogProbsFunction.apply(logits, targets, n_targets, top_k, bool(entropy), temperature, int(ignore_index)))
    with _ops.on_device_of(logits):
        return LogProbs(*S.log_probs(S.rows_of(logits), lead, targets, n_targets, top_k, bool(entropy), temperature,
                                     int(ignore_index), want_stats=False)[:5])
