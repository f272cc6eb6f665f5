"""Logit distillation: alpha * tau^2 * KL(teacher || student) at temperature tau plus
(1 - alpha) * cross entropy, with optional restriction to the teacher's top-k logits
(tunix/distillation/strategies/logit.py:28-169).

With a top-k the GPU runs two operators instead of passes over [.., V] in fp32: `top_logprobs` makes the teacher's list
(and its loss on integer labels) and `top_distill_loss` reads the student's logits once. A teacher's list may also stand
in the place of its logits: a `teacher_forward_fn` that returns `ops.functional.TopLogprobs`, computed on the spot or
stored earlier at temperature 1, keeps k numbers per token instead of V."""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from ...ops import _lib, functional, kernels
from .base_strategy import BaseStrategy, softmax_cross_entropy


def _class_ids(logits, labels):
  """Integer labels as ids, None for distributions over the vocabulary."""
  if labels.dtype in (torch.int32, torch.int64, torch.int16, torch.uint8) and labels.ndim == logits.ndim - 1:
    return labels.long()
  return None


def _refuse(outside, what):
  """Ids outside the vocabulary are an error, as in a lookup: on the host it is raised. On the GPU a lookup's assertion
  ends the process; here the answer is a factor for the loss instead, 1 or, where there are some, NaN."""
  if outside.is_cuda:
    return torch.where(outside.any(), math.nan, 1.0)
  if bool(outside.any()):
    raise RuntimeError(f"LogitStrategy: {what} outside the vocabulary")
  return None


def _times(x, factor):
  return x if factor is None else x * factor


class LogitStrategy(BaseStrategy):
  """Integer labels outside the vocabulary, and tokens among the teacher's top-k that the student does not have, are an
  error: raised on the CPU; on the GPU, where the host does not see them, the loss and its gradient are NaN with a
  teacher's list, and the lookup in torch asserts on the device where the formulas run."""

  def __init__(self, student_forward_fn, teacher_forward_fn, labels_fn, temperature: float = 2.0,
               alpha: float = 0.5, distill_top_k: int = 0):
    super().__init__(student_forward_fn, teacher_forward_fn, labels_fn)
    if temperature <= 0:
      raise ValueError(f"Temperature must be a positive number, got {temperature}")
    if not 0.0 <= alpha <= 1.0:
      raise ValueError(f"Alpha must be a float between 0.0 and 1.0, got {alpha}")
    self.temperature, self.alpha, self.distill_top_k = float(temperature), alpha, int(distill_top_k)

  def compute_eval_loss(self, student_output, labels):
    return softmax_cross_entropy(student_output, labels).mean(), {}

  def _compute_listed_loss(self, student_output, teacher_output, labels):
    V, stored = student_output.shape[-1], isinstance(teacher_output, functional.TopLogprobs)
    ids, sound = _class_ids(student_output, labels), None
    if ids is not None:
      known = ids.clamp(0, (V if stored else min(V, teacher_output.shape[-1])) - 1)
      ids, sound = known, _refuse(known != ids, "labels")
    if stored:
      top = teacher_output
      if top.temperature != 1.0:
        raise ValueError(f"LogitStrategy: a teacher's list is taken to its temperature here and has to come at temperature "
                         f"1, this one was made at {top.temperature}")
      if top.ids.shape[-1] < self.distill_top_k:
        raise ValueError(f"LogitStrategy: the teacher's list has {top.ids.shape[-1]} entries, too few for a top-k of "
                         f"{self.distill_top_k}")
      teacher = None if top.target is None else -top.target.mean()
    else:
      with torch.no_grad():
        top = functional.top_logprobs(teacher_output.detach(), self.distill_top_k, ids)
        teacher = -top.target.mean() if ids is not None else softmax_cross_entropy(teacher_output, labels).mean()
    k = self.distill_top_k or top.ids.shape[-1]
    if ids is None:                                                    # two gradients: they meet in fp32 and are rounded once
      student_output = student_output.float()
    listed = top.ids[..., :k]
    within = None
    if stored or teacher_output.shape[-1] > V:                         # negative ids are absent entries
      within = _refuse(listed >= V, "the teacher's tokens")
    terms = functional.top_distill_loss(student_output, listed, top.top.detach()[..., :k], ids, self.temperature, twice=True)
    kl = _times(terms.kl, within)
    soft = (kl * self.temperature ** 2).mean()
    hard = _times(terms.nll.mean() if ids is not None else softmax_cross_entropy(student_output, labels).mean(), sound)
    loss = self.alpha * soft + (1.0 - self.alpha) * hard
    metrics = {"distill/soft_loss": soft.detach(), "distill/hard_loss": hard.detach(),
               "distill/kl_div": kl.mean().detach()}
    if teacher is not None:
      metrics["distill/teacher_loss"] = _times(teacher.detach(), sound)
    return loss, metrics

  def _takes_list(self, student_output, teacher_output, labels) -> bool:
    """Whether these logits go through the teacher's list: what the operators do not take stays with the formulas."""
    s, t, k = student_output, teacher_output, self.distill_top_k
    if not s.is_cuda or not {s.dtype, t.dtype} <= {torch.float32, torch.bfloat16}:
      return False
    if not s.get_device() == t.get_device() == _lib.bind_thread():     # the kernels' GPU is the process's
      return False
    if not 0 < k <= min(kernels.MAX_TOP_K, t.shape[-1]) or s.shape[:-1] != t.shape[:-1]:
      return False
    ids = _class_ids(s, labels)
    if ids is not None and (ids.shape != s.shape[:-1] or ids.device != s.device):
      return False
    if not functional.MIN_TEMPERATURE <= self.temperature <= functional.MAX_TEMPERATURE:
      return False
    if t.requires_grad and torch.is_grad_enabled():                    # a list has no gradient for the teacher
      return False
    # forward mode and the transforms of torch.func
    return not (functional.is_dual(s) or functional.is_dual(t) or torch._C._are_functorch_transforms_active())

  def compute_loss(self, student_output, teacher_output, labels):
    if isinstance(teacher_output, functional.TopLogprobs) or self._takes_list(student_output, teacher_output, labels):
      return self._compute_listed_loss(student_output, teacher_output, labels)
    s, t = student_output.float(), teacher_output.float()
    sk, tk = s, t
    if self.distill_top_k > 0:
      tk, idx = torch.topk(t, self.distill_top_k, dim=-1)
      sk = s.gather(-1, idx)
    log_ps = F.log_softmax(sk / self.temperature, dim=-1)
    log_pt = F.log_softmax(tk / self.temperature, dim=-1)
    pt = log_pt.exp()
    kl = (pt * (torch.where(pt > 0, log_pt, torch.zeros_like(log_pt)) - log_ps)).sum(-1)
    soft = (kl * self.temperature ** 2).mean()
    hard = softmax_cross_entropy(s, labels).mean()
    with torch.no_grad():
      teacher = softmax_cross_entropy(t, labels).mean()
    loss = self.alpha * soft + (1.0 - self.alpha) * hard
    return loss, {"distill/soft_loss": soft.detach(), "distill/hard_loss": hard.detach(),
                  "distill/kl_div": kl.mean().detach(), "distill/teacher_loss": teacher}
