"""Plain-PyTorch statements of every hot op.

These are the oracle the CUDA kernels are tested against, and the execution path for CPU
tensors (unit tests, the fp32 plumbing configuration). They are differentiable through
ordinary autograd and make no assumption about dtype.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F

# Value the attention scores take where the mask forbids attention
# (tunix/models/llama3/model.py:382-396 uses the same large negative constant).
K_MASK = -2.3819763e38


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
  return F.linear(x, w, bias)


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float, w_offset: float = 0.0) -> torch.Tensor:
  """fp32 `x * rsqrt(mean(x^2) + eps) * (w + w_offset)`; Gemma uses w_offset = 1
  (tunix/models/gemma/model.py:715-740), Llama/Qwen use 0 (tunix/models/llama3/model.py:273-297)."""
  xf = x.float()
  y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * (w.float() + w_offset)
  return y.to(x.dtype)


def rope_cos_sin(positions: torch.Tensor, head_dim: int, theta: float, scale: float = 1.0):
  half = head_dim // 2
  inv = 1.0 / (theta ** (torch.arange(half, device=positions.device, dtype=torch.float32) * 2.0 / head_dim))
  ang = positions.float()[..., None] / scale * inv
  return ang.cos(), ang.sin()


def apply_rope(x: torch.Tensor, positions: torch.Tensor, theta: float, scale: float = 1.0) -> torch.Tensor:
  """Half-split rotary embedding on x[..., T, heads, H] with positions[..., T]
  (tunix/models/qwen3/model.py:404-425)."""
  H = x.shape[-1]
  cos, sin = rope_cos_sin(positions, H, theta, scale)
  cos, sin = cos[..., None, :], sin[..., None, :]
  xf = x.float()
  x1, x2 = xf[..., : H // 2], xf[..., H // 2:]
  return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1).to(x.dtype)


def glu(gu: torch.Tensor, kind: str) -> torch.Tensor:
  """`act(gate) * up` for gu = [gate | up] on the last axis; kind in {"silu", "gelu"} (tanh GELU)."""
  g, u = gu.chunk(2, dim=-1)
  a = F.gelu(g.float(), approximate="tanh") if kind == "gelu" else F.silu(g.float())
  return (a * u.float()).to(gu.dtype)


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
  out = F.embedding(ids, table)
  if scale != 1.0:
    out = (out.float() * scale).to(table.dtype)
  return out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: Optional[torch.Tensor], scale: float,
              softcap: float = 0.0) -> torch.Tensor:
  """Dense GQA attention. q [B,T,N,H], k/v [B,S,K,H], mask [B,T,S] bool (True = attend).
  fp32 scores and softmax (tunix/models/qwen3/model.py:674-686)."""
  B, T, N, H = q.shape
  K = k.shape[2]
  G = N // K
  qf = q.float().view(B, T, K, G, H) * scale
  s = torch.einsum("btkgh,bskh->bkgts", qf, k.float())
  if softcap > 0:
    s = torch.tanh(s / softcap) * softcap
  if mask is not None:
    s = torch.where(mask[:, None, None, :, :], s, torch.full_like(s, K_MASK))
  p = torch.softmax(s, dim=-1)
  o = torch.einsum("bkgts,bskh->btkgh", p, v.float())
  return o.reshape(B, T, N, H).to(q.dtype)


def selective_log_softmax(logits: torch.Tensor, targets: torch.Tensor, temperature: float = 1.0,
                          want_entropy: bool = False):
  """`logit[target] - logsumexp(logits)` in fp32 (tunix/rl/common.py:187-203), entropy optional."""
  z = logits.float()
  if temperature not in (0.0, 1.0):
    z = z / temperature
  lse = torch.logsumexp(z, dim=-1)
  lp = z.gather(-1, targets.long().unsqueeze(-1)).squeeze(-1) - lse
  ent = None
  if want_entropy:
    lsm = z - lse.unsqueeze(-1)
    ent = -(lsm.exp() * lsm).sum(-1)
  return lp, ent


def linear_logprob(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, temperature: float = 1.0,
                   softcap: float = 0.0, want_entropy: bool = False):
  """lm_head + selective log-softmax. hidden [T,D], weight [V,D], targets [T]."""
  logits = hidden.float() @ weight.float().t()
  if softcap > 0:
    logits = torch.tanh(logits / softcap) * softcap
  return selective_log_softmax(logits, targets, temperature, want_entropy)


def _masked_log_softmax(z: torch.Tensor, dim: int = -1) -> torch.Tensor:
  """log_softmax that takes a row of -inf for an empty distribution (all -inf, zero gradient) instead of NaN."""
  empty = (z == float("-inf")).all(dim, keepdim=True)
  lp = F.log_softmax(torch.where(empty, torch.zeros_like(z), z), dim)
  return torch.where(empty, torch.full_like(lp, float("-inf")), lp)


def _from_max(x: torch.Tensor) -> torch.Tensor:
  """Rows relative to their maximum, so that dividing by a temperature cannot overflow; rows of -inf stay as they are."""
  m = x.detach().amax(-1, keepdim=True)
  return x - torch.where(m == float("-inf"), torch.zeros_like(m), m)


def _wide(x: torch.Tensor) -> torch.Tensor:
  return x if x.dtype == torch.float64 else x.float()


def top_logprobs(logits: torch.Tensor, k: int, targets: Optional[torch.Tensor], temperature: float,
                 want_entropy: bool):
  """(ids, top, target, entropy) of `functional.top_logprobs` for logits [T, V]."""
  x = _wide(logits)
  V = x.shape[1]
  lp = _masked_log_softmax(_from_max(x) / temperature)
  ids = torch.sort(x.detach(), dim=1, descending=True, stable=True).indices[:, :k]
  top = lp.gather(1, ids)
  target = entropy = None
  if targets is not None:
    known = (targets >= 0) & (targets < V)
    target = torch.where(known, lp.gather(1, targets.clamp(0, V - 1)[:, None])[:, 0], torch.zeros_like(lp[:, 0]))
  if want_entropy:
    p = lp.exp()
    entropy = -(p * torch.where(p == 0, torch.zeros_like(lp), lp)).sum(1)
  return ids, top, target, entropy


def top_distill_loss(logits: torch.Tensor, ids: torch.Tensor, values: torch.Tensor, labels: Optional[torch.Tensor],
                     temperature: float, full: bool):
  """(kl, nll) of `functional.top_distill_loss` for logits [T, V], ids and values [T, k]."""
  x = _wide(logits)
  T, V = x.shape
  low = float("-inf")
  there = (ids >= 0) & (ids < V)
  at = ids.clamp(0, V - 1)
  empty = (x == low).all(1)
  safe = torch.where(empty[:, None], torch.zeros_like(x), x)     # rows without a finite logit: no loss, no gradient
  t = _wide(values).detach().to(x.dtype)
  t = torch.where(there, t, torch.full_like(t, low))
  if full:
    lq = t
    lp = F.log_softmax(_from_max(safe) / temperature, dim=1).gather(1, at)
    none = empty
  else:
    picked = torch.where(there, x.gather(1, at), torch.full_like(t, low))
    none = (t == low).all(1) | (picked == low).all(1)
    lq = _masked_log_softmax(_from_max(t) / temperature)
    lp = _masked_log_softmax(_from_max(torch.where(none[:, None], torch.zeros_like(picked), picked)) / temperature)
  q = lq.exp()
  use = (q != 0) & ~none[:, None]
  zero = torch.zeros_like(q)
  kl = (torch.where(use, q, zero) * (torch.where(use, lq, zero) - torch.where(use, lp, zero))).sum(1)
  nll = None
  if labels is not None:
    known = (labels >= 0) & (labels < V) & ~empty
    lp1 = F.log_softmax(safe, dim=1).gather(1, labels.clamp(0, V - 1)[:, None])[:, 0]
    nll = torch.where(known, -lp1, torch.zeros_like(lp1))
  return kl, nll
