"""Differentiable hot ops.

Every function here accepts CPU or CUDA tensors. CUDA bf16 tensors run on the hand-written
sm_100a kernels (`kernels.py`) through `torch.autograd.Function`s with explicit backward
passes; everything else runs the PyTorch statement in `ref.py` under ordinary autograd.

Gradient accumulation fusion: a parameter may carry a `main_grad` attribute (an fp32 tensor
of the same shape). The backward passes then add the weight gradient straight into it from
the GEMM epilogue / reduction kernel and return no `.grad`, so accumulation over
micro-batches costs no extra pass and no bf16 rounding.
"""
from __future__ import annotations

import math
import threading
from typing import NamedTuple, Optional, Tuple

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from . import _lib, kernels, ref

bf16 = torch.bfloat16


def _use_kernels(*ts: torch.Tensor) -> bool:
  t = ts[0]
  if not t.is_cuda:
    return False
  if t.dtype != bf16:
    return False
  _lib.require()  # a CUDA bf16 tensor without the library is an error, never a silent fallback
  return True


def is_dual(t: torch.Tensor) -> bool:
  """Whether `t` carries a tangent of forward-mode differentiation."""
  return forward_ad.unpack_dual(t).tangent is not None


def _differentiated(t: torch.Tensor) -> bool:
  """Whether an operator on `t` has to go through its `Function`: a backward pass may follow, or `t` carries a tangent,
  which the `Function` refuses where the kernel alone would drop it."""
  return t.requires_grad and torch.is_grad_enabled() or is_dual(t)


def _main_grad(p: torch.Tensor) -> Optional[torch.Tensor]:
  return getattr(p, "main_grad", None)


# ------------------------------------------------------------------------------ linear
class _LinearFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x2, w, holder):
    ctx.save_for_backward(x2, w)
    ctx.holder = holder
    return kernels.gemm(x2, w)

  @staticmethod
  def backward(ctx, dy):
    x2, w = ctx.saved_tensors
    dy = dy.contiguous()
    dx = dw = None
    if ctx.needs_input_grad[0]:
      dx = kernels.gemm(dy, w, b_mn=True)                      # dx[M,K] = dy[M,N] @ w[N,K]
    if ctx.needs_input_grad[1]:
      mg = _main_grad(ctx.holder) if ctx.holder is not None else None
      if mg is not None:
        kernels.gemm(dy, x2, a_mn=True, b_mn=True, out=mg, accumulate=True)   # dw[N,K] += dy^T @ x
      else:
        dw = kernels.gemm(dy, x2, a_mn=True, b_mn=True)
    return dx, dw, None


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
  """y = x @ w^T (+ bias); w is [out, in]."""
  if _use_kernels(x, w) and w.dtype == bf16:
    K = x.shape[-1]
    x2 = x.reshape(-1, K)
    if not x2.is_contiguous():
      x2 = x2.contiguous()
    M, N = x2.shape[0], w.shape[0]
    if (M <= 128 and not (torch.is_grad_enabled() and (x.requires_grad or w.requires_grad))
        and kernels.gemm_skinny_supported(x2, w) and (bias is None or (bias.dtype == bf16 and bias.is_contiguous()))):
      # decode-shaped product without a backward pass: one launch that streams w once
      return kernels.gemm_skinny(x2, w, bias=bias).view(*x.shape[:-1], N)
    if kernels.gemm_supported(M, N, K, x2, w) and w.is_contiguous():
      y = _LinearFn.apply(x2, w, w)
      y = y.view(*x.shape[:-1], N)
      if bias is not None:
        y = y + bias
      return y
  return ref.linear(x, w, bias)


# ------------------------------------------------------------------------------ rmsnorm
class _RMSNormFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x2, w, eps, offset, holder):
    y, _, rstd = kernels.rmsnorm_fwd(x2, w, eps, offset)
    ctx.save_for_backward(x2, w, rstd)
    ctx.eps, ctx.offset, ctx.holder = eps, offset, holder
    return y

  @staticmethod
  def backward(ctx, dy):
    x2, w, rstd = ctx.saved_tensors
    mg = _main_grad(ctx.holder)
    if mg is not None:
      dx, _ = kernels.rmsnorm_bwd(x2, w, dy.contiguous(), rstd, ctx.eps, ctx.offset, dw_out=mg, dw_accumulate=True)
      return dx, None, None, None, None
    dx, dw = kernels.rmsnorm_bwd(x2, w, dy.contiguous(), rstd, ctx.eps, ctx.offset)
    return dx, dw.to(w.dtype), None, None, None


class _AddRMSNormFn(torch.autograd.Function):
  """(x, res) -> (norm(x + res), x + res): the residual add fused into the norm's read."""

  @staticmethod
  def forward(ctx, x2, res2, w, eps, offset, holder):
    y, s, rstd = kernels.rmsnorm_fwd(x2, w, eps, offset, residual=res2)
    ctx.save_for_backward(s, w, rstd)
    ctx.eps, ctx.offset, ctx.holder = eps, offset, holder
    return y, s

  @staticmethod
  def backward(ctx, dy, ds):
    s, w, rstd = ctx.saved_tensors
    mg = _main_grad(ctx.holder)
    dres = ds.contiguous() if ds is not None else None
    if mg is not None:
      dx, _ = kernels.rmsnorm_bwd(s, w, dy.contiguous(), rstd, ctx.eps, ctx.offset, dres=dres, dw_out=mg,
                                  dw_accumulate=True)
      dw = None
    else:
      dx, dwf = kernels.rmsnorm_bwd(s, w, dy.contiguous(), rstd, ctx.eps, ctx.offset, dres=dres)
      dw = dwf.to(w.dtype)
    return dx, dx, dw, None, None, None


def _norm_ok(x: torch.Tensor, w: torch.Tensor) -> bool:
  D = x.shape[-1]
  return _use_kernels(x) and w.dtype == bf16 and D % 8 == 0 and D <= 8192


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-6, w_offset: float = 0.0) -> torch.Tensor:
  if _norm_ok(x, w):
    x2 = x.reshape(-1, x.shape[-1]).contiguous()
    return _RMSNormFn.apply(x2, w, eps, w_offset, w).view(x.shape)
  return ref.rms_norm(x, w, eps, w_offset)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, w: torch.Tensor, eps: float = 1e-6,
                 w_offset: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
  """Returns (rms_norm(x + residual), x + residual)."""
  if _norm_ok(x, w):
    D = x.shape[-1]
    y, s = _AddRMSNormFn.apply(x.reshape(-1, D).contiguous(), residual.reshape(-1, D).contiguous(), w, eps,
                               w_offset, w)
    return y.view(x.shape), s.view(x.shape)
  s = x + residual
  return ref.rms_norm(s, w, eps, w_offset), s


# ------------------------------------------------------------------------------ qk-norm + rope
_rope_tables = {}
_bound = threading.local()     # per host thread: a rollout thread's bound must not leak into a trainer thread


def _position_bound() -> int:
  return getattr(_bound, "n", 0)


def set_position_bound(n: int) -> int:
  """Declares that every position this thread passes to `qk_norm_rope` is below `n` until further
  notice (0 = unknown). With a bound the rotary table is sized once and the per-call
  device-to-host read of `positions.max()` is skipped, which also makes the call capturable in
  a CUDA graph. A position that breaks the promise is clamped by the kernel and reported through
  the status word (bit 8). Returns the previous bound."""
  old = _position_bound()
  _bound.n = int(n)
  return old


def rope_table(head_dim: int, theta: float, max_pos: int, device, scale: float = 1.0) -> torch.Tensor:
  key = (head_dim, float(theta), float(scale), str(device))
  t = _rope_tables.get(key)
  if t is None or t.shape[0] < max_pos:
    n = max(4096, 1 << (max(1, max_pos) - 1).bit_length())
    t = kernels.rope_table(n, head_dim, theta, device, scale)
    _rope_tables[key] = t
  return t


class _QKNormRopeFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, qkv2, positions, table, n_q, n_k, H, wq, wk, eps, offset, hq, hk):
    out = kernels.qknorm_rope_fwd(qkv2, positions, table, n_q, n_k, H, wq, wk, eps, offset)
    ctx.save_for_backward(qkv2, positions, table, wq, wk)
    ctx.cfg = (n_q, n_k, H, eps, offset)
    ctx.hq, ctx.hk = hq, hk
    return out

  @staticmethod
  def backward(ctx, dy):
    qkv2, positions, table, wq, wk = ctx.saved_tensors
    n_q, n_k, H, eps, offset = ctx.cfg
    dx, dwq, dwk = kernels.qknorm_rope_bwd(qkv2, dy.contiguous(), positions, table, n_q, n_k, H, wq, wk, eps, offset)
    gq = gk = None
    if wq is not None:
      mq, mk = _main_grad(ctx.hq), _main_grad(ctx.hk)
      if mq is not None:
        mq.add_(dwq)
        mk.add_(dwk)
      else:
        gq, gk = dwq.to(wq.dtype), dwk.to(wk.dtype)
    return dx, None, None, None, None, None, gq, gk, None, None, None, None


def qk_norm_rope(qkv: torch.Tensor, positions: torch.Tensor, n_q: int, n_k: int, head_dim: int, theta: float,
                 wq: Optional[torch.Tensor] = None, wk: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 w_offset: float = 0.0, rope_scale: float = 1.0, max_pos: int = 0) -> torch.Tensor:
  """qkv [..., (n_q + 2 n_k) * H] (q heads | k heads | v heads) -> same shape, with optional
  per-head RMSNorm on q and k (tunix/models/qwen3/model.py:531-554) followed by half-split
  rotary embedding; v is passed through."""
  lead = qkv.shape[:-1]
  if _use_kernels(qkv) and head_dim in (64, 128, 256):
    q2 = qkv.reshape(-1, qkv.shape[-1]).contiguous()
    pos = positions.reshape(-1).to(torch.int32)
    bound = _position_bound()
    table = rope_table(head_dim, theta, max_pos or bound or 4096, qkv.device, rope_scale)
    if max_pos == 0 and bound == 0 and table.shape[0] < 1 << 20:
      # positions are data; make sure the table covers them (rare: only beyond 4096 tokens)
      need = int(pos.max().item()) + 1 if pos.numel() else 1
      if need > table.shape[0]:
        table = rope_table(head_dim, theta, need, qkv.device, rope_scale)
    out = _QKNormRopeFn.apply(q2, pos, table, n_q, n_k, head_dim, wq, wk, eps, w_offset, wq, wk)
    return out.view(*lead, -1)
  x = qkv.reshape(*lead, n_q + 2 * n_k, head_dim)
  q, k, v = x[..., :n_q, :], x[..., n_q:n_q + n_k, :], x[..., n_q + n_k:, :]
  if wq is not None:
    q = ref.rms_norm(q, wq, eps, w_offset)
    k = ref.rms_norm(k, wk, eps, w_offset)
  q = ref.apply_rope(q, positions, theta, rope_scale)
  k = ref.apply_rope(k, positions, theta, rope_scale)
  return torch.cat([q, k, v], dim=-2).reshape(*lead, -1)


# ------------------------------------------------------------------------------ GLU
class _GLUFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, gu2, gelu):
    ctx.save_for_backward(gu2)
    ctx.gelu = gelu
    return kernels.glu_fwd(gu2, gelu)

  @staticmethod
  def backward(ctx, dout):
    (gu2,) = ctx.saved_tensors
    return kernels.glu_bwd(gu2, dout.contiguous(), ctx.gelu), None


def glu(gu: torch.Tensor, kind: str = "silu") -> torch.Tensor:
  """act(gate) * up with gu = [gate | up] along the last axis."""
  F2 = gu.shape[-1]
  if _use_kernels(gu) and (F2 // 2) % 8 == 0:
    out = _GLUFn.apply(gu.reshape(-1, F2).contiguous(), kind == "gelu")
    return out.view(*gu.shape[:-1], F2 // 2)
  return ref.glu(gu, kind)


# ------------------------------------------------------------------------------ embedding
class _EmbeddingFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, ids, table, scale):
    ctx.save_for_backward(ids)
    ctx.scale, ctx.holder, ctx.shape = scale, table, table.shape
    return kernels.embedding_fwd(ids, table, scale)

  @staticmethod
  def backward(ctx, dout):
    (ids,) = ctx.saved_tensors
    mg = _main_grad(ctx.holder)
    dout = dout.contiguous()
    if mg is not None:
      if mg.dtype != torch.float32:
        raise ValueError(f"embedding: main_grad must be fp32 to be added to, got {mg.dtype}")
      kernels.embedding_bwd(ids, dout, mg, ctx.scale)
      return None, None, None
    g = torch.empty(ctx.shape, dtype=dout.dtype, device=dout.device)
    kernels.embedding_bwd(ids, dout, g, ctx.scale)
    return None, g, None


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
  """Rows of `table` [V, D] times `scale`. The table's gradient is summed by sorted tokens: repeatable to the bit,
  fp32 sums rounded once, straight into `main_grad` where the table has one."""
  if _use_kernels(table) and table.shape[1] % 8 == 0:
    if not table.is_contiguous() or table.data_ptr() % 16:
      # the plain statement, with the kernels' rule for ids outside the table: the nearest row, which gets no gradient
      known = ids.clamp(0, table.shape[0] - 1)
      rows = ref.embedding(known, table, scale)
      return torch.where((known == ids)[..., None], rows, rows.detach())
    home = _lib.bind_thread()
    if ids.get_device() != home or table.get_device() != home:
      raise ValueError(f"embedding: ids are on {ids.device}, the table on {table.device}, "
                       f"this process drives cuda:{home}")
    flat = ids if ids.dim() == 1 else ids.reshape(-1)
    if _differentiated(table):
      out = _EmbeddingFn.apply(flat, table, scale)
    else:
      out = kernels.embedding_fwd(flat, table, scale)
    return out if ids.dim() == 1 else out.view(*ids.shape, table.shape[1])
  return ref.embedding(ids, table, scale)


# ------------------------------------------------------------------------------ attention
def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, mask: Optional[torch.Tensor] = None,
              causal: bool = False, scale: Optional[float] = None, softcap: float = 0.0) -> torch.Tensor:
  """GQA attention. q [B,T,N,H], k/v [B,S,K,H]; mask [B,T,S] bool or None.
  `causal=True` with mask=None means the plain lower-triangular mask (T == S)."""
  H = q.shape[-1]
  scale = (1.0 / math.sqrt(H)) if scale is None else scale
  if q.is_cuda and q.dtype in (bf16, torch.float16) and softcap == 0.0:
    from . import attention as _attn
    return _attn.attention_cuda(q, k, v, mask=mask, causal=causal, scale=scale)
  if mask is not None and not isinstance(mask, torch.Tensor):
    mask = mask.dense()          # a symbolic segment mask
  if mask is None and causal:
    T, S = q.shape[1], k.shape[1]
    mask = torch.ones(T, S, dtype=torch.bool, device=q.device).tril(S - T)[None].expand(q.shape[0], T, S)
  return ref.attention(q, k, v, mask, scale, softcap)


# ------------------------------------------------------------------------------ lm_head + log-softmax
_LOGITS_BUDGET_BYTES = 1 << 30   # size of one fp32 logits block kept live at a time


def _chunk_rows(T: int, V: int) -> int:
  rows = max(128, _LOGITS_BUDGET_BYTES // (4 * V))
  rows = (rows // 128) * 128
  return min(T, rows)


class _LinearLogprobFn(torch.autograd.Function):
  """Sequence-chunked lm_head -> selective log-softmax (tunix/rl/common.py:485-571 does the
  same with a rematerialised scan): the [T, V] logits are never resident, only one block."""

  @staticmethod
  def forward(ctx, h2, w, targets, inv_temp, softcap, want_entropy, holder):
    T, D = h2.shape
    V = w.shape[0]
    rows = _chunk_rows(T, V)
    logp = torch.empty(T, dtype=torch.float32, device=h2.device)
    lse = torch.empty(T, dtype=torch.float32, device=h2.device)
    ent = torch.empty(T, dtype=torch.float32, device=h2.device) if want_entropy else None
    buf = torch.empty((rows, V), dtype=torch.float32, device=h2.device)
    for s in range(0, T, rows):
      e = min(T, s + rows)
      lg = kernels.gemm(h2[s:e], w, out=buf[: e - s])
      lp, ls, en = kernels.logprob_fwd(lg, targets[s:e], inv_temp, softcap, want_entropy)
      logp[s:e], lse[s:e] = lp, ls
      if want_entropy:
        ent[s:e] = en
    ctx.save_for_backward(h2, w, targets, lse, ent)
    ctx.cfg = (inv_temp, softcap, rows)
    ctx.holder = holder
    if want_entropy:
      return logp, ent
    return logp, None

  @staticmethod
  def backward(ctx, g_logp, g_ent):
    h2, w, targets, lse, ent = ctx.saved_tensors
    inv_temp, softcap, rows = ctx.cfg
    T, D = h2.shape
    V = w.shape[0]
    need_dh, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
    dh = torch.empty_like(h2) if need_dh else None
    mg = _main_grad(ctx.holder) if need_dw else None
    dw_acc = None
    if need_dw and mg is None:
      dw_acc = torch.zeros((V, D), dtype=torch.float32, device=h2.device)
    g_logp = g_logp.contiguous().float() if g_logp is not None else None
    g_ent = g_ent.contiguous().float() if g_ent is not None else None
    buf = torch.empty((rows, V), dtype=torch.float32, device=h2.device)
    dbuf = torch.empty((rows, V), dtype=bf16, device=h2.device)
    for s in range(0, T, rows):
      e = min(T, s + rows)
      lg = kernels.gemm(h2[s:e], w, out=buf[: e - s])
      dl = kernels.logprob_bwd(lg, targets[s:e], lse[s:e], ent[s:e] if ent is not None else None,
                               g_logp[s:e] if g_logp is not None else None,
                               g_ent[s:e] if g_ent is not None else None, inv_temp, softcap, out=dbuf[: e - s])
      if need_dh:
        kernels.gemm(dl, w, b_mn=True, out=dh[s:e])
      if need_dw:
        kernels.gemm(dl, h2[s:e], a_mn=True, b_mn=True, out=mg if mg is not None else dw_acc, accumulate=True)
    dw = None if (not need_dw or mg is not None) else dw_acc.to(w.dtype)
    return dh, dw, None, None, None, None, None


def linear_logprob(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, temperature: float = 1.0,
                   softcap: float = 0.0, want_entropy: bool = False):
  """Per-token log-probability (and entropy) of `targets` under softmax(hidden @ weight^T / T).

  hidden [..., D], weight [V, D], targets [...] -> (logp [...], entropy [...] or None), fp32.
  Shared by the trainer, the reference policy and the rollout sampler so that log-probs agree.
  """
  vp = getattr(weight, "vocab_parallel", None)
  if vp is not None:        # (group, first vocabulary row of this rank's slice): see ops/vocab_parallel.py
    from . import vocab_parallel
    return vocab_parallel.linear_logprob(hidden, weight, targets, vp[0], vp[1], temperature, softcap, want_entropy)
  lead = targets.shape
  D = hidden.shape[-1]
  V = weight.shape[0]
  inv_temp = 1.0 if temperature in (0.0, 1.0) else 1.0 / temperature
  if _use_kernels(hidden, weight) and weight.dtype == bf16 and V % 8 == 0 and D % 8 == 0 and weight.is_contiguous():
    h2 = hidden.reshape(-1, D).contiguous()
    T = h2.shape[0]
    pad = (-T) % 8
    tg = targets.reshape(-1)
    if pad:
      h2 = torch.cat([h2, h2.new_zeros(pad, D)], 0)
      tg = torch.cat([tg, tg.new_zeros(pad)], 0)
    lp, ent = _LinearLogprobFn.apply(h2, weight, tg, inv_temp, softcap, want_entropy, weight)
    lp = lp[:T].view(lead)
    ent = ent[:T].view(lead) if ent is not None else None
    return lp, ent
  lp, ent = ref.linear_logprob(hidden.reshape(-1, D), weight, targets.reshape(-1), temperature, softcap, want_entropy)
  return lp.view(lead), (ent.view(lead) if ent is not None else None)


# ------------------------------------------------------------------------------ alternatives of a row of logits
MIN_TEMPERATURE, MAX_TEMPERATURE = 1e-18, 1e18       # the inverse and products with logits stay within fp32


class _TopLogprobs(NamedTuple):
  ids: torch.Tensor                    # int64 [..., k], likeliest first
  top: torch.Tensor                    # fp32 [..., k], their log-probabilities
  target: Optional[torch.Tensor]       # fp32 [...], log-probability of the given token
  entropy: Optional[torch.Tensor]      # fp32 [...]


class TopLogprobs(_TopLogprobs):
  """What `top_logprobs` says of every row of logits. `temperature`, at which it says so, is an attribute beside the four
  fields: copies, pickles and `_replace` keep it, a tuple built anew from the fields is at temperature 1."""
  temperature = 1.0

  def __new__(cls, ids, top, target, entropy, temperature: float = 1.0):
    self = super().__new__(cls, ids, top, target, entropy)
    if temperature != 1.0:
      self.temperature = float(temperature)
    return self

  def _replace(self, **fields):
    return TopLogprobs(*super()._replace(**fields), temperature=self.temperature)


class DistillLoss(NamedTuple):
  """Per-row terms of `top_distill_loss`."""
  kl: torch.Tensor                     # fp32 [...]
  nll: Optional[torch.Tensor]          # fp32 [...]


def _grad32(g: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
  if g is None or (g.dtype == torch.float32 and g.is_contiguous()):
    return g
  return g.float().contiguous()


def _once(dx: torch.Tensor) -> torch.Tensor:
  """A gradient that cannot be differentiated again: where a graph of the backward pass is built, an error is put
  behind it (the softmax's own derivative would silently be missing)."""
  if not torch.is_grad_enabled():
    return dx
  error = torch._C._functions.DelayedError(b"top_logprobs and top_distill_loss have no second derivative", 1)
  return error(dx.detach().requires_grad_())


class _TopLogprobsFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x2, k, targets, inv_temp, want_entropy):
    ids, top, target, ent, stats = kernels.top_logprobs_fwd(x2, k, targets, inv_temp, want_entropy)
    ctx.save_for_backward(x2, ids, targets, ent, stats)
    ctx.inv_temp = inv_temp
    ctx.mark_non_differentiable(ids)
    ctx.set_materialize_grads(False)
    return ids, top, target, ent

  @staticmethod
  def backward(ctx, _, g_top, g_target, g_ent):
    x2, ids, targets, ent, stats = ctx.saved_tensors
    if g_top is None and g_target is None and g_ent is None:
      return None, None, None, None, None
    dx = kernels.top_logprobs_bwd(x2, ids, targets, stats, ent, _grad32(g_top), _grad32(g_target), _grad32(g_ent),
                                  ctx.inv_temp)
    return _once(dx), None, None, None, None


class _TopDistillFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x2, ids, values, labels, inv_temp, full, temperature):
    kl, nll, stats = kernels.top_distill_fwd(x2, ids, values, labels, inv_temp, full)
    ctx.save_for_backward(x2, ids, values, labels, stats)
    ctx.cfg, ctx.again = (inv_temp, full), temperature
    ctx.set_materialize_grads(False)
    return kl, nll

  @staticmethod
  def backward(ctx, g_kl, g_nll):
    x2, ids, values, labels, stats = ctx.saved_tensors
    rest = (None,) * 6
    if g_kl is None and g_nll is None:
      return None, *rest
    if ctx.again is not None and torch.is_grad_enabled():
      outs = ref.top_distill_loss(x2, ids, values, labels, ctx.again, ctx.cfg[1])
      pairs = [(o, g) for o, g in zip(outs, (g_kl, g_nll)) if g is not None]
      return torch.autograd.grad([o for o, _ in pairs], x2, [g for _, g in pairs], create_graph=True)[0], *rest
    dx = kernels.top_distill_bwd(x2, ids, values, labels, stats, _grad32(g_kl), _grad32(g_nll), *ctx.cfg)
    return _once(dx), *rest


def _check_rows(name: str, logits: torch.Tensor, temperature: float) -> None:
  """Arguments that `top_logprobs` and `top_distill_loss` share: floating logits [..., V], a positive temperature."""
  if logits.dim() < 1 or not logits.is_floating_point():
    raise ValueError(f"{name}: logits must be a floating tensor [..., V], got {logits.dtype} {tuple(logits.shape)}")
  if not MIN_TEMPERATURE <= temperature <= MAX_TEMPERATURE:
    raise ValueError(f"{name}: temperature must be positive and finite (1e-18 to 1e18), got {temperature}")


def _check_index(name: str, what: str, t: torch.Tensor, shape, logits: torch.Tensor) -> None:
  """An integer tensor of this shape on the logits' device."""
  if t.dtype != torch.int64 and t.dtype != torch.int32:
    raise ValueError(f"{name}: {what} must be int32 or int64, got {t.dtype}")
  if t.shape != shape:
    raise ValueError(f"{name}: {what} must have shape {tuple(shape)}, got {tuple(t.shape)}")
  if t.device != logits.device:
    raise ValueError(f"{name}: {what} is on {t.device}, the logits on {logits.device}")


def _rows(name: str, logits: torch.Tensor) -> Optional[torch.Tensor]:
  """The logits as the kernels read them ([T, V], unit column stride), or None where the plain statement runs."""
  if not logits.is_cuda or logits.dtype not in (bf16, torch.float32):
    return None
  _lib.require()
  home = _lib.bind_thread()
  if logits.get_device() != home:
    raise ValueError(f"{name}: logits are on {logits.device}, this process drives cuda:{home}")
  x2 = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])     # a view is a node of the graph
  if max(x2.shape) > 0x7fff0000:
    raise ValueError(f"{name}: rows and columns are counted in 31 bits, got {tuple(x2.shape)}")
  if x2.stride(1) != 1 and x2.shape[1] > 1 or x2.stride(0) < x2.shape[1] and x2.shape[0] > 1:
    x2 = x2.contiguous()
  return x2


def _ids64(t: Optional[torch.Tensor], *shape) -> Optional[torch.Tensor]:
  if t is None or (t.dtype == torch.int64 and t.dim() == len(shape) and t.is_contiguous()):
    return t
  return t.reshape(shape).to(torch.int64).contiguous()


def _lead(t: Optional[torch.Tensor], *shape) -> Optional[torch.Tensor]:
  return t if t is None or t.dim() == len(shape) else t.view(shape)


def top_logprobs(logits: torch.Tensor, k: int, targets: Optional[torch.Tensor] = None, temperature: float = 1.0,
                 want_entropy: bool = False) -> TopLogprobs:
  """The `k` likeliest tokens of every row of logits [..., V] under softmax(logits / temperature), with their
  log-probabilities, the log-probability of `targets` [...] and the entropy; all differentiable but for the ids.

  Tokens of equal logits come by the lowest id, a NaN counts as the largest logit. A target outside the vocabulary
  is ignored (0, no gradient). Logits of -inf are masked out; a row that has nothing else gets log-probabilities of
  -inf, entropy 0 and no gradient. fp32 and bf16 logits on the GPU, rows of any alignment and stride, take one
  kernel in each direction; there `k` is at most 256, and a logit tensor with a tangent of forward mode is refused."""
  _check_rows("top_logprobs", logits, temperature)
  V, lead = logits.shape[-1], logits.shape[:-1]
  if targets is not None:
    _check_index("top_logprobs", "targets", targets, lead, logits)
  k = int(k)
  if not 1 <= k <= V:
    raise ValueError(f"top_logprobs: k must be between 1 and the vocabulary's {V}, got {k}")
  x2 = _rows("top_logprobs", logits)
  tg = _ids64(targets, -1)
  if x2 is None:
    ids, top, target, ent = ref.top_logprobs(logits.reshape(-1, V), k, tg, float(temperature), want_entropy)
  else:
    if k > kernels.MAX_TOP_K:
      raise ValueError(f"top_logprobs: k is at most {kernels.MAX_TOP_K} on the GPU, got {k}")
    if _differentiated(x2):
      ids, top, target, ent = _TopLogprobsFn.apply(x2, k, tg, 1.0 / float(temperature), bool(want_entropy))
    else:
      ids, top, target, ent, _ = kernels.top_logprobs_fwd(x2, k, tg, 1.0 / float(temperature), bool(want_entropy))
  return TopLogprobs(_lead(ids, *lead, k), _lead(top, *lead, k), _lead(target, *lead), _lead(ent, *lead),
                     temperature)


def top_distill_loss(logits: torch.Tensor, top_ids: torch.Tensor, top_values: torch.Tensor,
                     labels: Optional[torch.Tensor] = None, temperature: float = 1.0,
                     normalize: str = "top", twice: bool = False) -> DistillLoss:
  """Distillation from a teacher's best tokens: per row of the student's logits [..., V] the divergence from the
  teacher's list (`top_ids`, `top_values` [..., k]) and, with `labels` [...], the cross entropy at temperature 1.

  normalize="top": both sides are renormalised over the list, KL(softmax(values / T) || softmax(logits[ids] / T));
    the values may be logits or log-probabilities.
  normalize="full": the values are log-probabilities t of the teacher over its whole vocabulary at this temperature
    (`top_logprobs(teacher, k, temperature=T).top`), the student is normalised over its whole vocabulary:
    sum_i exp(t_i) (t_i - log p_T(ids_i)). What the list leaves out does not count.

  The gradient goes to the logits only. An id outside the vocabulary is an absent entry and a label outside it is
  ignored; an entry of probability 0 adds nothing. A row without a usable entry (no id left, teacher's values all
  -inf, student's logits there all -inf) has divergence 0 and no gradient, a row of -inf also no cross entropy.
  With `twice` a backward pass that builds a graph takes the plain statement, whose gradient can be differentiated
  again; without it such a gradient leads to an error.
  fp32 and bf16 logits on the GPU take one kernel in each direction (a list without labels two for its gradient); there
  the list has at most 1024 entries and a tangent of forward mode is refused."""
  _check_rows("top_distill_loss", logits, temperature)
  V, lead = logits.shape[-1], logits.shape[:-1]
  k = top_ids.shape[-1] if top_ids.dim() else 0
  _check_index("top_distill_loss", "top_ids", top_ids, (*lead, k), logits)
  if labels is not None:
    _check_index("top_distill_loss", "labels", labels, lead, logits)
  if normalize not in ("top", "full"):
    raise ValueError(f"top_distill_loss: normalize must be 'top' or 'full', got {normalize!r}")
  if k < 1 or V < 1:
    raise ValueError(f"top_distill_loss: needs a list of at least one entry and a vocabulary, got k={k}, V={V}")
  if top_values.shape != top_ids.shape or not top_values.is_floating_point():
    raise ValueError(f"top_distill_loss: top_values must be floating and shaped like top_ids {tuple(top_ids.shape)}, "
                     f"got {top_values.dtype} {tuple(top_values.shape)}")
  if top_values.device != logits.device:
    raise ValueError(f"top_distill_loss: top_values is on {top_values.device}, the logits on {logits.device}")
  if _differentiated(top_values):
    raise ValueError("top_distill_loss: the teacher's values get no gradient; detach them")
  x2 = _rows("top_distill_loss", logits)
  ids, tg = _ids64(top_ids, -1, k), _ids64(labels, -1)
  full = normalize == "full"
  if x2 is None:
    kl, nll = ref.top_distill_loss(logits.reshape(-1, V), ids, top_values.reshape(-1, k), tg, float(temperature), full)
  else:
    if k > kernels.MAX_TOP_LIST:
      raise ValueError(f"top_distill_loss: the list has at most {kernels.MAX_TOP_LIST} entries on the GPU, got {k}")
    values = top_values
    if values.dtype != torch.float32 or values.dim() != 2 or values.requires_grad or not values.is_contiguous():
      values = values.detach().reshape(-1, k).float().contiguous()
    if _differentiated(x2):
      kl, nll = _TopDistillFn.apply(x2, ids, values, tg, 1.0 / float(temperature), full,
                                    float(temperature) if twice else None)
    else:
      kl, nll, _ = kernels.top_distill_fwd(x2, ids, values, tg, 1.0 / float(temperature), full)
  return DistillLoss(_lead(kl, *lead), _lead(nll, *lead))
