"""`functional.top_logprobs` and `functional.top_distill_loss` against their definitions in 64 bits: values, ties,
masked and empty rows, gradients (formula and differences), refusals; on the CPU and, marked gpu, the kernels."""
import math

import pytest
import torch

from tunix_b200.ops import functional as F

LOW = float("-inf")
f64 = torch.float64


# ------------------------------------------------------------------------------ definitions in 64 bits
def log_softmax64(z):
  """Row-wise, a row of -inf gives -inf."""
  m = z.amax(1, keepdim=True)
  empty = m == LOW
  d = torch.where(empty, torch.full_like(z, LOW), z - torch.where(empty, torch.zeros_like(m), m))
  s = d.exp().sum(1, keepdim=True)
  return torch.where(empty, d, d - torch.where(empty, torch.ones_like(s), s).log())


def score64(x, k, targets, tau, g_top=None, g_target=None, g_ent=None):
  """Values and the gradient's formula for logits x [T, V]; the gradient of an empty row is zero."""
  x = x.to(f64)
  V = x.shape[1]
  empty = (x == LOW).all(1)
  lp = log_softmax64(x / tau)
  p = lp.exp()
  ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
  plp = torch.where(p == 0, torch.zeros_like(p), p * lp)
  out = {"ids": ids, "top": lp.gather(1, ids), "entropy": -plp.sum(1)}
  grad = torch.zeros_like(x)
  total = torch.zeros_like(x[:, 0])
  if g_top is not None:
    grad.scatter_add_(1, ids, g_top.to(f64))
    total = total + g_top.to(f64).sum(1)
  if targets is not None:
    known = (targets >= 0) & (targets < V)
    at = targets.long().clamp(0, V - 1)[:, None]
    out["target"] = torch.where(known, lp.gather(1, at)[:, 0], torch.zeros_like(total))
    if g_target is not None:
      g = torch.where(known, g_target.to(f64), torch.zeros_like(total))
      grad.scatter_add_(1, at, g[:, None])
      total = total + g
  grad = grad - p * total[:, None]
  if g_ent is not None:
    grad = grad - g_ent.to(f64)[:, None] * (plp + p * out["entropy"][:, None])
  out["grad"] = torch.where(empty[:, None], torch.zeros_like(grad), grad / tau)
  return out


def distill64(x, ids, values, labels, tau, full, g_kl=None, g_nll=None):
  x, t = x.to(f64), values.to(f64)
  T, V = x.shape
  grad = torch.zeros_like(x)
  kl = torch.zeros(T, dtype=f64, device=x.device)
  nll = torch.zeros_like(kl)
  lp_t, lp_1 = log_softmax64(x / tau), log_softmax64(x)
  empty = (x == LOW).all(1)
  for r in range(T):
    keep = (ids[r] >= 0) & (ids[r] < V)
    at, tv = ids[r][keep].long(), t[r][keep]
    if full:
      live = not empty[r]
      lq, lp = tv, lp_t[r][at]
      q = lq.exp()
    else:
      live = at.numel() > 0 and bool((tv != LOW).any()) and bool((x[r][at] != LOW).any())
      if live:
        lq, lp = log_softmax64(tv[None] / tau)[0], log_softmax64(x[r][at][None] / tau)[0]
        q = lq.exp()
    if live:
      kl[r] = (q * (lq - lp))[q != 0].sum()
      if g_kl is not None:
        g = float(g_kl[r]) / tau
        if full:
          grad[r] += g * q.sum() * lp_t[r].exp()
          grad[r].index_add_(0, at, -g * q)
        else:
          grad[r].index_add_(0, at, g * (lp.exp() - q))
    if labels is not None and 0 <= int(labels[r]) < V and not empty[r]:
      nll[r] = -lp_1[r, int(labels[r])]
      if g_nll is not None:
        grad[r] += float(g_nll[r]) * lp_1[r].exp()
        grad[r, int(labels[r])] -= float(g_nll[r])
  return {"kl": kl, "nll": nll, "grad": grad}


# ------------------------------------------------------------------------------ tolerances
U = 2.0 ** -24        # half a step of fp32, relative


def finite_span(z):
  """Largest distance of a finite entry from its row's maximum, and 1 for rows without any."""
  m = z.amax(1, keepdim=True)
  d = torch.where(torch.isfinite(z) & torch.isfinite(m), m - z, torch.zeros_like(z))
  return d.clamp(max=100.0)       # beyond exp(-100) a term does not count in fp32


def lse_tol(x, tau):
  """Bound of |ln s - exact|, relative error of s: a term's exponent is off by 3 roundings of an argument of d / tau
  (subtraction, scale, product; the scale itself holds two more), its exponential by 2^-22, and each of the additions
  a thread makes by U (a row is spread over at least 32 threads of 8 elements); ln itself by 2 U |ln s| + 2^-23."""
  V = x.shape[1]
  arg = 5 * U * (finite_span(x.to(f64) / tau) * log_softmax64(x.to(f64) / tau).exp().nan_to_num()).sum(1)
  return arg + 2 ** -22 + U * (V / 256 + 64) + 2 * U * math.log(V + 1) + 2 ** -23


def lp_tol(x, tau):
  """Bound per element of log p = d / tau - ln s: three roundings of d / tau, one of the difference."""
  span = (x.to(f64).amax(1, keepdim=True) - x.to(f64)).abs() / tau
  return 4 * U * span.nan_to_num(0, 0, 0) + lse_tol(x, tau)[:, None] * (1 + U) + 2 * U * math.log(x.shape[1] + 1)


def p_tol(x, tau):
  """Bound per element of p: p times the error of its exponent (at most 100, terms beyond are 0) and 2^-22."""
  p = log_softmax64(x.to(f64) / tau).exp()
  return p * (6 * U * finite_span(x.to(f64) / tau) + lse_tol(x, tau)[:, None] + 4 * U * math.log(x.shape[1] + 1) + 2 ** -21) \
      + 2.0 ** -126


def close(got, want, tol, what):
  got, want = got.to(f64), want.to(f64)
  assert got.shape == want.shape, what
  # a value beyond fp32 (the lowest float divided by a temperature below 1) rounds to infinity
  want = torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * math.inf, want)
  odd = ~torch.isfinite(want)
  same = (got[odd] == want[odd]) | (torch.isnan(got[odd]) & torch.isnan(want[odd]))
  assert bool(same.all()), f"{what}: {got[odd][~same][:4]} for {want[odd][~same][:4]}"
  off = (got - want).detach().abs()[~odd] - tol.to(f64).expand(want.shape)[~odd]
  assert off.numel() == 0 or float(off.nan_to_num(math.inf).max()) <= 0, f"{what}: {float(off.max()):.3e} above the bound"


def check_score(x, k, targets, tau, dtype_eps, seed=0, want_entropy=True):
  """Values and gradients of `top_logprobs` on x (a leaf is made of it) against 64 bits."""
  g = torch.Generator(device=x.device).manual_seed(seed)
  T, V = x.shape
  rnd = lambda *s: torch.randn(*s, generator=g, device=x.device)   # noqa: E731
  g_top, g_target, g_ent = rnd(T, k), rnd(T), rnd(T)
  leaf = x.detach().requires_grad_()
  got = F.top_logprobs(leaf, k, targets, temperature=tau, want_entropy=want_entropy)
  want = score64(x, k, targets, tau, g_top, g_target if targets is not None else None, g_ent if want_entropy else None)
  assert got.ids.dtype == torch.int64 and torch.equal(got.ids, want["ids"])
  lt = lp_tol(x, tau)
  close(got.top, want["top"], lt.gather(1, want["ids"]), "top")
  pt = p_tol(x, tau)
  outs, grads = [got.top], [g_top]
  mag = g_top.abs().sum(1)
  if targets is not None:
    close(got.target, want["target"], lt.gather(1, targets.long().clamp(0, V - 1)[:, None])[:, 0], "target")
    outs, grads, mag = outs + [got.target], grads + [g_target], mag + g_target.abs()
  else:
    assert got.target is None
  lp = log_softmax64(x.to(f64) / tau)
  surprise = torch.where(lp > -745, lp.abs(), torch.zeros_like(lp))      # where p is not 0
  if want_entropy:
    # H = ln s - sum w d / (tau s): the terms' errors weighted by their size, V / 256 + 64 additions of parts of the sum
    ht = (pt * (surprise + 2)).sum(1) * 2 + lse_tol(x, tau) * 2 + U * (V / 256 + 80) * ((lp.exp() * surprise).sum(1) + math.log(V + 1))
    close(got.entropy, want["entropy"], ht, "entropy")
    outs, grads = outs + [got.entropy], grads + [g_ent]
  else:
    assert got.entropy is None
    ht = torch.zeros_like(mag)
  dx, = torch.autograd.grad(outs, leaf, grads)
  assert dx.dtype == x.dtype and dx.shape == x.shape
  e = g_ent.abs() if want_entropy else torch.zeros_like(mag)
  p = lp.exp()
  tol = (pt * mag[:, None] + (k + 4) * U * mag[:, None] * p
         + e[:, None] * (pt * (surprise + math.log(V + 1) + 1) + p * (lt.nan_to_num(0, 0, 0) + ht[:, None])
                         + 6 * U * p * (surprise + math.log(V + 1)))) / tau
  listed = torch.zeros_like(p).scatter_add_(1, want["ids"], g_top.abs().to(f64))
  if targets is not None:
    listed.scatter_add_(1, targets.long().clamp(0, V - 1)[:, None], g_target.abs().to(f64)[:, None])
  tol = tol + 6 * U * listed / tau + dtype_eps / 2 * want["grad"].abs() * (1 + 2 ** -6) + 2.0 ** -130
  close(dx, want["grad"], tol, "gradient")


def check_distill(x, ids, values, labels, tau, full, dtype_eps, seed=0):
  g = torch.Generator(device=x.device).manual_seed(seed)
  T, V = x.shape
  g_kl = torch.rand(T, generator=g, device=x.device) + 0.1
  g_nll = torch.rand(T, generator=g, device=x.device) + 0.1 if labels is not None else None
  leaf = x.detach().requires_grad_()
  got = F.top_distill_loss(leaf, ids, values, labels, temperature=tau, normalize="full" if full else "top")
  want = distill64(x, ids, values, labels, tau, full, g_kl, g_nll)
  there = (ids >= 0) & (ids < V)
  at = ids.long().clamp(0, V - 1)
  t = torch.where(there, values.to(f64), torch.full_like(values, LOW, dtype=f64))
  xs = torch.where(there, x.to(f64).gather(1, at), torch.full_like(t, LOW))
  if full:
    q = t.exp()
    qt = q * (2 ** -22)                                           # expf: 2 ulp
    lpt = lp_tol(x, tau).gather(1, at)
    lq, lp = t, log_softmax64(x.to(f64) / tau).gather(1, at)
  else:
    q, qt = log_softmax64(t / tau).exp(), p_tol(t, tau)
    lpt = lp_tol(xs, tau) + lp_tol(t, tau)
    lq, lp = log_softmax64(t / tau), log_softmax64(xs / tau)
  diff = torch.where((q > 0) & torch.isfinite(lq - lp), (lq - lp).abs(), torch.zeros_like(q))
  mass = torch.where(q > 0, q * (diff + lq.abs().nan_to_num(0, 0, 0)), torch.zeros_like(q)).sum(1)
  klt = (qt * diff + q * lpt.nan_to_num(0, 0, 0)).sum(1) + U * (ids.shape[1] + 8) * mass
  close(got.kl, want["kl"], klt + 2.0 ** -120, "kl")
  pairs = [(got.kl, g_kl)]
  p1t = p_tol(x, 1.0)
  tol = torch.zeros_like(p1t)
  listed = torch.zeros_like(p1t)
  gk = g_kl.to(f64)[:, None] / tau
  if full:
    Q = q.sum(1, keepdim=True)
    p = log_softmax64(x.to(f64) / tau).exp()
    tol = tol + gk * (Q * p_tol(x, tau) + p * (qt.sum(1, keepdim=True) + U * (ids.shape[1] + 8) * Q))
    listed.scatter_add_(1, at, gk * (qt + 6 * U * q))
  else:
    ps = log_softmax64(xs / tau).exp()
    listed.scatter_add_(1, at, gk * (p_tol(xs, tau) + qt + 6 * U * (ps + q)))
  if labels is None:
    assert got.nll is None
  else:
    lab = labels.long().clamp(0, V - 1)[:, None]
    close(got.nll, want["nll"], lp_tol(x, 1.0).gather(1, lab)[:, 0], "nll")
    pairs.append((got.nll, g_nll))
    gn = g_nll.to(f64)[:, None]
    tol = tol + gn * (p1t + 4 * U * log_softmax64(x.to(f64)).exp())
    listed.scatter_add_(1, lab, 4 * U * gn)
  dx, = torch.autograd.grad([a for a, _ in pairs], leaf, [b for _, b in pairs])
  assert dx.dtype == x.dtype and dx.shape == x.shape
  tol = tol + listed + dtype_eps / 2 * want["grad"].abs() * (1 + 2 ** -6) + 2.0 ** -130
  close(dx, want["grad"], tol, "gradient")


def make_logits(T, V, dtype, device, seed=0):
  g = torch.Generator().manual_seed(seed)
  x = torch.randn(T, V, generator=g) * 2
  x[:, torch.randperm(V, generator=g)[:min(V, 9)]] += 6 * torch.rand(T, min(V, 9), generator=g)
  return x.to(device=device, dtype=dtype)


def odd_rows(V, dtype, device):
  """Rows in which a selection or a softmax can go wrong, one of each kind."""
  lowest = torch.finfo(dtype).min
  r = torch.randn(V, generator=torch.Generator().manual_seed(3))
  up = torch.linspace(-8, 8, V)
  few = torch.full((V,), LOW)
  few[V // 3], few[V - 1] = 1.5, 1.5
  some = r.clone()
  some[: V // 2] = LOW
  far = r.clone()
  far[V // 2] = 30000.0
  rows = [up, up.flip(0), torch.zeros(V), torch.full((V,), LOW), few, some, torch.full((V,), lowest),
          torch.where(torch.arange(V) % 3 == 0, r, torch.full((V,), lowest)), r.sign(), -torch.zeros(V),
          torch.where(torch.arange(V) % 2 == 0, torch.zeros(V), -torch.zeros(V)), r * 100, far, r * 1e-3]
  return torch.stack(rows).to(device=device, dtype=dtype)


def make_list(x, k, seed=0, tau=1.0):
  """A teacher's list near the student's logits."""
  g = torch.Generator().manual_seed(seed)
  t = x.detach().float().cpu().nan_to_num(0, 0, -30).clamp(-50, 50)
  t = t + torch.randn(t.shape, generator=g)
  top, ids = torch.topk(torch.log_softmax(t / tau, 1), k, dim=1)
  return ids.to(x.device), top.to(x.device)


DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16]


def eps(dtype):
  return torch.finfo(dtype).eps


# ------------------------------------------------------------------------------ values and gradients
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,k,tau,entropy", [
    (1, 1, 1, 1.0, True), (3, 7, 7, 0.5, True), (5, 257, 17, 1.0, False), (2, 256, 256, 2.0, True),
    (4, 1000, 64, 1.0, True), (3, 4097, 256, 1.3, True), (7, 9001, 5, 0.7, False), (2, 32003, 100, 1.0, True),
    (3, 70001, 256, 1.0, True), (2, 200003, 3, 0.9, True),
])
def test_top_logprobs(device, dtype, T, V, k, tau, entropy):
  x = make_logits(T, V, dtype, device, seed=V)
  targets = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(1)).to(device)
  check_score(x, k, targets, tau, eps(dtype), want_entropy=entropy)
  check_score(x, k, None, tau, eps(dtype), want_entropy=entropy)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(6, 3), (300, 40), (5000, 256), (20011, 33), (140001, 200)])
def test_top_logprobs_of_odd_rows(device, dtype, V, k):
  x = odd_rows(V, dtype, device)
  targets = torch.arange(x.shape[0], device=device) % V
  targets[1], targets[2] = -100, V                                  # ignored
  check_score(x, k, targets, 1.0, eps(dtype))
  check_score(x, k, targets, 0.6, eps(dtype))


@pytest.mark.parametrize("device", DEVICES)
def test_equal_logits_come_by_the_lowest_id(device):
  V = 30000
  x = torch.zeros(3, V, device=device)
  x[1] = torch.randint(0, 3, (V,), generator=torch.Generator().manual_seed(0)).float().to(device)
  x[2, V // 2:] = 1.0
  got = F.top_logprobs(x, 100)
  assert got.ids[0].tolist() == list(range(100))
  assert got.ids[1].tolist() == (x[1] == 2).nonzero()[:100, 0].tolist()
  assert got.ids[2].tolist() == list(range(V // 2, V // 2 + 100))
  assert got.target is None and got.entropy is None


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_nan_and_infinity_stay_in_their_row(device, dtype):
  x = make_logits(4, 5000, dtype, device)
  x[1, 4321] = float("nan")
  x[2, 17] = float("inf")
  want = score64(x[[0, 3]], 8, None, 1.0)
  got = F.top_logprobs(x, 8, torch.zeros(4, dtype=torch.long, device=device), want_entropy=True)
  assert torch.equal(got.ids[[0, 3]], want["ids"])
  close(got.top[[0, 3]], want["top"], lp_tol(x[[0, 3]], 1.0).gather(1, want["ids"]), "top")
  assert int(got.ids[1, 0]) == 4321 and int(got.ids[2, 0]) == 17
  for t in (got.top, got.target, got.entropy):
    assert bool(t[1].isnan().all()) and bool(t[2].isnan().all())
  ids, values = make_list(x, 8)
  loss = F.top_distill_loss(x, ids, values, torch.zeros(4, dtype=torch.long, device=device), normalize="full")
  assert bool(loss.kl.isnan().tolist() == [False, True, True, False]) and loss.nll.isnan().tolist() == [False, True, True, False]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("full", [False, True])
@pytest.mark.parametrize("T,V,k,tau,labelled", [
    (1, 1, 1, 1.0, True), (3, 7, 7, 0.5, True), (5, 257, 17, 1.0, False), (4, 1000, 64, 2.0, True),
    (2, 5000, 1000, 1.0, True), (7, 9001, 5, 1.7, False), (2, 32003, 100, 3.0, True),
])
def test_top_distill_loss(device, dtype, full, T, V, k, tau, labelled):
  x = make_logits(T, V, dtype, device, seed=V)
  ids, values = make_list(x, k, tau=tau if full else 1.0)
  labels = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(1)).to(device) if labelled else None
  check_distill(x, ids, values, labels, tau, full, eps(dtype))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("full", [False, True])
def test_top_distill_loss_of_odd_rows_and_lists(device, dtype, full):
  V, k = 5000, 24
  x = odd_rows(V, dtype, device)
  T = x.shape[0]
  ids, values = make_list(x, k)
  labels = torch.arange(T, device=device) % V
  labels[1], labels[2] = -100, V
  check_distill(x, ids, values, labels, 1.0, full, eps(dtype))
  x = make_logits(T, V, dtype, device)
  ids, values = make_list(x, k)
  ids[0] = -1                                                       # nothing listed
  ids[1, 5:] = -1                                                   # a shorter list
  ids[2, 3] = V                                                     # outside the vocabulary
  ids[3] = ids[3, 0]                                                # one column, many times
  ids[4, 1] = ids[4, 0]                                             # one twice
  labels[4] = ids[4, 0]                                             # and the label too
  values[5] = LOW                                                   # teacher has nothing
  values[6, ::2] = LOW
  x[7, ids[7]] = LOW                                                # student has nothing of the list
  x[8, ids[8, 1:]] = LOW
  values[8, 1:] = LOW
  check_distill(x, ids, values, labels, 1.4, full, eps(dtype))
  x[9, ids[9, 0]] = LOW                                             # the teacher's best is impossible
  got = F.top_distill_loss(x, ids, values, labels, normalize="full" if full else "top")
  assert float(got.kl[9]) == math.inf and bool(torch.isfinite(got.kl[:7]).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignments(device, dtype):
  V, k = 4999, 12
  for cut in (0, 1, 3, 5):
    wide = make_logits(5, V + 40, dtype, device)
    x = wide[:, cut:cut + V]
    targets = torch.arange(5, device=device)
    check_score(x, k, targets, 1.0, eps(dtype))
    ids, values = make_list(x, k)
    check_distill(x, ids, values, targets, 2.0, True, eps(dtype))
    check_distill(x, ids.to(torch.int32), values.to(torch.float64).float(), targets.to(torch.int32), 2.0, False, eps(dtype))
  x = make_logits(V, 6, dtype, device).t()                         # columns are not contiguous
  check_score(x, k, None, 1.0, eps(dtype))
  x = make_logits(1, V, dtype, device).expand(3, V)
  check_score(x, k, None, 1.0, eps(dtype))


@pytest.mark.parametrize("device", DEVICES)
def test_leading_dimensions_and_missing_gradients(device):
  x = make_logits(6, 50, torch.float32, device).view(2, 3, 50).requires_grad_()
  targets = torch.randint(0, 50, (2, 3), device=device)
  got = F.top_logprobs(x, 4, targets, want_entropy=True)
  assert got.ids.shape == got.top.shape == (2, 3, 4) and got.target.shape == got.entropy.shape == (2, 3)
  assert not got.ids.requires_grad and got.top.requires_grad
  want = torch.log_softmax(x, -1).gather(-1, targets[..., None])[..., 0]
  gw, = torch.autograd.grad(want.sum(), x)
  g, = torch.autograd.grad(got.target.sum(), x, retain_graph=True)   # an expanded gradient, the others missing
  torch.testing.assert_close(g, gw, rtol=1e-5, atol=1e-6)
  e, = torch.autograd.grad(got.entropy.mean(), x)
  h = -(torch.log_softmax(x, -1) * torch.softmax(x, -1)).sum(-1)
  torch.testing.assert_close(e, torch.autograd.grad(h.mean(), x)[0], rtol=1e-4, atol=1e-7)
  loss = F.top_distill_loss(x, got.ids, got.top.detach(), targets)
  assert loss.kl.shape == loss.nll.shape == (2, 3)
  g, = torch.autograd.grad(loss.nll.sum(), x, retain_graph=True)
  torch.testing.assert_close(g, -gw, rtol=1e-5, atol=1e-6)
  # the student is the teacher here: divergence 0 and no gradient, but for two log-probabilities (of at most 16 in
  # size) that are off by 4 U of that and the sums of four terms: 2 (4 U 16 + 8 U) < 1e-5
  assert float(loss.kl.detach().abs().max()) < 1e-5
  g, = torch.autograd.grad(loss.kl.sum(), x)
  assert float(g.abs().max()) < 1e-5
  empty = torch.zeros(0, 50, device=device, requires_grad=True)
  none = F.top_logprobs(empty, 4, torch.zeros(0, dtype=torch.long, device=device), want_entropy=True)
  assert none.ids.shape == (0, 4) and none.entropy.shape == (0,)
  assert torch.autograd.grad(none.top.sum(), empty)[0].shape == (0, 50)
  got = F.top_logprobs(x.detach()[0, 0], 3)                          # a single row
  assert got.ids.shape == (3,)


def test_gradients_by_differences():
  x = make_logits(4, 23, torch.float64, "cpu").requires_grad_()
  targets = torch.tensor([0, 5, 22, -1])
  assert torch.autograd.gradcheck(lambda z: F.top_logprobs(z, 6, targets, temperature=0.8, want_entropy=True)[1:], (x,))
  ids, values = make_list(x, 6)
  for normalize in ("top", "full"):
    assert torch.autograd.gradcheck(lambda z: tuple(F.top_distill_loss(z, ids, values.double(), targets, 1.7, normalize)), (x,))


@pytest.mark.gpu
def test_kernel_gradients_by_differences():
  """Central differences of the fp32 kernel: truncation h^2 / 6 times a third derivative of at most 2 / tau^3, and
  rounding 2 lp_tol / 2h of each of the 8 summed outputs."""
  x = make_logits(3, 700, torch.float32, "cuda")
  targets = torch.tensor([3, 699, 0], device="cuda")
  w = torch.randn(3, 6, generator=torch.Generator().manual_seed(2)).cuda()

  def total(z):
    got = F.top_logprobs(z, 6, targets, temperature=1.5, want_entropy=True)
    return (got.top * w).sum(1) + got.target - 0.5 * got.entropy

  leaf = x.clone().requires_grad_()
  grad, = torch.autograd.grad(total(leaf).sum(), leaf)
  h = 2.0 ** -6
  tol = float(w.abs().sum(1).max() + 3) * (h * h / 3 + float(lse_tol(x, 1.5).max() + lp_tol(x, 1.5).max()) / h)
  for col in [0, 3, 699] + F.top_logprobs(x, 6).ids[0].tolist():
    step = torch.zeros_like(x)
    step[:, col] = h
    diff = (total(x + step) - total(x - step)) / (2 * h)
    assert float((diff - grad[:, col]).abs().max()) <= tol


# ------------------------------------------------------------------------------ refusals
@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
  x = torch.randn(2, 40, device=device)
  ids, values = make_list(x, 5)
  t = torch.zeros(2, dtype=torch.long, device=device)
  for k in (0, -1, 41):
    with pytest.raises(ValueError, match="k must be between"):
      F.top_logprobs(x, k)
  for bad in (0.0, -1.0, 1e-19, 1e19, math.inf, math.nan):
    with pytest.raises(ValueError, match="temperature"):
      F.top_logprobs(x, 3, temperature=bad)
    with pytest.raises(ValueError, match="temperature"):
      F.top_distill_loss(x, ids, values, temperature=bad)
  with pytest.raises(ValueError, match="targets must have shape"):
    F.top_logprobs(x, 3, t[:1])
  with pytest.raises(ValueError, match="int32 or int64"):
    F.top_logprobs(x, 3, t.float())
  with pytest.raises(ValueError, match="floating"):
    F.top_logprobs(torch.zeros(2, 40, dtype=torch.long, device=device), 3)
  with pytest.raises(ValueError, match="normalize"):
    F.top_distill_loss(x, ids, values, normalize="tail")
  with pytest.raises(ValueError, match="shaped like top_ids"):
    F.top_distill_loss(x, ids, values[:, :4])
  with pytest.raises(ValueError, match="shaped like top_ids"):
    F.top_distill_loss(x, ids, ids)
  with pytest.raises(ValueError, match="top_ids must have shape"):
    F.top_distill_loss(x, ids[:1], values[:1])
  with pytest.raises(ValueError, match="labels must have shape"):
    F.top_distill_loss(x, ids, values, t[:1])
  with pytest.raises(ValueError, match="at least one entry"):
    F.top_distill_loss(x, ids[:, :0], values[:, :0])
  with pytest.raises(ValueError, match="detach"):
    F.top_distill_loss(x, ids, values.clone().requires_grad_())
  with pytest.raises(ValueError, match="meta"):
    F.top_logprobs(x, 3, t.to("meta"))


@pytest.mark.gpu
def test_refusals_of_the_kernels():
  x = torch.randn(2, 2000, device="cuda")
  with pytest.raises(ValueError, match="at most 256"):
    F.top_logprobs(x, 257)
  ids = torch.zeros(2, 1025, dtype=torch.long, device="cuda")
  with pytest.raises(ValueError, match="at most 1024"):
    F.top_distill_loss(x, ids, ids.float())
  with pytest.raises(ValueError, match="on cpu"):
    F.top_logprobs(x, 3, torch.zeros(2, dtype=torch.long))


@pytest.mark.gpu
def test_second_derivatives_are_refused():
  x = torch.randn(3, 500, device="cuda", requires_grad=True)
  ids, values = make_list(x, 4)
  for out in (F.top_logprobs(x, 4).top, F.top_distill_loss(x, ids, values).kl):
    g, = torch.autograd.grad(out.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
      g.sum().backward()


@pytest.mark.gpu
def test_blocks_of_logits_beyond_32_bits():
  """Rows behind the 2^31st element of a block, and their gradients."""
  T, V, k = 17000, 131072, 10
  x = torch.zeros(T, V, device="cuda", dtype=torch.bfloat16)
  x[-4:] = make_logits(4, V, torch.bfloat16, "cuda")
  x.requires_grad_()
  last = x.detach()[-4:]
  targets = torch.arange(T, device="cuda")
  got = F.top_logprobs(x, k, targets)
  want = score64(last, k, targets[-4:], 1.0, torch.ones(4, k, device="cuda"))
  assert torch.equal(got.ids[-4:], want["ids"])
  close(got.top[-4:], want["top"], lp_tol(last, 1.0).gather(1, want["ids"]), "top")
  assert torch.equal(got.ids[0], torch.arange(k, device="cuda"))
  g, = torch.autograd.grad(got.top, x, torch.ones(T, k, device="cuda"))
  tol = (k + 2) * p_tol(last, 1.0) + (k + 8) * U * (1 + log_softmax64(last.to(f64)).exp()) \
      + 2.0 ** -8 * want["grad"].abs() * (1 + 2 ** -6) + 2.0 ** -130
  close(g[-4:], want["grad"], tol, "gradient")
  del got, g
  ids, values = make_list(last, k)
  ids, values = ids.repeat(T // 4, 1), values.repeat(T // 4, 1)
  loss = F.top_distill_loss(x, ids, values, None, temperature=2.0)
  g, = torch.autograd.grad(loss.kl.sum(), x)
  alone = distill64(last, ids[-4:], values[-4:], None, 2.0, False, torch.ones(4))
  assert float((loss.kl[-4:].detach().to(f64) - alone["kl"]).abs().max()) <= 1e-4
  assert float((g[-4:].to(f64) - alone["grad"]).abs().max()) <= 2.0 ** -8
  assert int((g[0] != 0).sum()) <= k and int((g[T // 2] != 0).sum()) <= k


@pytest.mark.gpu
def test_another_device_than_the_process_is_refused(monkeypatch):
  from tunix_b200.ops import _lib
  x = torch.randn(2, 100, device="cuda")
  ids, values = make_list(x, 3)
  monkeypatch.setattr(_lib, "bind_thread", lambda: 1)
  with pytest.raises(ValueError, match="this process drives cuda:1"):
    F.top_logprobs(x, 3)
  with pytest.raises(ValueError, match="this process drives cuda:1"):
    F.top_distill_loss(x, ids, values)


@pytest.mark.gpu
def test_more_rows_than_31_bits_are_refused():
  x = torch.zeros(1, 1, device="cuda").expand(2 ** 31, 1)                  # no memory behind it
  with pytest.raises(ValueError, match="31 bits"):
    F.top_logprobs(x, 1)
  with pytest.raises(ValueError, match="31 bits"):
    F.top_distill_loss(x, torch.zeros(1, 1, dtype=torch.int64, device="cuda").expand(2 ** 31, 1), x)


@pytest.mark.gpu
def test_repeated_calls_agree_to_the_bit():
  """Candidates are collected in any order; what is reported does not depend on it."""
  x = make_logits(40, 50000, torch.bfloat16, "cuda")
  targets = torch.arange(40, device="cuda")
  first = F.top_logprobs(x, 64, targets, want_entropy=True)
  many = x.repeat(20, 1)                           # another number of blocks per row
  other = F.top_logprobs(many, 64, targets.repeat(20), want_entropy=True)
  for _ in range(5):
    again = F.top_logprobs(x, 64, targets, want_entropy=True)
    more = F.top_logprobs(many, 64, targets.repeat(20), want_entropy=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    assert all(torch.equal(a, b) for a, b in zip(other, more))
  assert torch.equal(first.ids, other.ids[:40])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tau", [1e-18, 1e-6, 1e-3, 1e3, 1e18])
def test_extreme_temperatures(device, tau):
  """Cold: one token takes everything (the smallest temperatures leave the range in which sums are taken in one pass).
  Hot: all tokens are alike."""
  x = make_logits(3, 6000, torch.float32, device)
  x[:, 77] = x.amax(1) + 1.0                                       # a clear best token
  got = F.top_logprobs(x, 5, torch.zeros(3, dtype=torch.long, device=device), temperature=tau, want_entropy=True)
  want = score64(x, 5, torch.zeros(3, dtype=torch.long, device=device), tau)
  assert torch.equal(got.ids, want["ids"])
  close(got.top, want["top"], lp_tol(x, tau).gather(1, want["ids"]), "top")
  close(got.target, want["target"], lp_tol(x, tau)[:, 0], "target")
  p, lp = log_softmax64(x.to(f64) / tau).exp(), log_softmax64(x.to(f64) / tau)
  size = torch.where(p > 0, p * lp.abs(), torch.zeros_like(p)).sum(1) + math.log(6001)
  close(got.entropy, want["entropy"], 4 * lse_tol(x, tau) * (1 + size) + U * 100 * size, "entropy")


# ------------------------------------------------------------------------------ derivatives of other kinds
@pytest.mark.parametrize("device", DEVICES)
def test_a_tangent_is_taken_along_or_refused(device):
  """Forward mode: the plain statement on the CPU has it, the kernels refuse a dual tensor rather than drop its tangent."""
  from torch.autograd import forward_ad
  x = make_logits(3, 50, torch.float32, device)
  v = torch.randn(3, 50, generator=torch.Generator().manual_seed(5)).to(device)
  ids, values = make_list(x, 4)
  table = torch.randn(9, 16, generator=torch.Generator().manual_seed(6)).to(device, torch.bfloat16 if device == "cuda" else torch.float32)
  at = torch.arange(6, device=device)
  calls = [(x, v, lambda z: F.top_logprobs(z, 4).top), (x, v, lambda z: F.top_distill_loss(z, ids, values).kl),
           (table, torch.ones_like(table), lambda z: F.embedding(at, z, 2.0))]
  with forward_ad.dual_level():
    for t, tangent, fn in calls:
      dual = forward_ad.make_dual(t, tangent)
      if device == "cuda":
        with pytest.raises(NotImplementedError):
          fn(dual)
        assert forward_ad.unpack_dual(fn(t)).tangent is None            # others are not affected
      else:
        assert forward_ad.unpack_dual(fn(dual)).tangent is not None
    with pytest.raises(ValueError, match="detach"):
      F.top_distill_loss(x, ids, forward_ad.make_dual(values, torch.ones_like(values)))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tau", [1e-18, 1e-9, 1e-3, 1e9])
def test_gradients_at_extreme_temperatures(device, tau):
  """With masked columns; the smallest temperatures make factors that overflow against an unbounded exponent."""
  x = make_logits(3, 6000, torch.float32, device)
  x[:, 77] = x.amax(1) + 1.0                                       # a clear best token
  x[:, 100:2000] = LOW
  x[1, 2000:2100] = -1e4
  check_score(x, 5, torch.full((3,), 77, device=device), tau, eps(x.dtype))
  check_score(x, 5, torch.full((3,), 2000, device=device), tau, eps(x.dtype))


@pytest.mark.gpu
def test_row_statistics_belong_to_the_graph():
  """What the backward pass reads is saved with the graph: seen by saved-tensor hooks and freed with it."""
  import weakref
  x = make_logits(3, 50, torch.float32, "cuda").requires_grad_()
  ids, values = make_list(x, 4)
  for call in (lambda: F.top_logprobs(x, 4).top, lambda: F.top_distill_loss(x, ids, values, normalize="full").kl):
    seen = []

    def pack(t):
      seen.append((tuple(t.shape), weakref.ref(t)))
      return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
      out = call()
    stats = [r for shape, r in seen if shape in ((3, 2), (3, 8))]
    assert len(stats) == 1
    out.sum().backward()
    del out
    assert stats[0]() is None


@pytest.mark.gpu
def test_both_exponentials_over_their_range():
  """With two temperatures a part of a row's exponentials is made by multiply-adds: one element of every such place and
  of every size, against 64 bits."""
  d = torch.cat([torch.linspace(0, 18, 6000), torch.linspace(18, 90, 1000)])
  d = torch.cat([-d, torch.full((1,), LOW)]).to(torch.bfloat16)
  T = d.numel()
  for place in range(1, 16):
    x = torch.full((T, 16), LOW, dtype=torch.bfloat16)
    x[:, 0] = 0.0
    x[:, place] = d
    x = x.cuda()
    ids, values = torch.zeros(T, 1, dtype=torch.long, device="cuda"), torch.zeros(T, 1, device="cuda")
    got = F.top_distill_loss(x, ids, values, torch.zeros(T, dtype=torch.long, device="cuda"), temperature=2.0, normalize="full")
    w2, w1 = torch.exp(d.to(f64).cuda() / 2), torch.exp(d.to(f64).cuda())
    # ln(1 + w): w off by 2^-22 of itself and by the rounding of its exponent (at most 2^7 in size, 2^-24 of that by
    # the scale and again by the product), the sum by U, the logarithm by 2 U of a number below 1
    for value, w in ((got.kl, w2), (got.nll, w1)):
      tol = w * (2.0 ** -22 + 2 * U * d.to(f64).cuda().abs().clamp_max(100.0)) + 4 * U
      assert float(((value.to(f64) - torch.log1p(w)).abs() - tol).max()) <= 0
