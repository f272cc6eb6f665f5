"""Distillation from a teacher's best tokens as a user runs it: `LogitStrategy` with a top-k or a stored list, the
trainer around it, and a step from the token embedding to the table's gradient; captured and on two streams."""
import math

import pytest
import torch
import torch.nn.functional as F

from tunix_b200 import optim
from tunix_b200.common.configs import TrainingConfig
from tunix_b200.distillation import DistillationTrainer, TrainingInput, strategies
from tunix_b200.models.transformer import ModelConfig, Transformer
from tunix_b200.ops import functional
from tunix_b200.sft import utils as sft_utils

bf16, f64 = torch.bfloat16, torch.float64
DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24


def strategy(**kw):
  return strategies.LogitStrategy(lambda m, **i: None, lambda m, **i: None, lambda **i: None, **kw)


def loss64(s, t, labels, k, tau, alpha):
  """The strategy's loss in 64 bits for integer or one-hot labels, the gradients of its two parts and a bound of the
  terms these are made of."""
  s = s.detach().to(f64).requires_grad_()
  t = t.detach().to(f64)
  rows = s[..., 0].numel()
  tk, idx = torch.topk(t, k, dim=-1)
  lq = F.log_softmax(tk / tau, -1)
  lp = F.log_softmax(s.gather(-1, idx) / tau, -1)
  soft = alpha * (lq.exp() * (lq - lp)).sum(-1).mean() * tau * tau
  lps = F.log_softmax(s, -1)
  hot = F.one_hot(labels, s.shape[-1]).to(f64) if labels.ndim == 2 else labels.to(f64)
  hard = (1 - alpha) * -(lps * hot).sum(-1).mean()
  terms = ((1 - alpha) * (lps.exp() + hot) / rows).scatter_add(-1, idx, alpha * tau * (lq.exp() + lp.exp()) / rows)
  return (soft + hard).detach(), torch.autograd.grad(soft, s)[0], torch.autograd.grad(hard, s)[0], terms.detach()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("one_hot", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, bf16])
def test_strategy_over_logits_and_over_a_list(device, one_hot, dtype):
  B, T, V, k, tau, alpha = 2, 9, 700, 12, 2.0, 0.6
  g = torch.Generator().manual_seed(0)
  # distinct teacher values in either type: no ties at the k-th place
  t = torch.stack([torch.randperm(V, generator=g) for _ in range(B * T)]).view(B, T, V).float().to(device).mul(0.0625).to(dtype)
  if dtype == bf16:
    t = (torch.stack([torch.randperm(V, generator=g) for _ in range(B * T)]).view(B, T, V) % 256).float().to(device)
    t = torch.where(t > 128, t, torch.zeros_like(t)).mul(0.0625)
    rank = torch.argsort(torch.rand(B, T, V, generator=g), -1)[..., :k].to(device)
    t.scatter_(-1, rank, (torch.arange(k, device=device) + 20.0).expand(B, T, k))
    t = t.to(bf16)
  s = (torch.randn(B, T, V, generator=g) * 2).to(device).to(dtype)
  ids = torch.randint(0, V, (B, T), generator=g).to(device)
  labels = F.one_hot(ids, V).float() if one_hot else ids
  want, g_soft, g_hard, terms = loss64(s, t, labels, k, tau, alpha)
  strat = strategy(temperature=tau, alpha=alpha, distill_top_k=k)
  listed = functional.top_logprobs(t, k + 5, ids)
  # fp32 throughout: log-probabilities of at most 64 in size off by 16 roundings each, means of 18 of them
  tol = 64 * 16 * U * (tau * tau + 1)
  for teacher in (t, listed):
    leaf = s.clone().requires_grad_()
    loss, m = strat.compute_loss(leaf, teacher, labels)
    assert abs(float(loss.detach()) - float(want)) <= tol
    assert set(m) == {"distill/soft_loss", "distill/hard_loss", "distill/kl_div", "distill/teacher_loss"}
    assert float(m["distill/teacher_loss"]) == pytest.approx(float(-F.log_softmax(t.double(), -1).gather(-1, ids[..., None]).mean()), abs=tol)
    grad, = torch.autograd.grad(loss, leaf)
    # one-hot labels: the two parts arrive separately, each rounded to the logits' type, and their sum is rounded; an
    # exponent of at most 64 in size off by 8 roundings and 2^-22 of an exponential is 1024 U of a term
    half = torch.finfo(dtype).eps / 2
    near = (grad.to(f64) - (g_soft + g_hard)).abs() - half * (1 + half) * (g_soft.abs() + g_hard.abs() + (g_soft + g_hard).abs()) \
        - 1024 * U * terms
    assert float(near.max()) <= 0


def test_a_list_without_targets_has_no_teacher_loss():
  t, s = torch.randn(2, 3, 40), torch.randn(2, 3, 40)
  _, m = strategy(distill_top_k=4).compute_loss(s, functional.top_logprobs(t, 4), torch.zeros(2, 3, dtype=torch.long))
  assert "distill/teacher_loss" not in m and math.isfinite(float(m["distill/soft_loss"]))
  # without a top-k of its own the strategy takes the whole list
  whole, _ = strategy(alpha=1.0).compute_loss(s, functional.top_logprobs(t, 4), torch.zeros(2, 3, dtype=torch.long))
  cut, _ = strategy(alpha=1.0, distill_top_k=4).compute_loss(s, t, torch.zeros(2, 3, dtype=torch.long))
  assert float(whole) == pytest.approx(float(cut), rel=1e-5)


V_MODEL = 512


def tiny(layers, width, seed, device, dtype):
  cfg = ModelConfig(num_layers=layers, vocab_size=V_MODEL, embed_dim=width, hidden_dim=2 * width, num_heads=2,
                    head_dim=64, num_kv_heads=1, dtype=dtype, weight_tying=True, embed_scale=True)
  return Transformer(cfg, device=device).init_weights(seed=seed, scale=0.05)


def forward_logits(m, input_tokens, input_mask):
  pos = sft_utils.build_positions_from_mask(input_mask)
  return m(input_tokens, pos, None, sft_utils.make_causal_attn_mask(input_mask))[0]


def teacher_list(m, input_tokens, input_mask):
  return functional.top_logprobs(forward_logits(m, input_tokens, input_mask), 16, torch.roll(input_tokens, -1, 1))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("stored", [False, True])
def test_trainer(device, stored):
  dtype = bf16 if device == "cuda" else torch.float32
  strat = strategies.LogitStrategy(forward_logits, teacher_list if stored else forward_logits,
                                   lambda input_tokens, input_mask: torch.roll(input_tokens, -1, 1), temperature=2.0,
                                   alpha=0.7, distill_top_k=16)
  tr = DistillationTrainer(tiny(1, 128, 0, device, dtype), tiny(2, 256, 1, device, dtype), strat, optim.adamw(1e-3),
                           TrainingConfig(eval_every_n_steps=100, max_steps=3, pbar_description=None))
  g = torch.Generator().manual_seed(0)
  before = tr.model.embedder.input_embedding.detach().clone()
  tr.train([TrainingInput(torch.randint(1, V_MODEL, (2, 24), generator=g), torch.ones(2, 24, dtype=torch.long)) for _ in range(3)])
  for name in ("distill/soft_loss", "distill/hard_loss", "distill/kl_div", "distill/teacher_loss"):
    h = tr.metrics_logger.get_metric_history("", name, "train")
    assert len(h) == 3 and all(math.isfinite(v) for v in h)
  assert not torch.equal(before, tr.model.embedder.input_embedding.detach())
  tr.close()


def step(table, ids, t_logits, labels, k, tau):
  """Token embedding -> tied head -> distillation from the teacher's list -> gradient of the table (both uses)."""
  h = functional.embedding(ids, table, 1.5)
  logits = h @ table.t()
  with torch.no_grad():
    top = functional.top_logprobs(t_logits, k, labels, temperature=tau)
  terms = functional.top_distill_loss(logits, top.ids, top.top, labels, temperature=tau, normalize="full")
  loss = (0.7 * terms.kl + 0.3 * terms.nll).mean()
  return loss, torch.autograd.grad(loss, table)[0], top


@pytest.mark.gpu
def test_chain_against_64_bits(kernel_lib):
  V, D, T, k, tau = 2003, 64, 300, 20, 1.3
  g = torch.Generator().manual_seed(0)
  table = (torch.randn(V, D, generator=g) * 0.3).to(bf16).cuda().requires_grad_()
  ids = torch.randint(0, 40, (T,), generator=g).cuda()
  labels = torch.randint(0, V, (T,), generator=g).cuda()
  t_logits = (torch.randn(T, V, generator=g) * 2).cuda()
  loss, grad, top = step(table, ids, t_logits, labels, k, tau)

  tb = table.detach().to(f64).requires_grad_()
  h = tb[ids] * 1.5
  h = h + (h.detach().to(bf16).to(f64) - h.detach())                # rounded where the operators round
  logits = h @ tb.t()
  logits = logits + (logits.detach().to(bf16).to(f64) - logits.detach())
  t = F.log_softmax(t_logits.to(f64) / tau, -1)
  tt, at = torch.topk(t, k, -1)
  lp = F.log_softmax(logits / tau, -1).gather(-1, at)
  kl = (tt.exp() * (tt - lp)).sum(-1)
  nll = -F.log_softmax(logits, -1).gather(-1, labels[:, None])[:, 0]
  want = (0.7 * kl + 0.3 * nll).mean()
  want_grad, = torch.autograd.grad(want, tb)
  assert torch.equal(top.ids, at)
  # a logit that lies within its product's fp32 error of a border rounds to the other side: half a step of 2^-8
  assert abs(float(loss.detach()) - float(want.detach())) <= 2.0 ** -8 * float(logits.detach().abs().max())
  # the gradients of the logits, of the hidden state and of each use of the table are rounded to bf16 (2^-8 each), a
  # logit on a border moves its probability by at most half a step of its size
  rel = float((grad.to(f64) - want_grad).norm() / want_grad.norm())
  assert rel <= 4 * 2.0 ** -8 + 2.0 ** -8 * float(logits.detach().abs().max())


@pytest.mark.gpu
def test_captured_step_and_two_streams(kernel_lib):
  V, D, T, k, tau = 5000, 64, 400, 20, 1.3
  g = torch.Generator().manual_seed(0)
  table = torch.nn.Parameter((torch.randn(V, D, generator=g) * 0.3).to(bf16).cuda())
  inputs = [(torch.randint(0, 40, (T,), generator=g).cuda(), (torch.randn(T, V, generator=g) * 2).cuda(),
             torch.randint(0, V, (T,), generator=g).cuda()) for _ in range(2)]

  def run(i):
    loss, grad, top = step(table, i[0], i[1], i[2], k, tau)
    return loss.detach(), grad, top.ids, top.top, top.target

  static = [x.clone() for x in inputs[0]]
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    for _ in range(2):
      run(static)
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = run(static)
  want = [[x.clone() for x in run(i)] for i in inputs]
  torch.cuda.synchronize()
  for which in (0, 1, 0):
    for dst, src in zip(static, inputs[which]):
      dst.copy_(src)
    graph.replay()
    for a, b in zip(captured, want[which]):
      assert torch.equal(a, b)
  torch.cuda.synchronize()
  streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
  for n, s in enumerate(streams):
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
      got.append([run(inputs[n]) for _ in range(4)])
  graph.replay()
  torch.cuda.synchronize()
  for n in range(2):
    for r in got[n]:
      assert all(torch.equal(a, b) for a, b in zip(r, want[n]))


# ------------------------------------------------------------------------------ what the strategy took before it had a list
def rows64(s, t, ids, k, tau, alpha):
  """The strategy's loss in 64 bits, differentiable in both logits."""
  s, t = s.to(f64), t.to(f64)
  tk, idx = torch.topk(t, k, dim=-1)
  lq, lp = F.log_softmax(tk / tau, -1), F.log_softmax(s.gather(-1, idx) / tau, -1)
  soft = (lq.exp() * (lq - lp)).sum(-1).mean() * tau * tau
  return alpha * soft + (1 - alpha) * -F.log_softmax(s, -1).gather(-1, ids[..., None]).mean()


def some_logits(T, V, device, seed=0):
  """Student, teacher with distinct values in every row, labels."""
  g = torch.Generator().manual_seed(seed)
  t = torch.stack([torch.randperm(V, generator=g) for _ in range(T)]).float() * 0.0625
  return (torch.randn(T, V, generator=g) * 2).to(device), t.to(device), torch.randint(0, V, (T,), generator=g).to(device)


@pytest.mark.parametrize("device", DEVICES)
def test_a_teacher_with_a_graph_gets_its_gradient(device):
  T, V, k, tau, alpha = 5, 300, 8, 2.0, 0.6
  s, t, ids = some_logits(T, V, device)
  t = t.requires_grad_()
  loss, _ = strategy(temperature=tau, alpha=alpha, distill_top_k=k).compute_loss(s, t, ids)
  grad, = torch.autograd.grad(loss, t)
  want, = torch.autograd.grad(rows64(s, t, ids, k, tau, alpha), t)
  tk, idx = torch.topk(t.detach().to(f64), k, dim=-1)
  lq, lp = F.log_softmax(tk / tau, -1), F.log_softmax(s.to(f64).gather(-1, idx) / tau, -1)
  # d/dt = alpha tau / T q (lq - lp - kl): logits of at most 64 in size make log-probabilities that are off by 8 roundings
  # of that, 512 U, so the bracket is off by 2048 U and every factor by 1024 U of its size
  size = alpha * tau / T * lq.exp() * (1 + (lq - lp).abs() + (lq.exp() * (lq - lp)).sum(-1, keepdim=True))
  tol = torch.zeros(T, V, dtype=f64, device=device).scatter_(-1, idx, 4096 * U * size)
  assert float(((grad.to(f64) - want).abs() - tol).max()) <= 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("way", ["dual", "jvp", "grad", "vmap"])
def test_forward_mode_and_function_transforms_of_the_strategy(device, way):
  from torch.autograd import forward_ad
  T, V, k, tau, alpha = 5, 300, 8, 2.0, 0.6
  s, t, ids = some_logits(T, V, device)
  strat = strategy(temperature=tau, alpha=alpha, distill_top_k=k)
  v = torch.randn(T, V, generator=torch.Generator().manual_seed(9)).to(device)
  fn = lambda z: strat.compute_loss(z, t, ids)[0]   # noqa: E731
  leaf = s.to(f64).requires_grad_()
  want, = torch.autograd.grad(rows64(leaf, t, ids, k, tau, alpha), leaf)
  terms = loss64(s[None], t[None], ids[None], k, tau, alpha)[3][0]
  if way == "grad":
    assert float(((torch.func.grad(fn)(s).to(f64) - want).abs() - 1024 * U * terms).max()) <= 0
  elif way == "vmap":
    two = torch.func.vmap(fn)(torch.stack([s, s + v]))
    alone = torch.stack([rows64(s, t, ids, k, tau, alpha), rows64(s + v, t, ids, k, tau, alpha)])
    # as in test_strategy_over_logits_and_over_a_list
    assert float((two.to(f64) - alone).abs().max()) <= 64 * 16 * U * (tau * tau + 1)
  else:
    if way == "dual":
      with forward_ad.dual_level():
        tangent = forward_ad.unpack_dual(fn(forward_ad.make_dual(s, v))).tangent
    else:
      tangent = torch.func.jvp(fn, (s,), (v,))[1]
    assert tangent is not None
    # every product of a gradient (1024 U of its terms) and the tangent, in a sum of T V terms in any order
    assert abs(float(tangent) - float((want * v).sum())) <= (1024 + T * V) * U * float((terms * v.abs()).sum())


@pytest.mark.gpu
def test_strategy_on_another_device_than_the_process(monkeypatch):
  from tunix_b200.ops import _lib
  s, t, ids = some_logits(5, 300, "cuda")
  strat = strategy(temperature=2.0, alpha=0.6, distill_top_k=8)
  want = rows64(s, t, ids, 8, 2.0, 0.6)
  monkeypatch.setattr(_lib, "bind_thread", lambda: 1)
  loss, _ = strat.compute_loss(s, t, ids)
  assert abs(float(loss) - float(want)) <= 64 * 16 * U * 5


@pytest.mark.parametrize("device", DEVICES)
def test_strategy_temperatures_and_rows_beyond_the_operators(device):
  """A temperature that the operators refuse, and a teacher of fewer rows than the student (compared over its own)."""
  s, t, ids = some_logits(6, 300, device)
  loss, _ = strategy(temperature=1e19, alpha=0.0, distill_top_k=8).compute_loss(s, t, ids)
  assert abs(float(loss) - float(rows64(s, t, ids, 8, 1.0, 0.0))) <= 64 * 16 * U * 2
  s3, t3 = s.view(2, 3, 300), t.view(2, 3, 300)[:, :2]
  strat = strategy(temperature=2.0, alpha=1.0, distill_top_k=8)
  fewer, _ = strat.compute_loss(s3, t3, torch.zeros(2, 1, 300, device=device))
  want = rows64(s3[:, :2].reshape(4, 300), t3.reshape(4, 300), ids[:4], 8, 2.0, 1.0)
  assert abs(float(fewer) - float(want)) <= 64 * 16 * U * 5


@pytest.mark.parametrize("device", DEVICES)
def test_second_derivatives_through_the_strategy(device):
  T, V, k, tau, alpha = 3, 40, 6, 2.0, 0.6
  s, t, ids = some_logits(T, V, device)
  v = torch.randn(T, V, generator=torch.Generator().manual_seed(9)).to(device)
  strat = strategy(temperature=tau, alpha=alpha, distill_top_k=k)
  for stored in (False, True):
    leaf, leaf64 = s.clone().requires_grad_(), s.to(f64).requires_grad_()
    teacher = functional.top_logprobs(t, k, ids) if stored else t
    g, = torch.autograd.grad(strat.compute_loss(leaf, teacher, ids)[0], leaf, create_graph=True)
    hv, = torch.autograd.grad((g * v).sum(), leaf)
    g64, = torch.autograd.grad(rows64(leaf64, t, ids, k, tau, alpha), leaf64, create_graph=True)
    hv64, = torch.autograd.grad((g64 * v).sum(), leaf64)
    # rows of H v: w p (v - p.v) for each of the two softmaxes, w <= 1 / T; a probability is off by 1024 U of its size,
    # its product with v - p.v by 4096 U of p (|v| + 1) max |v|
    lp, at = F.log_softmax(s.to(f64), -1).exp(), torch.topk(t, k, -1).indices
    ps = F.log_softmax(s.to(f64).gather(-1, at) / tau, -1).exp()
    size = (1 - alpha) / T * lp + torch.zeros_like(lp).scatter_(-1, at, alpha / T * ps)
    assert float(((hv.to(f64) - hv64).abs() - 4096 * U * size * (v.abs() + 1) * float(v.abs().max())).max()) <= 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("top_k", [0, 8])
@pytest.mark.parametrize("stored", [False, True])
@pytest.mark.parametrize("label", [-100, 300])
def test_labels_outside_the_vocabulary_are_an_error(device, top_k, stored, label):
  """On the host they raise, with and without a list; on the GPU the loss and its gradient are NaN with a list (without
  one the lookup's own assertion is the error, which no test may set off)."""
  if device == "cuda" and not stored and top_k == 0:
    pytest.skip("an assertion on the device")
  s, t, ids = some_logits(4, 300, device)
  s = s.requires_grad_()
  teacher = functional.top_logprobs(t, 8, ids) if stored else t
  strat = strategy(temperature=2.0, alpha=0.6, distill_top_k=top_k)
  good, _ = strat.compute_loss(s, teacher, ids)
  assert math.isfinite(float(good.detach()))
  ids = ids.clone()
  ids[2] = label
  if device == "cpu":
    with pytest.raises(RuntimeError, match="out of bounds|outside"):
      strat.compute_loss(s, teacher, ids)
    return
  loss, m = strat.compute_loss(s, teacher, ids)
  assert math.isnan(float(loss.detach())) and math.isnan(float(m["distill/hard_loss"]))
  assert bool(torch.autograd.grad(loss, s)[0].isnan().any())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("k", [8, 280])
@pytest.mark.parametrize("stored", [False, True])
def test_a_teacher_of_more_tokens_than_the_student(device, k, stored):
  """Fine as long as its list stays within the student's tokens; else an error, on the GPU a loss of NaN with a list."""
  s, t, ids = some_logits(4, 300, device)
  wide = torch.cat([t, torch.full((4, 60), -50.0, device=device)], 1)
  if stored and k > 256 and device == "cuda":
    pytest.skip("lists of the GPU end at 256")
  of = lambda z: functional.top_logprobs(z, k, ids) if stored else z   # noqa: E731
  strat = strategy(temperature=2.0, alpha=0.6, distill_top_k=k)
  loss, _ = strat.compute_loss(s, of(wide), ids)
  want = rows64(s, wide, ids, k, 2.0, 0.6)
  assert abs(float(loss) - float(want)) <= 64 * 16 * U * 5
  if k > 256 and device == "cuda":
    return                                                          # without a list: the lookup's assertion on the device
  wide[1, 310] = 60.0
  if device == "cpu":
    with pytest.raises(RuntimeError, match="out of bounds|outside"):
      strat.compute_loss(s, of(wide), ids)
  else:
    loss, m = strat.compute_loss(s, of(wide), ids)
    assert math.isnan(float(loss)) and math.isnan(float(m["distill/kl_div"]))


@pytest.mark.parametrize("device", DEVICES)
def test_a_list_of_another_temperature_is_refused(device):
  import copy
  import pickle
  from tunix_b200.sft.sharding_utils import shard_input
  s, t, ids = some_logits(4, 300, device)
  strat = strategy(temperature=2.0, alpha=0.6, distill_top_k=10)
  warm = functional.top_logprobs(t, 12, ids, temperature=2.0)
  for teacher in (warm, pickle.loads(pickle.dumps(warm)), copy.deepcopy(warm), warm._replace(entropy=None),
                  shard_input(warm, device=torch.device(device))):
    assert teacher.temperature == 2.0 and len(teacher) == 4
    with pytest.raises(ValueError, match="temperature"):
      strat.compute_loss(s, teacher, ids)
  kept = pickle.loads(pickle.dumps(functional.top_logprobs(t, 12, ids)))
  by_hand = functional.TopLogprobs(kept.ids, kept.top, None, None)
  for teacher in (kept, by_hand):
    loss, _ = strat.compute_loss(s, teacher, ids)
    assert abs(float(loss) - float(rows64(s, t, ids, 10, 2.0, 0.6))) <= 64 * 16 * U * 5


@pytest.mark.parametrize("device", DEVICES)
def test_a_list_shorter_than_the_top_k_is_refused(device):
  s, t, ids = some_logits(4, 300, device)
  for labels in (ids, F.one_hot(ids, 300).float()):
    with pytest.raises(ValueError, match="4 entries.* top-k of 10"):
      strategy(distill_top_k=10).compute_loss(s, functional.top_logprobs(t, 4, ids), labels)
    strategy(distill_top_k=4).compute_loss(s, functional.top_logprobs(t, 4, ids), labels)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("one_hot", [False, True])
def test_a_bf16_gradient_is_rounded_once(device, one_hot):
  T, V, k, tau, alpha = 6, 700, 12, 2.0, 0.6
  s, t, ids = some_logits(T, V, device)
  s = s.to(bf16)
  labels = F.one_hot(ids, V).float() if one_hot else ids
  _, g_soft, g_hard, terms = (z[0] if z.ndim else z for z in loss64(s[None], t[None], ids[None], k, tau, alpha))
  # 1024 U of a term before the one rounding, half a step of 2^-7 of the value
  off = 1024 * U * terms
  for teacher in (t, functional.top_logprobs(t, k, ids)):
    leaf = s.clone().requires_grad_()
    loss, _ = strategy(temperature=tau, alpha=alpha, distill_top_k=k).compute_loss(leaf, teacher, labels)
    grad, = torch.autograd.grad(loss, leaf)
    near = (grad.to(f64) - (g_soft + g_hard)).abs() - off - 2.0 ** -8 * ((g_soft + g_hard).abs() + off)
    assert float(near.max()) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("stored", [False, True])
def test_captured_strategy_step(stored):
  """A loss with its gradient replays on new inputs, labels outside the vocabulary among them."""
  T, V, k = 40, 500, 8
  strat = strategy(temperature=2.0, alpha=0.6, distill_top_k=k)
  inputs = [list(some_logits(T, V, "cuda", seed)) for seed in (0, 1)]
  bad = [x.clone() for x in inputs[1]]
  bad[2][3] = V

  def run(s, t, ids):
    leaf = s.detach().requires_grad_()
    loss, _ = strat.compute_loss(leaf, functional.top_logprobs(t, k, ids) if stored else t, ids)
    return loss.detach(), torch.autograd.grad(loss, leaf)[0]

  static = [x.clone() for x in inputs[0]]
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    for _ in range(2):
      run(*static)
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = run(*static)
  for case in (inputs[1], bad, inputs[0]):
    for dst, src in zip(static, case):
      dst.copy_(src)
    graph.replay()
    want = run(*case)
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(captured, want))
    assert bool(captured[0].isnan()) == (case is bad)
