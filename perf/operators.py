"""Measured cases of the vocabulary operators.

Three operators of a distillation or scoring step, each over the whole vocabulary of a model:

* `functional.top_logprobs`: log-probabilities of given tokens, entropy and the k best alternatives of every row
  of logits (a teacher or a rollout that is scored), and the gradient through them;
* `functional.top_distill_loss`: distillation from a teacher's k best alternatives plus cross entropy on labels,
  with the gradient of the student's logits;
* `functional.embedding`: the scaled lookup and the table's gradient, summed by sorted tokens.

`run` computes them in plain torch operations, or with `own` through the framework's entry points.
"""
import math

import torch

own = False

F32, BF16 = torch.float32, torch.bfloat16
_DTYPES = {"bf16": BF16, "fp32": F32}


# ---------------------------------------------------------------------------------------------------- the cases
def _score(name, rows, vocab, k, dtype, temperature=1.0, targets=True, entropy=False, grad=False, masked=0, pad=0):
  return {"name": name, "op": "score", "rows": rows, "vocab": vocab, "k": k, "dtype": dtype,
          "temperature": temperature, "targets": targets, "entropy": entropy, "grad": grad, "masked": masked,
          "pad": pad}


def _distill(name, rows, vocab, k, dtype, temperature, normalize, labels=True, masked=0, pad=0):
  return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "k": k, "dtype": dtype,
          "temperature": temperature, "normalize": normalize, "labels": labels, "masked": masked, "pad": pad}


def _embed(name, tokens, vocab, dim, main_grad, scaled, hot):
  return {"name": name, "op": "embed", "tokens": tokens, "vocab": vocab, "dim": dim, "main_grad": main_grad,
          "scaled": scaled, "hot": hot}


def listed():
  return [
      # one sequence's next token with a handful of alternatives: nothing but latency
      _score("score_one_token", 1, 262144, 5, "fp32"),
      # a decode step of eight sequences that reports alternatives and entropy
      _score("score_decode_8", 8, 151936, 20, "bf16", entropy=True),
      # a teacher's pass over two micro-batches of 4096 tokens: what a student will be trained on
      _score("score_teacher_8k", 8192, 128256, 64, "bf16"),
      # the model's fp32 logits at a sampling temperature, rows of a ragged batch, padded vocabulary masked out
      _score("score_fp32_entropy", 2047, 151936, 8, "fp32", temperature=0.7, entropy=True, masked=271),
      # a policy that is trained through its tokens, its alternatives and its entropy
      _score("score_train", 1000, 262144, 16, "bf16", entropy=True, grad=True),
      # a toy student with an odd vocabulary: launch costs
      _distill("distill_small", 64, 32003, 8, "fp32", 2.0, "top"),
      # a training micro-batch, teacher restricted to its best 64, with labels
      _distill("distill_top_bf16", 4096, 128256, 64, "bf16", 2.0, "top"),
      # the same without labels on fp32 logits: the gradient is zero but for 32 columns a row
      _distill("distill_soft_only_fp32", 2048, 151936, 32, "fp32", 1.0, "top", labels=False),
      # both normalised over the whole vocabulary, two temperatures in one pass
      _distill("distill_full_bf16", 4096, 151936, 100, "bf16", 1.5, "full"),
      # a toy model's step
      _embed("embed_small", 512, 2048, 512, False, False, 0.0),
      # a batch of four sequences of 4096 tokens into the fp32 gradient buffer
      _embed("embed_main_grad", 16384, 128256, 4096, True, False, 0.05),
      # a padded batch over a large vocabulary: half of the tokens are the padding id
      _embed("embed_padded", 65536, 262144, 1152, False, True, 0.5),
  ]


_MOST_LOGITS = 4096 * 151936          # elements of a drawn block of logits (bf16; half as many in fp32)


def _log_uniform(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  op = rng.choice(["score", "score", "distill", "distill", "embed"])
  if op == "embed":
    dim = 8 * _log_uniform(rng, 8, 640)
    vocab = min(_log_uniform(rng, 1000, 262144), 500_000_000 // dim)
    tokens = min(_log_uniform(rng, 1, 65536), 80_000_000 // dim)
    return _without_name(_embed("", tokens, vocab, dim, rng.random() < 0.5, rng.random() < 0.5,
                                rng.choice([0.0, 0.05, 0.5, 1.0])))
  dtype = rng.choice(["bf16", "fp32"])
  vocab = _log_uniform(rng, 1000, 262144)
  most = _MOST_LOGITS // (2 if dtype == "fp32" else 1) // vocab
  rows = _log_uniform(rng, 1, min(8192, most))
  k = _log_uniform(rng, 1, 128)
  masked = rng.choice([0, 0, rng.randrange(1, vocab // 4)])
  pad = rng.choice([0, 0, rng.randrange(1, 64)])
  temperature = rng.choice([1.0, round(rng.uniform(0.5, 3.0), 3)])
  if op == "score":
    return _without_name(_score("", rows, vocab, k, dtype, temperature, rng.random() < 0.8, rng.random() < 0.5,
                                rng.random() < 0.4, masked, pad))
  return _without_name(_distill("", rows, vocab, k, dtype, temperature, rng.choice(["top", "full"]),
                                rng.random() < 0.7, masked, pad))


def _without_name(case):
  del case["name"]
  return case


# ---------------------------------------------------------------------------------------------------- inputs
def _logits(case, gen):
  """Logits as a trained model gives them: a broad bulk and a few likely tokens in every row."""
  T, V = case["rows"], case["vocab"]
  x = torch.randn(T, V + case["pad"], generator=gen, device="cuda", dtype=F32).mul_(2.0)
  span = (V - case["masked"]) // 12                        # one likely token in each twelfth: no column twice
  at = torch.randint(0, span, (T, 12), generator=gen, device="cuda") + span * torch.arange(12, device="cuda")
  up = torch.rand(T, 12, generator=gen, device="cuda").mul_(10.0).add_(4.0)
  x.scatter_(1, at, up)
  if case["masked"]:
    x[:, V - case["masked"]:V] = float("-inf")
  return x


def _ids(case, gen):
  """Token ids with the frequencies of text: p(id) falls like 1 / rank; a share `hot` is one padding id."""
  V, T = case["vocab"], case["tokens"]
  u = torch.rand(T, generator=gen, device="cuda", dtype=torch.float64)
  ids = torch.exp(u * math.log(V)).long().sub_(1).clamp_(0, V - 1)
  ids = (ids * 7919) % V                                   # frequent ids are spread over the table
  pad = torch.rand(T, generator=gen, device="cuda") < case["hot"]
  return torch.where(pad, torch.zeros_like(ids), ids)


def prepare(case, seed):
  gen = torch.Generator(device="cuda")
  gen.manual_seed(seed)
  if case["op"] == "embed":
    V, D, T = case["vocab"], case["dim"], case["tokens"]
    table = torch.randn(V, D, generator=gen, device="cuda", dtype=F32).mul_(0.02).to(BF16)
    table = torch.nn.Parameter(table)
    ids = _ids(case, gen)
    dout = torch.randn(T, D, generator=gen, device="cuda", dtype=F32).mul_(1e-3).to(BF16)
    if case["main_grad"]:
      table.main_grad = torch.zeros(V, D, device="cuda", dtype=F32)
    return {"case": case, "table": table, "ids": ids, "dout": dout,
            "scale": math.sqrt(D) if case["scaled"] else 1.0}
  T, V, k = case["rows"], case["vocab"], case["k"]
  dtype = _DTYPES[case["dtype"]]
  wide = _logits(case, gen)
  state = {"case": case}
  live = torch.rand(T, generator=gen, device="cuda") >= 0.05        # the others are padding: no gradient
  if case["op"] == "score":
    state["targets"] = torch.randint(0, V - case["masked"], (T,), generator=gen, device="cuda") if case["targets"] else None
    if case["targets"]:                                             # most given tokens are likely ones
      best = wide[:, :V].argmax(1)
      state["targets"] = torch.where(torch.rand(T, generator=gen, device="cuda") < 0.7, best, state["targets"])
    if case["grad"]:
      w = live.float() / T
      state["g_top"] = torch.randn(T, k, generator=gen, device="cuda").mul_(w[:, None])
      state["g_target"] = torch.randn(T, generator=gen, device="cuda").mul_(w) if case["targets"] else None
      state["g_entropy"] = w * 0.01 if case["entropy"] else None
  else:
    tau = case["temperature"]
    teacher = wide[:, :V] + torch.randn(T, V, generator=gen, device="cuda", dtype=F32).mul_(0.5)
    top, ids = torch.topk(teacher, k, dim=1)
    state["ids"] = ids
    state["top"] = top / tau - torch.logsumexp(teacher / tau, 1, keepdim=True)
    random = torch.randint(0, V - case["masked"], (T,), generator=gen, device="cuda")
    labels = torch.where(torch.rand(T, generator=gen, device="cuda") < 0.8, ids[:, 0], random)
    state["labels"] = labels if case["labels"] else None
    state["g_kl"] = live.float() * (0.7 * tau * tau / T)
    state["g_nll"] = live.float() * (0.3 / T) if case["labels"] else None
    del teacher
  logits = wide.to(dtype)[:, :V]                # a row stride above V where the block is padded
  state["logits"] = logits.detach().requires_grad_(case["op"] == "distill" or case["grad"])
  return state


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
  case = state["case"]
  if own:
    return _run_own(state, case)
  with torch.no_grad():
    if case["op"] == "score":
      return _plain_score(state, case)
    if case["op"] == "distill":
      return _plain_distill(state, case)
    return _plain_embed(state, case)


def _run_own(state, case):
  from tunix_b200.ops import functional as F
  if case["op"] == "embed":
    table = state["table"]
    if case["main_grad"]:
      table.main_grad.zero_()
    out = F.embedding(state["ids"], table, state["scale"])
    grad, = torch.autograd.grad(out, table, state["dout"], allow_unused=True)
    return {"out": out, "grad": table.main_grad if case["main_grad"] else grad}
  logits = state["logits"]
  if case["op"] == "score":
    got = F.top_logprobs(logits, case["k"], state["targets"], temperature=case["temperature"],
                         want_entropy=case["entropy"])
    out = {"ids": got.ids, "top": got.top, "target": got.target, "entropy": got.entropy}
    if case["grad"]:
      pairs = [(got.top, state["g_top"]), (got.target, state["g_target"]), (got.entropy, state["g_entropy"])]
      pairs = [p for p in pairs if p[1] is not None]
      out["grad"], = torch.autograd.grad([p[0] for p in pairs], logits, [p[1] for p in pairs])
    return out
  got = F.top_distill_loss(logits, state["ids"], state["top"], state["labels"], temperature=case["temperature"],
                           normalize=case["normalize"])
  pairs = [(got.kl, state["g_kl"])] + ([(got.nll, state["g_nll"])] if case["labels"] else [])
  grad, = torch.autograd.grad([p[0] for p in pairs], logits, [p[1] for p in pairs])
  return {"kl": got.kl, "nll": got.nll, "grad": grad}


def _order_keys(x):
  """int64 keys that rank the values of a row from high to low, equal ones by the lowest index."""
  V = x.shape[1]
  bits = (x + 0.0).view(torch.int32)
  bits = bits ^ ((bits >> 31) & 0x7FFFFFFF)
  return (bits.long() << 32) + (V - 1 - torch.arange(V, device=x.device))


def _plain_score(state, case):
  x = state["logits"].float()
  T, V = x.shape
  k, inv = case["k"], 1.0 / case["temperature"]
  ids = V - 1 - (torch.topk(_order_keys(x), k, dim=1).values & 0xFFFFFFFF)
  m = x.amax(1, keepdim=True)
  d = (x - m) * inv
  e = d.exp()
  s = e.sum(1, keepdim=True)
  ls = s.log()
  out = {"ids": ids, "top": d.gather(1, ids) - ls, "target": None, "entropy": None}
  if case["targets"]:
    out["target"] = (d.gather(1, state["targets"][:, None]) - ls)[:, 0]
  if case["entropy"] or case["grad"]:
    p = e / s
    lp = d - ls
    h = -torch.where(p > 0, p * lp, 0.0).sum(1)
    if case["entropy"]:
      out["entropy"] = h
  if case["grad"]:
    g = p * -state["g_top"].sum(1, keepdim=True)
    g.scatter_add_(1, ids, state["g_top"])
    if case["targets"]:
      g -= p * state["g_target"][:, None]
      g.scatter_add_(1, state["targets"][:, None], state["g_target"][:, None])
    if case["entropy"]:
      g -= state["g_entropy"][:, None] * torch.where(p > 0, p * (lp + h[:, None]), 0.0)
    out["grad"] = (g * inv).to(state["logits"].dtype)
  return out


def _plain_distill(state, case):
  x = state["logits"].float()
  inv = 1.0 / case["temperature"]
  ids, t = state["ids"], state["top"]
  m = x.amax(1, keepdim=True)
  z = x - m
  picked = z.gather(1, ids) * inv
  if case["normalize"] == "top":
    t = t * inv
    t = t - t.amax(1, keepdim=True)
    q = t.exp()
    sq = q.sum(1, keepdim=True)
    q, lq = q / sq, t - sq.log()
    pm = picked.amax(1, keepdim=True)
    sp = (picked - pm).exp().sum(1, keepdim=True)
    lp = picked - pm - sp.log()
    kl = torch.where(q > 0, q * (lq - lp), 0.0).sum(1)
    g = torch.zeros_like(x).scatter_add_(1, ids, state["g_kl"][:, None] * inv * (lp.exp() - q))
  else:
    q = t.exp()
    e = (z * inv).exp()
    s = e.sum(1, keepdim=True)
    lp = picked - s.log()
    kl = torch.where(q > 0, q * (t - lp), 0.0).sum(1)
    g = e * (state["g_kl"][:, None] * inv * q.sum(1, keepdim=True) / s)
    g.scatter_add_(1, ids, state["g_kl"][:, None] * -inv * q)
  nll = None
  if case["labels"]:
    e = z.exp()
    s = e.sum(1, keepdim=True)
    at = state["labels"][:, None]
    nll = (s.log() - z.gather(1, at))[:, 0]
    g += e * (state["g_nll"][:, None] / s)
    g.scatter_add_(1, at, -state["g_nll"][:, None])
  return {"kl": kl, "nll": nll, "grad": g.to(state["logits"].dtype)}


def _plain_embed(state, case):
  table, ids = state["table"], state["ids"]
  out = (table[ids].float() * state["scale"]).to(table.dtype)
  grad = torch.zeros(table.shape, dtype=F32, device=table.device)
  grad.index_add_(0, ids, state["dout"].float() * state["scale"])
  return {"out": out, "grad": grad if case["main_grad"] else grad.to(table.dtype)}


# ---------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
  state = prepare(case, seed)
  if case["op"] == "embed":
    table, ids = state["table"].detach(), state["ids"]
    grad = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
    grad.index_put_((ids,), state["dout"].double(), accumulate=True)
    return {"out": table[ids].double() * state["scale"], "grad": grad * state["scale"]}
  parts = [_exact_rows(state, case, lo, lo + 512) for lo in range(0, case["rows"], 512)]
  return {n: None if parts[0][n] is None else torch.cat([p[n] for p in parts]) for n in parts[0]}


def _exact_rows(state, case, lo, hi):
  """Rows lo to hi by autograd on the definition; masked columns have no probability and no gradient."""
  V, live = case["vocab"], case["vocab"] - case["masked"]
  of = lambda name: None if state.get(name) is None else state[name][lo:hi]   # noqa: E731
  x = state["logits"].detach()[lo:hi, :live].double().requires_grad_()
  lp = torch.log_softmax(x / case["temperature"], dim=1)
  lp_all = torch.cat([lp, lp.new_full((lp.shape[0], case["masked"]), float("-inf"))], 1)
  if case["op"] == "score":
    raw = state["logits"].detach()[lo:hi].float()
    ids = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :case["k"]]
    out = {"ids": None, "top": lp_all.gather(1, ids), "target": None, "entropy": None}
    loss = 0.0
    if case["targets"]:
      out["target"] = lp_all.gather(1, of("targets")[:, None])[:, 0]
    if case["entropy"]:
      out["entropy"] = -(lp.exp() * lp).sum(1)
    if not case["grad"]:
      return {n: None if v is None else v.detach() for n, v in out.items()}
    for n in ("top", "target", "entropy"):
      if of("g_" + n) is not None:
        loss = loss + (out[n] * of("g_" + n).double()).sum()
  else:
    ids, t = of("ids"), of("top").double()
    if case["normalize"] == "top":
      lq = torch.log_softmax(t / case["temperature"], dim=1)
      lps = torch.log_softmax(torch.nn.functional.pad(x, (0, case["masked"]), value=float("-inf")).gather(1, ids)
                              / case["temperature"], dim=1)
    else:
      lq, lps = t, lp_all.gather(1, ids)
    q = lq.exp()
    there = q > 0
    kl = torch.where(there, q * (torch.where(there, lq, 0.0) - torch.where(there, lps, 0.0)), 0.0).sum(1)
    out = {"kl": kl, "nll": None}
    loss = (kl * of("g_kl").double()).sum()
    if case["labels"]:
      out["nll"] = -torch.log_softmax(x, dim=1).gather(1, of("labels")[:, None])[:, 0]
      loss = loss + (out["nll"] * of("g_nll").double()).sum()
  grad, = torch.autograd.grad(loss, x)
  out["grad"] = torch.nn.functional.pad(grad, (0, case["masked"]))
  return {n: None if v is None else v.detach() for n, v in out.items()}


# ---------------------------------------------------------------------------------------------------- floors
def work(case):
  if case["op"] == "embed":
    T, V, D = case["tokens"], case["vocab"], case["dim"]
    # rows of the table, of the output and of its gradient; the table's whole gradient is written
    return {"bytes": 3 * T * D * 2 + T * 8 + V * D * (4 if case["main_grad"] else 2), "flops": 2 * T * D}
  T, V, k = case["rows"], case["vocab"], case["k"]
  size = 2 if case["dtype"] == "bf16" else 4
  block = T * V * size
  if case["op"] == "score":
    some = T * k * 12 + T * (12 if case["targets"] else 0) + T * (4 if case["entropy"] else 0)
    grad = (2 * block + T * k * 4 + T * 8) if case["grad"] else 0      # read again for the gradient, and written
    return {"bytes": block + some + grad, "flops": T * V * (6 + (6 if case["grad"] else 0))}
  lists = T * k * 12 + T * (8 + 8 if case["labels"] else 4)
  reads = 2 if case["labels"] or case["normalize"] == "full" else 0    # forward and backward
  softmaxes = (1 if case["labels"] else 0) + (1 if case["normalize"] == "full" else 0)
  return {"bytes": (reads + 1) * block + lists, "flops": T * V * (1 + 8 * softmaxes)}
