"""The embedding's gradient, summed by sorted tokens: against 64 bits for every kind of id list, bitwise repeatable,
into a new table or an fp32 gradient buffer; on the CPU and, marked gpu, the kernels."""
import pytest
import torch

from tunix_b200.ops import functional as F

bf16, f64 = torch.bfloat16, torch.float64
U = 2.0 ** -24
DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]


def id_list(kind, T, V, seed=0):
  g = torch.Generator().manual_seed(seed)
  if kind == "one":
    return torch.full((T,), V // 2)
  if kind == "distinct":
    return torch.randperm(max(T, V), generator=g)[:T] % V
  if kind == "rising":
    return torch.arange(T) * V // max(T, 1)
  if kind == "falling":
    return (T - 1 - torch.arange(T)) * V // max(T, 1)
  ids = (torch.rand(T, generator=g) ** 6 * V).long().clamp(0, V - 1)      # a few frequent ones, a long tail
  if kind == "padded":
    ids[torch.rand(T, generator=g) < 0.6] = 0
  if kind == "outside":
    ids[::3] = -1
    ids[1::5] = V
    ids[2::7] = 2 ** 30
  return ids


def sums64(ids, dout, V, scale):
  """(sum, sum of magnitudes, number of terms) per row of the table."""
  keep = (ids >= 0) & (ids < V)
  d = dout.to(f64)[keep] * scale
  at = ids.long()[keep]
  total = torch.zeros(V, dout.shape[1], dtype=f64, device=dout.device).index_add_(0, at, d)
  mag = torch.zeros_like(total).index_add_(0, at, d.abs())
  return total, mag, torch.bincount(at, minlength=V).to(f64)[:, None]


def check(ids, D, V, scale, grad_dtype, seed=0):
  from tunix_b200.ops import kernels
  g = torch.Generator(device="cuda").manual_seed(seed)
  ids = ids.cuda()
  dout = torch.randn(ids.numel(), D, generator=g, device="cuda").to(bf16)
  base = torch.randn(V, D, generator=g, device="cuda") if grad_dtype == torch.float32 else torch.zeros(V, D, device="cuda", dtype=bf16)
  fresh = lambda: base.clone() if grad_dtype == torch.float32 else torch.full_like(base, 7.0)   # noqa: E731
  grad, again = fresh(), fresh()                                         # a bf16 gradient is written whole
  kernels.embedding_bwd(ids, dout, grad, scale)
  kernels.embedding_bwd(ids, dout, again, scale)
  assert torch.equal(grad, again)
  total, mag, n = sums64(ids, dout, V, scale)
  present = n[:, 0] > 0
  assert torch.equal(grad[~present], base[~present])                     # rows of other tokens are left as they were
  # n additions and the scale in fp32; then one addition to the buffer, or one rounding to bf16
  tol = (n + 2) * U * mag
  want = total
  if grad_dtype == torch.float32:
    want = base.to(f64) + total
    tol = tol + U * (want.abs() + tol)
  else:
    tol = tol + 2.0 ** -8 * (want.abs() + tol)      # 8 significant bits: a step is 2^-7 of the value, half of it 2^-8
  off = ((grad.to(f64) - want).abs() - tol)[present]
  assert off.numel() == 0 or float(off.max()) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("grad_dtype", [torch.float32, bf16])
@pytest.mark.parametrize("kind", ["one", "distinct", "rising", "falling", "tail", "padded", "outside"])
@pytest.mark.parametrize("T,V,D", [(1, 1, 8), (2, 5, 24), (8, 3, 8), (12, 1, 16), (16, 2, 8), (31, 1000, 64), (33, 7, 1152), (1000, 300, 520),
                                   (4096, 128256, 64), (4097, 1024, 256), (9001, 262144, 40)])
def test_sorted_sums(kernel_lib, grad_dtype, kind, T, V, D):
  check(id_list(kind, T, V), D, V, 1.0 if T % 2 else 2.5, grad_dtype)


@pytest.mark.gpu
def test_long_lists_and_large_tables(kernel_lib):
  check(id_list("padded", 150_001, 50_000), 16, 50_000, 1.0, torch.float32)
  check(id_list("tail", 20_000, 1_048_577), 8, 1_048_577, 1.0, bf16)       # three passes of the sort
  check(id_list("padded", 5000, 100), 4104, 100, 1.0, torch.float32)       # several column tiles
  check(id_list("one", 0, 10), 8, 10, 1.0, torch.float32)
  check(id_list("one", 0, 10), 8, 10, 1.0, bf16)
  for T in (5, 40, 700, 4096, 9000, 20_000):                               # runs that end on and around chunk borders
    for length in (1, 3, 4, 5, 8, 9, 15, 16, 31, 32, 33, 63, 64, 65, 97):
      check(torch.arange(T) // length, 8, T, 1.0, torch.float32)
  check(id_list("tail", 5000, 100).to(torch.int32), 64, 100, 1.0, torch.float32)


@pytest.mark.gpu
def test_buffer_at_an_odd_offset(kernel_lib):
  """A gradient that is a view into a flat buffer may begin at any element."""
  from tunix_b200.ops import kernels
  ids = id_list("padded", 500, 40).cuda()
  dout = torch.randn(500, 32, device="cuda").to(bf16)
  flat = torch.zeros(40 * 32 + 9, device="cuda")
  want = torch.zeros(40, 32, device="cuda")
  kernels.embedding_bwd(ids, dout, want)
  for off in (1, 2, 7):
    flat.zero_()
    kernels.embedding_bwd(ids, dout, flat[off:off + 40 * 32].view(40, 32))
    assert torch.equal(flat[off:off + 40 * 32].view(40, 32), want)
    assert float(flat[:off].abs().sum()) == 0 and float(flat[off + 40 * 32:].abs().sum()) == 0
  small = torch.full((40 * 32 + 9,), 3.0, device="cuda", dtype=bf16)
  kernels.embedding_bwd(ids, dout, small[3:3 + 40 * 32].view(40, 32))
  assert torch.equal(small[3:3 + 40 * 32].view(40, 32), want.to(bf16))
  assert bool((small[:3] == 3).all()) and bool((small[3 + 40 * 32:] == 3).all())


@pytest.mark.gpu
def test_tables_that_the_kernels_do_not_take(kernel_lib):
  """Views of wider tables and tables at odd offsets get the plain statement, ids on the host an error."""
  ids = id_list("padded", 50, 30).cuda()
  wide = torch.randn(30, 48, device="cuda").to(bf16)
  flat = torch.randn(30 * 32 + 1, device="cuda").to(bf16)
  for table in (wide[:, :32], flat[1:].view(30, 32)):
    leaf = table.detach().requires_grad_()
    out = F.embedding(ids, leaf, 2.0)
    assert torch.equal(out, (table[ids].float() * 2.0).to(bf16))
    out.float().sum().backward()
    assert leaf.grad.shape == (30, 32)
  with pytest.raises(ValueError, match="ids are on cpu"):
    F.embedding(ids.cpu(), wide.contiguous())


@pytest.mark.gpu
def test_other_devices_and_buffers_are_refused(kernel_lib, monkeypatch):
  from tunix_b200.ops import _lib
  ids = id_list("padded", 50, 30).cuda()
  table = torch.randn(30, 32, device="cuda").to(bf16).requires_grad_()
  table.main_grad = torch.zeros(30, 32, device="cuda", dtype=bf16)
  with pytest.raises(ValueError, match="main_grad must be fp32"):
    F.embedding(ids, table).sum().backward()
  monkeypatch.setattr(_lib, "bind_thread", lambda: 1)
  with pytest.raises(ValueError, match="this process drives cuda:1"):
    F.embedding(ids, table)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("main_grad", [False, True])
def test_gradient_through_the_lookup(device, main_grad):
  if device == "cpu" and main_grad:
    pytest.skip("gradient buffers belong to the kernels")
  V, D, scale = 50, 32, 5.0
  table = torch.randn(V, D, generator=torch.Generator().manual_seed(0)).to(device=device, dtype=bf16).requires_grad_()
  ids = id_list("padded", 60, V).view(3, 20).to(device)
  dout = torch.randn(3, 20, D, generator=torch.Generator().manual_seed(1)).to(device=device, dtype=bf16)
  if main_grad:
    table.main_grad = torch.ones(V, D, device=device)
  out = F.embedding(ids, table, scale)
  assert torch.equal(out, (table.detach()[ids].float() * scale).to(bf16))
  grad, = torch.autograd.grad(out, table, dout, allow_unused=True)
  total, mag, n = sums64(ids.reshape(-1), dout.reshape(-1, D), V, scale)
  if main_grad:
    assert grad is None
    assert float(((table.main_grad.to(f64) - 1 - total).abs() - (n + 3) * U * (mag + 1)).max()) <= 0
  else:
    # on the CPU every product with the scale and every addition rounds to bf16
    steps = (n + 2) * 2.0 ** -8 if device == "cpu" else 2.0 ** -8 * torch.ones_like(n)
    assert grad.dtype == bf16
    assert float(((grad.to(f64) - total).abs() - steps * mag - 2.0 ** -100).max()) <= 0


@pytest.mark.gpu
def test_captured_backward_and_two_streams(kernel_lib):
  """A captured gradient replays on new inputs; two streams and a replay share no workspace."""
  V, D, T = 300, 64, 5000
  table = torch.nn.Parameter(torch.randn(V, D, device="cuda").to(bf16))
  ids, dout = id_list("padded", T, V).cuda(), torch.randn(T, D, device="cuda").to(bf16)

  def grad_of(i, d):
    return torch.autograd.grad(F.embedding(i, table, 2.0), table, d)[0]

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    for _ in range(2):
      grad_of(ids, dout)
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = grad_of(ids, dout)
  ids2, dout2 = id_list("tail", T, V, seed=5).cuda(), torch.randn(T, D, device="cuda").to(bf16)
  first, second = grad_of(ids, dout), grad_of(ids2, dout2)
  graph.replay()
  assert torch.equal(captured, first)
  ids.copy_(ids2)
  dout.copy_(dout2)
  torch.cuda.synchronize()
  results = []
  for s in (torch.cuda.Stream(), torch.cuda.Stream()):
    with torch.cuda.stream(s):
      results.append([grad_of(ids, dout) for _ in range(5)])
  graph.replay()
  torch.cuda.synchronize()
  assert torch.equal(captured, second)
  assert all(torch.equal(r, second) for rs in results for r in rs)


@pytest.mark.gpu
def test_tables_and_batches_beyond_32_bits(kernel_lib):
  from tunix_b200.ops import kernels
  V, D = 600_000, 4096                                                   # 2.5e9 elements of the table
  ids = torch.tensor([V - 1, 5, V - 1, V - 2], device="cuda")
  dout = torch.randn(4, D, device="cuda").to(bf16)
  grad = torch.empty(V, D, device="cuda", dtype=bf16)
  kernels.embedding_bwd(ids, dout, grad)
  assert torch.equal(grad[V - 1], (dout[0].float() + dout[2].float()).to(bf16))
  assert torch.equal(grad[V - 2], dout[3]) and torch.equal(grad[5], dout[1])
  assert int((grad != 0).any(1).sum()) == 3
  assert torch.equal(kernels.embedding_fwd(ids, grad), grad[ids])
  del grad
  T, V = 600_000, 7                                                      # 2.5e9 elements of the batch
  ids = torch.full((T,), 3, device="cuda")
  ids[-2:] = 6
  dout = torch.zeros(T, D, device="cuda", dtype=bf16)
  dout[::1000] = 1.0
  dout[-2:] = torch.randn(2, D, device="cuda").to(bf16)
  grad = torch.zeros(V, D, device="cuda")
  kernels.embedding_bwd(ids, dout, grad)
  assert torch.equal(grad[6], dout[-2].float() + dout[-1].float())
  assert float((grad[3] - T / 1000).abs().max()) == 0.0                  # 600 ones: exact in fp32


def test_more_tokens_than_the_gradient_counts_are_refused(kernel_lib):
  """The sort's indices run past the last token by up to a tile: the limit leaves room for that. Nothing is allocated."""
  from tunix_b200.ops import kernels
  for T in (0x7fff0001, 2 ** 31 - 1, 2 ** 31):
    ids = torch.zeros(1, dtype=torch.long).expand(T)
    dout = torch.zeros(1, 8, dtype=bf16).expand(T, 8)
    with pytest.raises(ValueError, match="31 bits"):
      kernels.embedding_bwd(ids, dout, torch.zeros(4, 8))
  for T in (0x7fff0001, 2 ** 31 - 1):
    assert kernel_lib.tx_embedding_grad(None, 1, None, None, 0, T, 8, 4, 1.0, None, None) == 1


@pytest.mark.gpu
def test_ids_outside_a_table_that_the_kernels_do_not_take(kernel_lib):
  """As with the kernels: the nearest row is read and gets no gradient."""
  wide = torch.randn(30, 48, device="cuda").to(bf16)
  flat = torch.randn(30 * 32 + 1, device="cuda").to(bf16)
  ids = torch.tensor([-1, 0, 29, 30, 2 ** 40, 5], device="cuda")
  dout = torch.randn(6, 32, device="cuda").to(bf16)
  for table in (wide[:, :32], flat[1:].view(30, 32)):
    taken = table.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
    leaf = table.detach().requires_grad_()
    a, b = F.embedding(ids, leaf, 2.0), F.embedding(ids, taken, 2.0)
    assert torch.equal(a, b)
    ga, gb = torch.autograd.grad(a, leaf, dout)[0], torch.autograd.grad(b, taken, dout)[0]
    assert torch.equal(ga, gb) and bool((ga[0] == gb[0]).all())
