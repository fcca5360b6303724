"""actions.sample / log_prob / log_prob_backward and Engine.step_sampled (csrc/pcx_policy.hip) against the definitions in
64 bits.

Sampling is compared for equality.  What may differ is a row whose number falls on a border between two sums: weights are
64-bit on both sides, each good to a few units, so a border of A summands is known to (A + 16) 2^-52 of the total; rows
nearer than that (none is expected) are left out, and rows over 16,384 actions, whose top_p border is summed in fixed point
of 2^-(62 - log2 A), also those within A of such units of it.

log_prob, entropy and gradients are float32 sums of A terms with exp good to 2^-22 of its value: d = (x - max) / T is off by
2^-23 |d| in three roundings, which exp turns into 3 * 2^-23 |d| e^d <= 2^-22.  A sum of probabilities is then off by
(A_eff + 8) 2^-22 relative, A_eff = the longest chain of additions (a lane's share of the row and the joining of lanes): A / 64 + 16 at
worst here.  log s moves by that much absolutely, log-probabilities and entropies besides by 2^-22 of the terms they are made of
(|x - max| / T, log s), a gradient by that much of each of its two terms."""

import ctypes
import math

import numpy as np
import pytest

from pycolab_amd import _native as N
from pycolab_amd import actions as policy

torch = pytest.importorskip('torch')

DTYPES = ['float32', 'float16', 'bfloat16']


def logits_of(n, a, dtype, seed, spread=2.0):
  g = torch.Generator().manual_seed(seed)
  return (torch.randn(n, a, generator=g) * spread).to(getattr(torch, dtype)), torch.rand(n, generator=g)


def draw_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, legal=None):
  """(action, is its border too near to call) of one row, by sorting."""
  x = np.asarray(x, np.float64)
  ok = ~np.isnan(x) & (x > -np.inf)
  if legal is not None:
    ok &= np.asarray(legal, bool)
  index = np.flatnonzero(ok)
  if index.size == 0:
    return -1, False
  order = index[np.lexsort((index, -x[index]))]
  if not temperature > 0:
    return int(order[0]), False
  best = x[order[0]]
  with np.errstate(invalid='ignore', over='ignore'):
    w = np.where(x[order] == best, 1.0, np.exp((x[order] - best) / np.float64(np.float32(temperature))))
  if top_k > 0:
    order, w = order[:top_k], w[:top_k]
  near = (x.size + 16) * 2.0 ** -52
  fixed = x.size * 2.0 ** -(62 - math.ceil(math.log2(max(2, x.size)))) if x.size > 16384 else 0.0
  close = False
  if top_p < 1:
    ahead = np.concatenate([[0.0], np.cumsum(w)[:-1]])
    target = np.float64(np.float32(top_p)) * w.sum()
    exact = np.all(w == 1.0) and float(target).is_integer()  # (counts of equal weights are exact on both sides)
    close = not exact and bool(np.any(np.abs(ahead[1:] - target) <= near * w.sum() + fixed))
    keep = ahead < target
    keep[0] = True
    order, w = order[keep], w[keep]
  floor = min(np.float64(np.float32(min_p)), 1.0) if min_p > 0 else 0.0
  keep = w >= floor
  close = close or bool(np.any((np.abs(w - floor) <= 8 * 2.0 ** -52 * floor) & (w != 1.0) & (floor > 0)))
  order, w = order[keep], w[keep]
  by_index = np.argsort(order)
  order, w = order[by_index], w[by_index]
  cdf = np.cumsum(w)
  target = np.float64(u) * cdf[-1]
  exact = np.all(w == 1.0) and float(target).is_integer()
  close = close or (not exact and bool(np.any(np.abs(cdf - target) <= near * cdf[-1])))
  hit = (cdf > target) & (w > 0)
  return int(order[np.argmax(hit)] if hit.any() else order[np.flatnonzero(w > 0)[-1]]), close


def check_sample(x, u, legal=None, **rules):
  n = x.shape[0]
  dev = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in rules.items()}
  got = policy.sample(x.cuda(), u.cuda(), legal=None if legal is None else legal.cuda(), **dev)
  assert got.dtype == torch.int32 and tuple(got.shape) == (n,)
  got, skipped = got.cpu().numpy(), 0
  xs = x.double().numpy()
  for i in range(n):
    row = {k: float(v[i]) if isinstance(v, torch.Tensor) else v for k, v in rules.items()}
    if 'top_k' in row:
      row['top_k'] = int(row['top_k'])
    want, close = draw_row(xs[i], float(u[i]), legal=None if legal is None else legal[i].numpy(), **row)
    skipped += close
    assert close or got[i] == want, (i, got[i], want, row)
  assert skipped <= max(1, n // 50)
  return got


def soft64(x, legal, temperature):
  """(log p, p, entropy, some) in 64 bits; log p is -inf where not allowed."""
  x = x.double()
  ok = ~torch.isnan(x) & (x > -math.inf)
  if legal is not None:
    ok &= legal.bool()
  some = ok.any(1)
  z = torch.where(ok, x / float(np.float32(temperature)), torch.full_like(x, -math.inf))
  z = torch.where(some[:, None], z, torch.zeros_like(z))
  lp = torch.log_softmax(z, 1)
  lp = torch.where(ok, lp, torch.full_like(lp, -math.inf))
  p = torch.where(ok, lp.exp(), torch.zeros_like(lp))
  h = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
  return lp, p, h, some, ok


def check_log_prob(x, taken, legal=None, temperature=1.0, seed=0):
  n, a = x.shape
  lp, p, h, some, ok = soft64(x, legal, temperature)
  g = torch.Generator().manual_seed(seed)
  g_lp, g_h = torch.randn(n, generator=g), torch.randn(n, generator=g)
  leaf = x.cuda().requires_grad_()
  l_dev = None if legal is None else legal.cuda()
  got_lp, got_h = policy.log_prob(leaf, taken.cuda(), legal=l_dev, temperature=temperature)
  there = (taken >= 0) & some
  at = taken.long().clamp(min=0)[:, None]
  want = torch.where(there, lp.gather(1, at)[:, 0], torch.zeros(n, dtype=torch.float64))
  chain = (a / 64 + 24) * 2.0 ** -22
  depth = torch.where(torch.isfinite(want), want.abs(), torch.zeros_like(want))
  spread = math.log(a) + 1
  inf = torch.isinf(want)
  assert torch.equal(got_lp.cpu()[inf].double(), want[inf])
  assert ((got_lp.detach().cpu().double() - want)[~inf].abs() <= (chain + 2.0 ** -21 * (depth + spread))[~inf]).all()
  off_h = chain * (h + 2 * spread) + 2.0 ** -21 * spread
  assert ((got_h.detach().cpu().double() - h).abs() <= off_h).all()
  grad, = torch.autograd.grad([got_lp, got_h], [leaf], [g_lp.cuda(), g_h.cuda()])
  assert grad.dtype == x.dtype
  one = torch.zeros_like(p).scatter_(1, at, 1.0) * there[:, None]
  gl, gh = (g_lp.double() * there)[:, None], g_h.double()[:, None]
  term = torch.where(p > 0, p * (lp + h[:, None]), torch.zeros_like(p))
  want = torch.where(ok, (gl * (one - p) - gh * term) / float(np.float32(temperature)), torch.zeros_like(p))
  log_size = torch.where(p > 0, p * (lp.abs() + h[:, None]), torch.zeros_like(p))
  tol = ((gl.abs() * (one + p) + gh.abs() * log_size) * chain + gh.abs() * p * (chain + off_h[:, None]) + (gl.abs() * p + gh.abs() * log_size) * 2.0 ** -21 *
         torch.where(p > 0, lp.abs() + spread, torch.zeros_like(p))) / temperature
  tol = tol + torch.finfo(x.dtype).eps / 2 * (want.abs() + tol) + torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps + 2.0 ** -120
  bad = ~((grad.cpu().double() - want).abs() <= tol)
  assert not bad.any(), (int(bad.sum()), float((grad.cpu().double() - want).abs().max()))
  return got_lp, got_h, grad


# ---------------------------------------------------------------- without a GPU


def rows(**kw):
  d = N.LogitsDesc()
  d.n, d.row_stride, d.legal_stride, d.actions, d.dtype = 4, 5, 5, 5, N.F32
  for k, v in kw.items():
    setattr(d, k, v)
  return d


def rules(**kw):
  r = N.Sampling()
  r.temperature, r.top_p = 1.0, 1.0
  for k, v in kw.items():
    setattr(r, k, v)
  return r


def test_description_layouts_and_sizes():
  assert ctypes.sizeof(N.LogitsDesc) == 32 and ctypes.sizeof(N.Sampling) == 48
  lib, size = N.lib(), N.c_u64(9)
  assert lib.pcx_sample_size(ctypes.byref(rows(actions=16384)), ctypes.byref(size)) == 0 and size.value == 0
  assert lib.pcx_sample_size(ctypes.byref(rows(actions=16385)), ctypes.byref(size)) == 0 and size.value > 0
  assert lib.pcx_log_prob_size(ctypes.byref(rows()), ctypes.byref(size)) == 0 and size.value == 0


@pytest.mark.parametrize('kw,text', [(dict(dtype=N.I32), 'float32'), (dict(n=-1), 'rows'), (dict(n=(1 << 31) + 1), 'rows'), (dict(actions=0), 'actions'),
                                     (dict(actions=(1 << 24) + 1), 'actions'), (dict(row_stride=-1), 'stride'), (dict(legal_stride=-1), 'stride')])
def test_refused_descriptions(kw, text):
  lib, size = N.lib(), N.c_u64(0)
  for f in (lib.pcx_sample_size, lib.pcx_log_prob_size):
    assert f(ctypes.byref(rows(**kw)), ctypes.byref(size)) == N.E_INVALID
    assert text in lib.pcx_last_error().decode()


@pytest.mark.parametrize('kw', [dict(temperature=-1.0), dict(temperature=math.nan), dict(top_k=-1), dict(top_p=-0.5), dict(top_p=math.nan),
                                dict(min_p=-0.1), dict(min_p=1.5), dict(min_p=math.nan)])
def test_refused_rules(kw):
  at = 1 << 20
  assert N.lib().pcx_sample_actions(ctypes.byref(rows()), ctypes.byref(rules(**kw)), at, None, at, at, None, 0, None) == N.E_INVALID


def test_null_and_misaligned_pointers_are_refused_before_any_launch():
  lib, at = N.lib(), 1 << 20
  for logits, uniforms, out in ((None, at, at), (at, None, at), (at, at, None), (at + 1, at, at), (at, at + 2, at), (at, at, at + 1)):
    assert lib.pcx_sample_actions(ctypes.byref(rows()), ctypes.byref(rules()), logits, None, uniforms, out, None, 0, None) == N.E_INVALID
  assert lib.pcx_sample_actions(ctypes.byref(rows()), None, at, None, at, at, None, 0, None) == N.E_INVALID
  assert lib.pcx_sample_actions(ctypes.byref(rows(actions=100000)), ctypes.byref(rules()), at, None, at, at, at, 64, None) == N.E_INVALID  # workspace
  for i in range(5):
    args = [at] * 5
    args[i] = None
    assert lib.pcx_log_prob(ctypes.byref(rows()), 1.0, args[0], None, args[1], args[2], args[3], args[4], None, 0, None) == N.E_INVALID
    assert lib.pcx_log_prob_backward(ctypes.byref(rows()), 1.0, args[0], None, args[1], args[2], args[3], None, None, args[4], None) == N.E_INVALID
  for t in (0.0, -1.0, math.nan, math.inf):
    assert lib.pcx_log_prob(ctypes.byref(rows()), t, at, None, at, at, at, at, None, 0, None) == N.E_INVALID


def test_needs_a_gpu():
  if torch.cuda.is_available():
    pytest.skip('there is one')
  with pytest.raises(RuntimeError, match='PyTorch-ROCm'):
    policy.sample(torch.zeros(2, 3), torch.zeros(2))
  with pytest.raises(RuntimeError, match='PyTorch-ROCm'):
    policy.log_prob(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int32))


def test_the_reference_of_these_tests():
  assert draw_row([0, 0, 0, 0], 0.5) == (2, False)
  assert draw_row([0, 0, 0, 0], 0.99, top_p=0.5) == (1, False)
  assert draw_row([1, 2, 2, 0], 0.0, temperature=0) == (1, False)
  assert draw_row([1, 2, 2, 0], 0.99, top_k=1)[0] == 1
  assert draw_row([-np.inf, np.nan], 0.3) == (-1, False)


# ---------------------------------------------------------------- on the GPU

WIDTHS = [1, 2, 3, 5, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200, 511, 512, 513, 1000, 4095, 4096, 4097, 9001, 16384, 16385, 40000]


@pytest.mark.gpu
@pytest.mark.parametrize('a', WIDTHS)
def test_sample_widths(a):
  n = 70 if a < 5000 else 9
  for k, dtype in enumerate(DTYPES):
    x, u = logits_of(n, a, dtype, 100 * a + k)
    legal = torch.rand(n, a, generator=torch.Generator().manual_seed(a)) < 0.7
    legal[1] = False
    check_sample(x, u)
    check_sample(x, u, legal=legal, temperature=0.7)
    check_sample(x, u, top_k=3)
    check_sample(x, u, top_p=0.8, temperature=1.5)
    check_sample(x, u, min_p=0.1)
    check_sample(x, u, legal=legal, temperature=1.2, top_k=max(1, a // 3), top_p=0.9, min_p=0.01)


@pytest.mark.gpu
@pytest.mark.parametrize('a', [5, 16, 100, 300, 2000, 9000, 20000])
def test_sample_rules_row_by_row(a):
  n = 40
  g = torch.Generator().manual_seed(a)
  x, u = logits_of(n, a, 'float32', a + 1)
  pick = lambda values, dtype: torch.tensor(values, dtype=dtype)[torch.randint(0, len(values), (n,), generator=g)]
  check_sample(x, u, temperature=pick([0.0, 0.3, 1.0, 2.5, -1.0, math.nan], torch.float32), top_k=pick([0, 1, 2, 7, a, a + 5, -3], torch.int32),
               top_p=pick([0.0, 0.1, 0.6, 1.0, 2.0], torch.float32), min_p=pick([0.0, 0.05, 0.5, 1.0, 3.0], torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize('a', [4, 16, 120, 500, 4000, 10000, 30000])
@pytest.mark.parametrize('dtype', DTYPES)
def test_sample_ties_go_to_the_lowest_index(a, dtype):
  """Few distinct values, and rows of one value alone, whose sums are exact: the cuts fall within ties."""
  n = 24
  g = torch.Generator().manual_seed(a)
  x = torch.randint(-2, 3, (n, a), generator=g).to(getattr(torch, dtype))
  x[:8] = 1.5
  x[7] = torch.finfo(x.dtype).min  # (a row masked by the lowest value everywhere: all its actions are equal)
  u = torch.rand(n, generator=g)
  u[:4] = torch.tensor([0.0, 0.5, 0.75, 1 - 2.0 ** -24])
  for kw in (dict(), dict(top_k=1), dict(top_k=a // 2), dict(top_k=a - 1), dict(top_p=0.5), dict(top_p=0.25, top_k=a // 2), dict(min_p=1.0), dict(temperature=0.0)):
    check_sample(x, u, **kw)
  got = policy.sample(x.cuda(), u.cuda(), temperature=0.0).cpu()
  assert torch.equal(got, x.float().argmax(1).int()) or (x.gather(1, got.long()[:, None])[:, 0] == x.max(1).values).all()
  assert (policy.sample(x[:8].cuda(), u[:8].cuda(), top_k=1).cpu() == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize('a', [6, 40, 700, 6000, 20000])
@pytest.mark.parametrize('dtype', DTYPES)
def test_sample_infinities_and_no_numbers(a, dtype):
  x, u = logits_of(12, a, dtype, a)
  info = torch.finfo(x.dtype)
  x[0] = -math.inf
  x[1] = math.nan
  x[2, 3:] = -math.inf
  x[3, 4] = math.inf
  x[4, 1] = x[4, 5] = math.inf
  x[5, 2] = math.nan
  x[6] = info.max
  x[7, 0], x[7, 1:] = info.max, info.min
  x[8] = 0.0
  x[8, ::2] = -0.0
  legal = torch.ones(12, a, dtype=torch.bool)
  legal[9] = False
  legal[10, 1:] = False
  x[10, 1], x[11, 2] = math.nan, math.inf  # (in a place that is not allowed)
  legal[11, 2] = False
  for kw in (dict(), dict(top_k=2), dict(top_p=0.7), dict(min_p=0.3), dict(temperature=0.0), dict(top_k=3, top_p=0.5, temperature=0.5)):
    got = check_sample(x, u, legal=legal, **kw)
    assert got[0] == -1 and got[1] == -1 and got[9] == -1 and got[10] == 0 and got[3] == 4 and got[11] != 2


@pytest.mark.gpu
@pytest.mark.parametrize('a', [3, 16, 64, 3000, 20000])
def test_sample_numbers_outside_and_at_the_ends(a):
  """u = 0 takes the first kept action of positive weight; one or more, or no number, the last."""
  x, _ = logits_of(5, a, 'float32', a)
  x[:, 0] = -2000.0  # (weight 0 in 64 bits)
  x[:, -1] = -2000.0
  got = policy.sample(x.cuda(), torch.tensor([0.0, 1.0, 2.0, math.nan, 1 - 2.0 ** -24]).cuda()).cpu()
  assert got[0] == 1 and got[1] == got[2] == got[3] == a - 2 and 1 <= got[4] <= a - 2


@pytest.mark.gpu
def test_sample_strides_out_and_shapes():
  base, u = logits_of(30, 40, 'bfloat16', 5)
  for lo, hi in ((0, 9), (1, 14), (3, 40), (7, 24)):
    want = policy.sample(base[:, lo:hi].contiguous().cuda(), u.cuda(), top_p=0.9)
    view = base.cuda()[:, lo:hi]
    assert torch.equal(policy.sample(view, u.cuda(), top_p=0.9), want)
    legal = (torch.rand(30, 50, generator=torch.Generator().manual_seed(6)) < 0.5).cuda()
    assert torch.equal(policy.sample(view, u.cuda(), legal=legal[:, lo + 2:hi + 2]),
                       policy.sample(view.contiguous(), u.cuda(), legal=legal[:, lo + 2:hi + 2].contiguous()))
    one = legal[0, lo:hi].contiguous()
    assert torch.equal(policy.sample(view, u.cuda(), legal=one), policy.sample(view, u.cuda(), legal=one.to(torch.uint8).repeat(30, 1)))
  row = base.cuda()[:1].expand(30, 40)  # one row of logits for all
  assert torch.equal(policy.sample(row, u.cuda()), policy.sample(row.contiguous(), u.cuda()))
  out = torch.full((32,), 77, dtype=torch.int32).cuda()
  policy.sample(base.cuda(), u.cuda(), out=out[1:31])
  assert out[0] == 77 and out[31] == 77 and torch.equal(out[1:31], policy.sample(base.cuda(), u.cuda()))
  assert policy.sample(base[:0].cuda(), u[:0].cuda()).shape == (0,)


@pytest.mark.gpu
def test_sample_refusals():
  x, u = torch.zeros(4, 5).cuda(), torch.zeros(4).cuda()
  legal = torch.ones(4, 5, dtype=torch.bool).cuda()
  for kw in (dict(logits=x.cpu()), dict(logits=x[0]), dict(logits=x.t()[:4, :4]), dict(logits=x[:, :0]), dict(uniforms=u[:3]), dict(uniforms=u.double()),
             dict(uniforms=u.cpu()), dict(legal=legal[:, :4]), dict(legal=legal.float()), dict(legal=legal.cpu()), dict(legal=legal.t().contiguous().t()),
             dict(temperature=-0.5), dict(temperature=math.nan), dict(temperature=u.double()), dict(temperature=u[:3]), dict(top_k=-1), dict(top_k=1.5),
             dict(top_k=u), dict(top_p=-0.1), dict(min_p=1.1), dict(min_p=-0.1), dict(out=torch.zeros(4).cuda()), dict(out=torch.zeros(8, dtype=torch.int32).cuda()[::2])):
    with pytest.raises(ValueError):
      policy.sample(**dict(dict(logits=x, uniforms=u), **kw))
  with pytest.raises(TypeError):
    policy.sample(x.double(), u)
  taken = torch.zeros(4, dtype=torch.int32).cuda()
  for kw in (dict(actions=taken.long()), dict(actions=taken[:2]), dict(actions=taken.cpu()), dict(temperature=0.0), dict(temperature=math.inf), dict(legal=legal[:2])):
    with pytest.raises(ValueError):
      policy.log_prob(**dict(dict(logits=x, actions=taken), **kw))


@pytest.mark.gpu
def test_sample_frequencies():
  """The numbers k / n pick each action as often as its probability says, to one part in n for each border."""
  x = torch.tensor([0.3, -1.0, 2.0, 0.0, 1.1]).cuda()
  n = 1 << 16
  u = (torch.arange(n) / n).cuda()
  got = torch.bincount(policy.sample(x.expand(n, 5), u).long(), minlength=5).double().cpu() / n
  assert ((got - torch.softmax(x.double().cpu(), 0)).abs() <= 2.0 / n).all()


@pytest.mark.gpu
@pytest.mark.parametrize('a', WIDTHS + [70000])
def test_log_prob_widths(a):
  for k, dtype in enumerate(DTYPES):
    n = 50 if a < 5000 else 7
    x, u = logits_of(n, a, dtype, a + k)
    legal = torch.rand(n, a, generator=torch.Generator().manual_seed(a)) < 0.7
    legal[2] = False
    taken = (u * a).int().clamp(max=a - 1)
    check_log_prob(x, taken)
    check_log_prob(x, policy.sample(x.cuda(), u.cuda(), legal=legal.cuda()).cpu(), legal=legal, temperature=0.6)


@pytest.mark.gpu
@pytest.mark.parametrize('a', [5, 30, 300, 5000, 20000])
@pytest.mark.parametrize('dtype', DTYPES)
def test_log_prob_odd_rows(a, dtype):
  x, _ = logits_of(10, a, dtype, a)
  info = torch.finfo(x.dtype)
  taken = torch.ones(10, dtype=torch.int32)
  legal = torch.ones(10, a, dtype=torch.bool)
  x[0] = -math.inf
  taken[0] = -1
  x[1, 2:] = -math.inf
  x[2] = info.max
  x[3, 0] = info.max
  x[3, 1:] = info.min
  taken[3] = 0
  legal[4] = False
  taken[4] = -1
  taken[5] = -1  # an environment that did nothing although it could
  legal[6, 1] = False  # an action that was not allowed
  x[7, 3] = math.nan
  legal[8, 3] = False
  x[8, 3] = math.nan
  x[9] = info.min
  lp, h, grad = check_log_prob(x, taken, legal=legal, temperature=1.3)
  assert lp[0] == 0 and lp[4] == 0 and lp[5] == 0 and lp[6] == -math.inf
  assert h[0] == 0 and h[4] == 0 and not grad[0].any() and not grad[4].any() and grad[7, 3] == 0 and grad[8, 3] == 0
  for bad in (a, a + 100, -2, 2 ** 31 - 1):
    taken[3] = bad
    leaf = x.cuda().requires_grad_()
    lp, _ = policy.log_prob(leaf, taken.cuda(), legal=legal.cuda())
    assert torch.isnan(lp[3]) and lp[0] == 0
    grad, = torch.autograd.grad(lp[1:6].sum(), leaf)
    assert torch.isnan(grad[3]).all() and not torch.isnan(grad[1]).any()


@pytest.mark.gpu
def test_log_prob_infinite_logits():
  x = torch.zeros(3, 6)
  x[0, 1] = math.inf
  x[1, 1] = x[1, 4] = math.inf
  leaf = x.cuda().requires_grad_()
  lp, h = policy.log_prob(leaf, torch.tensor([1, 4, 0], dtype=torch.int32).cuda())
  lp_, h_ = lp, h
  lp, h = lp.detach(), h.detach()
  assert lp[0] == 0 and abs(float(lp[1]) + math.log(2)) < 1e-6 and h[0] == 0 and abs(float(h[1]) - math.log(2)) < 1e-6
  grad, = torch.autograd.grad(lp_.sum() + h_.sum(), leaf)
  assert torch.isfinite(grad).all() and not grad[0].any()


@pytest.mark.gpu
def test_log_prob_gradient_against_differences():
  """Of float64 log_softmax and of the kernel's own results, along one direction v: h = 2^-6 leaves h^2 / 6 of a third derivative
  bounded by 6 |v|^3 a row, and the kernel's own rounding 2^-18 / h."""
  x, u = logits_of(40, 12, 'float32', 3, spread=1.0)
  taken = (u * 12).int()
  v = torch.randn(40, 12, generator=torch.Generator().manual_seed(4)) / 4
  g_lp, g_h = torch.randn(40, generator=torch.Generator().manual_seed(5)), torch.randn(40, generator=torch.Generator().manual_seed(6))
  leaf = x.cuda().requires_grad_()
  out = policy.log_prob(leaf, taken.cuda(), temperature=0.8)
  grad, = torch.autograd.grad(out, [leaf], [g_lp.cuda(), g_h.cuda()])
  slope = float((grad.cpu().double() * v.double()).sum())
  h = 2.0 ** -6

  def own(t):
    lp, e = policy.log_prob((x + t * v).cuda(), taken.cuda(), temperature=0.8)
    return float((lp.cpu().double() * g_lp.double() + e.cpu().double() * g_h.double()).sum())

  def exact(t):
    lp, p, e, _, _ = soft64(x.double() + t * v.double(), None, 0.8)
    return float((lp.gather(1, taken.long()[:, None])[:, 0] * g_lp.double() + e * g_h.double()).sum())

  third = float(((g_lp.abs() + 4 * g_h.abs()).double() * 6 * (v.double().abs().max(1).values / 0.8) ** 3).sum())
  bound = h * h / 6 * third + 2.0 ** -18 / h
  for f in (own, exact):
    assert abs((f(h) - f(-h)) / (2 * h) - slope) <= bound
  assert bound < 0.1 * abs(slope) + 0.05


@pytest.mark.gpu
def test_log_prob_strides_one_gradient_and_no_gradient():
  base, u = logits_of(20, 50, 'float32', 8)
  taken = (u * 9).int().cuda()
  view = base.cuda()[:, 3:12]
  lp, h = policy.log_prob(view, taken)
  lp2, h2 = policy.log_prob(view.contiguous(), taken)
  assert torch.equal(lp, lp2) and torch.equal(h, h2) and not lp.requires_grad
  leaf = view.contiguous().requires_grad_()
  lp, h = policy.log_prob(leaf, taken)
  only, = torch.autograd.grad(lp.sum(), leaf, retain_graph=True)
  other, = torch.autograd.grad(h.sum(), leaf, retain_graph=True)
  both, = torch.autograd.grad(lp.sum() + h.sum(), leaf)
  assert ((both - only - other).abs() <= 8 * 2.0 ** -24 * (both.abs() + only.abs() + other.abs()) + 2.0 ** -24).all()
  wide = base.cuda().requires_grad_()  # a leaf read through a view
  lp, _ = policy.log_prob(wide[:, 3:12], taken)
  lp.sum().backward()
  assert torch.equal(wide.grad[:, 3:12], only) and not wide.grad[:, :3].any()
  assert policy.log_prob(base[:0].cuda(), taken[:0])[0].shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize('n,a', [(1000, 5), (300, 700), (20, 20000)])
def test_policy_in_graphs_and_on_other_streams(n, a):
  x, u = logits_of(n, a, 'float32', a)
  x, u = x.cuda(), u.cuda()
  g_lp, g_h = torch.randn(n).cuda(), torch.randn(n).cuda()

  def step():
    taken = policy.sample(x, u, top_k=a // 2 + 1, top_p=0.9)
    lp, h, stats = policy.log_prob(x, taken, return_stats=True)
    return taken, lp, h, policy.log_prob_backward(x, taken, h, stats, g_lp, g_h)

  want = step()
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    other = step()
  torch.cuda.current_stream().wait_stream(side)
  assert all(torch.equal(p, q) for p, q in zip(want, other))
  leaf = x.clone().requires_grad_()
  grad, = torch.autograd.grad(policy.log_prob(leaf, want[0]), [leaf], [g_lp, g_h])
  assert torch.equal(grad, want[3])
  torch.cuda.synchronize()
  graphs = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
  with torch.cuda.graph(graphs[0]):
    first = step()
  with torch.cuda.graph(graphs[1]):
    second = step()
  for i in range(4):
    x.copy_(x.roll(1, 1))
    u.copy_(u.roll(1))
    expect = step()
    graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    for got in (first, second):
      assert all(torch.equal(p, q) for p, q in zip(expect, got))
  with pytest.raises(RuntimeError, match='log_prob_backward'):
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
      policy.log_prob(leaf, want[0])
  torch.cuda.synchronize()


@pytest.mark.gpu
def test_a_rollout_and_a_gradient_step():
  """Boards -> project -> logits -> sample -> step, and the policy gradient over the boards kept, against float64."""
  import os
  from pycolab_amd import rendering
  from pycolab_amd.compiler import GameTemplate
  from pycolab_amd.engine import Engine
  path = os.path.join(os.path.dirname(__file__), 'golden', 'templates', 'scrolly_maze_L0.npz')
  B, T, H, layers = 128, 4, 64, 'P#@abc'
  g = torch.Generator().manual_seed(1)
  weight = (torch.randn(H, len(layers), 10, 30, generator=g) / 8).cuda()
  bias, head = (torch.randn(H, generator=g) / 8).cuda(), (torch.randn(5, H, generator=g) / 8).cuda()
  numbers = torch.rand(T, B, generator=g).cuda()
  engines = [Engine.from_template(GameTemplate.load(path), batch=B, auto_reset=True) for _ in range(2)]
  policy_net = rendering.ObservationProjection(layers, weight, bias, activation='tanh')
  obs = engines[0].its_showtime()[0]
  engines[1].its_showtime()
  boards, taken, legal = [], [], torch.tensor([1, 1, 1, 1, 0], dtype=torch.bool).cuda()  # (nobody quits)
  for t in range(T):
    boards.append(obs.board.clone())
    logits = policy_net(obs) @ head.t()
    drawn = engines[0].step_sampled(logits, numbers[t], legal=legal, top_p=0.95)
    obs = engines[0]._result()[0]
    same = policy.sample(logits, numbers[t], legal=legal, top_p=0.95)
    assert torch.equal(drawn, same)
    play_obs, reward, discount = engines[1].play(same)
    assert torch.equal(play_obs.board, obs.board) and torch.equal(reward, engines[0].buffers['reward'].tensor)
    taken.append(drawn)
  boards, taken = torch.cat(boards), torch.cat(taken)
  assert taken.min() >= 0 and taken.max() <= 3 and boards.shape == (T * B, 10, 30)
  gain = torch.randn(T * B, generator=g).cuda()
  leaves = [weight.clone().requires_grad_(), bias.clone().requires_grad_(), head.clone().requires_grad_()]
  hidden = rendering.project(boards, layers, leaves[0], leaves[1], activation='tanh')
  lp, h = policy.log_prob(hidden @ leaves[2].t(), taken, legal=legal)
  loss = -(lp * gain).mean() - 0.01 * h.mean()
  got = torch.autograd.grad(loss, leaves)
  exact = [p.detach().double().cpu().requires_grad_() for p in leaves]
  x = torch.stack([(boards.cpu() == ord(c)) for c in layers], 1).double().flatten(1)
  z = torch.tanh(x @ exact[0].flatten(1).t() + exact[1]) @ exact[2].t()
  log_p = torch.log_softmax(z.masked_fill(~legal.cpu(), -math.inf), 1)
  l64 = -(log_p.gather(1, taken.long().cpu()[:, None])[:, 0] * gain.double().cpu()).mean()
  # (over the four legal moves: autograd would multiply 0 by infinity at the fifth)
  log4 = torch.log_softmax(z[:, :4], 1)
  h64 = -(log4.exp() * log4).sum(1)
  want = torch.autograd.grad(l64 - 0.01 * h64.mean(), exact)
  for a, b in zip(got, want):
    assert (a.cpu().double() - b).abs().max() <= 2.0 ** -14 * b.abs().max()  # float32 throughout: some hundred roundings of 2^-24
  with pytest.raises(ValueError):
    engines[0].step_sampled(logits[:5], numbers[0][:5])
  for e in engines:
    e.close()


@pytest.mark.gpu
def test_results_changed_in_place():
  x = torch.randn(6, 5, device='cuda', requires_grad=True)
  taken = torch.tensor([0, 1, 2, 3, 4, -1], dtype=torch.int32, device='cuda')
  lp, h = policy.log_prob(x, taken)
  lp.mul_(2.0)
  (lp.sum() + h.sum()).backward()
  y = x.detach().clone().requires_grad_()
  lp, h = policy.log_prob(y, taken)
  (2.0 * lp.sum() + h.sum()).backward()
  assert torch.equal(x.grad, y.grad)
  lp, h = policy.log_prob(y, taken)
  h.add_(1.0)  # (the gradient needs it as it was)
  with pytest.raises(RuntimeError, match='inplace'):
    h.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('n,a', [(9, 16385), (5, 40001), (3, 262144), (2, 262145), (130, 270000)])
def test_sample_few_of_very_many(n, a, dtype):
  """Rows that no workgroup holds with a small top_k, or the best alone: random ones, ones of few values, ones of one value,
  masked ones, best ones at either end."""
  x, u = logits_of(n, a, dtype, a)
  g = torch.Generator().manual_seed(a)
  x[0] = torch.randint(-2, 3, (a,), generator=g).to(x.dtype)
  x[1] = 0.25
  legal = torch.ones(n, a, dtype=torch.bool)
  if n > 2:
    legal[2] = False
    legal[2, a - 1] = True
  if n > 4:
    x[3] = -math.inf
    x[3, a - 3:] = 1.0
    x[4, a - 1] = math.inf
    legal[4, :a // 2] = torch.rand(a // 2, generator=g) < 0.001
  rows = slice(0, min(n, 12))  # (the plain form sorts)
  for kw in (dict(top_k=1), dict(top_k=40, top_p=0.9), dict(top_k=256, temperature=0.7, min_p=0.01), dict(temperature=0.0), dict(top_k=257), dict(temperature=0.0, top_k=3)):
    got = policy.sample(x.cuda(), u.cuda(), legal=legal.cuda(), **kw).cpu()
    want = policy.sample(x[rows].cuda(), u[rows].cuda(), legal=legal[rows].cuda(), **kw).cpu()
    assert torch.equal(got[rows], want)  # (130 rows or 12 of them: another way there)
    check_sample(x[rows], u[rows], legal=legal[rows], **kw)
  per_row = torch.tensor([0.0, 0.5, 1.0, 2.0])[torch.arange(n) % 4]
  check_sample(x[rows], u[rows], legal=legal[rows], top_k=50, top_p=0.8, temperature=per_row[rows])


@pytest.mark.gpu
def test_tensors_with_a_tangent_are_told_apart():
  from pycolab_amd import device as dev
  plain = torch.ones(3)
  dev.refuse_tangents('f', plain, None)
  with torch.autograd.forward_ad.dual_level():
    dual = torch.autograd.forward_ad.make_dual(torch.ones(3), torch.ones(3))
    dev.refuse_tangents('f', plain, None)
    with pytest.raises(RuntimeError, match='forward'):
      dev.refuse_tangents('f', plain, dual)
  assert not dual.requires_grad  # (which is why nothing else notices)


@pytest.mark.gpu
def test_log_prob_refuses_forward_mode_and_function_transforms():
  x, taken = torch.randn(4, 5).cuda(), torch.zeros(4, dtype=torch.int32).cuda()
  with torch.autograd.forward_ad.dual_level():
    dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
    with pytest.raises(RuntimeError, match='forward'):
      policy.log_prob(dual, taken)
    policy.log_prob(x, taken)  # (no tangent)
  f = lambda x: policy.log_prob(x, taken)[0]
  for transform in (lambda: torch.func.jvp(f, (x,), (x,)), lambda: torch.func.grad(lambda x: f(x).sum())(x),
                    lambda: torch.func.vmap(f)(torch.stack([x] * 2)), lambda: torch.func.vjp(f, x)):
    with pytest.raises(RuntimeError):
      transform()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('log2a,bits', [(20, 43.5), (20, 46.0), (22, 41.5), (24, 39.25), (24, 50.0)])
def test_sample_long_tails(log2a, bits, dtype):
  """One action and 2^log2a - 1 equal ones of about 2^-bits of its weight each, itself the last one: what of the tail top_p
  keeps, counted in 64 bits.  u = 0 then takes the first action if any of the tail is kept, a number halfway through the
  kept tail's part of the total the action there."""
  a = 1 << log2a
  best = torch.tensor(0.0)
  low = float(torch.tensor(-bits * math.log(2.0)).to(getattr(torch, dtype)))
  w = math.exp(low)
  tail = (a - 1) * w
  total = 1.0 + tail
  x = torch.full((1, a), low).to(getattr(torch, dtype))
  x[0, a - 1] = best
  x = x.cuda()
  for k in range(1, 6):
    p = 1.0 - k * 2.0 ** -24  # (exact in float32)
    need = (p * total - 1.0) / w  # how many of the tail it takes
    if abs(need) < 64 or abs(need - (a - 1)) < 64:
      continue  # (on the border: the sums of the 64-bit formula are not that good)
    kept = 0 if need < 0 else min(a - 1, math.ceil(need))
    got = int(policy.sample(x, torch.zeros(1).cuda(), top_p=p).cpu())
    assert got == (0 if kept else a - 1), (k, kept, got)
    if not kept:
      continue
    u = float(np.float32(0.5 * kept * w / (1.0 + kept * w)))
    at = u * (1.0 + kept * w) / w
    got = int(policy.sample(x, torch.tensor([u]).cuda(), top_p=p).cpu())
    assert abs(got - at) <= 1.0 + at * 2.0 ** -30, (k, kept, got, at)


@pytest.mark.gpu
@pytest.mark.parametrize('a', [16385, 33380, 131072, 262144, 300000])
def test_sample_rules_as_numbers_and_as_rows_agree(a):
  """The same rule as a number and as an array row by row: the same actions, whichever kernels they take."""
  n = 8
  for dtype in DTYPES:
    x, u = logits_of(n, a, dtype, a)
    x[1] = -40.0
    x[1, a - 1] = 0.0  # a long tail
    x[2] = 0.5
    x, u = x.cuda(), u.cuda()
    u[1] = 0.0
    for rule in (dict(top_k=1), dict(top_k=40, top_p=0.9), dict(top_k=256, top_p=1 - 2.0 ** -24), dict(top_k=257, top_p=1 - 2.0 ** -24), dict(top_k=a // 2, top_p=0.95),
                 dict(top_p=1 - 2.0 ** -23), dict(temperature=0.0), dict(temperature=0.7, top_k=40, min_p=0.01), dict(min_p=0.001)):
      want = policy.sample(x, u, **rule)
      rows = {k: torch.full((n,), v, dtype=torch.int32 if k == 'top_k' else torch.float32).cuda() for k, v in rule.items()}
      assert torch.equal(policy.sample(x, u, **rows), want), rule
      for k in rule:
        assert torch.equal(policy.sample(x, u, **dict(rule, **{k: rows[k]})), want), (rule, k)
      assert torch.equal(policy.sample(x[1:4], u[1:4], **rule), want[1:4])
    # rules of both kinds in one batch
    ks = torch.tensor([1, 40, 0, 256, 257, a, 3, 0], dtype=torch.int32).cuda()
    ts = torch.tensor([1.0, 0.7, 1.0, 0.5, 1.0, 1.0, 0.0, 0.0]).cuda()
    got = policy.sample(x, u, top_k=ks, temperature=ts, top_p=0.9)
    for i in range(n):
      assert got[i] == policy.sample(x[i:i + 1], u[i:i + 1], top_k=int(ks[i]), temperature=float(ts[i]), top_p=0.9)[0], i


@pytest.mark.gpu
def test_backward_after_the_actions_were_drawn_anew_is_refused():
  """A buffer of actions that sample(out=...) writes again before the gradient of the old ones' log-probability."""
  x, u = logits_of(40, 9, 'float32', 60)
  leaf, u = x.cuda().requires_grad_(), u.cuda()
  taken = torch.empty(40, dtype=torch.int32, device='cuda')
  policy.sample(leaf, u, out=taken)
  lp, _ = policy.log_prob(leaf, taken)
  policy.sample(leaf, u.flip(0), out=taken)
  with pytest.raises(RuntimeError, match='modified by an inplace operation'):
    lp.sum().backward()
  with pytest.raises(RuntimeError, match='modified by an inplace operation'):  # a part of it is it, too
    both = policy.log_prob(leaf, taken)[0]
    policy.sample(leaf[:3], u[:3], out=taken[:3])
    both.sum().backward()
  policy.log_prob(leaf, taken)[0].sum().backward()
  want = policy.log_prob_backward(leaf, taken, *policy.log_prob(leaf, taken, return_stats=True)[1:], torch.ones(40, device='cuda'))
  assert torch.equal(leaf.grad, want)
  with torch.inference_mode():  # (a tensor of no version)
    held = torch.empty(40, dtype=torch.int32, device='cuda')
    assert torch.equal(policy.sample(x.cuda(), u, out=held), policy.sample(x.cuda(), u))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('a', [5, 200, 3000])
def test_log_prob_whose_saved_tensors_went_elsewhere(a, dtype):
  """What autograd saved comes back laid out in its own way: copies on the host, a forward pass made anew."""
  from torch.utils.checkpoint import checkpoint
  n = 30
  base, u = logits_of(n, 2 * a + 7, dtype, a)
  mask = torch.rand(n, 3 * a, generator=torch.Generator().manual_seed(a)) < 0.7
  taken = (u * a).int().cuda()
  g = torch.randn(2, n, generator=torch.Generator().manual_seed(1)).cuda()
  wide, legal = base.cuda(), mask.cuda()
  for allowed in (None, legal[:, a:2 * a], legal[0, :a]):
    view = wide[:, 5:5 + a]
    lp, h, stats = policy.log_prob(view, taken, legal=allowed, return_stats=True)
    want = policy.log_prob_backward(view, taken, h, stats, g[0], g[1], legal=allowed)

    def grads(run):
      leaf = wide.clone().requires_grad_()
      out = run(lambda x: policy.log_prob(x[:, 5:5 + a], taken, legal=allowed), leaf)
      assert torch.equal(out[0], lp) and torch.equal(out[1], h)
      torch.autograd.backward(out, [g[0], g[1]])
      assert not leaf.grad[:, :5].any() and not leaf.grad[:, 5 + a:].any()
      return leaf.grad[:, 5:5 + a]

    def on_the_host(f, x):
      with torch.autograd.graph.save_on_cpu():
        return f(x)

    assert torch.equal(grads(lambda f, x: f(x)), want)
    assert torch.equal(grads(on_the_host), want)
    for reentrant in (False, True):
      assert torch.equal(grads(lambda f, x: checkpoint(f, x, use_reentrant=reentrant)), want)


@pytest.mark.gpu
@pytest.mark.parametrize('n,a', [((1 << 22) + 37, 3), ((1 << 22) + 37, 16), ((1 << 22) + 37, 20), (1024 + 37, 16500), (1024 + 37, 270000)])
def test_more_rows_than_one_launch_takes(n, a):
  """The rows behind the first 2^22 (1,024 of more than 16,384 actions) give what they give by themselves."""
  dtype = torch.bfloat16 if a > 100 else torch.float32
  g = torch.Generator(device='cuda').manual_seed(a)
  x = torch.randn(n, a, generator=g, device='cuda', dtype=dtype).mul_(2)
  u, legal = torch.rand(n, generator=g, device='cuda'), torch.rand(n, a, generator=g, device='cuda', dtype=dtype) < 0.8
  legal[n - 3] = False
  rules = dict(temperature=torch.rand(n, generator=g, device='cuda') + 0.5, top_k=torch.randint(0, 300, (n,), generator=g, device='cuda', dtype=torch.int32),
               top_p=torch.rand(n, generator=g, device='cuda') * 0.3 + 0.75, min_p=torch.rand(n, generator=g, device='cuda') * 0.01)
  rules['temperature'][1::5] = 0.0
  g_lp, g_h = torch.randn(n, generator=g, device='cuda'), torch.randn(n, generator=g, device='cuda')
  for kw in (dict(), dict(top_p=0.9), dict(top_k=40, temperature=0.7), rules):
    got = policy.sample(x, u, legal=legal, **kw)
    lp, h, stats = policy.log_prob(x, got, legal=legal, temperature=0.8, return_stats=True)
    grad = policy.log_prob_backward(x, got, h, stats, g_lp, g_h, legal=legal, temperature=0.8)
    for part in (slice(0, 9), slice(n - 47, n)):
      some = {k: v[part] if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
      want = policy.sample(x[part], u[part], legal=legal[part], **some)
      assert torch.equal(got[part], want)
      # (log_prob may divide few long rows: other sums, so they are held against 64 bits)
      exact, p, h64, _, ok = soft64(x[part].cpu(), legal[part].cpu(), 0.8)
      at = want.cpu().long().clamp(min=0)[:, None]
      there = want.cpu() >= 0
      lp64 = torch.where(there, exact.gather(1, at)[:, 0], torch.zeros_like(h64))
      off = (a / 64 + 24) * 2.0 ** -22 + 2.0 ** -21 * (lp64.abs() + math.log(a) + 1)
      off_h = (a / 64 + 24) * 2.0 ** -22 * (h64 + 2 * (math.log(a) + 1)) + 2.0 ** -21 * (math.log(a) + 1)
      assert ((lp[part].cpu().double() - lp64).abs() <= off).all() and ((h[part].cpu().double() - h64).abs() <= off_h).all()
      one = torch.zeros_like(p).scatter_(1, at, 1.0) * there[:, None]
      gl, gh = (g_lp[part].cpu().double() * there)[:, None], g_h[part].cpu().double()[:, None]
      term = torch.where(p > 0, p * (exact + h64[:, None]), torch.zeros_like(p))
      want64 = torch.where(ok, (gl * (one - p) - gh * term) / 0.8, torch.zeros_like(p))
      # p is off by `off` of itself, log p and H by off + off_h
      size = gl.abs() * (one + p) + gh.abs() * p * (torch.where(p > 0, exact.abs(), torch.zeros_like(p)) + h64[:, None] + 1)
      tol = size * 4 * (off + off_h)[:, None] + torch.finfo(dtype).eps / 2 * want64.abs() + 2.0 ** -100
      assert ((grad[part].cpu().double() - want64).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize('n,a,stride', [((1 << 20) + 3, 2100, 2100), (300, 20000, 1 << 23), (40, 1 << 20, (1 << 26) + 8)])
def test_offsets_beyond_31_bits(n, a, stride):
  """Logits of 2^31 elements and more: the last rows give what they give by themselves."""
  g = torch.Generator(device='cuda').manual_seed(a)
  held = torch.empty((n - 1) * stride + a, dtype=torch.bfloat16, device='cuda')
  assert held.numel() > 1 << 31
  x = held.as_strided((n, a), (stride, 1))
  for lo in range(0, n, 1 << 16):
    x[lo:lo + (1 << 16)].normal_(0, 2, generator=g)
  u = torch.rand(n, generator=g, device='cuda')
  g_lp, g_h = torch.randn(n, generator=g, device='cuda'), torch.randn(n, generator=g, device='cuda')
  for kw in (dict(top_p=0.9), dict(top_k=40, temperature=0.7), dict(temperature=0.0)):
    got = policy.sample(x, u, **kw)
    lp, h, stats = policy.log_prob(x, got, return_stats=True)
    for part in (slice(0, 5), slice(n // 2, n // 2 + 5), slice(n - 5, n)):
      near = x[part].contiguous()
      assert torch.equal(got[part], policy.sample(near, u[part], **kw))
      exact, _, h64, _, _ = soft64(near.cpu(), None, 1.0)
      lp64 = exact.gather(1, got[part].cpu().long()[:, None])[:, 0]
      off = (a / 64 + 24) * 2.0 ** -22
      assert ((lp[part].cpu().double() - lp64).abs() <= off + 2.0 ** -21 * (lp64.abs() + math.log(a) + 1)).all()
      assert ((h[part].cpu().double() - h64).abs() <= off * (h64 + 2 * (math.log(a) + 1)) + 2.0 ** -21 * (math.log(a) + 1)).all()
  if n * a < 1 << 31:
    return
  grad = policy.log_prob_backward(x, got, h, stats, g_lp, g_h)
  for part in (slice(0, 5), slice(n // 2, n // 2 + 5), slice(n - 5, n)):
    assert torch.equal(grad[part], policy.log_prob_backward(x[part], got[part], h[part], stats[part], g_lp[part], g_h[part]))


@pytest.mark.gpu
@pytest.mark.parametrize('a', [5, 300, 20000])
def test_what_a_rollout_in_inference_mode_left(a):
  """Actions and masks made in inference mode serve a gradient afterwards."""
  x, u = (t.cuda() for t in logits_of(40, a, 'float32', 66))
  legal = torch.rand(40, a, generator=torch.Generator().manual_seed(5)).cuda() < 0.8
  with torch.inference_mode():
    mask, one = legal.clone(), legal[0].clone()
    taken, free = policy.sample(x, u, legal=mask), policy.sample(x, u, legal=one)
  for t, m, plain in ((taken, mask, legal), (free, one, legal[0])):
    assert t.is_inference() and m.is_inference()
    grads = []
    for allowed, drawn in ((m, t), (plain, t.clone())):
      leaf = x.clone().requires_grad_()
      lp, h = policy.log_prob(leaf, drawn, legal=allowed)
      grads += torch.autograd.grad(lp.sum() + 0.1 * h.sum(), leaf)
    assert torch.equal(*grads)
