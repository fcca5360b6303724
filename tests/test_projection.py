"""rendering.ObservationProjection / project / project_backward (csrc/pcx_project.hip): the product of a weight with the
layers of boards, its epilogue and its gradients, against the same formulas in 64 bits.

Tolerances.  A product with a set feature is exact and sums are float32: with S = sum |w| over the set features plus
|bias|, a sum of m terms is off by at most (m + 2) 2^-23 S (2^-23: a matrix unit may cut off where it adds).  The
activations are 1.13-Lipschitz (gelu's slope peaks at 1.129) and the device's exp / tanh / erf are good to a few units:
8 * 2^-24 (|y| + 1) is allowed.  Storing the result rounds by eps / 2 of it.  In the gradients the activation's slope and
dz are each rounded to the weight's type (eps |dz| together, nothing for float32 beyond its own eps), and the slope moves
with the sum's error by at most 1.1 of it (silu, tanh and gelu have second derivatives below 1.1)."""

import ctypes
import math

import numpy as np
import pytest

from pycolab_amd import _native as N
from pycolab_amd import rendering

torch = pytest.importorskip('torch')

CHARS = ' #.@Pabcdefghijklmnopqrstuvwxyz01234'
DTYPES = ['float32', 'float16', 'bfloat16']
ACTS = [None, 'relu', 'silu', 'tanh', 'gelu']


def make(n, layers, rows, cols, hidden, dtype, seed, stacked=False, grid=False):
  """Boards (one character of them is not stacked), weight, bias and residual on the CPU.  grid: numbers whose sums are
  exact in float32, so that no sum lies between zero and its rounding (relu's slope is then the same in any precision)."""
  g = torch.Generator().manual_seed(seed)
  dt = getattr(torch, dtype)
  chars = CHARS[:layers]
  if stacked:
    boards = (torch.rand(n, layers, rows, cols, generator=g) < 0.3).to(torch.uint8) * torch.randint(1, 256, (n, layers, rows, cols), generator=g).to(torch.uint8)
  else:
    table = torch.tensor([ord(c) for c in chars + '~'], dtype=torch.uint8)
    boards = table[torch.randint(0, layers + 1, (n, rows, cols), generator=g)]
  if grid:
    weight = torch.randint(-8, 9, (hidden, layers, rows, cols), generator=g).float() / 16
    bias = torch.randint(-8, 9, (hidden,), generator=g).float() / 16
  else:
    weight = torch.randn(hidden, layers, rows, cols, generator=g) / math.sqrt(rows * cols)
    bias = torch.randn(hidden, generator=g)
  residual = torch.randn(n, hidden, generator=g)
  return chars, boards, weight.to(dt), bias.to(dt), residual.to(dt)


def features(chars, boards):
  if boards.dim() == 4:
    return (boards != 0).double().flatten(1)
  return torch.stack([(boards == ord(c)).double() for c in chars], 1).flatten(1)


def act64(kind, z):
  if kind == 'relu':
    return z.clamp(min=0), (z > 0).double()
  if kind == 'tanh':
    return torch.tanh(z), 1 - torch.tanh(z) ** 2
  if kind == 'silu':
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s))
  if kind == 'gelu':
    c = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
    return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
  return z, torch.ones_like(z)


def reference(chars, boards, weight, bias, act, residual):
  """(y, bound on what may differ from it, slope, bound on the slope)"""
  x, w = features(chars, boards), weight.double().flatten(1)
  b = torch.zeros(w.shape[0], dtype=torch.float64) if bias is None else bias.double()
  z = x @ w.t() + b
  size = x @ w.abs().t() + b.abs()
  off = (x.sum(1, keepdim=True) + 2) * 2.0 ** -23 * size
  y, slope = act64(act, z)
  tol = 1.13 * off + 8 * 2.0 ** -24 * (y.abs() + 1)
  if residual is not None:
    y = y + residual.double()
    tol = tol + 2.0 ** -24 * y.abs()
  half = torch.finfo(weight.dtype).eps / 2
  tiny = torch.finfo(weight.dtype).tiny * half
  return y, tol + half * (y.abs() + tol) + tiny, slope, (1.1 * off if act not in (None, 'relu') else 0 * off) + 8 * 2.0 ** -24


def near(got, want, tol, what):
  got = got.detach().double().cpu()
  assert got.shape == want.shape, (what, got.shape, want.shape)
  bad = ~((got - want).abs() <= tol)
  assert not bad.any(), '{}: {} of {} off, worst {:.3g} where {:.3g} is allowed'.format(
      what, int(bad.sum()), bad.numel(), float((got - want).abs().max()), float(tol.flatten()[(got - want).abs().flatten().argmax()]))


def check(n, layers, rows, cols, hidden, dtype, act, seed, stacked=False, with_bias=True, with_residual=True, train=False):
  chars, boards, weight, bias, residual = make(n, layers, rows, cols, hidden, dtype, seed, stacked, grid=act == 'relu')
  bias, residual = bias if with_bias else None, residual if with_residual else None
  y, tol, slope, slope_tol = reference(chars, boards, weight, bias, act, residual)
  dev = [None if t is None else t.cuda() for t in (boards, weight, bias, residual)]
  got = rendering.ObservationProjection(chars, dev[1], dev[2], activation=act)(dev[0], residual=dev[3])
  assert got.dtype == weight.dtype
  near(got, y, tol, 'forward')
  if not train:
    return
  leaves = [t for t in dev[1:] if t is not None]
  for t in leaves:
    t.requires_grad_()
  out = rendering.project(dev[0], chars, dev[1], dev[2], activation=act, residual=dev[3])
  near(out, y, tol, 'forward of a training step')
  grad = torch.randn(n, hidden, generator=torch.Generator().manual_seed(seed + 1)).to(weight.dtype)
  grads = list(torch.autograd.grad(out, leaves, grad.cuda()))
  check_grads(chars, boards, weight, grad, slope, slope_tol, grads[0], grads[1] if with_bias else None)
  if with_residual:
    assert torch.equal(grads[-1].cpu(), grad)


def check_grads(chars, boards, weight, grad, slope, slope_tol, dw, db):
  x, eps = features(chars, boards), torch.finfo(weight.dtype).eps
  dz = grad.double() * slope
  off = grad.double().abs() * slope_tol + eps * (dz.abs() + grad.double().abs() * slope_tol) + torch.finfo(weight.dtype).tiny * eps
  n = x.shape[0]
  for got, left, what in ((dw, x, 'grad weight'), (db, torch.ones(n, 1, dtype=torch.float64), 'grad bias')):
    if got is None:
      continue
    want = (dz.t() @ left)
    tol = off.t() @ left + (n + 2) * 2.0 ** -23 * (dz.abs().t() @ left)
    tol = tol + eps / 2 * (want.abs() + tol) + torch.finfo(weight.dtype).tiny * eps
    near(got.flatten(1) if what == 'grad weight' else got[:, None], want, tol, what)


# ---------------------------------------------------------------- without a GPU


def desc(**kw):
  d = N.ProjectDesc()
  d.n, d.row_stride, d.cells, d.n_layers, d.hidden, d.dtype = 4, 300, 300, 3, 64, N.BF16
  for i, c in enumerate('P#@'):
    d.chars[i] = ord(c)
  for k, v in kw.items():
    setattr(d, k, v)
  return d


def sizes(d):
  out = [N.c_u64(77) for _ in range(3)]
  rc = N.lib().pcx_project_sizes(ctypes.byref(d), *[ctypes.byref(x) for x in out])
  return rc, [int(x.value) for x in out]


def test_description_layout():
  # n, row_stride, 32 offsets: 34 x 8; six int32; 32 characters
  assert ctypes.sizeof(N.ProjectDesc) == 34 * 8 + 6 * 4 + 32
  assert N.ProjectDesc.chars.offset == 34 * 8 + 24


def test_sizes():
  rc, (packed, forward, backward) = sizes(desc())
  assert rc == 0
  assert packed == 10 * 4 * 1 * 2 * 2048  # quads of 32 cells x octets x groups of 4 layers x tiles of 32 units x 2 KB
  assert forward > 0 and backward > 0
  assert sizes(desc(dtype=N.F32))[1][0] == 3 * packed
  assert sizes(desc(n=0))[1] == [packed, 0, 0]


@pytest.mark.parametrize('kw,text', [
    (dict(dtype=N.I32), 'float32, float16 or bfloat16'), (dict(activation=5), 'activation'), (dict(activation=-1), 'activation'),
    (dict(cells=0), 'range'), (dict(n_layers=0), 'range'), (dict(n_layers=33), 'range'), (dict(hidden=0), 'range'),
    (dict(hidden=1 << 17), 'range'), (dict(n=-1), 'boards'), (dict(n=(1 << 31) + 1), 'boards'), (dict(row_stride=-1), 'stride'),
    (dict(cells=1 << 20, hidden=1 << 16), 'too large')])
def test_refused_descriptions(kw, text):
  rc, _ = sizes(desc(**kw))
  assert rc == N.E_INVALID and text in N.lib().pcx_last_error().decode()


def test_a_layer_twice_is_refused():
  d = desc()
  d.chars[2] = ord('P')
  rc, _ = sizes(d)
  assert rc == N.E_INVALID and 'twice' in N.lib().pcx_last_error().decode()
  d.stacked = 1  # (stacked layers have no characters)
  assert sizes(d)[0] == 0


def test_null_and_misaligned_pointers_are_refused_before_any_launch():
  lib, d, at = N.lib(), desc(), 1 << 20
  assert lib.pcx_project_sizes(None, None, None, None) == N.E_INVALID
  assert lib.pcx_project_pack(ctypes.byref(d), None, at, None) == N.E_INVALID
  assert lib.pcx_project_pack(ctypes.byref(d), at, at + 8, None) == N.E_INVALID
  big = 1 << 40
  assert lib.pcx_project_forward(ctypes.byref(d), None, at, None, None, at, None, at, big, None) == N.E_INVALID
  assert lib.pcx_project_forward(ctypes.byref(d), at, at, None, None, None, None, at, big, None) == N.E_INVALID
  assert lib.pcx_project_forward(ctypes.byref(d), at, at, at + 1, None, at, None, at, big, None) == N.E_INVALID
  assert lib.pcx_project_forward(ctypes.byref(d), at, at, None, None, at, None, at, 16, None) == N.E_INVALID  # too small a workspace
  assert lib.pcx_project_backward(ctypes.byref(d), at, None, None, at, at, at, big, None) == N.E_INVALID
  assert lib.pcx_project_backward(ctypes.byref(d), at, at, None, at, at, None, 0, None) == N.E_INVALID
  assert lib.pcx_project_backward(ctypes.byref(desc(activation=N.ACT_RELU)), at, at, None, at, at, at, big, None) == N.E_INVALID  # slopes
  assert lib.pcx_project_backward(ctypes.byref(desc(n=0)), at, at, None, at, at, at, big, None) == N.E_INVALID


def test_needs_a_gpu():
  if torch.cuda.is_available():
    pytest.skip('there is one')
  with pytest.raises(RuntimeError, match='PyTorch-ROCm'):
    rendering.ObservationProjection('P', torch.zeros(4, 1, 2, 2))
  with pytest.raises(RuntimeError, match='PyTorch-ROCm'):
    rendering.project(torch.zeros(1, 2, 2, dtype=torch.uint8), 'P', torch.zeros(4, 1, 2, 2))


# ---------------------------------------------------------------- on the GPU


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('stacked', [False, True])
def test_one_board(dtype, stacked):
  check(1, 8, 10, 30, 256, dtype, 'relu', 1, stacked=stacked, train=True)


@pytest.mark.gpu
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('dtype', DTYPES)
def test_types_and_activations(dtype, act):
  check(70, 5, 6, 12, 40, dtype, act, 2, train=True)


@pytest.mark.gpu
@pytest.mark.parametrize('stacked', [False, True])
@pytest.mark.parametrize('layers', [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 32])
def test_layers(layers, stacked):
  check(130, layers, 5, 7, 33, 'bfloat16', 'tanh', 3, stacked=stacked, train=True)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,cols', [(1, 1), (1, 3), (2, 2), (3, 5), (4, 4), (1, 31), (4, 8), (3, 11), (9, 7), (8, 8), (45, 89)])
def test_cells(rows, cols):
  for stacked in (False, True):
    check(37, 6, rows, cols, 24, 'float16', 'silu', 4, stacked=stacked, train=True)


@pytest.mark.gpu
@pytest.mark.parametrize('hidden', [1, 2, 31, 32, 33, 64, 65, 96, 128, 130, 200, 257, 512])
def test_hidden(hidden):
  for n in (3, 600):  # (both launch shapes)
    check(n, 4, 5, 8, hidden, 'bfloat16', 'gelu', 5, train=True)


@pytest.mark.gpu
@pytest.mark.parametrize('n', [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 511, 512, 513, 1025, 5000])
def test_boards(n):
  check(n, 5, 6, 12, 72, 'float32', 'relu', 6, train=True)


@pytest.mark.gpu
def test_no_bias_no_residual():
  check(50, 3, 4, 9, 36, 'float16', None, 7, with_bias=False, with_residual=False, train=True)
  check(50, 3, 4, 9, 36, 'float32', 'silu', 8, with_bias=True, with_residual=False, train=True)


@pytest.mark.gpu
def test_many_boards():
  check(40000, 8, 10, 30, 96, 'bfloat16', 'relu', 9, train=True)


@pytest.mark.gpu
def test_float32_weights_keep_all_their_bits():
  g = torch.Generator().manual_seed(10)
  weight = torch.randn(64, 2, 1, 1, generator=g) * torch.exp2(torch.randint(-100, 100, (64, 2, 1, 1), generator=g).float())
  boards = torch.tensor([ord('a'), ord('b'), ord('c')], dtype=torch.uint8).reshape(3, 1, 1)
  y = rendering.project(boards.cuda(), 'ab', weight.cuda()).cpu()
  assert torch.equal(y[0], weight[:, 0, 0, 0]) and torch.equal(y[1], weight[:, 1, 0, 0]) and not y[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_largest_smallest_and_no_numbers(dtype):
  """One feature a board: the weight itself comes back, whatever it is; what is not finite stays where it is set."""
  dt, info = getattr(torch, dtype), torch.finfo(getattr(torch, dtype))
  values = torch.tensor([info.max, -info.max, info.tiny, info.smallest_normal * info.eps, 0.0, 1.0], dtype=dt)
  y = rendering.project(torch.full((1, 1, 1), ord('a'), dtype=torch.uint8).cuda(), 'a', values.reshape(6, 1, 1, 1).cuda()).cpu()[0]
  assert torch.equal(y[:3], values[:3]) and torch.equal(y[4:], values[4:])
  assert abs(float(y[3]) - float(values[3])) <= float(values[3])  # the smallest subnormal: itself, or flushed to zero
  w = torch.tensor([math.inf, -math.inf, math.nan, 2.0], dtype=dt).reshape(4, 1, 1, 1)
  y = rendering.project(torch.full((1, 1, 1), ord('a'), dtype=torch.uint8).cuda(), 'a', w.cuda()).cpu()[0]
  assert y[0] == math.inf and y[1] == -math.inf and torch.isnan(y[2]) and y[3] == 2


@pytest.mark.gpu
def test_strided_boards_and_planes():
  chars, boards, weight, bias, _ = make(40, 6, 5, 9, 48, 'float32', 11)
  y, tol, _, _ = reference(chars, boards, weight, bias, 'relu', None)
  proj = rendering.ObservationProjection(chars, weight.cuda(), bias.cuda(), activation='relu')
  wide = torch.zeros(40, 3, 53, dtype=torch.uint8).cuda()  # boards inside larger rows, starting at odd addresses
  for shift in (0, 1, 2, 3, 5):
    wide.zero_()
    inside = wide[:, 1, shift:shift + 45].unflatten(1, (5, 9))
    inside.copy_(boards.cuda())
    near(proj(inside), y, tol, 'shift {}'.format(shift))
  near(proj(boards.cuda().flip(0)), y.flip(0), tol.flip(0), 'flipped')
  first = boards[:1].cuda().expand(7, 5, 9)  # one board seven times
  near(proj(first), y[:1].expand(7, -1), tol[:1].expand(7, -1), 'expanded')


@pytest.mark.gpu
def test_last_board_of_an_allocation():
  """The bytes behind the last board are not read: a board at the very end of its allocation, at every cell count."""
  for cells in range(1, 40):
    pool = torch.full((4096,), ord('#'), dtype=torch.uint8).cuda()
    board = pool[4096 - cells:].reshape(1, 1, cells)
    w = torch.randn(8, 1, 1, cells)
    near(rendering.project(board, '#', w.cuda()), w.double().flatten(1).sum(1)[None], (cells + 4) * 2.0 ** -23 * w.double().abs().flatten(1).sum(1)[None], cells)


@pytest.mark.gpu
def test_refusals():
  w, b = torch.zeros(16, 3, 4, 5).cuda(), torch.zeros(2, 4, 5, dtype=torch.uint8).cuda()
  ok = rendering.ObservationProjection('P#@', w)
  ok(b)
  for bad in (b.cpu(), b[0], b.reshape(2, 20), b.reshape(1, 2, 4, 5), b.transpose(1, 2)[:, :, :], torch.zeros(2, 4, 6, dtype=torch.uint8).cuda(),
              torch.zeros(2, 5, 4, dtype=torch.uint8).cuda(), torch.zeros(2, 4, 10, dtype=torch.uint8).cuda()[:, :, ::2]):
    with pytest.raises(ValueError):
      ok(bad)
  with pytest.raises(TypeError):
    ok(b.float())
  with pytest.raises(TypeError):
    ok(b.bool())  # (one layer's bools are no characters)
  with pytest.raises(TypeError):
    ok('a board')
  for residual in (torch.zeros(2, 15).cuda(), torch.zeros(3, 16).cuda(), torch.zeros(2, 16).half().cuda(), torch.zeros(2, 16)):
    with pytest.raises(ValueError):
      ok(b, residual=residual)
  for kw in (dict(layers='P#'), dict(layers='P##'), dict(layers='P#一'), dict(activation='swish'), dict(weight=w.cpu()), dict(weight=w[:0]),
             dict(weight=w.reshape(16, 3, 20)), dict(bias=torch.zeros(15).cuda()), dict(bias=torch.zeros(16).half().cuda())):
    args = dict(dict(layers='P#@', weight=w), **kw)
    with pytest.raises(ValueError):
      rendering.ObservationProjection(**args)
    with pytest.raises(ValueError):
      rendering.project(b, **args)
  with pytest.raises(TypeError):
    rendering.project(b, 'P#@', w.double())
  with pytest.raises(NotImplementedError):
    rendering.project(b, '', w)
  with pytest.raises(ValueError):
    ok.load(w.half())
  with pytest.raises(ValueError):
    ok.load(w, torch.zeros(16).cuda())


@pytest.mark.gpu
def test_flat_weight_load_and_same_numbers():
  chars, boards, weight, bias, residual = make(300, 7, 10, 30, 160, 'bfloat16', 12)
  b, w, c, r = boards.cuda(), weight.cuda(), bias.cuda(), residual.cuda()
  proj = rendering.ObservationProjection(chars, w, c, activation='silu')
  first = proj(b, residual=r)
  assert torch.equal(first, rendering.ObservationProjection(chars, w.flatten(1), c, activation='silu')(b, residual=r))
  assert torch.equal(first, rendering.project(b, chars, w, c, activation='silu', residual=r))
  assert torch.equal(first, rendering.project(b, chars, w, c, activation='silu', residual=r))  # sums in a fixed order
  proj.load(w * 2, c)
  assert torch.equal(proj(b, residual=r), rendering.project(b, chars, w * 2, c, activation='silu', residual=r))
  stacked = torch.stack([(b == ord(ch)) for ch in chars], 1)  # bool layers of the same boards
  y, tol, _, _ = reference(chars, boards, weight * 2, bias, 'silu', residual)
  near(proj(stacked, residual=r), y, tol, 'bool layers')
  proj.load(w, c)
  y, tol, _, _ = reference(chars, boards, weight, bias, 'silu', residual)
  near(proj(stacked, residual=r), y, tol, 'bool layers after load()')


@pytest.mark.gpu
@pytest.mark.parametrize('name,stacked', [('scrolly_maze_L0', False), ('marauders_unoccluded', True), ('warehouse_L0', False)])
def test_observations_of_an_engine(name, stacked):
  import os
  from pycolab_amd.compiler import GameTemplate
  from pycolab_amd.engine import Engine
  path = os.path.join(os.path.dirname(__file__), 'golden', 'templates', name + '.npz')
  for batch in (1, 96):
    eng = Engine.from_template(GameTemplate.load(path), batch=batch, auto_reset=True)
    obs, _, _ = eng.its_showtime()
    layers = 'P' + ''.join(sorted(obs.layers)[:3]).replace('P', '') + '\x7f'  # the last one does not exist in the game
    g = torch.Generator().manual_seed(13)
    weight = torch.randn(48, len(layers), eng.rows, eng.cols, generator=g)
    proj = rendering.ObservationProjection(layers, weight.cuda())
    for step in range(3):
      obs = eng.play(torch.full((batch,), step % 2, dtype=torch.int32).cuda() if batch > 1 else step % 2)[0]
      cells = [torch.as_tensor(np.asarray(obs.layers[c].cpu() if batch > 1 else obs.layers[c])) for c in layers if c in obs.layers]
      cells = torch.stack([x.reshape(batch, eng.rows, eng.cols) for x in cells] + [torch.zeros(batch, eng.rows, eng.cols)] * (len(layers) - len(cells)), 1)
      y, tol, _, _ = reference(layers, (cells != 0).to(torch.uint8), weight, None, None, None)
      got = proj(obs)
      assert got.shape == ((48,) if batch == 1 else (batch, 48))
      near(got.reshape(batch, 48), y, tol, '{} step {}'.format(name, step))
      assert torch.equal(got.reshape(batch, 48), rendering.project(obs, layers, weight.cuda()).reshape(batch, 48))
    with pytest.raises(RuntimeError, match='actual feature'):
      rendering.project(obs, '\x7f', weight[:, :1].contiguous().cuda())
    eng.close()


@pytest.mark.gpu
def test_cropped_and_repainted_observations():
  import os
  from pycolab_amd import cropping
  from pycolab_amd.compiler import GameTemplate
  from pycolab_amd.engine import Engine
  path = os.path.join(os.path.dirname(__file__), 'golden', 'templates', 'better_scrolly_maze_L0.npz')
  eng = Engine.from_template(GameTemplate.load(path), batch=33, auto_reset=True)
  obs, _, _ = eng.its_showtime()
  cropper = cropping.ScrollingCropper(rows=10, cols=30, to_track=['P'], scroll_margins=(2, 3))
  cropper.set_engine(eng)
  window = cropper.crop(obs)
  weight = torch.randn(64, 4, 10, 30, generator=torch.Generator().manual_seed(14))
  want = rendering.ObservationToFeatureArray('P#@a')(window).cpu()
  y, tol, _, _ = reference('P#@a', (want != 0).to(torch.uint8), weight, None, 'tanh', None)
  near(rendering.ObservationProjection('P#@a', weight.cuda(), activation='tanh')(window), y, tol, 'window')
  repainter = rendering.ObservationCharacterRepainter({'a': '@', 'b': '@', 'c': '@'})
  full = repainter(obs)
  weight = torch.randn(40, 2, 45, 89, generator=torch.Generator().manual_seed(15))
  want = rendering.ObservationToFeatureArray('P@')(full).cpu()
  y, tol, _, _ = reference('P@', (want != 0).to(torch.uint8), weight, None, None, None)
  near(rendering.project(full, 'P@', weight.cuda()), y, tol, 'repainted')
  eng.close()


@pytest.mark.gpu
def test_gradient_against_differences():
  """d/dt f(w + t v) at 0 against (f(w + h v) - f(w - h v)) / 2h in float64 of the formula, and of the kernels' own forward
  pass: with |v| such that z moves by at most 1 per unit of t, h = 2^-5 leaves h^2 / 6 |f'''| <= 2^-12 |g| sums."""
  chars, boards, weight, bias, _ = make(64, 4, 3, 5, 24, 'float32', 16)
  v = torch.randn(weight.shape, generator=torch.Generator().manual_seed(17)) / 15
  grad = torch.randn(64, 24, generator=torch.Generator().manual_seed(18))
  w = weight.cuda().requires_grad_()
  out = rendering.project(boards.cuda(), chars, w, bias.cuda(), activation='silu')
  dw, = torch.autograd.grad(out, [w], grad.cuda())
  slope = float((dw.cpu().double() * v.double()).sum())
  h = 2.0 ** -5

  def own(t):
    return rendering.project(boards.cuda(), chars, (weight + t * v).cuda(), bias.cuda(), activation='silu').cpu().double()

  x = features(chars, boards)
  dz = (x @ v.double().flatten(1).t()).abs()
  bound = h * h / 6 * 1.0 * float((grad.double().abs() * dz ** 3).sum()) + 1e-5 * float(grad.abs().sum())
  for f in (own, lambda t: act64('silu', x @ (weight.double() + t * v.double()).flatten(1).t() + bias.double())[0]):
    difference = float((grad.double() * (f(h) - f(-h))).sum()) / (2 * h)
    assert abs(difference - slope) <= bound, (difference, slope, bound)
  assert bound < 0.05 * float((grad.double().abs() * dz).sum())  # (the bound says something)


@pytest.mark.gpu
def test_only_what_is_asked_for():
  chars, boards, weight, bias, residual = make(20, 3, 4, 4, 16, 'float32', 19)
  b = boards.cuda()
  for which in ((0,), (1,), (2,), (0, 2)):
    t = [weight.cuda(), bias.cuda(), residual.cuda()]
    for i in which:
      t[i].requires_grad_()
    out = rendering.project(b, chars, t[0], t[1], activation='tanh', residual=t[2])
    out.sum().backward()
    assert [x.grad is not None for x in t] == [i in which for i in range(3)]
  with torch.no_grad():
    assert not rendering.project(b, chars, t[0], t[1]).requires_grad
  shared = weight.cuda().requires_grad_()  # the same weight twice: its gradients add up
  g1, = torch.autograd.grad(rendering.project(b, chars, shared).sum(), shared)
  g2, = torch.autograd.grad(rendering.project(b, chars, shared).sum() + rendering.project(b, chars, shared).sum(), shared)
  assert torch.equal(g2, 2 * g1)
  half = torch.randn(20, 16).cuda()
  out = rendering.project(b, chars, shared)
  assert torch.equal(torch.autograd.grad(out, shared, half[:, :1].expand(20, 16), retain_graph=True)[0],
                     torch.autograd.grad(out, shared, half[:, :1].expand(20, 16).contiguous())[0])  # a broadcast gradient
  out = rendering.project(b, chars, shared)
  b.zero_()
  with pytest.raises(RuntimeError, match='modified by an inplace operation'):
    out.sum().backward()


@pytest.mark.gpu
def test_other_streams_and_graphs():
  chars, boards, weight, bias, residual = make(700, 8, 10, 30, 96, 'bfloat16', 20)
  b, w, c, r = boards.cuda(), weight.cuda(), bias.cuda(), residual.cuda()
  proj = rendering.ObservationProjection(chars, w, c, activation='relu')
  want = proj(b, residual=r)
  grad = torch.randn(700, 96).to(torch.bfloat16).cuda()
  y, slope = rendering.project(b, chars, w, c, activation='relu', residual=r, return_slope=True)
  dw, db = rendering.project_backward(b, chars, w, grad, slope)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    other = proj(b, residual=r)
  torch.cuda.current_stream().wait_stream(side)
  assert torch.equal(other, want)
  ones = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
  torch.cuda.synchronize()
  with torch.cuda.graph(ones[0]):
    first = proj(b, residual=r)
  with torch.cuda.graph(ones[1]):
    second, sl = rendering.project(b, chars, w, c, activation='relu', residual=r, return_slope=True)
    gw, gb = rendering.project_backward(b, chars, w, grad, sl)
  for i in range(4):
    b.copy_(boards.cuda().roll(i, 0))
    expect = proj(b, residual=r)
    ones[0].replay()
    ones[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(first, expect) and torch.equal(second, expect)
    _, s2 = rendering.project(b, chars, w, c, activation='relu', residual=r, return_slope=True)
    e2 = rendering.project_backward(b, chars, w, grad, s2)
    assert torch.equal(gw, e2[0]) and torch.equal(gb, e2[1])
  b.copy_(boards)
  proj.load(w * 2, c)
  ones[0].replay()
  assert torch.equal(first, proj(b, residual=r))
  leaf = w.clone().requires_grad_()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with pytest.raises(RuntimeError, match='project_backward'):
    with torch.cuda.graph(graph):
      rendering.project(b, chars, leaf, c)
  torch.cuda.synchronize()
  assert torch.equal(rendering.project_backward(boards.cuda(), chars, w, grad, slope)[0], dw) and db.shape == (96,)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_relu_stops_infinite_gradients(dtype):
  """Where relu is shut nothing comes through, whatever the gradient is; a sum that is no number is not shut."""
  for n, hidden in ((65, 16), (64, 13)):
    chars, boards, weight, bias, _ = make(n, 3, 5, 7, hidden, dtype, 21)
    bias[0], bias[1] = -1e4, float('nan')
    w, c = weight.cuda().requires_grad_(), bias.cuda().requires_grad_()
    out = rendering.project(boards.cuda(), chars, w, c, activation='relu')
    grad = torch.ones(n, hidden, dtype=w.dtype, device='cuda')
    grad[:, 0] = float('inf')
    out.backward(grad)
    assert not out[:, 0].any() and out[:, 1].isnan().all()
    assert not c.grad[0].any() and not w.grad[0].any()
    assert float(c.grad[1]) == n  # (whole numbers: exact)


@pytest.mark.gpu
def test_backward_after_the_observation_is_gone_is_refused():
  import os
  from pycolab_amd import cropping
  from pycolab_amd.compiler import GameTemplate
  from pycolab_amd.engine import Engine
  path = os.path.join(os.path.dirname(__file__), 'golden', 'templates', 'better_scrolly_maze_L0.npz')
  eng = Engine.from_template(GameTemplate.load(path), batch=9, auto_reset=True)
  obs, _, _ = eng.its_showtime()
  cropper = cropping.ScrollingCropper(rows=10, cols=30, to_track=['P'], scroll_margins=(2, 3))
  cropper.set_engine(eng)
  repainter = rendering.ObservationCharacterRepainter({'a': '@', 'b': '@', 'c': '@'})
  sources = lambda obs: (obs, cropper.crop(obs), repainter(obs), repainter(cropper.crop(obs)))
  shapes = ((45, 89), (10, 30), (45, 89), (10, 30))
  weights = [torch.randn(8, 2, r, c, device='cuda').requires_grad_() for r, c in shapes]
  for w, s in zip(weights, sources(obs)):  # in time
    rendering.project(s, 'P@', w).sum().backward()
    assert w.grad.abs().sum() > 0
  late = [rendering.project(s, 'P@', w) for w, s in zip(weights, sources(obs))]
  kept = rendering.project(obs.board.clone(), 'P@', weights[0])
  residual = torch.zeros(9, 8, device='cuda', requires_grad=True)
  only_residual = rendering.project(obs, 'P@', weights[0].detach(), residual=residual)
  eng.play(torch.zeros(9, dtype=torch.int32).cuda())
  for out in late:
    with pytest.raises(RuntimeError, match='overwritten by a later step'):
      out.sum().backward()
  kept.sum().backward()
  only_residual.sum().backward()
  assert (residual.grad == 1).all()
  out = rendering.project(eng.play(torch.zeros(9, dtype=torch.int32).cuda())[0], 'P@', weights[0])
  eng.close()
  with pytest.raises(RuntimeError, match='engine closed'):
    out.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('act', ACTS)
def test_the_explicit_pair(act, dtype):
  """project(return_slope=True) and project_backward(): the formula's gradients and autograd's own, whether or not the
  activation is named again."""
  for stacked in (False, True):
    chars, boards, weight, bias, residual = make(130, 5, 5, 7, 40, dtype, 30, stacked, grid=act == 'relu')
    y, tol, slope64, slope_tol = reference(chars, boards, weight, bias, act, residual)
    b, w, c, r = (t.cuda() for t in (boards, weight, bias, residual))
    grad = torch.randn(130, 40, generator=torch.Generator().manual_seed(31)).to(weight.dtype)
    out, slope = rendering.project(b, chars, w, c, activation=act, residual=r, return_slope=True)
    near(out, y, tol, 'forward')
    assert (slope is None) == (act is None)
    leaves = [w.clone().requires_grad_(), c.clone().requires_grad_()]
    auto = torch.autograd.grad(rendering.project(b, chars, *leaves, activation=act, residual=r), leaves, grad.cuda())
    for named in (dict(), dict(activation=act)):
      dw, db = rendering.project_backward(b, chars, w, grad.cuda(), slope, **named)
      check_grads(chars, boards, weight, grad, slope64, slope_tol, dw, db)
      assert torch.equal(dw, auto[0]) and torch.equal(db, auto[1])


def small_engine(batch, name='better_scrolly_maze_L0'):
  import os
  from pycolab_amd.compiler import GameTemplate
  from pycolab_amd.engine import Engine
  return Engine.from_template(GameTemplate.load(os.path.join(os.path.dirname(__file__), 'golden', 'templates', name + '.npz')), batch=batch, auto_reset=True)


@pytest.mark.gpu
def test_the_explicit_pair_of_one_observation():
  """A batch-1 Observation: the result is [hidden], and so may its gradient be."""
  eng = small_engine(1, 'scrolly_maze_L0')
  obs, _, _ = eng.its_showtime()
  w = torch.randn(24, 2, 10, 30, generator=torch.Generator().manual_seed(32)).cuda()
  out, slope = rendering.project(obs, 'P#', w, activation='tanh', return_slope=True)
  grad = torch.randn(24, generator=torch.Generator().manual_seed(33)).cuda()
  assert out.shape == grad.shape
  leaf = w.clone().requires_grad_()
  want, = torch.autograd.grad(rendering.project(obs, 'P#', leaf, activation='tanh'), leaf, grad)
  for g in (grad, grad[None]):
    assert torch.equal(rendering.project_backward(obs, 'P#', w, g, slope, activation='tanh')[0], want)
  with pytest.raises(ValueError):
    rendering.project_backward(obs, 'P#', w, grad[:23], slope)
  with pytest.raises(ValueError, match='slopes'):
    rendering.project_backward(obs, 'P#', w, grad, activation='tanh')
  eng.close()


@pytest.mark.gpu
def test_backward_after_import_state():
  """A checkpoint with its observation rewrites the planes, one without leaves them."""
  from pycolab_amd import cropping
  eng = small_engine(9)
  obs, _, _ = eng.its_showtime()
  cropper = cropping.ScrollingCropper(rows=10, cols=30, to_track=['P'], scroll_margins=(2, 3))
  cropper.set_engine(eng)
  cropper.crop(obs)
  with_planes, without = eng.export_state(with_observation=True), eng.export_state()
  obs = eng.play(torch.zeros(9, dtype=torch.int32).cuda())[0]
  big, small = (torch.randn(8, 2, r, c, device='cuda').requires_grad_() for r, c in ((45, 89), (10, 30)))
  out = rendering.project(obs, 'P@', big).sum()
  eng.import_state(without)
  torch.autograd.grad(out, big, retain_graph=True)
  window = rendering.project(cropper.crop(obs), 'P@', small).sum()
  eng.import_state(with_planes)
  for late, weight in ((out, big), (window, small)):
    with pytest.raises(RuntimeError, match='overwritten'):
      torch.autograd.grad(late, weight)
  eng.close()


@pytest.mark.gpu
def test_backward_after_a_cropper_let_go_of_its_window_is_refused():
  from pycolab_amd import cropping
  eng, other = small_engine(1), small_engine(1)
  small = torch.randn(8, 2, 10, 30, device='cuda').requires_grad_()
  obs, _, _ = eng.its_showtime()
  other.its_showtime()
  cropper = cropping.ScrollingCropper(rows=10, cols=30, to_track=['P'], scroll_margins=(2, 3))
  cropper.set_engine(eng)
  out = rendering.project(cropper.crop(obs), 'P@', small).sum()
  cropper.set_engine(other)
  with pytest.raises(RuntimeError, match='overwritten'):
    torch.autograd.grad(out, small)
  eng.close()
  other.close()


@pytest.mark.gpu
def test_backward_after_a_view_of_the_planes_was_overwritten_is_refused():
  """The kernels write an engine's, a cropper's, a repainter's and a converter's arrays where autograd does not see it: a
  backward pass over a tensor that lies in one of them is refused once it was written again."""
  from pycolab_amd import cropping
  eng = small_engine(9)
  obs, _, _ = eng.its_showtime()
  cropper = cropping.ScrollingCropper(rows=10, cols=30, to_track=['P'], scroll_margins=(2, 3))
  cropper.set_engine(eng)
  repainter = rendering.ObservationCharacterRepainter({'a': '@', 'b': '@', 'c': '@'})
  converter = rendering.ObservationToArray({c: ord(c) for c in obs.layers}, dtype=np.uint8)
  still = torch.zeros(9, dtype=torch.int32).cuda()
  big, small = (torch.randn(8, 2, r, c, device='cuda').requires_grad_() for r, c in ((45, 89), (10, 30)))
  run = lambda t, w: rendering.project(t, 'P@', w).sum()

  def written(make_tensor, weight, again):
    """make_tensor() -> a view; again() -> writes what it shows."""
    out = run(make_tensor(), weight)
    grad, = torch.autograd.grad(out, weight)  # in time
    assert grad.abs().sum() > 0
    out, copy = run(make_tensor(), weight), run(make_tensor().clone(), weight)
    again()
    torch.autograd.grad(copy, weight)
    with pytest.raises(RuntimeError, match='overwritten'):
      torch.autograd.grad(out, weight)

  for view in (lambda: obs.board, lambda: obs.board[2:7], lambda: eng.planes_view()[:, 0], lambda: eng.planes_view()[:, 1:3]):
    for again in (lambda: eng.step(still), lambda: eng.step_n(still[None]), lambda: eng.step_hashed(1, 0, 2), lambda: eng.reset()):
      written(view, big, again)
  written(lambda: cropper.crop(obs).board, small, lambda: cropper.crop(obs))
  window = cropper.crop(obs).board
  out = run(window, small)
  eng.step(still)  # (the window is written by crop() alone)
  torch.autograd.grad(out, small)
  written(lambda: repainter(obs).board, big, lambda: repainter(obs))
  written(lambda: converter(obs), big, lambda: converter(obs))
  out = run(obs.board, big)
  eng.close()  # (nobody writes the tensor any more)
  torch.autograd.grad(out, big)


@pytest.mark.gpu
def test_backward_after_what_a_step_writes_besides_its_planes_is_refused():
  """Fused croppers' windows and a fused converter's array are written by the step itself."""
  from pycolab_amd import cropping
  still = torch.zeros(9, dtype=torch.int32).cuda()
  small = torch.randn(8, 2, 10, 30, device='cuda').requires_grad_()
  eng = small_engine(9)
  obs, _, _ = eng.its_showtime()
  cropper = cropping.ScrollingCropper(rows=10, cols=30, to_track=['P'], scroll_margins=(2, 3))
  assert cropping.fuse_croppers(eng, [cropper])
  obs = eng.play(still)[0]
  out = rendering.project(cropper.crop(obs).board, 'P@', small).sum()
  eng.step(still)
  with pytest.raises(RuntimeError, match='overwritten'):
    torch.autograd.grad(out, small)
  eng.close()
  eng = small_engine(9, 'scrolly_maze_L0')
  obs, _, _ = eng.its_showtime()
  converter = rendering.ObservationToArray({c: ord(c) for c in obs.layers}, dtype=np.uint8)
  assert converter.fuse_into(eng, force=True)
  obs = eng.play(still)[0]
  out = rendering.project(converter(obs), 'P@', small).sum()
  eng.step(still)
  with pytest.raises(RuntimeError, match='overwritten'):
    torch.autograd.grad(out, small)
  converter.unfuse()
  eng.close()


@pytest.mark.gpu
def test_backward_over_a_view_after_import_state():
  eng = small_engine(9)
  obs, _, _ = eng.its_showtime()
  with_planes, without = eng.export_state(with_observation=True), eng.export_state()
  obs = eng.play(torch.zeros(9, dtype=torch.int32).cuda())[0]
  big = torch.randn(8, 2, 45, 89, device='cuda').requires_grad_()
  out = rendering.project(obs.board, 'P@', big).sum()
  eng.import_state(without)
  torch.autograd.grad(out, big, retain_graph=True)
  eng.import_state(with_planes)
  with pytest.raises(RuntimeError, match='overwritten'):
    torch.autograd.grad(out, big)
  eng.close()


@pytest.mark.gpu
def test_forward_mode_and_function_transforms_are_refused():
  chars, boards, weight, bias, residual = make(6, 3, 4, 5, 16, 'float32', 50)
  b, given = boards.cuda(), [t.cuda() for t in (weight, bias, residual)]
  for i in range(3):
    with torch.autograd.forward_ad.dual_level():
      args = list(given)
      args[i] = torch.autograd.forward_ad.make_dual(args[i], torch.ones_like(args[i]))
      with pytest.raises(RuntimeError, match='forward'):
        rendering.project(b, chars, args[0], args[1], residual=args[2])
      rendering.project(b, chars, given[0], given[1], residual=given[2])  # (no tangent)
  f = lambda w: rendering.project(b, chars, w, given[1])
  for transform in (lambda: torch.func.jvp(f, (given[0],), (given[0],)), lambda: torch.func.grad(lambda w: f(w).sum())(given[0]),
                    lambda: torch.func.vmap(f)(torch.stack([given[0]] * 2)), lambda: torch.func.vjp(f, given[0])):
    with pytest.raises(RuntimeError):
      transform()


# Boards and hidden units that reach every instance of the product's kernel (a wave's tiles of boards x hidden units, the
# workgroup's waves along them, and whether the cells are divided: a plan without a workspace is undivided).  450 units are 15
# tiles, 50 are two; 35 cells are two quads.
TILES = [(300, 450, True),     # 1 x 1, one wave x four
         (700, 450, True),     # 2 x 2, two waves x two
         (700, 50, True),      # 2 x 2, four waves x one
         (16300, 450, True),   # 4 x 2, two waves x two: 64 x 4 workgroups of 256 boards
         (16500, 450, False),  # ... 65 x 4
         (24700, 450, False),  # 4 x 2, four waves x two: 98,304 boards of four tiles each and more
         (130600, 50, True),   # 4 x 2, four waves x one: 256 workgroups of 512 boards
         (131200, 50, False)]  # ... 257
STACKED_TILES = [(700, 450, True), (5000, 450, False), (700, 50, True), (33000, 50, False)]  # 1 x 2, four waves x two and x one


def check_on_device(n, layers, rows, cols, hidden, dtype, act, seed, stacked=False, divided=None, train=True):
  """As check(), with the formulas in 64 bits on the device."""
  chars, boards, weight, bias, residual = make(n, layers, rows, cols, hidden, dtype, seed, stacked, grid=act == 'relu')
  if divided is not None:
    d = desc(n=n, row_stride=boards[0].numel(), cells=rows * cols, n_layers=layers, hidden=hidden, stacked=int(stacked),
             dtype={'float32': N.F32, 'float16': N.F16, 'bfloat16': N.BF16}[dtype])
    for i, c in enumerate(chars):
      d.chars[i] = ord(c)
    assert (sizes(d)[1][1] > 0) == divided
  boards, weight, bias, residual = (t.cuda() for t in (boards, weight, bias, residual))
  y, tol, slope64, slope_tol = reference(chars, boards, weight, bias, act, residual)
  got = rendering.ObservationProjection(chars, weight, bias, activation=act)(boards, residual=residual)
  near(got, y.cpu(), tol.cpu(), 'forward')
  out, slope = rendering.project(boards, chars, weight, bias, activation=act, residual=residual, return_slope=True)
  assert torch.equal(out, got)
  if slope is not None:
    # (besides: silu's 1 - s is off by some 2 * 2^-24, which |z|, here below 10, multiplies)
    near(slope, slope64.cpu(), (slope_tol + 24 * 2.0 ** -24).expand_as(slope64).cpu(), 'slope')
  if not train:
    return
  grad = torch.randn(n, hidden, generator=torch.Generator().manual_seed(seed + 1)).to(weight.dtype).cuda()
  dw, db = rendering.project_backward(boards, chars, weight, grad, slope, activation=act)
  x, eps, tiny = features(chars, boards), torch.finfo(weight.dtype).eps, torch.finfo(weight.dtype).tiny
  dz = grad.double() * slope64
  off = grad.double().abs() * slope_tol + eps * (dz.abs() + grad.double().abs() * slope_tol) + tiny * eps
  for g, left, what in ((dw.flatten(1), x, 'grad weight'), (db[:, None], torch.ones(n, 1, dtype=torch.float64, device='cuda'), 'grad bias')):
    want = dz.t() @ left
    tol = off.t() @ left + (n + 2) * 2.0 ** -23 * (dz.abs().t() @ left)
    near(g, want.cpu(), (tol + eps / 2 * (want.abs() + tol) + tiny * eps).cpu(), what)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('layers,act', [(3, 'silu'), (8, 'relu'), (11, 'tanh'), (16, 'gelu'), (20, None)])
@pytest.mark.parametrize('n,hidden,divided', TILES)
def test_every_tile_shape(n, hidden, divided, layers, act, dtype):
  check_on_device(n, layers, 5, 7, hidden, dtype, act, 40, divided=divided)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('n,hidden,divided', STACKED_TILES)
def test_every_tile_shape_of_stacked_layers(n, hidden, divided, dtype):
  for layers, act in ((1, 'gelu'), (7, 'relu'), (8, 'tanh'), (11, None), (12, 'silu')):
    check_on_device(n, layers, 5, 7, hidden, dtype, act, 41, stacked=True, divided=divided)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,n,layers,rows,cols,hidden', [('float32', 2048, 7, 45, 89, 200), ('bfloat16', 8192, 14, 16, 30, 512)])
def test_weights_beyond_the_cache(dtype, n, layers, rows, cols, hidden):
  """50 GB and more of boards times the weight's bytes: eight waves, the cells divided."""
  check_on_device(n, layers, rows, cols, hidden, dtype, 'gelu', 42, divided=True)


@pytest.mark.gpu
def test_a_projection_dropped_while_another_stream_uses_it():
  """Its laid-out weight must not become another tensor's memory before that stream has read it."""
  chars, boards, weight, bias, residual = make(700, 8, 10, 30, 96, 'bfloat16', 51)
  b, r = boards.cuda(), residual.cuda()
  for stacked in (False, True):
    x = torch.stack([(b == ord(c)) for c in chars], 1) if stacked else b
    want = rendering.project(x, chars, weight.cuda(), bias.cuda(), activation='tanh', residual=r)
    proj = rendering.ObservationProjection(chars, weight.cuda(), bias.cuda(), activation='tanh')
    proj(x)
    side, busy = torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
      torch.cuda._sleep(200_000_000)  # (some tens of milliseconds and more)
      got = proj(x, residual=r)
      busy.record()
    held = [(t.data_ptr(), t.numel() * t.element_size()) for t in (proj._packs[int(stacked)], proj._bias)]  # (what that call reads)
    del proj
    taken = [torch.empty(size, dtype=torch.uint8, device='cuda').fill_(255) for _, size in held for _ in range(3)]
    assert not busy.query(), 'the other stream was through too early to tell'
    for ptr, size in held:
      assert not any(t.data_ptr() < ptr + size and ptr < t.data_ptr() + t.numel() for t in taken)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('stacked', [False, True])
@pytest.mark.parametrize('dtype', DTYPES)
def test_gradients_whose_saved_tensors_went_elsewhere(dtype, stacked, act):
  """What autograd saved comes back laid out in its own way: copies on the host, a forward pass made anew."""
  from torch.utils.checkpoint import checkpoint
  n = 70
  chars, boards, weight, bias, residual = make(n, 6, 5, 9, 40, dtype, 61, stacked)
  many = torch.zeros((n, 3) + tuple(boards.shape[1:]), dtype=torch.uint8)  # the boards lie apart
  many[:, 1] = boards
  many, given, grad = many.cuda(), [t.cuda() for t in (weight, bias, residual)], torch.randn(n, 40, generator=torch.Generator().manual_seed(2)).to(weight.dtype).cuda()
  out, slope = rendering.project(boards.cuda(), chars, given[0], given[1], activation=act, residual=given[2], return_slope=True)
  want = rendering.project_backward(boards.cuda(), chars, given[0], grad, slope, activation=act) + (grad,)

  def on_the_host(f, *leaves):
    with torch.autograd.graph.save_on_cpu():
      return f(*leaves)

  for run, later in ((lambda f, *leaves: f(*leaves), False), (on_the_host, False), (on_the_host, True),
                     (lambda f, *leaves: checkpoint(f, *leaves, use_reentrant=False), False),
                     (lambda f, *leaves: checkpoint(f, *leaves, use_reentrant=True), False)):
    held = many.clone()
    leaves = [t.clone().requires_grad_() for t in given]
    y = run(lambda w, b, r: rendering.project(held[:, 1], chars, w, b, activation=act, residual=r), *leaves)
    assert torch.equal(y, out)
    if later:  # (the copy on the host is of the boards as they were)
      held.zero_()
    y.backward(grad)
    assert all(torch.equal(leaf.grad, w) for leaf, w in zip(leaves, want))


@pytest.mark.gpu
def test_a_frozen_weight_leaves_the_boards_free():
  """The gradients of bias and residual read no boards: those may be written again before."""
  chars, boards, weight, bias, residual = make(40, 5, 4, 8, 24, 'float32', 62)
  b, w, grad = boards.cuda(), weight.cuda(), torch.ones(40, 24).cuda()
  _, slope = rendering.project(b, chars, w, bias.cuda(), activation='tanh', return_slope=True)
  want = rendering.project_backward(b, chars, w, grad, slope, activation='tanh')[1]
  leaves = [bias.cuda().requires_grad_(), residual.cuda().requires_grad_()]
  y = rendering.project(b, chars, w, leaves[0], activation='tanh', residual=leaves[1])
  b.zero_()
  y.backward(grad)
  assert torch.equal(leaves[0].grad, want) and torch.equal(leaves[1].grad, grad)


@pytest.mark.gpu
def test_a_projection_made_in_inference_mode_takes_new_values():
  chars, boards, weight, bias, _ = make(40, 5, 4, 8, 24, 'bfloat16', 63)
  b, w, c = boards.cuda(), weight.cuda(), bias.cuda()
  with torch.inference_mode():
    proj = rendering.ObservationProjection(chars, -w, -c, activation='silu')
    proj(b)
  leaf = w.clone().requires_grad_()
  proj.load(leaf, c)
  want = rendering.project(b, chars, w, c, activation='silu')
  assert torch.equal(proj(b), want)
  other = rendering.ObservationProjection(chars, -w, -c, activation='silu')
  with torch.inference_mode():
    other.load(w, c)
    assert torch.equal(other(b), want)
  assert leaf._version == 0 and torch.equal(other(b), want)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('n,hidden', [(70, 64), (3000, 48), (70, 19)])
def test_arrays_at_any_element(n, hidden, dtype):
  """Bias, residual, gradient and slopes that begin in the middle of a word or of four elements: the same numbers."""
  chars, boards, weight, bias, residual = make(n, 6, 7, 9, hidden, dtype, 64)
  b, w = boards.cuda(), weight.cuda()

  def moved(t, by):  # the same numbers `by` elements into an allocation
    held = torch.empty(t.numel() + 8, dtype=t.dtype, device='cuda')[by:by + t.numel()].view(t.shape)
    return held.copy_(t)

  grad = torch.randn(n, hidden, generator=torch.Generator().manual_seed(3)).to(weight.dtype)
  shifted = torch.empty(b.numel() + 8, dtype=torch.uint8, device='cuda')
  for act in ('relu', 'gelu'):
    want, slope = rendering.project(b, chars, w, bias.cuda(), activation=act, residual=residual.cuda(), return_slope=True)
    grads = rendering.project_backward(b, chars, w, grad.cuda(), slope, activation=act)
    for by in (1, 2, 3):
      at = shifted[by:by + b.numel()].view(b.shape).copy_(b)
      out, k = rendering.project(at, chars, moved(weight, by), moved(bias, by), activation=act, residual=moved(residual, by), return_slope=True)
      assert torch.equal(out, want) and torch.equal(k, slope)
      got = rendering.project_backward(at, chars, w, moved(grad, by), moved(slope, by), activation=act)
      assert torch.equal(got[0], grads[0]) and torch.equal(got[1], grads[1])


@pytest.mark.gpu
@pytest.mark.parametrize('rows,cols,hidden,dtype,act,stacked', [(3, 4, 1056, 'bfloat16', 'relu', False), (3, 4, 1056, 'bfloat16', 'relu', True),
                                                                (42, 50, 8, 'float16', None, False), (42, 17, 8, 'float16', None, True)])
def test_offsets_beyond_31_bits(rows, cols, hidden, dtype, act, stacked):
  """Results of 2^31 elements and more, boards of 2^32 bytes and more.  All numbers are small multiples of 1/16 and all sums
  of them exact, so the last boards give what they give by themselves, and the gradients are whole numbers."""
  n, layers = (1 << 21) + 5, 3
  g = torch.Generator(device='cuda').manual_seed(rows)
  chars, cells = ' !"', rows * cols
  if stacked:
    boards = torch.randint(0, 2, (n, layers, rows, cols), generator=g, device='cuda', dtype=torch.uint8)
  else:
    boards = torch.randint(32, 36, (n, rows, cols), generator=g, device='cuda', dtype=torch.uint8)
  assert n * hidden >= 1 << 31 or boards.numel() >= 1 << 32
  dt = getattr(torch, dtype)
  weight = (torch.randint(-8, 9, (hidden, layers, rows, cols), generator=g, device='cuda').float() / 16).to(dt)
  bias = (torch.randint(-8, 9, (hidden,), generator=g, device='cuda').float() / 16).to(dt)
  out, slope = rendering.project(boards, chars, weight, bias, activation=act, return_slope=True)
  for part in (slice(0, 40), slice(n // 2, n // 2 + 40), slice(n - 40, n)):
    want, want_slope = rendering.project(boards[part], chars, weight, bias, activation=act, return_slope=True)
    assert torch.equal(out[part], want)
    assert slope is None or torch.equal(slope[part], want_slope)
  grad = torch.randint(-1, 2, (n, hidden), generator=g, device='cuda', dtype=torch.int8).to(dt)
  dw, db = rendering.project_backward(boards, chars, weight, grad, slope, activation=act)
  want, want_b = torch.zeros(hidden, layers * cells, dtype=torch.float64, device='cuda'), torch.zeros(hidden, dtype=torch.float64, device='cuda')
  for lo in range(0, n, 1 << 16):
    part = boards[lo:lo + (1 << 16)]
    x = part.flatten(1) if stacked else torch.stack([part == ord(c) for c in chars], 1).flatten(1)
    dz = grad[lo:lo + (1 << 16)].double()
    if slope is not None:
      dz = dz * slope[lo:lo + (1 << 16)]
    want += dz.t().contiguous() @ x.double()
    want_b += dz.sum(0)
  assert torch.equal(dw.flatten(1), want.to(dt)) and torch.equal(db, want_b.to(dt))


@pytest.mark.gpu
@pytest.mark.parametrize('stacked', [False, True])
@pytest.mark.parametrize('n,layers,rows,cols,hidden,dtype', [(5, 2, 1024, 1024, 3, 'bfloat16'), (700, 1, 512, 1024, 2, 'float16'), (3, 32, 100, 101, 5, 'float32'),
                                                             (70, 3, 2, 2, 1 << 16, 'float16'), (600, 2, 1, 1, 1 << 16, 'float32')])
def test_the_largest_boards_and_layers(n, layers, rows, cols, hidden, dtype, stacked):
  """A million cells a board, 65,536 units, 32 layers.  Small multiples of 1/16: all sums are exact."""
  chars, boards, weight, bias, residual = make(n, layers, rows, cols, hidden, dtype, 65, stacked, grid=True)
  b, w, c = boards.cuda(), weight.cuda(), bias.cuda()
  grad = torch.randint(-1, 2, (n, hidden), generator=torch.Generator().manual_seed(4)).to(weight.dtype).cuda()
  x = features(chars, b).float()  # (as are float32's products and sums of these numbers)
  want = x @ w.flatten(1).float().t().contiguous() + c.float()
  got = rendering.project(b, chars, w, c)
  assert torch.equal(got, want.to(w.dtype))
  dw, db = rendering.project_backward(b, chars, w, grad)
  assert torch.equal(dw.flatten(1), (grad.float().t().contiguous() @ x).to(w.dtype))
  assert torch.equal(db, grad.float().sum(0).to(w.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('stacked', [False, True])
def test_boards_that_a_rollout_in_inference_mode_left(stacked):
  chars, boards, weight, bias, _ = make(50, 5, 6, 7, 40, 'float32', 67, stacked)
  b, grad = boards.cuda(), torch.randn(50, 40, generator=torch.Generator().manual_seed(6)).cuda()
  with torch.inference_mode():
    kept = torch.stack([b, b], 1)[:, 1]
  assert kept.is_inference() and not kept.is_contiguous()
  grads = []
  for given in (b, kept):
    leaves = [weight.cuda().requires_grad_(), bias.cuda().requires_grad_()]
    grads.append(torch.autograd.grad(rendering.project(given, chars, *leaves, activation='tanh'), leaves, grad))
  assert all(torch.equal(p, q) for p, q in zip(*grads))
  frozen = bias.cuda().requires_grad_()
  only, = torch.autograd.grad(rendering.project(kept, chars, weight.cuda(), frozen, activation='tanh'), frozen, grad)
  assert torch.equal(only, grads[0][1])


@pytest.mark.gpu
def test_an_engine_stepped_in_inference_mode():
  eng = small_engine(9)
  with torch.inference_mode():
    obs, _, _ = eng.its_showtime()
    board = obs.board
  big = torch.randn(8, 2, 45, 89, generator=torch.Generator().manual_seed(7)).cuda().requires_grad_()
  want, = torch.autograd.grad(rendering.project(obs.board.clone(), 'P@', big).sum(), big)
  for boards in (board, obs):
    out = rendering.project(boards, 'P@', big).sum()
    got, = torch.autograd.grad(out, big)
    assert torch.equal(got, want)
  out, late = rendering.project(board, 'P@', big).sum(), rendering.project(obs, 'P@', big).sum()
  eng.step(torch.zeros(9, dtype=torch.int32).cuda())
  assert torch.equal(torch.autograd.grad(out, big)[0], want)  # (of a copy)
  with pytest.raises(RuntimeError, match='overwritten'):
    torch.autograd.grad(late, big)
  eng.close()
