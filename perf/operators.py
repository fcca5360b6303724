"""What the policy operators next to the engine are measured on.

Three operators sit between the engine's observations and its actions:

  project   act(features . weight^T + bias) + residual, with features the layers an
            ObservationToFeatureArray would stack -- read from the boards' characters
            (or from stacked uint8 layers, where layers overlap) -- and its backward pass
  sample    one action per environment from logits, by temperature, top-k, top-p and
            min-p, legal actions only, from one given uniform number per row
  log_prob  log-probability of the taken actions and the policy's entropy, and the
            gradient with respect to the logits

`run` computes them in elementary torch operations while `own` is false, and with the
calls a user makes of the package while it is true.
"""

import math

import torch

own = False

_DTYPES = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}
_SIZE = {'float32': 4, 'float16': 2, 'bfloat16': 2}
_CHARS = ' #.@Pabcdefghijklmnopqrstuvwxyz0'


def _project(name, n, rows, cols, layers, hidden, dtype, activation, residual=False, train=False, stacked=False):
  return dict(name=name, op='project', n=n, rows=rows, cols=cols, layers=layers, hidden=hidden, dtype=dtype,
              activation=activation, residual=residual, train=train, stacked=stacked)


def _sample(name, n, actions, dtype, legal=False, per_row=False, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
  return dict(name=name, op='sample', n=n, actions=actions, dtype=dtype, legal=legal, per_row=per_row,
              temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


def _log_prob(name, n, actions, dtype, legal=False, temperature=1.0):
  return dict(name=name, op='log_prob', n=n, actions=actions, dtype=dtype, legal=legal, temperature=temperature)


def listed():
  return [
      # one environment being played: scrolly_maze's board, latency counts
      _project('project_one_board', 1, 10, 30, 8, 256, 'bfloat16', 'relu'),
      # a batch of marauders boards, ten characters
      _project('project_marauders', 4096, 16, 39, 10, 512, 'float16', 'silu'),
      # every environment of a large scrolly_maze engine, a residual stream added
      _project('project_scrolly_maze', 262144, 10, 30, 8, 256, 'bfloat16', 'relu', residual=True),
      # warehouse_manager with occlusion_in_layers=False: layers overlap, so they come stacked
      _project('project_stacked_warehouse', 32768, 11, 10, 11, 128, 'bfloat16', 'tanh', stacked=True),
      # a training step over stored scrolly_maze boards
      _project('train_scrolly_maze', 65536, 10, 30, 8, 256, 'bfloat16', 'relu', residual=True, train=True),
      # the large uncropped board of better_scrolly_maze, an odd number of cells, weights in 32 bits
      _project('train_better_scrolly', 2048, 45, 89, 7, 200, 'float32', 'gelu', train=True),
      # the five moves of the shipped mazes, in every environment of the headline batch
      _sample('sample_moves', 1048576, 5, 'float32', legal=True),
      # a small batch whose environments each have their own exploration rules
      _sample('sample_rules_per_row', 1024, 16, 'bfloat16', legal=True, per_row=True),
      # a prefab game whose entities share one action code: 4,096 joint actions
      _sample('sample_joint', 4096, 4096, 'bfloat16', temperature=0.8, top_k=50, top_p=0.95, min_p=0.02),
      # the widest action code of a game with directives
      _sample('sample_widest', 8, 1048576, 'float32', temperature=1.3, top_p=0.9),
      # policy-gradient step of a million environments
      _log_prob('log_prob_moves', 1048576, 5, 'float32', legal=True),
      # policy-gradient step over joint actions
      _log_prob('log_prob_joint', 4096, 4096, 'bfloat16', temperature=0.8),
  ]


def _spread(rng, lo, hi):
  """A whole number of [lo, hi], its logarithm evenly spread."""
  return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
  op = rng.choice(['project', 'project', 'train', 'sample', 'sample', 'log_prob'])
  dtype = rng.choice(sorted(_DTYPES))
  if op in ('project', 'train'):
    while True:
      stacked = rng.random() < 0.25
      c = _project(None, _spread(rng, 1, 262144), rng.randint(3, 45), rng.randint(7, 89), rng.randint(3, 16),
                   _spread(rng, 8, 512), dtype, rng.choice([None, 'relu', 'silu', 'tanh', 'gelu']),
                   residual=rng.random() < 0.5, train=op == 'train', stacked=stacked)
      w = c['n'] * c['rows'] * c['cols'] * c['layers']
      if w * c['hidden'] * (2 if c['train'] else 1) <= 262144 * 300 * 8 * 256 and w <= 262144 * 300 * 8:
        break
  else:
    while True:
      n, a = _spread(rng, 1, 1048576), _spread(rng, 2, 1048576)
      if n * a <= 4096 * 4096:
        break
    if op == 'log_prob':
      c = _log_prob(None, n, a, dtype, legal=rng.random() < 0.5, temperature=rng.choice([1.0, 0.7, 1.5]))
    else:
      c = _sample(None, n, a, dtype, legal=rng.random() < 0.5, per_row=rng.random() < 0.3,
                  temperature=rng.choice([1.0, 0.6, 1.4]), top_k=rng.choice([0, 1, 3, 40, 1000]),
                  top_p=rng.choice([1.0, 0.95, 0.5]), min_p=rng.choice([0.0, 0.0, 0.05]))
  del c['name']
  return c


def _make(case, seed):
  """The inputs of a case, from the seed alone."""
  g = torch.Generator(device='cuda')
  g.manual_seed(seed)
  dt, n, dev = _DTYPES[case['dtype']], case['n'], 'cuda'
  s = dict(case=case)
  if case['op'] == 'project':
    r, c, l, h = case['rows'], case['cols'], case['layers'], case['hidden']
    # the characters of a game board: half of it blank, a third walls, the rest spread over the entities and one
    # character that the learner does not stack
    table = [' '] * 128 + ['#'] * 80
    table += [(_CHARS[2:l] + '~')[i % (l - 1)] for i in range(256 - len(table))]
    table = torch.tensor([ord(x) for x in table], dtype=torch.uint8, device=dev)
    pick = torch.randint(0, 256, (n, r, c), generator=g, device=dev, dtype=torch.uint8)
    boards = table[pick.int()]
    s['layers'] = _CHARS[:l]
    if case['stacked']:
      chars = torch.tensor([ord(x) for x in s['layers']], dtype=torch.uint8, device=dev)
      over = torch.randint(0, 256, (n, l, r, c), generator=g, device=dev, dtype=torch.uint8) < 20  # overlapping layers
      s['boards'] = ((boards[:, None] == chars[None, :, None, None]) | over).to(torch.uint8)
    else:
      s['boards'] = boards
    s['weight'] = (torch.randn(h, l, r, c, generator=g, device=dev) * (1.0 / math.sqrt(r * c))).to(dt)
    s['bias'] = (torch.randn(h, generator=g, device=dev) * 0.1).to(dt)
    s['residual'] = torch.randn(n, h, generator=g, device=dev).to(dt) if case['residual'] else None
    if case['train']:
      s['grad'] = torch.randn(n, h, generator=g, device=dev).to(dt)
    return s
  a = case['actions']
  s['logits'] = (torch.randn(n, a, generator=g, device=dev) * 2.0).to(dt)
  s['legal'] = None
  if case['legal']:
    s['legal'] = torch.rand(n, a, generator=g, device=dev) < 0.75
    s['legal'][3::257] = False  # an environment with nothing left to do
  if case['op'] == 'sample':
    s['uniforms'] = torch.rand(n, generator=g, device=dev)
    for key in ('temperature', 'top_k', 'top_p', 'min_p'):
      s[key] = case[key]
    if case['per_row']:
      s['temperature'] = torch.rand(n, generator=g, device=dev) * 1.5 + 0.25
      s['temperature'][::7] = 0.0  # greedy environments
      s['top_k'] = torch.randint(0, min(a, 100) + 1, (n,), generator=g, device=dev, dtype=torch.int32)
      s['top_p'] = 1.05 - 0.6 * torch.rand(n, generator=g, device=dev)
      s['min_p'] = (0.1 * torch.rand(n, generator=g, device=dev) - 0.03).clamp(min=0.0)
  else:
    key = torch.rand(n, a, generator=g, device=dev)
    if s['legal'] is not None:
      key = torch.where(s['legal'], key, torch.full_like(key, -1.0))
    best = key.max(1)
    s['actions'] = torch.where(best.values >= 0, best.indices, torch.full_like(best.indices, -1)).to(torch.int32)
    s['grad_log_prob'] = torch.randn(n, generator=g, device=dev)
    s['grad_entropy'] = torch.randn(n, generator=g, device=dev) * 0.01
  return s


def prepare(case, seed):
  s = _make(case, seed)
  if own and case['op'] == 'project':
    if case['train']:
      for key in ('weight', 'bias', 'residual'):
        if s[key] is not None:
          s[key].requires_grad_()
    else:  # a policy that is only asked keeps its weights laid out
      from pycolab_amd import rendering
      s['handle'] = rendering.ObservationProjection(s['layers'], s['weight'], s['bias'], activation=case['activation'])
  elif own and case['op'] == 'log_prob':
    s['logits'].requires_grad_()
  return s


def run(state):
  case = state['case']
  if own:
    return _run_own(case, state)
  if case['op'] == 'project':
    return _plain_project(case, state)
  if case['op'] == 'sample':
    return _plain_sample(case, state)
  return _plain_log_prob(case, state)


def _run_own(case, s):
  from pycolab_amd import actions
  from pycolab_amd import rendering
  if case['op'] == 'project' and not case['train']:
    return s['handle'](s['boards'], residual=s['residual'])
  if case['op'] == 'project':
    y = rendering.project(s['boards'], s['layers'], s['weight'], s['bias'], activation=case['activation'],
                          residual=s['residual'])
    leaves = [s[k] for k in ('weight', 'bias', 'residual') if s[k] is not None]
    return [y.detach()] + list(torch.autograd.grad(y, leaves, s['grad']))
  if case['op'] == 'sample':
    return actions.sample(s['logits'], s['uniforms'], temperature=s['temperature'], top_k=s['top_k'], top_p=s['top_p'],
                          min_p=s['min_p'], legal=s['legal'])
  log_prob, entropy = actions.log_prob(s['logits'], s['actions'], legal=s['legal'], temperature=case['temperature'])
  grad, = torch.autograd.grad([log_prob, entropy], [s['logits']], [s['grad_log_prob'], s['grad_entropy']])
  return [log_prob.detach(), entropy.detach(), grad]


# ---------------------------------------------------------------- plain forms


def _activate(kind, z):
  """(act(z), act'(z))"""
  if kind is None:
    return z, torch.ones_like(z)
  if kind == 'relu':
    return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).to(z.dtype)
  if kind == 'tanh':
    t = torch.tanh(z)
    return t, 1 - t * t
  if kind == 'silu':
    sg = 1 / (1 + torch.exp(-z))
    return z * sg, sg * (1 + z * (1 - sg))
  cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))  # gelu
  return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _plain_project(case, s):
  n, h = case['n'], case['hidden']
  if case['stacked']:
    features = (s['boards'] != 0).float()
  else:
    chars = torch.tensor([ord(x) for x in s['layers']], dtype=torch.uint8, device='cuda')
    features = (s['boards'][:, None] == chars[None, :, None, None]).float()
  features = features.reshape(n, -1)
  dt = s['weight'].dtype
  z = features @ s['weight'].reshape(h, -1).float().t() + s['bias'].float()
  y, slope = _activate(case['activation'], z)
  if s['residual'] is not None:
    y = y + s['residual'].float()
  if not case['train']:
    return y.to(dt)
  dz = s['grad'].float() * slope
  out = [y.to(dt), (dz.t() @ features).reshape(s['weight'].shape).to(dt), dz.sum(0).to(dt)]
  if s['residual'] is not None:
    out.append(s['grad'].clone())
  return out


def _column(value, n, dtype):
  if not isinstance(value, torch.Tensor):
    value = torch.full((n,), value, dtype=torch.float32 if dtype == torch.float64 else dtype, device='cuda')
  return value.to(dtype)[:, None]


def _plain_sample(case, s):
  # in 64 bits: an action is decided by where a number falls between two sums
  n, a = case['n'], case['actions']
  x = s['logits'].double()
  ok = ~torch.isnan(x) & (x > -math.inf)
  if s['legal'] is not None:
    ok = ok & s['legal']
  x = torch.where(ok, x, torch.full_like(x, -math.inf))
  temperature = _column(s['temperature'], n, torch.float64)
  top_k, top_p, min_p = _column(s['top_k'], n, torch.int64), _column(s['top_p'], n, torch.float64), _column(s['min_p'], n, torch.float64)
  greedy = ~(temperature > 0)
  value, index = torch.sort(x, dim=1, descending=True, stable=True)  # ties: the lowest index first
  best = value[:, :1]
  live = value > -math.inf
  w = torch.where(value == best, torch.ones_like(value), torch.exp((value - best) / torch.where(greedy, torch.ones_like(temperature), temperature)))
  w = torch.where(live, w, torch.zeros_like(w))
  rank = torch.arange(a, device='cuda')[None, :]
  keep = live & ((top_k <= 0) | (rank < top_k))
  w = torch.where(keep, w, torch.zeros_like(w))
  run_ = torch.cumsum(w, 1)
  ahead = torch.cat([torch.zeros_like(run_[:, :1]), run_[:, :-1]], 1)
  keep = keep & ((rank == 0) | ~(top_p < 1) | (ahead < top_p * run_[:, -1:]))
  keep = keep & ((rank == 0) | (w >= min_p.clamp(max=1.0)))
  keep = keep & ((rank == 0) | ~greedy)
  w = torch.where(keep, w, torch.zeros_like(w))
  w = torch.zeros_like(w).scatter_(1, index, w)  # back in the actions' own order
  cdf = torch.cumsum(w, 1)
  over = (cdf > s['uniforms'].double()[:, None] * cdf[:, -1:]) & (w > 0)
  action = torch.where(over, rank, torch.full_like(rank, a)).min(1).values
  return torch.where(ok.any(1), action, torch.full_like(action, -1)).to(torch.int32)


def _plain_log_prob(case, s):
  t = case['temperature']
  x = s['logits'].detach().float() / t
  ok = ~torch.isnan(x) & (x > -math.inf)
  if s['legal'] is not None:
    ok = ok & s['legal']
  x = torch.where(ok, x, torch.full_like(x, -math.inf))
  some = ok.any(1)
  best = torch.where(some, x.max(1).values, torch.zeros_like(x[:, 0]))[:, None]
  d = torch.where(ok, x - best, torch.zeros_like(x))
  e = torch.where(ok, torch.exp(d), torch.zeros_like(x))
  total = torch.where(some, e.sum(1), torch.ones_like(best[:, 0]))[:, None]
  p, lp = e / total, d - torch.log(total)
  zero = torch.zeros_like(p)
  entropy = -(torch.where(ok, p * lp, zero)).sum(1)
  taken = s['actions'].long()
  there = taken >= 0
  at = taken.clamp(min=0)[:, None]
  picked = torch.where(ok.gather(1, at)[:, 0], lp.gather(1, at)[:, 0], torch.full_like(entropy, -math.inf))
  log_prob = torch.where(there & some, picked, torch.zeros_like(entropy))
  g_lp = torch.where(there, s['grad_log_prob'], torch.zeros_like(entropy))[:, None]
  grad = -g_lp * p - s['grad_entropy'][:, None] * p * (lp + entropy[:, None])
  grad.scatter_add_(1, at, g_lp)
  grad = torch.where(ok, grad / t, zero)
  return [log_prob, entropy, grad.to(s['logits'].dtype)]


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
  n, size = case['n'], _SIZE[case['dtype']]
  if case['op'] == 'project':
    cells, l, h = case['rows'] * case['cols'], case['layers'], case['hidden']
    boards = n * cells * (l if case['stacked'] else 1)
    weight = h * l * cells * size
    out = n * h * size
    moved = boards + weight + h * size + out * (2 if case['residual'] else 1)
    flops = 2 * n * l * cells * h  # the product over all layers, as matrix units take it
    if case['train']:  # the step's gradient in; the weight's, the bias' and the residual's gradients out
      moved += out + weight + h * size + (out if case['residual'] else 0)
      flops *= 2
    return dict(bytes=moved, flops=flops)
  a = case['actions']
  moved = n * a * size + (n * a if case['legal'] else 0)
  if case['op'] == 'sample':
    moved += n * 8 + (n * 16 if case['per_row'] else 0)  # a uniform number in, an action out; the rows' rules
    return dict(bytes=moved, flops=n * a * 4)
  moved += n * a * size + n * 20  # the logits' gradient out; actions and two gradients in, two numbers out
  return dict(bytes=moved, flops=n * a * 12)


# ---------------------------------------------------------------- in 64 bits, from the definitions


def exact(case, seed):
  s = _make(case, seed)
  if case['op'] == 'sample':
    return None  # a choice, no computed number
  if case['op'] == 'project':
    return _exact_project(case, s)
  x = s['logits'].double().requires_grad_()
  allowed = torch.ones_like(x, dtype=torch.bool) if s['legal'] is None else s['legal']
  filled = (x / case['temperature']).masked_fill(~allowed, -1e300)
  lp = torch.log_softmax(filled, 1)
  inside = allowed.any(1).double()
  entropy = -(torch.where(allowed, lp.exp() * lp, torch.zeros_like(lp))).sum(1) * inside
  there = (s['actions'] >= 0).double() * inside
  log_prob = lp.gather(1, s['actions'].long().clamp(min=0)[:, None])[:, 0] * there
  grad, = torch.autograd.grad((log_prob * s['grad_log_prob'].double() + entropy * s['grad_entropy'].double()).sum(), x)
  return [log_prob.detach(), entropy.detach(), grad]


def _exact_project(case, s):
  n, h = case['n'], case['hidden']
  w, b = s['weight'].double().reshape(h, case['layers'], -1), s['bias'].double().requires_grad_()
  step = max(1, (1 << 28) // (case['rows'] * case['cols']))
  outs, dw, db = [], torch.zeros_like(w), torch.zeros(h, dtype=torch.float64, device='cuda')
  act = {None: lambda z: z, 'relu': torch.relu, 'tanh': torch.tanh, 'silu': lambda z: z * torch.sigmoid(z),
         'gelu': lambda z: z * torch.special.ndtr(z)}[case['activation']]
  for lo in range(0, n, step):
    part = s['boards'][lo:lo + step]
    m = part.shape[0]

    def layer(k):
      on = part[:, k] != 0 if case['stacked'] else part == ord(s['layers'][k])
      return on.reshape(m, -1).double()

    z = torch.zeros(m, h, dtype=torch.float64, device='cuda')
    for k in range(case['layers']):
      z += layer(k) @ w[:, k].t()
    z.requires_grad_()
    y = act(z + b)
    if case['train']:
      dz, db_ = torch.autograd.grad(y, [z, b], s['grad'][lo:lo + m].double())
      db += db_
      for k in range(case['layers']):
        dw[:, k] += dz.t() @ layer(k)
    y = y.detach()
    if s['residual'] is not None:
      y = y + s['residual'][lo:lo + m].double()
    outs.append(y)
  y = torch.cat(outs)
  if not case['train']:
    return y
  out = [y, dw.reshape(s['weight'].shape), db]
  if s['residual'] is not None:
    out.append(s['grad'].double())
  return out
