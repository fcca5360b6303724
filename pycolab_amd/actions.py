"""Actions: synthetic tapes shared by host, oracle and device, and actions drawn from a policy's logits.

`pcx_action_hash` (include/pcx.h) is the counter-based generator behind
`Engine.step_hashed`: action of environment `env` (its GLOBAL index in a
sharded batch) at step `t` = hash(seed, env, t) % n_actions.  This is its
vectorised host twin, so that a sharded run can stage on every rank exactly the
tape an unsharded engine would draw on the device (the global
environment index drives the actions, never the rank).

`sample` draws one action per environment from a policy's logits (what
`Engine.play()` / `Engine.step_sampled()` then takes), `log_prob` is the
log-probability of actions taken and the policy's entropy, differentiable in
the logits.  Both run as kernels of csrc/pcx_policy.hip on PyTorch tensors.
"""

import numpy as np

from pycolab_amd import _native as N
from pycolab_amd import device as dev

_M1, _M2, _M3 = np.uint64(0x9E3779B97F4A7C15), np.uint64(0xBF58476D1CE4E5B9), np.uint64(0x94D049BB133111EB)


def action_hash(seed, env, t):
  """uint32 array: pcx_action_hash(seed, env, t), broadcasting `env` and `t`."""
  with np.errstate(over='ignore'):
    env = np.asarray(env, dtype=np.uint64)
    t = np.asarray(t, dtype=np.uint64)
    x = np.uint64(seed & 0xFFFFFFFFFFFFFFFF) ^ (env * _M1) ^ (t * _M2)
    x = (x ^ (x >> np.uint64(30))) * _M2
    x = (x ^ (x >> np.uint64(27))) * _M3
    x = x ^ (x >> np.uint64(31))
    return (x >> np.uint64(32)).astype(np.uint32)


def hashed_tape(seed, env_lo, n_envs, t0, steps, n_actions):
  """int32 [steps, n_envs]: the actions `step_hashed(seed, t0, steps)` draws for
  global environments [env_lo, env_lo + n_envs)."""
  env = np.arange(env_lo, env_lo + n_envs, dtype=np.uint64)[None, :]
  t = np.arange(t0, t0 + steps, dtype=np.uint64)[:, None]
  return (action_hash(seed, env, t) % np.uint32(n_actions)).astype(np.int32)


# ---------------------------------------------------------------------- a policy's actions


def _rows(torch, logits, legal):
  """(description, legal tensor to keep, rows, actions, device index) of logits [n, actions] whose actions are contiguous."""
  if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dim() != 2:
    raise ValueError('logits must be a device tensor [n, actions]')
  dtype = dev.policy_dtype(logits, 'logits')
  n, actions = logits.shape
  row_stride, stride = logits.stride()
  if actions < 1:
    raise ValueError('logits of no action')
  if actions > 1 and stride != 1:
    raise ValueError('the actions of a row must be contiguous (strides {})'.format(logits.stride()))
  legal_stride = 0
  if legal is not None:
    if not isinstance(legal, torch.Tensor) or legal.device != logits.device or legal.dtype not in (torch.bool, torch.uint8):
      raise ValueError('legal must be a bool or uint8 tensor on {}'.format(logits.device))
    if legal.dim() == 1 and legal.shape[0] == actions:
      legal = legal.expand(n, actions)
    if legal.shape != logits.shape:
      raise ValueError('legal must be [{}, {}] or [{}]'.format(n, actions, actions))
    legal_stride, stride = legal.stride()
    if actions > 1 and stride != 1:
      raise ValueError('the actions of a row of `legal` must be contiguous')
  return N.LOGITS_DESC.pack(n, row_stride, legal_stride, actions, dtype), legal, n, actions, logits.device.index


def _per_row(torch, value, name, n, dtype, device):
  """A rule's device array [n], or None for a number."""
  if not isinstance(value, torch.Tensor):
    return None
  if value.dtype != dtype or value.device != device or tuple(value.shape) != (n,):
    raise ValueError('{} must be a number or a {} tensor [{}] on {}'.format(name, dtype, n, device))
  return value.contiguous()


def sample(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, legal=None, out=None):
  """One action per row of `logits` (float32, float16 or bfloat16 device tensor [n, actions]): int32 [n], what
  `Engine.play()` takes.

  `uniforms`: float32 [n], one number of [0, 1) per row; the result is a function of the row and its number alone, so a
  sharded batch draws what the whole one would.  `legal`: bool / uint8 [n, actions] or [actions]; an action is allowed where
  it is legal and its logit is neither -infinity nor a NaN.  Of the allowed actions, ordered by (logit descending, index
  ascending), the first `top_k` stay (0: all), of those each whose predecessors weigh less than `top_p` of the total, of
  those each at least `min_p` times as probable as the best; the best one always.  Weights are exp(logit / temperature);
  `temperature` 0 takes the best action.  Each of the four is a number or a device array [n] (float32; `top_k` int32), row by
  row.  A row that allows nothing gives `_native.ACTION_NONE` (-1), the engine's `None`.

  `out`: an int32 tensor [n] to write into (autograd counts it as a change in place: a backward pass that needs its old values
  is refused; of a replayed graph's writes it does not know).  Nothing waits for the device; calls can be captured into a graph."""
  torch = dev.require_torch('sample()')
  desc, legal, n, _, index = _rows(torch, logits, legal)
  device = logits.device
  if (not isinstance(uniforms, torch.Tensor) or uniforms.dtype != torch.float32 or uniforms.device != device or uniforms.dim() != 1 or
      uniforms.shape[0] != n):
    raise ValueError('uniforms must be float32 [{}] on {}'.format(n, device))
  t_row = _per_row(torch, temperature, 'temperature', n, torch.float32, device)
  k_row = _per_row(torch, top_k, 'top_k', n, torch.int32, device)
  p_row = _per_row(torch, top_p, 'top_p', n, torch.float32, device)
  m_row = _per_row(torch, min_p, 'min_p', n, torch.float32, device)
  if k_row is None:
    if int(top_k) != top_k:
      raise ValueError('top_k must be a whole number')
    top_k = max(-1, min(int(top_k), 1 << 30))
  rules = N.SAMPLING.pack(0.0 if t_row is not None else float(temperature), 0.0 if p_row is not None else float(top_p),
                          0.0 if m_row is not None else float(min_p), 0 if k_row is not None else top_k,
                          dev.pointer(t_row) or 0, dev.pointer(k_row) or 0, dev.pointer(p_row) or 0, dev.pointer(m_row) or 0)
  given = out is not None
  if not given:
    out = torch.empty((n,), dtype=torch.int32, device=device)
  elif out.dtype != torch.int32 or out.device != device or tuple(out.shape) != (n,) or not out.is_contiguous():
    raise ValueError('out must be a contiguous int32 tensor [{}] on {}'.format(n, device))
  uniforms = uniforms.contiguous()
  scratch, size = dev.workspace('pcx_sample_size', desc, device)
  dev.launch(index, N.lib().pcx_sample_actions, desc, rules, logits.data_ptr(), dev.pointer(legal), uniforms.data_ptr(), out.data_ptr(),
             dev.pointer(scratch), size)
  if given:  # (a log_prob() of the actions that lay there may still wait for its backward pass)
    torch.autograd.graph.increment_version(out)
  return out


def _taken(torch, actions, n, device):
  if not isinstance(actions, torch.Tensor) or actions.dtype != torch.int32 or actions.device != device or tuple(actions.shape) != (n,):
    raise ValueError('actions must be int32 [{}] on {}'.format(n, device))
  return actions.contiguous()


def _log_prob_forward(torch, desc, legal, logits, actions, temperature):
  n, device = logits.shape[0], logits.device
  stats = torch.empty((n, 2), dtype=torch.float32, device=device)
  log_prob, entropy = stats.new_empty(n), stats.new_empty(n)
  scratch, size = dev.workspace('pcx_log_prob_size', desc, device)
  dev.launch(device.index, N.lib().pcx_log_prob, desc, temperature, logits.data_ptr(), dev.pointer(legal), actions.data_ptr(),
             log_prob.data_ptr(), entropy.data_ptr(), stats.data_ptr(), dev.pointer(scratch), size)
  return log_prob, entropy, stats


def _log_prob_backward(torch, desc, legal, logits, actions, temperature, entropy, stats, grad_log_prob, grad_entropy):
  # (autograd calls this on a thread of its own, where every line costs several times what it does elsewhere)
  grad = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty(logits.shape)
  if grad_log_prob is not None and not grad_log_prob.is_contiguous():
    grad_log_prob = grad_log_prob.contiguous()
  if grad_entropy is not None and not grad_entropy.is_contiguous():
    grad_entropy = grad_entropy.contiguous()
  dev.launch(logits.get_device(), N.lib().pcx_log_prob_backward, desc, temperature, logits.data_ptr(), dev.pointer(legal), actions.data_ptr(),
             entropy.data_ptr(), stats.data_ptr(), dev.pointer(grad_log_prob), dev.pointer(grad_entropy), grad.data_ptr())
  return grad


def _layout(logits, actions, legal, entropy, stats):
  """Where and how the arrays of a backward pass lie: what the forward pass's description of them goes by."""
  return (logits.data_ptr(), logits.dtype, logits.shape, logits.stride(), None if legal is None else (legal.data_ptr(), legal.stride()), actions.data_ptr(),
          entropy.data_ptr(), stats.data_ptr())


_log_prob_function = None


def _log_prob_autograd():
  """The autograd function behind `log_prob()` (made on first use: PyTorch is optional here)."""
  global _log_prob_function
  if _log_prob_function is None:
    torch = dev.torch_module()
    grad_enabled = torch.is_grad_enabled

    class LogProb(torch.autograd.Function):

      @staticmethod
      def forward(ctx, logits, actions, legal, temperature, desc):
        ctx.set_materialize_grads(False)
        log_prob, entropy, stats = _log_prob_forward(torch, desc, legal, logits, actions, temperature)
        ctx.desc, ctx.temperature, ctx.layout = desc, temperature, _layout(logits, actions, legal, entropy, stats)
        ctx.save_for_backward(logits, actions, legal, entropy, stats)
        return log_prob, entropy

      @staticmethod
      def backward(ctx, grad_log_prob, grad_entropy):
        if grad_enabled():
          dev.refuse_twice('log_prob')
        logits, actions, legal, entropy, stats = ctx.saved_tensors
        if grad_log_prob is None and grad_entropy is None:
          return None, None, None, None, None
        if _layout(logits, actions, legal, entropy, stats) != ctx.layout:
          # (what was saved went elsewhere meanwhile -- torch.autograd.graph.saved_tensors_hooks, checkpoint -- and what came
          # back is laid out in its own way)
          return (log_prob_backward(logits, actions, entropy, stats, grad_log_prob, grad_entropy, legal, ctx.temperature), None, None, None,
                  None)
        return (_log_prob_backward(torch, ctx.desc, legal, logits, actions, ctx.temperature, entropy, stats, grad_log_prob, grad_entropy),
                None, None, None, None)

    _log_prob_function = LogProb
  return _log_prob_function


def _positive(temperature):
  temperature = float(temperature)
  if not 0.0 < temperature < float('inf'):
    raise ValueError('temperature must be a positive number, not {}'.format(temperature))
  return temperature


def log_prob(logits, actions, legal=None, temperature=1.0, return_stats=False):
  """(log-probability of `actions`, entropy) of every row's policy softmax(logits / temperature) over the allowed actions:
  two float32 tensors [n], differentiable in `logits` (float32, float16 or bfloat16 [n, actions]) once, in reverse mode.

  `actions`: int32 [n], as `sample()` returned them.  -1 (`_native.ACTION_NONE`: nothing was allowed) has log-probability 0
  and adds nothing to the gradient; so does a row that allows nothing, whose entropy is 0 too.  An action that is not
  allowed has -infinity, one that does not exist a NaN.  The gradient is 0 where an action is not allowed.  `legal`: as for
  `sample()`.

  `return_stats=True`: no autograd; returns (log_prob, entropy, stats), what `log_prob_backward` takes -- the pair to
  capture into a graph."""
  torch = dev.require_torch('log_prob()')
  if not return_stats and torch.is_grad_enabled():
    actions, legal = dev.saveable(torch, actions), dev.saveable(torch, legal)
  desc, legal, n, _, _ = _rows(torch, logits, legal)
  actions, temperature = _taken(torch, actions, n, logits.device), _positive(temperature)
  if return_stats:
    return _log_prob_forward(torch, desc, legal, logits.detach(), actions, temperature)
  dev.refuse_tangents('log_prob', logits)
  if logits.requires_grad and torch.is_grad_enabled():
    dev.refuse_recording_in_capture('log_prob', 'log_prob(..., return_stats=True) and log_prob_backward()')
    return _log_prob_autograd().apply(logits, actions, legal, temperature, desc)
  return _log_prob_forward(torch, desc, legal, logits, actions, temperature)[:2]


def log_prob_backward(logits, actions, entropy, stats, grad_log_prob=None, grad_entropy=None, legal=None, temperature=1.0):
  """The gradient with respect to `logits` of `log_prob()`'s two results, from theirs (float32 [n], None: zero) and from the
  `entropy` and `stats` it returned.  Records nothing for autograd and waits for nothing: it may be captured."""
  torch = dev.require_torch('log_prob_backward()')
  desc, legal, n, _, _ = _rows(torch, logits, legal)
  actions, temperature = _taken(torch, actions, n, logits.device), _positive(temperature)
  for t, shape, name in ((entropy, (n,), 'entropy'), (stats, (n, 2), 'stats')):
    if t.dtype != torch.float32 or tuple(t.shape) != shape or t.device != logits.device or not t.is_contiguous():
      raise ValueError('{} must be what log_prob(..., return_stats=True) returned'.format(name))
  for g, name in ((grad_log_prob, 'grad_log_prob'), (grad_entropy, 'grad_entropy')):
    if g is not None and (g.dtype != torch.float32 or tuple(g.shape) != (n,) or g.device != logits.device):
      raise ValueError('{} must be float32 [{}] on {}'.format(name, n, logits.device))
  return _log_prob_backward(torch, desc, legal, logits.detach(), actions, temperature, entropy, stats, grad_log_prob, grad_entropy)
