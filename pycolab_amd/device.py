"""Device memory and stream plumbing for the host facade.

PyTorch-ROCm, when present with a visible GPU, owns the allocations (so
observations are ordinary device tensors for the consumer) and supplies the
HIP stream; otherwise buffers come from the C ABI's own allocator and are
read back with synchronous copies.  Either way the step kernels are the ones
in csrc/ -- nothing here computes.
"""

import ctypes
import weakref

import numpy as np

from pycolab_amd import _native as N

from pycolab_amd._torchprobe import torch_module  # noqa: F401 (re-exported)


_NP_TO_TORCH = {'uint8': 'uint8', 'int32': 'int32', 'float32': 'float32', 'int64': 'int64', 'float64': 'float64'}


class DeviceBuffer(object):
  """A typed device array with `.ptr`, `.numpy()` and (with torch) `.tensor`."""

  def __init__(self, shape, dtype, device_id):
    self.shape = tuple(int(s) for s in shape)
    self.dtype = np.dtype(dtype)
    self.nbytes = int(np.prod(self.shape)) * self.dtype.itemsize
    self.device_id = device_id
    torch = torch_module()
    self.tensor = None
    self._raw = None
    if torch is not None:
      self.tensor = torch.zeros(self.shape, dtype=getattr(torch, _NP_TO_TORCH[self.dtype.name]),
                                device='cuda:%d' % device_id)
      self.ptr = self.tensor.data_ptr()
    else:
      p = ctypes.c_void_p()
      N.check(N.lib().pcx_device_malloc(ctypes.byref(p), max(self.nbytes, 1)))
      self._raw = p
      self.ptr = p.value
      self.upload(np.zeros(self.shape, self.dtype))

  @classmethod
  def view_of(cls, tensor, dtype, device_id):
    """A typed buffer over (a slice of) an existing device tensor: no allocation."""
    self = cls.__new__(cls)
    self.dtype = np.dtype(dtype)
    torch = torch_module()
    self.tensor = tensor.view(getattr(torch, _NP_TO_TORCH[self.dtype.name]))
    self.shape = tuple(self.tensor.shape)
    self.nbytes = int(np.prod(self.shape)) * self.dtype.itemsize
    self.device_id = device_id
    self._raw = None
    self.ptr = self.tensor.data_ptr()
    return self

  def numpy(self):
    if self.tensor is not None:
      return self.tensor.cpu().numpy()
    out = np.empty(self.shape, self.dtype)
    N.check(N.lib().pcx_memcpy_d2h(out.ctypes.data, self.ptr, self.nbytes))
    return out

  def upload(self, array):
    array = np.ascontiguousarray(array, dtype=self.dtype).reshape(self.shape)
    if self.tensor is not None:
      torch = torch_module()
      self.tensor.copy_(torch.from_numpy(array))
    else:
      N.check(N.lib().pcx_memcpy_h2d(self.ptr, array.ctypes.data, self.nbytes))

  def free(self):
    if self._raw is not None:
      N.lib().pcx_device_free(self._raw)
      self._raw = None
    self.tensor = None

  def __del__(self):
    try:
      self.free()
    except Exception:  # pylint: disable=broad-except
      pass


class Written(object):
  """How often kernels have written a device array that a caller may still be looking at (autograd's own counters do not see
  them).  Whoever launches the writes holds it, and it holds the array, if there is a tensor of it: while it lives, the
  tensor's storage can be found by its address and is no one else's."""

  __slots__ = ('count', 'tensor', '__weakref__')
  _by_storage = weakref.WeakValueDictionary()

  def __init__(self, tensor=None):
    self.count = 0
    self.tensor = tensor
    if tensor is not None and tensor.numel():
      Written._by_storage[tensor.untyped_storage().data_ptr()] = self

  @classmethod
  def of(cls, tensor):
    """The one of the array that `tensor` is a view of, or None."""
    return cls._by_storage.get(tensor.untyped_storage().data_ptr()) if tensor.numel() else None


def current_stream(device_id):
  torch = torch_module()
  if torch is None:
    return None
  return ctypes.c_void_p(torch.cuda.current_stream(device_id).cuda_stream)


def synchronize(device_id):
  torch = torch_module()
  if torch is not None:
    torch.cuda.synchronize(device_id)
  else:
    N.check(N.lib().pcx_stream_synchronize(None))


# ---- the policy operators (rendering.project, actions.sample, actions.log_prob) work on PyTorch tensors ----------------
# Their calls are small next to what they launch only if the way there is short: descriptions as packed bytes, the raw
# stream, no context manager on the device that is current anyway.


def require_torch(what):
  torch = torch_module()
  if torch is None:
    raise RuntimeError('{} needs PyTorch-ROCm and a GPU'.format(what))
  return torch


_kinds = None


def policy_dtype(tensor, name):
  """The C ABI's number for a floating tensor's type."""
  global _kinds
  if _kinds is None:
    torch = torch_module()
    _kinds = {torch.float32: N.F32, torch.float16: N.F16, torch.bfloat16: N.BF16}
  kind = _kinds.get(tensor.dtype)
  if kind is None:
    raise TypeError('{} must be float32, float16 or bfloat16, not {}'.format(name, tensor.dtype))
  return kind


def pointer(tensor):
  return None if tensor is None else tensor.data_ptr()


def raw_stream(device_id):
  """`device_id`'s current stream, as the C ABI takes it."""
  if _raw_stream is None:
    _find_stream()
  return _raw_stream(device_id)


def launch(device_id, function, *args):
  """function(*args, stream) of the C ABI on `device_id`'s current stream."""
  if _raw_stream is None:
    _find_stream()
  if _one_gpu or _current_device() == device_id:
    code = function(*args, _raw_stream(device_id))
  else:
    torch = torch_module()
    with torch.cuda.device(device_id):
      code = function(*args, torch.cuda.current_stream(device_id).cuda_stream)
  if code:
    N.check(code)


_raw_stream = _one_gpu = _current_device = None


def _find_stream():
  global _raw_stream, _one_gpu, _current_device
  torch = torch_module()
  _one_gpu, _current_device = torch.cuda.device_count() == 1, torch.cuda.current_device
  # (the stream without the Python object around it)
  _raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


_sizes = {}


def workspace(function, desc, device):
  """(tensor or None, bytes): the workspace that `function` (pcx_..._size) asks for a description, for this call alone."""
  key = (function, desc)
  size = _sizes.get(key)
  if size is None:
    out = N.c_u64(0)
    N.check(getattr(N.lib(), function)(desc, ctypes.byref(out)))
    if len(_sizes) > 4096:
      _sizes.clear()
    size = _sizes[key] = int(out.value)
  if not size:
    return None, 0
  torch = torch_module()
  return torch.empty(size, dtype=torch.uint8, device=device), size


def refuse_recording_in_capture(what, instead):
  """A backward pass captured while an eager graph of the same leaves lives would run on that graph's stream and end the
  process: differentiable calls are refused under capture, the explicit pair of calls is what a graph holds."""
  if torch_module().cuda.is_current_stream_capturing():
    raise RuntimeError('{}() does not record gradients while a graph is captured: capture {} instead'.format(what, instead))


def saveable(torch, tensor):
  """The tensor, or a copy where it was made in inference mode -- in a rollout, say: autograd saves no such tensor."""
  return tensor.clone() if isinstance(tensor, torch.Tensor) and tensor.is_inference() else tensor


def refuse_tangents(what, *tensors):
  """Forward mode is not recorded: a tensor with a tangent looks like any other (it does not ask for gradients), and its
  tangent would be dropped."""
  forward = torch_module().autograd.forward_ad
  if getattr(forward, '_current_level', 0) < 0:  # (nobody differentiates forward; without that number, ask each tensor)
    return
  for tensor in tensors:
    if tensor is not None and forward.unpack_dual(tensor).tangent is not None:
      raise RuntimeError('{}() has no forward-mode derivative'.format(what))


def refuse_twice(what):
  """Called in a backward pass: gradients are recorded there only when it is to be differentiated itself."""
  if torch_module().is_grad_enabled():
    raise RuntimeError('{}() cannot be differentiated twice'.format(what))
