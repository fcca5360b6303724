"""Observations and observation post-processors.

`Observation` is the reference's namedtuple (rendering.py:28-63).  In batched
mode `board` has shape [B, rows, cols] and every `layers[c]` has shape
[B, rows, cols]; all are zero-copy views of a planes array in HBM
([B, 1 + n_chars, pitch] uint8), valid until the next step -- the
reference's own aliasing rule.

`ObservationToArray`, `ObservationToFeatureArray` and
`ObservationCharacterRepainter` keep the reference's constructors
(rendering.py:304-661) and run as streaming epilogue kernels
(csrc/pcx_post.hip) over the planes the engine, a cropper or a repainter
just wrote.  With batch > 1 their results are device tensors the kernel wrote
in place (no copy, no synchronisation; `torch.utils.dlpack.to_dlpack(t)`
exports them to any DLPack consumer); batch 1 returns the reference's NumPy
types.  They accept observations produced by this package (those know where
their planes live); anything else is rejected -- there is no host path.
"""

import collections
import ctypes

import numpy as np

from pycolab_amd import _native as N
from pycolab_amd import device as dev


class Observation(collections.namedtuple('Observation', ['board', 'layers'])):
  """board + layers; instances made by engines/croppers remember their source."""
  _source = None


_DTYPES = {'uint8': N.U8, 'int32': N.I32, 'float32': N.F32, 'int64': N.I64, 'float64': N.F64}


class _Post(object):
  """One device post-processor bound to one planes source.

  The output array is a device tensor of ours that the C side writes into
  (`pcx_post_bind_output`): `run()` enqueues one kernel on the current stream
  and returns that tensor -- no copy and no wait (batch 1, or no PyTorch: a
  NumPy copy, after a synchronisation, in the reference's shapes).
  """

  def __init__(self, source, desc, out_dtype, out_shape):
    self.view, self.device_id = source._planes_view()
    self.key = _view_key(self.view)
    self.desc = desc
    self.out_dtype, self.out_shape = np.dtype(out_dtype), tuple(out_shape)
    handle = ctypes.c_void_p()
    lib = N.lib()
    N.check(lib.pcx_post_create(ctypes.byref(self.view), ctypes.byref(desc), self.device_id, ctypes.byref(handle)))
    self.handle = handle
    self.out = None
    if dev.torch_module() is not None:
      self.out = dev.DeviceBuffer(self.out_shape, self.out_dtype, self.device_id)
      N.check(lib.pcx_post_bind_output(handle, self.out.ptr, self.out.nbytes))
    self.written = dev.Written(None if self.out is None else self.out.tensor)

  def run(self, host):
    lib = N.lib()
    N.check(lib.pcx_post_run(self.handle, dev.current_stream(self.device_id)))
    self.written.count += 1
    if self.out is not None and self.out.tensor is not None and not host:
      seen = N.c_i32(0)
      N.check(lib.pcx_post_error_poll(self.handle, dev.current_stream(self.device_id), ctypes.byref(seen)))
      return self.out.tensor, bool(seen.value)
    dev.synchronize(self.device_id)
    if self.out is not None:
      return self.out.numpy(), self.errors().any()
    ptr, nbytes = ctypes.c_void_p(), N.c_u64()
    N.check(lib.pcx_post_output(self.handle, ctypes.byref(ptr), ctypes.byref(nbytes)))
    out = np.empty(self.out_shape, self.out_dtype)
    assert out.nbytes == nbytes.value, (out.nbytes, nbytes.value)
    N.check(lib.pcx_memcpy_d2h(out.ctypes.data, ptr, out.nbytes))
    return out, self.errors().any()

  def errors(self):
    errs = np.empty((int(self.view.batch),), np.uint8)
    N.check(N.lib().pcx_post_errors(self.handle, errs.ctypes.data))
    return errs

  def __del__(self):
    try:
      N.lib().pcx_post_destroy(self.handle)
    except Exception:  # pylint: disable=broad-except
      pass


def _view_key(view):
  """What a cached post-processor depends on: where the source planes live and
  their shape.  A cropper re-attached to another engine, or an engine that was
  closed and rebuilt, shows up as a different key (the old planes are gone)."""
  return (view.planes, int(view.batch), view.rows, view.cols, view.pitch, view.n_chars, bytes(view.chars))


def _bound(post, source):
  """The cached `_Post` if it still reads the planes `source` has now."""
  if post is None:
    return None
  view, _ = source._planes_view()
  return post if post.key == _view_key(view) else None


def _source_of(observation):
  source = getattr(observation, '_source', None)
  if source is None:
    raise TypeError('this post-processor runs on the device and needs an Observation returned by a '
                    'pycolab_amd Engine or cropper')
  if getattr(observation, '_planes_stale', False):
    raise RuntimeError('this Observation is a placeholder: its engine no longer writes the full-board planes '
                       '(fuse_croppers(..., only_crops=True) or fuse_into(..., skip_board=True)); only the fused '
                       'croppers / the fused converter have something to return')
  return source


# Where the general epilogue body loses to step + stand-alone kernel (profiles/r04_post_kernels.md: scrolly_maze at
# 1,048,576 environments, value array next to the planes 1.33 against 0.95 ms, repainter 1.94 against 1.42; hello_world
# at 262,144: 0.40 / 0.36 and 0.64 / 0.51) and where it wins (4,096: 0.018 / 0.027; marauders 32,768: 0.059 / 0.071):
# the dividing line is whether the step's own planes still fit the 256 MiB Infinity Cache -- beyond it the separate
# kernel streams the board back at cache speed while the fused body is bound by its scalar bookkeeping.
_FUSED_BODY_PAYS_UP_TO = 256 << 20


def _general_epilogue_pays(engine):
  """Do this engine's observation planes fit the Infinity Cache (the fused value-array / repainter body wins)?"""
  return engine.batch * (1 + len(engine.template.chars)) * engine._pitch <= _FUSED_BODY_PAYS_UP_TO


def _strides(shape3, permute):
  """Element strides of (d, r, c) in the contiguous array whose axes are
  `permute` of (d, r, c) -- np.transpose(result, permute) made contiguous."""
  permute = (0, 1, 2) if permute is None else tuple(permute)
  out_shape = [shape3[a] for a in permute]
  out_strides = [int(np.prod(out_shape[i + 1:])) for i in range(3)]
  stride = [0, 0, 0]
  for out_axis, a in enumerate(permute):
    stride[a] = out_strides[out_axis]
  return stride, out_shape


class ObservationToArray(object):
  """board characters -> values or value vectors (rendering.py:409-542)."""

  def __init__(self, value_mapping, dtype=None, permute=None):
    self._value_mapping = value_mapping
    first = next(iter(value_mapping.values()))
    self._dtype = np.dtype(dtype if dtype is not None else np.array(first).dtype)
    try:
      self._depth = len(first)
      self._is_3d = True
    except TypeError:
      self._depth = 1
      self._is_3d = False
    self._permute = tuple(permute) if permute is not None else None
    if permute is not None:
      if self._is_3d and set(permute) != {0, 1, 2}:
        raise ValueError('When the value mapping contains 1-D vectors, the '
                         'permute argument to the ObservationToArray '
                         'constructor must be a list or tuple containing some '
                         'permutation of the integers 0, 1, and 2.')
      elif not self._is_3d and set(permute) != {0, 1}:
        raise ValueError('When the value mapping contains scalars, the permute '
                         'argument to the ObservationToArray constructor must '
                         'be a list or tuple containing some permutation of '
                         'the integers 0 and 1.')
    if self._dtype.name not in _DTYPES:
      raise NotImplementedError('ObservationToArray on the device supports dtypes {}'.format(sorted(_DTYPES)))
    if self._depth > N.POST_MAX_DEPTH:
      raise NotImplementedError('value vectors longer than {}'.format(N.POST_MAX_DEPTH))
    self._post = None
    self._fused = None  # (engine, device tensor, step count) once fuse_into() succeeded

  def fuse_into(self, engine, skip_layers=False, skip_board=False, force=False):
    """Have `engine`'s step kernel write this array itself, as an epilogue of
    its render loop (the board dword is in a register there, the value table in
    LDS): from the next `play()` / `step()` on, calling this object with one of
    the engine's observations returns the tensor the step already filled.
    `skip_layers=True` also stops the step from writing the uint8 layer planes
    -- a consumer that ingests, say, an RGB image gets the board and the image
    and nothing else; `skip_board=True` leaves out the board plane too (the
    engine's observations then carry `board=None`): the step writes this one
    array (scrolly_maze, a million environments, RGB: 0.69 ms against 1.05 ms
    for step + post-processor).  Returns False, and changes nothing, where the
    engine's kernel cannot do it (batch 1, a permuted axis order, boards that
    are not a whole number of dwords, a character of the game without a value,
    the table-driven kernel, unoccluded layers, fused croppers) -- or where it
    would be SLOWER than the two kernels: with the planes kept (or only the
    layers dropped) on batches whose planes no longer fit the Infinity Cache
    (`_general_epilogue_pays`; `force=True` fuses regardless, for A/B runs).
    Calls then run the post-processor as its own kernel, as before."""
    torch = dev.torch_module()
    identity = self._permute is None or tuple(self._permute) == tuple(range(len(self._permute)))
    if not identity or torch is None or engine._native is None or engine.batch == 1:
      return False
    if not (force or skip_board or _general_epilogue_pays(engine)):
      return False
    tdtype = getattr(torch, self._dtype.name)
    shape = (self._depth, engine.rows, engine.cols) if self._is_3d else (engine.rows, engine.cols)
    out = torch.zeros((engine.batch,) + shape, dtype=tdtype, device='cuda:%d' % engine._device_id)
    lut = np.zeros((N.POST_MAX_DEPTH, 128), np.uint64)
    mapped = np.zeros((128,), np.uint8)
    for key, value in self._value_mapping.items():
      ch = ord(key)
      if ch > 127:
        continue
      mapped[ch] = 1
      comps = np.atleast_1d(np.array(value)).astype(self._dtype)
      for i in range(self._depth):
        lut[i, ch] = int.from_bytes(comps[i].tobytes().ljust(8, b'\0'), 'little')
    d = N.EpilogueDesc()
    d.depth = self._depth
    d.out_dev = out.data_ptr()
    d.skip_layers = 2 if skip_board else int(bool(skip_layers))
    d.to_array = 1
    d.dtype = _DTYPES[self._dtype.name]
    d.lut = lut.ctypes.data
    d.mapped = mapped.ctypes.data
    # start from the current observation (environments a later step leaves untouched keep values that match their
    # board) -- computed BEFORE the kernel's epilogue is switched: if the engine has no planes to start from (an
    # earlier epilogue with skip_board) the array starts as zeros and nothing is left half-installed
    try:
      seed = ObservationToArray(self._value_mapping, self._dtype, self._permute)(engine._result()[0])
    except RuntimeError:
      seed = None
    try:
      N.check(N.lib().pcx_engine_set_epilogue(engine._native, ctypes.byref(d)))
    except NotImplementedError:
      return False
    if seed is not None:
      out.copy_(seed)
    engine._install_epilogue(self, out, only=skip_board)  # the ENGINE owns the epilogue (see ObservationToFeatureArray.fuse_into)
    self._fused = (engine, out, engine._steps_launched)
    return True

  def unfuse(self):
    """Takes the epilogue out of the engine's step kernel again."""
    if self._fused is not None:
      self._fused[0]._clear_epilogue(self)

  def _epilogue_gone(self):
    self._fused = None

  def _after_import(self, engine, out, restored):
    """Engine.import_state(): `out` holds what the EXPORTING engine's kernel wrote.  With the observation restored it
    is refilled from the restored planes; without, it counts as not written until the next step."""
    if restored:
      out.copy_(ObservationToArray(self._value_mapping, self._dtype, self._permute)(engine._result()[0]))
      self._fused = (engine, out, engine._steps_launched - 1)
    else:
      self._fused = (engine, out, engine._steps_launched)

  def __call__(self, observation):
    """Batch 1: a NumPy array as in the reference.  Batch > 1: a device tensor
    [B, ...] written in place by the kernel (no copy, no synchronisation); an
    unmapped character is then reported at a later call or by
    `check_errors()`."""
    if self._fused is not None and getattr(observation, '_source', None) is self._fused[0]:
      engine, out, attached_at = self._fused
      if engine._steps_launched > attached_at:  # a step has run since: the kernel wrote `out`
        return out
    source = _source_of(observation)
    self._post = _bound(self._post, source)
    if self._post is None:
      view, _ = source._planes_view()
      R, C = view.rows, view.cols
      d = N.PostDesc()
      d.kind, d.dtype, d.depth = N.POST_TO_ARRAY, _DTYPES[self._dtype.name], self._depth
      for key, value in self._value_mapping.items():
        ch = ord(key)
        if ch > 127:
          continue
        d.mapped[ch] = 1
        comps = np.atleast_1d(np.array(value)).astype(self._dtype)
        for i in range(self._depth):
          d.lut[i][ch] = int.from_bytes(comps[i].tobytes().ljust(8, b'\0'), 'little')
      if self._is_3d:
        perm3 = self._permute
      else:  # (rows, cols) permutation of the 2-D result
        perm3 = None if self._permute is None else (0,) + tuple(1 + a for a in self._permute)
      stride, shape = _strides((self._depth, R, C), perm3)
      d.stride[0], d.stride[1], d.stride[2] = stride
      if not self._is_3d:
        shape = shape[1:]
      self._post = _Post(source, d, self._dtype, (int(view.batch),) + tuple(shape))
    single = self._post.out_shape[0] == 1
    out, bad = self._post.run(host=single)
    if bad:
      self.check_errors()
    return out[0] if single else out

  def check_errors(self):
    """Synchronises; raises if an observation held a character without a value."""
    if self._post is not None and self._post.errors().any():
      raise RuntimeError(
          'This ObservationToArray only knows array values for the '
          'characters {}, but it received an observation with a character '
          'not in that set'.format(str(''.join(self._value_mapping.keys()))))


class ObservationToFeatureArray(object):
  """float32 stack of selected layers (rendering.py:545-661)."""

  def __init__(self, layers, permute=None):
    self._layers = layers
    self._depth = len(layers)
    self._permute = tuple(permute) if permute is not None else None
    if permute is not None and sorted(permute) != [0, 1, 2]:
      raise ValueError('The permute argument to the ObservationToFeatureArray '
                       'constructor must be a list or tuple containing some '
                       'permutation of the integers 0, 1, and 2.')
    if self._depth > N.POST_MAX_DEPTH:
      raise NotImplementedError('more than {} layers'.format(N.POST_MAX_DEPTH))
    self._post = None
    self._fused = None  # (engine, device tensor) once fuse_into() succeeded
    self._fused_window = None  # (cropper, device tensor, step count): fuse_into(engine, source=cropper)

  def fuse_into(self, engine, skip_layers=False, skip_board=False, source=None):
    """Have `engine`'s step kernel write this feature array itself, as an
    epilogue of its render loop (the layer masks are in registers there):
    from the next `play()` / `step()` on, calling this object with one of the
    engine's observations returns the tensor the step already filled -- no
    second pass over the planes, no extra launch.  `skip_layers=True` also
    stops the step from writing the uint8 layer planes (`Observation.layers`
    then goes stale; the board stays valid) for consumers that only ingest
    the features.  Returns False, and changes nothing, where the engine's
    kernel cannot do it (batch > 1; the five hand-written step kernels with
    occluded layers and no fused croppers; axis order default or channels
    last, `permute=(1, 2, 0)` -- the latter on boards of whole dwords): calls
    then run the post-processor as its own kernel, as before.  The
    engine owns the installed epilogue: when this object goes away, or another
    post-processor fuses, the kernel stops writing into this one's tensor.

    `source=cropper` -- crop, THEN post-process, in the one launch (the order
    of the reference's pipeline: human_ui.py:252-265, better_scrolly_maze.py:
    237-247 into rendering.py:545-661): `cropper` must be fused into the
    engine's step kernel (`cropping.fuse_croppers`); the kernel then also
    writes the feature stack OF ITS WINDOW, [B, depth, rows, cols] of the
    window (channels last: [B, rows, cols, depth]), and calling this object
    with one of the cropper's observations returns that tensor.  Here
    `skip_layers` / `skip_board` stop the kernel from writing the WINDOW's
    uint8 layer planes / board plane (with `fuse_croppers(..., only_crops=
    True)` a learner that ingests the egocentric feature stack gets exactly
    that and nothing else: better_scrolly_maze, 10x30 window of the 45x89
    board, eight layers: 9.6 KB per environment instead of 32 KB of planes
    plus a second pass).  False for the table-driven kernel, more than 16
    layers, a cropper that is not fused."""
    if source is not None:
      return self._fuse_into_window(engine, source, skip_layers, skip_board)
    torch = dev.torch_module()
    if (self._permute not in (None, (0, 1, 2), (1, 2, 0)) or torch is None or engine._native is None or engine.batch == 1 or
        len(set(self._layers)) != len(self._layers) or any(ord(c) > 255 for c in self._layers)):
      return False
    channels_last = self._permute == (1, 2, 0)
    shape = (engine.rows, engine.cols, self._depth) if channels_last else (self._depth, engine.rows, engine.cols)
    out = torch.zeros((engine.batch,) + shape, dtype=torch.float32, device='cuda:%d' % engine._device_id)
    d = N.EpilogueDesc()
    d.depth = self._depth
    for i, ch in enumerate(self._layers):
      d.chars[i] = ord(ch)
    d.out_dev = out.data_ptr()
    d.skip_layers = 2 if skip_board else int(bool(skip_layers))  # skip_board: not even the board plane (observations carry board=None)
    d.channels_last = int(channels_last)
    # start from the current observation (environments a later step leaves untouched keep features that match their
    # planes), computed before the kernel's epilogue is switched (see ObservationToArray.fuse_into)
    try:
      seed = ObservationToFeatureArray(self._layers, self._permute)(engine._result()[0])
    except RuntimeError:
      seed = None
    try:
      N.check(N.lib().pcx_engine_set_epilogue(engine._native, ctypes.byref(d)))
    except NotImplementedError:
      return False
    if seed is not None:
      out.copy_(seed)
    # The ENGINE owns the epilogue: it keeps this converter and the tensor the
    # kernel writes alive for as long as it may launch (a converter that was
    # garbage-collected would leave the kernel writing freed memory), tells the
    # converter it replaces that it is no longer fed, and lets go in close().
    engine._install_epilogue(self, out, only=skip_board)
    self._fused = (engine, out, engine._steps_launched)
    return True

  def unfuse(self):
    """Takes the epilogue out of the engine's step kernel again (calls then run
    the post-processor as its own kernel)."""
    if self._fused is not None:
      self._fused[0]._clear_epilogue(self)
    if self._fused_window is not None:
      cropper = self._fused_window[0]
      if cropper._native is not None:
        N.check(N.lib().pcx_cropper_set_features(cropper._native, None))
      cropper._features = None
      cropper._feat_skip = 0
      self._fused_window = None

  def _epilogue_gone(self):
    self._fused = None

  def _fuse_into_window(self, engine, cropper, skip_layers, skip_board):
    torch = dev.torch_module()
    if (torch is None or engine._native is None or engine.batch == 1 or cropper._engine is not engine or not cropper._fused or
        cropper._native is None or self._permute not in (None, (0, 1, 2), (1, 2, 0)) or
        len(set(self._layers)) != len(self._layers) or any(ord(c) > 255 for c in self._layers) or self._depth > 16):
      return False
    channels_last = self._permute == (1, 2, 0)
    shape = (cropper.rows, cropper.cols, self._depth) if channels_last else (self._depth, cropper.rows, cropper.cols)
    out = torch.zeros((engine.batch,) + shape, dtype=torch.float32, device='cuda:%d' % engine._device_id)
    d = N.EpilogueDesc()
    d.depth = self._depth
    for i, ch in enumerate(self._layers):
      d.chars[i] = ord(ch)
    d.out_dev = out.data_ptr()
    d.skip_layers = 2 if skip_board else int(bool(skip_layers))
    d.channels_last = int(channels_last)
    # (the window as it stands, through the stand-alone kernel: environments a later step leaves alone keep it)
    seed = ObservationToFeatureArray(self._layers, self._permute)(cropper.crop(None))
    try:
      N.check(N.lib().pcx_cropper_set_features(cropper._native, ctypes.byref(d)))
    except NotImplementedError:
      return False
    out.copy_(seed)
    if cropper._features is not None and cropper._features[0] is not self:
      cropper._features[0]._window_gone()
    cropper._features = (self, out)
    cropper._feat_skip = int(d.skip_layers)
    cropper._feat_skip_since = engine._steps_launched
    self._fused_window = (cropper, out, engine._steps_launched)
    return True

  def _window_gone(self):
    self._fused_window = None

  def _window_after_import(self, cropper, out, restored=True):
    """Engine.import_state() with a stack fused into `cropper`'s window: the tensor holds what the step kernel wrote
    before the import.  Refill it from the restored window through the stand-alone kernels (the window's uint8 planes
    are restored with the checkpoint's observation or recut by crop()); a window whose planes the kernel no longer
    writes (skip_layers / skip_board) cannot be recomputed and counts as not written until the next step -- and so does
    every window when the checkpoint carried no observation (`restored` False: crop(None) would recut it from the
    engine's full-board planes, which then still show the frame BEFORE the import)."""
    if self._fused_window is None or self._fused_window[0] is not cropper:
      return
    engine = cropper._engine
    if getattr(cropper, '_feat_skip', 0) or not restored:
      self._fused_window = (cropper, out, engine._steps_launched)  # (stale until a step rewrites it)
      return
    out.copy_(ObservationToFeatureArray(self._layers, self._permute)(cropper.crop(None)))
    self._fused_window = (cropper, out, engine._steps_launched - 1)

  def _after_import(self, engine, out, restored):
    """Engine.import_state(): see ObservationToArray._after_import."""
    if restored:
      out.copy_(ObservationToFeatureArray(self._layers, self._permute)(engine._result()[0]))
      self._fused = (engine, out, engine._steps_launched - 1)
    else:
      self._fused = (engine, out, engine._steps_launched)

  def __call__(self, observation):
    if self._fused_window is not None and getattr(observation, '_source', None) is self._fused_window[0]:
      cropper, out, attached_at = self._fused_window
      if cropper._fused and cropper._engine is not None and cropper._engine._steps_launched > attached_at:
        return out  # the step kernel cut the window and wrote its stack
    if self._fused is not None and getattr(observation, '_source', None) is self._fused[0]:
      engine, out, attached_at = self._fused
      if engine._steps_launched > attached_at:  # a step has run since: the kernel wrote `out`
        return out
    if getattr(observation, '_planes_stale', False):
      _source_of(observation)  # (raises, saying what the placeholder is: BEFORE the layers check, which its empty `layers` would fail with a misleading text)
    if not any(l in observation.layers for l in self._layers):
      raise RuntimeError(
          'The layers argument to this ObservationToFeatureArray, {}, has no '
          'entry that refers to an actual feature in the input observation. '
          'Actual features in the observation are {}.'.format(
              repr(self._layers), repr(''.join(sorted(observation.layers)))))
    source = _source_of(observation)
    self._post = _bound(self._post, source)
    if self._post is None:
      view, _ = source._planes_view()
      d = N.PostDesc()
      d.kind, d.dtype, d.depth = N.POST_FEATURE_ARRAY, N.F32, self._depth
      for i, ch in enumerate(self._layers):
        d.chars[i] = ord(ch) if ord(ch) < 256 else 255
      stride, shape = _strides((self._depth, view.rows, view.cols), self._permute)
      d.stride[0], d.stride[1], d.stride[2] = stride
      self._post = _Post(source, d, np.float32, (int(view.batch),) + tuple(shape))
    single = self._post.out_shape[0] == 1
    out, _ = self._post.run(host=single)  # float32 device tensor [B, ...] for batch > 1 (zero-copy hand-off)
    return out[0] if single else out


class ObservationCharacterRepainter(object):
  """Repaints characters through a fixed mapping (rendering.py:304-406)."""

  def __init__(self, character_mapping):
    self._character_mapping = character_mapping
    self._post = None
    self._out_chars = None
    self._repainted = None
    self._fused = None  # (engine, step count) once fuse_into() succeeded

  def fuse_into(self, engine, skip_layers=False, skip_board=False, force=False):
    """Have `engine`'s step kernel write the repainted observation itself (the
    board dword through the character table, every output layer by a byte-wise
    compare): from the next `play()` / `step()` on, calling this object with
    one of the engine's observations returns the planes the step already
    filled; they are a planes source as before (`ObservationToArray(...)(
    repainter(observation))` chains).  `skip_layers` / `skip_board`: the step
    no longer writes the original layer planes / any original plane.  Returns
    False, and changes nothing, where the engine's kernel cannot do it (batch
    1, boards that are not a whole number of dwords, the table-driven kernel,
    unoccluded layers, fused croppers) or where it would be slower than step +
    stand-alone kernel: batches whose planes no longer fit the Infinity Cache
    (`_general_epilogue_pays`; `force=True` fuses regardless)."""
    torch = dev.torch_module()
    if torch is None or engine._native is None or engine.batch == 1:
      return False
    if not (force or _general_epilogue_pays(engine)):
      return False
    obs = engine._result()[0]
    if obs.board is None:
      return False
    self(obs)  # creates the output planes (and brings them up to date with the current observation)
    if self._post.out is None or self._post.out.tensor is None:
      return False
    lut = np.zeros((N.POST_MAX_DEPTH, 128), np.uint64)
    lut[0, :] = np.arange(128)
    for k, v in self._character_mapping.items():
      lut[0, ord(k)] = ord(v)
    mapped = np.ones((128,), np.uint8)
    d = N.EpilogueDesc()
    d.depth = len(self._out_chars)
    for i, ch in enumerate(self._out_chars):
      d.chars[i] = ord(ch)
    d.out_dev = self._post.out.ptr
    d.skip_layers = 2 if skip_board else int(bool(skip_layers))
    d.to_array = 2
    d.dtype = N.U8
    d.lut = lut.ctypes.data
    d.mapped = mapped.ctypes.data
    try:
      N.check(N.lib().pcx_engine_set_epilogue(engine._native, ctypes.byref(d)))
    except NotImplementedError:
      return False
    engine._install_epilogue(self, self._post.out, only=skip_board)
    self._fused = (engine, engine._steps_launched)
    return True

  def unfuse(self):
    if self._fused is not None:
      self._fused[0]._clear_epilogue(self)

  def _epilogue_gone(self):
    self._fused = None

  def _after_import(self, engine, out, restored):
    """Engine.import_state(): the repainted planes are the exporting engine's; the next call repaints the restored
    observation with the stand-alone kernel (into the same planes), later ones take what the step kernel writes."""
    del out, restored
    self._fused = (engine, engine._steps_launched)

  def __call__(self, original_observation):
    fused_now = (self._fused is not None and getattr(original_observation, '_source', None) is self._fused[0] and
                 self._fused[0]._steps_launched > self._fused[1])
    if fused_now:
      return self._wrap(self._post.out.tensor)  # the step kernel wrote the planes
    source = _source_of(original_observation)
    self._post = _bound(self._post, source)
    if self._post is None:
      view, device_id = source._planes_view()
      self._out_chars = sorted((set(original_observation.layers) - set(self._character_mapping))
                               .union(self._character_mapping.values()))
      if len(self._out_chars) > N.POST_MAX_DEPTH:
        raise NotImplementedError('a repainted observation with more than {} characters'.format(N.POST_MAX_DEPTH))
      d = N.PostDesc()
      d.kind, d.dtype, d.depth = N.POST_REPAINT, N.U8, len(self._out_chars)
      for ch in range(128):
        d.lut[0][ch] = ch
        d.mapped[ch] = 1
      for k, v in self._character_mapping.items():
        if ord(k) > 127 or ord(v) > 127:
          raise ValueError('ObservationCharacterRepainter on the device repaints ASCII characters only')
        d.lut[0][ord(k)] = ord(v)
      for i, ch in enumerate(self._out_chars):
        d.chars[i] = ord(ch)
      pitch = (view.rows * view.cols + 3) & ~3
      self._post = _Post(source, d, np.uint8, (int(view.batch), 1 + len(self._out_chars), pitch))
      self._repainted = _RepaintedPlanes(self._post, self._out_chars, view.rows, view.cols, pitch, device_id, _engine_of(source))
    B = self._post.out_shape[0]
    planes, bad = self._post.run(host=B == 1)
    if bad and self._post.errors().any():
      raise RuntimeError('ObservationCharacterRepainter met a character outside ASCII')
    return self._wrap(planes)

  def _wrap(self, planes):
    B = self._post.out_shape[0]
    R, C, pitch = self._repainted.rows, self._repainted.cols, self._repainted.pitch
    if B == 1:
      planes = np.ascontiguousarray(planes[0, :, :R * C]).reshape(-1, R, C)
      obs = Observation(board=planes[0],
                        layers={c: planes[1 + i].astype(np.bool_) for i, c in enumerate(self._out_chars)})
    else:
      P = 1 + len(self._out_chars)
      if hasattr(planes, 'as_strided'):   # device tensor: zero-copy [B, P, rows, cols] view of the pitched planes
        view4 = planes.as_strided((B, P, R, C), (P * pitch, pitch, C, 1))
      else:
        view4 = np.ascontiguousarray(planes[:, :, :R * C]).reshape(B, P, R, C)
      obs = Observation(board=view4[:, 0], layers={c: view4[:, 1 + i] for i, c in enumerate(self._out_chars)})
    obs._source = self._repainted  # lets ObservationToArray / ToFeatureArray run on the repainted planes
    return obs


class _RepaintedPlanes(object):
  """The planes a repainter wrote, as a source for further post-processors."""

  def __init__(self, post, out_chars, rows, cols, pitch, device_id, origin):
    self._post, self._out_chars, self._origin = post, out_chars, origin
    self.rows, self.cols, self.pitch, self._device_id = rows, cols, pitch, device_id

  def _planes_view(self):
    ptr, nbytes = ctypes.c_void_p(), N.c_u64()
    N.check(N.lib().pcx_post_output(self._post.handle, ctypes.byref(ptr), ctypes.byref(nbytes)))
    view = N.PlanesView()
    view.planes = ptr.value
    view.batch = self._post.out_shape[0]
    view.rows, view.cols, view.pitch = self.rows, self.cols, self.pitch
    view.n_chars = len(self._out_chars)
    for i, ch in enumerate(self._out_chars):
      view.chars[i] = ord(ch)
    return view, self._device_id


# ---------------------------------------------------------------------- the first layer of a policy
#
# What a learner does with the stack ObservationToFeatureArray makes is, first of all, to multiply it by a weight.  The
# operators below do that from the boards themselves (csrc/pcx_project.hip): the float32 stack -- 9.6 KB per scrolly_maze
# board of 300 bytes -- is never written.  They need PyTorch-ROCm.

_ACTIVATIONS = {None: N.ACT_NONE, 'relu': N.ACT_RELU, 'silu': N.ACT_SILU, 'tanh': N.ACT_TANH, 'gelu': N.ACT_GELU}


def _engine_of(source):
  """The engine whose steps change what a source of planes (itself, a cropper, repainted planes) holds."""
  return getattr(source, '_engine', None) or getattr(source, '_origin', None) or source


def _written_of(source):
  return source._post.written if isinstance(source, _RepaintedPlanes) else source._written


def _occluded(source):
  """Are this source's layers exactly `board == character`?"""
  engine = getattr(source, '_engine', None) or source
  return bool(getattr(engine, '_occlusion_in_layers', False))


class _Boards(object):
  """Where a projection's boards lie: an Observation of this package, a uint8 tensor [n, rows, cols] of characters, or a
  uint8 / bool tensor [n, layers, rows, cols] of stacked layers."""

  def __init__(self, boards, layers):
    torch = dev.require_torch('a projection of observations')
    self.single = False
    self.offsets = None  # stacked layers: byte offsets within a board
    self.written = []  # of an Observation, or after watch(): [(what has been written, how often)]
    self.engine = None
    if isinstance(boards, torch.Tensor):
      self.keep, shape = boards, boards.shape
      if not boards.is_cuda:
        raise ValueError('boards must be a device tensor')
      if boards.dim() == 4:
        if boards.dtype not in (torch.uint8, torch.bool):
          raise TypeError('stacked layers must be uint8 or bool, not {}'.format(boards.dtype))
        if shape[1] != len(layers):
          raise ValueError('{} stacked layers for the {} characters {}'.format(shape[1], len(layers), repr(layers)))
        self.offsets = [k * boards.stride(1) for k in range(len(layers))]
      elif boards.dim() == 3:
        if boards.dtype != torch.uint8:
          raise TypeError('boards must be uint8 characters, not {}'.format(boards.dtype))
      else:
        raise ValueError('boards must be [n, rows, cols] characters or [n, layers, rows, cols] stacked layers, not '
                         '{}'.format(list(shape)))
      self.n, self.rows, self.cols = int(shape[0]), int(shape[-2]), int(shape[-1])
      if (self.cols > 1 and boards.stride(-1) != 1) or (self.rows > 1 and boards.stride(-2) != self.cols):
        raise ValueError('the cells of a board must lie one after the other (rows * cols contiguous bytes)')
      self.strides = boards.stride()
      self.device_id, self.ptr, self.row_stride = boards.device.index, boards.data_ptr(), int(self.strides[0])
    else:
      source = _source_of(boards)
      view, self.device_id = source._planes_view()
      present = bytes(view.chars)[:view.n_chars]
      if not any(ord(c) < 256 and ord(c) in present for c in layers):
        raise RuntimeError('The layers {} have no entry that refers to an actual feature in the input observation, whose '
                           'features are {}.'.format(repr(layers), repr(present.decode('latin-1'))))
      self.keep = boards
      engine = _engine_of(source)
      self.engine, self.written = engine, [(w, w.count) for w in (engine._written, _written_of(source))]
      self.n, self.rows, self.cols = int(view.batch), view.rows, view.cols
      self.ptr, self.row_stride = view.planes, (1 + view.n_chars) * view.pitch
      self.single = self.n == 1
      if not _occluded(source):
        self.offsets = [(1 + present.index(ord(c))) * view.pitch if ord(c) in present else -1 for c in layers]

  def watch(self):
    """A backward pass is to come.  (Of a tensor's writes autograd knows, but for what this package's kernels write to it.)"""
    if isinstance(self.keep, dev.torch_module().Tensor):
      written = dev.Written.of(self.keep)
      self.written = [] if written is None else [(written, written.count)]
    return self

  def check_unchanged(self, what):
    """In a backward pass: do the boards still show what the forward pass read?"""
    if (self.engine is not None and self.engine._native is None) or any(w.count != count for w, count in self.written):
      raise RuntimeError('{}(): the boards were overwritten by a later step (or crop, or conversion), or their engine closed, '
                         'before the backward pass: pass a copy of the board, a tensor of its own'.format(what))


_NO_OFFSETS = bytes(8 * N.POST_MAX_DEPTH)
_project_sizes = {}


class _Projection(object):
  """The checked arguments of one projection: what the C ABI's description is made of."""

  def __init__(self, layers, weight, bias, activation):
    torch = dev.require_torch('a projection of observations')
    if activation not in _ACTIVATIONS:
      raise ValueError('activation must be one of {}, not {}'.format(list(_ACTIVATIONS), repr(activation)))
    depth = len(layers)
    if not 1 <= depth <= N.POST_MAX_DEPTH:
      raise NotImplementedError('a projection takes 1 to {} layers, not {}'.format(N.POST_MAX_DEPTH, depth))
    if any(ord(c) > 255 for c in layers) or len(set(layers)) != depth:
      raise ValueError('layers must be distinct one-byte characters, not {}'.format(repr(layers)))
    if not isinstance(weight, torch.Tensor) or not weight.is_cuda:
      raise ValueError('weight must be a device tensor')
    self.dtype = dev.policy_dtype(weight, 'weight')
    if weight.dim() not in (2, 4) or weight.numel() == 0 or (weight.shape[1] != depth if weight.dim() == 4 else weight.shape[1] % depth):
      raise ValueError('weight must be [hidden, {0}, rows, cols] or [hidden, {0} * rows * cols], not {1}'.format(depth, list(weight.shape)))
    self.layers, self.hidden, self.device = layers, int(weight.shape[0]), weight.device
    self.cells = int(weight.numel()) // (self.hidden * depth)
    self.board = tuple(weight.shape[2:]) if weight.dim() == 4 else None
    self.check_row(bias, 'bias', weight)
    if bias is not None and tuple(bias.shape) != (self.hidden,):
      raise ValueError('bias must be [{}], not {}'.format(self.hidden, list(bias.shape)))
    self.torch_dtype, self.activation = weight.dtype, _ACTIVATIONS[activation]
    chars = layers.encode('latin-1') if isinstance(layers, str) else bytes(ord(c) for c in layers)
    self.tails = [N.PROJECT_TAIL.pack(self.cells, depth, self.hidden, self.dtype, self.activation, stacked, chars) for stacked in (0, 1)]

  def check_row(self, tensor, name, weight):
    if tensor is not None and (tensor.dtype != weight.dtype or tensor.device != weight.device):
      raise ValueError('{} must be {} on {}, like the weight'.format(name, weight.dtype, weight.device))

  def slope_dtype(self):
    return self.torch_dtype if self.activation == N.ACT_RELU else dev.torch_module().float32

  def check_rows(self, tensor, name, n, dtype=None):
    if tensor is None:
      return
    if tensor.dtype != (dtype or self.torch_dtype) or tensor.device != self.device or tuple(tensor.shape) != (n, self.hidden):
      raise ValueError('{} must be {} [{}, {}] on {}'.format(name, dtype or self.torch_dtype, n, self.hidden, self.device))

  def at(self, boards):
    """The description (the bytes of a pcx_project_desc) for these boards."""
    if boards.device_id != self.device.index:
      raise ValueError('the boards are on GPU {}, the weight is on GPU {}'.format(boards.device_id, self.device.index))
    if boards.rows * boards.cols != self.cells or (self.board and self.board != (boards.rows, boards.cols)):
      raise ValueError('the weight is for boards of {} cells, these are {} x {}'.format(
          '{} x {}'.format(*self.board) if self.board else self.cells, boards.rows, boards.cols))
    if boards.offsets is None:
      return N.PROJECT_HEAD.pack(boards.n, boards.row_stride) + _NO_OFFSETS + self.tails[0]
    return (N.PROJECT_HEAD.pack(boards.n, boards.row_stride) +
            N.PROJECT_OFFSETS.pack(*boards.offsets, *([0] * (N.POST_MAX_DEPTH - len(boards.offsets)))) + self.tails[1])

  @staticmethod
  def sizes(desc):
    """Bytes of (the laid-out weight, the forward workspace, the backward workspace)."""
    found = _project_sizes.get(desc)
    if found is None:
      out = (N.c_u64(0), N.c_u64(0), N.c_u64(0))
      N.check(N.lib().pcx_project_sizes(desc, *[ctypes.byref(x) for x in out]))
      if len(_project_sizes) > 4096:
        _project_sizes.clear()
      found = _project_sizes[desc] = tuple(int(x.value) for x in out)
    return found

  def pack(self, desc, weight, packed=None):
    torch = dev.torch_module()
    if packed is None:
      packed = torch.empty(self.sizes(desc)[0], dtype=torch.uint8, device=self.device)
    if not weight.is_contiguous():
      weight = weight.detach().contiguous()
    dev.launch(self.device.index, N.lib().pcx_project_pack, desc, weight.data_ptr(), packed.data_ptr())
    return packed

  def forward(self, desc, boards, packed, bias, residual, want_slope=False):
    torch = dev.torch_module()
    if residual is not None:
      self.check_rows(residual, 'residual', boards.n)
      residual = residual.contiguous()
    out = torch.empty((boards.n, self.hidden), dtype=self.torch_dtype, device=self.device)
    slope = torch.empty_like(out, dtype=self.slope_dtype()) if want_slope else None
    size = self.sizes(desc)[1]
    scratch = packed.new_empty(size) if size else None
    if bias is not None and not bias.is_contiguous():
      bias = bias.contiguous()
    dev.launch(self.device.index, N.lib().pcx_project_forward, desc, boards.ptr, packed.data_ptr(), dev.pointer(bias), dev.pointer(residual),
               out.data_ptr(), dev.pointer(slope), dev.pointer(scratch), size)
    return out, slope

  def backward(self, desc, boards, grad, slope, want_weight, want_bias, weight_shape):
    # (autograd calls this on a thread of its own, where every line costs several times what it does elsewhere)
    make = grad.new_zeros if boards.n == 0 else grad.new_empty
    dw = make(weight_shape) if want_weight else None
    db = make(self.hidden) if want_bias else None
    if boards.n and (want_weight or want_bias):
      size = self.sizes(desc)[2]
      scratch = grad.new_empty(size, dtype=dev.torch_module().uint8)
      grad = grad.contiguous()
      slope = None if slope is None else slope.contiguous()
      dev.launch(self.device.index, N.lib().pcx_project_backward, desc, boards.ptr, grad.data_ptr(), dev.pointer(slope), dev.pointer(dw),
                 dev.pointer(db), scratch.data_ptr(), size)
    return dw, db


class ObservationProjection(object):
  """`act(features @ weight.T + bias) + residual` of every board, with `features` the stack that
  `ObservationToFeatureArray(layers)` would make of it -- for a policy that is only asked.

  `weight`: float32, float16 or bfloat16 device tensor, [hidden, len(layers), rows, cols] or the same flattened to two
  axes (a Linear layer's weight over the flattened stack); `bias`: [hidden] or None; `activation`: None, 'relu', 'silu',
  'tanh' or 'gelu' (the exact one).  The weight is copied and laid out once, here and in `load()`: later changes of the
  tensors do not show until `load()` is called.

  Calling it takes an Observation of this package (engine, cropper or repainter; nothing is copied), a uint8 device
  tensor [n, rows, cols] of board characters -- say, boards kept from a rollout -- or a uint8 / bool tensor
  [n, len(layers), rows, cols] of stacked layers, and returns [n, hidden] of the weight's type (a batch-1 Observation:
  [hidden]).  `residual`: [n, hidden] or None.  Boards whose layers are `board == character` (the default engine) are
  read as characters; with `occlusion_in_layers=False` the layer planes are read.  Characters of a board that are not
  among `layers` count nowhere.  Sums are float32.  Nothing waits for the device, so a call can be captured into a graph
  (keep this object as long as the graph); gradients are `project()`'s business."""

  def __init__(self, layers, weight, bias=None, activation=None):
    self._activation = activation
    self._layers = layers
    self._plan = _Projection(layers, weight, bias, activation)
    self._weight = weight.detach().clone()
    self._bias = None if bias is None else bias.detach().clone()
    self._packs = {}
    self._streams = set()  # (stacked, stream) that a laid-out weight has been used on
    self._lay_out(0)

  def _lay_out(self, stacked):
    """The weight in the order the kernel for characters (0) or stacked layers (1) reads it; waits until it lies there,
    so that calls on any stream may use it."""
    torch = dev.torch_module()
    if torch.cuda.is_current_stream_capturing():
      raise RuntimeError('this ObservationProjection has not laid its weight out for stacked layers yet: call it once before '
                         'capturing a graph')
    desc = N.PROJECT_HEAD.pack(0, 0) + _NO_OFFSETS + self._plan.tails[stacked]  # (the layout depends on the weight alone)
    self._packs[stacked] = self._plan.pack(desc, self._weight, self._packs.get(stacked))
    torch.cuda.current_stream(self._plan.device).synchronize()

  def load(self, weight, bias=None):
    """New values for weight and bias (same shapes and types), in place: graphs that captured a call see them.  Waits for
    the device, before and after."""
    torch = dev.torch_module()
    if torch.cuda.is_current_stream_capturing():
      raise RuntimeError('load() cannot be captured into a graph')
    if tuple(weight.shape) != tuple(self._weight.shape) or weight.dtype != self._weight.dtype or (bias is None) != (self._bias is None):
      raise ValueError('load() takes a weight {} {} and {} bias'.format(self._weight.dtype, list(self._weight.shape),
                                                                       'no' if self._bias is None else 'a'))
    _Projection(self._layers, weight, bias, self._activation)  # (checks)
    torch.cuda.synchronize(self._plan.device)  # nobody reads the old values any more
    with torch.inference_mode():  # (made in it, the copies can be written nowhere else)
      self._weight.copy_(weight)
      if bias is not None:
        self._bias.copy_(bias)
    for stacked in list(self._packs):
      self._lay_out(stacked)
    torch.cuda.synchronize(self._plan.device)

  def __call__(self, observation, residual=None):
    boards = _Boards(observation, self._layers)
    desc = self._plan.at(boards)
    stacked = int(boards.offsets is not None)
    if stacked not in self._packs:
      self._lay_out(stacked)
    used = stacked, dev.raw_stream(self._plan.device.index)
    if used not in self._streams:
      # (their memory is not given to others, when this object goes, before that stream has passed the calls made on it)
      stream = dev.torch_module().cuda.current_stream(self._plan.device)
      for kept in (self._packs[stacked], self._bias):
        if kept is not None:
          kept.record_stream(stream)
      self._streams.add(used)
    out, _ = self._plan.forward(desc, boards, self._packs[stacked], self._bias, None if residual is None else residual.detach())
    return out[0] if boards.single else out


_project_function = None


def _project_autograd():
  """The autograd function behind `project()` (made on first use: PyTorch is optional here)."""
  global _project_function
  if _project_function is None:
    torch = dev.torch_module()
    grad_enabled = torch.is_grad_enabled

    class ProjectBoards(torch.autograd.Function):

      @staticmethod
      def forward(ctx, weight, bias, residual, plan, boards, desc):
        out, slope = plan.forward(desc, boards, plan.pack(desc, weight), bias, residual, want_slope=plan.activation != N.ACT_NONE)
        ctx.plan, ctx.boards, ctx.desc, ctx.weight_shape = plan, boards, desc, weight.shape
        # (the boards are an input like any other, where they are a tensor and the weight's gradient reads them: a write to
        # them before backward() is noticed)
        ctx.save_for_backward(slope, boards.keep if ctx.needs_input_grad[0] and isinstance(boards.keep, torch.Tensor) else None)
        return out

      @staticmethod
      def backward(ctx, grad):
        if grad_enabled():
          dev.refuse_twice('project')
        slope, saved = ctx.saved_tensors
        plan, boards, desc, want = ctx.plan, ctx.boards, ctx.desc, ctx.needs_input_grad
        if saved is not None and (saved.data_ptr() != boards.ptr or saved.stride() != boards.strides):
          # (what was saved went elsewhere meanwhile -- torch.autograd.graph.saved_tensors_hooks, checkpoint -- and what came
          # back, as it was then, is laid out in its own way)
          boards = _Boards(saved, plan.layers)
          desc = plan.at(boards)
          if boards.n != ctx.boards.n:
            raise ValueError('project(): {} boards came back of {} saved'.format(boards.n, ctx.boards.n))
        elif want[0]:
          boards.check_unchanged('project')
        plan.check_rows(slope, 'slope', boards.n, plan.slope_dtype())
        dw, db = plan.backward(desc, boards, grad, slope, want[0], want[1], ctx.weight_shape)
        return dw, db, grad if want[2] else None, None, None, None

    _project_function = ProjectBoards
  return _project_function


def project(boards, layers, weight, bias=None, activation=None, residual=None, return_slope=False):
  """`act(features @ weight.T + bias) + residual`, differentiable in `weight`, `bias` and `residual` (once, in reverse
  mode): one training step's first layer.  Arguments, shapes and types as for `ObservationProjection`, which is the form for weights that stay; this
  one lays the weight out in every call.

  An Observation, its board and what a converter returned are views of arrays that the next step, crop or conversion
  overwrites: a backward pass after that is refused (where a replayed graph wrote them, nobody knows: do not); pass a copy
  of the board (`observation.board.clone()`).  A weight that is no finite number makes the results of the boards that use it
  no finite numbers, and of others some.

  `return_slope=True`: no autograd; returns (out, slope) with slope = act'(...) (None without an activation), what
  `project_backward` takes -- the pair to capture into a graph."""
  torch = dev.require_torch('project()')
  plan = _Projection(layers, weight, bias, activation)
  if not return_slope and weight.requires_grad and torch.is_grad_enabled():
    boards = dev.saveable(torch, boards)
  view = _Boards(boards, layers)
  desc = plan.at(view)
  plan.check_rows(residual, 'residual', view.n)
  if not return_slope:
    dev.refuse_tangents('project', weight, bias, residual)
  if not return_slope and torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (weight, bias, residual)):
    dev.refuse_recording_in_capture('project', 'project(..., return_slope=True) and project_backward()')
    out = _project_autograd().apply(weight, bias, residual, plan, view.watch(), desc)
    return out[0] if view.single else out
  bias, residual = (None if t is None else t.detach() for t in (bias, residual))
  out, slope = plan.forward(desc, view, plan.pack(desc, weight), bias, residual, want_slope=return_slope and activation is not None)
  out = out[0] if view.single else out
  return (out, slope) if return_slope else out


def project_backward(boards, layers, weight, grad, slope=None, activation=None):
  """(grad_weight, grad_bias) of `project()` for the gradient `grad` of its result ([n, hidden]; of a batch-1 Observation
  [hidden] too); `slope` as it returned it, `activation` as it was given.  The residual's gradient is `grad`.  Records
  nothing for autograd and waits for nothing: it may be captured.

  Without `activation`, the gradient is multiplied by the slopes, and where a slope is 0 nothing comes through; named, a
  smooth activation's slope of 0 makes an infinite gradient a NaN, as its formula does."""
  dev.require_torch('project_backward()')
  if activation is None and slope is not None:
    # (16-bit weights: relu's slopes have their type, the others' are float32.  float32 weights: relu's rule multiplies by
    # any slope and lets nothing through at 0.)
    activation = 'relu' if slope.dtype == weight.dtype else 'silu'
  elif activation is not None and slope is None:
    raise ValueError('project_backward() needs the slopes of {}'.format(activation))
  plan = _Projection(layers, weight, None, activation)
  view = _Boards(boards, layers)
  desc = plan.at(view)
  if view.single and grad.dim() == 1:
    grad = grad[None]
  plan.check_rows(grad, 'grad', view.n)
  plan.check_rows(slope, 'slope', view.n, plan.slope_dtype())
  return plan.backward(desc, view, grad.detach(), slope, True, True, weight.shape)
