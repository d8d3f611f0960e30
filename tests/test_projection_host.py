"""CPU: the host side of the pre-norm projections, on stand-ins for device tensors."""


class _OnDevice:
  """What _workspace asks of a tensor."""

  def __init__(self, device):
    self.device = device

  def get_device(self):
    return self.device

  def new_empty(self, shape, dtype):
    return self.device, shape


def test_workspace_sizes_are_kept_by_device(monkeypatch):
  """Two devices with different numbers of SMs need different workspaces for the same call; each size is asked once."""
  from faster_weathernext import _lib
  from faster_weathernext import projection
  monkeypatch.setattr(projection, "_WORKSPACE", {})
  desc = _lib.LinearDesc(64, 32, 48, 0, 0, 1, 0, 0, 0, 48, 48, 32, 32)
  asked = []

  def size_of(device):
    def call(_desc, _a, _b, need):
      asked.append(device)
      need.value = 256 * (device + 1)
      return _lib.FWN_OK
    return call

  for device in (0, 1, 0, 1):
    ws, size = projection._workspace(_OnDevice(device), desc, size_of(device), 256, 512)
    assert size == 256 * (device + 1) and ws == (device, (size,))
  assert asked == [0, 1]


def test_tensors_off_their_elements_are_refused():
  """A float32 tensor at an address off 4 bytes, a bf16 one off 2: refused by every entry point before any CUDA call."""
  from faster_weathernext import _lib
  lib, bad = _lib.lib(), _lib.FWN_ERR_INVALID_ARGUMENT
  rms = _lib.RmsDesc(4, 64, 1, 0, 1, 0, 0, 1e-6, 0, 64, 64)  # float32 x and weight, bf16 residual and out
  good = [256, 256, 256, 256, 256, None]                     # x, residual, weight, x_out, out, scale
  for i, off in enumerate((258, 257, 258, 258, 257)):
    assert lib.fwn_rms_norm(rms, *good[:i], off, *good[i + 1:], 0) == bad
  fp8 = _lib.RmsDesc(4, 64, 1, 0, 1, 2, 0, 1e-6, 0, 64, 64)
  assert lib.fwn_rms_norm(fp8, 256, None, None, None, 257, 258, 0) == bad  # the scale; e4m3 values start anywhere
  good = [256] * 8                                           # x, residual, weight, dh, ds, dx, d_residual, d_weight
  for i, off in enumerate((258, 257, 258, 257, 258, 258, 257, 258)):
    assert lib.fwn_rms_norm_bwd(rms, *good[:i], off, *good[i + 1:], 256, 1 << 30, 0) == bad
  lin = _lib.LinearDesc(4, 32, 48, 0, 1, 1, 1, 0, 0, 48, 48, 32, 32)       # float32 bias, residual and out
  good = [256, None, 256, None, 256, 256, 256, None]         # a, a_scale, b, b_scale, bias, x, out, d_bias
  for i, off in ((0, 257), (2, 257), (4, 258), (5, 258), (6, 258)):
    assert lib.fwn_linear(lin, *good[:i], off, *good[i + 1:], None, 0, 0) == bad
  lin8 = _lib.LinearDesc(4, 32, 48, 2, 1, 1, 1, 0, 0, 48, 48, 32, 32)
  for scales in ((258, 256), (256, 258)):
    assert lib.fwn_linear(lin8, 257, scales[0], 257, scales[1], None, None, 256, None, None, 0, 0) == bad
  assert lib.fwn_linear_pack(257, 48, 256, 48, 4, 48, 0, 0) == bad
  good = [256, 256, 256, 256, 256, 256, 256]                 # a, b, bias, dy, d_a, d_b, d_bias
  for i, off in enumerate((257, 257, 258, 258, 257, 257, 258)):
    assert lib.fwn_linear_bwd(lin, *good[:i], off, *good[i + 1:], 256, 1 << 30, 0) == bad
  assert b"elements" in lib.fwn_last_error_string()


def test_a_run_of_k_beyond_the_waits_limit_is_refused():
  """An output tile's run of k that takes seconds would end in a wait that gives up; few rows have none."""
  import ctypes
  from faster_weathernext import _lib
  lib, k = _lib.lib(), 2 ** 30
  size = ctypes.c_size_t(7)
  lin = lambda m, k, flags=0, act=0: _lib.LinearDesc(m, 32, k, 0, 0, 1, 0, act, flags, k, k, 32, 32)  # noqa: E731
  grad = lin(64, k, _lib.LINEAR_PRE_GRAD, _lib.ACT_GELU_TANH)     # the gradient of the pre-activation: k is not split
  assert lib.fwn_linear_workspace_size(grad, 256, 256, size) == _lib.FWN_ERR_UNSUPPORTED
  assert lib.fwn_linear(grad, 256, None, 256, None, 256, 256, 256, None, 256, 1 << 40, 0) == _lib.FWN_ERR_UNSUPPORTED
  assert lib.fwn_linear_workspace_size(lin(64, 2 ** 31 - 2048), 256, 256, size) == _lib.FWN_ERR_UNSUPPORTED
  assert lib.fwn_linear_workspace_size(lin(64, 2 ** 26), 256, 256, size) == _lib.FWN_OK and size.value > 0
  assert lib.fwn_linear_workspace_size(lin(8, k), 256, 256, size) == _lib.FWN_OK and size.value == 0
