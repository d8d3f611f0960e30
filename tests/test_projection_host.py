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
