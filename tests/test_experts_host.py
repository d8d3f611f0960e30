"""CPU: refusals of the products grouped by expert and of the routing (Python and C), before any CUDA call."""
import ctypes

import pytest
import torch


def _grouped(lib_mod, **kw):
  d = dict(m=64, groups=3, n=32, k=48, out_dtype=0, bias_dtype=1, x_dtype=0, act=0, flags=0, lda=48, ldb=48, b_stride=1536,
           ldx=32)
  d.update(kw)
  return lib_mod.GroupedDesc(*d.values())


def test_grouped_refusals():
  from faster_weathernext import _lib
  lib = _lib.lib()
  bad, no, room = _lib.FWN_ERR_INVALID_ARGUMENT, _lib.FWN_ERR_UNSUPPORTED, _lib.FWN_ERR_WORKSPACE

  def call(desc, a=256, b=256, bias=None, offsets=256, out=256, ws=None, n=0):
    return lib.fwn_linear_grouped(desc, a, b, bias, offsets, out, ws, n, 0)

  def back(desc, a=256, b=256, bias=None, offsets=256, dy=256, da=256, db=256, dbias=None, ws=None, n=0):
    return lib.fwn_linear_grouped_bwd(desc, a, b, bias, offsets, dy, da, db, dbias, ws, n, 0)

  for f in (call, back):
    assert f(None) == bad
    for kw in (dict(m=-1), dict(groups=0), dict(n=0), dict(k=0), dict(out_dtype=2), dict(bias_dtype=2), dict(x_dtype=2), dict(act=3),
               dict(flags=1), dict(flags=4), dict(lda=47), dict(ldb=47), dict(b_stride=47)):
      assert f(_grouped(_lib, **kw)) == bad, kw
    for kw in (dict(groups=1024), dict(m=2 ** 31 - 1), dict(n=2 ** 20 + 1, ldx=2 ** 20 + 1), dict(k=2 ** 20 + 1, lda=2 ** 21, ldb=2 ** 21, b_stride=2 ** 30),
               dict(lda=52), dict(ldb=52), dict(b_stride=1540)):
      assert f(_grouped(_lib, **kw)) == no, kw
    assert f(_grouped(_lib), a=None) == bad and f(_grouped(_lib), b=None) == bad and f(_grouped(_lib), offsets=None) == bad
    assert f(_grouped(_lib), a=257) == bad and f(_grouped(_lib), offsets=258) == bad
    assert f(_grouped(_lib), a=264) == no and f(_grouped(_lib), b=264) == no      # not where a TMA copy may start
    assert f(_grouped(_lib)) == room and f(_grouped(_lib), ws=256, n=100) == room and f(_grouped(_lib), ws=272, n=1 << 30) == room
  assert call(_grouped(_lib), out=None) == bad
  assert call(_grouped(_lib, m=0), a=None, b=None, offsets=None, out=None) == _lib.FWN_OK
  assert back(_grouped(_lib), dy=None) == bad and back(_grouped(_lib, ldx=31)) == bad
  assert back(_grouped(_lib), dbias=256) == bad                                   # d_bias without a bias
  size = ctypes.c_size_t(7)
  assert lib.fwn_linear_grouped_workspace_size(_grouped(_lib), None) == bad
  assert lib.fwn_linear_grouped_workspace_size(_grouped(_lib, m=0), size) == _lib.FWN_OK and size.value == 0
  assert lib.fwn_linear_grouped_workspace_size(_grouped(_lib, m=8), size) == _lib.FWN_OK and size.value == 0   # few rows
  assert lib.fwn_linear_grouped_bwd_workspace_size(_grouped(_lib, n=0), 256, size) == bad
  assert lib.fwn_linear_grouped_bwd_workspace_size(_grouped(_lib), 256, size) == _lib.FWN_OK and size.value > 0


@pytest.mark.parametrize("flags", [0, 2])
@pytest.mark.parametrize("act", [0, 1])
def test_grouped_plans(flags, act):
  """Every size has a plan; its workspace grows neither with what is not there nor beyond a few times the operands."""
  from faster_weathernext import _lib
  lib = _lib.lib()
  size = ctypes.c_size_t(0)
  for m in (1, 2, 9, 100, 5000, 163848, 2 ** 26):
    for groups in (1, 2, 8, 64, 1023):
      for n, k in ((8, 8), (64, 4096), (512, 2048), (2048, 512)):
        ldb, stride = (n, n * k) if flags else (k, n * k)
        desc = _lib.GroupedDesc(m, groups, n, k, 0, 1, 0, act, flags, k, ldb, stride, n)
        assert lib.fwn_linear_grouped_workspace_size(desc, size) == _lib.FWN_OK
        assert size.value <= 2 * 128 * 1024 + 16384
        assert lib.fwn_linear_grouped_bwd_workspace_size(desc, 256, size) == _lib.FWN_OK
        # d_pre, sums of 32 rows, maps, and parts of the weights' gradient: as many as fill the card, or as experts.
        assert size.value <= 2 * m * n + m * n // 4 + 8 * 128 * 1024 + 4 * n * (m // 32 + 8 * groups) + 4 * n * k * (260 + 2 * min(groups, m)) + 2 ** 20


def _route(lib_mod, **kw):
  d = dict(rows=300, experts=8, top=2, dtype=1, reserved=0)
  d.update(kw)
  return lib_mod.RouteDesc(*d.values())


def test_route_refusals():
  from faster_weathernext import _lib
  lib = _lib.lib()
  bad, no = _lib.FWN_ERR_INVALID_ARGUMENT, _lib.FWN_ERR_UNSUPPORTED

  def call(desc, logits=256, stride=8, experts=256, weights=256, order=256, position=256, offsets=256, ws=256, n=1 << 20):
    return lib.fwn_route(desc, logits, stride, experts, weights, order, position, offsets, ws, n, 0)

  assert call(None) == bad
  for kw in (dict(rows=-1), dict(experts=0), dict(top=0), dict(top=9), dict(dtype=2)):
    assert call(_route(_lib, **kw)) == bad, kw
  for kw in (dict(experts=1024), dict(experts=100, top=17), dict(rows=2 ** 30)):
    assert call(_route(_lib, **kw), stride=2000) == no, kw
  for kw in (dict(logits=None), dict(stride=7), dict(experts=None), dict(weights=None), dict(order=None), dict(position=None),
             dict(offsets=None), dict(logits=258), dict(order=257)):
    assert call(_route(_lib), **kw) == bad, kw
  assert call(_route(_lib), ws=None, n=0) == _lib.FWN_ERR_WORKSPACE and call(_route(_lib), n=8) == _lib.FWN_ERR_WORKSPACE
  size = ctypes.c_size_t(7)
  assert lib.fwn_route_workspace_size(_route(_lib, rows=128), size) == _lib.FWN_OK and size.value == 0
  assert lib.fwn_route_workspace_size(_route(_lib), None) == bad
  assert lib.fwn_route_bwd(_route(_lib), 256, 256, None, 256, 0) == bad and lib.fwn_route_bwd(_route(_lib, rows=0), None, None, None, None, 0) == _lib.FWN_OK
  spread = lambda desc, d=64, x=256, stride=64, pos=256, w=None, y=None, out=256, dots=None: lib.fwn_route_spread(  # noqa: E731
      desc, d, x, stride, pos, w, y, out, dots, 0)
  assert spread(_route(_lib), d=0) == bad and spread(_route(_lib), stride=63) == bad and spread(_route(_lib), x=None) == bad
  assert spread(_route(_lib), y=256) == bad and spread(_route(_lib), dots=256) == bad and spread(_route(_lib), out=None) == bad
  assert spread(_route(_lib), x=258) == bad and spread(_route(_lib, rows=0), x=None, pos=None, out=None) == _lib.FWN_OK
  gather = lambda desc, d=64, y=256, pos=256, w=None, out=256: lib.fwn_route_gather(desc, d, y, pos, w, out, 0)  # noqa: E731
  assert gather(_route(_lib), d=-1) == bad and gather(_route(_lib), y=None) == bad and gather(_route(_lib), out=None) == bad
  assert gather(_route(_lib, rows=0), y=None, pos=None, out=None) == _lib.FWN_OK


def test_python_refusals():
  from faster_weathernext import experts
  with pytest.raises(ValueError):
    experts.linear_grouped(torch.zeros(4, 8), torch.zeros(2, 3, 7), torch.zeros(3, dtype=torch.int32))
  with pytest.raises(TypeError):
    experts.linear_grouped(torch.zeros(4, 8), torch.zeros(2, 3, 8), torch.zeros(3, dtype=torch.int32))
  with pytest.raises(ValueError, match="CUDA"):
    experts.route(torch.zeros(4, 8), 2)
  with pytest.raises(ValueError):
    experts.route(torch.zeros(4), 1)
