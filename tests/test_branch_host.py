"""CPU: refusals of the residual branches (Python and C) and the oracle's generator against its published vectors."""
import ctypes

import numpy as np
import pytest
import torch


def test_philox_published_vectors():
  """The known answers that the generator's authors publish with it (Random123, kat_vectors: philox4x32, 10 rounds)."""
  from oracle import dropout
  got = lambda c, k: [f"{w:08x}" for w in dropout.philox4x32(np.array([c], np.uint64), k)[0]]  # noqa: E731
  assert got([0, 0, 0, 0], (0, 0)) == ["6627e8d5", "e169c58d", "bc57ac4c", "9b00dbd8"]
  f = 0xFFFFFFFF
  assert got([f, f, f, f], (f, f)) == ["408f276d", "41c83b0e", "a20bc7c6", "6d5451fd"]
  assert got([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], (0xa4093822, 0x299f31d0)) == \
      ["d16cfe09", "94fdcceb", "5001e420", "24126ea1"]


def test_mask_factors():
  from oracle import dropout
  f = dropout.factors((1000, 64), 0.25, 7)
  assert set(np.unique(f)) == {0.0, 65536 / (65536 - 16384)}
  assert abs((f == 0).mean() - 0.25) < 5 * (0.25 * 0.75 / f.size) ** 0.5
  assert np.array_equal(dropout.factors((64,), 0.25, 7, first=640), f.reshape(-1)[640:704])
  assert not np.array_equal(dropout.factors((1000, 64), 0.25, 7, site=1), f)
  assert not dropout.factors((5,), 1.0, 3).any() and (dropout.factors((5,), 1e-6, 3) == 1).all()


def _drop(lib_mod, **kw):
  d = dict(seed=1, seed_at=None, site=0, threshold=6554)
  d.update(kw)
  return lib_mod.DropoutDesc(*d.values())


def _branch(lib_mod, **kw):
  d = dict(rows=6, x_stride=64, y_stride=64, gate_span=6, d=64, x_dtype=1, y_dtype=0, post_dtype=1, weight_dtype=1,
           gate_dtype=1, out_dtype=0, eps=1e-6, residual_scale=1.0, reserved=0, drop=lib_mod.DropoutDesc())
  d.update(kw)
  return lib_mod.BranchDesc(*d.values())


def test_dropout_refusals():
  from faster_weathernext import _lib
  lib = _lib.lib()
  bad, no = _lib.FWN_ERR_INVALID_ARGUMENT, _lib.FWN_ERR_UNSUPPORTED
  assert lib.fwn_dropout(None, 256, 256, 8, 0, 0) == bad
  assert lib.fwn_dropout(_drop(_lib, threshold=65537), 256, 256, 8, 0, 0) == bad
  assert lib.fwn_dropout(_drop(_lib, seed_at=260), 256, 256, 8, 0, 0) == bad
  assert lib.fwn_dropout(_drop(_lib), 256, 256, -1, 0, 0) == bad and lib.fwn_dropout(_drop(_lib), 256, 256, 8, 2, 0) == bad
  assert lib.fwn_dropout(_drop(_lib), None, 256, 8, 0, 0) == bad and lib.fwn_dropout(_drop(_lib), 256, None, 8, 0, 0) == bad
  assert lib.fwn_dropout(_drop(_lib), 257, 256, 8, 0, 0) == bad and lib.fwn_dropout(_drop(_lib), 256, 258, 8, 1, 0) == bad
  assert lib.fwn_dropout(_drop(_lib), 256, 256, 2 ** 43, 0, 0) == no
  assert lib.fwn_dropout(_drop(_lib), None, None, 0, 0, 0) == _lib.FWN_OK


def test_branch_refusals():
  from faster_weathernext import _lib
  lib = _lib.lib()
  bad, no = _lib.FWN_ERR_INVALID_ARGUMENT, _lib.FWN_ERR_UNSUPPORTED

  def call(desc, x=256, y=256, pw=None, w=None, gate=None, s=256, h=256, scale=None, rstd=None):
    return lib.fwn_branch_norm(desc, x, y, pw, w, gate, s, h, scale, rstd, 0)

  assert call(None) == bad and call(_branch(_lib, rows=-1)) == bad and call(_branch(_lib, d=0)) == bad
  assert call(_branch(_lib, d=8193, x_stride=8193, y_stride=8193)) == no
  assert call(_branch(_lib, d=8191, x_stride=8191, y_stride=8191)) == no   # no room for rows that start anywhere
  assert call(_branch(_lib, rows=2 ** 31, gate_span=1)) == no
  assert call(_branch(_lib, x_dtype=2)) == bad and call(_branch(_lib, gate_dtype=2)) == bad
  assert call(_branch(_lib, out_dtype=3)) == bad and call(_branch(_lib, eps=-1.0)) == bad
  assert call(_branch(_lib, eps=float("nan"))) == bad
  assert call(_branch(_lib, x_stride=63)) == bad and call(_branch(_lib, y_stride=63)) == bad
  assert call(_branch(_lib, gate_span=4)) == bad and call(_branch(_lib, gate_span=0)) == bad
  assert call(_branch(_lib, gate_span=12)) == bad
  assert call(_branch(_lib, drop=_drop(_lib, threshold=70000))) == bad
  assert call(_branch(_lib), x=None) == bad and call(_branch(_lib), h=None) == bad and call(_branch(_lib), y=258, s=256, x=257) == bad
  assert call(_branch(_lib), x=260) == no                      # rows that no wide access reaches
  assert call(_branch(_lib, x_stride=66), x=256) == no         # and not contiguous
  assert call(_branch(_lib, out_dtype=2)) == bad and call(_branch(_lib), scale=256) == bad   # scale goes with e4m3
  assert call(_branch(_lib), rstd=260) == bad
  assert call(_branch(_lib, rows=0, gate_span=0), x=None, y=None, s=None, h=None) == _lib.FWN_OK
  size = ctypes.c_size_t(0)
  assert lib.fwn_branch_norm_bwd_workspace_size(_branch(_lib, out_dtype=2), size) == bad
  assert lib.fwn_branch_norm_bwd_workspace_size(_branch(_lib), None) == bad
  assert lib.fwn_branch_norm_bwd_workspace_size(_branch(_lib), size) == _lib.FWN_OK and size.value > 0

  def back(desc, pw=None, w=None, gate=None, rstd=256, dpw=None, dw=None, dgate=None, ws=256, n=1 << 30):
    return lib.fwn_branch_norm_bwd(desc, 256, 256, pw, w, gate, rstd, 256, 256, 256, 256, dpw, dw, dgate, ws, n, 0)

  assert back(_branch(_lib), dpw=256) == bad and back(_branch(_lib), dw=256) == bad and back(_branch(_lib), dgate=256) == bad
  assert back(_branch(_lib), rstd=None) == bad
  assert back(_branch(_lib), ws=None, n=0) == _lib.FWN_ERR_WORKSPACE and back(_branch(_lib), n=16) == _lib.FWN_ERR_WORKSPACE


def test_python_refusals():
  from faster_weathernext import branch
  x = torch.zeros(4, 8)
  with pytest.raises(ValueError, match="CUDA"):
    branch.dropout(x, 0.1, 1)
  with pytest.raises(TypeError):
    branch.dropout(x.double(), 0.1, 1)
  with pytest.raises(ValueError, match="CUDA"):
    branch.branch_norm(x, x)
  with pytest.raises(ValueError):
    branch.branch_norm(x, x, eps=-1.0)
  with pytest.raises(ValueError):
    branch.branch_norm(torch.zeros(4, 0), torch.zeros(4, 0))
