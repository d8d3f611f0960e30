"""CPU: the C entry points of the norm and the projections refuse bad arguments before any CUDA call."""
import ctypes


def _rms(lib_mod, **kw):
  d = dict(rows=4, d=64, x_dtype=1, residual_dtype=0, weight_dtype=1, out_dtype=0, flags=0, eps=1e-6, reserved=0,
           x_stride=64, residual_stride=64)
  d.update(kw)
  return lib_mod.RmsDesc(*d.values())


def _lin(lib_mod, **kw):
  d = dict(m=64, n=32, k=48, dtype=0, out_dtype=0, bias_dtype=1, x_dtype=0, act=0, flags=0, lda=48, ldb=48, ldx=32, ldo=32)
  d.update(kw)
  return lib_mod.LinearDesc(*d.values())


def test_rms_norm_refusals():
  from faster_weathernext import _lib
  lib = _lib.lib()
  call = lambda desc, x=256, r=None, w=None, xo=None, out=256, sc=None: lib.fwn_rms_norm(desc, x, r, w, xo, out, sc, 0)  # noqa: E731
  bad, no = _lib.FWN_ERR_INVALID_ARGUMENT, _lib.FWN_ERR_UNSUPPORTED
  assert call(None) == bad
  assert call(_rms(_lib, rows=-1)) == bad and call(_rms(_lib, d=0)) == bad
  assert call(_rms(_lib, d=16385, x_stride=16385)) == no
  assert call(_rms(_lib, x_dtype=2)) == bad and call(_rms(_lib, out_dtype=3)) == bad
  assert call(_rms(_lib, eps=-1.0)) == bad and call(_rms(_lib, eps=float("nan"))) == bad
  assert call(_rms(_lib, x_stride=63)) == bad and call(_rms(_lib, flags=2)) == bad
  assert call(_rms(_lib), x=None) == bad and call(_rms(_lib), out=None) == bad
  assert call(_rms(_lib), r=256) == bad                         # a residual without x_out
  assert call(_rms(_lib, out_dtype=2)) == bad                   # e4m3 without a scale
  assert call(_rms(_lib), sc=256) == bad                        # and a scale without e4m3
  assert call(_rms(_lib, rows=0), x=None, out=None) == _lib.FWN_OK
  size = ctypes.c_size_t(0)
  assert lib.fwn_rms_norm_bwd_workspace_size(_rms(_lib, out_dtype=2), size) == bad
  assert lib.fwn_rms_norm_bwd(_rms(_lib), 256, None, None, 256, None, 256, None, 256, None, 0, 0) == bad  # d_weight without weight


def test_linear_refusals():
  from faster_weathernext import _lib
  lib = _lib.lib()
  call = lambda desc, a=256, sa=None, b=256, sb=None, bias=None, x=None, out=256, db=None: lib.fwn_linear(  # noqa: E731
      desc, a, sa, b, sb, bias, x, out, db, None, 0, 0)
  bad, no = _lib.FWN_ERR_INVALID_ARGUMENT, _lib.FWN_ERR_UNSUPPORTED
  assert call(None) == bad
  assert call(_lin(_lib, m=-1)) == bad and call(_lin(_lib, n=0)) == bad and call(_lin(_lib, k=0)) == bad
  assert call(_lin(_lib, dtype=1)) == bad and call(_lin(_lib, act=3)) == bad and call(_lin(_lib, flags=8)) == bad
  assert call(_lin(_lib, lda=47)) == bad and call(_lin(_lib, ldb=47)) == bad and call(_lin(_lib, ldo=31)) == bad
  assert call(_lin(_lib, dtype=2, flags=_lib.LINEAR_B_N_CONTIGUOUS)) == no
  assert call(_lin(_lib, flags=_lib.LINEAR_PRE_GRAD)) == no     # no activation
  assert call(_lin(_lib), a=None) == bad and call(_lin(_lib), out=None) == bad
  assert call(_lin(_lib, dtype=2)) == bad and call(_lin(_lib), sa=256, sb=256) == bad   # scales go with e4m3
  assert call(_lin(_lib, x_dtype=1), x=256) == no               # a residual of another type
  assert call(_lin(_lib, ldx=31), x=256) == bad and call(_lin(_lib), db=256) == bad
  assert call(_lin(_lib, m=0), a=None, b=None, out=None) == _lib.FWN_OK
  size = ctypes.c_size_t(0)
  assert lib.fwn_linear_bwd_workspace_size(_lin(_lib, dtype=2), 256, 256, 256, size) == no
  assert lib.fwn_linear_bwd_workspace_size(_lin(_lib, m=0), 256, 256, 256, size) == bad
  assert lib.fwn_linear_pack(256, 10, 256, 17, 4, 10, 0, 0) == bad and lib.fwn_linear_pack(256, 9, 256, 16, 4, 10, 0, 0) == bad
  assert b"stride" in lib.fwn_last_error_string()
