"""Dropout's mask in NumPy (test infrastructure): Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011)."""
import numpy as np

_M = 0xFFFFFFFF


def philox4x32(counter, key, rounds=10):
  """Words of the counters [n, 4] (uint32) under the key (two 32-bit ints): uint32 [n, 4]."""
  c = [np.asarray(counter)[:, i].astype(np.uint64) for i in range(4)]
  k0, k1 = int(key[0]), int(key[1])
  s, m = np.uint64(32), np.uint64(_M)
  for _ in range(rounds):
    a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
    c = [(b >> s) ^ c[1] ^ np.uint64(k0), b & m, (a >> s) ^ c[3] ^ np.uint64(k1), a & m]
    k0, k1 = (k0 + 0x9E3779B9) & _M, (k1 + 0xBB67AE85) & _M
  return np.stack(c, 1).astype(np.uint32)


def factors(shape, p, seed, site=0, first=0):
  """The mask with its factors, float64 of `shape`: 0 or 1 / (1 - p) with p the nearest multiple of 2^-16. `first`: the
  index of the first value (a multiple of 8)."""
  n = int(np.prod(shape, dtype=np.int64))
  t = int(round(65536 * p))
  if t == 65536:
    return np.zeros(shape)
  i = np.arange((n + 7) // 8, dtype=np.uint64) + np.uint64(first // 8)
  counter = np.stack((i & np.uint64(_M), i >> np.uint64(32), np.full_like(i, site), np.zeros_like(i)), 1).astype(np.uint32)
  seed = int(seed) & (2 ** 64 - 1)
  words = philox4x32(counter, (seed & _M, seed >> 32))
  numbers = np.stack((words & np.uint32(0xFFFF), words >> np.uint32(16)), 2).reshape(-1)[:n]
  return np.where(numbers >= t, 65536.0 / (65536 - t), 0.0).reshape(shape)
