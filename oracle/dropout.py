"""Dropout's random numbers on the host: Philox-4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
1, 2, 3", 2011) in numpy, and which elements of rows are kept."""
import numpy as np

_LOW = np.uint64(0xffffffff)


def philox(counter, key):
  """The four words (uint64 arrays below 2^32) of counters (four words, arrays or numbers) and a key (two words)."""
  c = [np.asarray(w, np.uint64) for w in counter]
  k = [int(w) for w in key]
  for _ in range(10):
    a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
    c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & _LOW, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & _LOW]
    k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
  return c


def kept(rows, channels, p, seed, offset, first=0):
  """Whether each element of the rows first .. first + rows - 1 is kept: bool [rows, channels]."""
  seed, offset = seed % 2 ** 64, offset % 2 ** 64
  eights = -(-channels // 8)
  row = np.arange(first, first + rows, dtype=np.uint64)[:, None] + np.zeros((1, eights), np.uint64)
  eight = np.arange(eights, dtype=np.uint64)[None] + np.zeros((rows, 1), np.uint64)
  words = philox((eight, row, offset & 0xffffffff, offset >> 32), (seed & 0xffffffff, seed >> 32))
  halves = np.stack([h for w in words for h in (w & np.uint64(0xffff), w >> np.uint64(16))], -1)
  return halves.reshape(rows, eights * 8)[:, :channels] >= border(p)


def border(p):
  """Of 16 random bits: those below it are dropped."""
  return round(p * 65536)


def multiplier(p):
  """Of what is kept, in float32."""
  return np.float32(65536 / (65536 - border(p))) if border(p) < 65536 else np.float32(0)
