"""Philox4x32-10 (Salmon et al., SC 2011) in numpy, and the dropout mask of include/midman_gpu.h made from it."""
import numpy as np

LOW = np.uint64(0xFFFFFFFF)


def philox4x32_10(counter, key):
    """counter: four uint64 arrays (or numbers) of 32-bit words, key: two numbers -> four arrays of 32-bit words."""
    c = [np.asarray(w, np.uint64) for w in counter]
    k = [int(w) for w in key]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & LOW, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & LOW]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def kept(seed, offset, rows, cols, p):
    """The [rows, cols] truth values of the elements that dropout keeps."""
    blocks = -(-cols // 4)
    at = np.arange(rows * blocks, dtype=np.uint64)
    words = philox4x32_10([at & LOW, at >> np.uint64(32), np.full_like(at, offset & 0xFFFFFFFF),
                           np.full_like(at, offset >> 32)], [seed & 0xFFFFFFFF, seed >> 32])
    return np.stack(words, 1).reshape(rows, blocks * 4)[:, :cols] >= np.uint64(int(p * 2.0 ** 32))
