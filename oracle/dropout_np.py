"""Dropout by Philox 4x32-10 in numpy: the mask from the generator's definition (Salmon, Moraes,
Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC'11)."""
import numpy as np

_LOW = np.uint64(0xFFFFFFFF)
_HALF = np.uint64(32)


def philox(counter, key):
    """counter [..., 4], key [..., 2] (32-bit words) -> the block's four words, uint32."""
    c = [np.asarray(counter)[..., i].astype(np.uint64) for i in range(4)]
    k = [np.asarray(key)[..., i].astype(np.uint64) for i in range(2)]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> _HALF) ^ c[1] ^ k[0], b & _LOW, (a >> _HALF) ^ c[3] ^ k[1], a & _LOW]
        k = [(k[0] + np.uint64(0x9E3779B9)) & _LOW, (k[1] + np.uint64(0xBB67AE85)) & _LOW]
    return np.stack(c, -1).astype(np.uint32)


def threshold(p):
    return int(round(65536 * p))


def keep_mask(rows, cols, p, seed, offset=0):
    """bool [rows, cols]: the elements that stay."""
    blocks = -(-cols // 8)
    counter = np.zeros((rows, blocks, 4), dtype=np.uint64)
    counter[..., 0] = np.arange(blocks)
    counter[..., 1] = np.arange(rows)[:, None]
    offset, seed = offset & (2**64 - 1), seed & (2**64 - 1)
    counter[..., 2], counter[..., 3] = offset & 0xFFFFFFFF, offset >> 32
    words = philox(counter, np.array([seed & 0xFFFFFFFF, seed >> 32], dtype=np.uint64))
    halves = np.stack((words & 0xFFFF, words >> 16), -1).reshape(rows, blocks * 8)
    return halves[:, :cols] >= threshold(p)


def dropout(x, p, seed, offset=0, fill=None):
    """float64 dropout of x [rows, cols]; its gradient is the same of the gradient with fill 0
    (scaled for fill=None)."""
    keep = keep_mask(*x.shape, p, seed, offset)
    if fill is None:
        rest = 65536 - threshold(p)
        return np.where(keep, x * (65536.0 / rest if rest else 1.0), 0.0)
    return np.where(keep, x, fill)
