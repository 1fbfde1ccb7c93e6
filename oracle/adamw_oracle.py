"""AdamW on numpy arrays: the moments operation by operation in fp32 (their
8-bit codes follow bit for bit), the weights in 64 bits."""
import numpy as np

BLOCK = 256
M1, M2, STEP, ADD = 0x6A09C55D, 0x5D1B8E63, 0x9E2F4D8B, 0x3C7A15E9
U = np.uint64
_ALL = U(0xFFFFFFFF)


def padded(n):
    return -(-n // BLOCK) * BLOCK


def _mix(x, by):
    p = (np.asarray(x, dtype=U) & _ALL) * U(by)
    return (p >> U(32)) ^ (p & _ALL)


def words(seed, step, first, n):
    """Random words of elements first .. first + n: (for the moments, for the weight)."""
    i = np.arange(first, first + n, dtype=U)
    k = _mix(U((seed & 0xFFFFFFFF)) + U(ADD), M1)
    k = _mix(k ^ U(seed >> 32) ^ U(ADD), M2)
    k = _mix(k + U(step) + U(STEP), M1)
    b = i >> U(8)
    kb = _mix(k + (b & _ALL) + U(ADD), M1)
    kb = _mix((kb ^ (b >> U(32))) + U(STEP), M2)
    h = _mix(_mix((kb ^ ((i & U(255)) * U(STEP) & _ALL)) + U(ADD), M1) ^ U(STEP), M2)
    return h, _mix(h ^ U(ADD), M1)


def decode(codes, scale, first):
    """first: the first moment (sign, 4, 3 bits), else the second (5, 3)."""
    c = codes.astype(np.int64)
    size = c & 127 if first else c
    e, f = size >> 3, (size & 7) / 8.0
    top = 15 if first else 31
    v = np.where(e == 0, f * 2.0 ** (1 - top), (1 + f) * 2.0 ** (e - float(top)))
    v = np.float32(v).reshape(-1, BLOCK) * scale[:, None].astype(np.float32)
    v = v.reshape(-1).astype(np.float32)
    return np.where(c > 127, -v, v) if first else v


def encode(x, noise, first):
    """Codes and scales of fp32 x; noise: 20 random bits a value."""
    x = x.astype(np.float32).reshape(-1, BLOCK)
    scale = np.maximum(np.abs(x).max(1), np.float32(2.0 ** -100))
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        inv = np.float32(1) / scale
        y = np.abs(x) * inv[:, None] * np.float32(2.0 ** (-112 if first else -96))
    c = (np.ascontiguousarray(y).view(np.uint32).astype(U) + noise.reshape(y.shape).astype(U)) >> U(20)
    if first:
        c = np.minimum(c, U(127)) | ((x < 0).astype(U) << U(7))
    else:
        c = np.maximum(np.minimum(c, U(255)), (x > 0).astype(U))
    return c.astype(np.uint8).reshape(-1), scale


def moments(m, v, g, b1, b2):
    """The fp32 averages, each operation rounded."""
    f = np.float32
    m, v, g = m.astype(f), v.astype(f), g.astype(f)
    with np.errstate(under="ignore"):
        return m * f(b1) + g * f(1 - b1), v * f(b2) + (g * g) * f(1 - b2)


def weights(p, m, v, step, lr, b1, b2, eps, decay):
    """The updated weights in 64 bits, from the new moments."""
    m, v = m.astype(np.float64), v.astype(np.float64)
    p = p.astype(np.float64)
    down = np.sqrt(v / (1 - b2 ** step)) + eps
    with np.errstate(invalid="ignore", divide="ignore"):
        return p - lr * decay * p - lr * (m / (1 - b1 ** step)) / down


def noise(h, first):
    return ((h >> U(16) if first else h & U(0xFFFF)) << U(4)) | U(8)
