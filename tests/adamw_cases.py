"""Plain restatements for the AdamW tests: the step's formula in 64 bits, and the 8-bit moments' format (blocks of 256,
one exponent each, codes counting the cut float32 patterns) in integers."""
import numpy as np

BLOCK = 256
U = 2.0 ** -24                      # half a float32 step


def adamw64(w, g, m, v, t, lr, wd, b1, b2, eps):
    w, g, m, v = (np.asarray(x, np.float64) for x in (w, g, m, v))
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return w * (1 - lr * wd) - lr / (1 - b1 ** t) * m / (np.sqrt(v) / np.sqrt(1 - b2 ** t) + eps), m, v


def adamw32(g, m, v, b1, b2):
    """The moments in float32, each product and sum rounded (what the 8-bit codes are cut from)."""
    f = np.float32
    m = m * f(b1) + g * f(1 - b1)
    v = v * f(b2) + (g * g) * f(1 - b2)
    return m, v


def hash32(index, key):
    m32 = np.uint64(0xFFFFFFFF)
    i = np.asarray(index, np.uint64)
    with np.errstate(over="ignore"):
        x = (i + np.uint64(key) + (i >> np.uint64(32)) * np.uint64(0x6A09E667)) & m32
        x = (x * np.uint64(0x9E3779B9)) & m32
        x ^= x >> np.uint64(16)
        x = (x * np.uint64(0x6A09E667)) & m32
        x ^= x >> np.uint64(15)
        x = (x * np.uint64(0xBB67AE85)) & m32
    return (x ^ (x >> np.uint64(16))).astype(np.int64)


def base_of(e, signed):
    return np.maximum(0, 8 * (e + 1) - (127 if signed else 255))


def encode(x, noise, signed):
    """codes [n], exponents [blocks] of float32 x; noise: 16-bit numbers added below the last kept bit."""
    x = np.asarray(x, np.float32)
    n = x.size
    pad = -n % BLOCK
    bits = np.pad(x.view(np.uint32).astype(np.int64) & 0x7FFFFFFF, (0, pad)).reshape(-1, BLOCK)
    sign = np.pad((x.view(np.uint32) >> 31).astype(np.int64), (0, pad)).reshape(-1, BLOCK)
    noise = np.pad(np.broadcast_to(np.asarray(noise, np.int64), n), (0, pad)).reshape(-1, BLOCK)
    e = (bits.max(1, keepdims=True) >> 23) if bits.size else np.zeros((0, 1), np.int64)
    code = np.maximum(((bits + (noise << 4)) >> 20) - base_of(e, signed), 0)
    code = code + 128 * sign if signed else np.maximum(code, bits > 0)
    code = np.where(e == 255, 0, code)
    return code.reshape(-1)[:n].astype(np.uint8), e.reshape(-1).astype(np.uint8)


def decode(codes, exps, signed):
    n = codes.size
    c = np.pad(codes.astype(np.int64), (0, -n % BLOCK)).reshape(-1, BLOCK)
    e = exps.astype(np.int64)[:, None]
    size = c & 127 if signed else c
    x = np.where(size > 0, (size + base_of(e, signed)) << 20, 0).astype(np.uint32).view(np.float32)
    x = np.where(c > 127, -x, x) if signed else x
    return np.where(e == 255, np.float32("nan"), x).reshape(-1)[:n].astype(np.float32)


def split_bf16(w):
    """(bfloat16 bits, residual) of float32 w: nearest, halves away from zero."""
    bits = np.asarray(w, np.float32).view(np.uint32).astype(np.int64)
    hi = ((bits + 0x8000) >> 16) & 0xFFFF
    lo = bits - (hi << 16)
    return hi.astype(np.uint16), lo.astype(np.int16)
