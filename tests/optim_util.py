"""The optimiser operators restated in numpy: AdamW in 64 bits, and the 8-bit moments in single 32-bit operations."""
import numpy as np

F = np.float32
U32 = 2.0 ** -24   # half a step of f32


def adamw64(p, g, m, v, t, lr, b1, b2, eps, wd, scale):
    """(p, m, v, the update, the first moment's size, the step's divisor), in 64 bits."""
    p, g, m, v = (np.asarray(a, np.float64) for a in (p, g, m, v))
    g = g * scale
    m1 = b1 * m + (1 - b1) * g
    v1 = b2 * v + (1 - b2) * g * g
    div = (np.sqrt(v1 / (1 - b2 ** t)) + eps) * (1 - b1 ** t) / lr
    with np.errstate(divide="ignore", invalid="ignore"):
        up = m1 / div
    return p - lr * wd * p - up, m1, v1, up, b1 * np.abs(m) + (1 - b1) * np.abs(g), div


def bounds(p, up, size, div, bf16_of=None):
    """How far the kernel's m and p may be from 64 bits.

    m: beta, 1 - beta and grad_scale * g are rounded once each, then two products and a sum: 5 half steps of the size
    of its terms.  The update: that over the divisor, whose v has 7 (halved by the root), the root 2, the two corrections
    (log, product, expm1 of 2, rsqrt of 4) 8 each at most, the sum and products 4, the quotient 4: 32.  p: keep has 2,
    the product and the difference 1 each."""
    bm = 5 * U32 * size
    with np.errstate(divide="ignore", invalid="ignore"):
        bp = bm / div + 32 * U32 * np.abs(up) + 5 * U32 * np.abs(p)
    if bf16_of is not None:   # rounded to bf16 once more
        bp = bp + 2.0 ** -8 * np.abs(bf16_of)
    return bm, bp


def mix(x):
    x = np.asarray(x, np.uint32)
    x = x ^ (x >> np.uint32(16))
    x = x * np.uint32(0x6A09E667)
    x = x ^ (x >> np.uint32(15))
    x = x * np.uint32(0xBB67AE85)
    return x ^ (x >> np.uint32(16))


def random_bits(seed, t, tensor, n, first=0):
    """The 32 random bits of elements [first, first + n) of a tensor."""
    with np.errstate(over="ignore"):
        key = mix(mix(mix(np.uint32(seed & 0xFFFFFFFF)) ^ np.uint32(t & 0xFFFFFFFF)) ^ np.uint32(tensor))
        i = np.arange(first, first + n, dtype=np.uint64)
        key = key + (i >> np.uint64(32)).astype(np.uint32) * np.uint32(0xBB67AE85)
        return mix(key + i.astype(np.uint32) * np.uint32(0x9E3779B1))


def blocks(a, fill=0):
    n = -(-len(a) // 256) * 256
    out = np.full(n, fill, a.dtype)
    out[:len(a)] = a
    return out.reshape(-1, 256)


def power(e):
    return np.ldexp(F(1), np.asarray(e, np.int32) - 127).astype(F)


def e4m3(code):
    """The values of e4m3 codes (uint8)."""
    c = np.asarray(code, np.int32)
    e, f = (c >> 3) & 15, c & 7
    v = np.where(e == 0, np.ldexp(f.astype(np.float64), -9), np.ldexp(8.0 + f, e - 10))
    v = np.where((c & 0x7F) == 0x7F, np.nan, v)
    return np.where(c & 0x80, -v, v)


def held(code, exp):
    """The f32 values that codes [n] with exponents [ceil(n / 256)] stand for."""
    v = e4m3(blocks(code)) * power(exp).astype(np.float64)[:, None]
    return v.astype(F).reshape(-1)[:len(code)]


def encode(x, u, root):
    """x f32 [n] and 16 random bits each -> (codes [n], exponents): rounded down or up with the probability of the rest."""
    n = len(x)
    x, u = blocks(np.asarray(x, F)), blocks(np.asarray(u, np.uint32))
    size = np.abs(x)
    fine = np.isfinite(size)
    top = np.where(fine, size, F(0)).max(1)
    e = np.maximum(top.view(np.uint32).astype(np.int64) >> 23, 7) - 7
    y = np.where(fine, size, F(0)) * power(254 - e)[:, None]
    low = y < F(2.0 ** -6)
    z = np.where(low, y + F(2.0 ** -6), y).astype(F)
    code = ((z.view(np.uint32).astype(np.int64) + ((u.astype(np.int64) << 4) | 8)) >> 20) - np.where(low, 968, 960)
    if root:
        code = np.where((size > 0) & (code == 0), 1, code)
    code = np.where(np.signbit(x) & (not root), code | 0x80, code)
    code = np.where(fine, code, 0x7F)
    return code.astype(np.uint8).reshape(-1)[:n], e.astype(np.uint8)


def adamw8_moments(g, cm, em, cs, es, seed, t, tensor, b1, b2, scale):
    """New (m codes, m exponents, s codes, s exponents) of one tensor; every operation rounded to f32."""
    with np.errstate(over="ignore", invalid="ignore", under="ignore"):
        g = np.asarray(g, F) * F(scale)
        m = held(cm, em) * F(b1) + g * F(1 - b1)
        s = held(cs, es)
        s = np.sqrt(s * s * F(b2) + g * g * F(1 - b2))
        bits = random_bits(seed, t, tensor, len(g))
        return (*encode(m, bits & np.uint32(0xFFFF), False), *encode(s, bits >> np.uint32(16), True))
