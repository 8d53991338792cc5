"""AdamW with 32- and 8-bit moments from its formulas, in 64 bits on the CPU: what the device's step is checked against.

8-bit moments: blocks of 256 elements of one tensor; block exponent byte E with the block's largest finite magnitude in
[128, 256) * 2^(E - 127); a magnitude goes to the upper of its two e4m3 neighbours if its fraction of the way plus u >= 1."""
import numpy as np

A, B = 0x9E3779B9, 0xBB67AE85


def mix(x):
    x = np.asarray(x, dtype=np.uint64) & 0xFFFFFFFF
    x ^= x >> 15
    x = (x * B) & 0xFFFFFFFF
    return x ^ (x >> 13)


def dither(places, t, seed):
    key = mix(int(t) + int(mix(seed * A)))
    h = mix(np.asarray(places, dtype=np.uint64) * A + key)
    return (h >> 16).astype(np.float64) / 65536, (h & 0xFFFF).astype(np.float64) / 65536


def step_size(z):
    """Distance of the e4m3 numbers around the magnitude z."""
    e = np.floor(np.log2(np.maximum(z, 2.0 ** -6)))
    return 2.0 ** (e - 3)


def exponents(x):
    """E per block of x [n <= 256 k] (fp64)."""
    out = []
    for k in range(0, len(x), 256):
        b = np.abs(x[k:k + 256])
        top = np.max(np.where(np.isfinite(b), b, 0.0), initial=0.0)
        out.append(0 if top == 0 else max(0, int(np.floor(np.log2(top))) - 7 + 127))
    return np.array(out, dtype=np.int64)


def hold(x, u, least):
    """(values the codes stand for divided by the scale, E per block) of x, an fp32 value each: exact in fp64."""
    x = np.asarray(x, dtype=np.float64)
    E = exponents(x)
    z = np.abs(x) / np.repeat(2.0 ** (E - 127.0), 256)[:len(x)]
    q = step_size(z)
    down = np.floor(z / q)
    frac = z / q - down
    held = q * (down + (frac + u >= 1))
    held = np.where((x != 0), np.maximum(held, least), held)
    held = np.where(np.isfinite(x), np.copysign(held, x), np.nan)
    return held, E


def moments(m, v, g, b1, b2):
    """m', v' in fp32, each operation rounded (the order the 8-bit codes are defined with), and in fp64."""
    f = np.float32
    g32, m32, v32 = (np.asarray(x, f) for x in (g, m, v))
    m1 = m32 * f(b1) + g32 * f(1 - b1)
    v1 = v32 * f(b2) + (g32 * g32) * f(1 - b2)
    return m1, v1, m * b1 + g * (1 - b1), v * b2 + g * g * (1 - b2)


def weights(p, m, v, t, lr, b1, b2, eps, wd):
    return p - lr * wd * p - lr / (1 - b1 ** t) * m / (np.sqrt(v / (1 - b2 ** t)) + eps)
