"""4-bit floating point in numpy: the definition of codes and block scales, and products in 64 bits."""
import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
VALUES = np.concatenate([MAGNITUDES, -MAGNITUDES])
BORDERS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
MX, NV = 0, 1


def cpad(channels):
    return -(-channels // 64) * 64


def pitch(fmt, channels):
    return 4 * -(-cpad(channels) // 128) if fmt == MX else cpad(channels) // 16


def e4m3(t):
    """Nearest e4m3 value (ties to even, saturated at 448) of t >= 0, and its byte."""
    t = np.asarray(t, np.float64)
    e = np.clip(np.frexp(np.where(t > 0, t, 1.0))[1] - 1, -6, 8)
    step = np.ldexp(1.0, e - 3)
    v = np.minimum(np.rint(t / step) * step, 448.0)
    e = np.clip(np.frexp(np.where(v > 0, v, 1.0))[1] - 1, -6, 8)
    m = np.rint(v / np.ldexp(1.0, e - 3)).astype(np.int64)      # 8..15, below 8 for subnormal values
    byte = np.where(m >= 8, (e + 7) * 8 + m - 8, m)
    return v, byte.astype(np.uint8)


def quantize(x, fmt, g=1.0):
    """fp32 [rows, channels] -> codes [rows, cpad / 2], scales [rows, pitch], bit for bit as documented."""
    x = np.asarray(x, np.float32)
    rows, channels = x.shape
    b, cp = (32, 16)[fmt], cpad(channels)
    xb = np.zeros((rows, cp), np.float32)
    xb[:, :channels] = x
    xb = xb.reshape(rows, cp // b, b)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        amax = np.abs(xb).max(2)                # a NaN stays one
        bad = ~np.isfinite(amax)
        top = np.where(bad, 0, amax).astype(np.float32)
        if fmt == MX:
            e = np.clip(np.where(top > 0, np.frexp(np.where(top > 0, top, 1).astype(np.float64))[1] - 3, -127),
                        -127, 127)
            s = np.ldexp(1.0, e)
            byte = np.where(bad, 255, e + 127).astype(np.uint8)
            q = xb.astype(np.float64) / s[..., None]
        else:
            t = top / (np.float32(6) * np.float32(g))
            v, byte = e4m3(t)
            s = (v.astype(np.float32) * np.float32(g))
            byte = np.where(bad, 127, byte).astype(np.uint8)
            q = np.where(s[..., None] > 0, xb / s[..., None], 0).astype(np.float64)
        a = np.abs(np.where(bad[..., None], 0, q))
        i = np.zeros(a.shape, np.uint8)
        for k, c in enumerate(BORDERS):
            i += (a > c) | ((a == c) & (k % 2 == 1))
        i |= ((np.signbit(q) & ~bad[..., None] & (i > 0)).astype(np.uint8) << 3)
    i = i.reshape(rows, cp)
    scales = np.zeros((rows, pitch(fmt, channels)), np.uint8)
    scales[:, : byte.shape[1]] = byte
    return i[:, 0::2] | i[:, 1::2] << 4, scales


def magnitude_codes(codes):
    """Codes with the sign of zeros taken away (it is not specified)."""
    lo, hi = codes & 15, codes >> 4
    lo, hi = np.where(lo == 8, 0, lo), np.where(hi == 8, 0, hi)
    return (lo | hi << 4).astype(np.uint8)


def scale_values(scales, fmt, channels):
    """fp64 block scales without the tensor scale, [rows, blocks]."""
    s = scales[:, : cpad(channels) // (32, 16)[fmt]].astype(np.int64)
    if fmt == MX:
        return np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    e, m = s >> 3, s & 7
    v = np.where(e > 0, np.ldexp(1 + m / 8, e - 7), np.ldexp(m / 8, -6))
    return np.where(s == 127, np.nan, v)


def values(codes, scales, fmt, channels, g=1.0):
    """fp64 [rows, channels] of codes and scales, with S = scale * g rounded to fp32."""
    v = VALUES[np.stack([codes & 15, codes >> 4], 2).reshape(codes.shape[0], -1)]
    s = scale_values(scales, fmt, channels)
    if fmt == NV and g != 1.0:
        s = (s.astype(np.float32) * np.float32(g)).astype(np.float64)
    return (v.reshape(v.shape[0], s.shape[1], -1) * s[..., None]).reshape(v.shape[0], -1)[:, :channels]


def product(x, w, alpha, bias, relu, res=None, res_relu=False):
    """act(alpha x W^T + bias) in 64 bits, and how far an fp16 result may be from it.

    The products of two 4-bit values and two block scales have at most 12 significant bits and are exact; K of them and the
    partial sums are added in fp32, each addition off by at most 2^-23 of the sum of magnitudes (an adder that
    cuts instead of rounding); alpha, bias and their sum: three roundings of 2^-24; the store: half a step of fp16, 2^-11 of the
    value or 2^-25.  With a residual the sum is rounded to fp16 twice."""
    y = alpha * (x @ w.T)
    mass = abs(alpha) * (np.abs(x) @ np.abs(w).T)
    if bias is not None:
        y = y + bias
        mass = mass + np.abs(bias)
    off = mass * (x.shape[1] * 2.0 ** -23 + 3 * 2.0 ** -24)
    if relu:
        y = np.where(y < 0, 0, y)
    off = off + np.abs(y) * 2.0 ** -11 + 2.0 ** -25
    if res is not None:
        y = y + res
        if res_relu:
            y = np.where(y < 0, 0, y)
        off = off * (1 + 2.0 ** -11) + np.abs(y) * (2.0 ** -11 + 2.0 ** -24) + 2.0 ** -25
    return y, off
