"""The 8-bit paged K/V cache in numpy and 64 bits: the formats' values, the
rule by which rows are appended, and attention over what the bytes stand for."""
import numpy as np

import mslim_attn

E4M3, INT8 = mslim_attn.FORMAT_E4M3, mslim_attn.FORMAT_INT8
LARGEST = {E4M3: 448.0, INT8: 127.0}


def values(fmt):
    """What each of the 256 bytes stands for."""
    byte = np.arange(256)
    if fmt == INT8:
        return np.where(byte > 127, byte - 256, byte).astype(np.float64)
    e, m = byte >> 3 & 15, byte & 7
    x = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    x[(byte & 127) == 127] = np.nan
    return np.where(byte > 127, -x, x)


def nearest(x, fmt):
    """The format's value nearest to x, halves to even."""
    if fmt == INT8:
        return np.rint(x)
    _, e = np.frexp(x)
    step = 2.0 ** (np.maximum(e, -5) - 4.0)
    return np.rint(x / step) * step


def half_step(x, fmt):
    """Half the distance between the format's values around x."""
    if fmt == INT8:
        return np.full_like(x, 0.5)
    _, e = np.frexp(x)
    return 2.0 ** (np.maximum(e, -5) - 5.0)


def scale_of(amax, fmt):
    """The smallest power of two with amax <= largest * scale, 2^-126 at least; NaN where amax is not finite."""
    f, e = np.frexp(np.where(np.isfinite(amax), amax, 1.0))
    top, exponent = np.frexp(LARGEST[fmt])
    s = np.where(amax == 0, 2.0 ** -126, 2.0 ** np.maximum(e - exponent + (f > top), -126.0))
    return np.where(np.isfinite(amax), s, np.nan)


def rotate(x, positions, theta, scaling=None):
    """Rotate-half RoPE of x [rows][heads][d] in 64 bits; scaling: (factor, low, high, original maximum)."""
    half = x.shape[-1] // 2
    inv = float(np.float32(theta)) ** (-np.arange(half) / half)
    if scaling:
        factor, low, high, most = scaling
        wavelength = 2 * np.pi / inv
        smooth = np.clip((most / wavelength - low) / (high - low), 0, 1)
        inv = (1 - smooth) * inv / factor + smooth * inv
    angle = (np.asarray(positions, np.float64)[:, None] * inv)[:, None]
    a, b = x[..., :half], x[..., half:]
    return np.concatenate((a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)), -1)


class Pool:
    """A pool's bytes and scales on the host: bytes [page][head][token][d] for K and, put in order, for V."""

    def __init__(self, pages, kvh, page, d, fmt):
        self.pages, self.kvh, self.page, self.d, self.fmt = pages, kvh, page, d, fmt
        self.k8 = np.zeros((pages, kvh, page, d), np.uint8)
        self.v8 = np.zeros_like(self.k8)
        self.scales = np.ones((pages, kvh, page // 16, 2), np.float32)

    def v_bytes(self):
        """V in the order of the device pool: [page][head][block][4][d][4]."""
        return np.ascontiguousarray(self.v8.reshape(self.pages, self.kvh, self.page // 16, 4, 4, self.d)
                                    .swapaxes(-1, -2))

    def set_v_bytes(self, b):
        self.v8 = np.ascontiguousarray(b.reshape(self.pages, self.kvh, self.page // 16, 4, self.d, 4)
                                       .swapaxes(-1, -2)).reshape(self.k8.shape)

    def rows(self, table, tokens, which):
        """f64 [tokens][heads][d] of one sequence: which 0 K, 1 V; an entry that names no page gives zeros."""
        at = np.arange(tokens)
        page = table[at // self.page]
        known = (page >= 0) & (page < self.pages)
        page = np.where(known, page, 0)
        x = values(self.fmt)[(self.k8, self.v8)[which][page, :, at % self.page]]
        s = self.scales[page, :, at % self.page // 16, which].astype(np.float64)
        return np.where(known[:, None, None], x * s[..., None], 0.0), known


def attend(q, k, v, limit, known, scale):
    """f64 attention of q [rows][q_heads][d], row i over known tokens < limit[i]; also sum(p |v|)."""
    n, qh, d = q.shape
    kvh = k.shape[1]
    out, size = np.zeros((n, qh, d)), np.zeros((n, qh, d))
    for h in range(qh):
        kk, vv = k[:, h * kvh // qh], v[:, h * kvh // qh]
        for i in range(n):
            seen = known.copy()
            seen[limit[i]:] = False
            if not seen.any():
                continue
            x = kk[seen] @ q[i, h] * scale
            p = np.exp(x - x.max())
            out[i, h] = p @ vv[seen] / p.sum()
            size[i, h] = p @ np.abs(vv[seen]) / p.sum()
    return out, size


def bound(ref, size):
    """What BF16 outputs may be off: half a step of the value (2^-8), and of
    the probabilities, each rounded to BF16 (2^-8) and divided by the sum of
    the rounded ones (2^-8 again) against sum(p |v|); scores are sums in 32
    bits (256 terms and sum |q k| * scale < 128: an error below 2^-24 * 256 *
    128 = 2^-9, a worst case that no input here comes near, taken as 2^-10)."""
    return np.abs(ref) * 2.0 ** -8 + size * (2.0 ** -7 + 2.0 ** -10)
