"""The block-scaled FP4 key/value cache in numpy, from its definition: where a
token lies, how values become codes and back, and attention in 64 bits."""
import functools

import numpy as np

import oracle as O

MIDS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
MAGS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


@functools.lru_cache(None)
def scale_steps():
    """The values that a scale byte 0x00-0x7E stands for, ascending."""
    return O.e4m3_scale_values()[:127].astype(np.float64)


class Cache:
    """Host image of a cache: bytes [pages, page_stride]."""

    def __init__(self, pages, page, heads, dim, k_scale=1.0, v_scale=1.0, page_stride=0, fill=None, seed=0):
        self.pages, self.page, self.heads, self.dim = pages, page, heads, dim
        self.k_scale, self.v_scale = float(np.float32(k_scale)), float(np.float32(v_scale))
        self.codes, self.scales = page * dim // 2, page * dim // 16
        self.head_bytes = 2 * (self.codes + self.scales)
        self.stride = page_stride or heads * self.head_bytes
        if fill is None:
            self.data = np.random.default_rng(seed).integers(0, 256, (pages, self.stride), dtype=np.uint8)
        else:
            self.data = np.full((pages, self.stride), fill, dtype=np.uint8)

    def parts(self, page, head, place, is_v):
        """Slices of (codes, scales) of a token, into self.data[page]."""
        b = head * self.head_bytes + (self.codes + self.scales if is_v else 0)
        c0 = b + place * (self.dim // 2)
        s0 = b + self.codes + place * (self.dim // 16)
        return slice(c0, c0 + self.dim // 2), slice(s0, s0 + self.dim // 16)

    def write(self, page, place, k, v):
        """k, v: [heads, dim] float."""
        for is_v, x, g in ((False, k, self.k_scale), (True, v, self.v_scale)):
            c, s = quantize(x, g)
            for h in range(self.heads):
                cs, ss = self.parts(page, h, place, is_v)
                self.data[page, cs], self.data[page, ss] = c[h], s[h]

    def token(self, page, place, is_v):
        """[heads, dim] float32: codes times block scales (exact)."""
        out = np.empty((self.heads, self.dim), np.float32)
        for h in range(self.heads):
            cs, ss = self.parts(page, h, place, is_v)
            bits = O.decode_nvfp4(self.data[page, cs], self.data[page, ss], self.dim)
            out[h] = O.f16_bits_to_f32(bits)
        return out


def quantize(x, g):
    """Codes (two per byte, first high) and scale bytes of [rows, dim]; borders
    are products of few-bit numbers with the FP32 scale g, exact in 64 bits."""
    g = float(np.float32(g))
    x = np.asarray(x, np.float64)
    rows, dim = x.shape
    blk = x.reshape(rows, dim // 16, 16)
    steps = scale_steps()
    mids = (steps[1:] + steps[:-1]) / 2
    nan = np.isnan(blk).any(axis=2)
    amax = np.where(nan, 0, np.max(np.abs(np.where(np.isnan(blk), 0, blk)), axis=2))
    sb = np.searchsorted(6 * mids * g, amax, side="left")
    s = steps[sb]
    mag = (np.abs(blk)[..., None] > MIDS * (s * g)[..., None, None]).sum(axis=-1)
    code = np.where(np.signbit(blk), 8, 0) + mag
    code = np.where((s == 0)[..., None] | nan[..., None], 0, code).reshape(rows, dim).astype(np.uint8)
    return (code[:, 0::2] << 4) | code[:, 1::2], np.where(nan, 0x7F, sb).astype(np.uint8)


def sees(pos, tok, window, sinks):
    return (tok <= pos) & ((window <= 0) | (pos - tok < window) | (tok < sinks))


def attention(k, v, q, pos0, scale, window=0, sinks=0):
    """k, v [n, heads, dim] 64-bit values; q [rows, q_heads, dim]; the rows'
    positions start at pos0.  Returns out, lse and, for tolerances, the sum of
    p |v| / l, the largest sum |q k| scale of a visible score and the largest
    |score|, of each row and head."""
    n, heads, dim = k.shape
    rows, qh = q.shape[:2]
    out = np.zeros((rows, qh, dim))
    lse = np.full((rows, qh), -np.inf)
    absv = np.zeros((rows, qh, dim))
    reach = np.zeros((rows, qh))
    top = np.zeros((rows, qh))
    vis = sees(pos0 + np.arange(rows)[:, None], np.arange(n)[None, :], window, sinks)
    for h in range(qh):
        kk, vv = k[:, h // (qh // heads)], v[:, h // (qh // heads)]
        s = scale * (q[:, h] @ kk.T)
        mag = abs(scale) * (np.abs(q[:, h]) @ np.abs(kk).T)
        for i in range(rows):
            j = vis[i]
            if not j.any():
                continue
            x = s[i, j]
            m = x.max()
            p = np.exp(x - m)
            l = p.sum()
            out[i, h] = p @ vv[j] / l
            absv[i, h] = p @ np.abs(vv[j]) / l
            lse[i, h] = m + np.log(l)
            reach[i, h], top[i, h] = mag[i, j].max(), np.abs(x).max()
    return out, lse, absv, reach, top


def tolerances(out, lse, absv, reach, top, n, dim, eps_out):
    """Bounds of |error| of out and lse, from the kernels' arithmetic.

    A score is an FP32 sum of dim exact products (each step off by at most
    2^-23 of the sum of magnitudes), times a factor of three roundings and less
    a maximum, in log2 units: off by at most
        e = (dim + 8) 2^-23 reach + 2^-21 top + 2^-21 (the exponential).
    p is then off by e relative to itself, and by half an FP16 step (2^-11, or
    2^-25 of the largest p where it is subnormal: at most n 2^-25 of the sum);
    sums of n terms in FP32 add n 2^-23; the quotient carries e twice.  The
    output is rounded once more (eps_out of it, and half of FP16's smallest
    step, 2^-25)."""
    e = (dim + 8) * 2.0 ** -23 * reach + 2.0 ** -21 * top + 2.0 ** -21
    part = 2.0 ** -11 + np.expm1(2 * e) + n * 2.0 ** -23 + 2.0 ** -20
    vmax = np.max(np.abs(out), initial=0) + np.max(absv, initial=0)
    t_out = part[..., None] * absv * 1.01 + n * 2.0 ** -25 * vmax + eps_out * np.abs(out) + 2.0 ** -25
    t_lse = e + n * 2.0 ** -23 + 2.0 ** -22 * np.where(np.isfinite(lse), np.abs(lse), 0) + 2.0 ** -20
    return t_out, t_lse
