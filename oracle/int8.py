"""The operators of an attention block in 8 bits in plain numpy (TEST INFRASTRUCTURE ONLY): rows in 8-bit integers and
their product by exact integers, norms and rotation of heads in float64, and the paged 8-bit cache block by block."""

from __future__ import annotations

import numpy as np

F = np.float32
INV127 = F(1) / F(127)
TINY = F(2.0 ** -126)


def scale_of(top):
    """f32 scales for rows or blocks whose largest finite sizes are `top`."""
    top = np.asarray(top, F)
    return np.where(top > 0, np.maximum(top * INV127, TINY), F(0)).astype(F)


def inverse(scale):
    with np.errstate(divide="ignore"):
        return np.where(scale > 0, F(1) / scale, F(0)).astype(F)


def codes_at(x, scale):
    """Codes (int64) of f32 values under f32 scales; NaN as 0, infinities as the largest where the scale is not 0."""
    with np.errstate(invalid="ignore", over="ignore"):
        c = np.rint((np.asarray(x, F) * inverse(scale)).astype(F))
    return np.where(np.isnan(c), 0, np.clip(np.nan_to_num(c, nan=0, posinf=127, neginf=-127), -127, 127)).astype(np.int64)


def quantize(x):
    """(codes int64 [m, k], scales f32 [m]) of rows x, f32: NaN and zeros where a row holds an infinity or a NaN."""
    x = np.asarray(x, F)
    ok = np.isfinite(x).all(1)
    y = np.where(ok[:, None], x, F(0))
    s = scale_of(np.abs(y).max(1))
    return codes_at(y, s[:, None]), np.where(ok, s, F(np.nan)).astype(F)


def linear(codes, sx, w, sw, bias=None):
    """((float)sum * sw) * sx (+ bias), each step rounded to f32."""
    total = (codes @ w.T).astype(F)
    with np.errstate(invalid="ignore", over="ignore"):
        y = ((total * sw[None]).astype(F) * sx[:, None]).astype(F)
        return y if bias is None else (y + bias).astype(F)


def heads(x, weight, inv_freq, pos, eps):
    """Norm and rotation of heads x [m, h, d], float64; also the largest size that a rotated element's two parts and
    their sum may have, for the tolerance."""
    x, w = x.astype(np.float64), weight.astype(np.float64)
    half = len(inv_freq)
    z = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    a = (pos.astype(np.float64)[:, None] * inv_freq.astype(np.float64))[:, None]
    cos, sin = np.cos(a), np.sin(a)
    out, size = z.copy(), np.abs(z)
    u, v = z[..., :half], z[..., half:2 * half]
    out[..., :half], out[..., half:2 * half] = u * cos - v * sin, v * cos + u * sin
    size[..., :half] = size[..., half:2 * half] = np.abs(u) + np.abs(v)
    return out, size


def heads_tolerance(kind, ref, size, d):
    """|got - ref| of `heads`. In f32, u = 2^-24 a half step: the sum of d squares is off by (d + 1) u of itself, the
    mean, eps and root add 3 u and halve the sum's part, the reciprocal, x r and the weight 3 u; the angle, reduced to
    a turn in 64 bits, is rounded to f32 at up to pi (4 u at most, its 64-bit error far below), cosine and sine are off
    by 4 u more at most; two products and a sum 2 u of `size`. Then one rounding to the output's type."""
    u = 2.0 ** -24
    tol = size * ((d + 1) / 2 + 3 + 3 + 8 + 2) * u
    step = {"float32": u, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[kind]
    tiny = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}[kind]
    return tol + step * (np.abs(ref) + tol) + tiny


class Cache:
    """Codes (-127 .. 127) of every slot and the scales of every block of sixteen slots."""

    def __init__(self, P, S, H, D):
        self.P, self.S, self.H, self.D = P, S, H, D
        self.code = {w: np.zeros((P * S, H, D), np.int64) for w in "kv"}
        self.scale = {w: np.zeros((P * S // 16, H), F) for w in "kv"}

    # (what oracle.paged.attend reads of a cache, for a bound that has no part here)
    @property
    def d(self):
        return {w: np.zeros((self.P * self.S, self.H, self.D // 32), np.float16) for w in "kv"}

    def append(self, k, v, slots):
        """Blocks in the order in which rows enter them: the rows of the sixteen from the first one on, of a slot given
        twice the last."""
        block = [int(s) // 16 if 0 <= s < self.P * self.S else -1 - t for t, s in enumerate(slots)]
        for t, b in enumerate(block):
            if b < 0 or b in block[max(0, t - 15):t]:
                continue
            rows = {int(slots[u]) % 16: u for u in range(t, min(t + 16, len(slots))) if block[u] == b}
            at, u = list(rows), list(rows.values())
            for w, x in (("k", k), ("v", v)):
                self._join(w, np.asarray(x, F)[u], b, at)

    def _join(self, w, x, b, at):
        size = np.where(np.isfinite(x), np.abs(x), F(0)).max((0, 2))  # [H]
        fresh = 0 in at
        old = self.scale[w][b]
        old = np.where((not fresh) & (old > 0) & np.isfinite(old), old, F(0)).astype(F)
        new = np.maximum(old, scale_of(size)).astype(F)
        block = self.code[w][16 * b:16 * b + 16]
        if not fresh:
            with np.errstate(divide="ignore", invalid="ignore"):
                ratio = np.where(new > old, old / new, F(1)).astype(F)
            block[:] = np.rint((block.astype(F) * ratio[None, :, None]).astype(F)).astype(np.int64)
        block[at] = codes_at(x, new[None, :, None])
        self.scale[w][b] = new

    def rows(self, w, slots):
        slots = np.asarray(slots)
        return self.code[w][slots].astype(np.float64) * self.scale[w][slots // 16].astype(np.float64)[..., None]

    def planes(self):
        """(k_codes, k_scales, v_codes, v_scales), flat, by the index formulas of the layout."""
        P, S, H, D = self.P, self.S, self.H, self.D
        byte = {w: (self.code[w] + 128).astype(np.uint8).reshape(P, S, H, D) for w in "kv"}
        scale = {w: self.scale[w].reshape(P, S // 16, H).transpose(0, 2, 1).ravel().copy() for w in "kv"}
        kc = byte["k"].transpose(0, 2, 1, 3).ravel().copy()
        vc = byte["v"].reshape(P, S // 16, 16, H, D).transpose(0, 3, 1, 4, 2).ravel().copy()
        return kc, scale["k"], vc, scale["v"]

    def value_size(self):
        """The largest size that a value can have under the scales held."""
        s = self.scale["v"]
        return 127.0 * float(np.max(s[np.isfinite(s)], initial=0))


def tolerance(kind, ref, lse, pav, qk, keys, D, most):
    """Bounds on |got - ref| of out and lse of attention over a Cache. A half step is 2^-24 in f32 (u), 2^-11 in f16 (h),
    2^-8 in bf16; `most` the largest size of a value under the scales.

    Codes and 16-bit queries enter the products exactly. A score is off by e: the f32 sum of D products, its scale, an
    f32 query's split in two f16 parts and the argument of exp2, at most (D + 16) u of sum |q k|. A probability is then
    off by 2 e of itself; exp2, its block's share of the scale (2^-6 and more in the exponent, whose logarithm is off by
    2^-22 at most, 3 u of the probability) and the running rescales 12 u more. Of sum p |v| the output is off by that, by
    (keys / 16 + 64) u from the f32 sums (32 keys a product, products in sequence) and, 16-bit calls, by h where a
    probability is one f16 (two f16 parts: 4 u), twice that again allowed. A probability times its share is held at 2^6 or
    more times the row's largest one's size, so one in f16's subnormal range is off by at most 2^-31 of it, times a
    reference for the scales of at most twice their largest: 2^-30 most for each key. The output is rounded once."""
    u, h = 2.0 ** -24, 2.0 ** -11
    e = (D + 16) * u * qk
    rel = 2 * e + (keys / 16 + 80) * u
    out = pav * (rel[..., None] + (0 if kind == "float32" else 3 * h)) + 2.0 ** -30 * most * keys
    step = {"float32": u, "float16": h, "bfloat16": 2.0 ** -8}[kind]
    tiny = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}[kind]
    out = out + step * (np.abs(ref) + out) + tiny
    with np.errstate(invalid="ignore"):
        return out, e + (keys / 16 + 80) * u + 4 * u * np.abs(np.where(np.isfinite(lse), lse, 0))
