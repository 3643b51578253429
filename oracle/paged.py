"""The paged 4-bit key/value cache in plain numpy (TEST INFRASTRUCTURE ONLY): the page bookkeeping one request after
another, q4_0 blocks element by element, the four planes by their index formulas, and attention in float64."""

from __future__ import annotations

import numpy as np

MAX_SCALE = 8188.0


def plan(fresh, lens, table, page_size, free_pages, state, tokens):
    """tn_paged_plan, one request after another. Returns a dict of its outputs; inputs are left as they were."""
    n, width, P, S = len(fresh), table.shape[1], len(free_pages), page_size
    lens = [min(max(int(x), 0), width * S) for x in lens]
    table, stack = table.copy(), free_pages.copy()
    count = min(max(int(state[0]), 0), P)
    for r in range(n):
        if fresh[r] < 0:
            for j in range(-(-lens[r] // S)):
                if count < P:
                    stack[count] = table[r, j]
                    count += 1
            lens[r] = 0
    start, base, taken, lacking, out_of_pages, total = [0], [], 0, 0, False, 0
    for r in range(n):
        add = max(int(fresh[r]), 0)
        total += add
        held = -(-lens[r] // S)
        need = -(-(lens[r] + add) // S) - held
        if lens[r] + add > width * S or total > tokens:
            ok = False
        elif need == 0:
            ok = True
        else:
            out_of_pages = out_of_pages or taken + need > count
            ok = not out_of_pages
        base.append(lens[r] if ok else -1)
        if ok:
            for j in range(need):
                table[r, held + j] = stack[count - 1 - taken]
                taken += 1
            lens[r] += add
        else:
            lacking += max(need, min(add, 1))
        start.append(min(total, tokens))
    slots, pos = np.full(tokens, -1, np.int32), np.zeros(tokens, np.int32)
    for r in range(n):
        for t in range(start[r], start[r + 1]):
            p = base[r] + t - start[r]
            if base[r] >= 0 and 0 <= table[r, p // S] < P:
                slots[t], pos[t] = table[r, p // S] * S + p % S, p
    i32 = lambda x: np.asarray(x, np.int32)  # noqa: E731
    return {"lens": i32(lens), "base": i32(base), "table": table, "free": stack, "state": i32([count - taken, lacking]),
            "row_start": i32(start), "slots": slots, "pos": pos}


def blocks(x):
    """Codes (uint8 [..., nb, 32]) and f16 scales [..., nb] of f32 rows, one element of a block after another."""
    b = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    top = np.zeros(b.shape[:-1], np.float32)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        for j in range(32):
            top = np.where(np.abs(b[..., j]) > np.abs(top), b[..., j], top)
        d = np.clip(top / np.float32(-8), np.float32(-MAX_SCALE), np.float32(MAX_SCALE))
        inv = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
        v = b * inv[..., None] + np.float32(8.5)
    code = np.where(np.isnan(v), 0, np.clip(v, 0, 15)).astype(np.uint8)
    return code, d.astype(np.float16)


def values(code, d):
    """float64 values [..., D] of blocks."""
    y = (code.astype(np.float64) - 8) * d.astype(np.float64)[..., None]
    return y.reshape(*y.shape[:-2], 32 * y.shape[-2])


class Cache:
    """The codes and scales of every slot, and the planes that hold them."""

    def __init__(self, P, S, H, D):
        self.P, self.S, self.H, self.D = P, S, H, D
        self.code = {w: np.full((P * S, H, D // 32, 32), 8, np.uint8) for w in "kv"}
        self.d = {w: np.zeros((P * S, H, D // 32), np.float16) for w in "kv"}

    def append(self, k, v, slots):
        for w, x in (("k", k), ("v", v)):
            code, d = blocks(x)
            for t, s in enumerate(slots):
                if 0 <= s < self.P * self.S:
                    self.code[w][s], self.d[w][s] = code[t], d[t]

    def rows(self, w, slots):
        return values(self.code[w][slots], self.d[w][slots])

    def planes(self):
        """(k_codes, k_scales, v_codes, v_scales), flat, by the index formulas of the layout."""
        P, S, H, nb = self.P, self.S, self.H, self.D // 32
        byte = {w: (self.code[w][..., :16] | (self.code[w][..., 16:] << 4)).reshape(P, S, H, nb, 16) for w in "kv"}
        d = {w: self.d[w].reshape(P, S, H, nb) for w in "kv"}
        kc, vc = np.empty((P, H, S, 4, nb, 4), np.uint8), np.empty((P, H, S // 8, 16, nb, 8), np.uint8)
        for g in range(4):
            kc[:, :, :, g] = byte["k"][..., 4 * g:4 * g + 4].transpose(0, 2, 1, 3, 4)
        vd = np.empty((P, H, S // 8, nb, 8), np.float16)
        for place, token in enumerate((0, 2, 1, 3, 4, 6, 5, 7)):
            vc[..., place] = byte["v"][:, token::8].transpose(0, 2, 1, 4, 3)
        for token in range(8):
            vd[..., token] = d["v"][:, token::8].transpose(0, 2, 1, 3)
        return kc.ravel(), d["k"].transpose(0, 2, 1, 3).ravel().copy(), vc.ravel(), vd.ravel()


def attend(q, cache, row_start, lens, table, scale=None):
    """out, lse and, for the tolerance, sum p |v|, sum |v| and the largest scale sum |q k| and scale sum |q| |d| (d a
    key block's scale) of each row, float64.
    Rows that no request has are NaN in all of them."""
    T, Hq, D = q.shape
    G, S = Hq // cache.H, cache.S
    scale = D ** -0.5 if scale is None else scale
    out, pav, vsum = (np.full(q.shape, np.nan) for _ in range(3))
    lse, qk, qd = (np.full((T, Hq), np.nan) for _ in range(3))
    for r, length in enumerate(lens):
        a, z = row_start[r], row_start[r + 1]
        t = np.arange(length)
        page = table[r, t // S] if length else t
        good = (page >= 0) & (page < cache.P)
        slot = np.where(good, page * S + t % S, 0)
        k, v = cache.rows("k", slot), cache.rows("v", slot)
        kd = np.repeat(np.abs(cache.d["k"][slot].astype(np.float64)), 32, -1)
        m = np.maximum(0, length - (z - a) + np.arange(z - a) + 1)  # keys of each row
        none, seen = m == 0, t[None] < m[:, None]
        for h in range(Hq):
            kh, vh = k[:, h // G], v[:, h // G]
            with np.errstate(invalid="ignore", divide="ignore"):
                s = np.where(good, (q[a:z, h] @ kh.T) * scale, np.nan)
                s = np.where(seen, s, -np.inf)
                top = s.max(1, initial=-np.inf)
                e = np.exp(s - np.where(none, 0, top)[:, None])
                p = e / e.sum(1, keepdims=True)
                vz = np.where(good[:, None], vh, 0)
                out[a:z, h], lse[a:z, h] = p @ vz, top + np.log(e.sum(1))
                pav[a:z, h] = p @ np.abs(vz)
            vsum[a:z, h] = seen @ np.abs(vz)
            qk[a:z, h] = np.where(seen & good, np.abs(q[a:z, h]) @ np.abs(kh).T, 0).max(1, initial=0) * abs(scale)
            qd[a:z, h] = np.where(seen & good, np.abs(q[a:z, h]) @ kd[:, h // G].T, 0).max(1, initial=0) * abs(scale)
            out[a:z, h][none], lse[a:z, h][none], pav[a:z, h][none] = np.nan, -np.inf, 0
    return out, lse, pav, vsum, qk, qd


def row_keys(row_start, lens, T):
    """Keys that each of T rows attends; 0 for rows of no request."""
    m = np.zeros(T, np.int64)
    for r, length in enumerate(lens):
        a, z = row_start[r], row_start[r + 1]
        m[a:z] = np.maximum(0, length - (z - a) + np.arange(z - a) + 1)
    return m


def tolerance(kind, ref, lse, pav, vsum, qk, qd, keys, D, rounded=True, biased=True):
    """Bounds on |got - ref| of out and lse (arrays like them). A half step is 2^-24 in f32 (u), 2^-11 in f16 (h),
    2^-8 in bf16.

    A score is off by e: the f32 sum of D products, at most (D + 16) u of sum |q k| (the split of an f32 query in two
    f16 parts, the scale and the argument of exp2 among the 16); in bf16 calls a key may be rounded to f16, h of that
    sum, where `rounded` (a truth value, or one a row: rows of more than 1024 keys on the kernel of many rows). 16-bit
    calls of D <= 128 may, where `biased` (the kernel of few rows), multiply by codes 72 too large, c + 72 of 64 .. 79,
    and start a block's sum from z = -72 sum q. With Q = sum |q| of the block's 32 elements: z is 10 additions and a
    product of 72 Q at most, 11 * 72 u Q; of the 33 terms, any that are summed make at most 79 Q (with z they are -72 of
    the rest's q and c of their own), 33 * 79 u Q; together under 3400 u Q, times the block's scale d. A probability is
    then off by 2 e of itself, exp2 and the running rescales 8 u more. Of sum p |v| the output
    is off by that and by (keys / 16 + 64) u from the f32 sums (32 keys a product, products in sequence), by 2 h where
    probabilities and values are rounded to f16 (bf16 calls) and by h where one of them is (f16 calls). Probabilities
    are held at 2^6 or more times their size, so one in f16's subnormal range is off by at most 2^-31 of the row's
    largest: 2^-31 sum |v|. The output is rounded once."""
    u, h = 2.0 ** -24, 2.0 ** -11
    e = (D + 16) * u * qk
    if kind == "bfloat16":
        e = e + np.where(np.reshape(rounded, (-1, 1)), h * qk, 0)
    if biased and kind != "float32" and D <= 128:
        e = e + 3400 * u * qd
    rel = 2 * e + (keys / 16 + 72) * u
    out = pav * (rel[..., None] + {"float32": 0, "float16": h, "bfloat16": 2 * h}[kind]) + 2.0 ** -31 * vsum
    step = {"float32": u, "float16": h, "bfloat16": 2.0 ** -8}[kind]
    tiny = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}[kind]
    out = out + step * (np.abs(ref) + out) + tiny
    with np.errstate(invalid="ignore"):
        return out, e + (keys / 16 + 72) * u + 4 * u * np.abs(np.where(np.isfinite(lse), lse, 0))
