"""The operators of a paged 4-bit key/value cache, as cases that can be timed and checked: the step that hands pages
to requests (block tables, slot maps), the writer and the reader of the cache, and the attention over it.

Every case is one pass through a public entry point of include/tnhip.h on buffers that the caller owns, or (`own`
false) the same operator in elementary torch operations, in 32 bits, rounded once at the end. The sizes are those
of this package's own configurations and tests (9/3 heads of 64, 32/8 heads of 128, sixteen sequences of 512 to
4096 tokens, prompts of 2048), widened to what a program that serves such models asks for.

The cache of a layer is four planes, in pages of `ps` tokens (P pages, H key/value heads, D elements a row, nb =
D / 32 blocks of q4_0, each an f16 scale and 16 bytes, byte j holding element j low and element j + 16 high):
  k_codes  [P][H][ps][4][nb][4]      byte j of part g of block b: byte 4 g + j of the block
  k_scales [P][H][ps][nb]
  v_codes  [P][H][ps / 8][16][nb][8] the bytes c of block b of eight tokens, tokens in the order 0 2 1 3 4 6 5 7
  v_scales [P][H][ps / 8][nb][8]     tokens in order
"""

from __future__ import annotations

import math

import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_CODE = {"f32": 0, "bf16": 1, "f16": 2}  # TN_F32, TN_BF16, TN_F16
_ORDER = (0, 2, 1, 3, 4, 6, 5, 7)
MAX_SCALE = 8188.0  # 8 * 8188 = 65504


def listed():
    return [
        # sixteen sequences, one token each, two of them ended and one new with a prompt of 240: all latency
        _plan("plan decode step", 16, 16, 512, 256, "decode"),
        # prompts of several hundred requests admitted together into a large pool
        _plan("plan admit prompts", 500, 32, 256, 60000, "prompts"),
        # one token a sequence into the cache, and back as the values the attention sees
        _rows("append decode rows", "append", "bf16", 16, 8, 128, 16),
        # a long prompt's rows into the cache and back
        _rows("append prompt", "append", "bf16", 8192, 8, 128, 64),
        # a short request's cached rows read back for a small f32 model
        _rows("read short", "read", "f32", 250, 3, 64, 16),
        # a long context read back, to move it or to attend it with another kernel
        _rows("read long", "read", "bf16", 65536, 8, 128, 128),
        # one sequence of a small f32 model, one token: all latency
        _attn("decode small", "f32", 1, 9, 3, 64, 16, 300, 300, 1, 1),
        # sixteen sequences of 512 to 4096 cached tokens, one token each
        _attn("decode batch", "bf16", 16, 32, 8, 128, 16, 512, 4096, 1, 1),
        # long contexts, the cache's reason to be in 4 bits
        _attn("decode long", "f16", 12, 32, 8, 128, 64, 20000, 40000, 1, 1),
        # four drafted tokens a sequence to verify, another head dim
        _attn("verify drafts", "bf16", 8, 24, 8, 96, 32, 100, 3000, 4, 4),
        # a prompt whose rows were just appended
        _attn("prompt", "bf16", 1, 32, 8, 128, 64, 4096, 4096, 4096, 4096),
        # ragged chunks of prompts behind contexts of their own, some of them a single token
        _attn("ragged chunks", "f16", 6, 16, 4, 64, 16, 1000, 3000, 1, 700),
    ]


def _plan(name, n, ps, width, tokens, kind):
    return {"name": name, "op": "plan", "n": n, "ps": ps, "width": width, "tokens": tokens, "kind": kind}


def _rows(name, op, dtype, m, Hkv, D, ps):
    return {"name": name, "op": op, "dtype": dtype, "m": m, "Hkv": Hkv, "D": D, "ps": ps}


def _attn(name, dtype, n, Hq, Hkv, D, ps, lo, hi, qlo, qhi):
    """n requests of lo to hi cached tokens, the last qlo to qhi of which are the call's rows."""
    return {"name": name, "op": "attn", "dtype": dtype, "n": n, "Hq": Hq, "Hkv": Hkv, "D": D, "ps": ps, "lo": lo,
            "hi": hi, "qlo": qlo, "qhi": qhi}


def draw(rng):
    """One more case of the ranges above, sizes spread over their logarithm."""
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["plan"] * 2 + ["append"] * 2 + ["read"] * 2 + ["attn"] * 6)
    ps = rng.choice([16, 16, 32, 64, 128, 256])
    if op == "plan":
        kind = rng.choice(["decode", "prompts"])
        n = log(1, 1000)
        tokens = n + log(16, 2000) if kind == "decode" else log(max(64, 2 * n), 65536)
        c = _plan("", n, ps, max(1, 8192 // ps), tokens, kind)
    elif op in ("append", "read"):
        Hkv, D = rng.choice([1, 2, 3, 4, 8]), rng.choice([32, 64, 64, 96, 128, 128, 160, 256])
        most = 65536 * 1024 // (Hkv * D) if op == "read" else 8192 * 1024 // (Hkv * D)
        c = _rows("", op, rng.choice(["bf16", "bf16", "f16", "f32"]), log(1, min(most, 65536)), Hkv, D, ps)
    while op == "attn":
        D = rng.choice([64, 64, 128, 128, 128, 32, 96, 256])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        Hkv, rep = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 3, 4, 7, 8])
        n, hi = log(1, 64), log(16, 40000)
        lo = rng.randrange(max(1, hi // 4), hi + 1)
        qlo, qhi = rng.choice([(1, 1), (1, 1), (1, 1), (2, 5), (1, log(2, 4096)), (0, 0)])
        if qhi == 0:  # whole prompts
            n, qlo, qhi = min(n, 4), lo, hi
        qhi = min(qhi, lo) if qhi < hi else qhi
        qlo = min(qlo, qhi)
        pairs = n * hi * Hkv * rep * qhi
        if n * hi * Hkv * D > 12 * 40000 * 8 * 128 or pairs > 32 * 4096 * 4096 or pairs * D > 32 * 4096 * 4096 * 128:
            continue
        if dtype != "bf16" and pairs * D > 16 * 2048 * 2048 * 128:
            continue
        c = _attn("", dtype, n, Hkv * rep, Hkv, D, ps, lo, hi, qlo, qhi)
        break
    c.pop("name", None)
    return c


# --- inputs ------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _spread(lo, hi, n):
    """n whole numbers spread evenly from lo to hi: the same total for every seed."""
    return [lo + (hi - lo) * (2 * i + 1) // (2 * n) for i in range(n)]


def _blocks(x):
    """The q4_0 codes (uint8 [..., nb, 32]) and f16 scales [..., nb] of rows x: d is the element of largest size
    (the first of equals) over -8, held to 8188 in size, in f32; codes min(15, trunc(x / d + 8.5)), f32."""
    b = x.to(torch.float32).unflatten(-1, (-1, 32))
    a = b.abs()
    top = a.amax(-1, keepdim=True)
    first = torch.where(a == top, torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
    d = (b.gather(-1, first) / -8).clamp(-MAX_SCALE, MAX_SCALE)
    inv = torch.where(d != 0, 1 / d, torch.zeros_like(d))
    return (b * inv + 8.5).clamp(0, 15).to(torch.uint8), d.squeeze(-1).to(torch.float16)


def _planes(codes, d):
    """The four layouts of codes [P, H, ps, nb, 32] and scales [P, H, ps, nb]: (as K codes, as K scales, as V codes,
    as V scales)."""
    P, H, ps, nb = d.shape
    byte = codes[..., :16] | (codes[..., 16:] << 4)
    k = byte.view(P, H, ps, nb, 4, 4).transpose(3, 4).contiguous()
    v = byte.view(P, H, ps // 8, 8, nb, 16)[:, :, :, list(_ORDER)].permute(0, 1, 2, 5, 4, 3).contiguous()
    return k, d.contiguous(), v, d.view(P, H, ps // 8, 8, nb).transpose(3, 4).contiguous()


def _k_values(codes, d):
    """f32 values [..., D] of K rows: codes [..., 4, nb, 4], scales [..., nb]."""
    byte = codes.transpose(-3, -2).flatten(-2)
    c = torch.cat([byte & 15, byte >> 4], -1).to(torch.float32) - 8
    return (c * d.to(torch.float32)[..., None]).flatten(-2)


def _v_values(codes, d):
    """f32 values [..., 8, D] of groups of eight V rows: codes [..., 16, nb, 8], scales [..., nb, 8]."""
    byte = codes.movedim(-1, -3)[..., list(_ORDER), :, :].transpose(-1, -2)  # the order is its own inverse
    c = torch.cat([byte & 15, byte >> 4], -1).to(torch.float32) - 8
    return (c * d.to(torch.float32).transpose(-1, -2)[..., None]).flatten(-2)


def _cache(g, P, c):
    """A filled cache: the planes of normal rows."""
    H, ps, D = c["Hkv"], c["ps"], c["D"]
    k = _planes(*_blocks(_randn(g, P, H, ps, D)))
    v = _planes(*_blocks(_randn(g, P, H, ps, D)))
    return {"k_codes": k[0], "k_scales": k[1], "v_codes": v[2], "v_scales": v[3], "P": P, "H": H, "ps": ps, "D": D}


# --- pages for requests ------------------------------------------------------------


def _plan_inputs(c, seed):
    """Lengths and new tokens with the same totals for every seed, in another order; pages handed out at random."""
    n, ps, width = c["n"], c["ps"], c["width"]
    if c["kind"] == "decode":  # one token each; an eighth ended; the first slot newly taken by a short prompt
        lens = _spread(1, min(width * ps - 1, 4096), n)
        fresh = [-1 if i % 8 == 5 else 1 for i in range(n)]
        lens[0], fresh[0] = 0, max(1, min(width * ps, c["tokens"] - n))
    else:  # new requests, together most of the rows, the last two rows left over
        lens = [0] * n
        fresh = [max(1, min(width * ps, f)) for f in _spread(1, max(1, 2 * (c["tokens"] - 2) // n - 1), n)]
    g = _gen(seed)
    order = torch.randperm(n, generator=g, device="cuda")
    held = [-(-x // ps) for x in lens]
    need = [max(0, -(-(x + max(f, 0)) // ps) - h) for x, f, h in zip(lens, fresh, held)]
    P = sum(held) + sum(need) + 7
    lens, fresh = _ints(lens)[order], _ints(fresh)[order]
    pages = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    h = (lens + ps - 1) // ps
    at = torch.arange(width, device="cuda")
    before = torch.cumsum(h, 0) - h
    table = torch.where(at < h[:, None], pages[(before[:, None] + at).clamp(max=P - 1)], -1).to(torch.int32)
    free = torch.full((P,), -1, dtype=torch.int32, device="cuda")
    count = P - sum(held)
    free[:count] = pages[sum(held):]
    return {"n": n, "ps": ps, "width": width, "tokens": c["tokens"], "P": P, "lens": lens, "fresh": fresh,
            "table": table, "free": free, "state": _ints([count, 0])}


def _prepare_plan(c, seed):
    s = _plan_inputs(c, seed)
    n, T = s["n"], s["tokens"]
    return {**s, "op": "plan", "lens_out": _ints([0] * n), "state_out": _ints([0, 0]), "row_start": _ints([0] * (n + 1)),
            "base": _ints([0] * n), "slots": _ints([0] * T), "pos": _ints([0] * T)}


def _plan_plain(s):
    n, ps, width, T, P = s["n"], s["ps"], s["width"], s["tokens"], s["P"]
    lens, ended = s["lens"].clamp(0, width * ps).long(), s["fresh"] < 0
    add = s["fresh"].clamp(min=0).long()
    held = (lens + ps - 1) // ps
    at = torch.arange(width, device=lens.device)
    back = s["table"][ended[:, None] & (at < held[:, None])]  # in order of requests, then pages
    count = s["state"][0].long() + back.numel()
    free = s["free"].clone()
    free[s["state"][0].long() + torch.arange(back.numel(), device=lens.device)] = back
    lens, held = torch.where(ended, 0, lens), torch.where(ended, 0, held)
    need = (lens + add + ps - 1) // ps - held
    ends = torch.cumsum(add, 0)
    bad = (lens + add > width * ps) | (ends > T)
    asked = torch.cumsum(torch.where(bad, 0, need), 0)
    ok = ~bad & ((need == 0) | (asked <= count))
    first = asked - need
    got = ok[:, None] & (at >= held[:, None]) & (at < (held + need)[:, None])
    table = torch.where(got, free[(count - 1 - (first[:, None] + at - held[:, None])).clamp(0, P - 1)], s["table"])
    taken = torch.where(ok & (need > 0), asked, 0).amax()
    starts = torch.cat([ends.new_zeros(1), ends]).clamp(max=T)
    t = torch.arange(T, device=lens.device)
    r = (torch.searchsorted(ends, t, right=True)).clamp(max=n - 1)
    p = lens[r] + t - starts[r]
    page = table[r, (p // ps).clamp(0, width - 1)].long()
    live = ok[r] & (t < starts[n]) & (page >= 0) & (page < P)
    i32 = torch.int32
    return {"lens": torch.where(ok, lens + add, lens).to(i32), "base": torch.where(ok, lens, -1).to(i32), "table": table,
            "free": free, "state": torch.stack([count - taken, torch.where(ok, 0, need).sum()]).to(i32),
            "row_start": starts.to(i32), "slots": torch.where(live, page * ps + p % ps, -1).to(i32),
            "pos": torch.where(live, p, 0).to(i32)}


# --- rows into the cache and back ------------------------------------------------------


def _prepare_append(c, seed):
    g = _gen(seed)
    m, H, D, ps = c["m"], c["Hkv"], c["D"], c["ps"]
    P = -(-m // ps) + 3
    # k and v are parts of the projections' stacked rows [m, (2 + 1) H D], as q|k|v gives them
    x = _randn(g, m, 3, H, D).to(_TORCH[c["dtype"]])
    if m > 64:  # a prompt: tokens in order through pages at random
        at = torch.arange(m, device="cuda")
        slots = torch.randperm(P, generator=g, device="cuda")[at // ps] * ps + at % ps
    else:  # a token each of as many sequences
        slots = torch.randperm(P * ps, generator=g, device="cuda")[:m]
    nb = D // 32
    # pages that hold nothing yet
    z = lambda dt, *s: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
    cache = {"k_codes": z(torch.uint8, P, H, ps, 4, nb, 4), "k_scales": z(torch.float16, P, H, ps, nb),
             "v_codes": z(torch.uint8, P, H, ps // 8, 16, nb, 8), "v_scales": z(torch.float16, P, H, ps // 8, nb, 8),
             "P": P, "H": H, "ps": ps, "D": D}
    out = [torch.empty(m, H, D, dtype=_TORCH[c["dtype"]], device="cuda") for _ in range(2)]
    return {"op": "append", "cache": cache, "x": x, "slots": slots.to(torch.int32), "out": out, "dtype": c["dtype"],
            "m": m}


def _append_plain(s):
    c, x = s["cache"], s["x"]
    slots, ps = s["slots"].long(), c["ps"]
    page, row = slots // ps, slots % ps
    codes, d = _blocks(x[:, 1:])
    byte = codes[..., :16] | (codes[..., 16:] << 4)  # [m, 2, H, nb, 16]
    m, _, H, nb, _ = byte.shape
    c["k_codes"][page, :, row] = byte[:, 0].view(m, H, nb, 4, 4).transpose(2, 3)
    c["k_scales"][page, :, row] = d[:, 0]
    group, at = row // 8, torch.tensor(_ORDER, device=row.device)[row % 8]
    c["v_codes"][page, :, group, :, :, at] = byte[:, 1].transpose(2, 3)
    c["v_scales"][page, :, group, :, row % 8] = d[:, 1]
    return _read_plain(s)


def _prepare_read(c, seed):
    g = _gen(seed)
    m, ps = c["m"], c["ps"]
    P = -(-m // ps) + 3
    at = torch.arange(m, device="cuda")
    slots = torch.randperm(P, generator=g, device="cuda")[at // ps] * ps + at % ps  # a request's positions in order
    out = [torch.empty(m, c["Hkv"], c["D"], dtype=_TORCH[c["dtype"]], device="cuda") for _ in range(2)]
    return {"op": "read", "cache": _cache(g, P, c), "slots": slots.to(torch.int32), "out": out, "dtype": c["dtype"],
            "m": m}


def _read_plain(s):
    c, slots = s["cache"], s["slots"].long()
    ps, dt = c["ps"], _TORCH[s["dtype"]]
    page, row = slots // ps, slots % ps
    k = _k_values(c["k_codes"][page, :, row], c["k_scales"][page, :, row])
    at = torch.tensor(_ORDER, device=row.device)[row % 8]
    byte = c["v_codes"][page, :, row // 8, :, :, at].transpose(-1, -2)  # [m, H, nb, 16]
    v = torch.cat([byte & 15, byte >> 4], -1).to(torch.float32) - 8
    v = (v * c["v_scales"][page, :, row // 8, :, row % 8].to(torch.float32)[..., None]).flatten(-2)
    return [k.to(dt), v.to(dt)]


# --- attention --------------------------------------------------------------------------


def _lengths(c):
    """(rows, cached tokens) of each request, the same for every seed."""
    n = c["n"]
    lens = _spread(c["lo"], c["hi"], n)
    if c["qlo"] == c["lo"] and c["qhi"] == c["hi"]:
        return lens, lens  # whole prompts
    return [min(a, b) for a, b in zip(_spread(c["qlo"], c["qhi"], n)[::-1], lens)], lens


def _attn_inputs(c, seed):
    g = _gen(seed)
    n, ps = c["n"], c["ps"]
    rows, lens = _lengths(c)
    held = [-(-x // ps) for x in lens]
    P, width = sum(held) + 2, max(held)
    order = torch.randperm(n, generator=g, device="cuda")
    rows, lens = _ints(rows)[order], _ints(lens)[order]
    pages = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    h = (lens + ps - 1) // ps
    at = torch.arange(width, device="cuda")
    table = torch.where(at < h[:, None], pages[((torch.cumsum(h, 0) - h)[:, None] + at).clamp(max=P - 1)], -1)
    starts = torch.cat([rows.new_zeros(1), torch.cumsum(rows, 0)]).to(torch.int32)
    T = sum(_lengths(c)[0])
    q = _randn(g, T, c["Hq"], c["D"]).to(_TORCH[c["dtype"]])
    return q, starts, lens, table.to(torch.int32), _cache(g, P, c)


def _prepare_attn(c, seed):
    q, starts, lens, table, cache = _attn_inputs(c, seed)
    rows, ls = _lengths(c)
    max_rows, max_len = max(rows), max(ls)
    s = {"op": "attn", "q": q, "row_start": starts, "lens": lens, "table": table, "cache": cache, "n": c["n"],
         "Hq": c["Hq"], "max_rows": max_rows, "max_len": max_len, "dtype": c["dtype"], "out": torch.empty_like(q),
         "lse": torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")}
    return s


def _attn_plain(s):
    c, q, lens = s["cache"], s["q"], s["lens"].long()
    n, H, D, ps = s["n"], c["H"], c["D"], c["ps"]
    G, S, L = s["Hq"] // H, s["max_len"], s["max_rows"]
    W = -(-S // ps)
    page = s["table"][:, :W].long().clamp(min=0)  # pages past a request's length: masked below
    k = _k_values(c["k_codes"][page], c["k_scales"][page]).transpose(1, 2).reshape(n, H, W * ps, D)[:, :, :S]
    v = _v_values(c["v_codes"][page], c["v_scales"][page]).transpose(1, 2).reshape(n, H, W * ps, D)[:, :, :S]
    starts = s["row_start"].long()
    rows = starts[1:] - starts[:-1]
    j = torch.arange(L, device=q.device)
    live = j < rows[:, None]  # [n, L]
    qp = q.to(torch.float32)[(starts[:-1, None] + j).clamp(max=q.shape[0] - 1)]  # [n, L, Hq, D]
    qp = qp.view(n, L, H, G, D).permute(0, 2, 3, 1, 4).reshape(n * H, G * L, D)
    score = torch.bmm(qp, k.transpose(2, 3).contiguous().view(n * H, D, S)) / math.sqrt(D)
    last = (lens - rows)[:, None] + j  # the last key that each row attends
    keep = torch.arange(S, device=q.device) <= last[..., None]  # [n, L, S]
    score = score.view(n, H, G, L, S).masked_fill(~keep[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - top)
    total = e.sum(-1, keepdim=True)
    v = v.masked_fill((torch.arange(S, device=q.device) >= lens[:, None])[:, None, :, None], 0)
    o = torch.bmm(e.view(n * H, G * L, S), v.contiguous().view(n * H, S, D)).view(n, H, G, L, D) / total
    lse = (top + torch.log(total))[..., 0]
    o, lse = o.permute(0, 3, 1, 2, 4)[live], lse.permute(0, 3, 1, 2)[live]  # the rows in order
    return o.reshape(q.shape).to(q.dtype), lse.reshape(q.shape[:2])


# --- what a measuring program calls ---------------------------------------------------------

_PREPARE = {"plan": _prepare_plan, "append": _prepare_append, "read": _prepare_read, "attn": _prepare_attn}
_PLAIN = {"plan": _plan_plain, "append": _append_plain, "read": _read_plain, "attn": _attn_plain}


def prepare(case, seed):
    return _PREPARE[case["op"]](case, seed)


def _bind(s):
    """The C ABI calls of one pass with their arguments bound, as a host binding holds them, and its outputs."""
    import ctypes
    import functools

    from torchnative_amd import _lib

    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    if s["op"] == "plan":
        call = functools.partial(L.tn_paged_plan, st, s["n"], p(s["fresh"]), p(s["lens"]), p(s["lens_out"]),
                                 p(s["table"]), s["width"], s["ps"], p(s["free"]), s["P"], p(s["state"]),
                                 p(s["state_out"]), s["tokens"], p(s["row_start"]), p(s["base"]), p(s["slots"]),
                                 p(s["pos"]))
        return _lib.check, [call], {"lens": s["lens_out"], "base": s["base"], "table": s["table"], "free": s["free"],
                                    "state": s["state_out"], "row_start": s["row_start"], "slots": s["slots"],
                                    "pos": s["pos"]}
    c = s["cache"]
    pages = _lib.Q4Cache(p(c["k_codes"]), p(c["k_scales"]), p(c["v_codes"]), p(c["v_scales"]), c["P"], c["ps"], c["H"],
                         c["D"])
    ref, code = ctypes.byref(pages), _CODE[s["dtype"]]
    if s["op"] == "attn":
        q, n, Hq = s["q"], s["n"], s["Hq"]
        T = q.shape[0]
        floats = L.tn_sdpa_paged_q4_0_work_floats(ref, n, T, Hq, s["max_rows"], s["max_len"])
        s["work"] = torch.empty(floats, dtype=torch.float32, device="cuda")
        call = functools.partial(L.tn_sdpa_paged_q4_0, st, ref, code, p(q), Hq * c["D"], T, Hq, n, p(s["row_start"]),
                                 p(s["lens"]), p(s["table"]), s["table"].shape[1], s["max_rows"], s["max_len"],
                                 float("nan"), p(s["work"]), floats, p(s["out"]), p(s["lse"]))
        return _lib.check, [call], (s["out"], s["lse"])
    calls = []
    if s["op"] == "append":
        x = s["x"]
        calls.append(functools.partial(L.tn_kv_append_q4_0, st, ref, code, p(x[:, 1]), p(x[:, 2]), s["m"], x.stride(0),
                                       p(s["slots"])))
    calls.append(functools.partial(L.tn_kv_read_q4_0, st, ref, p(s["slots"]), s["m"], code, p(s["out"][0]),
                                   p(s["out"][1])))
    return _lib.check, calls, s["out"]


def run(state):
    if not own:
        return _PLAIN[state["op"]](state)
    if "calls" not in state:
        state["calls"] = _bind(state)
    check, calls, out = state["calls"]
    for call in calls:
        status = call()
        if status:
            check(status)
    return out


def exact(case, seed):
    c = case
    if c["op"] == "plan":
        return None  # whole numbers
    if c["op"] == "append":
        x = _prepare_append(c, seed)["x"][:, 1:].float().unflatten(-1, (-1, 32))
        top = torch.zeros_like(x[..., 0])  # the codes are defined by f32 steps, one element after another
        for j in range(32):
            top = torch.where(x[..., j].abs() > top.abs(), x[..., j], top)
        d = (top * -0.125).clamp(-MAX_SCALE, MAX_SCALE)
        inv = torch.where(d == 0, d, d.reciprocal())
        code = torch.floor((x * inv[..., None] + 8.5).double()).clamp(0, 15)
        y = ((code - 8) * d.to(torch.float16).double()[..., None]).flatten(-2)
        return [y[:, 0], y[:, 1]]

    def stored(cache):  # [P, H, ps, D] of K and of V, element by element out of the layouts above
        P, H, ps, D = cache["P"], cache["H"], cache["ps"], cache["D"]
        e, t = torch.arange(D, device="cuda"), torch.arange(ps, device="cuda")
        b, j, high = e // 32, e % 16, (e % 32) // 16
        k = cache["k_codes"][:, :, :, j // 4, b, j % 4]
        k = torch.where(high.bool(), k >> 4, k & 15)
        k = (k.double() - 8) * cache["k_scales"].double()[..., b]
        place = torch.empty(8, dtype=torch.long, device="cuda")
        place[list(_ORDER)] = torch.arange(8, device="cuda")
        t = t[:, None]
        v = cache["v_codes"][:, :, t // 8, j, b, place[t % 8]]
        v = torch.where(high.bool(), v >> 4, v & 15)
        return k, (v.double() - 8) * cache["v_scales"][:, :, t // 8, b, t % 8].double()

    if c["op"] == "read":
        s = _prepare_read(c, seed)
        k, v = stored(s["cache"])
        at = s["slots"].long()
        return [x.transpose(1, 2).reshape(-1, c["Hkv"], c["D"])[at] for x in (k, v)]
    q, starts, lens, table, cache = _attn_inputs(c, seed)
    if cache["P"] * c["Hkv"] * c["ps"] * c["D"] > 600e6:
        return None
    k, v = stored(cache)
    out, lse = torch.empty(q.shape, dtype=torch.float64, device="cuda"), torch.empty(q.shape[:2], dtype=torch.float64,
                                                                                       device="cuda")
    G, starts = c["Hq"] // c["Hkv"], starts.tolist()
    for r, S in enumerate(lens.tolist()):
        a, z = starts[r], starts[r + 1]
        pages = table[r, : -(-S // c["ps"])].long()
        keep = torch.arange(S, device="cuda") <= (S - (z - a) + torch.arange(z - a, device="cuda"))[:, None]
        for h in range(c["Hkv"]):
            kh, vh = (x[pages, h].reshape(-1, c["D"])[:S] for x in (k, v))
            for i in range(h * G, h * G + G):
                s = (q[a:z, i].double() @ kh.t()) / math.sqrt(c["D"])
                s = s.masked_fill(~keep, -math.inf)
                lse[a:z, i] = torch.logsumexp(s, -1)
                out[a:z, i] = torch.exp(s - lse[a:z, i, None]) @ vh
    return out, lse


def work(case):
    c = case
    if c["op"] == "plan":
        if c["kind"] == "decode":
            pages = c["n"] * 2
        else:
            pages = c["tokens"] // c["ps"] + c["n"] // 2
        return {"bytes": 4 * (5 * c["n"] + 2 * c["tokens"] + 2 * pages), "flops": 0}
    if c["op"] in ("append", "read"):
        row = 2 * c["m"] * c["Hkv"] * c["D"]
        return {"bytes": row * (_SIZE[c["dtype"]] * (2 if c["op"] == "append" else 1) + 4.5 / 8 * (
            2 if c["op"] == "append" else 1)) + 4 * c["m"], "flops": 0}
    rows, lens = _lengths(c)
    size, D = _SIZE[c["dtype"]], c["D"]
    pairs = sum(a * b - a * (a - 1) / 2 for a, b in zip(rows, lens))
    return {"bytes": sum(lens) * c["Hkv"] * D * 2 * 4.5 / 8 + sum(rows) * c["Hq"] * (2 * D * size + 4)
            + 4 * sum(-(-x // c["ps"]) for x in lens), "flops": 4 * pairs * c["Hq"] * D}
