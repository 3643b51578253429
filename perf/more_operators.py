"""The operators of an attention block held in 8 bits, as cases that can be timed and checked: the linear in 8-bit
integers with a scale for each token and channel, the norms of query and key heads with the rotation of their
positions, the writer and the reader of a paged cache in 8 bits, and the attention over it.

Every case is one pass through a public entry point of include/tnhip.h on buffers that the caller owns, or (`own`
false) the same operator in elementary torch operations, in 32 bits, rounded once at the end. The sizes are those
of this package's own configurations and tests (9/3 heads of 64, 32/8 heads of 128, [1536, 576], [14336, 4096], sixteen
sequences of 512 to 4096 tokens), widened to what a program that serves such models asks for.

Rows in 8 bits are codes [rows][pitch], pitch the length rounded up to 64 with zeros behind it, and an f32 scale a row.
The cache of a layer is four planes, in pages of `ps` tokens (P pages, H key/value heads, D elements a row): a byte is
its code + 128, and sixteen tokens of a head share a scale.
  k_codes  [P][H][ps][D]          k_scales [P][H][ps / 16] f32
  v_codes  [P][H][ps / 16][D][16] v_scales [P][H][ps / 16] f32
"""

from __future__ import annotations

import math

import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_CODE = {"f32": 0, "bf16": 1, "f16": 2}  # TN_F32, TN_BF16, TN_F16
TINY = 2.0**-126  # the smallest scale of a row or block that is not zero
EPS = 1e-6


def listed():
    return [
        # one token of a small f32 model: all latency
        _linear("linear one row", "f32", "f32", 1, 1536, 576, False),
        # sixteen sequences, one token each: the weight's bytes
        _linear("linear batch", "bf16", "bf16", 16, 14336, 4096, False),
        # a prompt, or the prompts of a batch
        _linear("linear prompt", "bf16", "bf16", 4096, 14336, 4096, True),
        # one token of a small f32 model
        _heads("heads one row", "f32", 1, 9, 3, 64, 64, 300),
        # a long prompt's rows out of the stacked projections
        _heads("heads prompt", "bf16", 8192, 32, 8, 128, 128, 8192),
        # one token a sequence into blocks that hold others, and those back as the values the attention sees
        _rows("append decode rows", "bf16", 16, 1, 1, 8, 128, 16),
        # a long prompt's rows into the cache and back
        _rows("append prompt", "bf16", 1, 8192, 8192, 8, 128, 64),
        # one sequence of a small f32 model, one token: all latency
        _attn("decode small", "f32", 1, 9, 3, 64, 16, 300, 300, 1, 1),
        # sixteen sequences of 512 to 4096 cached tokens, one token each
        _attn("decode batch", "bf16", 16, 32, 8, 128, 16, 512, 4096, 1, 1),
        # long contexts
        _attn("decode long", "f16", 12, 32, 8, 128, 64, 20000, 40000, 1, 1),
        # a prompt whose rows were just appended
        _attn("prompt", "bf16", 1, 32, 8, 128, 64, 4096, 4096, 4096, 4096),
        # ragged chunks of prompts behind contexts of their own, some of them a single token
        _attn("ragged chunks", "f16", 6, 16, 4, 64, 16, 1000, 3000, 1, 700),
    ]


def _linear(name, dtype, out, m, n, k, bias):
    return {"name": name, "op": "linear", "dtype": dtype, "out": out, "m": m, "n": n, "k": k, "bias": bias}


def _heads(name, dtype, m, Hq, Hkv, D, rot, far):
    """m tokens at positions below `far`, the first `rot` elements of a head rotated."""
    return {"name": name, "op": "heads", "dtype": dtype, "m": m, "Hq": Hq, "Hkv": Hkv, "D": D, "rot": rot, "far": far}


def _rows(name, dtype, n, lo, hi, Hkv, D, ps):
    """n requests that add lo to hi rows each."""
    return {"name": name, "op": "append", "dtype": dtype, "n": n, "lo": lo, "hi": hi, "Hkv": Hkv, "D": D, "ps": ps}


def _attn(name, dtype, n, Hq, Hkv, D, ps, lo, hi, qlo, qhi):
    """n requests of lo to hi cached tokens, the last qlo to qhi of which are the call's rows."""
    return {"name": name, "op": "attn", "dtype": dtype, "n": n, "Hq": Hq, "Hkv": Hkv, "D": D, "ps": ps, "lo": lo,
            "hi": hi, "qlo": qlo, "qhi": qhi}


def draw(rng):
    """One more case of the ranges above, sizes spread over their logarithm."""
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["linear"] * 4 + ["heads"] * 2 + ["append"] * 2 + ["attn"] * 5)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    ps = rng.choice([16, 16, 32, 64, 128, 256])
    c = None
    while c is None:
        if op == "linear":
            m, n, k = log(1, 8192), log(16, 20000), log(16, 16384)
            if m * n * k <= 4096 * 14336 * 4096 and m * k + n * k + 2 * m * n <= 200e6:
                c = _linear("", dtype, rng.choice([dtype, dtype, "f32"]), m, n, k, rng.random() < 0.5)
        elif op == "heads":
            D = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
            Hkv, rep, m = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 3, 4, 7, 8]), log(1, 16384)
            rot = rng.choice([D, D, D, D // 2])
            if m * Hkv * (rep + 1) * D * _SIZE[dtype] <= 8192 * 40 * 128 * 2:
                c = _heads("", dtype, m, Hkv * rep, Hkv, D, rot, log(m, 1000000))
        elif op == "append":
            Hkv, D = rng.choice([1, 2, 3, 4, 8]), rng.choice([32, 64, 64, 96, 128, 128, 160, 256])
            n, hi = log(1, 64), rng.choice([1, 1, 5, log(1, 8192)])
            if n * hi * Hkv * D * _SIZE[dtype] <= 8192 * 8 * 128 * 2:
                c = _rows("", dtype, n, max(1, hi // rng.choice([1, 2, 10])), hi, Hkv, D, ps)
        else:
            D = rng.choice([64, 64, 128, 128, 128, 32, 96, 256])
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
    c.pop("name")
    return c


# --- inputs ------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rand(g, lo, hi, *shape):
    return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32) * (hi - lo) + lo


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _spread(lo, hi, n):
    """n whole numbers spread evenly from lo to hi: the same total for every seed."""
    return [lo + (hi - lo) * (2 * i + 1) // (2 * n) for i in range(n)]


def _scale_of(top):
    """The f32 scale of codes for values of sizes up to `top`, f32."""
    return torch.where(top > 0, (top / 127).clamp(min=TINY), torch.zeros_like(top))


def _codes_at(x, scale):
    """The codes, f32 whole numbers, of f32 values x under `scale`."""
    inv = torch.where(scale > 0, 1 / scale, torch.zeros_like(scale))
    return torch.round(x * inv).clamp(-127, 127)


# --- the linear in 8-bit integers -----------------------------------------------------


def _prepare_linear(c, seed):
    g = _gen(seed)
    m, n, k = c["m"], c["n"], c["k"]
    x = _randn(g, m, k) * _rand(g, 0.2, 2.0, k)  # channels of unlike sizes, as behind a norm
    w = _randn(g, n, k) * 0.02
    scales = _scale_of(w.abs().amax(1))
    pitch = -(-k // 64) * 64
    codes = torch.zeros(n, pitch, dtype=torch.int8, device="cuda")
    codes[:, :k] = _codes_at(w, scales[:, None]).to(torch.int8)
    return {"op": "linear", "x": x.to(_TORCH[c["dtype"]]), "w": codes, "scales": scales,
            "bias": _randn(g, n) * 0.1 if c["bias"] else None, "dtype": c["dtype"], "out": c["out"],
            "y": torch.empty(m, n, dtype=_TORCH[c["out"]], device="cuda")}


def _linear_plain(s):
    x = s["x"].to(torch.float32)
    sx = _scale_of(x.abs().amax(1, keepdim=True))
    # sums of products of codes are whole numbers, below 2^24 but for rows far from any that are met
    total = _codes_at(x, sx) @ s["w"][:, : x.shape[1]].to(torch.float32).t().contiguous()
    y = total * s["scales"] * sx
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(_TORCH[s["out"]])


# --- norms of heads and their rotation ----------------------------------------------------


def _prepare_heads(c, seed):
    g = _gen(seed)
    m, Hq, H, D, rot = c["m"], c["Hq"], c["Hkv"], c["D"], c["rot"]
    dt = _TORCH[c["dtype"]]
    # q and k are parts of the projections' stacked rows [m, (Hq + 2 H) D], as q|k|v gives them
    x = (_randn(g, m, Hq + 2 * H, D) * _rand(g, 0.3, 3.0, Hq + 2 * H, 1)).to(dt)
    freq = 1e5 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float32) / rot)
    if c["far"] > m:  # rows of many requests
        pos = torch.randint(c["far"], (m,), generator=g, device="cuda", dtype=torch.int32)
    else:
        pos = torch.arange(m, device="cuda", dtype=torch.int32)
    weights = [1 + 0.2 * _randn(g, D) for _ in range(2)]
    out = [torch.empty(m, h, D, dtype=dt, device="cuda") for h in (Hq, H)]
    return {"op": "heads", "x": x, "Hq": Hq, "H": H, "weights": weights, "freq": freq, "pos": pos, "dtype": c["dtype"],
            "out": out}


def _heads_plain(s):
    x, Hq, H = s["x"], s["Hq"], s["H"]
    D, half = x.shape[2], s["freq"].shape[0]
    angle = s["pos"].to(torch.float64)[:, None, None] * s["freq"].to(torch.float64)
    cos, sin = torch.cos(angle).to(torch.float32), torch.sin(angle).to(torch.float32)
    w = torch.cat([s["weights"][0].expand(Hq, D), s["weights"][1].expand(H, D)])
    z = x[:, : Hq + H].to(torch.float32)
    z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS) * w
    a, b = z[..., :half], z[..., half : 2 * half]
    z = torch.cat([a * cos - b * sin, b * cos + a * sin, z[..., 2 * half :]], -1).to(x.dtype)
    return [z[:, :Hq], z[:, Hq:]]


# --- rows into the cache and back ---------------------------------------------------------


def _planes(codes):
    """The layouts of K and of V of codes, f32 whole numbers [P, H, ps, D]."""
    byte = (codes + 128).to(torch.uint8)
    P, H, ps, D = byte.shape
    return byte, byte.view(P, H, ps // 16, 16, D).transpose(3, 4).contiguous()


def _cache(g, P, c):
    """A filled cache: codes of normal rows under scales of unlike sizes."""
    H, ps, D = c["Hkv"], c["ps"], c["D"]
    k, v = (_planes((_randn(g, P, H, ps, D) * 36).round().clamp(-127, 127))[i] for i in range(2))
    ks, vs = (_rand(g, 0.5, 1.5, P, H, ps // 16) / 36 for _ in range(2))
    return {"k_codes": k, "k_scales": ks, "v_codes": v, "v_scales": vs, "P": P, "H": H, "ps": ps, "D": D}


def _prepare_append(c, seed):
    """Request i adds its rows behind 7 i mod 16 tokens of a block begun earlier, through pages at random."""
    g = _gen(seed)
    n, ps, H, D = c["n"], c["ps"], c["Hkv"], c["D"]
    rows, held = _spread(c["lo"], c["hi"], n), [7 * i % 16 for i in range(n)]
    pages = [-(-(a + b) // ps) for a, b in zip(rows, held)]
    P, m = sum(pages) + 3, sum(rows)
    order = torch.randperm(P, generator=g, device="cuda")
    rows, held, pages = _ints(rows).long(), _ints(held).long(), _ints(pages).long()
    first = torch.cumsum(pages, 0) - pages

    def slots(begin, count):  # positions begin .. begin + count - 1 of each request
        r = torch.repeat_interleave(torch.arange(n, device="cuda"), count)
        at = torch.arange(r.numel(), device="cuda") - (torch.cumsum(count, 0) - count)[r] + begin[r]
        return (order[first[r] + at // ps] * ps + at % ps).to(torch.int32)

    new, look = slots(held, rows), slots(torch.zeros_like(held), held + rows)
    # k and v are parts of the projections' stacked rows, heads of unlike sizes
    x = (_randn(g, m, 3, H, D) * _rand(g, 0.5, 2.0, H, 1)).to(_TORCH[c["dtype"]])
    out = [torch.empty(look.numel(), H, D, dtype=_TORCH[c["dtype"]], device="cuda") for _ in range(2)]
    return {"op": "append", "cache": _cache(g, P, c), "x": x, "slots": new, "look": look, "out": out,
            "dtype": c["dtype"]}


def _read_plain(s):
    c, slots = s["cache"], s["look"].long()
    page, row = slots // c["ps"], slots % c["ps"]
    k = (c["k_codes"][page, :, row].to(torch.float32) - 128) * c["k_scales"][page, :, row // 16, None]
    v = (c["v_codes"][page, :, row // 16, :, row % 16].to(torch.float32) - 128) * c["v_scales"][page, :, row // 16, None]
    return [k.to(_TORCH[s["dtype"]]), v.to(_TORCH[s["dtype"]])]


def _append_plain(s):
    c, slots = s["cache"], s["slots"].long()
    P, H, ps, D = c["P"], c["H"], c["ps"], c["D"]
    block, row = slots // 16, slots % 16
    begun = torch.zeros(P * ps // 16, dtype=torch.bool, device="cuda")
    begun[block[row == 0]] = True  # blocks that begin anew
    x = s["x"][:, 1:].to(torch.float32)  # [m, 2, H, D]
    top = torch.zeros(P * ps // 16, 2, H, device="cuda").index_reduce_(0, block, x.abs().amax(-1), "amax")
    planes = (c["k_codes"].view(P, H, ps // 16, 16, D), c["v_codes"].transpose(3, 4))
    for i, (codes, scales) in enumerate(zip(planes, (c["k_scales"], c["v_scales"]))):
        old = scales.transpose(1, 2).reshape(-1, H)
        old = torch.where(begun[:, None], torch.zeros_like(old), old)
        new = torch.maximum(old, _scale_of(top[:, i]))  # [blocks, H]
        ratio = torch.where(new > old, old / new, torch.ones_like(new))
        ratio = ratio.view(P, ps // 16, H).transpose(1, 2)[..., None, None]
        codes.copy_((torch.round((codes.to(torch.float32) - 128) * ratio) + 128).to(torch.uint8))
        page, b = block * 16 // ps, block % (ps // 16)
        codes[page, :, b, row] = (_codes_at(x[:, i], new[block][..., None]) + 128).to(torch.uint8)
        scales.copy_(torch.where(begun[:, None] | (top[:, i] > 0), new, scales.transpose(1, 2).reshape(-1, H))
                     .view(P, ps // 16, H).transpose(1, 2))
    return _read_plain(s)


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
    return {"op": "attn", "q": q, "row_start": starts, "lens": lens, "table": table, "cache": cache, "n": c["n"],
            "Hq": c["Hq"], "max_rows": max(rows), "max_len": max(ls), "dtype": c["dtype"], "out": torch.empty_like(q),
            "lse": torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")}


def _attn_plain(s):
    c, q, lens = s["cache"], s["q"], s["lens"].long()
    n, H, D, ps = s["n"], c["H"], c["D"], c["ps"]
    G, S, L = s["Hq"] // H, s["max_len"], s["max_rows"]
    W = -(-S // ps)
    page = s["table"][:, :W].long().clamp(min=0)  # pages past a request's length: masked below
    k = (c["k_codes"][page].to(torch.float32) - 128).view(n, W, H, ps // 16, 16, D) * c["k_scales"][page][..., None, None]
    k = k.transpose(1, 2).reshape(n, H, W * ps, D)[:, :, :S]
    v = (c["v_codes"][page].to(torch.float32) - 128) * c["v_scales"][page][..., None, None]
    v = v.transpose(4, 5).transpose(1, 2).reshape(n, H, W * ps, D)[:, :, :S]
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
    o = torch.bmm(e.view(n * H, G * L, S), v.contiguous().view(n * H, S, D)).view(n, H, G, L, D) / total
    lse = (top + torch.log(total))[..., 0]
    o, lse = o.permute(0, 3, 1, 2, 4)[live], lse.permute(0, 3, 1, 2)[live]  # the rows in order
    return o.reshape(q.shape).to(q.dtype), lse.reshape(q.shape[:2])


# --- what a measuring program calls ---------------------------------------------------------

_PREPARE = {"linear": _prepare_linear, "heads": _prepare_heads, "append": _prepare_append, "attn": _prepare_attn}
_PLAIN = {"linear": _linear_plain, "heads": _heads_plain, "append": _append_plain, "attn": _attn_plain}


def prepare(case, seed):
    return _PREPARE[case["op"]](case, seed)


def _bind(s):
    """The C ABI calls of one pass with their arguments bound, as a host binding holds them, and its outputs."""
    import ctypes
    import functools

    from torchnative_amd import _lib

    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    code = _CODE[s["dtype"]]
    if s["op"] == "linear":
        x, w = s["x"], s["w"]
        m, k = x.shape
        need = L.tn_i8_linear_work_bytes(m, k)
        s["work"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        call = functools.partial(L.tn_i8_linear, st, p(x), code, m, k, p(w), p(s["scales"]), w.shape[0],
                                 None if s["bias"] is None else p(s["bias"]), p(s["work"]), need, p(s["y"]),
                                 _CODE[s["out"]])
        return _lib.check, [call], s["y"]
    if s["op"] == "heads":
        x, Hq, H = s["x"], s["Hq"], s["H"]
        D = x.shape[2]
        call = functools.partial(L.tn_qk_norm_rope, st, code, p(x), x.stride(0), Hq, p(x[:, Hq:]), x.stride(0), H,
                                 x.shape[0], D, p(s["weights"][0]), p(s["weights"][1]), EPS, p(s["freq"]),
                                 2 * s["freq"].shape[0], p(s["pos"]), p(s["out"][0]), Hq * D, p(s["out"][1]), H * D)
        return _lib.check, [call], s["out"]
    c = s["cache"]
    pages = _lib.Q8Cache(p(c["k_codes"]), p(c["k_scales"]), p(c["v_codes"]), p(c["v_scales"]), c["P"], c["ps"], c["H"],
                         c["D"])
    ref = ctypes.byref(pages)
    if s["op"] == "attn":
        q, n, Hq = s["q"], s["n"], s["Hq"]
        T = q.shape[0]
        floats = L.tn_sdpa_paged_q8_work_floats(ref, n, T, Hq, s["max_rows"], s["max_len"])
        s["work"] = torch.empty(max(floats, 1), dtype=torch.float32, device="cuda")
        call = functools.partial(L.tn_sdpa_paged_q8, st, ref, code, p(q), Hq * c["D"], T, Hq, n, p(s["row_start"]),
                                 p(s["lens"]), p(s["table"]), s["table"].shape[1], s["max_rows"], s["max_len"],
                                 float("nan"), p(s["work"]), floats, p(s["out"]), p(s["lse"]))
        return _lib.check, [call], (s["out"], s["lse"])
    x = s["x"]
    append = functools.partial(L.tn_kv_append_q8, st, ref, code, p(x[:, 1]), p(x[:, 2]), x.shape[0], x.stride(0),
                               p(s["slots"]))
    read = functools.partial(L.tn_kv_read_q8, st, ref, p(s["look"]), s["look"].numel(), code, p(s["out"][0]),
                             p(s["out"][1]))
    return _lib.check, [append, read], s["out"]


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


def _exact_codes(x, top):
    """Codes and scales, which f32 steps define: (codes f64, scales f64) of f32 rows x whose largest size is `top`."""
    scale = torch.maximum(top / 127.0, torch.full_like(top, TINY)) * (top > 0)
    inv = torch.where(scale == 0, scale, scale.reciprocal())
    return (x * inv).double().round().clamp(-127, 127), scale.double()


def exact(case, seed):
    c = case
    if c["op"] == "linear":
        s = _prepare_linear(c, seed)
        x = s["x"].float()
        codes, sx = _exact_codes(x, x.abs().max(1, keepdim=True).values)
        y = torch.matmul(codes, s["w"][:, : c["k"]].double().t().contiguous()) * sx * s["scales"].double()
        return y if s["bias"] is None else y + s["bias"].double()
    if c["op"] == "heads":
        s = _prepare_heads(c, seed)
        half = c["rot"] // 2
        theta = torch.outer(s["pos"].double(), s["freq"].double())[:, None]
        parts = (s["x"][:, : c["Hq"]], s["x"][:, c["Hq"] : c["Hq"] + c["Hkv"]])
        out = []
        for z, w in zip(parts, s["weights"]):
            z = z.double()
            z = z / (z.pow(2).sum(-1, keepdim=True) / c["D"] + EPS).sqrt() * w.double()
            turned = z.clone()
            turned[..., :half] = z[..., :half] * theta.cos() - z[..., half : c["rot"]] * theta.sin()
            turned[..., half : c["rot"]] = z[..., half : c["rot"]] * theta.cos() + z[..., :half] * theta.sin()
            out.append(turned)
        return out

    def stored(cache):  # [P, H, ps, D] of K and of V, element by element out of the layouts above
        t = torch.arange(cache["ps"], device="cuda")
        k = (cache["k_codes"].double() - 128) * cache["k_scales"].double()[:, :, t // 16, None]
        v = cache["v_codes"][:, :, t // 16, :, t % 16].permute(1, 2, 0, 3)
        return k, (v.double() - 128) * cache["v_scales"].double()[:, :, t // 16, None]

    if c["op"] == "append":
        s = _prepare_append(c, seed)
        at, new = s["look"].long(), s["slots"].long()
        x = s["x"][:, 1:].float()
        H, D, ps = c["Hkv"], c["D"], c["ps"]
        blocks, of = torch.unique(at // 16, return_inverse=True)  # the blocks that are looked at, ascending
        which = torch.searchsorted(blocks, new // 16)
        seen = torch.zeros(blocks.numel(), 16, dtype=torch.bool, device="cuda")
        seen[which, new % 16] = True
        out = []
        for i, name in enumerate("kv"):
            codes = s["cache"][name + "_codes"]
            if name == "v":
                codes = codes.transpose(3, 4)
            codes = codes.reshape(-1, H, ps // 16, 16, D).transpose(1, 2).reshape(-1, H, 16, D)[blocks].float() - 128
            old = s["cache"][name + "_scales"].transpose(1, 2).reshape(-1, H)[blocks]
            old = torch.where(seen[:, :1], torch.zeros_like(old), old)
            rows = torch.zeros(blocks.numel(), 16, H, D, device="cuda")
            rows[which, new % 16] = x[:, i]
            top = rows.abs().amax((1, 3))
            scale = torch.maximum(old, torch.maximum(top / 127.0, torch.full_like(top, TINY)) * (top > 0))
            kept = torch.where((scale > old)[..., None, None], (codes * (old / scale)[..., None, None]).round(), codes)
            inv = torch.where(scale == 0, scale, scale.reciprocal())
            fresh = (rows.transpose(1, 2) * inv[..., None, None]).round().clamp(-127, 127)
            y = torch.where(seen[:, None, :, None], fresh, kept).double() * scale.double()[..., None, None]
            out.append(y[of, :, at % 16])
        return out
    q, starts, lens, table, cache = _attn_inputs(c, seed)
    if cache["P"] * c["Hkv"] * c["ps"] * c["D"] > 600e6:
        return None
    k, v = stored(cache)
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
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
    if c["op"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k * _SIZE[c["dtype"]] + n * k + 4 * n * (2 if c["bias"] else 1) + m * n * _SIZE[c["out"]],
                "flops": 2 * m * n * k}
    if c["op"] == "heads":
        row = (c["Hq"] + c["Hkv"]) * c["D"]
        return {"bytes": c["m"] * (2 * row * _SIZE[c["dtype"]] + 4), "flops": 8 * c["m"] * row}
    if c["op"] == "append":  # rows in and, of their blocks, out again; their codes written and read
        new = sum(_spread(c["lo"], c["hi"], c["n"]))
        look = new + sum(7 * i % 16 for i in range(c["n"]))
        row = 2 * c["Hkv"] * c["D"]
        return {"bytes": new * row * (_SIZE[c["dtype"]] + 1) + look * row * (_SIZE[c["dtype"]] + 1), "flops": 0}
    rows, lens = _lengths(c)
    size, D = _SIZE[c["dtype"]], c["D"]
    pairs = sum(a * b - a * (a - 1) / 2 for a, b in zip(rows, lens))
    return {"bytes": sum(lens) * c["Hkv"] * D * 2 + sum(rows) * c["Hq"] * (2 * D * size + 4)
            + 4 * sum(-(-x // c["ps"]) for x in lens), "flops": 4 * pairs * c["Hq"] * D}
