"""The token operators of ccnet_amd.ops as measurable cases: query/key normalisation with position rotation, the 8-bit
key/value cache (written, read back, attended over) and cross attention to states of another length.

`run` computes each in plain torch where `own` is false and through ccnet_amd.ops where it is true."""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
TINY = 2.0 ** -126  # a scale below the smallest normal number counts as zero


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one image's tokens of the Transformer at 640x640: 20x20 positions, d_model 256 in 2 heads, default precision
        {"name": "rope_frame", "op": "rope", "B": 400, "T": 1, "Hq": 2, "Hk": 2, "D": 128, "rot": 128, "pairs": "half", "dtype": "fp32", "far": 64},
        # a long prompt with shared key heads, far along its sequence, q and k as columns of one projection buffer
        {"name": "rope_prompt", "op": "rope", "B": 4, "T": 4099, "Hq": 32, "Hk": 8, "D": 128, "rot": 128, "pairs": "half", "dtype": "bf16", "far": 1 << 20},
        # one new token at each of the 20x20 positions, default precision
        {"name": "write_frame", "op": "write", "B": 400, "T": 1, "H": 2, "D": 128, "page": 16, "codes": "int8", "dtype": "fp32", "before": 63, "spread": 1},
        # prompts of different lengths written behind what the cache holds
        {"name": "write_prompt", "op": "write", "B": 6, "T": 4096, "H": 8, "D": 128, "page": 64, "codes": "fp8", "dtype": "bf16", "before": 1000, "spread": 2},
        # the tokens of up to 64 images read back
        {"name": "read_frame", "op": "read", "B": 400, "T": 64, "H": 2, "D": 128, "page": 16, "codes": "int8", "dtype": "fp32", "spread": 3},
        # long contexts read back for a consumer in 16 bits
        {"name": "read_prompt", "op": "read", "B": 8, "T": 8192, "H": 8, "D": 128, "page": 64, "codes": "fp8", "dtype": "bf16", "spread": 4},
        # the Transformer's decoder on 64 images against the states of 48 others, sequence-first as the framework lays it out
        {"name": "cross_frames", "op": "cross", "B": 400, "Sq": 64, "Sk": 48, "Hq": 2, "Hk": 2, "D": 128, "dtype": "fp32", "first": True, "mask": False, "spread": 0},
        # one token of a decoder against the 40x40 positions of a 1280x1280 image, padded, some of them masked
        {"name": "cross_token", "op": "cross", "B": 32, "Sq": 1, "Sk": 1600, "Hq": 16, "Hk": 16, "D": 64, "dtype": "bf16", "first": False, "mask": True, "spread": 5},
        # many queries against long states with shared heads
        {"name": "cross_long", "op": "cross", "B": 2, "Sq": 4096, "Sk": 8191, "Hq": 32, "Hk": 8, "D": 128, "dtype": "bf16", "first": False, "mask": False, "spread": 6},
        # one new image attends to those before it at each position, default precision
        {"name": "cache_frame", "op": "cache", "B": 400, "Sq": 1, "L": 64, "Hq": 2, "Hk": 2, "D": 128, "page": 16, "codes": "int8", "dtype": "fp32", "causal": True, "spread": 7},
        # a serving batch: one token each over contexts of different lengths
        {"name": "cache_batch", "op": "cache", "B": 64, "Sq": 1, "L": 8192, "Hq": 32, "Hk": 8, "D": 128, "page": 64, "codes": "fp8", "dtype": "bf16", "causal": True, "spread": 8},
        # a few tokens at once at the end of one very long context
        {"name": "cache_long", "op": "cache", "B": 1, "Sq": 5, "L": 131071, "Hq": 32, "Hk": 8, "D": 128, "page": 32, "codes": "int8", "dtype": "bf16", "causal": True, "spread": 0},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "cross", "cache"])
    dtype, codes = rng.choice(["bf16", "fp32"]), rng.choice(["int8", "fp8"])
    Hk = rng.choice([1, 2, 3, 4, 8])
    Hq, spread = Hk * rng.choice([1, 2, 4, 7]), rng.randrange(1, 1 << 20)
    page = rng.choice([16, 32, 64, 128])
    if op == "rope":
        D, T = rng.choice([32, 40, 64, 80, 96, 128, 256]), _spread(rng, 1, 4099)
        B = _spread(rng, 1, max(1, min(400, 16000 // T)))
        return {"op": op, "B": B, "T": T, "Hq": Hq, "Hk": Hk, "D": D, "rot": rng.choice([D, D // 2 // 4 * 4]), "pairs": rng.choice(["half", "even"]), "dtype": dtype,
                "far": _spread(rng, 1, 1 << 20)}
    D = rng.choice([32, 64, 80, 96, 128, 256] if op == "cross" else [32, 64, 80, 128, 256])
    if op == "cross":
        Sq, Sk = _spread(rng, 1, 4096), _spread(rng, 1, 8191)
        while Sq * Sk * Hq * D > (2.0e11 if dtype == "bf16" else 2.5e10) or Sq * Sk * Hq > 2.0e9:
            Sk = (Sk + 1) // 2
        B = _spread(rng, 1, max(1, min(400, int((2.0e10 if dtype == "bf16" else 4.0e9) / (Sq * float(Sk) * Hq * D)))))
        return {"op": op, "B": B, "Sq": Sq, "Sk": Sk, "Hq": Hq, "Hk": Hk, "D": D, "dtype": dtype, "first": rng.random() < 0.3, "mask": rng.random() < 0.4, "spread": spread}
    if op == "cache":
        Sq, L = _spread(rng, 1, 64), _spread(rng, 1, 131071)
        B = _spread(rng, 1, max(1, min(400, int(2.5e8 / (L * Hk * D * (1 + Sq // 8))))))
        return {"op": op, "B": B, "Sq": Sq, "L": L, "Hq": Hq, "Hk": Hk, "D": D, "page": page, "codes": codes, "dtype": dtype, "causal": rng.random() < 0.7, "spread": spread}
    T = _spread(rng, 1, 8192 if op == "read" else 4096)
    B = _spread(rng, 1, max(1, min(400, 32000 // T)))
    c = {"op": op, "B": B, "T": T, "H": Hk, "D": D, "page": page, "codes": codes, "dtype": dtype, "spread": spread}
    return {**c, "before": _spread(rng, 1, 2000)} if op == "write" else c


def _lengths(spread, count, most, least=1):
    """`count` lengths of [least, most], the longest among them; all `most` where spread is 0."""
    if not spread:
        return [most] * count
    r = random.Random(spread)
    got = [r.randint(least, most) for _ in range(count)]
    got[r.randrange(count)] = most
    return got


# ------------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _heads(g, B, T, H, D, dtype, first=False, total=None):
    """Normal values (B, T, H, D), each head with a size of its own, as the columns of a wider buffer; `first`: the
    buffer's rows are sequence-first."""
    total = H if total is None else total
    lead = (T, B) if first else (B, T)
    x = torch.randn(*lead, total, D, device=DEV, generator=g)
    x *= torch.rand(total, 1, device=DEV, generator=g) + 0.5
    x = x.to(dtype)[:, :, :H]
    return x.transpose(0, 1) if first else x


def _table(g, B, width, spare=3):
    """Page tables (B, width) of distinct pages in no order, and how many pages there are."""
    n = B * width + spare
    return torch.randperm(n, device=DEV, generator=g)[:B * width].to(torch.int32).view(B, width).contiguous(), n


def _filled(g, n, H, page, D, codes):
    """A cache of n pages that holds normal values."""
    k = torch.randn(n, H, page, D, device=DEV, generator=g)
    v = torch.randn(n, H, D, page, device=DEV, generator=g)
    out = []
    for x in (k, v):
        s = x.abs().amax((2, 3)) * (1.0 / QMAX[codes])
        x = x / s[:, :, None, None]
        out.append((x.round_() if codes == torch.int8 else x).to(codes))
        out.append(s)
    return out[0], out[2], out[1], out[3]


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["op"] == "rope":
        dt, B, T = DTYPES[c["dtype"]], c["B"], c["T"]
        both = _heads(g, B, T, c["Hq"] + c["Hk"], c["D"], dt, total=c["Hq"] + 2 * c["Hk"])
        s["q"], s["k"] = both[:, :, :c["Hq"]], both[:, :, c["Hq"]:]
        s["wq"], s["wk"] = (1 + 0.1 * torch.randn(c["D"], device=DEV, generator=g) for _ in range(2))
        at = torch.randint(0, c["far"], (B, 1), device=DEV, generator=g)
        s["pos"] = (at + torch.arange(T, device=DEV)).to(torch.int32)
        half = c["rot"] // 2
        s["freqs"] = 10000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
        return s
    dt = DTYPES[c["dtype"]]
    if c["op"] == "cross":
        B, first = c["B"], c["first"]
        s["q"] = _heads(g, B, c["Sq"], c["Hq"], c["D"], dt, first)
        kv = _heads(g, B, c["Sk"], 2 * c["Hk"], c["D"], dt, first)
        s["k"], s["v"] = kv[:, :, :c["Hk"]], kv[:, :, c["Hk"]:]
        s["lens"] = torch.tensor(_lengths(c["spread"], B, c["Sk"], 0), dtype=torch.int32, device=DEV) if c["spread"] else None
        s["mask"] = torch.rand(B, c["Sk"], device=DEV, generator=g) < 0.8 if c["mask"] else None
        return s
    codes, B, page, D = CODES[c["codes"]], c["B"], c["page"], c["D"]
    H = c["Hk"] if c["op"] == "cache" else c["H"]
    if c["op"] == "write":
        start = _lengths(c["spread"] + 1, B, c["before"], 0)
        s["lens"] = torch.tensor(_lengths(c["spread"], B, c["T"], 0), dtype=torch.int32, device=DEV)
        s["start"] = torch.tensor(start, dtype=torch.int32, device=DEV)
        s["k"], s["v"] = (_heads(g, B, c["T"], H, D, dt) for _ in range(2))
        most = c["before"] + c["T"]
    else:
        most = c["L"] if c["op"] == "cache" else c["T"]
        s["lens"] = torch.tensor(_lengths(c["spread"], B, most, 0), dtype=torch.int32, device=DEV)
    s["table"], n = _table(g, B, -(-most // page))
    s["cache"] = _filled(g, n, H, page, D, codes)
    if c["op"] == "cache":
        s["q"] = _heads(g, B, c["Sq"], c["Hq"], D, dt)
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _norm_rope(x, w, pos, freqs, pairs, eps=1e-6):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w
    angle = pos.double()[:, :, None, None] * freqs
    cos, sin = angle.cos().float(), angle.sin().float()
    n = freqs.numel()
    a, b = (y[..., :n], y[..., n:2 * n]) if pairs == "half" else (y[..., 0:2 * n:2], y[..., 1:2 * n:2])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat((a, b), -1) if pairs == "half" else torch.stack((a, b), -1).flatten(-2)
    return torch.cat((turned, y[..., 2 * n:]), -1).to(x.dtype)


def _to_codes(x, scale, dtype):
    inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    y = x * inv
    y = torch.where(scale.isfinite(), y, torch.zeros_like(y)).clamp(-QMAX[dtype], QMAX[dtype])
    return (y.round() if dtype == torch.int8 else y).to(dtype)


def _write(x, codes, scales, table, start, lens, page):
    """New tokens x (B, T, H, D) into codes (pages, H, page, D), seen through a transposed view for the values."""
    B, T = x.shape[:2]
    slots = min((T + page - 2) // page + 1, table.shape[1])
    at = start.long()[:, None] // page + torch.arange(slots, device=x.device)
    tok = at[:, :, None] * page + torch.arange(page, device=x.device)
    begin, end = start.long()[:, None, None], (start + lens).long()[:, None, None]
    new = (tok >= begin) & (tok < end)
    had = tok < begin
    touched = new.any(-1) & (at < table.shape[1])
    pages = table.gather(1, at.clamp(max=table.shape[1] - 1)).long()[touched]
    rows = torch.arange(B, device=x.device)[:, None, None]
    fresh = x[rows, (tok - begin).clamp(0, T - 1)][touched].float().transpose(1, 2)
    new, had = new[touched][:, None, :, None], had[touched][:, None, :, None]
    old = codes.view(torch.uint8)[pages].view(codes.dtype)
    before = torch.where(had.any(2)[..., 0], scales[pages], torch.zeros_like(scales[pages]))
    amax = torch.where(new, fresh.abs(), torch.zeros_like(fresh)).amax((2, 3))
    scale = torch.maximum(before, amax * (1.0 / QMAX[codes.dtype]))
    scale = torch.where(scale < TINY, torch.zeros_like(scale), scale)
    wide = scale[:, :, None, None]
    kept = _to_codes(old.float() * before[:, :, None, None], wide, codes.dtype)
    put = torch.where(new, _to_codes(fresh, wide, codes.dtype).view(torch.uint8), torch.where(had, kept.view(torch.uint8), old.view(torch.uint8)))
    codes.view(torch.uint8)[pages] = put
    scales[pages] = scale


def _gathered(codes, scales, table, page):
    """The values (B, H, tokens, D) behind the page tables, in 32 bits; codes (pages, H, page, D) or a transposed view."""
    at = table.long().clamp(min=0)
    x = codes.view(torch.uint8)[at].view(codes.dtype).float() * scales[at][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _attend(q, k, v, seen, scale):
    """q (B, Hk, rows, D), k and v (B, Hk, keys, D), seen (B, 1, rows or 1, keys): softmax(scale q k) v, 0 where nothing is seen."""
    p = torch.matmul(q * scale, k.transpose(2, 3).contiguous())
    p = p.masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)


def _by_group(q, Hk):
    """(B, S, Hq, D) -> (B, Hk, S * G, D), rows by query, then by head of the group."""
    B, S, Hq, D = q.shape
    return q.reshape(B, S, Hk, Hq // Hk, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, S * (Hq // Hk), D)


def _from_group(o, S):
    B, Hk, rows, D = o.shape
    return o.reshape(B, Hk, S, rows // S, D).permute(0, 2, 1, 3, 4).reshape(B, S, Hk * (rows // S), D)


def _seen_causal(lens, Sq, G, keys, causal):
    """Which of `keys` tokens each of the Sq * G rows sees: (B, 1, Sq * G, keys)."""
    ends = lens.long()[:, None] - (torch.arange(Sq - 1, -1, -1, device=lens.device) if causal else torch.zeros(Sq, device=lens.device, dtype=torch.long))
    return torch.arange(keys, device=lens.device) < ends.repeat_interleave(G, 1)[:, None, :, None]


def _plain(s):
    c = s["case"]
    if c["op"] == "rope":
        return [_norm_rope(s["q"], s["wq"], s["pos"], s["freqs"], c["pairs"]), _norm_rope(s["k"], s["wk"], s["pos"], s["freqs"], c["pairs"])]
    if c["op"] == "cross":
        B, Sk = c["B"], c["Sk"]
        seen = torch.ones(B, Sk, dtype=torch.bool, device=DEV)
        if s["lens"] is not None:
            seen = torch.arange(Sk, device=DEV) < s["lens"][:, None]
        if s["mask"] is not None:
            seen = seen & s["mask"]
        k, v = (t.float().transpose(1, 2).contiguous() for t in (s["k"], s["v"]))
        o = _attend(_by_group(s["q"].float(), c["Hk"]), k, v, seen[:, None, None], c["D"] ** -0.5)
        return _from_group(o, c["Sq"]).to(s["q"].dtype)
    page = c["page"]
    kc, vc, ks, vs = s["cache"]
    if c["op"] == "write":
        _write(s["k"], kc, ks, s["table"], s["start"], s["lens"], page)
        _write(s["v"], vc.transpose(2, 3), vs, s["table"], s["start"], s["lens"], page)
        return [kc, vc, ks, vs]
    k, v = _gathered(kc, ks, s["table"], page), _gathered(vc.transpose(2, 3), vs, s["table"], page)
    if c["op"] == "read":
        there = (torch.arange(c["T"], device=DEV) < s["lens"][:, None])[:, :, None, None]
        return [torch.where(there, x.transpose(1, 2)[:, :c["T"]], torch.zeros((), device=DEV)).to(DTYPES[c["dtype"]]) for x in (k, v)]
    seen = _seen_causal(s["lens"], c["Sq"], c["Hq"] // c["Hk"], k.shape[2], c["causal"])
    o = _attend(_by_group(s["q"].float(), c["Hk"]), k, v, seen, c["D"] ** -0.5)
    return _from_group(o, c["Sq"]).to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from ccnet_amd import ops
    c = s["case"]
    if c["op"] == "rope":
        q, k = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (s["q"], s["k"]))
        ops.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["freqs"], q, k, eps=1e-6, interleaved=c["pairs"] == "even")
        return [q, k]
    if c["op"] == "cross":
        out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=s["q"].device)
        ops.cross_attention(s["q"], s["k"], s["v"], out, lens=s["lens"], key_mask=s["mask"])
        return out
    cache = ops.Cache8(*s["cache"])
    if c["op"] == "write":
        ops.kv_cache_write(s["k"], s["v"], cache, s["table"], s["start"], lens=s["lens"])
        return list(s["cache"])
    if c["op"] == "read":
        k, v = (torch.zeros(c["B"], c["T"], c["H"], c["D"], dtype=DTYPES[c["dtype"]], device=DEV) for _ in range(2))
        ops.kv_cache_read(cache, s["table"], s["lens"], k, v)
        return [k, v]
    out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=s["q"].device)
    ops.cache_attention(s["q"], cache, s["table"], s["lens"], out, causal=c["causal"])
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    size = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "rope":
        n = c["B"] * c["T"] * (c["Hq"] + c["Hk"])
        return {"bytes": 2 * n * c["D"] * size, "flops": n * (4 * c["D"] + 3 * c["rot"])}
    if c["op"] == "cross":
        keys = sum(_lengths(c["spread"], c["B"], c["Sk"], 0))
        return {"bytes": (2 * c["B"] * c["Sq"] * c["Hq"] + 2 * keys * c["Hk"]) * c["D"] * size, "flops": 4 * keys * c["Sq"] * c["Hq"] * c["D"]}
    if c["op"] == "cache":
        keys = sum(_lengths(c["spread"], c["B"], c["L"], 0))
        return {"bytes": 2 * c["B"] * c["Sq"] * c["Hq"] * c["D"] * size + 2 * keys * c["Hk"] * (c["D"] + 4 / c["page"]), "flops": 4 * keys * c["Sq"] * c["Hq"] * c["D"]}
    tokens = sum(_lengths(c["spread"], c["B"], c["T"], 0))
    n = 2 * tokens * c["H"] * c["D"]
    return {"bytes": n * (size + 1), "flops": 2 * n}


# ------------------------------------------------------------------------------------------------------------ 64 bits
def _exact_softmax(q, k, v, ends):
    """One head's rows q (R, D) over k, v (n, D), row r seeing the first ends[r] keys."""
    z = (q @ k.t().contiguous()) / math.sqrt(q.shape[1])
    hidden = torch.arange(k.shape[0], device=q.device) >= ends[:, None]
    z[hidden] = -math.inf
    lse = torch.logsumexp(z, 1, keepdim=True)
    w = torch.where(lse > -math.inf, (z - lse).exp(), torch.zeros_like(z))
    return w @ v


def _exact_heads(q, k, v, ends):
    """q (S, Hq, D), k and v (n, Hk, D) in 64 bits, ends (S,): (S, Hq, D)."""
    G = q.shape[1] // k.shape[1]
    heads = [_exact_softmax(q[:, h], k[:, h // G].contiguous(), v[:, h // G].contiguous(), ends) for h in range(q.shape[1])]
    return torch.stack(heads, 1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rope":
        got = []
        for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
            x = x.double()
            y = x / (x.pow(2).sum(-1, keepdim=True) / c["D"] + 1e-6).sqrt() * w.double()
            n = c["rot"] // 2
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["pos"].double()[..., None] * s["freqs"])[:, :, None]
            if c["pairs"] == "half":
                z = torch.complex(y[..., :n].contiguous(), y[..., n:2 * n].contiguous()) * turn
                y[..., :n], y[..., n:2 * n] = z.real, z.imag
            else:
                y[..., :2 * n] = torch.view_as_real(torch.view_as_complex(y[..., :2 * n].unflatten(-1, (n, 2)).contiguous()) * turn).flatten(-2)
            got.append(y)
        return got
    if c["op"] == "cross":
        if c["B"] * c["Hq"] > 2000:
            return None
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        for b in range(c["B"]):
            keep = torch.ones(c["Sk"], dtype=torch.bool, device=DEV)
            if s["lens"] is not None:
                keep[int(s["lens"][b]):] = False
            if s["mask"] is not None:
                keep &= s["mask"][b]
            k, v = s["k"][b][keep].double(), s["v"][b][keep].double()
            if k.shape[0]:
                out[b] = _exact_heads(s["q"][b].double(), k, v, torch.full((c["Sq"],), k.shape[0], device=DEV))
        return out
    page = c["page"]
    kc, vc, ks, vs = s["cache"]
    lens = s["lens"].tolist()
    if c["op"] == "write":
        scales = []
        for x, sc in ((s["k"], ks), (s["v"], vs)):
            sc = sc.double()
            for b, (n, at) in enumerate(zip(lens, s["start"].tolist())):
                for p in range(at // page, -(-(at + n) // page) if n else 0):
                    i = int(s["table"][b, p])
                    a = x[b, max(0, p * page - at):max(0, min(n, (p + 1) * page - at))].double().abs().amax((0, 2)) / QMAX[kc.dtype]
                    sc[i] = torch.maximum(sc[i], a) if p * page < at else a
            scales.append(sc)
        return [None, None] + scales
    values = []
    for x, sc in ((kc, ks), (vc.transpose(2, 3), vs)):
        values.append([(x[s["table"][b, :-(-n // page)].long()].double() * sc[s["table"][b, :-(-n // page)].long()].double()[..., None, None])
                       .transpose(1, 2).reshape(-1, x.shape[1], c["D"])[:n] for b, n in enumerate(lens)])
    if c["op"] == "read":
        out = [torch.zeros(c["B"], c["T"], c["H"], c["D"], dtype=torch.float64, device=DEV) for _ in range(2)]
        for o, rows in zip(out, values):
            for b, r in enumerate(rows):
                o[b, :r.shape[0]] = r
        return out
    if c["B"] * c["Hq"] > 4000:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    back = torch.arange(c["Sq"] - 1, -1, -1, device=DEV) if c["causal"] else torch.zeros(c["Sq"], dtype=torch.long, device=DEV)
    for b, n in enumerate(lens):
        if n:
            out[b] = _exact_heads(s["q"][b].double(), values[0][b], values[1][b], n - back)
    return out
