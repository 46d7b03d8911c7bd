"""The token operators against plain 64-bit implementations: query/key norm + rotation, the 8-bit cache (written, read, attended over)
and cross attention.  Tolerances are bounds: half a step of the output type (finfo.eps / 2, relative), half a bf16 step for every
probability that a matrix instruction takes in bf16, and the roundings of 32-bit sums as counted beside each."""
import numpy as np
import pytest
import torch

from ccnet_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
U24 = 2.0 ** -24


def gen(seed):
    return torch.Generator().manual_seed(seed)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def heads(g, B, T, H, D, dtype, layout="plain"):
    """(B, T, H, D) on the GPU: contiguous, columns of a wider buffer, sequence-first, or heads before tokens."""
    if layout == "slice":
        return torch.randn(B, T, H + 3, D, generator=g).to(dtype).to(DEV)[:, :, 2:H + 2]
    if layout == "first":
        return torch.randn(T, B, H, D, generator=g).to(dtype).to(DEV).transpose(0, 1)
    if layout == "heads":
        return torch.randn(B, H, T, D, generator=g).to(dtype).to(DEV).transpose(1, 2)
    return torch.randn(B, T, H, D, generator=g).to(dtype).to(DEV)


def blank(shape, dtype, layout="plain"):
    B, T, H, D = shape
    if layout == "first":
        return torch.full((T, B, H, D), 7.0, dtype=dtype, device=DEV).transpose(0, 1)
    if layout == "slice":
        return torch.full((B, T, H + 3, D), 7.0, dtype=dtype, device=DEV)[:, :, 2:H + 2]
    return torch.full(shape, 7.0, dtype=dtype, device=DEV)


# ------------------------------------------------------------------------------------------------------------ norm + rotation
def rope_ref(x, w, pos, freqs, interleaved, eps):
    """(result, |n1| + |n2| of each element's pair) in 64 bits."""
    x = x.double().cpu()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w.double().cpu()
    a = pos.double().cpu()[:, :, None, None] * freqs.cpu()
    c, s = torch.cos(a), torch.sin(a)
    n = freqs.numel()
    out, mag = y.clone(), y.abs()
    i1 = torch.arange(0, 2 * n, 2) if interleaved else torch.arange(n)
    i2 = i1 + 1 if interleaved else i1 + n
    y1, y2 = y[..., i1], y[..., i2]
    out[..., i1], out[..., i2] = y1 * c - y2 * s, y2 * c + y1 * s
    mag[..., i1] = mag[..., i2] = y1.abs() + y2.abs()
    return out, mag


def check_rope(got, x, w, pos, freqs, interleaved, eps):
    ref, mag = rope_ref(x, w, pos, freqs, interleaved, eps)
    # 32-bit: the sum of squares adds at most 16 values per lane and 6 levels of lanes (22 U), halved by the root; root, quotient,
    # two products (4 U), cosine and sine 2 ulp each of an argument rounded once (pi/2 + 4 U), the rotation 3 U: under 32 U
    tol = half_step(got.dtype) * (ref.abs() + 32 * U24 * mag) + 32 * U24 * mag + 1e-37
    bad = (got.double().cpu() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float((got.double().cpu() - ref).abs().max()))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,Hq,Hk,D,rot,layout", [(1, 1, 1, 1, 8, 8, "plain"), (3, 5, 4, 2, 128, 128, "slice"), (2, 7, 3, 1, 64, 32, "first"), (1, 33, 2, 2, 40, 20, "plain"),
                                                    (2, 3, 7, 7, 80, 80, "plain"), (1, 9, 2, 1, 96, 24, "heads"), (1, 5, 3, 3, 256, 256, "plain"), (1, 4, 2, 1, 256, 10, "plain"),
                                                    (1, 6, 2, 2, 72, 0, "plain"), (2, 700, 32, 8, 128, 64, "plain"), (400, 1, 2, 2, 128, 128, "slice")])
def test_qk_norm_rope(dtype, interleaved, B, T, Hq, Hk, D, rot, layout):
    g = gen(B * 31 + T * 7 + D + rot)
    q, k = heads(g, B, T, Hq, D, dtype, layout), heads(g, B, T, Hk, D, dtype, layout)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(DEV) for _ in range(2))
    pos = torch.randint(0, 1 << 20, (B, T), generator=g, dtype=torch.int32).to(DEV)
    freqs = ops.rope_freqs(rot, device=DEV)
    qo, ko = blank(q.shape, dtype, layout), blank(k.shape, dtype, layout)
    ops.qk_norm_rope(q, k, wq, wk, pos, freqs, qo, ko, eps=1e-6, interleaved=interleaved)
    check_rope(qo, q, wq, pos, freqs, interleaved, 1e-6)
    check_rope(ko, k, wk, pos, freqs, interleaved, 1e-6)


def test_qk_norm_rope_in_place_far_positions_and_without_weights():
    g = gen(5)
    both = heads(g, 2, 9, 6, 128, F32)
    q, k = both[:, :, :4], both[:, :, 4:]
    q0, k0 = q.clone(), k.clone()
    pos = torch.tensor([[0, 1, -1, 2 ** 31 - 1, -2 ** 31, 123456789, 1 << 24, (1 << 24) + 1, 7]], dtype=torch.int32, device=DEV).expand(2, 9)
    freqs = ops.rope_freqs(128, base=500000.0, device=DEV)
    ops.qk_norm_rope(q, k, None, None, pos, freqs, q, k, eps=1e-5)
    check_rope(q, q0, None, pos, freqs, False, 1e-5)
    check_rope(k, k0, None, pos, freqs, False, 1e-5)
    # queries alone, a row of zeros stays zeros, nothing to do is no error
    z = torch.zeros(1, 2, 1, 64, dtype=BF, device=DEV)
    ops.qk_norm_rope(z, None, None, None, torch.zeros(1, 2, dtype=torch.int32, device=DEV), ops.rope_freqs(64, device=DEV), z, None)
    assert not z.any()
    e = torch.zeros(0, 3, 2, 64, dtype=BF, device=DEV)
    ops.qk_norm_rope(e, e, None, None, torch.zeros(0, 3, dtype=torch.int32, device=DEV), ops.rope_freqs(64, device=DEV), e, e)


# ------------------------------------------------------------------------------------------------------------ cache
def quant(x, scale, dtype):
    """The documented rule in 32-bit numpy: every operation is correctly rounded, so the codes are equal bit for bit."""
    x, scale = np.asarray(x, np.float32), np.float32(scale)
    inv = np.float32(1) / scale if scale > 0 else np.float32(0)
    with np.errstate(all="ignore"):
        y = x * inv if np.isfinite(scale) else np.zeros_like(x)
    y = np.clip(y, -QMAX[dtype], QMAX[dtype])
    if dtype == torch.int8:
        return np.rint(y).astype(np.int8).view(np.uint8)
    return torch.from_numpy(y).to(dtype).view(torch.uint8).numpy()


def dequant(codes, dtype):
    return torch.from_numpy(np.ascontiguousarray(codes)).view(dtype).float().numpy()


class RefCache:
    """A cache as plain numpy: codes [pages][H][page][D] for both, keys and values."""

    def __init__(self, pages, page, H, D, dtype):
        self.page, self.dtype = page, dtype
        self.codes = [np.zeros((pages, H, page, D), np.uint8) for _ in range(2)]
        self.scales = [np.zeros((pages, H), np.float32) for _ in range(2)]

    def write(self, kv, table, start, lens):
        pages, H = self.scales[0].shape
        cap = table.shape[1] * self.page
        for codes, scales, x in zip(self.codes, self.scales, kv):
            x = x.float().cpu().numpy()
            for b in range(x.shape[0]):
                s0, n = min(max(int(start[b]), 0), cap), min(max(int(lens[b]), 0), x.shape[1])
                end = min(s0 + n, cap)
                for p in range(s0 // self.page, -(-end // self.page) if end > s0 else 0):
                    i = int(table[b, p])
                    if not 0 <= i < pages:
                        continue
                    a, z = max(s0, p * self.page), min(end, (p + 1) * self.page)
                    for h in range(H):
                        new = x[b, a - s0:z - s0, h]
                        old = scales[i, h] if a > p * self.page else np.float32(0)
                        sc = np.maximum(old, np.abs(new).max() * np.float32(1.0 / QMAX[self.dtype]))
                        if sc < np.float32(2.0 ** -126):
                            sc = np.float32(0)
                        k = a - p * self.page
                        if k and not sc == old:
                            with np.errstate(all="ignore"):
                                codes[i, h, :k] = quant(dequant(codes[i, h, :k], self.dtype) * old, sc, self.dtype)
                        codes[i, h, k:z - p * self.page] = quant(new, sc, self.dtype)
                        scales[i, h] = sc

    def values(self, which, row, n):
        """Tokens [0, n) of a page-table row, (n, H, D) in 32 bits as the device computes them: code * scale, rounded once."""
        pages, H, page, D = self.codes[0].shape
        out = np.zeros((n, H, D), np.float32)
        for j in range(n):
            i = int(row[j // page])
            if 0 <= i < pages:
                out[j] = dequant(self.codes[which][i, :, j % page], self.dtype) * self.scales[which][i][:, None]
        return out


def same_cache(cache, ref):
    k, v = cache.k.view(torch.uint8).cpu().numpy(), cache.v.view(torch.uint8).cpu().numpy().transpose(0, 1, 3, 2)
    for name, got, want in (("k", k, ref.codes[0]), ("v", v, ref.codes[1])):
        # e4m3 has two zeros; they stand for the same value
        g, w = (np.where(x == 0x80, 0, x) if ref.dtype != torch.int8 else x for x in (got, want))
        assert np.array_equal(g, w), (name, int((g != w).sum()))
    for got, want in ((cache.k_scale, ref.scales[0]), (cache.v_scale, ref.scales[1])):
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def pages_of(g, B, width, spare=2):
    n = B * width + spare
    return torch.randperm(n, generator=g)[:B * width].to(torch.int32).view(B, width).contiguous(), n


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page,H,D,layout", [(16, 2, 128, "slice"), (32, 1, 16, "plain"), (64, 3, 80, "first"), (128, 2, 256, "heads")])
def test_kv_cache_write_in_steps_and_read_back(codes, dtype, page, H, D, layout):
    g = gen(page + D)
    B, width = 4, 3
    table, n = pages_of(g, B, width)
    cache = ops.Cache8.empty(n, page, H, D, codes, DEV)
    ref = RefCache(n, page, H, D, codes)
    at = [0, 3, page - 1, page]
    # a few tokens, one token (most of them louder than what is there: the block is rounded again), many, none
    for step, (T, lens, gain) in enumerate([(5, [5, 1, 0, 4], 1.0), (1, [1, 1, 1, 1], 3.0), (page + 7, [page + 7, 2, page, 0], 0.5), (1, None, 1.0), (1, [0, 0, 0, 0], 1.0)]):
        k, v = heads(g, B, T, H, D, dtype, layout) * gain, heads(g, B, T, H, D, dtype, layout) * gain
        ops.kv_cache_write(k, v, cache, table.to(DEV), ints(at), lens=None if lens is None else ints(lens))
        lens = [T] * B if lens is None else lens
        ref.write((k, v), table, at, lens)
        same_cache(cache, ref)
        at = [a + min(m, T) for a, m in zip(at, lens)]
    T = max(at) + 2
    lens = [at[0], 1, at[2], 0]
    ko, vo = blank((B, T, H, D), dtype, layout if layout != "heads" else "plain"), blank((B, T, H, D), dtype)
    ops.kv_cache_read(cache, table.to(DEV), ints(lens), ko, vo)
    for which, o in ((0, ko), (1, vo)):
        for b in range(B):
            want = torch.from_numpy(ref.values(which, table[b], lens[b])).to(dtype)
            assert torch.equal(o[b, :lens[b]].cpu(), want)
            assert (o[b, lens[b]:] == 7.0).all()   # rows behind the sequence are left as they were


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_kv_cache_without_pages(codes):
    """Every entry names no page: writes are dropped, reads give zeros, rows behind the lengths stay."""
    g = gen(12)
    none = ops.Cache8.empty(0, 32, 2, 48, codes, DEV)
    table = ints([0, 1, -1, 2]).view(2, 2)
    k, v = heads(g, 2, 70, 2, 48, BF), heads(g, 2, 70, 2, 48, BF)
    ops.kv_cache_write(k, v, none, table, ints([0, 3]))
    ko, vo = blank(k.shape, BF), blank(k.shape, BF)
    ops.kv_cache_read(none, table, ints([70, 33]), ko, vo)
    for b, n in enumerate([64, 33]):   # (a table of two pages holds 64 tokens)
        for o in (ko, vo):
            assert not o[b, :n].any() and (o[b, n:] == 7.0).all()


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_kv_cache_edges(codes):
    """Zeros, values of every size, non-finite ones, tokens past the table, entries that name no page, lengths out of range."""
    g = gen(11)
    page, H, D, B = 16, 2, 32, 6
    table = torch.tensor([[0, 1], [2, 99], [-1, 3], [4, 5], [6, 7], [8, 9]], dtype=torch.int32)
    cache = ops.Cache8.empty(10, page, H, D, codes, DEV)
    ref = RefCache(10, page, H, D, codes)
    k, v = heads(g, B, 24, H, D, F32), heads(g, B, 24, H, D, F32)
    k[0, :, 0] = 0.0
    k[1, :, 0] *= 1e-40
    k[1, :, 1] *= 1e37
    v[3, 2, 0, 5] = float("nan")
    v[4, 20, 1, 7] = float("inf")
    k[5, 0, 0, 3] = float("-inf")
    start, lens = [0, 0, 0, 20, -5, 8], [24, 24, 24, 24, 1000, 24]
    for _ in range(2):   # the second time the same tokens meet what they left
        ops.kv_cache_write(k, v, cache, table.to(DEV), ints(start), lens=ints(lens))
        with np.errstate(all="ignore"):
            ref.write((k, v), table, start, lens)
        same_cache(cache, ref)
    ko, vo = blank((B, 24, H, D), F32), blank((B, 24, H, D), F32)
    ops.kv_cache_read(cache, table.to(DEV), ints([24, 24, 40, -3, 24, 24]), ko, vo)
    for b, n in enumerate([24, 24, 24, 0, 24, 24]):
        for which, o in ((0, ko), (1, vo)):
            with np.errstate(all="ignore"):
                assert np.array_equal(o[b, :n].cpu().numpy(), ref.values(which, table[b], n), equal_nan=True)
            assert (o[b, n:] == 7.0).all()
    assert torch.isnan(vo[4, 16:24, 1]).all() and torch.isfinite(vo[4, :16]).all()   # one block, one head


# ------------------------------------------------------------------------------------------------------------ attention
def attend_ref(q, k, v, seen, scale, dtype, pround):
    """One batch entry: q (S, Hq, D), k, v (n, Hk, D), seen (S, n) -> (result, tolerance) in 64 bits."""
    S, Hq, D = q.shape
    n, Hk = k.shape[:2]
    out, tol = torch.zeros(S, Hq, D, dtype=torch.float64), torch.full((S, Hq, D), 1e-37, dtype=torch.float64)
    for h in range(Hq):
        kh, vh = k[:, h // (Hq // Hk)], v[:, h // (Hq // Hk)]
        z = (q[:, h] @ kh.T) * scale
        z[~seen] = -np.inf
        # a score's 32-bit sum of D products, and the two factors behind it
        ds = ((q[:, h].abs() @ kh.abs().T) * abs(scale) * (D + 4) * U24).masked_fill(~seen, 0.0).amax(1, keepdim=True) if n else torch.zeros(S, 1, dtype=torch.float64)
        top = z.amax(1, keepdim=True) if n else torch.zeros(S, 1, dtype=torch.float64)
        p = torch.exp(z - torch.where(torch.isinf(top), torch.zeros_like(top), top)) if n else z
        total = p.sum(1, keepdim=True)
        p = torch.where(total > 0, p / total.clamp(min=1e-300), torch.zeros_like(p))
        live = seen.any(0)
        vz = torch.where(live[:, None], vh, torch.zeros_like(vh))
        o, a = p @ vz, p @ vz.abs()
        out[:, h] = o
        # weights: e^(+-ds) above and below the line, exp itself 8 U (argument up to 2^7 in units of U: |z| stays below 128 here), sums of n
        # terms and the rescalings, the probability's own rounding
        w = 2 * ds + (128 * 4 + 2 * n + 64) * U24 + pround
        tol[:, h] += a * w + half_step(dtype) * (o.abs() + a * w)
    return out, tol


def pround_of(dtype):
    return 2.0 ** -8 if dtype == BF else 0.0


def close(got, ref, tol):
    d = (got.double().cpu() - ref).abs()
    assert torch.isfinite(d).all()
    assert (d <= tol).all(), "off by %.3g of the bound" % float((d / tol).max())


CROSS = [(1, 1, 1, 1, 1, 8, "plain"), (2, 1, 300, 4, 4, 64, "slice"), (3, 5, 17, 7, 1, 40, "plain"), (2, 33, 64, 2, 2, 128, "first"), (1, 64, 65, 6, 2, 96, "heads"),
         (2, 130, 129, 4, 1, 80, "plain"), (1, 300, 513, 2, 1, 256, "slice"), (1, 1, 4099, 8, 2, 128, "plain"), (5, 16, 48, 2, 2, 32, "first"), (1, 257, 1000, 4, 2, 128, "plain"),
         (2, 3, 1000, 14, 2, 72, "heads"), (1, 9, 2500, 3, 3, 16, "plain")]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("B,Sq,Sk,Hq,Hk,D,layout", CROSS)
def test_cross_attention(dtype, masked, B, Sq, Sk, Hq, Hk, D, layout):
    g = gen(Sq * 13 + Sk + D)
    q, k, v = heads(g, B, Sq, Hq, D, dtype, layout) * 2, heads(g, B, Sk, Hk, D, dtype, layout), heads(g, B, Sk, Hk, D, dtype, layout)
    out = blank(q.shape, dtype, layout if layout != "heads" else "plain")
    lens = key_mask = None
    seen = torch.ones(B, Sk, dtype=torch.bool)
    if masked:
        n = torch.randint(0, Sk + 1, (B,), generator=g)
        n[0] = Sk
        key_mask = torch.rand(B, Sk, generator=g) < 0.7
        key_mask[0, :min(Sk, 70)] = False   # the first tile of keys is hidden whole
        seen = (torch.arange(Sk) < n[:, None]) & key_mask
        lens, key_mask = n.to(torch.int32).to(DEV), key_mask.to(DEV)
        hidden = ~seen.to(DEV)
        # what hidden rows hold must not matter
        k = torch.where(hidden[:, :, None, None], torch.tensor(float("nan"), dtype=dtype, device=DEV), k)
        v = torch.where(hidden[:, :, None, None], torch.tensor(float("inf"), dtype=dtype, device=DEV), v)
    ops.cross_attention(q, k, v, out, lens=lens, key_mask=key_mask)
    for b in range(B):
        kb, vb = (torch.where(seen[b][:, None, None], t[b].double().cpu(), torch.zeros((), dtype=torch.float64)) for t in (k, v))
        ref, tol = attend_ref(q[b].double().cpu(), kb, vb, seen[b].expand(Sq, Sk), D ** -0.5, dtype, pround_of(dtype))
        close(out[b], ref, tol)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_cross_attention_edges(dtype):
    g = gen(3)
    # no keys at all, a batch of nothing, all hidden by length or mask
    q = heads(g, 2, 3, 4, 64, dtype)
    out = blank(q.shape, dtype)
    none = torch.empty(2, 0, 2, 64, dtype=dtype, device=DEV)
    ops.cross_attention(q, none, none, out)
    assert not out.any()
    e = q[:0]
    ops.cross_attention(e, none[:0], none[:0], out[:0])
    k, v = heads(g, 2, 100, 2, 64, dtype), heads(g, 2, 100, 2, 64, dtype)
    out = blank(q.shape, dtype)
    ops.cross_attention(q, k, v, out, lens=ints([0, 0]))
    assert not out.any()
    out = blank(q.shape, dtype)
    mask = torch.zeros(2, 100, dtype=torch.bool, device=DEV)
    mask[1, 57] = True
    ops.cross_attention(q, k, v, out, key_mask=mask)
    assert not out[0].any()
    assert torch.equal(out[1], v[1, 57].repeat_interleave(2, 0).expand(3, 4, 64))   # one key: its value, whatever the score
    # scores at the end of the type's range: the largest takes all
    big = torch.zeros(1, 2, 1, 64, dtype=dtype, device=DEV)
    big[0, 0, 0, 0], big[0, 1, 0, 0] = 1e30, -1e30
    kk = torch.zeros(1, 70, 1, 64, dtype=dtype, device=DEV)
    kk[0, 33, 0, 0], kk[0, 44, 0, 0] = 100.0, -100.0
    vv = heads(g, 1, 70, 1, 64, dtype)
    o = blank(big.shape, dtype)
    ops.cross_attention(big, kk, vv, o, scale=1.0)
    assert torch.equal(o[0, 0, 0], vv[0, 33, 0]) and torch.equal(o[0, 1, 0], vv[0, 44, 0])
    # a NaN in a row that is seen shows in the rows that see it, and there alone
    v2 = v.clone()
    v2[0, 5, 1, 7] = float("nan")
    ops.cross_attention(q, k, v2, out, lens=ints([100, 100]))
    bad = torch.isnan(out)
    assert bad[0, :, 2:, 7].all() and int(bad.sum()) == 3 * 2
    # a broadcast input
    kb, vb = k[:1].expand(2, 100, 2, 64), v[:1].expand(2, 100, 2, 64)
    a, b = blank(q.shape, dtype), blank(q.shape, dtype)
    ops.cross_attention(q, kb, vb, a)
    ops.cross_attention(q, kb.contiguous(), vb.contiguous(), b)
    assert torch.equal(a, b)


# two row tiles per wave (many workgroups), every padded head size, split keys, one row more than the few-row kernels take
MANY = [(128, 33, 100, 2, 2, 32, "plain"), (130, 40, 70, 2, 2, 64, "first"), (64, 65, 129, 8, 4, 96, "slice"), (128, 33, 64, 2, 2, 128, "plain"), (256, 66, 33, 2, 2, 128, "plain"),
        (256, 65, 40, 2, 2, 40, "first"), (64, 125, 100, 8, 4, 32, "plain"), (64, 125, 70, 8, 4, 64, "slice"), (64, 125, 100, 8, 4, 96, "plain"), (64, 125, 65, 8, 4, 128, "first"), (1, 33, 3000, 1, 1, 64, "plain"), (1, 70, 2100, 3, 1, 32, "plain"), (2, 200, 1500, 1, 1, 256, "heads"), (1, 128, 1030, 2, 1, 80, "plain")]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("B,Sq,Sk,Hq,Hk,D,layout", MANY)
def test_cross_attention_with_many_rows(dtype, masked, B, Sq, Sk, Hq, Hk, D, layout):
    """As test_cross_attention; the first, a middle and the last batch entry against 64 bits."""
    g = gen(Sq * 17 + Sk + D + B)
    q, k, v = heads(g, B, Sq, Hq, D, dtype, layout) * 2, heads(g, B, Sk, Hk, D, dtype, layout), heads(g, B, Sk, Hk, D, dtype, layout)
    out = blank(q.shape, dtype, layout if layout != "heads" else "plain")
    n = torch.randint(0, Sk + 1, (B,), generator=g) if masked else torch.full((B,), Sk)
    n[-1] = Sk
    mask = torch.rand(B, Sk, generator=g) < 0.6 if masked else torch.ones(B, Sk, dtype=torch.bool)
    seen = (torch.arange(Sk) < n[:, None]) & mask
    ops.cross_attention(q, k, v, out, lens=n.to(torch.int32).to(DEV) if masked else None, key_mask=mask.to(DEV) if masked else None)
    assert torch.isfinite(out).all()
    for b in {0, B // 2, B - 1}:
        ref, tol = attend_ref(q[b].double().cpu(), k[b].double().cpu(), v[b].double().cpu(), seen[b].expand(Sq, Sk), D ** -0.5, dtype, pround_of(dtype))
        close(out[b], ref, tol)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Sq", [1, 20, 150])
def test_attention_in_place_negative_scale_and_rows_apart(dtype, Sq):
    """out = q; a negative and a zero scale; a query that is not a number spoils its own row and no other; the same call twice gives the same bits."""
    g = gen(Sq)
    q, k, v = heads(g, 2, Sq, 4, 64, dtype), heads(g, 2, 333, 2, 64, dtype), heads(g, 2, 333, 2, 64, dtype)
    mask = (torch.rand(2, 333, generator=g) < 0.8)
    for scale in (-0.3, 0.0, 0.125):
        out = blank(q.shape, dtype)
        ops.cross_attention(q, k, v, out, key_mask=mask.to(DEV), scale=scale)
        for b in range(2):
            ref, tol = attend_ref(q[b].double().cpu(), k[b].double().cpu(), v[b].double().cpu(), mask[b].expand(Sq, 333), scale, dtype, pround_of(dtype))
            close(out[b], ref, tol)
    again, own = blank(q.shape, dtype), q.clone()
    ops.cross_attention(q, k, v, again, key_mask=mask.to(DEV), scale=0.125)
    ops.cross_attention(own, k, v, own, key_mask=mask.to(DEV), scale=0.125)
    assert torch.equal(out, again) and torch.equal(out, own)
    bad = q.clone()
    bad[1, 0, 3, 5] = float("nan")
    ops.cross_attention(bad, k, v, again, key_mask=mask.to(DEV), scale=0.125)
    assert torch.isnan(again[1, 0, 3]).all()
    again[1, 0, 3] = out[1, 0, 3]
    assert torch.equal(again, out)
    # the same over a cache
    table, n = pages_of(g, 2, 6)
    cache, ref = fill_cache(g, table, n, 64, 2, 64, torch.int8, [333, 100])
    for scale in (-0.3, 0.0, 0.125):
        ops.cache_attention(q, cache, table.to(DEV), ints([333, 100]), out, scale=scale)
        for b, m in enumerate([333, 100]):
            r, tol = attend_ref(q[b].double().cpu(), values64(ref, 0, table[b], m), values64(ref, 1, table[b], m), torch.ones(Sq, m, dtype=torch.bool), scale, dtype, pround_of(dtype))
            close(out[b], r, tol)
    own = q.clone()
    ops.cache_attention(own, cache, table.to(DEV), ints([333, 100]), own, scale=0.125)
    assert torch.equal(out, own)
    ops.cache_attention(bad, cache, table.to(DEV), ints([333, 100]), again, scale=0.125)
    assert torch.isnan(again[1, 0, 3]).all()
    again[1, 0, 3] = out[1, 0, 3]
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Sq,D", [(2, 64), (40, 128), (150, 64), (150, 256), (700, 128)])
def test_scores_at_the_end_of_the_range(dtype, Sq, D):
    """Rows whose largest score is 1e32, rows whose scores are all the same, rows far below zero: the weights are exact, 1 or 1/n."""
    g = gen(Sq + D)
    n = 1100
    q = torch.zeros(1, Sq, 1, D, dtype=dtype, device=DEV)
    q[0, 0::3, 0, 0] = 1e30        # the key with 100 takes all
    q[0, 1::3, 0, 0] = -1e30       # the key with -100 takes all
    k = torch.zeros(1, n, 1, D, dtype=dtype, device=DEV)
    k[0, 1033, 0, 0], k[0, 44, 0, 0] = 100.0, -100.0
    v = heads(g, 1, n, 1, D, dtype)
    out = blank(q.shape, dtype)
    ops.cross_attention(q, k, v, out, scale=1.0)
    assert (out[0, 0::3, 0] == v[0, 1033, 0]).all() and (out[0, 1::3, 0] == v[0, 44, 0]).all()
    even = torch.full((1, n), 1.0 / n, dtype=torch.float64) @ v[0, :, 0].double().cpu()
    size = torch.full((1, n), 1.0 / n, dtype=torch.float64) @ v[0, :, 0].double().cpu().abs()
    close(out[0, 2::3, 0], even.expand(len(range(2, Sq, 3)), D), (half_step(dtype) * even.abs() + size * (2 * n + 64) * U24 * (1 + half_step(dtype))).expand(len(range(2, Sq, 3)), D))
    # every visible score at -3e30: as good as zero
    k[0, :, 0, 1], q[0, 2::3, 0, 1] = -1.0, 3e30
    ops.cross_attention(q, k, v, out, scale=1.0)
    close(out[0, 2::3, 0], even.expand(len(range(2, Sq, 3)), D), (half_step(dtype) * even.abs() + size * (2 * n + 64) * U24 * (1 + half_step(dtype))).expand(len(range(2, Sq, 3)), D))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_is_run_to_run_identical(dtype):
    """Split keys, joined parts, many rows: the same bits every time, whatever else the GPU does."""
    g = gen(31)
    cases = [(heads(g, 2, s, 8, 128, dtype), heads(g, 2, n, 2, 128, dtype), heads(g, 2, n, 2, 128, dtype)) for s, n in ((1, 9000), (15, 4000), (300, 3000))]
    first = [blank(q.shape, dtype) for q, _, _ in cases]
    for (q, k, v), o in zip(cases, first):
        ops.cross_attention(q, k, v, o)
    side = torch.cuda.Stream()
    noise = torch.randn(2048, 2048, device=DEV)
    for _ in range(5):
        with torch.cuda.stream(side):
            noise = noise @ noise * 1e-3
        for (q, k, v), o in zip(cases, first):
            again = blank(q.shape, dtype)
            ops.cross_attention(q, k, v, again)
            assert torch.equal(o, again)


def test_every_code_means_what_its_type_says():
    """Each of the 256 codes, read back and as the one value that a query sees (e4m3: without its two NaN)."""
    for codes in (torch.int8, torch.float8_e4m3fn):
        raw = torch.arange(256, dtype=torch.uint8)
        if codes == torch.int8:
            raw[128] = 1        # -128 is no code
        else:
            raw[[127, 255]] = 1
        cache = ops.Cache8.empty(16, 16, 1, 256, codes, DEV)
        cache.k.view(torch.uint8)[:] = raw.to(DEV)
        cache.v.view(torch.uint8)[:] = raw.to(DEV)[:, None]
        cache.k_scale.fill_(1.0)
        cache.v_scale.fill_(0.5)
        table = torch.arange(16, dtype=torch.int32, device=DEV).view(16, 1)
        want = raw.view(codes).float()
        ko, vo = blank((16, 16, 1, 256), F32), blank((16, 16, 1, 256), F32)
        ops.kv_cache_read(cache, table, ints([16] * 16), ko, vo)
        assert (ko.cpu() == want).all() and (vo.cpu() == want * 0.5).all()
        for dtype in (BF, F32):
            q = torch.zeros(16, 1, 1, 256, dtype=dtype, device=DEV)
            out = blank(q.shape, dtype)
            ops.cache_attention(q, cache, table, ints([1] * 16), out)
            assert (out.float().cpu() == want * 0.5).all()


def fill_cache(g, table, n, page, H, D, codes, lens, dtype=F32):
    """A cache and its numpy twin holding normal values of lens[b] tokens."""
    B, T = table.shape[0], max(max(lens), 1)
    cache, ref = ops.Cache8.empty(n, page, H, D, codes, DEV), RefCache(n, page, H, D, codes)
    k, v = heads(g, B, T, H, D, dtype), heads(g, B, T, H, D, dtype)
    ops.kv_cache_write(k, v, cache, table.to(DEV), ints([0] * B), lens=ints(lens))
    ref.codes = [cache.k.view(torch.uint8).cpu().numpy(), np.ascontiguousarray(cache.v.view(torch.uint8).cpu().numpy().transpose(0, 1, 3, 2))]
    ref.scales = [cache.k_scale.cpu().numpy(), cache.v_scale.cpu().numpy()]
    return cache, ref


def values64(ref, which, row, n):
    """(n, H, D): code * scale in 64 bits."""
    pages, H, page, D = ref.codes[0].shape
    idx = np.asarray(row[:-(-n // page)], dtype=np.int64)
    x = torch.from_numpy(ref.codes[which][idx]).view(ref.dtype).double() * torch.from_numpy(ref.scales[which][idx]).double()[:, :, None, None]
    return x.transpose(1, 2).reshape(-1, H, D)[:n]


CACHE = [(16, 3, 1, 2, 2, 128, 64, "plain"), (16, 2, 1, 8, 2, 64, 33, "slice"), (32, 2, 5, 4, 4, 80, 200, "first"), (64, 3, 1, 32, 8, 128, 777, "plain"), (128, 2, 3, 7, 1, 16, 300, "heads"),
         (64, 1, 17, 6, 2, 96, 1500, "plain"), (16, 1, 1, 1, 1, 256, 5000, "plain"), (32, 1, 70, 2, 1, 128, 257, "first"), (64, 2, 2, 14, 2, 32, 130, "plain"), (128, 1, 64, 8, 1, 256, 400, "plain")]


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("page,B,Sq,Hq,H,D,L,layout", CACHE)
def test_cache_attention(codes, dtype, causal, page, B, Sq, Hq, H, D, L, layout):
    g = gen(page + Sq + D + L)
    table, n = pages_of(g, B, -(-L // page) + 1)
    lens = [L] + [int(x) for x in torch.randint(0, L + 1, (B - 1,), generator=g)]
    cache, ref = fill_cache(g, table, n, page, H, D, codes, lens)
    table[:, -(-max(lens) // page):] = 1 << 30   # entries behind the sequences name no page
    q = heads(g, B, Sq, Hq, D, dtype, layout) * 2
    out = blank(q.shape, dtype, layout if layout != "heads" else "plain")
    ops.cache_attention(q, cache, table.to(DEV), ints(lens), out, causal=causal)
    for b in range(B):
        m = lens[b]
        k, v = values64(ref, 0, table[b], m), values64(ref, 1, table[b], m)
        ends = torch.arange(Sq) - Sq + 1 + m if causal else torch.full((Sq,), m)
        seen = torch.arange(m)[None] < ends[:, None]
        r, tol = attend_ref(q[b].double().cpu(), k, v, seen, D ** -0.5, dtype, pround_of(dtype))
        close(out[b], r, tol)


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_cache_attention_edges(codes):
    """Lengths of 0 and 1, more queries than tokens, entries that name no page in the middle, codes left behind the last token, a block
    that holds a NaN."""
    g = gen(21)
    page, H, D = 16, 1, 64
    table = torch.tensor([[0, 1, 2, 3], [4, 99, 5, 6], [7, 8, -1, -1], [9, 10, 11, 12], [13, 14, 15, 16]], dtype=torch.int32)
    lens = [0, 64, 1, 40, 33]
    cache, ref = fill_cache(g, table, 17, page, H, D, codes, lens)
    # whatever bytes lie behind the last token of a page must not matter (e4m3 has a NaN: 0x7f)
    cache.k.view(torch.uint8)[7, :, 1:] = 0x7F
    cache.v.view(torch.uint8)[7, :, :, 1:] = 0x7F
    cache.k.view(torch.uint8)[15, :, 1:] = 0x7F
    cache.v.view(torch.uint8)[15, :, :, 1:] = 0x7F
    q = heads(g, 5, 3, 2, D, BF)
    out = blank(q.shape, BF)
    ops.cache_attention(q, cache, table.to(DEV), ints(lens), out, causal=True)
    assert not out[0].any() and not out[2, :2].any()
    for b in (1, 2, 3, 4):
        m = lens[b]
        there = torch.tensor([0 <= int(table[b, j // page]) < 17 for j in range(m)])
        row = [max(0, int(i)) % 17 for i in table[b]]
        k, v = values64(ref, 0, row, m), values64(ref, 1, row, m)
        seen = (torch.arange(m)[None] < (torch.arange(3) - 2 + m)[:, None]) & there
        r, tol = attend_ref(q[b].double().cpu(), k, v, seen, D ** -0.5, BF, 2.0 ** -8)
        close(out[b], r, tol)
    # lengths past the table and below zero
    again = blank(q.shape, BF)
    ops.cache_attention(q, cache, table[1:2].expand(5, 4).contiguous().to(DEV), ints([64, 1000, 64, -7, 64]), again)
    assert not again[3].any()
    full = blank(q.shape, BF)
    ops.cache_attention(q, cache, table[1:2].expand(5, 4).contiguous().to(DEV), ints([64] * 5), full)
    assert all(torch.equal(again[b], full[b]) for b in (0, 1, 2, 4))
    # no pages, no table, no batch
    none = ops.Cache8.empty(0, page, H, D, codes, DEV)
    ops.cache_attention(q, none, table.to(DEV), ints(lens), out)
    assert not out.any()
    ops.cache_attention(q, cache, torch.zeros(5, 0, dtype=torch.int32, device=DEV), ints(lens), full)
    assert not full.any()
    ops.cache_attention(q[:0], cache, table[:0].to(DEV), ints([]), out[:0])
    # a NaN written into the values of page 9 shows in sequence 3 alone
    k, v = heads(g, 1, 1, H, D, F32), heads(g, 1, 1, H, D, F32)
    v[0, 0, 0, 3] = float("nan")
    ops.kv_cache_write(k, v, cache, table[3:4].to(DEV), ints([3]))
    ops.cache_attention(q, cache, table.to(DEV), ints(lens), out)
    assert torch.isnan(out[3]).all() and torch.isfinite(out[[0, 1, 2, 4]]).all()


def test_caches_and_tensors_past_32_bits():
    """Pages beyond 2^32 bytes of codes, rows beyond 2^31 elements."""
    g = gen(77)
    page, H, D = 128, 8, 256
    n = (1 << 32) // (page * H * D) + 3
    cache = ops.Cache8.empty(n, page, H, D, torch.int8, DEV)
    table = torch.tensor([[n - 1, 0], [n - 2, 1]], dtype=torch.int32, device=DEV)
    k, v = heads(g, 2, 200, H, D, BF), heads(g, 2, 200, H, D, BF)
    ops.kv_cache_write(k, v, cache, table, ints([0, 0]))
    small = ops.Cache8.empty(4, page, H, D, torch.int8, DEV)
    t2 = torch.tensor([[3, 0], [2, 1]], dtype=torch.int32, device=DEV)
    ops.kv_cache_write(k, v, small, t2, ints([0, 0]))
    assert torch.equal(cache.k[-2:], small.k[2:]) and torch.equal(cache.v[-2:], small.v[2:])
    q = heads(g, 2, 2, 16, D, BF)
    a, b = blank(q.shape, BF), blank(q.shape, BF)
    ops.cache_attention(q, cache, table, ints([200, 200]), a)
    ops.cache_attention(q, small, t2, ints([200, 200]), b)
    assert torch.equal(a, b)
    ka, va, kb, vb = (blank(k.shape, BF) for _ in range(4))
    ops.kv_cache_read(cache, table, ints([200, 200]), ka, va)
    ops.kv_cache_read(small, t2, ints([200, 200]), kb, vb)
    assert torch.equal(ka, kb) and torch.equal(va, vb)
    del cache, ka, va, kb, vb
    big = torch.empty((1 << 31) + 4096 * 64, dtype=BF, device=DEV)
    far = big.as_strided((2, 70, 1, 64), (1 << 31, 64, 64, 1))
    far.copy_(heads(g, 2, 70, 1, 64, BF))
    near = far.contiguous()
    o = [blank((2, 70, 1, 64), BF) for _ in range(2)]
    for x, y in zip((far, near), o):
        ops.cross_attention(x, x, x, y)
    assert torch.equal(*o)
    pos = torch.arange(70, dtype=torch.int32, device=DEV).expand(2, 70)
    for x, y in zip((far, near), o):
        ops.qk_norm_rope(x, None, None, None, pos, ops.rope_freqs(64, device=DEV), y, None)
    assert torch.equal(*o)


# ------------------------------------------------------------------------------------------------------------ together
def one_step(g, cache, table, at, B, Hq, H, D, dtype, freqs, wq, wk, memory):
    """One token per sequence: norm + rotation, write, attention over the cache, then over another encoder's states."""
    qkv = torch.randn(B, 1, Hq + 2 * H, D, generator=g).to(dtype).to(DEV)
    return qkv, lambda q, o, o2, k: (
        ops.qk_norm_rope(qkv[:, :, :Hq], qkv[:, :, Hq:Hq + H], wq, wk, at.view(B, 1), freqs, q, k),
        ops.kv_cache_write(k, qkv[:, :, Hq + H:], cache, table, at),
        ops.cache_attention(q, cache, table, at + 1, o, causal=True),
        ops.cross_attention(o, memory[0], memory[1], o2, lens=memory[2]))


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_run_of_steps_together(codes, dtype):
    """Tokens one at a time through all four operators, each step against 64 bits on what the device's own cache holds."""
    g = gen(9)
    B, Hq, H, D, page, steps = 3, 4, 2, 64, 16, 20
    table, n = pages_of(g, B, 3)
    tab = table.to(DEV)
    cache, ref = ops.Cache8.empty(n, page, H, D, codes, DEV), RefCache(n, page, H, D, codes)
    freqs = ops.rope_freqs(D, device=DEV)
    wq, wk = ((1 + 0.1 * torch.randn(D, generator=g)).to(DEV) for _ in range(2))
    memory = (heads(g, B, 50, H, D, dtype), heads(g, B, 50, H, D, dtype), ints([50, 7, 31]))
    at = ints([0, 5, 15])
    for step in range(steps):
        qkv, go = one_step(g, cache, tab, at, B, Hq, H, D, dtype, freqs, wq, wk, memory)
        q, o, o2, k = blank((B, 1, Hq, D), dtype), blank((B, 1, Hq, D), dtype), blank((B, 1, Hq, D), dtype), blank((B, 1, H, D), dtype)
        go(q, o, o2, k)
        check_rope(q, qkv[:, :, :Hq], wq, at.view(B, 1), freqs, False, 1e-6)
        check_rope(k, qkv[:, :, Hq:Hq + H], wk, at.view(B, 1), freqs, False, 1e-6)
        ref.write((k, qkv[:, :, Hq + H:]), table, at.tolist(), [1] * B)
        same_cache(cache, ref)
        for b in range(B):
            m = int(at[b]) + 1
            r, tol = attend_ref(q[b].double().cpu(), values64(ref, 0, table[b], m), values64(ref, 1, table[b], m), torch.ones(1, m, dtype=torch.bool), D ** -0.5, dtype, pround_of(dtype))
            close(o[b], r, tol)
            m = int(memory[2][b])
            r, tol = attend_ref(o[b].double().cpu(), memory[0][b, :m].double().cpu(), memory[1][b, :m].double().cpu(), torch.ones(1, m, dtype=torch.bool), D ** -0.5, dtype, pround_of(dtype))
            close(o2[b], r, tol)
        at = at + 1


def test_recorded_plan_captured_graphs_and_other_streams_equal_the_eager_calls():
    g = gen(15)
    B, Hq, H, D, page, L = 2, 8, 2, 128, 64, 3000
    table, n = pages_of(g, B, -(-L // page))
    cache, _ = fill_cache(g, table, n, page, H, D, torch.int8, [L, 1234])
    tab, lens = table.to(DEV), ints([L, 1234])
    q = heads(g, B, 1, Hq, D, BF)
    mem = heads(g, B, 2000, H, D, BF), heads(g, B, 2000, H, D, BF)
    pos, freqs = ints([[9], [4]]), ops.rope_freqs(D, device=DEV)
    nk, nv = heads(g, B, 1, H, D, BF), heads(g, B, 1, H, D, BF)
    start = ints([L - 1, 1233])
    ws = [torch.empty(max(1, ops.cache_attention_workspace_bytes(cache, B, 1, Hq, tab.shape[1])), dtype=torch.uint8, device=DEV),
          torch.empty(max(1, ops.cross_attention_workspace_bytes(BF, B, 1, 2000, Hq, H, D)), dtype=torch.uint8, device=DEV)]

    def chain(bufs, own):
        ops.qk_norm_rope(q, None, None, None, pos, freqs, bufs[0], None)
        ops.kv_cache_write(nk, nv, cache, tab, start)
        ops.cache_attention(bufs[0], cache, tab, lens, bufs[1], workspace=ws[0] if own else None)
        ops.cross_attention(bufs[1], *mem, bufs[2], workspace=ws[1] if own else None)
        ops.kv_cache_read(cache, tab, lens, bufs[3], bufs[4])

    def fresh():
        return [blank(q.shape, BF) for _ in range(3)] + [torch.zeros(B, L, H, D, dtype=BF, device=DEV) for _ in range(2)]

    want = fresh()
    chain(want, False)
    # a plan
    bufs = fresh()
    with ops.Recorder() as rec:
        chain(bufs, True)
    plan = ops.Plan(rec.handle, [bufs, ws])
    assert plan.num_ops == 5
    for _ in range(3):
        for x in bufs:
            x.zero_()
        plan.run()
        assert all(torch.equal(x, y) for x, y in zip(bufs, want))
    assert len(plan.run_timed()) == 5
    # two graphs that share the workspaces and one with torch's, replayed one after the other between eager work
    graphs = []
    side = torch.cuda.Stream()
    for own in (True, True, False):
        bufs = fresh()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            chain(bufs, own)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            chain(bufs, own)
        graphs.append((gr, bufs))
    for _ in range(4):
        for gr, bufs in graphs:
            for x in bufs:
                x.zero_()
            eager = fresh()
            chain(eager, False)
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(bufs, want)) and all(torch.equal(x, y) for x, y in zip(eager, want))
    # many rows of 256 dims: more LDS than a kernel may take unasked
    big = heads(g, 1, 100, 2, 256, BF), heads(g, 1, 300, 2, 256, BF)
    eager, caught = blank(big[0].shape, BF), blank(big[0].shape, BF)
    ops.cross_attention(big[0], big[1], big[1], eager)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        ops.cross_attention(big[0], big[1], big[1], caught)
    for _ in range(3):
        caught.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(caught, eager)
    # another stream
    bufs = fresh()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(bufs, False)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(bufs, want))


def test_a_recorded_call_without_its_workspace_is_refused_where_it_needs_one():
    g = gen(2)
    q, k = heads(g, 1, 1, 2, 64, BF), heads(g, 1, 20000, 2, 64, BF)
    if ops.cross_attention_workspace_bytes(BF, 1, 1, 20000, 2, 2, 64) == 0:
        return
    rec = ops.Recorder()
    with pytest.raises(ValueError, match="workspace"):
        with rec:
            ops.cross_attention(q, k, k, blank(q.shape, BF))
    with pytest.raises(ValueError, match="workspace"):
        ops.cross_attention(q, k, k, blank(q.shape, BF), workspace=torch.empty(1, dtype=torch.uint8, device=DEV))


# ------------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    q = torch.zeros(2, 3, 4, 64, dtype=BF, device=DEV)
    k = torch.zeros(2, 5, 2, 64, dtype=BF, device=DEV)
    pos, freqs = torch.zeros(2, 3, dtype=torch.int32, device=DEV), ops.rope_freqs(64, device=DEV)
    cache = ops.Cache8.empty(4, 16, 2, 64, torch.int8, DEV)
    table, two = torch.zeros(2, 2, dtype=torch.int32, device=DEV), ints([1, 1])

    def refused(err, fn, *a, **kw):
        with pytest.raises(err):
            fn(*a, **kw)

    refused(TypeError, ops.cross_attention, q.half(), k.half(), k.half(), q.half())
    refused(ValueError, ops.cross_attention, q, k.float(), k.float(), q)
    refused(ValueError, ops.cross_attention, q, k, k[:, :4], q)
    refused(ValueError, ops.cross_attention, q, k, k, q[:1].expand(2, 3, 4, 64))
    refused(ValueError, ops.qk_norm_rope, q, q, None, None, pos, freqs, q, None)
    refused(ValueError, ops.cross_attention, q[0], k, k, q)
    refused(RuntimeError, ops.cross_attention, q, torch.zeros(2, 5, 3, 64, dtype=BF, device=DEV), torch.zeros(2, 5, 3, 64, dtype=BF, device=DEV), q)   # 4 % 3 heads
    refused(ValueError, ops.cross_attention, q, k, k, q, lens=torch.ones(2, dtype=torch.int64, device=DEV))
    refused(ValueError, ops.cross_attention, q, k, k, q, lens=ints([1]))
    refused(ValueError, ops.cross_attention, q, k, k, q, key_mask=torch.ones(2, 4, dtype=torch.bool, device=DEV))
    refused(ValueError, ops.cross_attention, q, k.cpu(), k.cpu(), q)
    refused(RuntimeError, ops.cross_attention, q.clone().requires_grad_(), k, k, q)
    refused(RuntimeError, ops.cross_attention, q[..., :20].contiguous(), k[..., :20].contiguous(), k[..., :20].contiguous(), q[..., :20].contiguous())
    refused(RuntimeError, ops.cross_attention, *(torch.zeros(2, 3, 2, 264, dtype=BF, device=DEV) for _ in range(4)))
    odd = torch.zeros(2 * 3 * 4 * 64 + 1, dtype=BF, device=DEV)[1:].view(2, 3, 4, 64)
    refused(RuntimeError, ops.cross_attention, odd, k, k, q)   # not on a 16-byte address
    refused(RuntimeError, ops.cross_attention, torch.zeros(2, 3, 4, 68, dtype=BF, device=DEV)[..., :64], k, k, q)   # head stride of 136 bytes
    refused(ValueError, ops.cross_attention, torch.zeros(2, 3, 64, 4, dtype=BF, device=DEV).transpose(2, 3), k, k, q)
    with torch.no_grad():
        ops.cross_attention(q.clone().requires_grad_(), k, k, torch.empty_like(q))

    refused(ValueError, ops.qk_norm_rope, q, None, None, None, pos.long(), freqs, q, None)
    refused(ValueError, ops.qk_norm_rope, q, None, None, None, pos[:, :2], freqs, q, None)
    refused(ValueError, ops.qk_norm_rope, q, None, None, None, pos, freqs.float(), q, None)
    refused(ValueError, ops.qk_norm_rope, q, None, freqs, None, pos, freqs, q, None)
    refused(RuntimeError, ops.qk_norm_rope, q, None, None, None, pos, ops.rope_freqs(66, device=DEV), q, None)   # rotates more than a head holds
    refused(RuntimeError, ops.qk_norm_rope, q, None, None, None, pos, freqs, q, None, eps=-1.0)

    refused(ValueError, ops.Cache8.empty, 4, 24, 2, 64, torch.int8, DEV)
    refused(ValueError, ops.Cache8, cache.k, cache.k, cache.k_scale, cache.v_scale)
    refused(ValueError, ops.Cache8, cache.k, cache.v, cache.k_scale[:3], cache.v_scale)
    refused(ValueError, ops.Cache8, cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)
    refused(ValueError, ops.kv_cache_write, q, q, cache, table, two)   # four heads into a cache of two
    refused(ValueError, ops.kv_cache_write, k, k[:, :2], cache, table, two)
    refused(ValueError, ops.kv_cache_write, k, k, cache, table.long(), two)
    refused(ValueError, ops.kv_cache_write, k, k, cache, table[:1], two)
    refused(ValueError, ops.kv_cache_read, cache, table, ints([1]), k, k)
    refused(RuntimeError, ops.kv_cache_write, *(torch.zeros(1, 1, 2, 24, dtype=BF, device=DEV) for _ in range(2)),
            ops.Cache8.empty(1, 16, 2, 24, torch.int8, DEV), table[:1], ints([0]))   # heads of 24
    refused(ValueError, ops.cache_attention, q[..., :32], cache, table, two, q[..., :32])
    refused(ValueError, ops.cache_attention, q, cache, table, two.long(), q)
    refused(RuntimeError, ops.cache_attention, q[:, :, :3].contiguous(), cache, table, two, q[:, :, :3].contiguous())   # 3 query heads, 2 cache heads


# few rows to 16 and 32, up to 64 rows over long keys, many rows; keys split over workgroups and not
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Sq,Sk,D", [(1, 200, 64), (16, 1500, 128), (20, 333, 128), (32, 2600, 64), (3, 90, 256), (64, 1200, 128), (150, 700, 64), (150, 2100, 128)])
def test_infinite_visible_values(dtype, Sq, Sk, D):
    """A visible value of infinity makes its dim infinite with its sign, infinities of both signs make it NaN, as a sum of weights above zero times
    values says; the other dims are the finite sums they are.  (Weights above zero in 32 bits: |score| stays below 30 here.)"""
    g = gen(Sq + Sk + D)
    q, k, v = heads(g, 2, Sq, 2, D, dtype), heads(g, 2, Sk, 2, D, dtype), heads(g, 2, Sk, 2, D, dtype)
    out = blank(q.shape, dtype)
    fin = v.clone()
    fin[..., [3, 7, 20]] = 0.0
    v[0, 5, :, 3] = float("inf")
    v[0, Sk - 1, :, 3] = float("inf")
    v[:, 9, :, 7] = float("-inf")
    v[1, 70, :, 20] = float("inf")
    v[1, 71, :, 20] = float("-inf")
    ops.cross_attention(q, k, v, out)
    assert (out[0, :, :, 3] == float("inf")).all() and (out[:, :, :, 7] == float("-inf")).all() and torch.isnan(out[1, :, :, 20]).all()
    out[..., [3, 7, 20]] = 0.0
    for b in range(2):
        ref, tol = attend_ref(q[b].double().cpu(), k[b].double().cpu(), fin[b].double().cpu(), torch.ones(Sq, Sk, dtype=torch.bool), D ** -0.5, dtype, pround_of(dtype))
        close(out[b], ref, tol)


def rising(dtype, Sq, n, D, top):
    """Queries and keys whose scores rise evenly from 0 to `top` (base 2, a step of bf16 apart at most) along the keys, with scale 1."""
    q, k = torch.zeros(1, Sq, 1, D, dtype=dtype, device=DEV), torch.zeros(1, n, 1, D, dtype=dtype, device=DEV)
    q[..., 0] = 1.0
    k[0, :, 0, 0] = (torch.arange(n, device=DEV) * (top * 0.6931471805599453 / n)).to(dtype)
    return q, k


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Sq,n,D", [(1, 700, 64), (20, 700, 128), (3, 900, 256), (1, 9000, 128), (64, 1100, 128), (150, 700, 64), (150, 900, 256), (300, 4000, 128)])
def test_values_at_the_end_of_the_range(dtype, Sq, n, D):
    """Values so large that n of them just stay below the largest number: sums of weights up to 1 times them are finite, so the results are."""
    g = gen(Sq + n + D)
    q, k = rising(dtype, Sq, n, D, 7.9)
    v = ((0.5 + 0.5 * torch.rand(1, n, 1, D, generator=g)) * 2.0 ** (127 - np.ceil(np.log2(n)))).to(dtype).to(DEV)
    out = blank(q.shape, dtype)
    ops.cross_attention(q, k, v, out, scale=1.0)
    ref, tol = attend_ref(q[0].double().cpu(), k[0].double().cpu(), v[0].double().cpu(), torch.ones(Sq, n, dtype=torch.bool), 1.0, dtype, pround_of(dtype))
    close(out[0], ref, tol)


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Sq,n,D", [(1, 700, 64), (20, 700, 128), (70, 700, 128), (3, 900, 256), (1, 9000, 128)])
def test_cached_values_at_the_end_of_the_range(codes, dtype, Sq, n, D):
    """As above, the values in a cache, and a block of the largest values there are under a weight that rises late."""
    g = gen(Sq + n + D)
    page = 64
    q, k = rising(F32, Sq, n, D, 7.9)
    v = (0.5 + 0.5 * torch.rand(1, n, 1, D, generator=g)).to(DEV) * 2.0 ** (127 - np.ceil(np.log2(n)))
    table, pages = pages_of(g, 1, -(-n // page))
    cache, ref = ops.Cache8.empty(pages, page, 1, D, codes, DEV), RefCache(pages, page, 1, D, codes)
    ops.kv_cache_write(k, v, cache, table.to(DEV), ints([0]))
    ref.codes = [cache.k.view(torch.uint8).cpu().numpy(), np.ascontiguousarray(cache.v.view(torch.uint8).cpu().numpy().transpose(0, 1, 3, 2))]
    ref.scales = [cache.k_scale.cpu().numpy(), cache.v_scale.cpu().numpy()]
    q, out = q.to(dtype), blank(q.shape, dtype)
    ops.cache_attention(q, cache, table.to(DEV), ints([n]), out, scale=1.0)
    r, tol = attend_ref(q[0].double().cpu(), values64(ref, 0, table[0], n), values64(ref, 1, table[0], n), torch.ones(Sq, n, dtype=torch.bool), 1.0, dtype, pround_of(dtype))
    close(out[0], r, tol)


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_causal_attention_with_lengths_past_the_table(codes):
    """Query i sees lens - (Sq - 1 - i) tokens, or all that the table holds: tokens past it were dropped, the queries behind them still count."""
    g = gen(43)
    table, n = pages_of(g, 4, 4)
    cache, ref = fill_cache(g, table, n, 16, 1, 64, codes, [64] * 4)
    q = heads(g, 4, 5, 2, 64, BF)
    out = blank(q.shape, BF)
    lens = [64, 66, 2 ** 31 - 1, 67]
    ops.cache_attention(q, cache, table.to(DEV), ints(lens), out, causal=True)
    for b in range(4):
        seen = torch.arange(64)[None] < (lens[b] - 4 + torch.arange(5))[:, None]
        r, tol = attend_ref(q[b].double().cpu(), values64(ref, 0, table[b], 64), values64(ref, 1, table[b], 64), seen, 0.125, BF, 2.0 ** -8)
        close(out[b], r, tol)


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,Hq,H,D,page,at,new", [(5, 4, 2, 64, 16, [0, 7, 100, 31, 15], [3, 5, 1, 0, 2]), (1, 2, 2, 128, 64, [0, 63, 64], [1, 0, 1]),
                                                  (40, 8, 2, 128, 32, [500, 0, 31], [17, 40, 33]), (70, 2, 1, 256, 64, [1000, 3], [70, 9]), (33, 3, 3, 80, 128, [2500], [21])])
def test_ragged_steps_write_and_attend(codes, dtype, T, Hq, H, D, page, at, new):
    """A step in which each sequence brings its own count of new tokens: they are written, then each sees the tokens up to itself; rows without a
    token give 0."""
    g = gen(T + D + page)
    B = len(at)
    width = -(-(max(at) + T) // page)
    table, n = pages_of(g, B, width)
    cache, ref = fill_cache(g, table, n, page, H, D, codes, at)
    q, k, v = heads(g, B, T, Hq, D, dtype) * 2, heads(g, B, T, H, D, dtype), heads(g, B, T, H, D, dtype)
    start, count = ints(at), ints(new)
    ops.kv_cache_write(k, v, cache, table.to(DEV), start, lens=count)
    ref.write((k, v), table, at, new)
    same_cache(cache, ref)
    out = blank(q.shape, dtype)
    ops.cache_attention(q, cache, table.to(DEV), start + count, out, causal=True, start=start)
    for b in range(B):
        m = at[b] + new[b]
        assert not out[b, new[b]:].any()
        if new[b]:
            seen = torch.arange(m)[None] <= (at[b] + torch.arange(new[b]))[:, None]
            r, tol = attend_ref(q[b, :new[b]].double().cpu(), values64(ref, 0, table[b], m), values64(ref, 1, table[b], m), seen, D ** -0.5, dtype, pround_of(dtype))
            close(out[b, :new[b]], r, tol)
    # where every sequence brings T tokens, it is the call without start
    full, same = blank(q.shape, dtype), blank(q.shape, dtype)
    ops.cache_attention(q, cache, table.to(DEV), start + T, full, causal=True, start=start)
    ops.cache_attention(q, cache, table.to(DEV), start + T, same, causal=True)
    assert torch.equal(full, same)


def test_ragged_steps_edges():
    """Starts below zero count as 0, as a write takes them; starts at, behind and far behind the length give zeros; no start without causal."""
    g = gen(41)
    table, n = pages_of(g, 5, 4)
    cache, ref = fill_cache(g, table, n, 16, 1, 64, torch.int8, [64] * 5)
    q = heads(g, 5, 3, 2, 64, BF)
    out = blank(q.shape, BF)
    lens = [2, 10, 10, 10, 64]
    ops.cache_attention(q, cache, table.to(DEV), ints(lens), out, causal=True, start=ints([-9, 10, 2 ** 31 - 1, -2 ** 31, 62]))
    assert not out[1].any() and not out[2].any() and not out[0, 2].any() and not out[4, 2].any()
    for b, first, live in ((0, 0, 2), (3, 0, 3), (4, 62, 2)):
        seen = torch.arange(lens[b])[None] <= (first + torch.arange(live))[:, None]
        r, tol = attend_ref(q[b, :live].double().cpu(), values64(ref, 0, table[b], lens[b]), values64(ref, 1, table[b], lens[b]), seen, 0.125, BF, 2.0 ** -8)
        close(out[b, :live], r, tol)
    for bad in (dict(start=ints([0] * 5)), dict(causal=True, start=ints([0] * 4)), dict(causal=True, start=torch.zeros(5, dtype=torch.int64, device=DEV)),
                dict(causal=True, start=torch.zeros(5, dtype=torch.int32))):
        with pytest.raises(ValueError, match="cache_attention"):
            ops.cache_attention(q, cache, table.to(DEV), ints(lens), out, **bad)


def test_autograd_sees_what_is_written_and_tangents_are_refused():
    """A tensor that autograd saved and an operator then wrote over fails in its backward pass instead of giving a gradient of other values; a
    tensor with a forward-mode tangent is refused, as one that asks for a gradient is."""
    import torch.autograd.forward_ad as fwd
    g = gen(51)
    q, k = heads(g, 1, 3, 2, 64, F32), heads(g, 1, 3, 2, 64, F32)
    pos, freqs = ints([[0, 1, 2]]), ops.rope_freqs(64, device=DEV)
    cache = ops.Cache8.empty(1, 16, 2, 64, torch.int8, DEV)
    table, lens = ints([[0]]), ints([3])
    writes = {"qk_norm_rope": (lambda: ops.qk_norm_rope(q, k, None, None, pos, freqs, q, k), (q, k)),
              "kv_cache_write": (lambda: ops.kv_cache_write(q, k, cache, table, ints([0])), (cache.k, cache.v, cache.k_scale, cache.v_scale)),
              "kv_cache_read": (lambda: ops.kv_cache_read(cache, table, lens, q, k), (q, k)),
              "cache_attention": (lambda: ops.cache_attention(q, cache, table, lens, q), (q,)),
              "cross_attention": (lambda: ops.cross_attention(q, k, k, q), (q,))}
    for name, (call, outs) in writes.items():
        for x in outs:
            saved = x.detach().float() if x.dtype == torch.int8 else x
            before = x._version
            w = torch.ones((), device=DEV, requires_grad=True)
            y = (w * saved).sum()
            call()
            assert x._version > before, name
            if saved is x:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    y.backward()
    with torch.inference_mode():   # tensors without a version counter
        z = torch.empty_like(q)
        ops.cross_attention(q, k, k, z)
    with fwd.dual_level():
        ops.cross_attention(q, k, k, torch.empty_like(q))   # (no tangent: as ever)
        dual = fwd.make_dual(q, torch.ones_like(q))
        for call in (lambda: ops.cross_attention(dual, k, k, torch.empty_like(q)), lambda: ops.qk_norm_rope(k, dual, None, None, pos, freqs, k, k),
                     lambda: ops.kv_cache_write(k, dual, cache, table, ints([0])), lambda: ops.cache_attention(dual, cache, table, lens, k)):
            with pytest.raises(RuntimeError, match="inference only"):
                call()


# ------------------------------------------------------------------------------------------------------------ precision
def plain32(q, k, v, seen, scale):
    """The elementary form in 32 bits on the GPU, rounded once to the inputs' type: q (B, Sq, Hq, D), k, v (B, n, Hk, D) float32, seen (Sq, n)."""
    B, Sq, Hq, D = q.shape
    G = Hq // k.shape[2]
    qf = q.float().transpose(1, 2).contiguous()
    kf, vf = (x.transpose(1, 2).repeat_interleave(G, 1).contiguous() for x in (k, v))
    z = torch.matmul(qf * scale, kf.transpose(2, 3).contiguous()).masked_fill(~seen.to(DEV), -torch.inf)
    p = torch.exp(z - z.amax(-1, keepdim=True))
    return (torch.matmul(p, vf) / p.sum(-1, keepdim=True)).transpose(1, 2).to(q.dtype)


def exact64(q, k, v, seen, scale, weights=None):
    """In 64 bits on the CPU: (result, root mean square of the visible scores); `weights` rounds the weights e^(score - maximum) first."""
    G = q.shape[2] // k.shape[2]
    qd = q.double().cpu().transpose(1, 2)
    kd, vd = (x.double().cpu().transpose(1, 2).repeat_interleave(G, 1) for x in (k, v))
    z = (qd @ kd.transpose(2, 3).contiguous() * scale).masked_fill(~seen, -np.inf)
    p = torch.exp(z - z.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    sigma = float(z[torch.isfinite(z)].square().mean().sqrt())
    return ((weights(p) if weights else p) @ vd / total).transpose(1, 2), sigma


def bf16_terms(p, terms):
    """The sum of the first `terms` bf16 terms of p, in 64 bits."""
    got = torch.zeros_like(p)
    for _ in range(terms):
        got = got + (p - got).to(torch.bfloat16).double()
    return got


def rms(x):
    return float(x.double().square().mean().sqrt())


def hold_precision(got, q, k, v, seen, scale, two_terms):
    """bfloat16: the plain form's error is the rounding of its result, half a step spread evenly.  Two bf16 terms of a weight (2^-14) add nothing
    that shows: 1.2 leaves room for the draw (some thousand results: 2 %).  One term rounds each weight as the result is rounded, and the values are as often
    below zero as above, so the errors of n weights add up to as much as the result's own: sqrt(2) = 1.41, 1.6 with room.
    float32, in units of U = 2^-24, each rounding at most U/sqrt(3) rms of what it rounds, partial sums growing as the root of their length: a score (rms
    sigma) D/6 sigma^2 U^2, the values' sum n/6 U^2, a dozen single roundings 8 U^2; twice the root of their sum.  A weight of two bf16 terms
    (2^-17 of its binade at most, 2^-19 rms = 32 U) is past it, and that is checked on the oracle."""
    exact, sigma = exact64(q, k, v, seen, scale)
    err = rms(got.double().cpu() - exact)
    if q.dtype == BF:
        ratio = err / rms(plain32(q, k, v, seen, scale).double().cpu() - exact)
        assert ratio <= (1.2 if two_terms else 1.6), ratio
        return
    n, D = k.shape[1], q.shape[3]
    bound = 2 * U24 * (sigma ** 2 * D / 6 + n / 6 + 8) ** 0.5 * rms(exact)
    short, _ = exact64(q, k, v, seen, scale, lambda p: bf16_terms(p, 2))
    assert rms(short - exact) > bound
    assert err <= bound, err / bound


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,Sq,n,Hq,Hk,D,two_terms", [(8, 1, 150, 16, 4, 64, True), (2, 16, 200, 4, 4, 64, True), (4, 8, 220, 8, 2, 32, True), (1, 1, 9000, 64, 2, 64, True), (4, 64, 1100, 2, 2, 64, False),
                                                      (1, 100, 220, 2, 2, 64, False), (2, 300, 128, 2, 1, 32, False), (1, 200, 180, 2, 2, 128, False)])
def test_errors_of_cross_attention_are_those_of_the_plain_form(dtype, B, Sq, n, Hq, Hk, D, two_terms):
    if dtype == F32 and n > 300:
        n = 300   # the sums' own roundings would cover a lost term
    g = gen(Sq + n + D)
    q, k, v = heads(g, B, Sq, Hq, D, dtype), heads(g, B, n, Hk, D, dtype), heads(g, B, n, Hk, D, dtype)
    out = blank(q.shape, dtype)
    ops.cross_attention(q, k, v, out)
    hold_precision(out, q, k.float(), v.float(), torch.ones(Sq, n, dtype=torch.bool), D ** -0.5, two_terms)


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Sq,n,Hq,H,D,two_terms", [(1, 200, 64, 4, 64, True), (8, 250, 16, 4, 64, True), (16, 130, 8, 4, 32, True), (5, 9000, 32, 8, 64, True), (64, 250, 4, 4, 64, False), (48, 200, 4, 4, 256, True)])
def test_errors_of_cache_attention_are_those_of_the_plain_form(codes, dtype, Sq, n, Hq, H, D, two_terms):
    """On the values that the cache holds."""
    if dtype == F32 and n > 300:
        n = 300
    g = gen(Sq + n + D)
    table, pages = pages_of(g, 1, -(-n // 32))
    cache, ref = fill_cache(g, table, pages, 32, H, D, codes, [n])
    q = heads(g, 1, Sq, Hq, D, dtype)
    out = blank(q.shape, dtype)
    ops.cache_attention(q, cache, table.to(DEV), ints([n]), out, causal=True)
    k, v = (values64(ref, w, table[0], n).float().to(DEV)[None] for w in (0, 1))
    seen = torch.arange(n)[None] < (n - Sq + 1 + torch.arange(Sq))[:, None]
    hold_precision(out, q, k, v, seen, D ** -0.5, two_terms)


def test_float32_queries_over_a_cache_keep_all_their_bits():
    """Two keys of opposite sign and queries of two dims that nearly cancel: a score is 127 (x - y), below 2 but summed from products of up to 254.  Their
    sum is rounded a few times (8 half steps of 256 with those of the scale, for either key), so a weight moves by a quarter of 2 * 8 * 256 U = 2^-14.  A query of two
    bf16 terms (2^-17 in [1, 2)) would move it by 2^-12 to 2^-11: checked on the oracle."""
    g = gen(61)
    cache = ops.Cache8.empty(1, 16, 1, 16, torch.int8, DEV)
    table = ints([[0]])
    k, v = torch.zeros(1, 2, 1, 16, device=DEV), torch.zeros(1, 2, 1, 16, device=DEV)
    k[0, :, 0, 0], k[0, :, 0, 1] = torch.tensor([127.0, -127.0], device=DEV), torch.tensor([-127.0, 127.0], device=DEV)
    v[0, 0, 0] = 1.0
    ops.kv_cache_write(k, v, cache, table, ints([0]))
    assert cache.k_scale.item() == 1.0
    q = torch.zeros(1, 400, 1, 16)
    q[0, :, 0, 0] = 1.0 + 0.99 * torch.rand(400, generator=g)
    q[0, :, 0, 1] = q[0, :, 0, 0] + (torch.rand(400, generator=g) - 0.5) * 0.01
    out = torch.empty(1, 400, 1, 16, device=DEV)
    ops.cache_attention(q.to(DEV), cache, table, ints([2]), out, scale=1.0)

    def weight(x):
        return torch.sigmoid(2 * 127.0 * (x[0, :, 0, 0] - x[0, :, 0, 1]))

    value = v[0, 0, 0, 0].double().cpu() * cache.v_scale.item() * 127.0
    tol = 2.0 ** -14
    assert (weight(bf16_terms(q.double(), 2)) - weight(q.double())).abs().max() > 4 * tol
    assert ((out[0, :, 0, 0].double().cpu() - weight(q.double()) * value).abs() <= tol).all()


def test_a_call_that_splits_its_keys_needs_its_workspace():
    g = gen(2)
    q, k = heads(g, 1, 1, 2, 64, BF), heads(g, 1, 20000, 2, 64, BF)
    assert ops.cross_attention_workspace_bytes(BF, 1, 1, 20000, 2, 2, 64) > 0
    rec = ops.Recorder()
    with pytest.raises(ValueError, match="workspace"):
        with rec:
            ops.cross_attention(q, k, k, blank(q.shape, BF))
    with pytest.raises(ValueError, match="workspace"):
        ops.cross_attention(q, k, k, blank(q.shape, BF), workspace=torch.empty(1, dtype=torch.uint8, device=DEV))


def test_sizes_past_32_bits_and_tables_without_axes_are_refused():
    """Broadcast inputs reach sizes that the C entry points cannot take: 2^32 keys must not become none."""
    q = torch.ones(1, 2, 1, 64, dtype=BF, device=DEV)
    far = q[:, :1].expand(1, 1 << 32, 1, 64)
    cache = ops.Cache8.empty(2, 16, 1, 64, torch.int8, DEV)
    table, one = ints([[0, 1]]), ints([1])

    def refused(fn, *a, **kw):
        with pytest.raises(ValueError, match="2.31|table"):
            fn(*a, **kw)

    refused(ops.cross_attention, q, far, far, torch.empty_like(q))
    refused(ops.cross_attention, far, q, q, far)
    refused(ops.kv_cache_write, far, far, cache, table, one)
    refused(ops.qk_norm_rope, far, None, None, None, one.view(1, 1).expand(1, 1 << 32), ops.rope_freqs(64, device=DEV), far, None)
    refused(ops.kv_cache_read, cache, one[0], one, q, q)
    refused(ops.kv_cache_write, q, q, cache, one, one)
    refused(ops.cache_attention, q, cache, table.view(1, 1, 2), one, torch.empty_like(q))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_ragged_steps_recorded_captured_in_place_and_on_another_stream(dtype):
    """cache_attention with start in a plan, in a graph that is replayed while the starts change, over its own queries and on a side stream."""
    g = gen(71)
    B, T, Hq, H, D, page, L = 3, 6, 8, 2, 64, 32, 2500
    table, n = pages_of(g, B, -(-L // page))
    cache, _ = fill_cache(g, table, n, page, H, D, torch.int8, [L, 900, 40])
    tab, q = table.to(DEV), heads(g, B, T, Hq, D, dtype)
    steps = [([L - 6, 890, 37], [L, 893, 38]), ([L - 3, 0, 0], [L, 1, 6]), ([0, 500, 39], [0, 506, 40])]
    start, lens = ints(steps[0][0]), ints(steps[0][1])

    def eager(s, e):
        out = blank(q.shape, dtype)
        ops.cache_attention(q, cache, tab, ints(e), out, causal=True, start=ints(s))
        return out

    ws = torch.empty(ops.cache_attention_workspace_bytes(cache, B, T, Hq, tab.shape[1]), dtype=torch.uint8, device=DEV)
    assert ws.numel() > 0
    recorded, captured = blank(q.shape, dtype), blank(q.shape, dtype)
    with ops.Recorder() as rec:
        ops.cache_attention(q, cache, tab, lens, recorded, causal=True, workspace=ws, start=start)
    plan = ops.Plan(rec.handle, [recorded, ws])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.cache_attention(q, cache, tab, lens, captured, causal=True, start=start)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(captured, eager(*steps[0]))
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        ops.cache_attention(q, cache, tab, lens, captured, causal=True, start=start)
    for s, e in steps + steps:
        start.copy_(ints(s))
        lens.copy_(ints(e))
        want = eager(s, e)
        recorded.fill_(7.0)
        captured.fill_(7.0)
        plan.run()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(recorded, want) and torch.equal(captured, want)
        own = q.clone()
        ops.cache_attention(own, cache, tab, lens, own, causal=True, start=start)
        assert torch.equal(own, want)
