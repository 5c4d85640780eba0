"""The paged 8-bit cache against its definition in float64: cache_append bit for bit
(scales, rescaled codes, roundings, what it leaves alone), cache_attention row by row
over the keys that the row sees -- every head width, tiles of rows, page size and
division of the keys among workgroups; tables with entries that are no page; caches
and inputs of any strides; what lies behind a length or in a later token; streams and
graph capture; both together; and what they refuse.

Tolerances of the attention.  The cache's elements enter exactly.  With e = 2^-24 a
score is off by at most e (D A + 2 |s| + 16), A the sum of |q k| scaled (one product
sum, its scaling, the exponential), and sums over n keys by n e relative to the sum of
magnitudes; d stands for both.  Probabilities are rounded to 8 bits for bfloat16 (u =
2^-8), 8 + 8 for float16 (2^-16), 8 + 8 + 8 for float32 (2^-24).  So an output is off by
at most (u + 4 d) times the mean of |v|, and half a step of its type; the LSE by 4 d +
4 e (1 + |lse|).  float16's largest value is 65504: what lies past 65520, halfway to the
next step of 32, is an infinity.
"""

import math

import pytest
import torch

from _helpers import DEV, randn

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
E = 2.0 ** -24
PARTS = {BF16: 2.0 ** -8, F16: 2.0 ** -16, F32: 2.0 ** -24}


# ---- a cache on the host -----------------------------------------------------

def _e4m3(x):
    """The nearest of k 2^(e - 3), e the exponent of x but at least -6; of two the even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _values(cache, which):
    """(codes, scales) as float64."""
    return cache[which].view(torch.uint8).cpu().view(E4M3).double(), \
        cache[2 + which].view(torch.uint8).cpu().view(E8M0).float().double()


def _append(state, x, tables, lens, new=None):
    """x [B, L, H, D] into state = (codes, scales), float64, in place."""
    codes, scales = state
    pages, _, size = codes.shape[:3]
    n = x.shape[1]
    for b in range(x.shape[0]):
        length = min(max(int(lens[b]), 0), tables.shape[1] * size)
        count = n if new is None else min(max(int(new[b]), 0), n)
        at = max(length - count, 0)
        while at < length:
            slot, page = at % size, int(tables[b, at // size])
            m = min(size - slot, length - at)
            row = x[b, n - length + at:n - length + at + m].double().transpose(0, 1)
            at += m
            if not 0 <= page < pages:
                continue
            top = torch.where(row.isfinite(), row.abs(), torch.zeros_like(row)).amax((1, 2))
            e = torch.ceil(torch.log2(top / 448)).clamp(-117, 119)
            sc = torch.exp2(e)
            if slot:
                sc = torch.maximum(sc, scales[page])
                codes[page, :, :slot] = _e4m3(codes[page, :, :slot] * (scales[page] / sc)[:, None, None])
            new_codes = _e4m3((row / sc[:, None, None]).clamp(-448, 448))
            codes[page, :, slot:slot + m] = torch.where(row.isfinite(), new_codes, torch.full_like(row, math.nan))
            scales[page] = sc


def _same(got, want, what=""):
    assert got.shape == want.shape, what
    bad = ~((got == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {got.numel()} differ, first at {bad.nonzero()[0].tolist()}"


def _fill(pages, heads, size, dim, seed):
    """A cache full of old tokens."""
    import natten_amd

    cache = natten_amd.paged_cache(pages, heads, dim, size, device="cpu")
    for i in (0, 1):
        x = randn((pages, heads, size, dim), F32, seed + i) * 100
        cache[i].view(torch.uint8).copy_(x.clamp(-448, 448).to(E4M3).view(torch.uint8))
        g = torch.Generator().manual_seed(seed + 2 + i)
        cache[2 + i].view(torch.uint8).copy_(torch.randint(116, 122, (pages, heads), generator=g))
    return cache


def _to(cache):
    import natten_amd

    return natten_amd.PagedCache(*(t.view(torch.uint8).to(DEV).view(t.dtype) for t in cache))


def _tables(b, per, pages, seed):
    g = torch.Generator().manual_seed(seed)
    assert b * per <= pages
    return torch.randperm(pages, generator=g)[:b * per].view(b, per).to(torch.int32)


# ---- cache_append ------------------------------------------------------------

# B, L, heads, dim, page, lengths with the new tokens, new tokens or None
APPENDS = {
    "one token": (5, 1, 2, 64, 16, [1, 16, 17, 33, 40], None),
    "one token of many heads": (3, 1, 9, 128, 64, [64, 65, 1], None),
    "a narrow head": (2, 3, 1, 16, 16, [3, 20], None),
    "some tokens": (3, 7, 2, 80, 32, [7, 50, 96], None),
    "across pages": (3, 45, 2, 48, 16, [45, 60, 79], None),
    "many pages": (2, 300, 3, 128, 64, [300, 411], None),
    "wide heads": (2, 140, 2, 256, 128, [140, 200], None),
    "wide heads, one token": (2, 1, 3, 256, 128, [128, 77], None),
    "before the start": (3, 20, 2, 32, 16, [5, 0, 20], None),
    "padded": (5, 20, 2, 64, 16, [50, 33, 16, 20, 7], [3, 20, 0, 1, 20]),
    "padded past the start": (2, 9, 2, 32, 16, [4, 30], [9, 2]),
    "clamped lengths": (3, 10, 2, 32, 16, [1000, -7, 90], [100, 5, -3]),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", list(APPENDS))
def test_append_bit_for_bit(case, dtype):
    import natten_amd

    B, L, H, D, size, lens, new = APPENDS[case]
    per = -(-max(min(max(lens), 96), L, *(n for n in lens if n < 500)) // size)
    pages = B * per + 3
    cache = _fill(pages, H, size, D, 7)
    tables = _tables(B, per, pages, 1)
    # per token other magnitudes: some pages' scales grow, others hold
    g = torch.Generator().manual_seed(5)
    mag = torch.exp2(torch.randint(-12, 4, (B, L, H, 1), generator=g).float())
    key, value = ((randn((B, L, H, D), F32, s) * mag).to(dtype) for s in (1, 2))
    want = [_values(cache, i) for i in (0, 1)]
    for st, x in zip(want, (key, value)):
        _append(st, x, tables, lens, new)
    dev = _to(cache)
    out = natten_amd.cache_append(dev, key.to(DEV), value.to(DEV), tables.to(DEV),
                                  torch.tensor(lens, dtype=torch.int32, device=DEV),
                                  None if new is None else torch.tensor(new, dtype=torch.int32, device=DEV))
    assert out is None
    for i in (0, 1):
        codes, scales = _values(dev, i)
        _same(scales, want[i][1], f"{case} scales {i}")
        _same(codes, want[i][0], f"{case} codes {i}")


@pytest.mark.gpu
@pytest.mark.parametrize("size", [16, 64])
def test_token_by_token_as_scales_grow(size):
    """Appended one at a time, with magnitudes that rise and fall over 2^20."""
    import natten_amd

    B, H, D, T = 2, 3, 32, 2 * size + 3
    cache = _fill(2 * 3, H, size, D, 3)
    tables = _tables(B, 3, 6, 2)
    want = [_values(cache, i) for i in (0, 1)]
    dev = _to(cache)
    g = torch.Generator().manual_seed(9)
    for t in range(T):
        mag = torch.exp2(torch.randint(-10, 11, (B, 1, H, 1), generator=g).float())
        key, value = (randn((B, 1, H, D), F32, 10 * t + s) * mag for s in (1, 2))
        lens = [t + 1, max(t - 4, 0)]
        for st, x in zip(want, (key, value)):
            _append(st, x, tables, lens)
        natten_amd.cache_append(dev, key.to(DEV), value.to(DEV), tables.to(DEV),
                                torch.tensor(lens, device=DEV))
    for i in (0, 1):
        codes, scales = _values(dev, i)
        _same(scales, want[i][1], "scales")
        _same(codes, want[i][0], "codes")


@pytest.mark.gpu
def test_every_rounding_of_an_element():
    """The values of e4m3, what lies halfway between two of them and next to that, at
    scale 1 (448 is among them) and, in front of a page's larger tokens, rescaled."""
    import natten_amd

    v = torch.arange(0, 127, dtype=torch.uint8).view(E4M3).float()
    mid = (v[1:] + v[:-1]) / 2
    x = torch.cat([v, mid, mid * (1 + 2.0 ** -23), mid * (1 - 2.0 ** -23)])
    x = torch.cat([x, -x])
    x = torch.cat([x, torch.zeros(-x.numel() % 64)]).view(1, -1, 1, 64)
    x[..., 0] = 448.0
    n = x.shape[1]
    assert n <= 64
    cache = natten_amd.paged_cache(1, 1, 64, 128, DEV)
    tables = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    want = [_values(cache, i) for i in (0, 1)]
    for grow in (0, 1, 5, 12, 30):
        y = torch.full((1, 1, 1, 64), 448.0 * 2.0 ** grow)
        for xx, length in ((x, n), (y, n + 1)):
            for st in want:
                _append(st, xx, tables.cpu(), [length])
            natten_amd.cache_append(cache, xx.to(DEV), xx.to(DEV), tables, torch.tensor([length], device=DEV))
            for i in (0, 1):
                codes, scales = _values(cache, i)
                _same(scales, want[i][1], f"scales {grow}")
                _same(codes, want[i][0], f"codes {grow}")


@pytest.mark.gpu
def test_scales_of_extreme_values():
    import natten_amd

    big = torch.finfo(F32).max
    rows = torch.zeros(12, 16)
    rows[1, 0], rows[2, 0], rows[3, 0] = 2.0 ** -149, 2.0 ** -126, 2.0 ** -100
    rows[4, :2], rows[5, 0] = torch.tensor([big, 2.0 ** 127]), 1.75 * 2.0 ** 127
    rows[6, 0], rows[7, 0] = 448.0, 448.0 * (1 + 2.0 ** -22)
    rows[8, :3] = torch.tensor([math.inf, 3.0, -3.0])
    rows[9, :3] = torch.tensor([math.nan, 5.0, -math.inf])
    rows[10] = math.nan
    rows[11, 0] = -0.0
    x = rows.view(12, 1, 1, 16)
    cache = natten_amd.paged_cache(12, 1, 16, 16, DEV)
    tables = torch.arange(12, dtype=torch.int32, device=DEV).view(12, 1)
    want = [_values(cache, i) for i in (0, 1)]
    for st in want:
        _append(st, x, tables.cpu(), [1] * 12)
    natten_amd.cache_append(cache, x.to(DEV), x.to(DEV), tables, torch.ones(12, dtype=torch.int32, device=DEV))
    for i in (0, 1):
        codes, scales = _values(cache, i)
        _same(scales, want[i][1], "scales")
        _same(codes, want[i][0], "codes")
        value = codes[:, 0, 0] * scales
        assert value[4, 0] == 1.75 * 2.0 ** 127 and value[8, 1] == 3.0 and value[8, 0].isnan()
        assert value[10].isnan().all() and scales[10] == 2.0 ** -117 and scales[8] == 2.0 ** -7
        assert scales[6] == 1.0 and scales[7] == 2.0


def test_the_host_twin_of_the_rounding():
    """The oracle's own rounding against torch's conversion."""
    x = torch.cat([randn((4000,), F32, 1) * 2.0 ** k for k in range(-12, 7)])
    x = torch.cat([x, torch.arange(0, 127, dtype=torch.uint8).view(E4M3).float(),
                   torch.tensor([2.0 ** -10, 3 * 2.0 ** -10, 5 * 2.0 ** -10, 17.0, 19.0, 448.0])])
    x = x[x.abs() <= 448]
    assert torch.equal(_e4m3(x.double()), x.to(E4M3).double())


@pytest.mark.gpu
def test_entries_that_are_no_page():
    import natten_amd

    B, L, H, D, size = 2, 40, 2, 32, 16
    cache = _fill(6, H, size, D, 3)
    tables = torch.tensor([[2, -1, 4], [6, 1, 1 << 30]], dtype=torch.int32)
    key, value = (randn((B, L, H, D), F32, s) for s in (1, 2))
    want = [_values(cache, i) for i in (0, 1)]
    for st, x in zip(want, (key, value)):
        _append(st, x, tables, [48, 45])
    dev = _to(cache)
    lens = torch.tensor([48, 45], device=DEV)
    wide = tables.long()
    wide[0, 1], wide[1, 2] = -(1 << 40), 1 << 40
    for form in (tables, wide):
        natten_amd.cache_append(dev, key.to(DEV), value.to(DEV), form.to(DEV), lens)
        for i in (0, 1):
            codes, scales = _values(dev, i)
            _same(scales, want[i][1], "scales")
            _same(codes, want[i][0], "codes")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_views(dtype):
    import natten_amd

    B, L, H, D, size = 3, 21, 2, 32, 16
    packed = randn((B, L, 3 * H, D), dtype, 1).to(DEV)
    odd = randn((B, L + 4, H, D + 3), dtype, 2).to(DEV)[:, 3:3 + L, :, 1:1 + D]
    heads_first = randn((B, H, L, D), dtype, 3).to(DEV).transpose(1, 2)
    spread = randn((B, L, H, D), dtype, 4).to(DEV).transpose(0, -1).contiguous().transpose(0, -1)
    one = randn((1, 1, H, D), dtype, 5).to(DEV).expand(B, L, H, D)
    views = [packed[:, :, H:2 * H], odd, heads_first, spread, one]
    tables = torch.stack([_tables(B, 3, 9, 4).to(DEV)] * 2, -1)[..., 0]
    lens = torch.tensor([30, 21, 48], dtype=torch.int32, device=DEV)
    base = _fill(9, H, size, D, 5)
    for i, key in enumerate(views):
        value = views[i - 1]
        a, b = _to(base), _to(base)
        natten_amd.cache_append(a, key.contiguous(), value.contiguous(), tables.contiguous(), lens)
        # the cache as every second page and head of a larger one, token by token
        big = torch.zeros(18, size, 2 * H, D, dtype=torch.uint8, device=DEV)
        view = big.permute(0, 2, 1, 3)[::2, ::2]
        view.copy_(b[0].view(torch.uint8))
        scales = torch.zeros(H, 9, dtype=torch.uint8, device=DEV).t()
        scales.copy_(b[2].view(torch.uint8))
        c = natten_amd.PagedCache(view.view(E4M3), b[1], scales.view(E8M0), b[3])
        natten_amd.cache_append(c, key, value, tables, lens)
        for x, y in zip(a, c):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        assert not big[1::2].any() and not big.permute(0, 2, 1, 3)[:, 1::2].any()
    # lengths on the host, of either type
    for form in (lens.cpu(), lens.long(), lens.cpu().long()):
        d = _to(base)
        natten_amd.cache_append(d, key, value, tables, form, torch.tensor([21, 21, 21]))
        for x, y in zip(a, d):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


# ---- cache_attention ---------------------------------------------------------

def _make(case, dtype, seed=0, std=1.5):
    B, L, H, Hk, D, size, lens, window = case
    lens = [lens[b % len(lens)] for b in range(B)]
    per = max(1, -(-max(lens) // size))
    pages = B * per + 2
    cache = _fill(pages, Hk, size, D, seed + 20)
    return dict(q=randn((B, L, H, D), dtype, seed, std), cache=cache, tables=_tables(B, per, pages, seed + 1),
                lens=torch.tensor(lens, dtype=torch.int32), window=window)


def _held(t):
    """Values of all pages, [pages, heads, size, D] each, float64."""
    out = []
    for i in (0, 1):
        codes, scales = _values(t["cache"], i)
        out.append(codes * scales[..., None, None])
    return out


def _reference(t, scale=None, tokens=None):
    """(out, tolerance), (lse, tolerance), each row over its own keys."""
    q = t["q"].double()
    B, L, H, D = q.shape
    keys, vals = _held(t)
    pages, Hk, size = keys.shape[:3]
    scale = D ** -0.5 if scale is None else scale
    fi, u = torch.finfo(t["q"].dtype), PARTS[t["q"].dtype]
    out, lse = torch.zeros_like(q), torch.full(q.shape[:-1], -math.inf, dtype=torch.float64)
    to, tl = torch.zeros_like(q), torch.zeros_like(lse)
    cap = t["tables"].shape[1] * size
    for b in range(B):
        n = min(max(int(t["lens"][b]), 0), cap)
        for j in range(L) if tokens is None else tokens:
            at = n - L + j
            lo = 0 if t["window"] is None else max(0, at - t["window"] + 1)
            if at < 0:
                continue
            pos = torch.arange(lo, at + 1)
            page = t["tables"][b].long()[pos // size]
            ok = (page >= 0) & (page < pages)
            pos, page = pos[ok], page[ok]
            if pos.numel() == 0:
                continue
            kk, vv = (x[page, :, pos % size].repeat_interleave(H // Hk, 1).transpose(0, 1)
                      for x in (keys, vals))  # [H, n, D]
            qq = q[b, j].unsqueeze(1)
            s = (qq * kk).sum(-1) * scale
            a = (qq.abs() * kk.abs()).sum(-1).amax(-1) * scale
            l = torch.logsumexp(s, -1)
            p = torch.exp(s - l.unsqueeze(-1))
            out[b, j] = (p.unsqueeze(-1) * vv).sum(1)
            lse[b, j] = l
            d = E * (D * a + 2 * s.abs().amax(-1) + 16 + kk.shape[1])
            mean = (p.unsqueeze(-1) * vv.abs()).sum(1)
            to[b, j] = (u + 4 * d.unsqueeze(-1)) * mean + out[b, j].abs() * fi.eps / 2 + fi.tiny
            tl[b, j] = 4 * d + 4 * E * (1 + l.abs())
    return (out, to), (lse, tl)


def _near(got, want, what):
    v, tol = want
    o = got.detach().cpu().double()
    assert o.shape == v.shape, what
    if got.dtype == F16:  # (and either where it is within the tolerance of 65520)
        near = (v.abs() - 65520).abs() <= tol
        v = torch.where(near, o, torch.where(v.abs() > 65520, v.sign() * math.inf, v))
    fin = v.isfinite()
    assert torch.equal(o.isfinite(), fin), f"{what}: finite pattern"
    assert torch.equal(o.isnan(), v.isnan()) and torch.equal(o[v.isinf()], v[v.isinf()]), what
    bad = ~((o - v).abs() <= tol)[fin]
    assert not bad.any(), (f"{what}: {int(bad.sum())}/{o.numel()} off, worst "
                           f"{float(((o - v).abs() - tol)[fin].max()):.3e} beyond")


def _run(t, **kw):
    import natten_amd

    kw = {"return_lse": True, **kw}
    return natten_amd.cache_attention(t["q"].to(DEV), _to(t["cache"]), t["tables"].to(DEV),
                                      t["lens"].to(DEV), kernel_size=t["window"], **kw)


def _check(t, what="", **kw):
    out, lse = _run(t, **kw)
    assert out.dtype == t["q"].dtype and lse.dtype == F32 and out.is_contiguous()
    ro, rl = _reference(t, kw.get("scale"))
    _near(out, ro, f"{what} out")
    _near(lse, rl, f"{what} lse")


# B, tokens, heads, kv heads, dim, page, lengths, window
CASES = {
    "one of everything": (1, 1, 1, 1, 16, 16, [1], None),
    "one page": (2, 1, 4, 2, 64, 128, [100, 37], None),
    "nothing to see": (2, 3, 2, 1, 16, 16, [0, 2], None),
    "small service": (4, 1, 8, 2, 64, 16, [131, 0, 1, 64], None),
    "ragged": (9, 1, 8, 2, 128, 64, [150, 0, 33, 1000, 129, 5], None),
    "long, few heads": (1, 1, 2, 1, 96, 32, [5000], None),
    "very long tables": (2, 1, 4, 1, 64, 16, [3100, 700], None),
    "two tiles of heads": (3, 1, 32, 1, 128, 64, [300, 0, 129], None),
    "very many heads": (1, 1, 70, 1, 80, 16, [40], None),
    "256 wide": (2, 1, 6, 2, 256, 32, [150, 7], None),
    "256 wide, tokens": (3, 3, 8, 1, 256, 64, [150, 7, 2], None),
    "208 wide": (3, 1, 4, 2, 208, 16, [40, 5, 0], None),
    "32 wide": (3, 2, 4, 2, 32, 16, [90, 33, 1], None),
    "tokens narrow": (3, 4, 4, 2, 64, 16, [80, 4, 2], None),
    "tokens wide": (2, 9, 4, 1, 64, 32, [200, 150], None),
    "tokens of several tiles": (2, 70, 4, 1, 32, 16, [333, 75], None),
    "tokens longer than the sequence": (2, 40, 2, 1, 32, 16, [25, 10], None),
    "window of one": (3, 1, 4, 2, 64, 16, [90, 1, 0], 1),
    "window": (3, 1, 4, 2, 80, 32, [400, 33, 300], 129),
    "window, tokens narrow": (2, 5, 3, 1, 64, 16, [300, 4], 7),
    "window, tokens wide": (2, 50, 4, 2, 64, 64, [300, 60], 37),
    "window over all": (2, 3, 2, 1, 64, 16, [60, 20], 5000),
    "window, tokens of several tiles": (1, 130, 3, 1, 48, 128, [390], 100),
    "tokens of 128 channels": (2, 33, 8, 2, 128, 64, [200, 33], None),
    "tokens of 96 channels": (2, 100, 6, 2, 96, 16, [330, 101], None),
    "many samples": (130, 1, 2, 2, 32, 16, [3, 0, 17, 40], None),
    "many samples and tiles": (40, 20, 4, 1, 64, 32, [64, 20, 5, 0, 33], 25),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", list(CASES))
def test_attention_against_the_definition(case, dtype):
    _check(_make(CASES[case], dtype), f"{case} {dtype}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("window", [None, 3500])
def test_a_long_prompt(dtype, window):
    """Rows and keys that fill the chip several times over; compared at some tokens."""
    t = _make((2, 1500, 8, 2, 64, 64, [6000, 1800], window), dtype, 11)
    out, lse = _run(t)
    at = (0, 1, 700, 1499)
    ro, rl = _reference(t, tokens=at)
    for j in at:
        _near(out[:, j], (ro[0][:, j], ro[1][:, j]), f"token {j}")
        _near(lse[:, j], (rl[0][:, j], rl[1][:, j]), f"token {j} lse")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scores_far_apart_and_scales(dtype):
    _check(_make((2, 3, 4, 2, 64, 16, [140, 70], None), dtype, 3, std=12.0), "far apart")
    _check(_make((2, 1, 4, 2, 64, 16, [140, 70], None), dtype, 3), "scale", scale=0.03)
    # rising scores: the reference point moves in every tile; scales 2^60 apart
    t = _make((1, 40, 2, 1, 32, 16, [320], None), dtype, 4)
    order = t["tables"][0].long()
    for i, page in enumerate(order.tolist()):
        t["cache"].key_scale.view(torch.uint8)[page] = 110 + i // 2
        t["cache"].value_scale.view(torch.uint8)[page] = 95 + 3 * (i % 20)
    _check(t, "rising")


def _unseen(t):
    """Mask [pages, size] of slots that no row of t sees."""
    size = t["cache"].key.shape[2]
    hidden = torch.ones(t["cache"].key.shape[0], size, dtype=torch.bool)
    L = t["q"].shape[1]
    for b, n in enumerate(t["lens"].tolist()):
        lo = 0 if t["window"] is None else max(0, n - L - t["window"] + 1)
        for p in range(lo, n):
            hidden[int(t["tables"][b, p // size]), p % size] = False
    return hidden


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", ["small service", "ragged", "tokens narrow", "tokens wide", "window",
                                  "window, tokens wide", "256 wide, tokens", "tokens of several tiles",
                                  "two tiles of heads", "window, tokens of several tiles",
                                  "tokens of 128 channels"])
def test_what_no_row_sees_is_not_read(case, dtype):
    """NaN in every slot behind a length and in front of every window, NaN scales on
    pages that hold no seen token, no page at all in the tables past the lengths."""
    t = _make(CASES[case], dtype)
    want = _run(t)
    hidden = _unseen(t)
    for i in (0, 1):
        codes = t["cache"][i].view(torch.uint8)
        codes.masked_fill_(hidden[:, None, :, None], 0x7f)
        t["cache"][2 + i].view(torch.uint8)[hidden.all(1)] = 255
    size = t["cache"].key.shape[2]
    t["tables"] = torch.cat([t["tables"], torch.full((t["tables"].shape[0], 3), -1, dtype=torch.int32)], 1)
    for a, b in zip(_run(t), want):
        assert torch.equal(a, b)
    for b, n in enumerate(t["lens"].tolist()):  # pages that no row sees are none
        for i in range(t["tables"].shape[1]):
            page = int(t["tables"][b, i])
            if page >= 0 and hidden[page].all():
                t["tables"][b, i] = (-1, 1 << 30)[i % 2]
    for a, b in zip(_run(t), want):
        assert torch.equal(a, b)
    assert size > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", ["small service", "ragged", "tokens wide", "window, tokens wide",
                                  "256 wide, tokens", "tokens of several tiles", "tokens of 128 channels"])
def test_entries_that_are_no_page_are_not_seen(case, dtype):
    t = _make(CASES[case], dtype)
    g = torch.Generator().manual_seed(2)
    out = torch.rand(t["tables"].shape, generator=g) < 0.4
    t["tables"][out] = torch.tensor([-1, 1 << 30, t["cache"].key.shape[0]], dtype=torch.int32)[
        torch.randint(0, 3, (int(out.sum()),), generator=g)]
    _check(t, case)
    t["tables"].fill_(-1)
    o, lse = _run(t)
    assert not o.any() and (lse == -math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", ["tokens narrow", "tokens wide", "window, tokens narrow",
                                  "window, tokens wide", "256 wide, tokens", "tokens of several tiles",
                                  "tokens of 128 channels", "tokens of 96 channels"])
def test_tokens_that_a_row_does_not_see(case, dtype):
    """A NaN reaches the rows that see its token alone: a value's its own channel, a
    key's the whole row."""
    t = _make(CASES[case], dtype)
    L, size = t["q"].shape[1], t["cache"].key.shape[2]
    n = int(t["lens"][0])
    at = n - 1 - (min(L, n) - 1) // 2  # seen by the later half of the sample's rows
    page, slot = int(t["tables"][0, at // size]), at % size
    for i in (1, 0):
        codes = t["cache"][i].view(torch.uint8)
        keep = codes[page, 0, slot, 5].item()
        codes[page, 0, slot, 5] = 0x7f
        (ro, _), _ = _reference(t)
        hit = ro.isnan()[0].any(-1)
        assert hit.any() and not hit.all() and int(ro[0, -1, 0].isnan().sum()) == (1 if i else ro.shape[-1])
        _check(t, f"{case} {i}")
        codes[page, 0, slot, 5] = keep


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_views(dtype):
    import natten_amd

    t = _make((3, 2, 8, 2, 64, 16, [90, 5, 41], None), dtype, 1)
    B, L, H, D = t["q"].shape
    lens, tables = t["lens"].to(DEV), t["tables"].to(DEV)
    dev = _to(t["cache"])
    pages = dev.key.shape[0]
    tokens_first = torch.zeros(pages, 16, 2, 64, dtype=torch.uint8, device=DEV)
    tokens_first.copy_(dev.key.view(torch.uint8).transpose(1, 2))
    spread = torch.zeros(2 * pages, 2, 16, 80, dtype=torch.uint8, device=DEV)[::2, :, :, 16:]
    spread.copy_(dev.value.view(torch.uint8))
    scales = dev.key_scale.view(torch.uint8).t().contiguous().t()
    odd = natten_amd.PagedCache(tokens_first.transpose(1, 2).view(E4M3), spread.view(E4M3), scales.view(E8M0),
                                dev.value_scale)
    q = t["q"].to(DEV)
    packed = torch.cat([q, q * 2], 2)[:, :, :H]
    wide = torch.cat([q[..., :3], q, q[..., :2]], -1)[..., 3:3 + D]
    want = natten_amd.cache_attention(q, dev, tables, lens, return_lse=True)
    for qq in (q, packed, wide, q.transpose(0, -1).contiguous().transpose(0, -1)):
        for cache in (dev, odd):
            for tb in (tables, tables.long(), torch.stack([tables] * 2, -1)[..., 0],
                       torch.cat([tables, tables], 1)[:, :tables.shape[1]]):
                for a, b in zip(natten_amd.cache_attention(qq, cache, tb, lens, return_lse=True), want):
                    assert torch.equal(a, b)
    for form in (lens.long(), lens.cpu(), lens.cpu().long(), torch.stack((lens, lens), 1)[:, 0]):
        assert torch.equal(natten_amd.cache_attention(q, dev, tables, form), want[0])
    cap = tables.shape[1] * 16
    for wild, same in (([1 << 40, 5, 41], [cap, 5, 41]), ([-5, 5, 41], [0, 5, 41])):
        assert torch.equal(natten_amd.cache_attention(q, dev, tables, torch.tensor(wild, device=DEV)),
                           natten_amd.cache_attention(q, dev, tables, torch.tensor(same, device=DEV)))
    # samples that share pages
    shared = tables[:1].expand(3, -1)
    lens3 = torch.tensor([90, 33, 64], device=DEV)
    both = natten_amd.cache_attention(q, dev, shared, lens3)
    for b in range(3):
        assert torch.equal(both[b:b + 1], natten_amd.cache_attention(q[b:b + 1], dev, tables[:1], lens3[b:b + 1]))


@pytest.mark.gpu
def test_empty_calls():
    import natten_amd

    cache = natten_amd.paged_cache(4, 2, 32, 16)
    for B, L in ((0, 1), (2, 0)):
        q = torch.randn(B, L, 4, 32, device=DEV)
        k = torch.randn(B, L, 2, 32, device=DEV)
        tables = torch.zeros(B, 2, dtype=torch.int32, device=DEV)
        lens = torch.zeros(B, dtype=torch.int32, device=DEV)
        natten_amd.cache_append(cache, k, k, tables, lens)
        out, lse = natten_amd.cache_attention(q, cache, tables, lens, return_lse=True)
        assert out.shape == q.shape and lse.shape == q.shape[:3]
    q, k = torch.randn(2, 3, 4, 32, device=DEV), torch.randn(2, 3, 2, 32, device=DEV)
    lens = torch.tensor([5, 3], device=DEV)
    for pages, per in ((0, 2), (4, 0), (0, 0)):
        cache = natten_amd.paged_cache(pages, 2, 32, 16)
        tables = torch.zeros(2, per, dtype=torch.int32, device=DEV)
        natten_amd.cache_append(cache, k, k, tables, lens)
        out, lse = natten_amd.cache_attention(q, cache, tables, lens, return_lse=True)
        assert not out.any() and (lse == -math.inf).all()


@pytest.mark.gpu
def test_streams_twin_and_capture():
    import natten_amd
    import natten_amd.autograd.fused as AF

    B, H, Hk, D, size, per = 6, 8, 2, 64, 16, 8
    base = _fill(B * per, Hk, size, D, 3)
    tables = _tables(B, per, B * per, 1).to(DEV)
    lens = torch.tensor([(37 * b) % 100 + 1 for b in range(B)], dtype=torch.int32, device=DEV)
    q, k, v = (randn((B, 1, h, D), BF16, h).to(DEV) for h in (H, Hk, Hk))
    start = _to(base)

    def step(cache):
        for t, s in zip(cache, start):
            t.view(torch.uint8).copy_(s.view(torch.uint8))
        natten_amd.cache_append(cache, k, v, tables, lens)
        return natten_amd.cache_attention(q, cache, tables, lens, return_lse=True)

    want = step(_to(base))
    with AF.python_autograd():
        twin = step(_to(base))
    side, second = torch.cuda.Stream(), torch.cuda.Stream()
    caches = [_to(base) for _ in range(4)]
    side.wait_stream(torch.cuda.current_stream())
    second.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(second):  # two calls at once, each with its own workspace
        beside = step(caches[0])
    graphs, helds = [], []
    with torch.cuda.stream(side):
        other = step(caches[1])
        torch.cuda.synchronize()
        for c in caches[2:]:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                with pytest.raises(RuntimeError, match="on the host"):
                    natten_amd.cache_attention(q, c, tables, torch.ones(B, dtype=torch.int32))
                helds.append(step(c))
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c, d in zip(want, twin, other, beside):
        assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)
    eager = _to(base)
    for r in range(3):
        lens.copy_(torch.tensor([(17 * r + 31 * b) % 127 + 1 for b in range(B)]))
        for i, x in enumerate((q, k, v)):
            x.copy_(randn(x.shape, BF16, 40 + 3 * r + i))
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        fresh = step(eager)
        for held, c in zip(helds, caches[2:]):
            for a, b in zip(fresh, held):
                assert torch.equal(a, b), r
            for a, b in zip(eager, c):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), r


@pytest.mark.gpu
def test_the_cache_and_its_attention_against_neighborhood_attention():
    """A prompt appended in two parts, then token by token: the attention is that of
    na1d, causal, on the values that the cache holds -- and merged with a prefix that
    the batch shares."""
    import natten_amd

    B, T, H, Hk, D, size, W, N = 2, 150, 4, 2, 64, 16, 31, 40
    q, k, v = (randn((B, T, h, D), F32, s).to(DEV) for s, h in ((1, H), (2, Hk), (3, Hk)))
    pk, pv = (randn((N, Hk, D), F32, s).to(DEV) for s in (4, 5))
    cache = natten_amd.paged_cache(2 * 10, Hk, D, size)
    tables = _tables(B, 10, 20, 1).to(DEV)
    at = 0
    for n in (77, 64, *([1] * 9)):
        lens = torch.full((B,), at + n, dtype=torch.int32, device=DEV)
        natten_amd.cache_append(cache, k[:, at:at + n], v[:, at:at + n], tables, lens)
        at += n
        got, gl = natten_amd.cache_attention(q[:, at - n:at], cache, tables, lens, kernel_size=W, return_lse=True)
        host = natten_amd.PagedCache(*(t.view(torch.uint8).cpu().view(t.dtype) for t in cache))
        keys, vals = (x[tables.cpu().long()].transpose(2, 3).reshape(B, -1, Hk, D)[:, :at].float().to(DEV)
                      for x in _held({"cache": host}))
        want, wl = natten_amd.na1d(q[:, :at], keys, vals, kernel_size=W, is_causal=True, return_lse=True)
        assert torch.allclose(got, want[:, at - n:], rtol=1e-5, atol=1e-5)
        assert torch.allclose(gl, wl[:, at - n:], rtol=1e-5, atol=1e-5)
    a, la = natten_amd.prefix_attention(q[:, -1:], pk, pv, return_lse=True)
    merged, _ = natten_amd.merge_attentions([a, got], [la, gl])
    whole = natten_amd.prefix_attention(q[:, -1:], pk, pv, keys.contiguous(), vals.contiguous(), kernel_size=W)
    assert torch.allclose(merged, whole, rtol=1e-5, atol=1e-5)
    # held to within e4m3's half step of 2^-4, and the subnormals' of 2^-10 of the scale
    step = k[:, :at].abs() * 2.0 ** -4 + k.abs().max() * 2.0 ** -17
    assert ((keys - k).abs() <= step).all()


@pytest.mark.gpu
def test_gradients_tangents_and_transforms_are_refused():
    import natten_amd
    import natten_amd.autograd.fused as AF

    cache = natten_amd.paged_cache(4, 2, 32, 16)
    tables, lens = torch.tensor([[0, 1], [2, 3]], device=DEV), torch.tensor([20, 3], device=DEV)
    q, k = torch.randn(2, 1, 4, 32, device=DEV), torch.randn(2, 1, 2, 32, device=DEV)

    def append(key, value):
        natten_amd.cache_append(cache, key, value, tables, lens)

    def attend(query):
        return natten_amd.cache_attention(query, cache, tables, lens)

    dual = torch.autograd.forward_ad.make_dual
    before = [t.view(torch.uint8).clone() for t in cache]
    for twin in (False, True):
        with AF.python_autograd(twin):
            for fn, ts in ((append, (k, k)), (attend, (q,))):
                for i in range(len(ts)):
                    with pytest.raises(RuntimeError, match="no backward"):
                        fn(*(x.detach().clone().requires_grad_(j == i) for j, x in enumerate(ts)))
                    with torch.autograd.forward_ad.dual_level():
                        with pytest.raises((NotImplementedError, RuntimeError), match="derivative|no backward"):
                            fn(*(dual(x, torch.ones_like(x)) if j == i else x for j, x in enumerate(ts)))
                with pytest.raises(RuntimeError, match="functorch"):
                    torch.vmap(lambda *a: fn(*a))(*(x[None] for x in ts))
    for a, b in zip(cache, before):
        assert torch.equal(a.view(torch.uint8), b)
    with torch.no_grad():
        append(k.clone().requires_grad_(True), k)
        attend(q.clone().requires_grad_(True))
    version = cache.key._version
    append(k, k)
    assert cache.key._version > version
    with pytest.raises(RuntimeError, match="devices|HIP"):
        natten_amd.cache_attention(q, cache, tables.cpu(), lens)
    with pytest.raises(ValueError, match="seq_lens must be in"):
        natten_amd.cache_attention(q, cache, tables, torch.tensor([1, 33]))
    with pytest.raises(ValueError, match="new_lens must be in"):
        natten_amd.cache_append(cache, k, k, tables, lens, torch.tensor([1, 2]))


def test_refusals():
    import natten_amd
    from natten_amd._core import _lib

    cache = natten_amd.paged_cache(5, 2, 32, 16, device="cpu")
    q, k = torch.randn(2, 3, 4, 32), torch.randn(2, 3, 2, 32)
    tables, lens = torch.zeros(2, 4, dtype=torch.int32), torch.tensor([5, 7])
    with pytest.raises(RuntimeError, match="HIP"):
        natten_amd.cache_append(cache, k, k, tables, lens)
    with pytest.raises(RuntimeError, match="HIP"):
        natten_amd.cache_attention(q, cache, tables, lens)
    for args, match in (((5, 2, 24), "multiple of 16"), ((5, 2, 272), "up to 256"), ((5, 2, 0), "multiple"),
                        ((5, 0, 32), "heads must"), ((-1, 2, 32), "pages must"), ((5, 2, 32, 48), "page_size"),
                        ((5, 2, 32, 256), "page_size"), ((2.0, 2, 32), "pages must")):
        with pytest.raises(ValueError, match=match):
            natten_amd.paged_cache(*args, device="cpu")
    PC = natten_amd.PagedCache
    wrong = natten_amd.paged_cache(5, 2, 48, 16, device="cpu")
    odd = torch.zeros(5, 2, 16, 40, dtype=torch.uint8).view(E4M3)[..., 8:]
    for c, match in ((None, "PagedCache"), (PC(cache[0], wrong[1], *cache[2:]), "cache.key and cache.value"),
                     (PC(cache[0][0], cache[1][0], *cache[2:]), "cache.key and"),
                     (PC(*cache[:2], cache[2][:3], cache[3]), "key_scale"),
                     (PC(cache[0].view(torch.uint8), *cache[1:]), "float8"),
                     (PC(*cache[:3], cache[3].view(torch.uint8)), "float8"),
                     (PC(odd, cache[1], *cache[2:]), "multiples of 16"),
                     (PC(cache[0].view(torch.uint8).transpose(2, 3).contiguous().transpose(2, 3).view(torch.uint8)
                         .as_strided((5, 2, 16, 32), (1024, 512, 1, 16)).view(torch.uint8), *cache[1:]), "float8")):
        with pytest.raises(ValueError, match=match):
            natten_amd.cache_append(c, k, k, tables, lens)
        with pytest.raises(ValueError, match=match):
            natten_amd.cache_attention(q, c, tables, lens)
    for args, kw, match in (
            ((k[0], k[0], tables, lens), {}, "key and value must"),
            ((k, k[:, :2], tables, lens), {}, "key and value must"),
            ((k[:, :, :1], k[:, :, :1], tables, lens), {}, "key and value must"),
            ((k[..., :16], k[..., :16], tables, lens), {}, "key and value must"),
            ((k, k.half(), tables, lens), {}, "same dtype"),
            ((k, k, tables[0], lens), {}, "tables must"),
            ((k, k, tables[:1], lens), {}, "tables must"),
            ((k, k, tables.float(), lens), {}, "tables must be int32"),
            ((k, k, tables, lens[:1]), {}, "length B=2"),
            ((k, k, tables, lens.float()), {}, "int32 or int64"),
            ((k, k, tables, lens, lens[None]), {}, "new_lens must be a 1-D"),
            ((k, k, tables, lens, lens.short()), {}, "new_lens must be int32"),
            ((k, k, tables[:, :1].expand(2, (1 << 26) + 1), lens), {}, "2\\^30")):
        with pytest.raises(ValueError, match=match):
            natten_amd.cache_append(cache, *args, **kw)
    for args, kw, match in (
            ((q[0], cache, tables, lens), {}, "query must"),
            ((q[..., :16], cache, tables, lens), {}, "query must"),
            ((q[:, :, :3], cache, tables, lens), {}, "divisible"),
            ((q, cache, tables[:1], lens), {}, "tables must"),
            ((q, cache, tables, lens[:1]), {}, "length B=2"),
            ((q, cache, tables, lens), dict(kernel_size=0), "kernel_size"),
            ((q, cache, tables, lens), dict(kernel_size=2.0), "kernel_size"),
            ((q, cache, tables, lens), dict(scale=0.0), "scale"),
            ((q, cache, tables, lens), dict(scale=math.nan), "scale"),
            ((q, cache, tables, lens), dict(scale=math.inf), "scale")):
        with pytest.raises(ValueError, match=match):
            natten_amd.cache_attention(*args, **kw)

    lib = _lib.load()

    def params(**kw):
        return _lib.NaCacheParams(**{**dict(batch=2, tokens=1, heads=4, kv_heads=2, head_dim=32, dtype=2,
                                            pages=5, page_size=16, table_pages=4, scale=0.25), **kw})

    def append(p, c=None, x=None):
        return lib.na_cache_append(p, c, x, x, x, x, None, None)

    def attend(p, c=None, x=None, ws=None, n=0):
        return lib.na_cache_attend(p, c, x, x, x, x, None, ws, n, None)

    pages = _lib.NaCache(key=256, value=256, key_scale=1, value_scale=1)
    for n in ("key_stride", "value_stride"):
        getattr(pages, n)[:] = (1024, 512, 32)
    assert append(params()) == 1 and b"non-NULL" in lib.na_last_error()
    assert append(params(), pages) == 1 and b"tables" in lib.na_last_error()
    assert attend(params()) == 1 and attend(params(), pages) == 1
    assert attend(params(), pages, 1) == 4 and b"workspace" in lib.na_last_error()
    assert lib.na_cache_attend_workspace_bytes(params()) > 0
    for n in ("key", "value"):
        bad = _lib.NaCache.from_buffer_copy(pages)
        setattr(bad, n, 264)
        assert append(params(), bad, 1) == 1 and attend(params(), bad, 1) == 1
        assert b"16 bytes" in lib.na_last_error()
        bad = _lib.NaCache.from_buffer_copy(pages)
        getattr(bad, n + "_stride")[2] = 40
        assert append(params(), bad, 1) == 1 and attend(params(), bad, 1) == 1
    for empty in (dict(batch=0), dict(tokens=0)):
        assert append(params(**empty)) == 0 and attend(params(**empty)) == 0
    assert append(params(pages=0)) == 0 and append(params(table_pages=0)) == 0
    for bad in (dict(kv_heads=0), dict(dtype=5), dict(pages=-1), dict(table_pages=-1), dict(batch=-1),
                dict(tokens=-1)):
        assert append(params(**bad)) == 1 and attend(params(**bad)) == 1, bad
    for bad in (dict(heads=3), dict(heads=0), dict(window=-1), dict(scale=0.0), dict(scale=math.inf),
                dict(scale=math.nan)):
        assert attend(params(**bad)) == 1, bad
        assert lib.na_cache_attend_workspace_bytes(params(**bad)) == 0
    for bad in (dict(head_dim=24), dict(head_dim=272), dict(page_size=8), dict(page_size=48),
                dict(page_size=256), dict(table_pages=(1 << 26) + 1), dict(tokens=(1 << 30) + 1)):
        assert append(params(**bad)) == 2 and attend(params(**bad)) == 2, bad
    assert attend(params(batch=1 << 20, tokens=1 << 9)) == 2
    assert append(params(batch=1 << 20, tokens=1 << 12, table_pages=1 << 12), pages, 1) == 2


# ---- layouts and sizes at the kernels' limits --------------------------------

def _codes(t):
    return t.view(torch.uint8)


def test_strides_and_sizes_that_are_refused():
    import natten_amd
    from natten_amd._core import _lib

    lib = _lib.load()
    p = dict(batch=2, tokens=1, heads=4, kv_heads=2, head_dim=32, dtype=2, pages=5, page_size=16,
             table_pages=4, scale=0.25)

    def both(n, strides, **kw):
        c = _lib.NaCache(key=256, value=256, key_scale=1, value_scale=1)
        for m in ("key_stride", "value_stride"):
            getattr(c, m)[:] = (1024, 512, 32)
        getattr(c, n)[:] = strides
        q = _lib.NaCacheParams(**{**p, **kw})
        return {lib.na_cache_append(q, c, 1, 1, 1, 1, None, None),
                lib.na_cache_attend(q, c, 1, 1, 1, 1, None, None, 0, None)}

    for n in ("key_stride", "value_stride"):
        for strides in ((1 << 31, 512, 32), (1024, 512, 1 << 24), (-1024, 512, 32), (1024, -512, 32),
                        (1024, 512, -32)):
            assert both(n, strides) == {2}, strides
            assert b"strides" in lib.na_last_error()
    # a call's units of 64 keys are counted in 31 bits; a window keeps them few
    big = dict(p, batch=1 << 13, kv_heads=64, heads=64, table_pages=1 << 16)
    assert lib.na_cache_attend_workspace_bytes(_lib.NaCacheParams(**big)) == 0
    assert b"too large" in lib.na_last_error()
    assert lib.na_cache_attend_workspace_bytes(_lib.NaCacheParams(**big, window=4096)) > 0
    cache = natten_amd.paged_cache(2, 2, 32, 16, device="cpu")
    tables, lens = torch.zeros(2, 4, dtype=torch.int32), torch.tensor([5, 7])
    k = torch.randn(2, 3, 2, 32)
    for st in ((1 << 31, 512, 32, 1), (1024, 512, 1 << 24, 1)):
        far = torch.empty_strided((2, 2, 16, 32), st, dtype=torch.uint8, device="meta").view(E4M3)
        with pytest.raises(ValueError, match="2\\^31"):
            natten_amd.cache_append(cache._replace(value=far), k, k, tables, lens)
        with pytest.raises(ValueError, match="2\\^31"):
            natten_amd.cache_attention(k, cache._replace(key=far), tables, lens)


def _twins(cache, twin, q, k, v, tables, lens, **kw):
    """Appends to both caches and attends over both: the same bits."""
    import natten_amd

    out = []
    for c in (cache, twin):
        natten_amd.cache_append(c, k, v, tables, lens)
        out.append(natten_amd.cache_attention(q, c, tables, lens, return_lse=True, **kw))
    for a, b in zip(*out):
        assert torch.equal(a, b)
    assert out[0][0].isfinite().all() and out[0][0].abs().max() > 0
    used = tables.unique().long()
    for a, b in zip(cache, twin):
        assert torch.equal(_codes(a)[used], _codes(b)[used])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40, 300])
def test_strides_at_their_limits(n):
    """Pages 2^31 - 16 bytes apart, tokens 2^24 - 16: offsets past 32 bits."""
    import natten_amd

    big = torch.zeros(3 << 31, dtype=torch.uint8, device=DEV)
    st = ((1 << 31) - 16, 64, (1 << 24) - 16, 1)
    cache = natten_amd.paged_cache(3, 2, 64, 128)
    k8, v8 = (big.as_strided((3, 2, 128, 64), st, at).view(E4M3) for at in (0, 4096))
    cache = cache._replace(key=k8, value=v8)
    twin = natten_amd.paged_cache(3, 2, 64, 128)
    tables = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)
    for length in (n, 384 if n > 84 else 300 + n) if n < 300 else (300,):
        k, v = (randn((1, length, 2, 64), BF16, s).to(DEV) for s in (1, 2))
        lens = torch.tensor([length], device=DEV)
        q = randn((1, n, 4, 64), BF16, 3).to(DEV)
        _twins(cache, twin, q, k, v, tables, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 24])
def test_a_pool_past_four_gigabytes(n):
    import natten_amd

    pages = (1 << 32) // (2 * 128 * 256) + 300
    cache = natten_amd.paged_cache(pages, 2, 256, 128)
    twin = natten_amd.paged_cache(6, 2, 256, 128)
    near = torch.arange(6, dtype=torch.int32, device=DEV).view(2, 3)
    far = torch.tensor([[pages - 1, 0, pages - 2], [32768, 65536, 65535]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([350, 129], device=DEV)
    k, v = (randn((2, 350, 2, 256), BF16, s).to(DEV) for s in (1, 2))
    q = randn((2, n, 8, 256), BF16, 3).to(DEV)
    outs = []
    for c, t in ((cache, far), (twin, near)):
        natten_amd.cache_append(c, k, v, t, lens)
        outs.append(natten_amd.cache_attention(q, c, t, lens))
    assert torch.equal(*outs) and outs[0].isfinite().all() and outs[0].abs().max() > 0
    for a, b in zip(cache, twin):
        assert torch.equal(_codes(a)[far.long().flatten()], _codes(b)[near.long().flatten()])


@pytest.mark.gpu
@pytest.mark.parametrize("python", [False, True])
def test_strides_of_dimensions_of_one(python, monkeypatch):
    """One head, whose stride is no multiple of 16 and means nothing."""
    import natten_amd
    from natten_amd.autograd import fused

    monkeypatch.setattr(fused, "_py_autograd", python)
    twin = natten_amd.paged_cache(4, 1, 32, 16)
    cache = natten_amd.paged_cache(4, 1, 32, 16)
    cache = natten_amd.PagedCache(*(_codes(t).as_strided((4, 1, 16, 32), (512, 7, 32, 1)).view(E4M3)
                                    for t in cache[:2]), *cache[2:])
    k, v = (randn((2, 20, 1, 32), BF16, s).to(DEV) for s in (1, 2))
    q = randn((2, 3, 2, 32), BF16, 3).to(DEV)
    tables = torch.tensor([[0, 2], [3, 1]], device=DEV)
    _twins(cache, twin, q, k, v, tables, torch.tensor([20, 17], device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 70, 200])
def test_pages_in_front_of_every_window_are_given_back(n):
    """Their entries are -1, or name pages of NaNs: the same bits either way."""
    import natten_amd

    cache = natten_amd.paged_cache(130, 2, 64, 16)
    tables = torch.randperm(128, generator=torch.Generator().manual_seed(1)).view(1, 128).int().to(DEV)
    k, v = (randn((1, 2000, 2, 64), BF16, s).to(DEV) for s in (1, 2))
    lens = torch.tensor([2000], device=DEV)
    natten_amd.cache_append(cache, k, v, tables, lens)
    _codes(cache[0])[129], _codes(cache[1])[129] = 127, 127
    q = randn((1, n, 8, 64), BF16, 3).to(DEV)
    want = natten_amd.cache_attention(q, cache, tables, lens, kernel_size=700, return_lse=True)
    for entry in (-1, 129):
        t = tables.clone()
        t[:, :(2000 - n - 699) // 16] = entry
        t[:, 125:] = entry
        got = natten_amd.cache_attention(q, cache, t, lens, kernel_size=700, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), entry


# ---- short and long tables ---------------------------------------------------
# Single tokens against short tables run without a division of the keys; entries behind
# every length that are no page make the tables long.

def _lengthen(t):
    size = t["cache"].key.shape[2]
    t["tables"] = torch.cat([t["tables"], torch.full((t["tables"].shape[0], 4096 // size), -1, dtype=torch.int32)], 1)
    return t


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", list(CASES))
def test_long_tables_of_short_sequences(case, dtype):
    t = _lengthen(_make(CASES[case], dtype, 3))
    _check(t, f"{case} {dtype}")
    want = _run(t)
    hidden = _unseen(t)
    for i in (0, 1):
        t["cache"][i].view(torch.uint8).masked_fill_(hidden[:, None, :, None], 0x7f)
        t["cache"][2 + i].view(torch.uint8)[hidden.all(1)] = 255
    for a, b in zip(_run(t), want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("pages", [15, 16, 17, 24, 25, 80, 81])
def test_on_both_sides_of_the_division(pages, dim, dtype):
    """Tables of up to 256, 384 and 1280 keys and one page more, all of them full."""
    _check(_make((2, 1, 4, 2, dim, 16, [16 * pages, 16 * pages - 9], None), dtype, pages))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("samples, pages", [(63, 128), (64, 128), (64, 129)])
def test_on_both_sides_of_the_division_of_many(samples, pages, dtype):
    """Half a chip's items, tables of up to 2048 keys and one page more."""
    lens = [16 * pages, 1, 777, 0, 1300, 16 * pages - 30]
    _check(_make((samples, 1, 4, 2, 64, 16, lens, None), dtype, pages))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_a_long_sequence_with_a_short_window(dtype):
    """Keys from 60000 on, windows on either side of the division."""
    for window in (1, 300, 1264, 1265, 3000):
        _check(_make((1, 1, 4, 2, 64, 64, [61001], window), dtype, window), f"{window}")
