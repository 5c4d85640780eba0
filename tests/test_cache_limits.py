"""The paged cache at the ends of what its calls take: arguments of the C entries, values
and scales at the types' limits."""

import pytest
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _entry(**kw):
    """(library, parameters, a cache block of addresses that no host call reads)."""
    from natten_amd._core import _lib

    p = _lib.NaCacheParams(**{**dict(batch=2, tokens=1, heads=4, kv_heads=2, head_dim=32, dtype=2, pages=5,
                                     page_size=16, table_pages=4, table_stride=4, scale=0.25), **kw})
    c = _lib.NaCache(key=256, value=256, key_scale=1, value_scale=1)
    for n in ("key_stride", "value_stride"):
        getattr(c, n)[:] = (1024, 512, 32)
    return _lib.load(), p, c


@pytest.mark.parametrize("pages", [0, 5])
def test_tables_are_needed_where_they_have_entries(pages):
    """The kernels read entries up to a length, whether or not there are pages."""
    lib, p, c = _entry(pages=pages)
    assert lib.na_cache_attend(p, c, 1, None, 1, 1, None, None, 0, None) == 1
    assert b"tables" in lib.na_last_error()
    lib, p, c = _entry(pages=pages, table_pages=0)  # none to read: as far as the workspace
    assert lib.na_cache_attend(p, c, 1, None, 1, 1, None, None, 0, None) == 4


@pytest.mark.parametrize("scale", [2.5e38, 3.4e38])
def test_scales_whose_product_with_log2_e_is_infinite(scale):
    import natten_amd

    lib, p, c = _entry(scale=scale)
    assert lib.na_cache_attend(p, c, 1, 1, 1, 1, None, None, 0, None) == 1 and b"scale" in lib.na_last_error()
    lib, p, c = _entry(scale=1.9e38)
    assert lib.na_cache_attend(p, c, 1, 1, 1, 1, None, None, 0, None) == 4  # as far as the workspace
    cache = natten_amd.paged_cache(4, 2, 32, 16, device="cpu")
    args = torch.zeros(2, 1, 4, 32), cache, torch.zeros(2, 2, dtype=torch.int32), torch.tensor([3, 1])
    for bad in (scale, 1e-46):  # (float32 holds nothing as small)
        with pytest.raises(ValueError, match="scale"):
            natten_amd.cache_attention(*args, scale=bad)


# ---- queries at the ends of their types ----------------------------------------

# B, tokens, heads, kv heads, dim, page, lengths, window: every kind of tile
TILES = {
    "a workgroup an item": (2, 1, 8, 2, 64, 16, [131, 40], None),
    "a workgroup an item, 128": (2, 1, 8, 2, 128, 64, [131, 40], None),
    "shared out, 256": (1, 1, 4, 1, 256, 32, [700], None),
    "32 rows": (2, 7, 4, 1, 64, 16, [90, 33], None),
    "64 rows": (2, 12, 4, 1, 128, 64, [200, 70], None),
    "128 rows": (1, 70, 4, 2, 64, 16, [300], 200),
    "256 rows": (1, 70, 4, 1, 96, 16, [300], None),
}


@pytest.mark.gpu
@pytest.mark.parametrize("case", list(TILES))
def test_queries_next_to_the_largest_float32(case):
    """They round to no infinity as they are split.  Keys are some 2^-110, so that scores
    are finite, and `scale` brings them back to some units."""
    import test_cache as C

    t = C._make(TILES[case], F32, 5)
    t["cache"].key_scale.view(torch.uint8).fill_(10)
    g = torch.Generator().manual_seed(1)
    most = torch.finfo(F32).max
    near = torch.rand(t["q"].shape, generator=g) * 2.0 ** -7
    big = torch.where(t["q"] < 0, -1.0, 1.0) * (most * (1 - near))
    big[..., 0] = most
    some = torch.rand(t["q"].shape, generator=g) < 0.25
    t["q"] = torch.where(some, big, t["q"] * 2.0 ** 120)
    assert t["q"].isfinite().all()
    C._check(t, case, scale=2.0 ** -20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", list(TILES))
def test_infinite_queries(case, dtype):
    """Scores of -inf weigh nothing, a row of them alone sees nothing; a row with one of
    +inf, or with infinities of both signs, is NaN, its LSE too."""
    import test_cache as C

    t = C._make(TILES[case], dtype, 6)
    codes = t["cache"].key.view(torch.uint8)
    low = codes[..., 3] & 0x7f
    codes[..., 3] = torch.where(low == 0, 0x38, low) | 0x80  # channel 3: negative, none 0
    codes[..., 5] = torch.where(codes[..., 5] & 0x7f == 0, 0x38, codes[..., 5] & 0x7f)  # 5: positive
    want, want_lse = C._run(t)
    q = t["q"]
    t["q"] = q.clone()
    t["q"][:, -1, 0, 3] = float("inf")   # every score -inf
    t["q"][:, -1, 1, 5] = float("-inf")
    t["q"][:, -1, 2, 5] = float("inf")   # every score +inf
    t["q"][:, -1, 3, [3, 5]] = float("inf")  # -inf + inf
    out, lse = C._run(t)
    for h, kind in ((0, "none"), (1, "none"), (2, "nan"), (3, "nan")):
        if kind == "none":
            assert not out[:, -1, h].any() and (lse[:, -1, h] == -float("inf")).all(), h
        else:
            assert out[:, -1, h].isnan().all() and lse[:, -1, h].isnan().all(), h
    rest = torch.ones(out.shape[:3], dtype=torch.bool, device=out.device)
    rest[:, -1, :4] = False
    assert torch.equal(out[rest], want[rest]) and torch.equal(lse[rest], want_lse[rest])


# ---- scales outside the append's range -----------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", list(TILES))
def test_scales_outside_the_range_are_its_ends(case, dtype):
    import test_cache as C

    t = C._make(TILES[case], dtype, 7)
    outs = []
    for byte in (0, 1, 9, 10):
        for i in (2, 3):
            t["cache"][i].view(torch.uint8).fill_(byte)
        outs.append(C._run(t, scale=2.0 ** 100))
    assert outs[-1][0].abs().max() > 0 or dtype == F16  # (float16 ends at 2^-24)
    for out, lse in outs[:-1]:
        assert torch.equal(out, outs[-1][0]) and torch.equal(lse, outs[-1][1])
    outs = []
    # (256 products of up to 8 * 448 * 2^119 would pass 2^128, and so would the sums of 700
    # values of 448 * 2^119 before their division: codes of 7 * 2^-9 at most, sums below 2^127)
    t["q"] = t["q"] * 2.0 ** -20
    t["cache"].value.view(torch.uint8).bitwise_and_(0x87)
    for byte in (247, 255, 246):
        for i in (2, 3):
            t["cache"][i].view(torch.uint8).fill_(byte)
        outs.append(C._run(t, scale=2.0 ** -110))
    assert outs[-1][1].isfinite().all() and not outs[-1][0].isnan().any()
    for out, lse in outs[:-1]:
        assert torch.equal(out, outs[-1][0]) and torch.equal(lse, outs[-1][1])


@pytest.mark.gpu
@pytest.mark.parametrize("byte, taken", [(0, 10), (9, 10), (247, 246), (255, 246)])
def test_appending_to_a_page_with_such_a_scale(byte, taken):
    """Tokens in front keep their codes' values by the scale that they were taken by."""
    import natten_amd
    from _helpers import DEV, randn

    caches = []
    for b in (byte, taken):
        cache = natten_amd.paged_cache(2, 2, 32, 16)
        x = randn((1, 5, 2, 32), F32, 1).to(DEV)
        tables = torch.tensor([[1, 0]], device=DEV)
        natten_amd.cache_append(cache, x, x, tables, torch.tensor([5], device=DEV))
        for s in cache[2:]:
            s.view(torch.uint8).fill_(b)
        y = randn((1, 3, 2, 32), F32, 2).to(DEV) * 2.0 ** -116
        natten_amd.cache_append(cache, y, y, tables, torch.tensor([8], device=DEV))
        caches.append(cache)
    used = caches[0].key_scale.view(torch.uint8)[1]
    assert ((used >= 10) & (used <= 246)).all()
    for a, b in zip(*caches):
        assert torch.equal(a.view(torch.uint8)[1], b.view(torch.uint8)[1])


# ---- refusals and bounds that other tests pass by -------------------------------

def test_caches_whose_channels_are_not_adjacent():
    import natten_amd

    cache = natten_amd.paged_cache(5, 2, 32, 16, device="cpu")
    apart = (cache.key.view(torch.uint8).transpose(2, 3).contiguous().transpose(2, 3)
             .view(torch.float8_e4m3fn))
    assert apart.shape == cache.key.shape and apart.stride(3) == 16
    k, q = torch.randn(2, 3, 2, 32), torch.randn(2, 3, 4, 32)
    tables, lens = torch.zeros(2, 4, dtype=torch.int32), torch.tensor([5, 7])
    for name in ("key", "value"):
        bad = cache._replace(**{name: apart})
        with pytest.raises(ValueError, match="adjacent channels"):
            natten_amd.cache_append(bad, k, k, tables, lens)
        with pytest.raises(ValueError, match="adjacent channels"):
            natten_amd.cache_attention(q, bad, tables, lens)


def test_appending_to_shared_elements_is_refused():
    import natten_amd

    cache = natten_amd.paged_cache(5, 2, 32, 16, device="cpu")
    one = natten_amd.paged_cache(1, 1, 32, 16, device="cpu")
    k, q = torch.randn(2, 3, 2, 32), torch.randn(2, 3, 4, 32)
    tables, lens = torch.zeros(2, 4, dtype=torch.int32), torch.tensor([5, 7])
    for name, t in zip(cache._fields, one):
        shared = t.view(torch.uint8).expand(getattr(cache, name).shape).view(t.dtype)
        with pytest.raises(ValueError, match="share memory"):
            natten_amd.cache_append(cache._replace(**{name: shared}), k, k, tables, lens)
        with pytest.raises(RuntimeError, match="HIP"):  # (reading them is no mistake)
            natten_amd.cache_attention(q, cache._replace(**{name: shared}), tables, lens)
    with pytest.raises(RuntimeError, match="HIP"):  # one page and head: nothing is shared
        natten_amd.cache_append(one, k[:, :, :1], k[:, :, :1], tables, lens)


@pytest.mark.gpu
def test_a_table_that_names_pages_again():
    """A ring of four pages under a window of 20: tokens one at a time and in steps of up
    to 16, against a table of as many pages as the sequence has."""
    import natten_amd
    from _helpers import DEV, randn

    n, window = 400, 20
    ring, flat = natten_amd.paged_cache(4, 2, 64, 16), natten_amd.paged_cache(25, 2, 64, 16)
    tables = torch.arange(25, dtype=torch.int32, device=DEV).view(1, 25)
    k, v = (randn((1, n, 2, 64), BF16, s).to(DEV) for s in (1, 2))
    at = 0
    for step in [1] * 70 + [16, 3, 11, 16, 1, 7, 16, 16, 16, 5] * 3:
        if at + step > n:
            break
        at += step
        lens = torch.tensor([at], device=DEV)
        q = randn((1, step, 8, 64), BF16, at).to(DEV)
        outs = []
        for cache, t in ((ring, tables % 4), (flat, tables)):
            natten_amd.cache_append(cache, k[:, at - step:at], v[:, at - step:at], t, lens)
            # (pages that have left every window are no longer the ring's)
            gone = torch.arange(25, device=DEV) * 16 + 16 <= at - step - window + 1
            outs.append(natten_amd.cache_attention(q, cache, t.masked_fill(gone, -1), lens, kernel_size=window))
        assert torch.equal(*outs), at
    assert at > 300


@pytest.mark.gpu
@pytest.mark.parametrize("case", list(TILES))
def test_float16_outputs_around_their_largest(case):
    """Values around 65520, halfway from 65504 to what would come next: an output past it
    by more than its tolerance is an infinity of its sign, one before it finite and within
    the tolerance and half a step of 32; between them it is one of the two, and never NaN."""
    import test_cache as C

    t = C._make(TILES[case], F16, 8)
    g = torch.Generator().manual_seed(3)
    codes = t["cache"].value.view(torch.uint8)
    # 1.75, 1.875, 2 and 2.25, times 2^15: 57344, 61440, 65536 and 73728
    codes.copy_(torch.tensor([0x3e, 0x3f, 0x40, 0x41], dtype=torch.uint8)[
        torch.randint(0, 4, codes.shape, generator=g)])
    codes[..., 1::2] |= 0x80
    t["cache"].value_scale.view(torch.uint8).fill_(127 + 15)
    out, _ = C._run(t)
    (v, tol), _ = C._reference(t)
    tol = tol - v.abs() * torch.finfo(F16).eps / 2  # without the output's own rounding
    o = out.cpu().double()
    assert not o.isnan().any() and ((o.sign() == v.sign()) | (v == 0)).all()
    past, before = v.abs() - tol > 65520, v.abs() + tol < 65520
    assert past.any() and before.any()
    assert o[past].isinf().all() and o[before].isfinite().all()
    fin = o.isfinite()
    assert ((o - v).abs()[fin] <= (tol + 16)[fin]).all()
    assert (v.abs()[o.isinf()] >= (65520 - tol)[o.isinf()]).all()


@pytest.mark.gpu
def test_rows_that_see_nothing_and_masked_values_of_every_kind():
    """Codes of NaN behind the lengths, in rows that see nothing and in pages of no one."""
    import natten_amd
    from _helpers import DEV

    for dim in (64, 128, 256):
        cache = natten_amd.paged_cache(8, 2, dim, 16)
        for t in cache[:2]:
            t.view(torch.uint8).fill_(0x7f)
        for t in cache[2:]:
            t.view(torch.uint8).fill_(255)
        tables = torch.tensor([[0, 1, -1, 7], [2, 3, 4, 5]], dtype=torch.int32, device=DEV)
        for n in (1, 5, 40):
            q = torch.randn(2, n, 8, dim, device=DEV, dtype=BF16)
            out, lse = natten_amd.cache_attention(q, cache, tables, torch.zeros(2, dtype=torch.int32, device=DEV),
                                                  return_lse=True)
            assert not out.any() and (lse == -float("inf")).all()
