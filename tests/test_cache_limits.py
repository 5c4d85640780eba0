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
