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
