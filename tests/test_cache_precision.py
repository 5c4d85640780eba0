"""cache_attention's rounding of probabilities, by every kernel that bfloat16 queries take:
an output is off by half a step of its own type, the products' and sums' float32, and
no more than 2^-16 of the mean of |v| by the probabilities (test_cache gives the bounds;
there a bfloat16 row may be off by 2^-8 of it)."""

import pytest
import torch

import test_cache as C

BF16 = torch.bfloat16

# B, tokens, heads, kv heads, dim, page, lengths, window: rows of a tile, channels
TILES = {
    "a workgroup an item, 64": (2, 1, 8, 2, 64, 16, [700, 90], None),
    "a workgroup an item, 128": (2, 1, 8, 2, 128, 64, [700, 90], None),
    "a workgroup an item, 256": (2, 1, 6, 2, 256, 32, [350, 90], None),
    "shared out, 64": (1, 1, 4, 1, 64, 16, [3100], None),
    "shared out, 128": (1, 1, 4, 1, 128, 16, [3100], None),
    "shared out, 256": (1, 1, 4, 1, 256, 32, [1500], None),
    "32 rows of 64": (2, 7, 4, 1, 64, 16, [900, 300], None),
    "64 rows of 64": (2, 9, 4, 1, 64, 32, [900, 300], None),
    "64 rows of 128": (2, 12, 4, 1, 128, 64, [900, 300], None),
    "64 rows of 256": (1, 12, 4, 1, 256, 64, [700], None),
    "128 rows of 64": (1, 70, 4, 2, 64, 16, [900], 600),
    "128 rows of 128": (1, 30, 4, 1, 128, 64, [900], None),
    "256 rows of 128": (1, 70, 4, 1, 128, 64, [900], None),
    "256 rows of 96": (1, 70, 4, 1, 96, 16, [400], 300),
}


@pytest.mark.gpu
@pytest.mark.parametrize("case", list(TILES))
def test_probabilities_of_bfloat16_queries(case, monkeypatch):
    monkeypatch.setitem(C.PARTS, BF16, 2.0 ** -16)
    C._check(C._make(TILES[case], BF16, 2), case)


# 65 to 128 rows of 65 to 128 channels: a bfloat16 tile of its own, through test_cache's
# tests of what a row sees
ROWS = {
    "100 rows of 128": (2, 25, 8, 2, 128, 64, [200, 33], None),
    "128 rows of 96": (2, 32, 4, 1, 96, 16, [330, 101], None),
    "window, 66 rows of 80": (2, 33, 4, 2, 80, 32, [300, 60], 37),
    "window, 120 rows of 128": (1, 40, 3, 1, 128, 128, [390], 100),
}


@pytest.mark.gpu
@pytest.mark.parametrize("test", [
    C.test_attention_against_the_definition, C.test_what_no_row_sees_is_not_read,
    C.test_entries_that_are_no_page_are_not_seen, C.test_tokens_that_a_row_does_not_see,
    C.test_long_tables_of_short_sequences], ids=lambda t: t.__name__)
@pytest.mark.parametrize("case", list(ROWS))
def test_tiles_of_128_rows(case, test, monkeypatch):
    monkeypatch.setitem(C.CASES, case, ROWS[case])
    test(case, BF16)
