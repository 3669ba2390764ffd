"""l2c_cache_attention over e4m3 pages of sizes that are no multiple of four: scales are read one a lane there, and rows of
a tile lie in pages of their own."""
import pytest
from paged import Cache
from test_cache_attention_gpu import check

pytestmark = pytest.mark.gpu


# Widths that are multiples of 16 and of 8 only, for both ways of reading a row.
@pytest.mark.parametrize("width", [64, 72, 128, 136])
@pytest.mark.parametrize("new", [1, 7, 100])
@pytest.mark.parametrize("page", [1, 3, 6, 50])
def test_page_sizes_of_e4m3(torch_gpu, l2c, page, new, width):
    lengths = [max(new, n) for n in (page, page + 1, 3 * page, 34, 211)]
    check(l2c, Cache(page + new + width, lengths, [new] * 5, 2, width, page, "e4m3"), 8)


@pytest.mark.parametrize("page", [3, 6])
@pytest.mark.parametrize("new,window", [(1, 0), (1, 77), (5, 33), (300, 0), (300, 65)])
def test_parts_of_e4m3(torch_gpu, l2c, new, window, page):
    """The same where the positions are divided, where pages are not there, and behind windows."""
    c = Cache(page + new, [3001, 1700], [new, new], 2, 128, page, "e4m3")
    none = [(0, 1), (0, 500), (1, 0), (1, 333)]
    for s, column in none:
        c.tables[s, column] = -1
    check(l2c, c, 6, window=window, no_page=none)
