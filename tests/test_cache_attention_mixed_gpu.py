"""l2c_cache_attention of calls whose sequences have very different numbers of new tokens and positions: single tokens beside
chunks, on both sides of what decides between small and large tiles, and one long sequence among short ones."""
import pytest
from paged import Cache
from test_cache_attention_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("singles,chunk,context", [(60, 150, 700), (60, 500, 700), (3, 300, 9000), (200, 1, 20000), (1, 40, 5000)])
@pytest.mark.parametrize("first", [False, True])
def test_chunks_beside_single_tokens(torch_gpu, l2c, first, singles, chunk, context, cache):
    lengths = [1 + (i * 53) % 130 for i in range(singles)]
    lengths, new = ([context, *lengths], [chunk] + [1] * singles) if first else ([*lengths, context], [1] * singles + [chunk])
    check(l2c, Cache(chunk + singles, lengths, new, 2, 64, 16, cache, rows_behind=2), 8)
    check(l2c, Cache(chunk, lengths, new, 2, 128, 16, cache), 8, window=100)
