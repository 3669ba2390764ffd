"""l2c_cache_append reads the rows of its sequences and no others: k and v may end where those do, in calls (captured
ones, say) of more rows."""
import pytest
import torch
from paged import NAN, Cache, fused
from test_cache_append_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("new", [[1, 1], [0, 0], [700, 500]], ids=str)
@pytest.mark.parametrize("behind", [1, 37, 40000])
def test_rows_behind_the_sequences(torch_gpu, l2c, behind, new, cache):
    """k and v have the sequences' rows alone, and all that is behind them is theirs to read: nothing is."""
    c = Cache(behind, [n + 3 for n in new], new, 8, 128, 16, cache)
    own = c.rows
    k, v = (torch.cat((fused(own, 8 * 128, c.gen), torch.full((1, 8 * 128), NAN, device="cuda").bfloat16())) for _ in "kv")
    before = {which: getattr(c, which).clone() for which in ("keys", "values")}
    c.rows = own + behind
    args = c.tables, c.device(c.lengths), 8, 128, 16, c.pages, c.most, 2
    l2c.cache_append(c.keys, c.values, k, v, *args, rows=c.rows, starts=c.device(c.starts), key_scales=c.key_scales,
                     value_scales=c.value_scales)
    torch.cuda.synchronize()
    got = {which: getattr(c, which).clone() for which in ("keys", "values")}
    for which in got:
        getattr(c, which).copy_(before[which])
    c.rows = own
    check(l2c, c, k=k[:own], v=v[:own])
    for which, x in got.items():
        assert torch.equal(x.view(torch.uint8), getattr(c, which).view(torch.uint8))


def test_rows_before_the_sequences(torch_gpu, l2c):
    """The first sequence's rows need not be the call's first."""
    c = Cache(1, [20, 9], [6, 9], 2, 64, 16)
    k, v = fused(c.rows, 2 * 64, c.gen), fused(c.rows, 2 * 64, c.gen)
    before = c.keys.clone()
    args = c.tables, c.device(c.lengths), 2, 64, 16, c.pages, c.most, 2
    ahead = torch.full((5, 2 * 64), NAN, device="cuda").bfloat16()
    l2c.cache_append(c.keys, c.values, torch.cat((ahead, k)), torch.cat((ahead, v)), *args, rows=c.rows + 8,
                     starts=c.device([s + 5 for s in c.starts]))
    torch.cuda.synchronize()
    got = c.keys.clone()
    c.keys.copy_(before)
    check(l2c, c, k=k, v=v)
    assert torch.equal(got.view(torch.int16), c.keys.view(torch.int16))
