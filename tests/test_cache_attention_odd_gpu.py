"""l2c_cache_attention over values that are not finite where some rows of a tile see them and others do not: they show in
the rows that see them, in their columns, and nowhere else, and the call takes about as long as without them."""
import math

import pytest
import torch
from paged import E4M3, NAN, Cache, fused
from test_cache_attention_gpu import call, check

pytestmark = pytest.mark.gpu


def spoil(c, s, positions, bad):
    """Some columns of the values at these positions; e4m3 has no infinities: NaN codes, and a scale at the last."""
    for at in positions:
        if c.kind == "bf16":
            row = torch.randn(1, c.kv, c.width, generator=c.gen, device="cuda")
            row[:, 0, at % 3::5] = bad
            row[:, -1, -1] = -bad
            c.dense[s][1][:, at] = c.put(s, at, "values", row)[:, 0]
            continue
        page, slot = c.place(s, at, 1)
        if at == positions[-1] and not math.isnan(bad):
            c.values[page, :, slot] = torch.full((1, c.kv, c.width), -2.0, device="cuda").to(E4M3).view(torch.uint8)
            c.value_scales[page, :, slot] = bad
            c.dense[s][1][:, at] = -bad
        else:
            codes = c.values[page, :, slot]
            codes[..., at % 3::5] = 0x7f
            c.values[page, :, slot] = codes
            c.dense[s][1][:, at, at % 3::5] = NAN


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("bad", [NAN, math.inf])
@pytest.mark.parametrize("width", [8, 64, 72, 128, 256])
@pytest.mark.parametrize("new,window,scale", [(4, 0, None), (5, 30, -0.1), (40, 0, None), (300, 0, -0.1), (300, 41, None),
                                              (200, 1, None)])
def test_rows_that_see_them(torch_gpu, l2c, new, window, scale, width, bad, cache):
    c = Cache(width + new, [new + 70, new + 9], [new, new], 2, width, 16, cache)
    for s, length in enumerate(c.lengths):
        spoil(c, s, sorted({length - new, length - 1 - new // 2, length - 3, length - 1, 2}), bad)
    check(l2c, c, 8, window=window, scale=scale)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("new", [3, 64, 256])
def test_every_value(torch_gpu, l2c, new, cache):
    """All values of a sequence, those of another as they were."""
    c = Cache(new, [new + 200, new + 77], [new, new], 1, 64, 16, cache)
    spoil(c, 0, list(range(c.lengths[0])), NAN)
    check(l2c, c, 4)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("new", [1500])
def test_tiles_of_256_rows(torch_gpu, l2c, new, cache):
    c = Cache(new, [new + 40, 90], [new, 90], 64, 104, 16, cache)
    spoil(c, 0, [30, 41, 700, 1111, new + 39], math.inf)
    q = fused(c.rows, 64 * 104, c.gen)
    check(l2c, c, 64, q=q)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("length,new", [(8192, 1024), (20000, 2)])
def test_time(torch_gpu, l2c, length, new, cache):
    """A value that is not finite costs a tile some steps, not all of its rows one by one: no more than 4 times as long."""
    c = Cache(new, [length], [new], 8, 128, 16, cache, spread=0.1)
    q = fused(c.rows, 32 * 128, c.gen)
    size = l2c.cache_attention_workspace_bytes(1, new, 32, 8, 128, 16, c.most)
    workspace = torch.empty(size + 64, device="cuda", dtype=torch.uint8).fill_(0xff)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    least = []
    for _ in range(2):
        times = []
        for _ in range(5):
            begin.record()
            call(l2c, c, q, 32, workspace=workspace)
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        least.append(min(times))
        spoil(c, 0, [length - 1 - i * (new // 7) for i in range(1 + min(new - 1, 6))], NAN)
    assert least[1] <= 4 * least[0], least
