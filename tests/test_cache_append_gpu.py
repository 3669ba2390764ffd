"""l2c_cache_append: bf16 rows as they are, e4m3 rows as l2c_quantize_fp8 leaves them, bit for bit; everything
else as it was."""
import math

import pytest
import torch
from paged import Cache, fused

pytestmark = pytest.mark.gpu


def check(l2c, c, starts=True, spare=0, k=None, v=None, stream=None):
    width = c.kv * c.width
    print(f"case append lengths={c.lengths[:6]} new={c.new[:6]} kv={c.kv} width={c.width} page={c.page} {c.kind}", flush=True)
    k = fused(c.rows, width, c.gen, spare) if k is None else k
    v = fused(c.rows, width, c.gen, 2 * spare) if v is None else v
    keep = {n: getattr(c, n).clone() for n in ("keys", "values") + (("key_scales", "value_scales") if c.key_scales is not None else ())}
    l2c.cache_append(c.keys, c.values, k, v, c.tables, c.device(c.lengths), c.kv, c.width, c.page, c.pages, c.most,
                     len(c.lengths), rows=c.rows, starts=c.device(c.starts) if starts else None, key_scales=c.key_scales,
                     value_scales=c.value_scales, k_stride=k.stride(0), v_stride=v.stride(0), stream=stream)
    torch.cuda.synchronize()
    for which, x in (("keys", k), ("values", v)):
        rows = x.float().reshape(c.rows, c.kv, c.width) if x.is_contiguous() else x.float().reshape(-1, c.kv, c.width)
        if c.kind == "e4m3":
            codes = torch.empty(c.rows * c.kv, c.width, device="cuda", dtype=torch.uint8)
            scales = torch.empty(c.rows * c.kv, device="cuda")
            finite = rows.isfinite().all(-1)
            l2c.quantize_fp8(codes, scales, torch.where(finite.unsqueeze(-1), rows, 0.0).contiguous(), c.rows * c.kv, c.width)
            codes, scales = codes.reshape(rows.shape), scales.reshape(rows.shape[:2])
            codes[~finite], scales[~finite] = 0, math.nan
        for s, n in enumerate(c.new):
            for i in range(n):
                p, row = c.lengths[s] - n + i, c.starts[s] + i
                if p < 0 or p >= c.most * c.page or not 0 <= int(c.tables[s, p // c.page]) < c.pages:
                    continue
                at = int(c.tables[s, p // c.page]), slice(None), p % c.page
                if c.kind == "bf16":
                    keep[which][at] = x[row].reshape(c.kv, c.width)
                else:
                    keep[which][at] = codes[row]
                    keep[which[:-1] + "_scales"][at] = scales[row]
    for name, want in keep.items():
        got = getattr(c, name)
        bits = torch.int16 if got.dtype is torch.bfloat16 else torch.int32 if got.dtype is torch.float32 else torch.uint8
        if got.dtype is torch.float32:
            assert torch.equal(got.isnan(), want.isnan())
            got, want = got.nan_to_num(), want.nan_to_num()
        assert torch.equal(got.view(bits), want.view(bits)), name


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("width", [8, 16, 24, 64, 80, 128, 200, 256])
@pytest.mark.parametrize("kv", [1, 3, 8])
def test_rows(torch_gpu, l2c, kv, width, cache):
    check(l2c, Cache(width + kv, [30, 1, 17], [14, 1, 9], kv, width, 16, cache, rows_behind=2), spare=16)
    check(l2c, Cache(width + kv, [30, 1, 17], [1, 1, 1], kv, width, 16, cache), starts=False)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [1, 5, 16, 48])
def test_places_that_are_not_there(torch_gpu, l2c, page, cache):
    """Tokens before the first position, past the tables, and on entries that are no pages are not written."""
    c = Cache(page, [40, 3, 25, 0, -2], [12, 9, 25, 4, 1], 2, 64, page, cache, spare_columns=0)
    c.tables[0, 39 // page] = -1
    c.tables[2, 0], c.tables[2, 20 // page] = c.pages, 2 ** 31 - 1
    c.lengths[0] += 5
    check(l2c, c)


def test_values_at_the_ends_of_the_range(torch_gpu, l2c):
    """Ties, subnormal codes, zeros of both signs, rows of 0, the smallest and largest numbers, Inf and NaN."""
    c = Cache(1, [9], [9], 2, 64, 16, "e4m3")
    x = torch.zeros(9, 2, 64, device="cuda")
    x[0] = torch.linspace(-448, 448, 64, device="cuda")
    x[1, :, 0], x[1, :, 1:] = 448, torch.arange(63, device="cuda") * 2.0 ** -10
    x[2] = -0.0
    x[3, :, 0], x[3, :, 1] = 3.0e38, -2.0 ** -126
    x[4, :, 0], x[4, :, 1] = 1e-38, -9e-41
    x[5, :, 3], x[6, :, 4], x[7, 0, 5] = math.inf, math.nan, -math.inf
    x[8] = torch.randn(2, 64, generator=c.gen, device="cuda") * 1e-30
    x = x.bfloat16().reshape(9, 128)
    check(l2c, c, k=x, v=x.flip(0).contiguous())


def test_another_stream(torch_gpu, l2c):
    c = Cache(2, [200, 40], [100, 40], 4, 128, 16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    check(l2c, c, stream=stream)


def test_offsets_past_31_bits(torch_gpu, l2c):
    kv, width, page, pages = 8, 128, 64, 40000
    keys = torch.zeros(pages, kv, page, width, device="cuda", dtype=torch.bfloat16)
    values = torch.zeros_like(keys)
    tables = torch.tensor([[39999, 39990]], device="cuda", dtype=torch.int32)
    k = torch.randn(100, kv * width, device="cuda").bfloat16()
    lengths, starts = (torch.tensor(x, device="cuda", dtype=torch.int32) for x in ([100], [0, 100]))
    l2c.cache_append(keys, values, k, -k, tables, lengths, kv, width, page, pages, 2, 1, rows=100, starts=starts)
    want = k.reshape(100, kv, width).transpose(0, 1)
    for cache, sign in ((keys, 1), (values, -1)):
        assert torch.equal(cache[39999], sign * want[:, :64]) and torch.equal(cache[39990, :, :36], sign * want[:, 64:])
        assert int(cache[39990, :, 36:].count_nonzero()) == 0 and int(cache[:39990].count_nonzero()) == 0
