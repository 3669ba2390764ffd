"""l2c_cache_attention against the formula in 64 bits (tests/paged.py derives the tolerance). Places that no
position has, and pages of nobody, hold NaN, so that whatever is read past an end shows."""
import math

import pytest
import torch
from paged import NAN, Cache, attend, fused

pytestmark = pytest.mark.gpu


def call(l2c, c, q, heads, window=0, scale=None, out=None, starts=True, workspace=None, stream=None, tables=None):
    width = heads * c.width
    if out is None:
        out = torch.full((c.rows, width), 7.0, device="cuda", dtype=torch.bfloat16)
    if workspace is None:
        size = l2c.cache_attention_workspace_bytes(len(c.lengths), c.rows, heads, c.kv, c.width, c.page, c.most)
        assert size <= (c.width + 2) << 19
        workspace = torch.full((size + 64,), 0xff, device="cuda", dtype=torch.uint8)
    l2c.cache_attention(out, q, c.keys, c.values, c.tables if tables is None else tables, c.device(c.lengths), heads, c.kv,
                        c.width, c.page, c.pages, c.most, len(c.lengths), workspace[:workspace.numel() - 64],
                        rows=c.rows, starts=c.device(c.starts) if starts else None, key_scales=c.key_scales,
                        value_scales=c.value_scales, window=window, scale=scale, q_stride=q.stride(0),
                        out_stride=out.stride(0), stream=stream)
    torch.cuda.synchronize()
    assert bool((workspace[workspace.numel() - 64:] == 0xff).all())
    return out


def check(l2c, c, heads, window=0, scale=None, spare=0, no_page=(), q=None, **more):
    print(f"case attention lengths={c.lengths[:6]} new={c.new[:6]} heads={heads}/{c.kv} width={c.width} page={c.page} "
          f"{c.kind} window={window}", flush=True)
    if q is None:
        q = fused(c.rows, heads * c.width, c.gen, spare)
    out = call(l2c, c, q, heads, window, scale, **more)
    want, tol = attend(c, q, heads, window, scale, no_page)
    got = out[:, :heads * c.width].double().reshape(want.shape)
    last = c.starts[-1]
    assert bool((got[last:] == 7).all())  # rows of no sequence
    got, want, tol = got[:last], want[:last], tol[:last]
    assert torch.equal(got.isnan(), want.isnan())
    fine = want.isfinite()
    assert torch.equal(got[~fine].nan_to_num(), want[~fine].nan_to_num())
    assert bool(((got - want).abs() <= tol)[fine].all()), ((got - want).abs() / tol)[fine].max()
    return out


# Lengths at the edges of tiles of 16 to 128 and of pages, one token each.
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (8, 2), (32, 8), (5, 1), (16, 1), (33, 1)])
def test_one_token(torch_gpu, l2c, heads, kv, cache):
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257]
    c = Cache(heads * 100 + kv, lengths, [1] * len(lengths), kv, 64, 16, cache)
    a = check(l2c, c, heads, starts=False)
    b = check(l2c, c, heads, starts=True)
    assert a.shape == b.shape


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("width", [8, 16, 24, 40, 64, 72, 80, 96, 120, 128, 136, 192, 248, 256])
def test_widths(torch_gpu, l2c, width, cache):
    lengths, new = [70, 5, 140], [3, 5, 70]
    check(l2c, Cache(width, lengths, new, 2, width, 16, cache), 6, spare=16)
    check(l2c, Cache(width, lengths, [1, 1, 1], 2, width, 16, cache), 6, spare=8)


@pytest.mark.parametrize("new", [1, 7, 100])
@pytest.mark.parametrize("page", [1, 3, 16, 20, 48, 64, 100, 128, 1000])
def test_page_sizes(torch_gpu, l2c, page, new):
    lengths = [max(new, n) for n in (page, page + 1, max(1, page - 1), 3 * page, 211)]
    check(l2c, Cache(page + new, lengths, [new] * 5, 2, 128, page), 8)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("new", [[2, 3, 5], [1, 0, 4], [0, 0, 9], [16, 17, 15], [33, 1, 64], [127, 128, 129], [1, 300, 2],
                                 [0, 0, 0]], ids=str)
@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 1), (6, 2)])
def test_chunks(torch_gpu, l2c, new, heads, kv, cache):
    lengths = [n + more for n, more in zip(new, (0, 37, 200))]
    check(l2c, Cache(sum(new) + heads, lengths, new, kv, 64, 16, cache, rows_behind=5), heads)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 64, 65, 130, 10000])
@pytest.mark.parametrize("new", [1, 6, 90, 300])
def test_windows(torch_gpu, l2c, window, new):
    lengths = [new, new + 1, new + 63, new + 400]
    check(l2c, Cache(window + new, lengths, [new] * 4, 2, 64, 16), 8, window=window)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("width", [64, 136, 256])
@pytest.mark.parametrize("window", [0, 300, 700, 3001])
@pytest.mark.parametrize("new", [[1, 1], [5, 7], [6, 20], [150, 10], [600, 500]], ids=str)
def test_parts_of_long_sequences(torch_gpu, l2c, new, window, width, cache):
    """Tiles of every kind, divided where a window leaves enough of their positions."""
    check(l2c, Cache(sum(new) + width, [5000, 2300], new, 2, width, 16, cache), 8, window=window)


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("new", [1, 9, 200])
def test_pages_that_are_not_there(torch_gpu, l2c, new, page):
    """Entries of -1 and past the last page: their positions are passed over; rows with nothing left are 0."""
    lengths = [new + 5, new + 160, new + 333]
    c = Cache(new + page, lengths, [new] * 3, 2, 64, page)
    none = [(0, i) for i in range(c.most)] + [(1, 0), (1, 3), (2, 1), (2, (lengths[2] - 1) // page)]
    for i, (s, column) in enumerate(none):
        c.tables[s, column] = (-1, c.pages, -2 ** 31, 2 ** 31 - 1)[i % 4]
    out = check(l2c, c, 4, no_page=none)
    assert bool((out[:new] == 0).all())


def test_tokens_before_the_first_position(torch_gpu, l2c):
    """More new tokens than positions, lengths of 0 and below: rows without a position are 0."""
    c = Cache(5, [3, 0, -4, 2, 20], [7, 2, 3, 1, 20], 2, 64, 16)
    out = check(l2c, c, 8)
    assert bool((out[:4] == 0).all()) and bool((out[7:12] == 0).all())
    c = Cache(6, [0, 4, -1], [1, 1, 1], 2, 64, 16)
    out = check(l2c, c, 8, starts=False)
    assert bool((out[0] == 0).all()) and bool((out[2] == 0).all())


@pytest.mark.parametrize("new", [1, 40])
def test_lengths_past_the_tables(torch_gpu, l2c, new):
    """Positions that the tables have no column for are passed over."""
    c = Cache(3, [64, 100], [new, new], 1, 64, 16, spare_columns=0)
    want, tol = None, None
    q = fused(c.rows, 4 * 64, c.gen)
    c.lengths = [150, 400]
    c.dense = [[torch.cat((x, torch.zeros(1, n - x.shape[1], 64, device="cuda", dtype=torch.float64)), 1) for x in d]
               for d, n in zip(c.dense, c.lengths)]
    c.tables[0, 4:] = -1
    cut = [(0, i) for i in range(4, 30)] + [(1, i) for i in range(7, 30)]
    c.dense[1][0][:, 100:] = 0
    # Row 100 to 111 of the last page are there, and poisoned: make them values.
    zeros = torch.zeros(12, 1, 64, device="cuda")
    c.put(1, 100, "keys", zeros), c.put(1, 100, "values", zeros)
    check(l2c, c, 4, no_page=cut, q=q)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
@pytest.mark.parametrize("new,window", [(1, 0), (5, 0), (5, 20), (64, 0), (200, 50), (200, 0)])
def test_masked_places_hold_anything(torch_gpu, l2c, new, window, bad, cache):
    """Keys and values that some tokens see and others do not: each shows in the rows that see it, and only there."""
    length = new + 70
    c = Cache(new + window, [length, length + 9], [new, new], 2, 64, 16, cache)
    for at in {length - 1, length - max(1, new // 2), length - new, 3}:
        for which, i in (("keys", 0), ("values", 1)):
            row = torch.zeros(1, 2, 64, device="cuda")
            if cache == "e4m3":
                page, slot = c.place(0, at, 1)
                getattr(c, which[:-1] + "_scales")[page, :, slot] = bad
                getattr(c, which)[page, :, slot] = torch.ones(1, 2, 64, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8)
                c.dense[0][i][:, at] = bad
            elif which == "values":
                row[:, :, 5::7] = bad
                c.dense[0][1][:, at] = c.put(0, at, which, row)[:, 0]
    if cache == "e4m3":  # the keys' scales decide alone: only NaN has a score of its own, which is NaN
        if not math.isnan(bad):
            for at in {length - 1, length - max(1, new // 2), length - new, 3}:
                c.dense[0][0][:, at] = c.put(0, at, "keys", torch.zeros(1, 2, 64, device="cuda"))[:, 0]
    check(l2c, c, 4, window=window)


def test_keys_of_nan_in_masked_places(torch_gpu, l2c):
    for new in (1, 40, 150):
        c = Cache(new, [new + 40], [new], 1, 64, 16)
        at = new + 40 - max(1, new // 3)
        c.dense[0][0][:, at] = c.put(0, at, "keys", torch.full((1, 1, 64), NAN, device="cuda"))[:, 0]
        check(l2c, c, 4)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("new,window", [(1, 0), (1, 37), (3, 9), (30, 0), (30, 21), (150, 77)])
def test_what_nobody_sees_leaves_no_trace(torch_gpu, l2c, new, window, cache):
    """Rows of pages without a position, and positions behind the window: the same bits whatever they hold."""
    bits = []
    for poison in (0.0, NAN, 1.0e30, math.inf):
        c = Cache(new + window, [new + 50, new + 7], [new, new], 2, 64, 16, cache, poison=poison)
        q = fused(c.rows, 8 * 64, c.gen)
        if window:
            for s, length in enumerate(c.lengths):
                behind = length - new - window + 1
                if behind > 0:
                    page, slot = c.place(s, 0, behind)
                    for which in ("keys", "values"):
                        getattr(c, which)[page, :, slot] = poison if cache == "bf16" else 0x7f
                        if cache == "e4m3":
                            getattr(c, which[:-1] + "_scales")[page, :, slot] = poison
        bits.append(call(l2c, c, q, 8, window).view(torch.int16))
        assert all(torch.equal(bits[0], b) for b in bits)


@pytest.mark.parametrize("new", [1, 20])
def test_scores_of_minus_infinity(torch_gpu, l2c, new):
    """Keys whose score is -Inf weigh nothing; a row with no other is 0."""
    c = Cache(9, [new + 30, new + 3], [new, new], 1, 64, 16)
    q = torch.ones(c.rows, 4 * 64, device="cuda").bfloat16()
    low = torch.full((1, 1, 64), 0.0, device="cuda")
    low[..., 0] = -math.inf
    for s, positions in ((0, (0, 5, new + 10)), (1, range(new + 3))):
        for at in positions:
            c.dense[s][0][:, at] = c.put(s, at, "keys", low)[:, 0]
    out = check(l2c, c, 4, q=q)
    assert bool((out[new:] == 0).all())


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 30.0])
@pytest.mark.parametrize("new", [1, 30])
def test_scales(torch_gpu, l2c, new, scale):
    check(l2c, Cache(4, [200, 31], [new, new], 2, 64, 16), 8, scale=scale)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 200, 2 ** 30])
@pytest.mark.parametrize("new", [1, 5, 300])
def test_windows_past_everything(torch_gpu, l2c, new, window):
    check(l2c, Cache(new, [new + 350, new, 1], [new, new, 1], 2, 64, 16), 8, window=window)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("length,new", [(3000, 1), (3000, 4), (900, 600)])
def test_large_values(torch_gpu, l2c, length, new, cache):
    """Values as large as `length` of them may be, 2^128 / length, and scores that grow from tile to tile: weights are
    never above 1, so their sums do not overflow."""
    c = Cache(length, [length], [new], 1, 64, 16, cache, spread=0.0)
    q = torch.ones(c.rows, 2 * 64, device="cuda").bfloat16()
    j = torch.arange(length, device="cuda").float().reshape(-1, 1, 1)
    c.dense[0][0] = c.put(0, 0, "keys", (j * (8.0 / length)).floor().expand(-1, 1, 64).contiguous() / 8)
    c.dense[0][1] = c.put(0, 0, "values", torch.full((length, 1, 64), 1e35, device="cuda"))
    out = check(l2c, c, 2, q=q)
    assert bool(out.isfinite().all())


def peaked(c, q, heads, at):
    """Keys along the first query row of head 0 at the given positions of sequence 0: they share the weight."""
    k = torch.zeros(1, c.kv, c.width, device="cuda")
    row = q[c.starts[1] - 1].float().reshape(heads, c.width)[::heads // c.kv]
    for j in at:
        k[0] = row * (12.0 * c.width ** 0.5) / (row * row).sum(-1, keepdim=True)
        c.dense[0][0][:, j] = c.put(0, j, "keys", k)[:, 0]


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("length,new,page,heads,kv,width", [
    (70000, 1, 16, 8, 2, 128), (70001, 1, 64, 4, 4, 64), (30011, 3, 32, 8, 1, 128), (5003, 1000, 16, 4, 1, 64),
    (9999, 77, 128, 6, 2, 256), (20000, 16, 48, 10, 10, 80)])
def test_long(torch_gpu, l2c, length, new, page, heads, kv, width, cache):
    """Few positions share the weight, at the ends of tiles, pages and of what the splits may be: each counts."""
    c = Cache(length, [length, 40, length // 3], [new, 1, min(new, 5)], kv, width, page, cache, spread=0.1)
    q = fused(c.rows, heads * width, c.gen)
    last = length - 1
    peaked(c, q, heads, [0, 1, page - 1, page, 127, 128, 255, 256, 1023, 1024, last // 2, last - 64, last - 1, last])
    check(l2c, c, heads, q=q)
    check(l2c, c, heads, q=q, window=length // 2 + 3)


def test_offsets_past_31_bits(torch_gpu, l2c):
    """Pages beyond 2^31 values and 2^32 bytes."""
    kv, width, page = 8, 128, 64
    pages = 40000  # 2.6e9 values, 5.2 GB each
    keys = torch.zeros(pages, kv, page, width, device="cuda", dtype=torch.bfloat16)
    values = torch.zeros_like(keys)
    c = Cache(1, [300, 129], [9, 1], kv, width, page)
    high = torch.arange(pages - c.pages, pages, device="cuda")
    keys[high], values[high] = c.keys, c.values
    c.keys, c.values, c.pages = keys, values, pages
    c.tables = torch.where(c.tables >= 0, c.tables + int(high[0]), -1).int()
    check(l2c, c, 16)


@pytest.mark.parametrize("new", [1, 200])
def test_many_sequences(torch_gpu, l2c, new):
    lengths = [(i * 37) % 90 + new for i in range(300)]
    check(l2c, Cache(2, lengths, [new - i % min(new, 3) for i in range(300)] if new > 1 else [1] * 300, 1, 64, 16), 4)


def test_strides_and_streams(torch_gpu, l2c):
    c = Cache(8, [100, 33, 64], [20, 1, 40], 2, 64, 16)
    stream = torch.cuda.Stream()
    wide = torch.full((c.rows, 8 * 64 + 24), 7.0, device="cuda", dtype=torch.bfloat16)
    stream.wait_stream(torch.cuda.current_stream())
    check(l2c, c, 8, spare=40, out=wide, stream=stream)
    assert bool((wide[:, 8 * 64:] == 7).all())


@pytest.mark.parametrize("new", [1, 5, 150])
def test_repeated_and_captured(torch_gpu, l2c, new):
    """Equal bits on every call; a graph of it replayed over other lengths, tables and inputs, with eager calls on the
    same workspace between the replays."""
    c = Cache(new, [3000, 40 + new, 700 + new], [new] * 3, 2, 128, 16)
    d = Cache(new + 1, [new, 3000, 11 + new], [new] * 3, 2, 128, 16)
    d.most, d.pages = c.most, c.pages
    assert d.tables.shape[1] <= c.most and d.keys.shape[0] <= c.pages
    heads = 8
    size = l2c.cache_attention_workspace_bytes(3, c.rows, heads, 2, 128, 16, c.most)
    ws = torch.full((size + 64,), 0xff, device="cuda", dtype=torch.uint8)
    qs = [fused(c.rows, heads * 128, x.gen) for x in (c, d)]
    grown = torch.full_like(c.tables, -1)
    grown[:, :d.tables.shape[1]] = d.tables
    d.tables = grown
    for name in ("keys", "values"):
        big = torch.full_like(getattr(c, name), NAN)
        big[:getattr(d, name).shape[0]] = getattr(d, name)
        setattr(d, name, big)
    want = [call(l2c, x, q, heads, workspace=ws) for x, q in zip((c, d), qs)]
    state = [t.clone() for t in (qs[0], c.keys, c.values, c.tables, c.device(c.lengths), c.device(c.starts))]
    out = torch.zeros_like(want[0])

    def run():
        q, keys, values, tables, lengths, starts = state
        l2c.cache_attention(out, q, keys, values, tables, lengths, heads, 2, 128, 16, c.pages, c.most, 3, ws[:size],
                            rows=c.rows, starts=starts)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(4):
        x, q = (c, d)[i % 2], qs[i % 2]
        for to, of in zip(state, (q, x.keys, x.values, x.tables, x.device(x.lengths), x.device(x.starts))):
            to.copy_(of)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want[i % 2].view(torch.int16))
        again = call(l2c, (d, c)[i % 2], qs[1 - i % 2], heads, workspace=ws)
        assert torch.equal(again.view(torch.int16), want[1 - i % 2].view(torch.int16))


# Chunks long enough, over heads enough, for tiles of 256 rows (64 key heads, and 2048 rows for each).
@pytest.mark.parametrize("width,page,window", [(64, 16, 0), (128, 16, 0), (80, 48, 0), (96, 5, 0), (128, 64, 130), (40, 16, 1),
                                               (120, 16, 1000)])
def test_many_rows_and_heads(torch_gpu, l2c, width, page, window):
    lengths, new = [1500, 700, 3, 90, 1333], [1400, 650, 0, 90, 1]
    c = Cache(width + window, lengths, new, 64, width, page, rows_behind=3)
    q = fused(c.rows, 64 * width, c.gen, 8)
    peaked(c, q, 64, [0, 1, 63, 64, 65, 127, 128, 700, 1435, 1436, 1498, 1499])
    check(l2c, c, 64, window=window, q=q)


@pytest.mark.parametrize("width,page,window", [(128, 16, 0), (104, 20, 300)])
def test_many_rows_of_e4m3(torch_gpu, l2c, width, page, window):
    lengths, new = [1500, 3, 900], [1400, 1, 850]
    c = Cache(width, lengths, new, 64, width, page, "e4m3")
    q = fused(c.rows, 64 * width, c.gen)
    peaked(c, q, 64, [0, 63, 64, 700, 1499])
    check(l2c, c, 64, window=window, q=q)


@pytest.mark.parametrize("scale", [None, -0.7, 0.0])
def test_many_rows_of_shared_heads(torch_gpu, l2c, scale):
    c = Cache(3, [800, 1111], [260, 777], 31, 64, 16)
    check(l2c, c, 31 * 4, scale=scale)


@pytest.mark.parametrize("bad", [NAN, math.inf])
def test_many_rows_over_masked_places(torch_gpu, l2c, bad):
    """Values that are not finite where some rows of a tile see them; pages that are not there; -Inf scores."""
    c = Cache(4, [2200, 300], [2000, 100], 64, 64, 16)
    for at in (2199, 1700, 201, 5):
        row = torch.zeros(1, 64, 64, device="cuda")
        row[:, 3, 5::7] = bad
        c.dense[0][1][:, at] = c.put(0, at, "values", row)[:, 0]
    none = [(0, 0), (0, 3), (0, 77), (1, 2)] + [(0, i) for i in range(100, 109)]
    for s, column in none:
        c.tables[s, column] = -1
    check(l2c, c, 64, no_page=none)
    check(l2c, c, 64, no_page=none, window=90)
