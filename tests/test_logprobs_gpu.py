"""l2c_decoder_logprobs against the formulas in 64 bits.

With d the mean distance of a row's logits from the largest, weighed by their probabilities (the distance is at
least 0): an exponential is off by at most 2^-22 of it, and one of a distance t by what the fp32 product t log2(e)
leaves, which the kernel corrects or the library does; 32 of them added in fp32 2^-19 of the sum, so log Z is off by
2^-19 + 2^-22 =: e. The entropy is log Z + d: d is off by e d for its sums, twice. All is rounded once, 2^-24 of it."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -19 + 2.0 ** -22
NEG = -math.inf


def want_of(x, tokens, top):
    """x: float32 [rows][vocab] on the GPU. The order of the alternatives is exact."""
    rows, vocab = x.shape
    y = x.double()
    m = y.amax(1, keepdim=True)
    bad = (y.isnan().any(1)) | (y == math.inf).any(1) | (y == NEG).all(1)
    away = torch.where(y == NEG, 0.0, y - m)
    w = torch.where(y == NEG, 0.0, away.exp())
    z = w.sum(1, keepdim=True)
    d = -(w * away).sum(1) / z.squeeze(1)
    lp = torch.where(y == NEG, NEG, y - m) - z.log()
    order = torch.sort(torch.where(y.isnan(), NEG, y), dim=1, descending=True, stable=True).indices[:, :top]
    alt = torch.full((rows, top), NEG, device="cuda", dtype=torch.float64)
    which = torch.full((rows, top), -1, device="cuda", dtype=torch.long)
    n = order.shape[1]
    alt[:, :n] = lp.gather(1, order)
    which[:, :n] = torch.where(alt[:, :n] > NEG, order, -1)
    inside = (tokens >= 0) & (tokens < vocab)
    mine = torch.where(inside, lp.gather(1, tokens.clamp(0, vocab - 1).long().unsqueeze(1)).squeeze(1), math.nan)
    entropy = z.log().squeeze(1) + d
    mine[bad], entropy[bad], alt[bad], which[bad] = math.nan, math.nan, math.nan, -1
    return mine, entropy, which, alt, d


def close(got, want, tol):
    got = got.double()
    want = torch.where(want < -3.4028235677973366e38, NEG, want)  # what rounds to fp32's -Inf: the last half step and beyond
    assert torch.equal(got.isnan(), want.isnan())
    same = ~want.isfinite()
    assert torch.equal(got[same].nan_to_num(), want[same].nan_to_num())
    off = (got - want).abs()[~same]
    assert bool((off <= (tol + want.abs() * 2.0 ** -24)[~same]).all()), off.max()


def check(l2c, x, top, tokens=None, offset=0, stream=None, fill=0xff):
    rows, vocab = x.shape
    print(f"case logprobs {rows}x{vocab} top={top}", flush=True)
    buf = torch.empty(rows * vocab + 8, device="cuda")
    logits = buf[offset:offset + rows * vocab].view(rows, vocab)
    logits.copy_(x)
    gen = torch.Generator("cuda").manual_seed(rows + vocab)
    if tokens is None:
        tokens = torch.randint(vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    size = l2c.decoder_logprobs_workspace_bytes(vocab, top, rows)
    assert size <= rows * -(-vocab // 1024) * (8 * top + 32)
    ws = torch.full((size + 64,), fill, device="cuda", dtype=torch.uint8)
    lp, en = (torch.full((rows + 1,), 7.0, device="cuda") for _ in range(2))
    tt = torch.full((rows * top + 1,), 7, device="cuda", dtype=torch.int32)
    tl = torch.full((rows * top + 1,), 7.0, device="cuda")
    if stream:
        stream.wait_stream(torch.cuda.current_stream())
    l2c.decoder_logprobs(lp, en, tt, tl, logits, tokens, vocab, top, rows, ws[:size], stream=stream)
    torch.cuda.synchronize()
    assert bool((ws[size:] == fill).all()) and lp[rows] == en[rows] == tt[-1] == tl[-1] == 7
    mine, entropy, which, alt, d = want_of(logits, tokens, top)
    assert torch.equal(tt[:-1].view(rows, top).long(), which)
    close(lp[:rows], mine, E)
    close(en[:rows], entropy, E + 2 * E * d)
    close(tl[:-1].view(rows, top), alt, E)
    return lp[:rows], en[:rows], tt[:-1], tl[:-1]


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 31, 63, 64, 65, 255, 257, 1000, 1023, 1024, 1025, 2047, 2048, 2049, 4099,
                                   8191, 8192, 8193, 16389, 32768, 40001])
@pytest.mark.parametrize("top", [0, 1, 4, 5, 20, 32])
def test_vocabularies(torch_gpu, l2c, vocab, top):
    gen = torch.Generator("cuda").manual_seed(vocab)
    check(l2c, 3 * torch.randn(3, vocab, generator=gen, device="cuda"), top)


@pytest.mark.parametrize("rows,vocab,top", [(1, 32000, 5), (1, 131072, 32), (7, 131075, 0), (300, 5003, 8), (2000, 2050, 3),
                                            (64, 32003, 32), (1, 300001, 10), (1100, 9001, 17), (5000, 40, 2),
                                            (2, 2000003, 32)])
def test_batches(torch_gpu, l2c, rows, vocab, top):
    gen = torch.Generator("cuda").manual_seed(rows)
    check(l2c, 3 * torch.randn(rows, vocab, generator=gen, device="cuda"), top, offset=rows % 4)


@pytest.mark.parametrize("vocab", [40, 3000, 40000, 140000])
@pytest.mark.parametrize("top", [1, 7, 32])
def test_ties(torch_gpu, l2c, vocab, top):
    """Few values, one value, zeros of both signs: the lower token first."""
    gen = torch.Generator("cuda").manual_seed(vocab)
    x = torch.randint(3, (5, vocab), generator=gen, device="cuda").float()
    x[1] = -2.5
    x[2] = torch.where(torch.rand(vocab, generator=gen, device="cuda") < 0.5, -0.0, 0.0)
    x[3] = torch.arange(vocab, device="cuda").float()
    x[4] = -x[3]
    check(l2c, x, top)


@pytest.mark.parametrize("vocab", [3, 50, 2500, 33000, 140000])
@pytest.mark.parametrize("top", [0, 2, 32])
def test_infinities_and_nan(torch_gpu, l2c, vocab, top):
    gen = torch.Generator("cuda").manual_seed(vocab)
    x = 3 * torch.randn(9, vocab, generator=gen, device="cuda")
    x[0] = NEG
    x[1, vocab // 2] = math.nan
    x[2, vocab - 1] = math.inf
    x[3, 1:] = NEG                     # one token
    x[4, torch.rand(vocab, generator=gen, device="cuda") < 0.9] = NEG
    x[4, 0] = 1.0
    x[5] = math.nan
    x[6, 0], x[6, 1:] = 3e38, -3e38    # distances past the largest number
    x[7] = -3.4028234663852886e38      # the lowest value everywhere
    x[8, ::2] = -3.4028234663852886e38
    tokens = torch.tensor([0, 0, 0, vocab - 1, 0, 0, vocab - 1, 1, 1], device="cuda", dtype=torch.int32)
    check(l2c, x, top, tokens)


def test_tokens_outside(torch_gpu, l2c):
    x = torch.randn(5, 100, device="cuda")
    tokens = torch.tensor([-1, 100, 2 ** 31 - 1, -2 ** 31, 99], device="cuda", dtype=torch.int32)
    lp, *_ = check(l2c, x, 2, tokens)
    assert lp.isnan().tolist() == [True] * 4 + [False]


def test_certain_and_even(torch_gpu, l2c):
    """Entropy 0 of one token, log(n) of n equal ones; steep rows."""
    x = torch.full((3, 4096), NEG, device="cuda")
    x[0, 17] = 5.0
    x[1] = 1.0
    x[2] = -torch.arange(4096, device="cuda").float() * 10
    lp, en, *_ = check(l2c, x, 3, torch.tensor([17, 3, 0], device="cuda", dtype=torch.int32))
    assert en[0] == 0 and lp[0] == 0 and abs(float(en[1]) - math.log(4096)) < 1e-5


def test_parts_alone(torch_gpu, l2c):
    x = 3 * torch.randn(4, 5000, device="cuda")
    tokens = torch.arange(4, device="cuda", dtype=torch.int32)
    lp, en, tt, tl = check(l2c, x, 6, tokens)
    ws = torch.empty(l2c.decoder_logprobs_workspace_bytes(5000, 6, 4), device="cuda", dtype=torch.uint8)
    a, b = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    l2c.decoder_logprobs(None, a, None, None, x, None, 5000, 0, 4, ws)
    l2c.decoder_logprobs(b, None, None, None, x, tokens, 5000, 0, 4, ws)
    assert torch.equal(a, en) and torch.equal(b, lp)
    t, l = torch.zeros_like(tt), torch.zeros_like(tl)
    l2c.decoder_logprobs(None, None, t, l, x, None, 5000, 6, 4, ws)
    assert torch.equal(t, tt) and torch.equal(l, tl)


def test_rows_past_31_bits(torch_gpu, l2c):
    rows, vocab = 66000, 33000
    x = torch.randn(rows, vocab, device="cuda")
    tokens = torch.full((rows,), 7, device="cuda", dtype=torch.int32)
    lp, en = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    tt, tl = torch.zeros(rows, 2, device="cuda", dtype=torch.int32), torch.zeros(rows, 2, device="cuda")
    ws = torch.empty(l2c.decoder_logprobs_workspace_bytes(vocab, 2, rows), device="cuda", dtype=torch.uint8)
    l2c.decoder_logprobs(lp, en, tt, tl, x, tokens, vocab, 2, rows, ws)
    torch.cuda.synchronize()
    at = [0, 40000, 65080, 65999]
    mine, entropy, which, alt, d = want_of(x[at], tokens[at], 2)
    assert torch.equal(tt[at].long(), which)
    close(lp[at], mine, E), close(en[at], entropy, E + 2 * E * d), close(tl[at], alt, E)


def test_captured_on_another_stream(torch_gpu, l2c):
    gen = torch.Generator("cuda").manual_seed(1)
    rows, vocab, top = 3, 40000, 9
    xs = [3 * torch.randn(rows, vocab, generator=gen, device="cuda") for _ in range(2)]
    tokens = torch.tensor([1, 2, 39999], device="cuda", dtype=torch.int32)
    want = [check(l2c, x, top, tokens, stream=torch.cuda.Stream()) for x in xs]
    ws = torch.empty(l2c.decoder_logprobs_workspace_bytes(vocab, top, rows), device="cuda", dtype=torch.uint8)
    x = xs[0].clone()
    out = [torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"),
           torch.zeros(rows * top, device="cuda", dtype=torch.int32), torch.zeros(rows * top, device="cuda")]

    def run():
        l2c.decoder_logprobs(*out, x, tokens, vocab, top, rows, ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(4):
        x.copy_(xs[i % 2])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 2]))
        check(l2c, xs[1 - i % 2], top, tokens)
