"""How precisely l2c_cache_attention weighs values where sequences have few rows: by exponentials that are not rounded to
bf16. Every other position has score 0 and value 1, the others score s and value -1, so with w = exp(-s) the result is
(w - 1) / (w + 1), where w lies about half way between two bf16 numbers: rounded to either it is off by 2^-9.

The bound: every |value| is 1, so A of tests/paged.py is 1. The weights are held to 2^-15 of each; scores are at most
M = 0.01 and off by M (width + 4) 2^-24, exponentials by 2^-21 more, which counts twice, once in their sum; sums of n
terms n 2^-24 each; the result is rounded by 2^-8 of it."""
import math

import pytest
import torch
from paged import E4M3, NAN, Cache
from test_cache_attention_gpu import call, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("width", [64, 80, 128, 256])
@pytest.mark.parametrize("length,new,heads,kv", [(64, 1, 1, 1), (64, 1, 8, 2), (130, 3, 4, 1), (1000, 1, 16, 1),
                                                 (900, 16, 2, 2)])
@pytest.mark.parametrize("below", [2.0 ** -9 * 1.01, 3 * 2.0 ** -9 * 0.99])
def test_weights_are_not_rounded_to_bf16(torch_gpu, l2c, below, length, new, heads, kv, width, cache):
    print(f"case weights {length} new={new} heads={heads}/{kv} width={width} {cache} below={below}", flush=True)
    c = Cache(width, [length], [new], kv, width, 16, cache, spread=0.0)
    odd = (torch.arange(length, device="cuda") % 2).float().reshape(length, 1, 1)
    key = torch.zeros(length, kv, width, device="cuda")
    key[:, :, :1] = odd
    keys = c.put(0, 0, "keys", key)
    values = c.put(0, 0, "values", (1 - 2 * odd).expand(length, kv, width))
    q = torch.zeros(c.rows, heads, width, device="cuda")
    q[:, :, 0] = 1
    s = -math.log(1 - below)  # w = 1 - below
    out = call(l2c, c, q.reshape(c.rows, -1).bfloat16(), heads, scale=s).double().reshape(c.rows, heads, width)
    for i in range(new):
        n = length - new + i + 1
        weight = torch.exp(s * (keys[0, :n, 0] - keys[0, 1, 0]))
        want = (weight.unsqueeze(1) * values[0, :n]).sum(0) / weight.sum()
        tol = 2.0 ** -15 + 2 * (0.01 * (width + 4) * 2.0 ** -24 + 2.0 ** -21) + 2 * n * 2.0 ** -24 + want.abs() * 2.0 ** -8
        off = (out[i] - want).abs()
        assert bool((off <= 1.02 * tol).all()), (off / tol).max()


@pytest.mark.parametrize("bad", [NAN, -math.inf])
@pytest.mark.parametrize("page", [5, 16])
@pytest.mark.parametrize("width", [64, 72])
@pytest.mark.parametrize("new,window", [(1, 0), (5, 0), (5, 99), (40, 0), (150, 0)])
def test_scales_beside_scores_of_minus_infinity(torch_gpu, l2c, new, window, width, page, bad):
    """A value that is not finite times the weight 0 is NaN in every kind of tile, also where the weight is 0 because the
    score is -Inf, and also where the value is not finite by its scale; rows that do not see it have none of it."""
    c = Cache(width, [new + 130, new + 3], [new, new], 1, width, page, "e4m3")
    q = torch.ones(c.rows, 4 * width, device="cuda").bfloat16()
    low = torch.zeros(1, 1, width, device="cuda")
    low[..., 0] = -1
    for at in (4, 40, new + 90, new + 128):
        where, slot = c.place(0, at, 1)
        c.keys[where, :, slot] = low.to(E4M3).view(torch.uint8)
        c.key_scales[where, :, slot] = math.inf
        c.dense[0][0][:, at] = torch.where(low[0] < 0, -math.inf, 0.0).double()  # the score of ones is -Inf
        c.values[where, :, slot] = torch.ones_like(low).to(E4M3).view(torch.uint8)
        c.value_scales[where, :, slot] = bad
        c.dense[0][1][:, at] = bad
    check(l2c, c, 4, window=window, q=q)
