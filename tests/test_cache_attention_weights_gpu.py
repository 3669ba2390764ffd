"""How precisely l2c_cache_attention weighs values where sequences have few rows: by exponentials that are not rounded to
bf16. Every other position has score 0 and value 1, the others score s and value -1, so with w = exp(-s) the result is
(w - 1) / (w + 1), where w lies about half way between two bf16 numbers: rounded to either it is off by 2^-9.

The bound: every |value| is 1, so A of tests/paged.py is 1. The weights are held to 2^-15 of each; scores are at most
M = 0.01 and off by M (width + 4) 2^-24, exponentials by 2^-21 more, which counts twice, once in their sum; sums of n
terms n 2^-24 each; the result is rounded by 2^-8 of it."""
import math

import pytest
import torch
from paged import Cache
from test_cache_attention_gpu import call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("width", [8, 64, 80, 96, 128, 192, 256])
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
