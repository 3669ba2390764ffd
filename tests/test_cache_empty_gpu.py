"""The operators over a cache that has no pages yet, or tables without columns, whose tensors are empty and lie nowhere:
no position holds anything, so nothing is written and attention is 0."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("new", [1, 5, 200])
@pytest.mark.parametrize("pages,most", [(0, 4), (3, 0), (0, 0)])
def test_a_cache_without_places(torch_gpu, l2c, pages, most, new, cache):
    print(f"case empty pages={pages} most={most} new={new} {cache}", flush=True)
    sequences, heads, kv, width, page = 2, 4, 2, 64, 16
    rows = sequences * new
    dev = lambda x: torch.tensor(x, device="cuda", dtype=torch.int32)  # noqa: E731
    shape = (pages, kv, page, width)
    keys, values = (torch.zeros(shape, device="cuda", dtype=torch.bfloat16 if cache == "bf16" else torch.uint8) for _ in "kv")
    scales = {} if cache == "bf16" else {n: torch.ones(shape[:3], device="cuda") for n in ("key_scales", "value_scales")}
    tables = torch.zeros(sequences, most, device="cuda", dtype=torch.int32)
    lengths, starts = dev([new, new + 3]), dev([0, new, rows])
    q = torch.randn(rows, heads * width, device="cuda").bfloat16()
    k = torch.randn(rows, kv * width, device="cuda").bfloat16()
    l2c.cache_append(keys, values, k, k, tables, lengths, kv, width, page, pages, most, sequences, rows=rows, starts=starts,
                     **scales)
    size = l2c.cache_attention_workspace_bytes(sequences, rows, heads, kv, width, page, most)
    workspace = torch.empty(size, device="cuda", dtype=torch.uint8)
    out = torch.full((rows, heads * width), 7.0, device="cuda", dtype=torch.bfloat16)
    l2c.cache_attention(out, q, keys, values, tables, lengths, heads, kv, width, page, pages, most, sequences, workspace,
                        rows=rows, starts=starts, **scales)
    assert not keys.view(torch.uint8).any()
    assert bool((out == 0).all())
