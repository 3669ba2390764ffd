"""l2c_cache_copy of more pages and groups than one launch has workgroups for."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count,groups,page_bytes", [
    (4096, 5000, 16),         # 2^24 workgroups and more by its groups,
    (300, 70000, 5),          # and more than 65535 of those, too
    (2 ** 24 + 3, 1, 16),     # by its pairs,
    (2 ** 23 + 1, 3, 20),     # by both
    (9, 9, 1 << 20),          # large pages, in one launch
])
def test_more_than_a_launch(torch_gpu, l2c, count, groups, page_bytes):
    print(f"case copy {count} pairs, {groups} groups of {page_bytes}", flush=True)
    pages = 8
    gen = torch.Generator("cuda").manual_seed(count)
    raw = torch.randint(256, (groups, pages, page_bytes), generator=gen, device="cuda", dtype=torch.uint8)
    copies = torch.full((count, 2), -1, device="cuda", dtype=torch.int32)
    pairs = {0: (1, 4), count // 2: (7, 0), count - 1: (3, 5)}
    want = raw.clone()
    for at, (a, b) in pairs.items():
        copies[at] = torch.tensor([a, b], dtype=torch.int32)
        want[:, b] = raw[:, a]
    l2c.cache_copy(raw, copies, count, pages, page_bytes, groups=groups)
    assert torch.equal(raw, want)
