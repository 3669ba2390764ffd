"""The kernels of the attention over a cache in pages and of the log probabilities (CPU: compiles the device
code only and reads the compiler's resource report): every one of them is reached by some call."""
import os
import re
import shutil

import pytest

from test_register_budget import HIPCC, PKG, resource_report

needs_hipcc = pytest.mark.skipif(not shutil.which(HIPCC) and not os.path.exists(HIPCC), reason="hipcc not available")


def attention(sequences, rows, heads, kv_heads, width, page_size, max_pages, starts, e4m3):
    """(The tiles' kernel, the join's or None, the parts' bytes) by the rules that the entry point's comments state."""
    group = heads // kv_heads
    packed = rows * group
    narrow = packed <= (16 if not e4m3 else 48 if width <= 64 else 24) * sequences
    many = 96 < width <= 128 and packed // 256 * kv_heads > 256
    m = 16 if narrow else 256 if many else 128
    slots = packed // m + sequences if starts else sequences * -(-group // m)
    tiles = slots * kv_heads
    least = (128 if tiles < 128 else 256) if narrow else max(256, min(tiles, 512) // 8 * 64)
    splits = min((2048 if narrow else 256 if width > 128 else 512) // tiles, -(-max_pages * page_size // least), 64)
    splits = max(1, min(splits, (1 << 17) // (rows * heads)))
    columns = next(c for c in (2, 3, 4, 6, 8) if width <= 32 * c)
    if narrow:
        pairs = e4m3 and width % 16 == 0
        kernel = "narrow", 4 if pairs and columns == 3 else columns, e4m3, pairs
    else:
        kernel = "wide", columns, 8 if many else 4, e4m3
    join = None if splits == 1 else (m, 32 if narrow else 64, splits > 8)
    return kernel, join, 0 if splits == 1 else rows * heads * splits * (width + 2) * 4


@needs_hipcc
def test_every_attention_kernel_is_reached():
    import l2c
    reached, joins = set(), set()
    for width in (8, 48, 64, 72, 80, 96, 104, 128, 136, 192, 200, 256):
        for sequences, rows, heads, kv_heads in ((1, 1, 8, 8), (1, 1, 32, 8), (64, 64, 32, 8), (1, 20, 8, 8),
                                                 (1, 256, 32, 8), (2, 3000, 32, 8), (1, 4096, 64, 8), (1, 700, 64, 64)):
            for max_pages in (1, 20, 1000):
                ways = [attention(sequences, rows, heads, kv_heads, width, 16, max_pages, starts, e4m3)
                        for starts in (True, False) if starts or rows == sequences for e4m3 in (True, False)]
                reached |= {kernel for kernel, _, _ in ways}
                joins |= {join for _, join, _ in ways if join}
                assert l2c.cache_attention_workspace_bytes(sequences, rows, heads, kv_heads, width, 16, max_pages) \
                    == max(size for _, _, size in ways)
    built, built_joins = set(), set()
    for name in resource_report(os.path.join(PKG, "csrc", "l2c_attention.hip")):
        if m := re.search(r"narrow_kernelILi(\d)ELb([01])ELb([01])E", name):
            built.add(("narrow", int(m[1]), m[2] == "1", m[3] == "1"))
        elif m := re.search(r"wide_kernelILi(\d)ELi(\d)ELb([01])E", name):
            built.add(("wide", int(m[1]), int(m[2]), m[3] == "1"))
        elif m := re.search(r"join_kernelILi(\d+)ELi(\d+)ELb([01])E", name):
            built_joins.add((int(m[1]), int(m[2]), m[3] == "1"))
    assert built == reached
    assert built_joins == joins


@needs_hipcc
def test_every_log_probability_kernel_is_reached():
    import l2c
    reached = set()
    for vocab in (1, 1024, 1025, 2048, 2049, 5000, 32003, 131072, 1 << 20, 0x7fffffff):
        for rows in (1, 3, 16, 100, 511, 512, 2048):
            chunks = min((vocab - 1) // 2048 + 1, 64, max(1, 1024 // rows)) if rows < 512 else 1
            chunk = (vocab - 1) // chunks + 1
            chunks = (vocab - 1) // chunk + 1
            reached.add((1 if chunk <= 1024 else 2 if chunk <= 2048 else 4, chunks == 1))
            for top in (0, 20, 32):
                assert l2c.decoder_logprobs_workspace_bytes(vocab, top, rows) == \
                    (rows * chunks * (24 + 8 * top) if chunks > 1 else 0)
    built = {(int(m[1]), m[2] == "1") for name in resource_report(os.path.join(PKG, "csrc", "l2c_logprobs.hip"))
             if (m := re.search(r"logprobs_kernelILi(\d)ELb([01])E", name))}
    assert built == reached
