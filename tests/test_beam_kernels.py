"""The kernels of the beam selection's chunks (CPU: compiles the device code only and reads the
compiler's resource report): every one of them is reached by some call, and those of one part a
chunk fit 64 registers, eight waves a SIMD."""
import os
import re
import shutil

import pytest

from test_register_budget import HIPCC, PKG, resource_report

PART = {2: 2048, 4: 4096, 8: 8192}  # logits of a part, by float4 a lane


def chosen(vocab, beams, batch):
    """(float4 a lane, several parts a chunk) by the rule that the entry point's comment states."""
    most = 1024 // beams
    for v in (2, 4):
        parts = -(-vocab // PART[v])
        if parts == 1 or (parts <= most and batch * beams * parts <= 2048):
            return v, False
    return 8, -(-vocab // PART[8]) > most


@pytest.mark.skipif(not shutil.which(HIPCC) and not os.path.exists(HIPCC), reason="hipcc not available")
def test_every_chunk_kernel_is_reached():
    import l2c
    reached = set()
    for vocab in (1, 2048, 2049, 32000, 65537, 131072, 262144, 262145, 300001, 1 << 20, 0x7fffffff):
        for beams in (1, 4, 17, 32):
            for batch in (1, 8, 64, 500):
                v, several = chosen(vocab, beams, batch)
                reached.add((v, several))
                parts = -(-vocab // PART[v])
                each = -(-parts // (1024 // beams)) if several else 1
                assert l2c.decoder_beam_workspace_bytes(vocab, beams, batch) == \
                    batch * beams * -(-parts // each) * (8 * beams + 16)
    report = resource_report(os.path.join(PKG, "csrc", "l2c_beam.hip"))
    built = {(int(m[1]), m[2] == "1"): registers for name, registers in report.items()
             if (m := re.search(r"beam_chunks_kernelILi(\d)ELb([01])E", name))}
    assert set(built) == reached
    for (_, several), registers in built.items():
        assert several or registers <= 64, built
