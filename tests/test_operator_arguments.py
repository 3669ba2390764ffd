"""What the residual norm, the MXFP4 product and the beam-search entry points refuse:
every case returns hipErrorInvalidValue before anything is launched, so the calls
return on a machine without a GPU. Calls with nothing to do return 0 there, too."""
import ctypes

import pytest

P = 1 << 20  # an address that is never dereferenced
INVALID = 1


def call(name, *args):
    import l2c
    fn = getattr(l2c.load(), name)
    return fn(*[ctypes.c_void_p(a) if t is ctypes.c_void_p else a for a, t in zip(args, fn.argtypes, strict=True)])


def norm(normalized=P, ntype=0, residual_out=2 * P, residual=3 * P, rtype=0, block=4 * P, btype=0, block_weight=P, gate=P,
         per=1, weight=P, size=64, batch=2):
    return call("l2c_residual_rmsnorm", normalized, ntype, residual_out, residual, rtype, block, btype, block_weight, gate,
                per, weight, size, batch, 1.0, 1e-5, None)


@pytest.mark.parametrize("bad", [
    dict(normalized=None), dict(residual=None), dict(block=None), dict(weight=None), dict(ntype=2), dict(rtype=-1),
    dict(btype=7), dict(size=0), dict(size=-1), dict(batch=-1), dict(per=0), dict(per=-3),
    dict(normalized=2 * P),                          # both outputs
    dict(normalized=3 * P, ntype=1),                 # an output over an input of another type
    dict(normalized=4 * P, btype=1), dict(residual_out=4 * P, btype=1),
    dict(normalized=P + 2), dict(residual=3 * P + 1, rtype=1), dict(block=4 * P + 2), dict(residual_out=2 * P + 3),
    dict(weight=P + 2), dict(gate=P + 1), dict(block_weight=P + 3),
    dict(batch=0x7fffffff),                          # more workgroups than one launch has
], ids=str)
def test_residual_rmsnorm_refuses(bad):
    assert norm(**bad) == INVALID


def test_residual_rmsnorm_of_nothing():
    assert norm(batch=0, normalized=None) == 0


def quantize(codes=P, scales=P, x=P, rows=3, cols=64):
    return call("l2c_quantize_mxfp4_bf16", codes, scales, x, rows, cols, None)


def product(out=P, x=P, xs=P, w=P, ws=P, batch=3, cols=64, rows=5):
    return call("l2c_matmul_mxfp4", out, x, xs, w, ws, batch, cols, rows, None)


@pytest.mark.parametrize("bad", [dict(codes=None), dict(scales=None), dict(x=None), dict(cols=0), dict(cols=48),
                                 dict(rows=-1), dict(x=P + 2), dict(codes=P + 8), dict(rows=0x7fffffff, cols=1 << 20)],
                         ids=str)
def test_quantize_mxfp4_bf16_refuses(bad):
    assert quantize(**bad) == INVALID


@pytest.mark.parametrize("bad", [dict(out=None), dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(cols=0),
                                 dict(cols=33), dict(batch=-1), dict(rows=-1), dict(x=P + 4), dict(w=P + 8),
                                 dict(cols=1 << 24), dict(batch=0x7fffffff, rows=0x7fffffff)], ids=str)
def test_matmul_mxfp4_refuses(bad):
    assert product(**bad) == INVALID


@pytest.mark.parametrize("batch,cols,rows", [(1, 48, 10), (1, 1 << 24, 10), (0, 64, 10), (3, 0, 10), (3, -64, 10),
                                             (3, 64, 0)])
def test_no_launch_shape_of_refused_products(batch, cols, rows):
    import l2c
    with pytest.raises(l2c.L2CError):
        l2c.launch_shape(l2c.OP_MATMUL_MXFP4, batch, cols, rows)


def test_products_of_nothing():
    assert quantize(rows=0, x=None) == 0
    assert product(batch=0, out=None) == 0 and product(rows=0, out=None) == 0


def select(scores_out=P, tokens_out=P, parents=P, generated=P, logits=P, scores=P, tokens=P, eos=-1, vocab=100, beams=4,
           batch=2, steps=8, step=3, workspace=P, size=1 << 30):
    return call("l2c_decoder_beam_select", scores_out, tokens_out, parents, generated, logits, scores, tokens, eos, vocab,
                beams, batch, steps, step, workspace, size, None)


@pytest.mark.parametrize("bad", [
    dict(scores_out=None), dict(tokens_out=None), dict(parents=None), dict(logits=None), dict(scores=None),
    dict(tokens=None), dict(workspace=None), dict(workspace=P + 8), dict(size=0), dict(size=2 * 4 * (8 * 4 + 16) - 1),
    dict(vocab=0), dict(beams=0), dict(beams=33), dict(batch=-1), dict(eos=100), dict(steps=0), dict(step=8),
    dict(step=-1), dict(batch=1 << 28, beams=32, size=1 << 60), dict(batch=1 << 24, vocab=0x7fffffff, size=1 << 62),
], ids=str)
def test_beam_select_refuses(bad):
    assert select(**bad) == INVALID


def test_beam_select_of_nothing():
    assert select(batch=0, logits=None) == 0


def test_beam_workspace_size():
    import l2c
    for vocab, beams, batch in [(1, 1, 1), (32000, 4, 1), (32003, 4, 256), (131072, 32, 8), (0x7fffffff, 32, 1)]:
        size = l2c.decoder_beam_workspace_bytes(vocab, beams, batch)
        assert 0 < size <= batch * beams * -(-vocab // 1024) * (8 * beams + 16)
    for bad in [(0, 4, 1), (100, 0, 1), (100, 33, 1), (100, 4, 0), (100, 4, -1)]:
        assert l2c.decoder_beam_workspace_bytes(*bad) == 0


def reorder(out=P, inp=1 << 40, parents=P, beams=4, batch=2, groups=1, pieces=1, group_stride=0, row_stride=256,
            piece_stride=0, piece_bytes=256):
    return call("l2c_decoder_beam_reorder", out, inp, parents, beams, batch, groups, pieces, group_stride, row_stride,
                piece_stride, piece_bytes, None)


@pytest.mark.parametrize("bad", [
    dict(out=None), dict(inp=None), dict(parents=None), dict(beams=0), dict(beams=33), dict(batch=-1), dict(groups=-1),
    dict(pieces=-1), dict(piece_bytes=-1), dict(row_stride=255), dict(row_stride=-256),
    dict(pieces=2, piece_stride=255, row_stride=1024), dict(pieces=2, piece_stride=300, row_stride=500),
    dict(groups=2, group_stride=8 * 256 - 1), dict(groups=2),
    dict(out=P, inp=P + 256), dict(out=P + 2047, inp=P),            # the two overlap
    dict(row_stride=1 << 62, batch=1 << 20),                        # past 63 bits
    dict(piece_bytes=1 << 36, row_stride=1 << 36),                  # more than 2^31 - 1 units a row
    dict(batch=1 << 26, piece_bytes=4096, row_stride=4096, inp=1 << 50),  # more workgroups than one launch has
], ids=str)
def test_beam_reorder_refuses(bad):
    assert reorder(**bad) == INVALID


@pytest.mark.parametrize("nothing", [dict(batch=0), dict(groups=0), dict(pieces=0), dict(piece_bytes=0)], ids=str)
def test_beam_reorder_of_nothing(nothing):
    assert reorder(**nothing, out=None) == 0


def test_wrappers_check_types_and_devices():
    """On CPU tensors: the wrappers' own checks come first."""
    import torch

    import l2c
    f, h = torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        l2c.residual_rmsnorm(f, h, f, f, f, 64, 4)  # residual_out of another type than residual
    with pytest.raises(ValueError):
        l2c.residual_rmsnorm(f, f, f.double(), f, f, 64, 4)
    for bad in (f.half(), f.int(), torch.zeros(4, 64, dtype=torch.uint8)):
        for args in ((bad, f, f, f), (f, bad, bad, f), (f, f, f, bad)):
            with pytest.raises(ValueError, match="fp32 and bf16"):
                l2c.residual_rmsnorm(*args, f, 64, 4)
    with pytest.raises(ValueError):
        l2c.residual_rmsnorm(f, None, f, f, f, 64, 4)  # not on the GPU
    with pytest.raises(ValueError):
        l2c.decoder_beam_reorder(f, f, f, 2, 2, 256)
