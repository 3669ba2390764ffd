"""What the cache's and the log probabilities' entry points refuse: hipErrorInvalidValue before anything is
launched, so the calls return on a machine without a GPU. Calls with nothing to do return 0 there, too."""
import pytest
import torch
from test_operator_arguments import INVALID, P, call

BF16, E4M3 = 1, 2


def append(keys=P, values=2 * P, key_scales=3 * P, value_scales=4 * P, cache_type=BF16, k=5 * P, k_stride=256, v=6 * P,
           v_stride=256, tables=P, lengths=P, starts=P, sequences=2, rows=5, kv_heads=2, width=128, page_size=16, pages=10,
           max_pages=4):
    return call("l2c_cache_append", keys, values, key_scales, value_scales, cache_type, k, k_stride, v, v_stride, tables,
                lengths, starts, sequences, rows, kv_heads, width, page_size, pages, max_pages, None)


def attention(out=P, out_stride=1024, q=2 * P, q_stride=1024, keys=3 * P, values=4 * P, key_scales=P, value_scales=P,
              cache_type=BF16, tables=P, lengths=P, starts=P, sequences=2, rows=5, heads=8, kv_heads=2, width=128,
              page_size=16, pages=10, max_pages=4, window=0, workspace=P, size=1 << 40, scale=1.0):
    return call("l2c_cache_attention", out, out_stride, q, q_stride, keys, values, key_scales, value_scales, cache_type,
                tables, lengths, starts, sequences, rows, heads, kv_heads, width, page_size, pages, max_pages, window, scale,
                workspace, size, None)


BOTH = [dict(keys=None), dict(values=None), dict(keys=P + 8), dict(values=P + 8), dict(cache_type=0), dict(cache_type=3),
        dict(cache_type=E4M3, key_scales=None), dict(cache_type=E4M3, value_scales=None), dict(tables=None),
        dict(lengths=None), dict(starts=None), dict(sequences=-1), dict(rows=-1), dict(kv_heads=0), dict(kv_heads=-2),
        dict(width=0), dict(width=132), dict(width=-8), dict(width=264, k_stride=1024, v_stride=1024, q_stride=4096,
                                                            out_stride=4096),
        dict(page_size=0), dict(page_size=-1), dict(pages=-1), dict(max_pages=-1), dict(max_pages=1 << 20, page_size=1 << 11)]


def only(function, bad):
    names = function.__code__.co_varnames[:function.__code__.co_argcount]
    return {k: v for k, v in bad.items() if k in names}


@pytest.mark.parametrize("bad", BOTH + [
    dict(k=None), dict(v=None), dict(k=P + 4), dict(v=P + 8), dict(k_stride=255), dict(k_stride=252), dict(v_stride=0),
    dict(v_stride=260), dict(rows=0x7fffffff, kv_heads=64, k_stride=1 << 14, v_stride=1 << 14)], ids=str)
def test_append_refuses(bad):
    assert append(**only(append, bad)) == INVALID


@pytest.mark.parametrize("bad", BOTH + [
    dict(q=None), dict(out=None), dict(q=P + 4), dict(out=P + 8), dict(q_stride=1016), dict(q_stride=1028),
    dict(out_stride=-1024), dict(out_stride=1025), dict(heads=0), dict(heads=7), dict(window=-1),
    dict(scale=float("nan")), dict(scale=float("-inf")),
    dict(heads=65536, kv_heads=1, q_stride=1 << 23, out_stride=1 << 23),
    dict(rows=0x7fffffff, heads=64, q_stride=1 << 14, out_stride=1 << 14)], ids=str)
def test_attention_refuses(bad):
    assert attention(**only(attention, bad)) == INVALID


def test_attention_refuses_small_workspaces():
    import l2c
    sizes = dict(sequences=1, rows=1, heads=8, kv_heads=2, width=128, page_size=16, max_pages=8192)
    need = l2c.cache_attention_workspace_bytes(*sizes.values())
    assert 0 < need <= 130 << 19  # one token over 131072 positions is split
    for bad in (dict(size=need - 1), dict(workspace=None), dict(workspace=P + 8)):
        assert attention(**{**sizes, "size": need, "workspace": P, **bad}) == INVALID


def test_attention_workspace_size():
    import l2c
    for sequences, rows, heads, kv, width, page, most in [
            (1, 1, 1, 1, 8, 1, 1), (64, 64, 32, 8, 128, 16, 256), (4, 4, 32, 8, 128, 64, 2048), (1, 4096, 32, 8, 128, 64, 256),
            (16, 80, 10, 10, 80, 32, 80), (3, 5000, 64, 1, 256, 16, 8000), (1, 2, 128, 128, 256, 1000, 2000000),
            (100000, 100000, 1, 1, 64, 16, 8), (1, 1, 65535, 1, 256, 16, 1 << 20)]:
        assert 0 <= l2c.cache_attention_workspace_bytes(sequences, rows, heads, kv, width, page, most) <= (width + 2) << 19
    for bad in [(-1, 1, 8, 2, 128, 16, 4), (1, 1, 7, 2, 128, 16, 4), (1, 1, 8, 2, 100, 16, 4), (1, 1, 8, 2, 128, 0, 4),
                (0, 0, 8, 2, 128, 16, 4), (1, 1, 8, 2, 264, 16, 4), (1, 1, 8, 0, 128, 16, 4)]:
        assert l2c.cache_attention_workspace_bytes(*bad) == 0


@pytest.mark.parametrize("nothing", [dict(sequences=0), dict(rows=0), dict(sequences=0, rows=0, starts=None)], ids=str)
def test_of_no_rows(nothing):
    assert append(**nothing, keys=None) == 0 and attention(**nothing, out=None) == 0


def test_append_to_no_pages():
    assert append(pages=0, keys=None) == 0 and append(max_pages=0, keys=None) == 0


def advance(tables_out=P, lengths_out=2 * P, uses=3 * P, copies=4 * P, shortage=5 * P, tables=6 * P, lengths=7 * P,
            parents=8 * P, beams=2, starts=None, held=None, sequences=4, page_size=16, pages=10, max_pages=4, window=0):
    return call("l2c_cache_advance", tables_out, lengths_out, uses, copies, shortage, tables, lengths, parents, beams,
                starts, held, sequences, page_size, pages, max_pages, window, None)


@pytest.mark.parametrize("bad", [
    dict(tables_out=None), dict(lengths_out=None), dict(uses=None), dict(copies=None), dict(shortage=None),
    dict(tables=None), dict(lengths=None), dict(beams=0), dict(beams=-1), dict(beams=3), dict(sequences=-1),
    dict(page_size=0), dict(pages=-1), dict(max_pages=-1), dict(window=-1), dict(max_pages=1 << 28),
    dict(tables_out=6 * P), dict(lengths_out=7 * P),  # in place, with parents
    dict(sequences=0x7ffffffe)], ids=str)
def test_advance_refuses(bad):
    assert advance(**bad) == INVALID


def test_advance_of_nothing():
    assert advance(sequences=0, tables=None) == 0


def copy(cache=P, copies=P, count=4, pages=10, groups=1, group_stride=0, page_stride=256, page_bytes=256):
    return call("l2c_cache_copy", cache, copies, count, pages, groups, group_stride, page_stride, page_bytes, None)


@pytest.mark.parametrize("bad", [
    dict(cache=None), dict(copies=None), dict(count=-1), dict(pages=-1), dict(groups=-1), dict(page_bytes=-1),
    dict(page_stride=255), dict(page_stride=-256), dict(groups=2), dict(groups=2, group_stride=2559),
    dict(page_stride=1 << 62), dict(page_bytes=1 << 40, page_stride=1 << 40),
    dict(count=0x7fffffff, page_bytes=8192, page_stride=8192), dict(count=1 << 20, groups=1 << 16, group_stride=1 << 20)],
    ids=str)
def test_copy_refuses(bad):
    assert copy(**bad) == INVALID


@pytest.mark.parametrize("nothing", [dict(count=0), dict(pages=0), dict(groups=0), dict(page_bytes=0)], ids=str)
def test_copy_of_nothing(nothing):
    assert copy(**nothing, cache=None) == 0


def logprobs(logprobs=P, entropies=P, top_tokens=P, top_logprobs=P, logits=P, tokens=P, vocab=100000, top=4, rows=2,
             workspace=P, size=1 << 40):
    return call("l2c_decoder_logprobs", logprobs, entropies, top_tokens, top_logprobs, logits, tokens, vocab, top, rows,
                workspace, size, None)


@pytest.mark.parametrize("bad", [
    dict(logprobs=None), dict(tokens=None), dict(top_tokens=None), dict(top_logprobs=None), dict(logits=None),
    dict(logits=P + 2), dict(vocab=0), dict(vocab=-1), dict(top=-1), dict(top=33), dict(rows=-1),
    dict(workspace=None), dict(workspace=P + 8), dict(size=0), dict(rows=0x7fffffff, size=1 << 62)], ids=str)
def test_logprobs_refuses(bad):
    assert logprobs(**bad) == INVALID


def test_logprobs_of_no_rows():
    assert logprobs(rows=0, logits=None) == 0


def test_logprobs_workspace_size():
    import l2c
    for vocab, top, rows in [(1, 0, 1), (32000, 5, 1), (32003, 20, 2048), (131072, 32, 8), (0x7fffffff, 32, 1)]:
        size = l2c.decoder_logprobs_workspace_bytes(vocab, top, rows)
        assert 0 <= size <= rows * -(-vocab // 1024) * (8 * top + 32)
    for bad in [(0, 4, 1), (100, -1, 1), (100, 33, 1), (100, 4, 0), (100, 4, -1)]:
        assert l2c.decoder_logprobs_workspace_bytes(*bad) == 0


def test_wrappers_check_types():
    """On CPU tensors: the wrappers' own checks come first."""
    import l2c
    f, h, i = torch.zeros(64), torch.zeros(64).bfloat16(), torch.zeros(64, dtype=torch.int32)
    b, l = i.to(torch.uint8), i.long()
    sizes = (8, 2, 16, 16, 4, 4, 1)
    for args, more in [((f, h, h, h, i, i), {}), ((h, f, h, h, i, i), {}), ((h, h, f, h, i, i), {}), ((h, h, h, f, i, i), {}),
                       ((h, h, h, h, l, i), {}), ((h, h, h, h, i, l), {}), ((h, h, b, h, i, i), {}),
                       ((h, h, b, b, i, i), {}), ((h, h, b, b, i, i), dict(key_scales=f, value_scales=h)),
                       ((h, h, h, h, i, i), dict(starts=l)), ((h, h, h, h, i, i), {})]:
        with pytest.raises(ValueError):
            l2c.cache_attention(*args, *sizes, **more)
    for args in [(f, f, h, h, i, i), (b, b, h, h, i, i), (h, h, f, h, i, i), (h, h, h, h, i, l), (h, h, h, h, i, i)]:
        with pytest.raises(ValueError):
            l2c.cache_append(*args, 2, 16, 16, 4, 4, 1)
    for wrong in range(8):
        args = [i] * 7
        if wrong < 7:
            args[wrong] = l
        with pytest.raises(ValueError):
            l2c.cache_advance(*args, 2, 4, 16, 10)
    with pytest.raises(ValueError):
        l2c.cache_copy(f, l, 2, 4, 16)
    for args in [(h, f, i, f, f, i), (f, h, i, f, f, i), (f, f, l, f, f, i), (f, f, i, h, f, i), (f, f, i, f, h, i),
                 (f, f, i, f, f, l), (f, f, i, f, f, i)]:
        with pytest.raises(ValueError):
            l2c.decoder_logprobs(*args, 100, 2, 1)
