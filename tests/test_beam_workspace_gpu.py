"""What l2c_decoder_beam_select leaves in its workspace, and that nothing it finds there shows. The
workspace holds 16 bytes for every chunk of every row, then the chunks' lists of candidates, a logit
and a token each (-1: none). Equal values cost a chunk time, each compared with all others, so
those that can never be chosen, -Inf, are in no list, however many of them there are."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NEG = -np.inf


def select(torch, l2c, logits, scores, tokens, eos, beams, fill):
    rows, vocab = logits.shape
    batch = rows // beams
    print(f"case beam_workspace {batch}x{beams}x{vocab} fill={fill}", flush=True)
    dev = lambda a, t: torch.from_numpy(np.ascontiguousarray(a.astype(t))).cuda()  # noqa: E731
    ws = torch.full((l2c.decoder_beam_workspace_bytes(vocab, beams, batch),), fill, dtype=torch.uint8, device="cuda")
    out = [torch.full((rows,), 7, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
    l2c.decoder_beam_select(*out, None, dev(logits, np.float32), dev(scores, np.float32), dev(tokens, np.int32), eos, vocab,
                            beams, batch, 1, 0, ws)
    torch.cuda.synchronize()
    raw = ws.cpu().numpy()
    lists = len(raw) // (16 + 8 * beams)  # chunks of all rows
    candidates = raw[16 * lists:].view([("logit", np.float32), ("token", np.int32)])
    return [o.cpu().numpy() for o in out], candidates.reshape(batch, beams, beams, lists // rows)  # [request][rank][beam][chunk]


@pytest.mark.parametrize("masked", [0.9, 0.999, 2.0])
@pytest.mark.parametrize("batch,beams,vocab", [(2, 4, 32003), (1, 16, 131072), (3, 32, 5000), (1, 32, 300001), (300, 2, 9001)])
def test_masked_logits_are_in_no_list(torch_gpu, l2c, batch, beams, vocab, masked):
    rng = np.random.default_rng(vocab + beams)
    logits = 3 * rng.standard_normal((batch * beams, vocab)).astype(np.float32)
    logits[rng.random(logits.shape) < masked] = NEG
    _, lists = select(torch_gpu, l2c, logits, np.full(batch * beams, -2.0), np.zeros(batch * beams), -1, beams, 0xA5)
    there = lists["token"] >= 0
    assert (lists["token"][~there] == -1).all()
    assert (lists["logit"][there] > NEG).all()
    for b in range(batch):
        for k in range(beams):  # a list's logits are those of its tokens, in order; no more than there are
            got = lists[b, :, k]
            row = logits[b * beams + k]
            mine = there[b, :, k]
            np.testing.assert_array_equal(row[got["token"][mine]], got["logit"][mine])
            assert (mine[1:] <= mine[:-1]).all()
            assert mine.sum() >= min(beams, int((row > NEG).sum()))
            assert mine.sum() <= int((row > NEG).sum())


@pytest.mark.parametrize("batch,beams,vocab", [(3, 4, 900), (2, 8, 32003), (2, 17, 9001), (1, 32, 300001)])
def test_old_contents_do_not_show(torch_gpu, l2c, batch, beams, vocab):
    """Rows that are ended, dead, masked, or of NaN leave their part of the workspace as it was, or with
    no candidates: whatever that is (NaN, the largest numbers, tokens that look like tokens), the results
    are the same."""
    rng = np.random.default_rng(vocab)
    rows = batch * beams
    logits = 3 * rng.standard_normal((rows, vocab)).astype(np.float32)
    scores, tokens = -20 - 4 * rng.random(rows), rng.integers(3, vocab, rows)
    kind = np.arange(rows) % 8
    tokens[kind == 1] = 2
    scores[kind == 2], scores[kind == 3], scores[kind == 4] = NEG, np.nan, np.inf
    logits[kind == 5] = NEG
    logits[kind == 6, vocab // 2] = np.nan
    tokens[0], scores[0] = 2, NEG  # ended and dead
    want = None
    for fill in (0xA5, 0x00, 0xFF, 0x7F, 0x01):
        got, _ = select(torch_gpu, l2c, logits, scores, tokens, 2, beams, fill)
        want = want or got
        for g, w in zip(got, want):
            np.testing.assert_array_equal(g, w)
    live = np.isin(kind, (0, 1, 7)) & np.isfinite(scores)
    parents = want[2].reshape(batch, beams)
    for b in range(batch):
        assert set(parents[b]) - {-1} <= set(np.flatnonzero(live[b * beams:(b + 1) * beams]))


@pytest.mark.parametrize("eos", [-1, 2])
@pytest.mark.parametrize("batch,beams,vocab", [(1, 6, 900), (3, 8, 32003), (1, 32, 300001)])
def test_dead_and_ended_rows_are_left_out(torch_gpu, l2c, batch, beams, vocab, eos):
    """The first step's scores, 0, -Inf, -Inf, ..., and the other values that end a beam: no chunk of
    such a row has written anything, whatever its logits, and the others' have."""
    rows = batch * beams
    rng = np.random.default_rng(beams)
    logits = 3 * rng.standard_normal((rows, vocab)).astype(np.float32)
    scores, tokens = np.full(rows, NEG), np.full(rows, 5)
    scores[::beams] = 0.0
    scores[1], scores[2], scores[3] = np.nan, np.inf, -3.0
    tokens[3] = 2
    logits[1, 7] = np.nan
    written = np.isfinite(scores) & ~((tokens == eos) & (eos >= 0))
    (s, t, p), lists = select(torch_gpu, l2c, logits, scores, tokens, eos, beams, 0xA5)
    untouched = lists.view(np.uint8).reshape(batch, beams, beams, -1) == 0xA5  # [request][rank][beam][bytes]
    for b in range(batch):
        for k in range(beams):
            assert untouched[b, :, k].all() != written[b * beams + k]
    assert set(p[:beams]) <= {0, 3} and (p[beams:] == 0).all() and (t >= 0).all() and np.isfinite(s).all()
