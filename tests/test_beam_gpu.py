"""Beam search: l2c_decoder_beam_select and l2c_decoder_beam_reorder against the formulas
in 64 bits, and a run of the steps they are made for.

The kernel's exponentials are fp32: each is within 2 ulp, 2^-22, of its value, and a lane
adds at most 32 of them, 2^-19 of the sum. So a row's log-sum, and every score of the row,
is off by at most TOL = 2^-19 + 2^-22, the same for the whole row: the order within a row is
exact, and between rows scores closer than 2 TOL may change places. What is stored is
rounded to fp32, half a step more."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -19 + 2.0 ** -22
NEG = -np.inf


def scores_of(logits, scores, tokens, eos):
    """64-bit scores [rows][vocab] of every continuation, -inf where there is none."""
    x = logits.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        top = x.max(1, keepdims=True)
        # In this order: added to a maximum of the type's lowest value, the sum's logarithm is lost.
        s = scores.astype(np.float64)[:, None] + ((x - top) - np.log(np.exp(x - top).sum(1, keepdims=True)))
    s[np.isnan(x).any(1) | (x == np.inf).any(1) | (x == NEG).all(1)] = NEG
    for r in np.flatnonzero((tokens == eos) & (eos >= 0)):
        s[r] = NEG
        s[r, eos] = scores[r]
    s[~np.isfinite(scores)] = NEG
    return s


def check_select(torch, l2c, logits, scores, tokens, eos, beams, steps=4, step=2, offset=0, alias=False):
    rows, vocab = logits.shape
    batch = rows // beams
    print(f"case beam_select {batch}x{beams}x{vocab} eos={eos}", flush=True)
    buf = torch.empty(rows * vocab + 8, device="cuda")
    x = buf[offset:offset + rows * vocab]
    x.copy_(torch.from_numpy(logits.reshape(-1).astype(np.float32)))
    s = torch.from_numpy(scores.astype(np.float32)).cuda()
    t = torch.from_numpy(tokens.astype(np.int32)).cuda()
    size = l2c.decoder_beam_workspace_bytes(vocab, beams, batch)
    ws = torch.full((size + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    so = s if alias else torch.full((rows + 2,), 7.0, device="cuda")
    to = t if alias else torch.full((rows + 2,), 7, device="cuda", dtype=torch.int32)
    parents = torch.full((rows + 2,), 7, device="cuda", dtype=torch.int32)
    generated = torch.full((rows, steps), 9, device="cuda", dtype=torch.int32)
    l2c.decoder_beam_select(so, to, parents, generated, x, s, t, eos, vocab, beams, batch, steps, step, ws[:size])
    torch.cuda.synchronize()
    assert bool((ws[size:] == 0xA5).all()) and bool((parents[rows:] == 7).all())
    if not alias:
        assert bool((so[rows:] == 7).all()) and bool((to[rows:] == 7).all())
    so, to, pa = so[:rows].cpu().numpy(), to[:rows].cpu().numpy(), parents[:rows].cpu().numpy()
    g = generated.cpu().numpy()
    np.testing.assert_array_equal(g[:, step], to)
    assert (np.delete(g, step, 1) == 9).all()

    every = scores_of(logits.astype(np.float32), scores.astype(np.float32), tokens, eos)
    for b in range(batch):
        mine = every[b * beams:(b + 1) * beams]
        flat = mine.reshape(-1)
        order = np.argsort(-flat, kind="stable")
        order = order[flat[order] > NEG][:beams]
        got_s, got_t, got_p = (a[b * beams:(b + 1) * beams] for a in (so, to, pa))
        n = len(order)
        assert (got_s[n:] == NEG).all() and (got_t[n:] == -1).all() and (got_p[n:] == -1).all()
        assert ((0 <= got_t[:n]) & (got_t[:n] < vocab) & (0 <= got_p[:n]) & (got_p[:n] < beams)).all()
        at = got_p[:n].astype(np.int64) * vocab + got_t[:n]
        assert len(set(at)) == n
        step_of = np.abs(flat[order]) * 2.0 ** -23 + TOL  # stores of fp32
        assert (np.abs(got_s[:n] - flat[order]) <= step_of).all()
        assert (np.abs(got_s[:n] - flat[at]) <= step_of).all()
        # Another candidate than the oracle's, only where the two scores are that close.
        other = at != order
        assert (np.abs(flat[at] - flat[order])[other] <= 2 * TOL).all()
        # Within a beam: the order of its logits, equal ones by token, none left out.
        for k in set(got_p[:n]):
            own = got_t[:n][got_p[:n] == k]
            np.testing.assert_array_equal(own, np.argsort(-mine[k], kind="stable")[:len(own)])
    return so, to, pa


def ordinary(rng, batch, beams, vocab, ended=0.0, eos=-1):
    rows = batch * beams
    tokens = rng.integers(0, vocab, rows)
    if eos >= 0:
        tokens[tokens == eos] = (eos + 1) % vocab
        tokens[rng.random(rows) < ended] = eos
    return 3 * rng.standard_normal((rows, vocab)).astype(np.float32), -20 - 4 * rng.random(rows), tokens


# Rows shorter than the beams, than a wave's lanes, at the edges of lanes, chunks and vectors.
@pytest.mark.parametrize("vocab", [1, 2, 5, 31, 63, 64, 257, 1000, 1023, 1024, 1025, 2047, 2048, 4099, 8192, 8195, 16384,
                                   16389])
@pytest.mark.parametrize("beams", [1, 3, 4, 32])
def test_vocabularies(torch_gpu, l2c, vocab, beams):
    rng = np.random.default_rng(vocab * 100 + beams)
    check_select(torch_gpu, l2c, *ordinary(rng, 2, beams, vocab), -1, beams)


@pytest.mark.parametrize("batch,beams,vocab", [(1, 4, 32000), (7, 5, 32003), (64, 8, 5000), (300, 2, 8004), (40, 16, 32000),
                                               (3, 32, 50257), (1, 1, 131072), (2, 17, 131075), (260, 4, 32003),
                                               (100, 31, 1500), (1, 32, 300001)])
def test_batches(torch_gpu, l2c, batch, beams, vocab):
    rng = np.random.default_rng(batch + beams + vocab)
    logits, scores, tokens = ordinary(rng, batch, beams, vocab, 0.2, 2)
    check_select(torch_gpu, l2c, logits, scores, tokens, 2, beams, offset=batch % 4, alias=batch % 2 == 0)


def test_first_step(torch_gpu, l2c):
    """Scores 0, -Inf, ...: all beams come from the first."""
    rng = np.random.default_rng(1)
    logits, _, tokens = ordinary(rng, 3, 6, 4000)
    scores = np.tile([0.0] + [NEG] * 5, 3)
    _, _, parents = check_select(torch_gpu, l2c, logits, scores, tokens, -1, 6)
    assert (parents == 0).all()


def test_ties(torch_gpu, l2c):
    """Logits of few values: equal ones in the order of their tokens; equal beams in theirs."""
    rng = np.random.default_rng(2)
    for vocab, beams in ((700, 4), (9000, 32), (5001, 7)):
        logits = rng.integers(0, 3, (2 * beams, vocab)).astype(np.float32)
        logits[beams:] = logits[beams]  # the second request's beams are all the same row
        scores = np.concatenate([-20 - 4 * rng.random(beams), np.full(beams, -3.0)])
        so, to, pa = check_select(torch_gpu, l2c, logits, scores, np.zeros(2 * beams, int), -1, beams)
        assert (pa[beams:] == 0).all()
        logits = np.where(rng.random((beams, vocab)) < 0.5, -0.0, 0.0).astype(np.float32)  # zeros of both signs
        _, to, pa = check_select(torch_gpu, l2c, logits, np.full(beams, -1.0), np.zeros(beams, int), -1, beams)
        np.testing.assert_array_equal(to, np.arange(beams))
        assert (pa == 0).all()


@pytest.mark.parametrize("vocab", [40, 255, 256, 300, 511, 512, 513, 767, 769, 1500, 2560, 4575])
@pytest.mark.parametrize("beams", [2, 5, 9, 27, 30])
def test_rows_shorter_than_a_chunk(torch_gpu, l2c, vocab, beams):
    """Waves with few values and with none, and as many lists as beams; logits as they are, and
    rounded, so that many are equal."""
    rng = np.random.default_rng(vocab * 40 + beams)
    logits, scores, tokens = ordinary(rng, 3, beams, vocab, 0.1, 1)
    check_select(torch_gpu, l2c, logits, scores, tokens, 1, beams)
    check_select(torch_gpu, l2c, np.round(2 * logits) / 2, np.round(scores), tokens, 1, beams)


@pytest.mark.parametrize("vocab", [300, 5000, 65540, 200001])
@pytest.mark.parametrize("beams", [1, 4, 16, 32])
def test_equal_scores_of_many_lists(torch_gpu, l2c, vocab, beams):
    """All continuations equal: beam 0's first tokens, in every chunk alike."""
    rows = beams
    s, t, p = check_select(torch_gpu, l2c, np.zeros((rows, vocab), np.float32), np.full(rows, -3.0),
                           np.zeros(rows, int), -1, beams)
    np.testing.assert_array_equal(t, np.arange(beams))
    np.testing.assert_array_equal(p, 0)


@pytest.mark.parametrize("vocab", [300, 5000, 65540, 200001])
@pytest.mark.parametrize("beams", [2, 4, 16, 32])
def test_scores_equal_where_logits_are_not(torch_gpu, l2c, vocab, beams):
    """Logits whose difference from the largest is the same in 64 bits: a beam's continuations
    follow its logits, equal scores of several beams the beam."""
    torch = torch_gpu
    rng = np.random.default_rng(vocab + beams)
    logits = np.zeros((beams, vocab), np.float32)
    logits[:] = 1e-30 * rng.permutation(vocab)
    logits[:, 7] = 10.0
    for live in {1, 2}:
        scores = np.where(np.arange(beams) < live, -1.0, -np.inf)
        x = torch.from_numpy(logits.reshape(-1)).cuda()
        dev = {n: torch.zeros(beams, dtype=torch.float32 if n == "s" else torch.int32, device="cuda") for n in "stp"}
        s0, t0 = torch.from_numpy(scores.astype(np.float32)).cuda(), torch.zeros(beams, dtype=torch.int32, device="cuda")
        ws = torch.empty(l2c.decoder_beam_workspace_bytes(vocab, beams, 1), dtype=torch.uint8, device="cuda")
        l2c.decoder_beam_select(dev["s"], dev["t"], dev["p"], None, x, s0, t0, -1, vocab, beams, 1, 1, 0, ws)
        rest = np.argsort(-logits[0], kind="stable")[1:beams - live + 1]
        np.testing.assert_array_equal(dev["t"].cpu().numpy(), [7] * live + list(rest))
        np.testing.assert_array_equal(dev["p"].cpu().numpy(), list(range(live)) + [0] * (beams - live))


def test_masks(torch_gpu, l2c):
    """Rows masked in part, but for less than the beams, wholly; with the lowest value instead;
    NaN and +Inf; dead beams; and requests that have fewer continuations than beams or none."""
    rng = np.random.default_rng(3)
    beams, vocab = 4, 3000
    logits, scores, tokens = ordinary(rng, 8, beams, vocab)
    logits[0:4, rng.random(vocab) < 0.9] = NEG
    logits[4:8] = NEG
    logits[4, 17], logits[6, [5, 2999]] = 1.0, (2.0, 1.0)      # three continuations
    logits[8:12] = NEG                                         # none
    logits[12, 100], logits[13, 2999], logits[14, 0] = np.nan, np.inf, np.nan
    logits[14, 1:] = NEG
    scores[16:20] = [NEG, np.nan, -5.0, np.inf]
    logits[20:24, :2999] = np.finfo(np.float32).min
    logits[24:28] = np.finfo(np.float32).min
    logits[28], logits[29], logits[30] = np.nan, np.inf, NEG
    logits[31, 1:] = NEG
    _, to, pa = check_select(torch_gpu, l2c, logits, scores, tokens, -1, beams)
    assert (to[4:8] >= 0).sum() == 3 and (to[8:12] == -1).all()
    assert (pa[12:16] == 3).all() and (pa[16:20] == 2).all()
    assert list(to[28:32]) == [0, -1, -1, -1]


def test_ended_beams(torch_gpu, l2c):
    """An ended beam keeps its score and its place; its logits are not looked at."""
    rng = np.random.default_rng(4)
    beams, vocab, eos = 5, 2500, 2499
    logits, scores, tokens = ordinary(rng, 4, beams, vocab, 0.3, eos)
    tokens[5:10] = eos                       # all of a request: its beams in order of score
    tokens[10], scores[10] = eos, -1.0       # the best one
    tokens[15], scores[15] = eos, NEG        # ended and dead
    logits[tokens == eos] = np.nan
    so, to, pa = check_select(torch_gpu, l2c, logits, scores, tokens, eos, beams)
    assert (to[5:10] == eos).all() and (np.diff(so[5:10]) <= 0).all()
    assert to[10] == eos and pa[10] == 0 and so[10] == -1.0


def test_many_candidates_over_the_bound(torch_gpu, l2c):
    """Rows whose best values crowd: in few lists of the join; in few lanes of a chunk, where more
    reach the bound than its list holds; and rows of one value."""
    rng = np.random.default_rng(6)
    beams, vocab = 32, 131072
    logits = rng.standard_normal((beams, vocab)).astype(np.float32) * 0.01 - 30
    for k in range(beams):
        for first in range(0, vocab, 1024):
            best = 10 + rng.random(40)
            if (k + first // 1024) % 64 < 31:
                logits[k, first + rng.choice(1024, 40, replace=False)] = best
            else:
                logits[k, first + 5] = 9.0 + rng.random() * 0.1
    check_select(torch_gpu, l2c, logits, np.full(beams, -2.0), np.zeros(beams, int), -1, beams)
    for beams, vocab in ((4, 20000), (32, 100000), (32, 1500), (9, 65536)):
        crowd = np.arange(vocab) // 4 % 64 < beams - 1  # the first lanes of every wave, four values each time
        logits = np.where(crowd, 10 + rng.random((beams, vocab)), rng.random((beams, vocab))).astype(np.float32)
        check_select(torch_gpu, l2c, logits, -rng.random(beams), np.zeros(beams, int), -1, beams)
    beams = 32
    same = np.zeros((beams, 40000), np.float32)  # every continuation has the same score
    _, to, pa = check_select(torch_gpu, l2c, same, np.zeros(beams), np.ones(beams, int), -1, beams)
    np.testing.assert_array_equal(to, np.arange(beams))
    assert (pa == 0).all()


def test_sorted_rows(torch_gpu, l2c):
    """Ascending and descending logits: all of the best in one lane's neighbourhood."""
    for beams in (4, 32):
        up = np.linspace(-10, 10, 20011, dtype=np.float32)
        logits = np.stack([up, up[::-1]] * (beams // 2))
        check_select(torch_gpu, l2c, logits, -np.arange(beams) * 0.37, np.zeros(beams, int), -1, beams)


def test_long_buffers(torch_gpu, l2c):
    """Logits whose offsets pass 32 bits: the last request's rows lie 4.3 GB in."""
    torch = torch_gpu
    beams, vocab, batch = 4, 65536, 4112
    rows = beams * batch
    x = torch.zeros(rows, vocab, device="cuda")
    rng = np.random.default_rng(7)
    last = 3 * rng.standard_normal((beams, vocab)).astype(np.float32)
    x[-beams:] = torch.from_numpy(last).cuda()
    s = torch.zeros(rows, device="cuda")
    t = torch.zeros(rows, device="cuda", dtype=torch.int32)
    parents = torch.zeros_like(t)
    ws = torch.empty(l2c.decoder_beam_workspace_bytes(vocab, beams, batch), dtype=torch.uint8, device="cuda")
    l2c.decoder_beam_select(s, t, parents, None, x, s, t, -1, vocab, beams, batch, 1, 0, ws)
    so, to, pa = check_select(torch, l2c, last, np.zeros(beams), np.zeros(beams, int), -1, beams)
    np.testing.assert_array_equal(s[-beams:].cpu().numpy(), so)
    np.testing.assert_array_equal(t[-beams:].cpu().numpy(), to)
    np.testing.assert_array_equal(parents[-beams:].cpu().numpy(), pa)


# ---------------------------------------------------------------------------

def moved(state, parents, live):
    """The oracle: state [groups][batch][beams][pieces][positions][bytes], the first `live` positions."""
    out = state.copy()
    groups, batch, beams = state.shape[:3]
    for b in range(batch):
        for k in range(beams):
            p = parents[b, k]
            if 0 <= p < beams:
                out[:, b, k, :, :live] = state[:, b, p, :, :live]
    return out


def check_reorder(torch, l2c, shape, live, seed=0, offset=0, parents=None):
    groups, batch, beams, pieces, positions, width = shape
    print(f"case beam_reorder {shape} live={live} offset={offset}", flush=True)
    rng = np.random.default_rng(seed + sum(shape))
    state = rng.integers(0, 256, shape, dtype=np.uint8)
    if parents is None:
        parents = rng.integers(-1, beams + 1, (batch, beams))  # with some of no beam
    want = moved(state, parents, live)
    p = torch.from_numpy(parents.astype(np.int32)).cuda()

    def buffer(a):
        t = torch.full((a.size + 32,), 0x3C, dtype=torch.uint8, device="cuda")
        t[offset:offset + a.size].copy_(torch.from_numpy(a.reshape(-1)))
        return t
    piece = positions * width
    row = pieces * piece
    how = dict(row_stride=row, pieces=pieces, piece_stride=piece, groups=groups, group_stride=batch * beams * row)
    src = buffer(state)
    l2c.decoder_beam_reorder(src[offset:], src[offset:], p, beams, batch, live * width, **how)  # in place
    assert torch.equal(src, buffer(want))
    src, dst = buffer(state), buffer(np.full(shape, 0x11, np.uint8))
    l2c.decoder_beam_reorder(dst[offset:], src[offset:], p, beams, batch, live * width, **how)
    untouched = np.full(shape, 0x11, np.uint8)
    valid = (parents >= 0) & (parents < beams)
    untouched[:, valid, :, :live] = want[:, valid, :, :live]
    assert torch.equal(dst, buffer(untouched)) and torch.equal(src, buffer(state))


# groups, batch, beams, pieces, positions, bytes a position; positions in use
@pytest.mark.parametrize("shape,live", [
    ((1, 1, 1, 1, 1, 1), 1), ((1, 3, 4, 1, 64, 4), 17), ((2, 2, 2, 3, 40, 26), 39), ((4, 5, 8, 2, 16, 256), 16),
    ((1, 2, 32, 2, 9, 160), 7), ((3, 1, 17, 5, 50, 33), 50), ((1, 70, 5, 1, 300, 4), 299), ((2, 3, 4, 8, 64, 256), 0),
    ((1, 1, 3, 1, 1, 100003), 1), ((2, 4, 4, 4, 128, 256), 100), ((1, 1, 16, 1, 4096, 4), 4095)])
def test_reorder(torch_gpu, l2c, shape, live):
    check_reorder(torch_gpu, l2c, shape, live)


@pytest.mark.parametrize("offset", [1, 2, 4, 8])
def test_reorder_unaligned(torch_gpu, l2c, offset):
    check_reorder(torch_gpu, l2c, (2, 3, 4, 2, 10, 64), 9, offset=offset)
    check_reorder(torch_gpu, l2c, (2, 2, 3, 2, 10, 37), 10, offset=offset)


def test_reorder_parents(torch_gpu, l2c):
    """Cycles, swaps, one parent for all, everyone its own, and none."""
    for row in ([1, 2, 3, 0], [3, 2, 1, 0], [2, 2, 2, 2], [0, 1, 2, 3], [-1, -1, -1, -1], [4, -7, 1 << 30, 2]):
        check_reorder(torch_gpu, l2c, (2, 2, 4, 2, 33, 48), 31, parents=np.array([row, row[::-1]]))


def test_reorder_long_state(torch_gpu, l2c):
    """Rows further apart than 32 bits reach, in place."""
    torch = torch_gpu
    beams, row = 3, (1 << 31) + 4096
    state = torch.zeros(beams * row, dtype=torch.uint8, device="cuda")
    for k in range(beams):
        state[k * row:k * row + 1000] = k + 1
        state[k * row + row - 5000:k * row + row] = 10 * (k + 1)
    p = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    l2c.decoder_beam_reorder(state, state, p, beams, 1, row)
    for k, parent in enumerate([2, 0, 1]):
        assert bool((state[k * row:k * row + 1000] == parent + 1).all())
        assert bool((state[k * row + row - 5000:(k + 1) * row] == 10 * (parent + 1)).all())
        assert int(state[k * row + 1000:k * row + 2000].sum()) == 0


def test_reorder_long_state_out_of_place(torch_gpu, l2c):
    torch = torch_gpu
    beams, row = 2, (1 << 32) + 48
    state = torch.empty(beams * row, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(state)
    for k in range(beams):
        state[k * row:(k + 1) * row] = k + 1
    p = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    l2c.decoder_beam_reorder(out, state, p, beams, 1, row)
    for k in range(beams):
        assert int(out[k * row:(k + 1) * row].min()) == int(out[k * row:(k + 1) * row].max()) == 2 - k


@pytest.mark.parametrize("groups,width", [(65536, 16), (70001, 20), (131075, 1)])
def test_reorder_many_groups(torch_gpu, l2c, groups, width):
    check_reorder(torch_gpu, l2c, (groups, 2, 3, 1, 2, width), 1)


@pytest.mark.parametrize("length", [126 * 16 + 3, 127 * 16 + 1, 128 * 16, 128 * 16 + 1, 255 * 16, 257 * 16 + 5])
def test_reorder_short_and_long_rows(torch_gpu, l2c, length):
    check_reorder(torch_gpu, l2c, (2, 5, 3, 1, 1, length), 1)
    check_reorder(torch_gpu, l2c, (1, 37, 7, 1, 1, length), 1)


@pytest.mark.parametrize("beams", [2, 4, 7, 16, 32])
def test_reorder_many_short_rows(torch_gpu, l2c, beams):
    check_reorder(torch_gpu, l2c, (1, 301, beams, 1, 128, 4), 25)
    check_reorder(torch_gpu, l2c, (2, 67, beams, 3, 5, 13), 4, offset=2)


# ---------------------------------------------------------------------------

def bf16(x):
    u = x.astype(np.float32).view(np.uint32)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


class Decoder:
    """Beam decoding of a small model: token embeddings, a residual norm around a block (a fixed
    product of the state), a 4-bit classifier, selection, and histories and states that follow."""

    def __init__(self, torch, l2c, batch, beams, width, vocab, steps, seed=0):
        rng = np.random.default_rng(seed)
        self.torch, self.l2c = torch, l2c
        self.batch, self.beams, self.width, self.vocab, self.steps = batch, beams, width, vocab, steps
        rows = batch * beams
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.embedding = dev(rng.standard_normal((vocab, width)).astype(np.float32))
        self.block = dev((rng.standard_normal((width, width)) / np.sqrt(width)).astype(np.float32))
        self.ones = dev(np.ones(width, np.float32))
        self.gate = dev(rng.random(width).astype(np.float32))
        self.wc = torch.empty(vocab, width // 2, dtype=torch.uint8, device="cuda")
        self.ws = torch.empty(vocab, width // 32, dtype=torch.uint8, device="cuda")
        w = dev((6 * rng.standard_normal((vocab, width)) / np.sqrt(width)).astype(np.float32))
        l2c.quantize_mxfp4(self.wc, self.ws, w, vocab, width)
        f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        i = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)  # noqa: E731
        self.h, self.y, self.state = f(rows, width), f(rows, width), f(rows, width)
        self.n = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16)
        self.xc = torch.empty(rows, width // 2, dtype=torch.uint8, device="cuda")
        self.xs = torch.empty(rows, width // 32, dtype=torch.uint8, device="cuda")
        self.logits, self.scores, self.tokens, self.parents = f(rows, vocab), f(rows), i(rows), i(rows)
        self.generated = i(rows, steps)
        self.work = torch.empty(l2c.decoder_beam_workspace_bytes(vocab, beams, batch), dtype=torch.uint8, device="cuda")
        self.start(0)

    def start(self, token):
        self.scores.view(self.batch, self.beams).fill_(-float("inf"))[:, 0] = 0.0
        self.tokens.copy_(self.torch.arange(self.batch * self.beams) // self.beams + token)
        self.generated.fill_(-5)
        self.state.zero_()

    def step(self, step):
        l, rows = self.l2c, self.batch * self.beams
        l.decoder_rmsnorm(self.h, self.tokens, self.embedding, self.ones, self.width, self.vocab, rows)
        l.matmul(self.y, self.state, self.block, rows, self.width, self.width)
        # The new state is the sum, the classifier's input its norm.
        l.residual_rmsnorm(self.n, self.state, self.h, self.y, self.ones, self.width, rows, block_weight=self.ones,
                           gate=self.gate, rows_per_gate=rows, residual_scale=0.5)
        l.quantize_mxfp4_bf16(self.xc, self.xs, self.n, rows, self.width)
        l.matmul_mxfp4(self.logits, self.xc, self.xs, self.wc, self.ws, rows, self.width, self.vocab)
        l.decoder_beam_select(self.scores, self.tokens, self.parents, self.generated, self.logits, self.scores, self.tokens,
                              1, self.vocab, self.beams, self.batch, self.steps, step, self.work)
        if step:
            l.decoder_beam_reorder(self.generated, self.generated, self.parents, self.beams, self.batch, 4 * step,
                                   row_stride=4 * self.steps)
        l.decoder_beam_reorder(self.state, self.state, self.parents, self.beams, self.batch, 4 * self.width)

    def run(self, token):
        self.start(token)
        for s in range(self.steps):
            self.step(s)
        self.torch.cuda.synchronize()
        return [t.clone() for t in (self.scores, self.tokens, self.generated, self.state)]


def test_decoding_follows_the_beams(torch_gpu, l2c):
    """Five steps, each checked on the host from the step's own logits: the histories and
    states are those of the chosen parents, and a beam's score is the sum of its tokens'."""
    torch = torch_gpu
    d = Decoder(torch, l2c, 3, 4, 96, 500, 5)
    histories = [[[] for _ in range(4)] for _ in range(3)]
    d.start(7)
    for step in range(5):
        scores, tokens = d.scores.cpu().numpy(), d.tokens.cpu().numpy()
        d.step(step)
        torch.cuda.synchronize()
        logits, parents = d.logits.cpu().numpy(), d.parents.cpu().numpy().reshape(3, 4)
        got_s, got_t = d.scores.cpu().numpy(), d.tokens.cpu().numpy().reshape(3, 4)
        every = scores_of(logits, scores, tokens, 1).reshape(3, 4, 500)
        for b in range(3):
            best = np.sort(every[b].reshape(-1))[::-1][:4]
            assert (np.abs(got_s[4 * b:4 * b + 4] - best) <= TOL + np.abs(best) * 2.0 ** -23).all()
            histories[b] = [histories[b][parents[b, k]] + [int(got_t[b, k])] for k in range(4)]
        g = d.generated.cpu().numpy().reshape(3, 4, 5)
        assert [[list(r[:step + 1]) for r in req] for req in g] == histories
    # The state of a beam is that of its parent, computed from the parent's token and state.
    state = d.state.clone().view(3, 4, 96)
    d.step(4)
    h = d.state.view(3, 4, 96)
    assert h.shape == state.shape and not bool(h.isnan().any())


def test_decoding_captured_and_replayed(torch_gpu, l2c):
    """The whole decode as one graph, replayed over new starts with eager decodes between."""
    torch = torch_gpu
    d = Decoder(torch, l2c, 2, 5, 256, 3000, 6, seed=1)
    eager = {token: d.run(token) for token in (3, 40, 700)}
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    d.start(3)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        for s in range(6):
            d.step(s)
    for token in (700, 3, 40, 3):
        d.start(token)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip((d.scores, d.tokens, d.generated, d.state), eager[token]):
            assert torch.equal(got, want)
        again = d.run(token)
        for got, want in zip(again, eager[token]):
            assert torch.equal(got, want)


def test_decoders_on_two_streams(torch_gpu, l2c):
    """Two decodes whose calls alternate on streams of their own, and two graphs of them replayed
    at once: each gives what it gives alone."""
    torch = torch_gpu
    pair = [Decoder(torch, l2c, 3, 12, 128, 20000, 5, seed=2), Decoder(torch, l2c, 5, 4, 352, 9000, 5, seed=3)]
    alone = [d.run(11) for d in pair]
    streams = [torch.cuda.Stream() for _ in pair]
    graphs = [torch.cuda.CUDAGraph() for _ in pair]
    for d in pair:
        d.start(11)
    torch.cuda.synchronize()
    for s in range(5):
        for d, stream in zip(pair, streams):
            with torch.cuda.stream(stream):
                d.step(s)
    torch.cuda.synchronize()
    for d, want in zip(pair, alone):
        for got, w in zip((d.scores, d.tokens, d.generated, d.state), want):
            assert torch.equal(got, w)
    for d, graph, stream in zip(pair, graphs, streams):
        with torch.cuda.graph(graph, stream=stream):
            for s in range(5):
                d.step(s)
    for _ in range(3):
        for d in pair:
            d.start(11)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for d, want in zip(pair, alone):
            for got, w in zip((d.scores, d.tokens, d.generated, d.state), want):
                assert torch.equal(got, w)
