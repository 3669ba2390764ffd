"""l2c_decoder_beam_select over rows so long that a workgroup goes through its chunk in several
parts (32 beams from 262145 logits on, 16 from 524289): what is kept from part to part, the sum
that is rescaled when a later part has a larger maximum, and the order of equal values across parts.

Tolerance, with u = 2^-24, x the logits and d = x - (the largest so far in the chunk), which is
no further from 0 than x - (the row's largest): d is rounded once, which changes exp(d) by |d| u of
itself; the exponential is within 2 ulp, 4 u; a lane adds at most 32 of them in fp32, 31 u; the
rest is in 64 bits. So the sum is off by at most u (E|d| + 35) of itself, where E weighs |d| with
the softmax, and the logarithm, and every score of the row, by as much, the products of these
errors and exponentials below 2^-126 aside (less than one u more). Within a row the order
is exact; rows whose scores are closer than their tolerances may change places. What is
stored is rounded to fp32, half a step more."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NEG = -np.inf
PART = 8192  # logits of a part


def row_sums(logits, rows):
    """(largest, log of the sum of exp(x - largest), its tolerance) of these rows; NaN where a row has no continuation."""
    top, log, tol = (np.full(len(logits), np.nan) for _ in range(3))
    for r in rows:
        x = logits[r].astype(np.float64)
        if np.isnan(x).any() or x.max() in (np.inf, NEG):
            continue
        d = x - x.max()
        e = np.exp(d)
        top[r], log[r] = x.max(), np.log(e.sum())
        tol[r] = U * ((e * -np.where(d == NEG, 0.0, d)).sum() / e.sum() + 36)
    return top, log, tol


def best_of(row, n):
    """The tokens of the n largest logits that are not -Inf, equal ones in the order of their tokens."""
    n = min(n, len(row))
    least = np.partition(row, len(row) - n)[len(row) - n]
    at = np.flatnonzero((row >= least) & (row > NEG))
    return at[np.argsort(-row[at], kind="stable")][:n]


def check(torch, l2c, logits, scores, tokens=None, eos=-1):
    beams, vocab = logits.shape
    print(f"case beam_select_long {beams}x{vocab} eos={eos}", flush=True)
    assert vocab > PART * (1024 // beams)  # several parts a chunk
    logits, scores = logits.astype(np.float32), np.asarray(scores, np.float32)
    tokens = np.zeros(beams, np.int32) if tokens is None else tokens.astype(np.int32)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    size = l2c.decoder_beam_workspace_bytes(vocab, beams, 1)
    ws = torch.full((size + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    out_s = torch.full((beams + 1,), 7.0, device="cuda")
    out_t, out_p = (torch.full((beams + 1,), 7, dtype=torch.int32, device="cuda") for _ in range(2))
    l2c.decoder_beam_select(out_s, out_t, out_p, None, dev(logits), dev(scores), dev(tokens), eos, vocab, beams, 1, 1, 0,
                            ws[:size])
    torch.cuda.synchronize()
    assert bool((ws[size:] == 0xA5).all()) and float(out_s[-1]) == int(out_t[-1]) == int(out_p[-1]) == 7
    got_s, got_t, got_p = (a[:-1].cpu().numpy() for a in (out_s, out_t, out_p))

    ended = (tokens == eos) & (eos >= 0)
    top, log, tol = row_sums(logits, np.flatnonzero(np.isfinite(scores) & ~ended))
    rows, score, within = [], [], []  # every beam's best tokens, their scores, the row's tolerance
    for k in range(beams):
        best = np.array([eos]) if ended[k] else best_of(logits[k], beams)
        if not np.isfinite(scores[k]) or not (ended[k] or np.isfinite(top[k])):
            best = best[:0]
        rows.append(best)
        score.append(np.float64(scores[k]) + (np.zeros(len(best)) if ended[k] else
                                              (logits[k, best].astype(np.float64) - top[k]) - log[k]))
        within.append(np.full(len(best), 0.0 if ended[k] else tol[k]))
    flat_s, flat_tol = np.concatenate(score), np.concatenate(within)
    order = np.argsort(-flat_s, kind="stable")[:beams]
    n = len(order)
    assert (got_s[n:] == NEG).all() and (got_t[n:] == -1).all() and (got_p[n:] == -1).all()
    assert ((0 <= got_p[:n]) & (got_p[:n] < beams)).all()
    most = flat_tol.max(initial=0.0)
    for place in range(n):
        k = got_p[place]
        # A beam's tokens come in the order of its logits, equal ones by token, none left out.
        i = int((got_p[:place] == k).sum())
        assert i < len(rows[k]) and rows[k][i] == got_t[place], (place, k, got_t[place], rows[k][:4])
        stored = abs(score[k][i]) * U
        assert abs(got_s[place] - score[k][i]) <= within[k][i] * (1 + U) + stored
        # Another candidate than the oracle's, only where the two scores are that close.
        assert abs(score[k][i] - flat_s[order[place]]) <= 2 * most
    return got_s, got_t, got_p


SHAPES = [(32, 262145), (32, 300001), (32, 540003), (17, 500000), (16, 532480)]


def normal(beams, vocab, seed=0):
    rng = np.random.default_rng(seed + vocab + beams)
    return rng, 3 * rng.standard_normal((beams, vocab)).astype(np.float32), -20 - 4 * rng.random(beams)


@pytest.mark.parametrize("beams,vocab", SHAPES)
def test_ordinary_and_rounded(torch_gpu, l2c, beams, vocab):
    """As they are, with ended beams; and rounded, so that many are equal in every part."""
    rng, logits, scores = normal(beams, vocab)
    tokens = np.where(rng.random(beams) < 0.2, 2, 3)
    check(torch_gpu, l2c, logits, scores, tokens, 2)
    check(torch_gpu, l2c, np.round(logits), np.round(scores))


@pytest.mark.parametrize("beams,vocab", SHAPES)
def test_ties(torch_gpu, l2c, beams, vocab):
    """One value, few values, zeros of both signs, and the largest once or twice a part: equal ones by token."""
    rng, logits, scores = normal(beams, vocab, 1)
    same = np.zeros((beams, vocab), np.float32)
    s, t, p = check(torch_gpu, l2c, same, np.full(beams, -3.0))
    np.testing.assert_array_equal(t, np.arange(beams))
    np.testing.assert_array_equal(p, 0)
    _, t, p = check(torch_gpu, l2c, np.where(rng.random((beams, vocab)) < 0.5, -0.0, 0.0), np.full(beams, -1.0))
    np.testing.assert_array_equal(t, np.arange(beams))
    np.testing.assert_array_equal(p, 0)
    check(torch_gpu, l2c, rng.integers(0, 3, (beams, vocab)), scores)
    rare = np.minimum(logits, 9.0)
    rare[:, PART - 1::PART] = 12.0   # a part's last value, the next one's first
    rare[:, PART::2 * PART] = 12.0
    check(torch_gpu, l2c, rare, scores)
    s, t, p = check(torch_gpu, l2c, rare, np.where(np.arange(beams) == 3, -1.0, NEG))
    np.testing.assert_array_equal(t, np.flatnonzero(rare[3] == 12.0)[:beams])
    np.testing.assert_array_equal(p, 3)


@pytest.mark.parametrize("beams,vocab", SHAPES)
def test_sorted(torch_gpu, l2c, beams, vocab):
    """Ascending rows: every part replaces all that is kept and rescales the sum, by little and by
    much; descending rows: no later part has any; and both at once."""
    _, _, scores = normal(beams, vocab, 2)
    for span in (0.5, 20.0, 2000.0):
        up = np.linspace(-span, span, vocab, dtype=np.float32)
        check(torch_gpu, l2c, np.tile(up, (beams, 1)), -0.37 * np.arange(beams))
        check(torch_gpu, l2c, np.tile(up[::-1], (beams, 1)), -0.37 * np.arange(beams))
        check(torch_gpu, l2c, np.stack([up, up[::-1]] * beams)[:beams], scores)
    steps = np.repeat(np.arange(-(-vocab // PART)), PART)[:vocab].astype(np.float32)  # equal within a part
    check(torch_gpu, l2c, np.tile(steps, (beams, 1)), scores)
    check(torch_gpu, l2c, np.tile(-steps, (beams, 1)), scores)


@pytest.mark.parametrize("beams,vocab", SHAPES)
def test_masks(torch_gpu, l2c, beams, vocab):
    """Parts that are wholly masked before, between and after others; less than a list's values
    in a chunk; one value in all, the first or the last; nothing; NaN and +Inf in a later part only;
    the lowest value for a mask."""
    rng, logits, scores = normal(beams, vocab, 3)
    part = np.arange(vocab) // PART
    rows = logits.copy()
    rows[0, part % 2 == 0] = NEG                  # a chunk's first part
    rows[1, part % 2 == 1] = NEG
    rows[2, part % 3 != 1] = NEG
    rows[3, rng.random(vocab) < 0.999] = NEG
    rows[4] = NEG
    rows[5, 1:], rows[6, :-1] = NEG, NEG
    rows[7, part < part[-1]] = NEG                # the last, short part alone
    rows[8, part > 0] = NEG
    rows[9, PART + 5], rows[10, PART + 5], rows[11, -1], rows[12, -1] = np.nan, np.inf, np.nan, np.inf
    rows[13, :PART], rows[14, :PART] = np.nan, np.inf
    rows[15, part % 2 == 0] = np.finfo(np.float32).min
    _, _, p = check(torch_gpu, l2c, rows, scores)
    assert not set(p) & {4, 9, 10, 11, 12, 13, 14}
    # The same rows one at a time, so that none is hidden behind the others.
    for k in range(16):
        _, t, _ = check(torch_gpu, l2c, rows, np.where(np.arange(beams) == k, -2.0, NEG))
        none = k in (4, 9, 10, 11, 12, 13, 14)
        left = 0 if none else min(beams, int((rows[k] > NEG).sum()))
        assert (t >= 0).sum() == left
    few = np.full((beams, vocab), NEG, np.float32)
    few[0, [3, PART - 1, PART, vocab - 1]] = [1.0, 2.0, 2.0, 1.0]
    _, t, p = check(torch_gpu, l2c, few, np.zeros(beams))
    np.testing.assert_array_equal(t[:5], [PART - 1, PART, 3, vocab - 1, -1])
    lowest = np.full((beams, vocab), np.finfo(np.float32).min, np.float32)
    check(torch_gpu, l2c, lowest, scores)
    lowest[:, PART:] = -lowest[:, PART:]          # the largest value after the lowest
    check(torch_gpu, l2c, lowest, scores)


@pytest.mark.parametrize("beams,vocab", SHAPES)
def test_crowds(torch_gpu, l2c, beams, vocab):
    """The best values in few lanes, in one part of every chunk, and in one chunk."""
    rng, logits, scores = normal(beams, vocab, 4)
    place, part = np.arange(vocab), np.arange(vocab) // PART
    for crowd in (place // 4 % 64 < beams - 1, place // 4 % 256 == 255, part % 2 == 1, part == 1):
        check(torch_gpu, l2c, np.where(crowd, 20 + rng.random((beams, vocab)), logits), scores)
        check(torch_gpu, l2c, np.where(crowd, 20 + rng.integers(0, 3, (beams, vocab)), logits), scores)


def test_repeats(torch_gpu, l2c):
    """The order of the lists' atomics does not show: the same call ten times over, many equal values."""
    rng, logits, scores = normal(32, 300001, 5)
    logits = np.round(logits)
    first = check(torch_gpu, l2c, logits, scores)
    for _ in range(9):
        for a, b in zip(first, check(torch_gpu, l2c, logits, scores)):
            np.testing.assert_array_equal(a, b)
