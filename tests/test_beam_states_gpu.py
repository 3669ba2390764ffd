"""States inside a beam decode: after every step each row's state is, bit for bit, what its
parent's was before the reordering, and the parents are the selection's. test_beam_gpu's
decode of a small model, its calls watched; and the graph of the same decode, by its result."""
import numpy as np
import pytest

import test_beam_gpu as base

pytestmark = pytest.mark.gpu


class Watched:
    """The binding, with what every reordering found and left."""

    def __init__(self, l2c):
        self.l2c, self.seen = l2c, []

    def __getattr__(self, name):
        return getattr(self.l2c, name)

    def decoder_beam_reorder(self, out, inp, parents, *args, **kwargs):
        before, which = inp.clone(), parents.clone()
        self.l2c.decoder_beam_reorder(out, inp, parents, *args, **kwargs)
        self.seen.append((before, which, out.clone()))


def follow(state, parents, batch, beams):
    """The oracle: rows of `state` that follow their parents; rows without a parent keep theirs."""
    out = state.copy()
    for b in range(batch):
        for k in range(beams):
            p = parents[b * beams + k]
            if 0 <= p < beams:
                out[b * beams + k] = state[b * beams + p]
    return out


@pytest.mark.parametrize("batch,beams,width,vocab", [(3, 4, 96, 500), (2, 5, 256, 3000), (3, 12, 128, 20000),
                                                     (5, 4, 352, 9000), (1, 32, 64, 40)])
def test_states_and_histories_follow_the_parents(torch_gpu, l2c, batch, beams, width, vocab):
    steps = 6
    watched = Watched(l2c)
    d = base.Decoder(torch_gpu, watched, batch, beams, width, vocab, steps, seed=width)
    d.start(7)
    moved = 0
    for step in range(steps):
        watched.seen.clear()
        d.step(step)
        torch_gpu.cuda.synchronize()
        parents = d.parents.cpu().numpy()
        assert len(watched.seen) == (2 if step else 1)  # the histories, but for the first step, then the state
        for before, which, after in watched.seen:
            np.testing.assert_array_equal(which.cpu().numpy(), parents)
        before, _, after = (t.cpu().numpy() for t in watched.seen[-1])
        assert before.shape == (batch * beams, width) and np.isfinite(before).all()
        np.testing.assert_array_equal(after, follow(before, parents, batch, beams))
        np.testing.assert_array_equal(d.state.cpu().numpy(), after)
        moved += int((after != before).any(1).sum())
        if step:
            before, _, after = (t.cpu().numpy() for t in watched.seen[0])
            want = before.copy()
            want[:, :step] = follow(before, parents, batch, beams)[:, :step]
            np.testing.assert_array_equal(after, want)
            np.testing.assert_array_equal(d.generated.cpu().numpy(), after)
    assert moved > batch  # parents other than the rows themselves, and states that differ
    # Unwatched, and as one graph replayed twice with an eager decode between: the same states.
    want = [t.clone() for t in (d.scores, d.tokens, d.generated, d.state)]
    d.l2c = l2c
    graph = torch_gpu.cuda.CUDAGraph()
    d.start(7)
    torch_gpu.cuda.synchronize()
    with torch_gpu.cuda.graph(graph):
        for step in range(steps):
            d.step(step)
    for _ in range(2):
        d.start(7)
        graph.replay()
        torch_gpu.cuda.synchronize()
        for got, w in zip((d.scores, d.tokens, d.generated, d.state), want):
            assert torch_gpu.equal(got, w)
        for got, w in zip(d.run(7), want):
            assert torch_gpu.equal(got, w)
