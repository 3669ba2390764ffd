"""The cache's operators together, as a beam search over them uses them: a prompt in one chunk, then steps of
advance, copy, append, attention, product, selection; and the log probabilities of what came out. The oracle keeps
every beam's whole history of keys and values and moves it after the parents; a graph of the steps gives the same."""
import math

import pytest
import torch
from paged import NAN

pytestmark = pytest.mark.gpu


class Model:
    """One layer: a token's row of `embedding` gives queries, keys and values; attention's output times the
    classifier gives the logits."""

    def __init__(self, l2c, batch, beams, heads, kv, width, vocab, page, cache, window, seed):
        self.l2c, self.batch, self.beams, self.heads, self.kv, self.width = l2c, batch, beams, heads, kv, width
        self.vocab, self.page, self.window, self.n = vocab, page, window, batch * beams
        gen = torch.Generator("cuda").manual_seed(seed)
        self.stride = (heads + 2 * kv) * width
        self.embedding = torch.randn(vocab, self.stride, generator=gen, device="cuda").bfloat16()
        self.classifier = (0.5 * torch.randn(vocab, heads * width, generator=gen, device="cuda")).bfloat16()
        self.prompts = [torch.randint(vocab, (n,), generator=gen, device="cuda")
                        for n in torch.randint(1, 70, (batch,), generator=torch.Generator().manual_seed(seed)).tolist()]
        self.steps, self.most = 6, 80 // page + 1
        self.pages = batch * self.most + 2 * self.n
        shape = (2, self.pages, kv, page, width)
        i32 = dict(device="cuda", dtype=torch.int32)
        if cache == "bf16":
            self.pool, self.scales = torch.full(shape, NAN, device="cuda", dtype=torch.bfloat16), None
        else:
            self.pool = torch.full(shape, 0x7f, device="cuda", dtype=torch.uint8)
            self.scales = torch.full(shape[:-1], NAN, device="cuda")
        self.tables = [torch.full((self.n, self.most), -1, **i32) for _ in range(2)]
        self.lengths = [torch.zeros(self.n, **i32) for _ in range(2)]
        self.uses, self.copies, self.short = (torch.zeros(s, **i32) for s in (self.pages, (self.n, 2), 1))
        self.scores, self.tokens, self.parents = torch.zeros(self.n, device="cuda"), torch.zeros(self.n, **i32), torch.zeros(self.n, **i32)
        self.out = torch.zeros(self.n, heads * width, device="cuda", dtype=torch.bfloat16)
        self.logits = torch.zeros(self.n, vocab, device="cuda")
        size = max(l2c.cache_attention_workspace_bytes(self.n, rows, heads, kv, width, page, self.most)
                   for rows in (self.n, sum(len(p) for p in self.prompts)))
        self.attend_ws = torch.empty(size, device="cuda", dtype=torch.uint8)
        self.beam_ws = torch.empty(l2c.decoder_beam_workspace_bytes(vocab, beams, batch), device="cuda", dtype=torch.uint8)

    def advance(self, turn, parents, starts):
        self.l2c.cache_advance(self.tables[turn ^ 1], self.lengths[turn ^ 1], self.uses, self.copies, self.short,
                               self.tables[turn], self.lengths[turn], self.n, self.most, self.page, self.pages,
                               parents=parents, beams=self.beams, starts=starts, window=self.window)
        page = self.kv * self.page * self.width * self.pool.element_size()
        self.l2c.cache_copy(self.pool, self.copies, self.n, self.pages, page, groups=2)
        if self.scales is not None:
            self.l2c.cache_copy(self.scales, self.copies, self.n, self.pages, self.kv * self.page * 4, groups=2)

    def layer(self, turn, x, out, starts):
        """x: the new tokens' fused rows."""
        scales = dict(key_scales=None if self.scales is None else self.scales[0],
                      value_scales=None if self.scales is None else self.scales[1])
        q, k, v = x.split([self.heads * self.width, self.kv * self.width, self.kv * self.width], 1)
        self.l2c.cache_append(self.pool[0], self.pool[1], k, v, self.tables[turn], self.lengths[turn], self.kv, self.width,
                              self.page, self.pages, self.most, self.n, rows=len(x), starts=starts, k_stride=self.stride,
                              v_stride=self.stride, **scales)
        self.l2c.cache_attention(out, q, self.pool[0], self.pool[1], self.tables[turn], self.lengths[turn], self.heads,
                                 self.kv, self.width, self.page, self.pages, self.most, self.n, self.attend_ws, rows=len(x),
                                 starts=starts, window=self.window, q_stride=self.stride, **scales)

    def start(self):
        """The prompts, each in the first beam of its request, the others empty."""
        for t in self.tables:
            t.fill_(-1)
        self.lengths[0].zero_()
        counts = [0] * self.n
        for b, p in enumerate(self.prompts):
            counts[b * self.beams] = len(p)
        starts = torch.tensor([0] + counts, device="cuda").cumsum(0).int()
        x = self.embedding[torch.cat(self.prompts)]
        hidden = torch.zeros(len(x), self.heads * self.width, device="cuda", dtype=torch.bfloat16)
        self.advance(0, None, starts)
        self.layer(1, x, hidden, starts)
        last = starts[1::self.beams].long() - 1
        self.out.zero_()
        self.out[::self.beams] = hidden[last]
        self.scores.fill_(-math.inf)
        self.scores[::self.beams] = 0.0
        self.choose()
        return hidden

    def choose(self):
        self.l2c.matmul_bf16(self.logits, self.out, self.classifier, self.n, self.heads * self.width, self.vocab)
        self.l2c.decoder_beam_select(self.scores, self.tokens, self.parents, None, self.logits, self.scores, self.tokens, -1,
                                     self.vocab, self.beams, self.batch, 1, 0, self.beam_ws)

    def step(self, turn):
        self.advance(turn, self.parents, None)
        self.layer(turn ^ 1, self.embedding[self.tokens.clamp(min=0).long()], self.out, None)
        self.choose()


def attended(m, x, kv, at, window):
    """One token's output in 64 bits over the rows kv (fused), position `at` the last."""
    w, h = m.width, m.heads
    q = x[:h * w].double().reshape(m.kv, h // m.kv, w)
    k, v = (kv[:, (h + i * m.kv) * w:(h + (i + 1) * m.kv) * w].double().reshape(-1, m.kv, w).transpose(0, 1).contiguous() for i in (0, 1))
    if m.scales is not None:  # as the pages hold them
        def held(y):  # quotients rounded to fp32, by way of 64 bits: torch's own on the GPU are not always the nearest
            largest = y.abs().amax(-1, keepdim=True)
            s = torch.where(largest > 0, (largest / 448.0).float().double(), 1.0)
            return (y / s).float().to(torch.float8_e4m3fn).double() * s
        k, v = held(k), held(v)
    first = max(0, at - window + 1) if window else 0
    out = []
    for i in range(m.kv):
        p = torch.softmax(q[i] @ k[i, first:at + 1].t() / w ** 0.5, 1)
        out.append(p @ v[i, first:at + 1])
    return torch.cat(out).reshape(-1)


@pytest.mark.parametrize("cache,window,page", [("bf16", 0, 16), ("e4m3", 0, 5), ("bf16", 20, 8), ("e4m3", 9, 16)])
@pytest.mark.parametrize("batch,beams,heads,kv,width", [(3, 4, 4, 2, 64), (2, 7, 6, 1, 128)])
def test_beam_search(torch_gpu, l2c, batch, beams, heads, kv, width, cache, window, page):
    print(f"case step {batch}x{beams} {heads}/{kv} width={width} page={page} {cache} window={window}", flush=True)
    m = Model(l2c, batch, beams, heads, kv, width, 160, page, cache, window, seed=page + batch)
    hidden = m.start()
    torch.cuda.synchronize()
    at = 0
    for p in m.prompts:  # the chunk, token by token
        rows = m.embedding[p]
        for i in range(len(p)):
            want = attended(m, rows[i], rows, i, window)
            assert bool(((hidden[at + i].double() - want).abs() <= 2.0 ** -6 * 4).all())
        at += len(p)
    history = [list(m.prompts[r // beams].tolist()) if r % beams == 0 else [] for r in range(m.n)]
    record = []
    for step in range(m.steps):
        parents, tokens = m.parents.tolist(), m.tokens.tolist()
        m.step(step % 2 ^ 1)
        torch.cuda.synchronize()
        history = [history[r - r % beams + parents[r]] + [tokens[r]] if parents[r] >= 0 else [] for r in range(m.n)]
        assert int(m.short) == 0
        assert m.lengths[step % 2].tolist() == [len(x) for x in history]
        used = m.tables[step % 2]
        assert int(m.uses.sum()) == int((used >= 0).sum())
        for r in range(m.n):
            if not history[r]:
                assert bool((m.out[r] == 0).all())
                continue
            rows = m.embedding[torch.tensor(history[r], device="cuda")]
            want = attended(m, rows[-1], rows, len(history[r]) - 1, window)
            # Values of up to 4 in magnitude: two roundings of 2^-8, and the scores' fp32.
            assert bool(((m.out[r].double() - want).abs() <= 2.0 ** -6 * 4).all())
        record.append([t.clone() for t in (m.out, m.scores, m.tokens, m.parents)])
    # The same from a graph, one of two steps, replayed.
    m.start()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step(1), m.step(0)
    torch.cuda.current_stream().wait_stream(side)
    m.start()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.step(1), m.step(0)
    for again in range(2):
        m.start()
        for step in range(1, m.steps, 2):
            graph.replay()
            torch.cuda.synchronize()
            for got, want in zip((m.out, m.scores, m.tokens, m.parents), record[step]):
                assert torch.equal(got, want)


@pytest.mark.parametrize("width", [64, 128])
def test_scored_prompt(torch_gpu, l2c, width):
    """A prompt in chunks of odd sizes and in one: each token's log probability after those before it."""
    heads, kv, vocab, page, n = 4, 2, 1000, 16, 150
    m = Model(l2c, 1, 1, heads, kv, width, vocab, page, "bf16", 0, seed=width)
    m.most = 10
    gen = torch.Generator("cuda").manual_seed(3)
    prompt = torch.randint(vocab, (n,), generator=gen, device="cuda", dtype=torch.int32)
    m.tables = [torch.full((1, 10), -1, device="cuda", dtype=torch.int32) for _ in range(2)]
    got = []
    for cuts in ([0, n], [0, 1, 38, 39, 100, n]):
        m.lengths[0].zero_()
        m.tables[0].fill_(-1)
        turn, parts = 0, []
        for a, b in zip(cuts, cuts[1:]):
            starts = torch.tensor([0, b - a], device="cuda", dtype=torch.int32)
            size = l2c.cache_attention_workspace_bytes(1, b - a, heads, kv, width, page, m.most)
            m.attend_ws = torch.empty(size, device="cuda", dtype=torch.uint8)
            m.advance(turn, None, starts)
            turn ^= 1
            out = torch.zeros(b - a, heads * width, device="cuda", dtype=torch.bfloat16)
            m.layer(turn, m.embedding[prompt[a:b].long()], out, starts)
            parts.append(out)
        hidden = torch.cat(parts)
        logits = torch.zeros(n, vocab, device="cuda")
        l2c.matmul_bf16(logits, hidden, m.classifier, n, heads * width, vocab)
        following = torch.cat((prompt[1:], prompt[:1]))
        lp, en = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        tt, tl = torch.zeros(n, 3, device="cuda", dtype=torch.int32), torch.zeros(n, 3, device="cuda")
        ws = torch.empty(l2c.decoder_logprobs_workspace_bytes(vocab, 3, n), device="cuda", dtype=torch.uint8)
        l2c.decoder_logprobs(lp, en, tt, tl, logits, following, vocab, 3, n, ws)
        want = torch.log_softmax(logits.double(), 1)
        assert bool(((lp - want.gather(1, following.long().unsqueeze(1)).squeeze(1)).abs() < 1e-5).all())
        assert torch.equal(tt.long(), torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :3])
        got.append(hidden)
    assert bool(((got[0].double() - got[1].double()).abs() <= 2.0 ** -6 * 4).all())
