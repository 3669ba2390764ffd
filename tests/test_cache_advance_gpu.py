"""l2c_cache_advance and l2c_cache_copy against the rules of include/l2c.h, step by step in Python."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def advance(tables, lengths, parents, beams, starts, held, page, pages, window):
    """The rules, one sequence after the other."""
    n_seq, most = tables.shape
    out, lens, copies, lost = np.full_like(tables, -1), [], np.full((n_seq, 2), -1, np.int64), 0
    news = []
    for r in range(n_seq):
        p = r if parents is None else r - r % beams + parents[r] if 0 <= parents[r] < beams else -1
        length = 0 if p < 0 else max(0, int(lengths[p]))
        n = 0 if p < 0 else 1 if starts is None else max(0, int(starts[r + 1]) - int(starts[r]))
        for i in range(min(most, -(-length // page))):
            gone = window and (i + 1) * page <= length - window + 1
            out[r, i] = -1 if gone else tables[p, i]
        lens.append(length + n)
        news.append((length, n))
    is_page = lambda e: 0 <= e < pages  # noqa: E731
    names = {}
    for r in range(n_seq):
        for e in out[r]:
            if is_page(e):
                names[int(e)] = names.get(int(e), 0) + 1
    writers = {}
    for r, (length, n) in enumerate(news):
        i = length // page
        if n and length % page and i < most and is_page(out[r, i]):
            writers.setdefault(int(out[r, i]), []).append(r)
    free = iter([e for e in range(pages) if e not in names and not (held is not None and held[e])])
    for r, (length, n) in enumerate(news):
        i = length // page
        page_of = int(out[r, i]) if n and length % page and i < most and is_page(out[r, i]) else -1
        if page_of >= 0:
            w = writers[page_of]
            keeps = names[page_of] == len(w) and w[0] == r and not (held is not None and held[page_of])
            if not keeps:
                e = next(free, None)
                out[r, i] = -1 if e is None else e
                lost += e is None
                if e is not None:
                    copies[r] = page_of, e
        for i in range(-(-length // page), -(-(length + n) // page)):
            if i >= most:
                lost += 1
                continue
            e = next(free, None)
            out[r, i] = -1 if e is None else e
            lost += e is None
    uses = np.zeros(pages, np.int64)
    for e in out.reshape(-1):
        if is_page(e):
            uses[e] += 1
    return out, np.array(lens), uses, copies, lost


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def check(l2c, tables, lengths, page, pages, parents=None, beams=1, starts=None, held=None, window=0, in_place=False):
    n, most = tables.shape
    print(f"case advance {n}x{most} page={page} pages={pages} beams={beams} window={window} in_place={in_place}", flush=True)
    t, l = dev(tables), dev(lengths)
    junk = lambda *s: torch.full(s, 77777, device="cuda", dtype=torch.int32)  # noqa: E731
    to, lo = (t, l) if in_place else (junk(n, most), junk(n))
    uses, copies, shortage = junk(pages + 1), junk(n + 1, 2), junk(2)
    l2c.cache_advance(to, lo, uses, copies, shortage, t, l, n, most, page, pages, parents=dev(parents), beams=beams,
                      starts=dev(starts), held=dev(held), window=window)
    torch.cuda.synchronize()
    want = advance(tables, lengths, parents, beams, starts, held, page, pages, window)
    for got, w, what in zip((to, lo, uses[:pages], copies[:n]), want, ("tables", "lengths", "uses", "copies")):
        np.testing.assert_array_equal(got.cpu().numpy(), w, what)
    assert shortage.tolist() == [want[4], 77777] and int(uses[pages]) == 77777 and copies[n].tolist() == [77777] * 2
    return want


def beam_tables(rng, batch, beams, page, longest, spare):
    """Requests whose beams share all but the last pages."""
    lengths = rng.integers(0, longest + 1, batch)
    lengths[0] = longest
    need = -(-lengths // page)
    most = int(need.max()) + 3
    pages = int(beams * need.sum()) + spare
    order = iter(rng.permutation(pages))
    tables = np.full((batch, beams, most), -1)
    for b in range(batch):
        for i in range(need[b]):
            if i < need[b] - 2:
                tables[b, :, i] = next(order)
            else:
                tables[b, :, i] = [next(order) for _ in range(beams)]
    return tables.reshape(batch * beams, most), np.repeat(lengths, beams), pages


@pytest.mark.parametrize("page", [1, 2, 16, 48])
@pytest.mark.parametrize("batch,beams", [(1, 1), (1, 4), (7, 3), (40, 8), (300, 5)])
def test_beams(torch_gpu, l2c, batch, beams, page):
    rng = np.random.default_rng(batch * 100 + beams + page)
    tables, lengths, pages = beam_tables(rng, batch, beams, page, 10 * page, 3 * batch * beams)
    n = batch * beams
    parents = rng.integers(0, beams, n)
    parents[rng.random(n) < 0.1] = rng.choice([-1, beams, -2 ** 31, 2 ** 31 - 1])
    held = (rng.random(pages) < 0.1).astype(int)
    check(l2c, tables, lengths, page, pages, parents, beams)
    check(l2c, tables, lengths, page, pages, parents, beams, held=held, window=3 * page + 1)
    starts = np.concatenate(([0], np.cumsum(rng.integers(0, 3 * page, n))))
    check(l2c, tables, lengths, page, pages, parents, beams, starts=starts)
    check(l2c, tables, lengths, page, pages, starts=starts, in_place=True)
    check(l2c, tables, lengths, page, pages, in_place=True, window=1)


@pytest.mark.parametrize("seed", range(6))
def test_pages_shared_by_anyone(torch_gpu, l2c, seed):
    """Tables with any entries, the same page in several places of several sequences, and too few pages."""
    rng = np.random.default_rng(seed)
    for n, most, page, pages in ((5, 4, 4, 9), (60, 6, 16, 50), (1500, 5, 3, 700), (2100, 3, 7, 5000)):
        tables = rng.integers(-1, pages + 1, (n, most))
        tables[rng.random((n, most)) < 0.2] = rng.integers(0, pages)
        lengths = rng.integers(-2, most * page + 3 * page, n)
        starts = np.concatenate(([0], np.cumsum(rng.integers(0, 2 * page, n))))
        held = (rng.random(pages) < 0.2).astype(int)
        check(l2c, tables, lengths, page, pages, starts=starts, held=held)
        check(l2c, tables, lengths, page, pages, held=held, window=page)
        if n % 5 == 0:
            check(l2c, tables, lengths, page, pages, rng.integers(-1, 5, n), 5, starts)


def test_few_pages_and_none(torch_gpu, l2c):
    tables, lengths = np.full((3, 4), -1), np.zeros(3, int)
    for pages in (0, 1, 2, 3):
        _, _, _, _, lost = check(l2c, tables, lengths, 16, pages)
        assert lost == 3 - pages
    check(l2c, np.full((3, 0), -1), np.array([0, 5, 16]), 16, 4)
    # Two sequences write one page, and there is no other: the first keeps it.
    want = check(l2c, np.array([[0, -1], [0, -1]]), np.array([5, 5]), 16, 1)
    assert want[0].tolist() == [[0, -1], [-1, -1]] and want[4] == 1


def test_starts_that_fall(torch_gpu, l2c):
    check(l2c, np.array([[0, 1], [2, -1]]), np.array([20, 3]), 16, 6, starts=np.array([5, 2, 9]))


def test_many_pages(torch_gpu, l2c):
    """Free pages far behind used ones."""
    pages = 300000
    held = np.ones(pages, int)
    held[[5, 100000, 299999]] = 0
    check(l2c, np.full((4, 2), -1), np.zeros(4, int), 16, pages, held=held)
    check(l2c, np.full((4, 2), -1), np.zeros(4, int), 16, pages)


@pytest.mark.parametrize("page_bytes,stride,groups,offset", [(16, 16, 1, 0), (7, 9, 3, 1), (8192, 8192, 4, 0), (4099, 4100, 2, 3),
                                                             (40000, 40960, 2, 0)])
def test_copy(torch_gpu, l2c, page_bytes, stride, groups, offset):
    pages = 37
    print(f"case copy {page_bytes} {stride} {groups}", flush=True)
    gen = torch.Generator("cuda").manual_seed(page_bytes)
    raw = torch.randint(256, (groups * pages * stride + 64,), generator=gen, device="cuda", dtype=torch.uint8)
    want = raw.clone()
    pairs = [(3, 9), (-1, -1), (3, 10), (36, 0), (5, 5), (-1, 7), (4, 37), (2 ** 31 - 1, 2), (20, -2 ** 31), (8, 11)]
    for a, b in pairs:
        if 0 <= a < pages and 0 <= b < pages and a != b:
            for g in range(groups):
                at = offset + g * pages * stride
                want[at + b * stride:at + b * stride + page_bytes] = raw[at + a * stride:at + a * stride + page_bytes]
    l2c.cache_copy(raw[offset:], dev(np.array(pairs)), len(pairs), pages, page_bytes, page_stride=stride, groups=groups)
    assert torch.equal(raw, want)


def test_copy_of_many_groups(torch_gpu, l2c):
    groups = 70000
    raw = torch.arange(groups * 3, device="cuda", dtype=torch.int32).reshape(groups, 3)
    l2c.cache_copy(raw, dev(np.array([[0, 2]])), 1, 3, 4, groups=groups)
    assert torch.equal(raw[:, 2], raw[:, 0]) and int(raw[69999, 1]) == 69999 * 3 + 1


def test_captured(torch_gpu, l2c):
    """Replayed over other tables, with eager calls between the replays."""
    rng = np.random.default_rng(3)
    cases = []
    for _ in range(2):
        tables, lengths, _ = beam_tables(rng, 6, 4, 16, 100, 0)
        grown = np.full((24, 12), -1)
        grown[:, :tables.shape[1]] = tables
        cases.append((grown, lengths, rng.integers(-1, 4, 24)))
    pages = 400
    t, l, p = (dev(x) for x in cases[0])
    out = [torch.zeros(s, device="cuda", dtype=torch.int32) for s in ((24, 12), (24,), (pages,), (24, 2), (1,))]
    pool = torch.zeros(2, pages, 64, device="cuda", dtype=torch.uint8)
    fresh = torch.randint(256, pool.shape, device="cuda", dtype=torch.uint8)

    def run():
        l2c.cache_advance(*out, t, l, 24, 12, 16, pages, parents=p, beams=4)
        l2c.cache_copy(pool, out[3], 24, pages, 64, groups=2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(4):
        tables, lengths, parents = cases[i % 2]
        for to, of in ((t, tables), (l, lengths), (p, parents)):
            to.copy_(dev(of))
        pool.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        want = advance(tables, lengths, parents, 4, None, None, 16, pages, 0)
        for got, w in zip(out, want):
            np.testing.assert_array_equal(got.cpu().numpy().reshape(np.shape(w) or 1), w)
        moved = fresh.clone()
        for a, b in want[3]:
            if a >= 0:
                moved[:, b] = fresh[:, a]
        assert torch.equal(pool, moved)
        check(l2c, *cases[1 - i % 2][:2], 16, pages, cases[1 - i % 2][2], 4)
