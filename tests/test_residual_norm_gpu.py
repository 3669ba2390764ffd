"""l2c_residual_rmsnorm against the formulas in 64 bits.

Tolerances, with u = 2^-24 and m the length of the longest chain of additions of a sum
of squares (no more than size / 64 + 32, whatever the kernel's split): a sum of squares
of s terms is off by at most m + 1 roundings, its root by half as many; dividing, adding
eps, the root and the quotient add four. So z is off by (m / 2 + 8) u |z|, h by that and
four roundings of its two terms' sizes, and the norm by its own (m / 2 + 8) u, by h's
error at this place and by h's error over the row (relative, 2-norm). Stores of bf16 add
half a step, 2^-8 of the value."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def value(t):
    return t.float().cpu().numpy().astype(np.float64)


def expected(x, y, w, pw, g, per, scale, eps):
    """(h, its tolerance, n, its tolerance) of fp32 arithmetic, before the stores' rounding."""
    x, y = value(x), value(y)
    rows, size = x.shape
    chain = (size / 64 + 32) / 2 + 8
    z = y
    if pw is not None:
        z = z / np.sqrt((z * z).mean(1, keepdims=True) + eps) * value(pw)
    if g is not None:
        z = z * value(g)[np.arange(rows) // per]
    h = scale * x + z
    dh = U * ((chain if pw is not None else 0.0) * np.abs(z) + 4 * (np.abs(scale * x) + np.abs(z)))
    r = 1.0 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    n = h * r * value(w)
    over = np.sqrt((dh * dh).sum(1, keepdims=True) / np.maximum((h * h).sum(1, keepdims=True), 1e-300))
    dn = np.abs(r * value(w)) * dh + np.abs(n) * (chain * U + over)
    return h, dh, n, dn


def check(got, want, tol, what):
    bf16 = got.element_size() == 2
    got = value(got)
    tol = tol + (2.0 ** -8 if bf16 else 2.0 ** -24) * (np.abs(want) + tol) + 1e-37
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} values off; first at {np.argwhere(bad)[0]}, {got[bad][0]} for {want[bad][0]}"


def make(torch, batch, size, xt, yt, post, gate, seed=0):
    gen = torch.Generator("cuda").manual_seed(1000 * batch + size + seed)
    rnd = lambda *s: torch.empty(*s, device="cuda").normal_(generator=gen)  # noqa: E731
    per = {"none": 1, "one": batch, "row": 1, "three": 3}[gate]
    return dict(x=(2 * rnd(batch, size)).to(xt), y=rnd(batch, size).to(yt), w=1 + 0.3 * rnd(size),
                pw=1 + 0.3 * rnd(size) if post else None, per=per,
                g=None if gate == "none" else rnd(-(-batch // per), size))


def run(torch, l2c, d, batch, size, nt, xt, scale=0.75, eps=1e-5, keep=True):
    # A row before and after the outputs shows stores outside them.
    n = torch.full((batch + 2, size), 7.0, device="cuda", dtype=nt)
    h = torch.full((batch + 2, size), 7.0, device="cuda", dtype=xt)
    l2c.residual_rmsnorm(n[1:-1], h[1:-1] if keep else None, d["x"], d["y"], d["w"], size, batch, block_weight=d["pw"],
                         gate=d["g"], rows_per_gate=d["per"], residual_scale=scale, eps=eps)
    torch.cuda.synchronize()
    for t in (n, h):
        assert bool((t[0] == 7.0).all()) and bool((t[-1] == 7.0).all())
    assert keep or bool((h == 7.0).all())
    return n[1:-1], h[1:-1]


def compare(torch, l2c, batch, size, xt, yt, nt, post, gate, **how):
    print(f"case residual_rmsnorm {batch}x{size} {xt} {yt} {nt} post={post} gate={gate} {how}", flush=True)
    d = make(torch, batch, size, xt, yt, post, gate)
    scale, eps = how.get("scale", 0.75), how.get("eps", 1e-5)
    want_h, dh, want_n, dn = expected(d["x"], d["y"], d["w"], d["pw"], d["g"], d["per"], scale, eps)
    n, h = run(torch, l2c, d, batch, size, nt, xt, scale, eps, how.get("keep", True))
    check(n, want_n, dn, "normalized")
    if how.get("keep", True):
        check(h, want_h, dh, "residual")


# One value to more than the kernels hold in registers; whole and partial vectors, at every
# boundary of lanes and chunks.
SIZES = [1, 2, 3, 7, 8, 31, 64, 255, 257, 1024, 1029, 2048, 2056, 4096, 4104, 5003, 8192, 8200, 12289, 16384, 16392, 20001,
         40000]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("post", [False, True])
def test_sizes(torch_gpu, l2c, size, post):
    t = torch_gpu
    for batch, xt, yt, nt in ((1, t.float32, t.float32, t.bfloat16), (3, t.bfloat16, t.bfloat16, t.bfloat16)):
        compare(t, l2c, batch, size, xt, yt, nt, post, "one")


@pytest.mark.parametrize("batch", [2, 130, 700, 1500])
@pytest.mark.parametrize("size", [1000, 1003, 4096, 11008])
def test_batches(torch_gpu, l2c, batch, size):
    t = torch_gpu
    compare(t, l2c, batch, size, t.float32, t.float32, t.float32, True, "three")
    compare(t, l2c, batch, size, t.bfloat16, t.float32, t.bfloat16, False, "row")


@pytest.mark.parametrize("size", [768, 5003])
@pytest.mark.parametrize("types", range(8))
@pytest.mark.parametrize("gate", ["none", "one", "row", "three"])
def test_types_and_gates(torch_gpu, l2c, size, types, gate):
    t = torch_gpu
    kinds = [t.bfloat16 if types >> i & 1 else t.float32 for i in range(3)]
    compare(t, l2c, 5, size, *kinds, types % 2 == 0, gate)


def test_without_residual_out(torch_gpu, l2c):
    t = torch_gpu
    for size in (512, 4097, 30000):
        compare(t, l2c, 4, size, t.float32, t.bfloat16, t.bfloat16, True, "none", keep=False)


@pytest.mark.parametrize("scale,eps", [(0.0, 1e-5), (1.0, 0.0), (-2.5, 1e-3)])
def test_scales(torch_gpu, l2c, scale, eps):
    t = torch_gpu
    compare(t, l2c, 3, 1111, t.float32, t.float32, t.float32, True, "one", scale=scale, eps=eps)


@pytest.mark.parametrize("size", [96, 4100, 16384, 20000])
def test_in_place(torch_gpu, l2c, size):
    """Outputs over inputs give what separate outputs give, bit for bit."""
    t = torch_gpu
    for xt in (t.float32, t.bfloat16):
        d = make(t, 6, size, xt, xt, True, "row")
        n, h = run(t, l2c, d, 6, size, xt, xt)
        for swap in (False, True):
            x, y = d["x"].clone(), d["y"].clone()
            on, oh = (x, y) if swap else (y, x)
            l2c.residual_rmsnorm(on, oh, x, y, d["w"], size, 6, block_weight=d["pw"], gate=d["g"], rows_per_gate=1,
                                 residual_scale=0.75)
            assert t.equal(oh, h) and t.equal(on, n)


@pytest.mark.parametrize("offset", [1, 2, 3, 5])
@pytest.mark.parametrize("size", [64, 2048, 4101])
def test_unaligned_addresses(torch_gpu, l2c, offset, size):
    """Tensors that start `offset` elements into their allocation, each another one."""
    t = torch_gpu
    for xt, nt in ((t.float32, t.bfloat16), (t.bfloat16, t.float32)):
        d = make(t, 3, size, xt, xt, True, "row")
        want_h, dh, want_n, dn = expected(d["x"], d["y"], d["w"], d["pw"], d["g"], 1, 0.75, 1e-5)

        def at(a, k):
            buf = t.empty(a.numel() + 8, device="cuda", dtype=a.dtype)
            view = buf[k:k + a.numel()].view(a.shape)
            view.copy_(a)
            return view
        x, y, w, pw, g = at(d["x"], offset), at(d["y"], 2 * offset % 8), at(d["w"], offset), at(d["pw"], 1), at(d["g"], 3)
        n, h = at(t.zeros(3, size, device="cuda", dtype=nt), offset), at(t.zeros(3, size, device="cuda", dtype=xt), 1)
        l2c.residual_rmsnorm(n, h, x, y, w, size, 3, block_weight=pw, gate=g, rows_per_gate=1, residual_scale=0.75)
        check(n, want_n, dn, "normalized")
        check(h, want_h, dh, "residual")


def test_rows_do_not_touch_each_other(torch_gpu, l2c):
    """Rows of zeros, NaN and Inf among ordinary ones: those keep their values, zeros give
    zeros and the others NaN."""
    t = torch_gpu
    for size in (200, 4096, 20000):
        d = make(t, 6, size, t.float32, t.float32, False, "none")
        n0, h0 = run(t, l2c, d, 6, size, t.float32, t.float32)
        d["x"][1], d["y"][1] = 0.0, 0.0
        d["x"][3, size // 2] = float("nan")
        d["y"][4, size - 1] = float("inf")
        n, h = run(t, l2c, d, 6, size, t.float32, t.float32)
        for r in (0, 2, 5):
            assert t.equal(n[r], n0[r]) and t.equal(h[r], h0[r])
        assert bool((n[1] == 0).all()) and bool((h[1] == 0).all())
        assert bool(n[3].isnan().all()) and int(h[3].isnan().sum()) == 1
        assert bool(n[4, size - 1].isnan()) and bool(h[4, size - 1].isinf())
        assert bool((n[4, :size - 1] == 0).all())


def test_graph_and_stream(torch_gpu, l2c):
    """Captured on a side stream and replayed over new inputs."""
    t = torch_gpu
    d = make(t, 40, 4096, t.bfloat16, t.float32, True, "one")
    n, h = t.empty(40, 4096, device="cuda", dtype=t.bfloat16), t.empty(40, 4096, device="cuda", dtype=t.bfloat16)
    call = lambda: l2c.residual_rmsnorm(n, h, d["x"], d["y"], d["w"], 4096, 40, block_weight=d["pw"], gate=d["g"],  # noqa: E731
                                        rows_per_gate=40, residual_scale=0.5)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        call()
    for seed in range(3):
        new = make(t, 40, 4096, t.bfloat16, t.float32, True, "one", seed=seed)
        d["x"].copy_(new["x"])
        d["y"].copy_(new["y"])
        graph.replay()
        t.cuda.synchronize()
        got = n.clone(), h.clone()
        n.zero_(), h.zero_()
        call()
        t.cuda.synchronize()
        assert t.equal(got[0], n) and t.equal(got[1], h)
