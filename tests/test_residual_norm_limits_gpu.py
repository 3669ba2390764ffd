"""l2c_residual_rmsnorm over the longest rows that its size, an int, can name."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_longest_row(torch_gpu, l2c):
    """2^31 - 1 values, of which the last 700 are 1 and the others 0, in place: nothing is read or
    written before the row or behind it, and the sum of squares, 2800, is exact. The norm of a 1 is
    2 / sqrt(2800 / size + eps), seven roundings of fp32 (the size, the quotient, eps, the sum, the root, its reciprocal,
    the product) and one of bf16 from it."""
    torch = torch_gpu
    size, ones, guard = 2 ** 31 - 1, 700, 64
    print(f"case residual_rmsnorm 1x{size}", flush=True)

    def row(fill):
        buf = torch.full((guard + size + guard,), fill, device="cuda", dtype=torch.bfloat16)
        return buf, buf[guard:guard + size]
    xbuf, x = row(5.0)
    nbuf, n = row(5.0)
    x[:-ones] = 0.0
    x[-ones:] = 1.0
    w = torch.ones(size, device="cuda")
    l2c.residual_rmsnorm(n, x, x, x, w, size, 1)
    torch.cuda.synchronize()
    for buf in (xbuf, nbuf):
        assert bool((buf[:guard] == 5.0).all()) and bool((buf[-guard:] == 5.0).all())
    assert float(x[:-ones].abs().max()) == 0.0 and bool((x[-ones:] == 2.0).all())
    assert float(n[:-ones].abs().max()) == 0.0
    want = 2.0 / np.sqrt(2800.0 / size + 1e-5)
    got = n[-ones:].double().cpu().numpy()
    assert (np.abs(got - want) <= want * (2.0 ** -8 + 8 * 2.0 ** -24)).all()
