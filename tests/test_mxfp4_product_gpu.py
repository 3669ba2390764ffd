"""l2c_quantize_mxfp4_bf16 and l2c_matmul_mxfp4: codes and scales exactly those of the
format, products to the bound that the other products of exact terms are held to."""
import numpy as np
import pytest

import lowprec_oracle as lo

pytestmark = pytest.mark.gpu

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantize(bits):
    """(codes [rows][cols], scale bytes [rows][cols / 32]) of bf16 patterns, by search."""
    rows, cols = bits.shape
    with np.errstate(invalid="ignore"):  # signalling NaN patterns
        x = (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64).reshape(rows, cols // 32, 32)
    special = ~np.isfinite(x).all(-1)
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    amax = a.max(-1)
    exponent = np.where(amax > 0, np.frexp(amax)[1] - 3, -127).clip(-127)
    v = a / np.ldexp(1.0, exponent)[..., None]
    mid = (GRID[1:] + GRID[:-1]) / 2
    code = np.zeros(v.shape, np.int64)
    for i, m in enumerate(mid):  # past a midpoint, or on it where the code above is even
        code += (v > m) | ((v == m) & ((i + 1) % 2 == 0))
    code = np.where((x < 0) & (code > 0), code + 8, code)
    code[special] = 0
    return code.reshape(rows, cols), np.where(special, 255, exponent + 127).astype(np.uint8)


def unpack(codes):
    return np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1)


def pack(code):
    return (code[:, 0::2] + 16 * code[:, 1::2]).astype(np.uint8)


def dequantize(code, scales):
    v = np.where(code > 7, -1.0, 1.0) * GRID[code & 7]
    with np.errstate(invalid="ignore"):
        s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v.reshape(*scales.shape, 32) * s[..., None]).reshape(code.shape)


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def run_quantize(torch, l2c, bits):
    rows, cols = bits.shape
    codes = torch.full((rows + 2, cols // 2), 0x77, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows + 2, cols // 32), 0x55, dtype=torch.uint8, device="cuda")
    x = dev(torch, bits.view(np.int16))
    # The row before keeps codes 16-byte aligned whatever the length.
    l2c.quantize_mxfp4_bf16(codes[1:], scales[1:], x, rows, cols)
    torch.cuda.synchronize()
    for t, fill in ((codes, 0x77), (scales, 0x55)):
        assert bool((t[0] == fill).all()) and bool((t[-1] == fill).all())
    return codes[1:-1].cpu().numpy(), scales[1:-1].cpu().numpy()


def bf16(x):
    u = x.astype(np.float32).view(np.uint32)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (1, 4096), (5, 5024), (130, 320), (1024, 1024)])
def test_quantize_exact(torch_gpu, l2c, rows, cols):
    print(f"case quantize_mxfp4_bf16 {rows}x{cols}", flush=True)
    rng = np.random.default_rng(rows + cols)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-12, 12, (rows, cols // 32)).repeat(32, 1))
    bits = bf16(x)
    code, scale = quantize(bits)
    got, got_scale = run_quantize(torch_gpu, l2c, bits)
    np.testing.assert_array_equal(got_scale, scale)
    np.testing.assert_array_equal(unpack(got), code)


@pytest.mark.parametrize("lead", [0x3f80, 0x3fff, 0x0001, 0x0080, 0x0100, 0x7f7f, 0x7f80, 0x7fc0, 0xff80])
def test_quantize_every_pattern(torch_gpu, l2c, lead):
    """All 65536 patterns beside a leading value that sets the scale wherever it is the largest:
    ties, subnormals, both zeros, the largest values, infinities and NaN."""
    bits = np.full((2048, 64), 0, np.uint16)
    bits.reshape(-1, 32)[:, 0] = lead
    fill = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    bits.reshape(-1, 32)[:, 1:17] = fill.reshape(4096, 16)
    bits.reshape(-1, 32)[:, 17:32] = fill.reshape(4096, 16)[::-1, :15]
    code, scale = quantize(bits)
    got, got_scale = run_quantize(torch_gpu, l2c, bits)
    np.testing.assert_array_equal(got_scale, scale)
    np.testing.assert_array_equal(unpack(got), code)


def operands(rng, n, cols, spread=3):
    code = rng.integers(0, 16, (n, cols))
    scales = rng.integers(127 - spread, 128 + spread, (n, cols // 32)).astype(np.uint8)
    return code, scales


def check_product(torch, l2c, batch, cols, rows, seed=0, shift=0):
    print(f"case matmul_mxfp4 {batch}x{cols}x{rows}", flush=True)
    rng = np.random.default_rng(seed + batch + cols + rows)
    xc, xs = operands(rng, batch, cols)
    wc, ws = operands(rng, rows, cols)
    buf = torch.full((batch + 2, rows), 7.0, dtype=torch.float32, device="cuda")

    def scales(a):  # `shift` bytes past an aligned address
        t = torch.zeros(a.size + 16, dtype=torch.uint8, device="cuda")
        t[shift:shift + a.size].copy_(torch.from_numpy(a.reshape(-1)))
        return t[shift:shift + a.size]
    l2c.matmul_mxfp4(buf[1:], dev(torch, pack(xc)), scales(xs), dev(torch, pack(wc)), scales(ws), batch, cols, rows)
    torch.cuda.synchronize()
    assert bool((buf[0] == 7.0).all()) and bool((buf[-1] == 7.0).all())
    exp, bound = lo.logit_bound(dequantize(xc, xs), dequantize(wc, ws), 1.0, cols)
    bad = np.abs(buf[1:-1].cpu().numpy().astype(np.float64) - exp) > bound
    assert not bad.any(), f"{bad.sum()} outputs outside the bound; first at {np.argwhere(bad)[0]}"


# One value a side to more than a tile, one block to many steps, every remainder of blocks.
@pytest.mark.parametrize("cols", [32, 64, 96, 128, 160, 256, 288, 480, 512, 544, 1120, 2080])
@pytest.mark.parametrize("batch,rows", [(1, 1), (1, 100), (15, 17), (16, 33), (17, 64), (33, 31), (70, 130)])
def test_product_edges(torch_gpu, l2c, batch, cols, rows):
    check_product(torch_gpu, l2c, batch, cols, rows, shift=(batch + cols // 32) % 4)


@pytest.mark.parametrize("batch,cols,rows", [(1, 4096, 2048), (8, 5024, 1501), (40, 5024, 2004), (64, 4096, 4096),
                                             (129, 2080, 1000), (200, 1024, 8192), (256, 4096, 2752), (513, 768, 1025),
                                             (1024, 2048, 2048), (1030, 608, 4099), (300, 16384, 260), (2, 16384, 300),
                                             (1021, 288, 3000), (1024, 8192, 4096)])
def test_product_shapes(torch_gpu, l2c, batch, cols, rows):
    check_product(torch_gpu, l2c, batch, cols, rows)


# Every kernel: lanes, batch rows and weight rows of its tile, and shapes that run on it, with
# ragged edges, one step to many, odd and even steps and a part of one at the end.
KERNELS = [((256, 16, 16), [(7, 544, 1003), (1, 11008, 500), (16, 4128, 900), (100, 192, 1009), (33, 4128, 1003)]),
           ((128, 32, 32), [(332, 288, 8012), (1000, 320, 2157), (17, 288, 30001), (200, 544, 3800), (50, 256, 9000)]),
           ((512, 32, 32), [(33, 288, 4001), (61, 1056, 3005), (128, 2080, 1003), (250, 14016, 300), (5, 4096, 8190)]),
           ((512, 32, 64), [(40, 5024, 8004), (100, 10016, 3003), (100, 1504, 3001)]),
           ((512, 64, 64), [(200, 1312, 3801), (64, 4064, 11001), (1021, 2016, 1003), (63, 11008, 9003)]),
           ((512, 64, 128), [(120, 3904, 10003), (505, 1312, 3003), (1000, 16384, 2001)]),
           ((512, 128, 128), [(240, 4096, 10001), (513, 2080, 4003), (1010, 11008, 4001)]),
           ((512, 128, 192), [(500, 1120, 10801), (400, 4192, 11002), (384, 608, 10901)]),
           ((512, 256, 128), [(1011, 768, 8001), (1000, 4192, 8190)])]


@pytest.mark.parametrize("kernel,shapes", KERNELS, ids=str)
def test_every_kernel(torch_gpu, l2c, kernel, shapes):
    lanes, bm, bn = kernel
    for batch, cols, rows in shapes:
        grid, block, per_cu = l2c.launch_shape(l2c.OP_MATMUL_MXFP4, batch, cols, rows)
        assert (grid, block) == (-(-batch // bm) * -(-rows // bn), lanes), (batch, cols, rows)
        assert per_cu >= 1
        check_product(torch_gpu, l2c, batch, cols, rows, shift=1)


@pytest.mark.parametrize("batch,cols,rows", [(2, 160, 40), (300, 608, 520), (1024, 1056, 1100)])
def test_nan_scales(torch_gpu, l2c, batch, cols, rows):
    """A row with a NaN scale in its last block gives NaN in all its outputs and no others."""
    torch = torch_gpu
    rng = np.random.default_rng(5)
    xc, xs = operands(rng, batch, cols)
    wc, ws = operands(rng, rows, cols)
    xs[1, -1] = 255
    xc.reshape(batch, -1, 32)[1, -1] = 0  # zero codes, as the quantizer leaves them
    ws[7, 0] = 255
    out = torch.zeros(batch, rows, device="cuda")
    l2c.matmul_mxfp4(out, dev(torch, pack(xc)), dev(torch, xs), dev(torch, pack(wc)), dev(torch, ws), batch, cols, rows)
    nan = out.isnan().cpu().numpy()
    want = np.zeros_like(nan)
    want[1], want[:, 7] = True, True
    np.testing.assert_array_equal(nan, want)


def test_extreme_scales(torch_gpu, l2c):
    """Scales from 2^-127 up whose products stay finite: 2^-127 * 2^127 and the reverse."""
    torch = torch_gpu
    for batch, cols, rows in ((3, 96, 20), (300, 512, 300)):
        xc, wc = np.full((batch, cols), 2), np.full((rows, cols), 4)  # 1 and 2
        xs, ws = np.zeros((batch, cols // 32), np.uint8), np.full((rows, cols // 32), 254, np.uint8)
        for a, b in ((xs, ws), (ws[:1].repeat(batch, 0), xs[:1].repeat(rows, 0))):
            out = torch.zeros(batch, rows, device="cuda")
            l2c.matmul_mxfp4(out, dev(torch, pack(xc)), dev(torch, a), dev(torch, pack(wc)), dev(torch, b), batch, cols,
                             rows)
            assert bool((out == 2.0 * cols).all())


@pytest.mark.parametrize("batch,cols,rows", [(3, 352, 50), (40, 4096, 700), (300, 1024, 520)])
def test_quantized_weights_and_activations(torch_gpu, l2c, batch, cols, rows):
    """The operands as a user has them: weights by l2c_quantize_mxfp4, activations on the way."""
    torch = torch_gpu
    rng = np.random.default_rng(cols)
    w = (rng.standard_normal((rows, cols)) / np.sqrt(cols)).astype(np.float32)
    bits = bf16(rng.standard_normal((batch, cols)))
    wc = torch.empty(rows, cols // 2, dtype=torch.uint8, device="cuda")
    ws = torch.empty(rows, cols // 32, dtype=torch.uint8, device="cuda")
    l2c.quantize_mxfp4(wc, ws, dev(torch, w), rows, cols)
    xc = torch.empty(batch, cols // 2, dtype=torch.uint8, device="cuda")
    xs = torch.empty(batch, cols // 32, dtype=torch.uint8, device="cuda")
    l2c.quantize_mxfp4_bf16(xc, xs, dev(torch, bits.view(np.int16)), batch, cols)
    out = torch.empty(batch, rows, device="cuda")
    l2c.matmul_mxfp4(out, xc, xs, wc, ws, batch, cols, rows)
    code, scale = quantize(bits)
    exp, bound = lo.logit_bound(dequantize(code, scale), dequantize(unpack(wc.cpu().numpy()), ws.cpu().numpy()), 1.0, cols)
    assert (np.abs(out.cpu().numpy().astype(np.float64) - exp) <= bound).all()
