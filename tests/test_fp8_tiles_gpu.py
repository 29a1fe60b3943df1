"""Every kernel of the e4m3 product, by name: the tiles for many rows and the kernels for few, over numbers of K blocks that wrap the ring of
four LDS buffers (5, 6 and 9) and that do not fill it, with ragged edges on both sides.

Tolerance, from the kernels' order of summation, in units of 2^-24 sum|terms| (mag):
 * a block's 128 products are exact and added in fp32, whatever the order; an addition that truncates is off by 2 of them: 256;
 * the product of the two scales is rounded once, and each of the K / 128 additions of a scaled block (fused) once: 1 + K / 128;
 * up to eight waves' sums are joined: 7;
 * bias times gain and its addition: 1 and 1, and the bias itself counts as a term; leaky slope and gain, two constants and two products: 4.
The gain multiplies all of it by sqrt(2).  16-bit outputs add the 8-bit matrix instruction's block sums (less than 7 2^-13 mag) and half a step
of their type.  At K = 1152 that is 279 2^-24 mag for fp32 outputs; K 2^-22 mag, for any order, would be 4608 2^-24."""
import math

import pytest
import torch

from tests.test_fp8_gpu import EPS, TINY, TYPES, blocks, make_mm, mm64

# (rows, outputs) that reach each kernel on 256 CUs
SHAPES = {
    "rows 16x16/8w widened": (37, 300), "rows 16x16/8w 8-bit": (37, 300), "rows 16x32/8w widened": (13, 16500), "rows 16x32/8w 8-bit": (13, 16500),
    "rows 32x32/8w widened": (33, 6001), "rows 32x32/8w 8-bit": (33, 6001), "rows 32x64/4w widened": (1001, 1001), "rows 32x64/4w 8-bit": (1001, 1001),
    "tile 64x64/4w widened": (1501, 1031), "tile 64x64/4w 8-bit": (1501, 1031), "tile 128x128/8w widened": (2001, 1901), "tile 128x128/8w 8-bit": (2001, 1901),
    "tile 128x256/8w widened": (2499, 3001), "tile 256x256/8w 8-bit": (3499, 4001),
}
NAMES = sorted(SHAPES)
BY_TYPE = [(name, t) for name in NAMES for t in TYPES if ("widened" in name) == (t == torch.float32)]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    if torch.cuda.get_device_properties(0).multi_processor_count != 256:
        pytest.skip("the shapes reach their kernels on 256 CUs")
    return torch.device("cuda:0")


def operands(dev, name, k, dtype, seed=0):
    """(q, scale, Fp8Weight, exact result, sum of magnitudes), on the kernel of that name"""
    from nerffaceediting_amd import dense_ops
    m, n = SHAPES[name]
    q, s, wq, ws = make_mm(m, n, k, seed=seed)
    if dtype == torch.float16:
        s = s * 1e-5
    assert dense_ops.describe_fp8_matmul(m, n, dtype, q.shape[1]) == name
    want, mag = mm64(q, s, wq, ws, dev)
    return q.to(dev), s.t().contiguous().to(dev).t(), dense_ops.fp8_weight_from(wq.to(dev), ws.to(dev)), want, mag


def check(got, want, mag, k, bias=None, gain=1.0):
    b = 0.0 if bias is None else bias.abs()
    tol = gain * ((blocks(k) + 264) * mag + 6 * (mag + b)) * 2.0 ** -24
    if got.dtype != torch.float32:
        tol = tol + gain * 7 * 2.0 ** -13 * mag + want.abs() * EPS[got.dtype] * 1.001 + TINY[got.dtype]
        if got.dtype == torch.float16:
            assert float(want.abs().max()) < 60000
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1, 200, 384, 512, 600, 700, 1100])
@pytest.mark.parametrize("name,dtype", BY_TYPE, ids=lambda v: str(v).replace("torch.", ""))
def test_every_kernel(dev, name, dtype, k):
    from nerffaceediting_amd import dense_ops
    q, s, W, want, mag = operands(dev, name, k, dtype)
    got = dense_ops.fp8_matmul(q, s, W, out_dtype=dtype)
    assert got.dtype == dtype and got.shape == want.shape
    check(got, want, mag, k)
    for _ in range(5):
        assert torch.equal(dense_ops.fp8_matmul(q, s, W, out_dtype=dtype), got)      # same call, same bits
    assert torch.equal(dense_ops.fp8_matmul(q, s.contiguous(), W, out_dtype=dtype), got)      # row-major scales


@pytest.mark.gpu
@pytest.mark.parametrize("bias,lrelu", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("name,dtype", BY_TYPE, ids=lambda v: str(v).replace("torch.", ""))
def test_epilogue_of_every_kernel(dev, name, dtype, bias, lrelu):
    from nerffaceediting_amd import dense_ops
    k = 640
    q, s, W, want, mag = operands(dev, name, k, dtype, seed=1)
    b = torch.randn(want.shape[1], generator=torch.Generator().manual_seed(4)).to(dev) * float(mag.mean()) * 0.01
    got = dense_ops.fp8_matmul(q, s, W, bias=b if bias else None, bias_gain=0.5, lrelu=lrelu, out_dtype=dtype)
    b = b.double() * 0.5 if bias else None
    if bias:
        want = want + b
    if lrelu:
        want = torch.where(want < 0, want * 0.2, want) * math.sqrt(2)
    check(got, want, mag, k, b, math.sqrt(2) if lrelu else 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_rows_and_outputs_of_every_kernel_are_apart(dev, name):
    """NaN in one row's values, one row's scale and one block of weights; q as columns of a wider buffer full of NaN."""
    from nerffaceediting_amd import dense_ops
    dtype = torch.float32 if "widened" in name else torch.bfloat16
    k, (m, n) = 700, SHAPES[name]
    q, s, W, _, _ = operands(dev, name, k, dtype, seed=2)
    clean = dense_ops.fp8_matmul(q, s, W, out_dtype=dtype)
    raw, s2 = q.view(torch.uint8).clone(), s.clone()
    a, b = 1, m - 1
    raw[a, 699] = 0x7F
    s2[b, 3] = float("nan")
    got = dense_ops.fp8_matmul(raw.view(torch.float8_e4m3fn), s2, W, out_dtype=dtype)
    keep = torch.ones(m, dtype=torch.bool, device=dev)
    keep[[a, b]] = False
    assert bool(torch.isnan(got[~keep]).all()) and torch.equal(got[keep], clean[keep])
    bad = torch.ones(n, dtype=torch.bool, device=dev)
    bad[128:256] = False
    scale = W.scale.clone()
    scale[1, 2] = float("nan")
    got = dense_ops.fp8_matmul(q, s, dense_ops.Fp8Weight(W.packed, scale, n, k), out_dtype=dtype)
    assert bool(torch.isnan(got[:, ~bad]).all()) and torch.equal(got[:, bad], clean[:, bad])
    wide = torch.full((m + 2, q.shape[1] + 512), 0x7F, dtype=torch.uint8, device=dev)
    wide[1:m + 1, 256:256 + q.shape[1]] = q.view(torch.uint8)
    got = dense_ops.fp8_matmul(wide.view(torch.float8_e4m3fn)[1:m + 1, 256:256 + q.shape[1]], s, W, out_dtype=dtype)
    assert torch.equal(got, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("name", [n for n in NAMES if "widened" in n])
@pytest.mark.parametrize("at", [0, 70])
def test_fp32_outputs_keep_every_product(dev, name, at):
    """One product of 2^16 beside 127 of 1 in every block: whole numbers below 2^24, so any fp32 sum of them is exact.  The 8-bit instruction's
    grid (8 beside 2^16) would drop at least seven of them."""
    from nerffaceediting_amd import dense_ops
    m, n = SHAPES[name]
    k = 640
    assert dense_ops.describe_fp8_matmul(m, n, torch.float32, k) == name
    q, w = torch.ones(m, k, device=dev), torch.ones(n, k, device=dev)
    q[:, at::128] = 256
    w[:, at::128] = 256
    W = dense_ops.fp8_weight_from(w.to(torch.float8_e4m3fn), torch.ones(blocks(n), 5, device=dev))
    got = dense_ops.fp8_matmul(q.to(torch.float8_e4m3fn), torch.ones(5, m, device=dev).t(), W)
    assert bool((got == 5 * (65536 + 127)).all()), got.flatten()[:4].tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(8128, 16), (40, 16), (8128, 300)])
def test_16_bit_outputs_lose_no_more_than_documented(dev, m, n):
    """+7168 and -7168 at every two places of a block, 126 products of 15/32 beside them, just below the grid of 2^-13 4096: they cancel, and what
    the grid took is all of the error.  Documented: less than 7 2^-13 sum|products| = 12.3 of 59.06; all of them dropped would be 59."""
    from nerffaceediting_amd import dense_ops
    pairs = [(i, j) for i in range(128) for j in range(i + 1, 128)][:m]
    q = torch.full((m, 128), 15 / 512)
    for r, (i, j) in enumerate(pairs):
        q[r, i], q[r, j] = 448, -448
    W = dense_ops.fp8_weight_from(torch.full((n, 128), 16.0, device=dev).to(torch.float8_e4m3fn), torch.ones(blocks(n), 1, device=dev))
    got = dense_ops.fp8_matmul(q.to(dev).to(torch.float8_e4m3fn), torch.ones(m, 1, device=dev), W, out_dtype=torch.float16)
    want, mag = 126 * 15 / 32, 2 * 7168 + 126 * 15 / 32
    assert float((got.double() - want).abs().max()) <= 7 * 2.0 ** -13 * mag + 256 * 2.0 ** -24 * mag + want * EPS[torch.float16]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (5, 4100, 8192), (1, 130, 20000), (300, 48, 16384), (16, 16500, 1100), (33, 64, 256), (1300, 1100, 8200)])
def test_long_sums(dev, m, n, k):
    from nerffaceediting_amd import dense_ops
    q, s, wq, ws = make_mm(m, n, k, seed=6)
    W = dense_ops.fp8_weight_from(wq.to(dev), ws.to(dev))
    want, mag = mm64(q, s, wq, ws, dev)
    for dtype in (torch.float32, torch.bfloat16):
        check(dense_ops.fp8_matmul(q.to(dev), s.to(dev), W, out_dtype=dtype), want, mag, k)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tile 256x256/8w 8-bit", "tile 128x256/8w widened"])
def test_widest_strides_of_a_tile(dev, name):
    """Rows 2^23 bytes and scales 2^21 values apart, the most that the tiles' 32-bit offsets take: 255 rows are 2^31 - 2^23 bytes."""
    from nerffaceediting_amd import dense_ops
    dtype = torch.float32 if "widened" in name else torch.bfloat16
    k, (m, n) = 300, SHAPES[name]
    q, s, W, _, _ = operands(dev, name, k, dtype, seed=3)
    clean = dense_ops.fp8_matmul(q, s, W, out_dtype=dtype)
    if torch.cuda.mem_get_info(dev)[0] < 2 * m << 23:
        pytest.skip("not enough memory")
    far = torch.empty(m << 23, dtype=torch.uint8, device=dev).as_strided(q.shape, (1 << 23, 1))
    far.copy_(q.view(torch.uint8))
    far_scale = torch.empty(m << 21, dtype=torch.float32, device=dev).as_strided(s.shape, (1 << 21, 1))
    far_scale.copy_(s)
    assert dense_ops.describe_fp8_matmul(m, n, dtype, 1 << 23, 1 << 21) == name
    assert torch.equal(dense_ops.fp8_matmul(far.view(torch.float8_e4m3fn), far_scale, W, out_dtype=dtype), clean)


def test_describe_refusals():
    import ctypes
    from nerffaceediting_amd import _lib, dense_ops
    lib = _lib.load()
    buf = ctypes.create_string_buffer(64)
    for args, word in (((0, 5, 128, 1, 0, buf, 64), b"sizes"), ((5, -1, 128, 1, 0, buf, 64), b"sizes"), ((5, 5, 128, 1, 7, buf, 64), b"out_dtype"),
                       ((5, 5, 128, 1, 0, None, 64), b"buffer"), ((5, 5, 128, 1, 0, buf, 0), b"buffer")):
        assert lib.nfe_fp8_matmul_describe(*args) == -1 and word in lib.nfe_last_error()
    if not torch.cuda.is_available():                                      # counted for 256 CUs then
        for name, (m, n) in SHAPES.items():
            for dtype in TYPES:
                if ("widened" in name) == (dtype == torch.float32):
                    assert dense_ops.describe_fp8_matmul(m, n, dtype) == name
    assert dense_ops.describe_fp8_matmul(130, 70, q_stride=(1 << 23) + 16) == "rows 32x64/4w widened"
