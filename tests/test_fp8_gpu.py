"""8-bit dense operators (nfe_rms_norm_fp8, nfe_quantize_fp8, nfe_fp8_weight_*, nfe_fp8_matmul) against plain implementations in 64 bits.

Tolerances.
 * A scale is max|y| / 448.  y carries the fp32 roundings of the sum x + r, of the mean's sum (below 2^-19 relative for the rows here: at
   most 128 serial additions a lane and ten joining steps, halved by the root), of the root (1 ulp of v_rsq_f32) and of three products:
   2^-18 relative is above their total.
 * q * scale is y off by half a step of e4m3: 2^-4 |y|, and under the smallest normal number 2^-6 half of the smallest step, 2^-10 scale;
   the rounding decision itself sees y off by the 2^-18 above.
 * fp8_matmul: products are exact; a sum of K values in fp32 in any order is off by at most K 2^-24 sum|terms| (2^-23 where the matrix unit
   truncates instead of rounding), scaling adds two roundings a block: K 2^-22 sum|terms| bounds it, plus half a step of the output's type.
   With bf16 and fp16 outputs the 8-bit matrix instruction adds eight products at a time on a grid of 2^-13 times the largest one's power
   of two, truncating each (measured with single products: next to 2^16 in the same eight, 2^3 counts and 2^2 does not; in the other
   groups 2^-7 counts).  The largest of the eight has 8 significant bits and loses nothing; the other seven lose less than 2^-13 of the
   largest each, which is at most the group's sum of magnitudes: less than 7 2^-13 sum|terms| in all."""
import math

import pytest
import torch

BLOCK = 128
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def blocks(n):
    return -(-n // BLOCK)


def padded(y):
    return torch.nn.functional.pad(y, (0, blocks(y.shape[-1]) * BLOCK - y.shape[-1]))


def norm64(x, weight, residual, eps=1e-8):
    h = x.double().cpu()
    if residual is not None:
        h = h + residual.double().cpu()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double().cpu()
    return y, h


def check_rows(q, scale, y, cols, rel=2.0 ** -18):
    """q, scale as returned for rows whose unrounded values are y [N, cols] (64 bits)."""
    n = y.shape[0]
    assert q.dtype == torch.float8_e4m3fn and tuple(q.shape) == (n, blocks(cols) * BLOCK)
    assert scale.dtype == torch.float32 and tuple(scale.shape) == (n, blocks(cols))
    yb = padded(y).view(n, -1, BLOCK)
    want = yb.abs().amax(-1).clamp_min(1e-30) / 448
    assert bool(((scale.double().cpu() - want).abs() <= want * rel).all())
    value = q.cpu().float().double().view(n, -1, BLOCK) * scale.double().cpu()[..., None]
    err = (value - yb).abs()
    tol = yb.abs() * (2.0 ** -4 + 2 * rel) + want[..., None] * (2.0 ** -10 + 448 * rel)
    assert bool((err <= tol).all()), float((err - tol).max())
    assert not bool(q.cpu().float()[:, cols:].any())


ROWS = [(1, 512), (4, 512), (3, 8), (5, 1), (2, 127), (7, 128), (6, 129), (257, 520), (9, 1031), (33, 1024), (3, 2048), (5, 2056), (2, 4096), (3, 4104),
        (4, 8192), (2, 8200), (3, 16391), (1, 40000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", ROWS)
@pytest.mark.parametrize("weight,residual", [(False, False), (True, True), (True, False)])
def test_rms_norm(dev, rows, cols, dtype, weight, residual):
    from nerffaceediting_amd import dense_ops
    g = torch.Generator().manual_seed(rows * 100003 + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(cols, generator=g))).to(dtype)
    x[rows // 2] = 0                                                       # a row of zeros
    w = torch.randn(cols, generator=g) if weight else None
    r = (torch.randn(rows, cols, generator=g) * 3).to(dtype) if residual else None
    if residual:
        r[rows // 2] = 0
    got = dense_ops.rms_norm_fp8(x.to(dev), None if w is None else w.to(dev), None if r is None else r.to(dev))
    y, h = norm64(x, w, r)
    check_rows(got[0], got[1], y, cols)
    assert len(got) == (3 if residual else 2)
    if residual:
        assert torch.equal(got[2].cpu(), (x.float() + r.float()).to(dtype))
    assert not bool(got[0].cpu().float()[rows // 2].any()) or cols == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 128), (130, 500), (3, 1031), (2, 9000)])
def test_quantize(dev, rows, cols, dtype):
    from nerffaceediting_amd import dense_ops
    g = torch.Generator().manual_seed(cols)
    x = (torch.randn(rows, cols, generator=g) * 5).to(dtype)
    q, scale = dense_ops.quantize_fp8(x.to(dev))
    check_rows(q, scale, x.double(), cols, rel=2.0 ** -22)


@pytest.mark.gpu
def test_every_e4m3_value_and_tie(dev):
    """A block that holds all finite e4m3 values and the midpoints between them, with 448 as its maximum: scale 1, ties to even."""
    from nerffaceediting_amd import dense_ops
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (codes[:-1] + codes[1:]) / 2
    x = torch.cat([codes, mid, -codes, -mid])
    x = torch.cat([x, torch.full((-(-len(x) // 127) * 127 - len(x),), 0.0)]).view(-1, 127)
    x = torch.cat([x, torch.full((x.shape[0], 1), 448.0)], 1)
    q, scale = dense_ops.quantize_fp8(x.to(dev))
    assert torch.equal(scale.cpu(), torch.ones_like(scale.cpu()))
    assert torch.equal(q.cpu().float(), x.to(torch.float8_e4m3fn).float())


@pytest.mark.gpu
def test_special_values(dev):
    from nerffaceediting_amd import dense_ops
    x = torch.ones(6, 384, device=dev)
    x[1, 200], x[2, 5], x[3, 383] = float("inf"), float("nan"), -float("inf")
    x[4] = 1e-38
    x[5, :128] = 3e38
    q, scale = dense_ops.quantize_fp8(x)
    value = q.float().view(6, 3, 128) * scale[..., None]
    bad = torch.isnan(value).all(-1).cpu()
    want = torch.zeros(6, 3, dtype=torch.bool)
    want[1, 1] = want[2, 0] = want[3, 2] = True
    assert torch.equal(bad, want) and torch.equal(torch.isnan(value).any(-1).cpu(), want)
    assert not bool(q[4].float().any()) and bool(torch.isfinite(scale[4]).all())             # below the smallest maximum: zeros
    assert torch.allclose(value[5, 0], x[5, :128], rtol=2.0 ** -4, atol=0)
    for t in (q[0].float() * scale[0].repeat_interleave(128), value[1, 0], value[1, 2]):      # neighbours are untouched
        assert torch.allclose(t, torch.ones_like(t), rtol=2.0 ** -22)


@pytest.mark.gpu
def test_out_buffers_and_strides(dev):
    """Rows written into a wider buffer leave its other columns alone; transposed and sliced inputs; row-major scales."""
    from nerffaceediting_amd import dense_ops
    g = torch.Generator().manual_seed(2)
    a, b = torch.randn(37, 256, generator=g), torch.randn(37, 130, generator=g)
    q = torch.full((37, 768), 3.0, device=dev).to(torch.float8_e4m3fn)
    scale = torch.full((37, 6), 7.0, device=dev)
    dense_ops.rms_norm_fp8(a.to(dev), out=(q, scale), out_offset=128)
    dense_ops.quantize_fp8(b.to(dev), out=(q, scale), out_offset=512)
    check_rows(q[:, 128:384], scale[:, 1:3], norm64(a, None, None)[0], 256)
    check_rows(q[:, 512:768], scale[:, 4:6], b.double(), 130, rel=2.0 ** -22)
    for lo, hi in ((0, 128), (384, 512)):
        assert bool((q[:, lo:hi].float() == 3).all()) and bool((scale[:, lo // 128:hi // 128] == 7).all())
    for x in (a.t().contiguous().to(dev).t(), torch.cat([a, a], 1).to(dev)[:, 256:], torch.cat([a.flatten()[:1], a.flatten()]).to(dev)[1:].view(37, 256)):
        for got, want in zip(dense_ops.quantize_fp8(x), dense_ops.quantize_fp8(a.to(dev))):
            assert torch.equal(got.float(), want.float())


def make_mm(m, n, k, seed=0):
    """Random e4m3 operands, all finite codes, with scales that differ by orders of magnitude: (q, scale, wq, w_scale) on the CPU."""
    g = torch.Generator().manual_seed(seed + m * 7 + n * 131 + k)
    code = lambda *s: torch.randint(0, 127, s, generator=g, dtype=torch.uint8) + 128 * torch.randint(0, 2, s, generator=g, dtype=torch.uint8)
    q = code(m, blocks(k) * BLOCK)
    q[:, k:] = 0
    wq = code(n, k)
    s = torch.exp(torch.randn(m, blocks(k), generator=g))
    ws = torch.exp(torch.randn(blocks(n), blocks(k), generator=g)) / 448
    return q.view(torch.float8_e4m3fn), s, wq.view(torch.float8_e4m3fn), ws


def mm64(q, s, wq, ws, dev):
    """(result, sum of the terms' magnitudes) in 64 bits, on the GPU for speed."""
    n, k = wq.shape
    a = q.to(dev).float().double().view(q.shape[0], -1, BLOCK) * s.to(dev).double()[..., None]
    a = a.view(q.shape[0], -1)[:, :k].contiguous()
    w = wq.to(dev).float().double() * ws.to(dev).double().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    w = w.t().contiguous()
    return a @ w, a.abs() @ w.abs()


def check_mm(got, want, mag, k, extra=None):
    block = 0.0 if got.dtype == torch.float32 else 7 * 2.0 ** -13
    tol = k * 2.0 ** -22 * (mag if extra is None else mag + extra) + block * mag + want.abs() * EPS[got.dtype] * 1.001 + TINY[got.dtype]
    err = (got.double() - want).abs()
    if got.dtype == torch.float16:                                           # beyond fp16's range: infinite
        over = want.abs() > 65504
        err, tol = err.masked_fill(over, 0), tol
        assert bool((got[over].float().abs() >= 65504).all())
    assert bool((err <= tol).all()), float((err - tol).max())


MM = [(1, 512, 1024), (1, 1, 1), (2, 3, 5), (16, 16, 128), (15, 17, 127), (17, 33, 129), (31, 500, 640), (33, 64, 256), (64, 512, 512), (65, 129, 1000),
      (100, 1000, 300), (128, 128, 128), (129, 257, 1031), (255, 256, 2048), (256, 255, 1920), (500, 513, 512), (1000, 100, 4096), (5, 4100, 8192),
      (1, 130, 20000), (300, 48, 16384), (1500, 1031, 384), (3, 8230, 300), (16, 16500, 1100), (20, 16500, 400)]


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", TYPES)
@pytest.mark.parametrize("m,n,k", MM)
def test_matmul(dev, m, n, k, out_dtype):
    from nerffaceediting_amd import dense_ops
    q, s, wq, ws = make_mm(m, n, k)
    if out_dtype == torch.float16:
        s = s * 1e-5
    W = dense_ops.fp8_weight_from(wq.to(dev), ws.to(dev))
    got = dense_ops.fp8_matmul(q.to(dev), s.t().contiguous().to(dev).t(), W, out_dtype=out_dtype)
    assert tuple(got.shape) == (m, n) and got.dtype == out_dtype
    want, mag = mm64(q, s, wq, ws, dev)
    check_mm(got, want, mag, k)
    again = dense_ops.fp8_matmul(q.to(dev), s.to(dev), W, out_dtype=out_dtype)          # row-major scales
    assert torch.equal(got, again)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (7, 30, 200), (64, 512, 512), (300, 515, 700)])
@pytest.mark.parametrize("bias,lrelu", [(True, False), (False, True), (True, True)])
def test_matmul_epilogue(dev, m, n, k, bias, lrelu):
    from nerffaceediting_amd import dense_ops
    q, s, wq, ws = make_mm(m, n, k, seed=1)
    b = torch.randn(n, generator=torch.Generator().manual_seed(4)) * 100
    W = dense_ops.fp8_weight_from(wq.to(dev), ws.to(dev))
    got = dense_ops.fp8_matmul(q.to(dev), s.to(dev), W, bias=b.to(dev) if bias else None, bias_gain=0.01, lrelu=lrelu)
    want, mag = mm64(q, s, wq, ws, dev)
    gain = float(torch.tensor(0.01))                                         # the fp32 number that the call passes on
    if bias:
        want = want + b.to(dev).double() * gain
    if lrelu:
        want = torch.where(want < 0, want * 0.2, want) * math.sqrt(2)
    check_mm(got, want, mag * 1.5, k, extra=b.abs().to(dev).double() if bias else None)


@pytest.mark.gpu
def test_matmul_rows_do_not_touch_each_other(dev):
    """NaN in one row's values or scale stays in that row; a NaN weight scale stays in its 128 outputs; strided q and rows beyond the last."""
    from nerffaceediting_amd import dense_ops
    m, n, k = 150, 300, 400
    q, s, wq, ws = make_mm(m, n, k, seed=2)
    W = dense_ops.fp8_weight_from(wq.to(dev), ws.to(dev))
    clean = dense_ops.fp8_matmul(q.to(dev), s.to(dev), W)
    raw = q.view(torch.uint8).clone()
    raw[7, 3] = 0x7F
    s2 = s.clone()
    s2[100, 2] = float("nan")
    got = dense_ops.fp8_matmul(raw.view(torch.float8_e4m3fn).to(dev), s2.to(dev), W)
    keep = torch.ones(m, dtype=torch.bool)
    keep[[7, 100]] = False
    assert bool(torch.isnan(got[~keep.to(dev)]).all()) and torch.equal(got[keep.to(dev)], clean[keep.to(dev)])
    ws2 = ws.clone()
    ws2[1, 0] = float("nan")
    got = dense_ops.fp8_matmul(q.to(dev), s.to(dev), dense_ops.fp8_weight_from(wq.to(dev), ws2.to(dev)))
    assert bool(torch.isnan(got[:, 128:256]).all()) and torch.equal(got[:, :128], clean[:, :128]) and torch.equal(got[:, 256:], clean[:, 256:])
    wide = torch.full((m + 9, 1024), float("nan"), device=dev).to(torch.float8_e4m3fn)
    wide[3:m + 3, 256:768] = q.to(dev)
    assert torch.equal(dense_ops.fp8_matmul(wide[3:m + 3, 256:768], s.to(dev), W), clean)
    q5, s5 = q.to(dev)[:1].expand(5, -1), s.to(dev)[:1].expand(5, -1)
    assert torch.equal(dense_ops.fp8_matmul(q5, s5, W), dense_ops.fp8_matmul(q5.contiguous(), s5.contiguous(), W))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(512, 1024), (1, 1), (130, 129), (48, 700), (257, 128)])
def test_weight_quantisation(dev, n, k, dtype):
    """The packed values are read back by multiplying with unit rows."""
    from nerffaceediting_amd import dense_ops
    g = torch.Generator().manual_seed(n + k)
    w = (torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(dtype)
    W = dense_ops.fp8_weight(w.to(dev), gain=0.25)
    full = torch.zeros(blocks(n) * BLOCK, blocks(k) * BLOCK, dtype=torch.float64)
    full[:n, :k] = w.double()
    want = full.view(blocks(n), BLOCK, blocks(k), BLOCK).abs().amax((1, 3)).clamp_min(1e-30) / 448
    assert bool(((W.scale.double().cpu() - want * 0.25).abs() <= want * 2.0 ** -23).all())
    eye = torch.zeros(blocks(k) * BLOCK, blocks(k) * BLOCK).fill_diagonal_(1.0).to(torch.float8_e4m3fn)
    got = dense_ops.fp8_matmul(eye.to(dev), torch.ones(blocks(k) * BLOCK, blocks(k), device=dev), W).double().cpu().t()
    ref = want.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    err = (got[:, :k] * 4 - w.double()).abs()
    assert bool((err <= w.double().abs() * (2.0 ** -4 + 2.0 ** -20) + ref * (2.0 ** -10 + 448 * 2.0 ** -22)).all())
    assert not bool(got[:, k:].any())


@pytest.mark.gpu
def test_empty_rows(dev):
    from nerffaceediting_amd import dense_ops
    W = dense_ops.fp8_weight(torch.ones(20, 30, device=dev))
    q, s = dense_ops.rms_norm_fp8(torch.empty(0, 30, device=dev))
    assert tuple(q.shape) == (0, 128) and tuple(s.shape) == (0, 1)
    assert tuple(dense_ops.fp8_matmul(q, s, W).shape) == (0, 20)
    q, s, h = dense_ops.rms_norm_fp8(torch.empty(0, 30, device=dev), residual=torch.empty(0, 30, device=dev))
    assert tuple(h.shape) == (0, 30)


@pytest.mark.gpu
def test_layers_together_stream_and_graph(dev):
    """norm -> product -> quantise -> product as a mapping network runs them: against the same steps in 64 bits on the kernels' own 8-bit
    values, on another stream, and replayed from two graphs with eager work between."""
    from nerffaceediting_amd import dense_ops
    g = torch.Generator().manual_seed(9)
    w1, w2 = torch.randn(384, 512, generator=g).to(dev), torch.randn(512, 384, generator=g).to(dev)
    b1 = torch.randn(384, generator=g).to(dev)
    W1, W2 = dense_ops.fp8_weight(w1, gain=1 / math.sqrt(512)), dense_ops.fp8_weight(w2, gain=1 / math.sqrt(384))

    def layers(x):
        q, s = dense_ops.rms_norm_fp8(x)
        y = dense_ops.fp8_matmul(q, s, W1, bias=b1, lrelu=True)
        q2, s2 = dense_ops.quantize_fp8(y)
        return q, s, y, q2, s2, dense_ops.fp8_matmul(q2, s2, W2, out_dtype=torch.bfloat16)

    def weights64(W, n, k):
        eye = torch.zeros(k, k, device=dev).fill_diagonal_(1.0).to(torch.float8_e4m3fn)
        return dense_ops.fp8_matmul(eye, torch.ones(k, k // 128, device=dev), W).double()

    x = torch.randn(70, 512, generator=g).to(dev)
    q, s, y, q2, s2, out = layers(x)
    a = q.float().double().view(70, -1, 128) * s.double()[..., None]
    a, u1, u2 = a.view(70, -1), weights64(W1, 384, 512), weights64(W2, 512, 384)
    want = a @ u1 + b1.double()
    want = torch.where(want < 0, want * 0.2, want) * math.sqrt(2)
    check_mm(y, want, (a.abs() @ u1.abs()) * 1.5 + b1.double().abs(), 512)
    a2 = (q2.float().double().view(70, -1, 128) * s2.double()[..., None]).view(70, -1)
    check_mm(out, a2 @ u2, a2.abs() @ u2.abs(), 384)

    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = layers(x)[-1]
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(other, out)
    bufs = [torch.empty_like(x), torch.empty_like(x)]
    graphs, outs = [], []
    for b in bufs:
        b.copy_(x)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(layers(b)[-1])
        graphs.append(gr)
    for i in range(4):
        new = [torch.randn(70, 512, generator=g).to(dev) for _ in bufs]
        for b, n, gr in zip(bufs, new, graphs):
            b.copy_(n)
            gr.replay()
        for n, o in zip(new, outs):
            want = layers(n)[-1]
            torch.cuda.synchronize()
            assert torch.equal(o, want)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 5, 300])
def test_mapping_network_fp8(dev, n):
    """MappingNetwork(fc_math='fp8') against its own fp32 path.  Elementwise bound, layer by layer: operands are off by 2^-4 relative (plus
    2^-10 of a block's scale, max / 448) each, so a layer's sum by (2 * 2^-4 + 2^-8) sum|x||w| and the floors; the typical error is far
    below that, and its norm is held to 6 %: 2^-4 / sqrt(3) an operand is 3.6 %, two operands a layer in quadrature 5.1 % if every value sat
    at the start of its binade; two layers of independent errors then stay under 7.3 %, and uniform mantissas halve the variance."""
    from nerffaceediting_amd.training.networks_stylegan2 import MappingNetwork
    torch.manual_seed(0)
    ref = MappingNetwork(512, 25, 512, 14, num_layers=2).to(dev)
    m = MappingNetwork(512, 25, 512, 14, num_layers=2, fc_math="fp8").to(dev)
    m.load_state_dict(ref.state_dict())
    z, c = torch.randn(n, 512, device=dev), torch.randn(n, 25, device=dev)
    want, got = ref(z, c), m(z, c)
    assert got.shape == want.shape == (n, 14, 512) and got.dtype == torch.float32
    err = float((got - want).norm() / want.norm())
    assert 1e-4 < err < 0.06, err
    assert torch.equal(m(z[:1], c[:1]), m(z, c)[:1]) or n > 16        # batch sizes that run the same kernel agree to the bit
    with torch.no_grad():
        m.fc0.weight.mul_(2.0)                                       # the packed image follows the parameter
    ref.load_state_dict(m.state_dict())
    assert float((m(z, c) - ref(z, c)).norm() / ref(z, c).norm()) < 0.06
    t = m(z, c, truncation_psi=0.5, truncation_cutoff=7)
    assert torch.allclose(t[:, 7:], m(z, c)[:, 7:]) and torch.allclose(t[:, :7], m(z, c)[:, :7] * 0.5)


@pytest.mark.gpu
def test_refusals(dev):
    from nerffaceediting_amd import dense_ops
    x = torch.ones(4, 200, device=dev)
    W = dense_ops.fp8_weight(torch.ones(20, 200, device=dev))
    q, s = dense_ops.quantize_fp8(x)
    for bad in (x.double(), x.int()):
        with pytest.raises(RuntimeError, match="expected float32"):
            dense_ops.quantize_fp8(bad)
    with pytest.raises(AssertionError, match="wrong shape"):
        dense_ops.rms_norm_fp8(x, weight=torch.ones(100, device=dev))
    with pytest.raises(AssertionError, match="wrong shape"):
        dense_ops.rms_norm_fp8(x, residual=torch.ones(4, 100, device=dev))
    with pytest.raises(RuntimeError, match="residual"):
        dense_ops.rms_norm_fp8(x, residual=x.half())
    for eps in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            dense_ops.rms_norm_fp8(x, eps=eps)
    with pytest.raises(RuntimeError, match="no gradient"):
        dense_ops.rms_norm_fp8(x.clone().requires_grad_(True))
    with torch.no_grad():
        dense_ops.rms_norm_fp8(x.clone().requires_grad_(True))
    for out, off in (((q, s), 64), ((q, s), 128), ((q[:, :128], s), 0), ((q, s[:, :1]), 0), ((q.float(), s), 0)):
        with pytest.raises(ValueError, match="out must be"):
            dense_ops.quantize_fp8(x, out=out, out_offset=off)
    with pytest.raises(TypeError, match="Fp8Weight"):
        dense_ops.fp8_matmul(q, s, x)
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        dense_ops.fp8_matmul(q.float(), s, W)
    with pytest.raises(AssertionError, match="wrong shape"):
        dense_ops.fp8_matmul(q[:, :128], s, W)
    with pytest.raises(RuntimeError, match="scale"):
        dense_ops.fp8_matmul(q, s[:, :1], W)
    with pytest.raises(RuntimeError, match="out_dtype"):
        dense_ops.fp8_matmul(q, s, W, out_dtype=torch.float64)
    with pytest.raises(AssertionError, match="bias"):
        dense_ops.fp8_matmul(q, s, W, bias=torch.ones(21, device=dev))
    with pytest.raises(ValueError, match="empty weight"):
        dense_ops.fp8_weight(torch.ones(0, 5, device=dev))
    with pytest.raises(AssertionError, match="scale"):
        dense_ops.fp8_weight_from(q, s[:2])


def test_refusals_without_a_gpu():
    import ctypes
    from nerffaceediting_amd import _lib, dense_ops
    from nerffaceediting_amd.training.networks_stylegan2 import MappingNetwork
    x = torch.ones(4, 200)
    for call in (lambda: dense_ops.rms_norm_fp8(x), lambda: dense_ops.quantize_fp8(x), lambda: dense_ops.fp8_weight(x),
                 lambda: dense_ops.fp8_weight_from(x.to(torch.float8_e4m3fn), torch.ones(1, 2))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(ValueError, match="multiples of 128"):
        MappingNetwork(100, 25, 512, 14, fc_math="fp8")
    with pytest.raises(ValueError, match="fc_math"):
        MappingNetwork(512, 25, 512, 14, fc_math="int4")
    lib = _lib.load()
    assert lib.nfe_fp8_weight_bytes(17, 129) == 2 * 2 * 2048 and lib.nfe_fp8_weight_bytes(0, 5) == 0
    err = lib.nfe_last_error
    assert lib.nfe_fp8_matmul(None, None) == -1 and b"args is null" in err()
    a = _lib.Fp8MatmulArgs()
    a.struct_size = 8
    assert lib.nfe_fp8_matmul(ctypes.byref(a), None) == -1 and b"struct_size" in err()

    def matmul(**kw):
        a = _lib.Fp8MatmulArgs()
        a.struct_size, a.m, a.n, a.k, a.q, a.q_stride, a.scale, a.packed, a.w_scale, a.out = ctypes.sizeof(a), 4, 8, 200, 4096, 256, 64, 4096, 64, 64
        for name, v in kw.items():
            setattr(a, name, v)
        return lib.nfe_fp8_matmul(ctypes.byref(a), None)

    for kw, word in ((dict(q=None), b"null"), (dict(m=0), b"m=0"), (dict(n=0), b"bad sizes"), (dict(q_stride=200), b"aligned"), (dict(q=4100), b"aligned"),
                     (dict(out_dtype=5), b"out_dtype"), (dict(out=65), b"misaligned")):
        assert matmul(**kw) == -1 and word in err(), (kw, err())
    norm = lambda rows=2, cols=200, dtype=0, res=None, h=None, q=4096, stride=256, eps=1e-8: lib.nfe_rms_norm_fp8(64, res, None, dtype, rows, cols, eps, h, q,
                                                                                                               stride, 64, 1, 2, None)
    for kw, word in ((dict(rows=0), b"rows"), (dict(cols=0), b"cols"), (dict(dtype=9), b"dtype"), (dict(res=64), b"pairs"), (dict(stride=200), b"at least"),
                     (dict(stride=260), b"aligned"), (dict(q=4097), b"aligned"), (dict(q=None), b"null"), (dict(eps=0.0), b"eps")):
        assert norm(**kw) == -1 and word in err(), (kw, err())


@pytest.mark.gpu
def test_mapping_network_fp8_weight_image(dev):
    """The packed image follows the parameter: in-place change, replaced storage, and a first call inside a graph capture."""
    from nerffaceediting_amd.training.networks_stylegan2 import FullyConnectedLayer
    from nerffaceediting_amd import dense_ops
    torch.manual_seed(3)
    layer = FullyConnectedLayer(256, 130).to(dev)
    q, s = dense_ops.quantize_fp8(torch.randn(9, 256, device=dev))
    want = lambda: dense_ops.fp8_matmul(q, s, dense_ops.fp8_weight(layer.weight.detach(), gain=layer.weight_gain), layer.bias.detach(), layer.bias_gain)
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer.forward_fp8(q, s)
    assert torch.equal(layer.forward_fp8(q, s), want())                # the capture ran nothing
    for i in range(3):
        with torch.no_grad():
            layer.weight.mul_(1.5)
        g.replay()
        ref = want()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(layer.forward_fp8(q, s), ref)
    for _ in range(2):
        layer.weight.data = torch.randn(130, 256, device=dev)
    assert torch.equal(layer.forward_fp8(q, s), want())
    layer.weight = torch.nn.Parameter(torch.randn(130, 256, device=dev))
    assert torch.equal(layer.forward_fp8(q, s), want())


@pytest.mark.gpu
def test_many_rows_and_wide_strides(dev):
    """More rows than one launch of the norm takes (2^22), and row strides beyond what a tile's 32-bit offsets reach (2^23 bytes)."""
    from nerffaceediting_amd import dense_ops
    rows = (1 << 22) + 37
    x = torch.randn(rows, 9, device=dev, dtype=torch.bfloat16)
    q, s = dense_ops.quantize_fp8(x)
    at = torch.tensor([0, 1, (1 << 22) - 1, 1 << 22, (1 << 22) + 1, rows - 1], device=dev)
    check_rows(q[at], s[at], x[at].double().cpu(), 9, rel=2.0 ** -22)
    m, n, k, stride = 130, 70, 300, (1 << 23) + 16
    qs, ss, wq, ws = make_mm(m, n, k, seed=5)
    store = torch.zeros(m * stride, dtype=torch.uint8, device=dev)
    wide = store.as_strided((m, 384), (stride, 1))
    wide.copy_(qs.view(torch.uint8))
    W = dense_ops.fp8_weight_from(wq.to(dev), ws.to(dev))
    got = dense_ops.fp8_matmul(wide.view(torch.float8_e4m3fn), ss.to(dev), W)
    want, mag = mm64(qs, ss, wq, ws, dev)
    check_mm(got, want, mag, k)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 7])
def test_rows_at_any_address(dev, rows):
    """Contiguous rows that begin anywhere (a view into a byte buffer) are copied where the kernel needs 16-byte alignment."""
    from nerffaceediting_amd import dense_ops
    q, s, wq, ws = make_mm(rows, 40, 300)
    W = dense_ops.fp8_weight_from(wq.to(dev), ws.to(dev))
    want = dense_ops.fp8_matmul(q.to(dev), s.to(dev), W)
    for start in (1, 8, 15, 16):
        flat = torch.full((start + q.numel() + 16,), 0x7F, dtype=torch.uint8, device=dev)
        view = flat[start:start + q.numel()].view(q.shape)
        view.copy_(q.view(torch.uint8))
        assert torch.equal(dense_ops.fp8_matmul(view.view(torch.float8_e4m3fn), s.to(dev), W), want), start


@pytest.mark.gpu
def test_sizes_beyond_the_library_are_refused(dev):
    """Widths that a 32-bit argument would take for smaller ones: refused before anything is copied or allocated (expanded rows hold one value)."""
    from nerffaceediting_amd import dense_ops
    one = torch.ones(1, 1, device=dev, dtype=torch.bfloat16)
    free = torch.cuda.mem_get_info(dev)[0]
    for cols in ((1 << 30) + 1, (1 << 32) + 1):
        wide = one.expand(1, cols)
        for call in (lambda: dense_ops.quantize_fp8(wide), lambda: dense_ops.rms_norm_fp8(wide), lambda: dense_ops.rms_norm_fp8(wide, residual=wide),
                     lambda: dense_ops.fp8_weight(wide), lambda: dense_ops.fp8_weight(wide.t()),
                     lambda: dense_ops.fp8_weight_from(one.to(torch.float8_e4m3fn).expand(1, cols), torch.ones(1, 1, device=dev))):
            with pytest.raises(ValueError, match="at most"):
                call()
    for rows in (1 << 31, (1 << 32) + 1):
        with pytest.raises(ValueError, match="at most"):
            dense_ops.quantize_fp8(one.expand(rows, 1))
    W = dense_ops.fp8_weight(torch.ones(3, 5, device=dev))
    rows = (1 << 30) + 1
    q = torch.zeros(1, 128, device=dev).to(torch.float8_e4m3fn).expand(rows, 128)
    with pytest.raises(ValueError, match="at most"):
        dense_ops.fp8_matmul(q, torch.ones(1, 1, device=dev).expand(rows, 1), W)
    assert free - torch.cuda.mem_get_info(dev)[0] < 1 << 30


def test_weight_objects_are_checked_when_made():
    """Fp8Weight's sizes say how far the kernel reads: buffers that do not hold them are refused."""
    from nerffaceediting_amd.dense_ops import Fp8Weight
    packed, scale = torch.zeros(3 * 2 * 2048, dtype=torch.uint8), torch.ones(1, 2)
    assert Fp8Weight(packed, scale, 33, 200).in_features == 200
    for bad in ((packed, scale, 49, 200), (packed, scale, 32, 200), (packed, scale, 33, 257), (packed[1:], scale, 33, 200), (packed.float(), scale, 33, 200),
                (packed, scale[:, :1], 33, 200), (packed, scale.double(), 33, 200), (packed, torch.ones(2, 2)[:, :1].expand(2, 2)[:1], 33, 200),
                (packed, torch.ones(1, 4)[:, ::2], 33, 200), (torch.zeros(2 * packed.numel(), dtype=torch.uint8)[::2], scale, 33, 200),
                (packed, scale, 0, 200), (packed, scale, 33, -200), (packed.tolist(), scale, 33, 200)):
        with pytest.raises((ValueError, TypeError), match="Fp8Weight"):
            Fp8Weight(*bad)


@pytest.mark.gpu
def test_smallest_eps(dev):
    """The reciprocal root's instruction takes subnormal numbers for zero: eps is at least the smallest normal number, and works there."""
    from nerffaceediting_amd import dense_ops
    x = torch.zeros(3, 200, device=dev)
    x[1] = 2.0 ** -70
    q, s = dense_ops.rms_norm_fp8(x, eps=2.0 ** -126)
    check_rows(q, s, norm64(x, None, None, eps=2.0 ** -126)[0], 200)
    for eps in (2.0 ** -127, 1e-40, 1e-50):
        with pytest.raises(ValueError, match="eps"):
            dense_ops.rms_norm_fp8(x, eps=eps)


def test_smallest_eps_of_the_library():
    from nerffaceediting_amd import _lib
    lib = _lib.load()
    for eps in (2.0 ** -127, 1e-45, float("nan")):
        assert lib.nfe_rms_norm_fp8(64, None, None, 0, 2, 200, eps, None, 4096, 256, 64, 1, 2, None) == -1 and b"eps" in lib.nfe_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [384, 700, 5000])
def test_special_values_in_the_norm(dev, cols):
    """The formula's: a NaN makes the mean and so its whole row NaN; an infinity makes its own block NaN (infinity times zero) and the row's
    other blocks zero; squares whose sum leaves fp32 make the row zero; a NaN weight makes its block of every row NaN."""
    from nerffaceediting_amd import dense_ops
    x = torch.ones(6, cols, device=dev)
    x[1, 200], x[2, 5], x[3, cols - 1] = float("inf"), float("nan"), -float("inf")
    x[4] = 1e25
    q, scale = dense_ops.rms_norm_fp8(x)
    bad = torch.isnan(q.float().view(6, -1, BLOCK) * scale[..., None]).cpu()
    want = torch.zeros(6, blocks(cols), dtype=torch.bool)
    want[1, 1], want[2], want[3, blocks(cols) - 1] = True, True, True
    assert torch.equal(bad.all(-1), want) and torch.equal(bad.any(-1), want)
    value = (q.float().view(6, -1, BLOCK) * scale[..., None]).cpu()
    for row in (1, 3):
        assert not bool(value[row][~want[row]].any())
    assert not bool(value[4].any()) and bool(torch.isfinite(scale[4]).all())
    for row in (0, 5):
        check_rows(q[row:row + 1], scale[row:row + 1], norm64(x[row:row + 1].cpu(), None, None)[0], cols)
    weight = torch.ones(cols, device=dev)
    weight[130] = float("nan")
    q, scale = dense_ops.rms_norm_fp8(x[:1], weight)
    bad = torch.isnan(q.float().view(-1, BLOCK) * scale[0][:, None])
    assert bool(bad[1].all()) and not bool(bad[0].any()) and not bool(bad[2:].any())
