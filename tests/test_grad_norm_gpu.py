"""Gradient norm and clipping (nfe_grad_norm / nfe_grad_clip) against sums in 64 bits.

Tolerances.  The norm is formed in fp64 and rounded to fp32 once: half a step, 2^-24 relative, plus the fp64 sums' own 2^-53 a term.
A scaled gradient is g * f with f rounded to fp32 (2^-24), the product rounded to fp32 (2^-24) and then to the gradient's type (2^-24,
2^-8, 2^-11); results under the type's smallest normal number are off by half of its smallest step instead."""
import math

import pytest
import torch

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
NORM_TOL = 2.0 ** -23


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def make(dev, sizes, types, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale * 2.0 ** (i % 5 - 2)).to(types[i % len(types)]).to(dev) for i, n in enumerate(sizes)]


def true_norm(ts):
    return math.sqrt(sum(float(t.double().cpu().square().sum()) for t in ts))


def check_clipped(got, before, norm, max_norm):
    f = min(1.0, max_norm / (norm + 1e-6))
    for a, b in zip(got, before):
        if f == 1.0:
            assert torch.equal(a, b)
            continue
        want = b.double().cpu() * f
        err = (a.double().cpu() - want).abs()
        tol = want.abs() * (EPS[b.dtype] * 1.001 + 2.0 ** -22) + TINY[b.dtype]
        assert bool((err <= tol).all()), (b.dtype, b.shape, float((err - tol).max()))


CASES = [
    [1], [0, 1, 0], [3], [192], [255, 256, 257], [4095, 4096, 4097], [16383, 16384, 16385], [1 << 20], [5] * 257, [7, 0, 70001] * 110, [3_000_001, 17],
]


@pytest.mark.gpu
@pytest.mark.parametrize("types", [[torch.float32], [torch.bfloat16], [torch.float16], [torch.float32, torch.bfloat16, torch.float16]])
@pytest.mark.parametrize("sizes", CASES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_clip(dev, sizes, types):
    from nerffaceediting_amd import ops
    ts = make(dev, sizes, types)
    norm = true_norm(ts)
    got = ops.grad_norm(ts)
    assert got.dtype == torch.float32 and got.shape == () and got.device == dev
    assert abs(float(got) - norm) <= NORM_TOL * norm
    biggest = max((float(t.double().abs().max()) for t in ts if t.numel()))
    assert float(ops.grad_norm(ts, float("inf"))) == biggest
    for limit in (0.3 * norm, 10.0 * norm):
        mine = [t.clone() for t in ts]
        ret = ops.clip_grad_norm(mine, limit)
        assert float(ret) == float(got)                              # same list, same bits
        check_clipped(mine, ts, norm, limit)
    mine = [t.clone() for t in ts]
    ops.clip_grad_norm(mine, 0.25 * biggest, norm_type=float("inf"))
    check_clipped(mine, ts, biggest, 0.25 * biggest)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_unaligned_views_of_a_bucket(dev, dtype):
    """Views that start at every offset within 16 bytes; what lies between them stays as it was."""
    from nerffaceediting_amd import ops
    g = torch.Generator().manual_seed(3)
    flat = torch.randn(40000, generator=g).to(dtype).to(dev)
    before = flat.clone()
    spans, at = [], 0
    for i in range(24):
        n = (1, 2, 7, 8, 9, 31, 1023, 4097)[i % 8]
        spans.append((at + 1, at + 1 + n))
        at += n + 2
    views = [flat[a:b] for a, b in spans]
    old = [v.clone() for v in views]
    norm = true_norm(old)
    assert abs(float(ops.clip_grad_norm(views, 0.4 * norm)) - norm) <= NORM_TOL * norm
    check_clipped(views, old, norm, 0.4 * norm)
    outside = torch.ones(flat.numel(), dtype=torch.bool)
    for a, b in spans:
        outside[a:b] = False
    assert torch.equal(flat.cpu()[outside], before.cpu()[outside])


@pytest.mark.gpu
def test_layouts_and_none_entries(dev):
    from nerffaceediting_amd import ops
    a = torch.randn(5, 7, 3, device=dev).permute(2, 0, 1)              # fills one stretch of memory
    b = torch.randn(8, 6, 4, 5, device=dev).contiguous(memory_format=torch.channels_last)
    c = torch.randn(10, 12, device=dev)[:, ::2]                        # does not
    d = torch.ones(4, 1, device=dev).expand(4, 6)
    want = true_norm([a, b, c, d])
    assert abs(float(ops.grad_norm([a, None, b, c, d])) - want) <= NORM_TOL * want
    assert float(ops.grad_norm(a)) == pytest.approx(true_norm([a]), rel=NORM_TOL)
    old, norm = [a.clone(), b.clone()], true_norm([a, b])
    ops.clip_grad_norm((t for t in (a, None, b)), 0.5 * norm)
    check_clipped([a, b], old, norm, 0.5 * norm)
    for bad in (c, d):
        with pytest.raises(RuntimeError, match="one stretch of memory"):
            ops.clip_grad_norm([bad], 1.0)


@pytest.mark.gpu
def test_range_and_special_values(dev):
    """fp64 sums: squares far outside fp32's range count; infinities and NaN behave as in torch.nn.utils.clip_grad_norm_."""
    from nerffaceediting_amd import ops
    big, small = torch.full((5000,), 1e30, device=dev), torch.full((5000,), 1e-30, device=dev)
    for t in (big, small):
        want = true_norm([t])
        assert abs(float(ops.grad_norm([t])) - want) <= NORM_TOL * want
    zero = torch.zeros(100, device=dev)
    assert float(ops.clip_grad_norm([zero], 1.0)) == 0.0 and not bool(zero.any())
    t = torch.ones(300, device=dev)
    ops.clip_grad_norm([t], 0.0)
    assert not bool(t.any())
    for value, norm_type in ((float("inf"), 2), (float("nan"), 2), (float("inf"), float("inf")), (float("nan"), float("inf"))):
        x, y = torch.ones(70, device=dev), torch.ones(20000, device=dev, dtype=torch.bfloat16)
        x[13] = value
        p = [torch.nn.Parameter(torch.zeros_like(v)) for v in (x, y)]
        p[0].grad, p[1].grad = x.clone(), y.clone()
        want = torch.nn.utils.clip_grad_norm_(p, 1.0, norm_type=norm_type)
        got = ops.clip_grad_norm([x, y], 1.0, norm_type=norm_type)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
        for mine, ref in zip((x, y), p):
            assert torch.allclose(mine.float(), ref.grad.float(), equal_nan=True, rtol=0, atol=0)


@pytest.mark.gpu
def test_streams_graph_and_version(dev):
    """A captured clip replays with new gradients, beside eager calls on another stream; in-place writes count as such for autograd."""
    from nerffaceediting_amd import ops
    ts = make(dev, [70001, 300, 5], [torch.float32, torch.bfloat16])
    v = [t._version for t in ts]
    ops.clip_grad_norm([t.clone() for t in ts], 1.0)
    ops.clip_grad_norm(ts, 1e9)
    assert [t._version for t in ts] == [x + 1 for x in v]
    fresh = [make(dev, [70001, 300, 5], [torch.float32, torch.bfloat16], seed=10 + i) for i in range(4)]
    bufs = [torch.empty_like(t) for t in ts]
    for b, t in zip(bufs, ts):
        b.copy_(t)
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        ops.clip_grad_norm(bufs, 2.0)
    torch.cuda.current_stream(dev).wait_stream(side)
    graphs, norms = [], []
    for limit in (2.0, 3.0):                                           # two graphs over the same buffers
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(ops.clip_grad_norm(bufs, limit))
        graphs.append(g)
    for set_ in fresh:
        for g, n, limit in zip(graphs, norms, (2.0, 3.0)):
            for b, t in zip(bufs, set_):
                b.copy_(t)
            g.replay()
            eager = [t.clone() for t in set_]
            want = ops.clip_grad_norm(eager, limit)
            torch.cuda.synchronize()
            assert float(n) == float(want)
            assert all(torch.equal(a, b) for a, b in zip(bufs, eager))


@pytest.mark.gpu
def test_more_than_2_31_values(dev):
    """Offsets beyond 32 bits: 2^31 + 12345 bf16 values, the last one the only large one."""
    from nerffaceediting_amd import ops
    n = (1 << 31) + 12345
    t = torch.zeros(n, device=dev, dtype=torch.bfloat16)
    t[-1], t[n // 2], t[0] = 4.0, 2.0, -4.0
    assert float(ops.clip_grad_norm([t], 3.0)) == 6.0
    f = 3.0 / (6.0 + 1e-6)
    for i, x in ((-1, 4.0), (n // 2, 2.0), (0, -4.0)):
        assert abs(float(t[i]) - x * f) <= abs(x * f) * 2.0 ** -8
    assert float(ops.grad_norm([t], float("inf"))) == 2.0


@pytest.mark.gpu
def test_refusals(dev):
    from nerffaceediting_amd import ops
    t = torch.ones(10, device=dev)
    with pytest.raises(RuntimeError, match="share memory"):
        ops.clip_grad_norm([t, t], 1.0)
    with pytest.raises(RuntimeError, match="share memory"):
        ops.clip_grad_norm([t[:6], t[5:]], 1.0)
    assert float(ops.grad_norm([t, t])) == pytest.approx(math.sqrt(20.0), rel=NORM_TOL)        # reading twice is fine
    for bad in (-1.0, float("nan")):
        with pytest.raises(RuntimeError, match="max_norm"):
            ops.clip_grad_norm([t], bad)
    with pytest.raises(RuntimeError, match="float64"):
        ops.grad_norm([t.double()])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.grad_norm([t, t.cpu()])
    with pytest.raises(RuntimeError, match="autograd graph"):
        ops.clip_grad_norm([t.clone().requires_grad_(True) * 2], 1.0)
    assert float(t.sum()) == 10.0


@pytest.mark.gpu
@pytest.mark.parametrize("optimize", ["norm", "stats"])
def test_optimize_planes_clips_before_the_step(dev, optimize, monkeypatch):
    """The editing loop with max_grad_norm: Adam sees gradients whose joint norm is at most the limit, and they are the loss's own
    gradients scaled."""
    from nerffaceediting_amd import editing, utils

    def decode(G, ws, cam, norm, denorm, **kw):
        return {"image_raw": denorm}

    monkeypatch.setattr(utils, "decode", decode)
    seen = []
    real = torch.optim.Adam.step

    def step(self, *a, **k):
        seen.append([p.grad.clone() for g in self.param_groups for p in g["params"]])
        return real(self, *a, **k)

    monkeypatch.setattr(torch.optim.Adam, "step", step)
    g = torch.Generator().manual_seed(1)
    norm = torch.randn(1, 3, 32, 8, 8, generator=g).to(dev)
    mean, var = torch.randn(1, 3, 32, 1, 1, generator=g).to(dev), torch.rand(1, 3, 32, 1, 1, generator=g).to(dev) + 0.5
    kw = dict(steps=2, lr=0.01, optimize=optimize)
    loss = lambda out: (out["image_raw"] ** 2).sum()
    editing.optimize_planes(None, None, None, norm, mean, var, loss, **kw)
    free, seen[:] = list(seen[:1]), []
    editing.optimize_planes(None, None, None, norm, mean, var, loss, max_grad_norm=0.5, **kw)
    assert all(true_norm(s) <= 0.5 * (1 + 2.0 ** -20) for s in seen) and len(seen) == 2
    check_clipped(seen[0], free[0], true_norm(free[0]), 0.5)


def test_refusals_without_a_gpu():
    import ctypes
    from nerffaceediting_amd import _lib, ops
    with pytest.raises(ValueError, match="no tensors"):
        ops.grad_norm([])
    with pytest.raises(ValueError, match="no tensors"):
        ops.clip_grad_norm([None], 1.0)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.clip_grad_norm([torch.ones(3)], 1.0)
    with pytest.raises(TypeError):
        ops.grad_norm([1.0])
    with pytest.raises(ValueError, match="norm_type"):
        ops.grad_norm([torch.ones(3)], norm_type=1)
    lib = _lib.load()
    assert lib.nfe_grad_workspace_bytes(0) == 0 and lib.nfe_grad_workspace_bytes(1000) >= lib.nfe_grad_workspace_bytes(1) > 0
    one = lambda c, v: (c * 1)(v)
    args = lambda p=64, n=4, t=0, count=1: (one(ctypes.c_uint64, p), one(ctypes.c_int64, n), one(ctypes.c_int32, t), count)
    for bad, word in ((args(n=-1), b"elements"), (args(n=1 << 40), b"elements"), (args(t=3), b"dtype"), (args(p=66), b"misaligned"), (args(p=0), b"null"),
                      (args(count=0), b"count")):
        assert lib.nfe_grad_norm(*bad, 0, 256, 256, 1 << 30, None) == -1 and word in lib.nfe_last_error()
    assert lib.nfe_grad_norm(*args(), 7, 256, 256, 1 << 30, None) == -1 and b"norm_type" in lib.nfe_last_error()
    assert lib.nfe_grad_norm(*args(), 0, 256, 256, 8, None) == -3 and b"workspace" in lib.nfe_last_error()
    assert lib.nfe_grad_clip(*args(), 0, -1.0, 256, 256, 1 << 30, None) == -1 and b"max_norm" in lib.nfe_last_error()
    two = ((ctypes.c_uint64 * 2)(64, 72), (ctypes.c_int64 * 2)(4, 4), (ctypes.c_int32 * 2)(0, 0), 2)
    assert lib.nfe_grad_clip(*two, 0, 1.0, 256, 256, 1 << 30, None) == -1 and b"share memory" in lib.nfe_last_error()


@pytest.mark.gpu
def test_clipping_leaves_the_render_calls_status_alone(dev):
    """optimize_planes clips between the backward and the callback: what ops.render and ops.render_backward left for
    render_call_status() and render_handoff_aborts() stays, a clean status and a lost hand-off alike."""
    from nerffaceediting_amd import ops
    from tests.test_render_backward_gpu import _editing_size_case
    args, kw = _editing_size_case(dev)                                   # one forward
    grads = [g for g in ops.render_backward(*args, need=(True, True), **kw)]
    small, many = torch.ones(5, device=dev), [torch.ones(9000, device=dev) for _ in range(300)]

    def clip_all():
        for norm_type in (2, float("inf")):
            ops.grad_norm(grads, norm_type)
            ops.clip_grad_norm([small] + grads, 1.0, norm_type)
            ops.clip_grad_norm(many, 1e-3, norm_type)

    def lost():
        return [ops.render_handoff_aborts(backward=b) for b in (False, True)]

    clip_all()
    assert lost() == [0, 0]
    ops.render_call_status()
    ops.render_call_status(backward=True)
    words = ops._workspaces[(0, ops._stream())].view(torch.int32)
    planted = words[:64].clone()
    words[0], words[2], words[6] = 5, 3, 4                               # the counts of a forward's two passes and of a backward
    before = lost()
    assert all(before)
    clip_all()
    assert lost() == before
    with pytest.raises(RuntimeError, match="hand-offs"):
        ops.render_call_status()
    words[:64].copy_(planted)
    assert lost() == [0, 0]


@pytest.mark.gpu
def test_two_threads_on_one_stream(dev):
    """Calls from two host threads interleave their launches on the stream that they share: each scales by its own norm."""
    import threading
    from nerffaceediting_amd import ops
    n, rounds, bad = 40000, 300, []

    def work(value):
        t = torch.full((n,), value, device=dev)
        norm, got = value * math.sqrt(n), []
        for _ in range(rounds):
            g = t.clone()
            got.append((ops.clip_grad_norm([g], 0.5 * norm), g[0], g[-1]))
        for total, a, b in got:
            for x, want in ((total, norm), (a, 0.5 * value), (b, 0.5 * value)):
                if abs(float(x) - want) > 2.0 ** -20 * want:
                    bad.append((value, float(x), want))

    threads = [threading.Thread(target=work, args=(v,)) for v in (1.0, 64.0)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad[:3]
