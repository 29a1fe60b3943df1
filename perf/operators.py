"""Measured cases of the 8-bit dense operators and of gradient clipping: each in a plain form (elementary torch operations) and as the
calls a user makes of nerffaceediting_amd.

    norm   RMS norm (optional residual addition and weight) with an e4m3 output and a scale for every 128 columns
    mm     product of such rows with e4m3 weights that carry a scale for every 128 x 128 block, bias and activation
    clip   global 2-norm of the gradients in a list of tensors, and clipping in place
"""
import math
import random

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
SMALLEST = 1e-30
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # the mapping network's own norm at the batch of one interactive request (z_dim 512): a call's latency
        {"name": "norm z 4 rows", "op": "norm", "rows": 4, "cols": 512, "dtype": "float32", "residual": False, "weight": False},
        # many narrow rows of a width that no vector load divides: ragged features
        {"name": "norm odd 10001x1031", "op": "norm", "rows": 10001, "cols": 1031, "dtype": "float16", "residual": False, "weight": True},
        # a wide layer's residual stream, all of a large batch: bandwidth
        {"name": "norm wide 16384x4096", "op": "norm", "rows": 16384, "cols": 4096, "dtype": "bfloat16", "residual": True, "weight": True},
        # first layer of the mapping network for one latent (z 512 + embedded camera 512 -> 512): latency
        {"name": "mm mapping 1 row", "op": "mm", "rows": 1, "out": 512, "cols": 1024, "dtype": "float32", "lrelu": True, "bias": True},
        # the same layer over the latents that estimate the mean w
        {"name": "mm mapping 10000 rows", "op": "mm", "rows": 10000, "out": 512, "cols": 1024, "dtype": "float32", "lrelu": True, "bias": True},
        # few rows against large weights: reading the weights once is all there is
        {"name": "mm stream 16x8192x8192", "op": "mm", "rows": 16, "out": 8192, "cols": 8192, "dtype": "bfloat16", "lrelu": False, "bias": False},
        # a square product that fills the card
        {"name": "mm square 4096", "op": "mm", "rows": 4096, "out": 4096, "cols": 4096, "dtype": "bfloat16", "lrelu": False, "bias": True},
        # the largest, with edges that end inside a tile on both sides
        {"name": "mm large 8191x8190x8192", "op": "mm", "rows": 8191, "out": 8190, "cols": 8192, "dtype": "float16", "lrelu": False, "bias": False},
        # appearance editing: mean and deviation of one plane set are the leaves
        {"name": "clip statistics 2x96", "op": "clip", "count": 2, "total": 192, "dtype": "float32", "clipped": True},
        # geometry editing: the planes of four views (4 x 96 x 256 x 256) twice
        {"name": "clip planes 50.3M", "op": "clip", "count": 2, "total": 50331648, "dtype": "float32", "clipped": True},
        # the same size of one view, inside the limit: nothing is to be written
        {"name": "clip idle 6.3M", "op": "clip", "count": 1, "total": 6291456, "dtype": "float32", "clipped": False},
        # all parameters of a generator (180 tensors, 30 M values), half of them held in bfloat16
        {"name": "clip model 180 tensors", "op": "clip", "count": 180, "total": 30000000, "dtype": "mixed", "clipped": True},
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(("norm", "mm", "clip"))
    if op == "norm":
        cols = _log(rng, 16, 8192)
        return {"op": op, "rows": _log(rng, 1, min(20000, 67108864 // cols)), "cols": cols, "dtype": rng.choice(sorted(TYPES)),
                "residual": rng.random() < 0.5, "weight": rng.random() < 0.5}
    if op == "mm":
        return {"op": op, "rows": _log(rng, 1, 8190), "out": _log(rng, 16, 8190), "cols": _log(rng, 32, 8192), "dtype": rng.choice(sorted(TYPES)),
                "lrelu": rng.random() < 0.5, "bias": rng.random() < 0.5}
    total = _log(rng, 256, 50331648)
    return {"op": op, "count": _log(rng, 1, min(300, total // 64)), "total": total, "dtype": rng.choice(sorted(TYPES) + ["mixed"]),
            "clipped": rng.random() < 0.75}


def _blocks(n):
    return -(-n // BLOCK)


def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 16 + salt)


def _lengths(case):
    """The tensors' lengths: `count` parts of `total`, from single values to most of it, the same for every seed."""
    rng = random.Random(case["count"] * 1000003 + case["total"])
    cuts = sorted(rng.sample(range(1, case["total"]), case["count"] - 1)) if case["total"] < 4096 else sorted(
        max(1, int(case["total"] * rng.random() ** 2)) for _ in range(case["count"] - 1))
    ends = [0] + cuts + [case["total"]]
    return [b - a for a, b in zip(ends, ends[1:]) if b > a]


def _parts(case, seed):
    """Gradients as views of flat buckets (16-byte aligned starts), one bucket for each type: ([bucket], [view])."""
    types = [torch.float32, torch.bfloat16] if case["dtype"] == "mixed" else [TYPES[case["dtype"]]]
    lengths = _lengths(case)
    flats, views = [], []
    for j, t in enumerate(types):
        mine = lengths[j::len(types)]
        starts, at = [], 0
        for n in mine:
            starts.append(at)
            at += -(-n // 8) * 8
        flat = torch.zeros(max(at, 1), device="cuda", dtype=t)
        g = _generator(seed, 7 + j)
        values = torch.randn(flat.numel(), generator=g, device="cuda") * 0.02
        for i, (a, n) in enumerate(zip(starts, mine)):      # layers' gradients differ in size by orders of magnitude
            view = flat[a:a + n]
            view.copy_(values[a:a + n] * 2.0 ** (i % 7 - 3))
            views.append(view)
        flats.append(flat)
    return flats, views


def prepare(case, seed):
    op = case["op"]
    if op == "clip":
        flats, views = _parts(case, seed)
        square = sum(float(f.double().square().sum()) for f in flats)
        return {"op": op, "flats": flats, "views": views, "limit": math.sqrt(square) * (0.3 if case["clipped"] else 4.0), "clipped": case["clipped"]}
    g, t = _generator(seed, 1), TYPES[case["dtype"]]
    if op == "norm":
        m, k = case["rows"], case["cols"]
        channel = torch.exp(0.7 * torch.randn(k, generator=g, device="cuda"))              # features of unequal size
        x = (torch.randn(m, k, generator=g, device="cuda") * channel).to(t)
        x[m // 2] = 0                                                                       # a padding row
        state = {"op": op, "x": x, "residual": None, "weight": None}
        if case["residual"]:
            state["residual"] = (torch.randn(m, k, generator=g, device="cuda") * 2).to(t)
            state["residual"][m // 2] = 0
        if case["weight"]:
            state["weight"] = 1 + 0.2 * torch.randn(k, generator=g, device="cuda")
        return state
    m, n, k = case["rows"], case["out"], case["cols"]
    kb, nb = _blocks(k), _blocks(n)
    x = torch.zeros(m, kb * BLOCK, device="cuda")
    x[:, :k] = torch.randn(m, k, generator=g, device="cuda")
    x = x.view(m, kb, BLOCK)
    x_scale = x.abs().amax(-1).clamp_min(SMALLEST) / E4M3_MAX
    q = (x / x_scale[..., None]).to(torch.float8_e4m3fn).view(m, kb * BLOCK)
    w = torch.zeros(nb * BLOCK, kb * BLOCK, device="cuda")
    w[:n, :k] = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
    w = w.view(nb, BLOCK, kb, BLOCK)
    w_scale = w.abs().amax((1, 3)).clamp_min(SMALLEST) / E4M3_MAX
    wq = (w / w_scale[:, None, :, None]).to(torch.float8_e4m3fn).view(nb * BLOCK, kb * BLOCK)[:n, :k].contiguous()
    state = {"op": op, "q": q, "scale": x_scale.t().contiguous().t(), "wq": wq, "w_scale": w_scale, "k": k, "dtype": t, "lrelu": case["lrelu"],
             "bias": torch.randn(n, generator=g, device="cuda") if case["bias"] else None}
    if own:
        from nerffaceediting_amd import dense_ops
        state["weight"] = dense_ops.fp8_weight_from(wq, w_scale)      # laid out once, when a model is loaded
    return state


def _norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-8)
    if s["weight"] is not None:
        y = y * s["weight"]
    m, k = y.shape
    y = torch.nn.functional.pad(y, (0, _blocks(k) * BLOCK - k)).view(m, _blocks(k), BLOCK)
    scale = y.abs().amax(-1).clamp_min(SMALLEST) / E4M3_MAX
    out = {"q": (y / scale[..., None]).to(torch.float8_e4m3fn).view(m, -1), "scale": scale}
    if s["residual"] is not None:
        out["h"] = h.to(s["x"].dtype)
    return out


def _mm(s):
    q, wq = s["q"], s["wq"]
    m, k = q.shape[0], s["k"]
    x = (q.float().view(m, -1, BLOCK) * s["scale"][..., None]).view(m, -1)[:, :k]
    w = wq.float() * s["w_scale"].repeat_interleave(BLOCK, 0)[:wq.shape[0]].repeat_interleave(BLOCK, 1)[:, :k]
    y = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["lrelu"]:
        y = torch.where(y < 0, y * 0.2, y) * math.sqrt(2)
    return y.to(s["dtype"])


def _limit(s):
    """Gradients are clipped in place, so a second pass over the same ones would find them inside the limit: it falls by 1e-4 a pass."""
    limit = s["limit"]
    if s["clipped"]:
        s["limit"] = limit * (1 - 1e-4)
    return limit


def _clip(s):
    limit = _limit(s)
    squares = torch.stack([v.float().square().sum(dtype=torch.float64) for v in s["views"]])
    norm = squares.sum().sqrt()
    factor = (limit / (norm + 1e-6)).clamp(max=1.0).float()
    _ = [v.copy_(v.float() * factor) for v in s["views"]]
    return {"norm": norm.float(), "grads": s["flats"]}


def run(state):
    if not own:
        return {"norm": _norm, "mm": _mm, "clip": _clip}[state["op"]](state)
    from nerffaceediting_amd import dense_ops, ops
    if state["op"] == "norm":
        got = dense_ops.rms_norm_fp8(state["x"], weight=state["weight"], residual=state["residual"], eps=1e-8)
        return dict(zip(("q", "scale", "h"), got))
    if state["op"] == "mm":
        return dense_ops.fp8_matmul(state["q"], state["scale"], state["weight"], bias=state["bias"], lrelu=state["lrelu"], out_dtype=state["dtype"])
    return {"norm": ops.clip_grad_norm(state["views"], _limit(state)), "grads": state["flats"]}


def work(case):
    if case["op"] == "norm":
        m, k, b = case["rows"], case["cols"], 4 if case["dtype"] == "float32" else 2
        wide = 3 if case["residual"] else 1                       # x, and the residual read and written
        return {"bytes": m * k * b * wide + m * k + 4 * m * _blocks(k) + (4 * k if case["weight"] else 0), "flops": 8 * m * k}
    if case["op"] == "mm":
        m, n, k, b = case["rows"], case["out"], case["cols"], 4 if case["dtype"] == "float32" else 2
        scales = 4 * _blocks(k) * (m + _blocks(n))
        return {"bytes": (m + n) * k + scales + m * n * b + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    size = {"float32": 4, "mixed": 3}.get(case["dtype"], 2)
    return {"bytes": case["total"] * size * (2 if case["clipped"] else 1), "flops": case["total"] * (3 if case["clipped"] else 2)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        parts = [f.to(torch.float64) for f in s["flats"]]
        norm = math.sqrt(sum(float((p * p).sum()) for p in parts))
        factor = min(1.0, s["limit"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [p * factor for p in parts]}
    if case["op"] == "norm":
        h = s["x"].to(torch.float64)
        if s["residual"] is not None:
            h += s["residual"]
        power = torch.einsum("mk,mk->m", h, h) / h.shape[1] + 1e-8
        y = h / power.sqrt()[:, None]
        if s["weight"] is not None:
            y *= s["weight"]
        width = _blocks(y.shape[1]) * BLOCK
        full = torch.zeros(y.shape[0], width, dtype=torch.float64, device=y.device)
        full[:, :y.shape[1]] = y
        top = full.abs().unflatten(1, (-1, BLOCK)).max(-1).values
        scale = torch.maximum(top, torch.full_like(top, SMALLEST)) / E4M3_MAX
        out = {"q": full / scale.repeat_interleave(BLOCK, 1), "scale": scale}      # q before its rounding to 8 bits
        if s["residual"] is not None:
            out["h"] = h
        return out
    m, n, k = case["rows"], case["out"], case["cols"]
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for b in range(_blocks(k)):                                   # block by block, scales applied to the block's sums
        a, z = b * BLOCK, min(k, (b + 1) * BLOCK)
        part = s["q"][:, a:z].to(torch.float64) @ s["wq"][:, a:z].to(torch.float64).t().contiguous()
        part *= s["scale"][:, b, None].to(torch.float64)
        y += part * s["w_scale"][:, b].to(torch.float64).repeat_interleave(BLOCK)[:n]
    if s["bias"] is not None:
        y += s["bias"]
    if s["lrelu"]:
        y = torch.where(y < 0, 0.2 * y, y) * math.sqrt(2.0)
    return y
