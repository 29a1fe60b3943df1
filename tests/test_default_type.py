"""Buffers that the library writes as fp32 are fp32 whatever torch.set_default_dtype says: under a 16-bit default type an unnamed one would be
half as large as what the kernels write."""
import ast
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MAKERS = {"empty": 1, "zeros": 1, "ones": 1, "full": 2, "empty_strided": 2, "rand": 1, "randn": 1, "eye": 1, "linspace": 3}


def _unnamed(path):
    """(line, call) of the calls in a file that make a tensor of torch's default type."""
    with open(path) as f:
        tree = ast.parse(f.read())
    for node in ast.walk(tree):
        if isinstance(node, ast.Call) and isinstance(node.func, ast.Attribute) and node.func.attr in MAKERS:
            if isinstance(node.func.value, ast.Name) and node.func.value.id == "torch" and not any(k.arg == "dtype" for k in node.keywords):
                yield node.lineno, ast.unparse(node)


@pytest.mark.parametrize("name", ["ops.py", "dense_ops.py"])
def test_every_buffer_names_its_type(name):
    found = list(_unnamed(os.path.join(ROOT, "nerffaceediting_amd", name)))
    assert not found, found


@pytest.fixture(params=[torch.bfloat16, torch.float64])
def default_type(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield request.param
    torch.set_default_dtype(before)


def test_scale_buffers(default_type):
    from nerffaceediting_amd import dense_ops
    q, scale = dense_ops._fp8_out("quantize_fp8", None, 0, 3, 200, torch.device("cpu"))
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32


@pytest.mark.gpu
def test_same_results_under_any_default_type(default_type):
    from nerffaceediting_amd import dense_ops, ops
    from nerffaceediting_amd.training.networks_stylegan2 import MappingNetwork
    dev = torch.device("cuda:0")

    def run():
        g = torch.Generator().manual_seed(1)
        randn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float32).to(dev)
        x, w = randn(37, 300), randn(130, 300)
        q, s, h = dense_ops.rms_norm_fp8(x, randn(300), randn(37, 300))
        W = dense_ops.fp8_weight(w)
        q2, s2 = dense_ops.quantize_fp8(dense_ops.fp8_matmul(q, s, W))
        grads = [randn(40000), randn(7).bfloat16()]
        norm = ops.clip_grad_norm(grads, 1.0)
        out = [q.view(torch.uint8), s, h, W.packed, W.scale, q2.view(torch.uint8), s2, norm, *grads]
        for m in nets:
            out.append(m(randn(5, 128), randn(5, 25)))
        return [(t.dtype, t.cpu()) for t in out]

    torch.set_default_dtype(torch.float32)
    torch.manual_seed(0)
    nets = [MappingNetwork(128, 25, 128, 4, num_layers=2, embed_features=128, fc_math=m).to(dev) for m in (None, "fp8")]
    want = run()
    torch.set_default_dtype(default_type)
    for (t, a), (u, b) in zip(run(), want):
        assert t == u and torch.equal(a, b)
