"""FullyConnectedLayer.forward_fp8's weight image: kept between eager calls, never out of date and never missing.  Every check compares with
dense_ops.fp8_weight of the parameter as it is, bit for bit (the same kernels on the same values)."""
import io

import pytest
import torch


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def make(dev, n=130, k=256, rows=9, seed=3):
    from nerffaceediting_amd import dense_ops
    from nerffaceediting_amd.training.networks_stylegan2 import FullyConnectedLayer
    torch.manual_seed(seed)
    layer = FullyConnectedLayer(k, n).to(dev)
    q, s = dense_ops.quantize_fp8(torch.randn(rows, k, device=dev))

    def want():
        w = dense_ops.fp8_weight(layer.weight.detach(), gain=layer.weight_gain)
        return dense_ops.fp8_matmul(q, s, w, None if layer.bias is None else layer.bias.detach(), layer.bias_gain)

    return layer, q, s, want


def capture(layer, q, s):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer.forward_fp8(q, s)
    return g, out


@pytest.mark.gpu
def test_replays_after_an_eager_call_follow_the_weights(dev):
    layer, q, s, want = make(dev)
    assert torch.equal(layer.forward_fp8(q, s), want())
    g, out = capture(layer, q, s)
    for i in range(4):
        with torch.no_grad():
            layer.weight.mul_(1.5)
            layer.bias.add_(1.0)
        g.replay()
        ref = want()
        torch.cuda.synchronize()
        assert torch.equal(out, ref), i


@pytest.mark.gpu
def test_replays_outlive_the_eager_image(dev):
    """Eager call, two captures, then eager calls that replace the kept image and allocations that take whatever became free."""
    layer, q, s, want = make(dev)
    layer.forward_fp8(q, s)
    graphs = [capture(layer, q, s), capture(layer, q, s)]
    for i in range(4):
        with torch.no_grad():
            layer.weight.mul_(-0.5)
        assert torch.equal(layer.forward_fp8(q, s), want())
        junk = [torch.full((1 << j,), float("nan"), device=dev) for j in range(4, 18)]
        for g, out in graphs:
            g.replay()
            ref = want()
            torch.cuda.synchronize()
            assert torch.equal(out, ref), i
        del junk


@pytest.mark.gpu
def test_image_replaced_while_another_stream_reads_it(dev):
    """Image made on one stream, product waiting on another, image replaced there: what the first stream allocates next is not the image that
    the product has still to read."""
    layer, q, s, want = make(dev)
    layer.forward_fp8(q, s)
    ref = want()
    torch.cuda.synchronize()
    side = torch.cuda.Stream(device=dev)
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)                                  # about half a second
        out = layer.forward_fp8(q, s)
        done = torch.cuda.Event()
        done.record()
        new = (layer.weight.detach() * 2).clone()
        layer.weight = torch.nn.Parameter(new)
        size = layer._fp8[2].packed.numel()
        del layer._fp8                                                    # what replacing it does, without the wait of making the next one
    junk = [torch.full((size,), 0x7F, dtype=torch.uint8, device=dev) for _ in range(8)]      # e4m3 NaN
    torch.cuda.current_stream(dev).synchronize()
    assert not done.query()                                               # the product has not run yet
    torch.cuda.synchronize()
    assert torch.equal(out, ref) and len(junk) == 8


def test_image_is_finished_on_its_own_device(monkeypatch):
    """Before the image is kept, the stream that makes it is waited for: the one of the weights' device, whichever device is current."""
    from nerffaceediting_amd.training import networks_stylegan2 as net
    layer = net.FullyConnectedLayer(8, 4)
    waited = []

    class Stream:
        def __init__(self, device):
            self.device = device

        def synchronize(self):
            waited.append(self.device)

    class Image:
        def used(self):
            pass

    with pytest.raises(RuntimeError, match="no CPU fallback"):
        layer.forward_fp8(None, None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(device))
    monkeypatch.setattr(net.dense_ops, "fp8_weight", lambda w, gain: Image())
    monkeypatch.setattr(net.dense_ops, "fp8_matmul", lambda *a: None)
    layer.forward_fp8(None, None)
    assert waited == [layer.weight.device]


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["save", "deepcopy"])
def test_copies_of_a_layer_make_their_own_image(dev, how):
    """Weights changed after the image was made, then the module saved and loaded (or copied): a loaded parameter's version starts anew, and
    must not meet the version that the image was made at."""
    import copy
    from nerffaceediting_amd import dense_ops
    for bumps in range(3):
        layer, q, s, _ = make(dev)
        with torch.no_grad():
            for _ in range(bumps):
                layer.weight.add_(0.25)
            layer.forward_fp8(q, s)
            layer.weight.mul_(-3.0)
        if how == "save":
            file = io.BytesIO()
            torch.save(layer, file)
            file.seek(0)
            other = torch.load(file, weights_only=False)
        else:
            other = copy.deepcopy(layer)
        ref = dense_ops.fp8_matmul(q, s, dense_ops.fp8_weight(other.weight.detach(), gain=other.weight_gain), other.bias.detach(), other.bias_gain)
        assert torch.equal(other.forward_fp8(q, s), ref), bumps
        assert torch.equal(layer.forward_fp8(q, s), ref), bumps


def test_a_saved_layer_carries_no_image():
    import copy
    from nerffaceediting_amd.training.networks_stylegan2 import FullyConnectedLayer
    layer = FullyConnectedLayer(8, 4)
    plain = set(layer.__dict__)
    layer._fp8 = (layer.weight.detach(), layer.weight._version, "image")
    file = io.BytesIO()
    torch.save(layer, file)
    file.seek(0)
    for other in (torch.load(file, weights_only=False), copy.deepcopy(layer)):
        assert set(other.__dict__) == plain and torch.equal(other.weight, layer.weight)
    assert layer._fp8[2] == "image"


@pytest.mark.gpu
def test_image_follows_strides_and_gain(dev):
    """Changes that leave the parameter's address, shape and version as they were."""
    layer, q, s, want = make(dev, n=256)
    layer.forward_fp8(q, s)
    layer.weight.data = layer.weight.data.t()
    assert torch.equal(layer.forward_fp8(q, s), want())
    layer.weight_gain = layer.weight_gain * 3
    assert torch.equal(layer.forward_fp8(q, s), want())


@pytest.mark.gpu
def test_image_follows_a_new_parameter_on_the_same_memory(dev):
    """Parameter(layer.weight.data) starts its versions at 0 again; setting the kept image to None makes it anew."""
    layer, q, s, want = make(dev)
    layer.forward_fp8(q, s)
    with torch.no_grad():
        layer.weight.mul_(-2.0)
    layer.weight = torch.nn.Parameter(layer.weight.data, requires_grad=False)
    assert torch.equal(layer.forward_fp8(q, s), want())
    layer.weight.data.mul_(0.5)
    layer._fp8 = (None, None, None)
    assert torch.equal(layer.forward_fp8(q, s), want())


@pytest.mark.gpu
def test_weights_without_versions(dev):
    """Parameters made under inference_mode track no versions: no image is kept of them, and the layer works as the fp32 one does."""
    from nerffaceediting_amd.training.networks_stylegan2 import MappingNetwork
    with torch.inference_mode():
        layer, q, s, want = make(dev)
        assert torch.equal(layer.forward_fp8(q, s), want())
        layer.weight.mul_(2.0)
        assert torch.equal(layer.forward_fp8(q, s), want())
        m = MappingNetwork(128, 25, 128, 4, num_layers=2, embed_features=128, fc_math="fp8").to(dev)
        assert m(torch.randn(3, 128, device=dev), torch.randn(3, 25, device=dev)).shape == (3, 4, 128)
    assert torch.equal(layer.forward_fp8(q, s), want())


def test_mapping_networks_saved_before_fc_math():
    """A module pickled when MappingNetwork had no fc_math loads as the fp32 network that it was."""
    from nerffaceediting_amd.training.networks_stylegan2 import MappingNetwork
    m = MappingNetwork(16, 4, 16, 2, num_layers=2)
    del m.__dict__["fc_math"]
    file = io.BytesIO()
    torch.save(m, file)
    file.seek(0)
    assert torch.load(file, weights_only=False).fc_math is None


def test_fp8_stack_without_layers_is_refused():
    from nerffaceediting_amd.training.networks_stylegan2 import MappingNetwork
    with pytest.raises(ValueError, match="num_layers"):
        MappingNetwork(128, 0, 128, 4, num_layers=0, fc_math="fp8")
    assert MappingNetwork(128, 0, 128, 4, num_layers=0).num_layers == 0
