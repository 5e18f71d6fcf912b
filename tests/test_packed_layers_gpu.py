"""Packed layers made from quantizers of every kind, and what stands around them in a model: shifted grids, layers that have
no packed form, quantizers and hooks, autocast, captured calls."""

import pytest
import torch

from aimet_amd import nn as qnn
from aimet_amd.quantization.affine import NotPackable, PackedWeight, QuantizeDequantize, packed_linear

pytestmark = pytest.mark.gpu
names = lambda d: str(d).split(".")[-1]  # noqa: E731
plain = lambda t: t.as_subclass(torch.Tensor)  # noqa: E731

SHIFTED = {
    "tensor": ((), None), "channel": ((96, 1), None), "block": ((96, 4), (1, 64)), "rows": ((12, 2), (8, 128)),
}


def _layer(wq, device, dtype=torch.float32, in_f=256, out_f=96, bias=True):
    torch.manual_seed(0)
    q = qnn.QuantizedLinear(in_f, out_f, bias=bias).to(device=device, dtype=dtype)
    q.param_quantizers["weight"] = None if wq is None else wq.to(device)
    q.input_quantizers[0] = QuantizeDequantize((), 16, symmetric=False).to(device)
    q.output_quantizers[0] = QuantizeDequantize((), 16, symmetric=False).to(device)
    x = torch.randn(9, in_f, device=device, dtype=dtype)
    with torch.no_grad(), qnn.compute_encodings(q):
        q(x)
    return q, x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=names)
@pytest.mark.parametrize("kind", list(SHIFTED))
def test_shifted_grids(device, kind, dtype):
    """Grids of half steps: the packed values are the quantizer's, up to a rounding of the scale and of the product to the
    weight's type; a code next to the right one would be off by a fifteenth of the largest value at least."""
    shape, block = SHIFTED[kind]
    q, x = _layer(QuantizeDequantize(shape, 4, symmetric=True, block_size=block, zero_point_shift=0.5), device, dtype)
    wq = q.param_quantizers["weight"]
    eye = torch.eye(256, device=device)
    with torch.no_grad():
        dense = plain(wq(q.weight)).float()
        for weight in (q.pack().weight, PackedWeight.from_encoding(q.weight, wq.get_encodings()),
                       PackedWeight.from_encoding(q.weight.T.contiguous().T, wq.get_encodings()),
                       PackedWeight.from_encoding(wq(q.weight).dequantize(), wq.get_encodings())):
            read = packed_linear(eye, weight).T
            assert bool(((read - dense).abs() <= 1.01 * torch.finfo(dtype).eps * read.abs()).all())
        # all the roundings of the layer: the weight's, products of 256 terms in float32, the output's and one of its steps
        eps, xin = torch.finfo(dtype).eps, plain(q.input_quantizers[0](x)).double()
        total = xin.abs() @ dense.double().abs().T + q.bias.double().abs()
        step = q.output_quantizers[0].get_encodings().scale.double()
        got, want = (plain(layer(x)).double() for layer in (q.pack(), q))
        assert bool(((got - want).abs() <= (1.01 * eps + 512 * 2.0 ** -23) * total + eps * want.abs() + step).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=names)
def test_codes_that_are_not_whole_are_refused(device, dtype):
    codes = torch.randint(-8, 8, (32, 64), generator=torch.Generator().manual_seed(0)).to(dtype).to(device)
    scale, offset = torch.full((32, 2), 0.25, device=device), torch.arange(64.0, device=device).view(32, 2)
    for args in ((scale,), (scale, offset, -8)):
        whole = PackedWeight.pack(codes, *args)
        assert torch.equal(whole.codes, PackedWeight.pack(codes.to(torch.int8), *args).codes)
        for place, value in (((5, 3), 0.5), ((0, 0), -7.75), ((31, 63), float("nan"))):
            bad = codes.clone()
            bad[place] = value
            with pytest.raises(RuntimeError):
                PackedWeight.pack(bad, *args)


def test_tangents_are_refused_at_every_entry(device):
    from torch.autograd import forward_ad

    from aimet_amd.quantization.kv_cache import QuantizedKVCache

    w = PackedWeight.pack(torch.ones(32, 64, device=device), torch.ones(32, 1, device=device))
    x, bias = torch.randn(3, 64, device=device), torch.randn(32, device=device)
    cache = QuantizedKVCache(1, 1, 64, 64, 64, device)
    k = torch.randn(1, 1, 2, 64, device=device)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: packed_linear(dual(x), w), lambda: packed_linear(x, w, dual(bias)), lambda: cache.append(dual(k), k, 0),
                     lambda: cache.append(k, dual(k), 0), lambda: cache.attend(dual(k), 2)):
            with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
                call()
        packed_linear(x, w, bias), cache.append(k, k, 0), cache.attend(k, 2)


def _mixed(device):
    """Layers with a packed form and without one: blocks of 16 columns, 8 bits, no weight quantizer."""
    return torch.nn.ModuleDict({
        "block64": _layer(QuantizeDequantize((96, 4), 4, symmetric=True, block_size=(1, 64)), device)[0],
        "block16": _layer(QuantizeDequantize((96, 16), 4, symmetric=True, block_size=(1, 16)), device)[0],
        "bits8": _layer(QuantizeDequantize((96, 1), 8, symmetric=True), device)[0],
        "none": _layer(None, device)[0],
        "channel": _layer(QuantizeDequantize((96, 1), 4, symmetric=False), device)[0]})


def test_layers_without_a_packed_form_stay(device):
    model = _mixed(device)
    before = dict(model.items())
    with pytest.raises(NotPackable, match="16 columns"):
        before["block16"].pack()
    x = torch.randn(5, 256, device=device)
    with torch.no_grad():
        want = {k: plain(m(x)) for k, m in model.items()}
        assert qnn.pack_linears(model) == 2
        for k, m in model.items():
            if k in ("block64", "channel"):
                assert isinstance(m, qnn.PackedLinear)
            else:
                assert m is before[k] and torch.equal(plain(m(x)), want[k])
        assert qnn.pack_linears(model) == 0


def test_an_error_leaves_the_model_whole(device):
    """A layer that cannot be packed for another reason than its encoding: its weight is not on the device."""
    model = _mixed(device)
    before = dict(model.items())
    before["channel"].weight.data = before["channel"].weight.data.cpu()
    with pytest.raises(RuntimeError):
        qnn.pack_linears(model)
    assert all(model[k] is m for k, m in before.items())


def test_activation_quantizers_of_packed_layers(device):
    """The model-level helpers treat a packed layer's activation quantizers as those of the layer it was made from."""
    q, x = _layer(QuantizeDequantize((96, 4), 4, symmetric=True, block_size=(1, 64)), device)
    p = q.pack()
    model = torch.nn.Sequential(p)
    with torch.no_grad():
        bare = packed_linear(x, p.weight, p.bias)
        quantized = plain(model(x))
        assert not torch.equal(quantized, bare)
        for remove in (qnn.remove_activation_quantizers, qnn.remove_all_quantizers):
            with remove(model):
                assert torch.equal(plain(model(x)), bare)
            assert torch.equal(plain(model(x)), quantized)
        with qnn.remove_input_quantizers(model):
            assert p.input_quantizers[0] is None and p.output_quantizers[0] is not None
        with qnn.remove_output_quantizers(model):
            assert p.input_quantizers[0] is not None and p.output_quantizers[0] is None
        with qnn.remove_param_quantizers(model):
            assert torch.equal(plain(model(x)), quantized)
        # calibrated anew on ten times the data, together with the model, alone, and before it was packed
        ranges = []
        for target, context in ((model, lambda: qnn.compute_encodings(model)), (p, p.compute_encodings), (q, q.compute_encodings)):
            p.input_quantizers[0].set_range(-1, 1)
            with context():
                target(10 * x)
            ranges.append([t.clone() for o in (p.input_quantizers[0], p.output_quantizers[0]) for t in (o.min, o.max)])
        assert ranges[0][1] > 20
        for a, b, c in zip(*ranges):
            # the layers' products differ by the roundings of 256 terms in float32, the asymmetric grid by a step of 16 bits
            assert torch.equal(a, b) and bool((a - c).abs() <= 2.0 ** -12 * c.abs().max() + 2.0 ** -12)
        assert p.export_input_encodings("1.0.0")[0] is not None and p.export_output_encodings("1.0.0")[0] is not None
        qnn.remove_activation_quantizers(model)
        assert p.input_quantizers[0] is None and p.output_quantizers[0] is None


def test_what_a_replaced_layer_had(device):
    """Training mode and forward hooks stay with the place of the layer; the handles still remove them."""
    q, x = _layer(QuantizeDequantize((96, 4), 4, symmetric=True, block_size=(1, 64)), device)
    other, _ = _layer(QuantizeDequantize((96, 1), 4, symmetric=True), device)
    model = torch.nn.ModuleDict({"a": q, "b": other.eval()})
    calls = []
    handles = [q.register_forward_pre_hook(lambda m, a: calls.append(type(m).__name__)),
               q.register_forward_hook(lambda m, a, k, out: out * 0 if k.get("input") is None else out, with_kwargs=True),
               q.register_forward_hook(lambda m, a, out: calls.append("always"), always_call=True)]
    with torch.no_grad():
        assert qnn.pack_linears(model) == 2
        assert model["a"].training and not model["b"].training
        assert not bool(plain(model["a"](x)).any()) and calls == ["PackedLinear", "always"]
        assert bool(plain(model["a"](input=x)).any())
        for h in handles:
            h.remove()
        calls.clear()
        assert bool(plain(model["a"](x)).any()) and not calls
        assert not other.eval().pack().training


def test_a_model_that_is_a_layer_is_refused(device):
    q, _ = _layer(QuantizeDequantize((96, 1), 4, symmetric=True), device)
    with pytest.raises(RuntimeError, match="pack()"):
        qnn.pack_linears(q)


@pytest.mark.parametrize("layer_dtype", [torch.float32, torch.bfloat16], ids=names)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=names)
def test_autocast(device, layer_dtype, dtype):
    """Under autocast the packed layer computes in autocast's type, as the layer it was made from."""
    q, x = _layer(QuantizeDequantize((96, 4), 4, symmetric=True, block_size=(1, 64)), device, layer_dtype)
    p = q.pack()
    for layer in (q, p):
        layer.output_quantizers[0] = None
    with torch.no_grad():
        with torch.autocast("cuda", dtype=dtype):
            got, want = plain(p(x)), plain(q(x))
            xin = plain(p.input_quantizers[0](x)).to(dtype)
        assert got.dtype == want.dtype == dtype
        assert torch.equal(got, packed_linear(xin, p.weight, p.bias.to(dtype)))
        # the layer's weight is rounded to autocast's type (and to its own before), the result once on either side
        total = xin.double().abs() @ plain(q.param_quantizers["weight"](q.weight)).double().abs().T + p.bias.double().abs()
        eps = torch.finfo(dtype).eps / 2
        own = torch.finfo(layer_dtype).eps
        assert bool(((got - want).double().abs() <= (eps + 1.01 * own + 512 * 2.0 ** -23) * total + 2 * eps * want.double().abs() * 1.01).all())
        assert plain(p(x)).dtype == layer_dtype
        p.input_quantizers[0] = None
        for other in (x.double(), x.long()):  # autocast leaves these as they are
            with torch.autocast("cuda", dtype=dtype), pytest.raises(RuntimeError):
                p(other)


@pytest.mark.parametrize("m,n,k", [(20, 320, 4096), (300, 4096, 1024), (1100, 4200, 512)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=names)
def test_captured_calls_with_large_shared_memory(device, m, n, k, dtype):
    """Kernels that ask for more than 64 KB of shared memory at their launch, captured as their process's first call of these
    shapes and replayed with other inputs."""
    g = torch.Generator().manual_seed(0)
    w = PackedWeight.pack(torch.randint(-8, 8, (n, k), generator=g).to(torch.int8).to(device), torch.rand(n, k // 64, generator=g).to(device))
    x = torch.randn(m, k, generator=g).to(dtype).to(device)
    packed_linear(x[:1], w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = packed_linear(x, w)
    for _ in range(3):
        x.copy_(torch.randn(m, k, generator=g))
        graph.replay()
        eager = packed_linear(x, w)
        torch.cuda.synchronize()
        assert torch.equal(y, eager) and bool(y.any())


@pytest.mark.parametrize("batch,queries", [(1, 2), (8, 50)])
def test_captured_attention_with_large_shared_memory(device, batch, queries):
    """Head size 256: 70 KB for few rows, 128 KB for many."""
    from aimet_amd.quantization.kv_cache import QuantizedKVCache

    g = torch.Generator().manual_seed(0)
    cache = QuantizedKVCache(batch, 16, 192, 256, 64, device)
    kv = torch.randn(batch, 16, 190, 256, generator=g).bfloat16().to(device)
    cache.append(kv, kv.flip(3).contiguous(), 0)
    q = torch.randn(batch, 16, queries, 256, generator=g).bfloat16().to(device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(q, 190)
    for _ in range(3):
        q.copy_(torch.randn(q.shape, generator=g))
        graph.replay()
        eager = cache.attend(q, 190)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and bool(out.any())
