"""packed_linear against its formula in 64 bits, the packed form of calibrated layers against the layers, refusals."""

import math

import pytest
import torch

from aimet_amd import _lib
from aimet_amd import nn as qnn
from aimet_amd.quantization.affine import (GroupedBlockQuantizeDequantize, PackedWeight, QuantizeDequantize,
                                           packed_linear)

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _case(n, k, group, symmetric, seed, device):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g) + (0 if symmetric else 8)
    scale = torch.rand(n, k // group, generator=g) * 0.02 + 1e-3
    offset = None if symmetric else torch.randint(-15, 1, (n, k // group), generator=g).float()
    return codes.to(torch.int8).to(device), scale.to(device), None if offset is None else offset.to(device)


def _dense(codes, scale, offset, shift=0.0):
    group = codes.shape[1] // scale.shape[1]
    w = codes.cpu().double()
    if offset is not None:
        w = w + offset.cpu().double().repeat_interleave(group, 1)
    return (w + shift) * scale.cpu().double().repeat_interleave(group, 1)


def _check(y, x, codes, scale, offset, bias=None, shift=0.0, qmin=None):
    """Exact factors, float32 sums, one rounding.  A matrix instruction adds 32 products (33 roundings, allowed to
    truncate: 2^-23 each), up to 4 x 3 of them make a group sum, K / 32 group sums and 16 waves' results follow: that
    many times 2^-23 of the sum of magnitudes, which the codes enter counted from the lower end of the grid."""
    k = codes.shape[1]
    group = k // scale.shape[1]
    xd, w = x.cpu().double(), _dense(codes, scale, offset, shift)
    want = xd @ w.T
    qmin = (-8 if offset is None else 0) if qmin is None else qmin
    zero = torch.full(scale.shape, float(qmin)).double() if offset is None else offset.cpu().double() + qmin
    size = (codes.cpu().double() - qmin + (zero + shift).abs().repeat_interleave(group, 1)) * scale.cpu().double().repeat_interleave(group, 1)
    total = xd.abs() @ size.T
    if bias is not None:
        want, total = want + bias.cpu().double(), total + bias.cpu().double().abs()
    eps = torch.finfo(x.dtype).eps / 2
    bound = (12 * 33 + k / 32 + 17) * 2.0 ** -23 * total + eps * want.abs() * (1 + 1e-3)
    err = (y.cpu().double() - want).abs()
    assert y.dtype == x.dtype and y.shape == want.shape
    assert bool((err <= bound).all()), f"{(err / bound).max().item()} of the bound"
    # as a random walk of that many float32 roundings, each of a partial sum up to 4 times the result's size
    rel = err.norm().item() / want.norm().item()
    assert rel <= 4 * math.sqrt(k / 32 + 64) * 2.0 ** -24 + eps, rel


SHAPES = [  # tokens, out, in, group
    (1, 16, 32, 32), (1, 1, 64, 64), (1, 17, 96, 32), (1, 2048, 2048, 64), (2, 33, 192, 192), (3, 100, 130, 130),
    (5, 999, 2016, 32), (8, 48, 1024, 128), (15, 64, 2304, 192), (16, 256, 512, 64), (17, 80, 640, 64),
    (31, 31, 31, 31), (32, 96, 4096, 4096), (33, 128, 1152, 96), (47, 200, 256, 256), (64, 112, 768, 64),
    (65, 130, 512, 32), (100, 1000, 1001, 1001), (128, 128, 128, 128), (129, 257, 384, 64), (200, 64, 8192, 64),
    (257, 512, 2048, 128), (300, 384, 1000, 1000), (513, 272, 640, 64), (1025, 144, 256, 32),
    # activations that LDS does not hold at once
    (16, 100, 8192, 64), (32, 50, 5000, 5000), (7, 40, 14336, 128), (3, 33, 20000, 20000), (29, 4100, 3840, 32),
    # blocks of 32 x 128, 64 x 128 and 64 x 256: whole steps, rows that end inside one, groups of 32
    (257, 2000, 192, 64), (300, 3300, 320, 32), (290, 3400, 130, 130), (1000, 2200, 256, 64), (999, 2201, 320, 32),
    (1000, 2200, 130, 130),
    # of 32 x 64 and 32 x 128, of 32 to a workgroup
    (64, 2100, 2048, 64), (63, 2100, 2050, 2050), (128, 4200, 2048, 32), (100, 4200, 2100, 2100), (130, 500, 4096, 128),
]


@pytest.mark.parametrize("symmetric", [True, False], ids=["sym", "asym"])
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d).split(".")[-1])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_linear(device, shape, dtype, symmetric):
    m, n, k, group = shape
    codes, scale, offset = _case(n, k, group, symmetric, m + n, device)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(k)).to(dtype).to(device)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dtype).to(device) if n % 2 else None
    w = PackedWeight.pack(codes, scale, offset)
    _check(packed_linear(x, w, bias), x, codes, scale, offset, bias)


@pytest.mark.parametrize("m", [1, 20, 150])
def test_every_code_is_exact(device, m):
    """All 16 codes at every place of a tile: rows of the identity read the weight back, value by value."""
    n, k = 40, 256
    codes = ((torch.arange(n * k).view(n, k) * 7 + torch.arange(n)[:, None]) % 16 - 8).to(torch.int8).to(device)
    scale = torch.full((n, 4), 0.25, device=device)
    w = PackedWeight.pack(codes, scale)
    for dtype in DTYPES:
        for first in range(0, k, m):
            x = torch.eye(k, dtype=dtype, device=device)[first:first + m]
            assert torch.equal(packed_linear(x, w).float(), codes.float().T[first:first + m] * 0.25)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d).split(".")[-1])
@pytest.mark.parametrize("m", [4, 70, 300])
def test_strides_and_alignment(device, dtype, m):
    n, k = 72, 320
    codes, scale, offset = _case(n, k, 64, False, 3, device)
    w = PackedWeight.pack(codes, scale, offset)
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(m, k + 3, generator=g).to(dtype).to(device)
    for x in (wide[:, 3:], wide[:, :k], torch.randn(k, m, generator=g).to(dtype).to(device).T,
              torch.randn(1, k, generator=g).to(dtype).to(device).expand(m, k),
              torch.randn(m, 2, k, generator=g).to(dtype).to(device)[:, 1]):
        _check(packed_linear(x, w), x, codes, scale, offset)
    x = torch.randn(2, 3, m, k, generator=g).to(dtype).to(device)
    assert torch.equal(packed_linear(x, w), packed_linear(x.view(-1, k), w).view(2, 3, m, n))
    assert packed_linear(x[0, 0, 0], w).shape == (n,)
    assert packed_linear(x[:, :0], w).shape == (2, 0, m, n)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d).split(".")[-1])
def test_large_strides(device, dtype):
    """Rows 64 MB apart, so that a block's last row lies past 32-bit offsets; one row that is repeated."""
    n, k, m = 40, 64, 70
    codes, scale, offset = _case(n, k, 32, False, 3, device)
    w = PackedWeight.pack(codes, scale, offset)
    base = torch.empty(m << 24, dtype=dtype, device=device)
    x = base.view(m, 1 << 24)[:, 8:8 + k]
    x.copy_(torch.randn(m, k, generator=torch.Generator().manual_seed(1)).to(dtype))
    want = packed_linear(x.contiguous(), w)
    _check(want, x, codes, scale, offset)
    assert torch.equal(packed_linear(x, w), want)
    assert torch.equal(packed_linear(x[:20], w), packed_linear(x[:20].contiguous(), w))


def test_grids(device):
    """Other whole zero points and grids: an unsigned grid with one offset, a shifted grid, two and three bits."""
    codes, scale, _ = _case(50, 128, 32, True, 5, device)
    x = torch.randn(7, 128, device=device)
    offset = torch.full_like(scale, -8.0)
    w = PackedWeight.pack(codes + 8, scale, offset)
    assert w.zero is None  # one zero point for all
    _check(packed_linear(x, w), x, codes + 8, scale, offset)
    w = PackedWeight.pack(codes, scale, zero_point_shift=0.5)
    _check(packed_linear(x, w), x, codes, scale, None, shift=0.5)
    small = codes.clamp(-2, 1)
    w = PackedWeight.pack(small, scale, qmin=-2)
    _check(packed_linear(x, w), x, small, scale, None, qmin=-2)
    high = torch.full_like(scale, -120.0)
    high[0] = 100.0
    w = PackedWeight.pack(codes + 8, scale, high)
    assert w.zero is not None
    _check(packed_linear(x, w), x, codes + 8, scale, high)


@pytest.mark.parametrize("m", [1, 40, 260])
def test_rows_are_separate(device, m):
    """NaN and infinities stay in their row, the result of a row repeats bit for bit, padded channels are not written."""
    codes, scale, offset = _case(37, 256, 64, False, 6, device)
    w = PackedWeight.pack(codes, scale, offset)
    x = torch.randn(m + 2, 256, device=device).bfloat16()
    clean = packed_linear(x[:m], w)
    x[m, 5], x[m + 1, 200] = float("nan"), float("inf")
    y = packed_linear(x, w)
    assert torch.equal(y[:m], packed_linear(x, w)[:m]) and bool(y[m].isnan().all()) and not bool(y[m + 1].isfinite().any())
    _check(y[:m], x[:m], codes, scale, offset)
    assert torch.equal(clean, packed_linear(x[:m], w))


def test_another_stream_and_graph(device):
    codes, scale, offset = _case(96, 512, 64, False, 7, device)
    w = PackedWeight.pack(codes, scale, offset)
    x = torch.randn(3, 512, device=device)
    want = packed_linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(packed_linear(x, w), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = packed_linear(x, w)
    for k in range(3):
        x.copy_(torch.randn(3, 512, device=device))
        graph.replay()
        eager = packed_linear(x, w)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


def test_refusals(device):
    codes, scale, offset = _case(32, 128, 64, False, 8, device)
    w = PackedWeight.pack(codes, scale, offset)
    x = torch.randn(2, 128, device=device)
    for bad in (x.double(), x[:, :64], x.long(), torch.tensor(1.0, device=device)):
        with pytest.raises(RuntimeError):
            packed_linear(bad, w)
    with pytest.raises(_lib.HipLibraryError):
        packed_linear(x.cpu(), w)
    for bad in (torch.randn(31, device=device), torch.randn(32, device=device).half(), torch.randn(32)):
        with pytest.raises(RuntimeError):
            packed_linear(x, w, bad)
    with pytest.raises(RuntimeError, match="no backward"):
        packed_linear(x.clone().requires_grad_(True), w)
    with torch.no_grad():
        packed_linear(x.clone().requires_grad_(True), w)
    for args in ((codes + 1, scale, offset), (codes, scale), (codes, scale, offset + 0.5), (codes, scale, offset * 100),
                 (codes, scale[:, :1], offset), (codes, scale[:16], offset[:16]), (codes[0], scale, offset),
                 (codes, torch.rand(32, 8, device=device), torch.zeros(32, 8, device=device)),
                 (codes, scale.cpu(), offset), (codes[:, :0], scale, offset)):
        with pytest.raises(RuntimeError):
            PackedWeight.pack(*args)
    with pytest.raises(RuntimeError):
        PackedWeight.pack(codes.cpu(), scale.cpu())
    with pytest.raises(RuntimeError):
        PackedWeight(w.codes[:-1], w.scale, w.zero, w.zero_const, w.shape, w.group)
    with pytest.raises(RuntimeError):
        PackedWeight(w.codes, w.scale[:1], w.zero, w.zero_const, w.shape, w.group)


# ------------------------------------------------------------------------------------------------------ layers --
def _layer(device, dtype, wq, bias=True, out_f=96, in_f=256):
    torch.manual_seed(0)
    q = qnn.QuantizedLinear(in_f, out_f, bias=bias).to(device=device, dtype=dtype)
    q.param_quantizers["weight"] = wq.to(device)
    q.input_quantizers[0] = QuantizeDequantize((), 16, symmetric=False).to(device)
    q.output_quantizers[0] = QuantizeDequantize((), 16, symmetric=False).to(device)
    x = torch.randn(9, in_f, device=device, dtype=dtype)
    with torch.no_grad(), qnn.compute_encodings(q):
        q(x)
    return q, x


WEIGHT_QUANTIZERS = {
    "tensor": lambda: QuantizeDequantize((), 4, symmetric=True),
    "channel": lambda: QuantizeDequantize((96, 1), 4, symmetric=True),
    "channel_asym": lambda: QuantizeDequantize((96, 1), 4, symmetric=False),
    "block": lambda: QuantizeDequantize((96, 4), 4, symmetric=True, block_size=(1, 64)),
    "block_asym_3bit": lambda: QuantizeDequantize((96, 8), 3, symmetric=False, block_size=(1, 32)),
    "block_rows": lambda: QuantizeDequantize((12, 2), 4, symmetric=True, block_size=(8, 128)),
    "grouped": lambda: GroupedBlockQuantizeDequantize((96, 4), 4, symmetric=True, block_size=(1, 64),
                                                      decompressed_bw=8, block_grouping=(1, 4)),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("kind", list(WEIGHT_QUANTIZERS))
def test_packed_layer(device, kind, dtype):
    """The packed layer is the quantized one: same encodings, exact codes.  The layer's own product rounds code * scale
    to the weight's type (half a step: eps / 2 of every term) and sums in float32."""
    q, x = _layer(device, dtype, WEIGHT_QUANTIZERS[kind]())
    p = q.pack()
    with torch.no_grad():
        encoding = q.param_quantizers["weight"].get_encodings()
        dense = q.param_quantizers["weight"](q.weight).as_subclass(torch.Tensor)
        eye = torch.eye(256, device=device, dtype=torch.float32)
        read = packed_linear(eye, p.weight).T
        eps = torch.finfo(dtype).eps
        # scale and product are each rounded once to the weight's type at most
        assert bool(((read - dense.float()).abs() <= 1.01 * eps * read.abs()).all()), kind
        xin = q.input_quantizers[0](x).as_subclass(torch.Tensor)
        raw = packed_linear(xin, p.weight, p.bias).double()
        want = xin.double() @ read.double().T + p.bias.double()
        total = xin.double().abs() @ read.double().abs().T + p.bias.double().abs()
        assert bool(((raw - want).abs() <= eps / 2 * want.abs() * 1.001 + 600 * 2.0 ** -23 * total).all())
        y = p(x)
        step = q.output_quantizers[0].get_encodings().scale.double()
        assert bool(((y.as_subclass(torch.Tensor).double() - want.clamp(*(v.double() for v in (q.output_quantizers[0].min, q.output_quantizers[0].max)))).abs()
                     <= eps * want.abs() + 600 * 2.0 ** -23 * total + step).all())
        assert y.encoding is not None
    assert encoding.qmax - encoding.qmin <= 15


def test_packed_model_round_trip(device):
    q, x = _layer(device, torch.bfloat16, WEIGHT_QUANTIZERS["block"]())
    wide = qnn.QuantizedLinear(256, 8, bias=False).to(device, torch.bfloat16)
    wide.param_quantizers["weight"] = QuantizeDequantize((8, 1), 8, symmetric=True).to(device)
    model = torch.nn.Sequential(q, torch.nn.Sequential(torch.nn.Linear(96, 256).to(device, torch.bfloat16), wide))
    with torch.no_grad(), qnn.compute_encodings(model):
        model(x)
    with torch.no_grad():
        assert qnn.pack_linears(model) == 1
        assert isinstance(model[0], qnn.PackedLinear) and isinstance(model[1][1], qnn.QuantizedLinear)
        y = model(x)
        state = {k: v.clone() if torch.is_tensor(v) else v for k, v in model[0].state_dict().items()}
        other, _ = _layer(device, torch.bfloat16, WEIGHT_QUANTIZERS["block"](), bias=True)
        other.weight.data.mul_(-0.5)
        with qnn.compute_encodings(other):
            other(x)
        fresh = other.pack()
        assert not torch.equal(fresh(x), model[0](x))
        fresh.load_state_dict(state)
        assert torch.equal(fresh(x).as_subclass(torch.Tensor), model[0](x).as_subclass(torch.Tensor))
        before = fresh.weight_scale.clone()
        fresh.half()
        assert fresh.weight_scale.dtype == torch.float32 and torch.equal(fresh.weight_scale, before)
        fresh.bfloat16()
        with qnn.inference_mode(model):
            assert torch.equal(model(x).as_subclass(torch.Tensor), y.as_subclass(torch.Tensor))
        import copy
        twin = copy.deepcopy(model[0])
        assert torch.equal(twin(x).as_subclass(torch.Tensor), model[0](x).as_subclass(torch.Tensor))


def test_a_shared_layer_stays_one_layer(device):
    layer, _ = _layer(device, torch.float32, WEIGHT_QUANTIZERS["channel"]())
    model = torch.nn.ModuleDict({"a": layer, "b": torch.nn.Sequential(layer, torch.nn.ReLU()), "c": layer})
    assert qnn.pack_linears(model) == 1
    assert model["a"] is model["b"][0] is model["c"] and isinstance(model["a"], qnn.PackedLinear)


def test_folded_weight_packs(device):
    q, x = _layer(device, torch.float32, WEIGHT_QUANTIZERS["block"]())
    want = q.pack()
    q.fold_param_quantizers()
    got = q.pack()
    assert torch.equal(got.weight_codes, want.weight_codes) and torch.equal(got.weight_scale, want.weight_scale)
    assert qnn.pack_linears(torch.nn.Sequential(q)) == 1


def test_layer_refusals(device):
    q = qnn.QuantizedLinear(64, 32).to(device)
    with pytest.raises(RuntimeError, match="affine encoding"):
        q.pack()
    q, x = _layer(device, torch.float32, QuantizeDequantize((96, 1), 8, symmetric=True))
    with pytest.raises(RuntimeError, match="16 levels"):
        q.pack()
    q, x = _layer(device, torch.float32, QuantizeDequantize((96, 16), 4, symmetric=True, block_size=(1, 16)))
    with pytest.raises(RuntimeError, match="16 columns"):
        q.pack()
    q, x = _layer(device, torch.float32, WEIGHT_QUANTIZERS["channel"]())
    with pytest.raises(RuntimeError, match="no backward"):
        q.pack()(x.clone().requires_grad_(True))
