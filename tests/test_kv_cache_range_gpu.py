"""The 8-bit cache and its attention where ranges and roundings end: probabilities that cancel, queries and maxima at the
ends of their types' ranges."""

import math

import pytest
import torch

from aimet_amd.quantization.kv_cache import QuantizedKVCache

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
names = lambda d: str(d).split(".")[-1]  # noqa: E731

# (batch, heads, queries, length): few rows; many rows, four waves to a workgroup; eight
FORMS = [(4, 2, 1, 64), (4, 2, 3, 704), (8, 16, 40, 192), (8, 16, 50, 768)]


def _stored(cache):
    """Keys and values [B, H, C, D] in 64 bits, from what the cache holds."""
    return tuple(c.cpu().double() * (a.cpu().double() / 127).repeat_interleave(cache.block_tokens, 2)[..., None]
                 for c, a in zip(cache.codes(), (cache.k_amax, cache.v_amax)))


def _attention(cache, q, length, scale):
    """(answer, sum of probability times magnitude, largest sum of |q k| of a row) in 64 bits; one query head a head."""
    k, v = (x[:, :, :length] for x in _stored(cache))
    qd = q.cpu().double()
    t = q.shape[2]
    hidden = torch.arange(length)[None] > (length - t + torch.arange(t))[:, None]
    p = torch.softmax((qd @ k.transpose(2, 3) * scale).masked_fill(hidden, -math.inf), 3)
    return p @ v, p @ v.abs(), (qd.abs() @ k.abs().transpose(2, 3)).amax(3, keepdim=True) * abs(scale)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("batch,heads,queries,length", FORMS)
def test_probabilities_that_cancel(device, batch, heads, queries, length, dtype):
    """Tokens in pairs, their keys one code apart and their values opposite: the answer is what is left of probabilities
    that cancel, a few hundredths of what they add up to, so that it is the probabilities' roundings that show and not
    the answer's own.

    In relation to the sum of magnitudes: a probability's error is 2^-19 for the exponential and the logarithm of the
    block's scale, 2^-22 for its two float16 parts, and the error of its score, of which five roundings of 2^-24 count as
    a random walk.  (One float16 part is 2^-11 a token at most and 2^-12 / sqrt(3) of the mean square, over some ten
    tokens a row: 2^-14 or 2^-15.)"""
    g = torch.Generator().manual_seed(length)
    d = 64
    k = torch.randn(batch, heads, length // 2, 1, d, generator=g).expand(-1, -1, -1, 2, -1).clone() * 3
    k[..., 1, 0] += k.abs().amax() / 100
    v = torch.randn(batch, heads, length // 2, 1, d, generator=g) * torch.tensor([1.0, -1.0])[:, None]
    cache = QuantizedKVCache(batch, heads, length, d, 64, device)
    cache.append(*(x.reshape(batch, heads, length, d).to(device) for x in (k, v)), 0)
    q = torch.randn(batch, heads, queries, d, generator=g).to(dtype)
    out = cache.attend(q.to(device), length).cpu().double()
    want, size, most = _attention(cache, q, length, 1 / math.sqrt(d))
    even = (length - queries + torch.arange(queries)) % 2 == 1  # rows that see whole pairs
    out, want, size = (x[:, :, even] for x in (out, want, size))
    assert want.norm() <= 0.05 * size.norm()
    eps = torch.finfo(dtype).eps / 2
    assert (out - want).norm() <= eps * want.norm() + (2.0 ** -19 + 2.0 ** -22 + 5 * 2.0 ** -24 * most.amax()) * size.norm()


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
def test_read_back_at_the_top_of_the_range(device, dtype):
    """Blocks whose maximum is the largest number of their type, zeros and negative values beside it: a quotient and a
    product in float32, and one rounding to the type asked for."""
    top = torch.finfo(dtype).max
    g = torch.Generator().manual_seed(0)
    x = (torch.rand(1, 2, 64, 64, generator=g, dtype=torch.float64) * 2 - 1) * top
    x[:, :, ::16, :3] = torch.tensor([top, -top, 0.0], dtype=torch.float64)
    x = x.to(dtype)
    cache = QuantizedKVCache(1, 2, 64, 64, 16, device)
    cache.append(x.to(device), x.neg().flip(3).to(device), 0)
    assert bool((cache.k_amax == top).all()) and bool((cache.v_amax == top).all())
    for out_dtype in {torch.float32, dtype}:
        eps = torch.finfo(out_dtype).eps / 2
        for got, want in zip(cache.dequantize(dtype=out_dtype), _stored(cache)):
            got = got.cpu().double()
            assert bool(got.isfinite().all()) and bool((got[:, :, ::16].abs().amax(3) == top).all())
            assert bool(((got - want).abs() <= (eps + 2.0 ** -23) * want.abs()).all())


def test_read_back_into_float16_from_beyond_its_range(device):
    x = torch.zeros(1, 1, 64, 64)
    x[0, 0, ::16, :3] = torch.tensor([3e38, -3e38, 0.0])
    cache = QuantizedKVCache(1, 1, 64, 64, 16, device)
    cache.append(x.to(device), x.to(device), 0)
    for got in cache.dequantize(dtype=torch.float16):
        assert torch.equal(got.cpu(), x.half())


def _fill_blocks(shape, sizes, seed):
    """Values [B, H, T, D] whose blocks of 16 tokens are of the given sizes, in turn."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g, dtype=torch.float64).clamp(-4, 4) / 4
    size = torch.tensor(sizes, dtype=torch.float64).repeat(shape[2] // 16 // len(sizes) + 1)[:shape[2] // 16]
    return x * size.repeat_interleave(16)[:, None]


def _check_sizes(cache, q, length):
    """Every answer against the formula, as accurate for values of any size: the roundings of scores (d products a float32
    sum in instructions of 32, five more) and of probabilities as in the other tests, 2^-25 of a weight that is at least 2^10 at
    the largest for every token, and 2^-72 of the largest value for blocks that are smaller than that."""
    d = q.shape[3]
    out = cache.attend(q, length).cpu().double()
    want, size, most = _attention(cache, q, length, 1 / math.sqrt(d))
    eps, parts = torch.finfo(q.dtype).eps / 2, 2 if q.dtype == torch.float32 else 1
    scale = (cache.v_amax.cpu().double() / 127).repeat_interleave(cache.block_tokens, 2)[:, :, None, :length]
    t = q.shape[2]
    hidden = torch.arange(length)[None] > (length - t + torch.arange(t))[:, None]
    s = (q.cpu().double() @ _stored(cache)[0][:, :, :length].transpose(2, 3) / math.sqrt(d)).masked_fill(hidden, -math.inf)
    heavy = (torch.softmax(s, 3) * scale).amax(3, keepdim=True)
    bound = eps * want.abs() + length * 2.0 ** -35 * 127 * heavy + 2.0 ** -72 * 127 * scale.amax()
    bound += (2 * (33 * parts * d / 32 + 5) * 2.0 ** -23 * most + 2.0 ** -19 + 2.0 ** -21 + (66 + cache.capacity / 32) * 2.0 ** -22) * size
    bound += torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    err = (out - want).abs()
    assert bool(out.isfinite().all())
    assert bool((err <= bound).all()), (err / bound).max().item()
    return out


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=names)
@pytest.mark.parametrize("batch,heads,queries,length", FORMS + [(1, 1, 1, 2560)])
@pytest.mark.parametrize("sizes", [
    (1e-24,), (1e-30, 4e-31, 0.0), (1e-37, 3e-38), (0.0, 0.0, 0.0, 0.0, 1e-33), (1e-33, 0.0, 0.0, 0.0, 0.0), (2e-38, 1e-24, 1e-10, 3e4),
    (3e38, 1e-20, 1.0), (3e4, 1e-10, 1e-24, 2e-38), (3.3e38,), (0.0,)], ids=lambda s: "-".join(map(str, s)))
def test_values_of_any_size(device, batch, heads, queries, length, dtype, sizes):
    cache = QuantizedKVCache(batch, heads, length, 64, 16, device)
    k = torch.randn(batch, heads, length, 64, generator=torch.Generator().manual_seed(1))
    v = _fill_blocks((batch, heads, length, 64), sizes, 2)
    cache.append(k.to(device), v.float().to(device), 0)
    q = torch.randn(batch, heads, queries, 64, generator=torch.Generator().manual_seed(3)).to(dtype)
    out = _check_sizes(cache, q.to(device), length)
    assert bool(out.any()) == any(sizes[:length // 16])


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=names)
@pytest.mark.parametrize("batch,heads,queries,length", FORMS)
@pytest.mark.parametrize("dim", [128, 256])
def test_values_of_any_size_in_wider_heads(device, dim, batch, heads, queries, length, dtype):
    cache = QuantizedKVCache(batch, heads, length, dim, 16, device)
    k = torch.randn(batch, heads, length, dim, generator=torch.Generator().manual_seed(1))
    v = _fill_blocks((batch, heads, length, dim), (1e-30, 1e-33, 0.0, 2e-38), 2)
    cache.append(k.to(device), v.float().to(device), 0)
    q = torch.randn(batch, heads, queries, dim, generator=torch.Generator().manual_seed(3)).to(dtype)
    _check_sizes(cache, q.to(device), length)


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=names)
@pytest.mark.parametrize("batch,heads,queries,length", FORMS)
def test_weight_on_blocks_of_zeros(device, batch, heads, queries, length, dtype):
    """Blocks of zeros that have nearly all of the weight, in front of and behind tiny and huge ones: answers go to zero, and
    neither infinities nor NaN come of it."""
    for sizes in ((1e-30, 0.0, 1e30, 0.0), (0.0, 1e-36), (1e30, 0.0, 1e-30, 1e-4)):
        cache = QuantizedKVCache(batch, heads, length, 64, 16, device)
        k = torch.randn(batch, heads, length, 64, generator=torch.Generator().manual_seed(1))
        v = _fill_blocks((batch, heads, length, 64), sizes, 2)
        k[..., 0] += 30 * (v.abs().amax(3) == 0)
        cache.append(k.to(device), v.float().to(device), 0)
        q = torch.randn(batch, heads, queries, 64, generator=torch.Generator().manual_seed(3))
        q[..., 0] = 8
        _check_sizes(cache, q.to(dtype).to(device), length)


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=names)
@pytest.mark.parametrize("queries", [1, 60])
def test_scales_of_discarded_tokens(device, queries, dtype):
    """Small values over a longer sequence of huge ones that were discarded: their blocks' scales play no part."""
    batch, heads, length = (2, 2, 70) if queries == 1 else (8, 16, 70)
    q = torch.randn(batch, heads, queries, 64, generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
    k, v = (torch.randn(batch, heads, 192, 64, generator=torch.Generator().manual_seed(s)).to(device) for s in (1, 2))
    outs = []
    for discarded in (1.0, 1e30):
        cache = QuantizedKVCache(batch, heads, 192, 64, 16, device)
        cache.append(k, v * discarded, 0)
        cache.append(k[:, :, :length], v[:, :, :length] * 1e-20, 0)
        outs.append(_check_sizes(cache, q, length))
    assert torch.equal(*outs)


@pytest.mark.parametrize("batch,heads,queries,length", FORMS)
@pytest.mark.parametrize("top", [1.0, 16384.0, 65504.0])
def test_float16_queries_are_exact(device, top, batch, heads, queries, length):
    """Queries of one large channel, whose keys are zero, and of the smallest numbers of float16 in the others: those make
    the scores, and a bit lost of them would be an error of 1 / 15 at least."""
    g = torch.Generator().manual_seed(0)
    d = 64
    q = torch.randint(-15, 16, (batch, heads, queries, d), generator=g).float() * 2.0 ** -24
    q[..., 0] = top
    k = torch.randn(batch, heads, length, d, generator=g) * 2.0 ** 20
    k[..., 0] = 0
    cache = QuantizedKVCache(batch, heads, length, d, 64, device)
    cache.append(k.to(device), torch.randn(batch, heads, length, d, generator=g).to(device), 0)
    q = q.half()
    assert bool((q[..., 1:] != 0).any()) and bool((q[..., 0] == top).all())
    _check_sizes(cache, q.to(device), length)


def test_rewound_block_keeps_its_scale(device):
    """A draft with one large token is discarded inside a block: what was there and what follows stay on its grid, the next
    block and a block that is begun anew do not."""
    g = torch.Generator().manual_seed(0)
    x = torch.rand(1, 1, 40, 64, generator=g) * 2 - 1
    x[0, 0, 0, 0], x[0, 0, 9, 3], x[0, 0, 20, 5] = 1.0, -1.0, 1.0
    draft = torch.randn(1, 1, 4, 64, generator=g)
    draft[0, 0, 2, 7] = 50.0
    cache = QuantizedKVCache(1, 1, 64, 64, 16, device)
    cache.append(x[:, :, :10].to(device), x[:, :, :10].to(device), 0)
    cache.append(draft.to(device), draft.to(device), 10)
    cache.append(x[:, :, 10:].to(device), x[:, :, 10:].to(device), 10)
    fine, coarse = (x.double() * 127).round(), (x.double() * 127 / 50).round()
    coarse[:, :, :10] = (fine[:, :, :10] / 50).round()
    for codes, amax in zip(cache.codes(), (cache.k_amax, cache.v_amax)):
        codes = codes.cpu().double()
        assert amax[0, 0, 0] == 50 and amax[0, 0, 1] == 1
        assert torch.equal(codes[:, :, :16], coarse[:, :, :16]) and torch.equal(codes[:, :, 16:32], fine[:, :, 16:32])
    cache.append(x[:, :, :16].to(device), x[:, :, :16].to(device), 0)
    assert cache.k_amax[0, 0, 0] == 1 and torch.equal(cache.codes()[0].cpu().double()[:, :, :16], fine[:, :, :16])
