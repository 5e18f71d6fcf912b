"""The 8-bit key/value cache: codes and scales against their definition, bit for bit; attention against the formula in 64
bits on what the cache holds; the decoder that generates with it."""

import math

import pytest
import torch

from aimet_amd import _lib
from aimet_amd import nn as qnn
from aimet_amd.quantization.kv_cache import QuantizedKVCache

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
names = lambda d: str(d).split(".")[-1]  # noqa: E731


class Model:
    """The cache's definition on the CPU, in 64 bits: codes [B, H, C, D] and maxima [B, H, C / block] of one tensor."""

    def __init__(self, cache):
        self.block = cache.block_tokens
        self.codes = torch.zeros(cache.batch, cache.kv_heads, cache.capacity, cache.head_dim, dtype=torch.float64)
        self.amax = torch.zeros(cache.batch, cache.kv_heads, cache.capacity // self.block, dtype=torch.float64)

    def append(self, x, start, counts):
        x = x.detach().cpu().double()
        cap = self.codes.shape[2]
        for b in range(x.shape[0]):
            s, n = int(start[b]), max(0, min(int(counts[b]), x.shape[2]))
            lo, end = max(s, 0), min(s + n, cap)
            for p in range(lo // self.block * self.block, end, self.block):
                a, z = max(lo, p), min(end, p + self.block)
                if a >= z:
                    continue
                new = x[b, :, a - s:z - s]
                size = torch.where(new.isfinite(), new.abs(), 0.0).amax((1, 2))
                had = self.amax[b, :, p // self.block] if a > p else torch.zeros_like(size)
                now = torch.maximum(had, size)
                safe = torch.where(now > 0, now, 1.0)[:, None, None]
                grown = (now > had)[:, None, None]
                old = self.codes[b, :, p:a]
                self.codes[b, :, p:a] = torch.where(grown, (old * had[:, None, None] / safe).round(), old)
                v = torch.where(new.isnan(), 0.0, new).clamp(min=-now[:, None, None], max=now[:, None, None])
                self.codes[b, :, a:z] = (v * 127 / safe).round()
                self.amax[b, :, p // self.block] = now

    def values(self):
        return self.codes * (self.amax / 127).repeat_interleave(self.block, 2)[..., None]


def _codes(cache):
    """Stored codes of keys and values in 64 bits, [B, H, C, D]."""
    return tuple(x.cpu().double() for x in cache.codes())


def _same(cache, models):
    for got, amax, m in zip(_codes(cache), (cache.k_amax, cache.v_amax), models):
        assert torch.equal(got, m.codes)
        assert torch.equal(amax.cpu().double(), m.amax)


def _tokens(b, h, t, d, dtype, seed, device):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, t, h, d, generator=g) * torch.exp(torch.randn(b, t, 1, 1, generator=g))
    return x.to(dtype).to(device).transpose(1, 2)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("dim,block", [(64, 16), (64, 64), (128, 32), (128, 64), (256, 16), (256, 64)])
def test_append_in_steps(device, dim, block, dtype):
    """Prompts, single tokens and ragged chunks behind each other; every state is the definition's, bit for bit."""
    cache = QuantizedKVCache(3, 2, 250, dim, block, device)
    assert cache.capacity == 256
    models = Model(cache), Model(cache)
    lengths = torch.zeros(3, dtype=torch.int32)
    steps = [(5, [5, 0, 3]), (1, [1, 1, 1]), (70, [70, 64, 1]), (1, [1, 0, 1]), (16, [16, 16, 16]), (100, [63, 65, 100])]
    for i, (t, counts) in enumerate(steps):
        k, v = _tokens(3, 2, t, dim, dtype, 2 * i, device), _tokens(3, 2, t, dim, dtype, 2 * i + 1, device)
        n = torch.tensor(counts, dtype=torch.int32)
        cache.append(k, v, lengths.to(device), counts=n.to(device))
        for m, x in zip(models, (k, v)):
            m.append(x, lengths, n)
        lengths += n
        _same(cache, models)
    for out_dtype in DTYPES:
        # a float32 product with a float32 quotient: two roundings, then one to the type asked for
        for got, m in zip(cache.dequantize(201, out_dtype), models):
            want = m.values()[:, :, :201]
            assert got.dtype == out_dtype
            # float16 steps are of one size below its smallest normal number: half of that step is added
            tiny = torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps
            assert bool(((got.cpu().double() - want).abs() <= (torch.finfo(out_dtype).eps / 2 + 2.0 ** -23) * want.abs() + tiny).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
def test_append_borders(device, dtype):
    """Values at half a code (half of the block's maximum is 63.5 codes), zeros, infinities, NaN, tiny and huge numbers."""
    cache = QuantizedKVCache(1, 1, 256, 64, 16, device)
    models = Model(cache), Model(cache)
    big = 60000.0 if dtype == torch.float16 else 2.0 ** 120
    # below float16's normal numbers, and below float32's once it is divided by 127
    small = 2.0 ** -20 if dtype == torch.float16 else 2.0 ** -125
    x = torch.zeros(1, 1, 128, 64)
    g = torch.Generator().manual_seed(0)
    for blk, top in enumerate((1.0, 127.0, 1.9921875, 0.7, big, small, 3.0)):
        rows = x[0, 0, 16 * blk:16 * blk + 16]
        codes = torch.randint(-254, 255, rows.shape, generator=g)
        rows.copy_((codes / 254.0 * top))
        rows[0, 0], rows[1, :8] = top, torch.tensor([top / 2, -top / 2, top / 4, 0.0, -0.0, top, -top, top / 254])
    x[0, 0, 5, 3], x[0, 0, 6, 3], x[0, 0, 7, 3] = float("nan"), float("inf"), float("-inf")
    x[0, 0, 96 + 2] = float("inf")
    x[0, 0, 112:, :] = 0.0
    x[0, 0, 113, 5], x[0, 0, 114, 5] = float("inf"), float("nan")  # nothing finite but zeros in this block
    x = x.to(dtype)
    cache.append(x.to(device), x.flip(3).to(device), 0)
    models[0].append(x, [0], [128])
    models[1].append(x.flip(3), [0], [128])
    _same(cache, models)
    assert bool(torch.isfinite(torch.stack(cache.dequantize())).all())


@pytest.mark.parametrize("dtype,amax", [(torch.float16, a) for a in (1.0, 127.0, 100.0625, 65504.0, 2.0 ** -14, 2.0 ** -24)]
                         + [(torch.bfloat16, a) for a in (1.0, 127.0, 0.7109375, 2.0 ** 127, 2.0 ** -100, 2.0 ** -126)]
                         + [(torch.float32, a) for a in (127.0, 0.1, 3e38, 1e-39)])
def test_append_every_code(device, dtype, amax):
    """All 16-bit values (float32: their multiples of the maximum) under one maximum, ties included: codes are exact."""
    amax = torch.tensor(amax, dtype=dtype)
    patterns = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    x = (patterns.view(torch.float16).float() / 65504 * amax if dtype == torch.float32 else patterns.view(dtype)).nan_to_num(0, 0, 0)
    x = torch.where(x.abs() > amax, amax, x).view(1, 16, 64, 64)
    x[:, :, 0, 0] = amax
    cache = QuantizedKVCache(1, 16, 64, 64, 64, device)
    cache.append(x.to(device), x.flip(3).to(device), 0)
    want = (x.double() * 127 / amax.double()).round()  # the quotient is exact to 2^-53, borders are 2^-40 apart at least
    k, v = _codes(cache)
    assert torch.equal(k, want) and torch.equal(v, want.flip(3))
    assert bool((cache.k_amax == amax.float().item()).all()) and bool((cache.v_amax == amax.float().item()).all())


def test_append_leaves_the_rest(device):
    """Tokens in front of the cache and behind it are dropped, padding is not read into scales, what lies behind the last
    token stays as it was, and a rewritten block starts a new scale at its first token."""
    cache = QuantizedKVCache(4, 1, 128, 64, 32, device)
    models = Model(cache), Model(cache)
    full = [_tokens(4, 1, 128, 64, torch.float32, s, device) * 50 for s in (0, 1)]
    cache.append(*full, 0)
    for m, x in zip(models, full):
        m.append(x, [0] * 4, [128] * 4)
    k, v = (_tokens(4, 1, 40, 64, torch.float32, s, device).contiguous() for s in (2, 3))
    start, counts = [-10, 100, 32, 200], [40, 40, 7, 9]
    for x in (k, v):
        x[2, :, 7:] = float("nan")
    cache.append(k, v, torch.tensor(start, dtype=torch.int32, device=device), torch.tensor(counts, dtype=torch.int32, device=device))
    for m, x in zip(models, (k, v)):
        m.append(x, start, counts)
    _same(cache, models)
    cache.append(k, v, torch.tensor([2 ** 31 - 1, -2 ** 31, 5, 128], dtype=torch.int32, device=device),
                 torch.tensor([2 ** 31 - 1, 40, -3, 40], dtype=torch.int32, device=device))
    _same(cache, models)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
def test_append_strides(device, dtype):
    b, h, t, d = 2, 3, 21, 64
    want = QuantizedKVCache(b, h, 64, d, 32, device)
    k, v = _tokens(b, h, t, d, dtype, 4, device).contiguous(), _tokens(b, h, t, d, dtype, 5, device).contiguous()
    want.append(k, v, 7)
    odd = torch.empty(b, t, h, d + 1, dtype=dtype, device=device)
    odd[..., 1:] = v.transpose(1, 2)
    for kk, vv in ((k.transpose(2, 3).contiguous().transpose(2, 3), odd[..., 1:].transpose(1, 2)),
                   (torch.stack([k, v], 2)[:, :, 0], torch.stack([k, v], 3)[:, :, :, 1])):
        cache = QuantizedKVCache(b, h, 64, d, 32, device)
        cache.append(kk, vv, 7)
        assert torch.equal(cache.k_codes, want.k_codes) and torch.equal(cache.v_codes, want.v_codes)
    # one token for all heads and sequences
    cache.append(k[:1, :1, :1].expand(b, h, 1, d), v[:1, :1, :1].expand(b, h, 1, d), 32)
    k, _ = cache.codes()
    assert torch.equal(k[1, 2, 32], k[0, 0, 32]) and bool(k[0, 0, 32].any())


# -------------------------------------------------------------------------------------------------------- attention --
def _reference(cache, q, lengths, counts, scale):
    """(answer, sum of probability times magnitude, largest sum of |q k| of the row, largest probability times scale of
    the values' block), in 64 bits."""
    kc, vc = _codes(cache)
    k = kc * (cache.k_amax.cpu().double() / 127).repeat_interleave(cache.block_tokens, 2)[..., None]
    v = vc * (cache.v_amax.cpu().double() / 127).repeat_interleave(cache.block_tokens, 2)[..., None]
    qd = q.cpu().double()
    b, hq, t, d = qd.shape
    g = hq // cache.kv_heads
    out, size = torch.zeros_like(qd), torch.zeros_like(qd)
    most, heavy = torch.zeros(b, hq, t, 1, dtype=torch.float64), torch.zeros(b, hq, t, 1, dtype=torch.float64)
    v_scale = (cache.v_amax.cpu().double() / 127).repeat_interleave(cache.block_tokens, 2)
    for i in range(b):
        n, c = max(0, min(int(lengths[i]), cache.capacity)), max(0, min(int(counts[i]), t))
        for h in range(hq):
            s = qd[i, h] @ k[i, h // g, :n].T * scale
            seen = torch.arange(n)[None] <= (n - c + torch.arange(t))[:, None]
            seen &= (torch.arange(t) < c)[:, None]
            p = torch.softmax(s.masked_fill(~seen, -1e300), 1) * seen if n else s
            out[i, h], size[i, h] = p @ v[i, h // g, :n], p @ v[i, h // g, :n].abs()
            if n:
                heavy[i, h] = (p * v_scale[i, h // g, None, :n]).amax(1, keepdim=True)
                most[i, h] = (qd[i, h].abs() @ k[i, h // g, :n].abs().T * abs(scale)).amax(1, keepdim=True)
    return out, size, most, heavy


def _attend_check(cache, q, lengths, counts=None, scale=None, given=()):
    b, _, t, d = q.shape
    n = [lengths] * b if isinstance(lengths, int) else lengths
    c = [t] * b if counts is None else [counts] * b if isinstance(counts, int) else counts
    out = cache.attend(q, *(given or (lengths, counts)), scale)
    want, size, most, heavy = _reference(cache, q, n, c, 1 / math.sqrt(d) if scale is None else scale)
    eps = torch.finfo(q.dtype).eps / 2
    # scores: queries in full or in two parts of 11 bits (2^-23), float32 sums of d products (2^-23 each) and four more
    # roundings; a probability is off by twice that and by 2^-19 (exponential, logarithm of the scale); as float16 it is
    # off by 2^-12 for 16-bit queries, by 2^-23 as two parts; sums of up to 2^-23 a token tile of 32
    wide = q.dtype == torch.float32
    tiles = cache.capacity / 32
    score = (33 * (2 if wide else 1) * d / 32 + 5) * 2.0 ** -23 * most
    bound = eps * want.abs() + (2 * score + 2.0 ** -19 + (2.0 ** -22 if wide else 2.0 ** -11) + (66 + tiles) * 2.0 ** -22) * size
    bound += torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    # weights (probability times scale) are float16 numbers of which the largest is at least 2^10: steps of 2^-24 near zero
    # take away at most half a step, 2^-35 of the largest, for each token, times a code of at most 127
    bound += max(n) * 2.0 ** -35 * 127 * heavy.nan_to_num(0.0, 0.0)
    err = (out.cpu().double() - want).abs()
    assert out.dtype == q.dtype and out.shape == q.shape
    worst = tuple(x.item() for x in torch.unravel_index((err / bound).argmax(), err.shape))
    assert bool((err <= bound).all()), f"{(err / bound).max().item()} of the bound at {worst}: {out[worst].item()}, {want[worst].item()}"
    # the roundings as a random walk, relative to the whole answer: float16's of the weights (rms 2^-12 / sqrt(3) at most),
    # and for a score the sums' and its scale's (four of 2^-24); an error of the score is the same error of the probability,
    # relative to it
    if want.norm() > 0:
        rel = err.norm().item() / want.norm().item()
        assert rel <= eps + (2.0 ** -19 if wide else 2.0 ** -12) * max(1.0, (size.norm() / want.norm()).item()) + 5 * 2.0 ** -24 * most.max().item(), rel
    return out


def _filled(b, h, length, d, block, dtype, device, capacity=None, seed=0):
    cache = QuantizedKVCache(b, h, capacity or max(length, 1), d, block, device)
    if length:
        cache.append(_tokens(b, h, length, d, dtype, seed, device), _tokens(b, h, length, d, dtype, seed + 1, device), 0)
    return cache


def _queries(b, h, t, d, dtype, device, seed=9):
    return torch.randn(b, t, h, d, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device).transpose(1, 2)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("dim,block", [(64, 16), (64, 64), (128, 32), (128, 64), (256, 16), (256, 64)])
@pytest.mark.parametrize("length", [1, 63, 64, 65, 300])
def test_attend_one_token(device, length, dim, block, dtype):
    cache = _filled(2, 2, length, dim, block, dtype, device)
    _attend_check(cache, _queries(2, 6, 1, dim, dtype, device), length)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("heads,groups,queries,length", [
    (1, 1, 2, 2), (2, 1, 5, 130), (1, 8, 3, 70), (2, 5, 7, 500), (1, 16, 1, 64), (1, 17, 2, 200), (3, 1, 64, 64),
    (1, 4, 100, 100), (2, 2, 129, 400), (1, 3, 333, 1000), (1, 1, 1, 2500), (1, 2, 513, 513)])
def test_attend_several_tokens(device, heads, groups, queries, length, dtype):
    cache = _filled(2, heads, length, 64, 32, dtype, device, capacity=length + 70)
    _attend_check(cache, _queries(2, heads * groups, queries, 64, dtype, device), length)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("queries,length", [(70, 70), (200, 331), (260, 1100)])
def test_attend_prompts(device, queries, length, dim, dtype):
    cache = _filled(1, 2, length, dim, 64, dtype, device)
    _attend_check(cache, _queries(1, 8, queries, dim, dtype, device), length)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("batch,heads,groups,queries,length,dim", [
    # four waves with rows of their own; eight in several splits; eight in one; a long cache in many splits
    (8, 16, 1, 40, 200, 64), (8, 16, 3, 40, 300, 128), (8, 16, 1, 64, 333, 256), (8, 16, 1, 50, 750, 64),
    (4, 32, 2, 70, 1100, 128), (8, 16, 1, 50, 770, 256), (8, 16, 1, 600, 600, 64), (1, 1, 1, 40, 140000, 64)])
def test_attend_many_prompts(device, batch, heads, groups, queries, length, dim, dtype):
    cache = _filled(batch, heads, length, dim, 32, dtype, device)
    _attend_check(cache, _queries(batch, heads * groups, queries, dim, dtype, device), length)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("capacity,dim", [(300, 64), (800, 64), (800, 128), (700, 256)])
def test_attend_many_ragged_prompts(device, capacity, dim, dtype):
    b, t = 64, 40
    cache = _filled(b, 2, capacity, dim, 16, dtype, device)
    g = torch.Generator().manual_seed(0)
    lengths, counts = (torch.randint(0, n + 1, (b,), generator=g, dtype=torch.int32) for n in (capacity, t))
    q = _queries(b, 2, t, dim, dtype, device).contiguous()
    clean = _attend_check(cache, q, lengths.tolist(), counts.tolist(), given=(lengths.to(device), counts.to(device)))
    q[(torch.arange(t) >= counts[:, None]).to(device)[:, None].expand(b, 2, t)] = float("nan")
    assert torch.equal(cache.attend(q, lengths.to(device), counts.to(device)), clean)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("dim,capacity", [(64, 33000), (128, 16500), (256, 8250)])
def test_attend_large_caches(device, dim, capacity, dtype):
    """Codes that the caches do not keep (32 MiB and more), few rows; short and long sequences in one call."""
    cache = _filled(4, 4, capacity, dim, 32, dtype, device)
    lengths = [capacity, 1, 700, capacity // 2]
    q = _queries(4, 8, 2, dim, dtype, device)
    _attend_check(cache, q, lengths, 2, given=(torch.tensor(lengths, dtype=torch.int32, device=device), 2))


@pytest.mark.parametrize("queries", [1, 4, 80, 150])
@pytest.mark.parametrize("dtype", DTYPES, ids=names)
def test_attend_ragged(device, dtype, queries):
    """Other lengths and numbers of queries for each sequence: empty sequences, more queries than tokens, padding with
    NaN, lengths and counts outside the cache."""
    b = 7
    cache = _filled(b, 2, 300, 64, 16, dtype, device)
    lengths, counts = [300, 0, 1, 2, 257, 1000, -4], [queries, queries, queries, 0, max(1, queries // 2), 1, 2]
    q = _queries(b, 4, queries, 64, dtype, device).contiguous()
    t = {k: torch.tensor(x, dtype=torch.int32, device=device) for k, x in (("lengths", lengths), ("counts", counts))}
    clean = _attend_check(cache, q, lengths, counts, given=(t["lengths"], t["counts"]))
    for i in range(b):
        n = max(0, min(counts[i], queries))
        q[i, :, n:] = float("nan")
    out = cache.attend(q, t["lengths"], t["counts"])
    assert torch.equal(out, clean)
    for i in (1, 3, 6):
        assert not bool(out[i].any())


def test_attend_int_and_tensor_lengths_agree(device):
    for length, cap in ((90, 4096), (1000, 1000)):
        cache = _filled(2, 2, length, 64, 64, torch.bfloat16, device, capacity=cap)
        q = _queries(2, 8, 1, 64, torch.bfloat16, device)
        a = _attend_check(cache, q, length)
        b = cache.attend(q, torch.full((2,), length, dtype=torch.int32, device=device))
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -7 * a.float().abs().max()


@pytest.mark.parametrize("queries", [1, 90])
def test_attend_scales_of_unlike_size(device, queries):
    """Blocks of values from 1e-6 to 1e4 and scores from -200 to 200."""
    cache = QuantizedKVCache(1, 1, 512, 64, 16, device)
    g = torch.Generator().manual_seed(0)
    size = (10.0 ** torch.randint(-6, 5, (1, 1, 32, 1), generator=g).float()).repeat_interleave(16, 2)
    k = torch.randn(1, 1, 512, 64, generator=g) * 6
    cache.append(k.to(device), (torch.randn(1, 1, 512, 64, generator=g) * size).to(device), 0)
    for dtype in DTYPES[:2]:
        _attend_check(cache, _queries(1, 3, queries, 64, dtype, device) * 4, 512)
        _attend_check(cache, _queries(1, 3, queries, 64, dtype, device), 512, scale=-0.3)
        _attend_check(cache, _queries(1, 3, queries, 64, dtype, device), 512, scale=0.0)


@pytest.mark.parametrize("queries", [1, 90])
def test_attend_nonfinite_queries_stay_in_their_row(device, queries):
    cache = _filled(1, 2, 100, 64, 32, torch.float32, device)
    q = _queries(1, 4, queries, 64, torch.float32, device).contiguous()
    clean = cache.attend(q, 100)
    q[0, 1, 0, 3] = float("nan")
    out = cache.attend(q, 100)
    assert bool(out[0, 1, 0].isnan().all())
    keep = torch.ones(4, queries, dtype=torch.bool)
    keep[1, 0] = False
    assert torch.equal(out[0][keep], clean[0][keep])


@pytest.mark.parametrize("queries", [1, 80])
def test_attend_does_not_read_behind_the_length(device, queries):
    cache = _filled(1, 1, 200, 64, 32, torch.float32, device)
    q = _queries(1, 2, queries, 64, torch.float32, device)
    want = cache.attend(q, 100)
    cache.k_codes[:, :, 2:] = 255  # tokens from 128 on
    cache.v_codes[:, :, 2:] = 0
    cache.k_codes[:, :, 1, :, :, :, 12:] = 255  # tokens 112 to 127
    cache.v_codes[:, :, 1, :, 3] = 0
    cache.k_codes[:, :, 1, 1:, :, :, 8:12] = 255  # tokens 100 to 111
    cache.v_codes[:, :, 1, :, 2, :, 4:] = 0
    cache.k_amax[:, :, 4:] = float("nan")
    cache.v_amax[:, :, 4:] = float("inf")
    assert torch.equal(cache.attend(q, 100), want)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("queries", [1, 70])
def test_attend_layouts(device, dtype, queries):
    cache = _filled(2, 2, 150, 64, 64, dtype, device)
    q = _queries(2, 4, queries, 64, dtype, device)
    want = _attend_check(cache, q, 150)
    assert want.stride() == torch.empty_like(q).stride()
    odd = torch.empty(2, 4, queries, 65, dtype=dtype, device=device)[..., 1:]
    odd.copy_(q)
    channels_first = q.transpose(2, 3).contiguous().transpose(2, 3)
    for other in (q.contiguous(), odd, channels_first):
        assert torch.equal(cache.attend(other, 150), want)
    assert cache.attend(q[:, :, :0], 150).shape == (2, 4, 0, 64)
    same = q[:, :1, :1].expand(2, 4, queries, 64)
    _attend_check(cache, same, 150)


def test_repeats_bit_for_bit(device):
    for length, queries in ((5000, 1), (700, 300)):
        cache = _filled(1, 2, length, 128, 64, torch.bfloat16, device)
        q = _queries(1, 8, queries, 128, torch.bfloat16, device)
        first = cache.attend(q, length)
        for _ in range(3):
            assert torch.equal(cache.attend(q, length), first)


def test_offsets_past_32_bits(device):
    """3.3e9 codes of keys and of values: the last heads' positions lie behind 2^31."""
    heads, cap, d = 32, 800000, 128
    cache = QuantizedKVCache(1, heads, cap, d, 64, device)
    assert cache.k_codes.numel() > 2 ** 31
    t = 130
    k, v = _tokens(1, heads, t, d, torch.float32, 0, device), _tokens(1, heads, t, d, torch.float32, 1, device)
    start = cache.capacity - t
    cache.append(k, v, start)
    end = QuantizedKVCache(1, heads, 192, d, 64, device)  # the last three tiles
    end.k_codes, end.v_codes = cache.k_codes[:, :, -3:], cache.v_codes[:, :, -3:]
    kd, vd = (x[0].double() for x in end.codes())
    kq, vq = kd[None, :, -64:], vd[None, :, -64:]
    assert bool(kq.any()) and bool(vq.any())
    for h in (0, 31):
        for x, codes, amax in ((k, kq, cache.k_amax), (v, vq, cache.v_amax)):
            want = (x[0, h, -64:].double() * 127 / amax[0, h, -1].double()).round()
            assert torch.equal(codes[0, h], want)
    q = _queries(1, heads, 1, d, torch.float32, device)
    out = cache.attend(q, cache.capacity)
    # all other tokens have the score 0 and the value 0
    kd = kd * (cache.k_amax[0, :, -3:].double() / 127).repeat_interleave(64, 1)[..., None]
    vd = vd * (cache.v_amax[0, :, -3:].double() / 127).repeat_interleave(64, 1)[..., None]
    s = (kd @ q[0].double().transpose(1, 2))[..., 0] / math.sqrt(d)
    p = torch.exp(s)
    want = (p[:, None] @ vd)[:, 0] / (p.sum(1, keepdim=True) + cache.capacity - 192)
    assert (out[0, :, 0].double() - want).norm() <= 1e-5 * want.norm()


def test_another_stream_and_graph(device):
    """A decoding step captured once and replayed: lengths advance on the device; eager work of the same shapes runs in
    between and gives the same answers."""
    b, h, d, cap = 3, 2, 64, 256
    mk = lambda: QuantizedKVCache(b, h, cap, d, 16, device)  # noqa: E731
    captured, eager = mk(), mk()
    prompt = _tokens(b, h, 60, d, torch.bfloat16, 0, device), _tokens(b, h, 60, d, torch.bfloat16, 1, device)
    for c in (captured, eager):
        c.append(*prompt, 0, counts=torch.tensor([60, 0, 13], dtype=torch.int32, device=device))
    lengths = torch.tensor([60, 0, 13], dtype=torch.int32, device=device)
    other = lengths.clone()
    k, v = _tokens(b, h, 1, d, torch.bfloat16, 2, device).clone(), _tokens(b, h, 1, d, torch.bfloat16, 3, device).clone()
    q = _queries(b, 2 * h, 1, d, torch.bfloat16, device).clone()
    warm = mk()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm.append(k, v, lengths)
        warm.attend(q, lengths)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.append(k, v, lengths)
        lengths.add_(1)
        out = captured.attend(q, lengths)
    for step in range(6):
        for i, x in enumerate((k, v, q)):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 * step + i)).to(x))
        graph.replay()
        eager.append(k, v, other)
        other += 1
        want = eager.attend(q, other)
        torch.cuda.synchronize()
        assert torch.equal(out, want), step
        assert torch.equal(captured.k_codes, eager.k_codes) and torch.equal(captured.v_codes, eager.v_codes)
    _attend_check(eager, q, other.tolist(), given=(other, None))


def test_two_graphs_and_streams_at_once(device):
    """Calls whose token axis is split, in two graphs replayed on two streams together: neither uses the other's scratch."""
    made = []
    for i, (queries, length) in enumerate(((1, 9000), (40, 140000))):
        cache = _filled(1, 1, length, 64, 64, torch.bfloat16, device, seed=i)
        q = _queries(1, 2, queries, 64, torch.bfloat16, device, seed=i).clone()
        want = cache.attend(q, length)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = cache.attend(q, length)
        made.append((graph, out, want, torch.cuda.Stream(), cache, q))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, out, _, stream, *_ in made:
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, *_ in made:
            assert torch.equal(out, want)


def test_copies_are_their_own(device):
    import copy

    cache = _filled(1, 2, 40, 64, 16, torch.float32, device)
    twin = copy.deepcopy(cache)
    q = _queries(1, 2, 1, 64, torch.float32, device)
    want = cache.attend(q, 40)
    twin.append(_tokens(1, 2, 24, 64, torch.float32, 8, device), _tokens(1, 2, 24, 64, torch.float32, 9, device), 10)
    assert torch.equal(cache.attend(q, 40), want) and not torch.equal(twin.attend(q, 40), want)


def test_refusals(device):
    cache = QuantizedKVCache(2, 2, 128, 64, 32, device)
    k = torch.randn(2, 2, 4, 64, device=device)
    lens = torch.zeros(2, dtype=torch.int32, device=device)
    for bad in ((k, k[:, :, :3]), (k, k.half()), (k[:1], k[:1]), (k[..., :32], k[..., :32]), (k[:, :1], k[:, :1]),
                (k.double(), k.double()), (k[0], k[0])):
        with pytest.raises(RuntimeError):
            cache.append(*bad, 0)
    with pytest.raises(_lib.HipLibraryError):
        cache.append(k.cpu(), k.cpu(), 0)
    for start in (-1, 125, 1.0, True, lens.long(), lens[:1], lens.cpu(), torch.zeros(4, dtype=torch.int32, device=device)[::2], None):
        with pytest.raises(RuntimeError):
            cache.append(k, k, start)
    for counts in (-1, 5, lens.float()):
        with pytest.raises(RuntimeError):
            cache.append(k, k, 0, counts=counts)
    with pytest.raises(RuntimeError, match="no backward"):
        cache.append(k.clone().requires_grad_(True), k, 0)
    assert bool((cache.k_codes == 128).all()) and not bool(cache.v_amax.any())
    q = torch.randn(2, 4, 1, 64, device=device)
    for bad in (q[:1], q[:, :3], q[:, :0], q[..., :32], q.double(), q[0]):
        with pytest.raises(RuntimeError):
            cache.attend(bad, 4)
    for lengths in (-1, 129, 2.0, lens.long(), lens[:1], None):
        with pytest.raises(RuntimeError):
            cache.attend(q, lengths)
    for bad in ({"scale": float("inf")}, {"scale": float("nan")}, {"scale": 1e300}, {"counts": 2}):
        with pytest.raises(RuntimeError):
            cache.attend(q, 4, **bad)
    with pytest.raises(RuntimeError, match="no backward"):
        cache.attend(q.clone().requires_grad_(True), 4)
    for bad in (-1, 129, 3.0):
        with pytest.raises(RuntimeError):
            cache.dequantize(bad)
    with pytest.raises(RuntimeError):
        cache.dequantize(4, torch.float64)
    assert cache.dequantize(0)[0].shape == (2, 2, 0, 64)


# ---------------------------------------------------------------------------------------------------------- decoder --
def test_generate(device):
    """The three operators together: a small quantized decoder with packed weights over 8-bit caches.  Its logits for a
    continuation that was fed token by token are those of one pass over the whole text through the same caches up to
    the codes (a block's scale grows in steps when it is filled in steps), and close to those without a cache."""
    import llama_harness as LH

    cfg = LH.LlamaConfig(layers=2, hidden=256, ffn=512, heads=4, vocab=320)
    model = LH.build(cfg, device)
    LH.quantize(model)
    batches = LH.calibration_batches(cfg, device, batches=2, seq=48, batch=2)
    LH.calibrate(model, batches)
    ids = batches[0][:, :40]
    with torch.no_grad():
        plain = model(ids)
        assert qnn.pack_linears(model) == 7 * cfg.layers + 1
        packed = model(ids).as_subclass(torch.Tensor).float()
        spread = plain.as_subclass(torch.Tensor).float().std()
        # the weight's bfloat16 rounding (2^-9 a weight) through two layers: a few times 2^-9 of the logits' size
        assert (packed - plain.as_subclass(torch.Tensor).float()).std() <= 2.0 ** -5 * spread
        whole = model(ids, LH.make_caches(model, 2, 64), 0).as_subclass(torch.Tensor).float()
        caches = LH.make_caches(model, 2, 64)
        steps = [model(ids[:, :30], caches, 0)] + [model(ids[:, i:i + 1], caches, i) for i in range(30, 40)]
        steps = torch.cat([s.as_subclass(torch.Tensor).float() for s in steps], 1)
        # 8 bits: half a code is 1/254 of a block's largest value
        assert (whole - packed).std() <= 2.0 ** -4 * spread
        assert (steps - whole).std() <= 2.0 ** -4 * spread
        text = LH.generate(model, ids[:, :16], 5)
        assert text.shape == (2, 21) and torch.equal(text[:, :16], ids[:, :16])
        assert torch.equal(text, LH.generate(model, ids[:, :16], 5))
