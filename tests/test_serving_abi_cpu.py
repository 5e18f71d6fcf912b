"""Host-side refusals of the packed linear layer and the 8-bit cache, without a GPU: every call here returns before
anything is launched."""

import ctypes
import math

import pytest
import torch

from aimet_amd import _lib
from aimet_amd.quantization.affine import PackedWeight, packed_linear
from aimet_amd.quantization.kv_cache import QuantizedKVCache


@pytest.fixture(scope="module")
def lib():
    import os

    if not os.path.exists(_lib.LIB_PATH):
        from aimet_amd.csrc.build import build

        build(verbose=False)
    return _lib.load()


def test_header_and_bindings_agree(lib, tmp_path):
    """Every declared function is exported and bound, every struct has its mirror's size and offsets."""
    import os
    import re
    import shutil
    import subprocess

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "aimet_amd_serving.h")
    header = re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)
    declared = set(re.findall(r"\b(ahq_[a-z0-9_]+)\s*\(", header))
    assert declared == set(_lib._SERVING_SIGNATURES) and all(hasattr(lib, name) for name in declared)
    mirrors = {"ahq_int4_weight": _lib.Int4Weight, "ahq_kv_cache": _lib.KvCache, "ahq_kv_tokens": _lib.KvTokens, "ahq_kv_queries": _lib.KvQueries}
    assert set(re.findall(r"^\} (ahq_\w+);", header, flags=re.M)) == set(mirrors)
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', f'#include "{path}"', "int main(void) {"]
    for name, cls in mirrors.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join([*lines, "  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, what, value = line.split()
        cls = mirrors[name]
        assert int(value) == (ctypes.sizeof(cls) if what == "size" else getattr(cls, what).offset), line


def test_packed_sizes(lib):
    assert lib.ahq_int4_packed_bytes(16, 128) == 1024
    assert lib.ahq_int4_packed_bytes(17, 129) == 4 * 1024
    assert lib.ahq_int4_packed_bytes(14336, 4096) == 14336 * 4096 // 2
    for n, k in ((0, 1), (1, 0), (-1, 5), (1 << 40, 1), (1, 1 << 21)):
        assert lib.ahq_int4_packed_bytes(n, k) == 0


def test_int4_refusals(lib):
    p = 1 << 12  # an aligned address that is never followed
    assert lib.ahq_int4_pack(None, 4, 4, -8, p, None) == 1 and lib.ahq_int4_pack(p, 4, 4, -8, None, None) == 1
    assert lib.ahq_int4_pack(p, 0, 4, -8, p, None) == 1 and lib.ahq_int4_pack(p, 4, 4, 113, p, None) == 1
    assert lib.ahq_int4_pack(p, 4, 4, -129, p, None) == 1 and lib.ahq_int4_pack(p, 4, 4, 0, p + 4, None) == 1
    good = dict(dtype=0, x=p, m=1, ldx=64, w=p, n=32, k=64, group=32, scale=p, zero=None, zc=-8.0, bias=None, y=p, ldy=32)

    def linear(**kw):
        a = {**good, **kw}
        w = _lib.Int4Weight(a["n"], a["k"], a["group"], a["w"], a["scale"], a["zero"], a["zc"])
        return lib.ahq_int4_linear(w, a["dtype"], a["x"], a["m"], a["ldx"], a["bias"], a["y"], a["ldy"], None)

    for bad in (dict(dtype=3), dict(dtype=-1), dict(x=None), dict(w=None), dict(scale=None), dict(y=None), dict(m=-1),
                dict(n=0), dict(k=0), dict(ldx=63), dict(ldy=31), dict(group=0), dict(group=48), dict(group=128),
                dict(w=p + 8), dict(scale=p + 4), dict(zero=p + 2), dict(x=p + 1), dict(y=p + 2), dict(bias=p + 1)):
        assert linear(**bad) == 1, bad
    assert lib.ahq_int4_linear(None, 0, p, 1, 64, None, p, 32, None) == 1
    assert linear(group=16) == _lib.AHQ_ERR_UNSUPPORTED and b"32" in lib.ahq_last_error()
    assert linear(m=(1 << 20) + 1) == _lib.AHQ_ERR_UNSUPPORTED
    assert linear(m=0, x=None, y=None) == 0


def _cache(**kw):
    p = 1 << 12
    a = {**dict(batch=2, heads=2, capacity=128, head_dim=64, block=32, k=p, v=p, ka=p, va=p), **kw}
    return _lib.KvCache(a["batch"], a["heads"], a["capacity"], a["head_dim"], a["block"], a["k"], a["v"], a["ka"], a["va"])


def _tokens(**kw):
    p = 1 << 12
    a = {**dict(dtype=0, tokens=4, k=p, v=p), **kw}
    return _lib.KvTokens(a["dtype"], a["tokens"], a["k"], a["v"], (1024, 1024), (512, 512), (64, 64), None, None, 0, a["tokens"])


def _queries(**kw):
    p = 1 << 12
    a = {**dict(dtype=0, heads=4, queries=1, q=p, out=p, lengths=None, length=100, scale=0.125), **kw}
    return _lib.KvQueries(a["dtype"], a["heads"], a["queries"], a["q"], a["out"], 256, 64, 64, 256, 64, 64, a["lengths"], None,
                          a["length"], a["queries"], a["scale"])


BAD_CACHES = [dict(batch=0), dict(heads=-1), dict(capacity=0), dict(capacity=100), dict(batch=40000), dict(k=None),
              dict(v=None), dict(ka=None), dict(va=None), dict(k=(1 << 12) + 8), dict(capacity=(1 << 30) + 64)]
NO_KERNEL = [dict(head_dim=96), dict(head_dim=0), dict(block=8), dict(block=128)]


def test_kv_refusals(lib):
    for bad in BAD_CACHES:
        assert lib.ahq_kv_append(_cache(**bad), _tokens(), None) == 1, bad
        assert lib.ahq_kv_dequantize(_cache(**bad), 0, 4, 4096, 4096, None) == 1, bad
        assert lib.ahq_kv_attend(_cache(**bad), _queries(), None, 0, None) == 1, bad
        assert lib.ahq_kv_attend_workspace_bytes(_cache(**bad), _queries()) == 0
    for bad in NO_KERNEL:
        assert lib.ahq_kv_append(_cache(**bad), _tokens(), None) == _lib.AHQ_ERR_UNSUPPORTED, bad
        assert lib.ahq_kv_dequantize(_cache(**bad), 0, 4, 4096, 4096, None) == _lib.AHQ_ERR_UNSUPPORTED, bad
        assert lib.ahq_kv_attend(_cache(**bad), _queries(), None, 0, None) == _lib.AHQ_ERR_UNSUPPORTED, bad
    null = ctypes.POINTER(_lib.KvCache)()
    assert lib.ahq_kv_append(null, _tokens(), None) == 1 and lib.ahq_kv_attend(null, _queries(), None, 0, None) == 1
    c = _cache()
    for bad in (dict(dtype=5), dict(tokens=-1), dict(k=None), dict(v=None), dict(k=(1 << 12) + 2)):
        assert lib.ahq_kv_append(c, _tokens(**bad), None) == 1, bad
    assert lib.ahq_kv_append(c, _tokens(tokens=0, k=None, v=None), None) == 0
    assert lib.ahq_kv_append(c, _tokens(tokens=(1 << 28) + 1), None) == _lib.AHQ_ERR_UNSUPPORTED
    for length in (-1, 129):
        assert lib.ahq_kv_dequantize(c, 0, length, 4096, 4096, None) == 1
    assert lib.ahq_kv_dequantize(c, 0, 4, None, 4096, None) == 1 and lib.ahq_kv_dequantize(c, 9, 4, 4096, 4096, None) == 1
    assert lib.ahq_kv_dequantize(c, 0, 4, 4096, 4100, None) == 1 and lib.ahq_kv_dequantize(c, 0, 0, None, None, None) == 0
    large = _cache(batch=1, heads=1, capacity=1 << 30)
    assert lib.ahq_kv_dequantize(large, 0, (1 << 29) + 1, 4096, 4096, None) == _lib.AHQ_ERR_UNSUPPORTED
    for bad in (dict(dtype=3), dict(heads=3), dict(heads=0), dict(queries=-1), dict(q=None), dict(out=None), dict(q=(1 << 12) + 1),
                dict(queries=1 << 20), dict(scale=math.inf), dict(scale=-math.inf), dict(scale=math.nan), dict(scale=3e38)):
        assert lib.ahq_kv_attend(c, _queries(**bad), None, 0, None) == 1, bad
    assert lib.ahq_kv_attend(c, _queries(queries=0, q=None, out=None), None, 0, None) == 0


def test_attend_workspace(lib):
    """Nothing while the token axis is not split; a split needs its partial answers and two numbers a row."""
    assert lib.ahq_kv_attend_workspace_bytes(_cache(), _queries()) == 0  # two tiles: one workgroup takes them
    long = _cache(capacity=1 << 17)
    need = lib.ahq_kv_attend_workspace_bytes(long, _queries(length=1 << 17))
    assert need > 0 and need % (16 * (64 + 2) * 4) == 0
    assert lib.ahq_kv_attend_workspace_bytes(long, _queries(lengths=4096)) >= need  # by the capacity
    assert lib.ahq_kv_attend_workspace_bytes(long, _queries(length=256)) == 0
    assert lib.ahq_kv_attend(long, _queries(length=1 << 17), None, 0, None) == _lib.AHQ_ERR_WORKSPACE
    assert lib.ahq_kv_attend(long, _queries(length=1 << 17), 4096, need - 1, None) == _lib.AHQ_ERR_WORKSPACE


def test_front_end_refusals():
    with pytest.raises(_lib.HipLibraryError):
        QuantizedKVCache(1, 1, 64, 64, device="cpu")
    for bad in ((0, 1, 64, 64), (1, 0, 64, 64), (1, 1, 0, 64), (1, 1, 64, 80), (1, 1, 64, 64, 48), (256, 256, 64, 64),
                (1, 1, (1 << 30) + 1, 64)):
        with pytest.raises(RuntimeError):
            QuantizedKVCache(*bad)
    with pytest.raises(_lib.HipLibraryError):
        PackedWeight.pack(torch.zeros(4, 32), torch.ones(4, 1))
    with pytest.raises(RuntimeError):
        PackedWeight.pack(torch.zeros(32), torch.ones(4, 1))
    with pytest.raises(_lib.HipLibraryError):
        w = PackedWeight.__new__(PackedWeight)
        w.shape = (4, 32)
        packed_linear(torch.zeros(1, 32), w)
