"""Linear layers that run on the codes of a 4-bit weight instead of on a quantize-dequantized copy of it.

``PackedWeight`` holds what a calibrated weight quantizer of at most 16 levels describes: the codes, two to a byte in the
order the kernel reads them, and one float32 scale (and, for grids that are not symmetric, one whole zero point) per
output channel and group of columns.  ``packed_linear`` is ``torch.nn.functional.linear`` on it, for up to 2^20 rows and
results of up to 2^22 blocks of 64 x 256 values (float32: 32 x 128):

    y[m, n] = sum_g scale[n, g] * sum_{k in g} x[m, k] * (code[n, k] + offset[n, g] + zero_point_shift)  +  bias[n]

Products are exact and sums are float32; the result is rounded once, to the activations' type.  (Quantize-dequantizing a
bfloat16 weight rounds code * scale to bfloat16; here the scale stays float32, so the two agree to that rounding.)
There is no backward pass and no forward-mode derivative: the weight is frozen and the calls are those of inference;
tensors that require gradients or carry tangents are refused.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd import forward_ad

from aimet_amd import _lib
from aimet_amd.quantization._utils import concretize_block_size

__all__ = ["PackedWeight", "NotPackable", "packed_linear"]


class NotPackable(RuntimeError):
    """A weight or an encoding that has no packed form."""


def _refuse_gradients(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad() or on tensors that do not "
                           "require gradients")
    # tangents are carried whether gradients are enabled or not
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None  # pylint: disable=protected-access
                                              for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative: call it on tensors without tangents")


class PackedWeight:
    """The codes of a weight [out_features, in_features] with at most 16 levels, packed for ``packed_linear``.

    Attributes: ``codes`` (uint8, the library's layout), ``scale`` (float32 [out_features / 16, groups, 16], channels in
    sixteens and padded to them), ``zero`` (int8 of the same shape, or None where one zero point serves all),
    ``zero_const``, ``shape``, ``group`` (columns that share a scale)."""

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor], zero_const: float,
                 shape, group: int):
        self.codes, self.scale, self.zero, self.zero_const = codes, scale, zero, float(zero_const)
        self.shape, self.group = tuple(int(d) for d in shape), int(group)
        n, k = self.shape
        nbytes = _lib.load().ahq_int4_packed_bytes(n, k)
        if nbytes == 0 or codes.dtype != torch.uint8 or codes.numel() != nbytes or not codes.is_contiguous():
            raise RuntimeError(f"{tuple(codes.shape)} bytes of {codes.dtype} are no packed weight of shape {self.shape}")
        if self.group <= 0 or k % self.group or (self.group != k and self.group % 32):
            raise RuntimeError(f"groups must be a multiple of 32 columns that divides {k}, or all of them; got {group}")
        expected = (-(-n // 16), k // self.group, 16)
        for name, t, dtype in (("scale", scale, torch.float32), ("zero", zero, torch.int8)):
            if t is not None and (tuple(t.shape) != expected or t.dtype != dtype or not t.is_contiguous()
                                  or t.device != codes.device):
                raise RuntimeError(f"{name} must be a contiguous {dtype} tensor of shape {expected} on {codes.device}")
        self._struct = _lib.Int4Weight(n, k, self.group, codes.data_ptr(), scale.data_ptr(), _lib.ptr(zero), self.zero_const)

    def __getstate__(self):
        # the structure handed to the library holds addresses: copies and pickles make their own
        return {k: v for k, v in self.__dict__.items() if k != "_struct"}

    def __setstate__(self, state):
        self.__init__(*(state[k] for k in ("codes", "scale", "zero", "zero_const", "shape", "group")))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @classmethod
    def pack(cls, codes: torch.Tensor, scale: torch.Tensor, offset: Optional[torch.Tensor] = None,
             qmin: Optional[int] = None, zero_point_shift: float = 0.0) -> "PackedWeight":
        """``codes``: whole numbers [out_features, in_features] in [qmin, qmin + 15] (any dtype that holds them; qmin
        defaults to -8 without offsets and to 0 with them).  ``scale`` / ``offset``: [out_features, groups], the
        offsets whole numbers.  Reads the codes' and offsets' range back, so it synchronises: it is called once per
        weight."""
        if codes.dim() != 2 or codes.numel() == 0:
            raise RuntimeError(f"a weight of two dimensions is expected; got shape {tuple(codes.shape)}")
        _lib.require_device(codes, "codes")
        n, k = codes.shape
        if scale.dim() != 2 or scale.shape[0] != n or scale.shape[1] == 0 or k % scale.shape[1]:
            raise RuntimeError(f"scale must be [{n}, groups] with groups dividing {k}; got {tuple(scale.shape)}")
        if offset is not None and offset.shape != scale.shape:
            raise RuntimeError(f"offset has shape {tuple(offset.shape)}, scale {tuple(scale.shape)}")
        if any(t is not None and t.device != codes.device for t in (scale, offset)):
            raise RuntimeError("codes, scale and offset must be on one device")
        groups = scale.shape[1]
        if groups > 1 and (k // groups) % 32:
            raise NotPackable(f"groups of {k // groups} columns are not supported: a multiple of 32, or the whole row")
        qmin = (-8 if offset is None else 0) if qmin is None else int(qmin)
        if not -128 <= qmin <= 112:
            raise NotPackable(f"qmin must be in [-128, 112]; got {qmin}")
        # everything that has to be known of the values is read back at once
        known = [t.double() for t in torch.aminmax(codes)]
        if codes.is_floating_point():
            known.append((codes == codes.round()).all().double())
        if offset is not None:
            off = offset.detach().float()
            known += [t.double() for t in (*torch.aminmax(off), (off == off.round()).all())]
        lo, hi, *about_offset = torch.stack(known).tolist()
        if codes.is_floating_point() and not about_offset.pop(0):
            raise RuntimeError("codes must be whole numbers")
        if not qmin <= lo <= hi <= qmin + 15:
            raise RuntimeError(f"codes in [{lo:g}, {hi:g}] do not fit the 16 levels from {qmin} on")
        npad = -(-n // 16) * 16

        def in_sixteens(t, dtype):
            # rows of the padding have the scale 0 and are never stored
            out = torch.zeros(npad, groups, dtype=dtype, device=codes.device)
            out[:n] = t
            return out.view(npad // 16, 16, groups).transpose(1, 2).contiguous()

        scales = in_sixteens(scale.detach(), torch.float32)
        zero, zero_const = None, qmin + float(zero_point_shift)
        if offset is not None:
            o_lo, o_hi, whole = about_offset
            if not (math.isfinite(o_lo) and math.isfinite(o_hi) and whole):
                raise NotPackable("offsets must be whole numbers")
            if o_lo == o_hi:
                zero_const += o_lo
            else:
                if o_lo + qmin < -128 or o_hi + qmin > 127:
                    raise NotPackable(f"offset + qmin in [{o_lo + qmin}, {o_hi + qmin}] does not fit 8 bits")
                zero = in_sixteens(off + qmin, torch.int8)
                zero_const = float(zero_point_shift)
        lib = _lib.load()
        nbytes = lib.ahq_int4_packed_bytes(n, k)
        if nbytes == 0:
            raise NotPackable(f"a weight of shape {(n, k)} is too large to pack")
        packed = torch.empty(nbytes, dtype=torch.uint8, device=codes.device)
        raw = codes.detach().to(torch.int8).contiguous()
        with torch.cuda.device(codes.device):
            _lib.check(lib.ahq_int4_pack(raw.data_ptr(), n, k, qmin, packed.data_ptr(),
                                         _lib.current_stream(codes.device)), "ahq_int4_pack")
        return cls(packed, scales, zero, zero_const, (n, k), k // groups)

    @classmethod
    def from_encoding(cls, weight: torch.Tensor, encoding) -> "PackedWeight":
        """The packed form of a weight under an affine encoding (per tensor, per channel or blockwise, grouped block
        scales included) of at most 16 levels: the codes are those of ``encoding.quantize``, and on a shifted grid those
        of the values of ``encoding.quantize_dequantize``."""
        if weight.dim() != 2:
            raise RuntimeError(f"a weight of two dimensions is expected; got shape {tuple(weight.shape)}")
        if encoding.qmax - encoding.qmin > 15:
            raise NotPackable(f"the grid [{encoding.qmin}, {encoding.qmax}] has more than 16 levels")
        n, k = weight.shape
        with torch.no_grad():
            weight = weight.detach().as_subclass(torch.Tensor)

            def spread(t):
                t = t.detach().as_subclass(torch.Tensor).float()
                if t.numel() == 1:
                    return t.reshape(1, 1).expand(n, 1)
                t = t.reshape((1,) * (2 - t.dim()) + tuple(t.shape)) if t.dim() < 2 else t
                rows = n // t.shape[0]
                return t.repeat_interleave(rows, 0) if rows > 1 else t

            scale, offset = spread(encoding.scale), spread(encoding.offset)
            if encoding.block_size is not None:
                concretize_block_size((n, k), tuple(encoding.scale.shape), encoding.block_size)  # its own errors
            if scale.shape[1] not in (1, k) and encoding.block_size is None:
                raise NotPackable(f"scale of shape {tuple(encoding.scale.shape)} does not describe a weight of {(n, k)}")
            shift = encoding.zero_point_shift or 0.0
            if shift == 0.0:
                codes = encoding.quantize(weight).as_subclass(torch.Tensor)
            else:
                # quantize() knows no shift: what lies on the shifted grid lies half-way between its codes
                if scale.shape[0] != n or k % scale.shape[1]:
                    raise NotPackable(f"scale of shape {tuple(encoding.scale.shape)} does not describe a weight of {(n, k)}")
                on_grid = encoding.quantize_dequantize(weight).as_subclass(torch.Tensor).float()
                levels = on_grid.reshape(n, scale.shape[1], -1) / scale[..., None] - offset[..., None] - shift
                codes = levels.round().clamp(encoding.qmin, encoding.qmax).reshape(n, k)
            return cls.pack(codes, scale, offset, encoding.qmin, shift)


def packed_linear(x: torch.Tensor, weight: PackedWeight, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ dequantized(weight).T + bias`` for activations [..., in_features] in float32, bfloat16 or float16; the
    result has their type.  An infinite or NaN activation makes its row NaN, as do sums of activations times codes that
    leave float32 before the scale is applied."""
    n, k = weight.shape
    _lib.require_device(x, "x")
    if x.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"activations must be float32, bfloat16 or float16; got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] != k:
        raise RuntimeError(f"activations of shape {tuple(x.shape)} do not fit a weight of shape {(n, k)}")
    device = x.device
    if weight.codes.device != device:
        raise RuntimeError(f"activations are on {device}, the weight on {weight.codes.device}")
    if bias is not None and (bias.shape != (n,) or bias.dtype != x.dtype or bias.device != device):
        raise RuntimeError(f"bias must have shape {(n,)} and the activations' type and device; got "
                           f"{tuple(bias.shape)}, {bias.dtype}, {bias.device}")
    _refuse_gradients("packed_linear", x, bias)
    if type(x) is not torch.Tensor:
        x = x.as_subclass(torch.Tensor)
    y = x.new_empty(x.shape[:-1] + (n,))
    m = y.numel() // n
    if m == 0:
        return y
    rows = x if x.dim() == 2 else x.reshape(m, k)
    if (k > 1 and rows.stride(1) != 1) or (m > 1 and rows.stride(0) < k):
        rows = rows.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    args = (weight._struct, _lib.DTYPE_CODE[x.dtype], rows.data_ptr(), m, rows.stride(0) if m > 1 else k, _lib.ptr(bias),
            y.data_ptr(), n)
    if device.index == torch.cuda.current_device():
        status = _lib.load().ahq_int4_linear(*args, _lib.current_stream(device))
    else:
        with torch.cuda.device(device):
            status = _lib.load().ahq_int4_linear(*args, _lib.current_stream(device))
    _lib.check(status, "ahq_int4_linear")
    return y
