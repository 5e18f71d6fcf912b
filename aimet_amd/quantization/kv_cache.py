"""A key/value cache held in 8 bits, and attention over it.

Keys and values are stored as codes in [-127, 127] on a symmetric grid whose scale belongs to a block of 16, 32 or 64
tokens of one sequence and head: a code stands for ``code * amax / 127``, amax being the block's largest magnitude.  A
block that is written in several steps keeps one scale: where a new token is larger than everything before it, the codes
the block already has are rounded onto the wider grid.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from aimet_amd import _lib
from aimet_amd.quantization.affine.packed import _refuse_gradients

__all__ = ["QuantizedKVCache"]

PerSequence = Union[int, torch.Tensor]


class QuantizedKVCache:
    """Keys and values of ``batch`` sequences and ``kv_heads`` heads, up to ``capacity`` tokens each.

    The cache keeps no lengths: the caller says where tokens go (``start``) and how many a sequence holds
    (``lengths``), as whole numbers for all sequences or as one int32 tensor entry for each.  Values of such a tensor
    are not read back; positions outside the cache are dropped by ``append``, and lengths are limited to the capacity
    by ``attend``.  Calls run on the current stream; two calls that touch the same cache on different streams have to be
    ordered by the caller."""

    def __init__(self, batch: int, kv_heads: int, capacity: int, head_dim: int, block_tokens: int = 64, device="cuda"):
        if min(batch, kv_heads, capacity) <= 0:
            raise RuntimeError(f"batch, kv_heads and capacity must be positive; got {batch}, {kv_heads}, {capacity}")
        if head_dim not in (64, 128, 256):
            raise RuntimeError(f"head_dim must be 64, 128 or 256; got {head_dim}")
        if block_tokens not in (16, 32, 64):
            raise RuntimeError(f"block_tokens must be 16, 32 or 64; got {block_tokens}")
        if batch * kv_heads > 65535:
            raise RuntimeError(f"batch * kv_heads must be at most 65535; got {batch * kv_heads}")
        if capacity > 1 << 30:
            raise RuntimeError(f"capacity must be at most 2**30 tokens; got {capacity}")
        device = torch.device(device)
        if device.type != "cuda":
            raise _lib.HipLibraryError(f"the cache lives on '{device}': the HIP backend only runs on GPU tensors and has "
                                       "no CPU fallback")
        self.batch, self.kv_heads, self.head_dim, self.block_tokens = batch, kv_heads, head_dim, block_tokens
        self.capacity = -(-capacity // 64) * 64  # in whole tiles of 64 tokens
        blocks = self.capacity // block_tokens
        # bytes hold code + 128, a tile of 64 tokens in the order in which the matrix cores take it
        self.k_codes = torch.full((batch, kv_heads, self.capacity // 64, 4, head_dim // 64, 4, 16, 16), 128,
                                  dtype=torch.uint8, device=device)
        self.v_codes = torch.full((batch, kv_heads, self.capacity // 64, head_dim // 16, 4, 16, 16), 128,
                                  dtype=torch.uint8, device=device)
        self.k_amax = torch.zeros(batch, kv_heads, blocks, dtype=torch.float32, device=device)
        self.v_amax = torch.zeros(batch, kv_heads, blocks, dtype=torch.float32, device=device)
        self.device = self.k_codes.device
        self._bind()

    def _bind(self) -> None:
        self._struct = _lib.KvCache(self.batch, self.kv_heads, self.capacity, self.head_dim, self.block_tokens,
                                    self.k_codes.data_ptr(), self.v_codes.data_ptr(), self.k_amax.data_ptr(),
                                    self.v_amax.data_ptr())

    def __getstate__(self):
        # the structure handed to the library holds addresses: copies and pickles make their own
        return {k: v for k, v in self.__dict__.items() if k != "_struct"}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._bind()

    def _per_sequence(self, n: PerSequence, what: str, most: int) -> Tuple[Optional[int], int]:
        """(device pointer or None, value for all sequences) of a whole number or an int32 tensor [batch]."""
        if isinstance(n, torch.Tensor):
            if n.dtype != torch.int32 or tuple(n.shape) != (self.batch,) or n.device != self.device:
                raise RuntimeError(f"{what} must be a whole number or an int32 tensor of shape {(self.batch,)} on "
                                   f"{self.device}; got {n.dtype}, {tuple(n.shape)}, {n.device}")
            if not n.is_contiguous():
                raise RuntimeError(f"{what} must be contiguous")
            return n.data_ptr(), 0
        if isinstance(n, bool) or not isinstance(n, int):
            raise RuntimeError(f"{what} must be a whole number or an int32 tensor; got {type(n).__name__}")
        if not 0 <= n <= most:
            raise RuntimeError(f"{what} must be in [0, {most}]; got {n}")
        return None, n

    def _check(self, t: torch.Tensor, what: str, heads: Optional[int] = None) -> None:
        _lib.require_device(t, what)
        if t.device != self.device:
            raise RuntimeError(f"{what} is on {t.device}, the cache on {self.device}")
        if t.dtype not in _lib.DTYPE_CODE:
            raise RuntimeError(f"{what} must be float32, bfloat16 or float16; got {t.dtype}")
        if t.dim() != 4 or t.shape[0] != self.batch or t.shape[3] != self.head_dim or (heads and t.shape[1] != heads):
            raise RuntimeError(f"{what} of shape {tuple(t.shape)} does not fit a cache of {self.batch} sequences, "
                               f"{self.kv_heads} heads and head size {self.head_dim}")

    def _call(self, name: str, *args) -> None:
        fn = getattr(_lib.load(), name)
        if self.device.index == torch.cuda.current_device():
            status = fn(*args, _lib.current_stream(self.device))
        else:
            with torch.cuda.device(self.device):
                status = fn(*args, _lib.current_stream(self.device))
        _lib.check(status, name)

    def codes(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """The stored codes of keys and values as two int8 tensors [batch, kv_heads, capacity, head_dim]."""
        shape = (self.batch, self.kv_heads, self.capacity, self.head_dim)
        k = self.k_codes.unflatten(6, (4, 4)).permute(0, 1, 2, 6, 3, 7, 4, 5, 8)  # tile, g, s, r, u, c, e
        v = self.v_codes.permute(0, 1, 2, 4, 6, 3, 5)                             # tile, c, e, u, i
        return tuple((x.reshape(shape).to(torch.int16) - 128).to(torch.int8) for x in (k, v))

    def append(self, k: torch.Tensor, v: torch.Tensor, start: PerSequence,
               counts: Optional[PerSequence] = None) -> None:
        """Stores keys and values [batch, kv_heads, tokens, head_dim] (any strides): token t of a sequence goes to
        position ``start + t``; of a padded batch only the first ``counts`` tokens of each sequence are stored.  Infinite
        values saturate and NaN is stored as 0; neither sets a block's scale.

        A block that ``start`` lies inside keeps the scale it has, and this is also that of tokens which stood at ``start`` or
        behind it: where those were discarded (rejected drafts), what the block holds and what is appended to it stay on their
        grid, until a call begins at the block's first token.  What stands behind the last new token of a block counts as
        discarded: its codes stay, but the scale may be another."""
        self._check(k, "k", self.kv_heads)
        self._check(v, "v", self.kv_heads)
        if k.shape != v.shape or k.dtype != v.dtype:
            raise RuntimeError(f"k ({tuple(k.shape)}, {k.dtype}) and v ({tuple(v.shape)}, {v.dtype}) differ")
        _refuse_gradients("QuantizedKVCache.append", k, v)
        tokens = k.shape[2]
        count_ptr, count = self._per_sequence(tokens if counts is None else counts, "counts", tokens)
        start_ptr, first = self._per_sequence(start, "start", self.capacity)
        if start_ptr is None and count_ptr is None and first + count > self.capacity:
            raise RuntimeError(f"{count} tokens from position {first} on do not fit a cache of {self.capacity} tokens")
        if tokens == 0:
            return
        if k.stride(3) != 1:
            k = k.contiguous()
        if v.stride(3) != 1:
            v = v.contiguous()
        ks, vs = k.stride(), v.stride()
        x = _lib.KvTokens(_lib.DTYPE_CODE[k.dtype], tokens, k.data_ptr(), v.data_ptr(), (ks[0], vs[0]), (ks[1], vs[1]),
                          (ks[2], vs[2]), start_ptr, count_ptr, first, count)
        self._call("ahq_kv_append", self._struct, x)

    def dequantize(self, length: Optional[int] = None, dtype: torch.dtype = torch.float32):
        """The values of the first ``length`` tokens (all by default) as two tensors [batch, kv_heads, length,
        head_dim].  Positions that were never written read 0."""
        length = self.capacity if length is None else length
        if isinstance(length, bool) or not isinstance(length, int) or not 0 <= length <= self.capacity:
            raise RuntimeError(f"length must be a whole number in [0, {self.capacity}]; got {length}")
        if dtype not in _lib.DTYPE_CODE:
            raise RuntimeError(f"dtype must be float32, bfloat16 or float16; got {dtype}")
        k = torch.empty(self.batch, self.kv_heads, length, self.head_dim, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        if length:
            self._call("ahq_kv_dequantize", self._struct, _lib.DTYPE_CODE[dtype], length, k.data_ptr(), v.data_ptr())
        return k, v

    def attend(self, q: torch.Tensor, lengths: PerSequence, counts: Optional[PerSequence] = None,
               scale: Optional[float] = None) -> torch.Tensor:
        """Causal attention of the queries [batch, query_heads, queries, head_dim] (any strides; query_heads a multiple
        of kv_heads, neighbouring query heads share a key head; fewer than 2^20 queries a key head) over the stored
        tokens.  A sequence holds ``lengths`` tokens and its queries are the last ``queries`` of them (of a padded
        batch: its first ``counts`` queries are the last ``counts`` tokens): query t sees the tokens up to its own
        position, ``lengths - counts + t``.  Queries that see nothing, and those behind ``counts``, are answered with 0.
        ``scale`` multiplies the scores (default 1 / sqrt(head_dim)).  The result has the queries' type, shape and,
        where they are dense, memory layout.

        16-bit queries are used as they are (bfloat16 down to 2^-30 of a row's largest value), float32 queries to 22
        bits, those far below a row's largest value to fewer; probabilities have 22 bits and are off by at most 2^-35 of
        the row's largest one where they are small (both weighted by the scale of their values' block); all sums are
        float32, and the result is rounded once.  Values may be of any size; blocks whose values are all below 2^-72 of
        the largest one that the call's queries see of their sequence and head count as up to that."""
        self._check(q, "q")
        heads, queries = q.shape[1], q.shape[2]
        if heads == 0 or heads % self.kv_heads:
            raise RuntimeError(f"{heads} query heads are no multiple of the cache's {self.kv_heads}")
        _refuse_gradients("QuantizedKVCache.attend", q)
        count_ptr, count = self._per_sequence(queries if counts is None else counts, "counts", queries)
        length_ptr, length = self._per_sequence(lengths, "lengths", self.capacity)
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale)
        if not abs(scale) < 2.0 ** 126:  # as float32, with room for a factor of log2(e)
            raise RuntimeError(f"scale must be finite; got {scale}")
        if type(q) is not torch.Tensor:
            q = q.as_subclass(torch.Tensor)
        out = torch.empty_like(q)
        if queries == 0:
            return out
        if out.stride(3) != 1:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if q.stride(3) != 1:
            q = q.contiguous()
        qs, os_ = q.stride(), out.stride()
        x = _lib.KvQueries(_lib.DTYPE_CODE[q.dtype], heads, queries, q.data_ptr(), out.data_ptr(), qs[0], qs[1], qs[2],
                           os_[0], os_[1], os_[2], length_ptr, count_ptr, length, count, scale)
        nbytes = _lib.load().ahq_kv_attend_workspace_bytes(self._struct, x)
        # allocated anew for each call: a captured graph then owns its scratch, and no two calls share one
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        self._call("ahq_kv_attend", self._struct, x, _lib.ptr(ws), nbytes)
        return out
