"""A key/value cache held in 8 bits, and the attention that reads it.

A program that answers many queries against a forecast state (stations, a path, one point, for each
member and lead time) keeps the state's keys and values on the card.  Here they are held in 8 bits, with
a scale for each block of tokens and kv head: half the bytes of bfloat16 to hold, and to read at each
query.

* ``KVCache(batch, capacity, kv_heads, block_size=64, dtype=torch.int8)``: the storage.
* ``kv_cache_write(cache, k, v, start=0, counts=None)``: quantises tokens as it writes them: a whole
  state, a run of tokens, or one token of each sequence.
* ``kv_cache_read(cache, start=0, count=None, dtype=torch.bfloat16)``: the values the cache holds.
* ``cache_attn(q, cache, block_indices=None, softmax_scale=None, kv_lens=None)``: attention of each query
  over the whole sequence, or over key blocks of its own.
* ``cache_query_attn(q, cache, block_count, ...)``: ``query_topk`` on the cache's own block means, then
  the attention.

None of them has a gradient.  They enqueue on the current stream of the cache's device and never
synchronise the host; calls that write to a cache and calls that read it are ordered by the program, as
for any tensor.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import forward_only
from .query import _as_bf16, _bf16_heads, _scale, _scratch, query_topk
from .rotary import _DT, _like, _on, _ptr, _rows, _same_device, _stream

__all__ = ["KVCache", "kv_cache_write", "kv_cache_read", "cache_attn", "cache_query_attn"]

_CODES = {torch.int8: _lib.CODE_INT8, torch.float8_e4m3fn: _lib.CODE_E4M3}


class KVCache:
    """Keys and values of ``batch`` sequences of up to ``capacity`` tokens in 8 bits.

    ``dtype``: ``torch.int8`` (codes -127 .. 127, even steps) or ``torch.float8_e4m3fn`` (codes up to 448,
    relative steps: for blocks with a few large values among small ones).  ``block_size`` (64, 128 or 256
    tokens) is the reach of a scale and the unit of ``block_indices``.  A new cache is empty: all zeros.

    The lengths of the sequences are the program's own (``kv_lens`` of the attention).  ``k_scale`` and
    ``v_scale`` (float32 [batch, num_blocks, kv_heads]), ``k_mean`` (bfloat16 [batch, num_blocks, kv_heads,
    64], the mean of the keys of each block: ``k_cmp`` of ``query_topk``), ``k_norm`` (float32 as the scales, the
    largest norm of a key of the block) and the codes, in an order of the library's
    own, are tensors of the cache: ``kv_cache_write`` changes them in place, as autograd sees.
    """

    def __init__(self, batch: int, capacity: int, kv_heads: int, block_size: int = 64, dtype: torch.dtype = torch.int8,
                 device="cuda"):
        batch, capacity, kv_heads, block_size = int(batch), int(capacity), int(kv_heads), int(block_size)
        if batch < 1 or capacity < 1 or not 1 <= kv_heads <= 65535:
            raise ValueError(f"KVCache: batch, capacity and kv_heads must be positive, kv_heads at most 65535, got {batch}, {capacity}, {kv_heads}")
        if block_size not in (64, 128, 256):
            raise ValueError(f"KVCache: block_size must be 64, 128 or 256, got {block_size}")
        if dtype not in _CODES:
            raise TypeError(f"KVCache: dtype must be torch.int8 or torch.float8_e4m3fn, got {dtype}")
        nb = -(-capacity // block_size)
        if nb * block_size > (1 << 31) - 1025 or nb * (block_size // 64) * kv_heads * batch > (1 << 31) - 1025:
            raise ValueError(f"KVCache: {batch} sequences of {capacity} tokens and {kv_heads} heads are more than 2^31 tiles of 64 tokens, "
                             "or a sequence more than 2^31 tokens")
        self._sizes = (batch, nb, kv_heads, block_size, capacity)
        self._dtype = dtype
        shape = (batch, nb, kv_heads)
        self._k_codes, self._v_codes = (torch.zeros(*shape, block_size * 64, dtype=torch.uint8, device=device) for _ in range(2))
        self._k_scale, self._v_scale, self._k_norm = (torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(3))
        self._k_mean = torch.zeros(*shape, 64, dtype=torch.bfloat16, device=device)
        self._describe()

    def _describe(self) -> None:
        """The storage as the library takes it: made once, the tensors being the cache's own for its life."""
        B, nb, Hk, bs, capacity = self._sizes
        self._device = self._k_codes.device
        self._tensors = (self._k_codes, self._v_codes, self._k_scale, self._v_scale, self._k_norm, self._k_mean)
        self._c = _lib.Cache(self._k_codes.data_ptr(), self._v_codes.data_ptr(), self._k_scale.data_ptr(), self._v_scale.data_ptr(),
                             self._k_norm.data_ptr(), self._k_mean.data_ptr(), B, nb, Hk, bs, _CODES[self._dtype], capacity)

    def __getstate__(self) -> dict:   # (copies and pickles: of the tensors, not of where they lie)
        return {name: x for name, x in self.__dict__.items() if name not in ("_c", "_device", "_tensors")}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self._describe()

    batch = property(lambda self: self._sizes[0])
    num_blocks = property(lambda self: self._sizes[1])
    kv_heads = property(lambda self: self._sizes[2])
    block_size = property(lambda self: self._sizes[3])
    capacity = property(lambda self: self._sizes[4])
    dtype = property(lambda self: self._dtype)
    device = property(lambda self: self._device)
    k_codes = property(lambda self: self._k_codes)
    v_codes = property(lambda self: self._v_codes)
    k_scale = property(lambda self: self._k_scale)
    v_scale = property(lambda self: self._v_scale)
    k_norm = property(lambda self: self._k_norm)
    k_mean = property(lambda self: self._k_mean)

    def __repr__(self) -> str:
        B, _, Hk, bs, capacity = self._sizes
        return (f"KVCache(batch={B}, capacity={capacity}, kv_heads={Hk}, block_size={bs}, dtype={self._dtype}, "
                f"device={str(self.device)!r})")


def _no_gradient(what: str, **tensors) -> None:
    """Refuses inputs that autograd would follow, in either mode."""
    if torch.is_grad_enabled():
        forward_only(what, *tensors.values())
    if forward_ad._current_level >= 0:
        for name, t in tensors.items():
            if forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no derivative in forward mode, and {name} carries a tangent")


def _per_sequence(what: str, name: str, t: torch.Tensor, batch: int) -> None:
    if tuple(t.shape) != (batch,):
        raise ValueError(f"{what}: {name} {tuple(t.shape)} must be [B] = ({batch},)")
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: {name} are {t.dtype}, not int64 or int32")


def _int32(t: torch.Tensor | None, low: int, high: int) -> torch.Tensor | None:
    """t as the kernels read it; clamped before the conversion, so that a far value stays one."""
    if t is None or (t.dtype is torch.int32 and t.is_contiguous()):
        return t
    return (t if t.dtype is torch.int32 else t.clamp(low, high).to(torch.int32)).contiguous()


def _run(what: str, cache: KVCache, start, count: int):
    """(start, starts): one of a number, checked, and a tensor of one for each sequence."""
    if isinstance(start, torch.Tensor):
        _per_sequence(what, "start", start, cache.batch)
        return 0, start
    start = int(start)
    if start < 0 or start + count > cache.capacity:
        raise ValueError(f"{what}: tokens {start} .. {start + count - 1} do not lie in a cache of {cache.capacity}")
    return start, None


def kv_cache_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, start: int | torch.Tensor = 0,
                   counts: torch.Tensor | None = None) -> None:
    """Quantises k and v ([B, n, kv_heads, 64], bfloat16 or float32, any strides) into the cache.

    Token i of sequence b goes to position ``start + i`` (``start``: a number, or integers [B] on the cache's
    device), for i below ``counts[b]`` where ``counts`` (integers [B]) is given, clamped to 0 .. n: a padded
    batch.  Positions outside the cache are left out where ``start`` is a tensor and refused where it is a
    number.  A sequence ends with the tokens written: earlier tokens stay, later ones of the blocks written to
    become zeros, and blocks behind those stay as they are (the attention's ``kv_lens`` leaves them out).

    Each block of tokens and head, of k and of v, has one scale: the largest magnitude among its new tokens
    over the largest code (127 or 448) as float32, and at least the scale it had where earlier tokens of the
    block are kept, whose codes are then set to the new scale (a rounding more for them each time it grows).
    A code is the value over the scale, to the nearest, ties to even.  A block without a magnitude of 2^-100 or
    more holds zeros; one with a value that is not finite holds NaN throughout.
    """
    what = "kv_cache_write"
    B, _, Hk, _, _ = cache._sizes
    shape, dtype, device = k.shape, k.dtype, cache._device
    if len(shape) != 4 or shape[0] != B or shape[2] != Hk or shape[3] != 64:
        raise ValueError(f"{what}: k {tuple(shape)} must be [B, n, kv_heads, 64] = {(B, '*', Hk, 64)}")
    if dtype not in _DT:
        raise TypeError(f"{what}: k is {dtype}; bfloat16 and float32 are quantised")
    if v.shape != shape or v.dtype != dtype:
        raise ValueError(f"{what}: k {tuple(shape)} {dtype} and v {tuple(v.shape)} {v.dtype} disagree")
    n = shape[1]
    if n >= 1 << 31:
        raise ValueError(f"{what}: {n} tokens are 2^31 or more")
    _no_gradient(what, k=k, v=v)
    start, starts = _run(what, cache, start, n)
    if counts is not None:
        _per_sequence(what, "counts", counts, B)
    _same_device(what, cache._k_codes, of="the cache", k=k, v=v, start=starts, counts=counts)
    if n == 0:
        return
    starts, counts = _int32(starts, -1 << 31, (1 << 31) - 1), _int32(counts, 0, n)
    (k, kb), (v, vb) = _rows(k), _rows(v)
    with _on(device):
        st = _lib.lib().mosaic_kv_cache_write(ctypes.byref(cache._c), kb, vb, _DT[dtype], 64, n, start, _ptr(starts), _ptr(counts), _stream(device))
    _lib.check(st, "mosaic_kv_cache_write")
    torch.autograd.graph.increment_version(cache._tensors)   # (what was saved of them for a backward is no longer there)


def kv_cache_read(cache: KVCache, start: int | torch.Tensor = 0, count: int | None = None,
                  dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The values of ``count`` tokens from position ``start`` on: (k, v), [B, count, kv_heads, 64] in ``dtype``.

    ``start`` is a number, or integers [B] on the cache's device: positions outside the cache are then zeros,
    where a number is refused.  ``count`` defaults to the rest of the cache (of a number).  A value is code
    times scale, rounded once to ``dtype`` (bfloat16 or float32).
    """
    what = "kv_cache_read"
    B, _, Hk, _, capacity = cache._sizes
    device = cache._device
    if dtype not in _DT:
        raise TypeError(f"{what}: dtype is {dtype}; bfloat16 and float32 are read")
    if count is None:
        if isinstance(start, torch.Tensor):
            raise ValueError(f"{what}: count is needed where start is a tensor")
        count = capacity - int(start)
    count = int(count)
    if not 0 <= count < 1 << 31:
        raise ValueError(f"{what}: count must be in [0, 2^31), got {count}")
    start, starts = _run(what, cache, start, count)
    _same_device(what, cache._k_codes, of="the cache", start=starts)
    k = torch.empty(B, count, Hk, 64, dtype=dtype, device=device)
    v = torch.empty_like(k)
    if count == 0:
        return k, v
    starts = _int32(starts, -1 << 31, (1 << 31) - 1)
    with _on(device):
        st = _lib.lib().mosaic_kv_cache_read(ctypes.byref(cache._c), _DT[dtype], 64, count, start, _ptr(starts), k.data_ptr(), v.data_ptr(),
                                             _stream(device))
    _lib.check(st, "mosaic_kv_cache_read")
    return k, v


def _check_queries(what: str, q: torch.Tensor, cache: KVCache, kv_lens: torch.Tensor | None) -> None:
    _bf16_heads(what, q=q)
    B, Nq, Hq, _ = q.shape
    Hk = cache.kv_heads
    if B != cache.batch:
        raise ValueError(f"{what}: q {tuple(q.shape)} and the cache disagree on the batch, {B} and {cache.batch}")
    if Nq >= 1 << 31:
        raise ValueError(f"{what}: the queries must be below 2^31, got {Nq}")
    if Hq == 0 or Hq % Hk or Hq // Hk > 16:
        raise ValueError(f"{what}: {Hq} query heads must be a multiple of {Hk} kv heads, at most 16 times as many")
    if kv_lens is not None:
        _per_sequence(what, "kv_lens", kv_lens, B)
    _no_gradient(what, q=q)


def cache_attn(q: torch.Tensor, cache: KVCache, block_indices: torch.Tensor | None = None, softmax_scale: float | None = None,
               kv_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each query token over a cache: [B, Nq, Hq, 64] in q's type.

    q [B, Nq, Hq, 64] attends to every token of its sequence below ``kv_lens[b]`` (integers [B]; the
    capacity where it is None), or, with ``block_indices`` (int64 or int32 [B, Nq, kv_heads, K], K at most
    1024), to those of the blocks of ``cache.block_size`` tokens named there: a set, as in
    ``query_sparse_attn``.  A token without a key gets zeros.  ``softmax_scale`` defaults to 1/8 and lies
    within 1e-30 .. 1e30.  Scores, sums and accumulators are fp32, the weights rounded to bfloat16, as
    float32 q is; a row with scores, or sums of values over its keys, past fp32's range (2e38) is not
    defined.  There is no gradient.
    """
    what = "cache_attn"
    _check_queries(what, q, cache, kv_lens)
    B, Nq, Hq, d = q.shape
    Hk, K = cache.kv_heads, 0
    if block_indices is not None:
        if block_indices.dim() != 4 or tuple(block_indices.shape[:3]) != (B, Nq, Hk) or block_indices.shape[3] > 1024:
            raise ValueError(f"{what}: block_indices {tuple(block_indices.shape)} must be [B, Nq, kv_heads, K] = {(B, Nq, Hk, '*')}, "
                             "K at most 1024")
        if block_indices.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"{what}: block_indices are {block_indices.dtype}, not int64 or int32")
        K = block_indices.shape[3]
    scale = _scale(what, softmax_scale)
    _same_device(what, q, cache=cache._k_codes, block_indices=block_indices, kv_lens=kv_lens)
    if q.numel() == 0 or (block_indices is not None and K == 0):   # no row, or no key for any
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    lens = _int32(kv_lens, 0, cache.capacity)
    idx = block_indices
    if idx is not None and (idx.dtype is not torch.int64 or not idx.is_contiguous()):
        idx = idx.to(torch.int64).contiguous()
    dtype, device = q.dtype, q.device
    q, qb = _as_bf16(q)
    out = _like(q)
    L, c = _lib.lib(), ctypes.byref(cache._c)
    nbytes = L.mosaic_cache_attn_fwd_workspace_size(c, Nq, Hq, K)
    ws = _scratch(nbytes, device)
    with _on(device):
        st = L.mosaic_cache_attn_fwd(qb, c, _ptr(idx), _ptr(lens), Nq, Hq, d, K, scale, out.data_ptr(), _ptr(ws), nbytes,
                                     _stream(device))
    _lib.check(st, "mosaic_cache_attn_fwd")
    return out if dtype is torch.bfloat16 else out.to(dtype)


def cache_query_attn(q: torch.Tensor, cache: KVCache, block_count: int, *, softmax_scale: float | None = None,
                     kv_lens: torch.Tensor | None = None, block_mask: torch.Tensor | None = None,
                     return_block_indices: bool = False):
    """Each query token chooses ``block_count`` blocks of the cache and attends to them: [B, Nq, Hq, 64].

    ``mosaic_query_attn`` on a cache: ``query_topk`` against ``cache.k_mean``, which ``kv_cache_write`` keeps,
    then ``cache_attn``.  Blocks that begin at or past ``kv_lens[b]``, and those that ``block_mask`` (bool [B,
    num_blocks]) leaves out, are not chosen.  The mean of the block that a length ends in is that of every token
    written to it, those past the length too, though the attention leaves them out: lengths are best where the last
    write ended, which sets that block's mean.  With ``return_block_indices`` the choice (int64 [B, Nq,
    kv_heads, block_count], -1 past the last) is returned too.
    """
    what = "cache_query_attn"
    _check_queries(what, q, cache, kv_lens)
    _same_device(what, q, cache=cache._k_codes, kv_lens=kv_lens, block_mask=block_mask)
    B, nb = cache.batch, cache.num_blocks
    if block_mask is not None and (tuple(block_mask.shape) != (B, nb) or block_mask.dtype != torch.bool):
        raise ValueError(f"{what}: block_mask must be bool [B, num_blocks] = {(B, nb)}, got {block_mask.dtype} {tuple(block_mask.shape)}")
    if kv_lens is not None:
        live = torch.arange(0, nb * cache.block_size, cache.block_size, device=q.device) < kv_lens[:, None]
        block_mask = live if block_mask is None else block_mask & live
    idx = query_topk(q, cache.k_mean, block_count, block_mask)
    out = cache_attn(q, cache, idx, softmax_scale, kv_lens)
    return (out, idx) if return_block_indices else out
