"""Block-sparse attention of query tokens that each choose their own key blocks.

The block-sparse op (``attn_topk`` and ``mosaic_sparse_attn``) chooses key blocks once for a whole
block of queries on the keys' own mesh.  Here every query token has its own blocks, and the queries
need not lie on the mesh: stations, points of another grid, one token.

* ``query_topk(q, k_cmp, block_count, block_mask=None)``: the blocks of the largest scores of each
  query token and kv head against pooled keys.
* ``query_sparse_attn(q, k, v, block_indices, block_size, softmax_scale=None, kv_lens=None)``:
  attention of each query token over its blocks, differentiable in q, k and v.
* ``mosaic_query_attn(q, k, v, block_size, block_count, ...)``: both, on keys it pools itself.

q is [B, Nq, Hq, 64], keys [B, Nk, Hk, 64], Hq a multiple of Hk with at most 16 query heads per kv
head.  The computation is bf16 with fp32 statistics; fp32 inputs are converted and fp16 is refused,
as in the block-sparse op.  The ops enqueue on the current stream of q's device and never
synchronise the host.
"""

from __future__ import annotations

import torch

from . import _lib
from .primitives import pool_mean
from .rotary import _like, _on, _ptr, _rows, _same_device, _stream, _wants_grad

__all__ = ["query_topk", "query_sparse_attn", "mosaic_query_attn"]


def _bf16_heads(what: str, **tensors) -> None:
    """The checks of [B, N, H, 64] tensors that need no device."""
    for name, t in tensors.items():
        if t.dtype is torch.bfloat16 and t.dim() == 4 and t.shape[3] == 64:
            continue
        if t.dim() != 4:
            raise ValueError(f"{what}: {name} must be [B, N, H, 64], got shape {tuple(t.shape)}")
        if t.dtype == torch.float16:
            raise TypeError(f"{what}: {name} is float16: these kernels compute in bfloat16 (run the model under "
                            "torch.autocast(..., dtype=torch.bfloat16), or convert the inputs)")
        if t.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"{what}: {name} is {t.dtype}; bfloat16 and float32 are taken")
        if t.shape[3] != 64:
            raise ValueError(f"{what}: head_dim of {name} must be 64, got {t.shape[3]}")


def _groups(what: str, q: torch.Tensor, k: torch.Tensor) -> None:
    (B, _, Hq, _), (Bk, _, Hk, _) = q.shape, k.shape
    if B != Bk:
        raise ValueError(f"{what}: q {tuple(q.shape)} and keys {tuple(k.shape)} disagree on the batch")
    if max(B, q.shape[1], k.shape[1]) >= 1 << 31:   # (views of few elements may be that long)
        raise ValueError(f"{what}: the batch, queries and keys must each be below 2^31, got {tuple(q.shape)}, {tuple(k.shape)}")
    if Hk == 0 or Hq == 0 or Hq % Hk or Hq // Hk > 16:
        raise ValueError(f"{what}: {Hq} query heads must be a multiple of {Hk} kv heads, at most 16 times as many")


def _as_bf16(t: torch.Tensor):
    """bf16 rows as the kernels read them: (tensor, its pointer and strides)."""
    return _rows(t if t.dtype == torch.bfloat16 else t.to(torch.bfloat16))


def _block_size(what: str, block_size) -> int:
    if not 0 < block_size < 1 << 31 or block_size % 64:
        raise ValueError(f"{what}: block_size must be a positive multiple of 64 below 2^31, got {block_size}")
    return int(block_size)


def _scale(what: str, softmax_scale) -> float:
    """The scale as fp32 carries it and its reciprocal, with the logarithms the backward divides by it."""
    scale = 0.125 if softmax_scale is None else float(softmax_scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"{what}: softmax_scale must be within 1e-30 .. 1e30, got {softmax_scale}")
    return scale


def query_topk(q: torch.Tensor, k_cmp: torch.Tensor, block_count: int, block_mask: torch.Tensor | None = None) -> torch.Tensor:
    """The ``block_count`` key blocks of each query token and kv head: int64 [B, Nq, Hk, K].

    q [B, Nq, Hq, 64] against pooled keys ``k_cmp`` [B, nb, Hk, 64] (``pool_mean``, say): the score of
    a block is the sum over the kv head's query heads of their dot products with it, and the largest
    exact scores are taken, whatever their magnitude, ties to the lower block; one that is NaN is not.
    Blocks come in ascending order; slots past the last are -1, where ``block_mask`` (bool [B, nb],
    False: never taken) and NaN leave fewer than ``block_count``.  ``block_count`` is at most 64.  No
    gradient passes through the choice.
    """
    what = "query_topk"
    _bf16_heads(what, q=q, k_cmp=k_cmp)
    _groups(what, q, k_cmp)
    B, Nq, Hq, d = q.shape
    nb, Hk = k_cmp.shape[1:3]
    block_count = int(block_count)
    if not 0 < block_count <= min(nb, 64):
        raise ValueError(f"{what}: block_count must be in [1, {min(nb, 64)}], got {block_count}")
    if block_mask is not None and (tuple(block_mask.shape) != (B, nb) or block_mask.dtype != torch.bool):
        raise ValueError(f"{what}: block_mask must be bool [B, nb] = {(B, nb)}, got {block_mask.dtype} {tuple(block_mask.shape)}")
    _same_device(what, q, k_cmp=k_cmp, block_mask=block_mask)
    idx = torch.empty(B, Nq, Hk, block_count, dtype=torch.int64, device=q.device)
    if idx.numel() == 0:
        return idx
    (q, qb), (k_cmp, kb) = _as_bf16(q.detach()), _as_bf16(k_cmp.detach())
    mask = None if block_mask is None else block_mask.contiguous()
    with _on(q.device):
        st = _lib.lib().mosaic_query_topk_fwd(qb, kb, _ptr(mask), B, Nq, nb, Hq, Hk, d, block_count, idx.data_ptr(), _stream(q.device))
    _lib.check(st, "mosaic_query_topk_fwd")
    return idx


def _scratch(nbytes: int, device: torch.device) -> torch.Tensor | None:
    """Workspace (torch's allocator aligns to 512 bytes; the library checks the 256 it needs)."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _attn_fwd(q, k, v, idx, block_size, scale, lens, want_lse):
    """(output bf16 [B, Nq, Hq, 64], lse fp32 [B, Nq, Hq] or None, workspace or None); q, k, v as (rows, their Bnhd)."""
    (q, qb), (k, kb), (v, vb) = q, k, v
    B, Nq, Hq, d = q.shape
    Nk, Hk = k.shape[1:3]
    K, device = idx.shape[-1], q.device
    out = _like(q)
    lse = torch.empty((B, Nq, Hq), dtype=torch.float32, device=device) if want_lse else None
    L = _lib.lib()
    nbytes = L.mosaic_query_attn_fwd_workspace_size(B, Nq, Hq, Hk, block_size, K)
    ws = _scratch(nbytes, device)
    with _on(device):
        st = L.mosaic_query_attn_fwd(qb, kb, vb, idx.data_ptr(), _ptr(lens), B, Nq, Nk, Hq, Hk, d, block_size, K, scale,
                                     out.data_ptr(), _ptr(lse), _ptr(ws), nbytes, _stream(device))
    _lib.check(st, "mosaic_query_attn_fwd")
    return out, lse, ws


class _QueryAttn(torch.autograd.Function):
    """Saves the bf16 rows the kernels read, the output and its log-sum-exp, and the order of the tokens."""

    @staticmethod
    def forward(ctx, q, k, v, idx, block_size, scale, lens):
        ctx.dtypes = (q.dtype, k.dtype, v.dtype)
        ctx.rest = (block_size, scale)
        rows = [_as_bf16(t) for t in (q, k, v)]
        out, lse, ctx.order = _attn_fwd(*rows, idx, block_size, scale, lens, True)
        ctx.save_for_backward(*(t for t, _ in rows), out, lse, idx, lens)
        return out.to(q.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, go):
        q, k, v, out, lse, idx, lens = ctx.saved_tensors
        block_size, scale = ctx.rest
        B, Nq, Hq, d = q.shape
        Nk, Hk = k.shape[1:3]
        device = q.device
        (q, qb), (k, kb), (v, vb), (go, gb) = (_as_bf16(t) for t in (q, k, v, go))
        gq, gk, gv = _like(q), _like(k), _like(v)
        L = _lib.lib()
        nbytes = L.mosaic_query_attn_bwd_workspace_size(B, Nq, Nk, Hq, Hk, block_size, idx.shape[-1])
        ws = _scratch(nbytes, device)
        with _on(device):
            st = L.mosaic_query_attn_bwd(qb, kb, vb, out.data_ptr(), lse.data_ptr(), gb, idx.data_ptr(), _ptr(lens), B, Nq, Nk,
                                         Hq, Hk, d, block_size, idx.shape[-1], scale, _ptr(ctx.order), gq.data_ptr(),
                                         gk.data_ptr(), gv.data_ptr(), ws.data_ptr(), nbytes, _stream(device))
        _lib.check(st, "mosaic_query_attn_bwd")
        return tuple(g.to(t) for g, t in zip((gq, gk, gv), ctx.dtypes)) + (None,) * 4


def query_sparse_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, block_indices: torch.Tensor, block_size: int,
                      softmax_scale: float | None = None, kv_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each query token over its own key blocks: [B, Nq, Hq, 64] in q's type.

    ``block_indices`` (int64 or int32 [B, Nq, Hk, K], on q's device, K at most 1024) names, for each
    query token and kv head, blocks of ``block_size`` keys (a multiple of 64; the last block of k may
    be short).  It is a set: an index counts once however often it stands there, and one outside the
    blocks (such as -1) not at all.  ``kv_lens`` (integers [B]): keys from ``kv_lens[b]`` on are not
    attended; what they hold does not matter.  A token without a key gets zeros.  ``softmax_scale``
    defaults to 1/8 and lies within 1e-30 .. 1e30.  Differentiable in q, k and v, once, in reverse mode.
    """
    what = "query_sparse_attn"
    _bf16_heads(what, q=q, k=k, v=v)
    _groups(what, q, k)
    if k.shape != v.shape:
        raise ValueError(f"{what}: k and v shapes differ: {tuple(k.shape)} vs {tuple(v.shape)}")
    B, Nq, Hk = q.shape[0], q.shape[1], k.shape[2]
    block_size = _block_size(what, block_size)
    if block_indices.dim() != 4 or tuple(block_indices.shape[:3]) != (B, Nq, Hk) or block_indices.shape[3] > 1024:
        raise ValueError(f"{what}: block_indices {tuple(block_indices.shape)} must be [B, Nq, Hk, K] = {(B, Nq, Hk, '*')}, "
                         "K at most 1024")
    if block_indices.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: block_indices are {block_indices.dtype}, not int64 or int32")
    scale = _scale(what, softmax_scale)
    if kv_lens is not None:
        if tuple(kv_lens.shape) != (B,):
            raise ValueError(f"{what}: kv_lens {tuple(kv_lens.shape)} must be [B] = ({B},)")
        if kv_lens.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"{what}: kv_lens are {kv_lens.dtype}, not int64 or int32")
    _same_device(what, q, k=k, v=v, block_indices=block_indices, kv_lens=kv_lens)
    if kv_lens is not None:   # clamped before the conversion: a far length stays one
        kv_lens = (kv_lens if kv_lens.dtype == torch.int32 else kv_lens.clamp(0, k.shape[1]).to(torch.int32)).contiguous()
    if q.numel() == 0 or k.numel() == 0 or block_indices.numel() == 0:   # no row, or no key for any
        # (a product with nothing, so that gradients of the inputs are zeros)
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device) + 0 * (q[:0].sum() + k[:0].sum() + v[:0].sum()).to(q.dtype)
    idx = block_indices
    if idx.dtype is not torch.int64 or not idx.is_contiguous():
        idx = idx.to(torch.int64).contiguous()
    if _wants_grad(q, k, v):
        return _QueryAttn.apply(q, k, v, idx, block_size, scale, kv_lens)
    out, _, _ = _attn_fwd(_as_bf16(q), _as_bf16(k), _as_bf16(v), idx, block_size, scale, kv_lens, False)
    return out if q.dtype is torch.bfloat16 else out.to(q.dtype)


def mosaic_query_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, block_size: int, block_count: int, *,
                      softmax_scale: float | None = None, block_mask: torch.Tensor | None = None,
                      k_cmp: torch.Tensor | None = None, return_block_indices: bool = False):
    """Each query token chooses ``block_count`` blocks of k and attends to them: [B, Nq, Hq, 64].

    The keys' blocks are pooled by their mean (``pool_mean``), or ``k_cmp`` [B, Nk / block_size, Hk,
    64] holds what a program pooled once for many calls; ``query_topk`` chooses (``block_mask`` bool
    [B, nb]), ``query_sparse_attn`` attends.  Nk must be a multiple of ``block_size``.  Gradients pass
    through the attention, not through the choice.  With ``return_block_indices`` the choice (int64
    [B, Nq, Hk, block_count]) is returned too.
    """
    what = "mosaic_query_attn"
    _bf16_heads(what, q=q, k=k, v=v)
    block_size = _block_size(what, block_size)
    if k.shape[1] % block_size:
        raise ValueError(f"{what}: block_size must be a multiple of 64 that divides {k.shape[1]} keys, got {block_size}")
    nb = k.shape[1] // block_size
    softmax_scale = _scale(what, softmax_scale)
    if k_cmp is None:
        _same_device(what, q, k=k)
        with torch.no_grad():
            k_cmp = pool_mean(k.detach(), block_size)
    elif k_cmp.dim() != 4 or tuple(k_cmp.shape) != (k.shape[0], nb, k.shape[2], 64):
        raise ValueError(f"{what}: k_cmp {tuple(k_cmp.shape)} must be {(k.shape[0], nb, k.shape[2], 64)}")
    idx = query_topk(q.detach(), k_cmp.detach(), block_count, block_mask)
    out = query_sparse_attn(q, k, v, idx, block_size, softmax_scale)
    return (out, idx) if return_block_indices else out
