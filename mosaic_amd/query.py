"""Block-sparse attention of query tokens that each choose their own key blocks.

The block-sparse op (``attn_topk`` and ``mosaic_sparse_attn``) chooses key blocks once for a whole
block of queries on the keys' own mesh.  Here every query token has its own blocks, and the queries
need not lie on the mesh: stations, points of another grid, one token.

* ``query_topk(q, k_cmp, block_count, block_mask=None)``: the blocks of the largest scores of each
  query token and kv head against pooled keys.

q is [B, Nq, Hq, 64], keys [B, Nk, Hk, 64], Hq a multiple of Hk with at most 16 query heads per kv
head.  The computation is bf16 with fp32 statistics; fp32 inputs are converted and fp16 is refused,
as in the block-sparse op.  The ops enqueue on the current stream of q's device and never
synchronise the host.
"""

from __future__ import annotations

import torch

from . import _lib
from .ops import stream_of
from .rotary import _bnhd, _rows, _same_device

__all__ = ["query_topk"]


def _bf16_heads(what: str, **tensors) -> None:
    """The checks of [B, N, H, 64] tensors that need no device."""
    for name, t in tensors.items():
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
    Hq, Hk = q.shape[2], k.shape[2]
    if q.shape[0] != k.shape[0]:
        raise ValueError(f"{what}: q {tuple(q.shape)} and keys {tuple(k.shape)} disagree on the batch")
    if Hk == 0 or Hq == 0 or Hq % Hk or Hq // Hk > 16:
        raise ValueError(f"{what}: {Hq} query heads must be a multiple of {Hk} kv heads, at most 16 times as many")


def _as_bf16(t: torch.Tensor) -> torch.Tensor:
    return _rows(t if t.dtype == torch.bfloat16 else t.to(torch.bfloat16))


@torch.no_grad()
def query_topk(q: torch.Tensor, k_cmp: torch.Tensor, block_count: int, block_mask: torch.Tensor | None = None) -> torch.Tensor:
    """The ``block_count`` key blocks of each query token and kv head: int64 [B, Nq, Hk, K].

    q [B, Nq, Hq, 64] against pooled keys ``k_cmp`` [B, nb, Hk, 64] (``pool_mean``, say): the score of
    a block is the sum over the kv head's query heads of their dot products with it, and the largest
    exact scores are taken, ties to the lower block.  Blocks come in ascending order; slots past the
    last are -1, where ``block_mask`` (bool [B, nb], False: never taken) leaves fewer than
    ``block_count``.  ``block_count`` is at most 64.  No gradient passes through the choice.
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
    q, k_cmp = _as_bf16(q), _as_bf16(k_cmp)
    mask = None if block_mask is None else block_mask.contiguous()
    with torch.cuda.device(q.device):
        st = _lib.lib().mosaic_query_topk_fwd(_bnhd(q), _bnhd(k_cmp), None if mask is None else mask.data_ptr(), B, Nq, nb,
                                              Hq, Hk, d, block_count, idx.data_ptr(), stream_of(q))
    _lib.check(st, "mosaic_query_topk_fwd")
    return idx
