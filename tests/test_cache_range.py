"""Attention over the cache where scores, queries and scales are far from ordinary, and what writes leave for autograd."""

import ctypes
import math

import pytest
import torch

import mosaic_amd as M
from kv_cache_model import attention
from mosaic_amd import _lib
from test_cache_attn import BF16, E4M3, F32, I8, check, filled, queries, sets

gpu = pytest.mark.gpu
CODES = pytest.mark.parametrize("code", [I8, E4M3], ids=["int8", "e4m3"])
F64 = torch.float64

# nq, tokens, query heads, kv heads, block size, entries of a token (0: whole sequences): few rows of one workgroup a head, of
# shares; many rows whole, in shares, in workgroups of either size; blocks of few rows, in shares, of a chip full of rows
LAYOUTS = [
    (1, 200, 4, 1, 64, 0), (3, 64 * 9, 4, 4, 128, 0), (1, 64 * 61, 16, 1, 64, 0), (40, 64 * 12, 4, 1, 64, 0), (37, 64 * 70 + 9, 12, 3, 64, 0),
    (6500, 500, 16, 1, 64, 0), (3, 64 * 9, 4, 2, 64, 5), (1, 64 * 200, 4, 1, 256, 20), (17, 64 * 40, 4, 2, 64, 16), (4200, 64 * 70, 8, 2, 64, 3),
]


def one_hot(cache, q, scale, idx=None, lens=None):
    """Rows whose largest score is further above the others than fp32 can be off by hold the value of its key.

    A score of fp32: 72 roundings of 2^-24 of sum |q k|, and 2^-22 of |score| (see ``attention``); beyond twice that, in scores
    of 2^20 and more, no other key has a weight.  The value: its output's rounding, 2^-8, and 16 of fp32.
    """
    got = M.cache_attn(q.cuda(), cache, None if idx is None else idx.cuda(), scale, None if lens is None else lens.cuda())
    assert got.isfinite().all()
    got = got.cpu().to(F64)
    k, v = (t.cpu().to(F64) for t in M.kv_cache_read(cache, dtype=F32))
    B, Nq, Hq, _ = q.shape
    Nk, Hk = k.shape[1:3]
    G, bs, nb = Hq // Hk, cache.block_size, cache.num_blocks
    sure = 0
    for b in range(B):
        end = Nk if lens is None else int(lens[b])
        for h in range(Hk):
            ok = (torch.arange(Nk) < end).expand(Nq, Nk)
            if idx is not None:
                i, member = idx[b, :, h], torch.zeros(Nq, nb + 1, dtype=torch.bool)
                member.scatter_(1, torch.where((i < 0) | (i >= nb), nb, i), True)
                ok = ok & member[:, :nb].repeat_interleave(bs, 1)[:, :Nk]
            for g in range(h * G, h * G + G):
                qq = q[b, :, g].to(F64)
                x = (qq @ k[b, :, h].t()).masked_fill(~ok, -math.inf)
                top, at = x.topk(2, dim=-1)
                e = 72 * 2.0 ** -24 * (qq.abs() @ k[b, :, h].abs().t()).masked_fill(~ok, 0.0).amax(-1) + 2.0 ** -22 * top[:, 0].abs()
                rows = ok.any(-1) & (top[:, 0] - top[:, 1] > 2 * e + 200 / scale)
                want = v[b, at[:, 0], h]
                assert bool(((got[b, :, g] - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * want.abs())[rows].all()), (b, h, g)
                assert not got[b, ~ok.any(-1), g].any()
                sure += int(rows.sum())
    assert sure > 0.8 * B * Nq * Hq * (1.0 if idx is None else 0.8)


@gpu
@CODES
@pytest.mark.parametrize("scale", [3e8, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("nq,n,Hq,Hk,bs,K", LAYOUTS)
def test_scores_past_fp32_s_units_choose_one_key(nq, n, Hq, Hk, bs, K, scale, code):
    cache = filled(1, n, Hk, bs, code, seed=nq + n)
    idx = sets(1, nq, Hk, K, cache.num_blocks) if K else None
    if nq == 1 and K:
        idx = idx.clamp(min=0).add(1) % cache.num_blocks
    one_hot(cache, queries(1, nq, Hq, 31), scale, idx)
    if nq < 1000:
        one_hot(cache, queries(1, nq, Hq, 32), scale, idx, torch.tensor([n - n // 4]))


@gpu
@CODES
@pytest.mark.parametrize("scale", [1.0, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("nq,n,Hq,Hk,bs,K", LAYOUTS)
def test_equal_keys_weigh_the_same_in_every_share(nq, n, Hq, Hk, bs, K, scale, code):
    """Values of keys that are all one key: their mean, however many of them a share or a wave has."""
    g = torch.Generator().manual_seed(nq + n)
    k, v = torch.randn(1, 1, Hk, 64, generator=g).expand(1, n, Hk, 64), torch.randn(1, n, Hk, 64, generator=g) + 1
    cache = M.KVCache(1, n, Hk, block_size=bs, dtype=code)
    M.kv_cache_write(cache, k.cuda(), v.cuda())
    idx = sets(1, nq, Hk, K, cache.num_blocks) if K else None
    if nq == 1 and K:
        idx = idx.clamp(min=0).add(1) % cache.num_blocks
    q, values = queries(1, nq, Hq, 33), M.kv_cache_read(cache, dtype=F32)[1].cpu()
    for lens in (n, n - n // 3 - 1):
        lens = torch.tensor([lens])
        got = M.cache_attn(q.cuda(), cache, None if idx is None else idx.cuda(), scale, lens.cuda()).cpu().to(F64)
        # scores of 0 are the same softmax; equal scores are equal in fp32 too, so their errors do not enter
        want, tol = attention(torch.zeros_like(q), torch.zeros(1, n, Hk, 64), values, scale, lens, idx, bs)
        assert bool(((got - want).abs() <= tol).all()), ((got - want).abs() / tol.clamp(min=1e-300)).max().item()


@gpu
@CODES
@pytest.mark.parametrize("size", [2.0 ** -64, 2.0 ** -76, 2.0 ** -90], ids=["2^-64", "2^-76", "2^-90"])
@pytest.mark.parametrize("K", [0, 3])
@pytest.mark.parametrize("nq", [1, 40, 700])
def test_queries_near_nothing_with_large_scales(nq, K, size, code):
    """Scores of hundreds, all of them below zero for half of the rows, from queries whose squares leave fp32."""
    n = 64 * 12
    g = torch.Generator().manual_seed(34)
    k, v = torch.randn(2, 1, n, 1, 64, generator=g)
    k[..., 0] = 30.0
    cache = M.KVCache(1, n, 1, dtype=code)
    M.kv_cache_write(cache, k.cuda(), v.cuda())
    q = queries(1, nq, 4, 35).float()
    q[..., 0] = torch.tensor([-8.0, 8.0, -16.0, -3.0])
    idx = sets(1, nq, 1, K, 12).clamp(min=0) if K else None
    check(cache, (q * size).to(BF16), idx, scale=1.0 / size)


@gpu
@CODES
@pytest.mark.parametrize("large,small,scale", [(1e36, 1e-28, 1e-9), (2e37, 1e-26, 1e-12), (1e33, 1e-29, 1e-30), (3e34, 1e-29, 1e-30), (1e30, 1.0, 1e-30), (1e36, 1e4, 1e-30), (1e25, 1.0, 1e-25)])
@pytest.mark.parametrize("K", [0, 3])
@pytest.mark.parametrize("nq", [1, 40, 700])
def test_queries_whose_products_with_codes_leave_fp32(nq, K, large, small, scale, code):
    """Ordinary scores of large queries with small keys or scales, beside rows of ordinary queries (scores of nothing)."""
    n = 64 * 12
    g = torch.Generator().manual_seed(36)
    k, v = torch.randn(2, 1, n, 1, 64, generator=g)
    cache = M.KVCache(1, n, 1, dtype=code)
    M.kv_cache_write(cache, (k * small).cuda(), v.cuda())
    q = queries(1, nq, 4, 37).float()
    q[:, :, :3] *= large
    q[:, 1::3] = queries(1, nq, 4, 38)[:, 1::3].float()
    check(cache, q.to(BF16), sets(1, nq, 1, K, 12).clamp(min=0) if K else None, scale=scale)


FAKE = 1 << 20


def c_cache(batch, num_blocks, heads, capacity):
    return ctypes.byref(_lib.Cache(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, batch, num_blocks, heads, 64, _lib.CODE_INT8, capacity))


@pytest.mark.parametrize("batch,heads,nq,hq,K", [
    (1, 64, 1 << 23, 64, 4),            # 2^24 workgroups of 256 threads would look for the tokens' order, 2^22 attend
    (1 << 18, 16, 9, 256, 1),           # 2^22 workgroups of 1024 threads would make it, 2^23 of 256 attend
])
def test_launches_of_the_order_that_cannot_be_counted_are_refused(batch, heads, nq, hq, K):
    L, c = _lib.lib(), c_cache(batch, 4, heads, 250)
    assert L.mosaic_cache_attn_fwd_workspace_size(c, nq, hq, K) == 0
    rows = _lib.Bnhd(FAKE, nq * hq * 64, hq * 64, 64)
    assert L.mosaic_cache_attn_fwd(rows, c, FAKE, None, nq, hq, 64, K, 0.0, FAKE, FAKE, 1 << 62, None) == 8


@pytest.mark.parametrize("start", [(1 << 63) - 1, (1 << 63) - 5, 246, -1, -1 << 63])
def test_starts_whose_end_leaves_64_bits_are_refused(start):
    L, c, rows = _lib.lib(), c_cache(2, 4, 3, 250), _lib.Bnhd(FAKE, 960, 192, 64)
    assert L.mosaic_kv_cache_write(c, rows, rows, 1, 64, 5, start, None, None, None) == 8
    assert L.mosaic_kv_cache_read(c, 1, 64, 5, start, None, FAKE, FAKE, None) == 8


def held(cache):
    return [cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale, cache.k_norm, cache.k_mean]


@gpu
def test_writes_are_seen_by_autograd():
    cache = filled(1, 200, 2, seed=39)
    w = torch.ones(64, dtype=BF16, device="cuda", requires_grad=True)
    versions = [t._version for t in held(cache)]
    y = (w * cache.k_mean).sum()
    M.kv_cache_read(cache)
    M.cache_query_attn(queries(1, 3, 2).cuda(), cache, 2)
    none = torch.zeros(1, 0, 2, 64, dtype=BF16, device="cuda")
    M.kv_cache_write(cache, none, none)
    assert [t._version for t in held(cache)] == versions
    y.backward()                                        # nothing was written
    y = (w * cache.k_mean).sum()
    one = torch.ones(1, 1, 2, 64, dtype=BF16, device="cuda")
    M.kv_cache_write(cache, one, one, 70)
    assert all(t._version > x for t, x in zip(held(cache), versions))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@gpu
def test_writes_in_inference_mode():
    with torch.inference_mode():
        cache = filled(1, 100, 1, seed=40)
        k, _ = M.kv_cache_read(cache)
        M.kv_cache_write(cache, k[:, :64] * 2, k[:, :64], 0)
    one = torch.ones(1, 1, 1, 64, dtype=BF16, device="cuda")
    M.kv_cache_write(cache, one, one, 64)
    assert torch.equal(M.kv_cache_read(cache, 64, 1)[0], one)


@gpu
def test_a_choice_takes_the_means_of_all_that_is_written():
    """Lengths below what is written: the attention leaves the later tokens out, the last block's mean does not, until it is cut."""
    g = torch.Generator().manual_seed(41)
    k, v = torch.randn(2, 1, 192, 1, 64, generator=g)
    k[0, 70:128] += 4.0                                     # past the length, in the block that it ends in
    k[0, 128:] += 8.0                                       # a block past the length
    cache = M.KVCache(1, 192, 1)
    M.kv_cache_write(cache, k.cuda(), v.cuda())
    q, lens = torch.ones(1, 2, 1, 64, dtype=BF16).cuda(), torch.tensor([70]).cuda()
    out, idx = M.cache_query_attn(q, cache, 1, kv_lens=lens, return_block_indices=True)
    assert torch.equal(idx, M.query_topk(q, cache.k_mean, 1, torch.tensor([[True, True, False]]).cuda())) and bool((idx == 1).all())
    check(cache, q.cpu(), idx.cpu(), lens.cpu())            # ... over tokens 64 .. 69
    k[0, :64] += 0.5
    k[0, 64:70] -= 4.0
    M.kv_cache_write(cache, k[:, :64].cuda(), v[:, :64].cuda())
    M.kv_cache_write(cache, k[:, 64:70].cuda(), v[:, 64:70].cuda(), 64)      # the sequence ends there
    out, idx = M.cache_query_attn(q, cache, 1, kv_lens=lens, return_block_indices=True)
    assert bool((idx == 0).all())
    assert torch.equal(out, M.cache_attn(q, cache, idx, kv_lens=lens))


def test_a_cache_in_host_memory_is_named_by_the_refusal():
    cache, x = M.KVCache(1, 64, 1, device="cpu"), torch.zeros(1, 1, 1, 64)
    with pytest.raises(ValueError, match="kv_cache_write: the cache must be on a ROCm device, got cpu"):
        M.kv_cache_write(cache, x, x)
    with pytest.raises(ValueError, match="kv_cache_read: the cache must be on a ROCm device, got cpu"):
        M.kv_cache_read(cache)


@gpu
def test_tensors_elsewhere_are_named_by_the_refusal():
    cache, x = M.KVCache(2, 64, 1), torch.zeros(2, 1, 1, 64)
    with pytest.raises(ValueError, match="kv_cache_write: k is on cpu, the cache on cuda"):
        M.kv_cache_write(cache, x, x.cuda())
    with pytest.raises(ValueError, match="kv_cache_write: counts is on cpu, the cache on cuda"):
        M.kv_cache_write(cache, x.cuda(), x.cuda(), counts=torch.tensor([1, 1]))
    with pytest.raises(ValueError, match="kv_cache_read: start is on cpu, the cache on cuda"):
        M.kv_cache_read(cache, torch.tensor([1, 1]), 1)
