"""Attention over the key/value cache in 8 bits, against the same in float64 on the values the cache holds."""

import ctypes
import math

import pytest
import torch

import mosaic_amd as M
from kv_cache_model import attention
from mosaic_amd import _lib

gpu = pytest.mark.gpu
BF16, F32, I8, E4M3 = torch.bfloat16, torch.float32, torch.int8, torch.float8_e4m3fn


def filled(B, n, H, bs=64, code=I8, seed=0, grow=1.0):
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn(2, B, n, H, 64, generator=g)
    cache = M.KVCache(B, n, H, block_size=bs, dtype=code)
    M.kv_cache_write(cache, (grow * k).cuda(), v.cuda())
    return cache


def queries(B, n, H, seed=1, dtype=BF16):
    return torch.randn(B, n, H, 64, generator=torch.Generator().manual_seed(seed)).to(dtype)


def sets(B, n, H, K, nb, seed=2):
    """Block indices with repeats and entries out of range among them."""
    g = torch.Generator().manual_seed(seed)
    idx = torch.randint(-1, nb + 1, (B, n, H, K), generator=g)
    idx[:, ::7] = -1                       # rows without a block
    return idx


def check(cache, q, idx=None, lens=None, scale=None, values=None):
    got = M.cache_attn(q.cuda(), cache, None if idx is None else idx.cuda(), scale, None if lens is None else lens.cuda())
    assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
    k, v = values or (t.cpu() for t in M.kv_cache_read(cache, dtype=F32))
    want, tol = attention(q.to(BF16), k, v, 0.125 if scale is None else scale, lens, idx, cache.block_size)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), ((err / tol.clamp(min=1e-300)).max().item(), (err > tol).sum().item())
    return got


SHAPES = [  # B, Nq, Nk, Hq, Hk, bs
    (1, 1, 1, 1, 1, 64), (1, 1, 64, 4, 1, 64), (2, 1, 65, 12, 3, 64), (1, 3, 1000, 16, 1, 128), (1, 37, 700, 12, 3, 64), (2, 33, 513, 5, 5, 256),
    (1, 130, 300, 6, 2, 128), (1, 9, 5000, 24, 2, 64), (1, 1, 9000, 20, 5, 256), (3, 300, 129, 8, 1, 64), (1, 2, 20000, 3, 1, 128),
]


@gpu
@pytest.mark.parametrize("code", [I8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("B,Nq,Nk,Hq,Hk,bs", SHAPES)
def test_whole_sequences(code, B, Nq, Nk, Hq, Hk, bs):
    cache = filled(B, Nk, Hk, bs, code, seed=Nk, grow=2.0)
    check(cache, queries(B, Nq, Hq))
    lens = torch.tensor([Nk - Nk // 3, 0, Nk + 5][:B][::-1])
    check(cache, queries(B, Nq, Hq, seed=3), lens=lens, scale=0.3)


@gpu
@pytest.mark.parametrize("code", [I8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("K", [1, 5, 20])
@pytest.mark.parametrize("B,Nq,Nk,Hq,Hk,bs", SHAPES)
def test_blocks_of_each_token(code, K, B, Nq, Nk, Hq, Hk, bs):
    cache = filled(B, Nk, Hk, bs, code, seed=Nk)
    idx = sets(B, Nq, Hk, K, cache.num_blocks)
    check(cache, queries(B, Nq, Hq), idx)
    lens = torch.tensor([Nk - Nk // 3, 0, Nk][:B][::-1]).int()
    check(cache, queries(B, Nq, Hq, seed=3), idx.int(), lens)


@gpu
@pytest.mark.parametrize("grow", [1.0, 20.0], ids=["bounded", "past the bounds"])
@pytest.mark.parametrize("B,Nq,Nk,Hq,Hk,bs,code", [
    (1, 6500, 500, 16, 1, 64, I8), (3, 2100, 700, 16, 1, 128, E4M3), (1, 1000, 3100, 4, 4, 64, E4M3), (2, 400, 2000, 6, 2, 256, I8),
    (1, 1, 40000, 4, 1, 64, I8), (1, 16, 2600, 1, 1, 64, E4M3), (1, 17, 40000, 1, 1, 64, I8),
])
def test_layouts_of_whole_sequences(B, Nq, Nk, Hq, Hk, bs, code, grow):
    """Full rounds of workgroups with the rest in shares, shares alone, many of them; lengths that leave shares empty."""
    cache = filled(B, Nk, Hk, bs, code, seed=Nk + 1, grow=grow)
    q = queries(B, Nq, Hq, 26)
    check(cache, q)
    check(cache, q, lens=torch.tensor([Nk - 70, 0, 65][:B]))
    check(cache, q, lens=torch.tensor([1, Nk, 130][:B]))


@gpu
@pytest.mark.parametrize("code", [I8, E4M3], ids=["int8", "e4m3"])
def test_a_full_round_and_a_rest_in_shares(code):
    """Many tokens over a long sequence; every 61st of them, and the last, against float64."""
    n = 6500
    cache = filled(1, 2000, 1, 64, code, seed=27)
    q = queries(1, n, 16, 28)
    k, v = (t.cpu() for t in M.kv_cache_read(cache, dtype=F32))
    rows = torch.cat([torch.arange(0, n, 61), torch.arange(n - 40, n)])
    for lens in (None, torch.tensor([1801])):
        got = M.cache_attn(q.cuda(), cache, kv_lens=None if lens is None else lens.cuda())[:, rows.cuda()]
        want, tol = attention(q[:, rows], k, v, 0.125, lens, None, 64)
        assert bool(((got.cpu().double() - want).abs() <= tol).all())


@gpu
@pytest.mark.parametrize("lens", [0, 1, 63, 64, 65, 127, 128, 129, 255, 256])
@pytest.mark.parametrize("bs", [64, 128, 256])
def test_lengths_at_the_edges(bs, lens):
    cache = filled(1, 256, 2, bs, seed=4)
    q, n = queries(1, 3, 4), torch.tensor([lens])
    got = check(cache, q, lens=n)
    check(cache, q, sets(1, 3, 2, 3, cache.num_blocks), n)
    if lens == 0:
        assert not got.any()


@gpu
def test_many_tokens_in_their_own_and_in_no_order():
    """More workgroups than are split, and tokens that are taken in another order."""
    cache = filled(1, 64 * 70, 2, 64, E4M3, seed=5)
    for seed, spread in ((6, 2), (7, 70)):
        g = torch.Generator().manual_seed(seed)
        n = 4200
        at = torch.arange(n) * 70 // n if spread == 2 else torch.randint(0, 70, (n,), generator=g)
        idx = (at[:, None, None] + torch.randint(0, spread, (n, 2, 3), generator=g)).clamp(max=69)[None]
        check(cache, queries(1, n, 8, seed), idx)


@gpu
def test_more_blocks_than_a_union_takes_at_once():
    cache = filled(1, 64 * 1500 + 7, 1, 64, seed=8)
    idx = torch.tensor([0, 3, 1023, 1024, 1100, 1500, 1499, 1501]).view(1, 1, 1, 8).expand(1, 5, 1, 8)
    check(cache, queries(1, 5, 2), idx)
    idx = torch.randint(0, 1501, (1, 40, 1, 300), generator=torch.Generator().manual_seed(9))
    check(cache, queries(1, 40, 1), idx)


@gpu
@pytest.mark.parametrize("sparse", [False, True])
def test_queries_of_other_strides_and_types(sparse):
    cache = filled(2, 200, 2, seed=10)
    idx = sets(2, 40, 2, 3, cache.num_blocks) if sparse else None
    q = queries(40, 2, 8).transpose(0, 1)                        # sequence-first
    check(cache, q.contiguous(), idx)
    want = M.cache_attn(q.contiguous().cuda(), cache, None if idx is None else idx.cuda())
    assert torch.equal(M.cache_attn(queries(40, 2, 8).cuda().transpose(0, 1), cache, None if idx is None else idx.cuda()), want)
    odd = torch.empty(2, 40, 8, 67, dtype=BF16, device="cuda")[..., 1:65].copy_(q)
    assert torch.equal(M.cache_attn(odd, cache, None if idx is None else idx.cuda()), want)
    wide = idx if idx is None else torch.cat([idx, idx], -1).cuda()[..., 3:]
    assert torch.equal(M.cache_attn(q.cuda().flip(3).flip(3), cache, wide), want)
    check(cache, queries(2, 40, 8, dtype=F32), idx)


@gpu
@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("nq", [1, 200])
def test_scales_far_apart(sparse, nq):
    """Blocks of values that no one reference of the exponent fits, of keys near nothing, and zeros."""
    n = 64 * 6
    g = torch.Generator().manual_seed(11)
    k, v = torch.randn(2, 1, n, 2, 64, generator=g)
    v[0, :64] *= 2.0 ** -90
    v[0, 64:128] *= 2.0 ** 80
    v[0, 128:192] = 0
    k[0, 192:256] = 0
    k[0, 256:320] *= 2.0 ** -60
    cache = M.KVCache(1, n, 2)
    M.kv_cache_write(cache, k.cuda(), v.cuda())
    idx = torch.tensor([[0, 2], [0, 1], [3, 4], [2, 2], [5, 0], [1, 2]])[torch.arange(nq) % 6].view(1, nq, 1, 2).expand(1, nq, 2, 2) if sparse else None
    check(cache, queries(1, nq, 4), idx)
    if not sparse:
        check(cache, queries(1, nq, 4), lens=torch.tensor([64]))
        check(cache, queries(1, nq, 4), lens=torch.tensor([190]))


@gpu
@pytest.mark.parametrize("nq", [1, 30, 700])
def test_what_a_row_has_not_chosen_does_not_reach_it(nq):
    """Blocks of NaN (a value in them was not finite), among the keys and among the values."""
    n = 64 * 8
    g = torch.Generator().manual_seed(12)
    k, v = torch.randn(2, 1, n, 1, 64, generator=g)
    k[0, 70] = math.nan
    v[0, 200, 0, 3] = math.inf
    cache = M.KVCache(1, n, 1)
    M.kv_cache_write(cache, k.cuda(), v.cuda())
    q = queries(1, nq, 4)
    idx = torch.randint(0, 8, (1, nq, 1, 3), generator=g)
    idx[0, 0] = torch.tensor([0, 2, 4])
    got = M.cache_attn(q.cuda(), cache, idx.cuda()).cpu()
    hit = ((idx == 1) | (idx == 3)).any(-1).expand(1, nq, 4)
    assert got[hit].isnan().all() and got[~hit].isfinite().all()
    kk, vv = (t.cpu() for t in M.kv_cache_read(cache, dtype=F32))
    clean = torch.where(hit[..., :1, None], -1, idx)
    want, tol = attention(q, kk.nan_to_num(), vv.nan_to_num(), 0.125, None, clean)
    assert ((got.double() - want).abs() <= tol)[~hit].all()
    dense = M.cache_attn(q.cuda(), cache, kv_lens=torch.tensor([64]).cuda()).cpu()       # past the length
    want, tol = attention(q, kk.nan_to_num(), vv.nan_to_num(), 0.125, torch.tensor([64]))
    assert ((dense.double() - want).abs() <= tol).all()


@gpu
def test_large_logits_and_infinite_queries():
    cache = filled(1, 300, 1, seed=13, grow=30.0)
    check(cache, queries(1, 5, 2) * 20, scale=1.0)
    q = queries(1, 3, 1)
    q[0, 1, 0, 0] = math.inf
    got = M.cache_attn(q.cuda(), cache).cpu()
    assert got[0, 1].isnan().all() and got[0, [0, 2]].isfinite().all()
    q = queries(1, 3, 1)
    for scale in (1e-30, 1e30):
        got = M.cache_attn(q.cuda(), cache, softmax_scale=scale)
        assert got.isfinite().all()
    # equal weights: each carries its block's scale of values, and so a rounding of its own, which is the bound's second term
    check(cache, q, scale=1e-30)


@gpu
def test_choice_and_attention_together():
    """A state written, grown by a run, and queried: cache_query_attn is its steps, over the blocks that have keys."""
    B, H, bs = 2, 2, 64
    cache = M.KVCache(B, 1000, H, block_size=bs, dtype=E4M3)
    g = torch.Generator().manual_seed(14)
    k, v = torch.randn(2, B, 700, H, 64, generator=g)
    k = (k + torch.randn(B, 11, H, 64, generator=g).repeat_interleave(64, 1)[:, :700]).to(BF16)
    M.kv_cache_write(cache, k[:, :600].cuda(), v[:, :600].to(BF16).cuda())
    start = torch.tensor([600, 450], dtype=torch.int32, device="cuda")
    M.kv_cache_write(cache, k[:, 600:].cuda(), v[:, 600:].to(BF16).cuda(), start)
    lens = start + 100
    q = queries(B, 50, 8, seed=15)
    out, idx = M.cache_query_attn(q.cuda(), cache, 4, kv_lens=lens, return_block_indices=True)
    live = torch.arange(cache.num_blocks)[None] * bs < lens.cpu()[:, None]
    assert bool(live.gather(1, idx.cpu().clamp(min=0).flatten(1)).all())
    assert torch.equal(idx, M.query_topk(q.cuda(), cache.k_mean, 4, live.cuda()))
    assert torch.equal(out, M.cache_attn(q.cuda(), cache, idx, kv_lens=lens))
    check(cache, q, idx.cpu(), lens.cpu())
    mask = torch.ones(B, cache.num_blocks, dtype=torch.bool)
    mask[:, 3:] = False
    out, idx = M.cache_query_attn(q.cuda(), cache, 4, kv_lens=lens, block_mask=mask.cuda(), return_block_indices=True)
    assert int(idx.max()) == 2 and int(idx.min()) == -1
    check(cache, q, idx.cpu(), lens.cpu())
    assert torch.equal(M.cache_query_attn(q.cuda(), cache, 16), M.cache_attn(q.cuda(), cache, torch.arange(16).cuda().expand(B, 50, H, 16)))


@gpu
def test_the_same_bits_each_time_and_on_another_stream():
    cache = filled(2, 3000, 3, 128, E4M3, seed=16)
    q, idx = queries(2, 500, 12).cuda(), sets(2, 500, 3, 6, cache.num_blocks).cuda()
    dense, sparse = M.cache_attn(q, cache), M.cache_attn(q, cache, idx)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        there = [M.cache_attn(q, cache), M.cache_attn(q, cache, idx)]
    here = [M.cache_attn(q, cache), M.cache_attn(q, cache, idx)]
    torch.cuda.synchronize()
    for got in (there, here):
        assert torch.equal(got[0], dense) and torch.equal(got[1], sparse)


@gpu
@pytest.mark.parametrize("code", [I8, E4M3], ids=["int8", "e4m3"])
def test_a_token_s_bits_do_not_depend_on_the_tokens_beside_it(code):
    """In calls that fill the chip: tokens in another order, and beside ones whose scores leave the bounds."""
    n, H = 4200, 2
    cache = filled(1, 64 * 70, H, 64, code, seed=21)
    g = torch.Generator().manual_seed(22)
    idx = torch.randint(0, 70, (1, n, H, 5), generator=g).cuda()
    q = queries(1, n, 8, 23).cuda()
    want = M.cache_attn(q, cache, idx)
    order = torch.randperm(n, generator=g).cuda()
    assert torch.equal(M.cache_attn(q[:, order], cache, idx[:, order]), want[:, order])
    large = torch.rand(n, generator=g).cuda() < 0.1
    got = M.cache_attn(torch.where(large[None, :, None, None], 64 * q, q), cache, idx)
    assert torch.equal(got[:, ~large], want[:, ~large]) and not torch.equal(got[:, large], want[:, large])


@gpu
@pytest.mark.parametrize("nq", [1, 40, 900])
def test_scores_past_the_bounds(nq):
    """Rows whose references move, up and down, from the first block or a later one, and rows at the bound."""
    n = 64 * 12
    g = torch.Generator().manual_seed(24)
    k, v = torch.randn(2, 1, n, 1, 64, generator=g)
    size = torch.tensor([1.0, 1, 8, 1, 30, 1, 1, 60, 1, 2, 1, 100]).repeat_interleave(64)
    k = k * size[None, :, None, None]
    k[0, :, 0, 0] = torch.where(size > 20, -size, k[0, :, 0, 0])
    cache = M.KVCache(1, n, 1)
    M.kv_cache_write(cache, k.cuda(), v.cuda())
    q = queries(1, nq, 4, 25)
    q[0, ::3, :, 0] = 30.0
    q[0, 1::3, :, 0] = -30.0
    check(cache, q, scale=0.5)
    check(cache, q, sets(1, nq, 1, 4, 12), scale=0.5)
    only = torch.tensor([11, 7]).expand(1, nq, 1, 2)     # nothing but scores far below zero, for a third of the rows
    check(cache, q, only, scale=1.0)


@gpu
def test_a_captured_step():
    """A token written and attended to, replayed over changing inputs; every replay against the eager call."""
    B, H, n = 2, 2, 300
    g = torch.Generator().manual_seed(17)
    k, v = (t.to(BF16).cuda() for t in torch.randn(2, B, n + 8, H, 64, generator=g))
    caches = [M.KVCache(B, n + 8, H) for _ in range(2)]
    for c in caches:
        M.kv_cache_write(c, k[:, :n], v[:, :n])
    at = torch.full((B,), n, dtype=torch.int32, device="cuda")
    lens = at + 1
    q, kt, vt = queries(B, 1, 8).cuda(), k[:, n:n + 1].clone(), v[:, n:n + 1].clone()

    def step(c):
        M.kv_cache_write(c, kt, vt, at)
        return M.cache_attn(q, c, kv_lens=lens), M.cache_query_attn(q, c, 3, kv_lens=lens)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    for i in range(6):
        at.fill_(n + i)
        lens.fill_(n + i + 1)
        kt.copy_(k[:, n + i:n + i + 1])
        vt.copy_(v[:, n + i:n + i + 1])
        q.copy_(queries(B, 1, 8, seed=20 + i))
        graph.replay()
        want = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        check(caches[1], q.cpu(), lens=lens.cpu())


# ------------------------------------------------------------------ refusals

def cpu_cache():
    return M.KVCache(2, 100, 3, device="cpu")


Q = torch.zeros(2, 5, 6, 64, dtype=BF16)
IDX = torch.zeros(2, 5, 3, 2, dtype=torch.int64)


@pytest.mark.parametrize("q,kw,error,match", [
    (Q[0], {}, ValueError, "q must be"), (Q.half(), {}, TypeError, "float16"), (Q.double(), {}, TypeError, "float64"), (Q[..., :32], {}, ValueError, "head_dim"),
    (Q[:1], {}, ValueError, "batch"), (Q[:, :, :5], {}, ValueError, "multiple of 3"), (torch.zeros(2, 5, 51, 64), {}, ValueError, "at most 16"),
    (Q, dict(block_indices=IDX[0]), ValueError, "block_indices"), (Q, dict(block_indices=IDX[:, :, :2]), ValueError, "block_indices"),
    (Q, dict(block_indices=IDX.float()), TypeError, "block_indices"), (Q, dict(block_indices=IDX[..., :1].expand(2, 5, 3, 1025)), ValueError, "at most 1024"),
    (Q, dict(kv_lens=torch.zeros(3, dtype=torch.int32)), ValueError, "kv_lens"), (Q, dict(kv_lens=torch.zeros(2)), TypeError, "kv_lens"),
    (Q, dict(softmax_scale=0.0), ValueError, "softmax_scale"), (Q, dict(softmax_scale=math.nan), ValueError, "softmax_scale"),
    (Q.clone().requires_grad_(), {}, RuntimeError, "no backward"), (Q, {}, ValueError, "device"),
])
def test_calls_that_are_refused(q, kw, error, match):
    with pytest.raises(error, match=match):
        M.cache_attn(q, cpu_cache(), **kw)


def test_choices_that_are_refused():
    with pytest.raises(ValueError, match="device"):
        M.cache_query_attn(Q, cpu_cache(), 1)
    with pytest.raises(ValueError, match="batch"):
        M.cache_query_attn(Q[:1], cpu_cache(), 1)
    with pytest.raises(RuntimeError, match="no backward"):
        M.cache_query_attn(Q.clone().requires_grad_(), cpu_cache(), 1)


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="forward mode"):
            M.cache_attn(fwad.make_dual(Q, Q), cpu_cache())


@gpu
def test_calls_without_rows_or_blocks():
    cache = filled(2, 100, 3, seed=18)
    assert M.cache_attn(Q[:, :0].cuda(), cache).shape == (2, 0, 6, 64)
    assert not M.cache_attn(queries(2, 5, 6).cuda(), cache, IDX[..., :0].cuda()).any()


FAKE = 1 << 20


def test_c_entry_refuses_arguments():
    L = _lib.lib()
    c = ctypes.byref(_lib.Cache(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 4, 3, 64, _lib.CODE_INT8, 250))
    rows = _lib.Bnhd(FAKE, 1920, 384, 64)

    def call(q=rows, idx=None, lens=None, n=5, hq=6, d=64, K=0, scale=0.0, out=FAKE, ws=FAKE, nbytes=1 << 40, cache=c):
        return L.mosaic_cache_attn_fwd(q, cache, idx, lens, n, hq, d, K, scale, out, ws, nbytes, None)

    assert call(cache=None) == 1 and call(q=_lib.Bnhd(None, 0, 0, 0)) == 1 and call(out=None) == 1
    assert call(n=0) == 8 and call(hq=0) == 3 and call(hq=7) == 3 and call(d=32) == 2 and call(hq=51) == 11
    assert call(K=-1) == 5 and call(K=3) == 5 and call(idx=FAKE) == 5 and call(idx=FAKE, K=1025) == 11
    assert call(scale=1e-31) == 11 and call(scale=1e31) == 11
    assert call(q=_lib.Bnhd(FAKE + 8, 1920, 384, 64)) == 7 and call(out=FAKE + 4) == 7 and call(idx=FAKE + 4, K=1) == 7 and call(lens=FAKE + 2) == 7
    big = ctypes.byref(_lib.Cache(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 1000, 3, 64, _lib.CODE_INT8, 64000))
    need = L.mosaic_cache_attn_fwd_workspace_size(big, 5, 6, 0)
    assert need > 0 and call(ws=None, cache=big) == 6 and call(nbytes=need - 1, cache=big) == 6 and call(ws=FAKE + 16, cache=big) == 6
    assert L.mosaic_cache_attn_fwd_workspace_size(c, 5, 51, 0) == 0
    many = ctypes.byref(_lib.Cache(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 20, 1, 16, 64, _lib.CODE_INT8, 64))   # 2^24 workgroups of 256 threads
    assert call(n=1, hq=16, cache=many) == 8 and call(n=40, hq=16, cache=many) == 8
