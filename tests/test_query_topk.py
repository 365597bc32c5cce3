"""query_topk: refusals (CPU) and the selection against float64 scores (GPU).

The selection is exact, so every test asks for equal indices.  The scores of the oracle are float64
sums of products of bf16 values (exact up to 2^-53), and the inputs are such that no two of a row's
scores differ by less than that unless they are equal.
"""

import os

import pytest
import torch

import mosaic_amd as M
from mosaic_amd import _lib

gpu = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call,error,match", [
    (lambda: M.query_topk(z(5, 4, 64), z(1, 9, 1, 64), 2), ValueError, "B, N, H, 64"),
    (lambda: M.query_topk(z(1, 5, 4, 64, dtype=torch.float16), z(1, 9, 1, 64), 2), TypeError, "bfloat16"),
    (lambda: M.query_topk(z(1, 5, 4, 64), z(1, 9, 1, 64, dtype=torch.float64), 2), TypeError, "float64"),
    (lambda: M.query_topk(z(1, 5, 4, 32), z(1, 9, 1, 32), 2), ValueError, "64"),
    (lambda: M.query_topk(z(2, 5, 4, 64), z(1, 9, 1, 64), 2), ValueError, "batch"),
    (lambda: M.query_topk(z(1, 5, 4, 64), z(1, 9, 3, 64), 2), ValueError, "multiple"),
    (lambda: M.query_topk(z(1, 5, 17, 64), z(1, 9, 1, 64), 2), ValueError, "16 times"),
    (lambda: M.query_topk(z(1, 5, 4, 64), z(1, 9, 1, 64), 0), ValueError, "block_count"),
    (lambda: M.query_topk(z(1, 5, 4, 64), z(1, 9, 1, 64), 10), ValueError, "block_count"),
    (lambda: M.query_topk(z(1, 5, 4, 64), z(1, 99, 1, 64), 65), ValueError, "block_count"),
    (lambda: M.query_topk(z(1, 5, 4, 64), z(1, 9, 1, 64), 2, torch.ones(1, 8, dtype=torch.bool)), ValueError, "block_mask"),
    (lambda: M.query_topk(z(1, 5, 4, 64), z(1, 9, 1, 64), 2, torch.ones(1, 9)), ValueError, "block_mask"),
    (lambda: M.query_topk(z(1, 5, 4, 64), z(1, 9, 1, 64), 2), ValueError, "ROCm"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


FAKE = 1 << 20


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libmosaic_bsa.so not built")
@pytest.mark.parametrize("change,status", [
    (dict(batch=0), 8), (dict(nq=0), 8), (dict(nb=0), 8), (dict(d=32), 2), (dict(hq=5), 3), (dict(hq=34), 11),
    (dict(K=0), 5), (dict(K=10), 5), (dict(nb=100, K=65), 11), (dict(q=_lib.Bnhd(None, 0, 0, 0)), 1), (dict(out=None), 1),
    (dict(q=_lib.Bnhd(FAKE + 2, 0, 0, 0)), 7), (dict(k=_lib.Bnhd(FAKE, 0, 4, 0)), 7), (dict(out=FAKE + 4), 7),
    (dict(nq=0x7fffffff, batch=0x7fff), 8),
])
def test_abi_validation(change, status):
    c = dict(q=_lib.Bnhd(FAKE, 0, 256, 64), k=_lib.Bnhd(FAKE, 0, 128, 64), batch=1, nq=7, nb=9, hq=4, hk=2, d=64, K=3, out=FAKE)
    c.update(change)
    assert _lib.lib().mosaic_query_topk_fwd(c["q"], c["k"], None, c["batch"], c["nq"], c["nb"], c["hq"], c["hk"], c["d"],
                                            c["K"], c["out"], None) == status


# ------------------------------------------------------------------------------- GPU

def oracle(q, kc, K, mask=None):
    B, Nq, Hq, _ = q.shape
    nb, Hk = kc.shape[1:3]
    qs = q.to(BF16).double().view(B, Nq, Hk, Hq // Hk, 64).sum(3).permute(0, 2, 1, 3).contiguous()
    s = torch.matmul(qs, kc.to(BF16).double().permute(0, 2, 3, 1).contiguous()).cpu()
    ok = torch.ones(B, nb, dtype=torch.bool) if mask is None else mask.cpu()
    ok = ok[:, None, None, :].expand_as(s)
    order = torch.where(ok, s, -torch.inf).sort(dim=-1, descending=True, stable=True).indices[..., :K]
    order = torch.where(ok.gather(-1, order), order, nb).sort(-1).values
    return torch.where(order == nb, -1, order).permute(0, 2, 1, 3).to(q.device)


def randn(gen, *shape, dtype=BF16):
    return torch.randn(*shape, generator=gen, device=DEV).to(dtype)


@gpu
@pytest.mark.parametrize("B,Nq,nb,Hq,Hk,K", [
    (1, 1, 1, 1, 1, 1), (1, 1, 768, 12, 3, 16), (2, 17, 63, 4, 2, 5), (1, 37, 65, 3, 1, 64), (3, 16, 257, 16, 1, 24),
    (1, 1000, 513, 5, 5, 7), (2, 33, 769, 6, 2, 33), (1, 50, 1025, 8, 4, 16), (1, 19, 2500, 4, 1, 64), (1, 5000, 96, 16, 4, 12),
    (1, 3, 64, 7, 7, 64),
])
def test_selection(B, Nq, nb, Hq, Hk, K):
    gen = torch.Generator(device=DEV).manual_seed(nb + K)
    q, kc = randn(gen, B, Nq, Hq, 64), randn(gen, B, nb, Hk, 64)
    assert torch.equal(M.query_topk(q, kc, K), oracle(q, kc, K))
    mask = torch.rand(B, nb, generator=gen, device=DEV) < 0.3
    mask[0] = False                                   # a sequence with nothing to read
    got = M.query_topk(q, kc, K, mask)
    assert torch.equal(got, oracle(q, kc, K, mask))
    assert bool((got[0] == -1).all())


@gpu
@pytest.mark.parametrize("nb", [40, 300, 1200])
def test_ties_go_to_the_lowest_block(nb):
    gen = torch.Generator(device=DEV).manual_seed(nb)
    # small integers: most scores are equal to others, exactly
    q = torch.randint(-1, 2, (1, 60, 4, 64), generator=gen, device=DEV).to(BF16)
    kc = torch.randint(-1, 2, (1, nb, 2, 64), generator=gen, device=DEV).to(BF16)
    q[:, 5] = 0                                       # every score zero
    kc[:, nb // 2:] = kc[:, :nb - nb // 2].clone()    # every block twice
    for K in (1, 16, 33):
        assert torch.equal(M.query_topk(q, kc, K), oracle(q, kc, K))
    same = kc[:, :1].expand(1, nb, 2, 64)             # one key, broadcast over the blocks
    assert torch.equal(M.query_topk(q, same, 16), torch.arange(16, device=DEV).expand(1, 60, 2, 16))


@gpu
def test_scores_closer_than_fp32_tells():
    # keys that are one key but for a step of bf16 in one dimension: the scores differ by little beside
    # their common offset of hundreds, which is what 256 roundings in fp32 are measured by
    gen = torch.Generator(device=DEV).manual_seed(4)
    nb, Nq = 700, 64
    q = randn(gen, 1, Nq, 4, 64)
    kc = randn(gen, 1, 1, 1, 64).float().mul(64).expand(1, nb, 1, 64).clone()
    at = torch.randint(0, 64, (nb,), generator=gen, device=DEV)
    kc[0, torch.arange(nb, device=DEV), 0, at] *= 1 + 2.0 ** -7 * (torch.arange(nb, device=DEV) % 3 - 1)
    kc = kc.to(BF16)
    assert torch.equal(M.query_topk(q, kc, 16), oracle(q, kc, 16))


@gpu
def test_masked_blocks_hold_nan_and_infinities():
    gen = torch.Generator(device=DEV).manual_seed(6)
    q, kc = randn(gen, 1, 40, 4, 64), randn(gen, 1, 130, 1, 64)
    mask = torch.rand(1, 130, generator=gen, device=DEV) < 0.5
    want = oracle(q, kc, 16, mask)
    bad = kc.clone()
    bad[~mask] = float("nan")
    bad[:, (~mask[0]).nonzero()[:3, 0]] = float("inf")
    assert torch.equal(M.query_topk(q, bad, 16, mask), want)


@gpu
def test_layouts_and_types():
    gen = torch.Generator(device=DEV).manual_seed(8)
    q, kc = randn(gen, 2, 50, 8, 64), randn(gen, 2, 90, 2, 64)
    want = oracle(q, kc, 9)
    assert torch.equal(M.query_topk(q.transpose(0, 1).contiguous().transpose(0, 1), kc, 9), want)          # sequence-first
    wide = torch.randn(2, 50, 11, 64, generator=gen, device=DEV).to(BF16)
    wide[:, :, 2:10] = q
    assert torch.equal(M.query_topk(wide[:, :, 2:10], kc, 9), want)
    odd = torch.zeros(2, 50, 8, 65, device=DEV, dtype=BF16)
    odd[..., 1:] = q
    assert torch.equal(M.query_topk(odd[..., 1:], kc, 9), want)                                            # unaligned rows
    assert torch.equal(M.query_topk(q.float(), kc.float(), 9), want)
    assert M.query_topk(q[:, :0], kc, 9).shape == (2, 0, 2, 9)


@gpu
def test_captured_and_on_another_stream():
    gen = torch.Generator(device=DEV).manual_seed(10)
    q, kc = randn(gen, 1, 300, 4, 64), randn(gen, 1, 200, 1, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(M.query_topk(q, kc, 8), oracle(q, kc, 8))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        idx = M.query_topk(q, kc, 8)
    for _ in range(3):
        q.copy_(randn(gen, 1, 300, 4, 64))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(idx, oracle(q, kc, 8))


@gpu
@pytest.mark.parametrize("B,Nq,nb,Hq,Hk,K,masked", [
    (1, 20011, 700, 4, 1, 16, True),        # forty row tiles a workgroup, the last one short
    (40, 49, 130, 4, 2, 9, False),          # more kv heads than a round of workgroups has for one
    (3, 2500, 1000, 6, 3, 5, True),         # two chunks for each of several row tiles
    (1, 3000, 768, 12, 2, 40, False),       # more than four query heads, more blocks than half the lanes
])
def test_several_row_tiles_a_workgroup(B, Nq, nb, Hq, Hk, K, masked):
    gen = torch.Generator(device=DEV).manual_seed(Nq)
    q, kc = randn(gen, B, Nq, Hq, 64), randn(gen, B, nb, Hk, 64)
    mask = torch.rand(B, nb, generator=gen, device=DEV) < 0.5 if masked else None
    assert torch.equal(M.query_topk(q, kc, K, mask), oracle(q, kc, K, mask))


def choice(q, kc, K, mask=None):
    """The oracle where scores may lie anywhere: the first K of the unmasked blocks by their scores in
    float64, a NaN never; products one by one, so that an infinity meets no other row's."""
    B, Nq, Hq, _ = q.shape
    nb, Hk = kc.shape[1:3]
    qs, k = q.cpu().double().view(B, Nq, Hk, Hq // Hk, 64).sum(3), kc.cpu().double()
    s = torch.stack([(qs[:, n, None] * k).sum(-1).transpose(1, 2) for n in range(Nq)], 1)       # [B, Nq, Hk, nb]
    ok = ~s.isnan() if mask is None else ~s.isnan() & mask.cpu()[:, None, None, :]
    # (those that may not be taken behind the -inf of those that may)
    order = torch.where(s.isnan(), 0.0, s).sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, (~ok.gather(-1, order)).to(torch.int8).sort(dim=-1, stable=True).indices)[..., :K]
    order = torch.where(ok.gather(-1, order), order, nb).sort(-1).values
    return torch.where(order == nb, -1, order).to(q.device)


@gpu
@pytest.mark.parametrize("nb,K", [(60, 9), (700, 16), (700, 40), (1200, 16)])
@pytest.mark.parametrize("scale_q,scale_k", [(70, 0), (0, 70), (70, 70), (120, -100), (-80, 0), (0, -80), (-70, -70), (-126, 0)])
def test_scores_whose_norms_leave_fp32(nb, K, scale_q, scale_k):
    # keys that are one key but for a small part in a dimension of theirs: scores of hundreds that are
    # closer than fp32 holds them, times powers of two, which change no order
    print(f"scales 2^{scale_q} 2^{scale_k} nb {nb} K {K}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(14)
    q = randn(gen, 1, 33, 4, 64)
    kc = randn(gen, 1, 1, 1, 64).float().mul(64).expand(1, nb, 1, 64).clone()
    kc[..., 40:] = 0
    at = torch.randint(40, 64, (nb,), generator=gen, device=DEV)
    kc[0, torch.arange(nb, device=DEV), 0, at] = torch.randn(nb, generator=gen, device=DEV) * 2.0 ** -12
    kc = kc.to(BF16)
    q, kc = (q.double() * 2.0 ** scale_q).to(BF16), (kc.double() * 2.0 ** scale_k).to(BF16)
    assert torch.equal(M.query_topk(q, kc, K), choice(q, kc, K))
    mask = torch.rand(1, nb, generator=gen, device=DEV) < 0.5
    assert torch.equal(M.query_topk(q, kc, K, mask), choice(q, kc, K, mask))


@gpu
@pytest.mark.parametrize("Hq,Hk,nb,K", [(2, 2, 40, 1), (2, 2, 40, 40), (8, 2, 300, 16), (3, 1, 300, 33), (4, 1, 1200, 16), (2, 2, 1200, 64)])
def test_keys_and_queries_that_are_not_finite(Hq, Hk, nb, K):
    print(f"not finite {Hq}/{Hk} nb {nb} K {K}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(nb + K)
    q, kc = randn(gen, 2, 20, Hq, 64), randn(gen, 2, nb, Hk, 64)
    inf = float("inf")
    kc[0, nb // 2, 0, 5], kc[0, nb - 1, 0, 6], kc[0, 3, 0, 7] = inf, -inf, float("nan")
    kc[1, 7] = -inf                       # every product of a sign of its own: NaN, or where q is one-signed an infinity
    q[1, 11] = q[1, 11].abs()
    q[:, 4] = 0                           # scores of zero, and NaN beside the infinities
    q[:, 9, :, 3] = inf
    q[:, 13, :, 20] = float("nan")
    assert torch.equal(M.query_topk(q, kc, K), choice(q, kc, K))
    mask = torch.rand(2, nb, generator=gen, device=DEV) < 0.6
    assert torch.equal(M.query_topk(q, kc, K, mask), choice(q, kc, K, mask))
