"""query_sparse_attn and mosaic_query_attn: refusals (CPU) and values against float64 (GPU).

Tolerances, fixed before the first run.  h = 2^-8, half a step of bf16 at most, relative:
* output: each p is off by h of itself (its rounding; l sums the unrounded ones) and by the exponent
  of an fp32 score (64 products: 64 u |q||k| c, u = 2^-24, below h / 16 for the scores here), so
  |o - exact| <= 1.25 h sum p |v| + h |o|;
* grad v = sum P do: 1.25 h sum P |do| + h |dv|;
* delta = sum o do of the rounded o: off by (1.25 h sum p |v| + h |o|) |do| =: e, per row;
* dS = P (dP - delta) is off by 1.25 h |dS| + P e; grad q and grad k are sums of it with |k| or
  |q| and the scale, and h of the result.
"""

import os

import pytest
import torch

import mosaic_amd as M
from mosaic_amd import _lib

gpu = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
H = 2.0 ** -8


def z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


Q, KV = (1, 5, 4, 64), (1, 130, 2, 64)
IDX = torch.zeros(1, 5, 2, 3, dtype=torch.int64)


@pytest.mark.parametrize("call,error,match", [
    (lambda: M.query_sparse_attn(z(5, 4, 64), z(*KV), z(*KV), IDX, 64), ValueError, "B, N, H, 64"),
    (lambda: M.query_sparse_attn(z(*Q, dtype=torch.float16), z(*KV), z(*KV), IDX, 64), TypeError, "bfloat16"),
    (lambda: M.query_sparse_attn(z(*Q), z(*KV), z(1, 131, 2, 64), IDX, 64), ValueError, "differ"),
    (lambda: M.query_sparse_attn(z(*Q), z(1, 130, 3, 64), z(1, 130, 3, 64), IDX, 64), ValueError, "multiple"),
    (lambda: M.query_sparse_attn(z(2, 5, 4, 64), z(*KV), z(*KV), IDX, 64), ValueError, "batch"),
    (lambda: M.query_sparse_attn(z(*Q), z(*KV), z(*KV), IDX, 96), ValueError, "block_size"),
    (lambda: M.query_sparse_attn(z(*Q), z(*KV), z(*KV), IDX, 0), ValueError, "block_size"),
    (lambda: M.query_sparse_attn(z(*Q), z(*KV), z(*KV), IDX[:, :4], 64), ValueError, "block_indices"),
    (lambda: M.query_sparse_attn(z(*Q), z(*KV), z(*KV), torch.zeros(1, 5, 2, 1025, dtype=torch.int64), 64), ValueError, "1024"),
    (lambda: M.query_sparse_attn(z(*Q), z(*KV), z(*KV), IDX.float(), 64), TypeError, "block_indices"),
    (lambda: M.query_sparse_attn(z(*Q), z(*KV), z(*KV), IDX, 64, softmax_scale=0.0), ValueError, "softmax_scale"),
    (lambda: M.query_sparse_attn(z(*Q), z(*KV), z(*KV), IDX, 64, kv_lens=torch.zeros(2, dtype=torch.int32)), ValueError, "kv_lens"),
    (lambda: M.query_sparse_attn(z(*Q), z(*KV), z(*KV), IDX, 64, kv_lens=torch.zeros(1)), TypeError, "kv_lens"),
    (lambda: M.query_sparse_attn(z(*Q), z(*KV), z(*KV), IDX, 64), ValueError, "ROCm"),
    (lambda: M.mosaic_query_attn(z(*Q), z(*KV), z(*KV), 64, 2), ValueError, "divides"),
    (lambda: M.mosaic_query_attn(z(*Q), z(1, 128, 2, 64), z(1, 128, 2, 64), 64, 2, k_cmp=z(1, 3, 2, 64)), ValueError, "k_cmp"),
    (lambda: M.mosaic_query_attn(z(*Q), z(1, 128, 2, 64), z(1, 128, 2, 64), 64, 2), ValueError, "ROCm"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


FAKE = 1 << 20
HAVE_LIB = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libmosaic_bsa.so not built")


def _call(fn, c):
    L = _lib.lib()
    if fn == "fwd":
        return L.mosaic_query_attn_fwd(c["q"], c["k"], c["k"], c["idx"], None, c["B"], c["nq"], c["nk"], c["hq"], c["hk"], c["d"],
                                       c["bs"], c["K"], 0.125, c["out"], c["lse"], c["ws"], c["n"], None)
    return L.mosaic_query_attn_bwd(c["q"], c["k"], c["k"], FAKE, c["lse"], c["q"], c["idx"], None, c["B"], c["nq"], c["nk"],
                                   c["hq"], c["hk"], c["d"], c["bs"], c["K"], 0.125, c.get("order"), c["out"], FAKE, FAKE, c["ws"], c["n"],
                                   None)


@HAVE_LIB
@pytest.mark.parametrize("fn", ["fwd", "bwd"])
@pytest.mark.parametrize("change,status", [
    (dict(B=0), 8), (dict(nq=0), 8), (dict(nk=0), 8), (dict(d=32), 2), (dict(hq=5), 3), (dict(hq=34), 11), (dict(bs=32), 4),
    (dict(K=0), 5), (dict(K=1025), 11), (dict(q=_lib.Bnhd(None, 0, 0, 0)), 1), (dict(k=_lib.Bnhd(FAKE, 0, 4, 0)), 7),
    (dict(idx=None), 1), (dict(idx=FAKE + 4), 7), (dict(out=None), 1), (dict(out=FAKE + 8), 7), (dict(lse=FAKE + 2), 7),
    (dict(ws=None), 6), (dict(ws=FAKE + 16), 6), (dict(n=64), 6), (dict(nk=0x7fffffff), 8), (dict(nq=0x7fffffff), 8),
    (dict(nq=1 << 30, B=1 << 10), 8),
])
def test_abi_validation(fn, change, status):
    c = dict(q=_lib.Bnhd(FAKE, 0, 256, 64), k=_lib.Bnhd(FAKE, 0, 128, 64), idx=FAKE, B=1, nq=7, nk=200, hq=4, hk=2, d=64, bs=64,
             K=12, out=FAKE, lse=FAKE, ws=FAKE, n=1 << 40)
    c.update(change)
    assert _call(fn, c) == status


@HAVE_LIB
def test_workspace_sizes():
    L = _lib.lib()
    # many tokens: their order alone (2 + 4 bytes each and kv head); few entries of few keys: nothing
    size = L.mosaic_query_attn_fwd_workspace_size
    assert 6 * 3 * 49152 <= size(1, 49152, 12, 3, 64, 16) < 7 * 3 * 49152
    assert size(1, 1, 12, 3, 64, 16) == size(1, 1, 12, 3, 64, 32) == 0
    one = size(1, 1, 12, 3, 64, 33)
    assert one >= 32 * 12 * (64 * 4 + 8) and one % 256 == 0
    assert size(1, 1, 12, 3, 128, 17) > 0
    assert size(1, 1, 12, 5, 64, 16) == size(1, 1, 12, 3, 96, 16) == 0       # refused shapes
    assert L.mosaic_query_attn_bwd_workspace_size(1, 100, 1000, 12, 3, 64, 5) >= 2 * 4 * 1200 + 3 * 16 * 16 * 4


# ------------------------------------------------------------------------------- GPU

def oracle(q, k, v, idx, bs, scale=0.125, lens=None, go=None):
    """float64 values and what their terms add up to: dict of (value, bound)."""
    B, Nq, Hq, _ = q.shape
    Nk, Hk = k.shape[1:3]
    G, nb = Hq // Hk, -(-Nk // bs)
    q64, k64, v64 = (t.detach().to(BF16).double() for t in (q, k, v))
    inside = (idx >= 0) & (idx < nb)
    member = torch.zeros(B, Nq, Hk, nb + 1, dtype=torch.bool, device=q.device)
    member.scatter_(-1, torch.where(inside, idx, nb), True)
    ok = member[..., :nb].repeat_interleave(bs, dim=-1)[..., :Nk]
    if lens is not None:
        ok = ok & (torch.arange(Nk, device=q.device) < lens.view(B, 1, 1, 1))
    ok = ok.permute(0, 2, 1, 3).repeat_interleave(G, dim=1)                         # [B, Hq, Nq, Nk]
    kh, vh = (t.permute(0, 2, 1, 3).repeat_interleave(G, dim=1) for t in (k64, v64))
    used = ok.any(2).unsqueeze(-1)
    kh, vh = torch.where(used, kh, 0.0), torch.where(used, vh, 0.0)                 # what nobody chose does not matter
    qh = q64.permute(0, 2, 1, 3)
    s = (qh @ kh.transpose(-1, -2).contiguous() * scale).masked_fill(~ok, -torch.inf)
    p = torch.where(ok.any(-1, keepdim=True), torch.softmax(s, dim=-1), 0.0)
    back = lambda x: x.permute(0, 2, 1, 3)                                          # noqa: E731
    o = p @ vh
    ob = 1.25 * H * (p @ vh.abs()) + H * o.abs()
    out = {"o": (back(o), back(ob))}
    if go is not None:
        g = go.detach().to(BF16).double().permute(0, 2, 1, 3)
        shared = lambda x: x.view(B, Hk, G, Nk, 64).sum(2).permute(0, 2, 1, 3)      # noqa: E731
        e = (ob * g.abs()).sum(-1, keepdim=True)
        ds = p * (g @ vh.transpose(-1, -2).contiguous() - (o * g).sum(-1, keepdim=True))
        dsb = 1.25 * H * ds.abs() + p * e
        dq, dqb = scale * ds @ kh, scale * dsb @ kh.abs()
        dst, dsbt, pt = (x.transpose(-1, -2).contiguous() for x in (ds, dsb, p))
        dk, dkb = scale * shared(dst @ qh), scale * shared(dsbt @ qh.abs())
        dv, dvb = shared(pt @ g), 1.25 * H * shared(pt @ g.abs())
        out |= {"dq": (back(dq), back(dqb) + H * back(dq).abs()), "dk": (dk, dkb + H * dk.abs()), "dv": (dv, dvb + H * dv.abs())}
    return out


def near(got, want, what):
    value, bound = want
    over = (got.double() - value).abs() - bound - 1e-30
    assert bool((over <= 0).all()), f"{what}: {over.max().item():.3g} over its bound"


def randn(gen, *shape, dtype=BF16):
    return torch.randn(*shape, generator=gen, device=DEV).to(dtype)


def choose(gen, B, Nq, Hk, nb, K, how):
    """Block indices: neighbours alike ('near'), anywhere ('far'), or with repeats, -1 and out of range ('ragged')."""
    if how == "near":
        centre = (torch.arange(Nq, device=DEV) * nb // max(Nq, 1)).view(1, Nq, 1, 1)
        return ((centre + torch.arange(K, device=DEV) * 3 + torch.randint(0, 2, (B, Nq, Hk, K), generator=gen, device=DEV)) % nb)
    idx = torch.rand(B, Nq, Hk, nb, generator=gen, device=DEV).argsort(-1)[..., :K]
    if how == "ragged":
        idx = torch.where(torch.rand(idx.shape, generator=gen, device=DEV) < 0.4, -1, idx)
        idx[..., -1] = idx[..., 0]
        idx[:, ::5] = -1
        idx[:, 1::5, :, 0] = nb + 3
        idx[:, 2::5, :, 0] = 1 << 40
        idx[:, 3::5, :, 0] = -(1 << 40)
    return idx


CASES = [
    # B, Nq, Nk, Hq, Hk, bs, K, how, lens
    (1, 1, 1, 1, 1, 64, 1, "far", None),
    (1, 1, 1000, 12, 3, 64, 9, "far", None),
    (2, 1, 4096, 4, 4, 128, 16, "near", None),
    (1, 17, 130, 4, 2, 64, 3, "ragged", None),
    (2, 70, 777, 3, 1, 64, 5, "ragged", (777, 0)),
    (3, 33, 500, 16, 1, 128, 4, "far", (1, 129, 500)),
    (1, 130, 640, 5, 5, 64, 10, "near", None),
    (1, 41, 900, 10, 2, 192, 5, "ragged", (833,)),
    (1, 100, 320, 7, 1, 64, 2, "far", (100000,)),
    (2, 90, 1500, 8, 1, 64, 12, "near", (1500, 700)),
    (1, 29, 600, 18, 2, 64, 3, "far", None),
    (1, 20, 66000, 4, 1, 64, 40, "far", (65999,)),
    (1, 700, 1290, 4, 1, 64, 6, "near", (1281,)),
    (1, 2100, 700, 2, 1, 64, 4, "ragged", None),
]


@gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "b{}q{}k{}h{}-{}bs{}K{}{}".format(*c[:8]))
def test_values_and_gradients(case):
    B, Nq, Nk, Hq, Hk, bs, K, how, lens = case
    gen = torch.Generator(device=DEV).manual_seed(Nq + Nk)
    q, k, v = randn(gen, B, Nq, Hq, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nk, Hk, 64)
    go = randn(gen, B, Nq, Hq, 64)
    idx = choose(gen, B, Nq, Hk, -(-Nk // bs), K, how)
    lens_t = None if lens is None else torch.tensor(lens, device=DEV, dtype=torch.int32 if Nk % 2 else torch.int64)
    want = oracle(q, k, v, idx, bs, lens=None if lens is None else lens_t.clamp(max=Nk), go=go)
    near(M.query_sparse_attn(q, k, v, idx, bs, kv_lens=lens_t), want["o"], "without a graph")
    ql, kl, vl = (t.clone().requires_grad_() for t in (q, k, v))
    out = M.query_sparse_attn(ql, kl, vl, idx, bs, kv_lens=lens_t)
    near(out.detach(), want["o"], "output")
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (ql, kl, vl), go)):
        assert got.dtype == BF16 and got.is_contiguous()
        near(got, want[name], name)


@gpu
def test_larger_mesh_and_two_runs_agree_bit_for_bit():
    gen = torch.Generator(device=DEV).manual_seed(2)
    B, N, Hq, Hk, bs, K = 1, 4096, 8, 2, 64, 8
    q, k, v = (randn(gen, B, N, h, 64).requires_grad_() for h in (Hq, Hk, Hk))
    go = randn(gen, B, N, Hq, 64)
    idx = choose(gen, B, N, Hk, N // bs, K, "near")
    idx[:, :, :, 0] = 5                       # one block that everyone has

    def step():
        out = M.query_sparse_attn(q, k, v, idx, bs, 0.2)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), go))
    first, second = step(), step()
    want = oracle(q, k, v, idx, bs, 0.2, go=go)
    for name, a, b in zip(("o", "dq", "dk", "dv"), first, second):
        near(a, want[name], name)
        assert torch.equal(a, b)


@gpu
def test_what_a_row_has_not_chosen_does_not_reach_it():
    gen = torch.Generator(device=DEV).manual_seed(3)
    B, Nq, Nk, Hq, Hk, bs = 1, 40, 640, 4, 1, 64
    q, k, v, go = randn(gen, B, Nq, Hq, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nq, Hq, 64)
    idx = torch.randint(0, 8, (B, Nq, Hk, 4), generator=gen, device=DEV)
    idx[:, 7] = torch.tensor([8, 1, 2, 3], device=DEV)        # only this token sees block 8, and 9 is nobody's
    lens = torch.tensor([630], device=DEV)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[:, 512:576], bad_v[:, 512:576] = float("nan"), float("inf")
    bad_k[:, 576:], bad_v[:, 576:] = float("inf"), float("nan")
    want = oracle(q, k, v, idx, bs, lens=lens, go=go)
    ql, kl, vl = (t.requires_grad_() for t in (q, bad_k, bad_v))
    out = M.query_sparse_attn(ql, kl, vl, idx, bs, kv_lens=lens)
    dq, dk, dv = torch.autograd.grad(out, (ql, kl, vl), go)
    rows = torch.arange(Nq, device=DEV) != 7
    for name, got in (("o", out.detach()), ("dq", dq)):
        near(got[:, rows], tuple(x[:, rows] for x in want[name]), name)
        assert not torch.isfinite(got[:, 7]).any()
    # keys that the token without a finite value has no part in
    others = torch.ones(Nk, dtype=torch.bool, device=DEV)
    for u in (8, 1, 2, 3):
        others[u * 64:u * 64 + 64] = False
    for name, got in (("dk", dk), ("dv", dv)):
        near(got[:, others], tuple(x[:, others] for x in want[name]), name)
    # keys past the end, in a block that is read
    lens = torch.tensor([100], device=DEV)
    idx = torch.randint(0, 2, (B, Nq, Hk, 2), generator=gen, device=DEV)
    bad_k, bad_v = k.detach().clone(), v.detach().clone()
    bad_k[:, 100:], bad_v[:, 100:] = float("nan"), float("inf")
    want = oracle(q, k, v, idx, bs, lens=lens, go=go)
    kl, vl = bad_k.requires_grad_(), bad_v.requires_grad_()
    out = M.query_sparse_attn(ql, kl, vl, idx, bs, kv_lens=lens)
    for name, got in zip(("o", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, (ql, kl, vl), go))):
        near(got, want[name], name)


@gpu
def test_large_and_small_scores():
    # scores of hundreds: the running maximum has to move; the exponent's fp32 error is 64 u |q||k| c
    # = 2^-18 * 8 * 8 * 40 * 0.2, below h / 8, and the bound's 1.25 h becomes 1.5 h
    gen = torch.Generator(device=DEV).manual_seed(4)
    q, k, v = randn(gen, 1, 50, 4, 64) * 20, randn(gen, 1, 1280, 1, 64) * 2, randn(gen, 1, 1280, 1, 64)
    q[:, 3] = 0
    idx = choose(gen, 1, 50, 1, 20, 9, "far")
    value, bound = oracle(q, k, v, idx, 64)["o"]
    near(M.query_sparse_attn(q, k, v, idx, 64), (value, 1.2 * bound), "output")


@gpu
def test_gradient_against_differences():
    gen = torch.Generator(device=DEV).manual_seed(5)
    q, k, v, go = (randn(gen, 1, n, h, 64) for n, h in ((6, 2), (128, 1), (128, 1), (6, 2)))
    idx = torch.tensor([0, 1, -1], device=DEV).view(1, 1, 1, 3).expand(1, 6, 1, 3)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(M.query_sparse_attn(*leaves, idx, 64), leaves, go)
    for i, g in enumerate(grads):
        e = randn(gen, *g.shape)
        step = 2.0 ** -3

        def f(s):
            moved = [t.double() for t in (q, k, v)]
            moved[i] = moved[i] + s * e.double()
            kk, vv = (t.expand(1, 128, 2, 64).permute(0, 2, 1, 3) for t in moved[1:])
            p = torch.softmax(moved[0].permute(0, 2, 1, 3) @ kk.transpose(-1, -2).contiguous() / 8, -1)
            return ((p @ vv).permute(0, 2, 1, 3) * go.double()).sum()
        diff = (8 * (f(step / 2) - f(-step / 2)) - (f(step) - f(-step))) / (6 * step)      # fourth order
        assert abs((g.double() * e.double()).sum() - diff) <= 4 * H * (g.double() * e.double()).abs().sum()


@gpu
def test_layouts_types_and_empty_calls():
    gen = torch.Generator(device=DEV).manual_seed(6)
    q, k, v = randn(gen, 2, 50, 8, 64), randn(gen, 2, 300, 2, 64), randn(gen, 2, 300, 2, 64)
    idx = choose(gen, 2, 50, 2, 5, 3, "far")
    want = M.query_sparse_attn(q, k, v, idx, 64)
    seq = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(M.query_sparse_attn(*seq, idx, 64), want)
    kv = torch.cat([k, v], dim=2)                                       # slices of one projection
    assert torch.equal(M.query_sparse_attn(q, kv[:, :, :2], kv[:, :, 2:], idx.to(torch.int32), 64), want)
    odd = torch.zeros(2, 50, 8, 65, device=DEV, dtype=BF16)
    odd[..., 1:] = q
    assert torch.equal(M.query_sparse_attn(odd[..., 1:], k, v, idx, 64), want)
    ql = q.float().requires_grad_()
    out = M.query_sparse_attn(ql, k.float(), v, idx, 64)
    assert out.dtype == torch.float32 and torch.equal(out.detach().to(BF16), want)
    (gq,) = torch.autograd.grad(out.sum(), ql)
    assert gq.dtype == torch.float32
    shared = k[:1].expand(2, 300, 2, 64)                                # one set of keys for the batch
    kl = k[:1].clone().requires_grad_()
    go = randn(gen, 2, 50, 8, 64)
    out = M.query_sparse_attn(q, kl.expand(2, 300, 2, 64), v, idx, 64)
    (gk,) = torch.autograd.grad(out, kl, go)
    assert gk.shape == kl.shape
    near(out.detach(), oracle(q, shared, v, idx, 64)["o"], "shared keys")
    for a, b, i in ((q[:, :0], k, idx[:, :0]), (q, k[:, :0], idx), (q, k, idx[..., :0])):
        leaves = [t.clone().requires_grad_() for t in (a, b, b)]
        out = M.query_sparse_attn(*leaves, i, 64)
        assert out.shape == a.shape and not out.any()
        assert all(not g.any() for g in torch.autograd.grad(out.sum(), leaves))


@gpu
@pytest.mark.parametrize("K", [4, 9])          # few keys a workgroup, and a union in shares
def test_captured_replayed_and_on_another_stream(K):
    gen = torch.Generator(device=DEV).manual_seed(7)
    q, k, v, go = randn(gen, 1, 60, 4, 64), randn(gen, 1, 640, 1, 64), randn(gen, 1, 640, 1, 64), randn(gen, 1, 60, 4, 64)
    idx = choose(gen, 1, 60, 1, 10, K, "far")

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = M.query_sparse_attn(*leaves, idx, 64)
        return (out.detach(), *torch.autograd.grad(out, leaves, go))
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.cuda.graph(other):              # a second graph of the same calls
        held2 = step()
    for i in range(3):
        q.copy_(randn(gen, 1, 60, 4, 64))
        idx.copy_(choose(gen, 1, 60, 1, 10, K, "ragged"))
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i
        assert all(torch.equal(a, b) for a, b in zip(held2, want)), i


@gpu
def test_key_offsets_past_32_bits():
    # key rows 2^25 elements apart: the last block starts past 2^32 elements (9 GB of bf16)
    apart, Nk = 1 << 25, 133
    gen = torch.Generator(device=DEV).manual_seed(8)
    k = torch.empty((Nk - 1) * apart + 64, device=DEV, dtype=BF16).as_strided((1, Nk, 1, 64), (0, apart, 64, 1))
    small, v, q = randn(gen, 1, Nk, 1, 64), randn(gen, 1, Nk, 1, 64), randn(gen, 1, 9, 2, 64)
    k.copy_(small)
    idx = torch.tensor([0, 2], device=DEV).view(1, 1, 1, 2).expand(1, 9, 1, 2)
    assert torch.equal(M.query_sparse_attn(q, k, v, idx, 64), M.query_sparse_attn(q, small, v, idx, 64))


@gpu
def test_the_run_of_operators_as_they_are_used():
    """Norm and rotate queries at points and keys on a mesh, pool, choose, attend; forward and backward."""
    gen = torch.Generator(device=DEV).manual_seed(9)
    B, Nq, Nk, Hq, Hk, bs, K = 2, 75, 1024, 8, 2, 64, 5
    q0, k0 = randn(gen, B, Nq, Hq, 64).requires_grad_(), randn(gen, B, Nk, Hk, 64).requires_grad_()
    v = randn(gen, B, Nk, Hk, 64).requires_grad_()
    wq, wk = ((1 + 0.1 * torch.randn(64, generator=gen, device=DEV)).requires_grad_() for _ in range(2))
    at_q, at_k = torch.randn(B, Nq, 3, generator=gen, device=DEV), torch.randn(Nk, 3, generator=gen, device=DEV)
    sections = (8, 12, 12)
    q, _ = M.qk_norm_rope(q0, None, wq, positions=at_q, sections=sections)
    k, _ = M.qk_norm_rope(k0, None, wk, positions=at_k, sections=sections)
    out, idx = M.mosaic_query_attn(q, k, v, bs, K, return_block_indices=True)
    assert torch.equal(idx, M.query_topk(q.detach(), M.pool_mean(k.detach(), bs), K))
    go = randn(gen, B, Nq, Hq, 64)
    want = oracle(q, k, v, idx, bs, go=go)
    near(out.detach(), want["o"], "output")
    got = torch.autograd.grad(out, (q, k, v), go, retain_graph=True)
    for name, g in zip(("dq", "dk", "dv"), got):
        near(g, want[name], name)
    # the graph to the leaves: the norm's backward of those gradients
    leaves = torch.autograd.grad(out, (q0, k0, wq, wk), go, retain_graph=True)
    again = torch.autograd.grad((q, k), (q0, k0, wq, wk), got[:2])
    for a, b in zip(leaves, again):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    with_cmp = M.mosaic_query_attn(q, k, v, bs, K, k_cmp=M.pool_mean(k.detach(), bs))
    assert torch.equal(with_cmp, out)
    mask = torch.zeros(B, Nk // bs, dtype=torch.bool, device=DEV)
    mask[0, 3] = True
    out, idx = M.mosaic_query_attn(q, k, v, bs, K, block_mask=mask, return_block_indices=True)
    assert bool((idx[0, ..., 0] == 3).all()) and bool((idx[0, ..., 1:] == -1).all()) and not out[1].any()


@gpu
@pytest.mark.parametrize("Hq,Hk,K", [(4, 1, 3), (6, 2, 5)])
def test_a_block_that_every_token_wants(Hq, Hk, K):
    """Its keys' gradients are shared out over workgroups and summed; twice the same bits."""
    gen = torch.Generator(device=DEV).manual_seed(10)
    B, Nq, Nk, bs = 1, 2000, 1250, 64
    q, k, v, go = randn(gen, B, Nq, Hq, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nq, Hq, 64)
    idx = choose(gen, B, Nq, Hk, 20, K, "far")
    idx[..., 0], idx[:, 1000:, :, 1] = 3, 19                       # one of them the ragged last block
    lens = torch.tensor([1230], device=DEV)
    want = oracle(q, k, v, idx, bs, lens=lens, go=go)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = M.query_sparse_attn(*leaves, idx, bs, kv_lens=lens)
    got = torch.autograd.grad(out, leaves, go, retain_graph=True)
    for name, g in zip(("o", "dq", "dk", "dv"), (out.detach(), *got)):
        near(g, want[name], name)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(out, leaves, go)))


@gpu
@pytest.mark.parametrize("Hq,Hk,Nq,K", [(2, 2, 1500, 40), (16, 1, 300, 70), (3, 1, 1000, 1)])
def test_scattered_tokens(Hq, Hk, Nq, K):
    """Tokens that share little with the ones beside them, in unions of more than 64 blocks.  A
    token's result does not depend on the order of the tokens (workgroups as many either way)."""
    gen = torch.Generator(device=DEV).manual_seed(11)
    B, Nk, bs = 2, 130 * 64, 64
    q, k, v, go = randn(gen, B, Nq, Hq, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nq, Hq, 64)
    idx = choose(gen, B, Nq, Hk, 130, K, "far")
    want = oracle(q, k, v, idx, bs, go=go)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = M.query_sparse_attn(*leaves, idx, bs)
    for name, g in zip(("o", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, go))):
        near(g, want[name], name)
    perm = torch.randperm(Nq, generator=gen, device=DEV)
    assert torch.equal(M.query_sparse_attn(q[:, perm], k, v, idx[:, perm], bs), out.detach()[:, perm])


@gpu
def test_more_blocks_than_are_united_at_a_time():
    gen = torch.Generator(device=DEV).manual_seed(12)
    B, Nq, nb, Hq, Hk, bs = 1, 37, 2100, 4, 1, 64
    Nk = nb * bs - 17
    q, k, v, go = randn(gen, B, Nq, Hq, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nq, Hq, 64)
    idx = choose(gen, B, Nq, Hk, nb, 6, "far")
    idx[..., :3] = torch.tensor([1023, 1024, nb - 1], device=DEV)
    idx[:, ::2, :, 0] = 2048
    want = oracle(q, k, v, idx, bs, go=go)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = M.query_sparse_attn(*leaves, idx, bs)
    for name, g in zip(("o", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, go))):
        near(g, want[name], name)


@gpu
def test_keys_whose_scores_are_minus_infinity():
    """They have no weight, wherever they stand among a row's keys; with nothing else a row is zeros."""
    gen = torch.Generator(device=DEV).manual_seed(13)
    for Nq in (3, 400):                                                     # with a share of the blocks each, and without
        q, k, v = randn(gen, 1, Nq, 4, 64), randn(gen, 1, 640, 1, 64), randn(gen, 1, 640, 1, 64)
        q[..., 0] = 1
        k[:, :128, :, 0] = -float("inf")                                    # blocks 0 and 1
        k[:, 300:310, :, 0] = -float("inf")                                 # and keys of block 4
        idx = torch.tensor([0, 4, 1, 7], device=DEV).expand(1, Nq, 1, 4).clone()
        idx[:, 2] = torch.tensor([0, 1, 1, -1], device=DEV)
        out = M.query_sparse_attn(q, k, v, idx, 64)
        assert torch.isfinite(out).all() and not out[:, 2].any()
        kf = k.clone()
        kf[:, 300:310, :, 0] = -1e30
        rows = torch.arange(Nq, device=DEV) != 2
        near(out[:, rows], tuple(x[:, rows] for x in oracle(q, kf, v, idx.clamp(4, 9), 64)["o"]), "output")


@gpu
def test_query_and_gradient_offsets_past_32_bits():
    # rows of q and of the gradient 2^25 elements apart: the last begin past 2^32 bytes and elements
    apart, Nq = 1 << 25, 140
    gen = torch.Generator(device=DEV).manual_seed(14)
    small = randn(gen, 1, Nq, 2, 64), randn(gen, 1, Nq, 2, 64)
    wide = [torch.empty((Nq - 1) * apart + 128, device=DEV, dtype=BF16).as_strided((1, Nq, 2, 64), (0, apart, 64, 1)) for _ in small]
    for w, s in zip(wide, small):
        w.copy_(s)
    k, v = randn(gen, 1, 256, 1, 64), randn(gen, 1, 256, 1, 64)
    idx = torch.tensor([0, 2], device=DEV).view(1, 1, 1, 2).expand(1, Nq, 1, 2)

    def run(q, go):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = M.query_sparse_attn(*leaves, idx, 64)
        return (out.detach(), *torch.autograd.grad(out, leaves, go))
    assert all(torch.equal(a, b) for a, b in zip(run(*wide), run(*small)))


@gpu
def test_calls_on_two_streams_at_once():
    gen = torch.Generator(device=DEV).manual_seed(15)
    sets = []
    for Nq in (2, 900):
        q, k, v, go = randn(gen, 1, Nq, 4, 64), randn(gen, 1, 2560, 1, 64), randn(gen, 1, 2560, 1, 64), randn(gen, 1, Nq, 4, 64)
        sets.append((q, k, v, go, choose(gen, 1, Nq, 1, 40, 8, "far")))

    def step(q, k, v, go, idx):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = M.query_sparse_attn(*leaves, idx, 64)
        return (out.detach(), *torch.autograd.grad(out, leaves, go))
    want = [step(*s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(step(*s))
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2])), i


@gpu
@pytest.mark.parametrize("B,Nq,Nk,Hq,Hk,bs,K,how,lens", [
    (1, 1, 196608, 12, 3, 128, 16, "far", None),          # 16 blocks of two tiles
    (2, 1, 5000, 4, 1, 256, 8, "far", (4999, 700)),       # the last blocks end inside a tile, and before
    (3, 5, 900, 8, 1, 64, 7, "ragged", (900, 1, 64)),     # four tokens a workgroup, then one
    (1, 9, 640, 4, 4, 64, 1, "ragged", None),             # one query head to a kv head
    (1, 2, 640, 32, 2, 64, 10, "near", (0,)),             # no key at all
    (2, 40, 2000, 14, 2, 64, 8, "far", (1999, 2000)),     # 28 rows of 32
    (1, 1, 5000, 16, 1, 2048, 1, "far", (4000,)),         # one block of 32 tiles
])
def test_few_tokens_with_few_keys(B, Nq, Nk, Hq, Hk, bs, K, how, lens):
    gen = torch.Generator(device=DEV).manual_seed(Nk + K)
    q, k, v, go = randn(gen, B, Nq, Hq, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nq, Hq, 64)
    idx = choose(gen, B, Nq, Hk, -(-Nk // bs), K, how)
    lens = None if lens is None else torch.tensor(lens, device=DEV)
    assert _lib.lib().mosaic_query_attn_fwd_workspace_size(B, Nq, Hq, Hk, bs, K) == 0
    want = oracle(q, k, v, idx, bs, lens=lens, go=go)
    near(M.query_sparse_attn(q, k, v, idx, bs, kv_lens=lens), want["o"], "output")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = M.query_sparse_attn(*leaves, idx, bs, kv_lens=lens)
    for name, g in zip(("o", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, go))):
        near(g, want[name], name)


@gpu
def test_few_tokens_and_values_that_are_not_finite():
    """NaN and infinities of one token's block reach that token alone, and none behind the sequence's end."""
    gen = torch.Generator(device=DEV).manual_seed(16)
    q, k, v = randn(gen, 1, 8, 4, 64), randn(gen, 1, 640, 1, 64), randn(gen, 1, 640, 1, 64)
    idx = torch.randint(0, 8, (1, 8, 1, 4), generator=gen, device=DEV)
    idx[:, 3, :, 0] = 8                                                 # only this token has block 8; nobody has 9
    lens = torch.tensor([630], device=DEV)
    value, bound = oracle(q, k, v, idx, 64, lens=lens)["o"]
    k[:, 512:], v[:, 512:] = float("inf"), float("nan")
    out = M.query_sparse_attn(q, k, v, idx, 64, kv_lens=lens)
    rows = torch.arange(8, device=DEV) != 3
    near(out[:, rows], (value[:, rows], bound[:, rows]), "output")
    assert not torch.isfinite(out[:, 3]).any()
    idx[:, 3, :, 0] = 7
    lens = torch.tensor([460], device=DEV)                              # ends inside block 7
    k, v = randn(gen, 1, 640, 1, 64), randn(gen, 1, 640, 1, 64)
    want = oracle(q, k, v, idx, 64, lens=lens)["o"]
    k[:, 460:], v[:, 460:] = float("nan"), float("inf")
    near(M.query_sparse_attn(q, k, v, idx, 64, kv_lens=lens), want, "output")


@HAVE_LIB
def test_backward_refuses_a_misplaced_order():
    c = dict(q=_lib.Bnhd(FAKE, 0, 256, 64), k=_lib.Bnhd(FAKE, 0, 128, 64), idx=FAKE, B=1, nq=7, nk=200, hq=4, hk=2, d=64, bs=64,
             K=12, out=FAKE, lse=FAKE, ws=FAKE, n=1 << 40, order=FAKE + 16)
    assert _call("bwd", c) == 7


@gpu
@pytest.mark.parametrize("Nq,K", [(60, 3), (500, 8), (4000, 20), (40, 20)])
def test_backward_with_and_without_the_forward_s_order(Nq, K):
    gen = torch.Generator(device=DEV).manual_seed(Nq)
    q, k, v, go = randn(gen, 1, Nq, 4, 64), randn(gen, 1, 3000, 1, 64), randn(gen, 1, 3000, 1, 64), randn(gen, 1, Nq, 4, 64)
    idx = choose(gen, 1, Nq, 1, 47, K, "far")

    def grads(keep):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = M.query_sparse_attn(*leaves, idx, 64)
        if not keep:
            out.grad_fn.order = None
        return torch.autograd.grad(out, leaves, go)
    assert all(torch.equal(a, b) for a, b in zip(grads(True), grads(False)))


@gpu
@pytest.mark.parametrize("B,Nq,Nk,Hq,Hk,bs,K", [(1, 2, 700, 8, 4, 64, 7), (2, 5, 3000, 20, 5, 128, 9), (1, 300, 2000, 2, 1, 64, 6)])
def test_gradients_of_few_tokens_keep_their_precision(B, Nq, Nk, Hq, Hk, bs, K):
    """P and dS in two parts are off by 2^-16 and the delta by fp32 sums: what remains beside the
    gradients' own rounding is the exponent's error, a fifth of the terms' part of the bound at most."""
    gen = torch.Generator(device=DEV).manual_seed(Nk)
    q, k, v, go = randn(gen, B, Nq, Hq, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nq, Hq, 64)
    idx = choose(gen, B, Nq, Hk, -(-Nk // bs), K, "far")
    want = oracle(q, k, v, idx, bs, go=go)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    _, dk, dv = torch.autograd.grad(M.query_sparse_attn(*leaves, idx, bs), leaves, go)
    for name, got in (("dk", dk), ("dv", dv)):
        value, bound = want[name]
        near(got, (value, H * value.abs() + (bound - H * value.abs()) / 4), name)


@pytest.mark.parametrize("scale", [1e-46, 1e-31, 1e31, 1e39, float("inf"), float("nan"), -1.0])
def test_scales_that_fp32_does_not_carry_are_refused(scale):
    with pytest.raises(ValueError, match="softmax_scale"):
        M.query_sparse_attn(z(*Q), z(*KV), z(*KV), IDX, 64, softmax_scale=scale)
    with pytest.raises(ValueError, match="softmax_scale"):
        M.mosaic_query_attn(z(*Q), z(1, 128, 2, 64), z(1, 128, 2, 64), 64, 2, softmax_scale=scale)


@HAVE_LIB
@pytest.mark.parametrize("scale", [1e-44, 1e-31, 1e31, float("inf"), float("nan")])
def test_abi_refuses_scales(scale):
    L, row = _lib.lib(), _lib.Bnhd(FAKE, 0, 256, 64)
    kv = _lib.Bnhd(FAKE, 0, 128, 64)
    assert L.mosaic_query_attn_fwd(row, kv, kv, FAKE, None, 1, 7, 500, 4, 2, 64, 64, 3, scale, FAKE, FAKE, FAKE, 1 << 30, None) == 11
    assert L.mosaic_query_attn_bwd(row, kv, kv, FAKE, FAKE, row, FAKE, None, 1, 7, 500, 4, 2, 64, 64, 3, scale, None, FAKE, FAKE,
                                   FAKE, FAKE, 1 << 30, None) == 11


@gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-6])
def test_scales_near_nothing(scale):
    # every key weighs the same: the output and grad v are those of the mean
    gen = torch.Generator(device=DEV).manual_seed(31)
    q, k, v, go = randn(gen, 1, 9, 2, 64), randn(gen, 1, 300, 1, 64), randn(gen, 1, 300, 1, 64), randn(gen, 1, 9, 2, 64)
    idx = choose(gen, 1, 9, 1, 5, 3, "far")
    want = oracle(q, k, v, idx, 64, scale=scale, go=go)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = M.query_sparse_attn(*leaves, idx, 64, softmax_scale=scale)
    grads = torch.autograd.grad(out, leaves, go)
    near(out.detach(), want["o"], "output")
    near(grads[2], want["dv"], "grad v")
    for g, name in zip(grads, ("dq", "dk")):
        near(g.double() / scale, tuple(t / scale for t in want[name]), name)


@pytest.mark.parametrize("call,match", [
    (lambda: M.query_sparse_attn(z(*Q), z(*KV), z(*KV), IDX, (1 << 32) + 64), "block_size"),
    (lambda: M.query_sparse_attn(z(*Q), z(*KV), z(*KV), IDX, 1 << 31), "block_size"),
    (lambda: M.mosaic_query_attn(z(*Q), z(1, 0, 2, 64), z(1, 0, 2, 64), (1 << 32) + 64, 2), "block_size"),
    (lambda: M.query_sparse_attn(z(*Q), *[z(1, 1, 2, 64).expand(1, (1 << 32) + 64, 2, 64)] * 2, IDX, 64), "2\\^31"),
    (lambda: M.query_sparse_attn(z(1, 1, 4, 64).expand(1, 1 << 31, 4, 64), z(*KV), z(*KV), IDX, 64), "2\\^31"),
    (lambda: M.query_topk(z(*Q), z(1, 1, 2, 64).expand(1, (1 << 32) + 64, 2, 64), 2), "2\\^31"),
    (lambda: M.query_topk(z(1, 1, 1, 64).expand((1 << 32) + 1, 1, 1, 64), z(1, 2, 1, 64).expand((1 << 32) + 1, 2, 1, 64), 2), "2\\^31"),
])
def test_sizes_that_32_bits_do_not_carry_are_refused(call, match):
    with pytest.raises(ValueError, match=match):
        call()


@HAVE_LIB
def test_partials_do_not_grow_with_the_call():
    # what a large call keeps in proportion to its tokens, blocks and bits; the partials beside it stay below 160 MiB
    for B, Nq, Nk, Hq, Hk, bs, K in [(24, 196608, 196608, 12, 3, 64, 16), (4, 49152, 49152, 12, 3, 64, 16), (1, 1000, 1 << 22, 8, 8, 64, 2),
                                     (1, 12288, 12288, 16, 4, 64, 12), (8, 100000, 512, 4, 4, 256, 2)]:
        nb, tiles = -(-Nk // bs), -(-Nk // 64) * Hk * B
        chosen = Nq * min(K, nb) * Hk * B
        rest = 8 * B * Nq * Hq + B * Hk * nb * (Nq + 511) // 512 * 64 + 8 * B * Hk * nb + 4 * chosen + 12 * tiles + 8 * chosen // 64 + 6 * B * Hk * Nq
        got = _lib.lib().mosaic_query_attn_bwd_workspace_size(B, Nq, Nk, Hq, Hk, bs, K)
        assert 0 < got <= rest + (160 << 20), (B, Nq, Nk, got / 2 ** 20, rest / 2 ** 20)


@gpu
def test_many_key_tiles_with_wanted_blocks():
    # 4096 key tiles, so that only blocks that most tokens want are divided
    gen = torch.Generator(device=DEV).manual_seed(33)
    B, Nq, Nk, Hk, K = 16, 500, 2048, 8, 8
    q, k, v, go = randn(gen, B, Nq, Hk, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nk, Hk, 64), randn(gen, B, Nq, Hk, 64)
    idx = choose(gen, B, Nq, Hk, Nk // 64, K, "far")
    idx[:, :, 0, 1] = 5
    idx[3, 20:, 2, 2:] = -1
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = M.query_sparse_attn(*leaves, idx, 64)
    grads = torch.autograd.grad(out, leaves, go)
    for b in range(0, B, 5):                     # (a sequence at a time: the oracle's scores are dense)
        want = oracle(q[b:b + 1], k[b:b + 1], v[b:b + 1], idx[b:b + 1], 64, go=go[b:b + 1])
        near(out.detach()[b:b + 1], want["o"], "output")
        for g, name in zip(grads, ("dq", "dk", "dv")):
            near(g[b:b + 1], want[name], name)


@gpu
@pytest.mark.parametrize("Nq,Nk,Hq,Hk,K", [(6, 128, 2, 1, 2), (40, 700, 4, 2, 5), (300, 500, 4, 1, 3)])
def test_gradients_along_themselves_against_differences(Nq, Nk, Hq, Hk, K):
    """The derivative along a gradient is its norm, in which nothing cancels: a gradient twice as large, or
    with a part left out, is far outside.  What rounding may do to it is the sum of the elements' bounds
    along that direction (the output's l sums the rounded P, its log-sum-exp, which the backward reads, the
    unrounded ones); the difference quotient in float64 is off by step^4, below 1e-6 of it."""
    gen = torch.Generator(device=DEV).manual_seed(Nq)
    q, k, v, go = (randn(gen, 1, n, h, 64) for n, h in ((Nq, Hq), (Nk, Hk), (Nk, Hk), (Nq, Hq)))
    idx = choose(gen, 1, Nq, Hk, -(-Nk // 64), K, "far")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(M.query_sparse_attn(*leaves, idx, 64), leaves, go)
    bounds = oracle(q, k, v, idx, 64, go=go)
    member = torch.zeros(1, Nq, Hk, -(-Nk // 64), dtype=torch.bool, device=DEV).scatter_(-1, idx, True)
    ok = member.repeat_interleave(64, -1)[..., :Nk].permute(0, 2, 1, 3).repeat_interleave(Hq // Hk, 1)

    def f(i, x):
        qh, kh, vh = (t.double().permute(0, 2, 1, 3) for t in (x if j == i else t for j, t in enumerate((q, k, v))))
        kh, vh = kh.repeat_interleave(Hq // Hk, 1), vh.repeat_interleave(Hq // Hk, 1)
        s = (qh @ kh.transpose(-1, -2).contiguous() / 8).masked_fill(~ok, -torch.inf)
        return ((torch.softmax(s, -1) @ vh).permute(0, 2, 1, 3) * go.double()).sum()

    for i, (g, x, name) in enumerate(zip(grads, (q, k, v), ("dq", "dk", "dv"))):
        size = g.double().norm()
        e, step = g.double() / size, 2.0 ** -5
        at = [f(i, x.double() + s * step * e) for s in (1, -1, 0.5, -0.5)]
        diff = (8 * (at[2] - at[3]) - (at[0] - at[1])) / (6 * step)
        slack = (bounds[name][1] * e.abs()).sum() + 1e-6 * size
        assert slack < diff / 2, (name, (slack / size).item())     # a gradient of twice or half the size is off by diff / 2 or more
        assert abs(size - diff) <= slack, (name, ((size - diff) / size).item(), (slack / size).item())
