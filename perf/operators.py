"""Cases of the query-side operators, with their plain forms and their values in float64.

* ``rope``: ``rope_axes``, rotary positions with several axes (time, longitude, latitude);
* ``norm``: ``qk_norm_rope``, the RMS norm of each query and key head and its rotation;
* ``topk``: ``query_topk``, the key blocks that a cheap score selects for each query token;
* ``attn``: ``query_sparse_attn``, attention of each query token over its own blocks.

A case with ``train`` set is a forward and a backward pass.  Sizes are those of the HEALPix
sequences of the model (768 tokens at nside 8 to 196608 at nside 128), its heads (12/3, 16/4,
20/5) and its selection blocks (64 and 128 tokens), with odd counts between.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TYPES = {"bf16": BF16, "f32": F32}


def _rope(name, seq, batch, hq, hk, sections, dtype="bf16", pairs="interleaved", train=False, integers=False,
          own_positions=False, d=64):
    return dict(name=name, kind="rope", seq=seq, batch=batch, hq=hq, hk=hk, sections=sections, dtype=dtype, pairs=pairs,
                train=train, integers=integers, own_positions=own_positions, d=d)


def _norm(name, seq, batch, hq, hk, dtype="bf16", pairs="interleaved", train=False, seq_first=False, d=64):
    return dict(name=name, kind="norm", seq=seq, batch=batch, hq=hq, hk=hk, dtype=dtype, pairs=pairs, train=train,
                seq_first=seq_first, d=d)


def _topk(name, queries, nb, batch, hq, hk, top, masked=False):
    return dict(name=name, kind="topk", queries=queries, nb=nb, batch=batch, hq=hq, hk=hk, top=top, masked=masked)


def _attn(name, queries, keys, batch, hq, hk, bs, top, scattered=False, ragged=False, train=False):
    return dict(name=name, kind="attn", queries=queries, keys=keys, batch=batch, hq=hq, hk=hk, bs=bs, top=top,
                scattered=scattered, ragged=ragged, train=train)


def listed():
    return [
        # one target point per ensemble member, each at its own time and place: a call's fixed cost
        _rope("rope_one_point_b24", 1, 24, 12, 3, "8,12,12", own_positions=True),
        # a training step on an odd number of points in fp32, integer grid coordinates, halves as pairs
        _rope("rope_train_f32_odd", 1537, 3, 16, 4, "16,8,8", dtype="f32", pairs="halves", train=True, integers=True),
        # the finest mesh: every token of nside 128 with time, longitude and latitude
        _rope("rope_nside128", 196608, 1, 12, 3, "8,12,12"),
        # a coarse stage at two members in fp32
        _norm("norm_nside8_f32", 768, 2, 20, 5, dtype="f32"),
        # the widest stage for four members, sequence-first as the model's projections leave it
        _norm("norm_nside64_b4", 49152, 4, 12, 3, seq_first=True),
        # a training step of the second stage
        _norm("norm_train_nside32_b4", 12288, 4, 16, 4, train=True),
        # a few stations against the blocks of nside 64
        _topk("topk_37_points", 37, 768, 1, 12, 3, 16, masked=True),
        # every token of nside 64 selects its own blocks
        _topk("topk_nside64", 49152, 768, 1, 12, 3, 16),
        # one point against the nside 128 state: the split over the selected keys counts
        _attn("attn_one_point", 1, 196608, 1, 12, 3, 128, 16),
        # scattered stations in no order, padded batch, some rows without a block
        _attn("attn_stations_b2", 10007, 49152, 2, 12, 3, 64, 16, scattered=True, ragged=True),
        # every token of nside 64 reads its own blocks
        _attn("attn_nside64", 49152, 49152, 1, 12, 3, 64, 16),
        # training the second stage's selection per token
        _attn("attn_train_nside32", 12288, 12288, 1, 16, 4, 64, 12, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    g = rng.choice((4, 4, 4, 2, 1, 3, 8))
    hk = rng.randint(1, 5 if g <= 4 else 2)
    return g * hk, hk


def draw(rng):
    kind = rng.choice(("rope", "norm", "topk", "attn", "attn"))
    hq, hk = _heads(rng)
    if kind in ("rope", "norm"):
        dtype, pairs = rng.choice(("bf16", "bf16", "f32")), rng.choice(("interleaved", "halves"))
        d = rng.choice((64, 64, 128, 32))
        train = rng.random() < 0.4
        unit = (hq + hk) * d * (2 if dtype == "f32" else 1) * (3 if train else 1)
        tokens = 196608 * 15 * 64 // unit       # at most the largest listed call's bytes
        seq = _log_int(rng, 1, min(196608, tokens))
        batch = _log_int(rng, 1, max(1, min(24, tokens // seq)))
        if kind == "norm":
            c = _norm("", seq, batch, hq, hk, dtype, pairs, train, rng.random() < 0.5, d)
        else:
            half = d // 2
            a = rng.randint(1, half - 2)
            b = rng.randint(1, half - a - 1)
            # two or three axes, the pairs past the last section unrotated
            sections = rng.choice((f"{half - a},{a}", f"{half - a - b},{a},{b}", f"{a},{b}"))
            c = _rope("", seq, batch, hq, hk, sections, dtype, pairs, train, rng.random() < 0.5, rng.random() < 0.5, d)
    elif kind == "topk":
        nb = _log_int(rng, 24, 1600)
        top = rng.randint(1, min(24, nb))
        queries = _log_int(rng, 1, min(49152, 49152 * 768 * 12 // (nb * hq)))
        c = _topk("", queries, nb, 1, hq, hk, top, rng.random() < 0.4)
        c["batch"] = _log_int(rng, 1, max(1, min(8, 49152 * 768 * 12 // (nb * hq * queries))))
    else:
        bs, train = rng.choice((64, 64, 128)), rng.random() < 0.4
        keys = _log_int(rng, 1000, 49152)
        top = rng.randint(1, min(24 if bs == 64 else 12, -(-keys // bs)))
        most = 12288 * 16 * 64 * 12 if train else 49152 * 12 * 64 * 16
        queries = _log_int(rng, 1, min(49152, most // (hq * bs * top)))
        batch = _log_int(rng, 1, max(1, min(4, most // (hq * bs * top * queries))))
        c = _attn("", queries, keys, batch, hq, hk, bs, top, rng.random() < 0.3, rng.random() < 0.4, train)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(2000003 + 7919 * int(seed))


def _randn(gen, *shape, dtype=BF16):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=F32).to(dtype)


def _field(gen, at, channels):
    """A smooth random field of the position ``at`` in [0, 1): waves of wavelengths from the whole
    sequence down to a hundredth of it, long ones strongest, so that neighbours are alike."""
    f = torch.exp(torch.rand(24, generator=gen, device=DEV) * math.log(100.0))
    amp = torch.randn(24, channels, generator=gen, device=DEV) / f.sqrt()[:, None]
    ph = 2 * math.pi * torch.rand(24, generator=gen, device=DEV)
    return torch.cos(2 * math.pi * at[:, None] * f + ph) @ (amp * (2.0 / (1.0 / f).sum().sqrt()))


def _pooled(case, gen, nq, nb, at):
    """Queries that vary smoothly with their place ``at``, and the means of as many key blocks: keys
    of a place resemble the queries of that place."""
    B, Hq, Hk = case["batch"], case["hq"], case["hk"]
    q, k = [], []
    for _ in range(B):
        place = torch.cat([at, (torch.arange(nb, device=DEV) + 0.5) / nb])
        base = _field(gen, place, Hk * 64).view(-1, Hk, 64)
        q.append(base[:nq].repeat_interleave(Hq // Hk, dim=1) + 0.5 * _field(gen, at, Hq * 64).view(nq, Hq, 64)
                 + 0.1 * torch.randn(nq, Hq, 64, generator=gen, device=DEV))
        k.append(base[nq:] + 0.3 * torch.randn(nb, Hk, 64, generator=gen, device=DEV))
    return torch.stack(q).to(BF16), torch.stack(k).to(BF16)


def _places(case, gen, n):
    at = (torch.arange(n, device=DEV) + 0.5) / n
    return torch.rand(n, generator=gen, device=DEV) if case.get("scattered") or n < 64 else at


def prepare(case, seed):
    gen = _gen(seed)
    kind = case["kind"]
    s = dict(case=case)
    if kind in ("rope", "norm"):
        B, N, d, dt = case["batch"], case["seq"], case["d"], TYPES[case["dtype"]]
        made = []
        for h in (case["hq"], case["hk"]):
            made.append(_randn(gen, N, B, h, d, dtype=dt).transpose(0, 1) if case.get("seq_first")
                        else _randn(gen, B, N, h, d, dtype=dt))
        s["q"], s["k"] = made
        if case["train"]:
            s["gq"], s["gk"] = (_randn(gen, B, N, h, d, dtype=dt) for h in (case["hq"], case["hk"]))
        if kind == "norm":
            s["wq"], s["wk"] = (1 + 0.2 * _randn(gen, d, dtype=F32) for _ in range(2))
            # the tables that a rotary module keeps: two axes of angles
            at = torch.rand(N, 2, generator=gen, device=DEV) * torch.tensor([360.0, 180.0], device=DEV) - 90.0
            n = d // 4
            f = 10000.0 ** (-torch.arange(n, device=DEV) / n)
            ang = (torch.deg2rad(at)[:, :, None] * f).reshape(N, 2 * n)
            s["cos"], s["sin"] = ang.cos(), ang.sin()
        else:
            s["sections"] = tuple(int(x) for x in case["sections"].split(","))
            shape = ((B,) if case["own_positions"] else ()) + (N, len(s["sections"]))
            if case["integers"]:
                s["pos"] = torch.randint(0, 100000, shape, generator=gen, device=DEV)
            else:   # hours since a far start, then radians
                p = (torch.rand(*shape, generator=gen, device=DEV) - 0.5) * 2 * math.pi
                p[..., 0] = torch.randint(0, 1 << 20, shape[:-1], generator=gen, device=DEV).float() / 4
                s["pos"] = p
        return s
    if kind == "topk":
        s["q"], s["kc"] = _pooled(case, gen, case["queries"], case["nb"], _places(case, gen, case["queries"]))
        s["mask"] = None
        if case["masked"]:   # the last sequence has no more than a few blocks that may be read
            s["mask"] = torch.rand(case["batch"], case["nb"], generator=gen, device=DEV) < 0.7
            s["mask"][-1, max(1, case["top"] // 2):] = False
        return s
    B, Nq, Nk, Hq, Hk, bs, K = (case[n] for n in ("batch", "queries", "keys", "hq", "hk", "bs", "top"))
    nb = -(-Nk // bs)
    q, kc = _pooled(case, gen, Nq, nb, _places(case, gen, Nq))
    lens = torch.full((B,), Nk, device=DEV, dtype=torch.int32)
    if case["ragged"]:   # a padded batch: the sequences end anywhere, inside a block too
        lens = torch.randint(max(1, Nk // 3), Nk + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
    live = torch.arange(nb, device=DEV) * bs < lens[:, None]
    score = torch.matmul(q.float().view(B, Nq, Hk, Hq // Hk, 64).mean(3).transpose(1, 2), kc.float().permute(0, 2, 3, 1).contiguous())
    score.masked_fill_(~live[:, None, None, :], -math.inf)
    best = score.topk(K, dim=-1)
    idx = torch.where(best.values.isinf(), -1, best.indices).transpose(1, 2).contiguous()
    if case["ragged"]:   # rows and slots without a block
        idx.masked_fill_((torch.rand(B, Nq, generator=gen, device=DEV) < 0.05)[:, :, None, None], -1)
        idx.masked_fill_(torch.rand(idx.shape, generator=gen, device=DEV) < 0.05, -1)
    k = kc.float().repeat_interleave(bs, dim=1)[:, :Nk] + _randn(gen, B, Nk, Hk, 64, dtype=F32)
    s.update(q=q, k=k.to(BF16), v=_randn(gen, B, Nk, Hk, 64), idx=idx, lens=lens if case["ragged"] else None)
    if case["train"]:
        s["go"] = _randn(gen, B, Nq, Hq, 64)
    return s


# ------------------------------------------------------------------------------------ one pass

def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    if case["kind"] == "rope":
        return _plain_rope(s, case)
    if case["kind"] == "norm":
        return _plain_norm(s, case)
    return _plain_topk(s, case) if case["kind"] == "topk" else _plain_attn(s, case)


def _own(s, case):
    import mosaic_amd as M

    kind, train = case["kind"], case.get("train")
    if kind == "topk":
        return M.query_topk(s["q"], s["kc"], case["top"], block_mask=s["mask"])
    leaves = [s["q"], s["k"]] + ([s["wq"], s["wk"]] if kind == "norm" else [s["v"]] if kind == "attn" else [])
    if train:
        leaves = [t.detach().requires_grad_() for t in leaves]
    if kind == "rope":
        out = M.rope_axes(leaves[0], leaves[1], s["pos"], s["sections"], interleaved=case["pairs"] == "interleaved")
        grads = (s["gq"], s["gk"]) if train else None
    elif kind == "norm":
        out = M.qk_norm_rope(*leaves, eps=1e-6, cos=s["cos"], sin=s["sin"], interleaved=case["pairs"] == "interleaved")
        grads = (s["gq"], s["gk"]) if train else None
    else:
        out = (M.query_sparse_attn(*leaves, s["idx"], case["bs"], kv_lens=s["lens"]),)
        grads = (s["go"],) if train else None
    if not train:
        return out
    return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, grads))


def _turn(x, c, s, pairs):
    """x [B, N, H, d] with each pair of dimensions turned by the angle of c = cos, s = sin [.., N, d/2]."""
    c, s = c.unsqueeze(-2), s.unsqueeze(-2)
    if pairs == "interleaved":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _angles(s, case):
    """Angles in 64 bits ([.., N, d/2], zero past the sections): far positions lose them in 32."""
    n = s["sections"]
    f = torch.cat([10000.0 ** (-torch.arange(m, device=DEV, dtype=F64) / m) for m in n])
    axis = torch.repeat_interleave(torch.arange(len(n), device=DEV), torch.tensor(n, device=DEV))
    ang = s["pos"].to(F64)[..., axis] * f
    return torch.nn.functional.pad(ang, (0, case["d"] // 2 - ang.shape[-1]))


def _plain_rope(s, case):
    ang = _angles(s, case)
    c, sn = ang.cos().float(), ang.sin().float()
    out = [_turn(s[n].float(), c, sn, case["pairs"]).to(s[n].dtype) for n in "qk"]
    if case["train"]:
        out += [_turn(s["g" + n].float(), c, -sn, case["pairs"]).to(s[n].dtype) for n in "qk"]
    return out


def _plain_norm(s, case):
    out, dx, dw = [], [], []
    for n in "qk":
        x, w = s[n].float(), s["w" + n]
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        h = x * r
        out.append(_turn(h * w, s["cos"], s["sin"], case["pairs"]).to(s[n].dtype))
        if case["train"]:
            u = _turn(s["g" + n].float(), s["cos"], -s["sin"], case["pairs"])
            dw.append((u * h).sum((0, 1, 2)))
            g = u * w
            dx.append((r * (g - h * (g * h).mean(-1, keepdim=True))).to(s[n].dtype))
    return out + dx + dw


def _plain_topk(s, case):
    # scores in 64 bits: they decide between values next to each other
    B, Nq, Hk, K = case["batch"], case["queries"], case["hk"], case["top"]
    q = s["q"].to(F64).view(B, Nq, Hk, -1, 64).sum(3).transpose(1, 2).contiguous()
    score = torch.matmul(q, s["kc"].to(F64).permute(0, 2, 3, 1).contiguous())          # [B, Hk, Nq, nb]
    if s["mask"] is not None:
        score.masked_fill_(~s["mask"][:, None, None, :], -math.inf)
    last = score.topk(K, dim=-1).values[..., -1:]
    tie = score == last
    keep = score > last
    keep |= tie & (tie.cumsum(-1, dtype=torch.int32) <= K - keep.sum(-1, keepdim=True))   # of equal ones the lowest
    idx = keep.nonzero()[:, -1].view(B, Hk, Nq, K)
    idx = torch.where(score.gather(-1, idx).isinf(), case["nb"], idx).sort(-1).values      # empty slots last
    return torch.where(idx == case["nb"], -1, idx).transpose(1, 2).contiguous()


def _plain_attn(s, case):
    B, Nq, Nk, Hq, Hk, bs, K = (case[n] for n in ("batch", "queries", "keys", "hq", "hk", "bs", "top"))
    nb = -(-Nk // bs)
    idx = s["idx"].transpose(1, 2)                                                       # [B, Hk, Nq, K]
    at = (idx[..., None] * bs + torch.arange(bs, device=DEV)).flatten(-2)                # keys of each row
    end = Nk if s["lens"] is None else s["lens"].view(B, 1, 1, 1)
    live = (at >= 0) & (at < end)
    pad = nb * bs - Nk
    kb, vb = (torch.nn.functional.pad(s[n], (0, 0, 0, 0, 0, pad)).float().transpose(1, 2).reshape(B * Hk * nb, bs * 64) for n in "kv")
    rows = (idx.clamp(min=0) + nb * torch.arange(B * Hk, device=DEV).view(B, Hk, 1, 1)).reshape(-1)
    q = s["q"].float().view(B, Nq, Hk, -1, 64).transpose(1, 2)                           # [B, Hk, Nq, G, 64]
    kg = kb.index_select(0, rows).view(B, Hk, Nq, K * bs, 64)
    x = torch.matmul(q, kg.transpose(-1, -2)) * 0.125
    x = x.masked_fill(~live.unsqueeze(-2), -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-30)                                     # rows without a key: zeros
    if not case["train"]:
        del kg, x, e
    vg = vb.index_select(0, rows).view(B, Hk, Nq, K * bs, 64)
    o = torch.matmul(p, vg)
    out = [o.transpose(1, 2).reshape(B, Nq, Hq, 64).to(BF16)]
    if case["train"]:
        g = s["go"].float().view(B, Nq, Hk, -1, 64).transpose(1, 2)
        ds = p * (torch.matmul(g, vg.transpose(-1, -2)) - (g * o).sum(-1, keepdim=True)) * 0.125
        out.append(torch.matmul(ds, kg).transpose(1, 2).reshape(B, Nq, Hq, 64).to(BF16))
        for left, right in ((ds, q), (p, g)):                                            # grad k, grad v
            part = torch.matmul(left.transpose(-1, -2), right).view(-1, bs * 64)
            whole = torch.zeros_like(kb).index_add_(0, rows, part)
            out.append(whole.view(B, Hk, nb * bs, 64)[:, :, :Nk].transpose(1, 2).to(BF16).contiguous())
    return out


# ------------------------------------------------------------------------------------ work

def work(case):
    kind = case["kind"]
    if kind in ("rope", "norm"):
        B, N, d = case["batch"], case["seq"], case["d"]
        one = (case["hq"] + case["hk"]) * d * B * N
        size = 4 if case["dtype"] == "f32" else 2
        passes = (5 if kind == "norm" else 4) if case["train"] else 2     # x, y and with a gradient g, dx (and x again)
        if kind == "norm":
            angles = 8 * N * (d // 2) * (2 if case["train"] else 1)
        else:
            angles = (8 if case["integers"] else 4) * N * (case["sections"].count(",") + 1) * (B if case["own_positions"] else 1)
        return dict(bytes=one * size * passes + angles, flops=one * (2 if case["train"] else 1) * (10 if kind == "norm" else 3))
    if kind == "topk":
        B, Nq, nb, Hq, Hk = (case[n] for n in ("batch", "queries", "nb", "hq", "hk"))
        return dict(bytes=2 * 64 * B * (Nq * Hq + nb * Hk) + 8 * B * Nq * Hk * case["top"], flops=2 * 64 * B * Nq * Hk * nb)
    B, Nq, Nk, Hq, Hk, bs, K = (case[n] for n in ("batch", "queries", "keys", "hq", "hk", "bs", "top"))
    qo, kv = 2 * 64 * B * Nq * Hq, 2 * 64 * B * Hk * min(Nk, Nq * K * bs)
    keys = min(Nk, K * bs)
    if case["train"]:   # q, k, v, grad of out and out in; out and three gradients out; two products and five
        return dict(bytes=5 * qo + 2 * kv + 4 * 64 * B * Hk * Nk + 8 * B * Nq * Hk * K, flops=2 * 64 * 7 * B * Nq * Hq * keys)
    return dict(bytes=2 * qo + 2 * kv + 8 * B * Nq * Hk * K, flops=2 * 64 * 2 * B * Nq * Hq * keys)


# ------------------------------------------------------------------------------------ float64

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "norm": _exact_norm, "topk": _exact_topk, "attn": _exact_attn}[case["kind"]](s, case)


def _spin(x, turn, pairs):
    """The pairs of x as complex numbers times ``turn`` [.., N, d/2]."""
    z = torch.complex(x[..., 0::2], x[..., 1::2]) if pairs == "interleaved" else torch.complex(*x.chunk(2, dim=-1))
    z = z * turn.unsqueeze(-2)
    return torch.view_as_real(z).flatten(-2) if pairs == "interleaved" else torch.cat([z.real, z.imag], dim=-1)


def _differentiated(s, leaves, outs):
    gs = [s["gq"].to(F64), s["gk"].to(F64)]
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, gs))


def _exact_rope(s, case):
    parts = []
    for a, n in enumerate(s["sections"]):
        for j in range(n):
            parts.append(s["pos"][..., a].to(F64) / 10000.0 ** (j / n))
    parts += [torch.zeros_like(parts[0])] * (case["d"] // 2 - len(parts))
    turn = torch.polar(torch.ones((), device=DEV, dtype=F64), torch.stack(parts, dim=-1))
    leaves = [s[n].to(F64).requires_grad_(case["train"]) for n in "qk"]
    outs = [_spin(x, turn, case["pairs"]) for x in leaves]
    return _differentiated(s, leaves, outs) if case["train"] else outs


def _exact_norm(s, case):
    turn = torch.complex(s["cos"].to(F64), s["sin"].to(F64))
    leaves = [s[n].to(F64).requires_grad_(case["train"]) for n in ("q", "k", "wq", "wk")]
    outs = [_spin(x / ((x * x).sum(-1, keepdim=True) / case["d"] + 1e-6).sqrt() * w, turn, case["pairs"])
            for x, w in zip(leaves[:2], leaves[2:])]
    return _differentiated(s, leaves, outs) if case["train"] else outs


def _exact_topk(s, case):
    """The first K of a stable sort of the float64 scores, one kv head at a time."""
    G, K, nb = case["hq"] // case["hk"], case["top"], case["nb"]
    q, kc = s["q"].to(F64), s["kc"].to(F64)
    out = torch.empty(case["batch"], case["queries"], case["hk"], K, device=DEV, dtype=torch.int64)
    for h in range(case["hk"]):
        score = sum(torch.matmul(q[:, :, h * G + g], kc[:, :, h].transpose(1, 2).contiguous()) for g in range(G))
        ok = torch.ones_like(score, dtype=torch.bool) if s["mask"] is None else s["mask"][:, None, :].expand_as(score)
        order = torch.where(ok, score, -math.inf).sort(dim=-1, descending=True, stable=True).indices[..., :K]
        got = ok.gather(-1, order)
        order = torch.where(got, order, nb).sort(-1).values
        out[:, :, h] = torch.where(order == nb, -1, order)
    return out


def _exact_attn(s, case):
    """Dense scores of a run of queries against every key, with the selection as a mask."""
    B, Nq, Nk, Hq, Hk, bs = (case[n] for n in ("batch", "queries", "keys", "hq", "hk", "bs"))
    G, nb = Hq // Hk, -(-Nk // bs)
    o, dq = (torch.zeros(B, Nq, Hq, 64, device=DEV, dtype=F64) for _ in range(2))
    dk, dv = (torch.zeros(B, Nk, Hk, 64, device=DEV, dtype=F64) for _ in range(2))
    run_of = max(1, (1 << 28) // (G * Nk))
    for b in range(B):
        end = Nk if s["lens"] is None else int(s["lens"][b])
        for h in range(Hk):
            k, v = s["k"][b, :, h].to(F64), s["v"][b, :, h].to(F64)
            for i in range(0, Nq, run_of):
                j = min(Nq, i + run_of)
                idx = s["idx"][b, i:j, h]
                member = torch.zeros(j - i, nb + 1, device=DEV, dtype=torch.bool)
                member.scatter_(1, torch.where(idx < 0, nb, idx), True)
                ok = member[:, :nb].repeat_interleave(bs, dim=1)[:, :Nk]
                ok = ok & (torch.arange(Nk, device=DEV) < end)
                at = slice(h * G, h * G + G)
                q = s["q"][b, i:j, at].to(F64)
                x = (q.reshape(-1, 64) @ k.t()).view(j - i, G, Nk) / 8
                x = x.masked_fill_(~ok[:, None, :], -math.inf)
                any_ = ok.any(-1)[:, None, None]
                p = torch.where(any_, torch.softmax(x, dim=-1), 0.0).view(-1, Nk)
                o[b, i:j, at] = (p @ v).view(j - i, G, 64)
                if case["train"]:
                    go = s["go"][b, i:j, at].to(F64).reshape(-1, 64)
                    dp = go @ v.t()
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / 8
                    dq[b, i:j, at] = (ds @ k).view(j - i, G, 64)
                    dk[b, :, h] += ds.t() @ q.reshape(-1, 64)
                    dv[b, :, h] += p.t() @ go
    return [o, dq, dk, dv] if case["train"] else [o]
