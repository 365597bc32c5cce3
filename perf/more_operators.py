"""Cases of the 8-bit key/value cache and the attention over it, with their plain forms and their values in float64.

* ``write``: ``kv_cache_write`` and ``kv_cache_read``, tokens quantised as they are written, with a
  scale for each block of tokens and kv head, and read back;
* ``read``: ``kv_cache_read`` alone, a window of a cache;
* ``step``: one token written for each member, then ``cache_attn`` of one query over all of the cache;
* ``dense``: ``cache_attn`` of queries over every token of a cache;
* ``sparse``: ``cache_attn`` of queries over key blocks of their own.

Sizes are those of the HEALPix sequences of the model (768 tokens at nside 8 to 196608 at nside 128),
its heads (12/3, 16/4, 20/5), its 24 ensemble members and its selection blocks (64 and 128 tokens),
with odd counts between.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TYPES = {"bf16": BF16, "f32": F32}
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def _write(name, seq, batch, hk, bs, codes, dtype="bf16", ragged=False, stacked=False):
    return dict(name=name, kind="write", seq=seq, batch=batch, hk=hk, bs=bs, codes=codes, dtype=dtype, ragged=ragged,
                stacked=stacked)


def _read(name, keys, start, count, batch, hk, bs, codes, dtype="bf16"):
    return dict(name=name, kind="read", keys=keys, start=start, count=count, batch=batch, hk=hk, bs=bs, codes=codes, dtype=dtype)


def _step(name, keys, batch, hq, hk, bs, codes):
    return dict(name=name, kind="step", keys=keys, batch=batch, hq=hq, hk=hk, bs=bs, codes=codes)


def _dense(name, queries, keys, batch, hq, hk, bs, codes, ragged=False):
    return dict(name=name, kind="dense", queries=queries, keys=keys, batch=batch, hq=hq, hk=hk, bs=bs, codes=codes, ragged=ragged)


def _sparse(name, queries, keys, batch, hq, hk, bs, top, codes, scattered=False, ragged=False):
    return dict(name=name, kind="sparse", queries=queries, keys=keys, batch=batch, hq=hq, hk=hk, bs=bs, top=top, codes=codes,
                scattered=scattered, ragged=ragged)


def listed():
    return [
        # the coarsest state of one member: the calls' fixed cost
        _write("write_nside8", 768, 1, 5, 64, "int8"),
        # fp32 observations appended to padded histories of three members, from the middle of blocks
        _write("write_ragged_f32", 10007, 3, 4, 128, "e4m3", dtype="f32", ragged=True),
        # the widest stage's keys and values of all members, views of the stacked projection's output
        _write("write_nside64_b24", 49152, 24, 3, 64, "int8", stacked=True),
        # a region of one member's state, an odd run from the middle of a block
        _read("read_region", 49152, 20011, 2995, 1, 3, 64, "e4m3"),
        # the finest state back in fp32
        _read("read_nside128_f32", 196608, 0, 196608, 1, 3, 128, "int8", dtype="f32"),
        # a track of each member grows by one point, which then reads its whole past
        _step("step_track_b24", 12288, 24, 16, 4, 64, "int8"),
        # one point against every token of nside 128
        _dense("dense_one_point", 1, 196608, 1, 12, 3, 128, "e4m3"),
        # a few stations against the states of two members, of unequal lengths
        _dense("dense_stations_b2", 37, 49152, 2, 12, 3, 64, "int8", ragged=True),
        # every token of nside 32 reads all of the finer mesh
        _dense("dense_nside32_on_64", 12288, 49152, 1, 12, 3, 64, "int8"),
        # one point, its own 16 blocks of nside 128
        _sparse("sparse_one_point", 1, 196608, 1, 12, 3, 128, 16, "int8"),
        # scattered stations in no order, padded batch, some rows without a block
        _sparse("sparse_stations_b2", 10007, 49152, 2, 12, 3, 64, 16, "e4m3", scattered=True, ragged=True),
        # every token of nside 64 reads its own blocks
        _sparse("sparse_nside64", 49152, 49152, 1, 12, 3, 64, 16, "int8"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    g = rng.choice((4, 4, 4, 2, 1, 3, 8, 16))
    hk = rng.randint(1, 5 if g <= 4 else 2)
    return g * hk, hk


def draw(rng):
    kind = rng.choice(("write", "write", "read", "step", "dense", "dense", "sparse", "sparse"))
    codes, bs = rng.choice(("int8", "e4m3")), rng.choice((64, 64, 128, 256))
    hq, hk = _heads(rng)
    if kind == "write":
        dtype = rng.choice(("bf16", "bf16", "f32"))
        most = 24 * 49152 * 3 // hk // (2 if dtype == "f32" else 1)
        seq = _log_int(rng, 1, 196608)
        batch = _log_int(rng, 1, max(1, min(24, most // seq)))
        ragged = seq * batch * hk < 1 << 21 and rng.random() < 0.6
        c = _write("", seq, batch, hk, bs, codes, dtype, ragged, rng.random() < 0.5)
    elif kind == "read":
        keys = _log_int(rng, 64, 196608)
        start = rng.choice((0, rng.randrange(keys)))
        count = rng.choice((keys - start, rng.randint(1, keys - start)))
        batch = _log_int(rng, 1, max(1, min(24, 24 * 49152 * 3 // (2 * hk * keys))))
        c = _read("", keys, start, count, batch, hk, bs, codes, rng.choice(("bf16", "bf16", "f32")))
    elif kind == "step":
        keys = _log_int(rng, 2, 100000)
        batch = _log_int(rng, 1, max(1, min(24, 24 * 12288 * 4 // (hk * keys))))
        c = _step("", keys, batch, hq, hk, bs, codes)
    elif kind == "dense":
        keys = _log_int(rng, 20, 196608)
        most = 12288 * 49152 * 12 // (hq * keys)
        queries = _log_int(rng, 1, max(1, min(12288, most)))
        batch = _log_int(rng, 1, max(1, min(8, most // queries)))
        c = _dense("", queries, keys, batch, hq, hk, bs, codes, rng.random() < 0.5)
    else:
        keys = _log_int(rng, 1000, 196608)
        top = rng.randint(1, min(1536 // bs, -(-keys // bs)))
        most = 49152 * 12 * 64 * 16
        queries = _log_int(rng, 1, min(49152, most // (hq * bs * top)))
        batch = _log_int(rng, 1, max(1, min(4, most // (hq * bs * top * queries))))
        c = _sparse("", queries, keys, batch, hq, hk, bs, top, codes, rng.random() < 0.3, rng.random() < 0.4)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(3000017 + 7919 * int(seed))


def _field(gen, at, channels):
    """A smooth random field of the position ``at`` in [0, 1): waves of wavelengths from the whole
    sequence down to a hundredth of it, long ones strongest, so that neighbours are alike."""
    f = torch.exp(torch.rand(24, generator=gen, device=DEV) * math.log(100.0))
    amp = torch.randn(24, channels, generator=gen, device=DEV) / f.sqrt()[:, None]
    ph = 2 * math.pi * torch.rand(24, generator=gen, device=DEV)
    return torch.cos(2 * math.pi * at[:, None] * f + ph) @ (amp * (2.0 / (1.0 / f).sum().sqrt()))


def _tokens(gen, batch, n, hk, dtype, stacked=False):
    """Keys and values of a mesh: a smooth field with noise, some channels larger than others."""
    at = (torch.arange(n, device=DEV) + 0.5) / n
    kv = torch.empty(batch, n, 2 * hk, 64, device=DEV, dtype=dtype)
    size = torch.exp(0.5 * torch.randn(2 * hk, 64, generator=gen, device=DEV))
    for b in range(batch):
        x = _field(gen, at, 2 * hk * 64).view(n, 2 * hk, 64) + 0.3 * torch.randn(n, 2 * hk, 64, generator=gen, device=DEV)
        kv[b] = x * size
    k, v = kv[:, :, :hk], kv[:, :, hk:]
    return (k, v) if stacked else (k.contiguous(), v.contiguous())


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
    return torch.stack(q).to(BF16), torch.stack(k)


def _inputs(case, seed):
    gen = _gen(seed)
    kind, B, Hk, bs = case["kind"], case["batch"], case["hk"], case["bs"]
    s = dict(case=case)
    if kind == "write":
        N = case["seq"]
        s["k"], s["v"] = _tokens(gen, B, N, Hk, TYPES[case["dtype"]], case["stacked"])
        s["start"], s["count"], s["keys"] = None, None, N
        if case["ragged"]:   # histories of up to a third of the run, and runs of unequal lengths
            past = N // 3 + 1
            s["hk"], s["hv"] = _tokens(gen, B, past, Hk, TYPES[case["dtype"]])
            s["start"] = torch.randint(0, past + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
            s["count"] = torch.randint(N // 2, N + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
            s["keys"] = past + N
        return s
    keys = case["keys"]
    s["keys"] = keys
    if kind in ("read", "step"):
        s["hk"], s["hv"] = _tokens(gen, B, keys, Hk, BF16)
        if kind == "step":   # the tracks have come to different lengths
            s["start"] = torch.randint(keys // 2, keys, (B,), generator=gen, device=DEV, dtype=torch.int32)
            s["lens"] = s["start"] + 1
            s["k"], s["v"] = _tokens(gen, B, 1, Hk, BF16)
            s["q"] = torch.randn(B, 1, case["hq"], 64, generator=gen, device=DEV).to(BF16)
        return s
    Nq, nb = case["queries"], -(-keys // bs)
    at = (torch.arange(Nq, device=DEV) + 0.5) / Nq
    if case.get("scattered") or Nq < 64:
        at = torch.rand(Nq, generator=gen, device=DEV)
    s["q"], kc = _pooled(case, gen, Nq, nb, at)
    lens = torch.full((B,), keys, device=DEV, dtype=torch.int32)
    if case["ragged"]:   # a padded batch: the sequences end anywhere, inside a block too
        lens = torch.randint(max(1, keys // 3), keys + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
    s["lens"] = lens if case["ragged"] else None
    s["hk"] = kc.repeat_interleave(bs, dim=1)[:, :keys]
    s["hk"] = (s["hk"] + torch.randn(s["hk"].shape, generator=gen, device=DEV)).to(BF16)
    s["hv"] = torch.randn(s["hk"].shape, generator=gen, device=DEV).to(BF16)
    if kind == "dense":
        return s
    live = torch.arange(nb, device=DEV) * bs < lens[:, None]
    mean = s["q"].float().view(B, Nq, Hk, -1, 64).mean(3).transpose(1, 2)
    score = torch.matmul(mean, kc.permute(0, 2, 3, 1).contiguous()).masked_fill_(~live[:, None, None, :], -math.inf)
    best = score.topk(case["top"], dim=-1)
    idx = torch.where(best.values.isinf(), -1, best.indices).transpose(1, 2).contiguous()
    if case["ragged"]:   # rows and slots without a block
        idx.masked_fill_((torch.rand(B, Nq, generator=gen, device=DEV) < 0.05)[:, :, None, None], -1)
        idx.masked_fill_(torch.rand(idx.shape, generator=gen, device=DEV) < 0.05, -1)
    s["idx"] = idx
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        import mosaic_amd as M

        s["cache"] = M.KVCache(case["batch"], s["keys"], case["hk"], block_size=case["bs"], dtype=CODES[case["codes"]][0], device=DEV)
        if "hk" in s:
            M.kv_cache_write(s["cache"], s["hk"], s["hv"])
    else:
        _held(s, case)
    for name in ("hk", "hv"):
        s.pop(name, None)
    return s


def _held(s, case):
    """The cache as plain tensors: codes [B, keys in whole blocks, Hk, 64] and scales [B, blocks, Hk]."""
    B, Hk, bs = case["batch"], case["hk"], case["bs"]
    nb, kind = -(-s["keys"] // bs), CODES[case["codes"]][0]
    for name in "kv":
        codes = torch.zeros(B, nb * bs, Hk, 64, device=DEV, dtype=kind)
        scale = torch.zeros(B, nb, Hk, device=DEV)
        if "h" + name in s:
            x = s["h" + name]
            for b in range(B):   # (a member at a time: the 32-bit values of all of them are many)
                new = torch.arange(nb * bs, device=DEV) < x.shape[1]
                c, scale[b:b + 1] = _quantise(codes[b:b + 1], scale[b:b + 1], x[b:b + 1], new[None], torch.zeros_like(new)[None], case)
                codes[b] = c[0].to(kind)
        s[name + "codes"], s[name + "scale"] = codes, scale


# ------------------------------------------------------------------------------------ one pass

def run(s):
    case = s["case"]
    return (_own if own else _plain)(s, case)


def _own(s, case):
    import mosaic_amd as M

    kind, cache = case["kind"], s["cache"]
    if kind == "write":
        M.kv_cache_write(cache, s["k"], s["v"], start=0 if s["start"] is None else s["start"], counts=s["count"])
        return M.kv_cache_read(cache, dtype=TYPES[case["dtype"]]) + (cache.k_scale, cache.v_scale, cache.k_mean)
    if kind == "read":
        return M.kv_cache_read(cache, case["start"], case["count"], dtype=TYPES[case["dtype"]])
    if kind == "step":
        M.kv_cache_write(cache, s["k"], s["v"], start=s["start"])
        out = M.cache_attn(s["q"], cache, kv_lens=s["lens"])
        return out, cache.k_scale, cache.v_scale, cache.k_mean
    return M.cache_attn(s["q"], cache, s.get("idx"), kv_lens=s["lens"])


def _blocks(x, bs):
    return x.unflatten(1, (x.shape[1] // bs, bs))


def _quantise(codes, scale, x, new, kept, case):
    """Codes (in 32 bits) and scales of a cache after x, one value for each True of ``new`` [B, keys] in
    order, is written; ``kept``: earlier tokens of the blocks written to, the others there become 0."""
    bs, (kind, top) = case["bs"], CODES[case["codes"]]
    old = codes.float()
    whole = new.shape == x.shape[:2] and bool(new.all())
    at = (new.cumsum(1) - 1).clamp(min=0, max=x.shape[1] - 1)
    y = x.float() if whole else x.float().gather(1, at[:, :, None, None].expand(-1, -1, *x.shape[2:])) * new[:, :, None, None]
    a = _blocks(y, bs).abs().amax((2, 4))                                           # [B, blocks, Hk]
    a = torch.where(a < 2.0 ** -100, 0.0, a)
    s_new = (a.double() / top).float()
    has = _blocks(kept, bs).any(2)[:, :, None]
    s_new = torch.where(has, torch.maximum(s_new, scale), s_new)
    touched = _blocks(new, bs).any(2)[:, :, None].expand_as(scale)
    s_new = torch.where(touched, torch.where(a.isfinite(), s_new, math.nan), scale)
    # quotients in 64 bits: which code is nearest is decided next to a border
    by = torch.where(s_new > 0, s_new, 1.0).repeat_interleave(bs, dim=1)[..., None].double()
    z = torch.where(kept[:, :, None, None], old.double() * scale.repeat_interleave(bs, dim=1)[..., None], y.double()) / by
    if case["codes"] == "e4m3":
        # to 32 bits by way of the odd neighbour, so that the second rounding goes as one would
        f = z.clamp(-top, top).float()
        off = (f.double() != z) & ((f.view(torch.int32) & 1) == 0) & (f.abs() < top)
        z = torch.where(off, torch.nextafter(f, torch.where(z > f, math.inf, -math.inf).float()), f).to(kind).float()
    else:
        z = z.round().clamp(-top, top).float()
    out = torch.where(touched.repeat_interleave(bs, dim=1)[..., None], z, old)
    return torch.where(out.isfinite(), out, 0.0), s_new


def _written(s, case):
    """Codes, scales and the keys' block means after the write, a name and a member at a time."""
    B, Hk, bs = case["batch"], case["hk"], case["bs"]
    nk = s["kcodes"].shape[1]
    start = torch.zeros(B, 1, device=DEV, dtype=torch.int64) if s["start"] is None else s["start"][:, None].long()
    n = s["k"].shape[1]
    end = start + (n if s.get("count") is None else s["count"][:, None])
    at = torch.arange(nk, device=DEV)
    new = (at >= start) & (at < end)
    kept = (at < start) & (at >= start // bs * bs) & (end > start)
    res = {name: [[], []] for name in "kv"}
    for name in "kv":
        for b in range(B):
            one = slice(b, b + 1)
            c, sc = _quantise(s[name + "codes"][one], s[name + "scale"][one], s[name][one], new[one], kept[one], case)
            res[name][0].append(c.to(s[name + "codes"].dtype))
            res[name][1].append(sc)
    (kc, ks), (vc, vs) = ([torch.cat(x) for x in res[name]] for name in "kv")
    return kc, ks, vc, vs, start, end


def _block_means(s, case, kc, ks, start, end):
    bs = case["bs"]
    edge = torch.arange(ks.shape[1], device=DEV) * bs
    left = (end - edge).clamp(min=0, max=bs)                                        # tokens up to the end of the write
    touched = (edge + bs > start) & (left > 0) & (end > start)
    n = torch.where(touched, left, (_past(s, case) - edge).clamp(min=0, max=bs)).clamp(min=1)
    sums = torch.cat([_blocks(kc[b:b + 1].float(), bs).sum(2) for b in range(kc.shape[0])])
    return (sums * ks[..., None] / n[:, :, None, None].float()).to(BF16)


def _past(s, case):
    """Tokens that the cache held before the write."""
    if case["kind"] == "step":
        return s["keys"]
    return case["seq"] // 3 + 1 if case["ragged"] else 0


def _values(codes, scale, bs, dtype, at=slice(None)):
    return (codes[:, at].float() * scale.repeat_interleave(bs, dim=1)[:, at, :, None]).to(dtype)


def _plain(s, case):
    kind, bs = case["kind"], case["bs"]
    if kind == "read":
        at = slice(case["start"], case["start"] + case["count"])
        return tuple(_values(s[n + "codes"], s[n + "scale"], bs, TYPES[case["dtype"]], at) for n in "kv")
    if kind in ("write", "step"):
        kc, ks, vc, vs, start, end = _written(s, case)
        state = (ks, vs, _block_means(s, case, kc, ks, start, end))
        if kind == "step":
            return (_attend_all(s["q"], kc, ks, vc, vs, s["lens"], s["keys"], case),) + state
        at = slice(0, s["keys"])
        return tuple(torch.cat([_values(c[b:b + 1], x[b:b + 1], bs, TYPES[case["dtype"]], at) for b in range(c.shape[0])])
                     for c, x in ((kc, ks), (vc, vs))) + state
    held = (s["kcodes"], s["kscale"], s["vcodes"], s["vscale"])
    if kind == "dense":
        return _attend_all(s["q"], *held, s["lens"], s["keys"], case)
    return _attend_blocks(s["q"], *held, s["lens"], s["idx"], s["keys"], case)


def _attend_all(q, kc, ks, vc, vs, lens, keys, case):
    B, Nq, Hq, _ = q.shape
    Hk, bs = case["hk"], case["bs"]
    kT = _values(kc, ks, bs, F32).permute(0, 2, 3, 1).contiguous()                  # [B, Hk, 64, keys]
    v = _values(vc, vs, bs, F32).transpose(1, 2).contiguous()
    live = torch.arange(kT.shape[-1], device=DEV) < (keys if lens is None else lens.view(B, 1, 1, 1))
    some = max(1, (1 << 29) // (B * Hq * kT.shape[-1]))
    out = []
    for i in range(0, Nq, some):
        part = q[:, i:i + some].float().view(B, -1, Hk, Hq // Hk, 64).transpose(1, 2).reshape(B, Hk, -1, 64)
        x = (torch.matmul(part, kT) * 0.125).masked_fill_(~live, -math.inf)
        e = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
        out.append(o.view(B, Hk, -1, Hq // Hk, 64).transpose(1, 2).reshape(B, -1, Hq, 64).to(BF16))
    return torch.cat(out, dim=1)


def _attend_blocks(q, kc, ks, vc, vs, lens, idx, keys, case):
    B, Nq, Hq, _ = q.shape
    Hk, bs, K = case["hk"], case["bs"], case["top"]
    nb = ks.shape[1]
    kb, vb = (_values(c, x, bs, F32).transpose(1, 2).reshape(B * Hk * nb, bs * 64) for c, x in ((kc, ks), (vc, vs)))
    end = keys if lens is None else lens.view(B, 1, 1, 1)
    some = max(1, (1 << 31) // (B * Hk * K * bs * 64))
    out = []
    for i in range(0, Nq, some):
        at = idx[:, i:i + some].transpose(1, 2)                                      # [B, Hk, n, K]
        n = at.shape[2]
        tok = (at[..., None] * bs + torch.arange(bs, device=DEV)).flatten(-2)
        live = ((tok >= 0) & (tok < end)).unsqueeze(-2)
        rows = (at.clamp(min=0) + nb * torch.arange(B * Hk, device=DEV).view(B, Hk, 1, 1)).reshape(-1)
        part = q[:, i:i + some].float().view(B, n, Hk, -1, 64).transpose(1, 2)
        x = torch.matmul(part, kb.index_select(0, rows).view(B, Hk, n, K * bs, 64).transpose(-1, -2)) * 0.125
        x = x.masked_fill_(~live, -math.inf)
        e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
        p = e / e.sum(-1, keepdim=True).clamp(min=1e-30)                             # rows without a key: zeros
        o = torch.matmul(p, vb.index_select(0, rows).view(B, Hk, n, K * bs, 64))
        out.append(o.transpose(1, 2).reshape(B, n, Hq, 64).to(BF16))
    return torch.cat(out, dim=1)


# ------------------------------------------------------------------------------------ work

def work(case):
    kind, B, Hk, bs = case["kind"], case["batch"], case["hk"], case["bs"]
    size = 4 if case.get("dtype") == "f32" else 2
    if kind == "write":   # values in and codes out; codes in and values out
        n = 2 * 64 * B * Hk * case["seq"]
        back = n * 7 // 6 if case["ragged"] else n     # (the histories are read back too: half of a third in the mean)
        return dict(bytes=n * (size + 1) + back * (size + 1), flops=4 * n)
    if kind == "read":
        n = 2 * 64 * B * Hk * case["count"]
        return dict(bytes=n * (size + 1), flops=n)
    Nq = case.get("queries", 1)
    qo, Hq = 4 * 64 * B * Nq * case["hq"], case["hq"]
    keys = case["keys"]
    if kind == "step":    # tracks of three quarters of the cache in the mean
        keys = keys * 3 // 4
    elif case["ragged"]:
        keys = keys * 2 // 3
    seen = keys if kind != "sparse" else min(keys, case["top"] * bs)
    held = keys if kind != "sparse" else min(keys, Nq * case["top"] * bs)
    idx = 8 * B * Nq * Hk * case["top"] if kind == "sparse" else 0
    return dict(bytes=qo + 2 * 64 * B * Hk * held + 8 * B * Hk * -(-held // bs) + idx, flops=2 * 2 * 64 * B * Nq * Hq * seen)


# ------------------------------------------------------------------------------------ float64

def _steps(z, case):
    """The nearest value of the code's grid, ties to even: whole numbers, or four significant bits down to 2^-9."""
    if case["codes"] == "int8":
        return torch.round(z).clamp(-127, 127)
    _, e = torch.frexp(z)
    unit = torch.ldexp(torch.ones_like(z), (e - 4).clamp(min=-9))
    return (torch.round(z / unit) * unit).clamp(-448, 448)


def _exact_write(s, case):
    """Values [B, keys, Hk, 64] and scales after the write, block by block."""
    B, Hk, bs = case["batch"], case["hk"], case["bs"]
    top = CODES[case["codes"]][1]
    start = [0] * B if s["start"] is None else s["start"].tolist()
    count = [s["k"].shape[1]] * B if s.get("count") is None else s["count"].tolist()
    out = []
    for name in "kv":
        scale = s[name + "scale"].to(F64)
        nb = scale.shape[1]
        codes = s[name + "codes"].to(F32).to(F64).view(B, nb, bs, Hk, 64)
        for b in range(B):
            i, j = start[b], start[b] + count[b]
            if j == i:
                continue
            first, last = i // bs, (j - 1) // bs
            x = torch.zeros((last + 1 - first) * bs, Hk, 64, device=DEV, dtype=F64)
            x[i - first * bs:j - first * bs] = s[name][b, :count[b]].to(F64)
            x = x.view(-1, bs, Hk, 64)
            sc = (x.abs().amax((1, 3)) / top).to(F32).to(F64)     # (a scale is a 32-bit number)
            if i % bs:
                old = codes[b, first, :i % bs] * scale[b, first, :, None]
                sc[0] = torch.maximum(sc[0], scale[b, first])
                x[0, :i % bs] = old
            codes[b, first:last + 1] = _steps(torch.where(sc[:, None, :, None] > 0, x / sc[:, None, :, None], 0.0), case)
            scale[b, first:last + 1] = sc
        out += [codes, scale]
    return out, start, count


def _exact_means(s, case, codes, scale, start, count):
    B, bs = case["batch"], case["bs"]
    nb = scale.shape[1]
    had = _past(s, case)
    n = torch.zeros(B, nb, 1, 1, device=DEV, dtype=F64)
    for b in range(B):
        for j in range(nb):
            n[b, j] = min(bs, max(0, had - j * bs))
        if count[b]:
            end = start[b] + count[b]
            for j in range(start[b] // bs, (end - 1) // bs + 1):
                n[b, j] = min(bs, end - j * bs)
    return codes.sum(2) * scale[..., None] / n.clamp(min=1)


def exact(case, seed):
    s = _inputs(case, seed)
    _held(s, case)
    kind, bs = case["kind"], case["bs"]
    if kind in ("write", "step"):
        if kind == "write" and case["batch"] * case["seq"] * case["hk"] > 1 << 21:
            return None     # (a block at a time in 64 bits, with its copies: too long)
        (kc, ks, vc, vs), start, count = _exact_write(s, case)
        state = [ks, vs, _exact_means(s, case, kc, ks, start, count)]
        k, v = ((c * x[:, :, None, :, None]).flatten(1, 2)[:, :s["keys"]] for c, x in ((kc, ks), (vc, vs)))
        if kind == "write":
            return [k, v] + state
        return [_exact_attn(s, case, k, v)] + state
    k, v = ((s[n + "codes"].to(F32).to(F64).unflatten(1, (-1, bs)) * s[n + "scale"].to(F64)[:, :, None, :, None]).flatten(1, 2)[:, :s["keys"]]
            for n in "kv")
    if kind == "read":
        return [x[:, case["start"]:case["start"] + case["count"]] for x in (k, v)]
    return _exact_attn(s, case, k, v)


def _exact_attn(s, case, k, v):
    """Scores of a run of queries against every key, with the selection as a mask, a kv head at a time."""
    B, Nq, Hq, Hk, bs, keys = case["batch"], s["q"].shape[1], case["hq"], case["hk"], case["bs"], s["keys"]
    G, nb = Hq // Hk, -(-keys // bs)
    o = torch.zeros(B, Nq, Hq, 64, device=DEV, dtype=F64)
    run_of = max(1, (1 << 28) // (G * keys))
    for b in range(B):
        end = keys if s["lens"] is None else int(s["lens"][b])
        for h in range(Hk):
            kh, vh = k[b, :, h].contiguous(), v[b, :, h].contiguous()
            for i in range(0, Nq, run_of):
                j = min(Nq, i + run_of)
                ok = (torch.arange(keys, device=DEV) < end).expand(j - i, keys)
                if case["kind"] == "sparse":
                    idx = s["idx"][b, i:j, h]
                    member = torch.zeros(j - i, nb + 1, device=DEV, dtype=torch.bool)
                    member.scatter_(1, torch.where(idx < 0, nb, idx), True)
                    ok = ok & member[:, :nb].repeat_interleave(bs, dim=1)[:, :keys]
                at = slice(h * G, h * G + G)
                x = (s["q"][b, i:j, at].to(F64).reshape(-1, 64) @ kh.t()).view(j - i, G, keys) / 8
                x = x.masked_fill_(~ok[:, None, :], -math.inf)
                p = torch.where(ok.any(-1)[:, None, None], torch.softmax(x, dim=-1), 0.0).view(-1, keys)
                o[b, i:j, at] = (p @ vh).view(j - i, G, 64)
    return o
