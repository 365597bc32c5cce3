"""A key/value cache in 8 bits in float64, token by token: what ``KVCache`` holds after a series of writes,
and the attention over it with a bound on what a kernel may be off by."""

import math

import torch

F64 = torch.float64
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def nearest_code(z, dtype):
    """Ties to even: whole numbers, or four significant bits down to 2^-9."""
    if dtype == torch.int8:
        return torch.round(z).clamp(-127, 127)
    _, e = torch.frexp(z)
    unit = torch.ldexp(torch.ones_like(z), (e - 4).clamp(min=-9))
    return (torch.round(z / unit) * unit).clamp(-448, 448)


class Model:
    def __init__(self, batch, capacity, heads, bs, dtype):
        nb = -(-capacity // bs)
        self.bs, self.dtype, self.capacity = bs, dtype, capacity
        self.codes = [torch.zeros(batch, nb * bs, heads, 64, dtype=F64) for _ in range(2)]
        self.scale = [torch.zeros(batch, nb, heads, dtype=F64) for _ in range(2)]
        self.mean = torch.zeros(batch, nb, heads, 64, dtype=F64)

    def write(self, k, v, start, counts=None):
        B, n, H, _ = k.shape
        for b in range(B):
            at = int(start[b]) if isinstance(start, torch.Tensor) else start
            c = n if counts is None else min(max(int(counts[b]), 0), n)
            first, last = max(at, 0), min(at + c, self.capacity)
            if last <= first:
                continue
            for j in range(first // self.bs, (last - 1) // self.bs + 1):
                t0 = j * self.bs
                lo, hi = max(first, t0), min(last, t0 + self.bs)
                for h in range(H):
                    for i, x in enumerate((k, v)):
                        self._block(i, b, j, h, x[b, lo - at:hi - at, h].to(F64), lo - t0)
                    held = self.codes[0][b, t0:hi, h].sum(0) * self.scale[0][b, j, h]
                    self.mean[b, j, h] = held / (hi - t0)

    def _block(self, i, b, j, h, x, kept):
        t0 = j * self.bs
        codes, before = self.codes[i][b, t0:t0 + self.bs, h], self.scale[i][b, j, h].clone()
        a = x.abs().amax()
        s = a / TOP[self.dtype] if not a < 2.0 ** -100 else torch.zeros((), dtype=F64)
        s = s.to(torch.float32).to(F64)                # a scale is a float32
        if kept:
            s = torch.maximum(s, before)               # (a NaN wins)
        old = codes[:kept].clone()
        codes.zero_()
        if not torch.isfinite(a) or torch.isnan(s):
            s = torch.full((), math.nan, dtype=F64)
        elif s > 0:
            codes[:kept] = nearest_code(old * before / s, self.dtype)
            codes[kept:kept + x.shape[0]] = nearest_code(x / s, self.dtype)
        self.scale[i][b, j, h] = s

    def values(self, i):
        """[B, capacity, H, 64] as float32: one rounding of the exact product"""
        full = self.codes[i] * self.scale[i].repeat_interleave(self.bs, dim=1)[..., None]
        return full[:, :self.capacity].to(torch.float32)


def attention(q, k, v, scale, lens=None, idx=None, bs=64):
    """(output, bound) in float64 of q [B, Nq, Hq, 64] (bfloat16 values) over k, v [B, Nk, Hk, 64].

    The bound of an element o = sum w_u v_u: the output's rounding (2^-8 |o|); the weights' rounding to bf16,
    shared by numerator and denominator (2^-8 of sum w |v - o|, and 2^-8 of that again); scores in fp32, each
    off by e (64 products, their sum and the factors: 72 roundings of 2^-24 of sum |q k| scale, and 2^-22 of
    |score| for its place in the exponent) which weigh 2 e sum w |v - o|; fp32 sums over the keys, 2^-24 each of
    sum w |v|, and 8 more for products with the scales, exponentials and joins; and weights
    that leave fp32 (and bf16): the reference of the scores, in powers of two, is 0 or up to 80 above the row's largest, and
    scales of values may take 20 more, so that what lies 2^-106 below the reference may be zeros.
    """
    q, k, v = (t.to(F64) for t in (q, k, v))
    B, Nq, Hq, d = q.shape
    Nk, Hk = k.shape[1:3]
    G = Hq // Hk
    out = torch.zeros(B, Nq, Hq, d, dtype=F64)
    tol = torch.zeros_like(out)
    for b in range(B):
        end = Nk if lens is None else min(max(int(lens[b]), 0), Nk)
        for h in range(Hk):
            ok = (torch.arange(Nk) < end).expand(Nq, Nk)
            if idx is not None:
                nb = -(-Nk // bs)
                member = torch.zeros(Nq, nb + 1, dtype=torch.bool)
                i = idx[b, :, h]
                member.scatter_(1, torch.where((i < 0) | (i >= nb), nb, i).to(torch.int64), True)
                ok = ok & member[:, :nb].repeat_interleave(bs, dim=1)[:, :Nk]
            some = ok.any(-1)[:, None]
            used = ok.any(0)
            kk, vv = k[b, used, h], v[b, used, h]      # (what no row has does not reach any)
            okk = ok[:, used]
            for g in range(h * G, h * G + G):
                x = q[b, :, g] @ kk.t() * scale
                p = torch.softmax(x.masked_fill(~okk, -math.inf), dim=-1)
                p = torch.where(okk & some, p, 0.0)
                o = p @ vv
                off = (p @ (vv * vv) - o * o).clamp(min=0).sqrt()      # not below sum w |v - o|, by Jensen
                size = p @ vv.abs()
                e = 72 * 2.0 ** -24 * scale * (q[b, :, g].abs() @ kk.abs().t()) + 2.0 ** -22 * x.abs()
                e = torch.where(okk, e, 0.0).amax(-1, keepdim=True) if kk.numel() else torch.zeros(Nq, 1, dtype=F64)
                most = (x.masked_fill(~okk, -math.inf).amax(-1, keepdim=True) / math.log(2.0) if kk.numel() else x.new_zeros(Nq, 1)).clamp(-80, 0)
                lost = okk.sum(-1, keepdim=True) * 2.0 ** (-106 - most) * (vv.abs().amax() if vv.numel() else 0.0)
                out[b, :, g] = o
                tol[b, :, g] = (2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -16 + 2 * e) * off
                                + (okk.sum(-1, keepdim=True) + 8) * 2.0 ** -24 * size + lost)
    return out, tol
