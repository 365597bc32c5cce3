"""rope_axes and qk_norm_rope: refusals (CPU) and values against float64 (GPU).

Tolerances, fixed before the first run (u = 2^-24, half a step of fp32):
* one rotation: products and sum round by at most 3 u of |a| + |b| (the pair's values); a cosine
  or sine is off by at most pi u (the reduced angle's rounding) + 4 u (the function) -- together
  below 16 u (|a| + |b|);
* the norm: 8 sequential and 4 tree additions of squares (halved by the root), mean, root, division
  and two products: below 16 u of each value, on top of the rotation: 32 u (|a| + |b|);
* its gradient: u = R(-a) g (16 u), v = w u, two means over d: below 64 u of r (|v| + |h| mean|v h|),
  taken over the pair;
* a weight gradient: at most 40 terms in a lane, 64 groups, 32 rows and 32 more: 176 u, and 32 u for
  each term: 256 u of the sum of |u h|;
* every bf16 output: 2^-8 of its value for the rounding, on top.
"""

import ctypes
import math

import pytest
import torch

import mosaic_amd as M
from mosaic_amd import _lib
from mosaic_amd.healpix import get_healpix_grid, rope_tables

U = 2.0 ** -24
gpu = pytest.mark.gpu
DEV = "cuda"


def heads(*shape, dtype=torch.float32, grad=False):
    x = torch.zeros(*shape, dtype=dtype)
    return x.requires_grad_() if grad else x


Q, K = (2, 5, 4, 64), (2, 5, 2, 64)


# ------------------------------------------------------------------------------- refusals (CPU)

@pytest.mark.parametrize("call,error,match", [
    (lambda: M.rope_axes(heads(5, 4, 64), None, torch.zeros(5, 1), (4,)), ValueError, "B, N, H, d"),
    (lambda: M.rope_axes(heads(*Q, dtype=torch.float16), None, torch.zeros(5, 1), (4,)), TypeError, "float16"),
    (lambda: M.rope_axes(heads(2, 5, 4, 48), None, torch.zeros(5, 1), (4,)), ValueError, "32, 64 or 128"),
    (lambda: M.rope_axes(heads(*Q), heads(2, 4, 2, 64), torch.zeros(5, 1), (4,)), ValueError, "disagree"),
    (lambda: M.rope_axes(heads(*Q), heads(*K, dtype=torch.bfloat16), torch.zeros(5, 1), (4,)), ValueError, "disagree"),
    (lambda: M.rope_axes(heads(*Q), heads(2, 5, 0, 64), torch.zeros(5, 1), (4,)), ValueError, "head"),
    (lambda: M.rope_axes(heads(*Q), None, torch.zeros(5, 2), (20, 13)), ValueError, "sections"),
    (lambda: M.rope_axes(heads(*Q), None, torch.zeros(5, 2), (20, -1)), ValueError, "sections"),
    (lambda: M.rope_axes(heads(*Q), None, torch.zeros(5, 9), (1,) * 9), ValueError, "sections"),
    (lambda: M.rope_axes(heads(*Q), None, torch.zeros(5, 3), (4, 4)), ValueError, "positions"),
    (lambda: M.rope_axes(heads(*Q), None, torch.zeros(3, 5, 2), (4, 4)), ValueError, "positions"),
    (lambda: M.rope_axes(heads(*Q), None, torch.zeros(5, 2, dtype=torch.complex64), (4, 4)), TypeError, "complex"),
    (lambda: M.rope_axes(heads(*Q), None, torch.zeros(5, 2), (4, 4), theta=-1.0), ValueError, "theta"),
    (lambda: M.rope_axes(heads(*Q), None, torch.zeros(5, 2), (4, 4), theta=(1.0, 2.0, 3.0)), ValueError, "theta"),
    (lambda: M.rope_axes(heads(*Q), None, torch.zeros(5, 2, requires_grad=True), (4, 4)), RuntimeError, "no gradient"),
    (lambda: M.rope_axes(heads(*Q), None, torch.zeros(5, 2), (4, 4)), ValueError, "ROCm"),
    (lambda: M.qk_norm_rope(heads(*Q), heads(*K), torch.ones(32)), ValueError, "q_weight"),
    (lambda: M.qk_norm_rope(heads(*Q), heads(*K), None, torch.ones(64, dtype=torch.long)), TypeError, "k_weight"),
    (lambda: M.qk_norm_rope(heads(*Q), None, None, torch.ones(64)), ValueError, "without k"),
    (lambda: M.qk_norm_rope(heads(*Q), None, eps=-1e-6), ValueError, "eps"),
    (lambda: M.qk_norm_rope(heads(*Q), None, eps=float("nan")), ValueError, "eps"),
    (lambda: M.qk_norm_rope(heads(*Q), None, cos=torch.zeros(5, 32)), ValueError, "together"),
    (lambda: M.qk_norm_rope(heads(*Q), None, positions=torch.zeros(5, 1)), ValueError, "together"),
    (lambda: M.qk_norm_rope(heads(*Q), None, cos=torch.zeros(5, 32), sin=torch.zeros(5, 32),
                            positions=torch.zeros(5, 1), sections=(4,)), ValueError, "not both"),
    (lambda: M.qk_norm_rope(heads(*Q), None, cos=torch.zeros(4, 32), sin=torch.zeros(5, 32)), ValueError, "d/2"),
    (lambda: M.qk_norm_rope(heads(*Q), None, cos=torch.zeros(5, 32, requires_grad=True), sin=torch.zeros(5, 32)),
     RuntimeError, "no gradient"),
    (lambda: M.qk_norm_rope(heads(*Q), heads(*K)), ValueError, "ROCm"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


FAKE = 1 << 20   # non-null, aligned, never read: every call below is refused on the host
HAVE_LIB = pytest.mark.skipif(not __import__("os").path.exists(_lib.LIB_PATH), reason="libmosaic_bsa.so not built")


def _rot(**kw):
    r = _lib.Rotation()
    r.positions, r.num_axes, r.position_type, r.interleaved = FAKE, 2, _lib.POS_F32, 1
    r.sections[0] = r.sections[1] = 16
    r.theta[0] = r.theta[1] = 10000.0
    for name, v in kw.items():
        if name in ("sections", "theta"):
            for i, x in enumerate(v):
                getattr(r, name)[i] = x
        else:
            setattr(r, name, v)
    return r


@HAVE_LIB
@pytest.mark.parametrize("change,status", [
    (dict(dtype=5), 10), (dict(batch=0), 8), (dict(seq=0), 8), (dict(batch=1 << 16, seq=1 << 15), 8), (dict(hq=0), 3),
    (dict(hk=-1), 3), (dict(d=48), 11), (dict(q=_lib.Bnhd(None, 0, 0, 0)), 1), (dict(q=_lib.Bnhd(FAKE + 2, 0, 0, 0)), 7),
    (dict(k=_lib.Bnhd(FAKE, 0, 4, 0)), 7), (dict(out=None), 1), (dict(out=FAKE + 8), 7), (dict(rot=None), 1),
    (dict(rot=_rot(positions=None)), 1), (dict(rot=_rot(num_axes=0)), 8), (dict(rot=_rot(num_axes=9)), 8),
    (dict(rot=_rot(position_type=4)), 10), (dict(rot=_rot(positions=FAKE + 2)), 7), (dict(rot=_rot(sections=(30, 3))), 8),
    (dict(rot=_rot(sections=(-1,))), 8), (dict(rot=_rot(theta=(0.0,))), 8), (dict(rot=_rot(cos=FAKE)), 1),
    (dict(rot=_rot(cos=FAKE, sin=FAKE + 4)), 7), (dict(norm=1, backward=1), 10), (dict(norm=1, eps=float("nan")), 10),
])
def test_abi_forward_validation(change, status):
    c = dict(q=_lib.Bnhd(FAKE, 0, 256, 64), k=_lib.Bnhd(FAKE, 0, 128, 64), dtype=_lib.DTYPE_BF16, batch=1, seq=8, hq=4, hk=2,
             d=64, rot=_rot(), backward=0, norm=0, eps=1e-6, out=FAKE)
    c.update(change)
    st = _lib.lib().mosaic_qk_rotate_fwd(c["q"], c["k"], c["dtype"], c["batch"], c["seq"], c["hq"], c["hk"], c["d"],
                                         None if c["rot"] is None else ctypes.byref(c["rot"]), c["backward"], c["norm"],
                                         None, None, c["eps"], c["out"], c["out"], None)
    assert st == status


@HAVE_LIB
def test_abi_backward_validation():
    L = _lib.lib()
    x = _lib.Bnhd(FAKE, 0, 256, 64)
    need = L.mosaic_qk_norm_bwd_workspace_size(1, 8, 64)
    assert need > 0 and L.mosaic_qk_norm_bwd_workspace_size(1, 8, 48) == 0

    def call(gq=x, dq=FAKE, ws=FAKE, n=need, eps=1e-6, rot=_rot(), wg=FAKE):
        return L.mosaic_qk_norm_rotate_bwd(gq, x, x, x, _lib.DTYPE_BF16, 1, 8, 4, 4, 64, ctypes.byref(rot), None, None, eps, dq,
                                           FAKE, wg, None, ws, n, None)
    assert call(gq=_lib.Bnhd(FAKE + 2, 0, 256, 64)) == 7
    assert call(dq=None) == 1
    assert call(dq=FAKE + 4) == 7
    assert call(ws=None) == 6
    assert call(ws=FAKE + 4) == 6
    assert call(n=need - 1) == 6
    assert call(eps=-1.0) == 10
    assert call(wg=FAKE + 2) == 7
    assert call(rot=_rot(sections=(33,))) == 8


# ------------------------------------------------------------------------------- values (GPU)

def _turn64(x, ang, rotated, inter):
    """x [B, N, H, d] in float64 turned by ang [.., N, d/2]; pairs past `rotated` kept."""
    c, s = ang.cos().unsqueeze(-2), ang.sin().unsqueeze(-2)
    a, b = (x[..., 0::2], x[..., 1::2]) if inter else x.chunk(2, dim=-1)
    on = torch.arange(x.shape[-1] // 2, device=x.device) < rotated
    y0, y1 = torch.where(on, a * c - b * s, a), torch.where(on, b * c + a * s, b)
    return torch.stack([y0, y1], -1).flatten(-2) if inter else torch.cat([y0, y1], -1)


def _pair_sum(x, inter):
    """|a| + |b| of each value's pair."""
    a, b = (x[..., 0::2], x[..., 1::2]) if inter else x.chunk(2, dim=-1)
    t = a.abs() + b.abs()
    return torch.stack([t, t], -1).flatten(-2) if inter else torch.cat([t, t], -1)


def _angles64(pos, sections, theta, half):
    cols = [pos[..., a].double() * th ** (-j / n) for a, (n, th) in enumerate(zip(sections, theta)) for j in range(n)]
    cols += [torch.zeros_like(cols[0] if cols else pos[..., 0].double())] * (half - len(cols))
    return torch.stack(cols, -1)


def _near(got, want, slack, what):
    """|got - want| within slack, and half a step of got's type."""
    lim = slack + (want.abs() * 2.0 ** -8 if got.dtype == torch.bfloat16 else 0.0)
    over = (got.double() - want).abs() - lim
    assert bool((over <= 0).all()), f"{what}: {over.max().item():.3g} over its bound"


def _make(shape, dtype, gen, layout="contiguous"):
    B, N, H, d = shape
    if layout == "seq_first":
        x = torch.randn(N, B, H, d, generator=gen, device=DEV).to(dtype).transpose(0, 1)
    elif layout == "slice":        # heads of a wider projection
        x = torch.randn(B, N, H + 3, d, generator=gen, device=DEV).to(dtype)[:, :, 1:H + 1]
    elif layout == "unaligned":    # rows that have to be copied
        x = torch.randn(B, N, H, d + 1, generator=gen, device=DEV).to(dtype)[..., 1:]
    elif layout == "broadcast":
        x = torch.randn(1, N, 1, d, generator=gen, device=DEV).to(dtype).expand(B, N, H, d)
    else:
        x = torch.randn(B, N, H, d, generator=gen, device=DEV).to(dtype)
    return x


ROPE_CASES = [
    # B, N, Hq, Hk, d, sections, inter, dtype, layout, position type, per member
    (1, 1, 12, 3, 64, (8, 12, 12), True, torch.bfloat16, "contiguous", torch.float32, False),
    (24, 1, 12, 3, 64, (8, 12, 12), True, torch.bfloat16, "seq_first", torch.float32, True),
    (2, 37, 5, 1, 64, (16, 16), False, torch.float32, "slice", torch.int64, False),
    (2, 130, 16, 4, 128, (16, 24, 24), False, torch.bfloat16, "unaligned", torch.int32, True),
    (3, 65, 1, 0, 32, (3, 0, 5), True, torch.float32, "contiguous", torch.float64, False),
    (1, 2049, 7, 2, 32, (16,), False, torch.bfloat16, "slice", torch.float32, False),
    (2, 9, 4, 4, 128, (1, 2, 3, 4, 5, 6, 7, 8), True, torch.float32, "seq_first", torch.float32, True),
    (1, 17001, 9, 5, 64, (10, 11, 9), True, torch.bfloat16, "contiguous", torch.float32, False),
    (2, 8, 4, 2, 64, (8, 8), True, torch.float32, "broadcast", torch.float16, False),
]


def _positions(case, gen):
    B, N, sections, ptype, per = case[0], case[1], case[5], case[9], case[10]
    shape = ((B,) if per else ()) + (N, len(sections))
    if ptype.is_floating_point:
        p = torch.randn(*shape, generator=gen, device=DEV) * 3
        if ptype != torch.float16:
            p[..., 0] = torch.randint(0, 1 << 22, shape[:-1], generator=gen, device=DEV) / 4   # far positions
        return p.to(ptype)
    return torch.randint(-50000, 1 << 20, shape, generator=gen, device=DEV).to(ptype)


@gpu
@pytest.mark.parametrize("case", ROPE_CASES, ids=lambda c: f"b{c[0]}n{c[1]}h{c[2]}-{c[3]}d{c[4]}" if isinstance(c, tuple) else None)
def test_rope_axes_values_and_gradient(case):
    B, N, Hq, Hk, d, sections, inter, dtype, layout, _, _ = case
    gen = torch.Generator(device=DEV).manual_seed(N + d)
    q = _make((B, N, Hq, d), dtype, gen, layout).requires_grad_()
    k = _make((B, N, Hk, d), dtype, gen, layout).requires_grad_() if Hk else None
    pos = _positions(case, gen)
    theta = tuple(10000.0 / (a + 1) for a in range(len(sections)))
    out = M.rope_axes(q, k, pos, sections, theta, interleaved=inter)
    ang, rotated = _angles64(pos, sections, theta, d // 2), sum(sections)
    for x, y in zip((q, k), out):
        if x is None:
            assert y is None
            continue
        assert y.dtype == dtype and y.is_contiguous() and y.shape == x.shape
        x64 = x.detach().double()
        _near(y.detach(), _turn64(x64, ang, rotated, inter), 16 * U * _pair_sum(x64, inter), "forward")
        g = torch.randn(x.shape, generator=gen, device=DEV).to(dtype)
        (dx,) = torch.autograd.grad(y, x, g, retain_graph=True)
        g64 = g.double()
        _near(dx, _turn64(g64, -ang, rotated, inter), 16 * U * _pair_sum(g64, inter), "gradient")


@gpu
def test_rope_axes_with_two_axes_is_the_rope_module():
    grid = get_healpix_grid(8)
    rope = M.RoPE(64)
    rope.initialize_rope(grid)
    rope = rope.to(DEV)
    gen = torch.Generator(device=DEV).manual_seed(0)
    q = torch.randn(2, 768, 4, 64, generator=gen, device=DEV)
    got, none = M.rope_axes(q, None, torch.deg2rad(grid).to(DEV), (16, 16))
    assert none is None
    # the module's fp32 tables hold angles below 2 pi to 2^-23 relative: 2 pi 2^-23 of |a| + |b|, and both sides' roundings
    lim = (2 * math.pi * 2 + 32) * U * _pair_sum(q.double(), True)
    assert bool(((got.double() - rope(q).double()).abs() <= lim).all())


@gpu
def test_rope_axes_keeps_unrotated_pairs_beside_infinities():
    q = torch.ones(1, 3, 2, 64, device=DEV)
    q[..., 40] = math.inf      # pair 20 of 32, interleaved
    q[..., 43] = math.nan
    out, _ = M.rope_axes(q, None, torch.ones(3, 1, device=DEV), (20,))
    assert torch.equal(out[..., 40:42], q[..., 40:42]) and torch.equal(out[..., 42], q[..., 42])
    assert torch.isfinite(out[..., :40]).all()


NORM_CASES = [
    # B, N, Hq, Hk, d, inter, dtype, layout, rotation, weights, eps
    (1, 1, 12, 3, 64, True, torch.bfloat16, "contiguous", "tables", True, 1e-6),
    (2, 33, 5, 2, 64, False, torch.float32, "slice", "tables", True, None),
    (2, 131, 16, 4, 128, True, torch.bfloat16, "seq_first", "positions", True, 1e-5),
    (3, 65, 3, 1, 32, False, torch.bfloat16, "unaligned", "none", True, 1e-6),
    (1, 700, 7, 7, 64, True, torch.float32, "broadcast", "none", False, 1e-6),
    (2, 90, 9, 0, 128, False, torch.float32, "contiguous", "positions", True, 1e-3),
]


@gpu
@pytest.mark.parametrize("case", NORM_CASES, ids=lambda c: f"b{c[0]}n{c[1]}h{c[2]}-{c[3]}d{c[4]}{c[8]}")
def test_qk_norm_rope_values_and_gradients(case):
    B, N, Hq, Hk, d, inter, dtype, layout, rotation, weighted, eps = case
    gen = torch.Generator(device=DEV).manual_seed(N)
    made = [_make((B, N, h, d), dtype, gen, layout) for h in (Hq, Hk) if h]
    xs = [x.detach().requires_grad_() for x in made]
    ws = [(1 + 0.3 * torch.randn(d, generator=gen, device=DEV)).requires_grad_() if weighted else None for _ in xs]
    kw, ang, rotated = {}, torch.zeros(N, d // 2, device=DEV, dtype=torch.float64), 0
    if rotation == "tables":
        a = torch.randn(N, d // 2, generator=gen, device=DEV) * 3
        kw = dict(cos=a.cos(), sin=a.sin())
        c64, s64, rotated = kw["cos"].double(), kw["sin"].double(), d // 2
    elif rotation == "positions":
        pos = torch.randn(N, 2, generator=gen, device=DEV) * 10
        kw = dict(positions=pos, sections=(d // 4, d // 8))
        ang, rotated = _angles64(pos, (d // 4, d // 8), (10000.0,) * 2, d // 2), d // 4 + d // 8
    if rotation != "tables":
        c64, s64 = ang.cos(), ang.sin()

    def turned(x, sign):
        c, s = c64.unsqueeze(-2), sign * s64.unsqueeze(-2)
        p, r = (x[..., 0::2], x[..., 1::2]) if inter else x.chunk(2, dim=-1)
        on = torch.arange(d // 2, device=DEV) < rotated
        y0, y1 = torch.where(on, p * c - r * s, p), torch.where(on, r * c + p * s, r)
        return torch.stack([y0, y1], -1).flatten(-2) if inter else torch.cat([y0, y1], -1)

    k, wk = (xs[1], ws[1]) if Hk else (None, None)
    out = M.qk_norm_rope(xs[0], k, ws[0], wk, eps=eps, interleaved=inter, **kw)
    e = torch.finfo(torch.float32).eps if eps is None else eps
    gs = [torch.randn(x.shape, generator=gen, device=DEV).to(dtype) for x in xs]
    leaves = xs + [w for w in ws if w is not None]
    grads = torch.autograd.grad([o for o in out if o is not None], leaves, gs)
    for i, (x, w, y, g) in enumerate(zip(xs, ws, out, gs)):
        x64, g64 = x.detach().double(), g.double()
        w64 = torch.ones(d, device=DEV, dtype=torch.float64) if w is None else w.detach().double()
        r = (x64.square().mean(-1, keepdim=True) + e).rsqrt()
        h = x64 * r
        assert y.dtype == dtype and y.is_contiguous()
        _near(y.detach(), turned(h * w64, 1), 32 * U * _pair_sum(h * w64, inter), "forward")
        u = turned(g64, -1)
        v = u * w64
        vh = (v * h).abs().mean(-1, keepdim=True)
        _near(grads[i], r * (v - h * (v * h).mean(-1, keepdim=True)),
              64 * U * r * (_pair_sum(g64, inter) * w64.abs() + h.abs() * (vh + (_pair_sum(g64, inter) * w64.abs() * h.abs()).mean(-1, keepdim=True))),
              "gradient of x")
        if w is not None:
            dw = grads[len(xs) + i]
            assert dw.dtype == torch.float32
            _near(dw, (u * h).sum((0, 1, 2)), 256 * U * (_pair_sum(g64, inter) * h.abs()).sum((0, 1, 2)), "weight gradient")


@gpu
def test_qk_norm_rope_gradient_against_differences():
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(1, 6, 2, 64, generator=gen, device=DEV)
    w = 1 + 0.2 * torch.randn(64, generator=gen, device=DEV)
    pos = torch.randn(6, 2, generator=gen, device=DEV)
    g = torch.randn(1, 6, 2, 64, generator=gen, device=DEV)

    def f(x, w):
        return M.qk_norm_rope(x, None, w, eps=1e-6, positions=pos, sections=(16, 16))[0]
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(f(xl, wl), (xl, wl), g)
    step = 2.0 ** -6
    ex, ew = torch.randn(x.shape, generator=gen, device=DEV), torch.randn(w.shape, generator=gen, device=DEV)
    for d, e, at in ((dx, ex, lambda s: f(x + s * ex, w)), (dw, ew, lambda s: f(x, w + s * ew))):
        diff = ((at(step).double() - at(-step).double()) * g.double()).sum() / (2 * step)
        # outputs of size 1 rounded by a few u: 768 values of g, random signs; the third derivative times step^2 / 6
        lim = 16 * U * math.sqrt(768) * 4 / step + step ** 2 * 100
        assert abs(diff.item() - (d.double() * e.double()).sum().item()) < lim


@gpu
def test_bf16_weights_float64_weights_and_one_needed_gradient():
    gen = torch.Generator(device=DEV).manual_seed(5)
    q = torch.randn(1, 20, 4, 64, generator=gen, device=DEV).to(torch.bfloat16)
    k = torch.randn(1, 20, 2, 64, generator=gen, device=DEV).to(torch.bfloat16).requires_grad_()
    for dt in (torch.bfloat16, torch.float64, torch.float16):
        w = torch.ones(64, device=DEV, dtype=dt).requires_grad_()
        qo, ko = M.qk_norm_rope(q, k, w, w)       # one weight for both
        dk, dw = torch.autograd.grad((qo, ko), (k, w), (torch.ones_like(qo), torch.ones_like(ko)))
        assert dk.dtype == torch.bfloat16 and dw.dtype == dt and torch.isfinite(dw).all()
    # only k's output is used: q's gradient is zeros
    ql = q.clone().requires_grad_()
    _, ko = M.qk_norm_rope(ql, k, None, None)
    dq, dk = torch.autograd.grad(ko.sum(), (ql, k), allow_unused=True)
    assert dq is None or not dq.any()
    with pytest.raises(RuntimeError):             # one derivative is what there is
        (dk,) = torch.autograd.grad(M.qk_norm_rope(q, k)[1].square().sum(), k, create_graph=True)
        dk.sum().backward()


@gpu
def test_empty_batch_and_sequence():
    for shape in ((0, 5, 2, 64), (2, 0, 2, 64)):
        x = torch.zeros(*shape, device=DEV).requires_grad_()
        w = torch.ones(64, device=DEV).requires_grad_()
        y, _ = M.rope_axes(x, None, torch.zeros(shape[1], 1, device=DEV), (4,))
        assert y.shape == shape
        y, _ = M.qk_norm_rope(x, None, w)
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == shape and not dw.any()


@gpu
def test_single_row_dimensions_with_odd_strides():
    base = torch.randn(3 * 64 + 7, device=DEV).to(torch.bfloat16)
    x = base.as_strided((1, 1, 3, 64), (7, 13, 64, 1))     # strides of single-element dimensions address nothing
    y, _ = M.qk_norm_rope(x, None)
    z, _ = M.qk_norm_rope(x.clone(memory_format=torch.contiguous_format).view(1, 1, 3, 64), None)
    assert torch.equal(y, z)


@gpu
def test_same_result_on_another_stream_and_twice():
    gen = torch.Generator(device=DEV).manual_seed(7)
    q = torch.randn(2, 3000, 4, 64, generator=gen, device=DEV).to(torch.bfloat16).requires_grad_()
    w = torch.ones(64, device=DEV).requires_grad_()
    g = torch.randn(q.shape, generator=gen, device=DEV).to(torch.bfloat16)

    def step():
        y, _ = M.qk_norm_rope(q, None, w, eps=1e-6)
        return (y.detach(), *torch.autograd.grad(y, (q, w), g))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)       # no atomics: bit for bit


@gpu
def test_captured_and_replayed():
    gen = torch.Generator(device=DEV).manual_seed(9)
    q = torch.randn(1, 500, 4, 64, generator=gen, device=DEV)
    w = torch.ones(64, device=DEV)
    g = torch.randn(q.shape, generator=gen, device=DEV)
    pos = torch.randn(500, 2, generator=gen, device=DEV)

    def step():
        ql, wl = q.detach().requires_grad_(), w.detach().requires_grad_()
        y, _ = M.qk_norm_rope(ql, None, wl, positions=pos, sections=(16, 8))
        return (y.detach(), *torch.autograd.grad(y, (ql, wl), g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=gen, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b), i


@gpu
def test_far_token_offsets_past_32_bits():
    # token rows 3 * 2^28 elements apart: the last starts past 2^31 elements (4.8 GB of bf16)
    N, H, apart = 4, 2, 3 << 28
    x = torch.empty(3 * apart + H * 64, device=DEV, dtype=torch.bfloat16).as_strided((1, N, H, 64), (0, apart, 64, 1))
    gen = torch.Generator(device=DEV).manual_seed(1)
    x.copy_(torch.randn(1, N, H, 64, generator=gen, device=DEV))
    pos = torch.randn(N, 1, generator=gen, device=DEV)
    a, _ = M.rope_axes(x, None, pos, (32,))
    b, _ = M.rope_axes(x.contiguous(), None, pos, (32,))
    assert torch.equal(a, b)


@gpu
def test_theta_is_read_at_each_call_and_weights_lie_anywhere():
    gen = torch.Generator(device=DEV).manual_seed(77)
    q, pos = torch.randn(1, 33, 2, 64, generator=gen, device=DEV), torch.randn(33, 1, generator=gen, device=DEV) * 50
    theta = torch.tensor(10000.0)
    first, _ = M.rope_axes(q, None, pos, (32,), theta)
    assert torch.equal(first, M.rope_axes(q, None, pos, (32,), 10000.0)[0])
    theta.fill_(100.0)
    assert torch.equal(M.rope_axes(q, None, pos, (32,), theta)[0], M.rope_axes(q, None, pos, (32,), 100.0)[0])
    w = torch.rand(131, generator=gen, device=DEV)
    for at in (1, 2, 3):                    # slices of a larger parameter
        got, _ = M.qk_norm_rope(q, None, w[at:at + 64], positions=pos, sections=(32,))
        assert torch.equal(got, M.qk_norm_rope(q, None, w[at:at + 64].clone(), positions=pos, sections=(32,))[0])


@pytest.mark.parametrize("eps", [1e39, float("inf"), float("nan")])
def test_eps_beyond_fp32_is_refused(eps):
    with pytest.raises(ValueError, match="eps"):
        M.qk_norm_rope(heads(1, 3, 2, 64), None, eps=eps)
