"""Rotary positions with several axes, and the norm of query and key heads with their rotation.

* ``rope_axes(q, k, positions, sections, theta)``: each head's pairs of dimensions turned by angles
  from a position of several axes (time, longitude, latitude; frame, row, column), where the
  reference's ``RoPE`` (primitives.py:108-135) has two axes in precomputed tables.
* ``qk_norm_rope(q, k, q_weight, k_weight, ...)``: the RMS norm of every query and key head and its
  rotation, by tables or by positions, in the same pass over q and k.  ``MosaicAttention`` calls it
  where its config sets ``head_norm``.

q is [B, N, Hq, d] and k [B, N, Hk, d] (or None), both bfloat16 or both float32, d 32, 64 or 128,
any strides with contiguous rows; outputs are new contiguous tensors of q's type.  Both ops are
differentiable once, in reverse mode: in q, k and the weights, not in positions or tables.  They enqueue on the
current stream of q's device and never synchronise the host.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad

from . import _lib

__all__ = ["rope_axes", "qk_norm_rope"]

_DT = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_POS = {torch.float32: _lib.POS_F32, torch.float64: _lib.POS_F64, torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64}
_WIDER = {torch.float16: torch.float32, torch.bfloat16: torch.float32, torch.int16: torch.int32,
          torch.int8: torch.int32, torch.uint8: torch.int32}


def _heads(what: str, q: torch.Tensor, k: torch.Tensor | None) -> None:
    """The checks of q and k that need no device."""
    for name, t in (("q", q), ("k", k)):
        if t is None and name == "k":
            continue
        if t.dim() != 4:
            raise ValueError(f"{what}: {name} must be [B, N, H, d], got shape {tuple(t.shape)}")
        if t.dtype not in _DT:
            raise TypeError(f"{what}: {name} is {t.dtype}; bfloat16 and float32 are computed")
    B, N, H, d = q.shape
    if d not in (32, 64, 128):
        raise ValueError(f"{what}: head_dim must be 32, 64 or 128, got {d}")
    Bk, Nk, Hk, dk = (B, N, 1, d) if k is None else k.shape
    if H == 0 or Hk == 0 or max(H, Hk) > 65535:
        raise ValueError(f"{what}: q and k need a head, and take 65535 at most")
    if Bk != B or Nk != N or dk != d or (k is not None and k.dtype != q.dtype):
        raise ValueError(f"{what}: q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} disagree")
    if B * N >= 1 << 31:
        raise ValueError(f"{what}: B * N must be below 2^31")


def _no_grad_through(what: str, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{what} has no gradient in {name}: pass it detached")


def _same_device(what: str, q: torch.Tensor, **tensors) -> None:
    if not q.is_cuda:
        raise ValueError(f"{what}: q must be on a ROCm device, got {q.device}")
    index = q.get_device()
    for name, t in tensors.items():
        if t is not None and (t.get_device() != index or not t.is_cuda):
            raise ValueError(f"{what}: {name} is on {t.device}, q on {q.device}")


_here = contextlib.nullcontext()


def _like(t: torch.Tensor) -> torch.Tensor:
    """A new contiguous tensor of t's shape and type (sooner made than by torch.empty)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _on(device: torch.device):
    """The device's context, entered only where another device is current (a call's host time counts
    where it has one row: the context takes longer than the comparison)."""
    return _here if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    """The handle of torch.cuda.current_stream(device), without making the stream object."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _strides(t: torch.Tensor) -> list[int]:
    """Strides with those of single-element dimensions, which address nothing, as 0."""
    return [s if n > 1 else 0 for n, s in zip(t.shape, t.stride())]


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, _lib.Bnhd]:
    """t with contiguous, 16-byte aligned rows (copied only where they are not), and as the kernels take it."""
    sb, sn, sh, sd = t.stride()
    unit = 3 if t.dtype == torch.float32 else 7
    ptr = t.data_ptr()
    if sd != 1 or ptr & 15 or (sb | sn | sh) & unit:
        sb, sn, sh, _ = _strides(t)
        if (sd != 1 and t.shape[3] > 1) or ptr & 15 or (sb | sn | sh) & unit:
            t = t.clone(memory_format=torch.contiguous_format)
            sb, sn, sh, _ = t.stride()
            ptr = t.data_ptr()
    return t, _lib.Bnhd(ptr, sb, sn, sh)


_NONE = _lib.Bnhd()


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=256)
def _axes(what: str, sections: tuple, theta, half: int):
    """(counts of pairs, their thetas) as the kernels take them, checked."""
    n = len(sections)
    if not 1 <= n <= _lib.MAX_AXES or min(sections) < 0 or sum(sections) > half:
        raise ValueError(f"{what}: sections {sections} must be 1 to {_lib.MAX_AXES} counts of pairs, at most {half} together")
    theta = theta if isinstance(theta, tuple) else (theta,) * n
    if len(theta) != n or not all(0 < x < math.inf for x in theta):
        raise ValueError(f"{what}: theta must be a positive number, or one for each of the {n} axes")
    pad = (0,) * (_lib.MAX_AXES - n)
    return (ctypes.c_int32 * _lib.MAX_AXES)(*(sections + pad)), (ctypes.c_double * _lib.MAX_AXES)(*(theta + pad))


def _positions(what: str, q: torch.Tensor, positions: torch.Tensor, sections, theta):
    """(positions as the kernels take them, counts and thetas), checked."""
    sections = tuple(map(int, sections))
    theta = tuple(map(float, theta)) if isinstance(theta, (list, tuple)) else float(theta)
    axes = _axes(what, sections, theta, q.shape[3] // 2)
    B, N, n, shape = q.shape[0], q.shape[1], len(sections), positions.shape
    if shape[-2:] != (N, n) or not (len(shape) == 2 or (len(shape) == 3 and shape[0] in (1, B))):
        raise ValueError(f"{what}: positions {tuple(shape)} must be [N, axes] or [B, N, axes] = {(B, N, n)}")
    if positions.dtype in _WIDER:
        positions = positions.to(_WIDER[positions.dtype])
    if positions.dtype not in _POS:
        raise TypeError(f"{what}: positions are {positions.dtype}; floating and integer types are taken")
    if n > 1 and positions.stride(-1) != 1:
        positions = positions.contiguous()
    return positions, axes


def _tables(what: str, q: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor):
    want = (q.shape[1], q.shape[3] // 2)
    if cos.shape != want or sin.shape != want:
        raise ValueError(f"{what}: cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must be [N, d/2] = {want}")
    made = []
    for t in (cos, sin):
        if t.dtype != torch.float32 or not t.is_contiguous():
            t = t.to(torch.float32).contiguous()
        made.append(t.clone() if t.data_ptr() % 16 else t)
    return made


def _rotation(cos, sin, positions, axes, interleaved: bool) -> _lib.Rotation | None:
    r = _lib.Rotation()
    r.interleaved = interleaved
    if cos is not None:
        r.cos, r.sin = cos.data_ptr(), sin.data_ptr()
        return r
    if positions is None:
        return None
    shape, stride = positions.shape, positions.stride()
    r.positions, r.position_type, r.num_axes = positions.data_ptr(), _POS[positions.dtype], shape[-1]
    r.stride_n = stride[-2]
    if len(shape) == 3 and shape[0] > 1:
        r.stride_b = stride[0]
    r.sections, r.theta = axes
    return r


def _wants_grad(*tensors) -> bool:
    """Whether autograd is to see the call: a tensor requires grad, or a forward-mode level is open, where
    the function refuses inputs that carry a tangent (it has none for its output)."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _rotate(q, k, rotation, backward: bool, norm: bool, wq=None, wk=None, eps: float = 0.0):
    """mosaic_qk_rotate_fwd on q and k (k may be None)."""
    B, N, Hq, d = q.shape
    dtype, device = q.dtype, q.device
    q_out = _like(q)
    Hk, k_out, kb, k_ptr = 0, None, _NONE, None
    if k is not None:
        Hk = k.shape[2]
        k_out = _like(k)
        k_ptr = k_out.data_ptr()
    if B * N == 0:
        return q_out, k_out
    q, qb = _rows(q)
    if k is not None:
        k, kb = _rows(k)
    with _on(device):
        st = _lib.lib().mosaic_qk_rotate_fwd(
            qb, kb, _DT[dtype], B, N, Hq, Hk, d, None if rotation is None else ctypes.byref(rotation), backward, norm,
            _ptr(wq), _ptr(wk), eps, q_out.data_ptr(), k_ptr, _stream(device))
    _lib.check(st, "mosaic_qk_rotate_fwd")
    return q_out, k_out


class _RopeAxes(torch.autograd.Function):
    """The rotation; its gradient is the rotation back."""

    @staticmethod
    def forward(ctx, q, k, positions, axes, interleaved):
        ctx.save_for_backward(positions)
        ctx.rest = (axes, interleaved)
        return _rotate(q, k, _rotation(None, None, positions, *ctx.rest), False, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        (positions,) = ctx.saved_tensors
        dq, dk = _rotate(gq, gk, _rotation(None, None, positions, *ctx.rest), True, False)
        return dq, dk, None, None, None


def rope_axes(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, sections, theta=10000.0, *,
              interleaved: bool = True):
    """q and k with each pair of dimensions turned by its axis of the position: ``(q', k')``.

    ``positions`` [N, axes] or [B, N, axes], floating or integer, on q's device.  ``sections``: the
    pairs of each axis, in order; pair j of an axis with n pairs turns by ``position *
    theta ** (-j / n)`` radians (``theta`` a number, or one for each axis), and pairs past the last
    section stay as they are.  The angle is formed in 64 bits and reduced there, so far positions
    keep it.  ``interleaved``: pair i is dimensions (2i, 2i + 1), else (i, i + d/2).

    ``rope_axes(q, k, deg2rad(grid), (d/4, d/4))`` is the reference's RoPE on that (longitude,
    latitude) grid (primitives.py:115-135), up to the rounding of its fp32 tables.
    """
    _heads("rope_axes", q, k)
    _no_grad_through("rope_axes", positions=positions)
    positions, axes = _positions("rope_axes", q, positions, sections, theta)
    _same_device("rope_axes", q, k=k, positions=positions)
    if _wants_grad(q, k):
        return _RopeAxes.apply(q, k, positions, axes, bool(interleaved))
    return _rotate(q, k, _rotation(None, None, positions, axes, bool(interleaved)), False, False)


def _fp32(w: torch.Tensor | None) -> torch.Tensor | None:
    return w if w is None or (w.dtype == torch.float32 and w.is_contiguous()) else w.to(torch.float32).contiguous()


class _QkNormRope(torch.autograd.Function):
    """The norm and rotation; the backward reads q and k again and forms the norms anew."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, eps, cos, sin, positions, axes, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.rest = (axes, interleaved)
        ctx.eps = eps
        return _rotate(q, k, _rotation(cos, sin, positions, *ctx.rest), False, True, _fp32(q_weight), _fp32(k_weight), eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        B, N, Hq, d = q.shape
        dtype, device = q.dtype, q.device
        dq = _like(q)
        Hk, dk, kb, gkb = 0, None, _NONE, _NONE
        if k is not None:
            Hk = k.shape[2]
            dk = _like(k)
        weights = (q_weight, k_weight)
        dw = [(torch.empty if B * N else torch.zeros)(d, dtype=torch.float32, device=device) if w is not None and need else None
              for w, need in zip(weights, ctx.needs_input_grad[2:4])]
        if B * N:
            gq, gqb = _rows(gq)
            q, qb = _rows(q)
            if k is not None:
                gk, gkb = _rows(gk)
                k, kb = _rows(k)
            wq, wk = map(_fp32, weights)
            rotation = _rotation(cos, sin, positions, *ctx.rest)
            L = _lib.lib()
            ws, nbytes = None, 0
            if dw[0] is not None or dw[1] is not None:
                nbytes = L.mosaic_qk_norm_bwd_workspace_size(B, N, d)
                ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
            with _on(device):
                st = L.mosaic_qk_norm_rotate_bwd(
                    gqb, gkb, qb, kb, _DT[dtype], B, N, Hq, Hk, d, None if rotation is None else ctypes.byref(rotation), _ptr(wq),
                    _ptr(wk), ctx.eps, dq.data_ptr(), _ptr(dk), _ptr(dw[0]), _ptr(dw[1]), _ptr(ws), nbytes, _stream(device))
            _lib.check(st, "mosaic_qk_norm_rotate_bwd")
        dw = [None if g is None else g.to(w.dtype) for g, w in zip(dw, weights)]
        return (dq, dk, *dw) + (None,) * 6


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, *, eps: float | None = None, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None, positions: torch.Tensor | None = None, sections=None,
                 theta=10000.0, interleaved: bool = True):
    """The RMS norm of every head of q and k over its d dimensions, then its rotation: ``(q', k')``.

    ``y = R (w * x * rsqrt(mean(x^2) + eps))`` with the statistics in fp32 and one rounding, of y.
    ``q_weight`` / ``k_weight`` [d] are shared by all heads (None: ones); ``eps`` None is torch's
    RMSNorm default, the epsilon of fp32.  The rotation comes from ``cos`` / ``sin`` (the RoPE
    module's tables, [N, d/2]), or from ``positions`` and ``sections`` as in ``rope_axes``, or is
    left out where neither is given.
    """
    what = "qk_norm_rope"
    _heads(what, q, k)
    if (cos is None) != (sin is None):
        raise ValueError(f"{what}: cos and sin go together")
    if (positions is None) != (sections is None):
        raise ValueError(f"{what}: positions and sections go together")
    if cos is not None and positions is not None:
        raise ValueError(f"{what}: tables or positions, not both")
    if k is None and k_weight is not None:
        raise ValueError(f"{what}: k_weight without k")
    eps = torch.finfo(torch.float32).eps if eps is None else float(eps)
    if not 0 <= eps <= torch.finfo(torch.float32).max:
        raise ValueError(f"{what}: eps must not be negative or beyond fp32, got {eps}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and tuple(w.shape) != (q.shape[3],):
            raise ValueError(f"{what}: {name} {tuple(w.shape)} must be [d] = ({q.shape[3]},)")
        if w is not None and not w.dtype.is_floating_point:
            raise TypeError(f"{what}: {name} is {w.dtype}")
    _no_grad_through(what, cos=cos, sin=sin, positions=positions)
    axes = None
    if cos is not None:
        cos, sin = _tables(what, q, cos, sin)
    elif positions is not None:
        positions, axes = _positions(what, q, positions, sections, theta)
    _same_device(what, q, k=k, q_weight=q_weight, k_weight=k_weight, cos=cos, sin=sin, positions=positions)
    interleaved = bool(interleaved)
    if _wants_grad(q, k, q_weight, k_weight):
        return _QkNormRope.apply(q, k, q_weight, k_weight, eps, cos, sin, positions, axes, interleaved)
    return _rotate(q, k, _rotation(cos, sin, positions, axes, interleaved), False, True, _fp32(q_weight), _fp32(k_weight), eps)
