"""Forward-mode derivatives of the query and rotary operators: there are none, and a call whose inputs carry
a tangent says so rather than return a value without one.

CPU: the wrappers with the library and the device stubbed out.  GPU: the same calls, and calls without
tangents inside a level, which are unchanged.
"""

import contextlib

import pytest
import torch
import torch.autograd.forward_ad as fwad

import mosaic_amd as M
from mosaic_amd import _lib, query, rotary

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


class _Stub:
    """Takes every call of the library and writes nothing."""

    def __getattr__(self, name):
        return (lambda *a: 256) if name.endswith("workspace_size") else (lambda *a: 0)


@pytest.fixture
def stubbed(monkeypatch):
    monkeypatch.setattr(_lib, "lib", lambda: _Stub())
    for module in (rotary, query):
        monkeypatch.setattr(module, "_same_device", lambda *a, **k: None)
        monkeypatch.setattr(module, "_on", lambda device: contextlib.nullcontext())
        monkeypatch.setattr(module, "_stream", lambda device: 0)


def calls(device):
    gen = torch.Generator().manual_seed(1)

    def t(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen).to(device, dtype)

    q, k, pos, w = t(1, 5, 4, 64), t(1, 5, 2, 64), t(5, 2), t(64)
    aq, ak, av = t(1, 5, 4, 64, dtype=BF16), t(1, 128, 2, 64, dtype=BF16), t(1, 128, 2, 64, dtype=BF16)
    idx = torch.zeros(1, 5, 2, 1, dtype=torch.int64, device=device)
    return {
        "rope_axes": (lambda q, k, pos: M.rope_axes(q, k, pos, (16, 16))[1], (q, k, pos)),
        "qk_norm_rope": (lambda q, k, wq, wk, pos: M.qk_norm_rope(q, k, wq, wk, positions=pos, sections=(16, 16))[0],
                         (q, k, w, w.clone(), pos)),
        "query_sparse_attn": (lambda q, k, v: M.query_sparse_attn(q, k, v, idx, 64), (aq, ak, av)),
        "mosaic_query_attn": (lambda q, k, v: M.mosaic_query_attn(q, k, v, 64, 1, k_cmp=ak[:, :2]), (aq, ak, av)),
    }


NAMED = [("rope_axes", 3), ("qk_norm_rope", 5), ("query_sparse_attn", 3), ("mosaic_query_attn", 3)]
EACH = [(name, i) for name, n in NAMED for i in range(n)]


def refuses_a_tangent(name, i, device):
    fn, args = calls(device)[name]
    for grad in (True, False):
        with torch.set_grad_enabled(grad), fwad.dual_level():
            moved = [fwad.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate(args)]
            with pytest.raises(RuntimeError, match="forward"):
                fn(*moved)


@pytest.mark.parametrize("name,i", EACH)
def test_a_tangent_is_refused(name, i, stubbed):
    refuses_a_tangent(name, i, "cpu")


@gpu
@pytest.mark.parametrize("name,i", EACH)
def test_a_tangent_is_refused_on_the_device(name, i):
    refuses_a_tangent(name, i, "cuda")


@gpu
@pytest.mark.parametrize("name", [n for n, _ in NAMED])
def test_calls_without_tangents_inside_a_level(name):
    fn, args = calls("cuda")[name]
    want = fn(*args)
    with fwad.dual_level():
        assert torch.equal(fn(*args), want)
        leaves = [a.clone().requires_grad_() if a.shape[-1] == 64 else a for a in args]
        out = fn(*leaves)
        assert torch.equal(out.detach(), want) and out.requires_grad
