"""``head_norm``: the RMS norm of query and key heads in ``MosaicAttention`` and the U-Net.

* CPU: the default has no new parameter and no new state; the flag adds one weight of head_dim per
  norm, or none where the model's norms have no weights; an older config object still works.
* GPU: the module against its own projections, normalised and rotated in 64 bits and rounded to
  bfloat16, through ``mosaic_attn_func`` and the output projection.  Every block is selected, so no
  tie of scores takes part.  Both sides' q and k round the same values once: they differ where fp32
  statistics (relative 2e-6) cross a rounding border, about one element in a thousand, by 2^-8.  What
  reaches the output is far below its own two bf16 roundings (of the heads and of the projection),
  whose relative L2 is at most 2^-9 each: bar 2^-8.
"""

import types

import pytest
import torch

from mosaic_amd.healpix import rope_tables
from mosaic_amd.model import BottleneckConfig, ModelConfig, StageConfig, Transformer
from mosaic_amd.primitives import MosaicAttention, mosaic_attn_func

DEV = "cuda"


def attention_config(**kw):
    base = dict(block_attn_size=128, sparse_block_size=64, sparse_block_count=8, num_heads=4, gqa_ratio=2, dim=256,
                qkv_compress_ratio=1, rope=True, rope_theta=10000)
    return types.SimpleNamespace(**{**base, **kw})


def model_config(**kw):
    stage = StageConfig(nside=8, dim=256, num_heads=4, block_attn_size=256, sparse_block_size=64, sparse_block_count=4,
                        encoder_depth=1, decoder_depth=1, mlp_ratio=2.0, gqa_ratio=2)
    bottleneck = BottleneckConfig(nside=4, dim=256, num_heads=4, block_attn_size=64, sparse_block_size=64,
                                  sparse_block_count=2, depth=1, mlp_ratio=2.0, gqa_ratio=2)
    base = dict(dim=256, num_heads=4, k_neighbors=8, qk_norm=False, rope=True, rope_theta=10000, sparse_every=1,
                variables=["a", "b"], static_variables=["s"], qkv_compress_ratio=1, cg_stage_cfgs=[stage],
                bottleneck_cfg=bottleneck)
    return ModelConfig(**{**base, **kw})


def test_default_has_no_norm():
    plain = MosaicAttention(attention_config(), block_attn_only=False)
    assert not plain.head_norm and not any("norm" in name for name in plain.state_dict())
    assert list(plain.state_dict()) == list(MosaicAttention(attention_config(head_norm=False), False).state_dict())


def test_flag_adds_one_weight_per_norm():
    m = MosaicAttention(attention_config(head_norm=True), block_attn_only=False)
    extra = set(m.state_dict()) - set(MosaicAttention(attention_config(), False).state_dict())
    assert extra == {"q_norm.weight", "k_norm.weight"}
    assert m.q_norm.weight.shape == m.k_norm.weight.shape == (64,)
    bare = MosaicAttention(attention_config(head_norm=True, rmsnorm_elementwise_affine=False), False)
    assert bare.head_norm and bare.q_norm.weight is None and "q_norm.weight" not in bare.state_dict()


def test_model_passes_the_flag():
    with_norm, without = Transformer(model_config(head_norm=True)), Transformer(model_config())
    extra = set(with_norm.state_dict()) - set(without.state_dict())
    blocks = [name for name, m in without.named_modules() if isinstance(m, MosaicAttention)]
    assert extra == {f"{name}.{n}_norm.weight" for name in blocks for n in "qk"}


def test_norm_is_not_the_fused_input_side():
    m = MosaicAttention(attention_config(head_norm=True), block_attn_only=False)
    m.fused_input_side = True
    assert not m._fused_input_side(torch.zeros(512, 1, 256, dtype=torch.bfloat16))


def turned(x, cos, sin):
    c, s = cos.double()[None, :, None], sin.double()[None, :, None]
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack((even * c - odd * s, odd * c + even * s), -1).flatten(-2)


def normed(x, norm, rope):
    x = x.double()
    x = x * (x.square().mean(-1, keepdim=True) + torch.finfo(torch.float32).eps).rsqrt()
    if norm.weight is not None:
        x = x * norm.weight.double()
    if rope is not None:
        x = turned(x, rope.cos_freqs, rope.sin_freqs)
    return x.to(torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("rope", ["shared", "apart", "none"])
@pytest.mark.parametrize("local", [False, True], ids=["sparse", "local"])
@pytest.mark.parametrize("affine", [True, False], ids=["weights", "ones"])
def test_attention_against_composition(rope, local, affine):
    print(f"head_norm rope={rope} local={local} affine={affine}", flush=True)
    S, B = 512, 3
    torch.manual_seed(1)
    m = MosaicAttention(attention_config(head_norm=True, rope=rope != "none", rmsnorm_elementwise_affine=affine),
                        block_attn_only=local)
    if affine:
        with torch.no_grad():
            m.q_norm.weight.uniform_(0.5, 2.0)
            m.k_norm.weight.uniform_(0.5, 2.0)
    pos = torch.rand(S, 2) * 3
    if rope != "none":
        m.q_rope.initialize_rope(pos)
        m.k_rope.initialize_rope(pos if rope == "shared" else pos + 0.25)
    m = m.to(DEV).to(torch.bfloat16)
    if rope != "none":              # the tables stay fp32, as under autocast
        for r in (m.q_rope, m.k_rope):
            r.cos_freqs, r.sin_freqs = r.cos_freqs.float(), r.sin_freqs.float()
    x = torch.randn(S, B, 256, generator=torch.Generator().manual_seed(2)).to(DEV, torch.bfloat16)
    with torch.no_grad():
        got = m(x)
        q, k, v, logits = m._projections(x)
        q, k, v = (t.unflatten(-1, (-1, 64)).transpose(0, 1) for t in (q, k, v))
        w = None if local else torch.softmax(
            logits.unflatten(-1, (4, 3)).permute(3, 1, 0, 2).float(), 0).to(x.dtype).unsqueeze(-1)
        o = mosaic_attn_func(normed(q, m.q_norm, m.q_rope), normed(k, m.k_norm, m.k_rope), v, w, block_attn_size=128,
                             sparse_block_size=64, sparse_block_count=8, block_attn_only=local, no_compression=False)
        ref = m.to_o(o.transpose(0, 1).flatten(-2))
    assert got.shape == ref.shape and torch.isfinite(got).all()
    err = ((got.double() - ref.double()).norm() / ref.double().norm()).item()
    assert err < 2 ** -8, err
    if rope != "none":              # the rotation took part
        with torch.no_grad():
            m.q_rope.cos_freqs.fill_(1.0)
            m.q_rope.sin_freqs.zero_()
            assert not torch.equal(m(x), got)


@pytest.mark.gpu
def test_scale_of_the_projections_cancels():
    """q / |q| does not change with q: to_q and to_k times 16 leave the output within the epsilon,
    where the module without the norm moves."""
    print("head_norm scale", flush=True)
    S, B = 512, 2
    x = torch.randn(S, B, 256, generator=torch.Generator().manual_seed(3)).to(DEV, torch.bfloat16)
    pos = torch.rand(S, 2, generator=torch.Generator().manual_seed(4)) * 3
    for head_norm in (True, False):
        torch.manual_seed(5)
        m = MosaicAttention(attention_config(head_norm=head_norm), block_attn_only=False)
        m.q_rope.initialize_rope(pos)
        m.k_rope.initialize_rope(pos)
        m = m.to(DEV)
        with torch.no_grad(), torch.autocast(DEV, dtype=torch.bfloat16):
            before = m(x)
            m.to_q.weight.mul_(16)
            m.to_k.weight.mul_(16)
            after = m(x)
        err = ((before.double() - after.double()).norm() / before.double().norm()).item()
        assert (err < 2 ** -8) == head_norm, (head_norm, err)


@pytest.mark.gpu
def test_unet_runs_with_head_norm():
    print("head_norm unet", flush=True)
    torch.manual_seed(0)
    model = Transformer(model_config(head_norm=True), seed=11)
    lon, lat = torch.linspace(0, 345, 24), torch.linspace(-90, 90, 13)
    model.initialize_interpolation(lon, lat)
    model.initialize_static_vars(torch.randn(24, 13, 1), lon, lat)
    model = model.to(DEV).eval()
    x, dyt = torch.randn(1, 1, 1, 24, 13, 2, device=DEV), torch.rand(1, 1, 2, device=DEV)
    with torch.no_grad(), torch.autocast(DEV, dtype=torch.bfloat16):
        out = model(x, dyt, 2)
    assert out.shape == (1, 2, 24, 13, 2) and torch.isfinite(out.float()).all()


def _module(**kw):
    torch.manual_seed(7)
    m = MosaicAttention(attention_config(head_norm=True, **kw), block_attn_only=False)
    with torch.no_grad():
        m.q_norm.weight.uniform_(0.5, 2.0)
        m.k_norm.weight.uniform_(0.5, 2.0)
    pos = torch.rand(512, 2, generator=torch.Generator().manual_seed(8)) * 3
    m.q_rope.initialize_rope(pos)
    m.k_rope.initialize_rope(pos)
    return m


class _Twice(torch.nn.Module):
    """A norm of the user's own."""

    def __init__(self, norm):
        super().__init__()
        self.norm = norm

    def forward(self, x):
        return 2 * self.norm(x)


CHANGES = {
    "hook": lambda m: m.q_norm.register_forward_hook(lambda mod, args, out: 2 * out),
    "pre-hook": lambda m: m.k_norm.register_forward_pre_hook(lambda mod, args: (args[0] * 0,)),
    "forward": lambda m: setattr(m.q_norm, "forward", lambda x: 2 * type(m.q_norm).forward(m.q_norm, x)),
    "module": lambda m: setattr(m, "k_norm", _Twice(m.k_norm)),
    "identity": lambda m: setattr(m, "q_norm", torch.nn.Identity()),
    "epsilon": lambda m: setattr(m.k_norm, "eps", 3.0),
}


@pytest.mark.parametrize("change", CHANGES)
def test_norms_that_are_not_plain_are_called(change):
    m = _module()
    assert m._fused_head_norm()
    CHANGES[change](m)
    assert not m._fused_head_norm()


def test_global_hooks_see_the_norms():
    m, seen = _module(), []
    handle = torch.nn.modules.module.register_module_forward_hook(lambda mod, args, out: seen.append(mod))
    try:
        assert not m._fused_head_norm()
    finally:
        handle.remove()
    assert m._fused_head_norm()


@pytest.mark.gpu
@pytest.mark.parametrize("change", [None, *CHANGES])
def test_norms_that_are_called_against_composition(change):
    """As the composition above, each norm's output rounded to bfloat16 before its rotation: four roundings
    of q and k where one was, 2^-9 each on scores that every block takes part in; bar 2^-7."""
    print(f"head_norm change={change}", flush=True)
    S, B = 512, 2
    m = _module().to(DEV)
    x = torch.randn(S, B, 256, generator=torch.Generator().manual_seed(2)).to(DEV, torch.bfloat16)
    with torch.no_grad(), torch.autocast(DEV, dtype=torch.bfloat16):
        before = m(x)
        if change is not None:
            CHANGES[change](m)
        got = m(x)
        q, k, v, logits = m._projections(x)
        q, k, v = (t.unflatten(-1, (-1, 64)).transpose(0, 1) for t in (q, k, v))
        w = torch.softmax(logits.unflatten(-1, (4, 3)).permute(3, 1, 0, 2).float(), 0).to(x.dtype).unsqueeze(-1)
        q, k = (turned(norm(t).double(), r.cos_freqs, r.sin_freqs).to(torch.bfloat16)
                for t, norm, r in ((q, m.q_norm, m.q_rope), (k, m.k_norm, m.k_rope)))
        o = mosaic_attn_func(q, k, v, w, block_attn_size=128, sparse_block_size=64, sparse_block_count=8,
                             block_attn_only=False, no_compression=False)
        ref = m.to_o(o.transpose(0, 1).flatten(-2))
    err = ((got.double() - ref.double()).norm() / ref.double().norm()).item()
    assert err < 2 ** -7, err
    if change is not None:
        assert ((got.double() - before.double()).norm() / before.double().norm()).item() > 2 ** -5


def test_configs_and_modules_from_before_the_flag():
    config = vars(model_config())
    del config["head_norm"]
    model = Transformer(types.SimpleNamespace(**config))
    assert not any(m.head_norm for m in model.modules() if isinstance(m, MosaicAttention))
    assert list(model.state_dict()) == list(Transformer(model_config()).state_dict())
    old = MosaicAttention(attention_config(), block_attn_only=False)     # as a pickled module has it
    old.__dict__.pop("head_norm", None)
    old.fused_input_side = True
    assert not old.head_norm and not old._fused_head_norm()
    assert not old._fused_input_side(torch.zeros(512, 1, 256, dtype=torch.bfloat16))
