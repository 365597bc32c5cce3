"""The key/value cache in 8 bits: writing and reading it, against its definition in float64 token by token."""

import ctypes
import math

import pytest
import torch

import mosaic_amd as M
from kv_cache_model import Model, attention, nearest_code
from mosaic_amd import _lib

gpu = pytest.mark.gpu
BF16, F32, I8, E4M3 = torch.bfloat16, torch.float32, torch.int8, torch.float8_e4m3fn
CODES = pytest.mark.parametrize("code", [I8, E4M3], ids=["int8", "e4m3"])


def tokens(B, n, H, dtype=BF16, seed=0, stacked=False):
    g = torch.Generator().manual_seed(seed)
    kv = torch.randn(B, n, 2 * H, 64, generator=g) * torch.exp(torch.randn(1, 1, 2 * H, 64, generator=g))
    kv = kv.to(dtype)
    k, v = kv[:, :, :H], kv[:, :, H:]
    return (k, v) if stacked else (k.contiguous(), v.contiguous())


def same(cache, model):
    """Codes (by the values they stand for), scales and means; the codes of tokens exactly."""
    k, v = M.kv_cache_read(cache, dtype=F32)
    for i, (got, scale) in enumerate(((k, cache.k_scale), (v, cache.v_scale))):
        assert torch.equal(scale.cpu().nan_to_num(-1.0), model.scale[i].float().nan_to_num(-1.0)), "kv"[i] + " scale"
        want = model.values(i)
        bad = (got.cpu() != want) & ~(got.cpu().isnan() & want.isnan())
        assert not bad.any(), ("kv"[i], int(bad.sum()), bad.nonzero()[:3].tolist())
    # the mean: exact sums (to 2^-22 for 256 of e4m3), two fp32 operations, half a step of bf16
    want = model.mean
    got = cache.k_mean.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    ok = (got - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * want.abs() + 2.0 ** -133
    assert bool((ok | want.isnan()).all())
    # the norm: a sum of 64 squares, its root and a product in fp32 (66 roundings of 2^-24, of the squares' half)
    norm = (model.codes[0] * model.scale[0].repeat_interleave(model.bs, 1)[..., None]).square().sum(-1).sqrt().unflatten(1, (-1, model.bs)).amax(2)
    got = cache.k_norm.cpu().double()
    assert torch.equal(got.isnan(), norm.isnan())
    assert bool((((got - norm).abs() <= norm * 2.0 ** -18) | norm.isnan() | (norm > 3e38)).all())


def made(B, capacity, H, bs, code):
    return M.KVCache(B, capacity, H, block_size=bs, dtype=code), Model(B, capacity, H, bs, code)


def write(cache, model, k, v, start=0, counts=None):
    on = lambda t: t.cuda() if isinstance(t, torch.Tensor) else t
    M.kv_cache_write(cache, k.cuda(), v.cuda(), on(start), on(counts))
    model.write(k, v, start, counts)


@gpu
@CODES
@pytest.mark.parametrize("B,n,H,bs,dtype", [(1, 1, 1, 64, BF16), (1, 64, 1, 64, F32), (2, 63, 3, 64, BF16), (1, 65, 5, 64, F32),
                                            (3, 129, 2, 128, BF16), (1, 300, 3, 128, F32), (2, 515, 1, 256, BF16), (1, 256, 4, 256, F32)])
def test_whole_states(code, B, n, H, bs, dtype):
    cache, model = made(B, n, H, bs, code)
    write(cache, model, *tokens(B, n, H, dtype, seed=n))
    same(cache, model)


@gpu
@CODES
def test_views_are_read_by_their_strides(code):
    cache, model = made(2, 200, 3, 64, code)
    k, v = tokens(2, 150, 3, seed=1, stacked=True)
    write(cache, model, k, v, 20)
    same(cache, model)
    k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in tokens(2, 70, 3, seed=2))       # sequence-first
    M.kv_cache_write(cache, k.transpose(0, 1).contiguous().cuda().transpose(0, 1), v.cuda(), 64)
    model.write(k, v, 64)
    same(cache, model)
    k, v = tokens(2, 70, 3, seed=3)
    odd = torch.empty(2, 70, 3, 67, dtype=BF16, device="cuda")[..., 1:65].copy_(k.cuda())            # rows of no alignment
    M.kv_cache_write(cache, odd, v.cuda()[:, :, :1].expand(-1, -1, 3, -1), 3)
    model.write(k, v[:, :, :1].expand(-1, -1, 3, -1), 3)
    same(cache, model)
    back = tokens(2, 70, 3, seed=4)
    M.kv_cache_write(cache, back[0].cuda().flip(1), back[1].cuda(), 0)
    model.write(back[0].flip(1), back[1], 0)
    same(cache, model)


@gpu
@CODES
@pytest.mark.parametrize("bs", [64, 128, 256])
def test_one_token_at_a_time(code, bs):
    """The scale grows now and then, and the tokens before are set to it."""
    cache, model = made(2, bs + 6, 2, bs, code)
    k, v = tokens(2, bs + 6, 2, seed=5)
    k[:, 10:] *= 3
    v[1, 30:] *= 7
    write(cache, model, k[:, :bs - 8], v[:, :bs - 8])
    for t in range(bs - 8, bs + 6):
        write(cache, model, k[:, t:t + 1], v[:, t:t + 1], t)
        same(cache, model)


@gpu
@CODES
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_padded_batches_and_positions_outside(code, dtype):
    B, capacity = 7, 330
    cache, model = made(B, capacity, 2, 64, code)
    write(cache, model, *tokens(B, capacity, 2, seed=6))
    start = torch.tensor([0, 1, 63, 200, -5, 328, 4000], dtype=dtype)
    counts = torch.tensor([100, 0, 2, 500, 70, 9, 3], dtype=dtype)
    write(cache, model, *tokens(B, 100, 2, F32, seed=7), start, counts)
    same(cache, model)
    write(cache, model, *tokens(B, 100, 2, seed=8), start)
    same(cache, model)
    write(cache, model, *tokens(B, 100, 2, seed=9), 17, counts)
    same(cache, model)
    if dtype is torch.int64:   # far positions stay far
        far = torch.tensor([1 << 32, -(1 << 32), 1 << 40, (1 << 32) + 5, -1 << 62, 1 << 62, 1 << 31])
        write(cache, model, *tokens(B, 100, 2, seed=10), far, counts * 0 + (1 << 33))
        same(cache, model)


@gpu
def test_later_blocks_are_left_and_the_last_one_is_cut():
    cache, model = made(1, 256, 1, 64, I8)
    write(cache, model, *tokens(1, 256, 1, seed=11))
    codes = cache.k_codes.clone()
    write(cache, model, *tokens(1, 10, 1, seed=12), 70)
    same(cache, model)
    k, _ = M.kv_cache_read(cache, dtype=F32)
    assert not k[0, 80:128].any() and k[0, 128:].any()
    assert torch.equal(cache.k_codes[:, 2:], codes[:, 2:]) and torch.equal(cache.k_codes[:, :1], codes[:, :1])


@gpu
@CODES
def test_ties_and_their_neighbours(code):
    """Values at and one float32 beside the middle between two codes, for scales that are exact and that are not."""
    top = 127.0 if code == I8 else 448.0
    for most in (top, top / 3 * 2.0 ** 20, 1.0, 3.3e-27):
        s = torch.tensor(most, dtype=torch.float64).div(top).float()
        if code == I8:
            mids = torch.arange(-126.5, 127.0, 1.0)
        else:
            grid = nearest_code(torch.arange(0, 448.5, 2.0 ** -9, dtype=torch.float64), code).unique()
            mids = ((grid[1:] + grid[:-1]) / 2).float()
            mids = torch.cat([mids, -mids])
        mid = (mids.double() * s.double()).float()
        x = torch.cat([mid, torch.nextafter(mid, torch.tensor(math.inf)), torch.nextafter(mid, torch.tensor(-math.inf))])
        x = x[x.abs() < most]
        n = -(-x.numel() // 63)
        x = torch.cat([x, x.new_zeros(63 * n - x.numel())]).view(1, n, 1, 63)
        x = torch.cat([torch.full((1, n, 1, 1), most), x], dim=-1)
        cache, model = made(1, n, 1, 64, code)
        write(cache, model, x, -x)
        same(cache, model)


@gpu
@CODES
def test_zeros_extremes_and_values_that_are_not_finite(code):
    cache, model = made(1, 64 * 8, 2, 64, code)
    k, v = tokens(1, 64 * 8, 2, F32, seed=13)
    k[0, :64] = 0
    v[0, 64:128] *= 2.0 ** -110            # zeros
    k[0, 128:192] = k[0, 128:192] / k[0, 128:192].abs().amax() * 2.0 ** -99
    v[0, 192:256] = v[0, 192:256] / v[0, 192:256].abs().amax() * 3.4e38
    k[0, 256:320, 0, 5] = math.inf
    v[0, 300, 1, 7] = math.nan
    k[0, 330, 0, 0] = -math.inf
    k[0, 400] = torch.finfo(F32).min
    write(cache, model, k, v)
    same(cache, model)
    got = M.kv_cache_read(cache, 256, 64, F32)
    assert got[0][0, :, 0].isnan().all() and got[0][0, :, 1].isfinite().all() and got[1][0, :, 1].isnan().all()
    # kept tokens of such a block keep it so; a block that begins anew is sound again
    k, v = tokens(1, 40, 2, F32, seed=14)
    write(cache, model, k, v, 300)
    same(cache, model)
    assert cache.k_scale[0, 4, 0].isnan() and cache.k_scale[0, 5, 0].isfinite()
    write(cache, model, k, v, 256)
    same(cache, model)
    assert cache.k_scale[0, 4].isfinite().all()


@gpu
@CODES
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("start,count", [(0, 0), (0, 1), (63, 2), (64, 64), (1, 199), (130, 70), (199, 1)])
def test_windows(code, dtype, start, count):
    cache, model = made(2, 200, 3, 128, code)
    write(cache, model, *tokens(2, 200, 3, seed=15))
    k, v = M.kv_cache_read(cache, start, count, dtype)
    for i, got in enumerate((k, v)):
        assert got.shape == (2, count, 3, 64) and got.dtype == dtype and got.is_contiguous()
        exact = (model.codes[i] * model.scale[i].repeat_interleave(128, 1)[..., None])[:, start:start + count]
        want = model.values(i)[:, start:start + count].to(dtype)
        if dtype == F32:
            assert torch.equal(got.cpu(), want)
        else:   # fp32, then bf16: half a step and 2^-24
            assert ((got.cpu().double() - exact).abs() <= (2.0 ** -8 + 2.0 ** -23) * exact.abs()).all()


@gpu
@CODES
def test_windows_of_each_sequence(code):
    cache, model = made(6, 200, 2, 64, code)
    write(cache, model, *tokens(6, 200, 2, seed=16))
    start = torch.tensor([0, 150, -30, 199, 200, -1000])
    for at in (start, start.int(), torch.tensor([1 << 33, -(1 << 33), 5, 64, 1 << 31, 77])):
        k, v = M.kv_cache_read(cache, at.cuda(), 90, F32)
        for i, got in enumerate((k, v)):
            pos = at.long()[:, None] + torch.arange(90)
            ok = (pos >= 0) & (pos < 200)
            want = model.values(i)[torch.arange(6)[:, None], pos.clamp(0, 199)] * ok[..., None, None]
            assert torch.equal(got.cpu(), want)


@gpu
@CODES
def test_offsets_past_32_bits(code):
    """A cache of 5.4 GB of codes for each of k and v: its last tokens, written, read and attended to."""
    n, H = 1 << 20, 80
    cache = M.KVCache(1, n, H, block_size=128, dtype=code)
    at = n - 150
    k, v = tokens(1, 150, H, seed=19)
    M.kv_cache_write(cache, k.cuda(), v.cuda(), at)
    M.kv_cache_write(cache, k[:, :3].cuda(), v[:, :3].cuda(), torch.tensor([5], device="cuda"))
    small = Model(1, 256, H, 128, code)               # the last two blocks
    small.write(k, v, 256 - 150)
    got = M.kv_cache_read(cache, at, 150, F32)
    for i in range(2):
        assert torch.equal(got[i].cpu(), small.values(i)[:, 106:])
    assert torch.equal(M.kv_cache_read(cache, torch.tensor([at], device="cuda"), 200, F32)[0][:, :150], got[0])
    q = torch.randn(1, 40, H, 64, generator=torch.Generator().manual_seed(20)).to(BF16)
    idx = torch.tensor([n // 128 - 1, n // 128 - 2]).expand(1, 40, H, 2)
    want, tol = attention(q, small.values(0), small.values(1), 0.125)
    for rows in (slice(0, 1), slice(0, 40)):          # one row, and many
        out = M.cache_attn(q[:, rows].cuda(), cache, idx[:, rows].cuda()).cpu().double()
        assert ((out - want[:, rows]).abs() <= tol[:, rows]).all()
    # the whole of it: keys of zeros all but the last, and the first few
    one = M.cache_attn(q[:, :1].cuda() * 0, cache).cpu().double()[0, 0]
    total = (small.values(1).double().sum(1)[0] + M.kv_cache_read(cache, 5, 3, F32)[1].cpu().double().sum(1)[0]) / n
    # equal scores: weights of 1, or of a block's scale each, off by 2^-8 at most
    size = (small.values(1).double().abs().sum(1)[0] + M.kv_cache_read(cache, 5, 3, F32)[1].cpu().double().abs().sum(1)[0]) / n
    assert ((one - total).abs() <= (2.0 ** -7 + 2.0 ** -12) * size + 2.0 ** -8 * total.abs()).all()


@gpu
def test_empty_writes_leave_the_cache():
    cache, model = made(2, 100, 1, 64, I8)
    write(cache, model, *tokens(2, 100, 1, seed=17))
    M.kv_cache_write(cache, *(t.cuda() for t in tokens(2, 0, 1)), 100)
    M.kv_cache_write(cache, *(t.cuda() for t in tokens(2, 5, 1)), 0, torch.zeros(2, dtype=torch.int32, device="cuda"))
    same(cache, model)


@gpu
def test_another_stream_and_a_captured_write():
    k, v = (t.cuda() for t in tokens(2, 200, 2, seed=18))
    cache, model = made(2, 256, 2, 64, I8)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        M.kv_cache_write(cache, k, v)
        got = M.kv_cache_read(cache, 0, 200, F32)
    torch.cuda.current_stream().wait_stream(stream)
    model.write(k.cpu(), v.cpu(), 0)
    assert torch.equal(got[0].cpu(), model.values(0)[:, :200])
    same(cache, model)
    # one token of each sequence at a position the graph reads: the program moves it between replays
    one = [t[:, :1].clone() for t in (k, v)]
    at = torch.tensor([200, 190], dtype=torch.int32, device="cuda")
    start = at.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        M.kv_cache_write(cache, *one, at)
        window = M.kv_cache_read(cache, at, 1, F32)
    for i in range(6):
        new = [t.cuda() for t in tokens(2, 1, 2, seed=30 + i)]
        for t, x in zip(one, new):
            t.copy_(x)
        at.copy_(start + i)
        graph.replay()
        model.write(new[0].cpu(), new[1].cpu(), (start + i).cpu())
        torch.cuda.synchronize()
        same(cache, model)
        assert torch.equal(window[1].cpu(), M.kv_cache_read(cache, at, 1, F32)[1].cpu())


# ------------------------------------------------------------------ refusals

def cpu_cache(**kw):
    return M.KVCache(**{**dict(batch=2, capacity=100, kv_heads=3, device="cpu"), **kw})


@pytest.mark.parametrize("kw,error", [
    (dict(batch=0), ValueError), (dict(capacity=0), ValueError), (dict(kv_heads=0), ValueError), (dict(kv_heads=65536), ValueError), (dict(block_size=32), ValueError),
    (dict(block_size=512), ValueError), (dict(dtype=torch.uint8), TypeError), (dict(dtype=torch.float8_e5m2), TypeError),
    (dict(capacity=1 << 31), ValueError), (dict(batch=1 << 20, capacity=1 << 20), ValueError),
])
def test_caches_that_are_refused(kw, error):
    with pytest.raises(error, match="KVCache"):
        cpu_cache(**kw)


def test_what_a_cache_says_of_itself():
    c = cpu_cache(capacity=130, block_size=128, dtype=E4M3)
    assert (c.batch, c.num_blocks, c.kv_heads, c.block_size, c.capacity, c.dtype) == (2, 2, 3, 128, 130, E4M3)
    assert c.k_scale.shape == (2, 2, 3) and c.k_mean.shape == (2, 2, 3, 64) and c.device.type == "cpu"
    assert "float8_e4m3fn" in repr(c)
    with pytest.raises(AttributeError):
        c.k_scale = None


def test_copies_have_storage_of_their_own():
    import copy
    import pickle

    c = cpu_cache()
    c.k_scale.fill_(2.0)
    for other in (copy.deepcopy(c), pickle.loads(pickle.dumps(c))):
        assert torch.equal(other.k_scale, c.k_scale) and other._c.k_scale == other.k_scale.data_ptr() != c.k_scale.data_ptr()
        assert (other._c.batch, other._c.capacity) == (2, 100) and other.device == c.device


K = torch.zeros(2, 5, 3, 64)


@pytest.mark.parametrize("k,v,kw,error,match", [
    (K[0], K, {}, ValueError, "k "), (K[:1], K[:1], {}, ValueError, "k "), (K[:, :, :2], K[:, :, :2], {}, ValueError, "k "),
    (K[..., :32], K[..., :32], {}, ValueError, "k "), (K, K[:, :4], {}, ValueError, "disagree"), (K, K[0], {}, ValueError, "disagree"), (K, K.bfloat16(), {}, ValueError, "disagree"),
    (K.half(), K.half(), {}, TypeError, "float16"), (K.double(), K.double(), {}, TypeError, "float64"),
    (K, K, dict(start=-1), ValueError, "cache of 100"), (K, K, dict(start=96), ValueError, "cache of 100"),
    (K, K, dict(start=torch.zeros(3, dtype=torch.int32)), ValueError, "start"), (K, K, dict(start=torch.zeros(2)), TypeError, "start"),
    (K, K, dict(counts=torch.zeros(2, 1, dtype=torch.int32)), ValueError, "counts"), (K, K, dict(counts=torch.zeros(2)), TypeError, "counts"),
    (K.clone().requires_grad_(), K, {}, RuntimeError, "no backward"), (K, K, {}, ValueError, "device"),
])
def test_writes_that_are_refused(k, v, kw, error, match):
    with pytest.raises(error, match=match):
        M.kv_cache_write(cpu_cache(), k, v, **kw)


@pytest.mark.parametrize("args,error,match", [
    ((0, 101), ValueError, "cache of 100"), ((-1, 5), ValueError, "cache of 100"), ((0, -1), ValueError, "count"),
    ((0, 5, torch.float16), TypeError, "float16"), ((torch.zeros(2, dtype=torch.int32),), ValueError, "count"),
    ((torch.zeros(1, dtype=torch.int32), 5), ValueError, "start"), ((0, 5), ValueError, "device"),
])
def test_reads_that_are_refused(args, error, match):
    with pytest.raises(error, match=match):
        M.kv_cache_read(cpu_cache(), *args)


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="forward mode"):
            M.kv_cache_write(cpu_cache(), K, fwad.make_dual(K, K))


FAKE = 1 << 20   # aligned host address; the checks fail before anything reads it


def c_cache(**kw):
    c = _lib.Cache(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 4, 3, 64, _lib.CODE_INT8, 250)
    for name, x in kw.items():
        setattr(c, name, x)
    return c


@pytest.mark.parametrize("kw,status", [
    (dict(k_codes=None), 1), (dict(v_codes=None), 1), (dict(k_scale=None), 1), (dict(v_scale=None), 1), (dict(k_norm=None), 1), (dict(k_mean=None), 1),
    (dict(batch=0), 8), (dict(num_blocks=0), 8), (dict(num_kv_heads=0), 3), (dict(num_kv_heads=65536), 3), (dict(block_size=32), 4), (dict(block_size=192), 4),
    (dict(code_type=2), 11), (dict(capacity=257), 8), (dict(capacity=0), 8), (dict(k_codes=FAKE + 8), 7), (dict(k_scale=FAKE + 2), 7),
    (dict(k_mean=FAKE + 4), 7), (dict(num_blocks=1 << 26, capacity=1), 8), (dict(batch=1 << 30), 8),
])
def test_c_entries_refuse_caches(kw, status):
    L, c, rows = _lib.lib(), c_cache(**kw), _lib.Bnhd(FAKE, 960, 192, 64)
    assert L.mosaic_kv_cache_write(ctypes.byref(c), rows, rows, 1, 64, 5, 0, None, None, None) == status
    assert L.mosaic_kv_cache_read(ctypes.byref(c), 1, 64, 5, 0, None, FAKE, FAKE, None) == status
    assert L.mosaic_cache_attn_fwd(rows, ctypes.byref(c), None, None, 5, 6, 64, 0, 0.0, FAKE, FAKE, 1 << 40, None) == status
    assert L.mosaic_cache_attn_fwd_workspace_size(ctypes.byref(c), 5, 6, 0) == 0


def test_c_entries_refuse_arguments():
    L, c, rows = _lib.lib(), ctypes.byref(c_cache()), _lib.Bnhd(FAKE, 960, 192, 64)
    put = lambda k=rows, dt=1, d=64, n=5, start=0, starts=None, counts=None, cache=c: L.mosaic_kv_cache_write(cache, k, rows, dt, d, n, start,
                                                                                                              starts, counts, None)
    assert put(cache=None) == 1 and put(k=_lib.Bnhd(None, 960, 192, 64)) == 1
    assert put(d=128) == 2 and put(dt=5) == 11 and put(n=0) == 8 and put(start=246) == 8 and put(start=-1) == 8
    assert put(k=_lib.Bnhd(FAKE + 8, 960, 192, 64)) == 7 and put(k=_lib.Bnhd(FAKE, 960, 190, 64)) == 7
    assert put(starts=FAKE + 2) == 7 and put(counts=FAKE + 1) == 7
    huge = ctypes.byref(c_cache(batch=1, num_blocks=1 << 24, num_kv_heads=1, capacity=1 << 30))   # 2^24 workgroups of 256 threads
    assert put(n=1 << 30, cache=huge) == 8 and L.mosaic_kv_cache_read(huge, 1, 64, 1 << 30, 0, None, FAKE, FAKE, None) == 8
    get = lambda n=5, start=0, k=FAKE, v=FAKE: L.mosaic_kv_cache_read(c, 1, 64, n, start, None, k, v, None)
    assert get(k=None) == 1 and get(v=FAKE + 8) == 7 and get(n=251) == 8 and get(start=1 << 40) == 8
