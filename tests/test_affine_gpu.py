"""The group-affine cache on the GPU against plain 64-bit forms (tests/affine_oracle.py)."""
import math

import pytest
import torch

import kaplumba_amd as K
from kaplumba_amd import AffineState, append_affine_kv, attention_affine, dequantize_affine
from kaplumba_amd.affine import affine_state
from tests import affine_oracle as A

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def vectors(seed, shape, dtype, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    scale = torch.exp(torch.randn(1, shape[1], 1, shape[3], generator=g) * spread)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def filled(seed, B, H, T, dim, bits, group, dtype, device, cap=None, spread=0.5, times=1.0):
    """(state viewing T tokens of capacity buffers on the device, f64 values) of quantized vectors."""
    x = (vectors(seed, (B, H, T, dim), torch.float32, spread) * times).to(dtype)
    words, params = A.quantize(x, bits, group)
    st = affine_state(B, H, cap or T, dim, bits, group, dtype, device)
    st.codes.view(torch.int32)[:, :, :T] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32).to(device)
    st.params[:, :, :T] = params.to(device)
    return AffineState(st.codes[:, :, :T], st.params[:, :, :T]), A.values(words, params, bits, group)


# ------------------------------------------------------------ write, read back ---
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kb,vb", [(4, 4), (8, 4), (4, 8), (8, 8)])
@pytest.mark.parametrize("D,Dv,group", [(32, 32, 32), (64, 64, 64), (128, 128, 64), (96, 160, 32), (192, 128, 64),
                                        (256, 128, 128), (512, 384, 128)])
def test_append_and_dequantize(device, dtype, kb, vb, D, Dv, group):
    dt, B, H, L, cap, at = DTYPES[dtype], 2, 3, 7, 20, 5
    k, v = vectors(1, (B, H, L, D), dt), vectors(2, (B, H, L, Dv), dt)
    ks, vs = (affine_state(B, H, cap, d, b, group, dt, device) for d, b in ((D, kb), (Dv, vb)))
    for st in (ks, vs):
        st.codes.view(torch.int32).fill_(-1234567)
        st.params.fill_(7.0)
    append_affine_kv(k.to(device), v.to(device), ks, vs, at, group)
    for x, st, bits in ((k, ks, kb), (v, vs, vb)):
        words, params = A.quantize(x, bits, group)
        assert torch.equal(A.words_of(st.codes)[:, :, at:at + L], words)
        assert bool((st.params[:, :, at:at + L].cpu() == params).all())
        # rows around the new ones keep what they held
        assert (st.codes.view(torch.int32)[:, :, :at] == -1234567).all() and (st.params[:, :, :at] == 7).all()
        assert (st.codes.view(torch.int32)[:, :, at + L:] == -1234567).all() and (st.params[:, :, at + L:] == 7).all()
        new = AffineState(st.codes[:, :, at:at + L], st.params[:, :, at:at + L])
        want = A.values(words, params, bits, group)
        for out in (None, torch.float32, torch.float16, torch.bfloat16):
            got = dequantize_affine(new, group, out)
            assert got.dtype == (out or dt) and got.is_contiguous()
            tol = want.abs() * (A.half_step(got.dtype) + 2.0 ** -24 * (out != torch.float32))
            if out == torch.float32 or (out is None and dt == torch.float32):
                # an f32 scale times a code is rounded with the sum: one rounding
                tol = want.abs() * 2.0 ** -24
            if got.dtype == torch.float16:
                tol = tol + 2.0 ** -25
            assert ((got.cpu().double() - want).abs() <= tol + 1e-45).all()
        # half a step of the stored scale, and what its rounding leaves at the top of the range
        step = params[..., 0].double().repeat_interleave(group, -1)
        left = (2 ** bits - 1) * A.half_step(dt)
        assert ((x.double() - want).abs() <= step * (0.5 + left) + 1e-30).all()


def test_append_strides_and_stream(device):
    B, H, L, D = 2, 4, 9, 128
    x = vectors(3, (B, H, L, 3 * D), torch.bfloat16).to(device)
    k, v = x[..., :D], x[..., D:2 * D].transpose(1, 2).contiguous().transpose(1, 2)
    odd = vectors(4, (B, H, L, D + 1), torch.bfloat16).to(device)[..., 1:]
    flat = vectors(5, (1, 1, 1, B * H * L * D + 1), torch.bfloat16).to(device).flatten()
    off = flat[1:].view(B, H, L, D)                      # contiguous, but not 16-byte aligned
    assert off.is_contiguous() and off.data_ptr() % 16
    for kk, vv in ((k, v), (odd, v), (off, v), (k, off), (k.transpose(2, 3).contiguous().transpose(2, 3), odd)):
        ks, vs = (affine_state(B, H, L, D, 4, 64, torch.bfloat16, device) for _ in range(2))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            append_affine_kv(kk, vv, ks, vs, 0)
        torch.cuda.current_stream().wait_stream(side)
        for t, st in ((kk, ks), (vv, vs)):
            words, params = A.quantize(t.cpu(), 4, 64)
            assert torch.equal(A.words_of(st.codes), words) and torch.equal(st.params.cpu(), params)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bits", [4, 8])
def test_append_special_values(device, dtype, bits):
    dt, group = DTYPES[dtype], 32
    big, tiny = torch.finfo(dt).max, torch.finfo(dt).tiny
    rows = [torch.zeros(64), torch.full((64,), -3.5), torch.linspace(-big, big, 64, dtype=torch.float64),
            torch.linspace(0, tiny, 64, dtype=torch.float64), torch.arange(64) * 0.5, -torch.arange(64) * 0.25,
            torch.tensor([math.inf] + [1.0] * 63), torch.tensor([1.0] * 40 + [math.nan] + [2.0] * 23),
            torch.tensor([-math.inf] * 64), torch.tensor([0.0, -0.0] * 32)]
    x = torch.stack([r.to(dt) for r in rows])[None, None]
    ks, vs = (affine_state(1, 1, len(rows), 64, bits, group, dt, device) for _ in range(2))
    append_affine_kv(x.to(device), x.to(device), ks, vs, 0, group)
    words, params = A.quantize(x, bits, group)
    for st in (ks, vs):
        assert torch.equal(A.words_of(st.codes), words)
        got = st.params.cpu()
        assert torch.equal(torch.nan_to_num(got.double(), nan=1e300), torch.nan_to_num(params.double(), nan=1e300))
    back = dequantize_affine(ks, group).cpu()
    assert torch.isnan(back[0, 0, 6, :32]).all() and torch.equal(back[0, 0, 6, 32:], x[0, 0, 6, 32:])
    assert torch.equal(back[0, 0, 0], x[0, 0, 0]) and torch.equal(back[0, 0, 1], x[0, 0, 1])


# ------------------------------------------------------------------- attention ---
def check(device, q, ks, vs, k64, v64, group, scale, dt, kb, **kw):
    got = attention_affine(q.to(device), ks, vs, group, scale, **{
        n: (x.to(device) if isinstance(x, torch.Tensor) else x) for n, x in kw.items()})
    assert got.shape == q.shape[:3] + (v64.shape[-1],) and got.dtype == dt
    want, _, p = A.attention(q, k64, v64, scale, **kw)
    rows = q.shape[1] // k64.shape[1] * q.shape[2]
    tol = A.attention_tolerance(q, ks.params.cpu(), kb, v64, want, p, scale, dt, group, rounded=rows > 16)
    off = (got.cpu().double() - want).abs()
    assert (off <= tol).all(), f"off by {(off / tol).max():.3g} of the tolerance at {(off / tol).argmax()}"
    return got


SHAPES = [  # B, Hq, Hkv, L, T, D, Dv, group
    (1, 4, 1, 1, 1, 128, 128, 64),
    (1, 32, 8, 1, 300, 128, 128, 64),
    (2, 8, 8, 1, 65, 64, 64, 32),
    (2, 14, 2, 1, 1000, 128, 128, 128),
    (1, 2, 1, 3, 77, 64, 64, 64),
    (3, 6, 2, 5, 130, 96, 96, 32),
    (1, 8, 2, 4, 513, 256, 256, 64),
    (1, 8, 1, 8, 257, 192, 128, 64),
    (1, 4, 2, 2, 40, 32, 160, 32),
    (1, 2, 1, 1, 90, 512, 384, 128),
    (1, 4, 2, 60, 190, 320, 96, 32),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kb,vb", [(4, 4), (8, 4), (8, 8), (4, 8)])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention(device, dtype, kb, vb, shape):
    B, Hq, Hkv, L, T, D, Dv, group = shape
    dt = DTYPES[dtype]
    ks, k64 = filled(5, B, Hkv, T, D, kb, group, dt, device, cap=T + 3)
    vs, v64 = filled(6, B, Hkv, T, Dv, vb, group, dt, device, cap=T + 3)
    q = vectors(7, (B, Hq, L, D), dt, 0.0)
    check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, kb, causal=L > 1)
    if L > 1:
        check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, kb)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("L,T,D,group", [(17, 64, 128, 64), (100, 100, 64, 32), (65, 400, 128, 128), (33, 129, 256, 64),
                                         (70, 333, 96, 32), (130, 700, 128, 64), (1, 500, 128, 64)])
def test_many_rows(device, dtype, L, T, D, group):
    dt, B, Hq, Hkv = DTYPES[dtype], 2, 8, 2
    ks, k64 = filled(8, B, Hkv, T, D, 4, group, dt, device, cap=T + 1)
    vs, v64 = filled(9, B, Hkv, T, D, 8, group, dt, device, cap=T + 1)
    q = vectors(10, (B, Hq, L, D), dt, 0.0)
    check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, 4, causal=True)
    check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, 4, causal=True,
          seq_lens=torch.tensor([T, max(1, T // 3)], dtype=torch.int32))


@pytest.mark.parametrize("kb,vb", [(4, 4), (8, 4), (8, 8)])
@pytest.mark.parametrize("D,Dv,group", [(64, 64, 32), (64, 64, 64), (96, 96, 32), (128, 128, 32), (128, 128, 64),
                                        (128, 128, 128), (192, 128, 32), (192, 128, 64), (256, 256, 32), (256, 256, 64),
                                        (256, 256, 128)])
def test_layouts(device, kb, vb, D, Dv, group):
    """Each layout's kernels: 2, 10, 40 and 180 query rows a kv head, with and without a mask; the last at enough
    tokens for the many-rows kernel at every head dim."""
    dt, B, Hq, Hkv = torch.bfloat16, 2, 4, 2
    for L, T in ((1, 130), (5, 70), (20, 577), (90, 12001)):
        ks, k64 = filled(30, B, Hkv, T, D, kb, group, dt, device)
        vs, v64 = filled(31, B, Hkv, T, Dv, vb, group, dt, device)
        q = vectors(32, (B, Hq, L, D), dt, 0.0)
        check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, kb, causal=True)
        if T < 1000:
            check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, kb, mask=mask_of("bool", B, Hq, L, T))


@pytest.mark.parametrize("L", [1, 3, 40])
@pytest.mark.parametrize("dtype,D,group", [("bf16", 128, 64), ("f16", 64, 32), ("f32", 128, 64), ("bf16", 384, 64)])
def test_ragged_and_padded(device, dtype, L, D, group):
    dt, B, Hq, Hkv, T = DTYPES[dtype], 6, 8, 2, 300
    ks, k64 = filled(11, B, Hkv, T, D, 8, group, dt, device, cap=512)
    vs, v64 = filled(12, B, Hkv, T, D, 4, group, dt, device, cap=512)
    q = vectors(13, (B, Hq, L, D), dt, 0.0)
    starts = torch.tensor([0, 299, 100, 0, 65, 300], dtype=torch.int32)
    lens = torch.tensor([300, 300, 100, 1, 256, 300], dtype=torch.int32)  # rows 2 and 5 hold no token
    for kw in (dict(seq_starts=starts), dict(seq_lens=lens), dict(seq_starts=starts, seq_lens=lens)):
        for causal in (False, True):
            if causal and L == 1:
                continue
            got = check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, 8, causal=causal, **kw)
            if len(kw) == 2:
                assert (got[2] == 0).all() and (got[5] == 0).all()


def mask_of(kind, B, Hq, L, T, seed=3):
    g = torch.Generator().manual_seed(seed)
    if kind == "bool":
        m = torch.rand(B, 1, L, T, generator=g) < 0.3
        m[0, 0, 0] = False                     # a row that sees nothing
        return m
    if kind == "window":
        i, t = torch.arange(T - L, T)[:, None], torch.arange(T)[None]
        return (t <= i) & (i < t + 20)
    m = torch.randn(B, Hq, L, T, generator=g)
    m[torch.rand(B, Hq, L, T, generator=g) < 0.3] = -math.inf
    m[0, 0, 0] = -math.inf                     # zeros come out
    m[-1, -1, -1] = torch.finfo(torch.float32).min
    if kind == "add_bf16":
        m = m.to(torch.bfloat16)
        m[-1, -1, -1] = torch.finfo(torch.bfloat16).min
    elif kind == "add_f16":
        m = m.to(torch.float16)
        m[-1, -1, -1] = torch.finfo(torch.float16).min
    return m


@pytest.mark.parametrize("kind", ["bool", "window", "add_f32", "add_f16", "add_bf16"])
@pytest.mark.parametrize("dtype,L,D,group", [("bf16", 1, 128, 64), ("f16", 5, 64, 64), ("f32", 3, 128, 64),
                                             ("bf16", 50, 128, 64), ("f16", 70, 64, 32), ("bf16", 37, 256, 128),
                                             ("bf16", 20, 288, 32)])
def test_masks(device, kind, dtype, L, D, group):
    dt, B, Hq, Hkv, T = DTYPES[dtype], 2, 8, 2, 210
    ks, k64 = filled(14, B, Hkv, T, D, 4, group, dt, device, cap=256)
    vs, v64 = filled(15, B, Hkv, T, D, 4, group, dt, device, cap=256)
    q = vectors(16, (B, Hq, L, D), dt, 0.0)
    m = mask_of(kind, B, Hq, L, T)
    got = check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, 4, mask=m)
    if kind.startswith("add"):
        assert (got[0, 0, 0] == 0).all()
    check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, 4, mask=m, seq_lens=torch.tensor([T, 77]),
          causal=L > 1)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("L,D", [(1, 128), (6, 128), (40, 128), (3, 384)])
def test_masked_tokens_may_hold_nan(device, dtype, L, D):
    dt, B, Hq, Hkv, T, group = DTYPES[dtype], 1, 4, 1, 150, 64
    ks, k64 = filled(17, B, Hkv, T, D, 4, group, dt, device)
    vs, v64 = filled(18, B, Hkv, T, D, 4, group, dt, device)
    keep = torch.ones(T, dtype=torch.bool)
    keep[20:60] = False
    keep[-1] = False
    for st, bad in ((ks, math.nan), (vs, math.inf), (vs, math.nan), (ks, -math.inf)):
        st.params[:, :, (~keep).nonzero().flatten().to(device)] = bad
        st.codes.view(torch.int32)[:, :, (~keep).nonzero().flatten().to(device)] = -1
    k64[:, :, ~keep], v64[:, :, ~keep] = 0.0, 0.0
    q = vectors(19, (B, Hq, L, D), dt, 0.0)
    add = torch.where(keep, 0.0, -math.inf).expand(L, T)
    for m in (keep.expand(L, T), add):
        got = attention_affine(q.to(device), ks, vs, group, 0.1, mask=m.to(device)).cpu()
        want, _, p = A.attention(q, k64, v64, 0.1, mask=m)
        tol = A.attention_tolerance(q, torch.nan_to_num(ks.params.cpu().double(), 0, 0, 0), 4, v64, want, p, 0.1, dt,
                                    group, rounded=Hq * L > 16)
        assert ((got.double() - want).abs() <= tol).all()
    # a token that is attended to and holds NaN shows
    ks.params[:, :, (~keep).nonzero().flatten().to(device)] = 0.1
    vs.params[:, :, (~keep).nonzero().flatten().to(device)] = math.nan
    out = attention_affine(q.to(device), ks, vs, group, 0.1)
    assert torch.isnan(out).all()


@pytest.mark.parametrize("L", [1, 5, 50])
@pytest.mark.parametrize("D,group", [(128, 64), (64, 32), (256, 128)])
@pytest.mark.parametrize("dtype,key,value", [("bf16", 1e6, 1e7), ("bf16", 1e-7, 1e-6), ("bf16", 2.0 ** -16, 2.0 ** -16),
                                             ("bf16", 1e20, 1e30), ("bf16", 1e-20, 1e-30), ("f16", 2000.0, 2000.0),
                                             ("f16", 2.0 ** -10, 2.0 ** -12)])
def test_sizes_of_keys_and_values(device, dtype, key, value, D, group, L):
    """Keys and values far from one, some tokens' alone and all of them: sixteen bits on the way to the products do not
    show in what comes out."""
    dt, B, Hq, Hkv, T = DTYPES[dtype], 1, 8, 2, 210
    ks, k64 = filled(26, B, Hkv, T, D, 4, group, dt, device, times=key)
    vs, v64 = filled(27, B, Hkv, T, D, 4, group, dt, device, times=value)
    q = (vectors(28, (B, Hq, L, D), torch.float32, 0.0) / key).to(dt)
    check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, 4, causal=True)
    check(device, q, ks, vs, k64, v64, group, -1 / math.sqrt(D), dt, 4, mask=mask_of("bool", B, Hq, L, T))
    # a few tokens of another size among ordinary ones
    k1, k164 = filled(26, B, Hkv, T, D, 4, group, dt, device)
    v1, v164 = filled(27, B, Hkv, T, D, 4, group, dt, device)
    for i in (0, 63, 64, 100, 209):
        for st, other, x, y in ((k1, ks, k164, k64), (v1, vs, v164, v64)):
            st.codes.view(torch.int32)[:, :, i] = other.codes.view(torch.int32)[:, :, i]
            st.params[:, :, i] = other.params[:, :, i]
            x[:, :, i] = y[:, :, i]
    q = vectors(28, (B, Hq, L, D), dt, 0.0)
    check(device, q, ks, v1, k64, v164, group, 0.0, dt, 4)
    check(device, q, k1, v1, k164, v164, group, 1 / math.sqrt(D) / max(key, 1.0), dt, 4)


# 512 query rows a kv head over 2999 tokens: past what the few-rows kernel takes at every head dim
MANY = [("bf16", 128, 128, 64), ("f16", 64, 64, 32), ("bf16", 96, 96, 32), ("f16", 192, 128, 64), ("bf16", 256, 256, 128)]


def many(seed, dtype, D, Dv, group, device, kb=4, vb=4, key=1.0, value=1.0):
    dt, B, Hq, Hkv, L, T = DTYPES[dtype], 2, 8, 2, 128, 2999
    ks, k64 = filled(seed, B, Hkv, T, D, kb, group, dt, device, cap=3001, times=key)
    vs, v64 = filled(seed + 1, B, Hkv, T, Dv, vb, group, dt, device, cap=3001, times=value)
    q = (vectors(seed + 2, (B, Hq, L, D), torch.float32, 0.0) / key).to(dt)
    return q, ks, vs, k64, v64, 1 / math.sqrt(D), dt


@pytest.mark.parametrize("kind", ["bool", "window", "add_f32", "add_f16", "add_bf16"])
@pytest.mark.parametrize("dtype,D,Dv,group", MANY)
def test_many_rows_masks(device, kind, dtype, D, Dv, group):
    q, ks, vs, k64, v64, scale, dt = many(40, dtype, D, Dv, group, device, 8, 8)
    m = mask_of(kind, 2, 8, 128, 2999)
    got = check(device, q, ks, vs, k64, v64, group, scale, dt, 8, mask=m)
    if kind.startswith("add"):
        assert (got[0, 0, 0] == 0).all()
    check(device, q, ks, vs, k64, v64, group, scale, dt, 8, mask=m, seq_lens=torch.tensor([2999, 1777]), causal=True)


@pytest.mark.parametrize("dtype,D,Dv,group", MANY)
def test_many_rows_ragged_and_padded(device, dtype, D, Dv, group):
    q, ks, vs, k64, v64, scale, dt = many(43, dtype, D, Dv, group, device, 8, 4)
    for starts, lens in (([0, 1500], [2999, 2000]), ([2998, 0], [2999, 1]), ([7, 2999], [71, 2999])):
        starts, lens = (torch.tensor(t, dtype=torch.int32) for t in (starts, lens))
        for causal in (False, True):
            check(device, q, ks, vs, k64, v64, group, scale, dt, 8, causal=causal, seq_lens=lens, seq_starts=starts)


@pytest.mark.parametrize("dtype,D,Dv,group", MANY)
def test_many_rows_masked_tokens_may_hold_nan(device, dtype, D, Dv, group):
    q, ks, vs, k64, v64, scale, dt = many(46, dtype, D, Dv, group, device)
    keep = torch.ones(2999, dtype=torch.bool)
    keep[torch.tensor([0, 1, 70, 500, 501, 1023, 2047, 2998])] = False
    hidden = (~keep).nonzero().flatten().to(device)
    for st, bad in ((ks, math.nan), (vs, math.inf), (vs, math.nan)):
        st.params[:, :, hidden] = bad
        st.codes.view(torch.int32)[:, :, hidden] = -1
    k64[:, :, ~keep], v64[:, :, ~keep] = 0.0, 0.0
    for m in (keep.expand(128, 2999), torch.where(keep, 0.0, -math.inf).expand(128, 2999)):
        got = attention_affine(q.to(device), ks, vs, group, scale, mask=m.to(device)).cpu()
        want, _, p = A.attention(q, k64, v64, scale, mask=m)
        tol = A.attention_tolerance(q, ks.params.cpu(), 4, v64, want, p, scale, dt, group, rounded=True)
        assert ((got.double() - want).abs() <= tol).all()
    ks.params[:, :, hidden] = 0.1
    assert torch.isnan(attention_affine(q.to(device), ks, vs, group, scale)).all()


@pytest.mark.parametrize("dtype,key,value", [("bf16", 1e6, 1e7), ("bf16", 1e-7, 1e-6), ("bf16", 2.0 ** -16, 2.0 ** -16),
                                             ("bf16", 1e20, 1e30), ("f16", 2000.0, 2000.0)])
@pytest.mark.parametrize("D,group", [(128, 64), (64, 32), (256, 128)])
def test_many_rows_sizes_of_keys_and_values(device, dtype, key, value, D, group):
    q, ks, vs, k64, v64, scale, dt = many(49, dtype, D, D, group, device, 8, 4, key, value)
    _, k1, v1, k164, v164, _, _ = many(49, dtype, D, D, group, device, 8, 4)
    for i in (0, 63, 64, 1000, 2998):  # a few tokens of another size among ordinary ones
        for st, other, x, y in ((k1, ks, k164, k64), (v1, vs, v164, v64)):
            st.codes.view(torch.int32)[:, :, i] = other.codes.view(torch.int32)[:, :, i]
            st.params[:, :, i] = other.params[:, :, i]
            x[:, :, i] = y[:, :, i]
    q1 = (q.double() * key).to(dt)
    check(device, q1, k1, v1, k164, v164, group, scale / max(key, 1.0), dt, 8, causal=True)
    check(device, q, ks, vs, k64, v64, group, -scale, dt, 8, causal=True)


@pytest.mark.parametrize("kind", ["bool", "window", "add_f16"])
@pytest.mark.parametrize("dtype,L,D,group", [("bf16", 1, 128, 64), ("f16", 5, 64, 64), ("bf16", 3, 192, 32)])
def test_masks_over_many_tokens(device, kind, dtype, L, D, group):
    """Few rows of enough tokens that the ranges of the mask are found first."""
    dt, B, Hq, Hkv, T = DTYPES[dtype], 2, 8, 2, 66001
    ks, k64 = filled(52, B, Hkv, T, D, 4, group, dt, device, cap=T + 3)
    vs, v64 = filled(53, B, Hkv, T, D, 4, group, dt, device, cap=T + 3)
    q = vectors(54, (B, Hq, L, D), dt, 0.0)
    m = mask_of(kind, B, Hq, L, T)
    check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, 4, mask=m)
    check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, 4, mask=m, causal=L > 1,
          seq_lens=torch.tensor([T, 777]), seq_starts=torch.tensor([60001, 0]))
    near = torch.zeros(L, T, dtype=torch.bool)  # a short window far into the cache, and a row without one
    near[:, 50000:50070] = True
    near[0, :] = L == 1
    check(device, q, ks, vs, k64, v64, group, 1 / math.sqrt(D), dt, 4, mask=near)


def test_many_splits_equal_few(device):
    """A long cache, whose tokens many workgroups share, and the same call over two halves joined by hand."""
    B, Hq, Hkv, T, D, group = 1, 8, 2, 20011, 128, 64
    dt = torch.bfloat16
    ks, k64 = filled(20, B, Hkv, T, D, 4, group, dt, device)
    vs, v64 = filled(21, B, Hkv, T, D, 4, group, dt, device)
    q = vectors(22, (B, Hq, 1, D), dt, 0.0)
    check(device, q, ks, vs, k64, v64, group, 0.3, dt, 4)
    q = vectors(22, (B, Hq, 4, D), dt, 0.0)
    check(device, q, ks, vs, k64, v64, group, 0.3, dt, 4, causal=True)


def test_large_scores(device):
    """Scores of thousands: one key has all the weight, whatever the split."""
    dt, T, D, group = torch.bfloat16, 700, 128, 64
    ks, k64 = filled(23, 1, 2, T, D, 8, group, dt, device)
    vs, v64 = filled(24, 1, 2, T, D, 8, group, dt, device)
    q = vectors(25, (1, 8, 1, D), dt, 0.0)
    got = attention_affine(q.to(device), ks, vs, group, 300.0).cpu().double()
    want, s, p = A.attention(q, k64, v64, 300.0)
    sure = p.amax(-1) > 1 - 2.0 ** -20
    assert sure.any()
    assert ((got - want).abs() <= want.abs() * 2.0 ** -8 + 1e-3)[sure].all()


# ------------------------------------------------------------ graphs and streams ---
def test_graph_replays(device):
    """Append, read back and attention captured together and replayed with eager work between."""
    dt, B, H, Hq, D, T, group = torch.bfloat16, 2, 2, 8, 128, 600, 64
    ks, _ = filled(26, B, H, T, D, 4, group, dt, device)
    vs, _ = filled(27, B, H, T, D, 4, group, dt, device)
    k, v = (vectors(s, (B, H, 1, D), dt).to(device) for s in (28, 29))
    q = vectors(30, (B, Hq, 1, D), dt, 0.0).to(device)

    def step():
        append_affine_kv(k, v, ks, vs, T - 1, group)
        return attention_affine(q, ks, vs, group, 0.1), dequantize_affine(ks, group)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, back = step()
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(31, 36):
        for t, s in ((k, seed), (v, seed + 50), (q, seed + 90)):
            t.copy_(vectors(s, t.shape, dt).to(device))
        graph.replay()
        torch.cuda.synchronize()
        got, got_back = out.clone(), back.clone()
        want, want_back = step()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(got_back, want_back)


def test_rows_do_not_depend_on_the_batch(device):
    """The same sequence alone and in a batch, and twice in one batch."""
    dt, D, T, group = torch.float16, 128, 333, 64
    ks, _ = filled(40, 1, 2, T, D, 8, group, dt, device)
    vs, _ = filled(41, 1, 2, T, D, 4, group, dt, device)
    q = vectors(42, (1, 8, 1, D), dt, 0.0).to(device)
    one = attention_affine(q, ks, vs, group, 0.1)
    twice = [AffineState(*(t.repeat(2, *([1] * (t.dim() - 1))) if t.dtype != torch.uint32 else
                           t.view(torch.int32).repeat(2, 1, 1, 1).view(torch.uint32) for t in st)) for st in (ks, vs)]
    two = attention_affine(q.repeat(2, 1, 1, 1), *twice, group, 0.1)
    assert torch.equal(two[0], two[1])
    off = (two[:1].double() - one.double()).abs().amax()
    assert off <= 2 * 2.0 ** -11 * one.double().abs().amax()


# ------------------------------------------------------------------- the cache ---
def test_cache_through_a_layer(device):
    """Prompt, decode steps, trim, growth, save and load, all through the cache class and the layer calls."""
    B, Hq, H, D, dt = 2, 8, 2, 128, torch.bfloat16
    caches = K.make_prompt_cache(num_layers=1, kv_bits=8, val_bits=4)
    cache = caches[0]
    assert isinstance(cache, K.QuantizedKVCache) and cache.empty()
    xs = [(vectors(50 + i, (B, Hq, L, D), dt, 0.0), vectors(60 + i, (B, H, L, D), dt), vectors(70 + i, (B, H, L, D), dt))
          for i, L in enumerate((250, 1, 1, 9))]
    k64, v64 = [], []
    for q, k, v in xs:
        L = q.shape[2]
        mask = cache.make_mask(L)
        ks, vs = cache.update_and_fetch(k.to(device), v.to(device))
        assert ks.shape == (B, H, cache.offset, D)
        out = K.scaled_dot_product_attention(q.to(device), ks, vs, cache, 0.1, mask)
        k64.append(A.values(*A.quantize(k, 8, 64), 8, 64))
        v64.append(A.values(*A.quantize(v, 4, 64), 4, 64))
        kk, vv = torch.cat(k64, 2), torch.cat(v64, 2)
        want, _, p = A.attention(q, kk, vv, 0.1, causal=L > 1)
        tol = A.attention_tolerance(q, cache.state[0].params.cpu(), 8, vv, want, p, 0.1, dt, 64, rounded=4 * L > 16)
        assert ((out.cpu().double() - want).abs() <= tol).all()
    assert cache.trim(9) == 9 and cache.offset == 252
    back = cache.dequantize(dtype=torch.float32)
    assert torch.allclose(back[0].cpu().double(), torch.cat(k64[:3], 2), rtol=2.0 ** -23, atol=0)
    assert cache.nbytes == 252 * B * H * (D + D // 2 + 2 * (D // 64) * 4)


def test_refused_first_append_leaves_the_cache_empty(device):
    cache = K.QuantizedKVCache(group_size=64, bits=4)
    k = vectors(60, (1, 2, 5, 128), torch.bfloat16).to(device)
    for v in (k.half(), k[:, :, :4], k[:, :1]):
        with pytest.raises(ValueError):
            cache.update_and_fetch(k, v)
        assert cache.empty() and cache.offset == 0 and cache.state == []
    other = k[..., :64].half()
    cache.update_and_fetch(other, other)
    assert cache.offset == 5
    with pytest.raises(ValueError):
        cache.update_and_fetch(k, k)
    assert cache.offset == 5
    cache.update_and_fetch(other, other)
    want = A.values(*A.quantize(other.cpu(), 4, 64), 4, 64)
    back = cache.dequantize(dtype=torch.float32)[0]
    assert back.shape == (1, 2, 10, 64)
    assert torch.allclose(back[:, :, 5:].cpu().double(), want, rtol=2.0 ** -23, atol=0)


def test_cache_files(device, tmp_path):
    q, k, v = (vectors(s, (1, h, 33, 64), torch.float16).to(device) for s, h in ((80, 4), (81, 2), (82, 2)))
    plain = K.KVCache()
    plain.update_and_fetch(k, v)
    cache = plain.to_quantized(group_size=32, bits=4)
    empty = K.QuantizedKVCache(group_size=128, bits=8, val_bits=4)
    f = str(tmp_path / "prompt.safetensors")
    K.save_prompt_cache(f, [cache, empty])
    got, none = K.load_prompt_cache(f, device=device)
    assert (got.group_size, got.key_bits, got.val_bits, got.offset) == (32, 4, 4, 33)
    assert (none.group_size, none.key_bits, none.val_bits, none.offset) == (128, 8, 4, 0) and none.empty()
    a = cache.quantized_attention(q, scale=0.2, mask="causal")
    assert torch.equal(a, got.quantized_attention(q, scale=0.2, mask="causal"))
    got.update_and_fetch(k, v)
    assert got.offset == 66


def test_compiled_layer_matches_eager(device):
    ks, _ = filled(90, 1, 2, 64, 128, 4, 64, torch.bfloat16, device)
    vs, _ = filled(91, 1, 2, 64, 128, 4, 64, torch.bfloat16, device)
    q, k, v = (vectors(s, (1, h, 1, 128), torch.bfloat16).to(device) for s, h in ((92, 8), (93, 2), (94, 2)))
    inv = (10000.0 ** (-torch.arange(0, 128, 2) / 128)).float().to(device)

    def layer(q, k, v, kc, kp, vc, vp):
        q, k = K.norm_rope(q, k, 63, inv)
        append_affine_kv(k, v, AffineState(kc, kp), AffineState(vc, vp), 63)
        return attention_affine(q, AffineState(kc, kp), AffineState(vc, vp), 64, 0.1)

    want = layer(q, k, v, *ks, *vs)
    got = torch.compile(layer, fullgraph=True, backend="eager")(q, k, v, *ks, *vs)
    assert torch.equal(want, got)
