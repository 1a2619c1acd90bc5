"""Norms and rotations of queries and keys against the formula in 64 bits."""
import math

import pytest
import torch

import kaplumba_amd as K
from kaplumba_amd import norm_rope
from tests import affine_oracle as A

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def frequencies(rot, base=10000.0):
    return (base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float()


def oracle(x, w, pos, inv, axis, eps, pairs, factor):
    """(result, how far f32 arithmetic and one rounding may be from it), element by element.

    A norm of D terms in f32 is off by (D / 4 + 8) 2^-24 of itself at most; cosine and sine by 2^-22 (an angle's
    rest rounded to f32 is off by 2^-24 turns of a half, and the functions by two ulps); the two products of a pair
    add up with three more roundings."""
    y = x.double()
    D = x.shape[-1]
    rel = 4 * 2.0 ** -24
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
        rel += (D / 4 + 8) * 2.0 ** -24
    out, size = y.clone(), y.abs()
    n = 0 if inv is None else len(inv)
    for i in range(n):
        p = (pos if axis is None else pos[axis[i]]).double() * inv[i].double()
        c, s = p.cos()[:, None] * factor, p.sin()[:, None] * factor
        j, k = (i, i + n) if pairs == "half" else (2 * i, 2 * i + 1)
        out[..., j], out[..., k] = y[..., j] * c - y[..., k] * s, y[..., j] * s + y[..., k] * c
        size[..., j] = size[..., k] = (y[..., j].abs() + y[..., k].abs()) * abs(factor)
    return out, size * (rel + 2.0 ** -21) + out.abs() * A.half_step(x.dtype) * 1.01 + \
        (2.0 ** -25 if x.dtype == torch.float16 else 1e-40)


def run(device, q, k, wq, wk, pos, inv, axis=None, eps=1e-6, pairs="half", factor=1.0):
    to = lambda t: t.to(device) if isinstance(t, torch.Tensor) else t  # noqa: E731
    got = norm_rope(q if q.is_cuda else q.to(device), k if k.is_cuda else k.to(device), to(pos), to(inv), axis=to(axis),
                    q_weight=to(wq), k_weight=to(wk), eps=eps, pairs=pairs, factor=factor)
    B, _, L, _ = q.shape
    at = torch.arange(L) + pos if not isinstance(pos, torch.Tensor) else pos
    if at.dim() == (1 if axis is None else 2):
        at = at.unsqueeze(-2)
    at = at.expand(at.shape[:-2] + (B, L))
    for x, w, g in ((q, wq, got[0]), (k, wk, got[1])):
        want, tol = oracle(x.cpu(), w, at, inv, axis, eps, pairs, factor)
        assert g.is_contiguous() and g.shape == x.shape and g.dtype == x.dtype
        off = (g.cpu().double() - want).abs()
        assert (off <= tol).all(), f"off by {(off / tol).max():.3g} of the tolerance"
    return got


def case(seed, B, Hq, Hk, L, D, dt):
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(B, h, L, D, generator=g).to(dt) for h in (Hq, Hk))
    return q, k, (1 + 0.2 * torch.randn(D, generator=g)).to(dt), (1 + 0.2 * torch.randn(D, generator=g)).to(dt)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("D,rot", [(64, 64), (80, 80), (80, 32), (96, 96), (128, 128), (128, 64), (192, 192), (256, 128),
                                   (256, 256), (512, 512), (13, 12), (13, 6), (100, 50), (2, 2), (130, 130), (72, 40)])
def test_dims(device, dtype, pairs, D, rot):
    dt = DTYPES[dtype]
    q, k, wq, wk = case(D + rot, 2, 6, 3, 5, D, dt)
    run(device, q, k, wq, wk, 17, frequencies(rot), pairs=pairs)
    run(device, q, k, None, None, 17, frequencies(rot), pairs=pairs)
    run(device, q, k, None, wk, 0, frequencies(rot), pairs=pairs, factor=1.25)


@pytest.mark.parametrize("B,Hq,Hk,L", [(1, 1, 1, 1), (1, 32, 8, 1), (32, 28, 4, 1), (1, 7, 1, 300), (3, 16, 16, 33),
                                       (1, 128, 2, 2), (2, 5, 0, 3), (2, 0, 5, 3)])
def test_heads_and_lengths(device, B, Hq, Hk, L):
    q, k, wq, wk = case(B + Hq, B, Hq, Hk, L, 128, torch.bfloat16)
    run(device, q, k, wq, wk, 1000, frequencies(128))


@pytest.mark.parametrize("far", [0, 32767, 131071, 1 << 20, (1 << 31) - 40, -5])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_far_positions(device, dtype, far):
    q, k, wq, wk = case(5, 1, 4, 2, 9, 128, DTYPES[dtype])
    run(device, q, k, wq, wk, far, frequencies(128))
    run(device, q, k, wq, wk, torch.arange(9, dtype=torch.int64) + far, frequencies(128))


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
@pytest.mark.parametrize("axes", [2, 3, 4])
def test_axes(device, axes, wide):
    B, L, D = 2, 21, 128
    q, k, wq, wk = case(axes, B, 8, 2, L, D, torch.float16)
    g = torch.Generator().manual_seed(axes)
    pos = torch.randint(0, 5000, (axes, B, L), generator=g).to(wide)
    sections = torch.arange(D // 2, dtype=torch.int32) * axes // (D // 2)
    mixed = (torch.arange(D // 2, dtype=torch.int32)) % axes
    for axis in (sections, mixed):
        run(device, q, k, wq, wk, pos, frequencies(D), axis)
        run(device, q, k, wq, wk, pos[:, :1], frequencies(D), axis)
        run(device, q, k, wq, wk, pos[:, 0], frequencies(D), axis)
    # the first axis alone is the rotation without axes
    zero = torch.zeros(D // 2, dtype=torch.int32)
    a = run(device, q, k, wq, wk, pos, frequencies(D), zero)
    b = run(device, q, k, wq, wk, pos[0], frequencies(D))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_strides(device):
    B, L, D = 2, 11, 128
    g = torch.Generator().manual_seed(1)
    x = torch.randn(B, L, 10 * D + 8, generator=g).to(torch.bfloat16).to(device)
    q = x[..., : 8 * D].unflatten(-1, (8, D)).transpose(1, 2)
    k = x[..., 8 * D: 10 * D].unflatten(-1, (2, D)).transpose(1, 2)
    odd = x[..., 3: 3 + 2 * D].unflatten(-1, (2, D)).transpose(1, 2)   # not 16-byte aligned
    w = torch.randn(D, generator=g)
    pos = torch.arange(2 * L, dtype=torch.int32)[::2].expand(B, L)
    run(device, q, k, w, w, pos, frequencies(D))
    run(device, q, odd, w, w.to(torch.bfloat16), pos, frequencies(D))
    run(device, q, k.transpose(2, 3).contiguous().transpose(2, 3), None, w, pos, frequencies(D))


def test_special_vectors(device):
    """Zeros, tiny and huge vectors; an infinity or NaN stays in its own vector."""
    D = 128
    q, k, wq, wk = case(9, 1, 4, 2, 6, D, torch.bfloat16)
    q[0, 0, 0], q[0, 1, 1] = 0, torch.finfo(torch.bfloat16).tiny
    q[0, 2, 2], k[0, 0, 3] = 1e18, 3e-20
    run(device, q, k, wq, wk, 3, frequencies(D))
    k[0, 1, 4, 7], q[0, 3, 5, 100] = math.nan, math.inf
    a, b = norm_rope(q.to(device), k.to(device), 3, frequencies(D).to(device), q_weight=wq.to(device), k_weight=wk.to(device))
    for got, (h, l) in ((b, (1, 4)), (a, (3, 5))):
        bad = ~torch.isfinite(got.cpu())
        assert bad[0, h, l].any()
        bad[0, h, l] = False
        assert not bad.any()


def test_norm_alone_and_nothing(device):
    q, k, wq, wk = case(11, 2, 4, 2, 3, 100, torch.float32)
    run(device, q, k, wq, wk, 0, None, eps=0.1)
    got = norm_rope(q.to(device), k.to(device), 0, None)
    assert torch.equal(got[0].cpu(), q) and torch.equal(got[1].cpu(), k)


def test_streams_and_graph(device):
    q, k, wq, wk = (t.to(device) for t in case(12, 2, 8, 2, 1, 128, torch.bfloat16))
    inv, pos = frequencies(128).to(device), torch.tensor([[5], [9]], dtype=torch.int32, device=device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm_rope(q, k, pos, inv, q_weight=wq, k_weight=wk)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = norm_rope(q, k, pos, inv, q_weight=wq, k_weight=wk)
    torch.cuda.current_stream().wait_stream(side)
    for n in range(4):
        pos += 1000
        q.mul_(-1.5)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = norm_rope(q, k, pos, inv, q_weight=wq, k_weight=wk)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind", ["turbo", "plain", "affine", "batch_turbo", "batch_plain"])
def test_attention_step(device, kind):
    """The layer's three calls by hand and through attention_step, over every cache."""
    B, Hq, H, D, dt = 2, 8, 2, 128, torch.bfloat16
    pads = [0, 3]

    def new():
        return {"turbo": lambda: K.TurboQuantKVCache(bits=3), "plain": K.KVCache,
                "affine": lambda: K.QuantizedKVCache(bits=4), "batch_turbo": lambda: K.BatchTurboQuantKVCache(pads, 3),
                "batch_plain": lambda: K.BatchKVCache(pads)}[kind]()

    a, b = new(), new()
    inv = frequencies(D).to(device)
    for i, L in enumerate((12, 1, 1)):
        q, k, wq, wk = (t.to(device) for t in case(20 + i, B, Hq, H, L, D, dt))
        v = case(30 + i, B, Hq, H, L, D, dt)[1].to(device)
        mask = a.make_mask(L)
        got = K.attention_step(q, k, v, a, 0.1, mask, inv_freq=inv, q_weight=wq, k_weight=wk)
        first = b.offset if not kind.startswith("batch") else \
            (b.offset[:, None] + torch.arange(L)).to(torch.int32).to(device)
        qq, kk = norm_rope(q, k, first, inv, q_weight=wq, k_weight=wk)
        want = K.scaled_dot_product_attention(qq, *b.update_and_fetch(kk, v), b, 0.1, b.make_mask(L) if L == 1 else mask)
        assert torch.equal(got, want) and torch.isfinite(got[0]).all()
