"""Refusals, shapes and host rules of the group-affine cache's operators (no GPU)."""
import ctypes
import itertools
import math

import pytest
import torch

import kaplumba_amd as K
from kaplumba_amd import _lib, affine, rope
from tests import affine_oracle as A

FAKE = ctypes.c_void_p(4096)


def append_args(**kw):
    a = dict(k=None, v=None, dtype=2, B=1, H=2, L=3, k_dim=128, v_dim=64, ksb=0, ksh=0, ksl=0, vsb=0, vsh=0, vsl=0,
             kb=4, vb=8, group=64, kc=None, kp=None, vc=None, vp=None, cap=16, offset=0, stream=None)
    a.update(kw)
    return list(a.values())


def attention_args(**kw):
    a = dict(q=None, dtype=2, B=0, Hq=8, Hkv=2, L=1, k_dim=128, v_dim=128, sb=0, sh=0, sl=0, scale=0.1, kc=None, kp=None,
             kb=4, vc=None, vp=None, vb=4, group=64, cap=64, T=64, starts=None, lens=None, causal=0, mask=None,
             mask_kind=0, strides=None, out=None, ws=None, wsb=0, stream=None)
    a.update(kw)
    return list(a.values())


def back_args(**kw):
    a = dict(codes=None, params=None, dtype=1, B=0, H=2, T=3, dim=64, bits=4, group=32, cap=8, out=None, out_dtype=0,
             stream=None)
    a.update(kw)
    return list(a.values())


def rope_args(**kw):
    a = dict(q=None, k=None, dtype=2, B=0, Hq=4, Hk=2, L=3, dim=128, qsb=0, qsh=0, qsl=0, ksb=0, ksh=0, ksl=0, wq=None,
             wk=None, wtype=0, eps=1e-6, rot=128, adjacent=0, inv=None, factor=1.0, axis=None, axes=1, pos=None,
             pos_bytes=0, start=0, psa=0, psb=0, psl=0, q_out=None, k_out=None, stream=None)
    a.update(kw)
    return list(a.values())


INVALID, UNSUPPORTED, WORKSPACE = _lib.TQ_ERR_INVALID_ARGUMENT, _lib.TQ_ERR_UNSUPPORTED, _lib.TQ_ERR_WORKSPACE


@pytest.mark.parametrize("call,args,code,text", [
    ("tq_append_affine_kv", append_args(kb=3), INVALID, b"bits"),
    ("tq_append_affine_kv", append_args(vb=16), INVALID, b"bits"),
    ("tq_append_affine_kv", append_args(group=48), UNSUPPORTED, b"groups"),
    ("tq_append_affine_kv", append_args(k_dim=100), UNSUPPORTED, b"head dim"),
    ("tq_append_affine_kv", append_args(v_dim=576), UNSUPPORTED, b"head dim"),
    ("tq_append_affine_kv", append_args(v_dim=0), UNSUPPORTED, b"head dim"),
    ("tq_append_affine_kv", append_args(offset=14), INVALID, b"capacity"),
    ("tq_append_affine_kv", append_args(offset=-1), INVALID, b"capacity"),
    ("tq_append_affine_kv", append_args(L=2 ** 31 - 1, offset=1), INVALID, b"capacity"),
    ("tq_append_affine_kv", append_args(L=-1), INVALID, b"sizes"),
    ("tq_append_affine_kv", append_args(dtype=3), INVALID, b"dtype"),
    ("tq_append_affine_kv", append_args(), INVALID, b"null"),
    ("tq_append_affine_kv", append_args(k=ctypes.c_void_p(4098), v=FAKE, kc=FAKE, kp=FAKE, vc=FAKE, vp=FAKE), INVALID, b"16-byte"),
    ("tq_append_affine_kv", append_args(k=FAKE, v=FAKE, kc=FAKE, kp=FAKE, vc=FAKE, vp=FAKE, vsl=65), INVALID, b"16-byte"),
    ("tq_dequantize_affine", back_args(bits=2), INVALID, b"bits"),
    ("tq_dequantize_affine", back_args(dim=48), UNSUPPORTED, b"head dim"),
    ("tq_dequantize_affine", back_args(cap=2), INVALID, b"sizes"),
    ("tq_dequantize_affine", back_args(out_dtype=7), INVALID, b"dtypes"),
    ("tq_dequantize_affine", back_args(B=1), INVALID, b"null"),
    ("tq_attention_affine", attention_args(kb=5), INVALID, b"bits"),
    ("tq_attention_affine", attention_args(dtype=-1), INVALID, b"q_dtype"),
    ("tq_attention_affine", attention_args(Hkv=3), INVALID, b"heads"),
    ("tq_attention_affine", attention_args(k_dim=96), UNSUPPORTED, b"head dims"),
    ("tq_attention_affine", attention_args(v_dim=1024), UNSUPPORTED, b"head dims"),
    ("tq_attention_affine", attention_args(T=65), INVALID, b"capacity"),
    ("tq_attention_affine", attention_args(mask_kind=9), INVALID, b"mask_kind"),
    ("tq_attention_affine", attention_args(mask_kind=1), INVALID, b"mask"),
    ("tq_attention_affine", attention_args(L=2 ** 30), UNSUPPORTED, b"query rows"),
    ("tq_attention_affine", attention_args(B=1), INVALID, b"null"),
    ("tq_attention_affine", attention_args(B=1, q=FAKE, kc=FAKE, kp=FAKE, vc=FAKE, vp=FAKE, out=FAKE, ws=FAKE, wsb=1), WORKSPACE,
     b"workspace"),
    ("tq_norm_rope", rope_args(dim=513), UNSUPPORTED, b"head dim"),
    ("tq_norm_rope", rope_args(rot=130), INVALID, b"rotated"),
    ("tq_norm_rope", rope_args(rot=7), INVALID, b"rotated"),
    ("tq_norm_rope", rope_args(axes=3), INVALID, b"axes"),
    ("tq_norm_rope", rope_args(axes=3, axis=FAKE), INVALID, b"axes"),
    ("tq_norm_rope", rope_args(pos=FAKE, pos_bytes=2), INVALID, b"positions"),
    ("tq_norm_rope", rope_args(eps=-1.0), INVALID, b"eps"),
    ("tq_norm_rope", rope_args(eps=math.nan), INVALID, b"eps"),
    ("tq_norm_rope", rope_args(wq=FAKE, wtype=5), INVALID, b"weight_dtype"),
    ("tq_norm_rope", rope_args(B=1), INVALID, b"null"),
    ("tq_norm_rope", rope_args(B=-1), INVALID, b"sizes"),
])
def test_entry_points_refuse(call, args, code, text):
    lib = _lib.load()
    assert getattr(lib, call)(*args) == code
    assert text in lib.tq_last_error(), lib.tq_last_error()


def test_empty_calls_succeed():
    lib = _lib.load()
    for args in (append_args(B=0), append_args(H=0), append_args(L=0)):
        assert lib.tq_append_affine_kv(*args) == _lib.TQ_OK
    assert lib.tq_dequantize_affine(*back_args()) == _lib.TQ_OK
    assert lib.tq_dequantize_affine(*back_args(B=1, T=0)) == _lib.TQ_OK
    assert lib.tq_attention_affine(*attention_args()) == _lib.TQ_OK
    assert lib.tq_attention_affine(*attention_args(B=1, L=0)) == _lib.TQ_OK
    for args in (rope_args(), rope_args(B=1, L=0), rope_args(B=1, Hq=0, Hk=0)):
        assert lib.tq_norm_rope(*args) == _lib.TQ_OK


def test_a_workspace_serves_every_smaller_problem():
    import numpy as np
    size = _lib.load().tq_attention_affine_workspace_size
    rng = np.random.default_rng(0)
    log = lambda lo, hi: int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))  # noqa: E731
    for Hq, Hkv, D, Dv in ((32, 8, 128, 128), (16, 8, 256, 256), (8, 1, 64, 64), (28, 4, 192, 128), (4, 4, 512, 512), (128, 16, 96, 96)):
        for _ in range(400):
            B, L, T = log(1, 64), log(1, 1024), log(1, 200000)
            b, l, t = log(1, B), log(1, L), log(1, T)
            assert 0 < size(b, Hq, Hkv, l, D, Dv, t) <= size(B, Hq, Hkv, L, D, Dv, T), (Hq, Hkv, D, B, L, T, b, l, t)
    assert size(1, 8, 3, 1, 128, 128, 5) == 0 and size(0, 8, 2, 1, 128, 128, 5) == 0 and size(1, 8, 2, 1, 576, 64, 5) == 0


def state(B, H, T, dim, bits=4, group=64, dtype=torch.bfloat16):
    return affine.affine_state(B, H, T, dim, bits, group, dtype, "cpu")


def test_wrappers_need_the_gpu():
    st = state(1, 2, 8, 128)
    x = torch.zeros(1, 2, 3, 128, dtype=torch.bfloat16)
    for call in (lambda: K.append_affine_kv(x, x, st, st, 0), lambda: K.dequantize_affine(st),
                 lambda: K.attention_affine(x, st, st), lambda: K.norm_rope(x, x, 0, None),
                 lambda: K.QuantizedKVCache().update_and_fetch(x, x)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()


@pytest.fixture
def on_any_device(monkeypatch):
    """The wrappers' own checks, up to the library call, on CPU tensors."""
    monkeypatch.setattr(affine, "_same_device", lambda *ts: None)
    monkeypatch.setattr(rope, "_same_device", lambda *ts: None)


def test_append_refuses(on_any_device):
    x = torch.zeros(1, 2, 3, 128, dtype=torch.bfloat16)
    ok = dict(k=x, v=x, k_state=state(1, 2, 8, 128), v_state=state(1, 2, 8, 128), offset=0, group_size=64)
    cut = state(1, 2, 8, 128)
    for kw, text in [
        (dict(group_size=48), "group_size"), (dict(group_size=32), "head dim"), (dict(offset=6), "outside"),
        (dict(offset=-1), "outside"), (dict(k=x[..., :64]), "head dim"), (dict(v=x[:, :1]), "share"),
        (dict(v=x.float()), "of torch.float32"), (dict(k=x.half(), v=x.half()), "float16"),
        (dict(v_state=state(1, 2, 9, 128)), "match"), (dict(v_state=state(1, 3, 8, 128)), "match"),
        (dict(k_state=K.AffineState(cut.codes[:, :, :4], cut.params[:, :, :4])), "contiguous"),
        (dict(k_state=K.AffineState(cut.codes.view(torch.int32), cut.params)), "uint32"),
        (dict(k_state=K.AffineState(cut.codes, cut.params[..., 0])), "shapes"),
    ]:
        with pytest.raises(ValueError, match=text):
            K.append_affine_kv(**{**ok, **kw})


def test_attention_refuses(on_any_device):
    q = torch.zeros(1, 8, 1, 128, dtype=torch.bfloat16)
    ok = dict(queries=q, k_state=state(1, 2, 8, 128), v_state=state(1, 2, 8, 64), group_size=64)
    for kw, text in [
        (dict(queries=q[..., :64]), "head dim"), (dict(queries=q[:, :7]), "multiple"), (dict(queries=q[0]), "B, Hq, L, D"),
        (dict(queries=q.half()), "over states"), (dict(v_state=state(1, 2, 9, 64)), "share"),
        (dict(v_state=state(1, 2, 8, 64, dtype=torch.float16)), "over states"), (dict(queries=q.repeat(2, 1, 1, 1)), "share"),
        (dict(k_state=state(1, 2, 8, 128, group=32)), "head dim|rows of"), (dict(group_size=7), "group_size"),
    ]:
        with pytest.raises(ValueError, match=text):
            K.attention_affine(**{**ok, **kw})
    wide = state(1, 2, 16, 64)
    with pytest.raises(ValueError, match="capacity"):
        K.attention_affine(**{**ok, "v_state": K.AffineState(wide.codes[:, :, :8], wide.params[:, :, :8])})
    with pytest.raises(ValueError, match="token range"):
        K.attention_affine(**{**ok, "v_state": K.AffineState(wide.codes[:, :, ::2], wide.params[:, :, ::2])})
    with pytest.raises(NotImplementedError, match="backward"):
        K.attention_affine(**{**ok, "queries": q.clone().requires_grad_()})
    with pytest.raises(ValueError, match="broadcast"):
        K.attention_affine(**ok, mask=torch.zeros(3, 1, 8))
    with pytest.raises(ValueError, match="per-sequence"):
        K.attention_affine(**ok, seq_lens=[1, 2])
    none = K.attention_affine(q, state(1, 2, 0, 128), state(1, 2, 0, 64))
    assert none.shape == (1, 8, 1, 64) and (none == 0).all()
    assert K.attention_affine(q[:, :, :0], state(1, 2, 8, 128), state(1, 2, 8, 64)).shape == (1, 8, 0, 64)


def test_norm_rope_refuses(on_any_device):
    x = torch.zeros(2, 4, 3, 128, dtype=torch.bfloat16)
    inv, ax = torch.ones(64), torch.zeros(64, dtype=torch.int32)
    pos = torch.zeros(2, 3, dtype=torch.int32)
    ok = dict(queries=x, keys=x, positions=0, inv_freq=inv)
    for kw, text in [
        (dict(keys=x.half()), "one dtype"), (dict(keys=x[:, :, :2]), "match"), (dict(queries=x[0]), "B, H, L, D"),
        (dict(pairs="both"), "pairs"), (dict(inv_freq=torch.ones(65)), "inv_freq"), (dict(inv_freq=torch.ones(2, 2)), "inv_freq"),
        (dict(axis=ax), "positions tensor"), (dict(axis=ax.long(), positions=pos[None]), "axis"),
        (dict(axis=ax[:3], positions=pos[None]), "axis"), (dict(positions=pos.float()), "int32 or int64"),
        (dict(positions=pos[:, :2]), "sequences"), (dict(positions=pos[None]), "are not"),
        (dict(axis=ax, positions=pos[0]), "are not"), (dict(positions=pos.repeat(2, 1)), "sequences"),
        (dict(q_weight=torch.ones(64)), "weight"), (dict(queries=x.double(), keys=x.double()), "dtype"),
    ]:
        with pytest.raises(ValueError, match=text):
            K.norm_rope(**{**ok, **kw})
    with pytest.raises(NotImplementedError, match="backward"):
        K.norm_rope(**ok, q_weight=torch.nn.Parameter(torch.ones(128)))


def test_cache_rules():
    for bad in (dict(bits=3), dict(group_size=16), dict(bits=4, key_bits=5), dict(val_bits=6)):
        with pytest.raises(ValueError):
            K.QuantizedKVCache(**bad)
    c = K.QuantizedKVCache()
    assert (c.group_size, c.key_bits, c.val_bits, c.size()) == (64, 8, 8, 0) and c.empty() and c.state == [] and c.nbytes == 0
    assert c.is_trimmable() and c.trim(4) == 0 and c.make_mask(1) is None and c.make_mask(3) == "causal"
    with pytest.raises(ValueError, match="no tokens"):
        c.quantized_attention(torch.zeros(1, 1, 1, 64))
    with pytest.raises(ValueError, match="single"):
        c.decode_attention(torch.zeros(1, 1, 2, 64))
    caches = K.make_prompt_cache(num_layers=3, kv_bits=4, kv_group_size=32)
    assert [type(c) for c in caches] == [K.QuantizedKVCache] * 3 and caches[0].group_size == 32 and caches[0].val_bits == 4
    with pytest.raises(ValueError):
        K.make_prompt_cache(num_layers=3, kv_bits=4, turbo_kv_bits=3)
    with pytest.raises(NotImplementedError):
        K.make_prompt_cache(num_layers=3, kv_bits=4, max_kv_size=100)
    with pytest.raises(ValueError, match="sinks"):
        K.scaled_dot_product_attention(torch.zeros(1, 1, 1, 64), None, None, c, 1.0, None, sinks=torch.zeros(1))


def test_cache_state_round_trip():
    a = K.QuantizedKVCache(group_size=32, bits=4, key_bits=8)
    a.reserve(20, 2, 3, 64, 96, "cpu", torch.float16)
    assert a.keys.codes.shape == (2, 3, 20, 16) and a.values.codes.shape == (2, 3, 20, 12) and a.keys.params.shape == (2, 3, 20, 2, 2)
    a.offset = 7
    a.keys.params.normal_()
    b = K.QuantizedKVCache.from_state(a.state, a.meta_state)
    assert (b.offset, b.group_size, b.key_bits, b.val_bits, b.bits) == (7, 32, 8, 4, 4)
    assert torch.equal(b.keys.params, a.state[0].params) and b.nbytes == a.nbytes
    for bad in (("7",), ("8", "32", "4"), ("-1", "32", "4"), ("7", "33", "4"), ("7", "32", "5"), ("7", "32", "4", "8", "1")):
        with pytest.raises(ValueError):
            K.QuantizedKVCache.from_state(a.state, bad)
    with pytest.raises(ValueError):
        K.QuantizedKVCache.from_state(a.state[:1], a.meta_state)


@pytest.mark.parametrize("bits,group", itertools.product((4, 8), (32, 64, 128)))
def test_oracle_round_trip(bits, group):
    """The plain form stores a value within half a step (and the scale's rounding at the top)."""
    x = torch.randn(3, 5, 256, generator=torch.Generator().manual_seed(bits * group)).to(torch.bfloat16)
    words, params = A.quantize(x, bits, group)
    back = A.values(words, params, bits, group)
    step = params[..., 0].double().repeat_interleave(group, -1)
    assert ((back - x.double()).abs() <= step * (0.5 + (2 ** bits - 1) * 2.0 ** -8)).all()
    assert (words >= 0).all() and (words < 2 ** 32).all()
