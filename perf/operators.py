"""The group-affine cache and the step before it, as they are measured: the work, its plain form and its calls.

A case is one call (or one write and read back) of a layer whose cache holds 4- or 8-bit codes with a scale
and a bias for each group of coordinates:

  rope    norms of the queries and keys of each head, and the rotation by their positions: ``norm_rope``
  codec   quantize L new tokens of keys and values into the cache, and read those tokens back:
          ``append_affine_kv`` and ``dequantize_affine``
  attend  attention of L query rows per head over the cache: ``attention_affine``

Keys and values are N(0, 1) times a log-normal scale per (head, channel), queries N(0, 1).
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
LOWEST = torch.finfo(torch.float32).min

ROPE = dict(kind="rope", B=1, L=1, Hq=32, Hkv=8, D=128, rot=128, axes=1, pairs="half", norm=True, far=0,
            dtype="bf16")
CODEC = dict(kind="codec", B=1, L=1, Hkv=8, D=128, Dv=128, kb=4, vb=4, group=64, tokens=0, dtype="bf16")
ATTEND = dict(kind="attend", B=1, L=1, Hq=32, Hkv=8, D=128, Dv=128, kb=4, vb=4, group=64, tokens=0, shortest=0,
              window=0, dtype="bf16")


def listed():
    rope = lambda name, **kw: dict(ROPE, name=name, **kw)  # noqa: E731
    codec = lambda name, **kw: dict(CODEC, name=name, **kw)  # noqa: E731
    attend = lambda name, **kw: dict(ATTEND, name=name, **kw)  # noqa: E731
    return [
        # one token of one request, far into a 32k context: launches, hardly any data
        rope("rope_decode", far=32767),
        # a whole 8192-token prompt of the headline heads
        rope("rope_prompt", L=8192),
        # two prompts with images or video: time, height and width positions, odd lengths, f16
        rope("rope_axes", B=2, L=2047, Hq=28, Hkv=4, axes=3, dtype="f16"),
        # the new token of each of 32 requests, 8-bit keys and 4-bit values
        codec("codec_step", B=32, kb=8, tokens=500),
        # a whole 8192-token prompt written in 4 bits, and read back
        codec("codec_prompt", L=8192),
        # a chunk of an odd length at head dim 256, 8-bit keys, small groups, f16
        codec("codec_d256", L=1999, B=2, D=256, Dv=256, kb=8, group=32, tokens=1001, dtype="f16"),
        # the first steps of a chat: latency
        attend("decode_short", tokens=512),
        # one layer of the headline benchmark: one token against 32k cached ones, 4 bits
        attend("decode_32k", tokens=32768),
        # a server's batch of 32 requests of unlike length, head dim 256, 8-bit keys and 4-bit values
        attend("decode_ragged_d256", B=32, Hq=16, D=256, Dv=256, kb=8, tokens=8192, shortest=2048, dtype="f16"),
        # four drafts verified in each of four long sequences
        attend("verify_131k", B=4, L=4, tokens=131076),
        # a chunk of a long prompt
        attend("prefill_d128", L=512, tokens=8192),
        # a chunk through a sliding-window layer (boolean array mask), head dim 64, 8 bits, f16, odd lengths
        attend("prefill_window", B=2, L=500, D=64, Dv=64, kb=8, vb=8, group=32, tokens=4097, window=1024, dtype="f16"),
    ]


# What a drawn case may cost: as much as the largest listed one does.
MOST_ROPE = 8192 * 40 * 128              # elements of queries and keys
MOST_NEW = 8192 * 8 * 256                # elements of keys and values written at once
MOST_CACHE = 4 * 131076 * 8 * 256        # elements of keys and values in a cache
MOST_PAIRS = 32 * 512 * 8192 * 256       # query rows x tokens x (Dk + Dv)


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(hi, lo + 1))))))


def draw(rng):
    kind = rng.choice(["rope", "codec", "attend", "attend", "attend"])
    hkv = rng.choice([1, 2, 4, 8, 8, 16])
    hq = hkv * rng.choice([1, 2, 4, 4, 7, 8])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "rope":
        c = dict(ROPE, Hkv=hkv, Hq=hq, dtype=rng.choice([dtype, dtype, "f32"]))
        c["D"] = rng.choice([64, 80, 96, 128, 128, 192, 256])
        c["rot"] = c["D"] if rng.random() < 0.7 else c["D"] // 2 // 16 * 16
        c["axes"] = rng.choice([1, 1, 3, 4])
        c["pairs"] = rng.choice(["half", "half", "adjacent"])
        c["norm"] = rng.random() < 0.8
        c["B"] = rng.choice([1, 1, 2, 8, 32])
        # a case of f32 holds half as many elements
        most = MOST_ROPE // (c["B"] * (hq + hkv) * c["D"] * (2 if c["dtype"] == "f32" else 1))
        c["L"] = 1 if rng.random() < 0.3 else _log_int(rng, 1, max(2, min(16384, most)))
        c["far"] = _log_int(rng, 1, 131072)
        return c
    d, dv = rng.choice([(64, 64), (128, 128), (128, 128), (256, 256), (96, 96), (192, 128)])
    kb, vb = rng.choice([(4, 4), (4, 4), (8, 4), (8, 8)])
    group = rng.choice([g for g in (32, 64, 64, 128) if d % g == 0 and dv % g == 0])
    common = dict(Hkv=hkv, D=d, Dv=dv, kb=kb, vb=vb, group=group, dtype=dtype)
    if kind == "codec":
        c = dict(CODEC, **common)
        c["B"] = rng.choice([1, 1, 2, 8, 32])
        c["L"] = 1 if rng.random() < 0.3 else _log_int(rng, 1, max(2, MOST_NEW // (c["B"] * hkv * (d + dv))))
        c["tokens"] = _log_int(rng, 1, 2000)
        return c
    c = dict(ATTEND, Hq=hq, **common)
    mode = rng.choice(["decode", "decode", "verify", "prefill", "prefill"])
    c["B"] = _log_int(rng, 1, 4 if mode == "prefill" else 32)
    c["L"] = {"decode": 1, "verify": rng.randint(2, 8), "prefill": _log_int(rng, 9, 1024)}[mode]
    if mode == "prefill" and rng.random() < 0.3:
        c["window"] = rng.choice([128, 512, 1024])
    # a query sees L tokens at least
    c["L"] = min(c["L"], math.isqrt(MOST_PAIRS // (c["B"] * hq * (d + dv))))
    # 8-bit codes and small groups take more bytes an element than the listed 4-bit cache's groups of 64
    bits = (d * kb + dv * vb) / (d + dv) + 32 / group
    most = min(131072, int(MOST_CACHE * 4.5 / bits) // (c["B"] * hkv * (d + dv)),
               MOST_PAIRS // (c["B"] * hq * c["L"] * (d + dv)))
    c["tokens"] = max(c["L"], _log_int(rng, 16, max(17, most)))
    if mode != "prefill" and c["B"] > 1 and rng.random() < 0.5:
        c["shortest"] = max(c["L"], int(c["tokens"] * rng.uniform(0.1, 1.0)))
    if mode == "decode" and rng.random() < 0.2:
        # f32 layers decode too: a quarter of the tokens keeps the cost
        c["dtype"], c["tokens"] = "f32", max(c["shortest"], c["tokens"] // 4, 1)
    return c


# ------------------------------------------------------------------- inputs ---
def _kv(g, shape, dtype):
    scale = torch.exp(torch.randn(1, shape[1], 1, shape[3], device="cuda", generator=g) * 0.5)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _lengths(case):
    """Tokens of each row of a batch, from ``shortest`` to ``tokens`` in mixed order; one row has all."""
    B, lo, hi = case["B"], case["shortest"], case["tokens"]
    return [hi - (hi - lo) * ((7 * b) % B) // max(B - 1, 1) for b in range(B)]


def _axis_of(case):
    """The axis that each frequency's position comes from: contiguous sections, the last axis has the rest."""
    n, a = case["rot"] // 2, case["axes"]
    part = n // a
    return [min(i // part, a - 1) if a > 1 else 0 for i in range(n)]


def _packed_row(dim, bits):
    return dim * bits // 32


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, B, L = DTYPES[case["dtype"]], case["B"], case["L"]
    if case["kind"] == "rope":
        D, rot = case["D"], case["rot"]
        # the layout a projection gives: (B, L, H, D), heads transposed to the front
        q = torch.randn(B, L, case["Hq"], D, device="cuda", generator=g).to(dtype).transpose(1, 2)
        k = torch.randn(B, L, case["Hkv"], D, device="cuda", generator=g).to(dtype).transpose(1, 2)
        wq, wk = ((1 + 0.2 * torch.randn(D, device="cuda", generator=g)).to(dtype) for _ in range(2))
        at = torch.arange(L, device="cuda", dtype=torch.int32) + case["far"]
        at = at.expand(B, L) + torch.arange(B, device="cuda", dtype=torch.int32)[:, None] * 3
        if case["axes"] > 1:
            # the other axes: rows and columns of a picture
            side = [torch.randint(0, 64, (B, L), device="cuda", generator=g, dtype=torch.int32)
                    for _ in range(case["axes"] - 1)]
            at = torch.stack([at] + side)
        inv = 1.0 / (10000.0 ** (torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot))
        return {"case": case, "q": q, "k": k, "wq": wq if case["norm"] else None, "wk": wk if case["norm"] else None,
                "positions": at.contiguous(), "inv_freq": inv.float(),
                "axis": torch.tensor(_axis_of(case), device="cuda", dtype=torch.int32) if case["axes"] > 1 else None}
    H, D, Dv, G = case["Hkv"], case["D"], case["Dv"], case["group"]
    if case["kind"] == "codec":
        cap = (case["tokens"] + L + 255) // 256 * 256
        state = {"case": case, "k": _kv(g, (B, H, L, D), dtype), "v": _kv(g, (B, H, L, Dv), dtype)}
        for side, dim, bits in (("ks", D, case["kb"]), ("vs", Dv, case["vb"])):
            state[side] = (torch.zeros(B, H, cap, _packed_row(dim, bits), dtype=torch.uint32, device="cuda"),
                           torch.zeros(B, H, cap, dim // G, 2, dtype=dtype, device="cuda"))
        return state
    T = case["tokens"]
    cap = (T + 255) // 256 * 256
    state = {"case": case, "scale": 1.0 / math.sqrt(D), "lens": None, "mask": None,
             "q": torch.randn(B, case["Hq"], L, D, device="cuda", generator=g).to(dtype)}
    for side, dim, bits in (("ks", D, case["kb"]), ("vs", Dv, case["vb"])):
        words = torch.empty(B, H, cap, _packed_row(dim, bits), dtype=torch.int32, device="cuda")
        params = torch.empty(B, H, cap, dim // G, 2, dtype=dtype, device="cuda")
        for b in range(B):
            w, p = _quantized(_kv(g, (1, H, cap, dim), dtype), bits, G)
            words[b], params[b] = w[0], p[0]
        state[side] = (words.view(torch.uint32)[:, :, :T], params[:, :, :T])
    if case["shortest"]:
        state["lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    if case["window"]:
        i = torch.arange(T - L, T, device="cuda")[:, None]
        t = torch.arange(T, device="cuda")[None, :]
        state["mask"] = (t <= i) & (i < t + case["window"])
    return state


# ------------------------------------------------------------ the plain form ---
def _quantized(x, bits, group):
    """Words (int32) and (scale, bias) pairs of x's last axis: a group's bias is its least value, its scale a
    (2^bits - 1)-th of its range in x's type; a code counts the half steps (k + 1/2) scale that x - bias reaches."""
    n = (1 << bits) - 1
    g = x.unflatten(-1, (-1, group))
    lo, hi = g.amin(-1).float(), g.amax(-1).float()
    scale = ((hi * 0.5 - lo * 0.5) / n * 2.0).to(x.dtype)
    step = scale.float()[..., None]
    away = g.float() - lo[..., None]
    code = torch.floor(away.double() / step + 0.5).clamp(0, n)
    code = torch.where(step > 0, code, 0.0).to(torch.int64).flatten(-2)
    code = code.unflatten(-1, (-1, 32 // bits)) << torch.arange(0, 32, bits, device=x.device)
    word = code.sum(-1)
    word = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
    return word, torch.stack([scale, lo.to(x.dtype)], -1)


def _values(words, params, bits, group):
    """The values in 32 bits that codes stand for."""
    w = words.view(torch.int32)
    code = (w[..., None] >> torch.arange(0, 32, bits, device=w.device, dtype=torch.int32)) & ((1 << bits) - 1)
    code = code.flatten(-2).unflatten(-1, (-1, group)).float()
    return (code * params[..., 0, None].float() + params[..., 1, None].float()).flatten(-2)


def _rope_plain(x, weight, state):
    case = state["case"]
    rot, dtype = case["rot"], x.dtype
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    at = state["positions"].double()
    if state["axis"] is None:
        at = at[..., None]
    else:
        at = at[state["axis"].long()].movedim(0, -1)
    angle = at * state["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if case["pairs"] == "half":
        a, b = y[..., : rot // 2], y[..., rot // 2: rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, y[..., rot:]], -1).to(dtype)


def _attend_plain(state):
    case = state["case"]
    B, L, Hq, H, T = case["B"], case["L"], case["Hq"], case["Hkv"], case["tokens"]
    k = _values(*state["ks"], case["kb"], case["group"])
    v = _values(*state["vs"], case["vb"], case["group"])
    q = state["q"].float().reshape(B, H, Hq // H * L, case["D"]) * state["scale"]
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).reshape(B, H, Hq // H, L, T)
    t = torch.arange(T, device=s.device)
    if state["mask"] is not None:
        s = torch.where(state["mask"], s, LOWEST)
    elif L > 1:
        end = state["lens"][:, None] if state["lens"] is not None else torch.full((1, 1), T, device=s.device)
        last = end - L + torch.arange(L, device=s.device)
        s = torch.where(t <= last[:, None, None, :, None], s, LOWEST)
    if state["lens"] is not None:
        s = torch.where(t < state["lens"][:, None, None, None, None], s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul((p / p.sum(-1, keepdim=True)).reshape(B, H, -1, T), v)
    return o.reshape(B, Hq, L, case["Dv"]).to(state["q"].dtype)


def run(state):
    case = state["case"]
    if case["kind"] == "rope":
        if own:
            from kaplumba_amd import norm_rope
            return norm_rope(state["q"], state["k"], state["positions"], state["inv_freq"], axis=state["axis"],
                             q_weight=state["wq"], k_weight=state["wk"], eps=1e-6, pairs=case["pairs"])
        return _rope_plain(state["q"], state["wq"], state), _rope_plain(state["k"], state["wk"], state)
    if case["kind"] == "codec":
        at, end, G = case["tokens"], case["tokens"] + case["L"], case["group"]
        (kw, kp), (vw, vp) = state["ks"], state["vs"]
        if own:
            from kaplumba_amd import AffineState, append_affine_kv, dequantize_affine
            append_affine_kv(state["k"], state["v"], AffineState(kw, kp), AffineState(vw, vp), at, group_size=G)
            new = [AffineState(w[:, :, at:end], p[:, :, at:end]) for w, p in ((kw, kp), (vw, vp))]
            return [dequantize_affine(st, group_size=G, dtype=state["k"].dtype) for st in new]
        out = []
        for x, w, p, bits in ((state["k"], kw, kp, case["kb"]), (state["v"], vw, vp, case["vb"])):
            w.view(torch.int32)[:, :, at:end], p[:, :, at:end] = _quantized(x, bits, G)
            out.append(_values(w[:, :, at:end], p[:, :, at:end], bits, G).to(x.dtype))
        return out
    if own:
        from kaplumba_amd import AffineState, attention_affine
        return attention_affine(state["q"], AffineState(*state["ks"]), AffineState(*state["vs"]), group_size=case["group"],
                                scale=state["scale"], causal=state["mask"] is None and case["L"] > 1,
                                seq_lens=state["lens"], mask=state["mask"])
    return _attend_plain(state)


# --------------------------------------------------------------- what it costs ---
def work(case):
    B, L, D, item = case["B"], case["L"], case["D"], DTYPES[case["dtype"]].itemsize
    if case["kind"] == "rope":
        n = B * L * (case["Hq"] + case["Hkv"]) * D
        small = 4 * B * L * case["axes"] + 4 * case["rot"] // 2 + 2 * D * item
        return {"bytes": 2 * n * item + small, "flops": 7 * n}
    Dv, H = case["Dv"], case["Hkv"]
    # one cached token of one head: codes, and a scale and a bias a group
    row = (D * case["kb"] + Dv * case["vb"]) / 8 + 2 * item * (D + Dv) / case["group"]
    if case["kind"] == "codec":
        n = B * H * L
        return {"bytes": n * (2 * (D + Dv) * item + 2 * row), "flops": 6 * n * (D + Dv)}
    T, W = case["tokens"], case["window"]
    lens = _lengths(case) if case["shortest"] else [T] * B
    seen = [min(n - L + i + 1, W or n) if L > 1 else n for n in lens for i in range(L)]
    read = sum(lens) if not W else B * min(T, W + L - 1)
    io = B * case["Hq"] * L * (D + Dv) * item + (L * T if W else 0)
    return {"bytes": H * read * row + io, "flops": 2 * case["Hq"] * sum(seen) * (D + Dv)}


# ------------------------------------------------------------ the same in 64 bits ---
def _codes64(words, bits):
    w = words.to(torch.int64)
    return torch.cat([(w // (1 << s) % (1 << bits))[..., None] for s in range(0, 32, bits)], -1).flatten(-2).double()


def _rope64(x, weight, state):
    case, D, rot = state["case"], x.shape[-1], state["case"]["rot"]
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / D + 1e-6) * weight.double()
    pos, out = state["positions"].double(), y.clone()
    for i, f in enumerate(state["inv_freq"].tolist()):
        p = (pos if case["axes"] == 1 else pos[_axis_of(case)[i]]) * f
        j, k = (i, i + rot // 2) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
        c, s = torch.cos(p)[:, None], torch.sin(p)[:, None]
        out[..., j] = c * y[..., j] - s * y[..., k]
        out[..., k] = s * y[..., j] + c * y[..., k]
    return out


def _back64(x, bits, group):
    n, x64 = (1 << bits) - 1, x.double()
    lo = torch.stack([c.min(-1).values for c in x64.split(group, -1)], -1)
    hi = torch.stack([c.max(-1).values for c in x64.split(group, -1)], -1)
    step = ((hi - lo) / n).to(x.dtype).double().repeat_interleave(group, -1)
    lo = lo.repeat_interleave(group, -1)
    steps = (x64 - lo) / step.clamp_min(1e-300)
    return lo + step * torch.floor(steps + 0.5).clamp(0, n)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rope":
        return _rope64(state["q"], state["wq"], state), _rope64(state["k"], state["wk"], state)
    if case["kind"] == "codec":
        return [_back64(state["k"], case["kb"], case["group"]), _back64(state["v"], case["vb"], case["group"])]
    B, L, Hq, H, T = case["B"], case["L"], case["Hq"], case["Hkv"], case["tokens"]
    R, G = Hq // H, case["group"]
    lens = _lengths(case) if case["shortest"] else [T] * B
    out = torch.empty(B, Hq, L, case["Dv"], dtype=torch.float64, device="cuda")
    for b in range(B):
        n = lens[b]
        for h in range(H):
            kv = []
            for (w, p), bits in ((state["ks"], case["kb"]), (state["vs"], case["vb"])):
                pair = p[b, h, :n].double().repeat_interleave(G, 1)
                kv.append(_codes64(w[b, h, :n], bits) * pair[..., 0] + pair[..., 1])
            s = state["q"][b, h * R:(h + 1) * R].double().reshape(R * L, -1) @ kv[0].T * state["scale"]
            if L > 1:
                i = torch.arange(n - L, n, device="cuda")[:, None]
                t = torch.arange(n, device="cuda")[None, :]
                seen = (t <= i) & (i - t < (case["window"] or n + 1))
                s = s.reshape(R, L, n).masked_fill(~seen, -math.inf).reshape(R * L, n)
            out[b, h * R:(h + 1) * R] = (torch.softmax(s, -1) @ kv[1]).reshape(R, L, -1)
    return out
