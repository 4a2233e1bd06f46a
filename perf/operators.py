"""What the framework's language-model operators are timed on: the gated linear recurrence, the per-head norm of queries
and keys with the position rotation, and the AdamW step over a whole list of tensors.

Every case names one operator, its sizes and its form.  `prepare` makes the inputs on the GPU, `run` is one pass through
the operator: in plain torch operations (`own` false) or through the framework (`own` true); `exact` is the definition
in 64 bits.  Both forms of a pass return the same outputs; states that a pass updates (AdamW) are updated in place.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    rec = dict(op="recurrence", form="gated", layout="sequence", ragged=False, h0=False, last=False, backward=True)
    qk = dict(op="qk", seq_len=0, rot=64, interleaved=False, base=10000.0, gain=True, pad=0, far=False, backward=True)
    return [
        # one new token for each of 128 running sequences, the state carried from the call before
        dict(rec, name="recurrence token step 128 x 512", n_seq=128, seq_len=1, dim=512, h0=True, last=True, backward=False),
        # the recurrent layer's benchmark size (128 steps, batch 128, 512 units, time-major), inference
        dict(rec, name="recurrence forward T128 B128 H512", n_seq=128, seq_len=128, dim=512, layout="time", backward=False),
        # a training step of a language-model block: 32 sequences of up to 512 tokens, width 1024, gate and input as the two
        # halves of one projection, sequences of different lengths
        dict(rec, name="recurrence training 32 x 512 x 1024 ragged", n_seq=32, seq_len=512, dim=1024, layout="fused", ragged=True),
        # one long document, few channels, odd sizes, decays given directly, state in and out
        dict(rec, name="recurrence training 1 x 65521 x 250 linear", form="linear", n_seq=1, seq_len=65521, dim=250, h0=True, last=True),
        # one new token for 8 sequences, grouped keys, positions far into a long context
        dict(qk, name="qk token step 8 rows 16+4 heads of 64", rows=8, heads_q=16, heads_k=4, d_head=64, far=True, backward=False),
        # the encoder block's training step (width 512, 8 heads, 32 sequences of 256), slices of one fused projection
        dict(qk, name="qk training 8192 rows 8+8 heads of 64", rows=8192, seq_len=256, heads_q=8, heads_k=8, d_head=64, pad=512),
        # the language model's training step (width 1024, 16 heads, 32 sequences of 512)
        dict(qk, name="qk training 16384 rows 16+16 heads of 64", rows=16384, seq_len=512, heads_q=16, heads_k=16, d_head=64),
        # odd row count and head width, part of each head rotated in neighbouring pairs, grouped keys, odd row stride
        dict(qk, name="qk training 4999 rows 12+3 heads of 80 partial", rows=4999, heads_q=12, heads_k=3, d_head=80, rot=32,
             interleaved=True, pad=7, far=True),
        # the MNIST classifier's six tensors: a step bound by launches
        dict(op="adamw", name="adamw 32-bit states MLP 784-128-64-10", model="mlp", bits=32),
        # one encoder block of width 512, states in 8 bits, nearest rounding
        dict(op="adamw", name="adamw 8-bit states block 512", model="lm", d=512, dff=2048, layers=1, vocab=0, bits=8, stochastic=False),
        # the six-layer language model (141 M parameters), states in 32 bits and in 8 with stochastic rounding
        dict(op="adamw", name="adamw 32-bit states language model", model="lm", d=1024, dff=4096, layers=6, vocab=32000, bits=32),
        dict(op="adamw", name="adamw 8-bit states language model", model="lm", d=1024, dff=4096, layers=6, vocab=32000, bits=8,
             stochastic=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "qk", "adamw"])
    if op == "recurrence":
        seq_len = _log(rng, 1, 65536)
        dim = _log(rng, 64, 2048)
        if rng.random() < 0.5:
            dim = max(64, dim // 64 * 64)
        n_seq = _log(rng, 1, max(1, min(256, 16000000 // (seq_len * dim)))) if seq_len * dim < 16000000 else 1
        seq_len = max(1, min(seq_len, 16000000 // (n_seq * dim)))
        return dict(op=op, form=rng.choice(["gated", "linear"]), n_seq=n_seq, seq_len=seq_len, dim=dim,
                    layout=rng.choice(["sequence", "time", "fused"]), ragged=rng.random() < 0.4, h0=rng.random() < 0.5,
                    last=rng.random() < 0.5, backward=rng.random() < 0.7)
    if op == "qk":
        d_head = rng.choice([32, 64, 64, 80, 96, 128, 160, 256])
        heads_k = rng.randint(1, 16)
        heads_q = heads_k * rng.choice([1, 1, 2, 4])
        rows = min(_log(rng, 1, 16384), 32000000 // (d_head * (heads_q + heads_k)))
        return dict(op=op, rows=rows, seq_len=rng.choice([0, 128, 512]), heads_q=heads_q, heads_k=heads_k, d_head=d_head,
                    rot=rng.choice([d_head, d_head, d_head // 2]), interleaved=rng.random() < 0.4,
                    base=rng.choice([10000.0, 500000.0]), gain=rng.random() < 0.8, pad=rng.choice([0, 0, 64, 5]),
                    far=rng.random() < 0.5, backward=rng.random() < 0.7)
    return dict(op="adamw", model="mixed", tensors=_log(rng, 1, 300), largest=_log(rng, 1000, 400000), shape_seed=rng.randint(0, 10**9),
                bits=rng.choice([8, 32]), stochastic=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------- sizes from the case
def _lens(case):
    """Length of each sequence: by the case alone, so that the work is known without the data."""
    if not case["ragged"]:
        return [case["seq_len"]] * case["n_seq"]
    r = random.Random(case["n_seq"] * 1000003 + case["seq_len"] * 101 + case["dim"])
    return [r.randint(0 if s % 7 == 3 else 1, case["seq_len"]) if s else case["seq_len"] for s in range(case["n_seq"])]


def _sizes(case):
    """Element counts of the tensors that one optimizer step updates."""
    if case["model"] == "mlp":
        w = (784, 128, 64, 10)
        return [n for a, b in zip(w[:-1], w[1:]) for n in (a * b, b)]
    if case["model"] == "lm":
        d, f, v = case["d"], case["dff"], case["vocab"]
        block = [d * d] * 4 + [d, d, d * f, f, f * d, d, d, d]   # q, k, v, output; norm; two dense layers; norm
        return ([v * d] if v else []) + block * case["layers"] + ([d * v, v] if v else [])
    r = random.Random(case["shape_seed"])
    return [_log(r, 1, case["largest"]) for _ in range(case["tensors"])]


def _blocks(case):
    return [-(-n // 256) for n in _sizes(case)]


def work(case):
    if case["op"] == "recurrence":
        n, one = sum(_lens(case)) * case["dim"], case["n_seq"] * case["dim"]
        ends = one * (bool(case["h0"]) + bool(case["last"]))
        total = 12 * n + 4 * ends
        flops = 10 * n
        if case["backward"]:   # gate, input, state and its gradient in, two gradients out
            total += 24 * n + 4 * ends
            flops += 14 * n
        return {"bytes": total, "flops": flops}
    if case["op"] == "qk":
        n = case["rows"] * (case["heads_q"] + case["heads_k"]) * case["d_head"]
        return {"bytes": 8 * n + (12 * n if case["backward"] else 0), "flops": 8 * n + (14 * n if case["backward"] else 0)}
    n = sum(_sizes(case))
    if case["bits"] == 32:
        return {"bytes": 28 * n, "flops": 15 * n}
    return {"bytes": 16 * n + 16 * sum(_blocks(case)), "flops": 40 * n}


# ----------------------------------------------------------------------------------------------------------- the inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape, scale=1.0, shift=0.0):
    return torch.randn(*shape, generator=g, device=DEV).mul_(scale).add_(shift)


def _strided(g, layout, S, L, D, scale=1.0, shift=0.0, base=None, half=0):
    """A [S, L, D] tensor in one of the three layouts (a view): sequence-major, time-major, or half of a fused projection."""
    if layout == "time":
        return _normal(g, L, S, D, scale=scale, shift=shift).transpose(0, 1)
    if layout == "fused":
        t = base if base is not None else torch.empty(S, L, 2 * D, device=DEV)
        t[..., half * D:(half + 1) * D] = _normal(g, S, L, D, scale=scale, shift=shift)
        return t[..., half * D:(half + 1) * D]
    return _normal(g, S, L, D, scale=scale, shift=shift)


def _empty_like_layout(layout, S, L, D):
    return torch.zeros(L, S, D, device=DEV).transpose(0, 1) if layout == "time" else torch.zeros(S, L, D, device=DEV)


def _prepare_recurrence(case, seed):
    g = _gen(seed)
    S, L, D, lay = case["n_seq"], case["seq_len"], case["dim"], case["layout"]
    s = {}
    base = torch.empty(S, L, 2 * D, device=DEV) if lay == "fused" else None
    if case["form"] == "gated":   # gates that keep most of the state, as trained ones do
        s["f"] = _strided(g, lay, S, L, D, scale=1.5, shift=2.0, base=base, half=0)
    else:                         # decays between about 0.5 and 1
        s["f"] = _strided(g, lay, S, L, D, scale=1.5, shift=2.5, base=base, half=0).sigmoid_()
    s["x"] = _strided(g, lay, S, L, D, base=base, half=1)
    s["h0"] = _normal(g, S, D) if case["h0"] else None
    s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=DEV) if case["ragged"] else None
    s["h"] = _empty_like_layout(lay, S, L, D)
    s["h_last"] = torch.zeros(S, D, device=DEV) if case["last"] else None
    if case["backward"]:
        s["dy"] = _normal(g, L, S, D).transpose(0, 1) if lay == "time" else _normal(g, S, L, D)
        s["dh_last"] = _normal(g, S, D) if case["last"] else None
        if lay == "fused":
            both = torch.zeros(S, L, 2 * D, device=DEV)
            s["df"], s["dx"] = both[..., :D], both[..., D:]
        else:
            s["df"], s["dx"] = _empty_like_layout(lay, S, L, D), _empty_like_layout(lay, S, L, D)
        s["dh0"] = torch.zeros(S, D, device=DEV) if case["h0"] else None
    return s


def _prepare_qk(case, seed):
    g = _gen(seed)
    R, d, pad = case["rows"], case["d_head"], case["pad"]
    wq, wk = case["heads_q"] * d, case["heads_k"] * d
    buf = _normal(g, R, wq + wk + pad)                      # [queries | keys | whatever else the projection holds]
    s = {"q": buf[:, :wq], "k": buf[:, wq:wq + wk], "q_out": torch.zeros(R, wq, device=DEV), "k_out": torch.zeros(R, wk, device=DEV)}
    if case["gain"]:
        s["gain_q"], s["gain_k"] = _normal(g, d, scale=0.1, shift=1.0), _normal(g, d, scale=0.1, shift=1.0)
    else:
        s["gain_q"] = s["gain_k"] = None
    high = 1000000 if case["far"] else 4096
    s["positions"] = None if case["seq_len"] else torch.randint(0, high, (R,), generator=g, device=DEV, dtype=torch.int32)
    if case["backward"]:
        s["dq_out"], s["dk_out"] = _normal(g, R, wq), _normal(g, R, wk)
        both = torch.zeros(R, wq + wk + pad, device=DEV)
        s["dq"], s["dk"] = both[:, :wq], both[:, wq:wq + wk]
        s["dgain_q"], s["dgain_k"] = (torch.zeros(d, device=DEV), torch.zeros(d, device=DEV)) if case["gain"] else (None, None)
    return s


def _prepare_adamw(case, seed):
    g = _gen(seed)
    sizes, blocks = _sizes(case), _blocks(case)
    NB = sum(blocks)
    first = [256 * sum(blocks[:i]) for i in range(len(blocks))]
    s = {"w": _normal(g, NB * 256, scale=0.02), "g": _normal(g, NB * 256, scale=1e-3), "t": 100, "hyper": (1e-3, 0.9, 0.999, 1e-8, 0.01)}
    size = torch.exp(_normal(g, NB, 1, scale=2.0)).expand(NB, 256).reshape(-1)   # gradients of very different size in the blocks
    s["g"].mul_(size)
    m = _normal(g, NB * 256, scale=3e-4).mul_(size)
    v = _normal(g, NB * 256, scale=1e-3).mul_(size).square_().mul_(0.8).add_(size.square().mul_(2e-7))
    for f, n, b in zip(first, sizes, blocks):               # the space behind each tensor's last element is no part of it
        for t in (s["w"], s["g"], m, v):
            t[f + n:f + 256 * b] = 0
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        s["m"], s["v"] = _pack(*_to_8(m, None, False)), _pack(*_to_8(v.sqrt_(), None, True))
        s["seed"] = 1234567 + int(seed) if case.get("stochastic") else -1
    s["at"] = list(zip(first, sizes))
    return s


def prepare(case, seed):
    s = {"recurrence": _prepare_recurrence, "qk": _prepare_qk, "adamw": _prepare_adamw}[case["op"]](case, seed)
    s["case"] = case
    if own:
        _hand_over(s)
    return s


# ------------------------------------------------------------------------------------------- through the framework
_ctx = None


def _hand_over(s):
    """The framework's context, its views of the buffers, and the optimizer's plan: what a program keeps between calls."""
    global _ctx
    from flutter_ml_b200 import _lib, ops
    if _ctx is None:
        _ctx = _lib.Context()
        _ctx.check(_ctx.lib.fml_set_stream(_ctx.h, torch.cuda.current_stream().cuda_stream))

    def arr(t):
        return _lib.DeviceArray(_ctx, t.data_ptr(), tuple(t.shape), np.int32 if t.dtype == torch.int32 else np.float32, owner=False)
    s["ops"], s["on"] = ops, {k: arr(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if s["case"]["op"] == "adamw":
        w, g = s["on"]["w"], s["on"]["g"]
        s["plan"] = ops.AdamWPlan(_ctx, [w.view(f, (n,)) for f, n in s["at"]], [g.view(f, (n,)) for f, n in s["at"]],
                                  s["on"]["m"], s["on"]["v"], stateBits=s["case"]["bits"])
    if s["case"]["op"] == "qk" and s["case"]["backward"]:
        s["scratch"] = _ctx.empty(ops.qk_norm_rope_scratch(s["case"]["d_head"]))


def _own_recurrence(s):
    c, o, ops = s["case"], s["on"], s["ops"]
    size = (c["n_seq"], c["seq_len"], c["dim"])
    at = dict(form=c["form"], h0=o.get("h0"), lens=o.get("lens"), strides_in=s["f"].stride()[:2], strides_h=s["h"].stride()[:2])
    ops.gated_recurrence_forward(_ctx, o["f"], o["x"], o["h"], *size, h_last=o.get("h_last"), **at)
    out = {"h": s["h"], "h_last": s["h_last"]}
    if c["backward"]:
        ops.gated_recurrence_backward(_ctx, o["f"], o["x"], o["h"], o["dy"], o["df"], o["dx"], *size, dh_last=o.get("dh_last"),
                                      dh0=o.get("dh0"), **at)
        out.update(df=s["df"], dx=s["dx"], dh0=s["dh0"])
    return out


def _own_qk(s):
    c, o, ops = s["case"], s["on"], s["ops"]
    at = dict(gain_q=o.get("gain_q"), gain_k=o.get("gain_k"), positions=o.get("positions"), seq_len=c["seq_len"], rot_dim=c["rot"],
              interleaved=c["interleaved"], base=c["base"], eps=1e-6, ld_q=s["q"].stride(0), ld_k=s["k"].stride(0))
    size = (c["rows"], c["heads_q"], c["heads_k"], c["d_head"])
    ops.qk_norm_rope_forward(_ctx, o["q"], o["k"], o["q_out"], o["k_out"], *size, **at)
    out = {"q": s["q_out"], "k": s["k_out"]}
    if c["backward"]:
        if c["gain"]:
            _ctx.zero(o["dgain_q"])
            _ctx.zero(o["dgain_k"])
        ops.qk_norm_rope_backward(_ctx, o["q"], o["k"], o["dq_out"], o["dk_out"], o["dq"], o["dk"], *size, scratch=s["scratch"],
                                  dgain_q=o.get("dgain_q"), dgain_k=o.get("dgain_k"), ld_dq=s["dq"].stride(0), ld_dk=s["dk"].stride(0), **at)
        out.update(dq=s["dq"], dk=s["dk"], dgain_q=s["dgain_q"], dgain_k=s["dgain_k"])
    return out


def _own_adamw(s):
    lr, b1, b2, eps, wd = s["hyper"]
    s["t"] += 1
    s["plan"].step(lr, b1, b2, eps, wd, s["t"], seed=s.get("seed", -1))
    return _adamw_out(s)


# --------------------------------------------------------------------------------------------------- the plain forms
def _scan(a, b, h0):
    """h_t = a_t h_{t-1} + b_t along dimension 1 by doubling; a and b are used up."""
    if h0 is not None:
        b[:, 0] += a[:, 0] * h0
    n, step = a.shape[1], 1
    while step < n:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _plain_recurrence(s):
    c, f, x, h0 = s["case"], s["f"], s["x"], s["h0"]
    L = c["seq_len"]
    gated = c["form"] == "gated"
    a = 1 / (1 + torch.exp(-f)) if gated else f.clone()
    keep = 1 / (1 + torch.exp(f)) if gated else None          # 1 - a, without the difference
    b = keep * x if gated else x.clone()
    inside = None
    if s["lens"] is not None:                                 # a step behind the end leaves the state as it is
        inside = (torch.arange(L, device=f.device)[None, :] < s["lens"][:, None])[..., None]
        a = torch.where(inside, a, torch.ones_like(a))
        b = torch.where(inside, b, torch.zeros_like(b))
    h = _scan(a.clone(), b, h0)
    out = {"h": h if inside is None else torch.where(inside, h, s["h"]), "h_last": h[:, -1].clone() if c["last"] else None}
    if not c["backward"]:
        return out
    first = h0[:, None] if h0 is not None else torch.zeros_like(h[:, :1])
    before = torch.cat([first, h[:, :-1]], 1)
    dy = s["dy"] if inside is None else torch.where(inside, s["dy"], torch.zeros_like(s["dy"]))
    dy = dy.flip(1)
    later = torch.cat([torch.ones_like(a[:, :1]), a.flip(1)[:, :-1]], 1)   # the decay behind each step, from the end
    G = _scan(later, dy.clone(), s["dh_last"]).flip(1)
    dx = keep * G if gated else G
    df = G * (before - x) * a * keep if gated else G * before
    if inside is not None:
        dx, df = torch.where(inside, dx, s["dx"]), torch.where(inside, df, s["df"])
    out.update(df=df, dx=dx, dh0=a[:, 0] * G[:, 0] if c["h0"] else None)
    return out


def _angles(s, dtype):
    c = s["case"]
    pos = s["positions"] if s["positions"] is not None else torch.arange(c["rows"], device=DEV) % c["seq_len"]
    i = torch.arange(c["rot"] // 2, device=DEV, dtype=torch.float64)
    ang = pos.double()[:, None, None] * c["base"] ** (-2.0 * i / c["rot"])
    return torch.cos(ang).to(dtype), torch.sin(ang).to(dtype)


def _rotate(z, cos, sin, rot, interleaved):
    if interleaved:
        a, b = z[..., 0:rot:2], z[..., 1:rot:2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = z[..., :rot // 2], z[..., rot // 2:rot]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([r, z[..., rot:]], -1)


def _plain_qk(s):
    c = s["case"]
    cos, sin = _angles(s, torch.float32)
    out, back = {}, {}
    for n in ("q", "k"):
        x = s[n].unflatten(1, (c["heads_" + n], c["d_head"]))
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        xh = x * r
        gain = s["gain_" + n]
        out[n] = _rotate(xh * gain if c["gain"] else xh, cos, sin, c["rot"], c["interleaved"]).flatten(1)
        if c["backward"]:
            dz = _rotate(s["d%s_out" % n].unflatten(1, (c["heads_" + n], c["d_head"])), cos, -sin, c["rot"], c["interleaved"])
            dxh = dz * gain if c["gain"] else dz
            back["d" + n] = (r * (dxh - xh * (dxh * xh).mean(-1, keepdim=True))).flatten(1)
            back["dgain_" + n] = (dz * xh).sum((0, 1)) if c["gain"] else None
    return {**out, **back}


def _mix(x):
    """A mixer of 32-bit numbers, held in 64 bits."""
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x85EBCA77) & 0xFFFFFFFF
    return x ^ (x >> 13)


def _random_words(NB, seed, t):
    """One 32-bit word for each element: by seed, step, block and place in the block."""
    one = lambda v: torch.tensor(v & 0xFFFFFFFF, dtype=torch.int64, device=DEV)  # noqa: E731
    key = _mix(_mix(_mix(one(seed)) ^ one(seed >> 32)) ^ one(t))
    block = _mix((key + torch.arange(NB, dtype=torch.int64, device=DEV) * 0x9E3779B1) & 0xFFFFFFFF)
    return _mix((block[:, None] + torch.arange(256, dtype=torch.int64, device=DEV)[None, :]) & 0xFFFFFFFF).reshape(-1)


def _to_8(x, words, root):
    """Blocks of 256 values in 8 bits (4 exponent and 3 fraction bits) times a power of two for each block: the smallest
    that brings the block's largest finite value to 448 at most.  `words` None rounds to the nearest, ties to even; else
    the dropped bits are rounded up with their own probability, from the upper (`root`: lower) half of each word.  What is
    not finite becomes NaN; a positive `root` stays positive.  Returns (codes, scales)."""
    x = x.view(-1, 256)
    size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    bits = size.amax(1).view(torch.int32)
    e = (((bits + 0x1FFFFF) >> 23) - 127 - 8).clamp(min=-126)
    scale = torch.exp2(e.double()).float()
    y = size * torch.exp2(-e.double()).float()[:, None]
    small = y < 2.0 ** -6
    z = torch.where(small, y + 2.0 ** -6, y).view(torch.int32)
    if words is None:
        up = 0x7FFFF + ((z >> 20) & 1)
    else:
        up = ((words & 0xFFFF if root else words >> 16) << 4).view(-1, 256).int()
    code = ((z + up) >> 20) - (120 << 3) - 8 * small.int()
    if root:
        code = torch.where((code == 0) & (x > 0), torch.ones_like(code), code)
    code = torch.where(torch.isfinite(x), code, torch.full_like(code, 127))
    return (code + 128 * torch.signbit(x).int() if not root else code).to(torch.uint8), scale


def _pack(codes, scale):
    """One buffer of 32-bit words: the codes of all blocks, then their scales."""
    return torch.cat([codes.reshape(-1).view(torch.float32), scale])


def _unpack(buf):
    NB = buf.numel() // 65
    return buf[:NB * 64].view(torch.float8_e4m3fn).view(NB, 256), buf[NB * 64:]


def _adamw_out(s):
    if s["case"]["bits"] == 32:
        return {"w": s["w"], "m": s["m"], "v": s["v"]}
    (mc, ms), (rc, rs) = _unpack(s["m"]), _unpack(s["v"])
    return {"w": s["w"], "m": mc, "m_scale": ms, "root_v": rc, "v_scale": rs}


def _plain_adamw(s):
    lr, b1, b2, eps, wd = s["hyper"]
    s["t"] += 1
    t, w, g, eight = s["t"], s["w"], s["g"], s["case"]["bits"] == 8
    if eight:
        (mc, ms), (rc, rs) = _unpack(s["m"]), _unpack(s["v"])
        m = (mc.float() * ms[:, None]).view(-1)
        v = (rc.float() * rs[:, None]).view(-1).square()
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = torch.sqrt(v)
    w -= (lr / (1 - b1 ** t)) * m / (root * (1 / math.sqrt(1 - b2 ** t)) + eps)
    w -= (lr * wd) * w
    if eight:
        words = _random_words(rs.numel(), s["seed"], t) if s["seed"] >= 0 else None
        s["m"].copy_(_pack(*_to_8(m, words, False)))
        s["v"].copy_(_pack(*_to_8(root, words, True)))
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _adamw_out(s)


def run(s):
    op = s["case"]["op"]
    if own:
        return {"recurrence": _own_recurrence, "qk": _own_qk, "adamw": _own_adamw}[op](s)
    return {"recurrence": _plain_recurrence, "qk": _plain_qk, "adamw": _plain_adamw}[op](s)


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_recurrence(case, s):
    S, L, D = case["n_seq"], case["seq_len"], case["dim"]
    f, x = s["f"].double(), s["x"].double()
    lens = s["lens"].long() if s["lens"] is not None else torch.full((S,), L, device=DEV)
    gated = case["form"] == "gated"
    a = torch.sigmoid(f) if gated else f
    keep = torch.sigmoid(-f) if gated else torch.ones_like(f)
    state = s["h0"].double() if case["h0"] else torch.zeros(S, D, dtype=torch.float64, device=DEV)
    H = torch.zeros(S, L + 1, D, dtype=torch.float64, device=DEV)
    H[:, 0] = state
    live = [(t < lens)[:, None] for t in range(L)] if case["ragged"] else None
    for t in range(L):
        new = a[:, t] * state + keep[:, t] * x[:, t]
        state = torch.where(live[t], new, state) if live else new
        H[:, t + 1] = state
    there = torch.arange(L, device=DEV)[None, :, None] < lens[:, None, None]
    out = {"h": torch.where(there, H[:, 1:], torch.zeros_like(x)), "h_last": state.clone() if case["last"] else None}
    if not case["backward"]:
        return out
    c = s["dh_last"].double() if case["last"] else torch.zeros(S, D, dtype=torch.float64, device=DEV)   # what flows back into h_t
    dy, df, dx = s["dy"].double(), torch.zeros_like(x), torch.zeros_like(x)
    for t in reversed(range(L)):
        G = dy[:, t] + c
        gx = keep[:, t] * G
        gf = G * ((H[:, t] - x[:, t]) * a[:, t] * keep[:, t] if gated else H[:, t])
        if live:
            G, gx, gf = (torch.where(live[t], v, torch.zeros_like(v)) for v in (G, gx, gf))
            c = torch.where(live[t], a[:, t] * G, c)
        else:
            c = a[:, t] * G
        dx[:, t], df[:, t] = gx, gf
    out.update(df=df, dx=dx, dh0=c if case["h0"] else None)
    return out


def _exact_qk(case, s):
    d, rot, R = case["d_head"], case["rot"], case["rows"]
    pos = s["positions"].double() if s["positions"] is not None else (torch.arange(R, device=DEV) % case["seq_len"]).double()
    theta = torch.tensor([case["base"] ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device=DEV)
    turn = torch.polar(torch.ones(R, rot // 2, dtype=torch.float64, device=DEV), pos[:, None] * theta)[:, None]   # e^{i angle}
    one = torch.arange(rot, device=DEV).view(-1, 2) if case["interleaved"] else torch.arange(rot, device=DEV).view(2, -1).t()

    def rotated(z, by):                                     # pairs as complex numbers
        pair = torch.complex(z[..., one[:, 0]], z[..., one[:, 1]]) * by
        z = z.clone()
        z[..., one[:, 0]], z[..., one[:, 1]] = pair.real, pair.imag
        return z
    out, back = {}, {}
    for n in ("q", "k"):
        H = case["heads_" + n]
        x = s[n].double().reshape(R, H, d)
        r = 1 / torch.sqrt(x.square().sum(-1, keepdim=True) / d + 1e-6)
        gain = s["gain_" + n].double() if case["gain"] else torch.ones(d, dtype=torch.float64, device=DEV)
        out[n] = rotated(x * r * gain, turn).reshape(R, -1)
        if case["backward"]:
            dz = rotated(s["d%s_out" % n].double().reshape(R, H, d), turn.conj())
            back["dgain_" + n] = torch.einsum("rhd,rhd->d", dz, x * r) if case["gain"] else None
            dz = dz * gain
            back["d" + n] = (r * dz - x * r ** 3 * (dz * x).sum(-1, keepdim=True) / d).reshape(R, -1)
    return {**out, **back}


def _exact_adamw(case, s):
    lr, b1, b2, eps, wd = s["hyper"]
    t, g = s["t"] + 1, s["g"].double()
    if case["bits"] == 8:
        (mc, ms), (rc, rs) = _unpack(s["m"]), _unpack(s["v"])
        m0, v0 = (mc.double() * ms.double()[:, None]).view(-1), (rc.double() * rs.double()[:, None]).view(-1) ** 2
    else:
        m0, v0 = s["m"].double(), s["v"].double()
    m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
    w = s["w"].double()
    w = w - lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    w = w - lr * wd * w
    if case["bits"] == 32:
        return {"w": w, "m": m, "v": v}
    return {"w": w, "m": None, "m_scale": None, "root_v": None, "v_scale": None}   # roundings have no 64-bit value


def exact(case, seed):
    kind = {"recurrence": _prepare_recurrence, "qk": _prepare_qk, "adamw": _prepare_adamw}[case["op"]]
    s = kind(case, seed)
    return {"recurrence": _exact_recurrence, "qk": _exact_qk, "adamw": _exact_adamw}[case["op"]](case, s)
