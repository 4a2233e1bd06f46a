"""Norm of queries and keys with the position rotation (fml_qk_norm_rope_*, ops, T.qkNormRope, MultiHeadAttention(qkNorm=True)).

Bounds from counting roundings, u = 2^-24 each.  Forward: the mean of squares is a sum of up to 13 nested additions of
positive terms, the root halves its error, with reciprocal, eps and the two products an element of z is off by at most 12 u;
a cosine by the rounding of the angle's fraction (pi u) and 2 ulp; two products and a sum: 32 u (|za| + |zb|).  Far positions
add what 53 bits leave of the angle, in the kernel and in the reference: 16 u (|za| + |zb|) more.  Backward: dz is off by
16 u (|dya| + |dyb|) = 16 u D, products with gain and xh by 14 u more, the mean by 14 u, r and the last two operations by
14 u: 64 u r (gain D + |xh| mean(gain D |xh|)).  dgain: each term off by 30 u D |xh|, and one rounding for each of the
at most rows * heads + 20 additions that a term passes through.
"""
import numpy as np
import pytest

U = 2.0 ** -24
f32 = np.float32


def pairs(rot, interleaved):
    i = np.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def turn(z, pos, rot, interleaved, base, sign=1.0):
    """z [rows, heads, d] turned by sign * angle; and |za| + |zb| for every element."""
    a, b = pairs(rot, interleaved)
    ang = pos[:, None].astype(np.float64) * base ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
    c, s = np.cos(ang)[:, None], sign * np.sin(ang)[:, None]
    out, size = z.copy(), np.abs(z)
    out[..., a], out[..., b] = z[..., a] * c - z[..., b] * s, z[..., a] * s + z[..., b] * c
    size[..., a] = size[..., b] = np.abs(z[..., a]) + np.abs(z[..., b])
    return out, size


def reference(x, gain, pos, rot, interleaved, base, eps, dy=None):
    """x, dy [rows, heads, d] float64 -> y, its bound; with dy also dx, dgain and their bounds."""
    rows, heads, d = x.shape
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xh = x * r
    y, size = turn(xh * gain, pos, rot, interleaved, base)
    far = 16 if np.abs(pos).max(initial=0) > 1 << 20 else 0
    out = [y, (32 + far) * U * size]
    if dy is not None:
        dz, D = turn(dy, pos, rot, interleaved, base, -1.0)
        gz, gD = dz * gain, D * np.abs(gain)
        dx = r * (gz - xh * (gz * xh).mean(-1, keepdims=True))
        out += [dx, (64 + far) * U * r * (gD + np.abs(xh) * (gD * np.abs(xh)).mean(-1, keepdims=True))]
        out += [(dz * xh).sum((0, 1)), (rows * heads + 50 + far) * U * (D * np.abs(xh)).sum((0, 1))]
    return out


def test_dividing_by_multiplying_is_exact_where_it_is_used():
    """The kernel counts a CTA's heads through and divides by the heads of a row with floor(n ceil(2^32 / h) / 2^32); it takes
    at most 2^31 / h^2 rows (or one) at a time, so n < 2^31 / h or n < h."""
    rng = np.random.default_rng(0)
    for h in [2, 3, 5, 7, 12, 100, 127, 128, 1000, 5792, 5793, 8191, 11585, 11586, 20000, 32767, 32768] + list(rng.integers(2, 32769, 200)):
        h = int(h)
        most = h * max(1, min(32, 2 ** 31 // (h * h)))
        n = np.unique(np.concatenate([np.arange(min(most, 5000)), most - 1 - np.arange(min(most, 5000)), np.arange(h - 1, most, h), np.arange(0, most, h)]))
        n = n.astype(np.uint64)
        assert np.array_equal((n * np.uint64(-(-2 ** 32 // h))) >> np.uint64(32), n // np.uint64(h)), h


def test_gains_of_another_head_width_are_refused():
    """The kernels read d_head elements of each gain, so a shorter one must not get that far."""
    from types import SimpleNamespace
    from flutter_ml_b200 import tensor as T
    gain = lambda n: SimpleNamespace(value=SimpleNamespace(size=n, shape=(n,)))  # noqa: E731
    for gq, gk in ((gain(63), None), (None, gain(63)), (gain(64), gain(128))):
        norm, x = T.QKNorm(gq, gk), SimpleNamespace(view=lambda *a: None)
        with pytest.raises(ValueError):
            norm.forward(None, x, x, 4, 4, 2, 2, 64, 256, 256)
        gradient = SimpleNamespace(grad=0)
        for g in norm.inputs:
            g.grad = gradient
        ctx = SimpleNamespace(empty=lambda *a: None)
        with pytest.raises(ValueError):
            norm.backward(ctx, x, x, x, 4, 4, 2, 2, 64, 256, 256, False)


@pytest.fixture(scope="module")
def ctx():
    from flutter_ml_b200 import _lib
    c = _lib.Context()
    yield c
    assert c.device_status() == 0
    c.close()


class Case:
    """Queries and keys as neighbouring slices of one [rows, hq d + hk d + pad] buffer that starts `shift` floats in."""

    def __init__(self, ctx, rows, hq, hk, d, rot, interleaved=False, pad=0, shift=0, positions="far", gain=True, base=10000.0, seed=0):
        rng = np.random.default_rng(seed + rows + d)
        self.ctx, self.rows, self.h, self.d, self.rot = ctx, rows, (hq, hk), d, rot
        self.inter, self.base, self.eps = interleaved, base, 1e-6
        self.w = (hq * d, hk * d)
        self.ld, self.shift = hq * d + hk * d + pad, shift
        self.host = rng.standard_normal(shift + rows * self.ld).astype(f32)
        if rows > 2:
            self.host[shift + self.ld:shift + self.ld + d] = 0        # a head of zeros
            self.host[shift + 2 * self.ld:shift + 2 * self.ld + d] *= f32(1e12)
        self.buf = ctx.upload(self.host)
        self.gains = [rng.standard_normal(d).astype(f32) if gain else None for _ in range(2)]
        self.dgains = [ctx.upload(g) if gain else None for g in self.gains]
        if positions == "far":
            self.pos = rng.integers(-5, 1 << 20, rows).astype(np.int32)
        elif positions == "farthest":
            self.pos = np.concatenate([[2 ** 31 - 1, -2 ** 31], rng.integers(1 << 30, 2 ** 31 - 1, rows)])[:rows].astype(np.int32)
        else:
            self.pos = (np.arange(rows) % positions if positions else np.arange(rows)).astype(np.int64)
        self.dpos = ctx.upload(self.pos) if isinstance(positions, str) else None
        self.seq_len = 0 if isinstance(positions, str) else positions
        self.dy = [rng.standard_normal((rows, w)).astype(f32) for w in self.w]

    def side(self, t):
        x = self.host[self.shift:].reshape(self.rows, self.ld)[:, t * self.w[0]:t * self.w[0] + self.w[t]]
        return x.reshape(self.rows, self.h[t], self.d).astype(np.float64)

    def views(self, buf, shift=None):
        o = self.shift if shift is None else shift
        return [buf.view(o, (self.rows, self.ld)), buf.view(o + self.w[0], ()) if self.h[1] else None]

    def ref(self, t, backward=False):
        g = self.gains[t].astype(np.float64) if self.gains[t] is not None else np.ones(self.d)
        return reference(self.side(t), g, self.pos, self.rot, self.inter, self.base, self.eps,
                         self.dy[t].reshape(self.rows, self.h[t], self.d).astype(np.float64) if backward else None)

    def options(self):
        return dict(gain_q=self.dgains[0], gain_k=self.dgains[1] if self.h[1] else None, positions=self.dpos, seq_len=self.seq_len, rot_dim=self.rot,
                    interleaved=self.inter, base=self.base, eps=self.eps, ld_q=self.ld, ld_k=self.ld)

    def forward(self, out=None, ld_out=None):
        from flutter_ml_b200 import ops
        q, k = self.views(self.buf)
        o = out or [self.ctx.upload(np.full((self.rows, w), 7, f32)) if w else None for w in self.w]
        ops.qk_norm_rope_forward(self.ctx, q, k, o[0], o[1], self.rows, *self.h, self.d, ld_q_out=ld_out, ld_k_out=ld_out, **self.options())
        return o

    def backward(self, grad, dgain, accumulate=False, dy=None):
        from flutter_ml_b200 import ops
        q, k = self.views(self.buf)
        gq, gk = self.views(grad)
        dy = dy or [self.ctx.upload(y) if y.size else None for y in self.dy]
        scratch = self.ctx.empty(ops.qk_norm_rope_scratch(self.d)) if dgain else None
        ops.qk_norm_rope_backward(self.ctx, q, k, dy[0], dy[1], gq, gk, self.rows, *self.h, self.d, scratch=scratch, accumulate=accumulate,
                                  dgain_q=dgain[0] if dgain else None, dgain_k=dgain[1] if dgain and self.h[1] else None, ld_dq=self.ld,
                                  ld_dk=self.ld, **self.options())


def close(got, ref, bound, what):
    assert got.shape == ref.shape, what
    bad = ~(np.abs(got.astype(np.float64) - ref) <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(np.abs(got - ref)[bad].max()), float(bound[bad].min()))


CASES = [
    dict(rows=1, hq=1, hk=0, d=1, rot=0),
    dict(rows=1, hq=1, hk=1, d=2, rot=2, interleaved=True),
    dict(rows=3, hq=2, hk=1, d=7, rot=4, pad=1),                                  # odd width: pairs, the last alone
    dict(rows=5, hq=3, hk=3, d=8, rot=8, gain=False),
    dict(rows=37, hq=4, hk=2, d=32, rot=32),
    dict(rows=33, hq=5, hk=1, d=32, rot=16, interleaved=True, pad=4),
    dict(rows=130, hq=16, hk=4, d=64, rot=64, positions=128),
    dict(rows=130, hq=16, hk=4, d=64, rot=64, positions="farthest"),
    dict(rows=65, hq=3, hk=2, d=64, rot=64, interleaved=True, positions="farthest", base=500000.0),
    dict(rows=64, hq=4, hk=4, d=64, rot=64, shift=1),                             # an address that float4 cannot take
    dict(rows=64, hq=4, hk=4, d=64, rot=64, pad=3, interleaved=True),             # a stride that float4 cannot take
    dict(rows=50, hq=12, hk=3, d=80, rot=32, interleaved=True, pad=7),
    dict(rows=50, hq=12, hk=3, d=80, rot=32, pad=8),
    dict(rows=51, hq=2, hk=2, d=96, rot=48),
    dict(rows=40, hq=2, hk=1, d=100, rot=100),                                    # not a multiple of 8
    dict(rows=40, hq=8, hk=8, d=128, rot=128, positions=0),
    dict(rows=40, hq=8, hk=1, d=160, rot=80, interleaved=True),
    dict(rows=31, hq=2, hk=2, d=255, rot=254),
    dict(rows=31, hq=2, hk=2, d=256, rot=256, gain=False),
    dict(rows=31, hq=2, hk=2, d=256, rot=0),
    dict(rows=20000, hq=2, hk=1, d=64, rot=64, positions=512),                    # more rows than one round of CTAs takes
    dict(rows=3001, hq=1, hk=1, d=10, rot=6),
    dict(rows=77, hq=5, hk=2, d=24, rot=8),
    dict(rows=1300, hq=700, hk=1, d=8, rot=8, gain=False),                        # many heads, two and three rows a CTA
    dict(rows=201, hq=7, hk=7, d=40, rot=40, shift=2),
    dict(rows=45, hq=9, hk=3, d=72, rot=64, interleaved=True),
    dict(rows=700, hq=1, hk=1, d=16, rot=0),
    dict(rows=4999, hq=12, hk=3, d=80, rot=32, interleaved=True, pad=7),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_forward_and_backward(ctx, case):
    c = Case(ctx, **case)
    out = c.forward()
    grad0 = np.random.default_rng(1).standard_normal(c.host.size).astype(f32)
    grad, dg = ctx.upload(grad0), [ctx.upload(np.full(c.d, 3, f32)) for _ in range(2)] if c.gains[0] is not None else None
    c.backward(grad, dg)
    g = grad.numpy()
    assert np.array_equal(g[:c.shift], grad0[:c.shift])
    g, g0 = g[c.shift:].reshape(c.rows, c.ld), grad0[c.shift:].reshape(c.rows, c.ld)
    assert np.array_equal(g[:, sum(c.w):], g0[:, sum(c.w):])                      # what lies behind the keys is left alone
    added = ctx.upload(grad0)
    c.backward(added, None, accumulate=True)
    added = added.numpy()[c.shift:].reshape(c.rows, c.ld)
    for t in range(2):
        if not c.h[t]:
            continue
        y, by, dx, bdx, dgain, bg = c.ref(t, True)
        shape = (c.rows, c.h[t], c.d)
        close(out[t].numpy().reshape(shape), y, by, "out")
        at = slice(t * c.w[0], t * c.w[0] + c.w[t])
        close(g[:, at].reshape(shape), dx, bdx, "gradient")
        old = g0[:, at].reshape(shape).astype(np.float64)
        close(added[:, at].reshape(shape), dx + old, bdx + U * (np.abs(dx) + np.abs(old) + bdx), "added gradient")
        if dg:
            close(dg[t].numpy(), dgain + 3, bg + 2 * U * (np.abs(dgain) + 3), "gain gradient")


@pytest.mark.gpu
def test_repeats_bit_for_bit_and_in_place(ctx):
    """Two runs agree exactly (no atomics); writing over the inputs gives the same values."""
    c = Case(ctx, rows=700, hq=6, hk=2, d=64, rot=32, pad=4)
    a = [o.numpy() for o in c.forward()]
    g1, g2 = ctx.zeros(c.host.size), ctx.zeros(c.host.size)
    d1, d2 = [ctx.zeros(64), ctx.zeros(64)], [ctx.zeros(64), ctx.zeros(64)]
    c.backward(g1, d1)
    c.backward(g2, d2)
    assert np.array_equal(g1.numpy(), g2.numpy()) and all(np.array_equal(x.numpy(), y.numpy()) for x, y in zip(d1, d2))
    # the gradient in place of the one that came in: dq_out holds dq afterwards
    q, k = c.views(ctx.upload(c.host))
    wide = np.zeros((c.rows, c.ld), f32)
    wide[:, :c.w[0]], wide[:, c.w[0]:sum(c.w)] = c.dy
    both = ctx.upload(wide)
    from flutter_ml_b200 import ops
    bq, bk = both, both.view(c.w[0], ())
    ops.qk_norm_rope_backward(ctx, q, k, bq, bk, bq, bk, c.rows, *c.h, c.d, ld_dq_out=c.ld, ld_dk_out=c.ld, ld_dq=c.ld, ld_dk=c.ld, **c.options())
    assert np.array_equal(both.numpy()[:, :sum(c.w)], g1.numpy().reshape(c.rows, c.ld)[:, :sum(c.w)])
    c.forward(out=c.views(c.buf), ld_out=c.ld)
    now = c.buf.numpy().reshape(c.rows, c.ld)
    assert np.array_equal(now[:, :c.w[0]], a[0]) and np.array_equal(now[:, c.w[0]:sum(c.w)], a[1])
    assert np.array_equal(now[:, sum(c.w):], c.host.reshape(c.rows, c.ld)[:, sum(c.w):])


@pytest.mark.gpu
def test_gradient_against_differences(ctx):
    """d(sum y dy) / dx and / dgain by central differences of the kernel's own forward pass, steps of 2^-6: the differences
    are off by the third derivative's share, below 2e-3 of the gradient's size here, and by rounding, 2^-24 * 2^6 * sqrt(n)."""
    c = Case(ctx, rows=2, hq=2, hk=1, d=16, rot=8)
    dg = [ctx.zeros(16), ctx.zeros(16)]
    grad = ctx.zeros(c.host.size)
    c.backward(grad, dg)
    g, h = grad.numpy(), 2.0 ** -6

    def loss():
        return sum(float((o.numpy().astype(np.float64) * y).sum()) for o, y in zip(c.forward(), c.dy))

    def slope(buf, host, i):
        v = []
        for sgn in (1, -1):
            x = host.copy()
            x[i] += sgn * h
            ctx.upload(x, out=buf)
            v.append(loss())
        ctx.upload(host, out=buf)
        return (v[0] - v[1]) / (2 * h)
    tol = 2e-3 * np.abs(g).max() + 2.0 ** -18 * 8
    for i in range(0, c.host.size, 5):
        assert abs(slope(c.buf, c.host, i) - g[i]) <= tol, i
    for t in range(2):
        for i in range(0, 16, 3):
            assert abs(slope(c.dgains[t], c.gains[t], i) - dg[t].numpy()[i]) <= 2.0 ** -18 * 8 * 8


@pytest.mark.gpu
def test_not_finite_values_stay_in_their_head(ctx):
    c = Case(ctx, rows=4, hq=3, hk=2, d=64, rot=64)
    clean = [o.numpy() for o in c.forward()]
    c.host[c.ld + 64 + 3] = np.nan       # row 1, second query head
    c.host[3 * c.ld + c.w[0] + 5] = np.inf   # row 3, first key head
    ctx.upload(c.host, out=c.buf)
    q, k = (o.numpy() for o in c.forward())
    assert np.isnan(q[1, 64:128]).all() and np.isnan(k[3, 5]) and not k[3, [i for i in range(64) if i not in (5, 37)]].any()
    q[1, 64:128], k[3, :64] = clean[0][1, 64:128], clean[1][3, :64]
    assert np.array_equal(q, clean[0]) and np.array_equal(k, clean[1])


@pytest.mark.gpu
def test_recorded_and_replayed(ctx):
    c = Case(ctx, rows=300, hq=4, hk=4, d=64, rot=64)
    grad, dg = ctx.zeros(c.host.size), [ctx.zeros(64), ctx.zeros(64)]
    dy = [ctx.upload(y) for y in c.dy]
    out = c.forward()
    c.backward(grad, dg, dy=dy)
    ref = [o.numpy() for o in out] + [grad.numpy(), dg[0].numpy(), dg[1].numpy()]
    ctx.sync()
    ctx.graph_begin()
    c.forward(out=out)
    for d in dg:
        ctx.zero(d)
    c.backward(grad, dg, dy=dy)
    gid = ctx.graph_end()
    for b in (*out, grad):
        ctx.zero(b)
    for _ in range(2):
        ctx.graph_launch(gid)
    ctx.sync()
    for got, want in zip([*out, grad, *dg], ref):
        assert np.array_equal(got.numpy(), want)
    ctx.check(ctx.lib.fml_graph_destroy(ctx.h, gid))


@pytest.mark.gpu
def test_no_rows_is_no_work(ctx):
    from flutter_ml_b200 import ops
    b = ctx.zeros(64)
    ops.qk_norm_rope_forward(ctx, b, None, b, None, 0, 1, 0, 64)
    ops.qk_norm_rope_backward(ctx, b, None, b, None, b, None, 0, 1, 0, 64)


@pytest.mark.gpu
def test_refusals(ctx):
    from flutter_ml_b200 import _lib, ops
    x, y = ctx.zeros(8, 256), ctx.zeros(8, 256)

    def fwd(**kw):
        a = dict(q=x, k=x.view(64, ()), q_out=y, k_out=y.view(64, ()), rows=8, heads_q=1, heads_k=1, d_head=64, ld_q=256, ld_k=256, ld_q_out=256,
                 ld_k_out=256)
        a.update(kw)
        ops.qk_norm_rope_forward(ctx, **a)
    fwd()
    for bad in (dict(d_head=257), dict(d_head=0), dict(heads_q=0), dict(heads_k=-1), dict(rows=-1), dict(rot_dim=63), dict(rot_dim=66),
                dict(eps=0.0), dict(base=0.0), dict(ld_q=32), dict(ld_k_out=63), dict(seq_len=-1), dict(q=None), dict(k_out=None),
                dict(q_out=x.view(32, ())),                    # over its own input, moved
                dict(q_out=x.view(64, ())),                    # over the keys
                dict(q_out=x, ld_q_out=128),                   # its own input at another stride
                dict(k_out=y.view(32, ()))):                   # over the other output
        with pytest.raises(_lib.FmlError):
            fwd(**bad)

    with pytest.raises(ValueError):
        fwd(positions=ctx.zeros(8))

    def bwd(**kw):
        a = dict(q=x, k=None, dq_out=y, dk_out=None, dq=y, dk=None, rows=8, heads_q=1, heads_k=0, d_head=64)
        a.update(kw)
        ops.qk_norm_rope_backward(ctx, **a)
    bwd()
    g, s = ctx.zeros(64), ctx.zeros(ops.qk_norm_rope_scratch(64))
    for bad in (dict(dq_out=None), dict(dgain_q=g, scratch=s), dict(gain_q=g, dgain_q=g), dict(accumulate=True), dict(gain_k=g, dgain_k=g, scratch=s)):
        with pytest.raises(_lib.FmlError):
            bwd(**bad)
    with pytest.raises(ValueError):
        bwd(gain_q=g, dgain_q=g, scratch=g)
    for bad in (dict(dgain_k=g), dict(dgain_k=s.view(100, (64,))), dict(dgain_q=s.view(0, (64,)), dgain_k=g)):   # sums into one place
        with pytest.raises(_lib.FmlError):
            bwd(**{**dict(k=x.view(64, ()), dk_out=ctx.zeros(8, 256), dk=ctx.zeros(8, 256), heads_k=1, gain_q=g, gain_k=g, dgain_q=g, scratch=s,
                          ld_k=256, ld_q=256), **bad})


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("twice", [False, True])
def test_attention_layer_with_norm_and_rotation(ctx, fused, twice):
    """MultiHeadAttention(qkNorm=True) on the tape, with the fused attention kernels and without, against torch in float64:
    output, input and parameter gradients within the TF32 bound of the attention and projection products that the other
    attention tests use (1e-3 relative for each product; three products and the attention forward, twice that backward).
    `twice` backpropagates a second output through the same projection, so gradients are added."""
    import torch
    from flutter_ml_b200 import layers, synth
    from flutter_ml_b200 import tensor as T
    S, n, d, H = 128, 2, 128, 2
    x0 = synth.normal(5, 0, (n * S, d))
    dout = synth.normal(5, 1, (n * S, d))
    old, T.FUSE_ATTENTION = T.FUSE_ATTENTION, fused
    try:
        calls = T.fused_attention_calls
        layer = layers.MultiHeadAttention(d, H, seq_len=S, causal=True, seed=3, qkNorm=True)
        x = T.Tensor(x0, ctx)
        layer.build(x)
        for i, g in enumerate((layer.gainQ, layer.gainK)):
            ctx.upload(synth.normal(6, i, (d // H,), 0.2) + np.float32(1), out=g.value)
        x.zeroGrad()
        assert len(layer.parameters) == 4
        qkv = T.denseMatrix(x, layer.Wqkv, None, None)
        outs = [T.attentionCore(qkv, n, S, H, d // H, True, -1, layer._qk_norm()) for _ in range(2 if twice else 1)]
        o = T.addMatrix(*outs) if twice else outs[0]
        y = T.denseMatrix(o, layer.Wo, None, None)
        assert (T.fused_attention_calls > calls) == fused
        y.grad = ctx.upload(dout)
        y.backward()
        if not twice:
            assert np.array_equal(layer(T.Tensor(x0, ctx)).numpy(), y.numpy())
    finally:
        T.FUSE_ATTENTION = old
    t = {k: torch.tensor(v.numpy().astype(np.float64), requires_grad=True) for k, v in
         dict(w=layer.Wqkv, o=layer.Wo, gq=layer.gainQ, gk=layer.gainK).items()}
    tx = torch.tensor(x0.astype(np.float64), requires_grad=True)
    qkv_t = (tx @ t["w"]).reshape(n, S, 3, H, d // H)

    def normed(z, g):
        z = z / torch.sqrt((z * z).mean(-1, keepdim=True) + 1e-6) * g
        half = d // H // 2
        ang = torch.arange(S, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
        c, s = torch.cos(ang)[None, :, None], torch.sin(ang)[None, :, None]
        a, b = z[..., :half], z[..., half:]
        return torch.cat([a * c - b * s, a * s + b * c], -1)
    q, k, v = normed(qkv_t[:, :, 0], t["gq"]), normed(qkv_t[:, :, 1], t["gk"]), qkv_t[:, :, 2]
    sc = torch.einsum("nihd,njhd->nhij", q, k) / np.sqrt(d // H)
    sc = sc.masked_fill(torch.triu(torch.ones(S, S, dtype=torch.bool), 1), -torch.inf)
    att = torch.einsum("nhij,njhd->nihd", torch.softmax(sc, -1), v).reshape(n * S, d) * (2 if twice else 1)
    yt = att @ t["o"]
    yt.backward(torch.tensor(dout.astype(np.float64)))

    def rel(a, b):
        b = b.detach().numpy()
        return np.linalg.norm(a.astype(np.float64) - b) / np.linalg.norm(b)
    assert rel(y.numpy(), yt) <= 4e-3
    for got, want in ((x.grad, tx.grad), (layer.Wqkv.grad, t["w"].grad), (layer.Wo.grad, t["o"].grad), (layer.gainQ.grad, t["gq"].grad),
                      (layer.gainK.grad, t["gk"].grad)):
        assert rel(got.numpy(), want) <= 8e-3


@pytest.mark.gpu
@pytest.mark.parametrize("heads_k", [0, 2])
def test_one_gain_for_queries_and_keys(ctx, heads_k):
    """The same Tensor as both gains (or with no keys): its gradient is the sum of both sides', added once each."""
    from flutter_ml_b200 import tensor as T
    rng = np.random.default_rng(6)
    C = (2 + heads_k) * 32
    x0, dy, g0 = (rng.standard_normal(s).astype(f32) for s in ((40, C), (40, C), 32))
    x, g = T.Tensor(x0, ctx), T.Tensor(g0, ctx)
    y = T.qkNormRope(x, 2, heads_k, 32, T.QKNorm(g, g), seq_len=40)
    assert y.creator.inputs == [x, g]
    y.grad = ctx.upload(dy)
    y.backward()
    r = reference(x0.reshape(40, -1, 32).astype(np.float64), g0.astype(np.float64), np.arange(40), 32, False, 10000.0, 1e-6,
                  dy.reshape(40, -1, 32).astype(np.float64))
    close(g.grad.numpy(), r[4], r[5] + 2 * U * np.abs(r[4]), "gain gradient")
    close(x.grad.numpy().reshape(40, -1, 32), r[2], r[3], "gradient")


@pytest.mark.gpu
def test_tape_node_leaves_the_values_out(ctx):
    """T.qkNormRope reads the first columns of a projection; the columns behind them get a zero gradient, or keep theirs."""
    from flutter_ml_b200 import tensor as T
    rng = np.random.default_rng(4)
    x0 = rng.standard_normal((24, 3 * 32 + 10)).astype(f32)
    dy = rng.standard_normal((24, 96)).astype(f32)
    g = rng.standard_normal(32).astype(f32)
    grads = []
    for start in (None, 2.0):
        x, gq = T.Tensor(x0, ctx), T.Tensor(g, ctx)
        if start is not None:
            x.grad = ctx.upload(np.full(x0.shape, start, f32))
        y = T.qkNormRope(x, 2, 1, 32, T.QKNorm(gain_q=gq, rot_dim=16), seq_len=8)
        y.grad = ctx.upload(dy)
        y.backward()
        grads.append((x.grad.numpy(), gq.grad.numpy()))
        pos = np.arange(24) % 8
        for cols, h, gain in ((slice(0, 64), 2, g.astype(np.float64)), (slice(64, 96), 1, np.ones(32))):
            xs, ys = x0[:, cols].reshape(24, h, 32).astype(np.float64), dy[:, cols].reshape(24, h, 32).astype(np.float64)
            r = reference(xs, gain, pos, 16, False, 10000.0, 1e-6, ys)
            close(y.numpy()[:, cols].reshape(24, h, 32), r[0], r[1], "out")
            add = start or 0.0
            close(x.grad.numpy()[:, cols].reshape(24, h, 32), r[2] + add, r[3] + 2 * U * (np.abs(r[2]) + add), "gradient")
        assert (x.grad.numpy()[:, 96:] == (start or 0.0)).all()
    assert np.array_equal(grads[0][1], grads[1][1])
    with pytest.raises(ValueError):
        T.qkNormRope(T.Tensor(x0, ctx), 3, 1, 32)


@pytest.mark.gpu
def test_misaligned_addresses_are_refused(ctx):
    """An address that is no multiple of four bytes would fault in the kernels; each buffer of both calls, one after the other."""
    import ctypes
    from flutter_ml_b200 import _lib
    d, rows = 64, 8
    b, s = ctx.zeros(8192), ctx.zeros(_lib.QK_NORM_ROPE_PARTS * 2 * d + 4)
    at = lambda o: ctypes.c_void_p(b.ptr + 4 * o)  # noqa: E731
    gq, gk, dgq, dgk, pos, scratch = at(7000), at(7064), at(7128), at(7192), at(7256), ctypes.c_void_p(s.ptr)
    fwd = [at(0), d, at(512), d, 1, at(1024), d, at(1536), d, 1, rows, d, gq, gk, pos, 0, d, 0, 10000.0, 1e-6]
    bwd = [at(0), d, at(512), d, at(1024), d, 1, at(1536), d, at(2048), d, at(2560), d, 1, rows, d, gq, gk, dgq, dgk, pos, 0, d, 0, 10000.0, 1e-6, 0, scratch]
    for name, args in (("fml_qk_norm_rope_fwd", fwd), ("fml_qk_norm_rope_bwd", bwd)):
        call = lambda a: getattr(ctx.lib, name)(ctx.h, *a)  # noqa: E731
        assert call(args) == 0
        for i, v in enumerate(args):
            if isinstance(v, ctypes.c_void_p):
                for k in (1, 2):
                    assert call(args[:i] + [ctypes.c_void_p(v.value + k)] + args[i + 1:]) != 0, (name, i)
                    assert b"misaligned" in ctx.lib.fml_last_error(ctx.h)
    ctx.sync()


# ---- gain gradients against a bound from the additions that a term really passes through
GAINS = [dict(rows=20000, hq=2, hk=1, d=64, rot=64, positions=512),                 # every place taken, two rounds of angles a CTA
         dict(rows=4999, hq=12, hk=3, d=80, rot=32, interleaved=True, pad=7),
         dict(rows=9001, hq=3, hk=3, d=128, rot=128, positions=1000),
         dict(rows=6000, hq=5, hk=2, d=24, rot=8),
         dict(rows=5000, hq=2, hk=2, d=256, rot=0, positions=0),
         dict(rows=3001, hq=1, hk=1, d=10, rot=6),                                    # pairs
         dict(rows=7000, hq=3, hk=2, d=100, rot=100, positions=64)]


def shares(case, sms):
    """(grid, first row of each CTA's share and the end, rows at once) of a backward launch."""
    rows, heads = case["rows"], max(case["hq"], case["hk"])
    grid = min(rows, 3 * sms, 592)
    first = [rows // grid * b + min(b, rows % grid) for b in range(grid + 1)]
    return grid, first, min(32, 8192 // max(case["rot"], 1), -(-rows // grid), max(1, 2 ** 31 // heads ** 2))


def additions(case, t, sms):
    """Additions on a term's way into the gain gradient of queries (t = 0) or keys: its lane's items, the heads beside it in
    the warp, the warps, the partial sums of the second kernel, its shuffles, the old value."""
    grid, first, at_once = shares(case, sms)
    d, heads = case["d"], (case["hq"], case["hk"])
    share = max(b - a for a, b in zip(first, first[1:]))
    groups = [min(at_once, share - r) for r in range(0, share, at_once)]
    if d % 8 or case["rot"] % 8:
        return sum(-(-n * sum(heads) // 8) for n in groups) + 8 + 19 + 5 + 1
    beside = 32 // (4 if d <= 32 else 8 if d <= 64 else 16 if d <= 128 else 32)
    return sum(-(-n * heads[t] // (8 * beside)) for n in groups) + int(np.log2(beside)) + 8 + 19 + 5 + 1


def gain_gradient(c, t, sms, case):
    """The reference, and its bound: 30 u of each term (16 more at far positions), and one rounding an addition."""
    r = c.ref(t, True)
    far = 16 if np.abs(c.pos).max() > 1 << 20 else 0
    terms = r[5] / ((c.rows * c.h[t] + 50 + far) * U)          # the sum of D |xh|
    return r[4], (30 + far + additions(case, t, sms)) * U * terms


@pytest.mark.parametrize("case", GAINS, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_the_gain_bound_sees_a_lost_share(case):
    """Without the rows of one CTA, the first, the last or one between, or without the second round of a CTA's rows, the gain
    gradients are off by more than the bound in most columns."""
    from types import SimpleNamespace
    c = Case(SimpleNamespace(upload=lambda a, **kw: a), **case)
    grid, first, at_once = shares(case, 148)
    lost = [(first[b], first[b + 1]) for b in (0, grid // 2, grid - 1)]
    if first[1] > at_once:
        lost.append((first[1] - (first[1] - at_once), first[1]))
    for t in range(2):
        want, bound = gain_gradient(c, t, 148, case)
        for a, b in lost:
            kept = np.r_[0:a, b:c.rows]
            g = c.gains[t].astype(np.float64)
            x, dy = c.side(t)[kept], c.dy[t].reshape(c.rows, c.h[t], c.d).astype(np.float64)[kept]
            less = reference(x, g, c.pos[kept], c.rot, c.inter, c.base, c.eps, dy)[4]
            assert np.mean(np.abs(less - want) > 3 * bound) > 0.8, (t, a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("case", GAINS, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_gain_gradients_of_whole_grids(ctx, case):
    c = Case(ctx, **case)
    dg = [ctx.zeros(c.d), ctx.zeros(c.d)]
    c.backward(ctx.zeros(c.host.size), dg)
    for t in range(2):
        want, bound = gain_gradient(c, t, ctx.sm_count(), case)
        close(dg[t].numpy(), want, bound, "gain gradient")
