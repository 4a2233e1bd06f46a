"""Gated linear recurrence (fml_gated_recurrence_*, ops, T.gatedRecurrence, GatedRecurrentLayer) against float64.

Bounds from counting roundings, u = 2^-24 each, to first order.  A gate is off by at most (8 + 1.25 |f|) u (the exponential's
argument, rounded in base 2 with a rounded constant: 1.25 |f| u; the exponential 4 u, the sum 1 u, the reciprocal 2 u, a
product), a LINEAR one is exact.  However the steps are grouped, a result is
the recurrence with every decay off by its own error, one product and one sum: with S_t = |a| S_{t-1} + |s x| the recurrence
of absolute values, the error obeys E_t = |a| E_{t-1} + k u (|a| S_{t-1} + |s x_t|), k = 4 and, GATED, the gate's, the joins
of segments, at most one a step, included; 4 u S_t more for the last roundings.  Backward the same with T_t = |dy_t| + C_{t+1},
C_t = |a| T_t; dx and df are products of G with gates (two of them: 2 (k - 4) + 8 u), and of the difference of two given numbers (2 u of each).
"""
import numpy as np
import pytest

U = 2.0 ** -24
f32 = np.float32


def gates(f, form):
    f = f.astype(np.float64)
    with np.errstate(over="ignore"):
        return (1 / (1 + np.exp(-f)), 1 / (1 + np.exp(f))) if form == "gated" else (f, np.ones_like(f))


def rounding(f, form):
    return 12 + 1.25 * np.abs(np.nan_to_num(f.astype(np.float64), posinf=80, neginf=80)) if form == "gated" else np.full(f.shape, 4.0)


def forward64(f, x, h0, lens, form):
    """[n_seq, seq_len, dim] -> h, its bound, the last state, its bound."""
    a, s = gates(f, form)
    k = rounding(f, form)
    x = x.astype(np.float64)
    state = h0.astype(np.float64).copy()
    S, E = np.abs(state), np.zeros_like(state)
    h, bound = np.zeros_like(x), np.zeros_like(x)
    for t in range(x.shape[1]):
        on = (t < lens)[:, None]
        add, dec = s[:, t] * x[:, t], np.abs(a[:, t])
        E = np.where(on, dec * E + k[:, t] * U * (dec * S + np.abs(add)), E)
        S = np.where(on, dec * S + np.abs(add), S)
        state = np.where(on, a[:, t] * state + add, state)
        h[:, t], bound[:, t] = state, E + 4 * U * S
    return h, 1.05 * bound + 1e-37, state, 1.05 * (E + 4 * U * S) + 1e-37


def backward64(f, x, h0, h, dy, dh_last, lens, form):
    """-> (df, its bound), (dx, its bound), (dh0, its bound), from the given h."""
    a, s = gates(f, form)
    k = rounding(f, form)
    x, h, dy = x.astype(np.float64), h.astype(np.float64), dy.astype(np.float64)
    before = np.concatenate([h0.astype(np.float64)[:, None], h[:, :-1]], 1)
    c = dh_last.astype(np.float64).copy()
    C, E = np.abs(c), np.zeros_like(c)
    df, dx, bf, bx = (np.zeros_like(x) for _ in range(4))
    for t in reversed(range(x.shape[1])):
        on = (t < lens)[:, None]
        G, T, EG = dy[:, t] + c, np.abs(dy[:, t]) + C, E + 2 * U * (np.abs(dy[:, t]) + C)
        d = before[:, t] - x[:, t] if form == "gated" else before[:, t]
        D = np.abs(before[:, t]) + np.abs(x[:, t]) if form == "gated" else np.abs(d)
        w = a[:, t] * s[:, t] if form == "gated" else np.ones_like(G)
        dx[:, t], bx[:, t] = s[:, t] * G, s[:, t] * (EG + 2 * k[:, t] * U * T)
        df[:, t], bf[:, t] = G * d * w, w * (np.abs(d) * (EG + 2 * k[:, t] * U * T) + 2 * U * D * T)
        E = np.where(on, np.abs(a[:, t]) * EG + k[:, t] * U * np.abs(a[:, t]) * T, E)
        C = np.where(on, np.abs(a[:, t]) * T, C)
        c = np.where(on, a[:, t] * G, c)
        for v in (df, dx, bf, bx):
            v[:, t] = np.where(on, v[:, t], 0)
    return (df, 1.05 * bf + 1e-37), (dx, 1.05 * bx + 1e-37), (c, 1.05 * (E + 4 * U * C) + 1e-37)


@pytest.fixture(scope="module")
def ctx():
    from flutter_ml_b200 import _lib
    c = _lib.Context()
    yield c
    assert c.device_status() == 0
    c.close()


class Case:
    def __init__(self, ctx, n_seq, seq_len, dim, form="gated", layout="sequence", ragged=False, ends=True, seed=0, lead=1):
        rng = np.random.default_rng(seed + n_seq * 7 + seq_len + dim)
        self.ctx, self.size, self.form, self.layout = ctx, (n_seq, seq_len, dim), form, layout
        self.f = (1.5 * rng.standard_normal((n_seq, seq_len, dim)) + 2).astype(f32)
        if form == "linear":
            self.f = (1 / (1 + np.exp(-self.f)) * np.where(rng.random(self.f.shape) < 0.1, -1, 1)).astype(f32)
        self.x = rng.standard_normal((n_seq, seq_len, dim)).astype(f32)
        self.dy = rng.standard_normal((n_seq, seq_len, dim)).astype(f32)
        self.h0 = rng.standard_normal((n_seq, dim)).astype(f32) if ends else np.zeros((n_seq, dim), f32)
        self.dh_last = rng.standard_normal((n_seq, dim)).astype(f32) if ends else np.zeros((n_seq, dim), f32)
        self.ends, self.lead = ends, lead   # lead: floats in front of every array
        self.lens = np.full(n_seq, seq_len)
        if ragged:
            self.lens = rng.integers(0, seq_len + 1, n_seq)
            self.lens[0] = seq_len
            self.lens[-1] = 0 if n_seq > 1 else self.lens[-1]
        self.dlens = ctx.upload(self.lens.astype(np.int32)) if ragged else None
        # strides in elements, and the distance of x from f
        gap = 3 if layout == "padded" else 0
        if layout == "time":
            self.si = self.sh = (dim, n_seq * dim)
            self.apart = n_seq * seq_len * dim
        elif layout == "fused":
            self.si, self.sh, self.apart = (seq_len * 2 * dim, 2 * dim), (seq_len * dim, dim), dim
        elif layout == "padded":
            self.si = self.sh = (seq_len * (dim + gap) + 5, dim + gap)
            self.apart = n_seq * (seq_len * (dim + gap) + 5) + 1
        else:
            self.si = self.sh = (seq_len * dim, dim)
            self.apart = n_seq * seq_len * dim
        span = (n_seq - 1) * self.si[0] + (seq_len - 1) * self.si[1] + dim
        self.n_in, self.n_h = span + self.apart + 1 + self.lead, (n_seq - 1) * self.sh[0] + (seq_len - 1) * self.sh[1] + dim + 1 + self.lead

    def index(self, strides, start=0):
        n, t, d = self.size
        return start + np.arange(n)[:, None, None] * strides[0] + np.arange(t)[None, :, None] * strides[1] + np.arange(d)

    def place(self, n, parts, fill=7.0):
        host = np.full(n, fill, f32)
        for idx, v in parts:
            host[idx] = v
        return host

    def inputs(self):
        b = self.ctx.upload(self.place(self.n_in, [(self.index(self.si, self.lead), self.f), (self.index(self.si, self.lead + self.apart), self.x)]))
        return b.view(self.lead, ()), b.view(self.lead + self.apart, ()), b

    def forward(self, h=None, h0=None, last=None):
        from flutter_ml_b200 import ops
        f, x, keep = self.inputs()
        h = h or self.ctx.upload(self.place(self.n_h, []))
        h0 = h0 or (self.ctx.upload(self.h0) if self.ends else None)
        last = last or self.ctx.upload(np.full(self.h0.shape, 7, f32))
        ops.gated_recurrence_forward(self.ctx, f, x, h.view(self.lead, ()), *self.size, form=self.form, h0=h0, lens=self.dlens, h_last=last,
                                     strides_in=self.si, strides_h=self.sh)
        return h, last

    def backward(self, h, out=None, dh0=None, accumulate=False, dy=True):
        from flutter_ml_b200 import ops
        f, x, keep = self.inputs()
        hd = self.ctx.upload(self.place(self.n_h, [(self.index(self.sh, self.lead), h)]))
        dyd = self.ctx.upload(self.place(self.n_h, [(self.index(self.sh, self.lead), self.dy)])) if dy else None
        out = out or self.ctx.upload(self.place(self.n_in, []))
        dh0 = dh0 or self.ctx.upload(np.full(self.h0.shape, 7, f32))
        ops.gated_recurrence_backward(self.ctx, f, x, hd.view(self.lead, ()), dyd.view(self.lead, ()) if dy else None, out.view(self.lead, ()),
                                      out.view(self.lead + self.apart, ()), *self.size, form=self.form, h0=self.ctx.upload(self.h0) if self.ends else None,
                                      lens=self.dlens, dh_last=self.ctx.upload(self.dh_last) if self.ends else None, dh0=dh0,
                                      strides_in=self.si, strides_h=self.sh, accumulate=accumulate)
        return out, dh0


def close(got, ref, bound, what):
    bad = ~(np.abs(got.astype(np.float64) - ref) <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(np.abs(got - ref)[bad].max()), float(bound[bad].min()))


SIZES = [(1, 1, 1), (128, 1, 512), (3, 2, 33), (2, 4, 70), (2, 5, 5), (1, 16, 32), (3, 17, 31), (2, 129, 64), (5, 127, 40), (80, 300, 32),
         (40, 257, 65), (5, 1000, 64), (3, 2049, 24), (1, 5000, 8), (1, 9001, 1), (1, 4097, 250), (300, 130, 96), (2, 700, 600), (1, 20000, 64), (1, 13000, 130), (40, 60, 130), (50, 40, 33), (3, 150, 1667)]


def both_directions(ctx, size, layout, ragged, form, lead):
    c = Case(ctx, *size, form=form, layout=layout, ragged=ragged, ends=layout != "fused", lead=lead)
    there = (np.arange(size[1])[None, :] < c.lens[:, None])[..., None] & np.ones(size, bool)
    ref, bound, last, blast = forward64(c.f, c.x, c.h0, c.lens, form)
    h, end = c.forward()
    flat = h.numpy()
    got = flat[c.index(c.sh, lead)]
    close(np.where(there, got, 0), np.where(there, ref, 0), bound, "h")
    assert (got[~there] == 7).all()                                      # rows behind the ends, and all around
    around = np.ones(c.n_h, bool)
    around[c.index(c.sh, lead)] = False
    assert (flat[around] == 7).all()
    close(end.numpy(), last, blast, "h_last")
    given = np.where(there, ref, 0).astype(f32)
    rf, rx, r0 = backward64(c.f, c.x, c.h0, given, c.dy, c.dh_last, c.lens, form)
    out, dh0 = c.backward(given)
    flat = out.numpy()
    for start, (r, b), what in ((lead, rf, "df"), (lead + c.apart, rx, "dx")):
        got = flat[c.index(c.si, start)]
        close(np.where(there, got, 0), r, b, what)
        assert (got[~there] == 7).all()
    around = np.ones(c.n_in, bool)
    around[c.index(c.si, lead)] = around[c.index(c.si, lead + c.apart)] = False
    assert (flat[around] == 7).all()
    close(dh0.numpy(), *r0, "dh0")
    again, dh0b = c.backward(given, ctx.upload(np.full(c.n_in, 2, f32)), ctx.upload(np.full(c.h0.shape, 2, f32)), accumulate=True)
    flat2 = again.numpy()
    for start in (lead, lead + c.apart):
        i = c.index(c.si, start)
        assert np.array_equal(flat2[i], np.where(there, flat[i] + f32(2), f32(2)))
    assert np.array_equal(dh0b.numpy(), dh0.numpy() + f32(2))


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["gated", "linear"])
@pytest.mark.parametrize("layout,ragged", [("sequence", False), ("sequence", True), ("time", True), ("fused", True), ("padded", False)])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward_and_backward(ctx, size, layout, ragged, form):
    both_directions(ctx, size, layout, ragged, form, 1)


# Addresses that let a lane take two or four channels at once, and among the sizes one for every way of sharing out the
# channels: many and few sequences, few and many channels, one CTA for all steps or clusters of them.
WIDE = [(4, s) for s in [(5, 3, 64), (150, 20, 512), (160, 20, 192), (8, 600, 1000), (75, 300, 64), (1, 5000, 64), (2, 2000, 192),
                         (1, 9001, 256), (1, 700, 2600), (3, 129, 20)]]
WIDE += [(2, s) for s in [(5, 4, 66), (300, 20, 130), (160, 20, 98), (8, 300, 1022), (50, 100, 50), (40, 300, 62), (1, 3000, 18),
                          (2, 2000, 250), (1, 2500, 1350), (3, 150, 64)]]
WIDE += [(1, (40, 300, 33))]


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["gated", "linear"])
@pytest.mark.parametrize("layout,ragged", [("sequence", False), ("time", True), ("fused", True)])
@pytest.mark.parametrize("lead,size", WIDE, ids=str)
def test_wide_loads(ctx, lead, size, layout, ragged, form):
    both_directions(ctx, size, layout, ragged, form, lead)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(2, 3, 40), (4, 300, 64), (1, 3000, 16)], ids=str)
def test_only_the_last_state_has_a_gradient(ctx, size):
    """dy = NULL is dy = 0."""
    c = Case(ctx, *size, ragged=True)
    c.dy[:] = 0
    h = forward64(c.f, c.x, c.h0, c.lens, "gated")[0].astype(f32)
    a, a0 = c.backward(h)
    b, b0 = c.backward(h, dy=False)
    assert np.array_equal(a.numpy(), b.numpy()) and np.array_equal(a0.numpy(), b0.numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(7, 260, 100), (1, 6000, 20)], ids=str)
def test_repeats_bit_for_bit_also_recorded(ctx, size):
    c = Case(ctx, *size, layout="time", ragged=True)
    h, last = c.forward()
    ref = h.numpy(), last.numpy()
    given = np.where(np.isin(ref[0][c.index(c.sh, 1)], 7.0), 0, ref[0][c.index(c.sh, 1)]).astype(f32)
    out, d0 = c.backward(given)
    refb = out.numpy(), d0.numpy()
    h2, last2 = c.forward()
    out2, d02 = c.backward(given)
    for x, y in zip((h2, last2, out2, d02), ref + refb):
        assert np.array_equal(x.numpy(), y)
    from flutter_ml_b200 import ops
    f, x, keep = c.inputs()
    h0, lens = ctx.upload(c.h0), c.dlens
    ctx.sync()
    ctx.graph_begin()
    ops.gated_recurrence_forward(ctx, f, x, h2.view(1, ()), *c.size, form=c.form, h0=h0, lens=lens, h_last=last2, strides_in=c.si, strides_h=c.sh)
    gid = ctx.graph_end()
    ctx.zero(last2)
    for _ in range(2):
        ctx.graph_launch(gid)
    ctx.sync()
    assert np.array_equal(h2.numpy(), ref[0]) and np.array_equal(last2.numpy(), ref[1])
    ctx.check(ctx.lib.fml_graph_destroy(ctx.h, gid))


@pytest.mark.gpu
def test_token_by_token_is_the_whole_sequence(ctx):
    """seq_len = 1 with the state handed on in place (h_last is h0), against one call over all steps: each within its bound."""
    c = Case(ctx, 6, 40, 48)
    ref, bound, last, blast = forward64(c.f, c.x, c.h0, c.lens, "gated")
    from flutter_ml_b200 import ops
    state = ctx.upload(c.h0)
    for t in range(40):
        f, x, h = ctx.upload(c.f[:, t].copy()), ctx.upload(c.x[:, t].copy()), ctx.empty(6, 48)
        ops.gated_recurrence_forward(ctx, f, x, h, 6, 1, 48, h0=state, h_last=state)
        close(h.numpy(), ref[:, t], bound[:, t], t)
    assert np.array_equal(h.numpy(), state.numpy())
    both, end = c.forward(h0=state, last=state)          # in place in the scan kernel too
    ref2, b2, last2, bl2 = forward64(c.f, c.x, h.numpy(), c.lens, "gated")
    close(state.numpy(), last2, bl2, "last")


@pytest.mark.gpu
@pytest.mark.parametrize("seq_len", [3, 200, 3000])
def test_values_that_are_not_finite(ctx, seq_len):
    """A NaN spoils its channel from its step on, an infinite gate is a gate of 0 or 1; the other channels are untouched."""
    c = Case(ctx, 2, seq_len, 20)
    clean = c.forward()[0].numpy()[c.index(c.sh, 1)]
    t = seq_len // 2
    c.x[0, t, 3] = np.nan
    c.f[1, t, 5], c.f[1, t, 6] = np.inf, -np.inf
    h, last = c.forward()
    h = h.numpy()[c.index(c.sh, 1)]
    assert np.isnan(h[0, t:, 3]).all() and np.array_equal(h[0, :t, 3], clean[0, :t, 3]) and np.isnan(last.numpy()[0, 3])
    assert h[1, t, 5] == (h[1, t - 1, 5] if t else c.h0[1, 5]) and h[1, t, 6] == c.x[1, t, 6]
    rest = np.ones(20, bool)
    rest[[3, 5, 6]] = False
    assert np.array_equal(h[..., rest], clean[..., rest])


@pytest.mark.gpu
def test_growing_decays_on_a_state_of_zero(ctx):
    """LINEAR with decays of 2: products of 512 of them overflow, a state of zero stays zero until the first input."""
    c = Case(ctx, 1, 2000, 8, form="linear", ends=False)
    c.f[:] = 2
    c.x[:] = 0
    c.x[0, 1990] = 1
    h = c.forward()[0].numpy()[c.index(c.sh, 1)]
    want = np.zeros(2000)
    want[1990:] = 2.0 ** np.arange(10)
    assert np.array_equal(h[0], np.repeat(want[:, None], 8, 1).astype(f32))


@pytest.mark.gpu
def test_gradient_against_differences(ctx):
    """Central differences of the kernel's forward pass, step 2^-7: off by the third derivative's share (below 1e-3 of the
    largest gradient for these gates) and by rounding, 2^-24 * 2^7 * the loss's size."""
    for form in ("gated", "linear"):
        c = Case(ctx, 2, 21, 4, form=form)
        h = forward64(c.f, c.x, c.h0, c.lens, form)[0].astype(f32)
        out, d0 = c.backward(h)
        flat = out.numpy()
        df, dx = flat[c.index(c.si, 1)], flat[c.index(c.si, 1 + c.apart)]

        def loss():
            hh, last = c.forward()
            hh = hh.numpy()[c.index(c.sh, 1)].astype(np.float64)
            return (hh * c.dy).sum() + (last.numpy().astype(np.float64) * c.dh_last).sum(), np.abs(hh * c.dy).sum()

        def slope(v, i, e=2.0 ** -7):
            old = v[i]
            v[i] = old + e
            up, size = loss()
            v[i] = old - e
            down = loss()[0]
            v[i] = old
            return (up - down) / (2 * e), size
        for arr, g in ((c.f, df), (c.x, dx), (c.h0, d0.numpy())):
            for i in list(np.ndindex(arr.shape))[::7]:
                s, size = slope(arr, i)
                assert abs(s - g[i]) <= 1e-3 * np.abs(g).max() + 2.0 ** -17 * size, (form, i)


@pytest.mark.gpu
@pytest.mark.parametrize("seq_len", [2, 9])
def test_offsets_beyond_32_bits(ctx, seq_len):
    """Rows 2^31 elements and more apart (steps of a projection whose rows are very wide)."""
    from flutter_ml_b200 import ops
    dim, rng = 24, np.random.default_rng(0)
    ts = (1 << 31) // (seq_len - 1) + 8
    f, x = rng.standard_normal((seq_len, dim)).astype(f32), rng.standard_normal((seq_len, dim)).astype(f32)
    big = ctx.empty((seq_len - 1) * ts + 2 * dim)
    for t in range(seq_len):
        ctx.upload(f[t], out=big.view(t * ts, (dim,)))
        ctx.upload(x[t], out=big.view(t * ts + dim, (dim,)))
    h = ctx.empty(seq_len, dim)
    ops.gated_recurrence_forward(ctx, big, big.view(dim, ()), h, 1, seq_len, dim, strides_in=(0, ts), strides_h=(0, dim))
    ref, bound, _, _ = forward64(f[None], x[None], np.zeros((1, dim), f32), np.array([seq_len]), "gated")
    close(h.numpy(), ref[0], bound[0], "h")
    big.free()


@pytest.mark.gpu
def test_bad_lengths_are_reported_and_clamped():
    from flutter_ml_b200 import _lib, ops
    ctx = _lib.Context()
    for seq_len in (3, 50):
        f, x, h = ctx.zeros(3, seq_len, 8), ctx.upload(np.ones((3, seq_len, 8), f32)), ctx.zeros(3, seq_len, 8)
        last = ctx.zeros(3, 8)
        ops.gated_recurrence_forward(ctx, f, x, h, 3, seq_len, 8, lens=ctx.upload(np.array([-4, seq_len, seq_len + 9], np.int32)), h_last=last)
        with pytest.raises(_lib.FmlError, match="sequence length"):
            ctx.device_status()
        assert ctx.device_status() == 0
        out = h.numpy()
        assert not out[0].any() and np.array_equal(out[1], out[2]) and out[1].all() and not last.numpy()[0].any()
    ctx.close()


@pytest.mark.gpu
def test_empty_calls(ctx):
    from flutter_ml_b200 import ops
    h0, last = ctx.upload(np.arange(8, dtype=f32)), ctx.zeros(8)
    ops.gated_recurrence_forward(ctx, None, None, None, 2, 0, 4, h0=h0, h_last=last)
    assert np.array_equal(last.numpy(), np.arange(8))
    ops.gated_recurrence_backward(ctx, None, None, None, None, None, None, 2, 0, 4, dh_last=h0, dh0=last)
    assert np.array_equal(last.numpy(), np.arange(8))
    ops.gated_recurrence_forward(ctx, None, None, None, 0, 5, 4)


@pytest.mark.gpu
def test_refusals(ctx):
    from flutter_ml_b200 import _lib, ops
    b = ctx.zeros(4096)
    at = lambda o: b.view(o, ())  # noqa: E731
    n = 2 * 5 * 8

    def fwd(**kw):
        a = dict(f=at(0), x=at(n), h=at(2 * n), n_seq=2, seq_len=5, dim=8, h0=at(3 * n), h_last=at(3 * n + 16))
        a.update(kw)
        ops.gated_recurrence_forward(ctx, **a)
    fwd()
    fwd(strides_in=(0, 8))                       # a gate shared by the sequences is only read
    for bad in (dict(n_seq=-1), dict(seq_len=-1), dict(dim=0), dict(f=None), dict(x=None), dict(h=None), dict(strides_in=(-40, 8)),
                dict(strides_h=(40, 4)), dict(strides_h=(8, 8)), dict(h=at(0)), dict(h=at(n - 8)), dict(h=at(3 * n - 4)), dict(h_last=at(2 * n)),
                dict(h_last=at(3 * n + 8)), dict(h_last=at(4))):
        with pytest.raises(_lib.FmlError):
            fwd(**bad)
    with pytest.raises(KeyError):
        fwd(form="other")
    with pytest.raises(ValueError):
        fwd(lens=at(3 * n))
    with pytest.raises(_lib.FmlError):
        ctx.call("fml_gated_recurrence_fwd", 2, 2, 5, 8, at(0), at(n), 40, 8, None, None, at(2 * n), 40, 8, None)

    def bwd(**kw):
        a = dict(f=at(0), x=at(n), h=at(2 * n), dy=at(3 * n), df=at(4 * n), dx=at(5 * n), n_seq=2, seq_len=5, dim=8, h0=at(6 * n),
                 dh_last=at(6 * n + 16), dh0=at(6 * n + 32))
        a.update(kw)
        ops.gated_recurrence_backward(ctx, **a)
    bwd()
    bwd(dh0=at(6 * n + 16))                      # dh_last in place
    fused = dict(f=at(0), x=at(8), df=at(4 * n), dx=at(4 * n + 8), strides_in=(80, 16))
    bwd(**fused)
    for bad in (dict(df=None), dict(dx=None), dict(h=None), dict(df=at(5 * n)), dict(df=at(0)), dict(dx=at(3 * n)), dict(dx=at(2 * n + 8)),
                dict(dh0=at(6 * n + 16), accumulate=True), dict(dh0=at(6 * n)), dict(dh0=at(0)), dict(strides_in=(0, 8)),
                dict(fused, dx=at(4 * n + 4)), dict(fused, dx=at(4 * n + 16)), dict(fused, dx=at(4 * n + 80))):
        with pytest.raises(_lib.FmlError):
            bwd(**bad)


@pytest.mark.gpu
@pytest.mark.parametrize("output", ["all", "last"])
@pytest.mark.parametrize("ragged", [False, True])
def test_layer_on_the_tape(ctx, output, ragged):
    """GatedRecurrentLayer (products in FP32 mode) against torch autograd in float64: 1e-5 relative, the FP32 bound of the
    dense products (TOL_FP32 of the other tests)."""
    import torch
    from flutter_ml_b200 import _lib, layers, synth
    from flutter_ml_b200 import tensor as T
    n, S, I, H = 3, 37, 20, 24
    layer = layers.GatedRecurrentLayer(H, seq_len=S, returnSequences=output == "all", seed=4, precision=_lib.PREC_FP32)
    x = T.Tensor(synth.normal(1, 0, (n * S, I)), ctx)
    layer.build(x)
    x.zeroGrad()
    lens = np.array([S, 0, 11], np.int32) if ragged else np.full(3, S, np.int32)
    h0 = T.Tensor(synth.normal(1, 1, (n, H)), ctx)
    h0.grad = ctx.upload(np.full((n, H), 0.5, f32))       # an existing gradient is added to
    y = layer.forward(x, lens=ctx.upload(lens) if ragged else None, h0=h0)
    dy = synth.normal(1, 2, y.shape)
    y.grad = ctx.upload(dy)
    y.backward()
    tt = {k: torch.tensor(v.numpy().astype(np.float64), requires_grad=True) for k, v in dict(x=x, w=layer.weights, b=layer.biases, h0=h0).items()}
    z = (tt["x"] @ tt["w"] + tt["b"]).reshape(n, S, 2 * H)
    a, state, out = torch.sigmoid(z[..., :H]), tt["h0"], []
    for t in range(S):
        on = torch.tensor((t < lens)[:, None])
        state = torch.where(on, a[:, t] * state + (1 - a[:, t]) * z[:, t, H:], state)
        out.append(torch.where(on, state, torch.zeros_like(state)))
    want = torch.stack(out, 1).reshape(n * S, H) if output == "all" else state
    want.backward(torch.tensor(dy.astype(np.float64)))
    rel = lambda p, q: np.linalg.norm(p.astype(np.float64) - q.detach().numpy()) / np.linalg.norm(q.detach().numpy())  # noqa: E731
    assert rel(y.numpy(), want) <= 1e-5
    # adding to 0.5 rounds each of the n H sums by at most u (0.5 + |g|), so the difference's norm by u (0.5 sqrt(n H) + |g|)
    g0 = tt["h0"].grad.numpy()
    off = np.linalg.norm(h0.grad.numpy().astype(np.float64) - 0.5 - g0)
    assert off <= 1e-5 * np.linalg.norm(g0) + U * (0.5 * np.sqrt(n * H) + np.linalg.norm(g0))
    for p, q in ((x, "x"), (layer.weights, "w"), (layer.biases, "b")):
        assert rel(p.grad.numpy(), tt[q].grad) <= 1e-5
    for bad in (dict(n_seq=2, seq_len=S), dict(n_seq=n, seq_len=S, output="first"), dict(n_seq=n, seq_len=S, lens=ctx.zeros(3))):
        with pytest.raises(ValueError):
            T.gatedRecurrence(T.Tensor(np.zeros((n * S, 2 * H), f32), ctx), **bad)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["sequence", "fused"])
@pytest.mark.parametrize("lead,size", [(1, (2, 3, 20)), (1, (2, 300, 20)), (1, (1, 9001, 12)), (4, (1, 5000, 64)), (4, (1, 9001, 256)), (2, (1, 6000, 18)),
                                       (4, (160, 2000, 64)), (4, (75, 3000, 64))], ids=str)
def test_an_infinite_state_stays_infinite(ctx, lead, size, layout):
    """GATED: all gates are positive, so a state that has become infinite stays so through any number of them, also where
    their product is far below float32's range; likewise an infinite gradient on its way back."""
    n, seq_len, _ = size
    c = Case(ctx, *size, layout=layout, lead=lead)
    clean = c.forward()[0].numpy()[c.index(c.sh, lead)]
    t, s = seq_len // 3, n - 1
    c.x[s, t, 3], c.x[s, t, 4], c.h0[s, 5] = np.inf, -np.inf, np.inf
    h, last = c.forward()
    h, last = h.numpy()[c.index(c.sh, lead)], last.numpy()
    assert (h[s, t:, 3] == np.inf).all() and (h[s, t:, 4] == -np.inf).all() and (h[s, :, 5] == np.inf).all()
    assert last[s, 3] == np.inf and last[s, 4] == -np.inf and last[s, 5] == np.inf
    assert np.array_equal(h[s, :t, 3:5], clean[s, :t, 3:5])
    rest = np.ones(size, bool)
    rest[s, :, 3:6] = False
    assert np.array_equal(h[rest], clean[rest])
    c.x[s, t, 3:5], c.h0[s, 5] = 0, 0
    given = forward64(c.f, c.x, c.h0, c.lens, "gated")[0].astype(f32) if seq_len < 4000 else clean
    clean, clean0 = (v.numpy() for v in c.backward(given))
    clean = [clean[c.index(c.si, lead + o)] for o in (0, c.apart)]
    c.dy[s, t, 3], c.dy[s, t, 4], c.dh_last[s, 5] = np.inf, -np.inf, np.inf
    out, dh0 = (v.numpy() for v in c.backward(given))
    df, dx = out[c.index(c.si, lead)], out[c.index(c.si, lead + c.apart)]
    assert (dx[s, :t + 1, 3] == np.inf).all() and (dx[s, :t + 1, 4] == -np.inf).all() and (dx[s, :, 5] == np.inf).all()
    assert np.array_equal(dh0[s, 3:6], np.array([np.inf, -np.inf, np.inf], f32))
    assert np.isinf(df[s, :t + 1, 3:5]).all() and np.isinf(df[s, :, 5]).all()
    for got, want in ((df, clean[0]), (dx, clean[1])):
        assert np.array_equal(got[s, t + 1:, 3:5], want[s, t + 1:, 3:5]) and np.array_equal(got[rest], want[rest])
    rest0 = rest[:, 0]
    assert np.array_equal(dh0[rest0], clean0[rest0])


@pytest.mark.gpu
def test_misaligned_addresses_are_refused(ctx):
    """An address that is no multiple of four bytes would fault in the kernels; each buffer of both calls, one after the other."""
    import ctypes
    b = ctx.zeros(4096)
    at = lambda o: ctypes.c_void_p(b.ptr + 4 * o)  # noqa: E731
    off = lambda v, k: ctypes.c_void_p(v.value + k)  # noqa: E731
    fwd = [0, 2, 3, 8, at(0), at(100), 24, 8, at(200), at(300), at(400), 24, 8, at(500)]
    bwd = [0, 2, 3, 8, at(0), at(100), 24, 8, at(200), at(300), at(400), at(500), 24, 8, at(600), at(700), at(800), at(900), 0]
    for name, args in (("fml_gated_recurrence_fwd", fwd), ("fml_gated_recurrence_bwd", bwd)):
        call = lambda a: getattr(ctx.lib, name)(ctx.h, *a)  # noqa: E731
        assert call(args) == 0
        for i, v in enumerate(args):
            if isinstance(v, ctypes.c_void_p):
                for k in (1, 2):
                    assert call(args[:i] + [off(v, k)] + args[i + 1:]) != 0, (name, i)
                    assert b"misaligned" in ctx.lib.fml_last_error(ctx.h)
    ctx.sync()


@pytest.mark.gpu
@pytest.mark.parametrize("backward", [0, 1])
def test_a_cluster_that_waits_in_vain_gives_up(backward):
    """One CTA of a cluster keeps its pairs (the failure is made by what is not sent, not by a fault): the others give up
    after the limit, the host reads FML_ERR_TIMEOUT with code 130 once, and the context then runs clusters correctly."""
    import ctypes
    import time
    from flutter_ml_b200 import _lib
    ctx = _lib.Context()
    ctx.check(ctx.lib.fml_selftest_cluster_wait(ctx.h, backward, 2000))
    start, code = time.time(), ctypes.c_int32(0)
    assert ctx.lib.fml_device_status(ctx.h, ctypes.byref(code)) == -4
    assert code.value == 130 and b"bounded wait expired" in ctx.lib.fml_last_error(ctx.h)
    assert time.time() - start < 1.0      # limits of 2 ms, not of every round or of the usual wait
    assert ctx.device_status() == 0
    c = Case(ctx, 1, 9001, 8)
    ref, bound, last, blast = forward64(c.f, c.x, c.h0, c.lens, "gated")
    h, end = c.forward()
    close(h.numpy()[c.index(c.sh, 1)], ref, bound, "h")
    close(end.numpy(), last, blast, "h_last")
    assert ctx.device_status() == 0
    for bad in (0, -1, 1000001):
        assert ctx.lib.fml_selftest_cluster_wait(ctx.h, backward, bad) != 0
    ctx.close()


@pytest.mark.gpu
def test_ragged_sequences_may_come_first(ctx):
    """`forward` with lengths is the only way to hand over ragged sequences, so it may be the layer's first call."""
    from flutter_ml_b200 import layers, synth
    from flutter_ml_b200 import tensor as T
    x, lens = T.Tensor(synth.normal(1, 0, (20, 6)), ctx), ctx.upload(np.array([10, 4], np.int32))
    first, built = (layers.GatedRecurrentLayer(8, seq_len=10, seed=2) for _ in range(2))
    built.build(x)
    y = first.forward(x, lens=lens).numpy()
    assert np.array_equal(y, built.forward(x, lens=lens).numpy()) and not y[14:].any() and y[:14].any()
    assert [p.shape for p in first.parameters] == [(6, 16), (16,)]
