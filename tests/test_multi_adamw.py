"""AdamW over a list of tensors (fml_adamw_plan_*, ops.AdamWPlan, optimizers.MultiTensorAdamW).

The 8-bit states are checked bit for bit against a restatement in numpy float32 (every operation of the moments is one
rounded float32 operation, scales are powers of two), the 32-bit ones and the parameters against float64 with bounds from
counting roundings, u = 2^-24 each:
  m   two products with rounded constants, the scaled gradient, the sum:  5 u (|b1 m| + |(1 - b1) g|)
  v   the same, all terms positive, one more for the square:              8 u v
  w   the step is a product and a two-ulp division (4 u) of terms off by at most 7 u each, plus the constants; two
      subtractions and the decay round w:                                24 u |step| + 4 u |w|
"""
import numpy as np
import pytest

U = 2.0 ** -24
f32 = np.float32


# ------------------------------------------------------------------------------------------------- restatement
def mix(x):
    x = np.asarray(x, dtype=np.uint64) & 0xFFFFFFFF
    x ^= x >> np.uint64(16)
    x = (x * np.uint64(0x9E3779B1)) & np.uint64(0xFFFFFFFF)
    x ^= x >> np.uint64(15)
    x = (x * np.uint64(0x85EBCA77)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(13))


def words(n_blocks, seed, t):
    key = mix(mix(mix(seed & 0xFFFFFFFF) ^ np.uint64(seed >> 32)) ^ np.uint64(t))
    block = mix(key + np.arange(n_blocks, dtype=np.uint64) * np.uint64(0x9E3779B1))
    return mix(block[:, None] + np.arange(256, dtype=np.uint64)[None]).astype(np.uint32)


def to_values(codes, scale):
    """float32 values of [blocks, 256] codes with one scale a block."""
    c = codes.astype(np.int64) & 127
    e, frac = c >> 3, c & 7
    v = np.where(e > 0, (8 + frac) * 2.0 ** (e - 10.0), frac * 2.0 ** -9.0)
    v = np.where(c == 127, np.nan, v) * np.where(codes & 128, -1.0, 1.0)
    return (v * scale[:, None].astype(np.float64)).astype(f32)


def to_codes(x, rnd, root):
    """[blocks, 256] float32 -> codes, scales; rnd = None rounds to the nearest (ties to even), else 16-bit integers."""
    fin = np.isfinite(x)
    size = np.where(fin, np.abs(x), f32(0)).astype(f32)
    amax = size.max(1).astype(np.float64)
    e = np.full(len(x), -126.0)
    nz = amax > 0
    e[nz] = np.maximum(np.ceil(np.log2(amax[nz] / 448.0)), -126)
    for i in np.nonzero(nz)[0]:   # log2 may be off by one at the border
        while e[i] > -126 and amax[i] <= 448 * 2.0 ** (e[i] - 1):
            e[i] -= 1
        while amax[i] > 448 * 2.0 ** e[i]:
            e[i] += 1
    y = size.astype(np.float64) / 2.0 ** e[:, None]
    if True:   # the float32 value that a subnormal place is rounded from
        small = y < 2.0 ** -6
        y = np.where(small, (y.astype(f32) + f32(2.0 ** -6)).astype(np.float64), y)
    step = 2.0 ** (np.floor(np.log2(y)) - 3)
    k = y / step                                    # 8 <= k < 16, exact
    if rnd is None:
        q = np.round(k)                             # ties to even
    else:
        q = np.floor(k + rnd / 65536.0)
    val = q * step - np.where(small, 2.0 ** -6, 0.0)
    code = np.where(val < 2.0 ** -6, val * 512, 0)
    big = val >= 2.0 ** -6
    ex = np.floor(np.log2(np.where(big, val, 1.0)))
    code = np.where(big, (ex + 7) * 8 + (val / 2.0 ** ex - 1) * 8, code).astype(np.int64)
    if root:
        code = np.where((code == 0) & (x > 0), 1, code)
    code = np.where(fin, code, 127)
    if not root:
        code = code + 128 * np.signbit(x)
    return code.astype(np.uint8), (2.0 ** e).astype(f32)


def moments32(m, v, g, b1, b2, gs=1.0):
    g = (g * f32(gs)).astype(f32)
    m = (m * f32(b1)).astype(f32) + (g * f32(1 - b1)).astype(f32)
    v = (v * f32(b2)).astype(f32) + ((g * g).astype(f32) * f32(1 - b2)).astype(f32)
    return m.astype(f32), v.astype(f32)


def step64(w, m, v, g, lr, b1, b2, eps, wd, t, gs=1.0):
    """float64 AdamW; returns w, m, v and the bounds of their float32 forms."""
    w, m, v, g = (np.asarray(a, np.float64) for a in (w, m, v, g * gs))
    size = np.abs(b1 * m) + np.abs((1 - b1) * g)
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    den = np.sqrt(v / (1 - b2 ** t)) + eps
    step = lr / (1 - b1 ** t) * size / den
    w = w - lr * (m / (1 - b1 ** t)) / den
    w = w - lr * wd * w
    return w, m, v, 24 * U * step + 4 * U * np.abs(w), 5 * U * size, 8 * U * v


def blocks_of(sizes):
    return [-(-n // 256) for n in sizes]


# ------------------------------------------------------------------------------------------------------ CPU tests
def test_state_floats():
    from flutter_ml_b200.ops import AdamWPlan
    from flutter_ml_b200._lib import FmlError
    assert AdamWPlan.state_floats([1], 32) == 256 and AdamWPlan.state_floats([1], 8) == 65
    assert AdamWPlan.state_floats([256, 257, 0, 1000], 32) == 256 * (1 + 2 + 0 + 4)
    assert AdamWPlan.state_floats([256, 257, 0, 1000], 8) == 65 * 7
    for sizes, bits in (([], 32), ([-1], 32), ([4], 16), ([2 ** 40], 8)):
        with pytest.raises(FmlError):
            AdamWPlan.state_floats(sizes, bits)


def test_random_words_are_uniform_and_differ():
    """Both halves of the words that decide the rounding: means within 5 standard errors of one half, bits independent of
    the neighbour, block, step and seed (correlation within 5 / sqrt(n))."""
    w = words(64, 12345, 7)
    n = w.size
    for part in (w >> 16, w & 0xFFFF):
        x = part.reshape(-1) / 65536.0
        assert abs(x.mean() - 0.5) <= 5 * np.sqrt(1 / 12 / n)
        assert abs(np.corrcoef(x[:-1], x[1:])[0, 1]) <= 5 / np.sqrt(n)
        assert abs(np.corrcoef(x[:-256], x[256:])[0, 1]) <= 5 / np.sqrt(n)
    for other in (words(64, 12345, 8), words(64, 12346, 7), words(64, 12345 + (1 << 32), 7)):
        assert abs(np.corrcoef(w.reshape(-1).astype(float), other.reshape(-1).astype(float))[0, 1]) <= 5 / np.sqrt(n)
    assert abs(np.corrcoef((w >> 16).reshape(-1).astype(float), (w & 0xFFFF).reshape(-1).astype(float))[0, 1]) <= 5 / np.sqrt(n)


def test_restated_format_is_float8_and_within_half_a_step():
    """The restatement against torch's own 8-bit type: the codes' values, nearest rounding within half a step (2^-4 of the
    value, 2^-10 of the scale where subnormal), random rounding to one of the two neighbours and right on average."""
    import torch
    codes = np.arange(256, dtype=np.uint8).reshape(1, 256)
    ref = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(to_values(codes, np.ones(1, f32))[0], ref, equal_nan=True)
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 256)) * np.exp(3 * rng.standard_normal((50, 256)))).astype(f32)
    x[3] = 0
    x[4, 1:] = 0
    c, s = to_codes(x, None, False)
    err = np.abs(to_values(c, s).astype(np.float64) - x)
    assert (err <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s[:, None]) * (1 + 1e-6)).all()
    assert (np.abs(x).max(1) <= 448 * s).all()
    total, reps = np.zeros_like(x, dtype=np.float64), 400
    for k in range(reps):
        c, s = to_codes(x, (words(50, 1, k) >> 16), False)
        y = to_values(c, s).astype(np.float64)
        step = np.maximum(2.0 ** np.floor(np.log2(np.maximum(np.abs(x), 1e-30))) / 8, 2.0 ** -9 * s[:, None])
        assert (np.abs(y - x) <= step * (1 + 1e-6)).all()
        total += (y - x) / step
    # each error has a standard deviation of at most half a step; over all elements the mean of the means has far less
    assert abs(total.mean() / reps) <= 5 * 0.5 / np.sqrt(reps * x.size)
    assert np.abs(total / reps).max() <= 6 * 0.5 / np.sqrt(reps)


# ------------------------------------------------------------------------------------------------------ GPU tests
@pytest.fixture(scope="module")
def ctx():
    from flutter_ml_b200 import _lib
    c = _lib.Context()
    yield c
    assert c.device_status() == 0
    c.close()


HYPER = dict(lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.01)


class Setup:
    """Tensors of the given sizes at the given offset (floats) inside one buffer each, with guard values around them."""

    def __init__(self, ctx, sizes, bits, seed=0, shift=0, scale=1.0):
        from flutter_ml_b200.ops import AdamWPlan
        rng = np.random.default_rng(seed)
        self.ctx, self.sizes, self.bits = ctx, sizes, bits
        gap = 3
        self.off, o = [], 4 + shift
        for n in sizes:
            self.off.append(o)
            o += n + gap if shift else (n + gap + 3) // 4 * 4
        self.total = o + 8
        self.w = rng.standard_normal(self.total).astype(f32) * f32(0.02)
        self.g = (rng.standard_normal(self.total) * np.exp(2 * rng.standard_normal(self.total)) * scale).astype(f32)
        self.dw, self.dg = ctx.upload(self.w), ctx.upload(self.g)
        floats = AdamWPlan.state_floats(sizes, bits)
        self.m, self.v = ctx.zeros(floats), ctx.zeros(floats)
        self.plan = AdamWPlan(ctx, [self.dw.view(o, (n,)) for o, n in zip(self.off, sizes)],
                              [self.dg.view(o, (n,)) for o, n in zip(self.off, sizes)], self.m, self.v, bits)

    def tensors(self, flat):
        return [flat[o:o + n].copy() for o, n in zip(self.off, self.sizes)]

    def states(self, buf):
        """Per tensor [blocks, 256] float32 values (32 bits), or (codes, scales)."""
        nb, out, b = blocks_of(self.sizes), [], 0
        flat, total = buf.numpy(), sum(nb)
        for k in nb:
            if self.bits == 32:
                out.append(flat.reshape(-1, 256)[b:b + k])
            else:
                out.append((flat[:total * 64].view(np.uint8).reshape(total, 256)[b:b + k], flat[total * 64:][b:b + k]))
            b += k
        return out

    def step(self, t, **kw):
        h = HYPER
        self.plan.step(h["lr"], h["b1"], h["b2"], h["eps"], h["wd"], t, **kw)


def padded(x):
    return np.concatenate([x, np.zeros(-len(x) % 256, f32)]).reshape(-1, 256)


SIZES = [[1], [255, 256, 257], [0, 5, 0, 2048, 2049], [4096 * 3 + 1, 7, 100000], [2047, 2303, 1, 1, 1]]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("shift", [0, 1, 2])
def test_states_in_32_bits(ctx, sizes, shift):
    s = Setup(ctx, sizes, 32, seed=len(sizes) + shift, shift=shift)
    w, g = s.tensors(s.w), s.tensors(s.g)
    m = [np.zeros(n) for n in sizes]
    v = [np.zeros(n) for n in sizes]
    for t in (1, 2, 3):
        s.step(t, grad_scale=0.5)
        now, ms, vs = s.dw.numpy(), s.states(s.m), s.states(s.v)
        for i, n in enumerate(sizes):
            rw, rm, rv, bw, bm, bv = step64(w[i], m[i], v[i], g[i], HYPER["lr"], 0.9, 0.999, 1e-8, 0.01, t, 0.5)
            w[i], m[i], v[i] = s.tensors(now)[i], ms[i].reshape(-1)[:n], vs[i].reshape(-1)[:n]   # the next step from the same place
            assert (np.abs(w[i] - rw) <= bw).all() and (np.abs(m[i] - rm) <= bm).all() and (np.abs(v[i] - rv) <= bv).all()
            assert not ms[i].reshape(-1)[n:].any() and not vs[i].reshape(-1)[n:].any()
    inside = np.zeros(s.total, bool)
    for o, n in zip(s.off, sizes):
        inside[o:o + n] = True
    assert np.array_equal(now[~inside], s.w[~inside]) and np.array_equal(s.dg.numpy(), s.g)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("seed", [-1, 0, 99 + (5 << 32)])
@pytest.mark.parametrize("shift", [0, 1])
def test_states_in_8_bits_bit_for_bit(ctx, sizes, seed, shift):
    s = Setup(ctx, sizes, 8, seed=3 + len(sizes), shift=shift)
    w, g = s.tensors(s.w), s.tensors(s.g)
    m = [np.zeros((b, 256), f32) for b in blocks_of(sizes)]
    r = [np.zeros((b, 256), f32) for b in blocks_of(sizes)]
    for t in (1, 2, 3, 4):
        s.step(t, seed=seed)
        now, ms, rs = s.dw.numpy(), s.states(s.m), s.states(s.v)
        rnd = words(sum(blocks_of(sizes)), seed, t) if seed >= 0 else None
        b = 0
        for i, n in enumerate(sizes):
            k = blocks_of(sizes)[i]
            gi, v0 = padded(g[i]), (r[i] * r[i]).astype(f32)
            rw, _, _, bw, _, _ = step64(w[i], m[i].reshape(-1)[:n], v0.reshape(-1)[:n], g[i], HYPER["lr"], 0.9, 0.999, 1e-8, 0.01, t)
            assert (np.abs(s.tensors(now)[i] - rw) <= bw).all()
            w[i] = s.tensors(now)[i]
            m1, v1 = moments32(m[i], v0, gi, 0.9, 0.999)
            for got, x, half, root in ((ms[i], m1, 16, False), (rs[i], np.sqrt(v1), 0, True)):
                if n:
                    code, scale = to_codes(x, None if rnd is None else (rnd[b:b + k] >> half) & 0xFFFF, root)
                    assert np.array_equal(got[0], code) and np.array_equal(got[1], scale)
            m[i] = to_values(*ms[i]) if n else m[i]
            r[i] = to_values(*rs[i]) if n else r[i]
            b += k


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_zero_grad_clears_only_the_tensors(ctx, bits):
    a, b = Setup(ctx, [300, 2048, 5], bits, seed=1, shift=1), Setup(ctx, [300, 2048, 5], bits, seed=1, shift=1)
    a.step(1, zero_grad=True)
    b.step(1)
    assert np.array_equal(a.dw.numpy(), b.dw.numpy()) and np.array_equal(a.m.numpy().view(np.int32), b.m.numpy().view(np.int32))
    left, inside = a.dg.numpy(), np.zeros(a.total, bool)
    for o, n in zip(a.off, a.sizes):
        inside[o:o + n] = True
    assert not left[inside].any() and np.array_equal(left[~inside], a.g[~inside])


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_places(ctx):
    """A NaN or infinite gradient makes its own element NaN and nothing else; extreme blocks keep their scale in range."""
    s = Setup(ctx, [1024], 8, seed=2)
    g = s.tensors(s.g)[0]
    g[5], g[300] = np.nan, np.inf
    g[512:768] = 0                      # a block of zeros
    g[768:] = 1e-38                     # a block whose roots are near the smallest numbers
    g[800] = 3e38                       # and its square overflows
    s.dg.ctx.upload(g, out=s.dg.view(s.off[0], (1024,)))
    s.step(1, seed=4)
    w = s.tensors(s.dw.numpy())[0]
    bad = np.zeros(1024, bool)
    bad[[5, 300]] = True
    assert np.isnan(w[bad]).all() and np.isfinite(w[~bad]).all()
    (mc, ms), (rc, rs) = s.states(s.m)[0], s.states(s.v)[0]
    m, r = to_values(mc, ms).reshape(-1), to_values(rc, rs).reshape(-1)
    assert np.isnan(m[bad]).all() and np.isfinite(m[~bad]).all()
    assert np.isnan(r[[5, 300, 800]]).all() and np.isfinite(np.delete(r, [5, 300, 800])).all()
    assert not m[512:768].any() and not r[512:768].any()
    s.step(2, seed=4)                   # the states can be read again
    w = s.tensors(s.dw.numpy())[0]
    assert np.isnan(w[bad]).all() and np.isfinite(np.delete(w, [5, 300, 800])).all()


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [-1, 7])
def test_blocks_of_extreme_size_bit_for_bit(ctx, seed):
    """Blocks around 1e15 (scales above 2^29), 1e-15 and 1e-30 (subnormal products), values of 40 orders of magnitude in one."""
    s = Setup(ctx, [2048], 8, seed=9)
    rng = np.random.default_rng(9)
    g = rng.standard_normal(2048).astype(f32)
    for i, size in enumerate((1e15, 1e17, 1e-15, 1e-18, 1e-30, 1.0, 1e9)):
        g[256 * i:256 * (i + 1)] *= f32(size)
    g[1792:] *= np.exp(rng.uniform(-46, 40, 256)).astype(f32)
    ctx.upload(g, out=s.dg.view(s.off[0], (2048,)))
    m, r = np.zeros((8, 256), f32), np.zeros((8, 256), f32)
    for t in (1, 2, 3):
        s.step(t, seed=seed)
        (mc, ms), (rc, rs) = s.states(s.m)[0], s.states(s.v)[0]
        with np.errstate(over="ignore"):
            m1, v1 = moments32(m, (r * r).astype(f32), padded(g), 0.9, 0.999)
        rnd = words(8, seed, t) if seed >= 0 else None
        for got, sc, x, half, root in ((mc, ms, m1, 16, False), (rc, rs, np.sqrt(v1), 0, True)):
            code, scale = to_codes(x, None if rnd is None else (rnd >> half) & 0xFFFF, root)
            assert np.array_equal(got, code) and np.array_equal(sc, scale)
        m, r = to_values(mc, ms), to_values(rc, rs)


@pytest.mark.gpu
def test_small_roots_are_never_rounded_to_zero(ctx):
    """One gradient a million times its neighbours': the neighbours' m and root fall below the block's range, and the root
    stays at 2^-9 of the scale, so a later step with no gradient is bounded by |m| over that."""
    s = Setup(ctx, [256], 8, seed=5)
    g = np.full(256, 1e-4, f32)
    g[0] = 1e4
    s.dg.ctx.upload(g, out=s.dg.view(s.off[0], (256,)))
    s.step(1)
    rc, rs = s.states(s.v)[0]
    assert (rc.reshape(-1)[1:] == 1).all() and rs[0] > 0
    before = s.tensors(s.dw.numpy())[0]
    ctx.zero(s.dg)
    s.step(2)
    after = s.tensors(s.dw.numpy())[0]
    m = np.abs(to_values(*s.states(s.m)[0]).reshape(-1)[1:]).max()
    floor = rs[0] * 2.0 ** -9 * np.sqrt(0.999) / np.sqrt(1 - 0.999 ** 2)
    bound = 1e-3 / (1 - 0.9 ** 2) * max(m, 1e-4) / floor + 1e-5 * np.abs(before[1:]) * 1.01 + 1e-8
    assert (np.abs(after[1:] - before[1:]) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_recorded_step_counts_on_the_device(ctx, bits):
    """t = 0 three times through one recording gives what t = 1, 2, 3 give."""
    a, b = Setup(ctx, [700, 3000], bits, seed=6), Setup(ctx, [700, 3000], bits, seed=6)
    ctx.sync()
    ctx.graph_begin()
    a.step(0, seed=11)
    gid = ctx.graph_end()
    for t in (1, 2, 3):
        ctx.graph_launch(gid)
        b.step(t, seed=11)
    ctx.sync()
    assert np.allclose(a.dw.numpy(), b.dw.numpy(), rtol=4 * U, atol=1e-3 * 8 * U)   # pow on the device may be an ulp off the host's
    assert np.array_equal(a.m.numpy().view(np.int32), b.m.numpy().view(np.int32))
    assert np.array_equal(a.v.numpy().view(np.int32), b.v.numpy().view(np.int32))
    ctx.check(ctx.lib.fml_graph_destroy(ctx.h, gid))


@pytest.mark.gpu
def test_step_on_a_lane_and_two_plans_at_once(ctx):
    a, b, ref = Setup(ctx, [5000], 8, seed=7), Setup(ctx, [5000], 32, seed=7), Setup(ctx, [5000], 8, seed=7)
    ref32 = Setup(ctx, [5000], 32, seed=7)
    ctx.sync()
    for t in (1, 2):
        a.step(t, lane=0, seed=3)
        b.step(t, lane=1)
        ref.step(t, seed=3)
        ref32.step(t)
    for lane in (0, 1):
        ctx.check(ctx.lib.fml_lane_sync(ctx.h, lane))
    ctx.sync()
    assert np.array_equal(a.dw.numpy(), ref.dw.numpy()) and np.array_equal(b.dw.numpy(), ref32.dw.numpy())


@pytest.mark.gpu
def test_refusals(ctx):
    from flutter_ml_b200 import _lib
    from flutter_ml_b200.ops import AdamWPlan
    n = AdamWPlan.state_floats([512, 512], 32)
    buf, m, v = ctx.zeros(4096), ctx.zeros(n), ctx.zeros(n)
    at = lambda o, k=512: buf.view(o, (k,))  # noqa: E731
    ok = ([at(0), at(512)], [at(1024), at(1536)])
    for w, g, mm, vv, bits in (([at(0), at(256)], ok[1], m, v, 32),          # tensors overlap
                               (ok[0], [at(0), at(1536)], m, v, 32),          # a gradient is a tensor
                               (ok[0], ok[1], m, m, 32),                      # one buffer for both states
                               (ok[0], ok[1], buf.view(2047, (n,)), v, 32),   # a state buffer that is not aligned
                               (ok[0], ok[1], m, v, 16)):
        with pytest.raises(_lib.FmlError):
            AdamWPlan(ctx, w, g, mm, vv, bits)
    with pytest.raises(ValueError):
        AdamWPlan(ctx, ok[0], [at(1024)], m, v)
    with pytest.raises(ValueError):
        AdamWPlan(ctx, ok[0], ok[1], ctx.zeros(10), v)
    host = np.zeros(512, f32)
    fake = _lib.DeviceArray(ctx, host.ctypes.data, (512,), owner=False)
    with pytest.raises(_lib.FmlError, match="memory of the context"):
        AdamWPlan(ctx, [at(0), fake], ok[1], m, v)
    plan = AdamWPlan(ctx, *ok, m, v)
    good = dict(lr=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, weightDecay=0.0, t=1)
    for bad in (dict(beta1=1.0), dict(beta2=-0.1), dict(epsilon=0.0), dict(lr=float("nan")), dict(t=-1), dict(weightDecay=float("inf")), dict(lane=9)):
        with pytest.raises(_lib.FmlError):
            plan.step(**{**good, **bad})
    plan.step(**good)
    gone = plan.id
    plan.close()
    with pytest.raises(_lib.FmlError, match="unknown plan"):
        ctx.check(ctx.lib.fml_adamw_plan_destroy(ctx.h, gone))
    plan.id = gone
    with pytest.raises(_lib.FmlError, match="unknown plan"):
        plan.step(**good)
    plan.id = -1
    assert AdamWPlan(ctx, [at(0, 0)], [at(0, 0)], ctx.zeros(4), ctx.zeros(4)).step(**good) is None   # nothing to do


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_class_beside_adamw(ctx, bits):
    """MultiTensorAdamW on a dense layer's parameters against AdamW on the same: equal within the rounding of one step (32
    bits; the two order their operations differently), near it with 8-bit states; a moved gradient is noticed."""
    from flutter_ml_b200 import optimizers as O
    from flutter_ml_b200.tensor import Tensor
    rng = np.random.default_rng(8)
    shapes = [(33, 17), (17,), (300, 70), (1,)]
    init = [rng.standard_normal(s).astype(f32) for s in shapes]
    grads = [rng.standard_normal(s).astype(f32) for s in shapes]
    a = [Tensor(x, ctx) for x in init]
    b = [Tensor(x, ctx) for x in init]
    oa, ob = O.AdamW(a, 0.01), O.MultiTensorAdamW(b, 0.01, stateBits=bits)
    for t in range(3):
        for i, (p, q) in enumerate(zip(a, b)):
            p.grad = ctx.upload(grads[i])
            if t == 1:
                q.grad = ctx.upload(grads[i])    # another buffer
            else:
                ctx.upload(grads[i], out=q.grad)
        oa.step()
        ob.step()
    for p, q, x, gr in zip(a, b, init, grads):
        d, moved = np.abs(p.numpy() - q.numpy()), np.abs(q.numpy() - x)
        if bits == 32:
            # three steps of lr * 1: each off by at most 24 + 24 roundings of the step and a few of w
            assert (d <= 3 * (48 * U * 0.0101 + 8 * U * np.abs(x) + 1e-9)).all()
        else:
            # constant gradients: m and the root are off by at most an eighth (one step of the format) after each of two
            # roundings, and so the last two of the three steps by at most (1 + 1/8)^2 / (1 - 1/8)^2 - 1 < 2/3 of lr each;
            # an eighth holds down to 2^-6 of the scale, and a scale is at most 2 / 448 of the block's largest
            full = np.abs(gr) >= 2.0 ** -5 / 448 * np.abs(gr).max()
            assert (d[full] <= 2 * 0.67 * 0.0101 + 1e-6).all() and moved[full].min() > 0
    for q in b:
        q.grad = None
    with pytest.raises(ValueError, match="no gradient"):
        ob.step()
    with pytest.raises(ValueError):
        O.MultiTensorAdamW([], 0.01)
    with pytest.raises(ValueError):
        O.MultiTensorAdamW(a, 0.01, seed=-3)


@pytest.mark.gpu
def test_roots_at_the_borders_of_the_codes(ctx):
    """Nearest rounding where one unit in the last place of the root changes its code: beta1 = beta2 = 0 make v the rounded
    square of the gradient, and the gradients are the midpoints between neighbouring codes (and up to six units beside them),
    a block for each power of two from 2^-55 to 2^55 whose largest element, 448 of it, fixes the scale."""
    mids = np.array([m * 2.0 ** e for e in range(-2, 8) for m in (1.0625, 1.1875, 1.3125, 1.4375, 1.5625, 1.6875)], f32)
    blocks = np.concatenate([mids * f32(1 + k * 2.0 ** -23) for k in (0, 1, -1, 6)] + [np.full(16, 448, f32)])   # 256 elements
    assert blocks.size == 256
    exps = range(-55, 56)
    s = Setup(ctx, [256 * len(exps)], 8, seed=1)
    g = np.concatenate([blocks * f32(2.0 ** e) for e in exps]).astype(f32)
    ctx.upload(g, out=s.dg.view(s.off[0], (g.size,)))
    s.plan.step(1e-3, 0.0, 0.0, 1e-8, 0.0, 1, seed=-1)
    code, scale = to_codes(np.sqrt((g * g).astype(f32)).reshape(-1, 256), None, True)
    rc, rs = s.states(s.v)[0]
    assert np.array_equal(rs, scale) and np.array_equal(rc, code)
    code, scale = to_codes(g.reshape(-1, 256), None, False)
    mc, ms = s.states(s.m)[0]
    assert np.array_equal(ms, scale) and np.array_equal(mc, code)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [-1, 4])
def test_codes_of_values_that_are_not_finite(ctx, seed):
    """NaN and both infinities among ordinary gradients, and a square that overflows: the codes are the restatement's."""
    s = Setup(ctx, [1024], 8, seed=2)
    g = s.tensors(s.g)[0]
    g[[5, 300, 301, 700, 1023]] = np.nan, np.inf, -np.inf, -np.inf, 3e38
    ctx.upload(g, out=s.dg.view(s.off[0], (1024,)))
    s.step(1, seed=seed)
    with np.errstate(over="ignore"):
        m, v = moments32(np.zeros((4, 256), f32), np.zeros((4, 256), f32), g.reshape(4, 256), 0.9, 0.999)
    m[np.isnan(m)] = np.nan             # the sign of a NaN is the processor's choice
    rnd = words(4, seed, 1) if seed >= 0 else None
    for (got, sc), x, half, root in ((s.states(s.m)[0], m, 16, False), (s.states(s.v)[0], np.sqrt(v), 0, True)):
        code, scale = to_codes(x, None if rnd is None else (rnd >> half) & 0xFFFF, root)
        assert np.array_equal(got, code) and np.array_equal(sc, scale)
    mc = s.states(s.m)[0][0].reshape(-1)
    assert list(mc[[5, 300, 301, 700]]) == [0x7f, 0x7f, 0xff, 0xff]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("device", [True, False])
def test_training_goes_on_from_a_checkpoint(ctx, tmp_path, bits, device):
    """Three steps, a checkpoint, two more; an optimizer that loads the checkpoint takes the same two, bit for bit.  With the
    count on the device the steps are replays of a recording, which the host does not count."""
    from flutter_ml_b200 import checkpoint, optimizers as O
    from flutter_ml_b200.tensor import Tensor
    rng = np.random.default_rng(3)
    shapes, path = [(40, 50), (7,)], str(tmp_path / "state")
    init, grads = ([rng.standard_normal(s).astype(f32) for s in shapes] for _ in range(2))

    def start(values):
        ps = [Tensor(x, ctx) for x in values]
        for p, g in zip(ps, grads):
            p.grad = ctx.upload(g)
        return ps, O.MultiTensorAdamW(ps, 0.01, stateBits=bits, seed=5, deviceCounter=device)

    def run(opt, steps):
        if not device:
            for _ in range(steps):
                opt.step()
            return
        ctx.sync()
        ctx.graph_begin()
        opt.step()
        gid = ctx.graph_end()
        for _ in range(steps):
            ctx.graph_launch(gid)
        ctx.sync()
        ctx.check(ctx.lib.fml_graph_destroy(ctx.h, gid))
    a, oa = start(init)
    run(oa, 3)
    assert oa._t == 3
    checkpoint.save_training_state(ctx, path, oa)
    b, ob = start([np.zeros(s, f32) for s in shapes])
    checkpoint.load_training_state(ctx, path, ob)
    assert ob._t == 3
    for o in (oa, ob):
        run(o, 2)
        assert o._t == 5
    for p, q in zip([x.value for x in a] + [oa._m, oa._v], [x.value for x in b] + [ob._m, ob._v]):
        assert np.array_equal(p.numpy().view(np.int32), q.numpy().view(np.int32))
    with pytest.raises(Exception, match="negative"):
        oa._plan.count = -1
    oa._plan.close()
    with pytest.raises(Exception, match="unknown plan"):
        oa._plan.count


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_a_recording_outlives_its_plan(ctx, bits):
    """The plan is destroyed, others take the place of what it could have freed, and the recording is replayed: it updates
    what the plan updated, as steps with t = 1, 2, 3 do."""
    a, b = Setup(ctx, [700, 3000], bits, seed=6), Setup(ctx, [700, 3000], bits, seed=6)
    ctx.sync()
    ctx.graph_begin()
    a.step(0, seed=11)
    gid = ctx.graph_end()
    a.plan.close()
    with pytest.raises(Exception, match="unknown plan"):
        a.plan.count
    others = [Setup(ctx, [700, 3000], bits, seed=i) for i in range(4)]
    for t in (1, 2, 3):
        ctx.graph_launch(gid)
        b.step(t, seed=11)
        for o in others:
            o.step(t)
    ctx.sync()
    assert np.array_equal(a.m.numpy().view(np.int32), b.m.numpy().view(np.int32))
    assert np.array_equal(a.v.numpy().view(np.int32), b.v.numpy().view(np.int32))
    ctx.check(ctx.lib.fml_graph_destroy(ctx.h, gid))


@pytest.mark.gpu
def test_a_recorded_step_outlives_a_moved_gradient(ctx):
    """MultiTensorAdamW makes its plan anew where a gradient has moved; a recording of the step before goes on with the old
    addresses."""
    from flutter_ml_b200 import optimizers as O
    from flutter_ml_b200.tensor import Tensor
    p = Tensor(np.ones(3000, f32), ctx)
    p.grad = first = ctx.upload(np.full(3000, 0.5, f32))
    opt = O.MultiTensorAdamW([p], 0.01)
    ctx.sync()
    ctx.graph_begin()
    opt.step()
    gid = ctx.graph_end()
    old = opt._plan
    p.grad = ctx.upload(np.full(3000, 0.5, f32))
    opt.step()
    assert opt._plan is not old and old.id == -1
    once = p.numpy()
    ctx.zero(p.grad)                    # the recording reads the gradient that it was made with
    ctx.graph_launch(gid)
    ctx.sync()
    assert (p.numpy() < once).all() and first.size == 3000
    ctx.check(ctx.lib.fml_graph_destroy(ctx.h, gid))


@pytest.mark.gpu
def test_a_plain_call_with_8_bit_states_is_adamw(ctx):
    """1500 steps of normal gradients through `step` as it comes: the roots of the second moments stay with those of 32-bit
    states.  They are right on average but for the variance of the rounding: the root moves by about 1/2000 a step, so codes
    a step of d <= 1/8 apart are changed with probability 1 / (2000 d) and add d / 2000 <= 6.3e-5 to v's relative mean, which
    decays by 1/1000 a step: v at most 6.3 % high, its root 3.2 %; 6144 elements leave a standard error below 1 %."""
    n, ring = 6144, 32
    a, b = Setup(ctx, [n], 8, seed=1), Setup(ctx, [n], 32, seed=1)
    rng = np.random.default_rng(1)
    grads = [ctx.upload(rng.standard_normal(n).astype(f32)) for _ in range(ring)]
    for t in range(1, 1501):
        now = grads[int(rng.integers(ring))]
        for s in (a, b):
            ctx.copy(s.dg.view(s.off[0], (n,)), now)
            s.step(t)
    root = to_values(*a.states(a.v)[0]).reshape(-1).astype(np.float64)
    exact = np.sqrt(b.states(b.v)[0].reshape(-1).astype(np.float64))
    assert 0.96 <= root.mean() / exact.mean() <= 1.06
    assert 0.96 <= (root / exact).mean() <= 1.06
