"""The recurrence, the query/key norm with rotation and the multi-tensor optimizer in one model, as they are used: a training
step (tape, FP32 products) against torch autograd in float64, and the same model token by token.

Gradients: 1e-5 relative, the FP32 bound of the dense products that carry them; no operator's own bound is above that.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
f32 = np.float32
N, S, D, H, V = 2, 19, 32, 2, 11     # sequences, steps, width, heads, classes


@pytest.fixture(scope="module")
def ctx():
    from flutter_ml_b200 import _lib
    c = _lib.Context(precision=_lib.PREC_FP32)
    yield c
    assert c.device_status() == 0
    c.close()


class Model:
    """Dense -> gated recurrence -> attention with normed, turned queries and keys -> residual -> class scores."""

    def __init__(self, ctx, x):
        from flutter_ml_b200 import layers, synth
        from flutter_ml_b200 import tensor as T
        self.ctx, self.T = ctx, T
        self.rec = layers.GatedRecurrentLayer(D, seq_len=S, seed=1)
        self.att = layers.MultiHeadAttention(D, H, seq_len=S, causal=True, seed=2, qkNorm=True, rotaryDim=8)
        self.head = layers.DenseLayerMatrix(V, None, seed=3)
        for layer, i in ((self.rec, x), (self.att, T.Tensor(ctx.zeros(N * S, D))), (self.head, T.Tensor(ctx.zeros(N * S, D)))):
            layer.build(i)
        for i, g in enumerate((self.att.gainQ, self.att.gainK)):
            ctx.upload(f32(1) + synth.normal(9, i, (D // H,), 0.3), out=g.value)
        self.parameters = self.rec.parameters + self.att.parameters + self.head.parameters

    def loss(self, x, target):
        T = self.T
        h = self.rec(x)
        return T.mseMatrix(self.head(T.addMatrix(h, self.att(h))), target)


def torch_loss(p, x, target):
    import torch
    w, b, wqkv, wo, gq, gk, wh, bh = p
    z = (x @ w + b).reshape(N, S, 2 * D)
    a, state, hs = torch.sigmoid(z[..., :D]), torch.zeros(N, D, dtype=torch.float64), []
    for t in range(S):
        state = a[:, t] * state + (1 - a[:, t]) * z[:, t, D:]
        hs.append(state)
    h = torch.stack(hs, 1)
    qkv = (h @ wqkv).reshape(N, S, 3, H, D // H)

    def normed(u, g):
        u = u / torch.sqrt((u * u).mean(-1, keepdim=True) + 1e-6) * g
        ang = torch.arange(S, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(4, dtype=torch.float64) / 4)
        c, s = torch.cos(ang)[None, :, None], torch.sin(ang)[None, :, None]
        u1, u2 = u[..., :4], u[..., 4:8]
        return torch.cat([u1 * c - u2 * s, u1 * s + u2 * c, u[..., 8:]], -1)
    q, k, v = normed(qkv[:, :, 0], gq), normed(qkv[:, :, 1], gk), qkv[:, :, 2]
    sc = torch.einsum("nihd,njhd->nhij", q, k) / np.sqrt(D // H)
    sc = sc.masked_fill(torch.triu(torch.ones(S, S, dtype=torch.bool), 1), -torch.inf)
    o = torch.einsum("nhij,njhd->nihd", torch.softmax(sc, -1), v).reshape(N, S, D)
    y = (h + o @ wo) @ wh + bh
    return ((y.reshape(N * S, V) - target) ** 2).mean()


def data():
    rng = np.random.default_rng(0)
    return rng.standard_normal((N * S, D)).astype(f32), rng.standard_normal((N * S, V)).astype(f32)


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(ctx, bits):
    import torch
    from flutter_ml_b200 import optimizers, tensor as T
    x0, y0 = data()
    x, target = T.Tensor(x0, ctx), T.Tensor(y0, ctx)
    m = Model(ctx, x)
    opt = optimizers.MultiTensorAdamW(m.parameters, 0.01, stateBits=bits, seed=5)
    for step in (1, 2):
        before = [p.numpy().astype(np.float64) for p in m.parameters]
        ps = [torch.tensor(b, requires_grad=True) for b in before]
        want = torch_loss(ps, torch.tensor(x0.astype(np.float64)), torch.tensor(y0.astype(np.float64)))
        want.backward()
        loss = m.loss(x, target)
        loss.backward()
        assert abs(float(loss.numpy().reshape(-1)[0]) - float(want)) <= 1e-5 * float(want)
        for p, q in zip(m.parameters, ps):
            g, r = p.grad.numpy().astype(np.float64), q.grad.numpy()
            assert np.linalg.norm(g - r) <= 1e-5 * np.linalg.norm(r), p.shape
        grads = [p.grad.numpy().astype(np.float64) for p in m.parameters]
        opt.step(zero_grad=True)
        assert not any(p.grad.numpy().any() for p in m.parameters)
        if step == 1:   # from states of zero the first step is lr * sign-like g / (|g| + eps), whatever the states' format
            for p, b, g in zip(m.parameters, before, grads):
                w = b - 0.01 * g / (np.abs(g) + 1e-8)
                w -= 0.01 * 0.01 * w
                assert np.abs(p.numpy() - w).max() <= 40 * 2.0 ** -24 * (0.01 + np.abs(w).max())


def test_token_by_token(ctx):
    """The same model one token at a time: the recurrence with its state handed on, queries and keys with explicit positions,
    the keys and values so far kept.  Products of other shapes add in another order: 1e-5 relative as above."""
    from flutter_ml_b200 import ops, tensor as T
    x0, _ = data()
    x = T.Tensor(x0, ctx)
    m = Model(ctx, x)
    h_all = m.rec(x)
    att_all = m.att(h_all).numpy().reshape(N, S, D)
    h_all = h_all.numpy().reshape(N, S, D)
    state, keys, values = ctx.zeros(N, D), [], []
    dk = D // H
    for t in range(S):
        xt = T.Tensor(x0.reshape(N, S, D)[:, t].copy(), ctx)
        z = T.denseMatrix(xt, m.rec.weights, m.rec.biases, None)
        h = ctx.empty(N, D)
        ops.gated_recurrence_forward(ctx, z.value, z.value.view(D, ()), h, N, 1, D, h0=state, h_last=state, strides_in=(2 * D, 2 * D))
        qkv = T.denseMatrix(T.Tensor(h), m.att.Wqkv, None, None)
        pos = ctx.upload(np.full(N, t, np.int32))
        qk = ctx.empty(N, 2 * D)
        ops.qk_norm_rope_forward(ctx, qkv.value, qkv.value.view(D, ()), qk, qk.view(D, ()), N, H, H, dk, gain_q=m.att.gainQ.value,
                                 gain_k=m.att.gainK.value, positions=pos, rot_dim=8, ld_q=3 * D, ld_k=3 * D, ld_q_out=2 * D, ld_k_out=2 * D)
        both = qk.numpy().astype(np.float64).reshape(N, 2, H, dk)
        keys.append(both[:, 1])
        values.append(qkv.numpy().astype(np.float64).reshape(N, 3, H, dk)[:, 2])
        sc = np.einsum("nhd,tnhd->nht", both[:, 0], np.array(keys)) / np.sqrt(dk)
        w = np.exp(sc - sc.max(-1, keepdims=True))
        o = np.einsum("nht,tnhd->nhd", w / w.sum(-1, keepdims=True), np.array(values)).reshape(N, D)
        out = o @ m.att.Wo.numpy().astype(np.float64)
        assert np.linalg.norm(h.numpy() - h_all[:, t]) <= 1e-5 * np.linalg.norm(h_all[:, t])
        assert np.linalg.norm(out - att_all[:, t]) <= 1e-5 * np.linalg.norm(att_all[:, t])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_recorded_training_step(ctx, bits):
    """Loss, backward pass and optimizer step recorded once and replayed three times, against the same three steps launched one
    by one from the same place: the same parameters, gradients and moments, bit for bit."""
    import gc
    from flutter_ml_b200 import optimizers, tensor as T
    x0, y0 = data()

    def start():
        x, target = T.Tensor(x0, ctx), T.Tensor(y0, ctx)
        m = Model(ctx, x)
        opt = optimizers.MultiTensorAdamW(m.parameters, 0.01, stateBits=bits, seed=5, deviceCounter=True)

        def step():
            m.loss(x, target).backward()
            x.grad = m.att.lastAttentionWeights = None      # nothing of one step is freed in the next
            opt.step(zero_grad=True)
        step()
        gc.collect()
        return m, opt, step
    a, oa, step_a = start()
    b, ob, step_b = start()
    for _ in range(3):
        step_a()
    ctx.sync()
    gc.collect()                        # what was allocated outside the recording is not freed inside it
    ctx.graph_begin()
    step_b()
    gc.collect()                        # what the recording allocated is freed inside it
    gid = ctx.graph_end()
    for _ in range(3):
        ctx.graph_launch(gid)
    ctx.sync()
    assert oa._t == ob._t == 4
    for p, q in zip(a.parameters, b.parameters):
        assert np.array_equal(p.numpy(), q.numpy()) and np.array_equal(p.grad.numpy(), q.grad.numpy())
    for p, q in ((oa._m, ob._m), (oa._v, ob._v)):
        assert np.array_equal(p.numpy().view(np.int32), q.numpy().view(np.int32))
    ctx.check(ctx.lib.fml_graph_destroy(ctx.h, gid))
