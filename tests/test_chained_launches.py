"""Kernels that are set up while the kernel before them drains (fml_launch_chained in csrc/common.cuh): what they may read how,
and chains of them without a pause against the same calls one at a time."""
import os
import re

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "flutter_ml_b200", "csrc")
f32 = np.float32


def test_chained_kernels_read_by_plain_loads():
    """A chained kernel starts while its predecessor writes: no read-only loads, and no __restrict__ (whose loads may become
    such, or move up across the wait), but for the optimizer's table of work items, which is written when the plan is made."""
    seen = 0
    for name in sorted(os.listdir(CSRC)):
        text = open(os.path.join(CSRC, name)).read()
        if not name.endswith(".cu") or "fml_chain_wait" not in text:
            continue
        seen += 1
        code = re.sub(r"//[^\n]*", "", text).replace("const Item* __restrict__ items", "")
        for word in ("__ldg", "ld.global.nc", "__restrict__", "__ldcg", "__ldca"):
            assert word not in code, (name, word)
    assert seen == 3


@pytest.fixture(scope="module")
def ctx():
    from flutter_ml_b200 import _lib
    c = _lib.Context()
    yield c
    assert c.device_status() == 0
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_chain_is_its_calls_one_at_a_time(ctx, bits):
    """Recurrence, norm, its backward pass with gain sums, and an optimizer step on input and gains that the next round reads:
    forty rounds without a pause give bit for bit what they give with the device idle between any two calls."""
    from flutter_ml_b200 import ops
    n, S, heads, d = 8, 24, 4, 64
    R, W = n * S, 2 * heads * d
    rng = np.random.default_rng(2)
    z0, dy0 = rng.standard_normal(R * 2 * W).astype(f32), rng.standard_normal((R, W)).astype(f32)
    gains = rng.standard_normal(2 * d).astype(f32) * f32(0.1) + f32(1)

    def run(pause):
        z, g, dy, h, y, dh, dz = (ctx.upload(z0), ctx.upload(gains), ctx.upload(dy0), ctx.zeros(R, W), ctx.zeros(R, W), ctx.zeros(R, W),
                                  ctx.zeros(R * 2 * W))
        dg, scratch = ctx.zeros(2 * d), ctx.empty(ops.qk_norm_rope_scratch(d))
        sizes = [z.size, g.size]
        m, v = (ctx.zeros(ops.AdamWPlan.state_floats(sizes, bits)) for _ in range(2))
        plan = ops.AdamWPlan(ctx, [z, g], [dz, dg], m, v, bits)
        gq, gk, dq, dk = g, g.view(d, (d,)), dg, dg.view(d, (d,))
        heads_of = lambda b: (b, b.view(heads * d, ()))  # noqa: E731
        opt = dict(gain_q=gq, gain_k=gk, seq_len=S, ld_q=W, ld_k=W)
        st = dict(strides_in=(S * 2 * W, 2 * W))
        seen = []
        for _ in range(40):
            for call in (lambda: ops.gated_recurrence_forward(ctx, z, z.view(W, ()), h, n, S, W, **st),
                         lambda: ops.qk_norm_rope_forward(ctx, *heads_of(h), *heads_of(y), R, heads, heads, d, ld_q_out=W, ld_k_out=W, **opt),
                         lambda: ops.qk_norm_rope_backward(ctx, *heads_of(h), *heads_of(dy), *heads_of(dh), R, heads, heads, d, dgain_q=dq, dgain_k=dk,
                                                           scratch=scratch, ld_dq_out=W, ld_dk_out=W, ld_dq=W, ld_dk=W, **opt),
                         lambda: ops.gated_recurrence_backward(ctx, z, z.view(W, ()), h, dh, dz, dz.view(W, ()), n, S, W, **st),
                         lambda: plan.step(0.01, 0.9, 0.999, 1e-8, 0.0, 0, zero_grad=True, seed=1)):
                call()
                if pause:
                    ctx.sync()
        for b in (z, g, h, y, dh, m, v):
            seen.append(b.numpy().view(np.int32))
        plan.close()
        return seen
    want = run(True)
    for _ in range(3):
        for a, b in zip(run(False), want):
            assert np.array_equal(a, b)


@pytest.mark.gpu
def test_recorded_by_the_owner_of_the_stream():
    """The context works on a stream that torch owns and records: recurrence (in clusters, their first use), norm and optimizer
    step replayed three times against three eager rounds, also when the plan has been destroyed in between."""
    import torch
    from flutter_ml_b200 import _lib, ops
    S, W, d = 6000, 128, 64
    rng = np.random.default_rng(3)
    z0, dy0 = rng.standard_normal((S, 2 * W)).astype(f32), rng.standard_normal((S, W)).astype(f32)

    def run(record):
        stream = torch.cuda.Stream()
        ctx = _lib.Context()
        ctx.check(ctx.lib.fml_set_stream(ctx.h, stream.cuda_stream))
        z, dy, h, y, dz = ctx.upload(z0), ctx.upload(dy0), ctx.zeros(S, W), ctx.zeros(S, W), ctx.zeros(S, 2 * W)
        n = ops.AdamWPlan.state_floats([z.size], 8)
        m, v = ctx.zeros(n), ctx.zeros(n)
        plan = ops.AdamWPlan(ctx, [z], [dz], m, v, 8)

        def step():
            st = dict(strides_in=(S * 2 * W, 2 * W))
            ops.gated_recurrence_forward(ctx, z, z.view(W, ()), h, 1, S, W, **st)
            ops.qk_norm_rope_forward(ctx, h, h.view(d, ()), y, y.view(d, ()), S, 1, 1, d, ld_q=W, ld_k=W, ld_q_out=W, ld_k_out=W)
            ops.gated_recurrence_backward(ctx, z, z.view(W, ()), h, dy, dz, dz.view(W, ()), 1, S, W, **st)
            plan.step(0.01, 0.9, 0.999, 1e-8, 0.0, 0, seed=2)
        ctx.sync()
        if record:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step()
            plan.close()
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
        else:
            for _ in range(3):
                step()
        ctx.sync()
        out = [b.numpy().view(np.int32) for b in (z, h, y, dz, m, v)]
        assert ctx.device_status() == 0
        if record:
            graph.reset()
        ctx.close()
        return out
    for a, b in zip(run(True), run(False)):
        assert np.array_equal(a, b)
