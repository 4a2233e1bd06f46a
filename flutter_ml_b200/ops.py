"""Layer-level operations on device arrays, composed from the C-ABI kernels.

Each function names the reference code it stands in for.  Shapes follow the reference's
DenseLayerMatrix convention: activations are [rows x features], weights [in x out]
(lib/layertypes/denseLayer.dart:96-104).
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib
from ._lib import ACT_BY_NAME


def dense_forward(ctx, X, W, b, act, M, N, K, Y, Z=None, precision=-1):
    """Y = act(X.W + b), optionally saving the pre-activation Z: matMul + addMatrixAndVector +
    activation (denseLayer.dart:116-125) as ONE kernel (bias and activation in the epilogue)."""
    ctx.gemm(X, W, Y, M, N, K, bias=b, preact=Z, act=act, precision=precision)


def dense_backward(ctx, X, W, saved, dY, act, M, N, K, dZ, dX=None, dW=None, db=None, accumulate=False,
                   precision=-1, after_dW=None):
    """Gradients of dense_forward.  saved = Z for relu/gelu, Y for sigmoid/tanh.
    dZ = dY * act'(saved) and db = column sums (tensor.dart:1030, 698-704), then
    dX (+)= dZ.W^T (tensor.dart:918-924) and dW (+)= X^T.dZ (:935-941); the transposes are operand
    layout flags, nothing is copied.  db must be zeroed by the caller unless it accumulates.  The weight gradient is
    queued first; `after_dW()` (if given) runs on the host right behind it, which is where a data-parallel caller starts
    the exchange of dW and db so that it overlaps the dX product."""
    code = ACT_BY_NAME[act]
    if code == _lib.ACT_NONE and db is None:
        dZ = dY
    else:
        ctx.call("fml_act_bwd", code, saved, dY, dZ, M, N, 0, db)
    beta = 1.0 if accumulate else 0.0
    if dW is not None:
        ctx.gemm(X, dZ, dW, K, N, M, transA=True, beta=beta, precision=precision)
    if after_dW is not None:
        after_dW()
    if dX is not None:
        ctx.gemm(dZ, W, dX, M, K, N, transB=True, beta=beta, precision=precision)
    return dZ


class GradientExchange:
    """Data-parallel exchange of a layer's weight and bias gradient, overlapped with the product that follows: the
    all-reduce (sum over ranks, NCCL) is enqueued on side stream `lane` behind everything queued so far, the persistent
    products that run beside it leave `reserve_sms` SMs free for it, and `join` makes the main stream wait for it."""

    def __init__(self, ctx, world: int, lane: int = 2, reserve_sms: int = 0, ev_start: int = 60, ev_done: int = 61,
                 overlap_rows: int = 0):
        self.ctx, self.world, self.lane, self.reserve = ctx, world, lane, reserve_sms
        self.ev_start, self.ev_done = ev_start, ev_done
        # rows of the product that follows which are computed on the reduced SM set while the exchange runs; the rest of
        # it is launched with all SMs again (0: the whole product runs on the reduced set)
        self.overlap_rows = overlap_rows

    def start(self, buf, n):
        if self.world == 1:
            return
        c, L = self.ctx, self.ctx.lib
        c.check(L.fml_event_record_on(c.h, self.ev_start, -1))
        c.check(L.fml_wait_event(c.h, self.lane, self.ev_start))
        c.check(L.fml_dp_allreduce_sum_on(c.h, self.lane, buf.ptr, n))
        c.check(L.fml_event_record_on(c.h, self.ev_done, self.lane))
        if self.reserve:
            c.check(L.fml_set_sm_reserve(c.h, self.reserve))

    def release_sms(self):
        """Later launches may use every SM again (the exchange is expected to be over by the time they start)."""
        if self.world > 1 and self.reserve:
            self.ctx.check(self.ctx.lib.fml_set_sm_reserve(self.ctx.h, 0))

    def join(self):
        if self.world == 1:
            return
        c, L = self.ctx, self.ctx.lib
        self.release_sms()
        c.check(L.fml_wait_event(c.h, -1, self.ev_done))


class DenseFwdBwdHost:
    """The dense forward+backward step driven from HOST buffers, the way the reference's FFI
    binding is used (lib/cuda/cudacaller.dart:25-60: host lists in, host list out), but with
    device buffers and pinned staging kept between calls."""

    def __init__(self, ctx, M, N, K, act="gelu", precision=-1, exchange=None):
        self.ctx, self.M, self.N, self.K, self.act, self.precision = ctx, M, N, K, act, precision
        self.exchange = exchange     # GradientExchange or None: sums dB and dbias over the data-parallel ranks
        e = ctx.empty
        self.A, self.B, self.bias, self.dC = e(M, K), e(K, N), e(N), e(M, N)
        self.C, self.Z, self.dZ, self.dA = e(M, N), e(M, N), e(M, N), e(M, K)
        self._gb_off = (K * N + 3) & ~3          # bias gradient at a 16-byte aligned offset behind the weight gradient
        self.grads = e(self._gb_off + N)         # side by side: one exchange
        self.dB, self.dbias = self.grads.view(0, (K, N)), self.grads.view(self._gb_off, (N,))
        p = ctx.pinned
        self.h_in = {"A": p((M, K)), "B": p((K, N)), "bias": p((N,)), "dC": p((M, N))}
        self.h_out = {"C": p((M, N)), "dA": p((M, K)), "dB": p((K, N)), "dbias": p((N,))}
        self.h2d_bytes = sum(a.nbytes for a in self.h_in.values())
        self.d2h_bytes = sum(a.nbytes for a in self.h_out.values())

    def compute(self, d=None):
        """Forward, dZ + dbias, dW, [exchange of dW and dbias started], dA, [exchange joined] on buffer set `d`."""
        c = self.ctx
        d = d or {k: getattr(self, k) for k in ("A", "B", "bias", "dC", "C", "Z", "dZ", "dA", "dB", "dbias", "grads")}
        dense_forward(c, d["A"], d["B"], d["bias"], self.act, self.M, self.N, self.K, d["C"], d["Z"], self.precision)
        c.zero(d["dbias"])
        ex = self.exchange
        M, N, K = self.M, self.N, self.K
        split = ex.overlap_rows if (ex and ex.world > 1 and 0 < ex.overlap_rows < M) else 0
        dense_backward(c, d["A"], d["B"], d["Z"], d["dC"], self.act, M, N, K, d["dZ"], None if split else d["dA"], d["dB"],
                       d["dbias"], precision=self.precision,
                       after_dW=(lambda: ex.start(d["grads"], d["grads"].size)) if ex else None)
        if split:
            # dA in two row blocks: the first beside the exchange on the reduced SM set, the second on all SMs
            c.gemm(d["dZ"], d["B"], d["dA"], split, K, N, transB=True, precision=self.precision)
            ex.release_sms()
            c.gemm(d["dZ"].view(split * N, (M - split, N)), d["B"], d["dA"].view(split * K, (M - split, K)), M - split, K, N,
                   transB=True, precision=self.precision)
        if ex:
            ex.join()

    def pipelined(self, steps: int):
        """`steps` end-to-end steps with the copies on two side streams and two sets of device buffers,
        so the upload of step s+1, the kernels of step s and the download of step s-1 overlap (PCIe is
        full duplex).  Same bytes per step as __call__; every step still uploads and downloads everything."""
        c, L = self.ctx, self.ctx.lib
        if not hasattr(self, "_sets"):
            e, (M, N, K) = c.empty, (self.M, self.N, self.K)
            second = dict(A=e(M, K), B=e(K, N), bias=e(N), dC=e(M, N), C=e(M, N), Z=e(M, N), dZ=e(M, N), dA=e(M, K),
                          grads=e(self._gb_off + N))
            second["dB"], second["dbias"] = second["grads"].view(0, (K, N)), second["grads"].view(self._gb_off, (N,))
            first = {k: getattr(self, k) for k in second}
            self._sets = [first, second]
        EV_UP, EV_COMP, EV_DOWN = 40, 42, 44     # event slots, +0/+1 per buffer set
        chk = c.check

        def upload(s):
            b = s % 2
            if s >= 2:
                chk(L.fml_wait_event(c.h, 0, EV_COMP + b))   # the kernels of step s-2 have read this set
            for k in ("A", "B", "bias", "dC"):
                chk(L.fml_lane_h2d(c.h, 0, self._sets[b][k].ptr, self.h_in[k].ctypes.data, self.h_in[k].size))
            chk(L.fml_event_record_on(c.h, EV_UP + b, 0))

        upload(0)
        for s in range(steps):
            b = s % 2
            d = self._sets[b]
            if s + 1 < steps:
                upload(s + 1)
            chk(L.fml_wait_event(c.h, -1, EV_UP + b))
            if s >= 2:
                chk(L.fml_wait_event(c.h, -1, EV_DOWN + b))  # the download of step s-2 has drained this set
            self.compute(d)
            chk(L.fml_event_record_on(c.h, EV_COMP + b, -1))
            chk(L.fml_wait_event(c.h, 1, EV_COMP + b))
            for k in ("C", "dA", "dB", "dbias"):
                chk(L.fml_lane_d2h(c.h, 1, self.h_out[k].ctypes.data, d[k].ptr, d[k].size))
            chk(L.fml_event_record_on(c.h, EV_DOWN + b, 1))
        chk(L.fml_lane_sync(c.h, 1))
        chk(L.fml_lane_sync(c.h, 0))
        c.sync()
        return self.h_out

    def __call__(self):
        """One end-to-end step: pinned host -> device, compute, device -> pinned host."""
        c = self.ctx
        for k, dst in (("A", self.A), ("B", self.B), ("bias", self.bias), ("dC", self.dC)):
            c.upload_async(self.h_in[k], dst)
        self.compute()
        for k, src in (("C", self.C), ("dA", self.dA), ("dB", self.dB), ("dbias", self.dbias)):
            c.download_into(src, self.h_out[k])  # the last one synchronises
        return self.h_out


def _index_buffer(a, n, what):
    """An int32 buffer of at least n entries; a view without a shape is an address and has no length to check."""
    if a.dtype != np.int32 or (a.shape and a.size < n):
        raise ValueError(f"{what} must be int32, {n} of them")


def gated_recurrence_forward(ctx, f, x, h, n_seq, seq_len, dim, form="gated", h0=None, lens=None, h_last=None, strides_in=None, strides_h=None):
    """h_t = a_t h_{t-1} + (1 - a_t) x_t with a = sigmoid(f) (form "gated"), or h_t = f_t h_{t-1} + x_t ("linear"), along every
    sequence (`fml_gated_recurrence_fwd`).  strides_in (f and x) and strides_h are (sequence, step) strides in elements,
    sequence-major without gaps by default; lens: int32 lengths on the device."""
    if lens is not None:
        _index_buffer(lens, n_seq, "gated_recurrence: lens")
    dense = (seq_len * dim, dim)
    si, sh = strides_in or dense, strides_h or dense
    rc = ctx.lib.fml_gated_recurrence_fwd(ctx.h, _lib.RECURRENCE_BY_NAME[form], n_seq, seq_len, dim, f and f.ptr, x and x.ptr, si[0], si[1],
                                          h0 and h0.ptr, lens and lens.ptr, h and h.ptr, sh[0], sh[1], h_last and h_last.ptr)
    if rc:
        ctx.check(rc)
    ctx.launches += 1


def gated_recurrence_backward(ctx, f, x, h, dy, df, dx, n_seq, seq_len, dim, form="gated", h0=None, lens=None, dh_last=None, dh0=None,
                              strides_in=None, strides_h=None, accumulate=False):
    """Gradients of `gated_recurrence_forward` from its inputs and its h (`fml_gated_recurrence_bwd`); dy may be None (zero),
    df and dx lie at the strides of f and x, dy at those of h."""
    if lens is not None:
        _index_buffer(lens, n_seq, "gated_recurrence: lens")
    dense = (seq_len * dim, dim)
    si, sh = strides_in or dense, strides_h or dense
    rc = ctx.lib.fml_gated_recurrence_bwd(ctx.h, _lib.RECURRENCE_BY_NAME[form], n_seq, seq_len, dim, f and f.ptr, x and x.ptr, si[0], si[1],
                                          h0 and h0.ptr, lens and lens.ptr, h and h.ptr, dy and dy.ptr, sh[0], sh[1], dh_last and dh_last.ptr,
                                          df and df.ptr, dx and dx.ptr, dh0 and dh0.ptr, 1 if accumulate else 0)
    if rc:
        ctx.check(rc)
    ctx.launches += 1


def qk_norm_rope_scratch(d_head: int) -> int:
    """Floats of the scratch buffer that the gain gradients of `qk_norm_rope_backward` go through."""
    return _lib.QK_NORM_ROPE_PARTS * 2 * d_head


def qk_norm_rope_forward(ctx, q, k, q_out, k_out, rows, heads_q, heads_k, d_head, gain_q=None, gain_k=None, positions=None, seq_len=0,
                         rot_dim=None, interleaved=False, base=10000.0, eps=1e-6, ld_q=None, ld_k=None, ld_q_out=None, ld_k_out=None):
    """Norm of every query and key head, its gain, and the rotation by position, in one launch (`fml_qk_norm_rope_fwd`).
    Row strides default to rows that lie end to end; rot_dim defaults to the whole head; k may be None with heads_k = 0."""
    if positions is not None:
        _index_buffer(positions, rows, "qk_norm_rope: positions")
    wq, wk = heads_q * d_head, heads_k * d_head
    rc = ctx.lib.fml_qk_norm_rope_fwd(ctx.h, q and q.ptr, ld_q or wq, q_out and q_out.ptr, ld_q_out or wq, heads_q, k and k.ptr, ld_k or wk,
                                      k_out and k_out.ptr, ld_k_out or wk, heads_k, rows, d_head, gain_q and gain_q.ptr, gain_k and gain_k.ptr,
                                      positions and positions.ptr, seq_len, d_head if rot_dim is None else rot_dim, 1 if interleaved else 0, base, eps)
    if rc:
        ctx.check(rc)
    ctx.launches += 1


def qk_norm_rope_backward(ctx, q, k, dq_out, dk_out, dq, dk, rows, heads_q, heads_k, d_head, gain_q=None, gain_k=None, dgain_q=None,
                          dgain_k=None, positions=None, seq_len=0, rot_dim=None, interleaved=False, base=10000.0, eps=1e-6, ld_q=None,
                          ld_k=None, ld_dq_out=None, ld_dk_out=None, ld_dq=None, ld_dk=None, accumulate=False, scratch=None):
    """Gradients of `qk_norm_rope_forward` (`fml_qk_norm_rope_bwd`); dgain_q and dgain_k are added to, through `scratch` of
    `qk_norm_rope_scratch(d_head)` floats."""
    if positions is not None:
        _index_buffer(positions, rows, "qk_norm_rope: positions")
    wq, wk = heads_q * d_head, heads_k * d_head
    if scratch is not None and scratch.size < qk_norm_rope_scratch(d_head):
        raise ValueError(f"qk_norm_rope_backward: the scratch buffer needs {qk_norm_rope_scratch(d_head)} floats")
    rc = ctx.lib.fml_qk_norm_rope_bwd(ctx.h, q and q.ptr, ld_q or wq, dq_out and dq_out.ptr, ld_dq_out or wq, dq and dq.ptr, ld_dq or wq, heads_q,
                                      k and k.ptr, ld_k or wk, dk_out and dk_out.ptr, ld_dk_out or wk, dk and dk.ptr, ld_dk or wk, heads_k, rows,
                                      d_head, gain_q and gain_q.ptr, gain_k and gain_k.ptr, dgain_q and dgain_q.ptr, dgain_k and dgain_k.ptr,
                                      positions and positions.ptr, seq_len, d_head if rot_dim is None else rot_dim, 1 if interleaved else 0, base,
                                      eps, 1 if accumulate else 0, scratch and scratch.ptr)
    if rc:
        ctx.check(rc)
    ctx.launches += 2 if dgain_q is not None or dgain_k is not None else 1


class AdamWPlan:
    """AdamW (lib/optimizers/adamw.dart:82-89) over a list of tensors in one launch (`fml_adamw_plan_*`).  `w` and `g` are
    lists of device arrays, `m` and `v` the two state buffers of `state_floats(sizes, stateBits)` floats, zeroed before the
    first step; all must keep their addresses while the plan lives (the plan holds a reference to each)."""

    def __init__(self, ctx, w, g, m, v, stateBits: int = 32):
        if len(w) != len(g) or any(a.size != b.size for a, b in zip(w, g)):
            raise ValueError("AdamWPlan: every tensor needs a gradient of its size")
        if any(a.dtype != np.float32 for a in (*w, *g, m, v)):
            raise ValueError("AdamWPlan: tensors, gradients and states are float32 buffers")
        sizes = [a.size for a in w]
        need = self.state_floats(sizes, stateBits)
        if m.size < need or v.size < need:
            raise ValueError(f"AdamWPlan: the state buffers need {need} floats")
        self.ctx, self._keep, self.id, self.stateBits = ctx, (list(w), list(g), m, v), -1, stateBits
        n = len(w)
        wp, gp = np.array([a.ptr for a in w], dtype=np.uint64), np.array([a.ptr for a in g], dtype=np.uint64)
        sz, pid = np.array(sizes, dtype=np.int64), ctypes.c_int32(-1)
        ctx.check(ctx.lib.fml_adamw_plan_create(ctx.h, n, wp.ctypes.data, gp.ctypes.data, sz.ctypes.data, m.ptr, v.ptr, stateBits,
                                                ctypes.byref(pid)))
        self.id = pid.value

    @staticmethod
    def state_floats(sizes, stateBits: int = 32) -> int:
        """Floats of each of the two state buffers for tensors of these element counts."""
        lib, sz, out = _lib.load(), np.array(sizes, dtype=np.int64), ctypes.c_int64(0)
        if lib.fml_adamw_state_floats(len(sz), sz.ctypes.data, stateBits, ctypes.byref(out)) != 0:
            raise _lib.FmlError(lib.fml_last_error(None).decode())
        return out.value

    def step(self, lr, beta1, beta2, epsilon, weightDecay, t, grad_scale=1.0, zero_grad=False, seed=0, lane=-1):
        """One update; t = 0 counts on the device (for recorded steps).  8-bit states are rounded at random by `seed`, or to
        the nearest code where it is negative, which with a beta2 near 1 is not AdamW (see `fml_adamw_plan_step`)."""
        self.ctx.check(self.ctx.lib.fml_adamw_plan_step(self.ctx.h, self.id, lane, lr, beta1, beta2, epsilon, weightDecay, t, grad_scale,
                                                        1 if zero_grad else 0, seed))
        self.ctx.launches += 1 if t else 2

    @property
    def count(self) -> int:
        """Steps counted on the device so far (those with t = 0); setting it goes on from a checkpoint."""
        t = ctypes.c_int32(0)
        self.ctx.check(self.ctx.lib.fml_adamw_plan_count(self.ctx.h, self.id, ctypes.byref(t)))
        return t.value

    @count.setter
    def count(self, t: int):
        self.ctx.check(self.ctx.lib.fml_adamw_plan_set_count(self.ctx.h, self.id, t))

    def close(self):
        if self.id >= 0 and self.ctx.h:
            self.ctx.check(self.ctx.lib.fml_adamw_plan_destroy(self.ctx.h, self.id))
        self.id = -1

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
