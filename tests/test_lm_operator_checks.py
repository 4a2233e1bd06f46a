"""Checks of arguments that the Python side of the language-model operators makes before any launch (CPU)."""
from types import SimpleNamespace

import numpy as np
import pytest


class Reached(Exception):
    """The call got as far as the library."""


class Library:
    def __getattr__(self, name):
        def call(*args):
            raise Reached(name)
        return call


CTX = SimpleNamespace(lib=Library(), h=None)


def buffer(shape, dtype=np.float32):
    return SimpleNamespace(ptr=4096, shape=shape, dtype=dtype, size=int(np.prod(shape)) if shape else 1)


def calls():
    from flutter_ml_b200 import ops
    b = buffer(())
    yield "lens", 5, lambda lens: ops.gated_recurrence_forward(CTX, b, b, b, 5, 3, 8, lens=lens)
    yield "lens", 5, lambda lens: ops.gated_recurrence_backward(CTX, b, b, b, b, b, b, 5, 3, 8, lens=lens)
    yield "positions", 7, lambda pos: ops.qk_norm_rope_forward(CTX, b, b, b, b, 7, 2, 2, 64, positions=pos)
    yield "positions", 7, lambda pos: ops.qk_norm_rope_backward(CTX, b, b, b, b, b, b, 7, 2, 2, 64, positions=pos)


@pytest.mark.parametrize("which", range(4))
def test_lengths_and_positions_too_few(which):
    """The kernels read one length for each sequence and one position for each row."""
    what, n, call = list(calls())[which]
    for bad in (buffer((n - 1,), np.int32), buffer((0,), np.int32), buffer((n,), np.int64), buffer((n,), np.float32), buffer((), np.float32)):
        with pytest.raises(ValueError, match=what):
            call(bad)
    for good in (None, buffer((n,), np.int32), buffer((n + 3,), np.int32), buffer((n, 1), np.int32), buffer((), np.int32)):
        with pytest.raises(Reached):
            call(good)
