"""Results over inputs: what may be replaced in place gives the bits of a call with tensors of its own."""
import numpy as np
import pytest

from sequence_util import DTYPES, put
from test_gpu_selective_scan import inputs
from theano_b200 import sequence as Q
from theano_b200 import shim

pytestmark = pytest.mark.gpu
F32 = np.dtype(np.float32)
S, T, C = 2, 40, 24


def rand(ctx, *shape, dtype=F32, seed=0):
    return put(ctx, np.random.RandomState(seed).standard_normal(shape), dtype)


def test_gradient_of_the_initial_tokens_in_their_place():
    """Blocks read the tokens before a sequence while others write their gradient."""
    ctx = shim.get_context(0)
    x, dy, w, b = rand(ctx, S, T, C), rand(ctx, S, T, C, seed=1), rand(ctx, C, 4), rand(ctx, C)
    init = lambda: rand(ctx, S, 3, C, seed=4)  # noqa: E731
    want = [a.to_host() for a in Q.device_causal_conv1d_grad(dy, x, w, b, silu=True, initial=init(), dinitial=Q.DeviceArray(ctx, (S, 3, C), F32))]
    for _ in range(3):
        i = init()
        got = Q.device_causal_conv1d_grad(dy, x, w, b, silu=True, initial=i, dinitial=i)
        assert all(np.array_equal(a.to_host(), b) for a, b in zip(got, want))


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("T,C,N", [(9, 24, 16), (300, 24, 16), (300, 11, 40)])       # uncut, cut into pieces, states of several lanes
def test_gradient_of_the_initial_states_in_their_place(dt, T, C, N):
    """The first piece writes them, all pieces read the states."""
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    v = inputs(3, [T] * 2, C, N, 1, dtype)
    x, steps, z, B, Cm = (put(ctx, np.stack(v[k]), dtype) for k in ("x", "dt", "z", "B", "C"))
    A = put(ctx, v["A"], F32)
    initial = lambda: put(ctx, v["initial"], F32)  # noqa: E731
    want = {k: a.to_host() for k, a in Q.device_selective_scan_grad(z, x, steps, A, B, Cm, softplus=True, initial=initial(), dfinal=initial()).items()}
    for both in (False, True):
        i = initial()
        got = Q.device_selective_scan_grad(z, x, steps, A, B, Cm, softplus=True, initial=i, dfinal=i if both else initial(), grads=dict(initial=i))
        assert all(np.array_equal(got[k].to_host(), want[k]) for k in want)
