"""The selective scan where decays leave float32's range, grow, or are no numbers: prompts give what single tokens and the formulas give."""
import numpy as np
import pytest

import sequence_plain as P
from sequence_util import DTYPES, close, put
from theano_b200 import sequence as Q
from theano_b200 import shim

pytestmark = pytest.mark.gpu
F32 = np.dtype(np.float32)
TYPES = pytest.mark.parametrize("dt", list(DTYPES))
STATES = pytest.mark.parametrize("C,N", [(8, 1), (8, 2), (24, 16), (16, 5), (8, 40)])       # every lane's first states, in each form
# delta * A of one token: raw steps of these sizes (exact in 16 bits) and A = 1; beyond 88.7 the exponential exceeds float32
POWERS = np.array([-3000, -100, -88, -20, -1, -0.0625, 0, 0.0625, 1, 20, 80, 88, 92, 104, 140, 208, 1000, 30000], np.float32)


def run(ctx, dtype, x, dt, A, B, C, initial, **more):
    final = Q.DeviceArray(ctx, initial.shape, np.float32)
    y = Q.device_selective_scan(put(ctx, x, dtype), put(ctx, dt, dtype), put(ctx, A, F32), put(ctx, B, dtype), put(ctx, C, dtype),
                                initial=put(ctx, initial, F32), final=final, **more)
    return y.to_host(), final.to_host()


@TYPES
@STATES
def test_decays_of_every_size(dt, C, N):
    """One token that drives nothing: the final state is exp(delta A) times the initial one, infinite where that exceeds float32."""
    ctx, S = shim.get_context(0), len(POWERS)
    x, B = np.zeros((S, 1, C)), np.ones((S, 1, N))
    steps = np.broadcast_to(POWERS[:, None, None], (S, 1, C))
    _, final = run(ctx, DTYPES[dt], x, steps, np.ones((C, N)), B, B, np.full((S, C, N), 0.5, np.float32))
    with np.errstate(over="ignore"):
        want = np.exp(POWERS.astype(np.float64)) * 0.5
    for i, w in enumerate(want):
        if w > 3.4e38:
            assert (final[i] == np.inf).all(), (POWERS[i], final[i].min(), final[i].max())
        else:      # the exponential's 2^-22, three roundings of its argument (log2(e), times A, times delta; 2^-24 of it each) and one
            # of the product; below 2^-126 zero
            assert np.abs(final[i] - w).max() <= w * (2.0 ** -22 + 2.0 ** -24 * (1 + 3 * abs(POWERS[i]))) + 2.0 ** -126, POWERS[i]


@TYPES
@STATES
def test_prompts_and_steps_agree_beyond_the_range(dt, C, N):
    """Growing states: the same tokens as a prompt and one by one overflow at the same token, to the same sign."""
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    S, T = 2, 12
    steps = np.zeros((S, T, C))
    steps[0, 3], steps[0, 7], steps[1, 5] = 104, 12, 0.5
    x, B = np.ones((S, T, C)), np.ones((S, T, N))
    A, init = np.ones((C, N)), np.full((S, C, N), 0.25, np.float32)
    init[:, 1::2] *= -1
    x[:, :, 1::2] *= -1
    y, final = run(ctx, dtype, x, steps, A, B, B, init)
    state = put(ctx, init, F32)
    for t in range(T):
        part = lambda a: put(ctx, a[:, t], dtype)  # noqa: E731
        one = Q.device_selective_scan_step(part(x), part(steps), put(ctx, A, F32), part(B), part(B), state).to_host()
        inf = np.isinf(one)
        assert inf[0].all() == (t >= 3) and not inf[1].any()
        assert np.array_equal(y[:, t][inf], one[inf])
        # values of one sign: on either side an exponential of 2^-22, sums of N + 4 terms, a result rounded to the type
        assert np.allclose(y[:, t][~inf], one[~inf], rtol=2 * (2.0 ** -22 + (N + 4) * 2.0 ** -24 + (0 if dt == "f32" else 2.0 ** -8)), atol=0)
    assert np.isinf(final[0]).all() and np.array_equal(final[0], state.to_host()[0])


@TYPES
@STATES
def test_not_a_number_in_A(dt, C, N):
    """It reaches every output of its channel, and passes by a sequence without tokens."""
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    lengths = [5, 0, 60]
    rows = sum(lengths)
    for n in {0, min(1, N - 1), N - 1}:
        A = np.full((C, N), -1.0, np.float32)
        A[3, n] = np.nan
        ones = lambda *s: np.ones(s)  # noqa: E731
        y, final = run(ctx, dtype, ones(rows, C), ones(rows, C) * 0.125, A, ones(rows, N), ones(rows, N), np.ones((3, C, N), np.float32),
                       sequences=Q.Sequences(ctx, lengths))
        bad = np.zeros((C, N), bool)
        bad[3, n] = True
        assert np.array_equal(np.isnan(final[0]), bad) and np.array_equal(np.isnan(final[2]), bad) and (final[1] == 1).all()
        assert np.isnan(y[:, 3]).all() and np.isfinite(np.delete(y, 3, 1)).all()


@TYPES
@pytest.mark.parametrize("C,N", [(8, 2), (24, 16), (8, 40)])
def test_gradients_behind_an_overflow(dt, C, N):
    """dC[t] = dy h[t], from the states that the gradient keeps: infinite from the token on at which they overflow; NaN with a NaN in A."""
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    T, at = 12, 3
    steps = np.zeros((1, T, C))
    steps[:, at] = 208
    ones = lambda *s: put(ctx, np.ones(s), dtype)  # noqa: E731

    def gradient(A):
        init = put(ctx, np.ones((1, C, N)), F32)
        args = (ones(1, T, C), put(ctx, np.zeros((1, T, C)), dtype), put(ctx, steps, dtype), put(ctx, A, F32), ones(1, T, N), ones(1, T, N))
        return Q.device_selective_scan_grad(*args, initial=init)["C"].to_host()[0]
    dC = gradient(np.ones((C, N)))
    assert (dC[:at] == C).all() and (dC[at:] == np.inf).all()
    A = np.full((C, N), -1.0)
    A[2, 0] = np.nan
    dC = gradient(A)
    assert np.isnan(dC[:, 0]).all() and (dC[:at, 1:] == C).all()


def test_states_of_zero_stay_zero_while_decays_grow():
    """A prompt that begins with tokens of no input and large growing steps, long enough to be cut: a piece's decays together exceed float32,
    the states do not."""
    ctx = shim.get_context(0)
    C, N, T, quiet = 8, 16, 400, 250
    rs = np.random.RandomState(2)
    x, steps = rs.standard_normal((T, C)).astype(np.float32), np.full((T, C), 2.0 ** -7, np.float32)
    B, Cm = rs.standard_normal((2, T, 1, N)).astype(np.float32)
    x[:quiet], steps[:quiet] = 0, 4
    A = np.full((C, N), 1.0, np.float32)
    want, m = (P.selective_scan([x], [steps], A, [B], [Cm], magnitudes=k) for k in (False, True))
    # a path through the T - quiet tokens behind the growth (an exponential of 4 and three roundings of an argument below 1 each), their
    # pieces' sums of deltas, sums over states
    e = (60 + 7.4 * (T - quiet)) * 2.0 ** -24
    for initial in (0.0, -0.0):
        y, final = run(ctx, F32, x[None], steps[None], A, B[None], Cm[None], np.full((1, C, N), initial, np.float32))
        assert (y[0, :quiet] == 0).all()
        close(y[0], want["y"][0], F32, e * m["y"][0])
        close(final, want["final"], F32, e * m["final"])
