"""Results over inputs and over each other: what may be replaced in place gives the bits of a call with tensors of its own, the rest is refused."""
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


def refused(ctx, call):
    before = ctx.launches
    with pytest.raises(ValueError, match="overlap"):
        call()
    assert ctx.launches == before


def test_convolution_over_its_input_is_refused():
    ctx = shim.get_context(0)
    x, dy, w, b, init = rand(ctx, S, T, C), rand(ctx, S, T, C), rand(ctx, C, 4), rand(ctx, C), rand(ctx, S, 3, C)
    wide = rand(ctx, S, T + 1, C)
    flat = rand(ctx, S * T, C)
    seqs = Q.Sequences(ctx, [30, 50])
    for call in (lambda: Q.device_causal_conv1d(x, w, out=x), lambda: Q.device_causal_conv1d(wide[:, 1:], w, out=wide[:, :T]),
                 lambda: Q.device_causal_conv1d(flat, w, sequences=seqs, out=flat), lambda: Q.device_causal_conv1d(x, w, initial=init, final=x[:, :3]),
                 lambda: Q.device_causal_conv1d_grad(dy, x, w, b, out=x), lambda: Q.device_causal_conv1d_grad(dy, x, w, b, out=dy),
                 lambda: Q.device_causal_conv1d_grad(dy, x, w, b, dw=flat[:C, :4]), lambda: Q.device_causal_conv1d_step(x[:, 0], x[:, 1:4], w),
                 lambda: Q.device_causal_conv1d_step(wide[:, 1], init, w, out=Q.DeviceArray(ctx, (S, C), F32, (0, 1), _ptr=wide.ptr))):
        with pytest.raises(ValueError):
            call()
    refused(ctx, lambda: Q.device_causal_conv1d(x, w, out=x))
    refused(ctx, lambda: Q.device_causal_conv1d(wide[:, 1:], w, out=wide[:, :T]))
    refused(ctx, lambda: Q.device_causal_conv1d_grad(dy, x, w, b, out=dy))


def test_halves_of_a_wider_tensor_are_no_overlap():
    """Rows that interleave, as a projection's halves do, and the first and second half of the tokens."""
    ctx = shim.get_context(0)
    w = rand(ctx, C, 4)
    host = np.random.RandomState(1).standard_normal((S, 2 * T, 2 * C))
    for at in (np.s_[:, :T, :C], np.s_[:, T:, C:]):
        for to in (np.s_[:, :T, C:], np.s_[:, T:, :C]):
            wide = put(ctx, host, F32)
            want = Q.device_causal_conv1d(wide[at], w).to_host()
            Q.device_causal_conv1d(wide[at], w, out=wide[to])
            got = wide.to_host()
            assert np.array_equal(got[to], want)
            got[to] = host[to]
            assert np.array_equal(got, host.astype(np.float32))


@pytest.mark.parametrize("dt", list(DTYPES))
def test_norms_in_place(dt):
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    for C in (24, 30, 20000):                          # vectors, single elements, rows that are read three times
        g = rand(ctx, C, dtype=dtype, seed=3)
        xr = lambda: (rand(ctx, 2, 5, C, dtype=dtype, seed=1), rand(ctx, 2, 5, C, dtype=dtype, seed=2))  # noqa: E731
        x, r = xr()
        total, stats = Q.DeviceArray(ctx, x.shape, dtype), Q.DeviceArray(ctx, (2, 5, 2), F32)
        want = Q.device_layer_norm(x, g, residual=r, total=total, stats=stats).to_host()
        sums = total.to_host()
        for over in ("x", "residual"):
            x, r = xr()
            out, tot = (x, r) if over == "x" else (r, x)
            assert np.array_equal(Q.device_layer_norm(x, g, residual=r, total=tot, out=out).to_host(), want) and np.array_equal(tot.to_host(), sums)
        x, r = xr()
        refused(ctx, lambda: Q.device_layer_norm(x, g, residual=r, total=x, out=x))
        refused(ctx, lambda: Q.device_layer_norm(x[:, :4], out=x[:, 1:]))
        refused(ctx, lambda: Q.device_layer_norm(x, x[0, 0], out=x))
        grads = Q.device_layer_norm_grad(r, total, g, stats, dtotal=x)
        want = [a.to_host() for a in grads]
        for over in range(3):
            t = [rand(ctx, 2, 5, C, dtype=dtype, seed=2), put(ctx, sums, dtype), rand(ctx, 2, 5, C, dtype=dtype, seed=1)]
            gamma = rand(ctx, C, dtype=dtype, seed=3)
            got = Q.device_layer_norm_grad(t[0], t[1], gamma, stats, dtotal=t[2], out=t[over], dgamma=gamma)
            assert all(np.array_equal(a.to_host(), b) for a, b in zip(got, want))
        refused(ctx, lambda: Q.device_layer_norm_grad(r, total, g, stats, dgamma=grads[1], dbeta=grads[1]))


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("T,C,N", [(9, 24, 16), (300, 24, 16), (300, 11, 40)])       # uncut, cut into pieces, states of several lanes
def test_scans_in_place(dt, T, C, N):
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    v = inputs(3, [T] * 2, C, N, 1, dtype)

    def tensors():
        t = {k: put(ctx, np.stack(v[k]), dtype) for k in ("x", "dt", "z", "B", "C")}
        t.update({k: put(ctx, v[k], F32) for k in ("A", "D", "dt_bias", "initial")})
        t.update(dy=put(ctx, np.stack(v["z"])[:, ::-1], dtype), dfinal=put(ctx, v["initial"][:, ::-1], F32))
        return t

    def scan(t, **out):
        return Q.device_selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"], dt_bias=t["dt_bias"], softplus=True, initial=t["initial"], **out)

    def grad(t, grads):
        return Q.device_selective_scan_grad(t["dy"], t["x"], t["dt"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"], dt_bias=t["dt_bias"], softplus=True,
                                            initial=t["initial"], dfinal=t["dfinal"], grads=grads)
    want = scan(tensors()).to_host()
    for over in ("x", "dt", "z"):
        t = tensors()
        assert np.array_equal(scan(t, out=t[over]).to_host(), want), over
    want = {k: a.to_host() for k, a in grad(tensors(), {}).items()}
    for grads in (dict(x="x", dt="dt", z="z", B="B", C="C", A="A", D="D", dt_bias="dt_bias", initial="initial"), dict(x="dy", dt="x", z="dt", initial="dfinal"),
                  dict(z="dy")):
        t = tensors()
        got = grad(t, {k: t[o] for k, o in grads.items()})
        for k in want:
            assert np.array_equal(got[k].to_host(), want[k]), (grads, k)
    t = tensors()
    for call in (lambda: scan(t, out=t["x"], final=Q.DeviceArray(ctx, t["initial"].shape, F32, _ptr=t["z"].ptr)),
                 lambda: grad(t, dict(x=t["x"], dt=t["x"])), lambda: grad(t, dict(D=t["dt_bias"], dt_bias=t["dt_bias"])),
                 lambda: grad(t, dict(A=Q.DeviceArray(ctx, t["A"].shape, F32, _ptr=t["initial"].ptr)))):
        refused(ctx, call)


def test_steps_over_their_state_are_refused():
    ctx = shim.get_context(0)
    one = lambda *s: rand(ctx, *s)  # noqa: E731
    state = one(S, C, 4)
    x = Q.DeviceArray(ctx, (S, C), F32, (C * 4, 1), _ptr=state.ptr)
    refused(ctx, lambda: Q.device_selective_scan_step(x, one(S, C), one(C, 4), one(S, 4), one(S, 4), state, out=one(S, C)))
    refused(ctx, lambda: Q.device_selective_scan_step(one(S, C), one(S, C), one(C, 4), one(S, 4), one(S, 4), state, out=x))
    B = one(S, C)
    refused(ctx, lambda: Q.device_selective_scan_step(one(S, C), one(S, C), one(C, 24), B, one(S, 24), one(S, C, 24), out=B))
