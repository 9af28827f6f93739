"""The selective scan: prompts, packed prompts and single tokens against float64."""
import numpy as np
import pytest

import sequence_plain as P
from sequence_util import DTYPES, E32, close, frame_intact, framed, normal, put
from theano_b200 import sequence as Q
from theano_b200 import shim

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dt", list(DTYPES))
# (sequences, tokens, channels, states, groups): one token, a tile's ends, odd channels and states, lanes of each state size, sequences cut
# into pieces, groups narrower than a block
SHAPES = [(1, 1, 8, 16, 1), (2, 31, 16, 16, 1), (1, 32, 40, 16, 2), (2, 33, 13, 5, 1), (1, 70, 24, 1, 3), (2, 40, 16, 32, 1), (1, 37, 16, 64, 2),
          (1, 21, 24, 128, 1), (1, 19, 10, 100, 2), (3, 300, 64, 16, 1), (1, 700, 24, 13, 1), (1, 300, 136, 16, 17)]


def inputs(seed, lengths, C, N, G, dtype, decay=1.0):
    """x, dt, z, B, C per sequence and A, D, dt_bias; step sizes from 0.001 to some, decays of 1 to N per step of 1."""
    rs = np.random.RandomState(seed)
    per = lambda *s: [normal(rs, (n,) + s, dtype) for n in lengths]  # noqa: E731
    v = dict(x=per(C), dt=per(C), z=per(C), B=per(G, N), C=per(G, N))
    v["A"] = (-decay * (1 + np.arange(N)) * np.exp(rs.standard_normal((C, N)) * 0.2)).astype(np.float32)
    v["D"] = rs.standard_normal(C).astype(np.float32)
    v["dt_bias"] = rs.uniform(-6, 1, C).astype(np.float32)
    v["initial"] = rs.standard_normal((len(lengths), C, N)).astype(np.float32)
    return v


def plain(v, which, softplus, **more):
    opt = {k: v[k] for k in ("D", "dt_bias") if k in which}
    return P.selective_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], zs=v["z"] if "z" in which else None, softplus=softplus,
                            initials=v["initial"] if "initial" in which else None, **opt, **more)


def units(v):
    """Relative errors, in 2^-24, of a product along any path through the tokens: of each decay the exponential's 4, the argument's 3 per unit
    of its size and, where sequences are cut, the sum of deltas' one per token; 60 for deltas, gates and the sums over states."""
    T = max(len(x) for x in v["x"])
    delta = max([np.logaddexp(0, np.abs(d) + np.abs(v["dt_bias"]).max()).max() if d.size else 0 for d in v["dt"]])
    return 60 + T * (4 + min(4, 3 * delta)) + 0.4 * T


def on_device(ctx, v, dtype, which):
    S = len(v["x"])
    t = {k: put(ctx, np.stack(v[k]), dtype) for k in ("x", "dt", "B", "C")}
    more = {k: put(ctx, v[k], np.float32) for k in ("D", "dt_bias", "initial") if k in which}
    if "z" in which:
        more["z"] = put(ctx, np.stack(v["z"]), dtype)
    assert S == len(v["z"])
    return (t["x"], t["dt"], put(ctx, v["A"], np.float32), t["B"], t["C"]), more


@TYPES
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("which,softplus", [(("D", "z", "dt_bias", "initial"), True), ((), True), (("D", "initial"), False)], ids=["all", "none", "raw"])
def test_prompts(dt, shape, which, softplus):
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    S, T, C, N, G = shape
    v = inputs(C + N, [T] * S, C, N, G, dtype)
    if not softplus:
        v["dt"] = [np.abs(d) for d in v["dt"]]
    args, more = on_device(ctx, v, dtype, which)
    wide, out = framed(ctx, (S, T, C), dtype)
    _, xin = framed(ctx, (S, T, C), dtype, value=np.stack(v["x"]))
    final = Q.DeviceArray(ctx, (S, C, N), np.float32)
    Q.device_selective_scan(xin, *args[1:], softplus=softplus, final=final, out=out, **more)
    want, m = plain(v, which, softplus), plain(v, which, softplus, magnitudes=True)
    e = units(v) * E32
    close(out.to_host(), np.stack(want["y"]), dtype, e * np.stack(m["y"]))
    close(final.to_host(), want["final"], np.float32, e * m["final"])
    assert frame_intact(wide, (S, T, C))


LENGTHS = [[5], [1, 1, 0, 2], [0, 0, 7], [3, 170, 0, 1, 230, 2, 0], [33, 32, 31, 64, 1, 9], [0], [4] * 40, [1, 500, 60]]


@TYPES
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda l: "-".join(map(str, l[:7])))
@pytest.mark.parametrize("C,N,G", [(16, 16, 1), (11, 5, 1), (48, 16, 3), (24, 40, 1)])
def test_packed(dt, lengths, C, N, G):
    """Sequences one behind the other, states moved on in place; rows of none hold NaN and stay as they were."""
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    v = inputs(sum(lengths) + C, lengths, C, N, G, dtype)
    which = ("D", "z", "dt_bias", "initial")
    n = sum(lengths)
    nan = lambda k: np.concatenate(v[k] + [np.full((9,) + v[k][0].shape[1:], np.nan, np.float32)])  # noqa: E731
    t = {k: put(ctx, nan(k), dtype) for k in ("x", "dt", "z", "B", "C")}
    out, state = put(ctx, np.full((n + 9, C), 5.0), dtype), put(ctx, v["initial"], np.float32)
    f32 = {k: put(ctx, v[k], np.float32) for k in ("A", "D", "dt_bias")}
    Q.device_selective_scan(t["x"], t["dt"], f32["A"], t["B"], t["C"], D=f32["D"], z=t["z"], dt_bias=f32["dt_bias"], softplus=True, initial=state,
                            final=state, sequences=Q.Sequences(ctx, lengths), out=out)
    want, m = plain(v, which, True), plain(v, which, True, magnitudes=True)
    e = units(v) * E32
    got = out.to_host()
    close(got[:n], np.concatenate(want["y"]), dtype, e * np.concatenate(m["y"]))
    assert (got[n:] == 5).all()
    close(state.to_host(), want["final"], np.float32, e * m["final"])


@TYPES
@pytest.mark.parametrize("S,C,N,G", [(1, 8, 16, 1), (3, 5, 7, 1), (65, 48, 16, 2), (2, 16, 64, 1), (2, 6, 128, 3)])
def test_steps(dt, S, C, N, G):
    """Single tokens behind a prompt's state, against the prompt with those tokens."""
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    T, cut = 9, 5
    v = inputs(S + C, [T] * S, C, N, G, dtype)
    which = ("D", "z", "dt_bias", "initial")
    want, m = plain(v, which, True), plain(v, which, True, magnitudes=True)
    e = units(v) * E32
    part = lambda k, at: put(ctx, np.stack(v[k])[:, at], dtype)  # noqa: E731
    state = put(ctx, v["initial"], np.float32)
    f32 = {k: put(ctx, v[k], np.float32) for k in ("A", "D", "dt_bias")}
    more = dict(D=f32["D"], dt_bias=f32["dt_bias"], softplus=True)
    head = slice(0, cut)
    y = Q.device_selective_scan(part("x", head), part("dt", head), f32["A"], part("B", head), part("C", head), z=part("z", head), initial=state, final=state,
                                **more)
    close(y.to_host(), np.stack(want["y"])[:, :cut], dtype, e * np.stack(m["y"])[:, :cut])
    for t in range(cut, T):
        x = part("x", t)
        y = Q.device_selective_scan_step(x, part("dt", t), f32["A"], part("B", t), part("C", t), state, z=part("z", t), out=x if t % 2 else None, **more)
        close(y.to_host(), np.stack(want["y"])[:, t], dtype, e * np.stack(m["y"])[:, t])
    close(state.to_host(), want["final"], np.float32, e * m["final"])


def test_states_without_groups_axis():
    ctx = shim.get_context(0)
    v = inputs(3, [20] * 2, 8, 16, 1, np.float32)
    args, more = on_device(ctx, v, np.dtype(np.float32), ("D",))
    a = Q.device_selective_scan(*args, softplus=True, **more).to_host()
    flat = [put(ctx, np.stack(v[k])[:, :, 0], np.float32) for k in ("B", "C")]
    assert np.array_equal(a, Q.device_selective_scan(*args[:3], *flat, softplus=True, **more).to_host())


def test_large_steps_forget_and_small_ones_keep():
    """softplus at both ends: steps of 1e-30 leave the state alone, steps of 1e4 end it at once; no overflow on the way."""
    ctx = shim.get_context(0)
    C, N = 8, 16
    x, B = np.ones((1, 4, C), np.float32), np.ones((1, 4, N), np.float32)
    A, init = np.full((C, N), -1.0, np.float32), np.full((1, C, N), 3.0, np.float32)
    final = Q.DeviceArray(ctx, (1, C, N), np.float32)
    for raw, want in ((-70.0, 3.0), (1e4, 1e4)):
        dt = np.full((1, 4, C), raw, np.float32)
        y = Q.device_selective_scan(*(put(ctx, a, np.float32) for a in (x, dt, A, B, B)), softplus=True, initial=put(ctx, init, np.float32), final=final)
        assert np.allclose(final.to_host(), want, rtol=2e-6) and np.allclose(y.to_host(), N * want, rtol=2e-6)


def test_infinities_stay_with_their_channel():
    ctx = shim.get_context(0)
    v = inputs(4, [50] * 2, 24, 16, 1, np.float32)
    args, more = on_device(ctx, v, np.dtype(np.float32), ("D", "z"))
    clean = Q.device_selective_scan(*args, softplus=True, **more).to_host()
    v["x"][0][20, 5], v["z"][1][30, 7] = np.inf, np.nan
    args, more = on_device(ctx, v, np.dtype(np.float32), ("D", "z"))
    got = Q.device_selective_scan(*args, softplus=True, **more).to_host()
    assert not np.isfinite(got[0, 20:, 5]).any() and np.isnan(got[1, 30, 7])
    got[0, 20:, 5], got[1, 30, 7] = clean[0, 20:, 5], clean[1, 30, 7]
    assert np.array_equal(got, clean)


def test_no_tokens_pass_the_state_on():
    ctx = shim.get_context(0)
    e, b = Q.DeviceArray(ctx, (2, 0, 8), np.float32), Q.DeviceArray(ctx, (2, 0, 4), np.float32)
    init = put(ctx, np.arange(64).reshape(2, 8, 4), np.float32)
    final = Q.DeviceArray(ctx, (2, 8, 4), np.float32)
    Q.device_selective_scan(e, e, put(ctx, -np.ones((8, 4)), np.float32), b, b, initial=init, final=final)
    assert np.array_equal(final.to_host(), init.to_host())
    Q.device_selective_scan(e, e, put(ctx, -np.ones((8, 4)), np.float32), b, b, final=final)
    assert (final.to_host() == 0).all()


def test_same_bits_every_time_and_in_a_graph():
    """Also for sequences that are cut into pieces, whose workspace each graph has for itself."""
    ctx = shim.get_context(0)
    v = inputs(9, [600] * 2, 48, 16, 1, np.float32)
    args, more = on_device(ctx, v, np.dtype(np.float32), ("D", "z", "dt_bias", "initial"))
    y, final = Q.DeviceArray(ctx, args[0].shape, np.float32), Q.DeviceArray(ctx, (2, 48, 16), np.float32)

    def call():
        Q.device_selective_scan(*args, softplus=True, final=final, out=y, **more)
    call()
    first = y.to_host(), final.to_host()
    graph, other = ctx.capture(call), ctx.capture(call)
    for t in (y, final):
        ctx.memset(t.ptr, 0x11, t.size * 4)
    graph.launch()
    call()
    other.launch()
    graph.launch()
    assert np.array_equal(first[0], y.to_host()) and np.array_equal(first[1], final.to_host())


def test_steps_of_more_sequences_than_a_grid_is_high():
    """65536 and more sequences: the states behind the 65535th move on as the first ones."""
    ctx = shim.get_context(0)
    S, C, N = 65540, 2, 4
    one = lambda *s: put(ctx, np.ones(s), np.float32)  # noqa: E731
    state = put(ctx, np.tile(np.arange(C * N, dtype=np.float32).reshape(1, C, N), (S, 1, 1)), np.float32)
    y = Q.device_selective_scan_step(one(S, C), one(S, C), put(ctx, -np.ones((C, N)), np.float32), one(S, N), one(S, N), state).to_host()
    h = state.to_host()
    assert (h == h[:1]).all() and (y == y[:1]).all()
    # one decay of e^-1 and a step of one: 4 roundings of 2^-24 of the value, of which exp2's 2^-22 is the largest
    assert np.abs(h[0] - (np.arange(8).reshape(C, N) * np.exp(-1) + 1)).max() < 8 * 2 ** -22
