"""The short causal convolution: prompts, packed prompts, single tokens and gradients, against float64."""
import numpy as np
import pytest

import sequence_plain as P
from sequence_util import DTYPES, E32, close, frame_intact, framed, normal, put, rounded
from theano_b200 import sequence as Q
from theano_b200 import shim

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dt", list(DTYPES))
# (sequences, tokens, channels, taps): shorter than the taps, one token, ends inside of a run, odd channels, many channel blocks
SHAPES = [(1, 1, 8, 4), (2, 2, 16, 4), (3, 3, 5, 4), (2, 17, 24, 2), (1, 65, 40, 3), (2, 131, 33, 4), (1, 40, 1032, 4), (2, 37, 16, 5), (1, 9, 8, 6),
          (2, 50, 8, 7), (1, 77, 72, 8), (5, 300, 64, 4)]


def magnitude(xs, w, bias, inits):
    """sum over k of |w[k] x[t - k]| + |bias|, per sequence."""
    return P.causal_conv([np.abs(x) for x in xs], np.abs(w), None if bias is None else np.abs(bias), False, True,
                         None if inits is None else [np.abs(i) for i in inits])[0]


def forward_slack(xs, w, bias, silu, flip, inits):
    ww = w if flip else w[:, ::-1]
    pres = P.causal_conv(xs, ww, bias, False, True, inits)[0]
    out = []
    for pre, m in zip(pres, magnitude(xs, ww, bias, inits)):
        s = (w.shape[1] + 2) * E32 * m
        # silu's slope is below 1.1; exp of v and the quotient are off by some 2^-24 (|v| + 10) of the result
        out.append(1.1 * s + (np.abs(pre) + 10) * E32 * np.abs(pre) if silu else s)
    return out


def gradient_slack(dys, xs, w, bias, silu, flip, inits):
    """(dx, dw, dbias, dinitial) slacks: each g is off by dy (slope's change with pre, and its own evaluation)."""
    ww = (w if flip else w[:, ::-1]).astype(np.float64)
    gs, mags = [], magnitude(xs, ww, bias, inits)
    for dy, m in zip(dys, mags):
        gs.append(np.abs(dy) * ((0.5 * (w.shape[1] + 2) * E32 * m + 24 * E32) if silu else 0 * m) + 2 * E32 * np.abs(dy))
    n = sum(len(x) for x in xs) + 60
    lin = lambda g: P.causal_conv_grad(g, [np.abs(x) for x in xs], np.abs(ww), None, False, True, None if inits is None else [np.abs(i) for i in inits])  # noqa: E731
    own, sums = lin(gs), lin([1.1 * np.abs(d) for d in dys])
    dx = [a + (w.shape[1] + 2) * E32 * b for a, b in zip(own[0], sums[0])]
    dw = own[1] + n * E32 * sums[1]
    return dx, dw if flip else dw[:, ::-1], own[2] + n * E32 * sums[2], own[3] + (w.shape[1] + 2) * E32 * sums[3]


def inputs(rs, S, T, C, K, dtype):
    return (normal(rs, (S, T, C), dtype), normal(rs, (C, K), dtype, K ** -0.5), normal(rs, (C,), dtype, 0.3), normal(rs, (S, K - 1, C), dtype))


@TYPES
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("silu,flip,more", [(True, True, True), (False, False, True), (True, False, False)])
def test_prompts(dt, shape, silu, flip, more):
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    S, T, C, K = shape
    x, w, b, init = inputs(np.random.RandomState(C + K), S, T, C, K, dtype)
    if not more:
        b = init = None
    wide, out = framed(ctx, x.shape, dtype)
    _, xin = framed(ctx, x.shape, dtype, value=x)
    final = Q.DeviceArray(ctx, (S, K - 1, C), dtype)
    dev = lambda a: None if a is None else put(ctx, a, dtype)  # noqa: E731
    Q.device_causal_conv1d(xin, dev(w), dev(b), silu=silu, filter_flip=flip, initial=dev(init), final=final, out=out)
    ys, fin = P.causal_conv(list(x), w, b, silu, flip, init)
    close(out.to_host(), np.stack(ys), dtype, np.stack(forward_slack(list(x), w, b, silu, flip, init)))
    assert np.array_equal(final.to_host(), fin)
    assert frame_intact(wide, x.shape)
    # the same bits from tensors without gaps
    assert np.array_equal(Q.device_causal_conv1d(dev(x), dev(w), dev(b), silu=silu, filter_flip=flip, initial=dev(init)).to_host(), out.to_host())


@TYPES
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("silu,flip,f32_params", [(True, True, False), (False, False, False), (True, False, True)])
def test_gradients(dt, shape, silu, flip, f32_params):
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    ptype = DTYPES["f32"] if f32_params else dtype
    S, T, C, K = shape
    rs = np.random.RandomState(C + K + 1)
    x, w, b, init = inputs(rs, S, T, C, K, dtype)
    dy = normal(rs, x.shape, dtype)
    wide, out = framed(ctx, x.shape, dtype)
    dinit = Q.DeviceArray(ctx, init.shape, dtype)
    _, dw, db, _ = Q.device_causal_conv1d_grad(put(ctx, dy, dtype), put(ctx, x, dtype), put(ctx, w, ptype), put(ctx, b, ptype), silu=silu, filter_flip=flip,
                                               initial=put(ctx, init, dtype), out=out, dinitial=dinit)
    want = P.causal_conv_grad(list(dy), list(x), w, b, silu, flip, init)
    slack = gradient_slack(list(dy), list(x), w, b, silu, flip, init)
    close(out.to_host(), np.stack(want[0]), dtype, np.stack(slack[0]))
    close(dw.to_host(), want[1], ptype, slack[1])
    close(db.to_host(), want[2], ptype, slack[2])
    close(dinit.to_host(), want[3], dtype, slack[3])
    assert frame_intact(wide, x.shape)


def packed(xs, tail, C):
    return np.concatenate([x for x in xs] + [np.full((tail, C), np.nan, np.float32)])


LENGTHS = [[5], [1, 1, 1, 0, 2], [0, 0, 7], [3, 70, 0, 1, 130, 2, 0], [33, 32, 31, 64, 1, 9], [0], [4] * 40]


@TYPES
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("C,K", [(16, 4), (11, 3), (520, 4), (8, 8)])
def test_packed(dt, lengths, C, K):
    """Sequences one behind the other; rows of none are left as they were, whatever they hold."""
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    rs = np.random.RandomState(sum(lengths) + C)
    xs, dys = ([normal(rs, (n, C), dtype) for n in lengths] for _ in range(2))
    _, w, b, _ = inputs(rs, 1, 1, C, K, dtype)
    init = normal(rs, (len(lengths), K - 1, C), dtype)
    X = put(ctx, packed(xs, 9, C), dtype)
    seqs = Q.Sequences(ctx, lengths)
    n = sum(lengths)
    out, dx = put(ctx, np.full((n + 9, C), 5.0), dtype), put(ctx, np.full((n + 9, C), 5.0), dtype)
    state = put(ctx, init, dtype)                      # moved on in place
    W, B, I = put(ctx, w, dtype), put(ctx, b, dtype), put(ctx, init, dtype)
    Q.device_causal_conv1d(X, W, B, silu=True, initial=state, final=state, sequences=seqs, out=out)
    ys, fin = P.causal_conv(xs, w, b, True, True, init)
    got = out.to_host()
    close(got[:n], np.concatenate(ys), dtype, np.concatenate(forward_slack(xs, w, b, True, True, init)))
    assert (got[n:] == 5).all() and np.array_equal(state.to_host(), fin)
    dinit = Q.DeviceArray(ctx, init.shape, dtype)
    _, dw, db, _ = Q.device_causal_conv1d_grad(put(ctx, packed(dys, 9, C), dtype), X, W, B, silu=True, initial=I, sequences=seqs, out=dx, dinitial=dinit)
    want = P.causal_conv_grad(dys, xs, w, b, True, True, init)
    slack = gradient_slack(dys, xs, w, b, True, True, init)
    got = dx.to_host()
    close(got[:n], np.concatenate(want[0]), dtype, np.concatenate(slack[0]))
    assert (got[n:] == 5).all()
    for a, b_, s in zip((dw, db, dinit), want[1:], slack[1:]):
        close(a.to_host(), b_, dtype, s)


@TYPES
@pytest.mark.parametrize("S,C,K", [(1, 8, 4), (3, 5, 2), (64, 136, 4), (2, 16, 8), (300, 33, 3)])
def test_steps_follow_a_prompt(dt, S, C, K):
    """Tokens one by one behind a prompt's state give the bits of the whole prompt."""
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    x, w, b, init = inputs(np.random.RandomState(S), S, 9, C, K, dtype)
    W, B = put(ctx, w, dtype), put(ctx, b, dtype)
    whole = Q.device_causal_conv1d(put(ctx, x, dtype), W, B, silu=True, initial=put(ctx, init, dtype)).to_host()
    state = put(ctx, init, dtype)
    first = Q.device_causal_conv1d(put(ctx, x[:, :4], dtype), W, B, silu=True, initial=state, final=state).to_host()
    assert np.array_equal(first, whole[:, :4])
    for t in range(4, 9):
        tok = put(ctx, x[:, t], dtype)
        y = Q.device_causal_conv1d_step(tok, state, W, B, silu=True, out=tok if t % 2 else None)
        assert np.array_equal(y.to_host(), whole[:, t])
    assert np.array_equal(state.to_host(), P.causal_conv(list(x), w, b, True, True, init)[1])


def test_image_rows_and_their_pads():
    """A channels-last image of one row of pixels; the pad channels of results are zeros."""
    ctx = shim.get_context(0)
    rs = np.random.RandomState(2)
    img, w = rs.standard_normal((2, 11, 1, 30)).astype(np.float16), rs.standard_normal((11, 4)).astype(np.float16)
    t = shim.DeviceTensor.from_host(ctx, img, "nhwc")
    out = Q.device_causal_conv1d(t, put(ctx, w, np.float16))
    rows = img[:, :, 0].transpose(0, 2, 1).astype(np.float32)
    ys, _ = P.causal_conv(list(rows), w.astype(np.float32), None, False, True)
    close(out.to_host()[:, :, 0].transpose(0, 2, 1), np.stack(ys), np.float16, np.stack(forward_slack(list(rows), w.astype(np.float32), None, False, True, None)))
    dx, _, _, _ = Q.device_causal_conv1d_grad(t, t, put(ctx, w, np.float16))
    for r in (out, dx):
        raw = np.empty((2, 30, r.stored_channels), np.float16)
        ctx.d2h(raw, r.ptr)
        ctx.sync()
        assert (raw[..., 11:] == 0).all()


def test_gradient_against_differences():
    ctx = shim.get_context(0)
    rs = np.random.RandomState(8)
    x, w, b, init, dy = (rs.standard_normal(s) for s in ((2, 7, 6), (6, 4), (6,), (2, 3, 6), (2, 7, 6)))
    f = lambda x, w, b, i: sum((y * d).sum() for y, d in zip(P.causal_conv(list(x), w, b, True, True, i)[0], dy))  # noqa: E731
    dinit = Q.DeviceArray(ctx, init.shape, np.float32)
    X, W, B, I, DY = (put(ctx, v, np.float32) for v in (x, w, b, init, dy))
    got = [t.to_host() for t in Q.device_causal_conv1d_grad(DY, X, W, B, silu=True, initial=I, dinitial=dinit)]
    h = 1e-5
    for which, value in enumerate((x, w, b, init)):
        for _ in range(3):
            at = np.unravel_index(rs.randint(value.size), value.shape)
            args = [x.copy(), w.copy(), b.copy(), init.copy()]
            args[which][at] += h
            up = f(*args)
            args[which][at] -= 2 * h
            assert abs((up - f(*args)) / (2 * h) - got[which][at]) < 1e-4 * max(1.0, np.abs(got[which]).max())


def test_infinities_reach_the_windows_that_hold_them():
    """... and nothing else: an infinite token of one sequence, of another channel, behind the last sequence."""
    ctx = shim.get_context(0)
    rs = np.random.RandomState(4)
    x, w = rs.standard_normal((20, 16)).astype(np.float32), rs.standard_normal((16, 4)).astype(np.float32)
    seqs = Q.Sequences(ctx, [8, 9])
    clean = Q.device_causal_conv1d(put(ctx, x, np.float32), put(ctx, w, np.float32), sequences=seqs).to_host()
    x[7, 3], x[17:] = np.inf, np.nan
    got = Q.device_causal_conv1d(put(ctx, x, np.float32), put(ctx, w, np.float32), sequences=seqs).to_host()
    clean[7, 3] = got[7, 3]
    assert np.isinf(got[7, 3]) and np.array_equal(got[:17], clean[:17])


def test_no_tokens():
    ctx = shim.get_context(0)
    w, init = put(ctx, np.ones((8, 4)), np.float32), put(ctx, np.arange(48).reshape(2, 3, 8), np.float32)
    e, final = Q.DeviceArray(ctx, (2, 0, 8), np.float32), Q.DeviceArray(ctx, (2, 3, 8), np.float32)
    Q.device_causal_conv1d(e, w, initial=init, final=final)
    assert np.array_equal(final.to_host(), init.to_host())
    dinit = Q.DeviceArray(ctx, (2, 3, 8), np.float32)
    _, dw, _, _ = Q.device_causal_conv1d_grad(e, e, w, initial=init, dinitial=dinit)
    assert (dw.to_host() == 0).all() and (dinit.to_host() == 0).all()


def test_same_bits_every_time_and_in_a_graph():
    ctx = shim.get_context(0)
    rs = np.random.RandomState(1)
    x, dy, w, b = (put(ctx, rs.standard_normal(s), np.float16) for s in ((3, 400, 128), (3, 400, 128), (128, 4), (128,)))
    y, dx, dw, db = (Q.DeviceArray(ctx, t.shape, np.float16) for t in (x, x, w, b))

    def both():
        Q.device_causal_conv1d(x, w, b, silu=True, out=y)
        Q.device_causal_conv1d_grad(dy, x, w, b, silu=True, out=dx, dw=dw, dbias=db)
    both()
    first = [t.to_host() for t in (y, dx, dw, db)]
    graph, other = ctx.capture(both), ctx.capture(both)
    for t in (y, dx, dw, db):
        ctx.memset(t.ptr, 0x11, t.size * 2)
    graph.launch()
    both()
    other.launch()
    graph.launch()
    assert all(np.array_equal(a, t.to_host()) for a, t in zip(first, (y, dx, dw, db)))
