"""The sequence operators together, as a layer of a model uses them: norm of the residual stream, causal convolution, scan."""
import threading

import numpy as np
import pytest

import sequence_plain as P
from sequence_util import DTYPES, put
from theano_b200 import sequence as Q
from theano_b200 import shim

pytestmark = pytest.mark.gpu
C, N, K, S, T, EPS = 48, 16, 4, 3, 70, 1e-5
# Three operators, each within some 300 roundings of 2^-24 of its terms' magnitudes (2e-5), and each less than five times as sensitive to its
# input as to its own roundings: 3e-4 of the largest value
TOL = 3e-4


def weights(seed=0):
    rs = np.random.RandomState(seed)
    f = lambda *s, k=1.0: (rs.standard_normal(s) * k).astype(np.float32)  # noqa: E731
    return dict(gamma=1 + f(C, k=.2), beta=f(C, k=.2), w=f(C, K, k=.5), bias=f(C, k=.2), A=-np.exp(f(C, N, k=.3)) * (1 + np.arange(N, dtype=np.float32)), D=f(C),
                dt_bias=rs.uniform(-5, -1, C).astype(np.float32))


def inputs(seed=1):
    rs = np.random.RandomState(seed)
    f = lambda *s: rs.standard_normal(s).astype(np.float32)  # noqa: E731
    return dict(x=f(S, T, C), stream=f(S, T, C) * 2, dt=f(S, T, C), z=f(S, T, C), B=f(S, T, N), C=f(S, T, N))


def plain(w, v):
    """float64: (y, new stream, conv state, scan state)"""
    total = v["x"].astype(np.float64) + v["stream"]
    n, _, _ = P.layer_norm(total, w["gamma"], w["beta"], EPS)
    u, conv = P.causal_conv(list(n), w["w"], w["bias"], True, True)
    o = P.selective_scan(u, list(v["dt"]), w["A"], list(v["B"][:, :, None]), list(v["C"][:, :, None]), w["D"], list(v["z"]), w["dt_bias"], True)
    return np.stack(o["y"]), total, conv, o["final"]


class Layer(object):
    def __init__(self, ctx, w):
        self.ctx, self.w = ctx, {k: put(ctx, a, np.float32) for k, a in w.items()}
        self.conv = Q.DeviceArray(ctx, (S, K - 1, C), np.float32)
        self.state = Q.DeviceArray(ctx, (S, C, N), np.float32)

    def prompt(self, t, keep=None):
        w = self.w
        keep = {} if keep is None else keep
        keep["total"] = Q.DeviceArray(self.ctx, t["x"].shape, np.float32)
        keep["stats"] = Q.DeviceArray(self.ctx, t["x"].shape[:-1] + (2,), np.float32)
        keep["n"] = Q.device_layer_norm(t["x"], w["gamma"], w["beta"], EPS, residual=t["stream"], total=keep["total"], stats=keep["stats"])
        keep["u"] = Q.device_causal_conv1d(keep["n"], w["w"], w["bias"], silu=True, final=self.conv)
        keep["y"] = Q.device_selective_scan(keep["u"], t["dt"], w["A"], t["B"], t["C"], D=w["D"], z=t["z"], dt_bias=w["dt_bias"], softplus=True, final=self.state)
        return keep["y"]

    def token(self, t):
        w = self.w
        n = Q.device_layer_norm(t["x"], w["gamma"], w["beta"], EPS, residual=t["stream"])
        u = Q.device_causal_conv1d_step(n, self.conv, w["w"], w["bias"], silu=True)
        return Q.device_selective_scan_step(u, t["dt"], w["A"], t["B"], t["C"], self.state, D=w["D"], z=t["z"], dt_bias=w["dt_bias"], softplus=True)


def near(got, want):
    assert np.abs(got - want).max() <= TOL * np.abs(want).max()


def test_prompt_then_tokens():
    ctx = shim.get_context(0)
    w, v = weights(), inputs()
    y, total, conv, state = plain(w, v)
    layer, cut = Layer(ctx, w), T - 6
    part = lambda at: {k: put(ctx, a[:, at], np.float32) for k, a in v.items()}  # noqa: E731
    keep = {}
    near(layer.prompt(part(slice(0, cut)), keep).to_host(), y[:, :cut])
    near(keep["total"].to_host(), total[:, :cut])
    for t in range(cut, T):
        near(layer.token(part(t)).to_host(), y[:, t])
    near(layer.conv.to_host(), conv)
    near(layer.state.to_host(), state)


def test_captured_token_loop_moves_the_states_on():
    """A graph of a token's step, replayed with new tokens in the same buffers."""
    ctx = shim.get_context(0)
    w, v = weights(), inputs()
    y, _, _, state = plain(w, v)
    layer = Layer(ctx, w)
    for t in (layer.conv, layer.state):
        ctx.memset(t.ptr, 0, t.size * 4)
    buf = {k: put(ctx, a[:, 0], np.float32) for k, a in v.items()}
    out = {}

    def step():
        out["y"] = layer.token(buf)
    step()
    for t in (layer.conv, layer.state):
        ctx.memset(t.ptr, 0, t.size * 4)
    graph = ctx.capture(step)
    got = out["y"]
    for t in range(T):
        for k in buf:
            ctx.h2d(buf[k].ptr, np.ascontiguousarray(v[k][:, t]))
        graph.launch()
        near(got.to_host(), y[:, t])
    near(layer.state.to_host(), state)


def test_training_step():
    """All gradients of the layer against the formulas' in float64."""
    ctx = shim.get_context(0)
    w, v = weights(), inputs()
    rs = np.random.RandomState(5)
    dy, dstream = (rs.standard_normal((S, T, C)).astype(np.float32) for _ in range(2))
    total = v["x"].astype(np.float64) + v["stream"]
    n, _, _ = P.layer_norm(total, w["gamma"], w["beta"], EPS)
    u, _ = P.causal_conv(list(n), w["w"], w["bias"], True, True)
    o = P.selective_scan(u, list(v["dt"]), w["A"], list(v["B"][:, :, None]), list(v["C"][:, :, None]), w["D"], list(v["z"]), w["dt_bias"], True, dys=list(dy))
    dn, dw, dbias, _ = P.causal_conv_grad(o["dx"], list(n), w["w"], w["bias"], True, True)
    dx, dgamma, dbeta = P.layer_norm_grad(np.stack(dn), total, w["gamma"], EPS)
    layer, keep = Layer(ctx, w), {}
    t, W = {k: put(ctx, a, np.float32) for k, a in v.items()}, layer.w
    layer.prompt(t, keep)
    g = Q.device_selective_scan_grad(put(ctx, dy, np.float32), keep["u"], t["dt"], W["A"], t["B"], t["C"], D=W["D"], z=t["z"], dt_bias=W["dt_bias"], softplus=True)
    gn, gw, gb, _ = Q.device_causal_conv1d_grad(g["x"], keep["n"], W["w"], W["bias"], silu=True)
    gx, gg, gbeta = Q.device_layer_norm_grad(gn, keep["total"], W["gamma"], keep["stats"], dtotal=put(ctx, dstream, np.float32))
    for got, want in ((g["dt"], np.stack(o["ddt"])), (g["B"], np.stack(o["dB"])[:, :, 0]), (g["C"], np.stack(o["dC"])[:, :, 0]), (g["z"], np.stack(o["dz"])), (g["A"], o["dA"]),
                      (g["D"], o["dD"]), (g["dt_bias"], o["ddt_bias"]), (gw, dw), (gb, dbias), (gg, dgamma), (gbeta, dbeta), (gx, dx + dstream)):
        near(got.to_host(), want)


def test_images_between_convolutions():
    """A norm between two 2-D convolutions of channels-last images, pad channels and all."""
    ctx = shim.get_context(0)
    rs = np.random.RandomState(3)
    x, w = rs.standard_normal((2, 12, 6, 6)).astype(np.float16), (rs.standard_normal((20, 12, 3, 3)) * .1).astype(np.float16)
    w2 = (rs.standard_normal((8, 20, 1, 1)) * .2).astype(np.float16)
    X, W, W2 = shim.DeviceTensor.from_host(ctx, x, "nhwc"), shim.DeviceTensor.from_host(ctx, w), shim.DeviceTensor.from_host(ctx, w2)
    mid = shim.device_conv2d(X, W, border_mode="half")
    out = shim.device_conv2d(Q.device_layer_norm(mid), W2)
    m = mid.to_host().astype(np.float64).transpose(0, 2, 3, 1)
    n = P.layer_norm(m, None, None, EPS)[0].astype(np.float16).astype(np.float64)
    want = np.einsum("nhwc,kc->nkhw", n, w2[:, :, 0, 0].astype(np.float64))
    # the normalised values rounded one way or the other (2^-11), float16 results: the repository's bound of the convolutions
    assert np.abs(out.to_host() - want).max() <= 2e-2 * np.abs(want).max()


def test_host_calls_give_the_device_calls_results():
    ctx = shim.get_context(0)
    w, v = weights(), inputs()
    D = lambda a: put(ctx, a, np.float32)  # noqa: E731
    assert np.array_equal(Q.layer_norm(v["x"], w["gamma"], w["beta"]), Q.device_layer_norm(D(v["x"]), D(w["gamma"]), D(w["beta"])).to_host())
    y, final = Q.causal_conv1d(v["x"], w["w"], w["bias"], silu=True)
    assert np.array_equal(y, Q.device_causal_conv1d(D(v["x"]), D(w["w"]), D(w["bias"]), silu=True).to_host()) and np.array_equal(final, v["x"][:, T - K + 1:])
    args = [v[k] if k in v else w[k] for k in ("x", "dt", "A", "B", "C")]
    y, final = Q.selective_scan(*args, D=w["D"], z=v["z"], dt_bias=w["dt_bias"], softplus=True)
    assert np.array_equal(y, Q.device_selective_scan(*map(D, args), D=D(w["D"]), z=D(v["z"]), dt_bias=D(w["dt_bias"]), softplus=True).to_host())
    g = Q.selective_scan_grad(v["z"], *args, D=w["D"], softplus=True)
    assert set(g) == {"x", "dt", "A", "B", "C", "D"} and g["A"].shape == w["A"].shape
    dx, dw, db, dinit = Q.causal_conv1d_grad(v["z"], v["x"], w["w"], initial=np.zeros((S, K - 1, C), np.float32))
    assert dx.shape == v["x"].shape and dw.shape == (C, K) and db is None and dinit.shape == (S, K - 1, C)
    dx, dg, db = Q.layer_norm_grad(v["z"], v["x"])
    assert dx.shape == v["x"].shape and dg.shape == db.shape == (C,) and dg.dtype == np.float32
    # packed rows, some of no sequence: zeros there
    flat = [a.reshape(S * T, -1) if a.ndim == 3 else a for a in args]
    y, final = Q.selective_scan(*flat, softplus=True, lengths=[5, 100, 0, 60])
    assert (y[165:] == 0).all() and (final[2] == 0).all() and np.isfinite(y).all()
    assert (Q.causal_conv1d(flat[0], w["w"], lengths=[200])[0][200:] == 0).all()


def test_two_contexts_at_once():
    """Threads with a context each: streams, pools and plans do not disturb each other."""
    w, v = weights(), inputs()
    want, errors = plain(w, v)[0], []

    def work():
        try:
            ctx = shim.Context(0)
            layer = Layer(ctx, w)
            t = {k: put(ctx, a, np.float32) for k, a in v.items()}
            for _ in range(20):
                near(layer.prompt(t).to_host(), want)
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=work) for _ in range(3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors


def test_one_context_from_several_threads():
    ctx = shim.get_context(0)
    w, v = weights(), inputs()
    want, errors = plain(w, v)[0], []

    def work():
        try:
            layer = Layer(ctx, w)
            t = {k: put(ctx, a, np.float32) for k, a in v.items()}
            for _ in range(10):
                near(layer.prompt(t).to_host(), want)
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=work) for _ in range(3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors


@pytest.mark.parametrize("dt", list(DTYPES))
def test_wrong_offsets_stay_inside_of_the_tensors(dt):
    """Device offsets that decrease or lie outside: wrong results, no access outside (the neighbours keep their values)."""
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    rows, ch = 40, 16
    ones = lambda *s: put(ctx, np.ones(s), dtype)  # noqa: E731
    frame = put(ctx, np.full((rows + 8, ch), 7.0), dtype)
    out = frame[4:4 + rows]
    for starts in ([0, 100, 30, 40], [-5, 10, 20, 1000], [50, 60, 70, 80], [40, 30, 20, 10], [0, 0, 0, 0]):
        seqs = Q.Sequences(ctx, [10, 10, 20])
        ctx.h2d(seqs.starts.ptr, np.array(starts, np.int32))
        ctx.sync()
        state = put(ctx, np.zeros((3, ch, 16)), np.float32)
        Q.device_causal_conv1d(ones(rows, ch), ones(ch, 4), silu=True, sequences=seqs, out=out)
        Q.device_selective_scan(ones(rows, ch), ones(rows, ch), put(ctx, -np.ones((ch, 16)), np.float32), ones(rows, 16), ones(rows, 16), softplus=True,
                                initial=state, final=state, sequences=seqs, out=out)
        Q.device_causal_conv1d_grad(ones(rows, ch), ones(rows, ch), ones(ch, 4), silu=True, sequences=seqs, out=out)
        Q.device_selective_scan_grad(ones(rows, ch), ones(rows, ch), ones(rows, ch), put(ctx, -np.ones((ch, 16)), np.float32), ones(rows, 16), ones(rows, 16),
                                     softplus=True, sequences=seqs, grads=dict(x=out))
    a = frame.to_host()
    assert (a[:4] == 7).all() and (a[4 + rows:] == 7).all()
