"""Gradients of the selective scan against float64 and against differences."""
import numpy as np
import pytest

import sequence_plain as P
from sequence_util import DTYPES, E32, close, frame_intact, framed, normal, put
from test_gpu_selective_scan import LENGTHS, SHAPES, inputs, plain, units
from theano_b200 import sequence as Q
from theano_b200 import shim

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dt", list(DTYPES))
ALL = ("D", "z", "dt_bias", "initial")


def sums(v):
    """Units of 2^-24 for a gradient: a path through the tokens and back, and sums over tokens and channels."""
    return 2 * units(v) + sum(len(x) for x in v["x"]) + v["A"].shape[0] / 4


def check(v, which, softplus, dys, dfinal, got, dtype, n=None):
    want = plain(v, which, softplus, dys=dys, dfinals=dfinal)
    m = plain(v, which, softplus, dys=dys, dfinals=dfinal, magnitudes=True)
    e = sums(v) * E32
    for name in ("x", "dt", "z", "B", "C"):
        if name == "z" and "z" not in which:
            assert "z" not in got
            continue
        a = got[name].to_host()
        join = np.stack if n is None else np.concatenate
        close(a if n is None else a[:n], join(want["d" + name]), dtype, e * join(m["d" + name]))
        assert n is None or (a[n:] == 5).all()
    for name in ("A", "D", "dt_bias", "initial"):
        if name == "A" or name in which:
            close(got[name].to_host(), want["d" + name], np.float32, e * m["d" + name])


@TYPES
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("which,softplus", [(ALL, True), ((), True), (("D", "initial"), False)], ids=["all", "none", "raw"])
def test_gradients(dt, shape, which, softplus):
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    S, T, C, N, G = shape
    v = inputs(C + N + 1, [T] * S, C, N, G, dtype)
    if not softplus:
        v["dt"] = [np.abs(d) for d in v["dt"]]
    rs = np.random.RandomState(7)
    dys = [normal(rs, (T, C), dtype) for _ in range(S)]
    dfinal = rs.standard_normal((S, C, N)).astype(np.float32) if "initial" in which else None
    dev = lambda k: put(ctx, np.stack(v[k]), dtype)  # noqa: E731
    f32 = lambda a: None if a is None else put(ctx, a, np.float32)  # noqa: E731
    more = {k: f32(v[k]) for k in ("D", "dt_bias", "initial") if k in which}
    if "z" in which:
        more["z"] = dev("z")
    wide, out = framed(ctx, (S, T, C), dtype)
    got = Q.device_selective_scan_grad(put(ctx, np.stack(dys), dtype), dev("x"), dev("dt"), f32(v["A"]), dev("B"), dev("C"), softplus=softplus,
                                       dfinal=f32(dfinal), grads=dict(x=out), **more)
    check(v, which, softplus, dys, dfinal, got, dtype)
    assert frame_intact(wide, (S, T, C))


@TYPES
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda l: "-".join(map(str, l[:7])))
@pytest.mark.parametrize("C,N,G", [(16, 16, 1), (11, 5, 1), (48, 16, 3), (24, 40, 1)])
def test_packed(dt, lengths, C, N, G):
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    v = inputs(sum(lengths) + C + 1, lengths, C, N, G, dtype)
    rs, n = np.random.RandomState(8), sum(lengths)
    dys = [normal(rs, (k, C), dtype) for k in lengths]
    dfinal = rs.standard_normal(v["initial"].shape).astype(np.float32)
    nan = lambda parts: put(ctx, np.concatenate(parts + [np.full((9,) + parts[0].shape[1:], np.nan, np.float32)]), dtype)  # noqa: E731
    t = {k: nan(v[k]) for k in ("x", "dt", "z", "B", "C")}
    f32 = {k: put(ctx, v[k], np.float32) for k in ("A", "D", "dt_bias", "initial")}
    grads = {k: put(ctx, np.full(t[k].shape, 5.0), dtype) for k in t}
    passed = put(ctx, dfinal, np.float32)              # the states' gradients pass through one array
    grads["initial"] = passed
    got = Q.device_selective_scan_grad(nan(dys), t["x"], t["dt"], f32["A"], t["B"], t["C"], D=f32["D"], z=t["z"], dt_bias=f32["dt_bias"], softplus=True,
                                       initial=f32["initial"], dfinal=passed, sequences=Q.Sequences(ctx, lengths), grads=grads)
    check(v, ALL, True, dys, dfinal, got, dtype, n)


def test_against_differences():
    ctx = shim.get_context(0)
    v = inputs(5, [6, 6], 4, 3, 2, np.dtype(np.float32), decay=0.5)
    rs = np.random.RandomState(6)
    dys, dfinal = [rs.standard_normal((6, 4)) for _ in range(2)], rs.standard_normal((2, 4, 3))

    def loss(v):
        o = plain(v, ALL, True)
        return sum((a * b).sum() for a, b in zip(o["y"], dys)) + (o["final"] * dfinal).sum()
    dev = lambda k: put(ctx, np.stack(v[k]), np.float32)  # noqa: E731
    f32 = {k: put(ctx, v[k], np.float32) for k in ("A", "D", "dt_bias", "initial")}
    got = Q.device_selective_scan_grad(put(ctx, np.stack(dys), np.float32), dev("x"), dev("dt"), f32["A"], dev("B"), dev("C"), D=f32["D"], z=dev("z"),
                                       dt_bias=f32["dt_bias"], softplus=True, initial=f32["initial"], dfinal=put(ctx, dfinal, np.float32))
    h = 1e-4
    for name, g in got.items():
        g = g.to_host()
        value = np.stack(v[name]) if isinstance(v[name], list) else v[name]
        for _ in range(4):
            at = np.unravel_index(rs.randint(value.size), value.shape)
            ends = []
            for sign in (1, -1):
                moved = value.astype(np.float64)
                moved[at] += sign * h
                ends.append(loss({**v, name: list(moved) if isinstance(v[name], list) else moved}))
            # central differences: h^2 / 6 of a third derivative of order 100, and float32 gradients
            assert abs((ends[0] - ends[1]) / (2 * h) - g[at]) < 2e-5 * max(1.0, np.abs(g).max()), name


def test_no_tokens():
    ctx = shim.get_context(0)
    e, b = Q.DeviceArray(ctx, (2, 0, 8), np.float32), Q.DeviceArray(ctx, (2, 0, 4), np.float32)
    A, init = put(ctx, -np.ones((8, 4)), np.float32), put(ctx, np.ones((2, 8, 4)), np.float32)
    dfinal = put(ctx, np.arange(64).reshape(2, 8, 4), np.float32)
    got = Q.device_selective_scan_grad(e, e, e, A, b, b, initial=init, dfinal=dfinal)
    assert np.array_equal(got["initial"].to_host(), dfinal.to_host()) and (got["A"].to_host() == 0).all()


def test_same_bits_every_time_and_in_a_graph():
    ctx = shim.get_context(0)
    v = inputs(9, [400] * 2, 48, 16, 1, np.dtype(np.float32))
    rs = np.random.RandomState(1)
    dev = lambda k: put(ctx, np.stack(v[k]), np.float32)  # noqa: E731
    f32 = {k: put(ctx, v[k], np.float32) for k in ("A", "D", "dt_bias", "initial")}
    args = (put(ctx, rs.standard_normal((2, 400, 48)), np.float32), dev("x"), dev("dt"), f32["A"], dev("B"), dev("C"))
    more = dict(D=f32["D"], z=dev("z"), dt_bias=f32["dt_bias"], softplus=True, initial=f32["initial"])
    grads = Q.device_selective_scan_grad(*args, **more)
    call = lambda: Q.device_selective_scan_grad(*args, grads=grads, **more)  # noqa: E731
    first = {k: t.to_host() for k, t in grads.items()}
    graph, other = ctx.capture(call), ctx.capture(call)
    for t in grads.values():
        ctx.memset(t.ptr, 0x11, t.size * 4)
    graph.launch()
    call()
    other.launch()
    graph.launch()
    assert all(np.array_equal(first[k], t.to_host()) for k, t in grads.items())


@pytest.mark.parametrize("T", [8, 300])
@pytest.mark.parametrize("C,N,G", [(48, 16, 3), (10, 40, 1), (4, 16, 1)])
def test_nothing_of_an_earlier_call_is_left(T, C, N, G):
    """Blocks with fewer channels than lanes, behind calls that filled every SM's shared memory with NaN: the sums over channels
    hold nothing of what lies there."""
    ctx = shim.get_context(0)
    f32 = np.dtype(np.float32)
    v = inputs(3, [T] * 2, C, N, G, f32)
    dev = lambda k: put(ctx, np.stack(v[k]), f32)  # noqa: E731
    args = (dev("x"), dev("x"), dev("dt"), put(ctx, v["A"], f32), dev("B"), dev("C"))
    want = plain(v, (), True, dys=v["x"])
    m = plain(v, (), True, dys=v["x"], magnitudes=True)
    nan = lambda *s: put(ctx, np.full(s, np.nan), f32)  # noqa: E731
    wide = (nan(300, 16, 128), nan(300, 16, 128), nan(300, 16, 128), nan(128, 16), nan(300, 16, 16), nan(300, 16, 16))
    for _ in range(3):
        Q.device_selective_scan(*wide[1:], softplus=True)
        Q.device_selective_scan_grad(*wide, softplus=True)
        got = Q.device_selective_scan_grad(*args, softplus=True)
        for k in ("x", "dt", "B", "C"):
            close(got[k].to_host(), np.stack(want["d" + k]), f32, sums(v) * E32 * np.stack(m["d" + k]))
        close(got["A"].to_host(), want["dA"], f32, sums(v) * E32 * m["dA"])
