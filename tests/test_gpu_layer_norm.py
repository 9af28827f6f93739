"""Layer norm, forward and backward, against float64."""
import numpy as np
import pytest

import sequence_plain as P
from sequence_util import DTYPES, E32, HALF, close, frame_intact, framed, normal, put, rounded
from theano_b200 import sequence as Q
from theano_b200 import shim

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dt", list(DTYPES))
EPS = 1e-5
# channel counts on both sides of each kernel form: a warp, a quarter block, a block, a block of 512, rows beyond registers
SHAPES = [(1, 1, 1), (1, 1, 8), (2, 3, 7), (1, 5, 256), (3, 2, 264), (2, 2, 1000), (1, 3, 1001), (1, 2, 2056), (2, 2, 4104), (1, 2, 5000), (1, 2, 16392), (1, 3, 20001)]


def sums_slack(C):
    """Roundings on the way of one sum over a row: at most 40 terms per thread, or a row's 512th, and 30 levels above."""
    return (30 + max(40, C / 512)) * E32


def check_forward(x, gamma, beta, dtype, y, stats, eps=EPS):
    want, mean, rstd = P.layer_norm(x, gamma, beta, eps)
    C = x.shape[-1]
    x64 = x.astype(np.float64)
    e = sums_slack(C)
    d_mean = e * np.abs(x64).mean(-1)
    # rstd moves by half of the variance's relative error: the sum of squares, and differences that the mean's error shifts
    d_rstd = rstd * (e + d_mean ** 2 * rstd ** 2 + 4 * E32)
    g = np.abs(gamma) if gamma is not None else np.ones(C)
    b = np.abs(beta) if beta is not None else np.zeros(C)
    dist = np.abs(x64 - mean[..., None])
    slack = g * ((d_mean[..., None] + E32 * (dist + np.abs(mean)[..., None])) * rstd[..., None] + dist * d_rstd[..., None]) + 4 * E32 * (g * dist * rstd[..., None] + b)
    close(y, want, dtype, slack)
    if stats is not None:
        close(stats[..., 0], mean, np.float32, d_mean)
        close(stats[..., 1], rstd, np.float32, d_rstd)
    return mean, rstd


@TYPES
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("residual", [False, True])
def test_forward(dt, shape, residual):
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    rs = np.random.RandomState(shape[-1])
    x = normal(rs, shape, dtype) + 0
    x[0, 0] += rounded(20, dtype)                      # a row far from zero
    x = rounded(x, dtype)
    r = normal(rs, shape, dtype, 2.0) if residual else None
    gamma, beta = normal(rs, shape[-1:], dtype), normal(rs, shape[-1:], dtype)
    stats = Q.DeviceArray(ctx, shape[:2] + (2,), np.float32)
    total = Q.DeviceArray(ctx, shape, dtype) if residual else None
    wide, out = framed(ctx, shape, dtype)
    Q.device_layer_norm(put(ctx, x, dtype), put(ctx, gamma, dtype), put(ctx, beta, dtype), EPS, residual=put(ctx, r, dtype) if residual else None,
                        total=total, stats=stats, out=out)
    t = x
    if residual:
        t = rounded(x + r, dtype)
        assert np.array_equal(total.to_host(), t)
    check_forward(t, gamma, beta, dtype, out.to_host(), stats.to_host())
    assert frame_intact(wide, shape)


@TYPES
@pytest.mark.parametrize("shape", SHAPES + [(2, 700, 40), (1, 331, 1024)], ids=str)
@pytest.mark.parametrize("f32_params", [False, True])
def test_backward(dt, shape, f32_params):
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    rs = np.random.RandomState(shape[-1] + 1)
    ptype = DTYPES["f32"] if f32_params else dtype
    C, rows = shape[-1], shape[0] * shape[1]
    x = normal(rs, shape, dtype)
    dy, extra = normal(rs, shape, dtype), normal(rs, shape, dtype)
    gamma = normal(rs, (C,), ptype)
    X, G = put(ctx, x, dtype), put(ctx, gamma, ptype)
    stats = Q.DeviceArray(ctx, shape[:2] + (2,), np.float32)
    Q.device_layer_norm(X, G, None, EPS, stats=stats)
    wide, out = framed(ctx, shape, dtype)
    dx, dg, db = Q.device_layer_norm_grad(put(ctx, dy, dtype), X, G, stats, dtotal=put(ctx, extra, dtype), out=out)
    want, wg, wb = P.layer_norm_grad(dy, x, gamma, EPS)
    _, mean, rstd = P.layer_norm(x, None, None, EPS)
    hat = np.abs((x.astype(np.float64) - mean[..., None]) * rstd[..., None])
    e = sums_slack(C)
    # of the normalised values: the mean's error on the scale of the row, rstd's relative one
    d_hat = (e * np.abs(x).mean(-1) * rstd)[..., None] + hat * (2 * e + 8 * E32) + 2 * E32 * (np.abs(x) + np.abs(mean)[..., None]) * rstd[..., None]
    g = np.abs(dy * gamma).astype(np.float64)
    m0, m1 = g.mean(-1, keepdims=True), (g * hat).mean(-1, keepdims=True)
    slack = rstd[..., None] * ((e + 8 * E32) * (g + m0 + 2 * hat * m1) + hat * (g * d_hat).mean(-1, keepdims=True) + d_hat * m1) + 4 * E32 * np.abs(extra)
    close(out.to_host(), want + extra, dtype, slack)
    assert frame_intact(wide, shape)
    n = (rows + 60) * E32                              # more than any thread adds one after the other
    close(dg.to_host(), wg, ptype, (n * np.abs(dy) * hat + np.abs(dy) * d_hat).sum((0, 1)))
    close(db.to_host(), wb, ptype, (n * np.abs(dy)).sum((0, 1)))


def test_gradient_against_differences():
    ctx = shim.get_context(0)
    rs = np.random.RandomState(3)
    x, gamma, beta = rs.standard_normal((2, 3, 24)), rs.standard_normal(24), rs.standard_normal(24)
    dy = rs.standard_normal(x.shape)
    f = lambda x, g, b: (P.layer_norm(x, g, b, EPS)[0] * dy).sum()  # noqa: E731
    stats = Q.DeviceArray(ctx, (2, 3, 2), np.float32)
    X, G, B = (put(ctx, v, np.float32) for v in (x, gamma, beta))
    Q.device_layer_norm(X, G, B, EPS, stats=stats)
    got = [t.to_host() for t in Q.device_layer_norm_grad(put(ctx, dy, np.float32), X, G, stats)]
    h = 1e-5
    for which, value in enumerate((x, gamma, beta)):
        at = np.unravel_index(rs.randint(value.size), value.shape)
        for sign in (1,):
            args = [x.copy(), gamma.copy(), beta.copy()]
            args[which][at] += h
            up = f(*args)
            args[which][at] -= 2 * h
            down = f(*args)
            # differences of a function of order 30 in float64 over 2e-5, and float32 inputs: 1e-4 of the gradients' scale
            assert abs((up - down) / (2 * h) - got[which][at]) < 1e-4 * max(1.0, np.abs(got[which]).max())


@TYPES
def test_images_strides_and_in_place(dt):
    """A channels-last image is a tensor of rows whose pad channels stay zero; views with gaps; results over inputs."""
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    rs = np.random.RandomState(5)
    if dt != "bf16":
        img = rs.standard_normal((2, 13, 3, 5)).astype(dtype)
        t = shim.DeviceTensor.from_host(ctx, img, "nhwc")
        out = Q.device_layer_norm(t)
        rows = img.transpose(0, 2, 3, 1).reshape(2, 15, 13).astype(np.float32)
        got = out.to_host().transpose(0, 2, 3, 1).reshape(2, 15, 13)
        check_forward(rows, None, None, dtype, got, None)
        raw = np.empty((2, 15, out.stored_channels), dtype)
        ctx.d2h(raw, out.ptr)
        ctx.sync()
        assert (raw[..., 13:] == 0).all()
    x = normal(rs, (3, 9, 64), dtype)
    X = put(ctx, x, dtype)
    Q.device_layer_norm(X, out=X)
    check_forward(x, None, None, dtype, X.to_host(), None)
    # tokens first: the sequences interleave
    Y = put(ctx, x.transpose(1, 0, 2), dtype)
    turned = Q.DeviceArray(ctx, (3, 9, 64), dtype, (64, 192, 1), Y.ptr)
    a, b = Q.device_layer_norm(turned).to_host(), Q.device_layer_norm(put(ctx, x, dtype)).to_host()
    assert np.array_equal(a, b)
    # the sum over its own first operand
    r = normal(rs, x.shape, dtype)
    X, R = put(ctx, x, dtype), put(ctx, r, dtype)
    y = Q.device_layer_norm(X, residual=R, total=X)
    assert np.array_equal(X.to_host(), rounded(x + r, dtype))
    check_forward(rounded(x + r, dtype), None, None, dtype, y.to_host(), None)


def test_infinities_stay_in_their_row():
    ctx = shim.get_context(0)
    x = np.random.RandomState(0).standard_normal((1, 4, 300)).astype(np.float32)
    clean = Q.device_layer_norm(put(ctx, x, np.float32)).to_host()
    x[0, 1, 7], x[0, 2, 9] = np.inf, np.nan
    y = Q.device_layer_norm(put(ctx, x, np.float32)).to_host()
    assert np.isnan(y[0, 1:3]).all() and np.array_equal(y[0, ::3], clean[0, ::3])


def test_constant_rows_and_no_rows():
    ctx = shim.get_context(0)
    y = Q.device_layer_norm(put(ctx, np.full((1, 2, 96), 3.0), np.float32), None, put(ctx, np.arange(96), np.float32)).to_host()
    assert np.array_equal(y[0, 0], np.arange(96, dtype=np.float32))
    e = Q.DeviceArray(ctx, (0, 4, 16), np.float32)
    assert Q.device_layer_norm(e).to_host().shape == (0, 4, 16)
    stats = Q.DeviceArray(ctx, (0, 4, 2), np.float32)
    _, dg, db = Q.device_layer_norm_grad(e, e, None, stats)
    assert (dg.to_host() == 0).all() and (db.to_host() == 0).all()


def test_same_bits_every_time_and_in_a_graph():
    ctx = shim.get_context(0)
    rs = np.random.RandomState(1)
    x, dy, gamma = (put(ctx, rs.standard_normal(s), np.float16) for s in ((4, 300, 512), (4, 300, 512), (512,)))
    stats, y = Q.DeviceArray(ctx, (4, 300, 2), np.float32), Q.DeviceArray(ctx, x.shape, np.float16)
    outs = [Q.DeviceArray(ctx, s, np.float16) for s in (x.shape, (512,), (512,))]

    def both():
        Q.device_layer_norm(x, gamma, None, EPS, stats=stats, out=y)
        Q.device_layer_norm_grad(dy, x, gamma, stats, out=outs[0], dgamma=outs[1], dbeta=outs[2])
    both()
    first = [t.to_host() for t in [y] + outs]
    graph, other = ctx.capture(both), ctx.capture(both)
    for t in [y] + outs:
        ctx.memset(t.ptr, 0x11, t.size * 2)
    graph.launch()
    both()
    other.launch()
    graph.launch()
    assert all(np.array_equal(a, t.to_host()) for a, t in zip(first, [y] + outs))


@TYPES
@pytest.mark.parametrize("C", [24, 300, 20001])
@pytest.mark.parametrize("over", ["dy", "dtotal"])
def test_gradient_over_its_input(dt, C, over):
    """dx in the place of dy or of the gradient that is added: the bits of a call with an array of its own."""
    ctx, dtype = shim.get_context(0), DTYPES[dt]
    rs = np.random.RandomState(C)
    x, dy, extra = (normal(rs, (2, 5, C), dtype) for _ in range(3))
    X, G, stats = put(ctx, x, dtype), put(ctx, normal(rs, (C,), dtype), dtype), Q.DeviceArray(ctx, (2, 5, 2), np.float32)
    Q.device_layer_norm(X, G, None, EPS, stats=stats)
    t = dict(dy=put(ctx, dy, dtype), dtotal=put(ctx, extra, dtype))
    want = [a.to_host() for a in Q.device_layer_norm_grad(t["dy"], X, G, stats, dtotal=t["dtotal"])]
    got = [a.to_host() for a in Q.device_layer_norm_grad(t["dy"], X, G, stats, dtotal=t["dtotal"], out=t[over])]
    assert all(np.array_equal(a, b) for a, b in zip(got, want))


def test_elements_off_their_boundaries_are_refused():
    ctx = shim.get_context(0)
    a = Q.DeviceArray(ctx, (2, 3, 8), np.float32)
    for off in (1, 2):
        bad = Q.DeviceArray(ctx, (1, 3, 8), np.float32, (24, 8, 1), a.ptr + off)
        with pytest.raises(ValueError):
            Q.device_layer_norm(bad)
    half = Q.DeviceArray(ctx, (1, 3, 8), np.float16, (24, 8, 1), a.ptr + 2)
    Q.device_layer_norm(half, out=Q.DeviceArray(ctx, (1, 3, 8), np.float16))
    with pytest.raises(ValueError):
        Q.device_layer_norm(a[:1], stats=Q.DeviceArray(ctx, (1, 3, 2), np.float32, (6, 2, 1), a.ptr + 4))
    ctx.sync()


def test_no_channels_refused_by_the_library():
    ctx = shim.get_context(0)
    d = Q.NormDesc(1, 1, 0, Q.F32, 0, 0.0)
    assert ctx.lib.b200conv_layer_norm(ctx.h, Q.ctypes.byref(d), None, None, None, None, None, None, None) == shim.E_INVALID
    assert ctx.lib.b200conv_layer_norm(ctx.h, None, None, None, None, None, None, None, None) == shim.E_INVALID
    assert ctx.lib.b200conv_layer_norm(None, Q.ctypes.byref(d), None, None, None, None, None, None, None) == shim.E_INVALID
