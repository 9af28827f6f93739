"""What the sequence operators refuse, before anything reaches the library; no GPU needed."""
import ctypes
import os
import re

import numpy as np
import pytest

from theano_b200 import sequence as Q
from theano_b200 import shim

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class _Library(object):
    """Counts the calls that pass the checks."""
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 0
        return call


class _Context(object):
    def __init__(self):
        self.lib, self.h, self.top = _Library(), 1, 4096

    def malloc(self, n):
        self.top += (n + 511) // 256 * 256
        return self.top

    def free(self, p):
        pass

    def h2d(self, p, a):
        pass

    def sync(self):
        pass

    def memset(self, *a):
        pass

    def check(self, rc):
        raise AssertionError(rc)


@pytest.fixture()
def ctx():
    return _Context()


def arr(ctx, *shape, dtype=np.float32):
    return Q.DeviceArray(ctx, shape, dtype)


def test_descriptors_match_the_header():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "b200conv.h")).read(), flags=re.S)
    sizes = {"int64_t": 8, "int32_t": 4, "float": 4, "b200conv_rows": ctypes.sizeof(Q.Rows)}
    for name, struct in (("rows", Q.Rows), ("norm_desc", Q.NormDesc), ("causal_desc", Q.CausalDesc), ("scan_desc", Q.ScanDesc)):
        body = re.search(r"typedef struct b200conv_%s \{(.*?)\} b200conv_%s;" % (name, name), text, re.S).group(1)
        fields = []
        for kind, names in re.findall(r"(\w+) ([^;]+);", body):
            fields += [(n.strip(), sizes[kind]) for n in names.split(",")]
        assert [f[0] for f in fields] == [f[0] for f in struct._fields_], name
        assert [f[1] for f in fields] == [ctypes.sizeof(f[1]) for f in struct._fields_], name
    assert re.search(r"B200CONV_BF16 = (\d+)", text).group(1) == str(Q.BF16)


def test_bfloat16_rounds_to_nearest_even():
    a = np.array([1.0, 1.00390625, 1.01171875, -3.0, 0.0, 65504.0, np.inf, -np.inf, 3.4e38, 1e-40], np.float32)
    want = np.array([1.0, 1.0, 1.015625, -3.0, 0.0, 65536.0, np.inf, -np.inf, np.inf, 2.0 ** -133], np.float32)      # subnormals are multiples of 2^-133
    assert np.array_equal(Q.from_bfloat16(Q.to_bfloat16(a)), want)
    assert np.isnan(Q.from_bfloat16(Q.to_bfloat16(np.array([np.nan], np.float32)))).all()
    with pytest.raises(TypeError):
        shim._dtype_code(Q.BFLOAT16)                   # the convolutions have no such type


def test_arrays(ctx):
    a = arr(ctx, 4, 6, 8)
    v = a[1:3, 2, 4:]
    assert v.shape == (2, 4) and v.strides == (48, 1) and v.ptr == a.ptr + 4 * (48 + 16 + 4) and v.span == 52
    for key in (np.s_[::2], np.s_[..., 0], np.s_[0, 0, 0], np.s_[9], np.s_[0, 0, :, 0]):
        with pytest.raises(IndexError):
            a[key]
    for shape, strides in (((2, 3), (3, 2)), ((2, 3), (-3, 1)), ((2, 3), (1,)), ((1, 1, 1, 1, 1), None), ((), None), ((-1, 2), None)):
        with pytest.raises(ValueError):
            Q.DeviceArray(ctx, shape, np.float32, strides, _ptr=4096)
    with pytest.raises(ValueError):
        Q.DeviceArray(ctx, (2, 3), np.float32, (3, 1))       # strides without memory of the caller's


def test_lengths(ctx):
    s = Q.Sequences(ctx, [3, 0, 5])
    assert (s.count, s.total, s.longest) == (3, 8, 5)
    for bad in ([], [[1, 2]], [1, -1], [1.5], [2 ** 31]):
        with pytest.raises(ValueError):
            Q.Sequences(ctx, bad)


NORM = dict(x=(2, 3, 8), gamma=(8,), beta=(8,), residual=(2, 3, 8), total=(2, 3, 8), out=(2, 3, 8))


@pytest.mark.parametrize("change,error", [
    (dict(x=(8,)), ValueError), (dict(x=(2, 3, 4, 8)), ValueError), (dict(gamma=(7,)), ValueError), (dict(beta=(8, 1)), ValueError), (dict(residual=(2, 3, 7)), ValueError),
    (dict(total=(6, 8)), ValueError), (dict(out=(2, 4, 8)), ValueError), (dict(stats=(2, 3)), ValueError), (dict(eps=-1.0), ValueError),
    (dict(eps=float("nan")), ValueError), (dict(x=(2, 3, 0), gamma=(0,), beta=(0,), residual=None, total=None, out=None), ValueError),
    (dict(residual="float16"), TypeError), (dict(gamma="float16", beta="bfloat16"), TypeError), (dict(x="int32"), TypeError)])
def test_layer_norm(ctx, change, error):
    def call(c):
        kw = {k: c.get(k, s) for k, s in NORM.items()}
        kw = {k: None if s is None else arr(ctx, *NORM[k], dtype=s) if isinstance(s, str) else arr(ctx, *s) for k, s in kw.items()}
        if "stats" in c:
            kw["stats"] = arr(ctx, *c["stats"])
        Q.device_layer_norm(kw.pop("x"), eps=c.get("eps", 1e-5), **kw)
    call({})
    assert ctx.lib.calls == ["b200conv_layer_norm"]
    with pytest.raises(error):
        call(change)
    assert len(ctx.lib.calls) == 1


def test_layer_norm_gradient(ctx):
    x, g, st = arr(ctx, 2, 3, 8), arr(ctx, 8), arr(ctx, 2, 3, 2)
    Q.device_layer_norm_grad(x, x, g, st, dgamma=False)
    for bad in (lambda: Q.device_layer_norm_grad(x, x, g, None), lambda: Q.device_layer_norm_grad(x, arr(ctx, 2, 4, 8), g, st),
                lambda: Q.device_layer_norm_grad(x, x, g, arr(ctx, 2, 3, 3)), lambda: Q.device_layer_norm_grad(x, x, g, st, dbeta=arr(ctx, 9)),
                lambda: Q.device_layer_norm_grad(x, x, g, arr(ctx, 2, 4, 2)[:, :3])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        Q.device_layer_norm_grad(x, x, g, st, dgamma=arr(ctx, 8, dtype=np.float16))
    assert ctx.lib.calls == ["b200conv_layer_norm_grad"]


def test_causal_convolution(ctx):
    x, w, init = arr(ctx, 2, 9, 8), arr(ctx, 8, 4), arr(ctx, 2, 3, 8)
    Q.device_causal_conv1d(x, w, arr(ctx, 8), initial=init, final=init)
    packed, seqs = arr(ctx, 9, 8), Q.Sequences(ctx, [4, 5])
    Q.device_causal_conv1d(packed, w, sequences=seqs)
    calls = list(ctx.lib.calls)
    for bad in (lambda: Q.device_causal_conv1d(x, arr(ctx, 7, 4)), lambda: Q.device_causal_conv1d(x, arr(ctx, 8, 9)), lambda: Q.device_causal_conv1d(x, arr(ctx, 8, 1)),
                lambda: Q.device_causal_conv1d(x, arr(ctx, 8)), lambda: Q.device_causal_conv1d(x, w, arr(ctx, 9)), lambda: Q.device_causal_conv1d(x, w, initial=arr(ctx, 2, 4, 8)),
                lambda: Q.device_causal_conv1d(x, w, final=arr(ctx, 3, 3, 8)), lambda: Q.device_causal_conv1d(packed, w), lambda: Q.device_causal_conv1d(x, w, sequences=seqs),
                lambda: Q.device_causal_conv1d(packed, w, sequences=Q.Sequences(ctx, [4, 6])), lambda: Q.device_causal_conv1d(x, w, out=arr(ctx, 2, 8, 8)),
                lambda: Q.device_causal_conv1d(x, arr(ctx, 8, 6)[:, :4]), lambda: Q.device_causal_conv1d_step(x, init, w), lambda: Q.device_causal_conv1d_step(arr(ctx, 3, 8), init, w),
                lambda: Q.device_causal_conv1d_grad(arr(ctx, 2, 8, 8), x, w), lambda: Q.device_causal_conv1d_grad(x, x, w, dw=arr(ctx, 8, 3))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: Q.device_causal_conv1d(x, arr(ctx, 8, 4, dtype=np.float16)), lambda: Q.device_causal_conv1d(x, w, initial=arr(ctx, 2, 3, 8, dtype="bfloat16")),
                lambda: Q.device_causal_conv1d(np.zeros((2, 9, 8), np.float32), w)):
        with pytest.raises(TypeError):
            bad()
    assert ctx.lib.calls == calls


SCAN = dict(x=(2, 9, 8), dt=(2, 9, 8), A=(8, 4), B=(2, 9, 2, 4), C=(2, 9, 2, 4), D=(8,), z=(2, 9, 8), dt_bias=(8,), initial=(2, 8, 4), final=(2, 8, 4))


@pytest.mark.parametrize("change,error", [
    (dict(dt=(2, 9, 7)), ValueError), (dict(A=(8, 5)), ValueError), (dict(A=(7, 4)), ValueError), (dict(A=(8, 129), B=(2, 9, 129), C=(2, 9, 129), initial=None, final=None), ValueError),
    (dict(A=(8, 0), B=(2, 9, 0), C=(2, 9, 0), initial=None, final=None), ValueError), (dict(B=(2, 9, 4)), ValueError), (dict(B=(2, 9, 3, 4), C=(2, 9, 3, 4)), ValueError),
    (dict(B=(2, 8, 2, 4)), ValueError), (dict(D=(7,)), ValueError), (dict(z=(2, 9, 9)), ValueError), (dict(dt_bias=(8, 1)), ValueError), (dict(initial=(2, 4, 8)), ValueError),
    (dict(final=(1, 8, 4)), ValueError), (dict(x=(9, 8)), ValueError), (dict(B="float16"), TypeError), (dict(A="float16"), TypeError), (dict(initial="float16"), TypeError),
    (dict(z="bfloat16"), TypeError)])
def test_selective_scan(ctx, change, error):
    def call(c):
        kw = {k: c.get(k, s) for k, s in SCAN.items()}
        kw = {k: None if s is None else arr(ctx, *SCAN[k], dtype=s) if isinstance(s, str) else arr(ctx, *s) for k, s in kw.items()}
        Q.device_selective_scan(*[kw.pop(k) for k in ("x", "dt", "A", "B", "C")], softplus=True, **kw)
    call({})
    with pytest.raises(error):
        call(change)
    assert ctx.lib.calls == ["b200conv_selective_scan"]


def test_selective_scan_gradient_and_step(ctx):
    t = {k: arr(ctx, *s) for k, s in SCAN.items()}
    args = [t[k] for k in ("x", "x", "dt", "A", "B", "C")]
    more = dict(D=t["D"], z=t["z"], dt_bias=t["dt_bias"], initial=t["initial"])
    assert set(Q.device_selective_scan_grad(*args, **more)) == {"x", "dt", "A", "B", "C", "D", "z", "dt_bias", "initial"}
    assert set(Q.device_selective_scan_grad(*args)) == {"x", "dt", "A", "B", "C"}
    for bad in (dict(grads=dict(y=t["x"])), dict(grads=dict(B=arr(ctx, 2, 9, 4, 2))), dict(grads=dict(A=arr(ctx, 8, 3))), dict(dfinal=arr(ctx, 2, 8, 5))):
        with pytest.raises(ValueError):
            Q.device_selective_scan_grad(*args, **more, **bad)
    with pytest.raises(ValueError):
        Q.device_selective_scan_grad(*args, grads=dict(z=t["x"]))
    step = [arr(ctx, 2, 8), arr(ctx, 2, 8), t["A"], arr(ctx, 2, 2, 4), arr(ctx, 2, 2, 4)]
    Q.device_selective_scan_step(*step, t["initial"])
    for bad in ((step[:4] + [arr(ctx, 2, 4)], t["initial"]), (step, arr(ctx, 3, 8, 4)), ([t["x"]] + step[1:], t["initial"])):
        with pytest.raises(ValueError):
            Q.device_selective_scan_step(*bad[0], bad[1])
    assert len(ctx.lib.calls) == 3


def test_pad_channels_of_an_image_are_no_scan_results(ctx):
    wide = Q.DeviceArray(ctx, (2, 9, 6), np.float32, (72, 8, 1), 4096, 8)
    with pytest.raises(ValueError):
        Q.device_selective_scan(wide, wide, arr(ctx, 6, 4), arr(ctx, 2, 9, 4), arr(ctx, 2, 9, 4), out=wide)


def test_tensors_of_another_context(ctx):
    other = _Context()
    x, w = arr(ctx, 2, 9, 8), arr(other, 8, 4)
    for bad in (lambda: Q.device_causal_conv1d(x, w), lambda: Q.device_layer_norm(x, arr(other, 8)), lambda: Q.device_layer_norm(x, out=arr(other, 2, 9, 8)),
                lambda: Q.device_causal_conv1d(arr(ctx, 9, 8), arr(ctx, 8, 4), sequences=Q.Sequences(other, [9]))):
        with pytest.raises(ValueError):
            bad()
    assert not ctx.lib.calls and not other.lib.calls


def test_a_checked_call_does_not_vouch_for_another(ctx):
    """Plans are found by what was checked: another shape, type, stride or option is checked again."""
    x, w = arr(ctx, 2, 9, 8), arr(ctx, 8, 4)
    for _ in range(2):
        Q.device_causal_conv1d(x, w)
    with pytest.raises(ValueError):
        Q.device_causal_conv1d(arr(ctx, 2, 9, 7), w)
    with pytest.raises(TypeError):
        Q.device_causal_conv1d(arr(ctx, 2, 9, 8, dtype=np.float16), w, out=x)


@pytest.mark.parametrize("call", [lambda a: Q.layer_norm(a), lambda a: Q.causal_conv1d(a, a[0]), lambda a: Q.selective_scan(a, a, a[0], a, a)])
def test_host_arrays_of_other_types(call):
    with pytest.raises(TypeError):
        call(np.zeros((2, 3, 4)))
