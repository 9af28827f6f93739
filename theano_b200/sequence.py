"""Layers of sequence models on the GPU: layer norm, the short causal convolution and the selective state space scan.

Beside the convolutions of ``theano_b200.shim`` and in the same two forms: numpy arrays in and out (what an op's
``perform`` calls) and ``device_*`` calls on tensors that stay in HBM, which are asynchronous on their context's stream.
Sequence tensors are ``(sequences, tokens, channels)`` with contiguous channels; sequences of several lengths may lie one
behind the other in a ``(rows, channels)`` tensor (`Sequences`).  A channels-last ``shim.DeviceTensor`` counts as one with
its pixels as tokens.  Data types: float32, float16 and bfloat16; sums and states are float32.  A result's memory is that of an input
only where a call says so; other overlaps raise ValueError.

The reference runs causal convolutions through its 2-D convolution (theano/tensor/nnet/abstract_conv.py, causal_conv1d) and
recurrences through its scan op, one op call per token; nothing here computes on the CPU.
"""
import ctypes
import itertools

import numpy as np

from . import shim
from .shim import DeviceTensor, _P

F32, F16, BF16 = shim.F32, shim.F16, 2
# numpy has no bfloat16: its bits in a field of that name, so that no calculation takes them for integers
BFLOAT16 = np.dtype([("bfloat16", np.uint16)])
_CODES = {np.dtype(np.float32): F32, np.dtype(np.float16): F16, BFLOAT16: BF16}
_DTYPES = {F32: np.dtype(np.float32), F16: np.dtype(np.float16), BF16: BFLOAT16}
_INT32 = np.dtype(np.int32)
_OTHER = -1                              # code of tensors that are no operands (offsets)
_FREED = "the memory of this tensor has been freed"


_signatures = {}                         # what plans need to know of an array -> a number that stands for it
_numbers = itertools.count(1)


def _signature(*what):
    """A number for a shape with its strides and type: plans are looked up on every call, and hashing ten nested tuples cost
    as much host time as the launch.  Equal signatures may get two numbers (the table is emptied at times), never two one."""
    n = _signatures.get(what)
    if n is None:
        if len(_signatures) >= 1 << 16:
            _signatures.clear()
        n = _signatures[what] = next(_numbers)
    return n


def _dtype(dt):
    return BFLOAT16 if isinstance(dt, str) and dt == "bfloat16" else np.dtype(dt)


def to_bfloat16(a):
    """float32 values as bfloat16 bits (`BFLOAT16`), rounded to nearest even."""
    bits = np.ascontiguousarray(a, dtype=np.float32).view(np.uint32)
    nan = (bits & 0x7fffffff) > 0x7f800000
    out = ((bits + 0x7fff + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    out[nan] = 0x7fc0
    return out.view(BFLOAT16).reshape(np.shape(a))


def from_bfloat16(a):
    """The float32 values of bfloat16 bits."""
    return (np.ascontiguousarray(a).view(np.uint16).astype(np.uint32) << 16).view(np.float32).reshape(np.shape(a))


class DeviceArray(object):
    """An array in HBM of up to four axes, the last one contiguous; ``strides`` are in elements.

    ``a[:, 3:9]`` and the like are views (integers and slices of step 1), which keep the array alive.  Arrays that wrap a
    pointer (``_ptr``) own nothing.  ``stored``: channels that a row holds in memory, those beyond the shape's last
    extent being zeros that the operators write (pad channels of an image)."""

    def __init__(self, ctx, shape, dtype, strides=None, _ptr=None, stored=0, _base=None):
        self.ctx, self.shape, self.dtype = ctx, tuple(int(s) for s in shape), _dtype(dtype)
        if not 1 <= len(self.shape) <= 4 or any(s < 0 for s in self.shape):
            raise ValueError("a device array has one to four axes of extent 0 or more, not %s" % (self.shape,))
        if strides is None:
            strides, n = [], 1
            for s in reversed(self.shape):
                strides.insert(0, n)
                n *= s
        elif _ptr is None:
            raise ValueError("strides belong to arrays that wrap memory")
        self.strides = tuple(int(s) for s in strides)
        if len(self.strides) != len(self.shape) or any(s < 0 for s in self.strides) or (self.shape[-1] > 1 and self.strides[-1] != 1):
            raise ValueError("the last axis must be contiguous and no stride negative: shape %s, strides %s" % (self.shape, self.strides))
        self.stored, self._base = int(stored), _base
        self.code = _CODES.get(self.dtype, _OTHER)
        self.sig = _signature(self.shape, self.strides, self.code, self.stored)
        self.owner = _ptr is None
        self.ptr = ctx.malloc(self.size * self.dtype.itemsize) if self.owner else _ptr

    @property
    def size(self):
        n = 1
        for s in self.shape:
            n *= s
        return n

    @property
    def span(self):
        """Elements from the first to behind the last one."""
        return 1 + sum((n - 1) * s for n, s in zip(self.shape, self.strides)) if self.size else 0

    @property
    def freed(self):
        return self.ptr is None or (self._base is not None and self._base.ptr is None)

    def __getitem__(self, key):
        if self.freed:
            raise ValueError(_FREED)
        key = key if isinstance(key, tuple) else (key,)
        if len(key) > len(self.shape) or any(k is Ellipsis or k is None for k in key):
            raise IndexError("too many indices, or neither integers nor slices")
        shape, strides, at = [], [], 0
        for axis, n in enumerate(self.shape):
            k = key[axis] if axis < len(key) else slice(None)
            if isinstance(k, slice):
                a, b, step = k.indices(n)
                if step != 1:
                    raise IndexError("slices of a device array have step 1")
                shape.append(max(0, b - a))
                strides.append(self.strides[axis])
                at += a * self.strides[axis]
            else:
                k = k.__index__()
                if not -n <= k < n or axis == len(self.shape) - 1:
                    raise IndexError("index %d of axis %d (extent %d; the last axis takes slices)" % (k, axis, n))
                at += (k % n) * self.strides[axis]
        whole = shape[-1] == self.shape[-1]
        return _View(self.ctx, shape, self.dtype, strides, self.ptr + at * self.dtype.itemsize, self.stored if whole else 0,
                     self if self._base is None else self._base)

    @staticmethod
    def rows_of(image):
        """The (N, H * W, C) rows of a channels-last `shim.DeviceTensor`."""
        if image.layout != "nhwc":
            raise ValueError("sequence operators take channels-last tensors")
        if image.ptr is None:
            raise ValueError(_FREED)
        n, c, h, w = image.shape
        cp = image.stored_channels
        return _View(image.ctx, (n, h * w, c), image.dtype, (h * w * cp, cp, 1), image.ptr, cp, image)

    @classmethod
    def from_host(cls, ctx, arr, dtype=None):
        """Upload a numpy array, as `dtype` (default: its own; 'bfloat16' rounds float32 values)."""
        dtype = _dtype(arr.dtype if dtype is None else dtype)
        arr = np.ascontiguousarray(arr)
        if arr.dtype != dtype:
            arr = to_bfloat16(arr) if dtype == BFLOAT16 else arr.astype(dtype)
        t = cls(ctx, arr.shape or (1,), dtype)
        ctx.h2d(t.ptr, arr)
        ctx.sync()
        return t

    def to_host(self):
        """A numpy array of the values (bfloat16: as float32)."""
        if self.freed:
            raise ValueError(_FREED)
        flat = np.empty(self.span, self.dtype)
        self.ctx.d2h(flat, self.ptr)
        self.ctx.sync()
        es = self.dtype.itemsize
        if not self.size:
            a = np.empty(self.shape, self.dtype)
        else:
            a = np.array(np.lib.stride_tricks.as_strided(flat, self.shape, [s * es for s in self.strides]))
        return from_bfloat16(a) if self.dtype == BFLOAT16 else a

    def free(self):
        if self.ptr and self.owner:
            self.ctx.free(self.ptr)
        self.ptr = None

    def __del__(self):
        try:
            if self.owner and self.ctx.h:
                self.free()
        except Exception:
            pass


class _View(DeviceArray):
    """Memory of another tensor: checked on every use, since that one may be freed before its views are gone."""


class Sequences(object):
    """The lengths of sequences that lie one behind the other in the rows of a (rows, channels) tensor; rows behind the
    last sequence belong to none: they are neither read nor written.  Made once per batch and kept by the program."""

    def __init__(self, ctx, lengths):
        lengths = np.asarray(lengths)
        if lengths.ndim != 1 or lengths.size == 0 or lengths.dtype.kind not in "iu":
            raise ValueError("lengths must be a vector of integers with one entry or more")
        if lengths.min() < 0 or int(lengths.astype(np.int64).sum()) > np.iinfo(np.int32).max:
            raise ValueError("lengths must not be negative nor add up to over 2^31 - 1")
        self.ctx, self.count = ctx, int(lengths.size)
        self.lengths = tuple(int(n) for n in lengths)
        self.total, self.longest = int(lengths.astype(np.int64).sum()), int(lengths.max())
        self.starts = DeviceArray.from_host(ctx, np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32))
        self.sig = _signature("sequences", self.count, self.total, self.longest)


# ======================================================================================
# plans: descriptors of calls that have been checked
# ======================================================================================
class Rows(ctypes.Structure):
    """``b200conv_rows`` of include/b200conv.h."""
    _fields_ = [("row", ctypes.c_int64), ("seq", ctypes.c_int64), ("stored", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class NormDesc(ctypes.Structure):
    """``b200conv_norm_desc``."""
    _fields_ = [("sequences", ctypes.c_int64), ("length", ctypes.c_int64), ("C", ctypes.c_int32), ("dtype", ctypes.c_int32),
                ("param_f32", ctypes.c_int32), ("eps", ctypes.c_float)] + [
                    (n, Rows) for n in ("x", "residual", "y", "total", "dy", "dtotal", "dx")]


_plans = {}                              # signature of a call -> its checked descriptor; emptied when it holds _LIMIT
_LIMIT = 4096


def _plan(key, make, *args):
    plan = _plans.get(key)
    if plan is None:
        plan = make(*args)
        if len(_plans) >= _LIMIT:
            _plans.clear()
        _plans[key] = plan
    return plan


def _array(t):
    """A tensor argument as a DeviceArray: channels-last images as their rows, other DeviceTensors as a vector."""
    if t is None or type(t) is DeviceArray:
        return t
    if isinstance(t, DeviceTensor):
        if t.layout == "nhwc":
            return DeviceArray.rows_of(t)
        if t.ptr is None:
            raise ValueError(_FREED)
        n = t.shape[0] * t.shape[1] * t.shape[2] * t.shape[3]
        return DeviceArray(t.ctx, (n,), t.dtype, (1,), t.ptr, 0, t)
    if isinstance(t, DeviceArray):
        if t.freed:
            raise ValueError(_FREED)
        return t
    raise TypeError("expected a DeviceArray or a channels-last DeviceTensor, not %s" % type(t).__name__)


def _sig(t):
    return 0 if t is None else t.sig


def _ptr(t):
    """Of an argument that may be left out; one that was freed is not (for the others the library refuses a null pointer)."""
    if t is None:
        return None
    if t.ptr is None:
        raise ValueError(_FREED)
    return t.ptr


def _one_context(ctx, *tensors):
    for t in tensors:
        if t is not None and t.ctx is not ctx:
            raise ValueError("tensors of one call must belong to one context (another context's stream is not waited for)")


def _like(t, original):
    """A new tensor for a result of `t`'s shape: an image where the argument was one."""
    if isinstance(original, DeviceTensor):
        return DeviceTensor(t.ctx, original.shape, t.dtype, "nhwc")
    return DeviceArray(t.ctx, t.shape, t.dtype)


def _same(what, t, shape, code):
    if t is None:
        return
    if t.shape != tuple(shape):
        raise ValueError("%s must have shape %s, not %s" % (what, tuple(shape), t.shape))
    if t.code != code:
        raise TypeError("%s must be %s, not %s" % (what, _DTYPES[code], t.dtype))


def _operand_code(t):
    if t.code == _OTHER:
        raise TypeError("sequence operators handle float32, float16 and bfloat16, not %s" % t.dtype)
    return t.code


def _params(what, code, *tensors):
    """Whether the parameters are float32 beside tensors of another type; all of them share one."""
    codes = {t.code for t in tensors if t is not None}
    if len(codes) > 1 or not codes <= {code, F32}:
        raise TypeError("%s must share one data type: the tensors' or float32" % what)
    return int(code != F32 and codes == {F32})


def _rows(t):
    if t is None:
        return Rows()
    seq, row = (t.strides[0], t.strides[1]) if len(t.shape) == 3 else (0, t.strides[0])
    return Rows(row, seq, t.stored, 0)


# ======================================================================================
# layer norm
# ======================================================================================
def _norm_shape(x):
    if len(x.shape) not in (2, 3):
        raise ValueError("layer norm takes (rows, channels) or (sequences, tokens, channels), not %s" % (x.shape,))
    return (x.shape[:2] if len(x.shape) == 3 else (1, x.shape[0])) + (x.shape[-1],)


def _plan_norm(eps, x, gamma, beta, stats, **tensors):
    code = _operand_code(x)
    S, T, C = _norm_shape(x)
    if C == 0:
        raise ValueError("layer norm over no channels")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    for name, t in tensors.items():
        _same(name, t, x.shape, code)
    for name, t in (("gamma", gamma), ("beta", beta)):
        if t is not None and t.shape != (C,):
            raise ValueError("%s must have one value per channel (%d), not shape %s" % (name, C, t.shape))
    _same("stats", stats, x.shape[:-1] + (2,), F32)
    if stats is not None and stats.strides != DeviceArray(x.ctx, stats.shape, np.float32, _ptr=0).strides:
        raise ValueError("stats must be contiguous")
    d = NormDesc(S, T, C, code, _params("gamma and beta", code, gamma, beta), eps)
    d.x = _rows(x)
    for name, t in tensors.items():
        setattr(d, name, _rows(t))
    return ctypes.byref(d)


def device_layer_norm(x, gamma=None, beta=None, eps=1e-5, residual=None, total=None, stats=None, out=None):
    """Layer norm over the channels of every row of x (+ residual): ``(t - mean) * rstd * gamma + beta``.

    `gamma`, `beta`: vectors of the tensors' type or float32.  `residual`: added to x first; `total` receives the sum,
    rounded to the tensors' type, which is what is normalised (it may be x or residual themselves).  `stats`: float32 of
    x's shape with (mean, rstd) in place of the channels, for the gradient.  Returns `out` (which may be x or residual, not `total`)."""
    given, x = x, _array(x)
    ctx = x.ctx
    gamma, beta, residual, total, stats = _array(gamma), _array(beta), _array(residual), _array(total), _array(stats)
    if out is None:
        out = _like(x, given)
    y = _array(out)
    _one_context(ctx, gamma, beta, residual, total, stats, y)
    d = _plan(("norm", eps, x.sig, _sig(gamma), _sig(beta), _sig(stats), _sig(residual), _sig(total), y.sig), lambda: _plan_norm(
        eps, x, gamma, beta, stats, residual=residual, total=total, y=y))
    rc = ctx.lib.b200conv_layer_norm(ctx.h, d, x.ptr, _ptr(residual), _ptr(gamma), _ptr(beta), y.ptr, _ptr(total), _ptr(stats))
    if rc:
        ctx.check(rc)
    return out


def device_layer_norm_grad(dy, x, gamma, stats, dtotal=None, out=None, dgamma=None, dbeta=None):
    """Gradients (dx, dgamma, dbeta) of `device_layer_norm`; x is what was normalised (`total` where there was a
    residual) and `stats` what the forward call left.  `dtotal`, the gradient that reaches the sum on other ways, is added to
    dx, which may be dy, x or dtotal.  dgamma and dbeta have gamma's type (float32 without one); False leaves one out."""
    given, dy = dy, _array(dy)
    ctx = dy.ctx
    x, gamma, stats, dtotal = _array(x), _array(gamma), _array(stats), _array(dtotal)
    if out is None:
        out = _like(dy, given)
    ptype = gamma.dtype if gamma is not None else np.float32
    grads = [None if g is False else g if g is not None else DeviceArray(ctx, (dy.shape[-1],), ptype) for g in (dgamma, dbeta)]
    dg, db = (_array(g) for g in grads)
    dx = _array(out)
    _one_context(ctx, x, gamma, stats, dtotal, dx, dg, db)
    if stats is None:
        raise ValueError("the gradient needs the statistics of the forward call")

    def make():
        _params("gamma and its gradients", dy.code, gamma, dg, db)
        for name, t in (("dgamma", dg), ("dbeta", db)):
            if t is not None and t.shape != (dy.shape[-1],):
                raise ValueError("%s must have one value per channel (%d), not shape %s" % (name, dy.shape[-1], t.shape))
        d = _plan_norm(0.0, x, gamma, None, stats, dy=dy, dtotal=dtotal, dx=dx)
        d._obj.param_f32 = _params("gamma and its gradients", dy.code, gamma, dg, db)
        return d
    d = _plan(("norm grad", dy.sig, x.sig, _sig(gamma), stats.sig, _sig(dtotal), dx.sig, _sig(dg), _sig(db)), make)
    rc = ctx.lib.b200conv_layer_norm_grad(ctx.h, d, dy.ptr, x.ptr, _ptr(gamma), stats.ptr, _ptr(dtotal), dx.ptr, _ptr(dg), _ptr(db))
    if rc:
        ctx.check(rc)
    return out, grads[0], grads[1]


# ======================================================================================
# the short causal convolution
# ======================================================================================
class CausalDesc(ctypes.Structure):
    """``b200conv_causal_desc``."""
    _fields_ = [("sequences", ctypes.c_int64), ("length", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in (
        "C", "width", "dtype", "param_f32", "flip", "silu", "packed", "reserved")] + [(n, Rows) for n in ("x", "y", "dy", "dx")]


def _contiguous(what, t):
    if t is not None:
        n = 1
        for size, stride in zip(reversed(t.shape), reversed(t.strides)):
            if size > 1 and stride != n:
                raise ValueError("%s must be contiguous" % what)
            n *= size


def _batch(x, sequences, what):
    """(sequences, tokens of each or rows of the tensor, channels) of a call's main tensor."""
    if sequences is None:
        if len(x.shape) != 3:
            raise ValueError("%s takes (sequences, tokens, channels), not %s" % (what, x.shape))
        return x.shape[0], x.shape[1], x.shape[2]
    if len(x.shape) != 2:
        raise ValueError("%s takes packed sequences as (rows, channels), not %s" % (what, x.shape))
    if sequences.total > x.shape[0]:
        raise ValueError("the sequences have %d tokens, the tensor has %d rows" % (sequences.total, x.shape[0]))
    return sequences.count, x.shape[0], x.shape[1]


def _plan_causal(x, w, bias, silu, flip, packed, S, T, C, states, tensors, grads):
    code = _operand_code(x)
    if len(w.shape) != 2 or w.shape[0] != C:
        raise ValueError("the filters must have shape (%d, taps), not %s" % (C, w.shape))
    width = w.shape[1]
    if not 2 <= width <= 8:
        raise ValueError("a short causal convolution has 2 to 8 taps, not %d" % width)
    _contiguous("the filters", w)
    if bias is not None and bias.shape != (C,):
        raise ValueError("bias must have one value per channel (%d), not shape %s" % (C, bias.shape))
    for name, t, like in grads:
        if t is not None and t.shape != like:
            raise ValueError("%s must have shape %s, not %s" % (name, like, t.shape))
        _contiguous(name, t)
    for name, t in states:
        _same(name, t, (S, width - 1, C), code)
        _contiguous(name, t)
    for name, t in tensors:
        _same(name, t, x.shape, code)
    d = CausalDesc(S, T, C, width, code, _params("filters, bias and their gradients", code, w, bias, *[t for _, t, _ in grads]), int(bool(flip)),
                   int(bool(silu)), int(packed), 0)
    d.x = _rows(x)
    for name, t in tensors:
        if t is not None:
            setattr(d, name, _rows(t))
    return ctypes.byref(d)


def device_causal_conv1d(x, w, bias=None, silu=False, filter_flip=True, initial=None, final=None, sequences=None, out=None):
    """Every channel's own short filter over the tokens up to each one: ``y[t] = sum_k w[:, k] x[t - k]`` (without
    `filter_flip` the last weight meets token t), + `bias`, then v * sigmoid(v) with `silu`.

    `w`: (channels, taps), 2 to 8 taps; `initial`: (sequences, taps - 1, channels), the tokens before the first, oldest
    first (default: zeros); `final` receives the same behind the last token and may be `initial`.  With `sequences`
    x is (rows, channels).  Returns `out`, which is none of the inputs."""
    given, x, w, bias = x, _array(x), _array(w), _array(bias)
    ctx = x.ctx
    initial, final = _array(initial), _array(final)
    if out is None:
        out = _like(x, given)
    y = _array(out)
    _one_context(ctx, w, bias, initial, final, y, sequences)
    d = _plan(("causal", silu, filter_flip, x.sig, w.sig, _sig(bias), _sig(initial), _sig(final), y.sig, _sig(sequences)), lambda: _plan_causal(
        x, w, bias, silu, filter_flip, sequences is not None, *_batch(x, sequences, "a causal convolution"),
        (("initial", initial), ("final", final)), (("y", y),), ()))
    rc = ctx.lib.b200conv_causal_conv(ctx.h, d, x.ptr, w.ptr, _ptr(bias), _ptr(initial), sequences and sequences.starts.ptr, y.ptr, _ptr(final))
    if rc:
        ctx.check(rc)
    return out


def device_causal_conv1d_grad(dy, x, w, bias=None, silu=False, filter_flip=True, initial=None, sequences=None, out=None, dw=None, dbias=None,
                              dinitial=None):
    """Gradients (dx, dw, dbias, dinitial) of `device_causal_conv1d`.  dw and dbias have the types of w and bias (False
    leaves one out, dbias exists with a bias only), dinitial is computed where it is given and may be `initial`.  dx is none of the
    inputs."""
    given, dy, x, w, bias = dy, _array(dy), _array(x), _array(w), _array(bias)
    ctx = x.ctx
    initial, dinitial = _array(initial), _array(dinitial)
    if out is None:
        out = _like(dy, given)
    dx = _array(out)
    dw = None if dw is False else dw if dw is not None else DeviceArray(ctx, w.shape, w.dtype)
    dbias = None if dbias is False or bias is None else dbias if dbias is not None else DeviceArray(ctx, bias.shape, bias.dtype)
    gw, gb = _array(dw), _array(dbias)
    _one_context(ctx, dy, w, bias, initial, dx, gw, gb, dinitial, sequences)
    d = _plan(("causal grad", silu, filter_flip, dy.sig, x.sig, w.sig, _sig(bias), _sig(initial), dx.sig, _sig(gw), _sig(gb), _sig(dinitial),
               _sig(sequences)), lambda: _plan_causal(
        x, w, bias, silu, filter_flip, sequences is not None, *_batch(x, sequences, "a causal convolution"),
        (("initial", initial), ("dinitial", dinitial)), (("dy", dy), ("dx", dx)),
        (("dw", gw, w.shape), ("dbias", gb, (w.shape[0],)))))
    rc = ctx.lib.b200conv_causal_conv_grad(ctx.h, d, dy.ptr, x.ptr, w.ptr, _ptr(bias), _ptr(initial), sequences and sequences.starts.ptr, dx.ptr,
                                           _ptr(gw), _ptr(gb), _ptr(dinitial))
    if rc:
        ctx.check(rc)
    return out, dw, dbias, dinitial


def device_causal_conv1d_step(x, state, w, bias=None, silu=False, filter_flip=True, out=None):
    """One token of every sequence, x (sequences, channels): the token `device_causal_conv1d` would give behind `state`,
    (sequences, taps - 1, channels), which moves on in place.  `out` may be x."""
    x, w, bias, state = _array(x), _array(w), _array(bias), _array(state)
    ctx = x.ctx
    if out is None:
        out = DeviceArray(ctx, x.shape, x.dtype)
    y = _array(out)
    _one_context(ctx, w, bias, state, y)

    def make():
        if len(x.shape) != 2:
            raise ValueError("a step takes (sequences, channels), not %s" % (x.shape,))
        d = _plan_causal(x, w, bias, silu, filter_flip, False, x.shape[0], 1, x.shape[1], (("state", state),), (("y", y),), ())
        for name, t in (("x", x), ("y", y)):
            setattr(d._obj, name, Rows(x.shape[1], t.strides[0], t.stored, 0))
        return d
    d = _plan(("causal step", silu, filter_flip, x.sig, w.sig, _sig(bias), state.sig, y.sig), make)
    rc = ctx.lib.b200conv_causal_conv_step(ctx.h, d, x.ptr, w.ptr, _ptr(bias), state.ptr, y.ptr)
    if rc:
        ctx.check(rc)
    return out


# ======================================================================================
# the selective state space scan
# ======================================================================================
class ScanDesc(ctypes.Structure):
    """``b200conv_scan_desc``."""
    _fields_ = [("sequences", ctypes.c_int64), ("length", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in (
        "C", "N", "groups", "dtype", "softplus", "packed", "longest", "reserved")] + [
            (n, Rows) for n in ("x", "dt", "z", "B", "Cm", "y", "dy", "dx", "ddt", "dz", "dB", "dCm")]


def _group_rows(what, t, lead):
    """B or C as (leading axes..., groups, N): its rows, groups and states."""
    if t is None:
        return Rows(), None, None
    if len(t.shape) not in (len(lead) + 1, len(lead) + 2) or t.shape[:len(lead)] != lead:
        raise ValueError("%s must have shape %s + (groups, states) or (states,), not %s" % (what, lead, t.shape))
    groups, N = (t.shape[-2] if len(t.shape) == len(lead) + 2 else 1), t.shape[-1]
    if groups > 1 and N > 0 and t.strides[-2] != N:
        raise ValueError("the groups of %s must follow each other without gaps" % what)
    seq, row = (t.strides[0], t.strides[1]) if len(lead) == 2 else (0, t.strides[0])
    return Rows(row, seq, 0, 0), groups, N


def _plan_scan(x, A, vectors, softplus, sequences, states, tensors, grouped):
    """`tensors`: (field, tensor) like x; `grouped`: (field, tensor) like B; `vectors`: float32 values per channel."""
    code = _operand_code(x)
    S, T, C = _batch(x, sequences, "a selective scan")
    if len(A.shape) != 2 or A.shape[0] != C:
        raise ValueError("A must have shape (%d, states), not %s" % (C, A.shape))
    N = A.shape[1]
    if not 1 <= N <= 128:
        raise ValueError("a selective scan has 1 to 128 states per channel, not %d" % N)
    _same("A", A, (C, N), F32)
    _contiguous("A", A)
    d = ScanDesc(S, T, C, N, 1, code, int(bool(softplus)), int(sequences is not None), sequences.longest if sequences else 0, 0)
    d.x = _rows(x)
    for name, t in tensors:
        _same(name, t, x.shape, code)
        if t is not None and t.stored > C and name in ("y", "dx", "ddt", "dz"):
            raise ValueError("a selective scan writes no pad channels: %d channels are stored as %d" % (C, t.stored))
        setattr(d, name, _rows(t))
    shape = None
    for name, t in grouped:
        rows, groups, n = _group_rows(name.replace("Cm", "C"), t, x.shape[:-1])
        if t is None:
            continue
        if t.code != code:
            raise TypeError("%s must have the tensors' data type" % name.replace("Cm", "C"))
        shape = shape or (groups, n)
        if (groups, n) != shape or n != N:
            raise ValueError("B, C and A disagree about groups or states: %s of %s, A has %d states" % ((groups, n), shape, N))
        setattr(d, name, rows)
    d.groups = shape[0]
    if d.groups < 1 or C % d.groups:
        raise ValueError("%d channels cannot share %d groups of B and C" % (C, d.groups))
    for name, t in vectors:
        _same(name, t, (C,) if not name.endswith("A") else (C, N), F32)
        _contiguous(name, t)
    for name, t in states:
        _same(name, t, (S, C, N), F32)
        _contiguous(name, t)
    return ctypes.byref(d)


def device_selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=False, initial=None, final=None, sequences=None, out=None):
    """The selective state space scan over the tokens of every sequence and channel:

        delta = dt + dt_bias (softplus of it);  h = exp(delta * A) * h + delta * x * B;  y = (sum(C * h) + D * x) * (z * sigmoid(z))

    x, dt, z: (sequences, tokens, channels), or (rows, channels) with `sequences`; B, C: the same rows of (groups, states) or
    (states,), shared by the channels of a group; A (channels, states), D and dt_bias (channels,) float32.  `initial` and `final`:
    float32 (sequences, channels, states), which may be one array.  Returns `out`, which may be x, dt or z."""
    given, x, dt, A, B, C = x, _array(x), _array(dt), _array(A), _array(B), _array(C)
    ctx = x.ctx
    D, z, dt_bias, initial, final = _array(D), _array(z), _array(dt_bias), _array(initial), _array(final)
    if out is None:
        out = _like(x, given)
    y = _array(out)
    _one_context(ctx, dt, A, B, C, D, z, dt_bias, initial, final, y, sequences)
    d = _plan(("scan", softplus, x.sig, dt.sig, A.sig, B.sig, C.sig, _sig(D), _sig(z), _sig(dt_bias), _sig(initial), _sig(final), y.sig,
               _sig(sequences)), lambda: _plan_scan(
        x, A, (("D", D), ("dt_bias", dt_bias)), softplus, sequences, (("initial", initial), ("final", final)),
        (("dt", dt), ("z", z), ("y", y)), (("B", B), ("Cm", C))))
    rc = ctx.lib.b200conv_selective_scan(ctx.h, d, x.ptr, dt.ptr, A.ptr, B.ptr, C.ptr, _ptr(D), _ptr(z), _ptr(dt_bias), _ptr(initial),
                                         sequences and sequences.starts.ptr, y.ptr, _ptr(final))
    if rc:
        ctx.check(rc)
    return out


def device_selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, softplus=False, out=None):
    """One token of every sequence: x, dt, z (sequences, channels), B, C (sequences, groups, states) or (sequences,
    states); `state`, float32 (sequences, channels, states), moves on in place.  `out` may be x, dt or z."""
    x, dt, A, B, C, state = _array(x), _array(dt), _array(A), _array(B), _array(C), _array(state)
    ctx = x.ctx
    D, z, dt_bias = _array(D), _array(z), _array(dt_bias)
    if out is None:
        out = DeviceArray(ctx, x.shape, x.dtype)
    y = _array(out)
    _one_context(ctx, dt, A, B, C, D, z, dt_bias, state, y)

    def make():
        if len(x.shape) != 2:
            raise ValueError("a step takes (sequences, channels), not %s" % (x.shape,))

        def token(t):                    # one token per sequence: the sequences' stride is that of the rows
            return None if t is None else DeviceArray(t.ctx, (t.shape[0], 1) + t.shape[1:], t.dtype, (t.strides[0], t.strides[0]) + t.strides[1:], t.ptr, t.stored, t)
        return _plan_scan(token(x), A, (("D", D), ("dt_bias", dt_bias)), softplus, None, (("state", state),),
                          (("dt", token(dt)), ("z", token(z)), ("y", token(y))), (("B", token(B)), ("Cm", token(C))))
    d = _plan(("scan step", softplus, x.sig, dt.sig, A.sig, B.sig, C.sig, state.sig, _sig(D), _sig(z), _sig(dt_bias), y.sig), make)
    rc = ctx.lib.b200conv_selective_scan_step(ctx.h, d, x.ptr, dt.ptr, A.ptr, B.ptr, C.ptr, _ptr(D), _ptr(z), _ptr(dt_bias), state.ptr, y.ptr)
    if rc:
        ctx.check(rc)
    return out


def device_selective_scan_grad(dy, x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=False, initial=None, dfinal=None, sequences=None,
                               grads=None):
    """Gradients of `device_selective_scan` for dy and, where given, `dfinal`, the gradient of the final states: a dict with
    x, dt, A, B, C and, where the call has them, D, z, dt_bias and initial.  `grads`: tensors to write them into, of the inputs'
    shapes and types, which may be the inputs themselves (that of x, dt and z also dy, that of initial also dfinal); those that it
    lacks are made."""
    dy, x, dt, A, B, C = _array(dy), _array(x), _array(dt), _array(A), _array(B), _array(C)
    ctx = x.ctx
    D, z, dt_bias, initial, dfinal = _array(D), _array(z), _array(dt_bias), _array(initial), _array(dfinal)
    inputs = dict(x=x, dt=dt, A=A, B=B, C=C, D=D, z=z, dt_bias=dt_bias, initial=initial)
    grads = dict(grads or {})
    for name in grads:
        if name not in inputs:
            raise ValueError("no input is called %r" % name)
    if grads.get("initial") is not None and initial is None:
        _same("the gradient of the initial states", _array(grads["initial"]), (x.shape[0] if sequences is None else sequences.count,) + A.shape, F32)
    for name, t in inputs.items():
        if t is not None and grads.get(name) is None:
            grads[name] = DeviceArray(ctx, t.shape, t.dtype)
        elif t is None and name != "initial" and grads.get(name) is not None:
            raise ValueError("the gradient of %s without %s" % (name, name))
    g = {name: _array(grads.get(name)) for name in inputs}
    _one_context(ctx, dy, dt, A, B, C, D, z, dt_bias, initial, dfinal, sequences, *g.values())

    def make():
        for name in ("B", "C"):
            if g[name].shape != inputs[name].shape:
                raise ValueError("the gradient of %s must have shape %s, not %s" % (name, inputs[name].shape, g[name].shape))
        return _plan_scan(x, A, (("D", D), ("dt_bias", dt_bias), ("dA", g["A"]), ("dD", g["D"]), ("ddt_bias", g["dt_bias"])), softplus, sequences,
                          (("initial", initial), ("dfinal", dfinal), ("dinitial", g["initial"])),
                          (("dt", dt), ("z", z), ("dy", dy), ("dx", g["x"]), ("ddt", g["dt"]), ("dz", g["z"])),
                          (("B", B), ("Cm", C), ("dB", g["B"]), ("dCm", g["C"])))
    d = _plan(("scan grad", softplus, dy.sig, x.sig, dt.sig, A.sig, B.sig, C.sig, _sig(D), _sig(z), _sig(dt_bias), _sig(initial), _sig(dfinal),
               _sig(sequences)) + tuple(map(_sig, g.values())), make)
    rc = ctx.lib.b200conv_selective_scan_grad(
        ctx.h, d, dy.ptr, x.ptr, dt.ptr, A.ptr, B.ptr, C.ptr, _ptr(D), _ptr(z), _ptr(dt_bias), _ptr(initial), _ptr(dfinal),
        sequences and sequences.starts.ptr, g["x"].ptr, g["dt"].ptr, g["A"].ptr, g["B"].ptr, g["C"].ptr, _ptr(g["D"]), _ptr(g["z"]),
        _ptr(g["dt_bias"]), _ptr(g["initial"]))
    if rc:
        ctx.check(rc)
    return grads


# ======================================================================================
# numpy in / numpy out (float32 and float16; synchronous)
# ======================================================================================
def _upload(ctx, dtype, *arrays):
    return [None if a is None else DeviceArray.from_host(ctx, np.asarray(a), dtype) for a in arrays]


def _common_dtype(*arrays):
    dt = np.result_type(*[np.asarray(a).dtype for a in arrays if a is not None])
    if dt not in (np.dtype(np.float32), np.dtype(np.float16)):
        raise TypeError("sequence operators on host arrays handle float32 and float16, not %s" % dt)
    return dt


def layer_norm(x, gamma=None, beta=None, eps=1e-5, ctx=None):
    """Layer norm over the last axis of a host array of (rows, channels) or (sequences, tokens, channels)."""
    dt = _common_dtype(x, gamma, beta)
    ctx = ctx or shim.get_context()
    x, gamma, beta = _upload(ctx, dt, x, gamma, beta)
    return device_layer_norm(x, gamma, beta, eps).to_host()


def layer_norm_grad(dy, x, gamma=None, eps=1e-5, ctx=None):
    """Gradients (dx, dgamma, dbeta) of `layer_norm`; without gamma those of gamma and beta are float32."""
    dt = _common_dtype(dy, x, gamma)
    ctx = ctx or shim.get_context()
    dy, x, gamma = _upload(ctx, dt, dy, x, gamma)
    stats = DeviceArray(ctx, x.shape[:-1] + (2,), np.float32)
    device_layer_norm(x, gamma, None, eps, stats=stats)
    return tuple(t.to_host() for t in device_layer_norm_grad(dy, x, gamma, stats))


def causal_conv1d(x, w, bias=None, silu=False, filter_flip=True, initial=None, lengths=None, ctx=None):
    """`device_causal_conv1d` on host arrays; returns (y, final state).  `lengths`: of packed sequences."""
    dt = _common_dtype(x, w, bias, initial)
    ctx = ctx or shim.get_context()
    x, w, bias, initial = _upload(ctx, dt, x, w, bias, initial)
    seqs = None if lengths is None else Sequences(ctx, lengths)
    S, _, C = _batch(x, seqs, "a causal convolution")
    final = DeviceArray(ctx, (S, max(w.shape[-1] - 1, 0), C), dt)
    y = device_causal_conv1d(x, w, bias, silu, filter_flip, initial=initial, final=final, sequences=seqs, out=_zeros(ctx, x.shape, dt))
    return y.to_host(), final.to_host()


def causal_conv1d_grad(dy, x, w, bias=None, silu=False, filter_flip=True, initial=None, lengths=None, ctx=None):
    """Gradients (dx, dw, dbias, dinitial) of `causal_conv1d`; None for those of absent inputs, zeros in rows of no sequence."""
    dt = _common_dtype(dy, x, w, bias, initial)
    ctx = ctx or shim.get_context()
    dy, x, w, bias, initial = _upload(ctx, dt, dy, x, w, bias, initial)
    seqs = None if lengths is None else Sequences(ctx, lengths)
    grads = device_causal_conv1d_grad(dy, x, w, bias, silu, filter_flip, initial=initial, sequences=seqs, out=_zeros(ctx, x.shape, dt),
                                      dinitial=None if initial is None else DeviceArray(ctx, initial.shape, dt))
    return tuple(None if t is None else t.to_host() for t in grads)


def _scan_inputs(ctx, dt, x, dts, A, B, C, D, z, dt_bias, initial, lengths):
    x, dts, B, C, z = _upload(ctx, dt, x, dts, B, C, z)
    A, D, dt_bias, initial = _upload(ctx, np.float32, A, D, dt_bias, initial)
    return (x, dts, A, B, C), dict(D=D, z=z, dt_bias=dt_bias, initial=initial, sequences=None if lengths is None else Sequences(ctx, lengths))


def _zeros(ctx, shape, dt):
    t = DeviceArray(ctx, shape, dt)
    ctx.memset(t.ptr, 0, t.size * t.dtype.itemsize)
    return t


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=False, initial=None, lengths=None, ctx=None):
    """`device_selective_scan` on host arrays; returns (y, final states).  `lengths`: of packed sequences."""
    dtype = _common_dtype(x, dt, B, C, z)
    ctx = ctx or shim.get_context()
    args, more = _scan_inputs(ctx, dtype, x, dt, A, B, C, D, z, dt_bias, initial, lengths)
    S = more["sequences"].count if lengths is not None else args[0].shape[0]
    final = DeviceArray(ctx, (S,) + args[2].shape, np.float32)
    y = device_selective_scan(*args, softplus=softplus, final=final, out=_zeros(ctx, args[0].shape, dtype), **more)
    return y.to_host(), final.to_host()


def selective_scan_grad(dy, x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=False, initial=None, dfinal=None, lengths=None, ctx=None):
    """Gradients of `selective_scan` by input name (`device_selective_scan_grad`); zeros in rows of no sequence."""
    dtype = _common_dtype(dy, x, dt, B, C, z)
    ctx = ctx or shim.get_context()
    args, more = _scan_inputs(ctx, dtype, x, dt, A, B, C, D, z, dt_bias, initial, lengths)
    dy, = _upload(ctx, dtype, dy)
    dfinal, = _upload(ctx, np.float32, dfinal)
    named = dict(x=args[0], dt=args[1], B=args[3], C=args[4], z=more["z"])
    grads = {k: _zeros(ctx, t.shape, dtype) for k, t in named.items() if t is not None}
    grads = device_selective_scan_grad(dy, *args, softplus=softplus, dfinal=dfinal, grads=grads, **more)
    return {k: t.to_host() for k, t in grads.items()}
