"""Tensors and tolerances of the sequence operators' tests.

A rounding to a type is off by at most half a step of the value; a float32 sum of n terms by at most n * 2^-24 of the sum of their
magnitudes.  `close` allows the half step and a slack that each test derives from such sums.

The scan's decays below 2^-126 are zero (the hardware's exponential has no subnormal results): such a decay, and every product with it, is
off by less than 2^-126 times its other factors and the number of terms that it enters, below 2^26 for the tests' inputs (values up to 2^4,
five of them in a product, at most 700 tokens): TINY."""
import numpy as np

from theano_b200 import sequence as Q

DTYPES = {"f32": np.dtype(np.float32), "f16": np.dtype(np.float16), "bf16": Q.BFLOAT16}
HALF = {DTYPES["f32"]: 2.0 ** -24, DTYPES["f16"]: 2.0 ** -11, DTYPES["bf16"]: 2.0 ** -8}
E32 = 2.0 ** -24
TINY = 2.0 ** -100
SENTINEL = 77.0


def rounded(a, dtype):
    """The values as the type holds them, as float32."""
    a = np.asarray(a, np.float32)
    return Q.from_bfloat16(Q.to_bfloat16(a)) if dtype == Q.BFLOAT16 else a.astype(dtype).astype(np.float32)


def normal(rs, shape, dtype, scale=1.0):
    return rounded(rs.standard_normal(shape) * scale, dtype)


def close(got, want, dtype, slack):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (got.shape, want.shape)
    assert np.isfinite(got).all()
    slack = np.broadcast_to(slack, want.shape)
    over = np.abs(got - want) - (HALF[np.dtype(dtype)] * (np.abs(want) + slack) + slack + TINY + (2.0 ** -25 if dtype == np.float16 else 0))
    assert (over <= 0).all(), "off by %.3g at %s: %.9g, not %.9g, slack %.3g" % (
        np.abs(got - want).flat[over.argmax()], np.unravel_index(over.argmax(), over.shape), got.flat[over.argmax()], want.flat[over.argmax()],
        slack.flat[over.argmax()])


def put(ctx, a, dtype):
    return Q.DeviceArray.from_host(ctx, np.asarray(a, np.float32), "bfloat16" if dtype == Q.BFLOAT16 else dtype)


def framed(ctx, shape, dtype, pad=5, value=None):
    """A tensor inside of a wider one filled with sentinels: (the wider one, the view).  `pad` columns on each side and a row
    behind; `value`: what the view holds."""
    lead = shape[:-1]
    wide = np.full((lead[0], lead[1] + 1, shape[-1] + 2 * pad) if len(shape) == 3 else (lead[0] + 1, shape[-1] + 2 * pad), SENTINEL, np.float32)
    inner = (slice(None), slice(0, lead[1]), slice(pad, pad + shape[-1])) if len(shape) == 3 else (slice(0, lead[0]), slice(pad, pad + shape[-1]))
    if value is not None:
        wide[inner] = value
    w = put(ctx, wide, dtype)
    return w, w[inner]


def frame_intact(w, shape, pad=5):
    a = w.to_host()
    inner = (slice(None), slice(0, shape[1]), slice(pad, pad + shape[-1])) if len(shape) == 3 else (slice(0, shape[0]), slice(pad, pad + shape[-1]))
    a[inner] = SENTINEL
    return (a == SENTINEL).all()
