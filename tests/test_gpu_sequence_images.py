"""The scan of channels-last images whose channels are padded in memory: the bits of a call on the same rows without pads."""
import numpy as np
import pytest

from sequence_util import put
from theano_b200 import sequence as Q
from theano_b200 import shim

pytestmark = pytest.mark.gpu
F32 = np.dtype(np.float32)


@pytest.mark.parametrize("C", [6, 8])
def test_scan_and_its_gradient(C):
    ctx = shim.get_context(0)
    rs = np.random.RandomState(0)
    S, H, W, N = 2, 5, 7, 4
    images = {k: rs.standard_normal((S, C, H, W)).astype(np.float32) for k in ("x", "dt", "z", "dy")}
    A, B, Cm = -np.exp(rs.standard_normal((C, N))), rs.standard_normal((S, H * W, N)), rs.standard_normal((S, H * W, N))
    rest = [put(ctx, a, F32) for a in (A, B, Cm)]

    def calls(x, dt, z, dy):
        y = Q.device_selective_scan(x, dt, *rest, z=z, softplus=True, out=Q.DeviceArray(ctx, (S, H * W, C), F32))
        grads = {k: Q.DeviceArray(ctx, (S, H * W, C), F32) for k in ("x", "dt", "z")}
        g = Q.device_selective_scan_grad(dy, x, dt, *rest, z=z, softplus=True, grads=grads)
        return [y.to_host()] + [g[k].to_host() for k in sorted(g)]
    flat = calls(**{k: put(ctx, a.reshape(S, C, -1).transpose(0, 2, 1), F32) for k, a in images.items()})
    got = calls(**{k: shim.DeviceTensor.from_host(ctx, a, "nhwc") for k, a in images.items()})
    assert all(np.array_equal(a, b) for a, b in zip(got, flat))
