"""Tensors of the sequence operators that no longer hold memory, and pad channels of inputs; no GPU needed."""
import numpy as np
import pytest

from test_sequence_refusals import _Context, arr
from theano_b200 import sequence as Q
from theano_b200 import shim


class _Images(_Context):
    def padded_channels(self, c, dtype):
        return -(-c // 8) * 8


@pytest.fixture()
def ctx():
    return _Images()


def test_a_freed_tensor_is_no_absent_one(ctx):
    """Optional arguments that were freed are refused, not left out of the computation."""
    x, w, states = arr(ctx, 2, 9, 8), arr(ctx, 8, 4), arr(ctx, 2, 3, 8)

    def freed(*shape):
        t = arr(ctx, *shape)
        t.free()
        return t
    scan = [x, x, arr(ctx, 8, 4), arr(ctx, 2, 9, 4), arr(ctx, 2, 9, 4)]
    token = [arr(ctx, 2, 8), arr(ctx, 2, 8), arr(ctx, 8, 4), arr(ctx, 2, 4), arr(ctx, 2, 4), arr(ctx, 2, 8, 4)]
    stats = arr(ctx, 2, 9, 2)
    for call in (lambda: Q.device_layer_norm(x, freed(8)), lambda: Q.device_layer_norm(x, beta=freed(8)), lambda: Q.device_layer_norm(x, residual=freed(2, 9, 8)),
                 lambda: Q.device_layer_norm(x, total=freed(2, 9, 8)), lambda: Q.device_layer_norm(x, stats=freed(2, 9, 2)),
                 lambda: Q.device_layer_norm_grad(x, x, freed(8), stats),
                 lambda: Q.device_layer_norm_grad(x, x, None, stats, dtotal=freed(2, 9, 8)), lambda: Q.device_layer_norm_grad(x, x, None, stats, dgamma=freed(8)),
                 lambda: Q.device_causal_conv1d(x, w, freed(8)), lambda: Q.device_causal_conv1d(x, w, initial=freed(2, 3, 8)),
                 lambda: Q.device_causal_conv1d(x, w, final=freed(2, 3, 8)), lambda: Q.device_causal_conv1d_grad(x, x, w, initial=freed(2, 3, 8)),
                 lambda: Q.device_causal_conv1d_grad(x, x, w, dinitial=freed(2, 3, 8)), lambda: Q.device_causal_conv1d_grad(x, x, w, dw=freed(8, 4)),
                 lambda: Q.device_causal_conv1d_step(token[0], states, w, freed(8)),
                 lambda: Q.device_selective_scan(*scan, D=freed(8)), lambda: Q.device_selective_scan(*scan, z=freed(2, 9, 8)),
                 lambda: Q.device_selective_scan(*scan, dt_bias=freed(8)), lambda: Q.device_selective_scan(*scan, initial=freed(2, 8, 4)),
                 lambda: Q.device_selective_scan(*scan, final=freed(2, 8, 4)), lambda: Q.device_selective_scan_step(*token, D=freed(8)),
                 lambda: Q.device_selective_scan_grad(x, *scan, dfinal=freed(2, 8, 4)), lambda: Q.device_selective_scan_grad(x, *scan, D=arr(ctx, 8), grads=dict(D=freed(8)))):
        with pytest.raises(ValueError, match="freed"):
            call()
    assert not ctx.lib.calls


def test_views_of_a_freed_tensor(ctx):
    """Views made before and after, views of views, rows of images: none of them reaches memory that is another's by now, or address 0."""
    a = arr(ctx, 2, 12, 8)
    view = a[:, 2:11]
    deep = view[:, 1:9][:, :8]
    Q.device_layer_norm(view, out=arr(ctx, 2, 9, 8))
    image = shim.DeviceTensor(ctx, (2, 6, 3, 3), np.float32, "nhwc")
    rows = Q.DeviceArray.rows_of(image)
    Q.device_layer_norm(rows, out=arr(ctx, 2, 9, 6))
    calls = list(ctx.lib.calls)
    a.free()
    image.free()
    for call in (lambda: a[:, 1:], lambda: view[:, 1:], lambda: deep[0], lambda: Q.device_layer_norm(view), lambda: Q.device_layer_norm(deep),
                 lambda: Q.device_layer_norm(rows), lambda: Q.device_layer_norm(image), lambda: view.to_host(), lambda: a.to_host()):
        with pytest.raises(ValueError, match="freed"):
            call()
    assert ctx.lib.calls == calls


def test_wrapped_memory_and_empty_tensors_are_not_freed_ones(ctx):
    mine = Q.DeviceArray(ctx, (2, 9, 8), np.float32, (72, 8, 1), _ptr=1 << 20)
    Q.device_layer_norm(mine, out=mine[:, :9])
    empty = Q.DeviceArray(ctx, (0, 9, 8), np.float32, (72, 8, 1), _ptr=0)
    Q.device_layer_norm(empty, out=Q.DeviceArray(ctx, (0, 9, 8), np.float32))
    assert len(ctx.lib.calls) == 2


def test_pad_channels_of_a_scans_inputs(ctx):
    """Inputs may be images with pad channels; results, whose pad channels a scan does not write, may not: in steps neither."""
    padded = lambda: Q.DeviceArray(ctx, (2, 9, 6), np.float32, (72, 8, 1), 1 << 20, 8)  # noqa: E731
    A, bc = arr(ctx, 6, 4), lambda: arr(ctx, 2, 9, 4)  # noqa: E731
    Q.device_selective_scan(padded(), padded(), A, bc(), bc(), z=padded(), out=arr(ctx, 2, 9, 6))
    own = dict(x=arr(ctx, 2, 9, 6), dt=arr(ctx, 2, 9, 6), z=arr(ctx, 2, 9, 6))
    Q.device_selective_scan_grad(padded(), padded(), padded(), A, bc(), bc(), z=padded(), grads=own)
    token, states, b = padded()[:, 0], arr(ctx, 2, 6, 4), arr(ctx, 2, 4)
    Q.device_selective_scan_step(token, token, A, b, b, states, z=token, out=arr(ctx, 2, 6))
    assert len(ctx.lib.calls) == 3
    for call in (lambda: Q.device_selective_scan(padded(), padded(), A, bc(), bc(), out=padded()),
                 lambda: Q.device_selective_scan_grad(padded(), padded(), padded(), A, bc(), bc(), z=padded(), grads=dict(own, dt=padded())),
                 lambda: Q.device_selective_scan_grad(padded(), padded(), padded(), A, bc(), bc(), z=padded(), grads=dict(own, z=padded())),
                 lambda: Q.device_selective_scan_grad(padded(), padded(), padded(), A, bc(), bc(), grads=dict(x=padded())),
                 lambda: Q.device_selective_scan_step(token, token, A, b, b, states, out=padded()[:, 1])):
        with pytest.raises(ValueError, match="pad channels"):
            call()
    assert len(ctx.lib.calls) == 3
