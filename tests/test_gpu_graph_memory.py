"""Memory that a captured graph uses stays with it: blocks freed while it is captured, and blocks made then and freed later."""
import numpy as np
import pytest

from sequence_util import put
from theano_b200 import sequence as Q
from theano_b200 import shim

pytestmark = pytest.mark.gpu
SHAPE = (3, 50, 64)


def fill(ctx, n):
    """Arrays of the results' size, as a program makes them after the capture."""
    return [put(ctx, np.full(SHAPE, 5.0 + i), np.float32) for i in range(n)]


def untouched(arrays):
    return all((a.to_host() == 5.0 + i).all() for i, a in enumerate(arrays))


@pytest.mark.parametrize("keep", [True, False])
def test_intermediate_results_of_a_graph_are_nobody_elses(keep):
    """Two norms in a row, the first one's result dropped inside of the captured function, the second one's kept or dropped behind it."""
    ctx = shim.Context(0)
    x = np.random.RandomState(0).standard_normal(SHAPE).astype(np.float32)
    X, gamma, out = put(ctx, x, np.float32), put(ctx, np.full(64, 3.0), np.float32), {}

    def layer():
        out["y"] = Q.device_layer_norm(Q.device_layer_norm(X), gamma)
    layer()
    want = out["y"].to_host()
    graph = ctx.capture(layer)
    if not keep:
        del out["y"]
    others = fill(ctx, 6)
    graph.launch()
    ctx.sync()
    assert untouched(others)
    if keep:
        assert np.array_equal(out["y"].to_host(), want)
    del graph
    more = fill(ctx, 6)
    assert untouched(others) and untouched(more)


def test_a_graph_gives_its_memory_back():
    """Captures and ends of graphs again and again take no more memory than the first few."""
    ctx = shim.Context(0)
    X = put(ctx, np.ones(SHAPE), np.float32)

    def layer():
        Q.device_layer_norm(Q.device_layer_norm(X))
    layer()
    seen = []
    for _ in range(6):
        graph = ctx.capture(layer)
        graph.launch()
        del graph
        ctx.sync()
        seen.append(ctx.memory_info()[0])
    assert len(set(seen[2:])) == 1, seen


def test_a_result_outlives_its_graph():
    ctx = shim.Context(0)
    X, out = put(ctx, np.arange(3 * 50 * 64).reshape(SHAPE), np.float32), {}

    def layer():
        out["y"] = Q.device_layer_norm(X)
    layer()
    want = out["y"].to_host()
    graph = ctx.capture(layer)
    graph.launch()
    ctx.sync()
    del graph
    others = fill(ctx, 4)
    assert np.array_equal(out["y"].to_host(), want) and untouched(others)
