"""The training operators at the edges of what a call may ask, without a GPU: what is refused, and by whom."""
import importlib

import numpy as np
import pytest

import training_ref as ref

P = "tensor-compiler-webgpu_b200"


# ---------------------------------------------------------------- positions that a gradient reaches
def _scaled_positions(pkg, through=None):
    g = pkg.ir.Graph()
    x, gain, s = g.input("x", [1, 3, 2, 4]), g.input("gain", [4]), g.input("s", [])
    pos = g.mul(g.const([0, 1, 2], [3]), s)
    if through is not None:
        pos = getattr(g, through)(pos)
    return g, x, gain, s, g.head_norm_rope(x, gain, pos)


def test_positions_have_no_gradient(pkg):
    """Positions computed from a wanted value: refused, never a silent zero."""
    g, x, gain, s, y = _scaled_positions(pkg)
    for wrt in ([s], [x, s], [s, gain]):
        with pytest.raises(pkg.autodiff.GradientError, match="positions"):
            pkg.autodiff.grad(g, [y], wrt)
    h = pkg.ir.Graph()   # the positions themselves
    pos = h.input("p", [3])
    with pytest.raises(pkg.autodiff.GradientError, match="positions"):
        pkg.autodiff.grad(h, [h.head_norm_rope(h.input("x", [1, 3, 2, 4]), h.input("g", [4]), pos)], [pos])
    pkg.autodiff.grad(g, [y], [x, gain])   # not asked for: as before


def test_positions_behind_a_stop_have_gradient_zero(pkg):
    g, x, gain, s, y = _scaled_positions(pkg, "stop_gradient")
    G = pkg.autodiff.grad(g, [y], [x, s])
    rng = np.random.default_rng(0)
    inputs = {"x": rng.standard_normal((1, 3, 2, 4)), "gain": rng.standard_normal(4), "s": 1.5, "d0": rng.standard_normal((1, 2, 3, 4))}
    vals = ref.evaluate(G.graph, inputs)
    assert not vals[G.grads[1]].any()
    a = g.nodes[y].attrs
    assert np.allclose(vals[G.grads[0]], ref.head_grad(inputs["x"], inputs["gain"], 1.5 * np.arange(3), a, inputs["d0"])["x"])


def test_stopped_inputs_of_a_node_cost_nothing(pkg):
    """Of a weight behind a stop no gradient is computed, and its gradient is zero."""
    g = pkg.ir.Graph()
    h, w = g.input("h", [5, 3]), g.input("w", [3, 4])
    y = g.linear_nll(h, g.stop_gradient(w), None, g.input("t", [5]))
    G = pkg.autodiff.grad(g, [y], [h, w])
    assert [n.attrs["wrt"] for n in G.graph.nodes if n.op == "linearNllGrad"] == ["h"]
    assert G.graph.nodes[G.grads[1]].op == "const"
