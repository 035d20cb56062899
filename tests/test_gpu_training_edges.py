"""The training operators on the B200 at the edges of what a call may ask: confident rows, masks at the end of the
range, mixed magnitudes, memory left by other launches."""
import importlib

import numpy as np
import pytest

import training_ref as ref
from test_gpu_training_ops import check_nll, check_orth, f32, mods, nll_case, nll_loss_case, run_graph, small_graphs, within  # noqa: F401
from test_training_edges import _graphs_with_waits

pytestmark = pytest.mark.gpu
P = "tensor-compiler-webgpu_b200"
U = ref.U


# ---------------------------------------------------------------- rows whose target is all but certain
def _dz_bound(x, p, onehot):
    """dz of a row (cotangent 1) from logits off by up to ez each: p (1 - p) 2 ez, since what all logits share is
    subtracted with the maximum; the sum of exponentials off by es, which moves a probability by es p (1 - p); and
    the exponential's 2^-22, the subtraction of s, the division and the product, half a step each."""
    h, w, b = x["h"], x["w"], x["b"]
    d, V = w.shape
    ez = (ref.product_bound(d, 256) * U * (np.abs(h) @ np.abs(w) + np.abs(b)).max(1)
          + 2.0 ** -39 * d * np.abs(h).max() * np.abs(w).max())[:, None]
    es = U * (32 + 2 * (11 + V / 64) + 8)
    return (2 * ez + es) * p * (1 - p) + 8 * U * p * (1 - p) + 4 * U * (p + onehot) * 2 + 2.0 ** -39


@pytest.mark.parametrize("R,d,V,level,pieces", [(40, 16, 33, 0.0, 1), (300, 40, 300, 100.0, 1), (300, 40, 300, -1000.0, 1),
                                                (200, 40, 900, 100.0, 4), (150, 600, 500, 100.0, 1), (1500, 64, 2600, 300.0, 1)])
def test_nll_confident_rows(pkg, mods, runner, monkeypatch, R, d, V, level, pieces):
    """A row's dz, read as db under a cotangent of that row alone, where the target has a probability of 1 - 1e-2 to
    1 - 1e-13 and all logits stand far from 0: the gradient's error is of the probabilities' size, not of the logits'."""
    to = importlib.import_module(P + ".training_ops")
    if pieces > 1:
        monkeypatch.setattr(to, "DZ_BYTES", 4 * R * 256)
        assert to.nll_pieces(R, V)[1] == pieces
    graph, y, grads, x = nll_case(pkg, R, d, V, wrt="b", seed=V)
    rng = np.random.default_rng(R)
    x["w"] = f32(rng.standard_normal((d, V)))
    t = x["t"].astype(int)
    margin = np.linspace(8, 34, R)      # the target's logit above the rest's noise
    x["h"] = f32(0.05 * rng.standard_normal((R, d)) + x["w"].T[t] * (margin / (x["w"].T[t] ** 2).sum(1))[:, None])
    x["b"] = f32(level + 0.1 * rng.standard_normal(V))
    _, p, _ = ref.nll(x["h"], x["w"], x["b"], x["t"])
    onehot = np.zeros_like(p)
    onehot[np.arange(R), t] = 1.0
    bound = _dz_bound(x, p, onehot)
    for r in (0, R // 3, R // 2, 2 * R // 3, R - 1):
        x["d0"] = (np.arange(R) == r).astype(np.float64)
        db = run_graph(mods, runner, graph, x, [grads["b"]])[0]
        within(db, p[r] - onehot[r], bound[r], f"dz of row {r}")


@pytest.mark.parametrize("V", [33, 65, 300, 5000])
def test_nll_gradients_of_a_row_add_up_to_zero(pkg, mods, runner, V):
    """The mean over 8192 rows of what dz adds up to.  The forward takes an exponential against its half tile's
    maximum and one to move that sum to the row's, the backward one against the row's: at most 2^-22 each (the
    exponential's bound), and a half step for each of s, the division and the product."""
    graph, y, grads, x = nll_case(pkg, 8192, 40, V, seed=V, wrt="b")
    x["d0"][:] = 1.0
    db = run_graph(mods, runner, graph, x, [grads["b"]])[0].astype(np.float64)
    assert abs(db.sum()) / 8192 <= 3 * 2.0 ** -22 + 3 * U


# ---------------------------------------------------------------- masks at the end of the range
LOWEST = -3.4028234663852886e38


@pytest.mark.parametrize("R,train", [(6, False), (40, False), (40, True)])
@pytest.mark.parametrize("bias", [LOWEST, -3e38, -2.5e38, -2e38, -1e30])
def test_nll_target_masked_by_a_finite_bias(pkg, mods, runner, R, train, bias):
    """A target that a finite bias masks: its loss is that bias's size, also where log2(e) times it leaves the range
    of float32.  The bound: half a step of the product by log2(e), of the one by log 2 and of the result, and of both
    constants."""
    if train:
        graph, y, grads, x = nll_case(pkg, R, 24, 200, seed=R)
    else:
        graph, y, x = nll_loss_case(pkg, R, 24, 200, seed=R)
        grads = {}
    x["b"][150:] = bias
    x["t"][:] = np.arange(R) % 150
    x["t"][1] = 170
    out = run_graph(mods, runner, graph, x, [y, *grads.values()])
    want, p, _ = ref.nll(x["h"], x["w"], x["b"], x["t"])
    assert abs(out[0][1] - want[1]) <= 6 * U * abs(bias)
    keep = np.arange(R) != 1
    assert np.allclose(out[0][keep], want[keep], rtol=1e-4, atol=1e-5)
    if train:
        want = ref.nll_grad(x["h"], x["w"], x["b"], x["t"], x["d0"])
        for k, got in zip(grads, out[1:]):
            assert np.allclose(got, want[k], rtol=1e-3, atol=1e-5), k


def test_nll_every_class_at_the_lowest_float(pkg, mods, runner):
    """A bias that masks every class leaves them alike, as adding it in float32 or float64 does: p = 1 / V."""
    R, V = 40, 100
    graph, y, grads, x = nll_case(pkg, R, 24, V, seed=1, wrt="b")
    x["b"][:] = LOWEST
    loss, db = run_graph(mods, runner, graph, x, [y, grads["b"]])
    want = np.full(V, x["d0"].sum() / V)
    np.subtract.at(want, x["t"].astype(int), x["d0"])
    assert np.allclose(loss, np.log(V), rtol=8 * U)
    assert np.allclose(db, want, rtol=0, atol=(R + 8) * U * x["d0"].sum())


# ---------------------------------------------------------------- mixed magnitudes
@pytest.mark.parametrize("what", ["rows", "cotangents", "classes"])
def test_nll_mixed_magnitudes(pkg, mods, runner, what):
    """One scale for the whole of h, of W and of dz: beside its own 22 bits a value keeps 2^-39 of its operand's
    largest, and every result stands within what that makes of it."""
    case = nll_case(pkg, 130, 48, 200, seed=11)
    x = case[3]
    if what == "rows":
        x["h"] = f32(x["h"] * 10.0 ** np.linspace(-9, 1, 130)[:, None])
    elif what == "cotangents":
        x["d0"] = f32(10.0 ** np.linspace(-20, 0, 130))
    else:
        x["b"] = f32(np.linspace(-60, 0, 200))
    check_nll(mods, runner, case)


# ---------------------------------------------------------------- pieces and operands of odd shapes
@pytest.mark.parametrize("bn,ctas", [(64, 1), (128, 1), (128, 2), (256, 2)])
def test_nll_last_piece_of_one_column(pkg, mods, runner, monkeypatch, bn, ctas):
    """The vocabulary in five pieces by the forward's tile, the last one column wide: most of its tile lies beyond."""
    to = importlib.import_module(P + ".training_ops")
    # (dW's products of one column take the narrowest tile whatever it costs)
    monkeypatch.setattr(to, "F16_COST", {to.Tile(64, 1): (10 ** 6, 0, 10 ** 9, 0), to.Tile(bn, ctas): (100, 1000, 10 ** 9, 0)})
    monkeypatch.setattr(to, "DZ_BYTES", 4 * 300 * 256)
    assert to.nll_pieces(300, 1025) == (256, 5)
    check_nll(mods, runner, nll_case(pkg, 300, 70, 1025, seed=bn), runs=2)


def test_operands_that_are_one_value(pkg, mods, runner):
    """Rows and weight of a head the same square matrix: its gradient is the sum of both; the gain of a head norm its
    positions too."""
    g = pkg.ir.Graph()
    x = g.input("x", [90, 90])
    y = g.linear_nll(x, x, None, g.input("t", [90]))
    G = pkg.autodiff.grad(g, [y], [x])
    rng = np.random.default_rng(5)
    v = {"x": f32(rng.standard_normal((90, 90)) / 9), "t": rng.integers(-1, 90, 90).astype(np.float64), "d0": f32(rng.random(90))}
    loss, dx = run_graph(mods, runner, G.graph, v, [y, G.grads[0]])
    eloss, eg = ref.nll_bounds(v["x"], v["x"], None, v["t"], v["d0"])
    within(loss, ref.nll(v["x"], v["x"], None, v["t"])[0], eloss, "loss")
    want = ref.nll_grad(v["x"], v["x"], None, v["t"], v["d0"])
    within(dx, want["h"] + want["w"], eg["h"] + eg["w"] + U * (np.abs(want["h"]) + np.abs(want["w"])), "dx")
    g = pkg.ir.Graph()
    x, gain = g.input("x", [2, 16, 3, 16]), g.input("gain", [16])
    y = g.head_norm_rope(x, gain, gain)
    v = {"x": f32(rng.standard_normal((2, 16, 3, 16))), "gain": f32(1 + 0.1 * rng.standard_normal(16))}
    a = g.nodes[y].attrs
    within(run_graph(mods, runner, g, v, [y])[0], ref.head(v["x"], v["gain"], v["gain"], a),
           ref.head_bounds(v["x"], v["gain"], v["gain"], a, None)["y"], "y")


# ---------------------------------------------------------------- memory that other launches left
def test_one_off_runs_over_what_others_left_in_scratch(pkg, mods, runner):
    """The runner's scratch full of ones' bits (error words, counters, partial sums): a one-off run clears what it
    relies on, and gives what a resident program gives."""
    rt, cg = mods
    for graph, keep, x in small_graphs(pkg):
        want = run_graph(mods, runner, graph, x, keep)
        low = cg.lower(graph, matmul="tiled")
        need = max(lau.scratch_bytes for lau in low["launches"])
        ptr = runner.scratch(need)
        rt.check(rt.lib().tc_memset32(runner.ctx, ptr, 0xFFFFFFFF, need // 4))
        out = runner.run(graph, low, x)
        for i, w in zip(keep, want):
            assert np.array_equal(out["values"][i].reshape(w.shape), w), graph.nodes[i].op
    g = pkg.ir.Graph()   # many matrices on one SM each
    y = g.orthogonalize(g.input("x", [400, 20, 30]))
    x = {"x": f32(np.random.default_rng(2).standard_normal((400, 20, 30)))}
    want = run_graph(mods, runner, g, x, [y])[0]
    rt.check(rt.lib().tc_memset32(runner.ctx, runner.scratch(256), 0xFFFFFFFF, 64))
    assert np.array_equal(runner.run(g, cg.lower(g), x)["values"][y].reshape(want.shape), want)


@pytest.mark.parametrize("capture", [False, True])
def test_control_blocks_are_not_cleared_by_a_run(pkg, mods, runner, capture):
    """The words beside a resident launch's error word, which nothing reads, last through its runs: an error there
    would too."""
    rt, cg = mods
    for graph, keep in _graphs_with_waits(pkg):
        prog = rt.Program(runner, graph, cg.lower(graph, matmul="tiled"), keep=keep, capture=capture)
        try:
            rng = np.random.default_rng(3)
            for n in graph.inputs():
                prog.write(n.id, rng.random(n.shape) if n.attrs["name"] != "t" else np.zeros(n.shape))
            mark = np.array([0, 11, 12, 13], np.uint32)
            for off in prog.err_slot.values():
                rt.check(rt.lib().tc_memcpy_htod(runner.ctx, prog.errs.ptr + off, mark.ctypes.data, 16))
            runner.sync()
            for _ in range(2):
                prog.run()
            prog.check_errors()
            words = prog.errs.download(prog.errs_bytes // 4, np.uint32)
            for off in prog.err_slot.values():
                assert np.array_equal(words[off // 4:off // 4 + 4], mark)
                assert not words[off // 4 + 4:off // 4 + 16].any()   # the counters are back at zero
        finally:
            prog.free()


# ---------------------------------------------------------------- Muon, data parallel
def test_data_parallel_trainer_with_muon(pkg, runner):
    """One rank of the data-parallel trainer with Muon against the single trainer: losses as the gradient programs'
    orders of sums allow, and the weights after three steps."""
    rt = importlib.import_module(P + ".runtime")
    dp = importlib.import_module(P + ".dp")
    s, V, B = pkg.steps, 300, 3
    cfg = s.make_config(T=40, d=64, H=4, L=1, ff=128, targets="index", rope=10000.0)
    params = {n: np.asarray(v, np.float32) for n, v in s.init_params_normal(V, 0, 0.05, cfg).items()}
    step = s.build_step3b(V, B, cfg, opt=s.MUON)
    state = s.initial_state(step["names"], s.param_shapes(V, cfg), s.MUON)
    one = rt.FusedTrainer(runner, rt.fused_step(step, matmul="tiled"), params, state)
    many = dp.DPTrainer(runner, V, B, cfg, params, opt=s.MUON)
    try:
        for t in range(3):
            toks = np.random.default_rng(t).integers(0, V, (B, cfg["T"] + 1))
            x, y = s.encode_batch([list(map(int, r)) for r in toks], V, cfg["T"], "index")
            a, b = one.train(x.reshape(-1), y), many.train(x.reshape(-1), y)
            assert abs(a - b) <= 1e-4 * abs(a), t
        names = s.muon_names(step["names"])
        u, v = one.read(names), many.read(names)
        for n in names:   # three updates of norm about lr sqrt(short side) each, equal to 1 % of one
            assert np.linalg.norm(u[n] - v[n]) <= 1e-2 * s.MUON["lr"] * np.sqrt(min(s.param_shapes(V, cfg)[n])), n
    finally:
        one.destroy()
        many.destroy()


def test_node_local_runs_of_launches_with_several_outputs(pkg, mods, runner):
    """run_local: both gradients of a head norm in one launch, each read back; an operand that has no value by the
    definition (what the loss saves) is asked for by name."""
    rt, cg = mods
    from test_training_edges import _multi_output
    (nll, vals), (head, hv) = _multi_output(pkg)
    out = rt.run_local(runner, head, cg.lower(head), hv, canary=True)
    for n in head.nodes:
        if n.op == "headNormRopeGrad":
            assert np.allclose(out[n.id].reshape(n.shape), hv[n.id], rtol=1e-5, atol=1e-5)
    vals[next(n.id for n in nll.nodes if n.attrs.get("out") == "saved")] = None
    with pytest.raises(ValueError, match="no value"):
        rt.run_local(runner, nll, cg.lower(nll), vals)
