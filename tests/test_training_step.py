"""The decoder's training step with the training operators: index targets, head norm with rotation, Muon."""
import importlib

import numpy as np
import pytest

import training_ref as ref


def tiny(pkg, **kw):
    return pkg.steps.make_config(T=6, d=8, H=2, L=1, ff=16, **kw)


def batch(pkg, V, B, T, seed, targets):
    toks = np.random.default_rng(seed).integers(0, V, (B, T + 1))
    return pkg.steps.encode_batch([list(map(int, t)) for t in toks], V, T, targets)


def values(pkg, step, V, cfg, opt, seed=0):
    s = pkg.steps
    rng = np.random.default_rng(seed)
    out = {}
    for name, shape, init in s.param_spec(V, cfg):
        out[name] = (1.0 if init[0] == "ones" else 0.0) + 0.3 * rng.standard_normal(shape)
    for name, v in s.initial_state(step["names"], s.param_shapes(V, cfg), opt).items():
        out[name] = np.asarray(v, np.float64)
    out[step["cotangent"]] = np.ones(())
    return out


def test_index_targets_give_the_one_hot_loss(pkg):
    """The same loss and gradients as from one-hot rows through the logits."""
    s, V, B = pkg.steps, 11, 2
    out = []
    for targets in ("one-hot", "index"):
        cfg = tiny(pkg, targets=targets)
        step = s.build_step3b(V, B, cfg)
        x, y = batch(pkg, V, B, cfg["T"], 1, targets)
        vals = ref.evaluate(step["graph"], {**values(pkg, step, V, cfg, s.ADAM_3B), "x": x, "y": y})
        out.append([vals[step["loss"]]] + [vals[step["grads"][n]] for n in step["names"]])
    for a, b in zip(*out):
        assert np.allclose(a, b, rtol=1e-10, atol=1e-13)


def test_padding_tokens_take_no_part(pkg):
    s, V, B = pkg.steps, 11, 2
    cfg = tiny(pkg, targets="index")
    step = s.build_step3b(V, B, cfg)
    x, y = batch(pkg, V, B, cfg["T"], 1, "index")
    y[4:] = -1
    vals = ref.evaluate(step["graph"], {**values(pkg, step, V, cfg, s.ADAM_3B), "x": x, "y": y})
    each = vals[step["logits"]]
    assert each[:4].all() and not each[4:].any() and np.isclose(vals[step["loss"]], each.sum() / (B * cfg["T"]))


@pytest.mark.parametrize("name", ["b0.wq", "b0.kn", "b0.qn", "b0.w1", "head", "tok"])
def test_gradient_against_differences(pkg, name):
    s, V, B = pkg.steps, 7, 2
    cfg = tiny(pkg, targets="index", rope=100.0)
    assert "pos" not in s.param_names(V, cfg)
    step = s.build_step3b(V, B, cfg)
    x, y = batch(pkg, V, B, cfg["T"], 2, "index")
    y[3] = -1
    inputs = {**values(pkg, step, V, cfg, s.ADAM_3B), "x": x, "y": y}
    g = ref.evaluate(step["graph"], inputs)[step["grads"][name]].reshape(-1)
    fwd = s.build_forward(V, B, cfg)
    for k in np.random.default_rng(3).choice(g.size, min(g.size, 8), replace=False):
        lo, hi = (np.array(inputs[name], np.float64).reshape(-1) for _ in range(2))
        lo[k] -= 1e-5
        hi[k] += 1e-5
        d = [ref.evaluate(fwd["graph"], {**inputs, name: v})[fwd["loss"]] for v in (lo, hi)]
        assert np.isclose(g[k], (d[1] - d[0]) / 2e-5, rtol=1e-5, atol=1e-8)   # eps^2 and 2^-53 / eps


def test_muon_update_formula(pkg):
    s, V, B = pkg.steps, 7, 2
    cfg = tiny(pkg, targets="index", rope=100.0)
    opt = {**s.MUON_3B, "weightDecay": 0.1}
    step = s.build_step3b(V, B, cfg, opt=opt)
    assert s.muon_names(step["names"]) == [f"b0.{k}" for k in s.MUON_KEYS]
    x, y = batch(pkg, V, B, cfg["T"], 4, "index")
    inputs = {**values(pkg, step, V, cfg, opt), "x": x, "y": y}
    rng = np.random.default_rng(5)
    for n in s.muon_names(step["names"]):
        inputs[f"{n}.buf"] = rng.standard_normal(np.shape(inputs[n]))
    vals = ref.evaluate(step["graph"], inputs)
    for n in step["names"]:
        g, new = vals[step["grads"][n]], vals[step["outputs"][n]]
        if n in s.muon_names(step["names"]):
            buf = 0.95 * inputs[f"{n}.buf"] + g
            o = ref.newton_schulz(g + 0.95 * buf, 5, (3.4445, -4.7750, 2.0315), 1e-7)
            m, k = g.shape
            assert np.allclose(vals[step["outputs"][f"{n}.buf"]], buf)
            assert np.allclose(new, inputs[n] * (1 - 0.02 * 0.1) - 0.02 * max(1, m / k) ** 0.5 * o)
        else:   # Adam's first step: lr against the gradient's sign
            assert np.allclose(new, inputs[n] - 2e-3 * g / (np.abs(g) + 1e-8), atol=1e-9)


def test_defaults_build_the_same_graphs(pkg):
    """Without the new settings every graph is node for node what it was: no new operator in it."""
    s = pkg.steps
    step = s.build_step3b(9, 2, tiny(pkg))
    assert not any(n.op in pkg.ir.TRAINING_OPS for n in step["graph"].nodes)
    assert step["stateNames"][0] == "tok.m" and "pos" in step["names"]


@pytest.mark.gpu
@pytest.mark.parametrize("capture", [False, True])
def test_trainer_on_the_gpu(pkg, runner, capture):
    """All of them in one resident step: loss, gradients' effect and state over three steps against float64."""
    rt = importlib.import_module("tensor-compiler-webgpu_b200.runtime")
    s, V, B = pkg.steps, 300, 3
    cfg = s.make_config(T=40, d=64, H=4, L=2, ff=128, targets="index", rope=10000.0)
    opt = s.MUON_3B
    step = s.build_step3b(V, B, cfg, opt=opt)
    init = values(pkg, step, V, cfg, opt, seed=7)
    names = step["names"]
    params = {n: np.asarray(init[n] * 0.3, np.float32) for n in names}
    state = {n: np.asarray(init[n], np.float32) for n in step["stateNames"]}
    trainer = rt.FusedTrainer(runner, rt.fused_step(step, matmul="tiled"), params, state, capture=capture)
    now = {n: np.asarray(v, np.float64) for n, v in {**params, **state}.items()}
    now[step["cotangent"]] = np.ones(())
    try:
        for t in range(3):
            x, y = batch(pkg, V, B, cfg["T"], t, "index")
            y[::7] = -1
            loss = trainer.train(x, y)
            vals = ref.evaluate(step["graph"], {**now, "x": x, "y": y})
            # some 60 chained operations of a few 2^-24 each, passed on by norms and softmaxes a few times over:
            # 1e-4 of a gradient's norm; a Muon update moves by lr a step, Adam's by its lr where a gradient is
            # that near zero that its sign is not certain
            assert abs(loss - vals[step["loss"]]) <= 2e-5 * abs(vals[step["loss"]])
            got = trainer.read(names + [n for n in step["stateNames"] if n.endswith(".buf")])
            for n, v in got.items():
                want = vals[step["outputs"][n]].reshape(-1)
                if n.endswith(".buf"):
                    assert np.linalg.norm(v - want) <= 1e-4 * np.linalg.norm(want), (t, n)
                elif n in s.muon_names(names):
                    moved = np.linalg.norm(want - now[n].reshape(-1))
                    assert np.linalg.norm(v - want) <= 1e-2 * moved, (t, n)
                else:
                    assert np.linalg.norm(v - want) <= 0.05 * np.linalg.norm(want - now[n].reshape(-1)) + 1e-6, (t, n)
            for n in [*names, *step["stateNames"]]:   # the next step from the device's own values
                now[n] = trainer.read([n])[n].astype(np.float64).reshape(np.shape(now[n]))
    finally:
        trainer.destroy()


@pytest.mark.gpu
def test_data_parallel_trainer_takes_the_new_model(pkg, runner):
    """The data-parallel trainer (one rank) on the model with rotation and index targets: the gradient program's
    losses are the single trainer's, as for the plain model."""
    rt = importlib.import_module("tensor-compiler-webgpu_b200.runtime")
    dp = importlib.import_module("tensor-compiler-webgpu_b200.dp")
    s, V, B = pkg.steps, 300, 3
    cfg = s.make_config(T=40, d=64, H=4, L=1, ff=128, targets="index", rope=10000.0)
    params = {n: np.asarray(v, np.float32) for n, v in s.init_params_normal(V, 0, 0.05, cfg).items()}
    names = s.param_names(V, cfg)
    state = s.initial_state(names, s.param_shapes(V, cfg))
    one = rt.FusedTrainer(runner, rt.fused_step(s.build_step3b(V, B, cfg), matmul="tiled"), params, state)
    many = dp.DPTrainer(runner, V, B, cfg, params)
    try:
        for t in range(3):
            x, y = batch(pkg, V, B, cfg["T"], t, "index")
            a, b = one.train(x.reshape(-1), y), many.train(x.reshape(-1), y)
            # the folded program orders some sums otherwise: a few 2^-24 of the loss
            assert abs(a - b) <= 1e-5 * abs(a), t
    finally:
        one.destroy()
        many.destroy()
