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


# ---------------------------------------------------------------- numbers that a float32 does not hold
def _lower(rt, js):
    """(status, message) of the library's lowering of a graph's JSON."""
    import ctypes
    import json
    out = ctypes.c_void_p()
    status = rt.lib().tc_lower_json(json.dumps(js).encode(), b"{}", ctypes.byref(out))
    message = rt.lib().tc_last_error().decode() if status else ""
    if not status:
        rt.lib().tc_lowered_free(out)
    return status, message


def _orth(g, **kw):
    return g.orthogonalize(g.input("x", [4, 4]), **kw)


def _head(g, **kw):
    return g.head_norm_rope(g.input("x", [1, 3, 2, 4]), g.input("gain", [4]), g.input("pos", [3]), **kw)


@pytest.mark.parametrize("build", [_orth, _head])
@pytest.mark.parametrize("eps", [1e-46, 1e39, 1e300, 10 ** 400, -1e-46])
def test_eps_is_a_float32(pkg, build, eps):
    """The kernels take eps as a float32: a positive one that rounds to 0 would divide a zero norm by zero, one
    beyond the range would make every value 0."""
    rt = importlib.import_module(P + ".runtime")
    g = pkg.ir.Graph()
    with pytest.raises(pkg.ir.ShapeError, match="eps"):
        build(g, eps=eps)
    g = pkg.ir.Graph()
    y = build(g)
    js = g.to_json()
    if abs(eps) < 1e308:
        js["nodes"][y]["attrs"]["eps"] = eps
        status, message = _lower(rt, js)
        assert status == 1 and "eps" in message
        with pytest.raises(pkg.ir.ShapeError, match="eps"):
            pkg.ir.Graph.from_json(js)


@pytest.mark.parametrize("eps", [0, 0.0, 1e-45, 3e38])
def test_eps_at_the_ends_is_taken(pkg, eps):
    rt = importlib.import_module(P + ".runtime")
    for build in (_orth, _head):
        g = pkg.ir.Graph()
        build(g, eps=eps)
        assert _lower(rt, g.to_json()) == (0, "")


def test_coefficients_are_float32(pkg):
    rt = importlib.import_module(P + ".runtime")
    g = pkg.ir.Graph()
    with pytest.raises(pkg.ir.ShapeError, match="coeffs"):
        _orth(g, steps=1, coeffs=(1e39, 0.0, 0.0))
    g = pkg.ir.Graph()
    y = _orth(g, steps=1)
    js = g.to_json()
    js["nodes"][y]["attrs"]["coeffs"] = [1e39, 0, 0]
    status, message = _lower(rt, js)
    assert status == 1 and "coeffs" in message


# ---------------------------------------------------------------- graphs that are not well formed
def test_the_library_refuses_short_constants(pkg):
    """A constant with fewer values than its shape: refused when lowered (its upload ended the process)."""
    rt = importlib.import_module(P + ".runtime")
    g = pkg.ir.Graph()
    g.add(g.input("x", [5]), g.const([1, 2, 3, 4, 5], [5]))
    js = g.to_json()
    assert _lower(rt, js) == (0, "")
    for value in ([1, 2], [], [1, 2, 3, 4, 5, 6]):
        js["nodes"][1]["attrs"]["value"] = value
        status, message = _lower(rt, js)
        assert status == 1 and "const" in message


def test_the_library_refuses_deep_json(pkg):
    """Brackets without end are an error, not a stack overflow."""
    import ctypes
    rt = importlib.import_module(P + ".runtime")
    out = ctypes.c_void_p()
    for text in (b'{"nodes":' + b"[" * 200000, b'{"nodes":' * 200000):
        assert rt.lib().tc_lower_json(text, b"{}", ctypes.byref(out)) == 1
        assert b"nested" in rt.lib().tc_last_error()


# ---------------------------------------------------------------- sizes beyond any device
def _big(pkg, which):
    g = pkg.ir.Graph()
    if which == "orth-square":
        g.orthogonalize(g.input("x", [1 << 32, 1 << 32]))
    elif which == "orth-long":
        g.orthogonalize(g.input("x", [1 << 31, 4]))
    elif which == "nll-rows":
        g.linear_nll(g.input("h", [1 << 62, 1]), g.input("w", [1, 5]), None, g.input("t", [1 << 62]))
    elif which == "nll-wide":
        g.linear_nll(g.input("h", [5, 1 << 24]), g.input("w", [1 << 24, 1 << 24]), None, g.input("t", [5]))
    elif which == "head-batch":
        g.head_norm_rope(g.input("x", [1 << 33, 1 << 33, 3, 8]), g.input("gain", [8]), g.input("pos", [1 << 33]))
    else:
        g.head_norm_rope(g.input("x", [1, 1 << 33, 3, 8]), g.input("gain", [8]), g.input("pos", [1 << 33]))
    return g


@pytest.mark.parametrize("which", ["orth-square", "orth-long", "nll-rows", "nll-wide", "head-batch", "head-tokens"])
def test_sizes_beyond_any_device_are_refused(pkg, monkeypatch, which):
    """Counts that leave 64 bits (a product of two sides became 0, and the process died dividing by it) or the 31
    bits of a kernel's rows and columns: refused by both hosts."""
    rt = importlib.import_module(P + ".runtime")
    with pytest.raises(pkg.ir.ShapeError, match="beyond"):
        _big(pkg, which)
    monkeypatch.setattr(pkg.ir, "MAX_DIM", 1 << 70)
    monkeypatch.setattr(pkg.ir, "MAX_VALUES", 1 << 200)
    js = _big(pkg, which).to_json()
    status, message = _lower(rt, js)
    assert status == 1 and "beyond" in message


def test_a_gradient_of_sizes_beyond_any_device_is_refused(pkg):
    rt = importlib.import_module(P + ".runtime")
    g = pkg.ir.Graph()
    y = g.linear_nll(g.input("h", [5, 3]), g.input("w", [3, 4]), None, g.input("t", [5]))
    js = pkg.autodiff.grad(g, [y], [0]).graph.to_json()
    node = next(n for n in js["nodes"] if n["op"] == "linearNllGrad")
    node["attrs"]["d"] = 1 << 45
    status, message = _lower(rt, js)
    assert status == 1 and "sizes" in message
    with pytest.raises(pkg.ir.ShapeError, match="sizes"):
        pkg.ir.Graph.from_json(js)


# ---------------------------------------------------------------- Muon after the allreduce
def _tiny_step(pkg, opt, **kw):
    s = pkg.steps
    cfg = s.make_config(T=6, d=8, H=2, L=1, ff=32, targets="index", rope=100.0, **kw)
    return s, cfg, s.build_step3b(11, 2, cfg, opt=opt)


def test_the_update_graph_is_the_steps_update(pkg):
    """Gradients in, parameters and state out: what the whole step makes of the same gradients, for both optimizers."""
    rng = np.random.default_rng(0)
    for opt in (pkg.steps.ADAM_3B, pkg.steps.MUON):
        s, cfg, step = _tiny_step(pkg, opt)
        up = s.build_adam_graph(11, cfg, opt)
        shapes = s.param_shapes(11, cfg)
        inputs = {n: rng.standard_normal(shapes[n]) for n in step["names"]}
        inputs |= {n: np.asarray(0.9) if n.endswith("Pow") else np.abs(rng.standard_normal(sh))
                   for n, sh in s.state_spec(step["names"], shapes, opt)}
        inputs |= {"x": np.eye(11)[rng.integers(0, 11, 12)], "y": rng.integers(-1, 11, 12), step["cotangent"]: 1.0}
        vals = ref.evaluate(step["graph"], inputs)
        got = ref.evaluate(up["graph"], {**inputs, **{f"g:{n}": vals[i] for n, i in step["grads"].items()}})
        assert set(up["outputs"]) == set(step["outputs"])
        for n, i in step["outputs"].items():
            assert np.allclose(got[up["outputs"][n]], vals[i], rtol=1e-12, atol=1e-14), n


def test_data_parallel_trainer_takes_muon(pkg, monkeypatch):
    """The trainer's two programs over Muon's state: every launch reads values still in place."""
    from test_program_plan import Recorder, _replay
    rt = importlib.import_module(P + ".runtime")
    dp = importlib.import_module(P + ".dp")
    rec = Recorder(rt.lib())
    monkeypatch.setattr(rt, "lib", lambda: rec)
    monkeypatch.setattr(rt.GpuRunner, "pipeline", lambda self, code: rt.Module(hash(code) & 0xFFFF, self))
    s, cfg, step = _tiny_step(pkg, pkg.steps.MUON)
    params = s.init_params_normal(11, 0, 0.02, cfg)
    tr = dp.DPTrainer(rt.GpuRunner(1, 0), 11, 2, cfg, params, opt=s.MUON, capture=False)
    _replay(tr.grad_prog, tr.fg.graph)
    _replay(tr.adam_prog, tr.fa.graph)
    assert sorted(tr.state_names) == sorted(step["stateNames"])
    assert any(lau.kind == "orthogonalize" for lau in tr.adam_prog.launches)


def test_muon_scales_by_fan_out_over_fan_in(pkg):
    """Muon's factor is sqrt(max(1, fan-out / fan-in)), whatever way round a weight is stored: here w1 is
    [d, 4 d] and gets 2, w2 [4 d, d] gets 1."""
    s = pkg.steps
    opt = {**s.MUON, "momentum": 0.0}
    g = pkg.ir.Graph()
    shapes = {"b0.w1": [4, 16], "b0.w2": [16, 4], "b0.wq": [4, 4]}
    ids = {n: g.input(n, sh) for n, sh in shapes.items()}
    grads = {n: g.input(f"g:{n}", sh) for n, sh in shapes.items()}
    state = {n: g.input(n, sh) for n, sh in s.state_spec(list(shapes), shapes, opt)}
    out = s.muon_update(g, list(shapes), ids, grads, state, opt)
    rng = np.random.default_rng(1)
    inputs = {n.attrs["name"]: rng.standard_normal(n.shape) for n in g.inputs()} | {"beta1Pow": 0.9, "beta2Pow": 0.9}
    vals = ref.evaluate(g, inputs)
    for n, factor in (("b0.w1", 2.0), ("b0.w2", 1.0), ("b0.wq", 1.0)):
        o = ref.newton_schulz(inputs[f"g:{n}"], 5, (3.4445, -4.7750, 2.0315), 1e-7)
        assert np.allclose(inputs[n] - vals[out[n]], 0.02 * factor * o, rtol=1e-9, atol=1e-12), n
    with pytest.raises(ValueError, match="factor"):
        s.muon_update(g, list(shapes), ids, grads, state, {**opt, "factor": "fan"})


def test_optimizer_settings_without_a_kind_are_adams(pkg):
    """Adam's settings alone, as before there was a second optimizer."""
    s = pkg.steps
    cfg = s.make_config(T=4, d=8, H=2, L=1, ff=16)
    bare = {k: v for k, v in s.ADAM_3B.items() if k != "kind"}
    for build in (lambda opt: s.build_step3b(7, 1, cfg, opt=opt), lambda opt: s.build_adam_graph(7, cfg, opt)):
        assert build(bare)["graph"].to_json() == build(s.ADAM_3B)["graph"].to_json()


def test_unknown_targets_are_refused(pkg):
    """A word that is neither form of the targets built the one-hot model before."""
    s = pkg.steps
    with pytest.raises(ValueError, match="targets"):
        s.build_forward(7, 1, s.make_config(T=4, d=8, H=2, L=1, ff=16, targets="indices"))
    with pytest.raises(ValueError, match="targets"):
        s.encode_batch([[0, 1, 2, 3, 4]], 7, 4, "indices")
    s.build_forward(7, 1, s.make_config(T=4, d=8, H=2, L=1, ff=16))


# ---------------------------------------------------------------- a resident program's error words
def _graphs_with_waits(pkg):
    """(graph, kept nodes): a launch of each kind that has a control block."""
    g = pkg.ir.Graph()
    h, w, b = g.input("h", [300, 260]), g.input("w", [260, 700]), g.input("b", [700])
    y = g.linear_nll(h, w, b, g.input("t", [300]))
    G = pkg.autodiff.grad(g, [y], [h, w, b])
    yield G.graph, [y, *G.grads]
    for shape in ([3, 64, 50], [3, 200, 300]):
        g = pkg.ir.Graph()
        yield g, [g.orthogonalize(g.input("x", shape))]
    g = pkg.ir.Graph()
    yield g, [g.matmul(g.input("a", [512, 4096]), g.input("b", [4096, 512]))]


def test_replays_leave_the_error_words_alone(pkg, monkeypatch):
    """What clears a control block in reused scratch does not get a resident program's private one, so an error
    stays until it is read, however many runs come between; what waits gets it."""
    from test_program_plan import Recorder
    rt = importlib.import_module(P + ".runtime")
    cg = importlib.import_module(P + ".codegen")
    real = rt.lib()
    rec = Recorder(real)
    monkeypatch.setattr(rt.GpuRunner, "pipeline", lambda self, code: rt.Module(hash(code) & 0xFFFF, self))
    kinds = set()
    for graph, keep in _graphs_with_waits(pkg):
        low = cg.lower(graph, matmul="tiled")
        monkeypatch.setattr(rt, "lib", lambda: rec)
        prog = rt.Program(rt.GpuRunner(1, 0), graph, low, keep=keep)
        monkeypatch.setattr(rt, "lib", lambda: real)
        issued = [(c, e) for (c, e) in zip([c for lau in prog.launches for c in rt.program_calls(lau)], rec.plans[prog.plan.value])]
        lo, hi = prog.errs.ptr, prog.errs.ptr + prog.errs_bytes
        for c, (_, name, _, args, maps) in issued:
            assert c.name == name
            if c.err_offset is None:
                continue
            waits = bool(maps) or name == "tcb_orth_small"
            kinds.add((name.split("_")[1], waits))
            assert lo <= args["p"][15] < hi if waits else args["p"][15] == 0, name
    assert kinds >= {("nll", True), ("nll", False), ("orth", True), ("orth", False), ("gemm", True)}


def test_trainers_raise_a_step_whose_wait_ran_out(pkg, monkeypatch):
    """train() reads the error words after its step: a wait that ran out is not a loss like any other."""
    import ctypes
    from test_program_plan import Recorder
    rt, dp = importlib.import_module(P + ".runtime"), importlib.import_module(P + ".dp")
    words = []

    class Device(Recorder):
        def tc_download(self, h, host, nbytes, offset):
            ctypes.memset(host, 0, int(nbytes))
            if words:
                ctypes.memmove(host, (ctypes.c_uint32 * 1)(words[0]), 4)
            return 0

        def tc_memcpy_dtoh(self, ctx, host, src, nbytes):
            ctypes.memset(host, 0, int(nbytes))
            return 0

        def tc_plan_run(self, plan):
            return 0
    rec = Device(rt.lib())
    monkeypatch.setattr(rt, "lib", lambda: rec)
    monkeypatch.setattr(rt.GpuRunner, "pipeline", lambda self, code: rt.Module(hash(code) & 0xFFFF, self))
    s, cfg, step = _tiny_step(pkg, pkg.steps.MUON)
    params = s.init_params_normal(11, 0, 0.02, cfg)
    state = s.initial_state(step["names"], s.param_shapes(11, cfg), s.MUON)
    runner = rt.GpuRunner(1, 0)
    x, y = np.zeros(12 * 11), np.zeros(12)
    for tr in (rt.FusedTrainer(runner, rt.fused_step(step, matmul="tiled"), params, state, capture=False),
               dp.DPTrainer(runner, 11, 2, cfg, params, opt=s.MUON, capture=False)):
        words[:] = []
        assert tr.train(x, y) == 0.0
        words[:] = [7]
        with pytest.raises(rt.TcError, match="ran out"):
            tr.train(x, y)


@pytest.fixture(scope="module")
def check_program(pkg, tmp_path_factory):
    import os
    import subprocess
    from conftest import ROOT
    rt = importlib.import_module(P + ".runtime")
    rt.lib()
    exe = str(tmp_path_factory.mktemp("check") / "check_program")
    lib = os.path.join(ROOT, P)
    subprocess.run(["gcc", "-O1", "-rdynamic", "-o", exe, os.path.join(ROOT, "tests", "c", "check_program.c"),
                    "-I" + os.path.join(ROOT, "include"), "-L" + lib, "-ltcb200", "-Wl,-rpath," + lib], check=True)
    return exe


def test_the_library_clears_whole_control_blocks(pkg, check_program, tmp_path):
    """tc_program_check after a wait that ran out: every arrival counter is zeroed with the error words, so the next
    run does not take a part of a tile for the last; and no planned call clears a private block before."""
    import json
    import os
    import subprocess
    for k, (graph, keep) in enumerate(_graphs_with_waits(pkg)):
        path = tmp_path / f"{k}.json"
        path.write_text(json.dumps(graph.to_json()))
        r = subprocess.run([check_program, str(path), ",".join(map(str, keep))], capture_output=True, text=True, timeout=60,
                           env={**os.environ, "TCB_KERNEL_CACHE": str(tmp_path / "cubins")})
        assert r.returncode == 0, r.stderr
        *calls, last = r.stdout.splitlines()
        rt = importlib.import_module(P + ".runtime")
        for line in calls:
            _, name, off = line.split()
            assert name not in rt.CLEARING or off == "-1", line
        assert any(int(line.split()[2]) >= 0 for line in calls)
        words = last.split()
        assert words[:4] == ["check", "5", "left", "0"] and words[-2:] == ["again", "0"], last


# ---------------------------------------------------------------- launches with several outputs, by every host
def _multi_output(pkg):
    """(graph, values of its nodes in 64 bits): a loss with its gradients, a head norm with both of its."""
    rng = np.random.default_rng(4)
    g = pkg.ir.Graph()
    h, w = g.input("h", [30, 8]), g.input("w", [8, 20])
    y = g.linear_nll(h, w, None, g.input("t", [30]))
    G = pkg.autodiff.grad(g, [y], [h, w]).graph
    yield G, ref.evaluate(G, {"h": rng.standard_normal((30, 8)), "w": rng.standard_normal((8, 20)), "t": rng.integers(0, 20, 30),
                              "d0": rng.random(30)})
    g = pkg.ir.Graph()
    x, gain = g.input("x", [2, 5, 3, 8]), g.input("gain", [8])
    G = pkg.autodiff.grad(g, [g.head_norm_rope(x, gain, g.input("pos", [5]))], [x, gain]).graph
    yield G, ref.evaluate(G, {"x": rng.standard_normal((2, 5, 3, 8)), "gain": rng.standard_normal(8), "pos": np.arange(5),
                              "d0": rng.standard_normal((2, 3, 5, 8))})


def test_timed_programs_of_launches_with_several_outputs(pkg, monkeypatch):
    """A graph timed (timing.graph_program): every output of a launch goes to its own node's buffer."""
    from test_program_plan import Recorder
    rt, cg, timing = (importlib.import_module(f"{P}.{m}") for m in ("runtime", "codegen", "timing"))
    rec = Recorder(rt.lib())
    for G, vals in _multi_output(pkg):
        low = cg.lower(G)
        prog = timing.graph_program(G, low, {n.attrs["name"]: vals[n.id] for n in G.inputs()}, [])
        with monkeypatch.context() as m:
            m.setattr(rt, "lib", lambda: rec)
            m.setattr(rt.GpuRunner, "pipeline", lambda self, code: rt.Module(1, self))
            bench = object.__new__(timing.Bench)
            bench.runner, bench.counts = rt.GpuRunner(1, 0), {}
            bench.pipeline, bench._count = bench.runner.pipeline, lambda what: None
            made = bench.prepare(prog)
        multi = [lau for lau in low["launches"] if len(getattr(lau, "nodes", [])) > 1]
        assert multi
        used = {v for e in rec.plans[made["plan"].value] for v in (e[3]["out"], *e[3]["p"])}
        for lau in multi:
            for i in lau.nodes:
                assert made["buffers"][i].ptr in used


# ---------------------------------------------------------------- the backward's logits are the forward's
@pytest.mark.parametrize("R,d,V", [(1, 16, 2), (64, 64, 65), (150, 600, 500), (33, 1030, 300), (40, 3000, 90), (4095, 256, 8192),
                                   (8192, 1024, 50001), (16384, 17, 131072), (70000, 64, 600), (16, 64, 1 << 24), (200000, 32, 700),
                                   (2048, 64, 131072), (131073, 8, 257)])
def test_logits_are_computed_again_by_the_same_tiles(pkg, R, d, V):
    """dz subtracts the maximum that the forward found, so its logits have to be the forward's bit for bit: the same
    tile, and where K is divided among CTAs the same division (several pieces are never divided)."""
    cg, to = importlib.import_module(P + ".codegen"), importlib.import_module(P + ".training_ops")
    g = pkg.ir.Graph()
    h, w = g.input("h", [R, d]), g.input("w", [d, V])
    y = g.linear_nll(h, w, None, g.input("t", [R]))
    G = pkg.autodiff.grad(g, [y], [h, w]).graph
    calls = [c for lau in cg.lower(G)["launches"] for c in lau.calls]
    (logits,) = [c for c in calls if c.name.startswith("tcb_nll_logits")]
    dz = [c for c in calls if c.name.startswith("tcb_nll_dz")]
    tile = logits.name.rsplit("_", 1)[1]
    assert len(dz) == to.nll_pieces(R, V)[1] and all(c.name.rsplit("_", 1)[1] == tile for c in dz)
    if len(dz) == 1:
        assert dz[0].grid == logits.grid and dz[0].params[:3] == logits.params[:3]
    else:
        ctas = 2 if tile.endswith("x2") else 1
        for c in (logits, *dz):
            M, N = c.params[0] & 0xFFFFFFFF, c.params[0] >> 32
            assert c.params[2] & 0xFFFFFFFF == to.f16_tiles(M, N, to.Tile(int(tile.split("x")[0]), ctas), False)
