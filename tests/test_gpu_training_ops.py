"""The training operators on the B200, against float64 formulas with bounds from counted roundings."""
import importlib

import numpy as np
import pytest

import training_ref as ref

pytestmark = pytest.mark.gpu
P = "tensor-compiler-webgpu_b200"


@pytest.fixture(scope="module")
def mods(pkg):
    return importlib.import_module(P + ".runtime"), importlib.import_module(P + ".codegen")


def run_graph(mods, runner, graph, inputs, keep, capture=False, runs=1):
    """A resident program of the fused graph; every kept value after `runs` runs."""
    rt, cg = mods
    pkg = importlib.import_module(P)
    f = pkg.fuse.fuse(graph, keep=keep)
    low = cg.lower_fused(f.graph, matmul="tiled", keep=[f.index[i] for i in keep])
    prog = rt.Program(runner, f.graph, low, keep=[f.index[i] for i in keep], batch=True, capture=capture)
    try:
        for n in f.graph.inputs():
            prog.write(n.id, inputs[n.attrs["name"]])
        for _ in range(runs):
            prog.run()
        prog.check_errors()
        return [prog.read(f.index[i]).reshape(graph.shape(i)) for i in keep]
    finally:
        prog.free()


def f32(x):
    return np.asarray(x, np.float32).astype(np.float64)


def within(got, want, bound, what):
    """A result is a float32: beside its bound, half of its own step and, where the exact value lies below
    2^-126, half of the subnormal step 2^-149 for each of the two scalings that made it."""
    d = np.abs(got.astype(np.float64) - want)
    bound = bound + ref.U * np.abs(want) + 2.0 ** -149
    bad = ~(d <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} values off, worst {np.nanmax(d / np.maximum(bound, 1e-300)):.3g} of the bound"


# ---------------------------------------------------------------- cross entropy
def nll_case(pkg, R, d, V, bias=True, wrt="hwb", seed=0, scale=1.0):
    g = pkg.ir.Graph()
    ids = {"h": g.input("h", [R, d]), "w": g.input("w", [d, V])}
    if bias:
        ids["b"] = g.input("b", [V])
    y = g.linear_nll(ids["h"], ids["w"], ids.get("b"), g.input("t", [R]))
    G = pkg.autodiff.grad(g, [y], [ids[k] for k in wrt if k in ids])
    rng = np.random.default_rng(seed)
    x = {"h": f32(rng.standard_normal((R, d)) * scale), "w": f32(rng.standard_normal((d, V)) * 2 / np.sqrt(d)),
         "t": rng.integers(0, V, R).astype(np.float64), "d0": f32(rng.random(R) / R)}
    if bias:
        x["b"] = f32(rng.standard_normal(V) * 0.1)
    return G.graph, y, dict(zip([k for k in wrt if k in ids], G.grads)), x


def check_nll(mods, runner, case, **kw):
    graph, y, grads, x = case
    out = run_graph(mods, runner, graph, x, [y, *grads.values()], **kw)
    a = (x["h"], x["w"], x.get("b"), x["t"])
    loss, _, _ = ref.nll(*a)
    eloss, eg = ref.nll_bounds(*a, x["d0"])
    within(out[0], loss, eloss, "loss")
    want = ref.nll_grad(*a, x["d0"])
    for k, got in zip(grads, out[1:]):
        within(got, want[k], eg[k], f"d{k}")
    return out


@pytest.mark.parametrize("R,d,V", [(1, 1, 1), (1, 16, 2), (5, 3, 7), (64, 64, 65), (128, 32, 256), (129, 33, 257),
                                   (100, 70, 513), (300, 256, 1000), (1000, 96, 4099), (33, 1030, 300), (2500, 8, 2500)])
def test_nll(pkg, mods, runner, R, d, V):
    check_nll(mods, runner, nll_case(pkg, R, d, V, seed=R))


@pytest.mark.parametrize("wrt", ["h", "w", "b", "hb", "wb"])
def test_nll_some_gradients(pkg, mods, runner, wrt):
    check_nll(mods, runner, nll_case(pkg, 200, 40, 300, wrt=wrt))


def test_nll_without_bias(pkg, mods, runner):
    check_nll(mods, runner, nll_case(pkg, 200, 40, 300, bias=False))


@pytest.mark.parametrize("share", [0.3, 1.0])
def test_nll_padding_rows(pkg, mods, runner, share):
    """Rows with no class: loss 0, no gradient, whatever their rows of h hold; a target of V or above too."""
    case = nll_case(pkg, 300, 40, 300, seed=1)
    x = case[3]
    out = np.random.default_rng(2).random(300) < share
    x["t"][out] = np.resize([-1.0, 300.0, -7.0, 1e9, np.nan], out.sum())
    plain = check_nll(mods, runner, case)
    x["h"][out] = np.resize([np.nan, np.inf, -np.inf, 3e38], (out.sum(), 40))
    again = run_graph(mods, runner, case[0], x, [case[1], *case[2].values()])
    for a, b in zip(plain, again):
        assert np.array_equal(a, b)
    assert not plain[0][out].any() and not plain[1][out].any()


def test_nll_masked_classes(pkg, mods, runner):
    """A bias of -inf takes classes out of the vocabulary (whole tiles of them); the lowest float does too."""
    case = nll_case(pkg, 150, 32, 1500, seed=3)
    x = case[3]
    x["b"][100:1300] = -np.inf
    x["b"][1400:] = -3.4028234663852886e38
    x["t"] = np.random.default_rng(4).integers(0, 100, 150).astype(np.float64)
    graph, y, grads, _ = case
    out = run_graph(mods, runner, graph, x, [y, *grads.values()])
    live = np.r_[0:100, 1300:1400]
    small = {"h": x["h"], "w": x["w"][:, live], "b": x["b"][live], "t": x["t"]}
    eloss, eg = ref.nll_bounds(*small.values(), x["d0"])
    within(out[0], ref.nll(*small.values())[0], eloss, "loss")
    want = ref.nll_grad(*small.values(), x["d0"])
    within(out[1], want["h"], eg["h"], "dh")
    within(out[2][:, live], want["w"], eg["w"], "dw")
    within(out[3][live], want["b"], eg["b"], "db")
    dead = np.setdiff1d(np.arange(1500), live)
    assert not out[2][:, dead].any() and not out[3][dead].any()


def test_nll_target_is_masked(pkg, mods, runner):
    """A target whose logit is -inf: the loss is inf, as -log 0."""
    case = nll_case(pkg, 4, 16, 20, seed=5)
    x = case[3]
    x["b"][7] = -np.inf
    x["t"][:] = [7, 1, 2, 3]
    out = run_graph(mods, runner, case[0], x, [case[1]])[0]
    assert out[0] == np.inf and np.isfinite(out[1:]).all()


def test_nll_nan_stays_in_its_row(pkg, mods, runner):
    case = nll_case(pkg, 140, 24, 100, seed=6)
    x = case[3]
    good = run_graph(mods, runner, case[0], x, [case[1], case[2]["h"]])
    x["h"][17, 3] = np.nan
    bad = run_graph(mods, runner, case[0], x, [case[1], case[2]["h"]])
    rest = np.arange(140) != 17
    assert np.isnan(bad[0][17]) and np.isnan(bad[1][17]).all()
    # the row's value leaves the scale of the others as it was unless it held the largest
    assert np.allclose(bad[0][rest], good[0][rest], rtol=1e-5) and np.allclose(bad[1][rest], good[1][rest], atol=1e-7)


@pytest.mark.parametrize("sh,sw,sg", [(1e-20, 1e20, 1.0), (1e15, 1e-15, 1e-30), (1.0, 1.0, 1e25), (1e-42, 1.0, 1.0)])
def test_nll_magnitudes(pkg, mods, runner, sh, sw, sg):
    """Scales are powers of two taken from the data: extreme operands keep float32's relative accuracy."""
    case = nll_case(pkg, 130, 48, 200, seed=7)
    x = case[3]
    x["h"], x["w"], x["d0"] = f32(x["h"] * sh), f32(x["w"] * sw), f32(x["d0"] * sg)
    check_nll(mods, runner, case)


@pytest.mark.parametrize("sh,sw,sg,wrt", [(1e36, 1e-36, 1e-30, "hwb"), (1e-36, 1e36, 1e30, "wb"), (1e36, 1e-36, 1.0, "w")])
def test_nll_magnitudes_that_cancel(pkg, mods, runner, sh, sw, sg, wrt):
    """The scale of h, or of its gradient's operand, alone takes the sums out of the range; both together do not."""
    case = nll_case(pkg, 70, 33, 90, seed=9, wrt=wrt)
    x = case[3]
    x["h"], x["w"], x["d0"] = f32(x["h"] * sh), f32(x["w"] * sw), f32(x["d0"] * sg)
    check_nll(mods, runner, case)


def test_nll_pieces(pkg, mods, runner, monkeypatch):
    """The vocabulary in several pieces: dh is added up over them, dW and db land at their columns."""
    to = importlib.import_module(P + ".training_ops")
    monkeypatch.setattr(to, "DZ_BYTES", 4 * 200 * 256)
    assert to.nll_pieces(200, 900) == (256, 4)   # the last piece narrower than a block
    check_nll(mods, runner, nll_case(pkg, 200, 40, 900, seed=8))


@pytest.mark.parametrize("V", [2, 5, 32])
def test_nll_few_classes_add_up_to_one(pkg, mods, runner, V):
    """A row's probabilities add up to 1, so its gradients of the logits to 0: what each row has left are a few
    roundings of half a step (2^-25) that do not lean to one side.  Their mean over 8192 rows has a standard deviation
    below 4 * 2^-25 / 90 = 1.3e-9; a lean of the exponential itself, 4e-8, would stand out."""
    case = nll_case(pkg, 8192, 40, V, seed=V)
    x = case[3]
    x["d0"][:] = 1.0
    out = run_graph(mods, runner, case[0], x, [case[1], *case[2].values()])
    assert abs(out[3].astype(np.float64).sum()) / 8192 <= 1e-8


def test_nll_is_deterministic_and_replays(pkg, mods, runner):
    case = nll_case(pkg, 700, 80, 3001, seed=9)
    keep = [case[1], *case[2].values()]
    a = run_graph(mods, runner, case[0], case[3], keep)
    b = run_graph(mods, runner, case[0], case[3], keep, capture=True, runs=3)
    for u, v in zip(a, b):
        assert np.array_equal(u, v)


# ---------------------------------------------------------------- head norm and rotation
def head_case(pkg, B, T, H, D, rot, inter=False, shared=True, first=True, wrt=("x", "gain"), start=0, seed=0):
    g = pkg.ir.Graph()
    x, gain = g.input("x", [B, T, H, D]), g.input("gain", [D])
    y = g.head_norm_rope(x, gain, g.input("pos", [T] if shared else [B, T]), rotary=rot, interleaved=inter, heads_first=first)
    G = pkg.autodiff.grad(g, [y], [{"x": x, "gain": gain}[k] for k in wrt])
    rng = np.random.default_rng(seed)
    pos = start + (np.arange(T) if shared else rng.integers(0, 2000, (B, T)))
    v = {"x": f32(rng.standard_normal((B, T, H, D))), "gain": f32(1 + 0.1 * rng.standard_normal(D)), "pos": f32(pos),
         "d0": f32(rng.standard_normal(g.shape(y)))}
    return G.graph, y, dict(zip(wrt, G.grads)), v


def check_head(mods, runner, case, **kw):
    graph, y, grads, v = case
    out = run_graph(mods, runner, graph, v, [y, *grads.values()], **kw)
    a = graph.nodes[y].attrs
    want = {"y": ref.head(v["x"], v["gain"], v["pos"], a), **ref.head_grad(v["x"], v["gain"], v["pos"], a, v["d0"])}
    e = ref.head_bounds(v["x"], v["gain"], v["pos"], a, v["d0"])
    for k, got in zip(["y", *grads], out):
        within(got, want[k], e[k], k)
    return out


@pytest.mark.parametrize("B,T,H,D,rot", [(1, 1, 1, 1, 0), (1, 1, 4, 64, 64), (2, 3, 1, 2, 2), (2, 3, 5, 7, 6), (3, 101, 5, 80, 40),
                                         (2, 33, 3, 48, 24), (1, 9, 2, 256, 128), (1, 5, 3, 512, 512), (2, 17, 7, 128, 0),
                                         (9, 1, 33, 32, 32), (40, 3, 2, 64, 64), (1, 700, 1, 96, 8)])
@pytest.mark.parametrize("inter,shared,first", [(False, True, True), (True, False, True), (False, False, False)])
def test_head(pkg, mods, runner, B, T, H, D, rot, inter, shared, first):
    check_head(mods, runner, head_case(pkg, B, T, H, D, rot, inter, shared, first, seed=D))


@pytest.mark.parametrize("wrt", [("x",), ("gain",), ("gain", "x")])
def test_head_some_gradients(pkg, mods, runner, wrt):
    check_head(mods, runner, head_case(pkg, 2, 50, 3, 64, 64, wrt=wrt))


@pytest.mark.parametrize("start", [1000, 1000000, 16000000])
def test_head_far_positions(pkg, mods, runner, start):
    check_head(mods, runner, head_case(pkg, 1, 40, 2, 128, 128, start=start))


def test_head_fractional_and_negative_positions(pkg, mods, runner):
    case = head_case(pkg, 1, 30, 2, 32, 32)
    case[3]["pos"] = f32(np.linspace(-700.3, 900.7, 30))
    check_head(mods, runner, case)


def test_head_zero_rows(pkg, mods, runner):
    """A head of zeros stays zero (eps keeps the root from dividing by zero) and hands on a finite gradient."""
    case = head_case(pkg, 1, 4, 2, 16, 16)
    case[3]["x"][0, 1] = 0.0
    out = check_head(mods, runner, case)
    assert not out[0][0, :, 1].any() and np.isfinite(out[1]).all()


def test_head_unaligned_operands(pkg, mods, runner):
    """Operands that start 4 bytes off a 16-byte boundary take the scalar path, with the same values."""
    rt, cg = mods
    case = head_case(pkg, 2, 50, 3, 64, 64)
    graph, y, grads, v = case
    keep = [y, *grads.values()]
    want = run_graph(mods, runner, graph, v, keep)
    f = pkg.fuse.fuse(graph, keep=keep)
    low = cg.lower_fused(f.graph, keep=[f.index[i] for i in keep])
    bufs, place = [], {}
    for n in f.graph.nodes:
        if n.op == "input" or n.id in [f.index[i] for i in keep]:
            b = rt.DeviceBuffer(runner, 4 * pkg.ir.size(n.shape) + 16)
            bufs.append(b)
            place[n.id] = b.ptr + 4
    prog = rt.Program(runner, f.graph, low, keep=[f.index[i] for i in keep], place=place)
    try:
        for n in f.graph.inputs():
            prog.write(n.id, v[n.attrs["name"]])
        prog.run()
        for i, w in zip(keep, want):
            got = prog.read(f.index[i]).reshape(w.shape)
            assert np.allclose(got, w, rtol=1e-5, atol=1e-5)
        a = graph.nodes[y].attrs
        within(prog.read(f.index[y]).reshape(want[0].shape), ref.head(v["x"], v["gain"], v["pos"], a),
               ref.head_bounds(v["x"], v["gain"], v["pos"], a, None)["y"], "y")
    finally:
        prog.free()
        for b in bufs:
            b.free()


# ---------------------------------------------------------------- Newton-Schulz
def orth_case(pkg, shape, **kw):
    g = pkg.ir.Graph()
    return g, g.orthogonalize(g.input("x", shape), **kw)


def check_orth(mods, runner, pkg, x, **kw):
    g, y = orth_case(pkg, list(x.shape), **kw)
    got = run_graph(mods, runner, g, {"x": x}, [y])[0].astype(np.float64)
    a = g.nodes[y].attrs
    want = ref.newton_schulz(x, a["steps"], a["coeffs"], a["eps"])
    flat = lambda v: v.reshape(-1, *v.shape[-2:])  # noqa: E731
    for k, (p, q, r) in enumerate(zip(flat(got), flat(want), flat(x))):
        bound = ref.newton_schulz_bound(r, a["steps"], a["coeffs"], a["eps"])
        assert np.linalg.norm(p - q) <= bound, (k, np.linalg.norm(p - q) / bound)
    return got


@pytest.mark.parametrize("shape", [(1, 1), (3, 64, 50), (64, 512), (500, 63), (17, 511), (1, 300), (128, 128), (2, 127, 65), (66, 128),
                                   (40, 130), (64, 257), (256, 64)])
def test_orthogonalize_both_forms(pkg, mods, runner, monkeypatch, shape):
    """What fits one SM, and the same by the launches of larger matrices."""
    to = importlib.import_module(P + ".training_ops")
    x = f32(np.random.default_rng(shape[-1]).standard_normal(shape))
    assert to.orth_small(min(shape[-2:]), max(shape[-2:])) if len(shape) > 1 else True
    a = check_orth(mods, runner, pkg, x)
    monkeypatch.setattr(to, "orth_small", lambda s, long: None)
    b = check_orth(mods, runner, pkg, x)
    assert np.allclose(a, b, atol=1e-3)


@pytest.mark.parametrize("shape", [(1, 1), (2, 3), (16, 16), (64, 64), (65, 64), (64, 65), (100, 70), (3, 70, 300),
                                   (2, 2, 129, 128), (128, 257), (257, 130), (256, 1024), (700, 512), (5, 1000), (1000, 5)])
def test_orthogonalize(pkg, mods, runner, shape):
    check_orth(mods, runner, pkg, f32(np.random.default_rng(shape[-1]).standard_normal(shape)))


@pytest.mark.parametrize("steps,coeffs", [(1, (1.5, -0.5, 0.0)), (8, (1.5, -0.5, 0.0)), (2, (3.4445, -4.7750, 2.0315)),
                                          (3, (1.875, -1.25, 0.375))])
def test_orthogonalize_coefficients(pkg, mods, runner, steps, coeffs):
    check_orth(mods, runner, pkg, f32(np.random.default_rng(1).standard_normal((80, 50))), steps=steps, coeffs=coeffs)


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1e18, 1e35])
def test_orthogonalize_magnitudes(pkg, mods, runner, scale):
    """The norm is taken in double: no square of a float32 overflows or vanishes."""
    check_orth(mods, runner, pkg, f32(np.random.default_rng(2).standard_normal((60, 90)) * scale), eps=0.0)


def test_orthogonalize_degenerate(pkg, mods, runner):
    """Zero matrices stay zero; rank one and a repeated row are as the formula has them."""
    assert not check_orth(mods, runner, pkg, np.zeros((2, 40, 30))).any()
    rng = np.random.default_rng(3)
    check_orth(mods, runner, pkg, f32(np.outer(rng.standard_normal(50), rng.standard_normal(70))))
    x = f32(rng.standard_normal((40, 40)))
    x[20:] = x[:20]
    check_orth(mods, runner, pkg, x)


def test_orthogonalize_stack_members_do_not_meet(pkg, mods, runner):
    """Each matrix of a stack gets what it gets alone, bit for bit, a NaN in one leaves the others."""
    x = f32(np.random.default_rng(4).standard_normal((3, 130, 70)))
    alone = [check_orth(mods, runner, pkg, m) for m in x]
    x[1, 5, 5] = np.nan
    g, y = orth_case(pkg, [3, 130, 70])
    got = run_graph(mods, runner, g, {"x": x}, [y])[0]
    assert np.array_equal(got[0], alone[0]) and np.array_equal(got[2], alone[2]) and np.isnan(got[1]).all()


def nll_loss_case(pkg, R, d, V, bias=True, seed=0):
    g = pkg.ir.Graph()
    y = g.linear_nll(g.input("h", [R, d]), g.input("w", [d, V]), g.input("b", [V]) if bias else None, g.input("t", [R]))
    rng = np.random.default_rng(seed)
    x = {"h": f32(rng.standard_normal((R, d))), "w": f32(rng.standard_normal((d, V)) * 2 / np.sqrt(d)),
         "t": rng.integers(0, V, R).astype(np.float64)}
    if bias:
        x["b"] = f32(rng.standard_normal(V) * 0.1)
    return g, y, x


def few_rows_bound(h, w, b, t):
    """A few rows' loss on the CUDA cores: a term passes through at most d / 8 fused steps of a warp (an eighth and
    one more of each 256 indices), 8 + 8 sums of warps and parts, one more of the bias, each off by half a step of
    the sums so far.  Sums of exponentials: 4 terms of each of V / 4096 steps, 40 joins of two roundings,
    exponentials of 2 steps."""
    loss, _, ok = ref.nll(h, w, b, t)
    (R, d), V = h.shape, w.shape[1]
    z = np.abs(np.where(ok[:, None], h, 0.0)) @ np.abs(w) + (0.0 if b is None else np.abs(b))
    top = (d / 8 + d / 256 + 20) * ref.U * z.max(1)
    return loss, 2 * top + ref.U * (4 * (V / 4096 + 1) + 2 * (V / 4096 + 40) + 8) + 6 * ref.U * (np.abs(loss) + z.max(1))


@pytest.mark.parametrize("R,d,V", [(1, 1, 1), (1, 64, 5000), (3, 70, 7), (4, 513, 4096), (5, 1000, 129), (8, 33, 128), (16, 257, 10001),
                                   (15, 16, 3), (16, 2048, 1000), (7, 300, 5003), (17, 300, 5003), (33, 300, 5003)])
@pytest.mark.parametrize("bias", [True, False])
def test_nll_loss_of_a_few_rows(pkg, mods, runner, R, d, V, bias):
    g, y, x = nll_loss_case(pkg, R, d, V, bias, seed=R)
    a = (x["h"], x["w"], x.get("b"), x["t"])
    loss, bound = few_rows_bound(*a)
    if R > 16:   # more than the CUDA cores' form takes
        bound = ref.nll_bounds(*a, np.zeros(R))[0]
    within(run_graph(mods, runner, g, x, [y], runs=2)[0], loss, bound, "loss")


def test_nll_loss_of_a_few_rows_masks(pkg, mods, runner):
    """Padding rows with NaN in h, classes out of the vocabulary, a target among them."""
    case = nll_loss_case(pkg, 6, 40, 700)
    x = case[2]
    x["b"][100:600], x["b"][650:] = -np.inf, -3.4028234663852886e38
    x["t"][:] = [3, -1, 99, 700, 620, 200]
    x["h"][1] = np.nan
    got = run_graph(mods, runner, case[0], x, [case[1]])[0]
    assert got[1] == 0 and got[3] == 0 and got[5] == np.inf
    live = np.r_[0:100, 600:650]
    keep = np.array([0, 2, 4])
    within(got[keep], *few_rows_bound(x["h"][keep], x["w"][:, live], x["b"][live], np.array([3.0, 99.0, 120.0])), "loss")


def test_nll_loss_of_a_few_rows_unaligned_weight(pkg, mods, runner):
    """W where the caller has it, 4 bytes past a 128-bit boundary: the scalar loads."""
    rt, cg = mods
    g, y, x = nll_loss_case(pkg, 5, 65, 260)
    ids = {n.attrs["name"]: n.id for n in g.inputs()}
    buf = rt.DeviceBuffer(runner, 4 * 65 * 260 + 16)
    prog = rt.Program(runner, g, cg.lower_fused(g, keep=[y]), keep=[y], place={ids["w"]: buf.ptr + 4})
    try:
        for name, i in ids.items():
            prog.write(i, x[name])
        prog.run()
        got = prog.read(y).ravel()
    finally:
        prog.free()
        buf.free()
    within(got, *few_rows_bound(x["h"], x["w"], x["b"], x["t"]), "loss")


@pytest.mark.parametrize("divide", [False, True])
@pytest.mark.parametrize("bn,ctas", [(64, 1), (128, 1), (128, 2), (256, 2)])
def test_every_tile_whole_and_divided(pkg, mods, runner, monkeypatch, bn, ctas, divide):
    """The products by each tile alone, their tiles whole or divided along K, at sizes with ragged edges."""
    to = importlib.import_module(P + ".training_ops")
    monkeypatch.setattr(to, "F16_COST", {to.Tile(bn, ctas): (100, 1000, 0, 0) if divide else (100, 1000, 10 ** 9, 0)})
    for R, d, V in ((150, 140, 257), (300, 200, 700), (900, 513, 1300)):
        check_nll(mods, runner, nll_case(pkg, R, d, V, seed=R), runs=2)
    for shape in ((140, 150), (390, 130), (2, 257, 600), (2, 300, 520)):
        x = np.random.default_rng(shape[-1]).standard_normal(shape).astype(np.float32).astype(np.float64)
        check_orth(mods, runner, pkg, x)


# ---------------------------------------------------------------- through the runner
def test_runner_reads_every_node_with_canaries(pkg, mods, runner):
    """GpuRunner.run: a buffer per node, canaries behind each; several gradients of one launch among them."""
    rt, cg = mods
    graph, y, grads, x = nll_case(pkg, 150, 30, 200)
    out = runner.run(graph, cg.lower(graph, matmul="tiled"), x, canary=True)
    assert all(out["canaryIntact"])
    want = ref.nll_grad(x["h"], x["w"], x["b"], x["t"], x["d0"])
    _, eg = ref.nll_bounds(x["h"], x["w"], x["b"], x["t"], x["d0"])
    for k, i in grads.items():
        within(out["values"][i].reshape(graph.shape(i)), want[k], eg[k], k)
    graph, y, grads, v = head_case(pkg, 2, 21, 3, 20, 20)
    out = runner.run(graph, cg.lower(graph), v, canary=True)
    assert all(out["canaryIntact"])
    graph, y = orth_case(pkg, [2, 70, 33])
    out = runner.run(graph, cg.lower(graph), {"x": np.ones((2, 70, 33))}, canary=True)
    assert all(out["canaryIntact"])


def small_graphs(pkg):
    graph, y, grads, x = nll_case(pkg, 150, 30, 200)
    yield graph, [y, *grads.values()], x
    graph, y, grads, x = nll_case(pkg, 700, 260, 3000, bias=False)
    yield graph, [y, *grads.values()], x
    graph, y, grads, x = nll_case(pkg, 1500, 520, 2600)   # tiles of pairs of SMs
    yield graph, [y, *grads.values()], x
    graph, y, x = nll_loss_case(pkg, 6, 300, 5000)
    yield graph, [y], x
    graph, y, grads, x = head_case(pkg, 2, 21, 3, 20, 20, True)
    yield graph, [y, *grads.values()], x
    for shape in ([2, 70, 33], [3, 200, 300], [520, 4000]):
        graph, y = orth_case(pkg, shape)
        yield graph, [y], {"x": f32(np.random.default_rng(1).standard_normal(shape))}


def test_c_abi_runs_them_bit_for_bit(pkg, mods, runner):
    """tc_lower_json -> tc_lowered_run and tc_program_*: the Python host's values."""
    import ctypes
    import json
    rt, cg = mods
    lib = rt.lib()
    for graph, keep, x in small_graphs(pkg):
        want = run_graph(mods, runner, graph, x, keep)
        low = ctypes.c_void_p()
        rt.check(lib.tc_lower_json(json.dumps(graph.to_json()).encode(), b'{"matmul": "tiled"}', ctypes.byref(low)))
        N = len(graph.nodes)
        ins, outs = (ctypes.c_void_p * N)(), (ctypes.c_void_p * N)()
        held, got, intact = [], {}, (ctypes.c_int * N)()
        for n in graph.nodes:
            if n.op == "input":
                held.append(np.ascontiguousarray(np.asarray(x[n.attrs["name"]], np.float32)))
                ins[n.id] = held[-1].ctypes.data
        for i in keep:
            got[i] = np.zeros(graph.shape(i), np.float32)
            outs[i] = got[i].ctypes.data
        rt.check(lib.tc_lowered_run(runner.ctx, low, ins, outs, 1, intact))
        assert all(intact)
        k = (ctypes.c_int32 * len(keep))(*keep)
        prog = ctypes.c_void_p()
        rt.check(lib.tc_program_create(runner.ctx, low, k, len(keep), None, 0, 1, ctypes.byref(prog)))
        for n in graph.nodes:
            if n.op == "input":
                a = np.ascontiguousarray(np.asarray(x[n.attrs["name"]], np.float32).reshape(-1))
                rt.check(lib.tc_program_write(prog, n.id, a.ctypes.data, a.size))
        for _ in range(2):
            rt.check(lib.tc_program_run(prog))
        rt.check(lib.tc_program_check(prog))
        for i, w in zip(keep, want):
            assert np.array_equal(got[i], w), graph.nodes[i].op
            a = np.zeros(w.size, np.float32)
            rt.check(lib.tc_program_read(prog, i, a.ctypes.data, a.size))
            assert np.array_equal(a.reshape(w.shape), w), graph.nodes[i].op
        rt.check(lib.tc_program_free(prog))
        rt.check(lib.tc_lowered_free(low))


def test_programs_on_two_streams_at_once(pkg, mods, runner):
    """Captured programs share no workspace: run side by side, again and again, each gives its own values."""
    import ctypes
    rt, cg = mods
    lib = rt.lib()
    cases = [c for c in small_graphs(pkg)]
    want = [run_graph(mods, runner, g, x, keep) for g, keep, x in cases]
    progs, streams = [], []
    try:
        for g, keep, x in cases:
            p = rt.Program(runner, g, cg.lower_fused(g, matmul="tiled", keep=keep), keep=keep, capture=True)
            for n in g.inputs():
                p.write(n.id, x[n.attrs["name"]])
            progs.append(p)
            s = ctypes.c_uint64()
            rt.check(lib.tc_stream_create(runner.ctx, ctypes.byref(s)))
            streams.append(s.value)
        for _ in range(20):
            for p, s in zip(progs, streams):
                rt.check(lib.tc_plan_run_on(p.plan, s))
        ev = rt.Events(runner, len(progs))
        for k, s in enumerate(streams):
            rt.check(lib.tc_event_record_on(runner.ctx, ev.ev[k], s))
            rt.check(lib.tc_event_sync(ev.ev[k], 20000))
        ev.free()
        for p, (g, keep, x), w in zip(progs, cases, want):
            p.check_errors()
            for i, v in zip(keep, w):
                assert np.array_equal(p.read(i).reshape(v.shape), v)
    finally:
        for p in progs:
            p.free()
        for s in streams:
            rt.check(lib.tc_stream_destroy(runner.ctx, s))
