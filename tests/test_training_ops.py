"""The training operators without a GPU: shapes and refusals, gradients against differences, launches."""
import importlib
import itertools

import numpy as np
import pytest

import training_ref as ref


@pytest.fixture(scope="module")
def mods(pkg):
    P = "tensor-compiler-webgpu_b200"
    return pkg, importlib.import_module(P + ".codegen"), importlib.import_module(P + ".training_ops"), \
        importlib.import_module(P + ".runtime")


def nll_graph(pkg, R, d, V, bias=True):
    g = pkg.ir.Graph()
    h, w = g.input("h", [R, d]), g.input("w", [d, V])
    b = g.input("b", [V]) if bias else None
    return g, h, w, b, g.linear_nll(h, w, b, g.input("t", [R]))


def head_graph(pkg, B, T, H, D, shared=True, **kw):
    g = pkg.ir.Graph()
    x, gain = g.input("x", [B, T, H, D]), g.input("gain", [D])
    return g, x, gain, g.head_norm_rope(x, gain, g.input("pos", [T] if shared else [B, T]), **kw)


def test_shapes(pkg):
    g, *_, y = nll_graph(pkg, 5, 3, 7)
    assert g.shape(y) == [5]
    g, *_, y = head_graph(pkg, 2, 5, 3, 8)
    assert g.shape(y) == [2, 3, 5, 8]
    g, *_, y = head_graph(pkg, 2, 5, 3, 8, heads_first=False)
    assert g.shape(y) == [2, 5, 3, 8]
    g = pkg.ir.Graph()
    assert g.shape(g.orthogonalize(g.input("x", [3, 4, 5, 6]))) == [3, 4, 5, 6]


@pytest.mark.parametrize("h,w,b,t", [([5, 3], [4, 7], [7], [5]), ([5, 3], [3, 7], [6], [5]), ([5, 3], [3, 7], [7], [4]),
                                     ([5, 3], [3, 7], [7], [5, 1]), ([2, 5, 3], [3, 7], [7], [5]),
                                     ([5, 3], [3, (1 << 24) + 1], None, [5])])
def test_nll_refusals(pkg, h, w, b, t):
    g = pkg.ir.Graph()
    ids = [g.input(k, s) if s else None for k, s in zip("hwbt", (h, w, b, t))]
    with pytest.raises(pkg.ir.ShapeError):
        g.linear_nll(*ids)


@pytest.mark.parametrize("kw", [{"rotary": 3}, {"rotary": 10}, {"rotary": -2}, {"rotary": 4.0}, {"eps": -1.0},
                                {"eps": float("nan")}, {"eps": 1e39}, {"base": 0.0}, {"base": float("inf")},
                                {"interleaved": 1}, {"heads_first": None}])
def test_head_refusals(pkg, kw):
    with pytest.raises(pkg.ir.ShapeError):
        head_graph(pkg, 2, 5, 3, 8, **kw)


@pytest.mark.parametrize("x,gain,pos", [([2, 5, 24], [8], [5]), ([2, 5, 3, 8], [9], [5]), ([2, 5, 3, 8], [8], [4]),
                                        ([2, 5, 3, 8], [8], [5, 2]), ([1, 1, 1, 514], [514], [1])])
def test_head_shape_refusals(pkg, x, gain, pos):
    g = pkg.ir.Graph()
    with pytest.raises(pkg.ir.ShapeError):
        g.head_norm_rope(g.input("x", x), g.input("g", gain), g.input("p", pos))


@pytest.mark.parametrize("shape,kw", [([4], {}), ([65536, 2, 2], {}), ([4, 4], {"steps": 0}), ([4, 4], {"steps": 33}),
                                      ([4, 4], {"coeffs": (1.0, 2.0)}), ([4, 4], {"coeffs": (1.0, float("inf"), 0.0)}),
                                      ([4, 4], {"coeffs": (400.0, 0.0, 0.0)}), ([4, 4], {"eps": -1e-9}),
                                      ([4, 4], {"coeffs": (3.0, 3.0, 3.0), "steps": 9})])
def test_orthogonalize_refusals(pkg, shape, kw):
    g = pkg.ir.Graph()
    with pytest.raises(pkg.ir.ShapeError):
        g.orthogonalize(g.input("x", shape), **kw)


def test_raw_emit_is_checked(pkg):
    """Graphs may come from JSON: the attributes are checked there too."""
    g, h, w, b, y = nll_graph(pkg, 5, 3, 7)
    js = g.to_json()
    assert pkg.ir.Graph.from_json(js).nodes[y].shape == [5]
    for attrs in ({"bias": False, "out": "loss"}, {"bias": True}, {"bias": True, "out": "logits"}, {"out": "loss"}):
        js["nodes"][y]["attrs"] = attrs
        with pytest.raises(pkg.ir.ShapeError):
            pkg.ir.Graph.from_json(js)
    t, gy = g.input_id("t"), g.input("gy", [5])
    saved = g.emit("linearNll", [h, w, b, t], {"bias": True, "out": "saved"})
    ok = {"bias": True, "d": 3, "V": 7, "wrt": "h"}
    assert g.shape(g.emit("linearNllGrad", [t, saved, gy], ok)) == [5, 3]
    for bad in ({"wrt": "t"}, {"wrt": None}, {"d": 40}, {"V": 800}, {"V": 0}, {"d": 3.0}, {"bias": False, "wrt": "b"}):
        with pytest.raises(pkg.ir.ShapeError):
            g.emit("linearNllGrad", [t, saved, gy], {**ok, **bad})
    with pytest.raises(pkg.ir.ShapeError):
        g.emit("linearNllGrad", [t, gy, saved], ok)
    with pytest.raises(pkg.autodiff.GradientError):
        pkg.autodiff.grad(g, [saved], [h])


def test_orthogonalize_has_no_gradient(pkg):
    g = pkg.ir.Graph()
    x = g.input("x", [4, 4])
    with pytest.raises(pkg.autodiff.GradientError):
        pkg.autodiff.grad(g, [g.orthogonalize(x)], [x])


def test_scales_hold_every_step(pkg):
    """The largest entries of X, S and P stay within fp16 under their scales, whatever the spectrum."""
    rng = np.random.default_rng(0)
    for steps, co in ((5, pkg.ir.NEWTON_SCHULZ), (1, (1.5, -0.5, 0.0)), (12, (1.5, -0.5, 0.0)), (3, (2.0, 0.0, 0.0)),
                      (4, (1.875, -1.25, 0.375))):
        ex, es, ep = pkg.ir.newton_schulz_scales(steps, co)
        for trial in range(20):
            s = rng.random(40) ** rng.integers(1, 6)
            s = s / np.linalg.norm(s) if trial else np.eye(1, 40)[0]
            for _ in range(steps):
                p = co[1] * s ** 2 + co[2] * s ** 4
                for v, k in ((s, ex), (s * s, es), (p, ep)):
                    assert np.abs(v).max() * 2.0 ** k < 65504
                s = np.abs(co[0] * s + co[1] * s ** 3 + co[2] * s ** 5)


# ---------------------------------------------------------------- gradients against differences
def _differences(graph, node, inputs, name, cot, eps=1e-5):
    base = np.asarray(inputs[name], np.float64)
    out = np.zeros(base.size)
    for k in range(base.size):
        vals = []
        for s in (eps, -eps):
            x = base.copy().reshape(-1)
            x[k] += s
            vals.append((ref.evaluate(graph, {**inputs, name: x})[node] * cot).sum())
        out[k] = (vals[0] - vals[1]) / (2 * eps)
    return out


def _check_gradients(pkg, g, out, wrt, inputs, seed):
    cot = np.random.default_rng(seed).standard_normal(g.shape(out))
    G = pkg.autodiff.grad(g, [out], list(wrt.values()))
    vals = ref.evaluate(G.graph, {**inputs, G.cotangents[0]: cot})
    for (name, _), i in zip(wrt.items(), G.grads):
        # central differences in 64 bits: eps^2 of third derivatives of order 1 and 2^-53 / eps of rounding
        assert np.allclose(vals[i].reshape(-1), _differences(g, out, inputs, name, cot), rtol=1e-6, atol=1e-7), name


@pytest.mark.parametrize("bias", [True, False])
def test_nll_gradient(pkg, bias):
    g, h, w, b, y = nll_graph(pkg, 5, 3, 4, bias)
    rng = np.random.default_rng(1)
    inputs = {"h": rng.standard_normal((5, 3)), "w": rng.standard_normal((3, 4)), "b": rng.standard_normal(4),
              "t": np.array([0, 3, -1, 2, 4])}
    _check_gradients(pkg, g, y, {"h": h, "w": w, **({"b": b} if bias else {})}, inputs, 2)


@pytest.mark.parametrize("shared,inter,rot,first", [(True, False, 6, True), (False, True, 4, False), (True, False, 0, True)])
def test_head_gradient(pkg, shared, inter, rot, first):
    g, x, gain, y = head_graph(pkg, 2, 3, 2, 6, shared, rotary=rot, interleaved=inter, heads_first=first)
    rng = np.random.default_rng(3)
    inputs = {"x": rng.standard_normal((2, 3, 2, 6)), "gain": rng.standard_normal(6),
              "pos": rng.integers(0, 50, (3,) if shared else (2, 3))}
    _check_gradients(pkg, g, y, {"x": x, "gain": gain}, inputs, 4)


def test_shared_gain_gradients_add_up(pkg):
    """One gain for queries and keys: its gradients of both nodes are added."""
    g = pkg.ir.Graph()
    gain, pos = g.input("gain", [4]), g.input("pos", [3])
    q, k = (g.head_norm_rope(g.input(n, [1, 3, 2, 4]), gain, pos) for n in "qk")
    y = g.matmul(q, g.transpose_last2(k))
    rng = np.random.default_rng(5)
    inputs = {"q": rng.standard_normal((1, 3, 2, 4)), "k": rng.standard_normal((1, 3, 2, 4)),
              "gain": rng.standard_normal(4), "pos": np.arange(3)}
    _check_gradients(pkg, g, y, {"gain": gain, "q": g.input_id("q")}, inputs, 6)


def test_orthogonalize_reference_is_orthogonal():
    """The formula itself: singular values come near 1, the singular vectors stay."""
    x = np.random.default_rng(7).standard_normal((12, 30))
    o = ref.newton_schulz(x, 5, (3.4445, -4.7750, 2.0315), 1e-7)
    s = np.linalg.svd(o, compute_uv=False)
    assert 0.6 < s.min() and s.max() < 1.25
    u, _, v = np.linalg.svd(x, full_matrices=False)
    d = u.T @ o @ v.T
    assert np.allclose(d, np.diag(np.diag(d)), atol=1e-10)


# ---------------------------------------------------------------- launches
def _grads(pkg, g, out, wrt):
    G = pkg.autodiff.grad(g, [out], wrt)
    return G.graph, G.grads


def test_gradients_of_a_node_are_one_launch(mods):
    pkg, cg, to, rt = mods
    g, h, w, b, y = nll_graph(pkg, 300, 64, 1000)
    G, grads = _grads(pkg, g, y, [h, w, b])
    lau = [l for l in cg.lower_fused(G)["launches"] if l.kind == "linear-nll-grad"]
    assert len(lau) == 1 and sorted(lau[0].nodes) == sorted(grads)
    # only what is asked for: no weight gradient, no product for it
    G, grads = _grads(pkg, g, y, [h])
    lau = [l for l in cg.lower(G)["launches"] if l.kind == "linear-nll-grad"]
    assert len(lau) == 1 and [c.name.rsplit("_", 1)[0] for c in lau[0].calls if c.tma] == ["tcb_nll_dz", "tcb_nll_dh"]
    assert not hasattr(lau[0], "nodes")
    # the loss and what it saves are one launch too; without a backward nothing is saved
    (fwd,) = [l for l in cg.lower(G)["launches"] if l.kind == "linear-nll"]
    assert fwd.nodes[0] == y and len(fwd.nodes) == 2
    (fwd,) = cg.lower(g)["launches"]
    assert not hasattr(fwd, "nodes")


def test_equal_nodes_are_launches_of_their_own(mods):
    """The same loss emitted twice: either is computed, neither is taken for the other's sibling."""
    pkg, cg, to, rt = mods
    g, h, w, b, y = nll_graph(pkg, 30, 8, 10)
    y2 = g.linear_nll(h, w, b, g.input_id("t"))
    assert [l.node for l in cg.lower(g)["launches"]] == [y, y2]
    G, grads = _grads(pkg, g, g.add(y, y2), [h])
    made = [i for l in cg.lower_fused(G)["launches"] for i in (getattr(l, "nodes", None) or [l.node])]
    assert len(made) == len(set(made)) and {n.id for n in G.nodes if n.op in pkg.ir.TRAINING_OPS} <= set(made)


def test_two_nodes_keep_their_gradients_apart(mods):
    pkg, cg, to, rt = mods
    g, h, w, b, y = nll_graph(pkg, 300, 64, 1000)
    y2 = g.linear_nll(h, w, b, g.input("t2", [300]))
    G, _ = _grads(pkg, g, g.add(y, y2), [h, w, b])
    assert len([l for l in cg.lower_fused(G)["launches"] if l.kind == "linear-nll-grad"]) == 2


@pytest.mark.parametrize("R,d,V", [(1, 1, 1), (64, 64, 65), (4095, 256, 8192), (8192, 1024, 50001), (16384, 17, 131072),
                                   (3, 2048, 1 << 24), (1 << 20, 64, 65)])
def test_nll_maps_stay_inside(mods, R, d, V):
    """Every tensor map starts on 16 bytes and ends inside its region; a piece of dz is bounded."""
    pkg, cg, to, rt = mods
    g, h, w, b, y = nll_graph(pkg, R, d, V)
    inner, floats = pkg.ir.linear_nll_saved(R, d, V)
    def blocked(n):
        return -(-n // 256) * min(256, to._up(n, 32))
    parts = sorted([(0, 12), (256, 4 * to._up(V, 256)), (inner["lse"], 4 * R), (inner["h"], 4 * R * blocked(d)),
                    (inner["w"], 4 * d * blocked(V))])
    assert all(o + n <= o2 for (o, n), (o2, _) in itertools.pairwise(parts)) and sum(parts[-1]) <= 4 * floats
    piece, pieces = to.nll_pieces(R, V)
    assert piece * pieces >= V > piece * (pieces - 1) and (pieces == 1 or piece % 256 == 0)
    assert 4 * R * piece <= max(to.DZ_BYTES, 4 * R * 256)
    G, _ = _grads(pkg, g, y, [h, w, b])
    for graph in (g, G):
        for lau in cg.lower_fused(graph)["launches"]:
            sizes = {"scratch": lau.scratch_bytes, "out": 4 * floats, "in_at": 4 * floats}
            for c in lau.calls:
                for region, off, cols, rows, batch, rs, bs, bc, br in c.tma or []:
                    if region == "in_at":
                        assert off & 7 == 1
                        off >>= 3
                    end = off + (batch - 1) * bs + (rows - 1) * rs + 2 * cols
                    assert off % 16 == 0 and rs % 16 == 0 and bs % 16 == 0 and end <= sizes[region] and 2 * cols <= rs


@pytest.mark.parametrize("M,N,K,batch,chunk,sym", [(64, 50, 16384, 1, 256, False), (1, 1, 1, 1, 256, False), (57, 1365, 55301, 1, 256, False),
                                                   (256, 256, 1024, 4, 128, True), (1000, 1000, 4095, 1, 128, True),
                                                   (4095, 256, 8192, 1, 256, False), (8192, 1024, 4096, 1, 256, False),
                                                   (1024, 512, 32000, 1, 256, False), (1300, 1300, 9000, 1, 128, True),
                                                   (18, 18, 3593, 14, 128, True), (300, 4099, 700, 1, 128, False),
                                                   (128, 2048, 12345, 1, 128, False)])
def test_division_of_a_product(mods, M, N, K, batch, chunk, sym):
    """The device's division of tiles among CTAs, restated: every chunk of every tile once, the pieces of a
    divided tile found by the warp that adds them, no two in one slot."""
    pkg, cg, to, rt = mods
    tile, ctas, whole, q = to.f16_plan(M, N, K, batch, chunk, sym)
    assert ctas % tile.ctas == 0 and 1 <= ctas <= 148 and M > 128 * (tile.ctas - 1)
    tiles, grid = batch * to.f16_tiles(M, N, tile, sym), ctas // tile.ctas   # pairs work as one
    chunks = -(-K // chunk)
    per = -(-chunks // q)
    total = (tiles - whole) * per
    assert (total == 0 or grid <= total) and (tiles - whole) * tile.ctas <= 148 and (tile.bn == 64 or N > tile.bn // 2)
    seen, slots = {}, {}
    for c in range(grid):
        for t in range(c, whole, grid):
            seen.setdefault(t, []).append((0, chunks, c))
        at, end = c * total // grid, (c + 1) * total // grid
        while at < end:
            t, k = divmod(at, per)
            n = min(end - at, per - k)
            piece = (k * q, min((k + n) * q, chunks), c)
            seen.setdefault(whole + t, []).append(piece)
            if piece[:2] != (0, chunks):
                slot = 2 * c + (k == 0)
                assert slot not in slots
                slots[slot] = (whole + t, piece)
            at += n
    assert sorted(seen) == list(range(tiles))
    for t, pieces in seen.items():
        pieces.sort()
        assert pieces[0][0] == 0 and pieces[-1][1] == chunks and all(a[1] == b[0] for a, b in itertools.pairwise(pieces))
        if len(pieces) > 1:
            first = (t - whole) * per
            ca, cb = (((x + 1) * grid - 1) // total for x in (first, first + per - 1))
            assert [p[2] for p in pieces] == list(range(ca, cb + 1))
            assert [slots[2 * c + (c == ca)][1] for c in range(ca, cb + 1)] == pieces
    assert to.f16_partial_bytes(ctas, whole, tiles, tile) >= (max(slots) + 1 if slots else 0) * 128 * tile.ctas * tile.bn * 4


@pytest.mark.parametrize("shape", [[1, 1], [64, 64], [100, 70], [3, 70, 300], [4095, 1000], [2, 2, 256, 1024]])
def test_orthogonalize_scratch(mods, shape):
    pkg, cg, to, rt = mods
    g = pkg.ir.Graph()
    g.orthogonalize(g.input("x", shape))
    (lau,) = cg.lower(g)["launches"]
    if to.orth_small(min(shape[-2:]), max(shape[-2:])):
        assert len(lau.calls) == 1 and lau.calls[0].smem <= 227 * 1024 and lau.calls[0].err_offset is not None
        return
    assert len(lau.calls) == 2 + 15
    for c in lau.calls:
        for region, off, cols, rows, batch, rs, bs, bc, br in c.tma or []:
            end = off + (batch - 1) * bs + (rows - 1) * rs + 2 * cols
            assert region == "scratch" and off % 16 == 0 and rs % 16 == 0 and bs % 16 == 0 and end <= lau.scratch_bytes
        if c.tma:
            assert c.err_offset is not None and c.smem <= 227 * 1024


@pytest.mark.parametrize("B,T,H,D,rot", [(1, 1, 4, 64, 64), (3, 1001, 5, 80, 40), (512, 256, 4, 64, 64), (2, 8191, 32, 128, 128),
                                         (1, 1, 1, 1, 0), (2, 3, 1, 7, 6), (1, 5, 3, 512, 512), (9, 1, 33, 33, 2)])
def test_head_launch_geometry(mods, B, T, H, D, rot):
    pkg, cg, to, rt = mods
    g, x, gain, y = head_graph(pkg, B, T, H, D, rotary=rot)
    G, _ = _grads(pkg, g, y, [x, gain])
    for lau in cg.lower_fused(G)["launches"]:
        main = lau.calls[0]
        heads = main.params[4]
        assert 1 <= main.grid[0] <= 148 * 4 and main.grid[0] <= B * T * H
        for v in ((4, 1) if rot % 8 == 0 and D % 4 == 0 else (1,)):
            lanes, rows = to._head_rows(D, rot, v)
            assert lanes <= 32 and 256 % lanes == 0 and main.smem <= 48 * 1024
            assert main.smem in (0,) or main.smem >= 4 * D * rows
        assert heads & (heads - 1) == 0
        if lau.kind == "head-norm-rope-grad":
            assert lau.scratch_bytes == main.grid[0] * D * 4


@pytest.mark.parametrize("which", ["nll", "nll-bias", "orth", "orth-64", "orth-128", "head-64", "head-odd", "head-none"])
def test_sources_compile(mods, which):
    pkg, cg, to, rt = mods
    code = {"nll": lambda: to.nll_source(False), "nll-bias": lambda: to.nll_source(True),
            "orth": lambda: to.orth_source(5, pkg.ir.NEWTON_SCHULZ, 1e-7),
            "orth-64": lambda: to.orth_source(5, pkg.ir.NEWTON_SCHULZ, 1e-7, (64, 512)),
            "orth-128": lambda: to.orth_source(5, pkg.ir.NEWTON_SCHULZ, 1e-7, (128, 128)), "head-64": lambda: to.head_source(64, 64, False),
            "head-odd": lambda: to.head_source(33, 6, True), "head-none": lambda: to.head_source(7, 0, False)}[which]()
    assert rt.compile_check(code) > 0


# ---------------------------------------------------------------- the library's own lowering
def _graphs(pkg):
    for R, d, V, bias, wrt in ((1, 1, 1, True, "hwb"), (64, 64, 65, True, "hwb"), (300, 64, 1000, False, "hw"), (2500, 8, 2500, True, "wb"),
                               (4095, 256, 8192, True, "hwb"), (8192, 1024, 50001, True, "hwb"), (16384, 1024, 131072, True, ""),
                               (57, 1365, 55301, True, "h"), (16384, 39, 50, True, "hwb"), (100, 513, 3, True, "b"),
                               (70000, 64, 600, False, "hw"), (3, 40, 1 << 24, True, "hwb")):
        g, h, w, b, y = nll_graph(pkg, R, d, V, bias)
        ids = [{"h": h, "w": w, "b": b}[k] for k in wrt]
        yield pkg.autodiff.grad(g, [y], ids).graph if wrt else g
    for B, T, H, D, kw in ((1, 1, 4, 64, {}), (3, 1001, 5, 80, {"rotary": 40, "interleaved": True, "shared": False}), (2, 8191, 32, 128, {}),
                           (512, 256, 4, 64, {"heads_first": False}), (1, 5, 3, 7, {"rotary": 6, "base": 500000, "eps": 0}),
                           (2, 3, 1, 512, {"rotary": 0}), (9, 1, 33, 33, {"rotary": 2, "base": 0.5})):
        g, x, gain, y = head_graph(pkg, B, T, H, D, **kw)
        yield g
        for wrt in ([x, gain], [x], [gain]):
            yield pkg.autodiff.grad(g, [y], wrt).graph
    for shape, kw in (([1, 1], {}), ([64, 64], {}), ([3, 128, 128], {}), ([63, 513], {}), ([4, 256, 1024], {}), ([4095, 1000], {}), ([4096, 4096], {}),
                      ([2, 2, 129, 18], {"steps": 8, "coeffs": (1.5, -0.5, 0)}), ([700, 512], {"steps": 1, "coeffs": (1.875, -1.25, 0.375), "eps": 0}),
                      ([14, 3593, 18], {}), ([1, 16384], {})):
        g = pkg.ir.Graph()
        g.orthogonalize(g.input("x", shape), **kw)
        yield g


def test_library_lowers_identically(mods):
    """tc_lower_json makes the Python host's records, field for field."""
    from test_lower_abi import _compare
    pkg, cg, to, rt = mods
    n = 0
    for g in _graphs(pkg):
        n += _compare(rt.lib(), cg, g)
        n += _compare(rt.lib(), cg, g, fused=False)
    assert n > 100
    g, h, w, b, y = nll_graph(pkg, 300, 64, 1000)
    y2 = g.linear_nll(h, w, b, g.input_id("t"))
    assert _compare(rt.lib(), cg, pkg.autodiff.grad(g, [g.add(y, y2)], [h, b]).graph) > 4


def test_library_lowers_the_training_step_identically(mods):
    from test_lower_abi import _compare
    pkg, cg, to, rt = mods
    s = pkg.steps
    cfg = s.make_config(T=40, d=64, H=4, L=2, ff=300, targets="index", rope=10000.0)
    step = s.build_step3b(300, 3, cfg, opt=s.MUON_3B)
    keep = [step["loss"], *step["outputs"].values()]
    f = pkg.fuse.fuse(step["graph"], keep=keep)
    kept = [f.index[i] for i in keep]
    for kw in ({}, {"fold": True, "keep": kept, "colfuse": True, "mofuse": True}):
        assert _compare(rt.lib(), cg, f.graph, matmul="tiled", **kw) > 100


@pytest.mark.parametrize("change", [{"bias": False}, {"out": "logits"}, {"out": None}, {"bias": 1}])
def test_library_refuses_bad_attributes(mods, change):
    import ctypes
    import json
    pkg, cg, to, rt = mods
    g, h, w, b, y = nll_graph(pkg, 5, 3, 7)
    js = g.to_json()
    js["nodes"][y]["attrs"].update(change)
    out = ctypes.c_void_p()
    assert rt.lib().tc_lower_json(json.dumps(js).encode(), b"{}", ctypes.byref(out)) == 1
    assert b"linearNll" in rt.lib().tc_last_error()


@pytest.mark.parametrize("node,shape", [("w", [4, 7]), ("t", [6]), ("b", [8]), ("y", [6]), ("h", [3])])
def test_library_refuses_bad_shapes(mods, node, shape):
    import ctypes
    import json
    pkg, cg, to, rt = mods
    g, h, w, b, y = nll_graph(pkg, 5, 3, 7)
    js = g.to_json()
    for n in js["nodes"]:
        if n["attrs"].get("name") == node or (node == "y" and n["op"] == "linearNll"):
            n["shape"] = shape
    out = ctypes.c_void_p()
    assert rt.lib().tc_lower_json(json.dumps(js).encode(), b"{}", ctypes.byref(out)) == 1


@pytest.mark.parametrize("op,change", [("head", {"rotary": 10}), ("head", {"rotary": 3}), ("head", {"eps": -1}), ("head", {"base": 0}),
                                       ("head", {"headsFirst": 0}), ("head", {"interleaved": None}), ("orth", {"steps": 0}), ("orth", {"steps": 2.5}),
                                       ("orth", {"coeffs": [1, 2]}), ("orth", {"coeffs": [400, 0, 0]}), ("orth", {"eps": -1})])
def test_library_refuses_bad_settings(mods, op, change):
    import ctypes
    import json
    pkg, cg, to, rt = mods
    if op == "head":
        g, _, _, y = head_graph(pkg, 2, 5, 3, 8)
    else:
        g = pkg.ir.Graph()
        y = g.orthogonalize(g.input("x", [4, 4]))
    js = g.to_json()
    js["nodes"][y]["attrs"].update(change)
    out = ctypes.c_void_p()
    assert rt.lib().tc_lower_json(json.dumps(js).encode(), b"{}", ctypes.byref(out)) == 1
