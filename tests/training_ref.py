"""A float64 evaluation of whole graphs in numpy, with the training operators written from their formulas.

The oracle of the training-operator tests: nothing here shares code with the package.  Beside each
operator stands the bound of its float32 kernel's error, by counting roundings (U is half a float32 step).
"""
import math

import numpy as np

U = 2.0 ** -24


# ---------------------------------------------------------------- the operators
def nll(h, w, b, t):
    """(loss [R], probabilities [R, V], valid rows) of a linear head."""
    R, V = h.shape[0], w.shape[1]
    ok = (t >= 0) & (t < V)
    z = np.where(ok[:, None], h, 0.0) @ w + (0.0 if b is None else b)
    m = z.max(1, keepdims=True)
    m = np.where(np.isneginf(m), 0.0, m)
    e = np.exp(z - m)
    s = e.sum(1, keepdims=True)
    idx = np.where(ok, t, 0).astype(np.int64)
    loss = np.where(ok, (np.log(s) + m)[:, 0] - z[np.arange(R), idx], 0.0)
    return loss, e / s, ok


def nll_grad(h, w, b, t, gy):
    _, p, ok = nll(h, w, b, t)
    dz = p.copy()
    rows = np.arange(len(t))[ok]
    dz[rows, t[ok].astype(np.int64)] -= 1.0
    dz = np.where(ok[:, None], dz * gy[:, None], 0.0)
    hh = np.where(ok[:, None], h, 0.0)
    return {"h": dz @ w.T, "w": hh.T @ dz, "b": dz.sum(0)}


def product_bound(K, chunk):
    """A split-fp16 product's error as a multiple of U sum |a| |b|: three roundings of 2^-22 a term (hi + lo of
    either operand, lo.lo dropped), and per chain of `chunk` indices three accumulations every 16, each
    truncated by up to a whole step (2 U) and as much again for the alignment within the instruction; the
    chains are added with one rounding each."""
    return 12 + 3 * (min(K, chunk) / 16 + 1) * 4 + math.ceil(K / chunk) + 4


def nll_bounds(h, w, b, t, gy):
    """Error bounds of the loss and the gradients."""
    R, d = h.shape
    V = w.shape[1]
    loss, p, ok = nll(h, w, b, t)
    hh = np.abs(np.where(ok[:, None], h, 0.0))
    z = hh @ np.abs(w) + (0.0 if b is None else np.abs(b))
    # the operands' absolute floor: 2^-40 of the largest magnitude in place of 2^-22 of the value
    floor = 2.0 ** -39 * d * hh.max(initial=0.0) * np.abs(w).max()
    ez = product_bound(d, 256) * U * z + floor
    top = ez.max(1)
    # the sums of exponentials: 32 in each of 4 chains, then 3 + 8 + tiles of joins of two roundings, expf of 2 steps
    es = U * (32 + 2 * (11 + V / 64) + 8)
    eloss = 2 * top + es + 6 * U * (np.abs(loss) + z.max(1))
    dz = np.abs(p)
    rows = np.arange(R)[ok]
    onehot = np.zeros_like(p)
    onehot[rows, t[ok].astype(np.int64)] = 1.0
    edz = p * (ez + top[:, None] + (es + 8 * U) + eloss[:, None]) + 4 * U * (p + onehot)
    g = np.where(ok, np.abs(gy), 0.0)[:, None]
    edz = g * edz + 2.0 ** -39 * g.max(initial=0.0)
    dz = g * (dz + onehot)
    aw = np.abs(w)
    return eloss, {"h": edz @ aw.T + (product_bound(V, 256) + V / 256) * U * (dz @ aw.T) + 2.0 ** -39 * V * g.max(initial=0.0) * aw.max(),
                   "w": hh.T @ edz + product_bound(R, 256) * U * (hh.T @ dz) + 2.0 ** -39 * R * g.max(initial=0.0) * hh.max(initial=0.0),
                   "b": edz.sum(0) + U * (5 + R / 256 + 8) * dz.sum(0)}


def rotate(x, pos, base, rotary, interleaved, back=False):
    """x [B,T,H,D] turned by pos [T] or [B,T]."""
    k = rotary // 2
    T = x.shape[1]
    ang = pos.reshape(-1, T)[:, :, None, None] * base ** (-np.arange(k) / max(k, 1))
    c, s = np.cos(ang), np.sin(ang) * (-1 if back else 1)
    y = x.copy()
    i = 2 * np.arange(k) if interleaved else np.arange(k)
    j = i + 1 if interleaved else i + k
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    return y


def head(x, gain, pos, a):
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + a["eps"]) * gain
    y = rotate(n, pos, a["base"], a["rotary"], a["interleaved"])
    return y.transpose(0, 2, 1, 3) if a["headsFirst"] else y


def head_grad(x, gain, pos, a, gy):
    gy = gy.transpose(0, 2, 1, 3) if a["headsFirst"] else gy
    u = rotate(gy, pos, a["base"], a["rotary"], a["interleaved"], back=True)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + a["eps"])
    ug = u * gain
    return {"gain": (u * x * r).sum((0, 1, 2)),
            "x": r * (ug - x * r * r * (ug * x).mean(-1, keepdims=True))}


def head_bounds(x, gain, pos, a, gy):
    """r: at most 16 + 5 additions, a division, a root and a sum, 12 U relative with the squares' halves; an
    angle: U of half a turn (pi U) and sincospi's 2 steps; then five products and sums.  40 U of the pair's
    magnitudes covers them.  dx has a second sum; dgain adds up every row."""
    k, i = a["rotary"] // 2, None
    n = np.abs(x) / np.sqrt((x * x).mean(-1, keepdims=True) + a["eps"]) * np.abs(gain)

    def pair(v):
        out = v.copy()
        i = 2 * np.arange(k) if a["interleaved"] else np.arange(k)
        j = i + 1 if a["interleaved"] else i + k
        out[..., i] = out[..., j] = v[..., i] + v[..., j]
        return out
    ey = 40 * U * pair(n)
    out = {"y": ey.transpose(0, 2, 1, 3) if a["headsFirst"] else ey}
    if gy is not None:
        g = np.abs(gy.transpose(0, 2, 1, 3) if a["headsFirst"] else gy)
        u = pair(g)
        r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + a["eps"])
        ax = np.abs(x)
        ug = u * np.abs(gain)
        rows = x.size / x.shape[-1]
        out["x"] = 100 * U * r * (ug + ax * r * r * (ug * ax).mean(-1, keepdims=True))
        out["gain"] = (60 + rows) * U * (u * ax * r).sum((0, 1, 2))
    return out


def newton_schulz(x, steps, coeffs, eps):
    a, b, c = coeffs
    x = x / (np.sqrt((x * x).sum((-2, -1), keepdims=True)) + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.swapaxes(-1, -2) if tall else x
    for _ in range(steps):
        s = x @ x.swapaxes(-1, -2)
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.swapaxes(-1, -2) if tall else x


def newton_schulz_bound(x, steps, coeffs, eps):
    """A bound, to first order, of the Frobenius norm of the error for one matrix.

    Every product is off by up to `kap` of its own norm: 24 accumulations in a chain of 128, each truncated
    by at most a step (2 U) of the running sum, twice for the alignment within, and 2^-22 for the splits.
    An error E of a step's X reaches the result multiplied by the derivative of the later steps.  Each acts
    on the singular values by f(t) = a t + b t^3 + c t^5, so its derivative's norm is the largest of
    |f(s) - f(t)| / |s - t|, |f(s) + f(t)| / (s + t) and |f'(s)| over the singular values s, t."""
    a, b, c = coeffs
    kap = 24 * 4 * U + 2.0 ** -22
    s = np.linalg.svd(x / (np.linalg.norm(x) + eps), compute_uv=False)
    f = lambda t: a * t + b * t ** 3 + c * t ** 5  # noqa: E731
    total = 4 * U * np.linalg.norm(s)
    for _ in range(steps):
        g, t = s * s, f(s)
        fro, two = np.linalg.norm, s.max()
        ds = kap * fro(g)
        dp = (abs(b) + 2 * abs(c) * g.max()) * ds + kap * (abs(b) * fro(g) + abs(c) * fro(g * g))
        dx = dp * two + kap * (fro((b * g + c * g * g) * s) + abs(a) * fro(s))
        d = np.abs(a + 3 * b * g + 5 * c * g * g).max()
        gap, add = np.abs(s[:, None] - s), s[:, None] + s
        lip = max(d, (np.abs(t[:, None] + t) / np.maximum(add, 1e-300)).max(),
                  np.where(gap > 1e-12, np.abs(t[:, None] - t) / np.maximum(gap, 1e-12), 0.0).max())
        if x.shape[0] != x.shape[1]:
            lip = max(lip, np.abs(a + b * g + c * g * g).max())
        total = total * lip + dx
        s = np.abs(t)
    return total


# ---------------------------------------------------------------- whole graphs
def evaluate(graph, inputs):
    """Every node's float64 value."""
    vals = []
    for n in graph.nodes:
        v = [vals[i] for i in n.inputs]
        a = n.attrs
        op = n.op
        if op == "input":
            r = np.asarray(inputs[a["name"]], np.float64).reshape(n.shape)
        elif op == "const":
            r = np.broadcast_to(np.asarray(a["value"], np.float64).reshape(n.shape if not isinstance(a["value"], (int, float)) else ()), n.shape)
        elif op in ("add", "sub", "mul", "div"):
            r = {"add": np.add, "sub": np.subtract, "mul": np.multiply, "div": np.divide}[op](*v)
        elif op in ("exp", "log", "tanh", "sqrt"):
            r = getattr(np, op)(v[0])
        elif op == "neg":
            r = -v[0]
        elif op == "relu":
            r = np.where(v[0] > 0, v[0], 0.0)
        elif op == "step":
            r = (v[0] > 0).astype(np.float64)
        elif op == "stopGradient":
            r = v[0]
        elif op == "matmul":
            r = v[0] @ v[1]
        elif op in ("sum", "max"):
            r = getattr(np, op)(v[0], axis=a["axis"], keepdims=bool(a.get("keepDims")))
        elif op == "broadcast":
            r = np.broadcast_to(v[0], n.shape)
        elif op == "reshape":
            r = v[0].reshape(n.shape)
        elif op == "transpose":
            r = v[0].transpose(a["perm"])
        elif op == "linearNll":
            # (opaque: the oracle's gradients go back to the operands)
            r = np.zeros(n.shape) if a["out"] == "saved" else nll(v[0], v[1], v[2] if a["bias"] else None, v[-1])[0]
        elif op == "linearNllGrad":
            ops = [vals[i] for i in graph.nodes[n.inputs[1]].inputs]
            r = nll_grad(ops[0], ops[1], ops[2] if a["bias"] else None, ops[-1], v[-1])[a["wrt"]]
        elif op == "headNormRope":
            r = head(*v, a)
        elif op == "headNormRopeGrad":
            r = head_grad(*v[:3], a, v[3])[a["wrt"]]
        elif op == "orthogonalize":
            r = newton_schulz(v[0], a["steps"], a["coeffs"], a["eps"])
        else:
            raise ValueError(op)
        vals.append(np.asarray(r, np.float64))
    return vals
